"""What the norm and the expert operators are measured on.

`listed()` holds the fixed cases, `draw()` makes more of the same ranges.  `run()` makes one pass: the framework's calls
where `own` is true, otherwise the same operators in their plain form, elementary torch operations in 32 bits (64 where a
choice between near neighbours hangs on it).  `exact()` computes the definition in 64 bits.

kind             one pass
norm             root-mean-square norm with the residual's addition; the output in the input's type or in 8 bits with scales
norm_train       the same with its backward pass
route            scores, groups, top-k and weights of each token's experts
route_train      the same with its backward pass
dispatch         counting sort of the tokens by expert and the copy of their rows, 8-bit codes and their scales
exchange         counting sort, copy of the rows, and the weighted sum of the experts' outputs
exchange_train   the same with its backward pass and the update of the balance bias
"""

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16,
          "float8_e4m3fn": torch.float8_e4m3fn, "float8_e5m2": torch.float8_e5m2}
LARGEST = {"float8_e4m3fn": 448.0, "float8_e5m2": 57344.0}  # largest finite value of the 8-bit types
SMALLEST_AMAX = 2.0 ** -40  # groups whose largest value is below this take this one's scale
EPS = 1e-6
TINY = 1e-20  # added to the sum that the weights are divided by


def listed():
    return [
        # One new token of a serving model: latency, not bandwidth.
        {"name": "norm_one_token", "kind": "norm", "rows": 1, "cols": 4096, "dtype": "bfloat16", "wtype": "bfloat16",
         "residual": True, "out": "float8_e4m3fn", "group": 128},
        # The activation shard of the all-gather workload, quantised before it travels.
        {"name": "norm_8bit_8192x4096", "kind": "norm", "rows": 8192, "cols": 4096, "dtype": "bfloat16", "wtype": "float32",
         "residual": True, "out": "float8_e4m3fn", "group": 128},
        # The same shard in training: forward and backward, weights in float32 as the fused optimizers take them.
        {"name": "norm_train_8192x4096", "kind": "norm_train", "rows": 8192, "cols": 4096, "dtype": "bfloat16",
         "wtype": "float32", "residual": True, "out": "", "group": 0},
        # A width that no vector divides, in full precision, without a residual.
        {"name": "norm_train_odd", "kind": "norm_train", "rows": 2053, "cols": 771, "dtype": "float32", "wtype": "float32",
         "residual": False, "out": "", "group": 0},
        # A few tokens of a decoding batch over few experts.
        {"name": "route_four_tokens", "kind": "route", "tokens": 4, "experts": 64, "k": 6, "dtype": "float32",
         "scores": "softmax", "bias": False, "groups": 1, "keep": 1, "best": 1, "renorm": True, "scale": 1.0, "pad": False},
        # A prompt batch, many experts in groups, sigmoid scores with a balance bias.
        {"name": "route_groups_8192x256", "kind": "route", "tokens": 8192, "experts": 256, "k": 8, "dtype": "bfloat16",
         "scores": "sigmoid", "bias": True, "groups": 8, "keep": 4, "best": 2, "renorm": True, "scale": 2.5, "pad": False},
        # A large training batch, softmax scores.
        {"name": "route_train_65536x128", "kind": "route_train", "tokens": 65536, "experts": 128, "k": 8, "dtype": "float32",
         "scores": "softmax", "bias": False, "groups": 1, "keep": 1, "best": 1, "renorm": True, "scale": 1.0, "pad": False},
        # A padded batch, an odd number of experts, a bias on softmax scores, weights that are not renormalised.
        {"name": "route_train_odd", "kind": "route_train", "tokens": 1537, "experts": 61, "k": 5, "dtype": "float16",
         "scores": "softmax", "bias": True, "groups": 1, "keep": 1, "best": 1, "renorm": False, "scale": 1.5, "pad": True},
        # Three new tokens of a serving model.
        {"name": "exchange_three_tokens", "kind": "exchange", "tokens": 3, "experts": 256, "k": 8, "cols": 4096,
         "dtype": "bfloat16", "align": 1, "residual": True, "pad": False},
        # A prompt batch in 8 bits, the experts' blocks aligned for their products.
        {"name": "dispatch_8bit_8192x4096", "kind": "dispatch", "tokens": 8192, "experts": 256, "k": 8, "cols": 4096,
         "dtype": "float8_e4m3fn", "align": 128, "residual": False, "pad": False},
        # A training batch: forward, backward and the balance update.
        {"name": "exchange_train_8192x2048", "kind": "exchange_train", "tokens": 8192, "experts": 64, "k": 8, "cols": 2048,
         "dtype": "bfloat16", "align": 1, "residual": True, "pad": False},
        # A padded batch of odd sizes in full precision.
        {"name": "exchange_train_odd", "kind": "exchange_train", "tokens": 1021, "experts": 7, "k": 3, "cols": 769,
         "dtype": "float32", "align": 8, "residual": False, "pad": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_train", "route", "route_train", "dispatch", "exchange", "exchange_train"])
    if kind in ("norm", "norm_train"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = -(-cols // 64) * 64
        rows = _log(rng, 1, max(2, min(65536, (32 << 20) // cols)))
        case = {"kind": kind, "rows": rows, "cols": cols, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
                "residual": rng.random() < 0.7, "out": "", "group": 0}
        case["wtype"] = rng.choice(["float32", case["dtype"]])
        if kind == "norm" and rng.random() < 0.6:
            case["out"] = rng.choice(["float8_e4m3fn", "float8_e4m3fn", "float8_e5m2"])
            case["group"] = rng.choice([0, 32, 64, 128, 128])
        return case
    experts = _log(rng, 4, 512)
    if kind in ("route", "route_train"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = max(groups * 2, experts // groups * groups)
        keep = rng.randint(1, groups)
        return {"kind": kind, "tokens": _log(rng, 1, min(65536, (16 << 20) // experts)), "experts": experts,
                "k": rng.randint(1, min(16, experts // groups * keep)), "dtype": rng.choice(["float32", "bfloat16", "float16"]),
                "scores": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "keep": keep,
                "best": rng.choice([1, 2]), "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]),
                "pad": rng.random() < 0.3}
    cols = _log(rng, 64, 8192)
    if rng.random() < 0.7:
        cols = -(-cols // 128) * 128
    k = rng.randint(1, min(10, experts))
    dtype = "float8_e4m3fn" if kind == "dispatch" else rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    row = cols * {"float8_e4m3fn": 1, "float32": 4}.get(dtype, 2)
    tokens = _log(rng, 1, min(32768, (192 << 20) // (row * (k + 1))))
    align = rng.choice([1, 8, 128])
    if min(experts, tokens * k) * align * row > 256 << 20:
        align = 8  # the blocks' last rows would outweigh the tokens'
    return {"kind": kind, "tokens": tokens, "experts": experts, "k": k, "cols": cols, "dtype": dtype, "align": align,
            "residual": kind != "dispatch" and rng.random() < 0.5, "pad": rng.random() < 0.3}


# ---- inputs --------------------------------------------------------------------------------


def _capacity(case):
    """Rows that the experts' blocks take at most, each block rounded up to `align`."""
    slots = case["tokens"] * case["k"]
    return slots + min(case["experts"], slots) * (case["align"] - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    state = {"case": case}
    if kind in ("norm", "norm_train"):
        t, shape = DTYPES[case["dtype"]], (case["rows"], case["cols"])
        state["x"] = normal(*shape, dtype=t)
        state["residual"] = (2 * normal(*shape)).to(t) if case["residual"] else None
        state["weight"] = (1 + 0.1 * normal(case["cols"])).to(DTYPES[case["wtype"]])
        if kind == "norm_train":
            state["grad_output"] = normal(*shape, dtype=t)
            state["grad_hidden"] = normal(*shape, dtype=t) if case["residual"] else None
        return state
    tokens, experts, k = case["tokens"], case["experts"], case["k"]
    popular = 0.3 * normal(experts)  # some experts are asked for more often
    logits = normal(tokens, experts) + popular
    # A padded batch: sequences of up to 64 places, each of them partly filled.
    mask = None
    if case["pad"]:
        filled = torch.randint(1, 65, (-(-tokens // 64), 1), generator=g, device="cuda")
        mask = (torch.arange(64, device="cuda") < filled).reshape(-1)[:tokens].contiguous()
    if kind in ("route", "route_train"):
        state["logits"] = logits.to(DTYPES[case["dtype"]])
        state["bias"] = (0.02 if case["scores"] == "softmax" else 0.1) * normal(experts) if case["bias"] else None
        state["mask"] = mask
        if kind == "route_train":
            state["grad_weights"] = normal(tokens, k)
        return state
    chosen = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k].to(torch.int32)
    state["indices"] = (torch.where(mask[:, None], chosen, -1) if mask is not None else chosen).contiguous()
    capacity, cols = _capacity(case), case["cols"]
    if kind == "dispatch":
        state["x"] = (64 * normal(tokens, cols)).clamp(-448, 448).to(DTYPES[case["dtype"]])
        state["scale"] = torch.rand(tokens, -(-cols // 128), generator=g, device="cuda") * 0.01
        state["rows"] = torch.zeros(capacity, cols, dtype=DTYPES[case["dtype"]], device="cuda")
        state["scale_rows"] = torch.zeros(capacity, state["scale"].shape[1], device="cuda")
        return state
    t = DTYPES[case["dtype"]]
    state["x"] = normal(tokens, cols, dtype=t)
    state["weights"] = torch.softmax(normal(tokens, k), dim=1)
    state["outputs"] = normal(capacity, cols, dtype=t)  # what the experts made of their rows
    state["residual"] = normal(tokens, cols, dtype=t) if case["residual"] else None
    state["rows"] = torch.zeros(capacity, cols, dtype=t, device="cuda")
    if kind == "exchange_train":
        state["bias"] = 0.02 * normal(experts)
        state["grad_output"] = normal(tokens, cols, dtype=t)
        state["grad_inputs"] = normal(capacity, cols, dtype=t)  # the gradient of the experts' inputs
        state["grad_rows"] = torch.zeros(capacity, cols, dtype=t, device="cuda")
    return state


# ---- one pass ------------------------------------------------------------------------------


def run(state):
    if own:
        return _RUN_OWN[state["case"]["kind"]](state)
    return _RUN_PLAIN[state["case"]["kind"]](state)


def _own_norm(s):
    from dragon_b200.normalization import rms_norm
    case = s["case"]
    r = rms_norm(s["x"], s["weight"], s["residual"], EPS, out_dtype=DTYPES[case["out"]] if case["out"] else None,
                 group_size=case["group"])
    return {"output": r.output, "scale": r.scale, "hidden": r.hidden if case["residual"] else None, "rstd": r.rstd}


def _own_norm_train(s):
    from dragon_b200.normalization import rms_norm, rms_norm_grad
    r = rms_norm(s["x"], s["weight"], s["residual"], EPS)
    grad_x, grad_weight = rms_norm_grad(s["grad_output"], r.hidden, r.rstd, s["weight"], s["grad_hidden"])
    return {"output": r.output, "grad_x": grad_x, "grad_weight": grad_weight}


def _own_route(s):
    from dragon_b200.experts import route
    c = s["case"]
    indices, weights = route(s["logits"], c["k"], s["bias"], s["mask"], scores=c["scores"], groups=c["groups"],
                             keep_groups=c["keep"], group_best=c["best"], renormalize=c["renorm"], scale=c["scale"])
    return {"indices": indices, "weights": weights}


def _own_route_train(s):
    from dragon_b200.experts import route_grad
    c = s["case"]
    r = _own_route(s)
    r["grad_logits"] = route_grad(s["grad_weights"], s["logits"], r["indices"], scores=c["scores"],
                                  renormalize=c["renorm"], scale=c["scale"])
    return r


def _own_dispatch(s):
    from dragon_b200.experts import dispatch, plan
    p = plan(s["indices"], s["case"]["experts"], s["case"]["align"])
    return {"counts": p.counts, "offsets": p.offsets, "positions": p.positions,
            "rows": dispatch(s["x"], p, out=s["rows"]), "scale_rows": dispatch(s["scale"], p, out=s["scale_rows"])}


def _own_exchange(s):
    from dragon_b200.experts import combine, dispatch, plan
    p = plan(s["indices"], s["case"]["experts"], s["case"]["align"])
    return {"rows": dispatch(s["x"], p, out=s["rows"]), "output": combine(s["outputs"], p, s["weights"], s["residual"])}


def _own_exchange_train(s):
    from dragon_b200.experts import combine, combine_grad, dispatch, dispatch_grad, plan, update_bias
    p = plan(s["indices"], s["case"]["experts"], s["case"]["align"])
    rows = dispatch(s["x"], p, out=s["rows"])
    output = combine(s["outputs"], p, s["weights"], s["residual"])
    grad_rows, grad_weights = combine_grad(s["grad_output"], s["outputs"], p, s["weights"], out=s["grad_rows"])
    return {"rows": rows, "output": output, "grad_rows": grad_rows, "grad_weights": grad_weights,
            "grad_x": dispatch_grad(s["grad_inputs"], p),
            "bias": update_bias(s["bias"], p.counts, 1e-3, out=torch.empty_like(s["bias"]))}


_RUN_OWN = {"norm": _own_norm, "norm_train": _own_norm_train, "route": _own_route, "route_train": _own_route_train,
            "dispatch": _own_dispatch, "exchange": _own_exchange, "exchange_train": _own_exchange_train}


def _plain_norm(s):
    case, t = s["case"], s["x"].dtype
    hidden = (s["x"].float() + s["residual"].float()).to(t) if case["residual"] else s["x"]
    h = hidden.float()
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
    y = h * rstd * s["weight"].float()
    out = {"hidden": hidden if case["residual"] else None, "rstd": rstd[:, 0], "scale": None}
    if not case["out"]:
        out["output"] = y.to(t)
        return out
    rows, cols = y.shape
    width = case["group"] or cols
    n = -(-cols // width)
    padded = torch.nn.functional.pad(y, (0, n * width - cols)).view(rows, n, width)
    amax = padded.abs().amax(2).clamp(min=SMALLEST_AMAX)
    largest = LARGEST[case["out"]]
    codes = (padded * (largest / amax)[:, :, None]).clamp(-largest, largest)
    out["scale"] = amax / largest
    out["output"] = codes.view(rows, n * width)[:, :cols].contiguous().to(DTYPES[case["out"]])
    return out


def _plain_norm_train(s):
    t = s["x"].dtype
    r = _plain_norm(s)
    h = s["x"].float() if r["hidden"] is None else r["hidden"].float()
    rstd, w, dy = r["rstd"][:, None], s["weight"].float(), s["grad_output"].float()
    normed = h * rstd
    g = dy * w
    grad = rstd * (g - normed * (g * normed).mean(1, keepdim=True))
    if s["grad_hidden"] is not None:
        grad = grad + s["grad_hidden"].float()
    return {"output": r["output"], "grad_x": grad.to(t), "grad_weight": (dy * normed).sum(0).to(s["weight"].dtype)}


def _scores(logits, kind):
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    e = torch.exp(logits - logits.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True)


def _largest_first(x, k):
    """Places of the k largest of each row, equal ones in their order."""
    return torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]


def _plain_route(s):
    c, logits = s["case"], s["logits"]
    tokens, experts = logits.shape
    # The choice hangs on values next to each other: 64 bits.
    exact = _scores(logits.double(), c["scores"])
    key = logits.double() if s["bias"] is None else exact + s["bias"].double()
    if c["groups"] > 1:
        value = exact if s["bias"] is None and c["best"] > 1 else key
        best = torch.sort(value.view(tokens, c["groups"], -1), dim=2, descending=True)[0][:, :, :c["best"]].sum(2)
        kept = torch.zeros(tokens, c["groups"], dtype=torch.bool, device=key.device)
        kept.scatter_(1, _largest_first(best, c["keep"]), True)
        key = torch.where(kept.repeat_interleave(experts // c["groups"], 1), key, -math.inf)
    chosen = _largest_first(key, c["k"])
    w = _scores(logits.float(), c["scores"]).gather(1, chosen)
    if c["renorm"]:
        w = w / (w.sum(1, keepdim=True) + TINY)
    w = w * c["scale"]
    if s["mask"] is not None:
        chosen, w = torch.where(s["mask"][:, None], chosen, -1), torch.where(s["mask"][:, None], w, 0.0)
    return {"indices": chosen.to(torch.int32), "weights": w}


def _plain_route_train(s):
    c = s["case"]
    r = _plain_route(s)
    there = r["indices"] >= 0
    at = r["indices"].clamp(min=0).long()
    score = _scores(s["logits"].float(), c["scores"])
    ds = c["scale"] * s["grad_weights"]
    if c["renorm"]:
        mine = score.gather(1, at)
        total = mine.sum(1, keepdim=True) + TINY
        ds = (ds - (ds * mine).sum(1, keepdim=True) / total) / total
    grad_scores = torch.zeros_like(score).scatter_(1, at, torch.where(there, ds, 0.0))
    if c["scores"] == "sigmoid":
        grad = grad_scores * score * (1 - score)
    else:
        grad = score * (grad_scores - (grad_scores * score).sum(1, keepdim=True))
    r["grad_logits"] = grad.to(s["logits"].dtype)
    return r


def _plain_plan(indices, experts, align, capacity):
    flat = indices.reshape(-1).long()
    there = flat >= 0
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device)
    counts.scatter_add_(0, torch.where(there, flat, experts), torch.ones_like(flat))
    counts = counts[:experts]
    blocks = (counts + align - 1) // align * align
    offsets = torch.cat([torch.zeros_like(counts[:1]), blocks.cumsum(0)])
    order = torch.sort(torch.where(there, flat, experts), stable=True)[1]
    first = torch.cat([torch.zeros_like(counts[:1]), counts.cumsum(0)])
    expert = torch.where(there, flat, experts)[order]
    rank = torch.arange(flat.numel(), device=flat.device) - first[expert]
    # Slots without an expert go to a row behind the last.
    at = torch.where(expert < experts, offsets[expert] + rank, capacity)
    place = torch.empty_like(flat)
    place[order] = at
    return {"counts": counts.to(torch.int32), "offsets": offsets.to(torch.int32),
            "positions": torch.where(there, place, -1).to(torch.int32).view(indices.shape), "place": place}


def _plain_move(x, place, k, capacity):
    """Row t of x at each of its places, zeros elsewhere."""
    eight = x.dtype == torch.float8_e4m3fn
    source = x.view(torch.uint8) if eight else x
    rows = torch.zeros(capacity + 1, x.shape[1], dtype=source.dtype, device=x.device)
    rows[place] = source.repeat_interleave(k, 0)
    return rows[:capacity].view(x.dtype) if eight else rows[:capacity]


def _plain_gather(rows, place, tokens, k):
    """[tokens, k, cols] in 32 bits; zeros where a slot has no expert."""
    there = place < rows.shape[0]
    got = rows[torch.where(there, place, 0)].float()
    return torch.where(there[:, None], got, 0.0).view(tokens, k, -1)


def _plain_dispatch(s):
    c = s["case"]
    p = _plain_plan(s["indices"], c["experts"], c["align"], _capacity(c))
    place = p.pop("place")
    p["rows"] = _plain_move(s["x"], place, c["k"], _capacity(c))
    p["scale_rows"] = _plain_move(s["scale"], place, c["k"], _capacity(c))
    return p


def _plain_combine(s, place, t):
    c = s["case"]
    total = (_plain_gather(s["outputs"], place, c["tokens"], c["k"]) * s["weights"][:, :, None]).sum(1)
    if s["residual"] is not None:
        total = total + s["residual"].float()
    return total.to(t)


def _plain_exchange(s):
    c, t = s["case"], s["x"].dtype
    place = _plain_plan(s["indices"], c["experts"], c["align"], _capacity(c))["place"]
    return {"rows": _plain_move(s["x"], place, c["k"], _capacity(c)), "output": _plain_combine(s, place, t)}


def _plain_exchange_train(s):
    c, t = s["case"], s["x"].dtype
    tokens, k, capacity = c["tokens"], c["k"], _capacity(c)
    p = _plain_plan(s["indices"], c["experts"], c["align"], capacity)
    place = p["place"]
    grad = s["grad_output"].float()
    grad_rows = torch.zeros(capacity + 1, c["cols"], dtype=t, device=place.device)
    grad_rows[place] = (grad[:, None, :] * s["weights"][:, :, None]).to(t).view(tokens * k, -1)
    counts = p["counts"].long()
    lacking = (counts.sum() - c["experts"] * counts).sign()  # 1 where an expert had fewer tokens than the mean
    return {"rows": _plain_move(s["x"], place, k, capacity), "output": _plain_combine(s, place, t),
            "grad_rows": grad_rows[:capacity],
            "grad_weights": (_plain_gather(s["outputs"], place, tokens, k) * grad[:, None, :]).sum(2),
            "grad_x": _plain_gather(s["grad_inputs"], place, tokens, k).sum(1).to(t), "bias": s["bias"] + 1e-3 * lacking}


_RUN_PLAIN = {"norm": _plain_norm, "norm_train": _plain_norm_train, "route": _plain_route, "route_train": _plain_route_train,
              "dispatch": _plain_dispatch, "exchange": _plain_exchange, "exchange_train": _plain_exchange_train}


# ---- what a pass cannot do without -----------------------------------------------------------


def work(case):
    kind = case["kind"]
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if kind in ("norm", "norm_train"):
        n, wsize = case["rows"] * case["cols"], torch.empty((), dtype=DTYPES[case["wtype"]]).element_size()
        weight = case["cols"] * wsize
        read = n * size * (2 if case["residual"] else 1) + weight
        if kind == "norm":
            groups = -(-case["cols"] // (case["group"] or case["cols"]))
            written = n * (1 + 4 * groups / case["cols"]) if case["out"] else n * size
            written += 4 * case["rows"] + (n * size if case["residual"] else 0)
            return {"bytes": read + written, "flops": 6 * n}
        # Forward: the output; backward: its gradient and the hidden values' in, the inputs' gradient out.
        written = n * size + n * size + weight
        read += n * size * (2 if case["residual"] else 1)
        return {"bytes": read + written, "flops": 16 * n}
    tokens, k = case["tokens"], case["k"]
    slots = tokens * k
    if kind in ("route", "route_train"):
        n = tokens * case["experts"]
        data = n * size + 8 * slots + (4 * case["experts"] if case["bias"] else 0) + (tokens if case["pad"] else 0)
        if kind == "route_train":
            data += n * size + 4 * slots
        return {"bytes": data, "flops": n * (k + 6) + (8 * n if kind == "route_train" else 0)}
    row = case["cols"] * size
    data = 4 * slots + tokens * row + slots * row
    if kind == "dispatch":
        scale = 4 * -(-case["cols"] // 128)
        return {"bytes": data + tokens * scale + slots * scale + 4 * slots + 8 * case["experts"], "flops": 8 * slots}
    combined = slots * row + tokens * row * (2 if case["residual"] else 1) + 4 * slots
    if kind == "exchange":
        return {"bytes": data + combined, "flops": 2 * slots * case["cols"]}
    # Backward: the output's gradient in, the experts' outputs' out; the experts' inputs' in, the tokens' out.
    back = tokens * row + slots * row + 4 * slots + slots * row + tokens * row + 8 * case["experts"]
    return {"bytes": data + combined + back, "flops": 7 * slots * case["cols"]}


# ---- the definition in 64 bits -----------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "norm_train": _exact_norm, "route": _exact_route, "route_train": _exact_route,
            "dispatch": _exact_exchange, "exchange": _exact_exchange, "exchange_train": _exact_exchange}[case["kind"]](s)


def _exact_norm(s):
    c, t = s["case"], s["x"].dtype
    hidden = s["x"].double()
    if c["residual"]:
        hidden = (hidden + s["residual"].double()).to(t).double()
    rstd = (torch.linalg.vector_norm(hidden, dim=1).square() / c["cols"] + EPS).rsqrt()
    w = s["weight"].double()
    y = torch.einsum("rc,r,c->rc", hidden, rstd, w)
    if c["kind"] == "norm":
        out = {"output": y, "scale": None, "hidden": hidden if c["residual"] else None, "rstd": rstd}
        if c["out"]:
            width = c["group"] or c["cols"]
            spans = [slice(a, min(a + width, c["cols"])) for a in range(0, c["cols"], width)]
            largest = torch.stack([y[:, a].abs().max(1).values for a in spans], 1).clamp(min=SMALLEST_AMAX)
            out["scale"] = largest / LARGEST[c["out"]]
            codes = torch.empty_like(y)
            for i, a in enumerate(spans):
                codes[:, a] = y[:, a] / out["scale"][:, i:i + 1]
            out["output"] = codes.float().to(DTYPES[c["out"]]).double()
        return out
    dy = s["grad_output"].double()
    # The Jacobian of y / w with respect to the hidden values is rstd (I - n n^T / cols), n the normalised row.
    n = hidden * rstd[:, None]
    inner = torch.einsum("rc,c,rc->r", dy, w, n) / c["cols"]
    grad = torch.einsum("r,rc->rc", rstd, dy * w - inner[:, None] * n)
    if s["grad_hidden"] is not None:
        grad += s["grad_hidden"].double()
    return {"output": y, "grad_x": grad, "grad_weight": torch.einsum("rc,rc->c", dy, n)}


def _exact_route(s):
    c = s["case"]
    l = s["logits"].double()
    tokens, experts = l.shape
    score = torch.sigmoid(l) if c["scores"] == "sigmoid" else torch.softmax(l, 1)
    key = l if s["bias"] is None else score + s["bias"].double()
    open_ = torch.ones(tokens, c["groups"], dtype=torch.bool, device=l.device)
    if c["groups"] > 1:
        value = (score if s["bias"] is None and c["best"] > 1 else key).reshape(tokens, c["groups"], -1)
        best = value.max(2).values if c["best"] == 1 or value.shape[2] == 1 else value.topk(2, dim=2).values.sum(2)
        open_.zero_()
        for _ in range(c["keep"]):  # one group after the other, the first of equal ones
            at = torch.where(open_, -math.inf, best).argmax(1, keepdim=True)
            first = (torch.where(open_, -math.inf, best) == best.gather(1, at)).int().argmax(1, keepdim=True)
            open_.scatter_(1, first, True)
    left = torch.where(open_[:, :, None], key.reshape(tokens, c["groups"], -1), -math.inf).reshape(tokens, experts)
    chosen = []
    for _ in range(c["k"]):
        top = left.max(1, keepdim=True).values
        first = (left == top).int().argmax(1, keepdim=True)
        chosen.append(first)
        left = left.scatter(1, first, -math.inf)
    chosen = torch.cat(chosen, 1)
    live = torch.ones(tokens, 1, dtype=torch.float64, device=l.device) if s["mask"] is None else s["mask"][:, None].double()
    mine = score.gather(1, chosen)
    total = mine.sum(1, keepdim=True) + TINY if c["renorm"] else torch.ones_like(mine[:, :1])
    out = {"indices": torch.where(live > 0, chosen, -1).to(torch.int32), "weights": c["scale"] * live * mine / total}
    if c["kind"] == "route":
        return out
    # d weights_j / d scores_i = scale (delta_ij - weights_j / scale) / total, or scale delta_ij.
    dw = s["grad_weights"].double() * live
    shared = (dw * out["weights"]).sum(1, keepdim=True) / total if c["renorm"] else 0.0
    ds = c["scale"] * dw / total - shared * live
    if c["scores"] == "sigmoid":
        out["grad_logits"] = torch.zeros_like(l).scatter_(1, chosen, ds * mine * (1 - mine))
    else:
        picked = torch.zeros_like(l).scatter_(1, chosen, ds * mine)
        out["grad_logits"] = picked - score * picked.sum(1, keepdim=True)
    return out


def _exact_exchange(s):
    c, device = s["case"], s["x"].device
    tokens, k, experts, align, capacity = c["tokens"], c["k"], c["experts"], c["align"], _capacity(c)
    slots = s["indices"].reshape(-1).tolist()
    counts = [0] * experts
    for e in slots:
        if e >= 0:
            counts[e] += 1
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + -(-n // align) * align)
    following, positions, source = list(offsets[:experts]), [], [tokens] * capacity
    for i, e in enumerate(slots):
        positions.append(following[e] if e >= 0 else -1)
        if e >= 0:
            source[following[e]] = i // k
            following[e] += 1
    owner = torch.tensor(source, device=device)
    at = torch.tensor(positions, device=device).view(tokens, k)

    def moved(x):
        return torch.cat([x.double(), torch.zeros(1, x.shape[1], dtype=torch.float64, device=device)])[owner]

    out = {"rows": moved(s["x"])}
    if c["kind"] == "dispatch":
        out["scale_rows"] = moved(s["scale"])
        out["counts"] = torch.tensor(counts, dtype=torch.int32, device=device)
        out["offsets"] = torch.tensor(offsets, dtype=torch.int32, device=device)
        out["positions"] = at.to(torch.int32)
        return out
    w = torch.where(at >= 0, s["weights"].double(), 0.0)
    total = torch.zeros(tokens, c["cols"], dtype=torch.float64, device=device)
    if s["residual"] is not None:
        total += s["residual"].double()
    for j in range(k):
        total += w[:, j:j + 1] * s["outputs"][at[:, j].clamp(min=0)].double()
    out["output"] = total
    if c["kind"] == "exchange":
        return out
    dout = s["grad_output"].double()
    grad_rows = torch.zeros(capacity + 1, c["cols"], dtype=torch.float64, device=device)
    grad_x, grad_w = torch.zeros_like(dout), torch.zeros_like(w)
    for j in range(k):
        there = (at[:, j:j + 1] >= 0).double()
        row = at[:, j].clamp(min=0)
        grad_rows[torch.where(at[:, j] >= 0, at[:, j], capacity)] = w[:, j:j + 1] * dout
        grad_w[:, j] = (dout * s["outputs"][row].double() * there).sum(1)
        grad_x += s["grad_inputs"][row].double() * there
    mean = sum(counts) / experts
    step = [1e-3 * ((n < mean) - (n > mean)) for n in counts]
    out.update(grad_rows=grad_rows[:capacity], grad_weights=grad_w, grad_x=grad_x,
               bias=s["bias"].double() + torch.tensor(step, dtype=torch.float64, device=device))
    return out

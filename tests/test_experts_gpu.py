"""The operators of a layer of experts against plain implementations in 64 bits.

Tolerances.  u = 2^-24 is half a step of float32.  A score is an exponential
(4 u: 2 steps of expf and its argument's rounding times the argument, below 16)
over a sum of up to 1024 positive ones; weights, their sums and quotients add a
few roundings each: 40 u relative.  Sums over columns are bounded by the sum of
their terms' magnitudes times the additions that follow one another."""

import math

import pytest
import torch

from dragon_b200 import experts
from dragon_b200.experts import combine, combine_grad, dispatch, dispatch_grad, plan, route, route_grad, update_bias

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
FLOATS = [torch.float32, torch.bfloat16, torch.float16]
DEV = "cuda:0"
INF = float("inf")


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def normal(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(DEV)


def close(got, want, bound, what=""):
    off = (got.double() - want).abs() - bound
    assert not torch.isnan(off).any() and off.max() <= 0, "{}: {} past its bound".format(what, off.max().item())


# ---- choice --------------------------------------------------------------------------------


def first(values, count):
    """Places of the largest, NaN before all, equal ones in their order."""
    rank = lambda i: (not math.isnan(values[i]), -values[i] if not math.isnan(values[i]) else 0.0, i)  # noqa: E731
    return sorted((i for i in range(len(values)) if values[i] != -INF), key=rank)[:count]


def route_reference(logits, k, bias=None, mask=None, scores="softmax", groups=1, keep_groups=1, group_best=1,
                    renormalize=True, scale=1.0):
    l = logits.double().cpu()
    tokens, num = l.shape
    score = (1 / (1 + torch.exp(-l))) if scores == "sigmoid" else torch.softmax(l, 1)
    indices, weights = torch.full((tokens, k), -1, dtype=torch.int32), torch.zeros(tokens, k, dtype=torch.float64)
    for t in range(tokens):
        if mask is not None and not mask[t]:
            continue
        s = score[t].tolist()
        ls = l[t].tolist()
        s = [0.0 if ls[e] == -INF else s[e] for e in range(num)]
        key = ls if bias is None else [-INF if ls[e] == -INF else s[e] + float(bias[e]) for e in range(num)]
        if groups > 1:
            width, value = num // groups, (s if bias is None and group_best == 2 else key)
            best = []
            for g in range(groups):
                members = [value[e] if key[e] != -INF else -INF for e in range(g * width, g * width + width)]
                top = first(members, group_best)
                best.append(sum(members[i] for i in top) if top else -INF)
            kept = first(best, keep_groups)
            key = [key[e] if e // width in kept else -INF for e in range(num)]
        chosen = first(key, k)
        total = sum(s[e] for e in chosen) + 1e-20 if renormalize else 1.0
        for j, e in enumerate(chosen):
            indices[t, j], weights[t, j] = e, scale * s[e] / total
    return indices, weights


def check_route(logits, k, **kwargs):
    indices, weights = route(logits, k, **kwargs)
    host = {n: v.cpu() if isinstance(v, torch.Tensor) else v for n, v in kwargs.items()}
    want_i, want_w = route_reference(logits, k, **host)
    assert torch.equal(indices.cpu(), want_i)
    fine = torch.isfinite(want_w)
    assert torch.equal(torch.isnan(weights.cpu()), torch.isnan(want_w))
    close(weights.cpu()[fine], want_w[fine], 40 * U * want_w[fine].abs() + 1e-37, "weights")


CHOICES = [  # experts, k, groups, keep, best
    (1, 1, 1, 1, 1), (2, 1, 1, 1, 1), (7, 7, 1, 1, 1), (32, 4, 1, 1, 1), (33, 5, 1, 1, 1), (64, 6, 8, 3, 1), (64, 8, 4, 2, 2),
    (96, 32, 1, 1, 1), (128, 8, 1, 1, 1), (160, 6, 32, 9, 2), (256, 8, 8, 4, 2), (257, 9, 1, 1, 1), (384, 8, 2, 1, 2),
    (512, 10, 4, 3, 1), (600, 3, 3, 2, 2), (1024, 32, 1, 1, 1), (1024, 8, 32, 4, 2), (96, 8, 3, 2, 2), (96, 4, 6, 3, 1),
    (48, 4, 2, 1, 2), (192, 6, 6, 2, 2), (320, 8, 5, 3, 2), (24, 3, 3, 1, 2)]


@pytest.mark.parametrize("num,k,groups,keep,best", CHOICES)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", FLOATS)
def test_route(dgn_lib, num, k, groups, keep, best, scores, with_bias, dtype):
    bias = normal(num, seed=2, scale=0.1) if with_bias else None
    kwargs = dict(scores=scores, bias=bias, groups=groups, keep_groups=keep, group_best=best)
    for tokens, renormalize, scale in ((1, True, 1.0), (37, False, 2.5)):
        check_route(normal(tokens, num, seed=tokens, dtype=dtype), k, renormalize=renormalize, scale=scale, **kwargs)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("num,k", [(8, 3), (64, 8), (256, 8), (320, 16)])
def test_equal_experts_are_taken_in_their_order(dgn_lib, scores, num, k):
    g = torch.Generator().manual_seed(3)
    logits = torch.randint(-2, 3, (64, num), generator=g).float().to(DEV)
    check_route(logits, k, scores=scores)
    check_route(logits * 0, k, scores=scores)
    check_route(logits, k, scores=scores, bias=torch.zeros(num, device=DEV))
    check_route(logits, k, scores=scores, groups=4, keep_groups=2)
    check_route(logits, k, scores=scores, bias=torch.zeros(num, device=DEV), groups=2, keep_groups=1 if num // 2 >= k else 2)


def test_neighbours_are_told_apart_as_in_64_bits(dgn_lib):
    """Keys that differ by far less than a step of float32."""
    num, k = 64, 8
    logits = normal(256, num, seed=4, scale=0.01)
    for e in range(1, num, 2):  # pairs of neighbours, one step of float32 apart
        logits[:, e] = torch.nextafter(logits[:, e - 1], torch.full_like(logits[:, 0], INF))
    bias = normal(num, seed=5, scale=0.1).repeat_interleave(2)[:num].contiguous()
    for scores in ("softmax", "sigmoid"):
        check_route(logits, k, scores=scores)
        check_route(logits, k, scores=scores, bias=bias)
        check_route(logits, k, scores=scores, bias=bias, groups=8, keep_groups=3, group_best=2)
        # A bias that undoes the scores: all keys nearly equal.
        s = torch.sigmoid(logits[0].double()) if scores == "sigmoid" else torch.softmax(logits[0].double(), 0)
        check_route(logits[:1].repeat(4, 1).contiguous(), k, scores=scores, bias=(0.9 - s).float())


def test_masks_and_values_that_are_not_finite(dgn_lib):
    for num, k, dtype in ((16, 4, torch.float32), (64, 6, torch.bfloat16), (256, 8, torch.float16)):
        logits = normal(12, num, seed=6).to(dtype)
        lowest = torch.finfo(dtype).min
        logits[0] = -INF                       # nothing left
        logits[1, 2:] = -INF                   # fewer than k
        logits[2] = lowest                     # a mask by the lowest value: still a choice
        logits[3, 3:] = lowest
        logits[4, 5] = float("nan")
        logits[5, 7] = INF
        logits[6, ::2] = -INF
        logits[7] = torch.finfo(dtype).max
        mask = torch.ones(12, dtype=torch.bool, device=DEV)
        mask[8] = mask[11] = False
        logits[8] = float("nan")
        for scores in ("softmax", "sigmoid"):
            for kwargs in (dict(), dict(bias=normal(num, seed=7, scale=0.1)), dict(groups=4, keep_groups=2),
                           dict(groups=2, keep_groups=1, group_best=2)):
                check_route(logits, k, scores=scores, mask=mask, **kwargs)
        bias = normal(num, seed=8, scale=0.1)
        bias[1:num - 1] = -INF                 # two experts are open
        check_route(logits[6:8].clone(), k, bias=bias)


def test_scores_that_vanish(dgn_lib):
    logits = torch.full((3, 8), -200.0, device=DEV)
    logits[:, 0] = 0
    bias = torch.zeros(8, device=DEV)
    bias[0] = -5  # chosen last: the others' softmax scores are below float32
    check_route(logits, 3, bias=bias)
    check_route(logits, 3, scores="sigmoid", bias=bias)


def route_grad_reference(grad_weights, logits, indices, scores, renormalize, scale):
    l = logits.double()
    there = (indices >= 0) & (indices < logits.shape[1])
    at = torch.where(there, indices, 0).long()
    score = torch.sigmoid(l) if scores == "sigmoid" else torch.softmax(l, 1)
    mine = torch.where(there, score.gather(1, at), 0.0)
    ds = scale * torch.where(there, grad_weights.double(), 0.0)
    size = ds.abs()
    if renormalize:
        total = mine.sum(1, keepdim=True) + 1e-20
        size = (size + (size * mine).sum(1, keepdim=True) / total) / total
        ds = torch.where(there, (ds - (ds * mine).sum(1, keepdim=True) / total) / total, 0.0)
    size = torch.where(there, size, 0.0)
    ds, size = (torch.zeros_like(l).scatter_add_(1, at, v) for v in (ds, size))
    if scores == "sigmoid":
        slope = torch.sigmoid(l) * torch.sigmoid(-l)
        return ds * slope, size * slope
    return score * (ds - (ds * score).sum(1, keepdim=True)), score * (size + (size * score).sum(1, keepdim=True))


@pytest.mark.parametrize("num,k", [(1, 1), (2, 2), (7, 3), (33, 5), (64, 8), (128, 8), (256, 8), (300, 32), (512, 6), (1024, 10)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", FLOATS)
def test_route_grad(dgn_lib, num, k, scores, renormalize, dtype):
    tokens = 41
    logits, grad_weights = normal(tokens, num, seed=1, dtype=dtype), normal(tokens, k, seed=2)
    mask = torch.ones(tokens, dtype=torch.bool, device=DEV)
    mask[5] = False
    indices, _ = route(logits, k, mask=mask, scores=scores)
    grad = route_grad(grad_weights, logits, indices, scores=scores, renormalize=renormalize, scale=1.5)
    want, size = route_grad_reference(grad_weights, logits, indices, scores, renormalize, 1.5)
    close(grad, want, 100 * U * size + half(dtype) * want.abs() + tiny(dtype), "grad_logits")
    assert (grad[5] == 0).all()


def test_route_grad_of_odd_lists(dgn_lib):
    """Missing choices, an expert twice, indices that do not exist; padded rows that hold NaN."""
    logits, grad_weights = normal(4, 16, seed=1), normal(4, 3, seed=2)
    indices = torch.tensor([[3, -1, 7], [5, 5, 2], [16, 1, -9], [-1, -1, -1]], dtype=torch.int32, device=DEV)
    logits[3] = float("nan")
    for scores in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            grad = route_grad(grad_weights, logits, indices, scores=scores, renormalize=renormalize)
            want, size = route_grad_reference(grad_weights[:3], logits[:3], indices[:3], scores, renormalize, 1.0)
            close(grad[:3], want, 100 * U * size)
            assert (grad[3] == 0).all()
    logits = normal(2, 16, seed=1)
    logits[:, 4:] = -INF
    indices, _ = route(logits, 4)
    grad = route_grad(normal(2, 4, seed=3), logits, indices)
    assert (grad[:, 4:] == 0).all() and torch.isfinite(grad).all()


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_grad_sees_differences_only(dgn_lib, scores):
    """Renormalised weights of one choice are constant, and so are those under a gradient that all choices share."""
    logits = normal(200, 24, seed=5)
    one, _ = route(logits, 1, scores=scores)
    grad = route_grad(normal(200, 1, seed=6), logits, one, scores=scores)
    assert grad.abs().max() <= 1e-15  # 1e-20 over the score and its square, times a gradient of a few units
    four, _ = route(logits, 4, scores=scores)
    dw = normal(200, 4, seed=7)
    a, b = (route_grad(w, logits, four, scores=scores) for w in (dw, dw + 64))
    shifted = (dw + 64) - 64  # what the addition leaves of dw: differences of neighbours are exact
    want, size = route_grad_reference(shifted, logits, four, scores, True, 1.0)
    close(b, want, 100 * U * size, "shifted")
    close(a, route_grad_reference(dw, logits, four, scores, True, 1.0)[0], 100 * U * size + 100 * U * size.amax(), "plain")


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_grad_against_differences(dgn_lib, scores, renormalize):
    logits, dw = normal(5, 48, seed=1), normal(5, 6, seed=2)
    indices, _ = route(logits, 6, scores=scores)
    grad = route_grad(dw, logits, indices, scores=scores, renormalize=renormalize, scale=2.0)

    def loss(l):
        s = (torch.sigmoid(l) if scores == "sigmoid" else torch.softmax(l, 1)).gather(1, indices.long())
        return (2.0 * (s / (s.sum(1, keepdim=True) + 1e-20) if renormalize else s) * dw.double()).sum()

    _, size = route_grad_reference(dw, logits, indices, scores, renormalize, 2.0)
    for seed in range(3):
        d = normal(5, 48, seed=10 + seed).double()
        slope = (loss(logits.double() + 1e-5 * d) - loss(logits.double() - 1e-5 * d)) / 2e-5
        bound = (d.abs() * size).sum()
        assert ((grad.double() * d).sum() - slope).abs() <= (100 * U + 1e-8) * bound


# ---- plan and moves --------------------------------------------------------------------------


def plan_reference(indices, num, align):
    flat = indices.reshape(-1).tolist()
    counts = [0] * num
    for e in flat:
        if 0 <= e < num:
            counts[e] += 1
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + -(-n // align) * align)
    following, positions = offsets[:num], []
    for e in flat:
        positions.append(following[e] if 0 <= e < num else -1)
        if 0 <= e < num:
            following[e] += 1
    return counts, offsets, positions


def choices(tokens, k, num, seed=0, missing=0.1):
    g = torch.Generator().manual_seed(seed)
    skew = (torch.rand(tokens, k, generator=g) ** 2 * num).int().clamp(max=num - 1)
    return torch.where(torch.rand(tokens, k, generator=g) < missing, -1, skew).int().to(DEV)


@pytest.mark.parametrize("tokens,k,num,align", [
    (0, 2, 4, 1), (1, 1, 1, 1), (1, 8, 256, 1), (3, 8, 256, 16), (31, 1, 7, 8), (100, 3, 5, 1), (513, 8, 64, 128),
    (1365, 3, 33, 4), (1366, 3, 33, 4), (5000, 8, 1024, 1), (20000, 32, 300, 64), (70000, 10, 128, 1), (40, 8, 768, 1), (9000, 2, 768, 1)])
def test_plan(dgn_lib, tokens, k, num, align):
    indices = choices(tokens, k, num)
    p = plan(indices, num, align)
    counts, offsets, positions = plan_reference(indices, num, align)
    assert p.counts.tolist() == counts
    assert p.offsets.tolist() == offsets
    assert p.ends.tolist() == [a + n for a, n in zip(offsets, counts)]
    assert p.positions.reshape(-1).tolist() == positions
    assert offsets[-1] <= p.capacity


def test_plan_passes_over_indices_that_do_not_exist(dgn_lib):
    indices = torch.tensor([[0, 5], [4, -7], [2147483647, 1], [-2147483648, 0]], dtype=torch.int32, device=DEV)
    p = plan(indices, 5, 2)
    assert p.counts.tolist() == [2, 1, 0, 0, 1] and p.offsets.tolist() == [0, 2, 4, 4, 4, 6]
    assert p.positions.tolist() == [[0, -1], [4, -1], [-1, 2], [-1, 1]]
    same = plan(torch.full((100, 8), 3, dtype=torch.int32, device=DEV), 6)  # all to one expert
    assert same.counts.tolist() == [0, 0, 0, 800, 0, 0] and same.positions.reshape(-1).tolist() == list(range(800))


MOVES = [(1, 1, 1, 16, 1), (3, 8, 256, 4096, 1), (5, 2, 4, 1, 4), (65, 3, 7, 769, 8), (200, 4, 16, 100, 128), (17, 32, 40, 1032, 1),
         (300, 2, 9, 2048, 16), (2, 2, 2, 20000, 1), (40, 3, 8, 4099, 1), (9, 2, 3, 263, 8)]


@pytest.mark.parametrize("tokens,k,num,cols,align", MOVES)
@pytest.mark.parametrize("dtype", FLOATS + [torch.uint8, torch.float8_e4m3fn, torch.int64])
def test_dispatch(dgn_lib, tokens, k, num, cols, align, dtype):
    p = plan(choices(tokens, k, num, seed=1), num, align)
    g = torch.Generator().manual_seed(2)
    size = torch.empty((), dtype=dtype).element_size()
    raw = torch.randint(0, 256, (tokens, cols * size), generator=g, dtype=torch.uint8).to(DEV)
    x = raw.view(dtype)
    filler = torch.full((p.capacity + 3, cols * size), 77, dtype=torch.uint8, device=DEV)
    out = dispatch(x, p, out=filler.view(dtype))
    assert out.data_ptr() == filler.data_ptr()
    want = torch.full((p.capacity + 3, cols * size), 77, dtype=torch.uint8)
    want[:int(p.offsets[-1])] = 0
    for t, row in enumerate(p.positions.tolist()):
        for at in row:
            if at >= 0:
                want[at] = raw[t].cpu()
    assert torch.equal(filler.cpu(), want)
    new = dispatch(x, p)
    assert new.shape == (p.capacity, cols)
    n = int(p.offsets[-1])
    assert torch.equal(new.view(torch.uint8)[:n].cpu(), want[:n])


def test_dispatch_of_strided_rows_and_short_buffers(dgn_lib):
    p = plan(choices(50, 3, 6, seed=1), 6, 4)
    for dtype in (torch.float32, torch.bfloat16, torch.uint8):
        for start, cols in ((0, 64), (1, 64), (3, 61)):
            wide = (100 * normal(50, 80, seed=2)).abs().to(dtype)
            x = wide[:, start:start + cols]
            n = int(p.offsets[-1])
            assert torch.equal(dispatch(x, p)[:n], dispatch(x.contiguous(), p)[:n])
    whole = dispatch(x, p)
    guard = torch.full((20, 61), 9, dtype=torch.uint8, device=DEV)
    short = dispatch(x, p, out=guard[:10])  # rows that do not exist are not written
    assert torch.equal(short, whole[:10]) and (guard[10:] == 9).all()


def combine_reference(rows, positions, weights, residual, tokens):
    at = positions.long()
    there = (at >= 0).double()[:, :, None]
    got = rows[at.clamp(min=0)].double()
    if weights is not None:
        got = got * weights.double()[:, :, None]
    got = torch.where(there > 0, got, 0.0)  # a NaN behind or on a missing slot counts for nothing
    total, size = got.sum(1), got.abs().sum(1)
    if residual is not None:
        total, size = total + residual.double(), size + residual.double().abs()
    return total, size


@pytest.mark.parametrize("tokens,k,num,cols,align", MOVES)
@pytest.mark.parametrize("dtype", FLOATS)
def test_combine_and_its_gradient(dgn_lib, tokens, k, num, cols, align, dtype):
    p = plan(choices(tokens, k, num, seed=1), num, align)
    n = int(p.offsets[-1])
    rows = normal(p.capacity, cols, seed=2, dtype=dtype)
    weights, residual = normal(tokens, k, seed=3), normal(tokens, cols, seed=4, dtype=dtype)
    if p.capacity > n:
        rows[n:] = float("nan")  # nobody's rows
    weights[p.positions < 0] = float("nan")
    for w, r in ((weights, residual), (weights, None), (None, residual), (None, None)):
        want, size = combine_reference(rows, p.positions, w, r, tokens)
        got = combine(rows, p, w, r)
        # k products and sums in a row, each half a step of float32, then the type's rounding.
        close(got, want, (k + 2) * U * size + half(dtype) * want.abs() + tiny(dtype), "combine")
    assert torch.equal(dispatch_grad(rows, p), combine(rows, p))
    grad = normal(tokens, cols, seed=5, dtype=dtype)
    filler = torch.full((p.capacity, cols), 7.0, dtype=dtype, device=DEV)
    grad_rows, grad_weights = combine_grad(grad, rows, p, weights, out=filler)
    want_rows = torch.full((p.capacity, cols), 7.0, dtype=torch.float64)
    want_rows[:n] = 0
    want_w, size_w = torch.zeros(tokens, k, dtype=torch.float64), torch.zeros(tokens, k, dtype=torch.float64)
    wd, gd, rd = weights.double().cpu(), grad.double().cpu(), rows.double().cpu()
    for t, row in enumerate(p.positions.tolist()):
        for j, at in enumerate(row):
            if at >= 0:
                want_rows[at] = wd[t, j] * gd[t]
                want_w[t, j], size_w[t, j] = (gd[t] * rd[at]).sum(), (gd[t] * rd[at]).abs().sum()
    close(grad_rows.cpu(), want_rows, (U + half(dtype)) * want_rows.abs() + tiny(dtype), "grad_rows")
    # A thread adds at most cols / 128 + 8 products, 5 + 8 more additions join the threads.
    close(grad_weights.cpu(), want_w, (cols / 64 + 24) * U * size_w, "grad_weights")
    new_rows, new_weights = combine_grad(grad, rows, p, weights)
    assert torch.equal(new_rows[:n], grad_rows[:n]) and torch.equal(new_weights, grad_weights)


def test_counts_are_the_callers_to_change(dgn_lib):
    """The group's counts may be added up in place before the rows move."""
    p = plan(choices(30, 2, 5, seed=1), 5, 8)
    n, x, weights = int(p.offsets[-1]), normal(30, 12, seed=2), normal(30, 2, seed=3)
    want = dispatch(x, p)
    grads = combine_grad(x, want, p, weights)
    p.counts.mul_(1000)
    ones = torch.ones(p.capacity, 12, device=DEV)
    assert torch.equal(dispatch(x, p, out=ones.clone())[:n], want[:n])
    assert torch.equal(combine_grad(x, want, p, weights, out=ones)[0][:n], grads[0][:n])


def test_combine_of_strided_tensors(dgn_lib):
    p = plan(choices(40, 3, 6, seed=1), 6)
    for dtype in FLOATS:
        rows, weights = normal(p.capacity, 64, seed=2, dtype=dtype), normal(40, 3, seed=3)
        wide = normal(40, 90, seed=4, dtype=dtype)
        for start in (0, 1, 8):
            cut = wide[:, start:start + 64]
            assert torch.equal(combine(rows, p, weights, cut), combine(rows, p, weights, cut.contiguous()))
            a, b = combine_grad(cut, rows, p, weights), combine_grad(cut.contiguous(), rows, p, weights)
            n = int(p.offsets[-1])
            assert torch.equal(a[0][:n], b[0][:n])
            close(a[1], b[1].double(), 100 * U * (cut.double().abs().sum(1) * 5)[:, None])


def test_combine_grad_against_differences(dgn_lib):
    p = plan(choices(6, 3, 4, seed=1), 4)
    rows, weights, dy = normal(p.capacity, 40, seed=2), normal(6, 3, seed=3), normal(6, 40, seed=5)
    grad_rows, grad_weights = combine_grad(dy, rows, p, weights)
    n = int(p.offsets[-1])

    def loss(r, w):
        return (combine_reference(r, p.positions, w, None, 6)[0] * dy.double()).sum()

    for seed in range(3):
        dr, dw = normal(p.capacity, 40, seed=10 + seed).double(), normal(6, 3, seed=20 + seed).double()
        slope = (loss(rows.double() + 1e-5 * dr, weights.double() + 1e-5 * dw)
                 - loss(rows.double() - 1e-5 * dr, weights.double() - 1e-5 * dw)) / 2e-5
        got = (grad_rows[:n].double() * dr[:n]).sum() + (grad_weights.double() * dw).sum()
        size = (grad_rows[:n].double() * dr[:n]).abs().sum() + (dw.abs() * 40 * 16).sum()
        assert (got - slope).abs() <= (64 * U + 1e-9) * size


@pytest.mark.parametrize("num", [1, 2, 33, 256, 1024])
def test_update_bias(dgn_lib, num):
    g = torch.Generator().manual_seed(num)
    counts = torch.randint(0, 1 << 30, (num,), generator=g).int()
    counts[0] = counts.long().sum().item() // num if num > 1 else 5
    bias = normal(num, seed=1)
    total = sum(counts.tolist())
    sign = torch.tensor([(c * num < total) - (c * num > total) for c in counts.tolist()], dtype=torch.float32, device=DEV)
    want = bias + torch.tensor(1e-3, device=DEV) * sign
    out = torch.empty_like(bias)
    assert update_bias(bias, counts.to(DEV), 1e-3, out=out) is out and torch.equal(out, want)
    update_bias(bias, counts.to(DEV), 1e-3)
    assert torch.equal(bias, want)


def test_refusals_on_the_device(dgn_lib):
    logits = torch.ones(4, 8, device=DEV)
    for kwargs in (dict(k=0), dict(k=9), dict(k=2, groups=3), dict(k=2, groups=4, keep_groups=5), dict(k=2, group_best=3),
                   dict(k=2, bias=torch.ones(7, device=DEV)), dict(k=2, bias=torch.ones(8)),
                   dict(k=2, mask=torch.ones(3, dtype=torch.bool, device=DEV))):
        with pytest.raises(ValueError):
            route(logits, **kwargs)
    with pytest.raises(TypeError):
        route(logits, 2, bias=torch.ones(8, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        route(torch.ones(8, 4, device=DEV).t(), 2)
    with pytest.raises(ValueError):
        route(torch.ones(1, 8, device=DEV).expand(4, 8), 2)
    with pytest.raises(ValueError):
        route(torch.ones(2, 1025, device=DEV), 2)
    indices, weights = route(logits, 2)
    with pytest.raises(TypeError):
        route_grad(weights, logits, indices.long())
    with pytest.raises(ValueError):
        route_grad(weights[:3], logits, indices)
    with pytest.raises(ValueError):
        plan(indices, 0)
    with pytest.raises(ValueError):
        plan(indices, 8, align=0)
    p = plan(indices, 8)
    x = torch.ones(4, 16, device=DEV)
    for call in (lambda: dispatch(x[:3], p), lambda: dispatch(x.cpu(), p), lambda: dispatch(x[:, :0], p),
                 lambda: dispatch(x, p, out=torch.empty(8, 15, device=DEV)), lambda: combine(x.t(), p),
                 lambda: combine(x, p, weights[:3]), lambda: combine(x, p, residual=x[:3]),
                 lambda: combine_grad(x[:3], x, p, weights), lambda: combine_grad(x, x, p, weights, out=x[:2]),
                 lambda: update_bias(torch.zeros(4, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV), 0.1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        combine(x.double(), p)
    with pytest.raises(TypeError):
        combine(x, p, residual=x.half())
    with pytest.raises(TypeError):
        dispatch(x, p, out=torch.empty(8, 16, device=DEV, dtype=torch.float16))


def test_a_stream_of_no_use_is_refused(dgn_lib):
    x = torch.ones(4, 8)
    with pytest.raises((ValueError, RuntimeError)):
        route(x, 2, stream=torch.cuda.Stream())


def test_empty_batches(dgn_lib):
    logits = torch.empty(0, 8, device=DEV)
    indices, weights = route(logits, 2)
    assert indices.shape == (0, 2) and route_grad(weights, logits, indices).shape == (0, 8)
    p = plan(indices, 8, 4)
    assert p.capacity == 0 and p.counts.tolist() == [0] * 8 and p.offsets.tolist() == [0] * 9
    x = torch.empty(0, 16, device=DEV)
    rows = dispatch(x, p)
    assert rows.shape == (0, 16) and combine(rows, p, weights).shape == (0, 16)
    assert combine_grad(x, rows, p, weights)[1].shape == (0, 2)
    every = plan(torch.full((5, 2), -1, dtype=torch.int32, device=DEV), 8, 4)  # tokens, but none with an expert
    assert every.counts.sum().item() == 0
    y = combine(torch.empty(0, 16, device=DEV), every, residual=torch.ones(5, 16, device=DEV))
    assert torch.equal(y, torch.ones(5, 16, device=DEV))


def test_streams_and_graphs(dgn_lib):
    tokens, num, k, cols = 3000, 64, 4, 256
    logits, x, dy = normal(tokens, num, seed=1), normal(tokens, cols, seed=2), normal(tokens, cols, seed=3)
    bias = normal(num, seed=4, scale=0.05)

    def all_of_it(**kwargs):
        indices, weights = route(logits, k, bias, **kwargs)
        p = plan(indices, num, **kwargs)
        rows = dispatch(x, p, **kwargs)
        y = combine(rows, p, weights, x, **kwargs)
        grad_rows, grad_weights = combine_grad(dy, rows, p, weights, **kwargs)
        grad_x = dispatch_grad(grad_rows, p, **kwargs)
        grad_logits = route_grad(grad_weights, logits, indices, **kwargs)
        new = update_bias(bias, p.counts, 1e-3, out=torch.empty_like(bias), **kwargs)
        return [indices, weights, p.positions, p.offsets, rows, y, grad_rows, grad_x, grad_logits, new]

    want = all_of_it()
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    # Allocated on the side stream, so that nothing is reused before it is done with it.
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        a = all_of_it(stream=side)
    with torch.cuda.stream(other):
        b = all_of_it(stream=other.cuda_stream)
    torch.cuda.synchronize()
    for got in (a, b):
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(all_of_it())
        graphs.append(graph)
    logits.mul_(-1)
    x.mul_(0.5)
    want = all_of_it()
    torch.cuda.synchronize()
    for graph, stream in zip(graphs, (side, other)):
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_a_layer_of_experts_trains_across_ranks(dgn_lib):
    """Norm, choice, exchange, experts and their backward pass on two virtual ranks, the
    group's token counts and gradients by all-reduce, the fused optimizer's step; against
    autograd over the same layer in 64 bits."""
    from dragon_b200.comm import Communicator
    from dragon_b200.fused_optim import FusedSGD
    from dragon_b200.normalization import rms_norm, rms_norm_grad
    ranks, tokens, cols, num, k, lr, rate = 2, 24, 64, 8, 2, 0.1, 1e-2
    start = {"norm": 1 + normal(cols, seed=1, scale=0.1), "router": normal(num, cols, seed=2, scale=0.3),
             "experts": normal(num, cols, cols, seed=3, scale=0.1)}
    bias0 = normal(num, seed=4, scale=0.1)
    xs = [normal(tokens, cols, seed=10 + r) for r in range(ranks)]
    dys = [normal(tokens, cols, seed=20 + r) for r in range(ranks)]

    # The layer in 64 bits; the choices come from route(), which has tests of its own.
    def oracle(x, dy, params, indices):
        w = {n: v.double().requires_grad_() for n, v in params.items()}
        h = x.double()
        y = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w["norm"]
        s = torch.softmax(y @ w["router"].t(), 1).gather(1, indices.long())
        s = s / (s.sum(1, keepdim=True) + 1e-20)
        out = h + sum(s[:, j:j + 1] * torch.einsum("tc,tcd->td", y, w["experts"][indices[:, j].long()]) for j in range(k))
        return out, torch.autograd.grad(out, list(w.values()), dy.double())

    comms = Communicator.emulated(ranks, 0)
    try:
        params = [{n: v.clone() for n, v in start.items()} for _ in range(ranks)]
        biases = [bias0.clone() for _ in range(ranks)]
        opts = [FusedSGD(list(params[r].values()), lr, comm=comms[r]) for r in range(ranks)]
        plans, want = [], {n: torch.zeros_like(v, dtype=torch.float64) for n, v in start.items()}
        for r in range(ranks):
            w = params[r]
            n = rms_norm(xs[r], w["norm"])
            logits = n.output @ w["router"].t()
            indices, weights = route(logits, k, biases[r])
            p = plan(indices, num, align=4)
            rows = dispatch(n.output, p)
            blocks = [slice(a, b) for a, b in zip(p.offsets.tolist(), p.offsets.tolist()[1:])]
            outputs = torch.zeros_like(rows)
            for e, b in enumerate(blocks):
                outputs[b] = rows[b] @ w["experts"][e]
            y = combine(outputs, p, weights, xs[r])
            grad_outputs, grad_weights = combine_grad(dys[r], outputs, p, weights)
            w["experts"].grad, grad_rows = torch.zeros_like(w["experts"]), torch.zeros_like(rows)
            for e, b in enumerate(blocks):
                w["experts"].grad[e] = rows[b].t() @ grad_outputs[b]
                grad_rows[b] = grad_outputs[b] @ w["experts"][e].t()
            grad_logits = route_grad(grad_weights, logits, indices)
            w["router"].grad = grad_logits.t() @ n.output
            grad_y = dispatch_grad(grad_rows, p) + grad_logits @ w["router"]
            _, w["norm"].grad = rms_norm_grad(grad_y, n.hidden, n.rstd, w["norm"], dys[r])
            plans.append(p)
            out, grads = oracle(xs[r], dys[r], start, indices)
            # Six operators and two products of 64 terms in a row, each within 100 u of its terms' magnitudes.
            assert (y.double() - out).norm() <= 1e-5 * out.norm()
            for (name, total), g in zip(want.items(), grads):
                assert (w[name].grad.double() - g).norm() <= 3e-5 * g.norm(), name
                total += g / ranks
        local = [p.counts.tolist() for p in plans]
        for r in range(ranks):
            comms[r].all_reduce([plans[r].counts])
        for r in range(ranks):
            update_bias(biases[r], plans[r].counts, rate)
        for r in range(ranks):
            opts[r].step()
        torch.cuda.synchronize()
        total = [a + b for a, b in zip(*local)]
        mean = sum(total) / num
        for r in range(ranks):
            assert plans[r].counts.tolist() == total
            moved = ((biases[r] - bias0) / rate).round().tolist()
            assert moved == [float((c < mean) - (c > mean)) for c in total]
            for name in start:
                assert torch.equal(params[0][name], params[r][name])
                step = start[name].double() - params[r][name].double()
                assert (step - lr * want[name]).norm() <= 4e-5 * lr * want[name].norm() + 2 * U * start[name].double().norm()
            assert comms[r].status() == 0
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()


def test_sync_expert_bias(dgn_lib):
    """With a group of one, without a group, outside of one, and where virtual ranks would read too early."""
    from dragon_b200 import distributed
    from dragon_b200.gradient_sync import sync_expert_bias
    distributed.finalize()
    try:
        for group in (distributed.new_group([0]), None):
            p = plan(choices(50, 2, 6, seed=3), 6)
            bias, counts = normal(6, seed=1), p.counts.clone()
            want = update_bias(bias.clone(), counts, 1e-2)
            assert sync_expert_bias(bias, p.counts, 1e-2, group) is bias
            assert torch.equal(bias, want) and torch.equal(p.counts, counts)
        distributed.init_emulated_world(2, 0)
        both, other = distributed.new_group([0, 1]), distributed.new_group([1])
        with distributed.as_rank(0):
            with pytest.raises(RuntimeError, match="virtual ranks"):
                sync_expert_bias(bias, p.counts, 1e-2, both)
            assert torch.equal(sync_expert_bias(bias, p.counts, 1e-2, other), want)  # not a member
    finally:
        torch.cuda.synchronize()
        distributed.finalize()


def test_a_device_that_does_not_exist_is_an_error(dgn_lib):
    from dragon_b200 import _C
    bias, counts = torch.zeros(4, device=DEV), torch.ones(4, dtype=torch.int32, device=DEV)
    args = (bias.data_ptr(), counts.data_ptr(), bias.data_ptr(), 4, 0.5)
    assert dgn_lib.dgn_expert_update_bias(*args, 4096, None) == _C.ERR_CUDA
    assert dgn_lib.dgn_last_error_string()
    assert torch.equal(update_bias(bias, counts, 0.5), torch.zeros(4, device=DEV))  # and nothing of it stays behind


def test_eight_bit_rows_travel(dgn_lib):
    """The norm's 8-bit rows and scales through all-gather and dispatch stand for the same values."""
    from dragon_b200.comm import Communicator
    from dragon_b200.normalization import rms_norm
    comms = Communicator.emulated(2, 0)
    try:
        norms = [rms_norm(normal(32, 256, seed=r, dtype=torch.bfloat16), out_dtype=torch.float8_e4m3fn, group_size=128)
                 for r in range(2)]
        codes = [torch.empty(64, 256, dtype=torch.uint8, device=DEV) for _ in range(2)]
        scales = [torch.empty(64, 2, device=DEV) for _ in range(2)]
        for c, n, out in zip(comms, norms, codes):
            c.all_gather(n.output.view(torch.uint8), out)
        for c, n, out in zip(comms, norms, scales):
            c.all_gather(n.scale, out)
        torch.cuda.synchronize()
        value = lambda q, s: q.view(torch.float8_e4m3fn).float() * s.repeat_interleave(128, 1)  # noqa: E731
        want = torch.cat([value(n.output, n.scale) for n in norms])
        assert all(torch.equal(value(q, s), want) for q, s in zip(codes, scales))
        p = plan(choices(64, 2, 4, missing=0.0), 4)
        rows = value(dispatch(codes[0], p), dispatch(scales[0], p))
        assert torch.equal(rows[p.positions.long()], want[:, None].expand(64, 2, 256))
    finally:
        torch.cuda.synchronize()
        for c in comms:
            c.destroy()


def test_module_limits_match_the_library(dgn_lib):
    assert (experts.MAX_EXPERTS, experts.MAX_CHOICES, experts.MAX_GROUPS) == (1024, 32, 32)

"""Operators of a layer of experts on torch CUDA tensors (dgn_route and
dgn_expert_* of include/dgn.h).

    indices, weights = route(logits, k, bias, mask)       # each token's experts
    p = plan(indices, num_experts)                        # where its rows go
    rows = dispatch(x, p)                                 # rows in the order of the experts
    ...                                                   # expert e: rows[p.offsets[e]:p.offsets[e] + p.counts[e]]
    y = combine(outputs, p, weights, residual)            # the weighted sum back

    grad_outputs, grad_weights = combine_grad(grad_y, outputs, p, weights)
    grad_x = dispatch_grad(grad_rows, p)
    grad_logits = route_grad(grad_weights, logits, indices)

    comm.all_reduce([p.counts])                           # the group's token counts
    update_bias(bias, p.counts, rate)                     # the same new bias on every rank

Like the collectives these calls enqueue work on a stream and return: nothing
is synchronised, so the number of rows of each expert stays on the device, and
no autograd graph is recorded, the backward pass is the ``_grad`` calls.
"""

import torch

from dragon_b200 import _C
from dragon_b200.comm import _TORCH_TO_DGN, _enter_stream, _raw_stream

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_SCORES = {"softmax": _C.SCORE_SOFTMAX, "sigmoid": _C.SCORE_SIGMOID}
MAX_EXPERTS, MAX_CHOICES, MAX_GROUPS = 1024, 32, 32


def _matrix(t, name, dtypes=_FLOATS):
    """Row stride of a CUDA matrix with contiguous rows that do not overlap."""
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError("Unsupported data type of <{}>: {}".format(name, t.dtype))
    if t.dim() != 2:
        raise ValueError("<{}> must have two dimensions".format(name))
    if not t.is_cuda:
        raise ValueError("<{}> must be a CUDA tensor (got {})".format(name, t.device))
    rows, cols = t.shape
    if cols > 1 and t.stride(1) != 1:
        raise ValueError("the rows of <{}> must be contiguous".format(name))
    if rows < 2:
        return cols
    if t.stride(0) < cols:
        raise ValueError("the rows of <{}> must not overlap".format(name))
    return t.stride(0)


def _exactly(t, name, device, shape, dtypes):
    """Checks a contiguous tensor of one device, shape and type."""
    if t.dtype not in dtypes:
        raise TypeError("Unsupported data type of <{}>: {}".format(name, t.dtype))
    if t.device != device:
        raise ValueError("<{}> must live on {} (got {})".format(name, device, t.device))
    if tuple(t.shape) != tuple(shape):
        raise ValueError("<{}> must have the shape {}, got {}".format(name, tuple(shape), tuple(t.shape)))
    if not t.is_contiguous():
        raise ValueError("<{}> must be contiguous".format(name))


def _score_code(scores):
    code = _SCORES.get(scores)
    if code is None:
        raise ValueError("Unsupported scores: {}".format(scores))
    return code


def _check_choice(k, experts):
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError("there must be 1 to {} experts, got {}".format(MAX_EXPERTS, experts))
    if not 1 <= k <= min(MAX_CHOICES, experts):
        raise ValueError("<k> must be 1 to {} and at most the number of experts, got {}".format(MAX_CHOICES, k))


def route(logits, k, bias=None, mask=None, scores="softmax", groups=1, keep_groups=1, group_best=1, renormalize=True,
          scale=1.0, stream=None):
    """Each token's k experts and their weights: (indices int32 [tokens, k], weights float32 [tokens, k]).

    logits: [tokens, experts], float16, bfloat16 or float32, up to 1024 experts.
    scores: "softmax" or "sigmoid" of the logits.  Experts are chosen by the
    logits, or by score + bias where a bias (float32 [experts]) is given; the
    weights are the scores without it, divided by their sum if `renormalize`, times
    `scale`.  groups > 1: the experts lie in equal runs, and only those of the
    `keep_groups` best runs count, a run's value being the sum of its best
    `group_best` (1 or 2) members.  Equal experts are taken in their order, and
    choices are made as if computed in 64 bits, so that every rank and every
    recomputation makes the same ones.

    An expert whose logit is -inf is never chosen, a NaN first.  mask (bool
    [tokens]): tokens where it is False, and slots that find no expert, get index
    -1 and weight 0; the other calls of this module pass over them."""
    if stream is not None:
        with _enter_stream(stream, logits.device):
            return route(logits, k, bias, mask, scores, groups, keep_groups, group_best, renormalize, scale)
    code = _score_code(scores)
    stride = _matrix(logits, "logits")
    tokens, experts = logits.shape
    _check_choice(k, experts)
    if not 1 <= groups <= MAX_GROUPS or experts % groups:
        raise ValueError("<groups> must be 1 to {} and divide the number of experts".format(MAX_GROUPS))
    if not 1 <= keep_groups <= groups:
        raise ValueError("<keep_groups> must be 1 to <groups>, got {}".format(keep_groups))
    if group_best not in (1, 2):
        raise ValueError("<group_best> must be 1 or 2, got {}".format(group_best))
    device = logits.device
    if bias is not None:
        _exactly(bias, "bias", device, (experts,), (torch.float32,))
    if mask is not None:
        _exactly(mask, "mask", device, (tokens,), (torch.bool,))
    indices = torch.empty((tokens, k), dtype=torch.int32, device=device)
    weights = torch.empty((tokens, k), dtype=torch.float32, device=device)
    rc = _C.lib().dgn_route(
        logits.data_ptr(), stride, bias.data_ptr() if bias is not None else None,
        mask.data_ptr() if mask is not None else None, indices.data_ptr(), weights.data_ptr(), tokens, experts, k, code,
        groups, keep_groups, group_best, bool(renormalize), scale, _TORCH_TO_DGN[logits.dtype], device.index,
        _raw_stream(device.index))
    if rc != _C.OK:
        _C.check(rc)
    return indices, weights


def route_grad(grad_weights, logits, indices, scores="softmax", renormalize=True, scale=1.0, stream=None):
    """Gradient of the logits (contiguous, in their type) from that of route()'s weights, for the same arguments."""
    if stream is not None:
        with _enter_stream(stream, logits.device):
            return route_grad(grad_weights, logits, indices, scores, renormalize, scale)
    code = _score_code(scores)
    stride = _matrix(logits, "logits")
    tokens, experts = logits.shape
    device = logits.device
    if indices.dim() != 2:
        raise ValueError("<indices> must have two dimensions")
    k = indices.shape[1]
    _check_choice(k, experts)
    _exactly(indices, "indices", device, (tokens, k), (torch.int32,))
    _exactly(grad_weights, "grad_weights", device, (tokens, k), (torch.float32,))
    grad = torch.empty((tokens, experts), dtype=logits.dtype, device=device)
    rc = _C.lib().dgn_route_grad(
        grad_weights.data_ptr(), logits.data_ptr(), stride, indices.data_ptr(), grad.data_ptr(), tokens, experts, k, code,
        bool(renormalize), scale, _TORCH_TO_DGN[logits.dtype], device.index, _raw_stream(device.index))
    if rc != _C.OK:
        _C.check(rc)
    return grad


class ExpertPlan(object):
    """Where the rows of a batch go, all on the device (int32):

    counts [experts], the rows of each expert; offsets [experts + 1], the first
    row of each expert's block, a multiple of `align`, and the end of the last;
    positions [tokens, k], the row of each choice, -1 for none.  `capacity` is the
    number of rows that always suffices."""

    def __init__(self, counts, offsets, positions, align):
        self.counts, self.offsets, self.positions, self.align = counts, offsets, positions, align
        self.tokens, self.k = positions.shape
        self.num_experts = counts.shape[0]
        slots = self.tokens * self.k
        self.capacity = slots + min(self.num_experts, slots) * (align - 1)


def plan(indices, num_experts, align=1, stream=None):
    """Counting sort of the (token, choice) pairs by expert, equal ones in their order.

    indices: int32 [tokens, k] as from route(); values outside 0..num_experts-1
    take no part.  align: each expert's block starts at a multiple of it."""
    if stream is not None:
        with _enter_stream(stream, indices.device):
            return plan(indices, num_experts, align)
    _matrix(indices, "indices", (torch.int32,))
    if not indices.is_contiguous():
        raise ValueError("<indices> must be contiguous")
    tokens, k = indices.shape
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError("there must be 1 to {} experts, got {}".format(MAX_EXPERTS, num_experts))
    if not 1 <= k <= MAX_CHOICES:
        raise ValueError("a token has 1 to {} choices, got {}".format(MAX_CHOICES, k))
    slots = tokens * k
    if align < 1 or slots + min(num_experts, slots) * (align - 1) >= 1 << 31:
        raise ValueError("<align> must be positive and the rows fewer than 2^31")
    device = indices.device
    counts = torch.empty(num_experts, dtype=torch.int32, device=device)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    positions = torch.empty((tokens, k), dtype=torch.int32, device=device)
    lib = _C.lib()
    nbytes = lib.dgn_expert_plan_workspace(slots, num_experts)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    rc = lib.dgn_expert_plan(indices.data_ptr(), slots, num_experts, align, counts.data_ptr(), offsets.data_ptr(),
                             positions.data_ptr(), workspace.data_ptr() if nbytes else None, nbytes, device.index,
                             _raw_stream(device.index))
    if rc != _C.OK:
        _C.check(rc)
    return ExpertPlan(counts, offsets, positions, align)


def _buffer(out, name, p, cols, dtype, device):
    """The caller's rows, or new ones; any number of rows, those that do not exist are not written."""
    if out is None:
        return torch.empty((p.capacity, cols), dtype=dtype, device=device)
    if out.dim() != 2:
        raise ValueError("<{}> must have two dimensions".format(name))
    _exactly(out, name, device, (out.shape[0], cols), (dtype,))
    return out


def _check_plan(p, device):
    if p.positions.device != device:
        raise ValueError("the plan must live on {} (got {})".format(device, p.positions.device))


def dispatch(x, plan, out=None, stream=None):
    """Rows in the order of the experts: out[plan.positions[t, j]] = x[t].

    x: [tokens, columns] of any type (8-bit codes and their scales are two calls
    with one plan).  out: [rows, columns], by default new with plan.capacity rows; a
    shorter one takes the rows that it has.  The unused rows of an expert's block
    become zeros, rows behind the last block stay as they are."""
    if stream is not None:
        with _enter_stream(stream, x.device):
            return dispatch(x, plan, out)
    stride = _matrix(x, "x", None)
    tokens, cols = x.shape
    _check_plan(plan, x.device)
    if tokens != plan.tokens:
        raise ValueError("<x> must have the plan's {} rows, got {}".format(plan.tokens, tokens))
    if cols == 0:
        raise ValueError("<x> has no columns")
    out = _buffer(out, "out", plan, cols, x.dtype, x.device)
    size = x.element_size()
    rc = _C.lib().dgn_expert_dispatch(
        x.data_ptr(), stride * size, cols * size, plan.positions.data_ptr(), plan.counts.data_ptr(),
        plan.offsets.data_ptr(), out.data_ptr(), tokens, plan.k, plan.num_experts, out.shape[0], x.device.index,
        _raw_stream(x.device.index))
    if rc != _C.OK:
        _C.check(rc)
    return out


def combine(rows, plan, weights=None, residual=None, stream=None):
    """Weighted sum of each token's rows: residual[t] + sum_j weights[t, j] * rows[plan.positions[t, j]].

    rows: [rows, columns], float16, bfloat16 or float32.  weights: float32
    [tokens, k], or None for ones.  residual: [tokens, columns] of the rows' type.
    Sums are held in float32 and rounded once."""
    if stream is not None:
        with _enter_stream(stream, rows.device):
            return combine(rows, plan, weights, residual)
    _matrix(rows, "rows")
    if not rows.is_contiguous():
        raise ValueError("<rows> must be contiguous")
    capacity, cols = rows.shape
    device = rows.device
    _check_plan(plan, device)
    if cols == 0:
        raise ValueError("<rows> has no columns")
    if weights is not None:
        _exactly(weights, "weights", device, (plan.tokens, plan.k), (torch.float32,))
    residual_stride = 0
    if residual is not None:
        residual_stride = _matrix(residual, "residual", (rows.dtype,))
        if residual.device != device or tuple(residual.shape) != (plan.tokens, cols):
            raise ValueError("<residual> must be of {} and have the shape {}".format(device, (plan.tokens, cols)))
    out = torch.empty((plan.tokens, cols), dtype=rows.dtype, device=device)
    rc = _C.lib().dgn_expert_combine(
        rows.data_ptr(), plan.positions.data_ptr(), weights.data_ptr() if weights is not None else None,
        residual.data_ptr() if residual is not None else None, residual_stride, out.data_ptr(), plan.tokens, plan.k, cols,
        capacity, _TORCH_TO_DGN[rows.dtype], device.index, _raw_stream(device.index))
    if rc != _C.OK:
        _C.check(rc)
    return out


def dispatch_grad(grad_rows, plan, stream=None):
    """Gradient of dispatch()'s x: the sum of the gradients of each token's rows."""
    return combine(grad_rows, plan, stream=stream)


def combine_grad(grad_output, rows, plan, weights, out=None, stream=None):
    """Backward pass of combine: (grad_rows [rows, columns], grad_weights float32 [tokens, k]).

    grad_rows is laid out as dispatch() lays its rows out (`out` likewise).  The
    residual's gradient is grad_output itself; without weights the rows' gradient
    is dispatch(grad_output, plan)."""
    if stream is not None:
        with _enter_stream(stream, rows.device):
            return combine_grad(grad_output, rows, plan, weights, out)
    _matrix(rows, "rows")
    if not rows.is_contiguous():
        raise ValueError("<rows> must be contiguous")
    capacity, cols = rows.shape
    device = rows.device
    _check_plan(plan, device)
    if cols == 0:
        raise ValueError("<rows> has no columns")
    stride = _matrix(grad_output, "grad_output", (rows.dtype,))
    if grad_output.device != device or tuple(grad_output.shape) != (plan.tokens, cols):
        raise ValueError("<grad_output> must be of {} and have the shape {}".format(device, (plan.tokens, cols)))
    _exactly(weights, "weights", device, (plan.tokens, plan.k), (torch.float32,))
    if out is None:
        out = torch.empty_like(rows)
    _exactly(out, "out", device, (capacity, cols), (rows.dtype,))
    grad_weights = torch.empty_like(weights)
    rc = _C.lib().dgn_expert_combine_grad(
        grad_output.data_ptr(), stride, rows.data_ptr(), plan.positions.data_ptr(), weights.data_ptr(),
        plan.counts.data_ptr(), plan.offsets.data_ptr(), out.data_ptr(), grad_weights.data_ptr(), plan.tokens, plan.k,
        plan.num_experts, cols, capacity, _TORCH_TO_DGN[rows.dtype], device.index, _raw_stream(device.index))
    if rc != _C.OK:
        _C.check(rc)
    return out, grad_weights


def update_bias(bias, counts, rate, out=None, stream=None):
    """bias + rate * sign(mean(counts) - counts), in place unless `out` is given.

    counts: int32 [experts], the tokens that each expert had in the whole group: the
    sum over the ranks of plan().counts, by an all-reduce."""
    if stream is not None:
        with _enter_stream(stream, bias.device):
            return update_bias(bias, counts, rate, out)
    if bias.dim() != 1 or not 1 <= bias.shape[0] <= MAX_EXPERTS:
        raise ValueError("<bias> must be a vector of 1 to {} elements".format(MAX_EXPERTS))
    if not bias.is_cuda:
        raise ValueError("<bias> must be a CUDA tensor (got {})".format(bias.device))
    _exactly(bias, "bias", bias.device, bias.shape, (torch.float32,))
    _exactly(counts, "counts", bias.device, bias.shape, (torch.int32,))
    if out is None:
        out = bias
    _exactly(out, "out", bias.device, bias.shape, (torch.float32,))
    rc = _C.lib().dgn_expert_update_bias(bias.data_ptr(), counts.data_ptr(), out.data_ptr(), bias.shape[0], rate,
                                         bias.device.index, _raw_stream(bias.device.index))
    if rc != _C.OK:
        _C.check(rc)
    return out

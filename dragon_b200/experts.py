"""Operators of a layer of experts on torch CUDA tensors (dgn_route and
dgn_expert_* of include/dgn.h).

    indices, weights = route(logits, k, bias, mask)       # each token's experts
    p = plan(indices, num_experts)                        # where its rows go
    rows = dispatch(x, p)                                 # rows in the order of the experts
    ...                                                   # expert e: rows[p.offsets[e]:p.ends[e]]
    y = combine(outputs, p, weights, residual)            # the weighted sum back

    grad_outputs, grad_weights = combine_grad(grad_y, outputs, p, weights)
    grad_x = dispatch_grad(grad_rows, p)
    grad_logits = route_grad(grad_weights, logits, indices)

    gradient_sync.sync_expert_bias(bias, p.counts, rate)  # the group's counts, the same new bias on every rank

Like the collectives these calls enqueue work on a stream and return: nothing
is synchronised, so the number of rows of each expert stays on the device, and
no autograd graph is recorded, the backward pass is the ``_grad`` calls (a
process that passes tensors which require gradients, with gradients enabled, is
warned once).
"""

from dragon_b200 import _C
from dragon_b200.comm import _enter_stream

_SCORES = {"softmax": _C.SCORE_SOFTMAX, "sigmoid": _C.SCORE_SIGMOID}
MAX_EXPERTS, MAX_CHOICES, MAX_GROUPS = 1024, 32, 32  # the DGN_MAX_ of include/dgn.h, for callers that size a model


def _score_code(scores):
    code = _SCORES.get(scores)
    if code is None:
        raise ValueError("Unsupported scores: {}".format(scores))
    return code


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
    return _C.torch_ops().route(logits, k, bias, mask, _score_code(scores), groups, keep_groups, group_best, renormalize,
                                scale)


def route_grad(grad_weights, logits, indices, scores="softmax", renormalize=True, scale=1.0, stream=None):
    """Gradient of the logits (contiguous, in their type) from that of route()'s weights, for the same arguments."""
    if stream is not None:
        with _enter_stream(stream, logits.device):
            return route_grad(grad_weights, logits, indices, scores, renormalize, scale)
    return _C.torch_ops().route_grad(grad_weights, logits, indices, _score_code(scores), renormalize, scale)


class ExpertPlan(object):
    """Where the rows of a batch go, all on the device (int32):

    counts [experts], the rows of each expert (the caller's to change: an
    all-reduce may add up the group's in place); offsets [experts + 1], the first
    row of each expert's block, a multiple of `align`, and the end of the last;
    ends [experts], behind the last row in use of each block; positions [tokens, k],
    the row of each choice, -1 for none.  `capacity` is the number of rows that
    always suffices."""

    def __init__(self, counts, offsets, ends, positions, align):
        self.counts, self.offsets, self.ends, self.positions, self.align = counts, offsets, ends, positions, align
        self.tokens, self.k = positions.shape
        self.num_experts = ends.shape[0]
        slots = self.tokens * self.k
        self.capacity = slots + min(self.num_experts, slots) * (align - 1)


def plan(indices, num_experts, align=1, stream=None):
    """Counting sort of the (token, choice) pairs by expert, equal ones in their order.

    indices: int32 [tokens, k] as from route(); values outside 0..num_experts-1
    take no part.  align: each expert's block starts at a multiple of it."""
    if stream is not None:
        with _enter_stream(stream, indices.device):
            return plan(indices, num_experts, align)
    return ExpertPlan(*_C.torch_ops().plan(indices, num_experts, align), align)


def dispatch(x, plan, out=None, stream=None):
    """Rows in the order of the experts: out[plan.positions[t, j]] = x[t].

    x: [tokens, columns] of any type (8-bit codes and their scales are two calls
    with one plan).  out: [rows, columns], by default new with plan.capacity rows; a
    shorter one takes the rows that it has.  The unused rows of an expert's block
    become zeros, rows behind the last block stay as they are: in a new tensor
    whatever its memory held."""
    if stream is not None:
        with _enter_stream(stream, x.device):
            return dispatch(x, plan, out)
    return _C.torch_ops().dispatch(x, plan.offsets, plan.ends, plan.positions, plan.capacity, out)


def combine(rows, plan, weights=None, residual=None, stream=None):
    """Weighted sum of each token's rows: residual[t] + sum_j weights[t, j] * rows[plan.positions[t, j]].

    rows: [rows, columns], float16, bfloat16 or float32.  weights: float32
    [tokens, k], or None for ones.  residual: [tokens, columns] of the rows' type.
    Sums are held in float32 and rounded once."""
    if stream is not None:
        with _enter_stream(stream, rows.device):
            return combine(rows, plan, weights, residual)
    return _C.torch_ops().combine(rows, plan.offsets, plan.ends, plan.positions, weights, residual)


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
    return _C.torch_ops().combine_grad(grad_output, rows, plan.offsets, plan.ends, plan.positions, weights, out)


def update_bias(bias, counts, rate, out=None, stream=None):
    """bias + rate * sign(mean(counts) - counts), in place unless `out` is given.

    counts: int32 [experts], the tokens that each expert had in the whole group: the
    sum over the ranks of plan().counts, by an all-reduce."""
    if stream is not None:
        with _enter_stream(stream, bias.device):
            return update_bias(bias, counts, rate, out)
    return _C.torch_ops().update_bias(bias, counts, rate, out)

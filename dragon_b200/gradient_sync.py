"""What a data-parallel training step synchronises, as functions over torch CUDA
tensors: the two gradient-sync call sites of the reference, and the balance
bias of a layer of experts.

* torch frontend, ``Optimizer.step`` (torch/core/optim/optimizer.py:134-164,
  261-262): gradients are grouped by dtype, each group is all-reduced in place
  with ``reduction="SUM"`` and ``bucket_size`` (512 MiB by default), and the
  division by the group size is folded into the update's ``grad_scale``.
* native optimizers, ``apply_gradients``
  (dragon/python/core/training/optimizer.py:70-81): all gradients go through
  one ``Collective`` with ``reduction="MEAN"`` and no bucketing (one collective
  per tensor in the reference; still one operator run here).

They return without synchronising; the gradients are reduced in place.
"""

import collections

from dragon_b200 import experts
from dragon_b200.distributed import backend as dist_backend
from dragon_b200.distributed.ops import _execute


def sync_gradients_torch_style(grads, bucket_size=512 * 1024 * 1024, group=None):
    """SUM all-reduce per dtype, bucketed.  Returns the factor the caller folds
    into ``grad_scale`` (1 / group size, or 1.0 without a group)."""
    group = group or dist_backend.get_group()
    if group is None:
        return 1.0
    by_dtype = collections.defaultdict(list)
    for g in grads:
        if g is not None:
            by_dtype[g.dtype].append(g)
    for same in by_dtype.values():
        _execute(group, same, outputs=same, operation="ALLREDUCE", reduction="SUM", bucket_size=bucket_size)
    return 1.0 / group.size


def sync_gradients_native_style(grads, group=None):
    """MEAN all-reduce of every gradient, in place, unbucketed."""
    group = group or dist_backend.get_group()
    if group is None:
        return
    grads = [g for g in grads if g is not None]
    if grads:
        _execute(group, grads, outputs=grads, operation="ALLREDUCE", reduction="MEAN")


def sync_expert_bias(bias, counts, rate, group=None):
    """One step of the balance bias of experts.route(): the ranks' token counts
    (experts.plan().counts, int32) are summed in place by an all-reduce, and
    ``bias`` moves by ``rate`` towards the experts that had fewer than the mean, in
    place and to the same bits on every rank.  Without a group the counts are this
    process's own; a rank outside of the group leaves both alone.

    Virtual ranks of an emulated world (a collective runs when the last of them
    issues it) all-reduce first, each of them, and then call experts.update_bias."""
    group = group or dist_backend.get_group()
    if group is not None:
        if dist_backend.communicator(group) is None:
            return bias
        if group.size > 1 and isinstance(dist_backend._world(), dist_backend._EmulatedWorld):
            raise RuntimeError("virtual ranks all-reduce their counts before any of them updates its bias")
        _execute(group, [counts], outputs=[counts], operation="ALLREDUCE", reduction="SUM")
    return experts.update_bias(bias, counts, rate)

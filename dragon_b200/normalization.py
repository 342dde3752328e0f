"""Root-mean-square norm with the residual's addition, and its backward pass, on
torch CUDA tensors (dgn_rms_norm and dgn_rms_norm_grad of include/dgn.h).

Beside the statistics exchange of synchronized batch normalization
(op_lib.run_sync_bn_stats) this is the norm of a transformer's layers.  Its
8-bit output and the scales are ordinary tensors: the all-gather of
activations moves them at half the bytes of bfloat16
(``comm.all_gather(r.output.view(torch.uint8), ...)``).

Like the collectives these calls enqueue work on a stream and return; no
autograd graph is recorded, the backward pass is the ``_grad`` call (a process
that passes tensors which require gradients, with gradients enabled, is warned once).
"""

import collections

from dragon_b200 import _C
from dragon_b200.comm import _enter_stream

RMSNorm = collections.namedtuple("RMSNorm", ["output", "hidden", "rstd", "scale"])


def rms_norm(x, weight=None, residual=None, eps=1e-6, out_dtype=None, group_size=0, inplace_residual=False,
             stream=None):
    """hidden = x + residual; output = hidden / sqrt(mean(hidden^2) + eps) * weight, over the last dimension.

    x, residual: float16, bfloat16 or float32, rows at one distance (a slice of
    columns will do), 1 to 32768 columns.  weight: float32 or of x's type, or
    None.  `hidden` is rounded to x's type and is what the backward pass takes;
    without a residual it is x itself, with `inplace_residual` the residual's own
    memory.  out_dtype: None for x's type, or torch.int8, torch.float8_e4m3fn or
    torch.float8_e5m2: then output * scale stands for the value, with one float32
    scale per row and `group_size` columns (32, 64, 128, or 0 for the row).

    The sum of a row's squares is held in float32: rows where it passes 3.4e38
    (4096 columns of 2.9e17 each) come out as zeros, with rstd 0.

    Returns RMSNorm(output, hidden, rstd, scale)."""
    if stream is not None:
        with _enter_stream(stream, x.device):
            return rms_norm(x, weight, residual, eps, out_dtype, group_size, inplace_residual)
    return RMSNorm._make(_C.torch_ops().rms_norm(x, weight, residual, eps, out_dtype, group_size, inplace_residual))


def rms_norm_grad(grad_output, hidden, rstd, weight=None, grad_hidden=None, stream=None):
    """Backward pass of rms_norm: (grad_x, grad_weight).

    hidden, rstd: from the forward call.  grad_output has hidden's type (an
    8-bit output passes its gradient straight through).  grad_hidden: the
    gradient that reaches `hidden` along the residual, or None.  grad_x is the
    gradient of x and of the residual alike; grad_weight has the weight's type
    and is None without a weight.  The same inputs in the same layout give
    the same bits."""
    if stream is not None:
        with _enter_stream(stream, hidden.device):
            return rms_norm_grad(grad_output, hidden, rstd, weight, grad_hidden)
    return _C.torch_ops().rms_norm_grad(grad_output, hidden, rstd, weight, grad_hidden)

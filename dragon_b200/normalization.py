"""Root-mean-square norm with the residual's addition, and its backward pass, on
torch CUDA tensors (dgn_rms_norm and dgn_rms_norm_grad of include/dgn.h).

Beside the statistics exchange of synchronized batch normalization
(op_lib.run_sync_bn_stats) this is the norm of a transformer's layers.  Its
8-bit output and the scales are ordinary tensors: the all-gather of
activations moves them at half the bytes of bfloat16
(``comm.all_gather(r.output.view(torch.uint8), ...)``).

Like the collectives these calls enqueue work on a stream and return; no
autograd graph is recorded, the backward pass is the ``_grad`` call.
"""

import collections

import torch

from dragon_b200 import _C
from dragon_b200.comm import _TORCH_TO_DGN, _enter_stream, _raw_stream

RMSNorm = collections.namedtuple("RMSNorm", ["output", "hidden", "rstd", "scale"])

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_CODES = {torch.int8: _C.CODE_I8, torch.float8_e4m3fn: _C.CODE_E4M3, torch.float8_e5m2: _C.CODE_E5M2}
_GROUPS = (0, 32, 64, 128)


def _rows(t, name):
    """(rows, columns, stride) of a tensor of rows that lie at one distance."""
    if t.dim() == 0:
        raise ValueError("<{}> needs at least one dimension.".format(name))
    cols = t.shape[-1]
    if t.is_contiguous():
        return t.numel() // cols if cols else 0, cols, cols
    if t.stride(-1) != 1 and cols > 1:
        raise ValueError("the last dimension of <{}> must be contiguous".format(name))
    stride, span = None, 1
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = step
        elif step != stride * span:
            raise ValueError("the rows of <{}> must lie at one distance".format(name))
        span *= size
    if stride is None:
        stride = cols
    if stride < cols:
        raise ValueError("the rows of <{}> must not overlap".format(name))
    return span, cols, stride


def _like(t, x, name, dtypes=None):
    """Checks that `t` is a CUDA tensor of x's device, shape and type (or one of `dtypes`)."""
    if t.device != x.device:
        raise ValueError("<{}> must live on {} (got {})".format(name, x.device, t.device))
    if t.shape != x.shape:
        raise ValueError("<{}> must have the shape {}".format(name, tuple(x.shape)))
    if t.dtype not in (dtypes or (x.dtype,)):
        raise TypeError("Unsupported data type of <{}>: {}".format(name, t.dtype))


def _check_input(x, name):
    if x.dtype not in _FLOATS:
        raise TypeError("Unsupported data type: {}".format(x.dtype))
    if not x.is_cuda:
        raise ValueError("<{}> must be a CUDA tensor (got {})".format(name, x.device))


def _check_weight(weight, x, cols):
    if weight.dtype != x.dtype and weight.dtype != torch.float32:
        raise TypeError("<weight> must be float32 or {}, got {}".format(x.dtype, weight.dtype))
    if weight.device != x.device:
        raise ValueError("<weight> must live on {} (got {})".format(x.device, weight.device))
    if weight.dim() != 1 or weight.shape[0] != cols or not weight.is_contiguous():
        raise ValueError("<weight> must be a contiguous vector of {} elements".format(cols))


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

    Returns RMSNorm(output, hidden, rstd, scale)."""
    if stream is not None:
        with _enter_stream(stream, x.device):
            return rms_norm(x, weight, residual, eps, out_dtype, group_size, inplace_residual)
    _check_input(x, "x")
    rows, cols, stride = _rows(x, "x")
    if not 0 < eps < float("inf"):
        raise ValueError("<eps> must be a positive number, got {}".format(eps))
    if group_size not in _GROUPS:
        raise ValueError("<group_size> must be one of {}, got {}".format(_GROUPS, group_size))
    code = _C.CODE_NONE
    if out_dtype is not None and out_dtype != x.dtype:
        code = _CODES.get(out_dtype)
        if code is None:
            raise TypeError("Unsupported output type: {}".format(out_dtype))
    dtype = _TORCH_TO_DGN[x.dtype]
    weight_dtype = dtype
    if weight is not None:
        _check_weight(weight, x, cols)
        weight_dtype = _TORCH_TO_DGN[weight.dtype]
    hidden, residual_stride, hidden_stride = x, 0, 0
    if residual is not None:
        _like(residual, x, "residual")
        _, _, residual_stride = _rows(residual, "residual")
        if inplace_residual:
            hidden, hidden_stride = residual, residual_stride
        else:
            hidden, hidden_stride = torch.empty(x.shape, dtype=x.dtype, device=x.device), cols
    elif inplace_residual:
        raise ValueError("<inplace_residual> needs a residual")
    output = torch.empty(x.shape, dtype=out_dtype if code else x.dtype, device=x.device)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    scale = None
    if code:
        groups = -(-cols // group_size) if group_size else 1
        scale = torch.empty(x.shape[:-1] + (groups,), dtype=torch.float32, device=x.device)
    rc = _C.lib().dgn_rms_norm(
        x.data_ptr(), stride, residual.data_ptr() if residual is not None else None, residual_stride,
        weight.data_ptr() if weight is not None else None, weight_dtype,
        hidden.data_ptr() if residual is not None else None, hidden_stride, output.data_ptr(), code, group_size,
        scale.data_ptr() if code else None, rstd.data_ptr(), rows, cols, eps, dtype, x.device.index,
        _raw_stream(x.device.index))
    if rc != _C.OK:
        _C.check(rc)
    return RMSNorm(output, hidden, rstd, scale)


def rms_norm_grad(grad_output, hidden, rstd, weight=None, grad_hidden=None, stream=None):
    """Backward pass of rms_norm: (grad_x, grad_weight).

    hidden, rstd: from the forward call.  grad_output has hidden's type (an
    8-bit output passes its gradient straight through).  grad_hidden: the
    gradient that reaches `hidden` along the residual, or None.  grad_x is the
    gradient of x and of the residual alike; grad_weight has the weight's type
    and is None without a weight.  The same inputs give the same bits."""
    if stream is not None:
        with _enter_stream(stream, hidden.device):
            return rms_norm_grad(grad_output, hidden, rstd, weight, grad_hidden)
    _check_input(hidden, "hidden")
    rows, cols, hidden_stride = _rows(hidden, "hidden")
    _like(grad_output, hidden, "grad_output")
    _, _, grad_stride = _rows(grad_output, "grad_output")
    if rstd.device != hidden.device or rstd.dtype != torch.float32 or rstd.numel() != rows or not rstd.is_contiguous():
        raise ValueError("<rstd> must be the forward call's")
    dtype = _TORCH_TO_DGN[hidden.dtype]
    weight_dtype, grad_hidden_stride = dtype, 0
    if grad_hidden is not None:
        _like(grad_hidden, hidden, "grad_hidden")
        _, _, grad_hidden_stride = _rows(grad_hidden, "grad_hidden")
    lib = _C.lib()
    grad_weight, workspace, nbytes = None, None, 0
    if weight is not None:
        _check_weight(weight, hidden, cols)
        weight_dtype = _TORCH_TO_DGN[weight.dtype]
        grad_weight = torch.empty_like(weight)
        nbytes = lib.dgn_rms_norm_grad_workspace(rows, cols, dtype)
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=hidden.device)
    grad_x = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device)
    rc = lib.dgn_rms_norm_grad(
        grad_output.data_ptr(), grad_stride, grad_hidden.data_ptr() if grad_hidden is not None else None,
        grad_hidden_stride, hidden.data_ptr(), hidden_stride, weight.data_ptr() if weight is not None else None,
        weight_dtype, rstd.data_ptr(), grad_x.data_ptr(), grad_weight.data_ptr() if weight is not None else None,
        workspace.data_ptr() if weight is not None else None, nbytes, rows, cols, dtype, hidden.device.index,
        _raw_stream(hidden.device.index))
    if rc != _C.OK:
        _C.check(rc)
    return grad_x, grad_weight

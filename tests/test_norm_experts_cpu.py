"""Refusals of the norm and expert operators, and their argument checks at the
C-ABI: none of them reaches a device."""

import ctypes

import pytest
import torch

from dragon_b200 import _C, experts
from dragon_b200.normalization import rms_norm, rms_norm_grad

P = 1 << 20  # an aligned address that is never read: every call below is refused first


def test_python_refuses_what_is_not_on_a_gpu_or_not_a_float():
    x = torch.ones(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm(x)
    with pytest.raises(TypeError, match="float64"):
        rms_norm(x.double())
    with pytest.raises(ValueError, match="CUDA"):
        rms_norm_grad(x, x, torch.ones(4))
    with pytest.raises(ValueError, match="CUDA"):
        experts.route(x, 2)
    with pytest.raises(TypeError, match="int64"):
        experts.route(x.long(), 2)
    with pytest.raises(ValueError, match="Unsupported scores"):
        experts.route(x, 2, scores="tanh")
    with pytest.raises(ValueError, match="CUDA"):
        experts.plan(torch.zeros(4, 2, dtype=torch.int32), 8)
    with pytest.raises(TypeError, match="int64"):
        experts.plan(torch.zeros(4, 2, dtype=torch.int64), 8)
    with pytest.raises(ValueError, match="CUDA"):
        experts.update_bias(torch.zeros(4), torch.zeros(4, dtype=torch.int32), 1e-3)


def norm_args(**change):
    a = dict(x=P, x_stride=64, residual=P, residual_stride=64, weight=P, weight_dtype=_C.F32, hidden=P, hidden_stride=64,
             out=P, code=0, group=0, scales=P, rstd=P, rows=4, cols=64, eps=1e-6, dtype=_C.BF16, device=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(dtype=_C.F64), _C.ERR_UNSUPPORTED), (dict(dtype=_C.I8), _C.ERR_UNSUPPORTED), (dict(rows=-1), _C.ERR_ARG),
    (dict(rows=1 << 31), _C.ERR_ARG), (dict(cols=0), _C.ERR_ARG), (dict(cols=32769, x_stride=40000), _C.ERR_ARG),
    (dict(eps=0.0), _C.ERR_ARG), (dict(eps=float("nan")), _C.ERR_ARG), (dict(eps=float("inf")), _C.ERR_ARG),
    (dict(code=4), _C.ERR_ARG), (dict(code=-1), _C.ERR_ARG), (dict(group=48), _C.ERR_ARG),
    (dict(weight_dtype=_C.F16), _C.ERR_ARG), (dict(x=None), _C.ERR_ARG), (dict(out=None), _C.ERR_ARG),
    (dict(rstd=None), _C.ERR_ARG), (dict(hidden=None), _C.ERR_ARG), (dict(code=2, scales=None), _C.ERR_ARG),
    (dict(x_stride=63), _C.ERR_ARG), (dict(hidden_stride=63), _C.ERR_ARG), (dict(x=P + 1), _C.ERR_ARG),
    (dict(weight=P + 2), _C.ERR_ARG), (dict(rstd=P + 2), _C.ERR_ARG), (dict(hidden_stride=72), _C.ERR_ARG)])
def test_norm_refuses(dgn_lib, change, status):
    assert dgn_lib.dgn_rms_norm(*norm_args(**change)) == status
    assert dgn_lib.dgn_last_error_string()


def test_norm_of_no_rows_is_nothing(dgn_lib):
    assert dgn_lib.dgn_rms_norm(*norm_args(rows=0, x=None, out=None)) == _C.OK


def norm_grad_args(**change):
    a = dict(grad_out=P, grad_out_stride=64, grad_hidden=P, grad_hidden_stride=64, hidden=P, hidden_stride=64, weight=P,
             weight_dtype=_C.F32, rstd=P, grad_x=P, grad_weight=P, workspace=P, workspace_bytes=1 << 20, rows=4, cols=64,
             dtype=_C.BF16, device=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(dtype=_C.F64), _C.ERR_UNSUPPORTED), (dict(cols=40000), _C.ERR_ARG), (dict(weight=None), _C.ERR_ARG),
    (dict(weight_dtype=_C.F16), _C.ERR_ARG), (dict(grad_weight=P + 2), _C.ERR_ARG),
    (dict(workspace_bytes=4), _C.ERR_ARG), (dict(rstd=None), _C.ERR_ARG), (dict(grad_hidden_stride=63), _C.ERR_ARG)])
def test_norm_grad_refuses(dgn_lib, change, status):
    assert dgn_lib.dgn_rms_norm_grad(*norm_grad_args(**change)) == status


def test_norm_grad_workspace_covers_the_rows(dgn_lib):
    size = dgn_lib.dgn_rms_norm_grad_workspace
    assert size(0, 64, _C.BF16) == 0 and size(4, 64, _C.F64) == 0 and size(4, 0, _C.F32) == 0
    assert size(1, 4096, _C.BF16) == 4096 * 4
    assert size(1 << 20, 4096, _C.BF16) <= 1024 * 4096 * 4  # bounded by the blocks of a grid, not by the rows


def route_args(**change):
    a = dict(logits=P, stride=64, bias=P, mask=P, indices=P, weights=P, tokens=4, experts=64, k=8, score=0, groups=1, keep=1,
             best=1, renormalize=1, scale=1.0, dtype=_C.F32, device=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(dtype=_C.F64), _C.ERR_UNSUPPORTED), (dict(tokens=-1), _C.ERR_ARG), (dict(experts=0), _C.ERR_ARG),
    (dict(experts=1025, stride=1025), _C.ERR_ARG), (dict(k=0), _C.ERR_ARG), (dict(k=33), _C.ERR_ARG),
    (dict(experts=4, k=5), _C.ERR_ARG), (dict(score=2), _C.ERR_ARG), (dict(stride=63), _C.ERR_ARG),
    (dict(groups=0), _C.ERR_ARG), (dict(groups=7), _C.ERR_ARG), (dict(groups=64), _C.ERR_ARG), (dict(keep=0), _C.ERR_ARG),
    (dict(groups=4, keep=5), _C.ERR_ARG), (dict(best=3), _C.ERR_ARG), (dict(logits=None), _C.ERR_ARG),
    (dict(weights=None), _C.ERR_ARG), (dict(logits=P + 2), _C.ERR_ARG), (dict(bias=P + 2), _C.ERR_ARG)])
def test_route_refuses(dgn_lib, change, status):
    assert dgn_lib.dgn_route(*route_args(**change)) == status


def test_calls_without_tokens_do_nothing(dgn_lib):
    assert dgn_lib.dgn_route(*route_args(tokens=0, logits=None)) == _C.OK
    assert dgn_lib.dgn_route_grad(None, None, 64, None, None, 0, 64, 8, 0, 1, 1.0, _C.F32, 0, None) == _C.OK
    assert dgn_lib.dgn_expert_dispatch(None, 16, 16, None, None, None, None, 0, 2, 8, 8, 0, None) == _C.OK
    assert dgn_lib.dgn_expert_combine(None, None, None, None, 0, None, 0, 2, 8, 8, _C.F32, 0, None) == _C.OK
    assert dgn_lib.dgn_expert_combine_grad(None, 8, None, None, None, None, None, None, None, 0, 2, 8, 8, 8, _C.F32, 0,
                                           None) == _C.OK


@pytest.mark.parametrize("slots,num,align,ws,status", [
    (-1, 8, 1, 0, _C.ERR_ARG), (1 << 31, 8, 1, 0, _C.ERR_ARG), (8, 0, 1, 0, _C.ERR_ARG), (8, 1025, 1, 0, _C.ERR_ARG),
    (8, 8, 0, 0, _C.ERR_ARG), (1 << 20, 8, 1 << 30, 0, _C.ERR_ARG), (1 << 20, 8, 1, 0, _C.ERR_ARG)])
def test_plan_refuses(dgn_lib, slots, num, align, ws, status):
    assert dgn_lib.dgn_expert_plan(P, slots, num, align, P, P, P, P, None, ws, 0, None) == status


def test_moves_refuse(dgn_lib):
    dispatch = dgn_lib.dgn_expert_dispatch
    assert dispatch(P, 8, 16, P, P, P, P, 4, 2, 8, 8, 0, None) == _C.ERR_ARG        # stride shorter than the row
    assert dispatch(P, 16, 16, P, P, P, P, 4, 33, 8, 8, 0, None) == _C.ERR_ARG      # choices
    assert dispatch(P, 16, 16, P, P, P, P, 4, 2, 1025, 8, 0, None) == _C.ERR_ARG    # experts
    assert dispatch(P, 16, 16, P, P, P, P, 4, 2, 8, 1 << 31, 0, None) == _C.ERR_ARG  # rows
    assert dispatch(P, 16, 16, P + 2, P, P, P, 4, 2, 8, 8, 0, None) == _C.ERR_ARG   # alignment
    assert dispatch(P, 16, 16, P, P, P, None, 4, 2, 8, 8, 0, None) == _C.ERR_ARG
    combine = dgn_lib.dgn_expert_combine
    assert combine(P, P, P, P, 8, P, 4, 2, 8, 8, _C.F64, 0, None) == _C.ERR_UNSUPPORTED
    assert combine(P, P, P, P, 7, P, 4, 2, 8, 8, _C.F32, 0, None) == _C.ERR_ARG
    assert combine(P, None, P, P, 8, P, 4, 2, 8, 8, _C.F32, 0, None) == _C.ERR_ARG
    grad = dgn_lib.dgn_expert_combine_grad
    assert grad(P, 7, P, P, P, P, P, P, P, 4, 2, 8, 8, 8, _C.F32, 0, None) == _C.ERR_ARG
    assert grad(P, 8, P, P, None, P, P, P, P, 4, 2, 8, 8, 8, _C.F32, 0, None) == _C.ERR_ARG
    assert grad(P, 8, P, P, P, P, P, P, P, 4, 2, 8, 8, 8, _C.I32, 0, None) == _C.ERR_UNSUPPORTED
    bias = dgn_lib.dgn_expert_update_bias
    assert bias(P, P, P, 0, 1e-3, 0, None) == _C.ERR_ARG
    assert bias(P, None, P, 4, 1e-3, 0, None) == _C.ERR_ARG
    assert bias(P, P, P + 1, 4, 1e-3, 0, None) == _C.ERR_ARG


def test_signatures_take_pointers_as_integers(dgn_lib):
    """The binding passes addresses as plain integers and None as null."""
    assert dgn_lib.dgn_rms_norm.argtypes[0] is ctypes.c_void_p and len(dgn_lib.dgn_rms_norm.argtypes) == 19

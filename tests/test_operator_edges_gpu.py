"""Calls at the edges of what the norm and expert operators take."""

import os
import subprocess
import sys

import pytest
import torch

from dragon_b200.experts import combine, combine_grad, dispatch, plan, route
from dragon_b200.normalization import rms_norm, rms_norm_grad

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def normal(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def test_views_that_stand_for_other_values_are_refused(dgn_lib):
    """x.conj() and the imaginary part of one share x's memory, whose values they are not."""
    z = torch.complex(normal(6, 4, seed=1), normal(6, 4, seed=2))
    p = plan(torch.zeros(6, 1, dtype=torch.int32, device=DEV), 2)
    assert torch.equal(dispatch(z.conj().resolve_conj(), p), z.conj())
    with pytest.raises(ValueError, match="conjugate"):
        dispatch(z.conj(), p)
    negative = z.conj().imag  # a negative view, of rows that are not contiguous
    assert negative.is_neg()
    column, vector = negative[:, :1], torch._neg_view(normal(4, seed=3))
    x = normal(6, 4, seed=4)
    for call in (lambda: dispatch(column, p), lambda: combine(torch._neg_view(x), p), lambda: rms_norm(column),
                 lambda: rms_norm(x, vector), lambda: rms_norm(x, residual=torch._neg_view(x)),
                 lambda: rms_norm_grad(torch._neg_view(x), x, rms_norm(x).rstd), lambda: route(column, 1),
                 lambda: route(x, 1, bias=vector)):
        with pytest.raises(ValueError, match="view"):
            call()


def test_the_longest_odd_rows(dgn_lib):
    """Rows whose bytes pass 31 bits with the offset of an unaligned start."""
    cols = (1 << 30) - 1
    p = plan(torch.arange(2, dtype=torch.int32, device=DEV)[:, None].contiguous(), 2)
    rows = torch.empty(2, cols, dtype=torch.float16, device=DEV)
    rows[0], rows[1] = 1.0, 2.0
    rows[:, :64] = normal(2, 64, seed=1, dtype=torch.float16)
    rows[:, -64:] = normal(2, 64, seed=2, dtype=torch.float16)
    assert torch.equal(combine(rows, p), rows)
    del rows
    one, row = plan(torch.zeros(1, 1, dtype=torch.int32, device=DEV), 1), torch.ones(1, cols + 1, dtype=torch.float16, device=DEV)
    residual = torch.ones(1, cols + 9, dtype=torch.float16, device=DEV)
    residual[:, :64] = 3.0
    cut = residual[:, 1:cols + 2]
    assert torch.equal(combine(row, one, residual=cut), cut + 1)


def test_a_process_is_told_once_that_no_graph_is_recorded(dgn_lib):
    code = """
import warnings
import torch
from dragon_b200.experts import combine, combine_grad, dispatch, plan, route
from dragon_b200.normalization import rms_norm, rms_norm_grad
x = torch.ones(4, 8, device="cuda:0", requires_grad=True)
p = plan(torch.zeros(4, 1, dtype=torch.int32, device="cuda:0"), 2)
calls = [lambda x: rms_norm(x).output, lambda x: rms_norm(x.detach(), x[0]).output, lambda x: route(x, 2)[1], lambda x: dispatch(x, p),
         lambda x: combine(x, p)]
def run(inputs):
    with warnings.catch_warnings(record=True) as told:
        warnings.simplefilter("always")
        for call in calls:
            assert not call(inputs).requires_grad
    return [str(w.message) for w in told]
assert run(x.detach()) == []
with torch.no_grad():
    assert run(x) == []
for call in calls:  # a filter that makes it an error stops every one of them
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        try:
            call(x)
        except UserWarning:
            continue
        raise AssertionError("no word")
told = run(x)
assert len(told) == 1 and "rms_norm_grad" in told[0], told
assert run(x) == []
print("TOLD_ONCE")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert "TOLD_ONCE" in done.stdout, done.stdout + done.stderr


U = 2.0 ** -24  # half a step of float32


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [64, 61])
@pytest.mark.parametrize("start", [0, 1, 8])
def test_strided_rows_against_the_definition(dgn_lib, dtype, cols, start):
    """Whatever the order: a sum of n products is within n steps' halves of the sum of their magnitudes, then rounded once."""
    g = torch.Generator().manual_seed(1)
    indices = torch.stack([torch.randperm(6, generator=g)[:3] for _ in range(40)]).int().to(DEV)
    p = plan(indices, 6)
    rows, weights, wide = normal(120, cols, seed=2, dtype=dtype), normal(40, 3, seed=3), normal(40, 90, seed=4, dtype=dtype)
    cut, mine = wide[:, start:start + cols], rows[p.positions.long()].double()
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half  # below the normal numbers steps stop shrinking
    terms = mine * weights.double()[:, :, None]
    want, size = terms.sum(1) + cut.double(), terms.abs().sum(1) + cut.double().abs()
    got = combine(rows, p, weights, cut).double()
    assert ((got - want).abs() <= 4 * U * size + half * (want.abs() + 4 * U * size) + tiny).all()
    grad_rows, grad_weights = combine_grad(cut, rows, p, weights)
    terms = mine * cut.double()[:, None]
    assert ((grad_weights.double() - terms.sum(2)).abs() <= cols * U * terms.abs().sum(2)).all()
    want = weights.double()[:, :, None] * cut.double()[:, None]
    off = (grad_rows[p.positions.long()].double() - want).abs()
    assert (off <= U * want.abs() + half * (1 + U) * want.abs() + tiny).all()


def test_offsets_beyond_32_bits(dgn_lib):
    """Matrices of more than 2^32 bytes and 2^31 elements: their last rows are those of a small call with the same layout."""
    rows, cols, last = 530000, 4104, 300
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[:], x[-last:] = 1.0, normal(last, cols, seed=1, dtype=torch.bfloat16)
    weight = 1 + 0.1 * normal(cols, seed=2)
    for dtype, group in ((None, 0), (torch.float8_e4m3fn, 32)):
        big, small = (rms_norm(t, weight, out_dtype=dtype, group_size=group) for t in (x, x[-last:]))
        assert torch.equal(big.output[-last:].view(torch.uint8), small.output.view(torch.uint8))
        assert torch.equal(big.rstd[-last:], small.rstd) and (dtype is None or torch.equal(big.scale[-last:], small.scale))
    assert torch.equal(rms_norm_grad(x, x, big.rstd)[0][-last:], rms_norm_grad(x[-last:], x[-last:], small.rstd)[0])
    del big
    indices = torch.zeros(rows, 1, dtype=torch.int32, device=DEV)
    indices[-last:] = 1  # the second expert's block begins behind 2^31 elements
    p = plan(indices, 2)
    moved = dispatch(x, p)
    assert torch.equal(p.positions[-last:, 0], torch.arange(rows - last, rows, dtype=torch.int32, device=DEV))
    assert torch.equal(moved[-last:], x[-last:])
    weights = torch.full((rows, 1), 0.5, device=DEV)
    assert torch.equal(combine(moved, p, weights)[-last:], x[-last:] * 0.5)
    grad_rows, grad_weights = combine_grad(x, moved, p, weights)
    assert torch.equal(grad_rows[-last:], x[-last:] * 0.5)
    want = x[-last:].double().square().sum(1)
    assert ((grad_weights[-last:, 0].double() - want).abs() <= cols * U * want).all()

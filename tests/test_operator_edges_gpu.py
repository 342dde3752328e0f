"""Calls at the edges of what the norm and expert operators take."""

import pytest
import torch

from dragon_b200.experts import combine, dispatch, plan, route
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

"""rms_norm and rms_norm_grad against the definition in 64 bits.

Tolerances.  u = 2^-24 is half a step of float32.  A row's sums take at most 64
additions in a thread, 5 + 5 across lanes and warps: with the products' own
rounding a sum is off by at most SUM = 80 u of the sum of its terms'
magnitudes.  rstd inherits half of the relative error of mean(h^2) (all terms
positive) and a few roundings: RSTD = 45 u.  Outputs add their rounding, half a
step of their type, relative to the value."""

import pytest
import torch

from dragon_b200.normalization import rms_norm, rms_norm_grad

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SUM, RSTD = 80 * U, 45 * U
FLOATS = [torch.float32, torch.bfloat16, torch.float16]
CODES = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
DEV = "cuda:0"


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step below the smallest normal number, where steps stop shrinking."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def make(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(rows, cols, generator=g)).to(dtype).to(DEV)


def weight_of(cols, dtype, seed=5):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.2 * torch.randn(cols, generator=g)).to(dtype).to(DEV)


def reference(x, weight, residual, eps):
    hidden = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    h = hidden.double()
    rstd = (h.square().mean(-1) + eps).rsqrt()
    y = h * rstd[..., None]
    return hidden, rstd, y if weight is None else y * weight.double()


def close(got, want, bound, what):
    """|got - want| <= bound, element by element."""
    off = (got.double() - want).abs() - bound
    assert not torch.isnan(off).any() and off.max() <= 0, "{}: {} past its bound".format(what, off.max().item())


SHAPES = [(1, 1), (1, 4096), (3, 769), (5, 128), (33, 1024), (7, 100), (600, 64), (2, 8192), (2, 16384), (2, 32768),
          (3, 1030), (2, 5121), (1500, 520), (2, 20001)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("kind", ["plain", "weight", "residual"])
def test_forward(dgn_lib, rows, cols, dtype, kind):
    x = make(rows, cols, dtype, 1)
    weight = None if kind == "plain" else weight_of(cols, dtype if kind == "weight" else torch.float32)
    residual = make(rows, cols, dtype, 2, 2.0) if kind == "residual" else None
    r = rms_norm(x, weight, residual, 1e-5)
    hidden, rstd, y = reference(x, weight, residual, 1e-5)
    # x + r in float32 and then in the type: two roundings, against one of the exact sum.
    assert (r.hidden != hidden).float().mean() <= 1e-3
    close(r.hidden, hidden.double(), 2 * half(dtype) * hidden.double().abs(), "hidden")
    hidden, rstd, y = reference(r.hidden, weight, None, 1e-5)
    close(r.rstd, rstd, RSTD * rstd, "rstd")
    close(r.output, y, (RSTD + 4 * U + half(dtype)) * y.abs() + tiny(dtype), "output")
    assert r.scale is None


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 769), (5, 128), (4, 4096), (2, 32768), (9, 200), (130, 96), (3, 2056), (3, 1030),
                                       (5, 70), (2, 4228)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("out_dtype", list(CODES))
@pytest.mark.parametrize("group", [0, 32, 64, 128])
def test_codes(dgn_lib, rows, cols, dtype, out_dtype, group):
    x, residual, weight = make(rows, cols, dtype, 1), make(rows, cols, dtype, 2), weight_of(cols, torch.float32)
    x[0] *= 0  # a row of zeros
    residual[0] *= 0
    r = rms_norm(x, weight, residual, 1e-6, out_dtype=out_dtype, group_size=group)
    _, _, y = reference(r.hidden, weight, None, 1e-6)
    width, top = group or cols, CODES[out_dtype]
    groups = -(-cols // width)
    assert r.output.dtype == out_dtype and tuple(r.scale.shape) == (rows, groups)
    padded = torch.nn.functional.pad(y, (0, groups * width - cols)).view(rows, groups, width)
    scale = padded.abs().amax(2).clamp(min=2.0 ** -40) / top
    close(r.scale, scale, (RSTD + 8 * U) * scale, "scale")
    wide = r.scale.double().repeat_interleave(width, 1)[:, :cols]
    # Half a step of the code: 1/2 for int8; of the value, or of the smallest normal code, for the others.
    step = 0.5 * wide if out_dtype == torch.int8 else torch.maximum(
        half(out_dtype) * y.abs(), tiny(out_dtype) * wide)
    close(r.output.double() * wide, y, step + (RSTD + 12 * U) * y.abs() + 1e-30, "value")
    largest = (r.output.double().abs() * (y.abs() > 0)).amax()
    assert largest <= top


def test_code_scales_have_a_floor_and_report_what_is_not_finite(dgn_lib):
    x = torch.ones(4, 256, device=DEV)
    weight = torch.ones(256, device=DEV)
    weight[:128] = 1e-20  # a group far below the floor
    x[1, 200], x[2, 130] = float("nan"), float("inf")
    for out_dtype, top in CODES.items():
        r = rms_norm(x, weight, out_dtype=out_dtype, group_size=128)
        assert abs(r.scale[0, 0].item() * top * 2.0 ** 40 - 1) <= U  # one rounding to float32: half a step
        assert torch.isnan(r.scale[1]).all()               # rstd is NaN: the whole row
        assert torch.isnan(r.scale[2, 1])                  # inf * 0 in its own group
        assert torch.isfinite(r.scale[3]).all()
        back = r.output.float() * r.scale.repeat_interleave(128, 1)
        assert torch.isnan(back[1]).all() and torch.isfinite(back[3]).all()
        assert (back[0, 128:] - 1).abs().max() <= 2.0 ** -2  # half a step of the coarsest code


def test_rows_do_not_touch_each_other(dgn_lib):
    for cols in (64, 769, 4096):
        x = make(6, cols, torch.bfloat16, 3)
        want = rms_norm(x).output.clone()
        x[2, 0], x[4, cols - 1] = float("nan"), float("inf")
        r = rms_norm(x)
        for row in (0, 1, 3, 5):
            assert torch.equal(r.output[row], want[row])
        assert torch.isnan(r.output[2]).all() and r.rstd[4] == 0


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("cols,offset", [(64, 0), (64, 1), (1000, 8), (1000, 3)])
def test_strided_rows_and_unaligned_starts(dgn_lib, dtype, cols, offset):
    wide_x, wide_r, wide_g = (make(10, cols + 24, dtype, s) for s in (1, 2, 3))
    cut = lambda t: t[:, offset:offset + cols]  # noqa: E731
    weight = weight_of(cols + 3, torch.float32)[3:]
    a = rms_norm(cut(wide_x), weight, cut(wide_r))
    b = rms_norm(cut(wide_x).contiguous(), weight.clone(), cut(wide_r).contiguous())
    assert torch.equal(a.hidden, b.hidden)
    _, _, y = reference(a.hidden, weight, None, 1e-6)
    for r in (a, b):
        close(r.output, y, (RSTD + 4 * U + half(dtype)) * y.abs() + tiny(dtype), "output")
    # Aligned and other rows add in another order: each is held to the bound of the definition, as in test_backward.
    grad, grad_weight = rms_norm_grad(cut(wide_g), a.hidden, a.rstd, weight, cut(wide_r))
    want, bound, want_w, size_w = grad_reference(cut(wide_g), a.hidden, a.rstd, weight, cut(wide_r))
    close(grad, want, bound + half(dtype) * want.abs() + tiny(dtype), "grad_x")
    close(grad_weight, want_w, (10 / 148 + 80) * U * size_w + U * want_w.abs(), "grad_weight")
    kept = wide_r.clone()
    c = rms_norm(cut(wide_x), weight, cut(wide_r), inplace_residual=True)
    assert c.hidden.data_ptr() == cut(wide_r).data_ptr() and torch.equal(c.hidden, a.hidden)
    assert torch.equal(wide_r[:, :offset], kept[:, :offset]) and torch.equal(wide_r[:, offset + cols:], kept[:, offset + cols:])
    x3 = make(12, cols, dtype, 4).view(3, 4, cols)
    assert torch.equal(rms_norm(x3).output, rms_norm(x3.view(12, cols)).output.view(3, 4, cols))


def test_rows_of_more_dimensions(dgn_lib):
    """Dimensions that fold into rows at one distance are taken, others refused."""
    wide = make(12, 100, torch.float32, 7).view(3, 4, 100)
    cut = wide[:, :, 8:72]
    r, flat = rms_norm(cut, residual=wide[:, :, 20:84]), rms_norm(cut.reshape(12, 64), residual=wide[:, :, 20:84].reshape(12, 64))
    assert r.output.shape == (3, 4, 64) and r.rstd.shape == (3, 4)
    assert torch.equal(r.output.view(12, 64), flat.output) and torch.equal(r.hidden.view(12, 64), flat.hidden)
    grad, _ = rms_norm_grad(cut, r.hidden, r.rstd)
    assert torch.equal(grad.view(12, 64), rms_norm_grad(cut.reshape(12, 64), flat.hidden, flat.rstd)[0])
    for bad in (wide.transpose(0, 1), wide[:, ::3], wide[..., ::2]):
        with pytest.raises(ValueError):
            rms_norm(bad)
    assert rms_norm(make(1, 64, torch.float32, 8)[0]).output.shape == (64,)


def grad_reference(dy, hidden, rstd, weight, grad_hidden):
    dy, h, r = dy.double(), hidden.double(), rstd.double()[:, None]
    g = dy if weight is None else dy * weight.double()
    n = h * r
    grad = r * (g - n * (g * n).mean(1, keepdim=True))
    # What float32 sums and roundings may add: the mean's error, then a few roundings of each term.
    bound = SUM * r * n.abs() * (g * n).abs().mean(1, keepdim=True) + 8 * U * (r * g.abs() + (r * n * (g * n).mean(1, keepdim=True)).abs())
    if grad_hidden is not None:
        grad = grad + grad_hidden.double()
        bound = bound + 2 * U * grad.abs()
    return grad, bound, (dy * n).sum(0), (dy * n).abs().sum(0)


@pytest.mark.parametrize("rows,cols", SHAPES + [(4000, 256)])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("kind", ["plain", "weight", "residual"])
def test_backward(dgn_lib, rows, cols, dtype, kind):
    hidden, dy = make(rows, cols, dtype, 1), make(rows, cols, dtype, 2)
    weight = None if kind == "plain" else weight_of(cols, dtype if kind == "weight" else torch.float32)
    grad_hidden = make(rows, cols, dtype, 3) if kind == "residual" else None
    rstd = rms_norm(hidden).rstd
    grad, grad_weight = rms_norm_grad(dy, hidden, rstd, weight, grad_hidden)
    want, bound, want_w, size_w = grad_reference(dy, hidden, rstd, weight, grad_hidden)
    close(grad, want, bound + half(dtype) * want.abs() + tiny(dtype), "grad_x")
    if weight is None:
        assert grad_weight is None
        return
    # A column's sum: at most rows / blocks + 32 additions in a row of them, each of them half a step.
    steps = (rows / 148 + 80) * U
    close(grad_weight, want_w, steps * size_w + half(weight.dtype) * want_w.abs() + tiny(weight.dtype), "grad_weight")
    again, again_w = rms_norm_grad(dy, hidden, rstd, weight, grad_hidden)
    assert torch.equal(again, grad) and torch.equal(again_w, grad_weight)


@pytest.mark.parametrize("cols", [5, 64, 1001, 4096])
def test_backward_against_differences(dgn_lib, cols):
    """Central differences of the definition in 64 bits, along random directions."""
    x, dy, gh = (make(3, cols, torch.float32, s) for s in (1, 2, 3))
    weight = weight_of(cols, torch.float32)
    r = rms_norm(x, weight)
    grad, grad_weight = rms_norm_grad(dy, r.hidden, r.rstd, weight, gh)

    def loss(h, w):
        y = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w
        return (y * dy.double()).sum() + (h * gh.double()).sum()

    for seed in range(3):
        dx, dw = make(3, cols, torch.float64, 10 + seed), make(1, cols, torch.float64, 20 + seed)[0]
        step = 1e-5
        slope = (loss(x.double() + step * dx, weight.double() + step * dw)
                 - loss(x.double() - step * dx, weight.double() - step * dw)) / (2 * step)
        got = (grad.double() * dx).sum() + (grad_weight.double() * dw).sum()
        # Each gradient is within 200 u of the magnitudes that make it up; differences add step^2.
        size = (dx.abs() * (3 * dy.double().abs() + gh.double().abs() + 3)).sum() + (dw.abs() * dy.double().abs().sum(0) * 4).sum()
        assert (got - slope).abs() <= 200 * U * size + 1e-7 * size


def test_no_rows(dgn_lib):
    x, weight = torch.empty(0, 64, device=DEV), torch.ones(64, device=DEV)
    r = rms_norm(x, weight, out_dtype=torch.int8, group_size=32)
    assert r.output.shape == (0, 64) and r.scale.shape == (0, 2)
    grad, grad_weight = rms_norm_grad(x, x, r.rstd, weight)
    assert grad.shape == (0, 64) and torch.equal(grad_weight, torch.zeros(64, device=DEV))


def test_refusals_on_the_device(dgn_lib):
    x = torch.ones(4, 64, device=DEV)
    bad = [dict(weight=torch.ones(63, device=DEV)), dict(weight=torch.ones(64)), dict(residual=torch.ones(4, 63, device=DEV)),
           dict(residual=torch.ones(4, 64)), dict(residual=torch.ones(1, 64, device=DEV).expand(4, 64)), dict(eps=0.0),
           dict(group_size=16), dict(inplace_residual=True)]
    for kwargs in bad:
        with pytest.raises(ValueError):
            rms_norm(x, **kwargs)
    for kwargs in (dict(weight=torch.ones(64, device=DEV, dtype=torch.float16)), dict(out_dtype=torch.int32),
                   dict(residual=torch.ones(4, 64, device=DEV, dtype=torch.float16))):
        with pytest.raises(TypeError):
            rms_norm(x, **kwargs)
    with pytest.raises(ValueError):
        rms_norm(torch.ones(64, 4, device=DEV).t())
    with pytest.raises(ValueError):
        rms_norm_grad(x, x, torch.ones(3, device=DEV))
    from dragon_b200 import _C
    with pytest.raises(_C.DgnError):
        rms_norm(torch.ones(1, 32769, device=DEV))
    args = (x.data_ptr(), 64, None, 0, x.data_ptr(), 64, x.data_ptr(), _C.F32, x.data_ptr(), x.data_ptr(), x.data_ptr(),
            x.data_ptr(), 16, 4, 64, _C.F32, 0, None)
    assert dgn_lib.dgn_rms_norm_grad(*args) == _C.ERR_ARG and b"workspace" in dgn_lib.dgn_last_error_string()


def test_streams_and_graphs(dgn_lib):
    x, residual, dy = (make(300, 1024, torch.bfloat16, s) for s in (1, 2, 3))
    weight = weight_of(1024, torch.float32)

    def both(**kwargs):
        r = rms_norm(x, weight, residual, **kwargs)
        return [r.output, r.hidden, r.rstd, *rms_norm_grad(dy, r.hidden, r.rstd, weight, residual, **kwargs)]

    want = both()
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):  # two streams at once, one given as a raw handle: their workspaces are their own
        a, b = both(stream=side), both(stream=other.cuda_stream)
    torch.cuda.synchronize()
    for got in (a, b):
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both())
        graphs.append(graph)
    x.mul_(-1)
    want = both()
    for graph in graphs:  # replayed at once, on two streams
        with torch.cuda.stream(side if graph is graphs[0] else other):
            torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
            graph.replay()
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(g, w) for g, w in zip(got, want))

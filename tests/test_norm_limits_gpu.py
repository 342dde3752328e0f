"""rms_norm at the ends of its ranges.

u = 2^-24 is half a step of float32."""

import threading

import pytest
import torch

from dragon_b200 import _C
from dragon_b200.normalization import rms_norm, rms_norm_grad

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CODES = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
DEV = "cuda:0"


def normal(*shape, seed=0, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(*shape, generator=g)).to(dtype).to(DEV)


def grouped(t, width):
    return t.reshape(t.shape[0], t.shape[1] // width, width)


@pytest.mark.parametrize("out_dtype", list(CODES))
@pytest.mark.parametrize("cols,group", [(64, 0), (64, 32), (96, 32), (33, 0)])
def test_codes_of_products_whose_reciprocal_is_below_the_normal_numbers(dgn_lib, out_dtype, cols, group):
    """hidden * weight between 2^126 and the largest float32: the largest code over it is an ordinary number all the same.
    Groups whose largest value passes float32 (one in row 0, 3.9e38) report an infinity: their scale is NaN."""
    x = normal(5, cols, seed=1, scale=1e17)
    weight = torch.full((cols,), 1.2e38, device=DEV)
    weight[::3] *= -0.5
    x = x / x.abs().amax(1, keepdim=True) * 1.5
    x[0], x[1] = x[0] * 0.6, x[1] * 1.8  # |h w| from 1.08e38 (2^126.3) to 3.2e38 at its largest
    r = rms_norm(x, weight, out_dtype=out_dtype, group_size=group)
    h = x.double()
    y = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * weight.double()
    width, top = group or cols, CODES[out_dtype]
    largest = grouped(y, width).abs().amax(2)
    scale = torch.where(largest <= torch.finfo(torch.float32).max, largest / top, float("nan"))
    fits = torch.isfinite(scale)
    assert fits.float().mean() >= 0.8
    assert torch.equal(torch.isnan(r.scale), torch.isnan(scale))
    # The row's sum of at most 96 squares, its root, and three roundings.
    assert ((r.scale.double() - scale).abs() <= 64 * U * scale)[fits].all()
    wide = r.scale.double().repeat_interleave(width, 1)
    half = 0.5 * wide if out_dtype == torch.int8 else torch.maximum(
        torch.finfo(out_dtype).eps / 2 * y.abs(), torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps / 2 * wide)
    off = (r.output.double() * wide - y).abs() - half - 72 * U * y.abs()
    assert off[fits.repeat_interleave(width, 1)].max() <= 0


def test_the_root_is_rounded_once(dgn_lib):
    """One column: h^2 and its sum with eps are rounded, which the root halves, and the root: two times half a step."""
    x = normal(4096, 1, seed=2) * torch.exp(normal(4096, 1, seed=3, scale=8.0))
    x[0], x[1], x[2] = 0.0, 1e-30, 1.8e19
    r = rms_norm(x, eps=1e-5)
    want = (x.double().square()[:, 0] + torch.tensor(1e-5, dtype=torch.float32).double().item()).rsqrt()
    assert ((r.rstd.double() - want).abs() <= 2.01 * U * want).all()


@pytest.mark.parametrize("out_dtype", list(CODES))
@pytest.mark.parametrize("cols", [512, 514, 515, 4096])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_codes_are_the_nearest_ones_between_neighbours_too(dgn_lib, out_dtype, cols, group):
    """Products u of bfloat16 rows and weights have 16 bits, so that u L / m is often halfway between two codes and
    otherwise at least 2^-41 of itself away from where float32 rounds: whoever rounds the quotient once gets these codes."""
    x, weight = normal(256, cols, seed=4, dtype=torch.bfloat16), normal(cols, seed=5, dtype=torch.bfloat16)
    r = rms_norm(x, weight, out_dtype=out_dtype, group_size=group)
    u, width = x.double() * weight.double(), group or cols
    groups = -(-cols // width)
    m = torch.nn.functional.pad(u, (0, groups * width - cols)).view(256, groups, width).abs().amax(2)
    q = (u * CODES[out_dtype] / m.repeat_interleave(width, 1)[:, :cols]).float()
    want = (q.round() if out_dtype == torch.int8 else q).to(out_dtype)
    assert torch.equal(r.output.view(torch.uint8), want.view(torch.uint8))


def test_two_threads_with_kernels_of_different_size(dgn_lib):
    """Callers of the C-ABI on threads of their own: the same kernel with more and with less shared memory at the same time."""
    failed, outputs = [], {}

    def work(cols):
        dy, h, gh = (normal(64, cols, seed=s, dtype=torch.bfloat16) for s in (1, 2, 3))
        rstd, out = rms_norm(h).rstd, torch.empty_like(h)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        for _ in range(3000):
            rc = dgn_lib.dgn_rms_norm_grad(dy.data_ptr(), cols, gh.data_ptr(), cols, h.data_ptr(), cols, None, _C.F32,
                                           rstd.data_ptr(), out.data_ptr(), None, None, 0, 64, cols, _C.BF16, 0,
                                           stream.cuda_stream)
            if rc != _C.OK:
                failed.append((cols, rc))
                break
        stream.synchronize()
        outputs[cols] = (out, rms_norm_grad(dy, h, rstd, None, gh)[0])

    threads = [threading.Thread(target=work, args=(cols,)) for cols in (4096, 2560, 2048)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    torch.cuda.synchronize()
    assert len(outputs) == 3 and all(torch.equal(a, b) for a, b in outputs.values())


@pytest.mark.parametrize("cols,dtype", [(64, torch.float32), (4096, torch.float32), (4096, torch.bfloat16), (1025, torch.float32),
                                        (32768, torch.float32)])
def test_the_sum_of_squares_has_the_range_of_float32(dgn_lib, cols, dtype):
    """Whatever the order of the additions: right below 2^128, zeros from there on.

    At most 74 additions follow one another (64 in a thread, 10 across threads), each half a step, and with the products'
    own the sum is off by 80 u, its root by half of that and a few roundings: 45 u; the output adds four more and its type's."""
    edge = (2.0 ** 128 / cols) ** 0.5
    x = torch.stack([torch.full((cols,), f * edge) for f in (0.98, 0.9, 1.02, 10.0)]).to(dtype).to(DEV)
    r = rms_norm(x)
    assert ((r.output[:2].double() - 1).abs() <= 49 * U + torch.finfo(dtype).eps / 2).all()
    want = x[:2, 0].double().reciprocal()
    assert ((r.rstd[:2].double() - want).abs() <= 45 * U * want).all()
    assert (r.output[2:] == 0).all() and (r.rstd[2:] == 0).all()


@pytest.mark.parametrize("out_dtype", list(CODES))
@pytest.mark.parametrize("cols", [64, 65])
def test_the_smallest_eps(dgn_lib, out_dtype, cols):
    """Rows of zeros stay zeros, and the smallest scale is theirs; a smaller eps is refused."""
    r = rms_norm(torch.zeros(3, cols, device=DEV), eps=2.0 ** -126, out_dtype=out_dtype)
    assert (r.output.float() == 0).all() and (r.scale.double() * CODES[out_dtype] * 2.0 ** 40 - 1).abs().max() <= U
    for eps in (1e-45, 2.0 ** -127):
        with pytest.raises(ValueError, match="eps"):
            rms_norm(torch.zeros(3, cols, device=DEV), eps=eps, out_dtype=out_dtype)

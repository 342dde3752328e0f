"""Choices of route() between keys that float32 does not tell apart, many rows at a time.

The definition is computed in 64 bits on the CPU.  Its exponentials and the
kernel's may differ in their last bit, so that rows whose keys lie within 1e-15
of each other without being equal are left out; there is about one in 1e7."""

import pytest
import torch

from dragon_b200.experts import route, route_grad

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
INF = float("inf")


def generator(seed):
    return torch.Generator().manual_seed(seed)


def keys_of(logits, bias, scores):
    l = logits.double()
    s = torch.sigmoid(l) if scores == "sigmoid" else torch.softmax(l, 1)
    return torch.where(l == -INF, -INF, s + bias.double())


def check(logits, bias, k, scores, groups=1, keep=1, best=1, at_least=0.99):
    """The k first of the definition for every row that 64 bits decide."""
    key = keys_of(logits, bias, scores)
    tokens, num = key.shape
    clear = torch.ones(tokens, dtype=torch.bool)
    if groups > 1:
        top = key.view(tokens, groups, -1).sort(stable=True, dim=2, descending=True)[0][:, :, :best]
        value = torch.where(top == -INF, 0.0, top).sum(2).masked_fill(top[:, :, 0] == -INF, -INF)
        ranked, order = value.sort(stable=True, dim=1, descending=True)
        if keep < groups:
            gap = ranked[:, keep - 1] - ranked[:, keep]
            # Sums of keys: their own rounding in 64 bits.
            clear &= ~((gap > 0) & (gap <= 1e-15 + 2.0 ** -50 * top.abs().masked_fill(top == -INF, 0).amax((1, 2))))
        kept = torch.zeros(tokens, groups, dtype=torch.bool).scatter_(1, order[:, :keep], True)
        key = torch.where(kept.repeat_interleave(num // groups, 1), key, -INF)
    ranked, order = key.sort(stable=True, dim=1, descending=True)
    gaps = ranked[:, :k] - torch.nn.functional.pad(ranked, (0, 1), value=-INF)[:, 1:k + 1]
    clear &= ~((gaps > 0) & (gaps <= 1e-15)).any(1)
    assert clear.float().mean() >= at_least
    want = torch.where(ranked[:, :k] == -INF, -1, order[:, :k]).int()
    got = route(logits.to(DEV), k, bias.to(DEV), scores=scores, groups=groups, keep_groups=keep, group_best=best)[0].cpu()
    wrong = (got != want).any(1) & clear
    assert not wrong.any(), "{} of {} rows differ, the first of them {}: {} instead of {}".format(
        int(wrong.sum()), int(clear.sum()), int(wrong.nonzero()[0]), got[wrong][0].tolist(), want[wrong][0].tolist())


def level(num, scores, tokens, seed, spread=0.05):
    """A bias, and logits whose scores it undoes: all keys of a row are equal but for the rounding of the logits."""
    g = generator(seed)
    bias = spread * torch.rand(num, generator=g) / (num if scores == "softmax" else 1)
    if scores == "softmax":  # scores that add up to one, and a shift of the logits that does not move them
        score = (1 + bias.double().sum()) / num - bias.double()
        logits = torch.log(score) + torch.randn(tokens, 1, generator=g, dtype=torch.float64)
    else:
        score = 0.3 + 0.5 * torch.rand(tokens, 1, generator=g, dtype=torch.float64) - bias.double()
        logits = torch.log(score) - torch.log1p(-score)
    return logits.float(), bias


@pytest.mark.parametrize("num", [2, 3, 4, 5, 8, 16, 64, 256, 600])
@pytest.mark.parametrize("k", [1, 2])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_a_bias_that_undoes_the_scores(dgn_lib, num, k, scores):
    logits, bias = level(num, scores, 3000, seed=num)
    check(logits, bias, k, scores)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("k", [1, 2])
@pytest.mark.parametrize("how", ["logits", "bias", "groups"])
def test_two_open_experts(dgn_lib, scores, k, how):
    """Of 32 experts two are left, nearly equal: by logits of -inf, by a bias of -inf, or by the groups that are kept."""
    tokens, num = 3000, 32
    pair, low = level(2, scores, tokens, seed=7)
    logits, bias = torch.full((tokens, num), -INF), torch.zeros(num)
    logits[:, 6:8], bias[6:8] = pair, low
    if how == "logits":
        return check(logits, bias, k, scores)
    logits[:, :6] = logits[:, 8:] = -30.0
    if how == "bias":
        bias[:6] = bias[8:] = -INF
        return check(logits, bias, k, scores)
    check(logits, bias, k, scores, groups=16, keep=1)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_two_experts_far_apart_in_steps(dgn_lib, scores):
    """The largest and the smallest key of a row are as many steps apart as there are, however near they lie."""
    g = generator(3)
    bias = torch.tensor([0.03, -0.02])
    score = 0.4 + 0.2 * torch.rand(4000, 1, generator=g, dtype=torch.float64) - bias.double()
    if scores == "softmax":
        score = 0.5 - (bias - bias.mean()).double().expand(4000, 2)
        logits = torch.log(score) + torch.randn(4000, 1, generator=g, dtype=torch.float64)
    else:
        logits = torch.log(score) - torch.log1p(-score)
    logits = logits + 1e-7 * torch.randn(4000, 2, generator=g, dtype=torch.float64)
    check(logits.float(), bias, 1, scores)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("width", [32, 24])  # a power of two of vectors, and groups that go through shared memory
@pytest.mark.parametrize("offset", [0.5, 4.0, 8.0, 32.0, 512.0])
@pytest.mark.parametrize("groups", [2, 4])
def test_groups_whose_keys_cancel(dgn_lib, scores, width, offset, groups):
    """The two best of each group are one of bias +offset and one of -offset: their sum is small, its rounding is not."""
    tokens, g = 4000, generator(int(offset * 2) + groups)
    logits = torch.randn(tokens, 1, width, generator=g).repeat(1, groups, 1)
    logits += torch.randn(tokens, groups, width, generator=g) * 10 ** (-7 + 3 * torch.rand(tokens, 1, 1, generator=g))
    bias = torch.full((groups, width), -offset)
    bias[:, 3] = offset
    check(logits.view(tokens, -1), bias.view(-1), 2, scores, groups=groups, keep=1, best=2)
    check(logits.view(tokens, -1), bias.view(-1), 4, scores, groups=groups, keep=max(1, groups - 1), best=2)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("best", [1, 2])
def test_groups_of_nearly_equal_scores(dgn_lib, scores, best):
    """Without a bias, and with one of nothing: sums of scores, and logits that are compared as they are."""
    tokens, groups, width, g = 4000, 4, 16, generator(9)
    logits = torch.randn(tokens, 1, width, generator=g).repeat(1, groups, 1)
    logits += torch.randn(tokens, groups, width, generator=g) * 10 ** (-8 + 4 * torch.rand(tokens, 1, 1, generator=g))
    check(logits.view(tokens, -1), torch.zeros(groups * width), 3, scores, groups=groups, keep=2, best=best)


def test_experts_closed_by_a_low_bias(dgn_lib):
    """A bias of -1e9 closes an expert as -inf does, in groups that have open ones and in groups that have none."""
    tokens, groups, width, g = 500, 4, 8, generator(10)
    logits, bias = torch.randn(tokens, groups * width, generator=g), 0.1 * torch.randn(groups * width, generator=g)
    bias[1:8] = -1e9  # one expert is open in the first group, none in the second
    bias[8:16] = -1e9
    for scores in ("softmax", "sigmoid"):
        for best in (1, 2):
            check(logits, bias, 4, scores, groups=groups, keep=2, best=best)


U = 2.0 ** -24  # half a step of float32


@pytest.mark.parametrize("num", [8, 61, 256, 600])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_gradients_of_small_scores_have_the_bits_of_float32(dgn_lib, num, scores):
    """One choice and no renormalisation: dl_e = -dw s_c s_e for the softmax's other experts, dw s (1 - s) for the sigmoid.

    Distances up to 85 from the row's largest logit, which is 0, so that the exponentials' arguments are exact: 4 u each (two
    steps of expf).  Their sum: 4 u and 15 additions after one another, a reciprocal: 20 u, which both scores have.  The
    exponential of e 4 u, four products.  48 u in all."""
    tokens, g = 64, generator(num)
    logits = -85 * torch.rand(tokens, num, generator=g)
    chosen = torch.randint(0, num, (tokens, 1), generator=g)
    logits.scatter_(1, chosen, 0.0)
    dw = torch.randn(tokens, 1, generator=g)
    if scores == "sigmoid":
        logits.scatter_(1, chosen, 170 * torch.rand(tokens, 1, generator=g) - 85)
    got = route_grad(dw.to(DEV), logits.to(DEV), chosen.int().to(DEV), scores=scores, renormalize=False).cpu().double()
    l = logits.double()
    if scores == "sigmoid":
        want = torch.zeros_like(l).scatter_(1, chosen, dw.double() * (torch.sigmoid(l) * torch.sigmoid(-l)).gather(1, chosen))
        # One exponential of the logit itself, whose argument is exact, a sum, a quotient, three products.
        assert ((got - want).abs() <= 16 * U * want.abs() + 1e-44).all()
        return
    s = torch.softmax(l, 1)
    want = -dw.double() * s.gather(1, chosen) * s
    others = torch.ones_like(l, dtype=torch.bool).scatter_(1, chosen, False)
    assert ((got - want).abs() <= 48 * U * want.abs() + 1e-44)[others].all()


@pytest.mark.parametrize("num", [8, 61, 256, 600])
def test_weights_as_they_are_have_the_bits_of_float32(dgn_lib, num):
    """Without renormalisation a weight is its score: an exponential (4 u and its argument's rounding, differences below 12)
    over a sum of positive ones (4 u + 12 u, 22 additions), two roundings."""
    logits = 2 * torch.randn(2000, num, generator=generator(num))
    indices, weights = route(logits.to(DEV), 4, renormalize=False)
    want = torch.softmax(logits.double(), 1).gather(1, indices.cpu().long())
    assert ((weights.cpu().double() - want).abs() <= 60 * U * want).all()

"""More refusals of the norm and expert operators at the C-ABI: none of them reaches a device."""

import os
import re

import pytest

from dragon_b200 import _C, experts
from tests.test_norm_experts_cpu import P, norm_args, route_args


@pytest.mark.parametrize("eps", [1e-45, 1e-40, 1.1e-38])
def test_eps_below_the_normal_numbers(dgn_lib, eps):
    """A row of zeros in e5m2 would be 0 times an infinity."""
    assert dgn_lib.dgn_rms_norm(*norm_args(eps=eps, code=_C.CODE_E5M2)) == _C.ERR_ARG
    assert b"eps" in dgn_lib.dgn_last_error_string()


@pytest.mark.parametrize("tokens", [1 << 59, 1 << 60, (1 << 62) + 4])
def test_tokens_whose_choices_pass_64_bits(dgn_lib, tokens):
    """32 choices each: a product that comes round to a small number is no answer to how many there are."""
    assert dgn_lib.dgn_expert_dispatch(P, 16, 16, P, P, P, P, tokens, 32, 8, 8, 0, None) == _C.ERR_ARG
    assert dgn_lib.dgn_expert_combine(P, P, P, P, 8, P, tokens, 32, 8, 8, _C.F32, 0, None) == _C.ERR_ARG
    assert dgn_lib.dgn_expert_combine_grad(P, 8, P, P, P, P, P, P, P, tokens, 32, 8, 8, 8, _C.F32, 0, None) == _C.ERR_ARG


def test_the_limits_are_those_of_the_header(dgn_lib):
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dgn.h")).read()
    limits = {name: int(value) for name, value in re.findall(r"#define DGN_(MAX_EXPERTS|MAX_CHOICES|MAX_GROUPS) (\d+)", header)}
    assert limits == {name: getattr(experts, name) for name in ("MAX_EXPERTS", "MAX_CHOICES", "MAX_GROUPS")}
    most = experts.MAX_EXPERTS
    for beyond in (dict(experts=most + 1, stride=most + 1), dict(k=experts.MAX_CHOICES + 1),
                   dict(experts=most, stride=most, groups=2 * experts.MAX_GROUPS)):
        assert dgn_lib.dgn_route(*route_args(**beyond)) == _C.ERR_ARG
    at = dict(experts=most, stride=most, k=experts.MAX_CHOICES, groups=experts.MAX_GROUPS)
    assert dgn_lib.dgn_route(*route_args(tokens=0, **at)) == _C.OK

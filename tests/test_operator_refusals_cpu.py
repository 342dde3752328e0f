"""More refusals of the norm and expert operators at the C-ABI: none of them reaches a device."""

import pytest

from dragon_b200 import _C
from tests.test_norm_experts_cpu import norm_args


@pytest.mark.parametrize("eps", [1e-45, 1e-40, 1.1e-38])
def test_eps_below_the_normal_numbers(dgn_lib, eps):
    """A row of zeros in e5m2 would be 0 times an infinity."""
    assert dgn_lib.dgn_rms_norm(*norm_args(eps=eps, code=_C.CODE_E5M2)) == _C.ERR_ARG
    assert b"eps" in dgn_lib.dgn_last_error_string()

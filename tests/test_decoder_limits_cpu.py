"""CPU: limits that the C entries of gated layers, cross entropy and rotary heads check before any launch, and what they
choose and lay out for calls that want some of the gradients.  No GPU call."""

import ctypes

import pytest

from tests.test_decoder_cpu import _cross, _gated, _need, _rotary
from turboadam_amd import _lib


@pytest.mark.parametrize("eps,code", [(0.0, 0), (2.0 ** -126, 0), (1.0, 0), (2.0 ** -127, 1), (2.0 ** -149, 1), (float("inf"), 1)])
def test_rotary_eps_is_zero_or_a_normal_number(eps, code):
    for backward in (0, 1):
        rc, _, msg = _need(_lib.load().tam_rotary_workspace, _rotary(eps=eps), backward)
        assert rc == code and (rc == 0 or "eps" in msg), (rc, msg)

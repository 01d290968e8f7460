"""What a call of the selective scan asks for, without a GPU."""

from __future__ import annotations

import ctypes

import pytest

from trnfft_amd import _lib


def sizes(**changes):
    desc = _lib.ScanDesc(**{**dict(dtype=1, channels=2048, groups=1, states=16, softplus=1, batch=8, tokens=4096), **changes})
    out = [ctypes.c_size_t() for _ in range(3)]
    assert _lib.lib().tfa_selective_scan_sizes(desc, *out) == _lib.TFA_OK
    return [v.value for v in out]


@pytest.mark.parametrize("states", [4, 16, 20, 64])
def test_no_room_for_gradients_that_are_not_wanted(states):
    whole, fixed = sizes(states=states), sizes(states=states, bc_fixed=1)
    assert fixed[:2] == whole[:2]
    # what adds up the gradients of b and c: two sets of states for every token, from 4 waves of 16 channels at the most (8 and 4 channels
    # above 16 and 32 states)
    filled, channels = (64, 16) if states > 32 else (32, 64) if states > 16 else (16, 64) if states > 8 else (4, 64)
    assert whole[2] - fixed[2] == 8 * 4096 * 2 * filled * 4 * (2048 // channels)


def test_gradients_that_have_no_room_are_refused():
    desc = _lib.ScanDesc(dtype=0, channels=8, groups=2, states=4, softplus=1, batch=1, tokens=4, bc_fixed=1)
    far = 4096
    for name in "bc":
        grads = _lib.ScanGrads(grad_y=far, **{name: far})
        assert _lib.lib().tfa_selective_scan_backward(desc, far, far, far, far, far, None, None, None, None, None, None, grads, far,
                                                      None) == _lib.TFA_ERR_INVALID
        assert b"bc_fixed" in _lib.lib().tfa_last_error()

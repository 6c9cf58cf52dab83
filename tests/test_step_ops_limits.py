"""CPU: arguments of the scheduler-step entry points that only their values
rule out, refused before any CUDA call."""

import ctypes

import pytest

ARG = 1


@pytest.mark.parametrize("theta,status", [(1e-40, ARG), (1e-45, ARG), (1e-38, 0), (1.0, 0), (3e38, 0)])
def test_rope_axes_refuses_a_theta_whose_frequencies_overflow(theta, status):
    """f_d = theta^(-d / half) has to be a finite fp32: its fraction of a turn
    is what the angles are computed from."""
    from kessie_b200 import _lib
    lib = _lib.load()
    sections = (ctypes.c_int * 2)(40, 24)
    for _ in range(2):                                                # a refused table is not kept
        got = lib.kessie_rope_axes_remap_v2(16, 256, 128, 16, 256, 128, 1, 0, 2, 128, None, 0, 16, 4, sections, 2, 0,
                                            theta, None)
        assert got == status
        if status:
            assert "theta" in _lib.last_error()[1]

"""What the sequence-tower operators' C entries and Python calls take and refuse at the ends of their ranges: decided
before the GPU is touched."""
import pytest
import torch

from dssm_amd import _lib, api

Z = torch.zeros
P = 4096  # an aligned address that is never read: the checks come first
F32, BF = _lib.DSSM_F32, _lib.DSSM_BF16


def test_zero_rows_do_nothing():
    lib = _lib.load()
    for dtype in (F32, BF):
        assert lib.dssm_linear_recurrence(0, 0, 4, 0, 0, 4, dtype, 0, 0, 0, 3, 4, 0, 0, 0, 4, 0, 0, 0, 0, 0) == 0
        assert lib.dssm_linear_recurrence_bwd(0, 0, 4, 0, 0, 4, dtype, 0, 0, 0, 0, 0, 0, 0, 3, 4, 0, 0, 0, 4, 0, 0, 4, 0, 0, 0, 0) == 0
        assert lib.dssm_linear_recurrence_step(0, 4, 0, 4, dtype, 0, 4, 0, 4, 0, 4, 0) == 0
        assert lib.dssm_linear_recurrence_ws_bytes(0, 3, 4, dtype) == 0
    # no rows of no steps or no channels, of a strange type, or fewer than none
    assert lib.dssm_linear_recurrence(0, 0, 4, 0, 0, 4, F32, 0, 0, 0, 0, 4, 0, 0, 0, 4, 0, 0, 0, 0, 0) == -1
    assert lib.dssm_linear_recurrence(0, 0, 4, 0, 0, 4, F32, 0, 0, 0, 3, 0, 0, 0, 0, 4, 0, 0, 0, 0, 0) == -1
    assert lib.dssm_linear_recurrence_step(0, 4, 0, 4, 7, 0, 4, 0, 4, 0, 4, 0) == -1
    assert lib.dssm_linear_recurrence_step(P, 4, P, 4, F32, P, 4, P, 4, -1, 4, 0) == -1

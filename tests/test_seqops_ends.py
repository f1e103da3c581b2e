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


@pytest.mark.parametrize("eps", [0.0, -1e-6, float("nan"), float("inf"), 2.0 ** -150, 1e-46, 3.5e38])
def test_eps_is_positive_as_a_float32(eps):
    """An eps that is 0 as fp32 would make a row of zeros NaN."""
    for call in (api.rms_norm, api.rms_norm_blocks8):
        with pytest.raises(ValueError, match="eps"):
            call(Z(3, 4), Z(4), None, eps)
    lib = _lib.load()
    assert lib.dssm_rms_norm(0, 4, 0, 0, P, 0, 4, F32, eps, 0, 4, 0, 0, 0, 0) == -1
    assert lib.dssm_rms_norm_blocks8(0, 4, 0, 0, P, 0, 4, F32, eps, 0, 0, 0, 0, 0, 0) == -1


@pytest.mark.parametrize("eps", [1e-45, 1e-6, 3.4e38])
def test_eps_that_a_float32_holds_is_taken(eps):
    with pytest.raises(ValueError, match="GPU"):  # past the check of eps, to the one of the device
        api.rms_norm(Z(3, 4), Z(4), None, eps)
    assert _lib.load().dssm_rms_norm(0, 4, 0, 0, P, 0, 4, F32, eps, 0, 4, 0, 0, 0, 0) == 0


def test_the_8_bit_form_is_as_wide_as_the_product():
    """Rows that blocks8_matmul multiplies can be laid out: up to 2^22 columns, and no more."""
    wide = Z(1, 1).expand(1, 1 << 22)
    with pytest.raises(ValueError, match="GPU"):
        api.quantize_blocks8(wide)
    with pytest.raises(ValueError, match="columns"):
        api.quantize_blocks8(Z(1, 1).expand(1, (1 << 22) + 1))
    b = api.Blocks8(Z(1, 1 << 22, dtype=torch.uint8).view(torch.float8_e4m3fn),
                    Z(1, 1 << 15, dtype=torch.uint8).view(torch.float8_e8m0fnu), 1 << 22)
    with pytest.raises(ValueError, match="GPU"):
        api.dequantize_blocks8(b)
    lib = _lib.load()
    for cols, rc in ((16385, 0), (1 << 22, 0), ((1 << 22) + 1, -1)):
        assert lib.dssm_quantize_blocks8(0, cols, 0, cols, F32, 0, 0, 0) == rc
        assert lib.dssm_dequantize_blocks8(0, 0, 0, cols, 0, cols, F32, 0) == rc


def test_sizes_that_an_int_would_cut_are_refused():
    """2^32 + 4 columns are not 4."""
    i = Z(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="columns"):
        api.embedding_lookup(Z(1, 1).expand(5, (1 << 32) + 4), i)
    with pytest.raises(ValueError, match="out of range"):
        api.embedding_grad(Z(1, 1).expand(3, (1 << 32) + 4), i, 5)
    with pytest.raises(ValueError, match="out of range"):
        api.embedding_grad(Z(3, 4), i, (1 << 64) + 5)
    with pytest.raises(ValueError, match="out of range"):
        api.embedding_grad(Z(1, 1).expand(3, (1 << 20) + 1), i, 5)
    with pytest.raises(ValueError, match="GPU"):
        api.embedding_lookup(Z(1, 1).expand(5, 1 << 30), i)
    # columns whose numbers would pass 2^31 on their way
    assert _lib.load().dssm_embedding_lookup(P, F32, 2 ** 31 - 1, 4, 2 ** 31 - 1, 0, 0, 0, 1.0, 0, F32, 0) == -1
    assert _lib.load().dssm_embedding_lookup(P, F32, 1 << 30, 4, 1 << 30, 0, 0, 0, 1.0, 0, F32, 0) == 0


def test_a_steps_rows_that_overlap_are_refused():
    """Two rows of one state would be moved on by two lanes at once."""
    step = _lib.load().dssm_linear_recurrence_step
    assert step(P, 4, P, 4, F32, P, 3, P, 4, 2, 4, 0) == -1
    assert step(P, 4, P, 4, F32, P, 0, P, 4, 2, 4, 0) == -1
    assert step(P, 4, P, 4, F32, P, 4, P, -3, 2, 4, 0) == -1
    assert b"overlap" in _lib.load().dssm_last_error()


def test_no_recurrence_kernel_is_built_that_no_cut_takes():
    """Segments of time are summed by eight waves or not at all, so no other kernel for it is in the library."""
    import re

    names = re.findall(rb"k_recur_[fb]wdI[^_]*?Li\dELi(\d)ELb([01])E", open(_lib.LIB_PATH, "rb").read())
    assert {(int(nw), int(sums)) for nw, sums in names} == {(1, 0), (4, 0), (8, 0), (8, 1)}


def test_more_rows_than_a_call_takes_are_a_value_error():
    """As the module says of shapes that do not fit, before anything runs."""
    tall, w = Z(1, 1).expand(1 << 31, 1), Z(1)
    for call in (lambda: api.rms_norm(tall, w), lambda: api.rms_norm_blocks8(tall, w), lambda: api.quantize_blocks8(tall),
                 lambda: api.rms_norm_grad(tall, tall, w, Z(1).expand(1 << 31))):
        with pytest.raises(ValueError, match="rows"):
            call()
    with pytest.raises(ValueError, match="GPU"):
        api.quantize_blocks8(Z(1, 1).expand((1 << 31) - 1, 1))

"""The sequence-tower operators' checks of arguments: they come before the GPU is touched."""
import pytest
import torch

from dssm_amd import _lib, api

Z = torch.zeros


def b8(rows, cols, kp=None):
    kp = -(-cols // 128) * 128 if kp is None else kp
    return api.Blocks8(Z(rows, kp, dtype=torch.uint8).view(torch.float8_e4m3fn),
                       Z(rows, kp // 128, dtype=torch.uint8).view(torch.float8_e8m0fnu), cols)


I32, F64, BF = torch.int32, torch.float64, torch.bfloat16
CASES = {
    "table rank": (ValueError, lambda: api.embedding_lookup(Z(4), Z(3, dtype=I32))),
    "table empty": (ValueError, lambda: api.embedding_lookup(Z(0, 4), Z(3, dtype=I32))),
    "table type": (TypeError, lambda: api.embedding_lookup(Z(4, 4, dtype=F64), Z(3, dtype=I32))),
    "out type": (TypeError, lambda: api.embedding_lookup(Z(4, 4), Z(3, dtype=I32), 1.0, F64)),
    "ids type": (TypeError, lambda: api.embedding_lookup(Z(4, 4), Z(3))),
    "lookup on the CPU": (ValueError, lambda: api.embedding_lookup(Z(4, 4), Z(3, dtype=I32))),
    "dy shape": (ValueError, lambda: api.embedding_grad(Z(3, 4), Z(2, dtype=I32), 5)),
    "dy rank": (ValueError, lambda: api.embedding_grad(Z(3), Z(3, dtype=I32), 5)),
    "dy no columns": (ValueError, lambda: api.embedding_grad(Z(3, 0), Z(3, dtype=I32), 5)),
    "no words": (ValueError, lambda: api.embedding_grad(Z(3, 4), Z(3, dtype=I32), 0)),
    "too many words": (ValueError, lambda: api.embedding_grad(Z(3, 4), Z(3, dtype=I32), 1 << 30)),
    "grad on the CPU": (ValueError, lambda: api.embedding_grad(Z(3, 4), Z(3, dtype=I32), 5)),
    "gate rank": (ValueError, lambda: api.linear_recurrence(Z(3, 4), Z(3, 4))),
    "gate and cand differ": (ValueError, lambda: api.linear_recurrence(Z(3, 4, 2), Z(3, 4, 3))),
    "gate and cand types": (TypeError, lambda: api.linear_recurrence(Z(3, 4, 2), Z(3, 4, 2, dtype=BF))),
    "no channels": (ValueError, lambda: api.linear_recurrence(Z(3, 4, 0), Z(3, 4, 0))),
    "recurrence type": (TypeError, lambda: api.linear_recurrence(Z(3, 4, 2, dtype=F64), Z(3, 4, 2, dtype=F64))),
    "lens shape": (ValueError, lambda: api.linear_recurrence(Z(3, 4, 2), Z(3, 4, 2), Z(2, dtype=I32))),
    "lens type": (ValueError, lambda: api.linear_recurrence(Z(3, 4, 2), Z(3, 4, 2), Z(3))),
    "h0 shape": (ValueError, lambda: api.linear_recurrence(Z(3, 4, 2), Z(3, 4, 2), None, Z(3, 3))),
    "h0 type": (ValueError, lambda: api.linear_recurrence(Z(3, 4, 2), Z(3, 4, 2), None, Z(3, 2, dtype=BF))),
    "recurrence on the CPU": (ValueError, lambda: api.linear_recurrence(Z(3, 4, 2), Z(3, 4, 2))),
    "states shape": (ValueError, lambda: api.linear_recurrence_grad(Z(3, 17, 2), Z(3, 17, 2), Z(1, 3, 2), None)),
    "dh type": (ValueError, lambda: api.linear_recurrence_grad(Z(3, 4, 2), Z(3, 4, 2), Z(1, 3, 2), Z(3, 4, 2, dtype=BF))),
    "dlast shape": (ValueError, lambda: api.linear_recurrence_grad(Z(3, 4, 2), Z(3, 4, 2), Z(1, 3, 2), None, Z(2, 2))),
    "step state type": (ValueError, lambda: api.linear_recurrence_step(Z(3, 2, dtype=BF), Z(3, 2, dtype=BF), Z(3, 2, dtype=BF))),
    "step state rows": (ValueError, lambda: api.linear_recurrence_step(Z(3, 2), Z(3, 2), Z(1, 2).expand(3, 2))),
    "step state columns": (ValueError, lambda: api.linear_recurrence_step(Z(3, 2), Z(3, 2), Z(2, 3).t())),
    "step rank": (ValueError, lambda: api.linear_recurrence_step(Z(3, 4, 2), Z(3, 4, 2), Z(3, 2))),
    "norm type": (TypeError, lambda: api.rms_norm(Z(3, 4, dtype=F64), Z(4))),
    "norm weight": (ValueError, lambda: api.rms_norm(Z(3, 4), Z(3))),
    "norm weight type": (ValueError, lambda: api.rms_norm(Z(3, 4, dtype=BF), Z(4, dtype=BF))),
    "norm residual": (ValueError, lambda: api.rms_norm(Z(3, 4), Z(4), Z(3, 5))),
    "norm eps": (ValueError, lambda: api.rms_norm(Z(3, 4), Z(4), None, 0.0)),
    "norm columns": (ValueError, lambda: api.rms_norm(Z(1, 16385), Z(16385))),
    "norm no columns": (ValueError, lambda: api.rms_norm(Z(3, 0), Z(0))),
    "norm8 weight": (ValueError, lambda: api.rms_norm_blocks8(Z(3, 4), Z(3))),
    "norm grad s": (ValueError, lambda: api.rms_norm_grad(Z(3, 4), Z(3, 5), Z(4), Z(3))),
    "norm grad rstd": (ValueError, lambda: api.rms_norm_grad(Z(3, 4), Z(3, 4), Z(4), Z(4))),
    "norm grad ds": (ValueError, lambda: api.rms_norm_grad(Z(3, 4), Z(3, 4), Z(4), Z(3), Z(3, 4, dtype=BF))),
    "quantize type": (TypeError, lambda: api.quantize_blocks8(Z(3, 4, dtype=I32))),
    "quantize columns": (ValueError, lambda: api.quantize_blocks8(Z(1, 16385))),
    "dequantize type": (TypeError, lambda: api.dequantize_blocks8(b8(3, 4), I32)),
    "blocks shape": (ValueError, lambda: api.dequantize_blocks8(b8(3, 129, 128))),
    "blocks type": (TypeError, lambda: api.blocks8_matmul(b8(3, 4)._replace(q=Z(3, 128)), b8(2, 4))),
    "blocks strides": (ValueError, lambda: api.blocks8_matmul(b8(3, 256), b8(2, 256)._replace(
        scale=Z(2, 2, dtype=torch.uint8).t().view(torch.float8_e8m0fnu)))),
    "matmul columns": (ValueError, lambda: api.blocks8_matmul(b8(3, 4), b8(2, 5))),
    "matmul bias": (ValueError, lambda: api.blocks8_matmul(b8(3, 4), b8(2, 4), Z(3))),
    "matmul type": (TypeError, lambda: api.blocks8_matmul(b8(3, 4), b8(2, 4), None, F64)),
    "matmul to fp32": (TypeError, lambda: api.blocks8_matmul(b8(3, 4), b8(2, 4), None, torch.float32)),
    "matmul on the CPU": (ValueError, lambda: api.blocks8_matmul(b8(3, 4), b8(2, 4))),
}


@pytest.mark.parametrize("name", CASES)
def test_refused(name):
    kind, call = CASES[name]
    with pytest.raises(kind):
        call()


def test_c_entries_refuse():
    """The C entries check what reaches them: null pointers, leading dimensions, types, workspaces."""
    lib = _lib.load()
    p = 4096  # an aligned address that is never read: the checks come first
    L, B, F = _lib.DSSM_F32, _lib.DSSM_BF16, lib
    bad = [
        F.dssm_embedding_lookup(0, L, 4, 4, 4, p, 0, 3, 1.0, p, L, 0),
        F.dssm_embedding_lookup(p, L, 3, 4, 4, p, 0, 3, 1.0, p, L, 0),
        F.dssm_embedding_lookup(p, 2, 4, 4, 4, p, 0, 3, 1.0, p, L, 0),
        F.dssm_embedding_grad(p, B, 4, p, 0, 4000, 4, 4, 1.0, p, p, 16, 0),
        F.dssm_embedding_grad(p, B, 4, p, 0, 3, 4, 4, 1.0, p + 4, p, 1 << 20, 0),
        F.dssm_embedding_grad(p, B, 3, p, 0, 3, 4, 4, 1.0, p, p, 1 << 20, 0),
        F.dssm_linear_recurrence(p, 8, 4, 0, 8, 4, B, 0, 0, 2, 2, 4, 0, p, 8, 4, p, 0, 0, 0, 0),
        F.dssm_linear_recurrence(p, 8, 4, p, 8, 4, 7, 0, 0, 2, 2, 4, 0, p, 8, 4, p, 0, 0, 0, 0),
        F.dssm_linear_recurrence(p, 0, 4, p, 0, 4, B, 0, 0, 1, 1 << 16, 4, 0, p, 0, 4, p, 0, 0, 0, 0),
        F.dssm_linear_recurrence_bwd(p, 8, 4, p, 8, 4, B, 0, 0, p, 8, 4, 0, 2, 2, 4, 0, p, 8, 4, p, 8, 4, 0, 0, 0, 0),
        F.dssm_linear_recurrence_step(p, 4, p, 4, B, 0, 4, p, 4, 2, 4, 0),
        F.dssm_rms_norm(p, 4, 0, 0, p, 2, 16385, L, 1e-6, p, 16385, 0, 0, 0, 0),
        F.dssm_rms_norm(p, 3, 0, 0, p, 2, 4, L, 1e-6, p, 4, 0, 0, 0, 0),
        F.dssm_rms_norm_blocks8(p, 4, 0, 0, p, 2, 4, L, 1e-6, p + 8, p, 0, 0, 0, 0),
        F.dssm_rms_norm_bwd(p, 4, p, 4, p, p, 0, 0, 2, 4, L, p, 4, p, p, 4, 0),
        F.dssm_quantize_blocks8(p, 4, 2, 4, L, p, 0, 0),
        F.dssm_dequantize_blocks8(p, p, 2, 4, p, 3, L, 0),
        F.dssm_blocks8_matmul(p, p, p, p, 2, 2, 0, 0, p, 2, B, 0),
        F.dssm_blocks8_matmul(p + 8, p, p, p, 2, 2, 4, 0, p, 2, B, 0),
        F.dssm_blocks8_matmul(p, p, p, p, 2, 2, 4, 0, p, 1, B, 0),
        F.dssm_blocks8_matmul(p, p, p, p, 2, 2, 4, 0, p, 2, L, 0),
    ]
    assert bad == [-1] * len(bad)
    assert lib.dssm_last_error()
    assert lib.dssm_embedding_grad_ws_bytes(1 << 31, 4, 4, L) == 0
    assert lib.dssm_rms_norm_bwd_ws_bytes(4, 16385) == 0


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    p = 4096
    assert lib.dssm_embedding_lookup(p, 0, 4, 4, 4, 0, 0, 0, 1.0, 0, 0, 0) == 0
    assert lib.dssm_rms_norm(0, 4, 0, 0, p, 0, 4, 0, 1e-6, 0, 4, 0, 0, 0, 0) == 0
    assert lib.dssm_quantize_blocks8(0, 4, 0, 4, 0, 0, 0, 0) == 0
    assert lib.dssm_blocks8_matmul(0, 0, 0, 0, 0, 2, 4, 0, 0, 2, _lib.DSSM_BF16, 0) == 0


def test_the_states_pieces_are_the_librarys():
    import os
    import re

    from dssm_amd import seqops
    head = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dssm.h")
    assert int(re.search(r"#define DSSM_RECUR_PIECE (\d+)", open(head).read()).group(1)) == seqops._PIECE

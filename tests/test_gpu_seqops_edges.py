"""The sequence-tower operators at the ends of their ranges: infinities among the values that count, the largest
magnitudes, many digits of a token, wide rows, every call in a captured graph."""
import pytest
import torch

from dssm_amd import api
from tests import seqops_ref as ref
from tests.test_gpu_seqops import BF, F16, F32, gen, inputs, near, rounded

pytestmark = pytest.mark.gpu
INF = float("inf")


# ---- recurrence --------------------------------------------------------------------------------------
def same_ends(got, want, tol):
    """NaN where want is NaN, infinite (with its sign) where it is infinite, and near it everywhere else"""
    got = got.cpu()
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), (kind, int(kind(got).sum()), int(kind(want).sum()))
    fin = torch.isfinite(want)
    rounded(got[fin], want[fin], tol[fin])


# one wave a row; four and eight waves over time; segments of time.  Eight gates of -14 make a product of u of 2^-161,
# below fp32's smallest value, while u itself is an ordinary number
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("R,T,H,dtype", [(2100, 18, 64, F32), (2, 25, 8, BF), (2, 40, 9, F32), (3, 600, 8, F16), (2, 2500, 70, BF),
                                         (2, 2500, 12, F32)])
def test_infinite_states_stay_infinite(device, R, T, H, dtype, reverse):
    """Infinite states, candidates and gradients that count, under gates that all but forget: the same whichever way
    the work is cut, which is as the formulas have it step by step."""
    gate, cand, lens, h0, g = inputs(R, T, H, dtype, T + H)
    gate[:, T // 4: 3 * T // 4] = -14.0
    h0[:, 0], h0[:, 1] = INF, -INF
    cand[:, T // 3, 2], cand[:, 2, 3] = INF, -INF
    dh, dlast = torch.randn(R, T, H, generator=g).to(dtype), torch.randn(R, H, generator=g)
    dlast[:, 4], dlast[:, 5] = INF, -INF
    dh[:, T // 2, 6] = INF
    dev = [x.to(device) for x in (gate, cand, lens, h0, dh, dlast)]
    h, last, states = api.linear_recurrence(dev[0], dev[1], dev[2], dev[3], reverse, save=True)
    wh, wl, _, eh, el = ref.recurrence(gate, cand, lens, h0, reverse)
    assert torch.isinf(wl[1, :4]).all() and torch.isfinite(wl[:, 4:]).all()  # (row 1 has all steps)
    same_ends(h, wh, eh)
    same_ends(last, wl, el)
    dg, dc, d0 = api.linear_recurrence_grad(dev[0], dev[1], states, dev[4], dev[5], dev[2], reverse)
    wg, wc, w0, eg, ec, e0 = ref.recurrence_grad(gate, cand, dh, dlast, lens, h0, reverse)
    assert torch.isinf(w0[1, 4:7]).all() and torch.isfinite(w0[:, [0, 1, 2, 3, 7]]).all()
    same_ends(dg, wg, eg)
    same_ends(dc, wc, ec)
    same_ends(d0, w0, e0)

"""The sequence-tower operators at the ends of their ranges: infinities among the values that count, the largest
magnitudes, many digits of a token, wide rows, every call in a captured graph."""
import pytest
import torch

from dssm_amd import api
from tests import seqops_ref as ref
from tests.test_gpu_seqops import BF, F16, F32, NORM, U, check_blocks, gen, inputs, near, product, rounded

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


# ---- 8-bit form --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("rows,cols", [(3, 16385), (2, 16384 * 2), (700, 16391), (2, 40000), (1, 16384 * 3 + 129)])
def test_rows_wider_than_the_norms(device, rows, cols, dtype):
    """The 8-bit form of rows of more than 16384 columns, between rows' ends that are NaN."""
    g = gen(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[0, 16384:16512] = 0  # the first block behind a stretch
    x[rows - 1, :128] = 2.0 ** -12
    around = torch.full((rows, cols + 9), float("nan"), dtype=dtype, device=device)
    around[:, 5:5 + cols] = x.to(device)
    b = api.quantize_blocks8(around[:, 5:5 + cols])
    check_blocks(b, x.double(), torch.zeros(rows, cols, dtype=torch.float64))
    # block by block it is what rows of the norm's width have
    for c0 in range(0, cols, 16384):
        part = api.quantize_blocks8(x[:, c0:c0 + 16384].contiguous().to(device))
        kp = part.q.shape[1]
        assert torch.equal(part.q.view(torch.uint8), b.q.view(torch.uint8)[:, c0:c0 + kp])
        assert torch.equal(part.scale.view(torch.uint8), b.scale.view(torch.uint8)[:, c0 // 128:(c0 + kp) // 128])


@pytest.mark.parametrize("M,N,K", [(5, 40, 20000), (130, 300, 16384 + 77), (600, 700, 33000)])
def test_product_of_wide_rows(device, M, N, K):
    g = gen(K)
    a = api.quantize_blocks8(torch.randn(M, K, generator=g).to(device))
    w = api.quantize_blocks8((torch.randn(N, K, generator=g) * K ** -0.5).to(device))
    bias = torch.randn(N, generator=g)
    want, tol = product(a, w, bias, K)
    rounded(api.blocks8_matmul(a, w, bias.to(device)), want, tol)


# ---- norm --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("cols", [1, 7, 40, 200, 500, 1000, 2000, 4100, 8000, 16384])
def test_norm_of_the_largest_and_smallest_rows(device, cols, dtype):
    """Rows whose squares, and whose products with the weight, are past fp32's range; rows beside them as ever."""
    g = gen(cols)
    x = torch.randn(13, cols, generator=g).to(dtype)
    w = torch.rand(cols, generator=g) + 0.5
    w[cols // 2] = 1e12
    dy, ds = torch.randn(13, cols, generator=g).to(dtype), torch.randn(13, cols, generator=g).to(dtype)
    plain, _, _ = api.rms_norm(x.to(device), w.to(device))
    plain8, _ = api.rms_norm_blocks8(x.to(device), w.to(device))
    big = {1: 2.0 ** 60, 3: 2.0 ** 64, 4: 2.0 ** 100, 6: 2.0 ** 120, 9: 2.0 ** 125, 12: 2.0 ** -90}
    for r, f in big.items():
        x[r] *= f
    x[9] = x[9].sign() * 2.0 ** 127  # the largest power of two: the squares' sum is 2^254 times the columns
    y, s, rstd = api.rms_norm(x.to(device), w.to(device))
    eps = float(torch.tensor(1e-6))
    wy, ws, wr = ref.norm(x, w, None, eps)
    rounded(y, wy, NORM * wy.abs())
    rounded(rstd, wr[:, 0], NORM * wr[:, 0])
    y8, _ = api.rms_norm_blocks8(x.to(device), w.to(device))
    check_blocks(y8, wy, NORM * wy.abs())
    others = [r for r in range(13) if r not in big]
    assert torch.equal(y[others], plain[others])
    assert torch.equal(y8.q.view(torch.uint8)[others], plain8.q.view(torch.uint8)[others])
    dx, dw = api.rms_norm_grad(dy.to(device), s, w.to(device), rstd, ds.to(device))
    wx, wdw, mx, mw = ref.norm_grad(dy, ws, w, wr, ds)
    rounded(dx, wx, 2 * NORM * mx)
    near(dw, wdw, 53 * U * mw)
    # an eps as small as the squares of such rows
    x[12] = (torch.randn(cols, generator=g) * 2.0 ** -74).to(dtype)
    y, _, rstd = api.rms_norm(x.to(device), w.to(device), None, 2.0 ** -147)
    wy, _, wr = ref.norm(x, w, None, 2.0 ** -147)
    rounded(y, wy, NORM * wy.abs())
    rounded(rstd, wr[:, 0], NORM * wr[:, 0])


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("cols", [5, 96, 300, 1500, 9000])
def test_norm_to_8_bits_keeps_what_its_gradient_takes(device, cols, dtype):
    g = gen(cols)
    x, res, dy = (torch.randn(2, 7, cols, generator=g).to(dtype).to(device) for _ in range(3))
    w = (torch.rand(cols, generator=g) + 0.5).to(device)
    for residual in (res, None):
        _, s, rstd = api.rms_norm(x, w, residual)
        b, s8 = api.rms_norm_blocks8(x, w, residual)
        b2, s2, rstd2 = api.rms_norm_blocks8(x, w, residual, save=True)
        assert torch.equal(s2, s) and torch.equal(s8, s) and torch.equal(rstd2, rstd)
        assert torch.equal(b2.q.view(torch.uint8), b.q.view(torch.uint8))
        for p, q in zip(api.rms_norm_grad(dy, s2, w, rstd2), api.rms_norm_grad(dy, s, w, rstd)):
            assert torch.equal(p, q)
    assert api.rms_norm_blocks8(x[:0], w, save=True)[2].shape == (0,)

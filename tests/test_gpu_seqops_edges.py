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


# ---- embedding ---------------------------------------------------------------------------------------
# (bits a digit, pairs a thread, sums of the counts): vocabularies from 2^20 words on take three digits, the third pass
# of which leaves the pairs where the first one did; ids outside the table sort behind all others in every digit
@pytest.mark.parametrize("n,V,E", [(4097, 1 << 20, 3), (70000, (1 << 20) + 5, 2), (600001, (1 << 21) - 1, 1),
                                   (2200003, (1 << 20) + 1, 1), (5000, (1 << 27) + 3, 1), (70001, (1 << 28) - 1, 1),
                                   (300001, (1 << 29) + 7, 1), (4500, (1 << 30) - 1, 1)])
def test_lookup_grad_of_three_digits(device, n, V, E):
    g = torch.Generator(device).manual_seed(n)
    dy = torch.randn(n, E, generator=g, device=device)
    ids = (torch.rand(n, generator=g, device=device, dtype=torch.float64) ** 6 * V).long().clamp_(0, V - 1)
    ids[::7] = ids[0]  # a token in all parts of the list
    ids[3::11] = V - 1 - ids[3::11] // 2  # and large ones
    ids[5::13], ids[6::17] = -1, V
    dy[(ids < 0) | (ids >= V)] = float("nan")  # never read
    got = api.embedding_grad(dy, ids.to(torch.int32) if n % 2 else ids, V, 0.5)
    ok = (ids >= 0) & (ids < V)
    words, at = torch.unique(ids[ok], return_inverse=True)
    want, mag, count = ref.lookup_grad(dy[ok].cpu(), at.cpu(), len(words), 0.5)
    near(got[words], want, U * (count + 2) * mag)
    got[words] = 0
    assert not got.any()  # every other word's row is zero


# ---- graphs ------------------------------------------------------------------------------------------
def test_every_call_in_one_graph(device):
    """Each call captured, several replays with other inputs and eager work between them, against the eager results."""
    g = torch.Generator(device).manual_seed(4)
    R, T, H, E, V = 3, 2400, 64, 130, 700
    normal = lambda *s: torch.randn(*s, generator=g, device=device)  # noqa: E731
    ids = torch.randint(0, V, (5000,), generator=g, device=device)
    few = torch.randint(0, V, (9,), generator=g, device=device, dtype=torch.int32)
    lens = torch.randint(0, T + 1, (R,), generator=g, device=device)
    floats = dict(table=normal(V, E), dy=normal(5000, E), gate=normal(R, T, H), cand=normal(R, T, H), dh=normal(R, T, H),
                  state=normal(R, H), x=normal(300, E), res=normal(300, E), w=normal(E), lin=normal(90, E), bias=normal(90))

    def work(a):
        out = [api.embedding_lookup(a["table"], ids, 2.0, BF), api.embedding_grad(a["dy"], ids, V),
               api.embedding_grad(a["dy"][:9], few, V)]
        h, last, states = api.linear_recurrence(a["gate"], a["cand"], lens, a["state"], True, save=True)
        out += [h, last, *api.linear_recurrence_grad(a["gate"], a["cand"], states, a["dh"], a["state"], lens, True)]
        running = a["state"].clone()
        out += [api.linear_recurrence_step(a["gate"][:, 0], a["cand"][:, 1], running), running]
        y, s, rstd = api.rms_norm(a["x"], a["w"], a["res"])
        out += [y, s, rstd, *api.rms_norm_grad(y, s, a["w"], rstd, a["x"])]
        b, s8, rstd8 = api.rms_norm_blocks8(a["x"], a["w"], a["res"], save=True)
        lin = api.quantize_blocks8(a["lin"])
        wide = api.quantize_blocks8(a["dy"].view(-1, 65000))
        out += [b.q.view(torch.uint8), b.scale.view(torch.uint8), s8, rstd8, lin.q.view(torch.uint8),
                lin.scale.view(torch.uint8), api.dequantize_blocks8(b, F32), api.dequantize_blocks8(wide, BF)]
        out += [api.blocks8_matmul(b, lin, a["bias"], F16), api.blocks8_matmul(lin, b)]
        return out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(floats)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work(floats)
    for k in range(4):
        for v in floats.values():
            v.copy_(torch.randn(v.shape, generator=g, device=device))
        for c in captured:
            c.zero_()
        want = [w.clone() for w in work(floats)]
        graph.replay()
        eager = work(floats)
        torch.cuda.synchronize()
        for i, (a, b, c) in enumerate(zip(captured, want, eager)):
            assert torch.equal(a, b) and torch.equal(a, c), (k, i)


@pytest.mark.parametrize("M,N,K", [(5, 20, 700), (300, 260, 700), (64, 1000, 1100), (2100, 2100, 260)])
def test_product_of_the_furthest_scales(device, M, N, K):
    """Scales at both ends of their range: of rows in fp32's subnormals, of the largest, and results near both ends."""
    g = gen(M)
    for ex, ey in ((-136, 120), (120, -136), (-120, -20), (100, 20), (-60, -60)):
        x, y = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g) * 2.0 ** ey
        a, w = (api.quantize_blocks8(t.to(device)) for t in (x * 2.0 ** (ex // 2) * 2.0 ** (ex - ex // 2), y))
        want, tol = product(a, w, None, K)
        rounded(api.blocks8_matmul(a, w), want, tol)

"""The sequence-tower operators (dssm_amd/seqops.py) on the GPU against their formulas in float64
(tests/seqops_ref.py), at the sizes and masks where they can go wrong.  Tolerances are sums of roundings, written
where they are used; `stored` is the one rounding into the output's type."""
import pytest
import torch

from dssm_amd import _lib, api, seqops
from tests import seqops_ref as ref

pytestmark = pytest.mark.gpu

F32, BF, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF, F16]
U = 2.0 ** -24  # half a unit of fp32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def near(got, want, tol):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape
    bad = ~(((got - want).abs() <= tol) | (got == want))
    assert not bad.any(), (int(bad.sum()), (got - want).abs().max(), got[bad][:4], want[bad][:4])


def rounded(got, want, tol):
    """got, stored once, is within tol of want before its rounding"""
    near(got, want, tol + ref.stored(want.abs() + tol, got.dtype))


# ---- embedding ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,out", [(F32, BF), (F32, F32), (BF, BF), (F16, F32), (BF, F16), (F32, F16)])
@pytest.mark.parametrize("n,V,E", [(1, 1, 1), (3, 7, 4), (77, 50, 33), (130, 1000, 128), (5, 9, 513), (1031, 300, 100),
                                   (300, 20, 17), (90, 40, 131), (60, 8, 39), (50, 9, 11)])
def test_lookup(device, n, V, E, dtype, out):
    g = gen(n * 1000 + E)
    table = torch.randn(V, E, generator=g).to(dtype)
    ids = torch.randint(0, V, (n,), generator=g)
    got = api.embedding_lookup(table.to(device), ids.to(device), 1.7, out)
    assert got.dtype == out
    want = ref.lookup(table, ids, float(torch.tensor(1.7)))  # the scale is an fp32 number
    rounded(got, want, U * want.abs())  # one fp32 product


def test_lookup_shapes_and_strange_ids(device):
    g = gen(3)
    table = torch.randn(11, 24, generator=g).to(device)
    ids = torch.tensor([[0, -1, 10], [11, 3, -2 ** 31]], dtype=torch.int32)
    got = api.embedding_lookup(table, ids.to(device), 2.0)
    assert got.shape == (2, 3, 24)
    near(got, ref.lookup(table.cpu(), ids, 2.0), 0.0)
    big = torch.tensor([2 ** 40, 5, -2 ** 60])  # int64 ids that would wrap to valid ones in 32 bits
    got = api.embedding_lookup(table, big.to(device))
    near(got, ref.lookup(table.cpu(), big, 1.0), 0.0)
    assert api.embedding_lookup(table, torch.zeros(0, 4, dtype=torch.int64, device=device)).shape == (0, 4, 24)
    # a table of strided rows, and ids of another order
    part = table[:, 5:18]
    ids = torch.arange(10, device=device).view(2, 5).t()
    near(api.embedding_lookup(part, ids), ref.lookup(part.cpu(), ids.cpu(), 1.0), 0.0)
    # an infinity in a row that no id names stays there
    table[4] = float("inf")
    assert torch.isfinite(api.embedding_lookup(table, torch.tensor([3, 5, -1], device=device))).all()


def check_grad(device, dy, ids, V, scale=0.5):
    got = api.embedding_grad(dy.to(device), ids.to(device), V, scale)
    want, mag, count = ref.lookup_grad(dy, ids, V, scale)
    near(got, want, U * (count + 2) * mag)  # count - 1 fp32 additions in any order, the scale, and one to spare
    assert (got.cpu()[count[:, 0] == 0] == 0).all()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,E", [(1, 1, 1), (2, 5, 3), (31, 3, 8), (32, 3, 8), (33, 1, 7), (64, 2, 16), (100, 1, 1), (1000, 40, 100),
                                   (4096, 700, 20), (4097, 700, 20), (5000, 1023, 9), (9000, 1024, 5), (12345, 70000, 12),
                                   (5000, 300, 33), (3000, 200, 131), (2000, 90, 17), (700, 60, 513), (6000, 7, 39),
                                   (3, 1 << 21, 2)])
def test_lookup_grad(device, n, V, E, dtype):
    g = gen(n + V + E)
    dy = torch.randn(n, E, generator=g).to(dtype)
    ids = (torch.rand(n, generator=g) ** 3 * V).long().clamp_(0, V - 1)  # some tokens often, most never
    check_grad(device, dy, ids.to(torch.int32) if n % 2 else ids, V)


@pytest.mark.parametrize("n,E", [(300, 64), (4096, 8), (40000, 130), (300001, 3)])
@pytest.mark.parametrize("kind", ["all the same", "all different", "two", "padding", "outside"])
def test_lookup_grad_patterns(device, n, E, kind):
    """Runs that fill every span, none, straddle them, and ids that are left out; 300001 ids take the counts'
    own launch."""
    g = gen(n + E)
    V = n + 5
    dy = torch.randn(n, E, generator=g)
    ids = {"all the same": torch.full((n,), 3), "all different": torch.randperm(n, generator=g),
           "two": torch.arange(n) % 2 * (V - 1), "padding": torch.where(torch.rand(n, generator=g) < 0.5, 0, torch.arange(n)),
           "outside": torch.where(torch.arange(n) % 3 == 0, -1, torch.where(torch.arange(n) % 3 == 1, V, 7))}[kind]
    dy[(ids < 0) | (ids >= V)] = float("nan")  # never read
    check_grad(device, dy, ids, V)


def test_lookup_grad_runs_of_about_256_spans(device):
    """Runs whose last span is found by one look at the next 256, just so, and by further ones; rows of 130 columns
    have spans of 32 entries."""
    g = gen(21)
    ids = torch.cat([torch.full((32 * k + d,), i) for i, (k, d) in enumerate(
        [(255, 0), (256, 0), (257, 31), (258, 1), (3, 5), (254, 30), (513, 2), (9, 0), (256, 31), (600, 7)])])
    check_grad(device, torch.randn(len(ids), 130, generator=g), ids, 12)
    check_grad(device, torch.randn(len(ids), 130, generator=g), ids[torch.randperm(len(ids), generator=g)], 12)


def test_lookup_grad_repeats_bit_for_bit_and_strides(device):
    g = gen(8)
    ids = (torch.rand(30000, generator=g) ** 4 * 500).long().to(device)
    dy = torch.randn(30000, 72, generator=g).to(device)
    first = api.embedding_grad(dy, ids, 500)
    for _ in range(3):
        assert torch.equal(api.embedding_grad(dy, ids, 500), first)
    wide = torch.randn(30000, 100, generator=g).to(device)
    wide[:, 3:75] = dy
    assert torch.equal(api.embedding_grad(wide[:, 3:75], ids, 500), first)
    assert torch.equal(api.embedding_grad(dy.view(300, 100, 72), ids.view(300, 100), 500), first)
    assert (api.embedding_grad(dy[:0], ids[:0], 9) == 0).all()


def test_lookup_past_32_bits(device):
    V, E = (1 << 22) + 3, 640  # 2.7e9 elements
    table = torch.zeros(V, E, dtype=BF, device=device)
    table[-1] = torch.arange(E, device=device).to(BF)
    got = api.embedding_lookup(table, torch.tensor([V - 1, 0, V], device=device))
    near(got, torch.stack([table[-1].cpu(), torch.zeros(E), torch.zeros(E)]), 0.0)
    del table
    grad = api.embedding_grad(got, torch.tensor([V - 1, 1, V], device=device), V)
    near(grad[-1], got[0].double().cpu(), 0.0)
    assert (grad[:-1].view(-1)[-1000:] == 0).all() and (grad[:5] == 0).all()


# ---- recurrence --------------------------------------------------------------------------------------
def inputs(R, T, H, dtype, seed, lens=True, h0=True):
    g = gen(seed)
    gate, cand = (torch.randn(R, T, H, generator=g) * 2 + 1).to(dtype), torch.randn(R, T, H, generator=g).to(dtype)
    ln = None
    if lens:
        ln = torch.randint(0, T + 1, (R,), generator=g, dtype=torch.int32)
        ln[0] = 0
        if R > 1:
            ln[1] = T
    return gate, cand, ln, torch.randn(R, H, generator=g) if h0 else None, g


def check_recurrence(device, gate, cand, lens, h0, reverse, g, grad=True):
    dev = lambda t: None if t is None else t.to(device)  # noqa: E731
    dt = gate.dtype
    h, last, states = api.linear_recurrence(dev(gate), dev(cand), dev(lens), dev(h0), reverse, save=True)
    wh, wlast, _, eh, el = ref.recurrence(gate, cand, lens, h0, reverse)
    assert h.dtype == dt and last.dtype == F32
    rounded(h, wh, eh)
    rounded(last, wlast, el)
    if not grad:
        return h, last
    dh = torch.randn(gate.shape, generator=g).to(dt)
    dlast = torch.randn(last.shape, generator=g)
    got = api.linear_recurrence_grad(dev(gate), dev(cand), states, dev(dh), dev(dlast), dev(lens), reverse)
    dg, dc, dh0, ge, ce, he = ref.recurrence_grad(gate, cand, dh, dlast, lens, h0, reverse)
    rounded(got[0], dg, ge)
    rounded(got[1], dc, ce)
    rounded(got[2], dh0, he)
    return h, last


# channels and steps that reach every way the work is cut: one wave a piece (many channels), four and eight
# waves over time, and segments of time
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("R,T,H,dtype", [(1, 1, 1, F32), (3, 1, 5, BF), (2, 16, 6, F16), (5, 17, 33, BF), (4, 40, 64, BF),
                                         (3, 63, 10, F32), (2, 129, 130, F16), (600, 33, 128, BF), (2100, 18, 64, F32),
                                         (1050, 20, 65, F16), (2, 256, 6, BF), (2, 257, 6, F32), (3, 300, 7, BF),
                                         (1, 1029, 3, F32), (2, 2500, 20, BF), (20, 2500, 63, BF), (14, 3400, 66, F16)])
def test_recurrence(device, R, T, H, dtype, reverse):
    gate, cand, lens, h0, g = inputs(R, T, H, dtype, R + T + H)
    check_recurrence(device, gate, cand, lens, h0, reverse, g)


def test_recurrence_without_extras(device):
    gate, cand, _, _, g = inputs(3, 50, 12, BF, 5, lens=False, h0=False)
    check_recurrence(device, gate, cand, None, None, False, g)
    # no dh, no dlast
    h, last, states = api.linear_recurrence(gate.to(device), cand.to(device), save=True)
    dlast = torch.randn(3, 12, generator=g)
    got = api.linear_recurrence_grad(gate.to(device), cand.to(device), states, None, dlast.to(device))
    dg, dc, dh0, ge, ce, he = ref.recurrence_grad(gate, cand, None, dlast)
    for x, w, e in zip(got, (dg, dc, dh0), (ge, ce, he)):
        rounded(x, w, e)
    dh = torch.randn(3, 50, 12, generator=g).to(BF)
    got = api.linear_recurrence_grad(gate.to(device), cand.to(device), states, dh.to(device))
    dg, dc, dh0, ge, ce, he = ref.recurrence_grad(gate, cand, dh)
    for x, w, e in zip(got, (dg, dc, dh0), (ge, ce, he)):
        rounded(x, w, e)
    plain = api.linear_recurrence(gate.to(device), cand.to(device))
    assert torch.equal(plain[0], h) and torch.equal(plain[1], last)


@pytest.mark.parametrize("reverse", [False, True])
def test_recurrence_does_not_read_behind_the_end(device, reverse):
    for R, T, H in ((4, 50, 9), (2, 3000, 8)):
        gate, cand, lens, h0, g = inputs(R, T, H, F32, 11)
        lens[-1] = T // 2
        dh, dlast = torch.randn(R, T, H, generator=g), torch.randn(R, H, generator=g)
        want = api.linear_recurrence(gate.to(device), cand.to(device), lens.to(device), h0.to(device), reverse, save=True)
        wgrad = api.linear_recurrence_grad(gate.to(device), cand.to(device), want[2], dh.to(device), dlast.to(device),
                                           lens.to(device), reverse)
        past = torch.arange(T)[None, :] >= lens[:, None]
        for x, bad in ((gate, float("nan")), (cand, float("inf")), (dh, float("nan"))):
            x[past] = bad
        got = api.linear_recurrence(gate.to(device), cand.to(device), lens.to(device), h0.to(device), reverse, save=True)
        ggrad = api.linear_recurrence_grad(gate.to(device), cand.to(device), got[2], dh.to(device), dlast.to(device),
                                           lens.to(device), reverse)
        for a, b in zip(got + ggrad, want + wgrad):
            assert torch.equal(a, b)
        assert torch.equal(got[1][0].cpu(), h0[0])  # the empty row keeps its state
        assert torch.equal(ggrad[2][0].cpu(), dlast[0])
        # lengths past either end are the ends
        odd = torch.where(lens == T, T + 100, torch.where(lens == 0, -5, lens))
        again = api.linear_recurrence(gate.to(device), cand.to(device), odd.long().to(device), h0.to(device), reverse)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


def test_recurrence_gate_ends(device):
    """Gates at and past the ends of what a sigmoid can tell apart: u is 0 or 1, nothing overflows."""
    inf = float("inf")
    gate = torch.tensor([-inf, -3e38, -200.0, -90.0, -88.0, -1e-30, 0.0, 88.0, 90.0, 200.0, 3e38, inf])
    cand = torch.full((1, 2, 12), 2.0)
    h0 = torch.full((1, 12), -1.0)
    got, last, states = api.linear_recurrence(gate.expand(1, 2, 12).to(device), cand.to(device), None, h0.to(device), save=True)
    want, _, _, e, _ = ref.recurrence(gate.expand(1, 2, 12), cand, None, h0)
    rounded(got, want, e + 2.0 ** -120)  # exp(-88) and below may be flushed
    grads = api.linear_recurrence_grad(gate.expand(1, 2, 12).to(device), cand.to(device), states,
                                       torch.ones(1, 2, 12, device=device))
    assert all(torch.isfinite(x).all() for x in grads)
    # a NaN stays in its own row and channel, and reaches its later steps alone
    g2 = torch.zeros(2, 40, 6)
    g2[1, 20, 3] = float("nan")
    h, _ = api.linear_recurrence(g2.to(device), torch.ones(2, 40, 6, device=device))
    bad = torch.isnan(h.cpu())
    assert bad[1, 20:, 3].all() and bad.sum() == 20


@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_strides(device, dtype):
    R, T, H = 5, 37, 22
    gate, cand, lens, h0, g = inputs(R, T, H, dtype, 17)
    dh = torch.randn(R, T, H, generator=g).to(dtype)
    args = [x.to(device) for x in (gate, cand, lens, h0, dh)]
    want = api.linear_recurrence(args[0], args[1], args[2], args[3], True, save=True)
    wgrad = api.linear_recurrence_grad(args[0], args[1], want[2], args[4], None, args[2], True)

    def same(gate, cand, dh, h0):
        got = api.linear_recurrence(gate, cand, args[2], h0, True, save=True)
        for a, b in zip(got + api.linear_recurrence_grad(gate, cand, got[2], dh, None, args[2], True), want + wgrad):
            assert torch.equal(a, b)
    both = torch.cat([args[0], args[1]], 2)  # halves of one projection
    same(both[..., :H], both[..., H:], args[4], args[3])
    tm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (args[0], args[1], args[4])]  # time-major
    same(tm[0], tm[1], tm[2], args[3])
    odd = torch.zeros(R, T, 2 * H + 1, dtype=dtype, device=device)  # rows that start anywhere
    odd[..., 1:H + 1] = args[0]
    same(odd[..., 1:H + 1], args[1], args[4], args[3].t().contiguous().t())
    cf = [x.permute(0, 2, 1).contiguous().permute(0, 2, 1) for x in (args[0], args[1], args[4])]  # channels apart
    same(cf[0], cf[1], cf[2], args[3])
    # rows so far apart that a wave's offsets pass 32 bits
    far = 40_000_000
    away = [torch.zeros(far * (R - 1) + T * H, dtype=dtype, device=device).as_strided((R, T, H), (far, H, 1)) for _ in range(3)]
    for x, y in zip(away, (args[0], args[1], args[4])):
        x.copy_(y)
    same(away[0], away[1], away[2], args[3])
    del away
    # one gate for all rows
    h, _ = api.linear_recurrence(args[0][:1].expand(R, T, H), args[1])
    h2, _ = api.linear_recurrence(args[0][:1].repeat(R, 1, 1), args[1])
    assert torch.equal(h, h2)


def test_recurrence_strides_of_long_rows(device):
    """An odd number of 16-bit channels, two a lane, in segments of time; rows that start anywhere, and rows so far
    apart that a wave's offsets pass 32 bits."""
    R, T, H, far = 2, 24011, 65, 340_000_000
    g = torch.Generator(device).manual_seed(3)
    args = [torch.randn(R, T, H, generator=g, device=device).to(BF) for _ in range(3)]
    want = api.linear_recurrence(args[0], args[1], save=True)
    wgrad = api.linear_recurrence_grad(args[0], args[1], want[2], args[2])
    odd = torch.zeros(R, T, 3 * H + 2, dtype=BF, device=device)
    near_ = [odd[..., k * H + 1:(k + 1) * H + 1] for k in range(3)]
    away = [torch.zeros(far * (R - 1) + T * H, dtype=BF, device=device).as_strided((R, T, H), (far, H, 1)) for _ in range(3)]
    for xs in (near_, away):
        for x, y in zip(xs, args):
            x.copy_(y)
        got = api.linear_recurrence(xs[0], xs[1], save=True)
        for a, b in zip(got + api.linear_recurrence_grad(xs[0], xs[1], got[2], xs[2]), want + wgrad):
            assert torch.equal(a, b)


def test_recurrence_empty(device):
    z = lambda *s: torch.zeros(*s, device=device)  # noqa: E731
    h, last = api.linear_recurrence(z(0, 4, 3), z(0, 4, 3))
    assert h.shape == (0, 4, 3) and last.shape == (0, 3)
    h0 = torch.randn(2, 3, device=device)
    h, last, states = api.linear_recurrence(z(2, 0, 3), z(2, 0, 3), None, h0, save=True)
    assert h.shape == (2, 0, 3) and torch.equal(last, h0)
    dg, dc, dh0 = api.linear_recurrence_grad(z(2, 0, 3), z(2, 0, 3), states, None, h0)
    assert torch.equal(dh0, h0)
    assert api.linear_recurrence_step(z(0, 3), z(0, 3), z(0, 3)).shape == (0, 3)


def test_recurrence_gradient_against_differences(device):
    """<gradient, d> of the kernels against central differences of the float64 formula along d."""
    R, T, H = 3, 45, 5
    gate, cand, lens, h0, g = inputs(R, T, H, F32, 23)
    dh, dlast = torch.randn(R, T, H, generator=g), torch.randn(R, H, generator=g)
    for reverse in (False, True):
        _, _, states = api.linear_recurrence(gate.to(device), cand.to(device), lens.to(device), h0.to(device), reverse, save=True)
        grads = api.linear_recurrence_grad(gate.to(device), cand.to(device), states, dh.to(device), dlast.to(device),
                                           lens.to(device), reverse)

        def loss(*x):
            h, last, *_ = ref.recurrence(x[0], x[1], lens, x[2], reverse)
            return float((h * dh.double()).sum() + (last * dlast.double()).sum())
        at = [x.double() for x in (gate, cand, h0)]
        for k in range(3):
            d = [torch.randn(x.shape, generator=g).double() if i == k else torch.zeros_like(x) for i, x in enumerate(at)]
            eps = 1e-5  # the difference is off by O(eps^2) and 2^-53 / eps of a loss of size ~100: 1e-8 together
            diff = (loss(*(x + eps * y for x, y in zip(at, d))) - loss(*(x - eps * y for x, y in zip(at, d)))) / (2 * eps)
            dot = float((grads[k].double().cpu() * d[k]).sum())
            mag = float((grads[k].double().cpu() * d[k]).abs().sum())
            assert abs(dot - diff) <= 1e-5 * mag + 1e-6, (k, dot, diff)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,H", [(1, 1), (3, 7), (256, 512), (33, 100)])
def test_step(device, R, H, dtype):
    gate, cand, _, h0, g = inputs(R, 6, H, dtype, R + H, lens=False)
    wide = torch.zeros(R, H + 3, device=device)
    state = wide[:, 1:H + 1]
    state.copy_(h0)
    wh, wl, _, eh, el = ref.recurrence(gate, cand, None, h0)
    gd, cd = gate.to(device), cand.to(device)
    for t in range(6):
        h = api.linear_recurrence_step(gd[:, t], cd[:, t], state)
        assert h.dtype == dtype
        rounded(h, wh[:, t], eh[:, t])
    rounded(state, wl, el)
    assert (wide[:, 0] == 0).all() and (wide[:, H + 1:] == 0).all()


def test_recurrence_past_32_bits(device):
    R, T, H = 1, 65536 + 24, 32768 + 64  # 2.15e9 elements each
    gate = torch.zeros(R, T, H, dtype=BF, device=device)
    cand = torch.zeros(R, T, H, dtype=BF, device=device)
    torch.manual_seed(0)
    gate[:, -64:, -64:] = torch.randn(1, 64, 64, device=device).to(BF)
    cand[:, -64:, -64:] = torch.randn(1, 64, 64, device=device).to(BF)
    h, last, states = api.linear_recurrence(gate, cand, save=True)
    # before the last 64 steps nothing but zeros came in, so the state there is zero
    want, wl, _, e, el = ref.recurrence(gate[:, -64:, -64:].cpu(), cand[:, -64:, -64:].cpu())
    rounded(h[:, -64:, -64:], want, e)
    rounded(last[:, -64:], wl, el)
    dlast = torch.randn(R, H, device=device)
    del h
    dg, dc, dh0 = api.linear_recurrence_grad(gate, cand, states, None, dlast)
    wg, wc, _, ge, ce, _ = ref.recurrence_grad(gate[:, -64:, -64:].cpu(), cand[:, -64:, -64:].cpu(), None, dlast[:, -64:].cpu())
    rounded(dg[:, -64:, -64:], wg, ge)
    rounded(dc[:, -64:, -64:], wc, ce)


# ---- norm --------------------------------------------------------------------------------------------
# the mean square is a sum of at most 16 squares a thread and 10 + 16 further additions; with the square root,
# the quotients and the two products every y is within 40 half units of fp32
NORM = 40 * U


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 3), (33, 8), (7, 127), (16, 128), (17, 129), (6, 500), (9, 513), (5, 1000),
                                       (4, 1025), (3, 2049), (2, 4100), (2, 8200), (3, 16384), (2000, 20)])
def test_norm(device, rows, cols, dtype):
    g = gen(rows + cols)
    x, res = torch.randn(rows, cols, generator=g).to(dtype), (torch.randn(rows, cols, generator=g) * 3).to(dtype)
    w = torch.rand(cols, generator=g) + 0.5
    dy, ds = torch.randn(rows, cols, generator=g).to(dtype), torch.randn(rows, cols, generator=g).to(dtype)
    for residual, add in ((res, ds), (None, None)):
        rd = None if residual is None else residual.to(device)
        y, s, rstd = api.rms_norm(x.to(device), w.to(device), rd, 1e-5)
        eps = float(torch.tensor(1e-5))
        wy, ws, wr = ref.norm(x, w, residual, eps)
        assert torch.equal(s.cpu(), ws) and y.dtype == dtype and rstd.dtype == F32
        rounded(y, wy, NORM * wy.abs())
        near(rstd, wr[:, 0], NORM * wr[:, 0])
        dx, dw = api.rms_norm_grad(dy.to(device), s, w.to(device), rstd, None if add is None else add.to(device))
        wx, wdw, mx, mw = ref.norm_grad(dy, ws, w, wr, add)
        rounded(dx, wx, 2 * NORM * mx)
        near(dw, wdw, (rows + 40) * U * mw)  # rows - 1 additions in any order over the norm's own error
        y8, s8 = api.rms_norm_blocks8(x.to(device), w.to(device), rd, 1e-5)
        assert torch.equal(s8.cpu(), ws)
        check_blocks(y8, wy, NORM * wy.abs())


def check_blocks(b, want, tol):
    """Values within half a step of e4m3 (2^-4 relative, 2^-10 of the scale below its normal range) of
    want +- tol; scales the smallest power of two that brings the block into +-448."""
    rows, cols = want.shape
    kp = -(-cols // 128) * 128
    assert b.cols == cols and b.q.shape == (rows, kp) and b.scale.shape == (rows, kp // 128)
    got = ref.values8(b.q, b.scale, kp)
    assert (got[:, cols:] == 0).all()
    scale = torch.exp2(b.scale.view(torch.uint8).double().cpu() - 127)
    pad = torch.nn.functional.pad(want.abs(), (0, kp - cols)).view(rows, -1, 128)
    tp = torch.nn.functional.pad(tol, (0, kp - cols)).view(rows, -1, 128)
    hi, lo = (pad + tp).amax(2), (pad - tp).amax(2)
    zero = pad.amax(2) == 0
    small = scale == 2.0 ** -127
    assert ((lo <= 448 * scale) | zero).all() and ((hi > 224 * scale) | zero | small).all() and (scale[zero] == 1).all()
    half = torch.maximum((want.abs() + tol) * 2.0 ** -4, scale.repeat_interleave(128, 1)[:, :cols] * 2.0 ** -10)
    near(got[:, :cols], want, tol + half)
    for dt in TYPES:
        v = api.dequantize_blocks8(b, dt)
        assert v.dtype == dt
        near(v, got[:, :cols].to(F32).to(dt).double(), 0.0)


def test_norm_rows_are_apart(device):
    """A NaN or infinite row is its own row's matter, also in the 8-bit form."""
    for cols in (40, 300, 3000):
        x = torch.randn(9, cols)
        w = torch.ones(cols)
        want, _, _ = api.rms_norm(x.to(device), w.to(device))
        b, _ = api.rms_norm_blocks8(x.to(device), w.to(device))
        want8 = api.dequantize_blocks8(b)
        x[3, 7], x[6, 1], x[8] = float("nan"), float("inf"), 0.0
        y, _, _ = api.rms_norm(x.to(device), w.to(device))
        y8 = api.dequantize_blocks8(api.rms_norm_blocks8(x.to(device), w.to(device))[0])
        keep = [0, 1, 2, 4, 5, 7]
        assert torch.equal(y[keep], want[keep]) and torch.equal(y8[keep], want8[keep])
        assert torch.isnan(y[3]).all() and torch.isnan(y8[3]).all() and (y[8] == 0).all() and (y8[8] == 0).all()
        assert torch.isnan(y[6, 1]) and torch.isnan(y8[6, 1]) and (y[6, 2:] == 0).all() and (y8[6, 2:] == 0).all()


def test_norm_shapes_and_strides(device):
    g = gen(2)
    x = torch.randn(3, 5, 90, generator=g).to(BF).to(device)
    w = torch.rand(90, generator=g).to(device)
    y, s, rstd = api.rms_norm(x, w, x)
    assert y.shape == x.shape and s.shape == x.shape and rstd.shape == (15,)
    y2, s2, rstd2 = api.rms_norm(x.view(15, 90), w, x.view(15, 90))
    assert torch.equal(y.view(15, 90), y2) and torch.equal(rstd, rstd2)
    wide = torch.zeros(15, 101, dtype=BF, device=device)
    wide[:, 7:97] = x.view(15, 90)
    a, b, c = api.rms_norm(wide[:, 7:97], w, wide[:, 7:97])
    assert torch.equal(a, y2) and torch.equal(b, s2) and torch.equal(c, rstd2)
    q, q2 = api.rms_norm_blocks8(wide[:, 7:97], w)[0], api.rms_norm_blocks8(x.view(15, 90), w)[0]
    assert torch.equal(q.q.view(torch.uint8), q2.q.view(torch.uint8))
    dy = torch.randn(15, 90, generator=g).to(BF).to(device)
    wide2 = torch.zeros(15, 93, dtype=BF, device=device)
    wide2[:, 3:] = dy
    for p, r in zip(api.rms_norm_grad(wide2[:, 3:], wide[:, 7:97], w, c, wide2[:, 3:]),
                    api.rms_norm_grad(dy, x.view(15, 90), w, c, dy)):
        assert torch.equal(p, r)
    assert api.rms_norm(x[:0], w)[0].shape == (0, 5, 90)
    dx, dw = api.rms_norm_grad(dy[:0], dy[:0], w, c[:0])
    assert dx.shape == (0, 90) and (dw == 0).all()
    # a column of all rows: one column, rows far apart
    col = x.view(15, 90)[:, 4:5]
    near(api.rms_norm(col, w[:1])[0], ref.norm(col.cpu(), w[:1].cpu(), None, 1e-6)[0], 0.02)


def test_norm_ragged_rows(device):
    """Every width of a ragged end, in rows whose surroundings are NaN: what lies beside a row is not used."""
    g = gen(5)
    for dtype in TYPES:
        for cols in list(range(1, 25)) + [133, 262, 1030, 4099]:
            x, dy = torch.randn(19, cols, generator=g).to(dtype), torch.randn(19, cols, generator=g).to(dtype)
            w = torch.rand(cols, generator=g) + 0.5
            base = torch.full((2, 19, cols + 11), float("nan"), dtype=dtype, device=device)
            xs, dys = base[0, :, 5:5 + cols], base[1, :, 5:5 + cols]
            xs.copy_(x)
            dys.copy_(dy)
            y, s, rstd = api.rms_norm(xs, w.to(device), dys)
            eps = float(torch.tensor(1e-6))
            wy, ws, wr = ref.norm(x, w, dy, eps)
            assert torch.equal(s.cpu(), ws)
            rounded(y, wy, NORM * wy.abs())
            dx, dw = api.rms_norm_grad(dys, s, w.to(device), rstd, xs)
            wx, wdw, mx, mw = ref.norm_grad(dy, ws, w, wr, x)
            rounded(dx, wx, 2 * NORM * mx)
            near(dw, wdw, 59 * U * mw)
            y8, _ = api.rms_norm_blocks8(xs, w.to(device), dys)
            check_blocks(y8, wy, NORM * wy.abs())


# rows enough that a workgroup walks several, at every number of threads a row; the outputs over the inputs, as the
# C entry points allow: s over x or the residual, dx over dy or ds
@pytest.mark.parametrize("rows,cols,dtype", [(40000, 24, BF), (40001, 21, F16), (9000, 200, F32), (9001, 501, BF),
                                             (8500, 1000, F16), (2500, 2041, BF), (2200, 4096, BF), (1100, 4103, F32),
                                             (1500, 8192, F16), (600, 8203, F32), (600, 12000, BF), (530, 16384, F32)])
def test_norm_many_rows_in_place(device, rows, cols, dtype):
    g = torch.Generator(device).manual_seed(rows)
    code = seqops._code(dtype, "x")
    x, res, dy, ds = (torch.randn(rows, cols, generator=g, device=device).to(dtype) for _ in range(4))
    w = torch.rand(cols, generator=g, device=device) + 0.5
    y, s, rstd = api.rms_norm(x, w, res)
    dx, dw = api.rms_norm_grad(dy, s, w, rstd, ds)
    pick = torch.unique(torch.cat([torch.arange(0, rows, max(rows // 40, 1)), torch.arange(rows - 3, rows)]))
    wy, ws, wr = ref.norm(x[pick].cpu(), w.cpu(), res[pick].cpu(), float(torch.tensor(1e-6)))
    assert torch.equal(s[pick].cpu(), ws)
    rounded(y[pick], wy, NORM * wy.abs())
    wx, _, mx, _ = ref.norm_grad(dy[pick].cpu(), ws, w.cpu(), wr, ds[pick].cpu())
    rounded(dx[pick], wx, 2 * NORM * mx)
    n = s.double() * rstd.double()[:, None]
    near(dw, (dy.double() * n).sum(0).cpu(), (rows + 40) * U * (dy.double() * n).abs().sum(0).cpu())
    need = int(_lib.load().dssm_rms_norm_bwd_ws_bytes(rows, cols))
    ws_ = torch.empty(need, dtype=torch.uint8, device=device)
    for turn in range(2):
        a, b, c, d = x.clone(), res.clone(), dy.clone(), ds.clone()
        over, back = (a, c) if turn else (b, d)
        y2, r2, w2 = torch.empty_like(y), torch.empty_like(rstd), torch.empty_like(dw)
        seqops._call(0, "dssm_rms_norm", a.data_ptr(), cols, b.data_ptr(), cols, w.data_ptr(), rows, cols, code, 1e-6,
                     y2.data_ptr(), cols, over.data_ptr(), cols, r2.data_ptr())
        assert torch.equal(y2, y) and torch.equal(over, s) and torch.equal(r2, rstd)
        seqops._call(0, "dssm_rms_norm_bwd", c.data_ptr(), cols, s.data_ptr(), cols, w.data_ptr(), rstd.data_ptr(),
                     d.data_ptr(), cols, rows, cols, code, back.data_ptr(), cols, w2.data_ptr(), ws_.data_ptr(), need)
        assert torch.equal(back, dx) and torch.equal(w2, dw)


def test_norm_gradient_against_differences(device):
    g = gen(31)
    x, w, dy, ds = (torch.randn(s, generator=g) for s in ((6, 70), (70,), (6, 70), (6, 70)))
    y, s, rstd = api.rms_norm(x.to(device), w.to(device))
    dx, dw = api.rms_norm_grad(dy.to(device), s, w.to(device), rstd, ds.to(device))

    def loss(x, w):
        n = x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6)
        return float((n * w * dy.double()).sum() + (x * ds.double()).sum())
    x, w = x.double(), w.double()
    for got, d in ((dx, (torch.randn(x.shape, generator=g).double(), 0 * w)), (dw, (0 * x, torch.randn(70, generator=g).double()))):
        e = 1e-6
        diff = (loss(x + e * d[0], w + e * d[1]) - loss(x - e * d[0], w - e * d[1])) / (2 * e)
        v = d[0] if got.dim() == 2 else d[1]
        dot = got.double().cpu() * v
        assert abs(float(dot.sum()) - diff) <= 1e-5 * float(dot.abs().sum()) + 1e-6


# ---- 8-bit form and product --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 128), (5, 129), (4, 700), (9, 1025), (2, 16384)])
def test_quantize(device, rows, cols, dtype):
    g = gen(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[0, :min(cols, 128)] = 0
    b = api.quantize_blocks8(x.to(device))
    check_blocks(b, x.double(), torch.zeros(rows, cols, dtype=torch.float64))
    again = api.quantize_blocks8(api.dequantize_blocks8(b))  # the form's own values come back as they are
    near(ref.values8(again.q, again.scale, cols), ref.values8(b.q, b.scale, cols), 0.0)


def test_quantize_ends(device):
    """The largest and smallest magnitudes, values at the scale's borders, ties, infinities and NaN."""
    x = torch.zeros(12, 128)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = 448.0, 448.0001, 3.4e38, 1e-45
    x[4, 0], x[5, 5], x[6, :4] = 2.0 ** -126, -2.0 ** -130, torch.tensor([448.0, 17.0, 19.0, -17.0])  # 17, 19: ties
    x[7, :3] = torch.tensor([float("inf"), 1.0, float("nan")])
    x[8, :2] = torch.tensor([float("-inf"), 0.0])
    x[9, :3] = torch.tensor([448.0, 2.0 ** -10, 3 * 2.0 ** -10])  # half a subnormal step, and three halves
    x[10, 0], x[11, 0] = 224.0, 224.0001
    b = api.quantize_blocks8(x.to(device))
    v = ref.values8(b.q, b.scale, 128)
    fin = [0, 1, 2, 3, 4, 5, 6, 9, 10, 11]
    check_blocks(api.quantize_blocks8(x[fin].to(device)), x[fin].double(), torch.zeros(10, 128, dtype=torch.float64))
    e = b.scale.view(torch.uint8).cpu()[:, 0].int() - 127
    assert e.tolist() == [0, 1, 120, -127, -127, -127, 0, -8, 0, 0, -1, 0]
    assert v[6, :4].tolist() == [448.0, 16.0, 20.0, -16.0]
    assert v[9, :3].tolist() == [448.0, 0.0, 2.0 ** -8]
    assert torch.isnan(v[7, 0]) and torch.isnan(v[7, 2]) and v[7, 1] == 1.0 and torch.isnan(v[8, 0]) and (v[8, 1:] == 0).all()


def product(a, w, bias, K):
    """(a w^T + bias, how far the matrix unit's sum may be off) in float64 from the forms' own values: products are exact;
    eight neighbouring ones are each cut to a grid of 2^-13 of the largest of them, which is at most the product of
    the eights' largest factors; the eights' sums, the chain and the bias are K / 8 + 9 additions at 2^-23 each,
    whether they round or cut, of partial sums no larger than the magnitudes' sum."""
    va, vw = (torch.nn.functional.pad(ref.values8(b.q, b.scale, K).nan_to_num(0), (0, -K % 8)) for b in (a, w))
    want, mag = va @ vw.t(), va.abs() @ vw.abs().t()
    cut = va.abs().view(len(va), -1, 8).amax(2) @ vw.abs().view(len(vw), -1, 8).amax(2).t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.abs().double()
    return want, 8 * 2.0 ** -13 * cut + (K / 8 + 9) * 2.0 ** -23 * mag


@pytest.mark.parametrize("out", [BF, F16])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 300, 128), (7, 17, 129), (16, 40, 1000), (17, 64, 2000), (33, 130, 257),
                                   (65, 300, 513), (64, 16, 4500), (200, 77, 640), (1100, 1030, 300), (257, 4100, 400),
                                   (3000, 3001, 130), (1500, 1500, 100), (1500, 1500, 1300), (200, 500, 3000),
                                   (100, 300, 200), (3000, 3001, 1100), (40, 4000, 1030), (250, 1000, 1700),
                                   (100, 1500, 2100), (9, 4200, 1300), (20, 4200, 200), (180, 700, 1024)])
def test_product(device, M, N, K, out):
    g = gen(M + N + K)
    a = api.quantize_blocks8((torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))).to(device))
    w = api.quantize_blocks8((torch.randn(N, K, generator=g) * K ** -0.5).to(device))
    bias = torch.randn(N, generator=g) if N % 2 else None
    want, tol = product(a, w, bias, K)
    got = api.blocks8_matmul(a, w, None if bias is None else bias.to(device), out)
    assert got.dtype == out and got.shape == (M, N)
    rounded(got, want, tol)
    assert torch.equal(api.blocks8_matmul(a, w, None if bias is None else bias.to(device), out), got)


def test_product_scales_and_rows_are_apart(device):
    """Every block's scale of both operands counts, and a NaN or a row of another size stays in its own row."""
    g = gen(77)
    for M, N, K in ((5, 20, 700), (300, 260, 700), (2100, 2100, 260)):
        x = torch.randn(M, K, generator=g)
        blocks = torch.exp2(torch.randint(-20, 20, (M, -(-K // 128)), generator=g).float())
        x *= blocks.repeat_interleave(128, 1)[:, :K]
        y = torch.randn(N, K, generator=g) * torch.exp2(torch.randint(-20, 20, (N, -(-K // 128)), generator=g).float()
                                                        ).repeat_interleave(128, 1)[:, :K]
        x[M // 2, K - 1] = float("nan")
        y[N - 1, 0] = float("inf")  # becomes NaN
        a, w = api.quantize_blocks8(x.to(device)), api.quantize_blocks8(y.to(device))
        got = api.blocks8_matmul(a, w)
        bad = torch.isnan(got.cpu())
        assert bad[M // 2].all() and bad[:, N - 1].all() and bad.sum() == M + N - 1
        want, tol = product(a, w, None, K)
        rounded(got.cpu()[~bad], want[~bad], tol[~bad])


def test_product_shares_of_k(device):
    """Four groups of waves share nine blocks: the shares that are not there add nothing, not even the NaN that the
    last block holds, and that one's scale."""
    M, N, K = 200, 500, 1100
    g = gen(77)
    x, y = torch.randn(M, K, generator=g), torch.randn(N, K, generator=g)
    x[3, K - 1], y[7, K - 2], x[150, 0] = float("nan"), float("inf"), float("nan")
    a, w = api.quantize_blocks8(x.to(device)), api.quantize_blocks8(y.to(device))
    a.scale.view(torch.uint8)[9, 8] = 255
    w.scale.view(torch.uint8)[11, 8] = 255
    bad = torch.isnan(api.blocks8_matmul(a, w).cpu())
    want = torch.zeros(M, N, dtype=torch.bool)
    want[[3, 9, 150]] = True
    want[:, [7, 11]] = True
    assert torch.equal(bad, want)


def test_product_empty(device):
    e = lambda r, c: api.quantize_blocks8(torch.zeros(r, c, device=device))  # noqa: E731
    assert api.blocks8_matmul(e(0, 5), e(3, 5)).shape == (0, 3)
    assert api.blocks8_matmul(e(4, 5), e(0, 5)).shape == (4, 0)
    assert api.dequantize_blocks8(e(0, 5)).shape == (0, 5)


# ---- as they are used --------------------------------------------------------------------------------
def tower(x, rows, steps, params, lens, H):
    """ids -> scaled embedding -> norm in 8 bits -> 8-bit projection -> recurrence: the rows' last states"""
    emb = api.embedding_lookup(params["table"], x, 3.0, BF)
    y8, s = api.rms_norm_blocks8(emb, params["norm"])
    proj = api.blocks8_matmul(y8, params["w"], params["bias"], BF).view(rows, steps, 2 * H)
    return proj, api.linear_recurrence(proj[..., :H], proj[..., H:], lens)


def test_tower_forward_and_single_tokens(device):
    """A run of the operators as a text tower serves with them: whole rows at once against the same rows token by
    token through the running state, and against the formulas on the same 8-bit values."""
    g = gen(5)
    V, E, H, R, T = 900, 96, 80, 6, 37
    params = {"table": torch.randn(V, E, generator=g).to(device), "norm": (torch.rand(E, generator=g) + 0.5).to(device),
              "w": api.quantize_blocks8((torch.randn(2 * H, E, generator=g) * E ** -0.5).to(device)),
              "bias": torch.randn(2 * H, generator=g).to(device)}
    ids = torch.randint(0, V, (R, T), generator=g, dtype=torch.int32).to(device)
    lens = torch.tensor([37, 0, 1, 16, 17, 30], dtype=torch.int32, device=device)
    proj, (h, last) = tower(ids, R, T, params, lens, H)
    wh, wl, _, eh, el = ref.recurrence(proj[..., :H].cpu(), proj[..., H:].cpu(), lens.cpu())
    rounded(h, wh, eh)
    rounded(last, wl, el)
    state = torch.zeros(R, H, device=device)
    for t in range(T):
        emb = api.embedding_lookup(params["table"], ids[:, t], 3.0, BF)
        y8, _ = api.rms_norm_blocks8(emb, params["norm"])
        p = api.blocks8_matmul(y8, params["w"], params["bias"], BF)
        live = lens > t
        kept = state.clone()
        one = api.linear_recurrence_step(p[:, :H], p[:, H:], state)
        state = torch.where(live[:, None], state, kept)
        # the projection's fp32 sums may differ in their last bits between the shapes, bf16 rounds that to at
        # most one step of one input here and there: gate and candidate move by 2^-7 of their size (~4), h by as much
        near(torch.where(live[:, None], one, 0.0), h[:, t].double().cpu(), 4 * 2.0 ** -7 * 4)
    near(state, last.double().cpu(), 4 * 2.0 ** -7 * 4)


def train(ids, lens, table, w, dout):
    """lookup -> norm with a residual -> recurrence, and back to the table"""
    R, T = ids.shape
    H = table.shape[1] // 2
    emb = api.embedding_lookup(table, ids, 2.0)
    y, s, rstd = api.rms_norm(emb, w, emb)
    h, last, states = api.linear_recurrence(y[..., :H], y[..., H:], lens, save=True)
    dg, dc, _ = api.linear_recurrence_grad(y[..., :H], y[..., H:], states, None, dout, lens)
    dx, dw = api.rms_norm_grad(torch.cat([dg, dc], 2), s, w, rstd)
    return last, api.embedding_grad(2 * dx, ids, table.shape[0], 2.0), dw


def train_inputs(device, seed=9, R=5, T=33, V=60, E=24):
    g = gen(seed)
    return (torch.randint(0, V, (R, T), generator=g).to(device), torch.randint(0, T + 1, (R,), generator=g).to(device),
            torch.randn(V, E, generator=g).to(device), (torch.rand(E, generator=g) + 0.5).to(device),
            torch.randn(R, E // 2, generator=g).to(device))


def test_training_run_against_differences(device):
    ids, lens, table, w, dout = train_inputs(device)
    last, dtable, dw = train(ids, lens, table, w, dout)
    H = table.shape[1] // 2

    def loss(table, w):
        emb = table[ids.cpu()] * 2.0
        s = emb + emb
        y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-6) * w
        _, last, *_ = ref.recurrence(y[..., :H], y[..., H:], lens.cpu())
        return float((last * dout.double().cpu()).sum())
    t, ww = table.double().cpu(), w.double().cpu()
    g = gen(1)
    for got, d in ((dtable, (torch.randn(t.shape, generator=g).double(), 0 * ww)),
                   (dw, (0 * t, torch.randn(ww.shape, generator=g).double()))):
        e = 1e-6
        diff = (loss(t + e * d[0], ww + e * d[1]) - loss(t - e * d[0], ww - e * d[1])) / (2 * e)
        dot = got.double().cpu() * (d[0] if got.dim() == 2 else d[1])
        assert abs(float(dot.sum()) - diff) <= 2e-5 * float(dot.abs().sum()) + 1e-6


def test_graphs_streams_and_two_at_once(device):
    """Two captured training runs of different sizes replayed in turn and on another stream with eager work between,
    every replay against the eager results."""
    runs = []
    for seed, R, T, V, E in ((1, 5, 33, 60, 24), (2, 2, 2600, 5000, 16)):
        args = train_inputs(device, seed, R, T, V, E)
        want = [x.clone() for x in train(*args)]
        other = train_inputs(device, seed + 10, R, T, V, E)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            train(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = train(*args)
        runs.append((graph, args, out, want, other))
    for k in range(4):
        for graph, args, out, want, other in runs:
            keep = [a.clone() for a in args]
            if k % 2:
                for a, b in zip(args, other):
                    a.copy_(b)
                want = train(*args)
            for o in out:
                o.zero_()
            graph.replay()
            eager = train(*other)
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(a, b)
            del eager
            for a, b in zip(args, keep):
                a.copy_(b)
    # the same work on two streams at once
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s, (_, args, _, _, _) in zip(streams, runs):
        with torch.cuda.stream(s):
            outs.append(train(*args))
    torch.cuda.synchronize()
    for out, (_, _, _, want, _) in zip(outs, runs):
        for a, b in zip(out, want):
            assert torch.equal(a, b)

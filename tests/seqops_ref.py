"""The sequence-tower operators from their formulas in float64 (CPU), step by step, with the running error
bounds that the GPU tests' tolerances are made of."""
import torch

TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # half a subnormal step


def stored(x, dtype):
    """How far x may move when it is stored as dtype (one rounding to nearest)."""
    half = torch.finfo(dtype).eps / 2
    return x.abs() * half + TINY[dtype]


def lookup(table, ids, scale):
    ids = ids.long()
    ok = (ids >= 0) & (ids < table.shape[0])
    return torch.where(ok[..., None], table.double()[ids.clamp(0, table.shape[0] - 1)] * scale, 0.0)


def lookup_grad(dy, ids, V, scale):
    """(gradient, sum of magnitudes, summands) per token"""
    E = dy.shape[-1]
    ids, dy = ids.reshape(-1).long(), dy.reshape(-1, E).double()
    ok = (ids >= 0) & (ids < V)
    ids, dy = ids[ok], dy[ok]
    g, a = torch.zeros(V, E, dtype=torch.float64), torch.zeros(V, E, dtype=torch.float64)
    g.index_add_(0, ids, dy)
    a.index_add_(0, ids, dy.abs())
    return g * scale, a * abs(scale), torch.bincount(ids, minlength=V).double()[:, None]


# One step's own error, relative to the magnitudes it adds: for fp32 gates u and v are within 4 units in the last
# place of fp32 (2^x 1, its correction 1/2, 1 + e 1/2, the reciprocal 1, a product 1/2; a unit is at most 2^-23),
# the two products and the sum add 3 half units: 4 * 2^-23 + 3 * 2^-24 < 2^-20.  For 16-bit gates the correction is
# left out: 2^x's argument -|f| log2 e is off by half a unit and by log2 e's own 1/4, which moves e, and with
# it the smaller of u and v (the larger less), by up to |f| * 1.5 * 2^-24.  A piece's product of u and the
# folds of pieces and segments make the same roundings in another order; twice the bound covers both walks.
# The roundings are relative to the magnitudes that are added, not to the sum: a piece's map A h + B is formed
# apart from the h it meets, so where A h and B cancel, the errors of each stay.  Both walks therefore carry the
# sum of magnitudes m (m_t = u m + |x|: |A| |h| + |B| summed over any cut is at most this) beside the value.
STEP = 2.0 ** -19


def step_error(gate):
    return STEP + (0.0 if gate.dtype == torch.float32 else 2 * 1.5 * 2.0 ** -24) * gate.double().abs()


def recurrence(gate, cand, lens=None, h0=None, reverse=False):
    """(h, last, states before each step, error bound of h and last)"""
    step = step_error(gate)
    gate, cand = gate.double(), cand.double()
    R, T, H = gate.shape
    lens = torch.full((R,), T) if lens is None else lens.long().clamp(0, T)
    u, v = torch.sigmoid(gate), torch.sigmoid(-gate)
    s = torch.zeros(R, H, dtype=torch.float64) if h0 is None else h0.double().clone()
    e, m = torch.zeros_like(s), s.abs()
    h, before, err = torch.zeros_like(gate), torch.zeros_like(gate), torch.zeros_like(gate)
    for t in (range(T - 1, -1, -1) if reverse else range(T)):
        on = (t < lens)[:, None]
        before[:, t] = s
        x, hu = v[:, t] * cand[:, t], u[:, t] * s
        nm = u[:, t] * m + x.abs()
        new, ne = hu + x, u[:, t] * e + step[:, t] * nm
        s, e, m = torch.where(on, new, s), torch.where(on, ne, e), torch.where(on, nm, m)
        h[:, t], err[:, t] = torch.where(on, s, 0.0), torch.where(on, e, 0.0)
    return h, s, before, err, e


def recurrence_grad(gate, cand, dh, dlast=None, lens=None, h0=None, reverse=False):
    """(dgate, dcand, dh0) and their error bounds"""
    h, _, before, herr, _ = recurrence(gate, cand, lens, h0, reverse)
    step = step_error(gate)
    gate, cand = gate.double(), cand.double()
    R, T, H = gate.shape
    lens = torch.full((R,), T) if lens is None else lens.long().clamp(0, T)
    u, v = torch.sigmoid(gate), torch.sigmoid(-gate)
    gam = torch.zeros(R, H, dtype=torch.float64) if dlast is None else dlast.double().clone()
    ge, m = torch.zeros_like(gam), gam.abs()
    emax = herr.amax(1)  # the error of any state of the row
    out = [torch.zeros_like(gate) for _ in range(4)]
    for t in (range(T) if reverse else range(T - 1, -1, -1)):
        on = (t < lens)[:, None]
        d = torch.zeros_like(gam) if dh is None else torch.where(on, dh[:, t].double(), 0.0)
        g = gam + d
        mg = m + d.abs()
        gerr = ge + 2.0 ** -24 * mg
        diff, uv = before[:, t] - cand[:, t], u[:, t] * v[:, t]
        dg, dc = g * diff * uv, g * v[:, t]
        dge = (gerr * diff.abs() + g.abs() * (emax + 2.0 ** -24 * diff.abs())) * uv + step[:, t] * 2 * dg.abs()
        dce = gerr * v[:, t] + step[:, t] * dc.abs()
        for o, val in zip(out, (dg, dc, dge, dce)):
            o[:, t] = torch.where(on, val, 0.0)
        gam, ge = torch.where(on, u[:, t] * g, gam), torch.where(on, u[:, t] * gerr + step[:, t] * u[:, t] * mg, ge)
        m = torch.where(on, u[:, t] * mg, m)
    return out[0], out[1], gam, out[2], out[3], ge


def norm(x, weight, residual, eps):
    s = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    f = s.double()
    rstd = 1 / torch.sqrt((f * f).mean(-1, keepdim=True) + eps)
    return f * rstd * weight.double(), s, rstd


def norm_grad(dy, s, weight, rstd, ds):
    """(dx, dweight, magnitudes that dx and dweight are sums of)"""
    n, d = s.double() * rstd, dy.double()
    wd = d * weight.double()
    m = (wd * n).mean(-1, keepdim=True)
    dx = rstd * (wd - n * m)
    mag = rstd * (wd.abs() + n.abs() * (wd * n).abs().mean(-1, keepdim=True))
    if ds is not None:
        dx, mag = dx + ds.double(), mag + ds.double().abs()
    return dx, (d * n).sum(0), mag, (d * n).abs().sum(0)


def values8(q, scale, cols):
    """The float64 values of the 8-bit form, decoded bit by bit."""
    b = torch.arange(256)
    e, f = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e > 0, (1 + f / 8) * torch.exp2(e.double() - 7), f / 8 * 2.0 ** -6)
    v = torch.where(b >= 128, -v, v)
    v[0x7F] = v[0xFF] = float("nan")
    q, s = q.view(torch.uint8).long().cpu(), scale.view(torch.uint8).double().cpu()
    s = torch.where(s == 255, float("nan"), torch.exp2(s - 127))
    return (v[q].view(len(q), -1, 128) * s[:, :, None]).view(len(q), -1)[:, :cols]

"""The sequence-tower operators as a user's program calls them, on the sizes that such programs meet.

One gated recurrent tower over token ids, the sibling of the GRU tower: the ids' embedding rows, scaled
(and the table's gradient by sorted tokens); the root-mean-square norm with the residual's addition, as
a training pair or with its output in 8 bits; the 8-bit product with a scale for each block of 128; and
the gated linear recurrence, over ragged batches of short texts, over a few very long ones, and for one
token of a running state.

`own` false: the operators' plain form, elementary torch operations in 32 bits, rounded once at the end.
`own` true: the framework's entry points (dssm_amd.api).
"""
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BLOCK = 128  # columns that share a scale in the 8-bit form


def listed():
    return [
        # one step's ids of the RNN tower's benchmark (6144 rows of 32 ids, the 21128-word vocabulary,
        # 128 columns), looked up into bf16 and scaled by sqrt(E); the gradient of the same lookup
        {"name": "embed_tower", "op": "embed", "n": 196608, "v": 21128, "e": 128, "dtype": "fp32", "out": "bf16"},
        {"name": "embed_grad_tower", "op": "embed_grad", "n": 196608, "v": 21128, "e": 128, "dtype": "bf16"},
        # a trigram-sized vocabulary times ten, odd width, few tokens: the dense gradient is mostly zeros
        {"name": "embed_grad_sparse", "op": "embed_grad", "n": 20011, "v": 300007, "e": 100, "dtype": "fp32"},
        # the tower's training step: ragged rows (some empty), both halves of one projection
        {"name": "recur_train_tower", "op": "recur_train", "r": 6144, "t": 32, "h": 128, "dtype": "bf16",
         "lens": True, "reverse": False, "h0": False},
        # training on a few long documents, backwards in time, from a carried state
        {"name": "recur_train_long", "op": "recur_train", "r": 4, "t": 16411, "h": 256, "dtype": "fp32",
         "lens": True, "reverse": True, "h0": True},
        # reading two very long documents
        {"name": "recur_long", "op": "recur", "r": 2, "t": 65537, "h": 512, "dtype": "bf16", "lens": False,
         "reverse": False, "h0": True},
        # serving: one token of each of 256 running states
        {"name": "recur_step", "op": "recur_step", "r": 256, "h": 512, "dtype": "bf16"},
        # the training pair over one step's tokens
        {"name": "norm_train_tower", "op": "norm_train", "rows": 196608, "cols": 256, "dtype": "bf16"},
        # serving: a handful of single tokens, then a long batch, with the output in 8 bits
        {"name": "norm8_tokens", "op": "norm8", "rows": 8, "cols": 4096, "dtype": "bf16"},
        {"name": "norm8_batch", "op": "norm8", "rows": 24571, "cols": 1024, "dtype": "bf16"},
        # the 8-bit product: single tokens against a square layer, and a long batch
        {"name": "product8_tokens", "op": "product8", "m": 7, "n": 4096, "k": 4096, "out": "bf16", "bias": True},
        {"name": "product8_batch", "op": "product8", "m": 8192, "n": 4096, "k": 8192, "out": "bf16", "bias": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "recur", "recur_train", "recur_step", "norm_train", "norm8", "product8"])
    dt = rng.choice(["bf16", "bf16", "fp32", "fp16"])
    flag = lambda: rng.random() < 0.5  # noqa: E731
    if op == "embed":
        return {"op": op, "n": _log(rng, 1, 200000), "v": _log(rng, 2, 300000), "e": _log(rng, 1, 512), "dtype": dt,
                "out": rng.choice(["bf16", "fp32", "fp16"])}
    if op == "embed_grad":
        return {"op": op, "n": _log(rng, 1, 200000), "v": _log(rng, 2, 300000), "e": _log(rng, 1, 256), "dtype": dt}
    if op in ("recur", "recur_train"):
        t = _log(rng, 1, 65537)
        h = _log(rng, 1, 1024)
        r = _log(rng, 1, max(1, min(8192, 25_000_000 // (t * h))))
        return {"op": op, "r": r, "t": t, "h": h, "dtype": dt, "lens": flag(), "reverse": flag(), "h0": flag()}
    if op == "recur_step":
        return {"op": op, "r": _log(rng, 1, 8192), "h": _log(rng, 1, 1024), "dtype": dt}
    if op in ("norm_train", "norm8"):
        cols = _log(rng, 1, 8192)
        return {"op": op, "rows": _log(rng, 1, max(1, min(200000, 25_000_000 // cols))), "cols": cols, "dtype": dt}
    k = _log(rng, 16, 8192)
    n = _log(rng, 1, 8192)
    return {"op": op, "m": _log(rng, 1, max(1, min(16384, 250_000_000_000 // (n * k)))), "n": n, "k": k,
            "out": rng.choice(["bf16", "fp16"]), "bias": flag()}


def work(case):
    op = case["op"]
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if op == "embed":
        # each token's id and output row, and each of the table's rows that can be met once
        n, v, e = case["n"], case["v"], case["e"]
        return {"bytes": n * 4 + n * e * size[case["out"]] + min(n, v) * e * size[case["dtype"]], "flops": n * e}
    if op == "embed_grad":
        n, v, e = case["n"], case["v"], case["e"]
        return {"bytes": n * 4 + n * e * size[case["dtype"]] + v * e * 4, "flops": n * e + v * e}
    if op in ("recur", "recur_train", "recur_step"):
        b = size[case["dtype"]]
        n = case["r"] * case.get("t", 1) * case["h"]
        # gate, candidate and h; in training also dh in and the two gradients out, with the inputs
        # read again by the backward call
        per = 3 * b if op != "recur_train" else 8 * b
        state = case["r"] * case["h"] * 4 * (4 if op == "recur_train" else 2)
        return {"bytes": n * per + state, "flops": n * (10 if op != "recur_train" else 30)}
    if op == "norm_train":
        n, b = case["rows"] * case["cols"], size[case["dtype"]]
        # x, residual -> y, s; then dy, s, ds -> dx
        return {"bytes": n * 8 * b + case["cols"] * 12 + case["rows"] * 8, "flops": n * 14}
    if op == "norm8":
        n, b = case["rows"] * case["cols"], size[case["dtype"]]
        # x, residual -> s and the 8-bit values with their scales; then the values they stand for
        return {"bytes": n * (3 * b + 2 + 2) + n * 2 // BLOCK + case["cols"] * 4, "flops": n * 8}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": (m + n) * (k + k // BLOCK) + m * n * size[case["out"]] + n * 4, "flops": 2 * m * n * k}


# ---- inputs ------------------------------------------------------------------------------------
def _tokens(g, n, v):
    """Token ids as texts have them: the i-th word about 1/i as often as the first."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * torch.log(torch.tensor(float(v), dtype=torch.float64))) - 1).long().clamp_(0, v - 1).to(torch.int32)


def _power(e):
    """2^(e - 127) of biased exponents, exactly."""
    return torch.where(e > 0, e.int() << 23, torch.full_like(e.int(), 1 << 22)).view(torch.float32)


def _blocks(x):
    """x [rows x K] fp32 in the 8-bit form: K padded with zeros to whole blocks of 128, e4m3 values and
    one power of two for each row's block, the smallest that brings the block into +-448."""
    rows, cols = x.shape
    pad = -cols % BLOCK
    x = torch.nn.functional.pad(x, (0, pad)).view(rows, -1, BLOCK)
    amax = x.abs().amax(2)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-127, 127) + 127
    q = (x / _power(e)[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(rows, cols + pad), e.to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(q, scale):
    """The 32-bit values that an 8-bit form stands for, padding and all."""
    rows, k = q.shape
    return (q.float().view(rows, -1, BLOCK) * _power(scale.view(torch.uint8))[:, :, None]).view(rows, k)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0, dtype="fp32"):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(DTYPES[dtype])

    op, s = case["op"], dict(case)
    if op == "embed":
        s["table"] = normal(case["v"], case["e"], std=case["e"] ** -0.5, dtype=case["dtype"])
        s["ids"] = _tokens(g, case["n"], case["v"])
        s["scale"] = float(case["e"]) ** 0.5
    elif op == "embed_grad":
        s["dy"] = normal(case["n"], case["e"], std=0.1, dtype=case["dtype"])
        s["ids"] = _tokens(g, case["n"], case["v"])
        s["scale"] = float(case["e"]) ** 0.5
    elif op in ("recur", "recur_train"):
        r, t, h, dt = case["r"], case["t"], case["h"], case["dtype"]
        proj = normal(r, t, 2 * h, dtype=dt)  # one projection: the gate's logits beside the candidate
        proj[..., :h] = proj[..., :h] * 1.5 + 2
        s["gate"], s["cand"] = proj[..., :h], proj[..., h:]
        s["lens"] = torch.randint(0, t + 1, (r,), generator=g, device="cuda", dtype=torch.int32) if case["lens"] else None
        s["h0"] = normal(r, h, std=0.5) if case["h0"] else None
        if op == "recur_train":
            s["dh"] = normal(r, t, h, std=0.1, dtype=dt)
            s["dlast"] = normal(r, h)
    elif op == "recur_step":
        proj = normal(case["r"], 2 * case["h"], dtype=case["dtype"])
        s["gate"], s["cand"] = proj[:, : case["h"]], proj[:, case["h"]:]
        s["state"] = normal(case["r"], case["h"], std=0.5)  # moves on with every pass, as it does in serving
    elif op in ("norm_train", "norm8"):
        shape = (case["rows"], case["cols"])
        s["x"], s["residual"] = normal(*shape, dtype=case["dtype"]), normal(*shape, std=2.0, dtype=case["dtype"])
        s["weight"] = normal(case["cols"], std=0.2, mean=1.0)
        if op == "norm_train":
            s["dy"], s["ds"] = normal(*shape, std=0.1, dtype=case["dtype"]), normal(*shape, std=0.1, dtype=case["dtype"])
    else:
        s["a"] = _blocks(normal(case["m"], case["k"]) * torch.exp(normal(case["m"], 1)))
        s["w"] = _blocks(normal(case["n"], case["k"], std=case["k"] ** -0.5))
        s["b"] = normal(case["n"]) if case["bias"] else None
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from dssm_amd import api
    op = s["op"]
    if op == "embed":
        return api.embedding_lookup(s["table"], s["ids"], s["scale"], DTYPES[s["out"]])
    if op == "embed_grad":
        return api.embedding_grad(s["dy"], s["ids"], s["v"], s["scale"])
    if op == "recur":
        return api.linear_recurrence(s["gate"], s["cand"], s["lens"], s["h0"], s["reverse"])
    if op == "recur_train":
        h, last, states = api.linear_recurrence(s["gate"], s["cand"], s["lens"], s["h0"], s["reverse"], save=True)
        grads = api.linear_recurrence_grad(s["gate"], s["cand"], states, s["dh"], s["dlast"], s["lens"], s["reverse"])
        return (h, last) + tuple(grads)
    if op == "recur_step":
        return api.linear_recurrence_step(s["gate"], s["cand"], s["state"]), s["state"]
    if op == "norm_train":
        y, total, rstd = api.rms_norm(s["x"], s["weight"], s["residual"], EPS)
        return (y, total) + tuple(api.rms_norm_grad(s["dy"], total, s["weight"], rstd, s["ds"]))
    if op == "norm8":
        y8, total = api.rms_norm_blocks8(s["x"], s["weight"], s["residual"], EPS)
        return api.dequantize_blocks8(y8, torch.bfloat16), total
    a, w = (api.Blocks8(q, scale, s["k"]) for q, scale in (s["a"], s["w"]))
    return api.blocks8_matmul(a, w, s["b"], DTYPES[s["out"]])


def _scan(u, x):
    """h_t = u_t h_{t-1} + x_t along dim 1 for all t at once: spans of doubling length are joined."""
    u, x, k = u.clone(), x.clone(), 1
    while k < u.shape[1]:
        x[:, k:] += u[:, k:] * x[:, :-k]
        u[:, k:] = u[:, k:] * u[:, :-k]
        k *= 2
    return x, u


def _active(s, t):
    if s["lens"] is None:
        return None
    return (torch.arange(t, device="cuda")[None, :] < s["lens"][:, None])[:, :, None]


def _recur_plain(s):
    gate, cand, dt = s["gate"].float(), s["cand"].float(), s["gate"].dtype
    r, t, h = gate.shape
    on = _active(s, t)
    u, c = torch.sigmoid(gate), cand
    v = torch.sigmoid(-gate)  # 1 - u, without its cancellation
    a, x = u, v * c
    if on is not None:
        a, x = torch.where(on, a, 1.0), torch.where(on, x, 0.0)
    if s["reverse"]:
        a, x = a.flip(1), x.flip(1)
    h0 = s["h0"] if s["h0"] is not None else torch.zeros(r, h, device="cuda")
    hs, span = _scan(a, x)
    hs = hs + span * h0[:, None]
    last = hs[:, -1].clone()
    before = torch.cat([h0[:, None], hs[:, :-1]], 1)
    back = (lambda z: z.flip(1)) if s["reverse"] else (lambda z: z)
    hs = back(hs)
    out = (hs if on is None else torch.where(on, hs, 0.0)).to(dt)
    if s["op"] == "recur":
        return out, last
    dh = s["dh"].float()
    dh = dh if on is None else torch.where(on, dh, 0.0)
    dh = back(dh).clone()
    dh[:, -1] += s["dlast"]
    # the gradient that reaches h_t: g_t = dh_t + a_{t+1} g_{t+1}, the same scan from the other end
    nxt = torch.cat([torch.zeros(r, 1, h, device="cuda"), a.flip(1)[:, :-1]], 1)
    g = _scan(nxt, dh.flip(1))[0].flip(1)
    dh0 = a[:, 0] * g[:, 0]
    g, before = back(g), back(before)
    dgate, dcand = g * (before - c) * u * v, g * v
    if on is not None:
        dgate, dcand = torch.where(on, dgate, 0.0), torch.where(on, dcand, 0.0)
    return out, last, dgate.to(dt), dcand.to(dt), dh0


def _run_plain(s):
    op = s["op"]
    if op == "embed":
        return (s["table"][s["ids"].long()].float() * s["scale"]).to(DTYPES[s["out"]])
    if op == "embed_grad":
        out = torch.zeros(s["v"], s["e"], device="cuda")
        out.index_add_(0, s["ids"].long(), s["dy"].float())
        return out * s["scale"]
    if op in ("recur", "recur_train"):
        return _recur_plain(s)
    if op == "recur_step":
        gate = s["gate"].float()
        h = torch.sigmoid(gate) * s["state"] + torch.sigmoid(-gate) * s["cand"].float()
        s["state"].copy_(h)
        return h.to(s["gate"].dtype), s["state"]
    if op in ("norm_train", "norm8"):
        dt = s["x"].dtype
        total = (s["x"].float() + s["residual"].float()).to(dt)
        f = total.float()
        rstd = torch.rsqrt((f * f).mean(1, keepdim=True) + EPS)
        norm = f * rstd
        y = norm * s["weight"]
        if op == "norm8":
            return _values(*_blocks(y))[:, : s["cols"]].to(torch.bfloat16), total
        dy = s["dy"].float()
        wdy = dy * s["weight"]
        dx = rstd * (wdy - norm * (wdy * norm).mean(1, keepdim=True)) + s["ds"].float()
        return y.to(dt), total, dx.to(dt), (dy * norm).sum(0)
    out = _values(*s["a"]) @ _values(*s["w"]).t()
    return (out if s["b"] is None else out + s["b"]).to(DTYPES[s["out"]])


# ---- the same from the definitions, in 64 bits -----------------------------------------------------
def _e4m3_grid(x):
    """x in 64 bits on the grid of e4m3 (three fraction bits, exponents from -6 up), ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _e4m3_table():
    b = torch.arange(256)
    e, f = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e > 0, (1 + f / 8) * torch.exp2(e.double() - 7), f / 8 * 2.0 ** -6)
    return torch.where(b >= 128, -v, v).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "embed":
        return torch.index_select(s["table"].double(), 0, s["ids"].long()) * s["scale"]
    if op == "embed_grad":
        ids, order = torch.sort(s["ids"].long())
        total = torch.cumsum(torch.nn.functional.pad(s["dy"].double()[order], (0, 0, 1, 0)), 0)
        at = torch.searchsorted(ids, torch.arange(s["v"] + 1, device="cuda"))
        return (total[at[1:]] - total[at[:-1]]) * s["scale"]
    if op in ("recur", "recur_train"):
        gate, c = s["gate"].double(), s["cand"].double()
        r, t, h = gate.shape
        u = 1 / (1 + torch.exp(-gate))
        v = 1 / (1 + torch.exp(gate))
        lens = s["lens"] if s["lens"] is not None else torch.full((r,), t, device="cuda")
        on = torch.arange(t, device="cuda")[:, None, None] < lens[None, :, None]  # [t, r, 1]
        # step by step, the past-the-end steps as u = 1 with nothing added and nothing learnt
        u1, x = torch.where(on, u.transpose(0, 1), 1.0).contiguous(), torch.where(on, (v * c).transpose(0, 1), 0.0).contiguous()
        hs, before = torch.empty_like(x), torch.empty_like(x)
        state = s["h0"].double() if s["h0"] is not None else torch.zeros(r, h, device="cuda", dtype=torch.float64)
        steps = range(t - 1, -1, -1) if s["reverse"] else range(t)
        for i in steps:
            before[i] = state
            state = torch.addcmul(x[i], u1[i], state)
            hs[i] = state
        out = [torch.where(on, hs, 0.0).transpose(0, 1), state]
        if op == "recur":
            return out
        dh = torch.where(on, s["dh"].double().transpose(0, 1), 0.0)
        g, gs = s["dlast"].double(), torch.empty_like(dh)
        for i in reversed(steps):
            g = g + dh[i]
            gs[i] = g
            g = g * u1[i]
        u, v, c = u.transpose(0, 1), v.transpose(0, 1), c.transpose(0, 1)
        dgate = torch.where(on, gs * (before - c) * u * v, 0.0).transpose(0, 1)
        return out + [dgate, torch.where(on, gs * v, 0.0).transpose(0, 1), g]
    if op == "recur_step":
        gate = s["gate"].double()
        u = 1 / (1 + torch.exp(-gate))
        h = u * s["state"].double() + s["cand"].double() / (1 + torch.exp(gate))
        return [h, h]
    if op in ("norm_train", "norm8"):
        f = (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()
        inv = 1 / torch.sqrt(torch.sum(f ** 2, 1) / s["cols"] + EPS)
        y = f * s["weight"].double() * inv[:, None]
        if op == "norm8":
            z = torch.nn.functional.pad(y, (0, -s["cols"] % BLOCK)).view(s["rows"], -1, BLOCK)
            amax = z.abs().amax(2, keepdim=True)
            scale = torch.exp2(torch.ceil(torch.log2(torch.where(amax > 0, amax, 448.0) / 448)).clamp(-127, 127))
            return [(_e4m3_grid(z / scale) * scale).view(s["rows"], -1)[:, : s["cols"]], f]
        dy, w = s["dy"].double(), s["weight"].double()
        dot = torch.sum(dy * w * f, 1) * inv ** 3 / s["cols"]
        dx = dy * w * inv[:, None] - f * dot[:, None] + s["ds"].double()
        return [y, f, dx, torch.einsum("rc,rc,r->c", dy, f, inv)]
    table = _e4m3_table()
    a, w = (table[q.view(torch.uint8).int()].view(len(q), -1, BLOCK)
            * torch.exp2(scale.view(torch.uint8).double() - 127)[:, :, None] for q, scale in (s["a"], s["w"]))
    out = torch.mm(a.view(len(a), -1), w.view(len(w), -1).t().contiguous())
    return out if s["b"] is None else out + s["b"].double()

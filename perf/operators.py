"""Cases of the sequence-model operators: the gated linear recurrence (forward pass, training pass, single tokens) and the
orthogonalised update of a weight matrix.

`run` computes a case either from elementary torch operations (`own` false) or through this package's entry points (`own` true);
`exact` computes the same outputs from the definitions in 64 bits.

    recurrence   h_t = a_t h_{t-1} + b_t  per channel, a_t = g, exp(g) or sigmoid(g) of the gate g ("decay", "log", "sigmoid"),
                 b_t = x_t, or (1 - a_t) x_t when coupled (the exact step of h' = r (x - h)); states restart at sequence starts
    update       u = g + beta m',  m' = beta m + g;  X = u / |u|;  five times X <- 3.4445 X - 4.7750 A X + 2.0315 A A X, A = X X'
"""
import math

import torch

own = False

COEFFS = (3.4445, -4.7750, 2.0315)
BETA = 0.95
TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a prompt of one user before the first answered token: few rows, the time axis has to be split
        dict(name="prefill_512", op="scan", batch=1, length=512, channels=2048, seqs=0, dtype="bf16", form="log", coupled=True, fused=True),
        # one whole document or recorded signal in one pass: the longest axis, the largest forward pass
        dict(name="prefill_65536", op="scan", batch=1, length=65536, channels=2048, seqs=0, dtype="bf16", form="log", coupled=False, fused=False),
        # prompts of several users packed without padding: ragged lengths, among them empty ones and single tokens, and a padded tail
        dict(name="packed_37", op="scan", batch=1, length=16381, channels=1024, seqs=37, dtype="f16", form="sigmoid", coupled=True, fused=False),
        # a training batch: input and gate are the two halves of one projection
        dict(name="train_8x4096", op="train", batch=8, length=4096, channels=2048, seqs=0, dtype="bf16", form="sigmoid", coupled=True, fused=True),
        # a small model in 32 bits with sizes that fit no tile
        dict(name="train_odd_f32", op="train", batch=2, length=2047, channels=777, seqs=0, dtype="f32", form="decay", coupled=False, fused=False),
        # one answered token of one user: nothing but latency
        dict(name="token_1", op="step", batch=1, slots=1, channels=2048, dtype="bf16", form="log", coupled=True),
        # one token for each of 256 running users, their states scattered over a pool of 512
        dict(name="token_256", op="step", batch=256, slots=512, channels=4096, dtype="bf16", form="log", coupled=True),
        # the hidden layer of a neural ODE, 128 wide
        dict(name="update_128", op="update", batch=1, rows=128, cols=128, dtype="f32", momentum=False),
        # a layer of sizes that fit no tile, in 32 bits
        dict(name="update_333x500", op="update", batch=1, rows=500, cols=333, dtype="f32", momentum=True),
        # the projections of all heads of a layer, orthogonalised one by one
        dict(name="update_heads", op="update", batch=16, rows=256, cols=1024, dtype="bf16", momentum=True),
        # a square projection
        dict(name="update_4096", op="update", batch=1, rows=4096, cols=4096, dtype="bf16", momentum=True),
        # the wide projection of a block, tall as it is stored
        dict(name="update_tall", op="update", batch=1, rows=8192, cols=2048, dtype="bf16", momentum=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "train", "train", "step", "update", "update"])
    form, coupled = rng.choice(["decay", "log", "sigmoid"]), rng.random() < 0.5
    if op in ("scan", "train"):
        dtype = rng.choice(["bf16", "bf16", "f16", "f32", "f64"])
        batch, length, channels = _log_int(rng, 1, 32), _log_int(rng, 1, 65536 if op == "scan" else 8192), _log_int(rng, 1, 4096)
        most = (1 << 26 if op == "scan" else 1 << 25) // {"f64": 4, "f32": 2}.get(dtype, 1)
        batch = max(1, min(batch, most // (length * channels)))
        channels = max(1, min(channels, most // (length * batch)))
        seqs = _log_int(rng, 1, 100) if rng.random() < 0.3 else 0
        return dict(op=op, batch=1 if seqs else batch, length=length, channels=channels, seqs=seqs, dtype=dtype, form=form, coupled=coupled, fused=rng.random() < 0.4)
    if op == "step":
        batch = _log_int(rng, 1, 512)
        return dict(op=op, batch=batch, slots=batch + rng.randrange(0, 2 * batch + 1), channels=_log_int(rng, 1, 4096), dtype=rng.choice(["bf16", "f16", "f32", "f64"]), form=form, coupled=coupled)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    most = 4096 if dtype == "bf16" else 640
    rows, cols, batch = _log_int(rng, 2, most), _log_int(rng, 2, most), _log_int(rng, 1, 16)
    batch = max(1, min(batch, (1 << 22) // (rows * cols)))
    return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=dtype, momentum=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _gate(gen, form, *shape):
    """Gates of a trained layer: every channel with a time constant of its own, from one token to a thousand, moved by each token."""
    rate = torch.exp(math.log(1e-3) * torch.rand(shape[-1], generator=gen, device="cuda"))        # 1 ... 1e-3 a token
    moved = _randn(gen, *shape).mul_(0.5).exp_().mul_(rate)
    if form == "log":
        return moved.neg_()
    if form == "decay":
        return moved.neg_().exp_()
    a = moved.neg_().exp_().clamp_(1e-3, 0.9995)
    return torch.logit(a)


def _offsets(case, seed):
    """Starts of the packed sequences and the end of the last: one empty sequence and one single token at least where there are three, and a tail without a sequence."""
    s, n = case["seqs"], case["length"]
    gen = torch.Generator().manual_seed(seed + 17)
    end = n - min(n // 50, 40)
    cuts = torch.randint(0, end + 1, (s - 1,), generator=gen).sort().values.tolist() if s > 1 else []
    at = [0] + cuts + [end]
    if s >= 3:
        at[2] = min(at[1] + 1, end)
        at[3] = max(at[3], at[2])
        at[1] = min(at[1], at[2])
        at[s - 1] = at[s]
        for i in range(1, s + 1):
            at[i] = max(at[i], at[i - 1])
    return at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    wide = torch.float64 if case["dtype"] == "f64" else torch.float32
    st = dict(case=case)
    if case["op"] == "update":
        b, r, c = case["batch"], case["rows"], case["cols"]
        k = max(1, min(r, c) // 8)
        # a gradient: a sum of outer products that spans few directions, and noise of the batch
        left, right = _randn(gen, b, r, k), _randn(gen, b, k, c)
        g = torch.bmm(left, right).mul_(1 / math.sqrt(k)).add_(_randn(gen, b, r, c), alpha=0.3).mul_(1e-3)
        st["grad"] = g.to(dt)
        st["momentum"] = _randn(gen, b, r, c).mul_(2e-3) if case["momentum"] else None
        return st
    d = case["channels"]
    if case["op"] == "step":
        b, s = case["batch"], case["slots"]
        st["x"], st["gate"] = _randn(gen, b, d).to(dt), _gate(gen, case["form"], b, d).to(dt)
        st["state"] = _randn(gen, s, d).to(wide)
        st["slots"] = torch.randperm(s, generator=gen, device="cuda")[:b].to(torch.int32) if s > b else None
        return st
    n, b = case["length"], case["batch"]
    shape = (n, d) if case["seqs"] else (b, n, d)
    if case["fused"]:
        both = torch.empty(*shape[:-1], 2 * d, dtype=dt, device="cuda")
        both[..., :d] = _randn(gen, *shape)
        both[..., d:] = _gate(gen, case["form"], *shape)
        st["x"], st["gate"] = both[..., :d], both[..., d:]
    else:
        st["x"], st["gate"] = _randn(gen, *shape).to(dt), _gate(gen, case["form"], *shape).to(dt)
    st["at"] = _offsets(case, seed) if case["seqs"] else None
    st["offsets"] = torch.tensor(st["at"], dtype=torch.int32, device="cuda") if case["seqs"] else None
    rows = case["seqs"] or b
    st["h0"] = _randn(gen, rows, d).to(wide)
    if case["op"] == "train":
        st["dh"] = _randn(gen, *shape).to(dt)
        st["dh_final"] = _randn(gen, rows, d).to(wide)
    return st


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        import scimlsensitivity_jl_amd as sa
        if case["op"] == "update":
            u = sa.orthogonalized_update(state["grad"], state["momentum"], beta=BETA)
            return [u] if state["momentum"] is None else [u, state["momentum"]]
        if case["op"] == "step":
            h = sa.gated_recurrence_step(state["x"], state["gate"], state["state"], form=case["form"], coupled=case["coupled"], slots=state["slots"])
            return [h, state["state"]]
        sol = sa.recurrence_solve(state["x"], state["gate"], state["h0"], form=case["form"], coupled=case["coupled"], offsets=state["offsets"], adjoint=case["op"] == "train")
        if case["op"] == "scan":
            return [sol.h, sol.h_final]
        dx, dgate, dh0 = sa.recurrence_adjoint(sol, state["dh"], state["dh_final"])
        return [sol.h, sol.h_final, dx, dgate, dh0]
    if case["op"] == "update":
        return _plain_update(state)
    if case["op"] == "step":
        return _plain_step(state)
    return _plain_scan(state)


def _wide(t):
    return t.double() if t.dtype == torch.float64 else t.float()


def _decay(case, gate):
    """a and 1 - a, each from the form that loses no digits."""
    g = _wide(gate)
    if case["form"] == "decay":
        return g, 1 - g
    if case["form"] == "log":
        return torch.exp(g), -torch.expm1(g)
    return torch.sigmoid(g), torch.sigmoid(-g)


def _shift(t, k, fill):
    """t moved by k rows along the time axis (rows from the other side are `fill`)."""
    out = torch.full_like(t, fill)
    if k >= 0:
        out[:, k:] = t[:, :t.shape[1] - k]
    else:
        out[:, :k] = t[:, -k:]
    return out


def _scan(a, b, backwards=False):
    """All h_t = a_t h_{t-1} + b_t from zero, by doubling: after step k a pair (a, b) spans 2^k rows."""
    k, n = 1, a.shape[1]
    sign = -1 if backwards else 1
    while k < n:
        b = b + a * _shift(b, sign * k, 0.0)
        a = a * _shift(a, sign * k, 1.0) if 2 * k < n else a
        k *= 2
    return b


def _plain_scan(state):
    case, x, gate, h0 = state["case"], state["x"], state["gate"], state["h0"]
    packed = state["offsets"] is not None
    if packed:
        x, gate = x[None], gate[None]
    a, rest = _decay(case, gate)
    xw = _wide(x)
    b = rest * xw if case["coupled"] else xw
    n = a.shape[1]
    if packed:
        off = state["offsets"].long()
        lens = off[1:] - off[:-1]
        row = torch.arange(n, device="cuda")
        seq = torch.searchsorted(off[1:].contiguous(), row, right=True).clamp_max(lens.numel() - 1)
        inside = ((row >= off[0]) & (row < off[-1]))[None, :, None]
        first = (row == off[seq])[None, :, None] & inside
        start = h0[seq][None]
    else:
        inside = torch.ones(1, n, 1, dtype=torch.bool, device="cuda")
        first = torch.zeros(1, n, 1, dtype=torch.bool, device="cuda")
        first[:, 0] = True
        start = h0[:, None]
    zero = torch.zeros((), dtype=a.dtype, device="cuda")
    keep = torch.where(first | ~inside, zero, a)                          # no state crosses a start
    src = torch.where(inside, b + torch.where(first, a * start, zero), zero)
    h = _scan(keep, src)
    if packed:
        empty = (lens == 0)[:, None]
        h_final = torch.where(empty, h0, h[0, (off[1:] - 1).clamp_min(0)])
    else:
        h_final = h[:, -1].clone()
    shape = state["x"].shape
    outs = [h.reshape(shape).to(x.dtype), h_final]
    if case["op"] == "scan":
        return outs
    dh, dhf = _wide(state["dh"].reshape(h.shape)), state["dh_final"]
    dh = torch.where(inside, dh, zero)
    if packed:
        dh = dh.index_add(1, (off[1:] - 1).clamp_min(0), torch.where(empty, zero, dhf)[None])
    else:
        dh[:, -1] += dhf
    G = _scan(_shift(keep, -1, 0.0), dh, backwards=True)
    before = torch.where(first, start, _shift(h, 1, 0.0))
    da = G * (before - xw if case["coupled"] else before)
    dx = G * rest if case["coupled"] else G
    if case["form"] == "log":
        da = da * a
    elif case["form"] == "sigmoid":
        da = da * a * rest
    da, dx = torch.where(inside, da, zero), torch.where(inside, dx, zero)
    if packed:
        at = off[:-1].clamp_max(n - 1)
        dh0 = torch.where(empty, dhf, a[0, at] * G[0, at])
    else:
        dh0 = a[:, 0] * G[:, 0]
    return outs + [dx.reshape(shape).to(x.dtype), da.reshape(shape).to(x.dtype), dh0]


def _plain_step(state):
    case, pool = state["case"], state["state"]
    a, rest = _decay(case, state["gate"])
    x = _wide(state["x"])
    at = slice(None) if state["slots"] is None else state["slots"].long()
    h = a * pool[at] + (rest * x if case["coupled"] else x)
    pool[at] = h
    return [h.to(state["x"].dtype), pool]


def _plain_update(state):
    g, m = state["grad"], state["momentum"]
    u = g.float()
    if m is not None:
        m.mul_(BETA).add_(u)
        u = u + BETA * m
    tall = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2).contiguous() if tall else u
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + 1e-7)
    for _ in range(5):
        p = torch.bmm(x, x.transpose(1, 2).contiguous())
        q = COEFFS[1] * p + COEFFS[2] * torch.bmm(p, p)
        x = COEFFS[0] * x + torch.bmm(q, x)
    x = (x.transpose(1, 2) if tall else x).to(g.dtype).contiguous()
    return [x] if m is None else [x, m]


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _walk(a, b, start, out, backwards=False):
    """out[t] = a[t] out[t-1] + b[t], row after row (the time axis is the first one)."""
    h = start
    rows = range(a.shape[0])
    for t in (reversed(rows) if backwards else rows):
        h = torch.addcmul(b[t], a[t], h, out=out[t])
    return h


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "update":
        x = st["grad"].double()
        outs = []
        if st["momentum"] is not None:
            m = BETA * st["momentum"].double() + x
            x = x + BETA * m
            outs = [m]
        done = []
        for y in x:
            flip = y.shape[0] > y.shape[1]
            y = y.t().contiguous() if flip else y
            y = y / (y.pow(2).sum().sqrt() + 1e-7)
            for _ in range(5):
                gram = y @ y.t().contiguous()
                once = gram @ y
                y = COEFFS[0] * y + COEFFS[1] * once + COEFFS[2] * (gram @ once)
            done.append(y.t() if flip else y)
        return [torch.stack(done)] + outs
    g, x = st["gate"].double(), st["x"].double()
    if case["form"] == "decay":
        a, one_less = g, 1 - g
    elif case["form"] == "log":
        a, one_less = g.exp(), -torch.expm1(g)
    else:
        a, one_less = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
    b = x * one_less if case["coupled"] else x
    if case["op"] == "step":
        pool = st["state"].double()
        at = torch.arange(case["batch"], device="cuda") if st["slots"] is None else st["slots"].long()
        h = a * pool[at] + b
        pool[at] = h
        return [h, pool]
    h0 = st["h0"].double()
    if case["seqs"]:
        pieces = [(slice(lo, hi), s) for s, (lo, hi) in enumerate(zip(st["at"][:-1], st["at"][1:]))]
        aT, bT, xT, startT = a, b, x, h0
        ends = [h0[s].clone() for _, s in pieces]
    else:
        pieces = [(slice(0, case["length"]), None)]
        aT, bT, xT = (t.transpose(0, 1).contiguous() for t in (a, b, x))
        startT, ends = h0, [h0]
    h = torch.zeros_like(aT)
    prev = torch.zeros_like(aT)
    for i, (cut, s) in enumerate(pieces):
        if cut.stop > cut.start:
            begin = startT if s is None else startT[s]
            ends[i] = _walk(aT[cut], bT[cut], begin, h[cut]).clone()
            prev[cut.start] = begin
            prev[cut.start + 1:cut.stop] = h[cut.start:cut.stop - 1]
    back = (lambda t: t) if case["seqs"] else (lambda t: t.transpose(0, 1))
    h_final = torch.stack(ends) if case["seqs"] else ends[0]
    outs = [back(h), h_final]
    if case["op"] == "scan":
        return outs
    dh = st["dh"].double() if case["seqs"] else st["dh"].double().transpose(0, 1).contiguous()
    dhf = st["dh_final"].double()
    G = torch.zeros_like(dh)
    dh0 = dhf.clone()
    for cut, s in pieces:
        if cut.stop > cut.start:
            aa, dd = aT[cut], dh[cut].clone()
            dd[-1] += dhf if s is None else dhf[s]
            follow = torch.cat([aa[1:], torch.zeros_like(aa[:1])])
            last = _walk(follow, dd, torch.zeros_like(dd[0]), G[cut], backwards=True)
            end = aa[0] * last
            if s is None:
                dh0 = end
            else:
                dh0[s] = end
    rest = one_less if case["seqs"] else one_less.transpose(0, 1)
    dx = G * rest if case["coupled"] else G
    dg = G * (prev - xT) if case["coupled"] else G * prev
    if case["form"] == "log":
        dg = dg * aT
    elif case["form"] == "sigmoid":
        dg = dg * aT * rest
    return outs + [back(dx), back(dg), dh0]


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    size = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    wide = 8 if case["dtype"] == "f64" else 4
    if case["op"] == "update":
        b, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
        # the two symmetric products need half their entries: X X' m m n, A A m m m, and B X 2 m m n
        return {"bytes": b * m * n * (2 * size + (8 if case["momentum"] else 0)), "flops": b * 5 * (3 * m * m * n + m * m * m)}
    d = case["channels"]
    if case["op"] == "step":
        return {"bytes": case["batch"] * d * (3 * size + 2 * wide), "flops": 2 * case["batch"] * d}
    cells, rows = case["batch"] * case["length"] * d, (case["seqs"] or case["batch"]) * d
    if case["op"] == "scan":
        return {"bytes": cells * 3 * size + 2 * rows * wide, "flops": 2 * cells}
    return {"bytes": cells * 6 * size + 4 * rows * wide, "flops": 8 * cells}

"""Plain row-by-row evaluation of the gated linear recurrence and of its gradients in extended precision (80 bits), with a bound of what a computation in
working precision u may be off.

The bound follows the recurrence: a step h = a h + b commits at most K u (|a h| + |b|) — the decay and 1 - a each within 4 u (exponential, its correction, reciprocal),
their products and the fused sum 2 u, and the same again because a state reaches a row through a product of decays formed apart from the row-by-row sum — and hands on
|a| times the error before it.  The reverse recurrence alike; products of computed factors add their relative errors.  Rounding the result to its type adds half a
step of the type."""
import numpy as np

K = 16
LD = np.longdouble


def decay(form, g):
    if form == "decay":
        return g, 1 - g
    if form == "log":
        return np.exp(g), -np.expm1(g)
    return 1 / (1 + np.exp(-g)), 1 / (1 + np.exp(g))


def solve(x, g, h0, form, coupled, u):
    """One sequence: x, g [L][D], h0 [D].  (h, h_final), each (value, bound)."""
    x, g, h0 = LD(x), LD(g), LD(h0)
    with np.errstate(all="ignore"):
        a, rest = decay(form, g)
        b = rest * x if coupled else x
    L, D = x.shape
    h = np.zeros((L, D), LD); E = np.zeros((L, D), LD)
    s, e = h0.copy(), np.zeros(D, LD)
    size = np.abs(h0)
    for t in range(L):
        size = np.abs(a[t]) * size + np.abs(b[t])
        e = np.abs(a[t]) * e + K * u * size
        s = a[t] * s + b[t]
        h[t], E[t] = s, e
    return (h, E), (s, e)


def adjoint(x, g, h0, form, coupled, u, dh, dhf):
    """(dx, dgate, dh0), each (value, bound)."""
    x, g, h0, dh, dhf = LD(x), LD(g), LD(h0), LD(dh), LD(dhf)
    a, rest = decay(form, g)
    (h, Eh), _ = solve(x, g, h0, form, coupled, u)
    L, D = x.shape
    dx = np.zeros((L, D), LD); Ex = np.zeros((L, D), LD); dg = np.zeros((L, D), LD); Eg = np.zeros((L, D), LD)
    R, eR, sR = dhf.copy(), np.zeros(D, LD), np.abs(dhf)
    for t in range(L - 1, -1, -1):
        G, eG, sG = dh[t] + R, eR + K * u * (np.abs(dh[t]) + sR), np.abs(dh[t]) + sR
        prev, eprev = (h[t - 1], Eh[t - 1]) if t else (h0, np.zeros(D, LD))
        d = prev - x[t] if coupled else prev
        ed = eprev + (u * (np.abs(prev) + np.abs(x[t])) if coupled else 0)
        val, err = G * d, np.abs(G) * ed + np.abs(d) * eG + eG * ed
        fac = a[t] if form == "log" else a[t] * rest[t] if form == "sigmoid" else np.ones(D, LD)
        dg[t], Eg[t] = val * fac, np.abs(fac) * (err + K * u * np.abs(val))
        f = rest[t] if coupled else np.ones(D, LD)
        dx[t], Ex[t] = G * f, np.abs(f) * (eG + K * u * np.abs(G))
        R, eR, sR = a[t] * G, np.abs(a[t]) * eG + K * u * np.abs(a[t]) * sG, np.abs(a[t]) * sG
    return (dx, Ex), (dg, Eg), (R, eR)


def whole(x, g, h0, form, coupled, u, pieces, dh=None, dhf=None):
    """All sequences of a [R][L][D] batch or, with pieces = offsets, of packed [1][L][D] rows: {name: (value, bound)}; rows of no sequence are zero."""
    B, L, D = x.shape
    seqs = [(b, 0, L) for b in range(B)] if pieces is None else [(0, lo, hi) for lo, hi in zip(pieces[:-1], pieces[1:])]
    S = len(seqs)
    h0 = np.zeros((S, D)) if h0 is None else h0
    o = {"h": np.zeros((2, B, L, D), LD), "h_final": np.zeros((2, S, D), LD)}
    if dh is not None:
        o.update(dx=np.zeros((2, B, L, D), LD), dgate=np.zeros((2, B, L, D), LD), dh0=np.zeros((2, S, D), LD))
    for s, (b, lo, hi) in enumerate(seqs):
        cut = (slice(None), b, slice(lo, hi))
        h, hf = solve(x[b, lo:hi], g[b, lo:hi], h0[s], form, coupled, u)
        o["h"][cut], o["h_final"][:, s] = np.stack(h), np.stack(hf)
        if dh is not None:
            dx, dg, d0 = adjoint(x[b, lo:hi], g[b, lo:hi], h0[s], form, coupled, u, dh[b, lo:hi], dhf[s])
            o["dx"][cut], o["dgate"][cut], o["dh0"][:, s] = np.stack(dx), np.stack(dg), np.stack(d0)
    return o

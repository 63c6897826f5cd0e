"""The operators as they are used together (`-m gpu`): a sequence layer whose gradients come from the recurrence's adjoint and whose weights take orthogonalised steps, and a neural ODE
trained by the adjoint solve and the same update; and what the calls refuse."""
import numpy as np
import pytest

import orthogonal_oracle as OO
import recurrence_oracle as RO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def layer(torch, x, W, V):
    """Input and gate of the recurrence from one projection, and its read-out: x [B][L][D], W [D][2 D], V [D][D]."""
    both = x @ W
    d = x.shape[-1]
    return both[..., :d], -torch.nn.functional.softplus(both[..., d:]), V


def test_sequence_layer_trains(sa, torch):
    """One projection -> (input, log-decay) -> recurrence -> read-out, in 32 bits: loss and gradients against the oracle's recurrence in 80 bits inside the same layer, then orthogonalised
    steps of both weights with momentum."""
    rng = np.random.default_rng(3)
    B, L, D = 2, 130, 24
    X, T = rng.standard_normal((B, L, D)), rng.standard_normal((B, L, D))
    W0, V0 = rng.standard_normal((D, 2 * D)) / D ** 0.5, rng.standard_normal((D, D)) / D ** 0.5
    dev = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda")        # noqa: E731
    x, t, W, V = dev(X), dev(T), dev(W0).requires_grad_(), dev(V0).requires_grad_()
    mW, mV = torch.zeros_like(W), torch.zeros_like(V)

    def loss_of():
        u, g, v = layer(torch, x, W, V)
        h, _ = sa.gated_recurrence(u, g, form="log", coupled=True)
        return ((h @ v - t) ** 2).mean()
    loss = loss_of()
    loss.backward()
    # the same layer in 64 bits around the oracle
    Wd, Vd = (np.float64(p.detach().cpu().numpy()) for p in (W, V))
    Xd, Td = (np.float64(a.cpu().numpy()) for a in (x, t))
    both = Xd @ Wd
    gate = -np.log1p(np.exp(both[..., D:]))
    o = RO.whole(both[..., :D], gate, None, "log", True, 0, None)
    h = np.float64(o["h"][0])
    e = h @ Vd - Td
    dy = 2 * e / e.size
    dh = dy @ Vd.T
    grads = RO.whole(both[..., :D], gate, None, "log", True, 0, None, dh, np.zeros((B, D)))
    dboth = np.concatenate([np.float64(grads["dx"][0]), np.float64(grads["dgate"][0]) * (-1 / (1 + np.exp(-both[..., D:])))], -1)
    want_W, want_V = np.einsum("bld,ble->de", Xd, dboth), np.einsum("bld,ble->de", h, dy)
    assert abs(loss.item() - np.mean(e ** 2)) < 1e-5 * np.mean(e ** 2)
    # sums of 260 products in 32 bits, each factor within a few 2^-24 of its size and the recurrence's memory of about ten rows: 1e-5 of the norm leaves a factor of ten
    for got, want in ((W.grad, want_W), (V.grad, want_V)):
        assert np.linalg.norm(got.double().cpu().numpy() - want) < 1e-5 * np.linalg.norm(want)
    for step in range(3):
        for p, m in ((W, mW), (V, mV)):
            g, before = p.grad.double().cpu().numpy(), m.double().cpu().numpy()
            u = sa.orthogonalized_update(p.grad, m, scale=0.02)
            want, want_m, v = OO.update(g, before, scale=0.02)
            norm, most = OO.allowance(v, 2.0 ** -20, scale=0.02)
            assert np.linalg.norm(u.double().cpu().numpy() - want) <= norm + 2.0 ** -24 * np.linalg.norm(want)
            with torch.no_grad():
                p -= u
            p.grad = None
        loss = loss_of()
        loss.backward()
        assert torch.isfinite(loss) and torch.isfinite(W.grad).all() and torch.isfinite(V.grad).all()


def test_prompt_then_tokens(sa, torch):
    """Serving: packed prompts of three users in one pass, their final states into a pool, then single tokens by slot: every state and output as in one solve of the whole sequences."""
    rng = np.random.default_rng(4)
    D, lens, more = 40, [37, 1, 90], 6
    full = [rng.standard_normal((n + more, D)) for n in lens]
    gate = [-np.exp(rng.standard_normal((n + more, D)) - 1) for n in lens]
    dev = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda")        # noqa: E731
    off = np.concatenate([[0], np.cumsum(lens)])
    sol = sa.recurrence_solve(dev(np.concatenate([f[:n] for f, n in zip(full, lens)])), dev(np.concatenate([g[:n] for g, n in zip(gate, lens)])), form="log", coupled=True,
                              offsets=torch.tensor(off, dtype=torch.int32, device="cuda"), adjoint=False)
    pool, slots = torch.zeros(8, D, device="cuda"), torch.tensor([5, 0, 3], dtype=torch.int32, device="cuda")
    pool[slots.long()] = sol.h_final
    got = [sa.gated_recurrence_step(dev(np.stack([f[n + i] for f, n in zip(full, lens)])), dev(np.stack([g[n + i] for g, n in zip(gate, lens)])), pool, form="log", coupled=True, slots=slots)
           for i in range(more)]
    for s, n in enumerate(lens):
        f32 = lambda a: np.float64(np.float32(a))             # noqa: E731
        (h, E), (last, e) = RO.solve(f32(full[s]), f32(gate[s]), np.zeros(D), "log", True, 2.0 ** -24)
        half = lambda v, b: b + 2.0 ** -24 * (np.abs(v) + b)  # noqa: E731
        assert np.all(np.abs(sol.h[off[s]:off[s + 1]].double().cpu().numpy() - h[:n]) <= half(h[:n], E[:n]))
        for i in range(more):
            assert np.all(np.abs(got[i][s].double().cpu().numpy() - h[n + i]) <= half(h[n + i], E[n + i]))
        assert np.all(np.abs(pool[slots[s]].double().cpu().numpy() - last) <= half(last, e))


def test_neural_ode_takes_orthogonalised_steps(sa, torch):
    """dense_chain -> solve -> adjoint_sensitivities -> WideDeviceFunction.orthogonalized_update -> solve: each weight's part against the definition, biases as they come."""
    rng = np.random.default_rng(5)
    fun = sa.WideDeviceFunction.dense_chain("update_chain", (2, 50, 2), input_power=3)
    p = 0.2 * rng.standard_normal(fun.np)
    u0, ts = np.array([[2.0, 0.0], [1.5, 0.3]]), np.linspace(0.0, 1.0, 6)
    momentum = torch.zeros(fun.np, dtype=torch.float32, device="cuda")
    for step in range(2):
        sol = sa.solve(sa.EnsembleProblem(sa.ODEProblem(fun, u0[0], (0.0, 1.0), p), u0), sa.RK4(), dt=0.02, saveat=ts, sensealg=sa.InterpolatingAdjoint())
        _, dp = sa.adjoint_sensitivities(sol, sa.RK4(), t=ts, dgdu_discrete=2.0 * (sol.u - 1.0))
        sol.engine.close()
        before = momentum.double().cpu().numpy()
        upd = fun.orthogonalized_update(dp, momentum)
        assert upd.shape == p.shape and upd.dtype == np.float64
        g = np.float64(np.float32(dp))
        for off, out, inp in fun.weight_blocks():
            at, bias = slice(off, off + out * inp), slice(off + out * inp, off + out * inp + out)
            want, want_m, v = OO.update(g[at].reshape(inp, out).T, before[at].reshape(inp, out).T, scale=max(1.0, out / inp) ** 0.5)
            norm, _ = OO.allowance(v, 2.0 ** -20, scale=max(1.0, out / inp) ** 0.5)
            assert np.linalg.norm(upd[at].reshape(inp, out).T - want) <= norm + 2.0 ** -24 * np.linalg.norm(want)
            m = 0.95 * before[bias] + g[bias]
            # beta m, its sum with g, beta m', its sum with g: five roundings (0.95 itself is one) of values of at most |g| + |m| + |m'|, which may cancel
            assert np.all(np.abs(upd[bias] - (g[bias] + 0.95 * m)) <= 5 * 2.0 ** -24 * (np.abs(g[bias]) + np.abs(before[bias]) + np.abs(m)))
        p = p - 0.05 * upd
    dense = torch.tensor(dp, device="cuda")
    assert torch.equal(fun.orthogonalized_update(dense), torch.tensor(fun.orthogonalized_update(dp), device="cuda"))
    other = sa.WideDeviceFunction("no_chain", 9, 1, "HIPADJ_W_FOR(i, N) du[i] = -p[0] * u[i];", "HIPADJ_W_FOR(i, N) dlam[i] = -p[0] * lam[i];", nacc=1)
    with pytest.raises(ValueError, match="not a dense_chain"):
        other.orthogonalized_update(np.zeros(1))
    with pytest.raises(ValueError, match="shape"):
        fun.orthogonalized_update(np.zeros(3))


def test_refusals(sa, torch):
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")    # noqa: E731
    x = z(2, 5, 4)
    off = torch.tensor([0, 2, 10], dtype=torch.int32, device="cuda")
    for text, call in [
            ("float64, float32", lambda: sa.recurrence_solve(x.int(), x.int())), ("x's type", lambda: sa.recurrence_solve(x, x.double())), ("x's type", lambda: sa.recurrence_solve(x, x.half())),
            ("shape", lambda: sa.recurrence_solve(x, z(2, 5, 3))), ("form", lambda: sa.recurrence_solve(x, x, form="exp")), ("channels", lambda: sa.recurrence_solve(x[0], x[0])),
            ("h0", lambda: sa.recurrence_solve(x, x, z(2, 3))), ("h0", lambda: sa.recurrence_solve(x, x, z(2, 4, t=torch.bfloat16))), ("h0 lives", lambda: sa.recurrence_solve(x, x, torch.zeros(2, 4))),
            ("offsets", lambda: sa.recurrence_solve(z(10, 4), z(10, 4), offsets=off.float())), ("offsets", lambda: sa.recurrence_solve(z(10, 4), z(10, 4), offsets=off[:1])),
            ("offsets", lambda: sa.recurrence_solve(z(10, 4), z(10, 4), offsets=off.cpu())),
            ("dh", lambda: sa.recurrence_adjoint(sa.recurrence_solve(x, x), z(2, 5, 3))), ("dh_final", lambda: sa.recurrence_adjoint(sa.recurrence_solve(x, x), x, z(2, 3))),
            ("state", lambda: sa.gated_recurrence_step(x[0], x[0], z(5, 4, t=torch.float16))), ("state", lambda: sa.gated_recurrence_step(x[0], x[0], z(5, 3))),
            ("as many states", lambda: sa.gated_recurrence_step(x[0], x[0], z(4, 4))), ("slots", lambda: sa.gated_recurrence_step(x[0], x[0], z(9, 4), slots=off)),
            ("overlap", lambda: sa.gated_recurrence_step(x[0], x[0], z(1, 4).expand(5, 4))),
            ("float32, bfloat16", lambda: sa.orthogonalized_update(z(4, 4, t=torch.float64))), ("rows, cols", lambda: sa.orthogonalized_update(z(4))),
            ("momentum", lambda: sa.orthogonalized_update(z(4, 4), z(4, 5))), ("momentum", lambda: sa.orthogonalized_update(z(4, 4), z(4, 4, t=torch.bfloat16))),
            ("momentum", lambda: sa.orthogonalized_update(z(4, 4), z(1, 4).expand(4, 4))), ("both be row-major", lambda: sa.orthogonalized_update(z(4, 6), z(6, 4).t(), out=z(4, 6))),
            ("coefficients", lambda: sa.orthogonalized_update(z(4, 4), coefficients=(1.0, 2.0)))]:
        with pytest.raises(ValueError, match=text):
            call()
    for bad in (dict(steps=0), dict(steps=65), dict(beta=float("inf")), dict(coefficients=(4.0, 0.0, 0.0)), dict(coefficients=(50.0, 0.0, 0.0))):
        with pytest.raises(sa.HipadjError):
            sa.orthogonalized_update(z(4, 4), **bad)


def test_offsets_that_do_not_ascend_stay_inside_the_arrays(sa, torch):
    """Their results are unspecified; the rows of h0, h_final and of the inputs around the given ones are neither read nor written."""
    for off in ([5, 3, 9, 1], [0, 100, 50, 20], [7, 7, 300, 2], [-5, 4, -1, 8]):
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        x = torch.full((20, 66), 0.5, device="cuda")
        sol = sa.recurrence_solve(x, -x, torch.zeros(3, 66, device="cuda"), form="log", offsets=o)
        grads = sa.recurrence_adjoint(sol, torch.ones_like(x), torch.ones(3, 66, device="cuda"))
        torch.cuda.synchronize()
        assert sol.h.shape == (20, 66) and grads[2].shape == (3, 66)

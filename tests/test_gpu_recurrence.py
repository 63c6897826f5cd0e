"""The gated linear recurrence on the device (`-m gpu`) against the row-by-row evaluation in extended precision (tests/recurrence_oracle.py), whose bound and half a step
of the output's type are the tolerance."""
import numpy as np
import pytest

import recurrence_oracle as O

pytestmark = pytest.mark.gpu

TYPES = ["float64", "float32", "bfloat16", "float16"]
HALF = {"float64": 2.0 ** -53, "float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}      # finfo.eps / 2
TINY = {"float64": 0.0, "float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -25}          # half a step below the normal range (float32: a flushed result)


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def unit(dtype):
    return 2.0 ** -53 if dtype == "float64" else 2.0 ** -24


def host(t):
    return t.detach().double().cpu().numpy()


def near(got, want, dtype, what):
    value, bound = want
    got = O.LD(host(got)).reshape(value.shape)
    tol = bound + HALF[dtype] * (np.abs(value) + bound) + TINY[dtype]
    assert np.array_equal(np.isnan(got), np.isnan(value)), f"{what}: NaN in other places"
    off = np.where(np.isfinite(value), np.abs(got - value) - tol, np.where(got == value, -1, np.where(np.isnan(value), -1, 1)))
    assert off.max(initial=-1) <= 0, f"{what}: {off.max()} over the bound at {np.unravel_index(off.argmax(), off.shape)}"


def gates(rng, form, shape):
    rate = np.exp(np.log(1e-3) * rng.random(shape[-1]))
    moved = np.exp(0.5 * rng.standard_normal(shape)) * rate
    if form == "log":
        return -moved
    a = np.clip(np.exp(-moved), 1e-3, 0.9995)
    return a if form == "decay" else np.log(a / (1 - a))


def inputs(torch, seed, shape, rows, form, dtype, gate_dtype=None):
    rng = np.random.default_rng(seed)
    wide = torch.float64 if dtype == "float64" else torch.float32
    dev = lambda a, t: torch.tensor(a, dtype=torch.float64).to(t).cuda()
    t, tg = getattr(torch, dtype), getattr(torch, gate_dtype or dtype)
    d = shape[-1]
    return dict(x=dev(rng.standard_normal(shape), t), gate=dev(gates(rng, form, shape), tg), h0=dev(rng.standard_normal((rows, d)), wide),
                dh=dev(rng.standard_normal(shape), t), dhf=dev(rng.standard_normal((rows, d)), wide))


def compare(sa, torch, q, form, coupled, dtype, offsets=None, gate_dtype=None, h0=True):
    packed = offsets is not None
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda") if packed else None
    start = q["h0"] if h0 else None
    sol = sa.recurrence_solve(q["x"], q["gate"], start, form=form, coupled=coupled, offsets=off)
    dx, dg, d0 = sa.recurrence_adjoint(sol, q["dh"], q["dhf"])
    as3 = (lambda t: host(t)[None]) if packed else host
    want = O.whole(as3(q["x"]), as3(q["gate"]), host(q["h0"]) if h0 else None, form, coupled, unit(dtype), offsets, as3(q["dh"]), host(q["dhf"]))
    state = "float64" if dtype == "float64" else "float32"
    for name, got, t in (("h", sol.h, dtype), ("h_final", sol.h_final, state), ("dx", dx, dtype), ("dgate", dg, gate_dtype or dtype), ("dh0", d0, state)):
        near(got, want[name], t, f"{name} {dtype} {form}")
    return sol, (dx, dg, d0)


@pytest.mark.parametrize("coupled", [False, True])
@pytest.mark.parametrize("form", ["decay", "log", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
def test_forms_and_types(sa, torch, dtype, form, coupled):
    compare(sa, torch, inputs(torch, 1, (2, 150, 96), 2, form, dtype), form, coupled, dtype)


@pytest.mark.parametrize("gate_dtype,dtype", [("float32", "bfloat16"), ("float32", "float16")])
def test_gate_in_32_bits_next_to_16(sa, torch, dtype, gate_dtype):
    compare(sa, torch, inputs(torch, 2, (1, 200, 130), 1, "log", dtype, gate_dtype), "log", True, dtype, gate_dtype=gate_dtype)


# lengths around the pieces (8, 16), the tiles (64, 128) and the groups of tiles (512, 1024); channel counts around the lanes and the two-channel path
@pytest.mark.parametrize("length", [0, 1, 2, 7, 8, 15, 16, 17, 63, 64, 65, 127, 128, 129, 511, 513, 1024, 1025, 1300])
def test_lengths(sa, torch, length):
    compare(sa, torch, inputs(torch, 3, (2, length, 6), 2, "sigmoid", "bfloat16"), "sigmoid", True, "bfloat16")
    compare(sa, torch, inputs(torch, 4, (1, length, 3), 1, "log", "float32"), "log", False, "float32")


@pytest.mark.parametrize("channels", [1, 2, 63, 64, 65, 127, 128, 129, 130, 257])
@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_channels(sa, torch, channels, dtype):
    compare(sa, torch, inputs(torch, 5, (3, 140, channels), 3, "log", dtype), "log", True, dtype)


def test_long_axis_of_many_groups(sa, torch):
    compare(sa, torch, inputs(torch, 6, (1, 9000, 5), 1, "log", "float32"), "log", False, "float32")


# one or two, three or four and more chains (of 64 float32 channels): groups of 32, 16 and 8 tiles of 128 rows (adjoint: 64), whole ones and one row more; float64 publishes in other words
@pytest.mark.parametrize("channels", [70, 200, 330])
@pytest.mark.parametrize("length", [2048, 2049, 4096, 4225])
def test_groups_of_tiles_by_the_number_of_chains(sa, torch, channels, length):
    compare(sa, torch, inputs(torch, 26, (1, length, channels), 1, "log", "float32"), "log", True, "float32")


@pytest.mark.parametrize("channels", [64, 192, 320])
def test_groups_of_tiles_in_64_bits(sa, torch, channels):
    compare(sa, torch, inputs(torch, 27, (1, 4100, channels), 1, "sigmoid", "float64"), "sigmoid", True, "float64")


PACKS = [[0, 5], [0, 0, 1, 1, 40], [0, 16, 32, 128, 128, 128, 300], [3, 70, 70, 71, 200, 290], [0, 1, 2, 3, 4, 5, 6, 7, 8, 20, 300], [0, 0, 0], [300, 300], [0, 300], [64, 128, 192, 256]]


@pytest.mark.parametrize("offsets", PACKS, ids=[str(i) for i in range(len(PACKS))])
@pytest.mark.parametrize("dtype,coupled,form", [("bfloat16", True, "sigmoid"), ("float32", False, "log"), ("float64", True, "decay")])
def test_packed_sequences(sa, torch, offsets, dtype, coupled, form):
    """Empty sequences, single rows, starts and ends on and off the borders of pieces and tiles, rows before the first and behind the last."""
    compare(sa, torch, inputs(torch, 7, (300, 70), len(offsets) - 1, form, dtype), form, coupled, dtype, offsets=offsets)


def test_packed_many_sequences_and_64_bit_offsets(sa, torch):
    rng = np.random.default_rng(8)
    offsets = [0] + sorted(rng.integers(0, 2001, 299).tolist()) + [2001]
    q = inputs(torch, 8, (2100, 34), 300, "log", "float32")
    sol, grads = compare(sa, torch, q, "log", True, "float32", offsets=offsets)
    again = sa.recurrence_solve(q["x"], q["gate"], q["h0"], form="log", coupled=True, offsets=torch.tensor(offsets, dtype=torch.int64, device="cuda"))
    assert torch.equal(again.h, sol.h) and torch.equal(again.h_final, sol.h_final)


# a wave looks at 64 sequences together: more empty ones than that between two rows of a piece, before the first and behind the last; 64, 65 and 4096 and more sequences of a row or none
EMPTY = [[0, 3] + [9] * 70 + [12, 300], [0] * 130 + [5, 300], [0, 200] + [300] * 200, [0] + [40] * 63 + [41], [0] + [40] * 64 + [41], list(range(0, 65)), list(range(0, 301)),
         [0] + [i // 16 for i in range(4800)] + [300]]


@pytest.mark.parametrize("offsets", EMPTY, ids=[str(i) for i in range(len(EMPTY))])
@pytest.mark.parametrize("dtype,coupled,form", [("bfloat16", False, "log"), ("float32", True, "sigmoid")])
def test_packed_windows_of_empty_sequences(sa, torch, offsets, dtype, coupled, form):
    compare(sa, torch, inputs(torch, 28, (300, 6), len(offsets) - 1, form, dtype), form, coupled, dtype, offsets=offsets)


def test_nothing_leaks_between_sequences(sa, torch):
    """NaN and infinities of one sequence, and in rows of no sequence, stay there: forward, backward and in the final states."""
    offsets = [2, 100, 230, 290]
    q = inputs(torch, 9, (300, 66), 3, "log", "bfloat16")
    clean = compare(sa, torch, q, "log", True, "bfloat16", offsets=offsets)
    bad = {k: v.clone() for k, v in q.items()}
    for k in ("x", "gate", "dh"):
        bad[k][:2] = float("nan"); bad[k][290:] = float("inf")
        bad[k][100:230] = float("nan")
    bad["h0"][1] = float("inf"); bad["dhf"][1] = float("nan")
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    sol = sa.recurrence_solve(bad["x"], bad["gate"], bad["h0"], form="log", coupled=True, offsets=off)
    grads = sa.recurrence_adjoint(sol, bad["dh"], bad["dhf"])
    for got, want in ((sol.h, clean[0].h), (grads[0], clean[1][0]), (grads[1], clean[1][1])):
        for a, b in ((0, 100), (230, 300)):
            assert torch.equal(got[a:b], want[a:b])
        assert torch.isnan(got[100:230]).all()
    for got, want in ((sol.h_final, clean[0].h_final), (grads[2], clean[1][2])):
        assert torch.equal(got[[0, 2]], want[[0, 2]]) and torch.isnan(got[1]).all()


def test_nan_and_infinite_rows_go_on_in_their_sequence(sa, torch):
    """A NaN state stays NaN however strong the later decays are (also where their product underflows); channels do not mix; a gate of -inf or of the type's lowest value
    forgets everything."""
    q = inputs(torch, 10, (1, 400, 8), 1, "log", "float32")
    q["gate"][0, :, 0] = -30.0; q["x"][0, 130, 0] = float("nan")
    q["gate"][0, 200, 1] = -float("inf"); q["gate"][0, 201, 2] = torch.finfo(torch.float32).min
    compare(sa, torch, q, "log", False, "float32")
    compare(sa, torch, q, "log", True, "float32")
    q["gate"][0, 200, 1] = float("inf"); q["gate"][0, 201, 2] = torch.finfo(torch.float32).max; q["gate"][0, 202, 3] = -float("inf"); q["gate"][0, :, 0] = 0.0
    compare(sa, torch, q, "sigmoid", True, "float32")


@pytest.mark.parametrize("form", ["decay", "log", "sigmoid"])
@pytest.mark.parametrize("packed", [False, True])
def test_gradient_of_a_start_behind_a_strong_decay(sa, torch, form, packed):
    """dh0 = a_1 G_1 leaves in 32 bits also for 16-bit data: exact where a_1 is tiny."""
    q = inputs(torch, 22, (1, 40, 34), 1, form, "bfloat16")
    q["gate"][0, 0] = {"decay": 2e-4, "log": -9.0, "sigmoid": -9.0}[form]
    if packed:
        q = {k: v[0] if v.dim() == 3 else v for k, v in q.items()}
    compare(sa, torch, q, form, True, "bfloat16", offsets=[0, 40] if packed else None)


def test_growing_decays_on_states_of_zero(sa, torch):
    """Decays of two overflow as a product over 128 rows; a state that is still exactly zero stays zero, forward and in the adjoint, and what starts later grows as it should."""
    q = inputs(torch, 21, (1, 700, 6), 1, "decay", "float32")
    q["gate"].fill_(2.0); q["x"].zero_(); q["h0"].zero_(); q["dh"].zero_(); q["dhf"].zero_()
    q["x"][0, 690, 1] = 3.0; q["dh"][0, 12, 2] = 1.5
    sol, (dx, dg, d0) = compare(sa, torch, q, "decay", False, "float32")
    assert float(sol.h[0, 699, 1]) == 3.0 * 2.0 ** 9 and float(dx[0, 0, 2]) == 1.5 * 2.0 ** 12 and float(d0[0, 2]) == 1.5 * 2.0 ** 13
    assert int(torch.count_nonzero(sol.h)) == 10 and int(torch.count_nonzero(dx)) == 13


def test_strides_of_fused_projections_and_broadcast_gates(sa, torch):
    q = inputs(torch, 11, (2, 150, 64), 2, "log", "bfloat16")
    both = torch.empty(2, 150, 128, dtype=torch.bfloat16, device="cuda")
    both[..., :64], both[..., 64:] = q["x"], q["gate"]
    plain = compare(sa, torch, q, "log", True, "bfloat16")
    views = dict(q, x=both[..., :64], gate=both[..., 64:], dh=q["dh"].transpose(0, 1).contiguous().transpose(0, 1))
    viewed = compare(sa, torch, views, "log", True, "bfloat16")
    assert torch.equal(plain[0].h, viewed[0].h) and all(torch.equal(a, b) for a, b in zip(plain[1], viewed[1]))
    odd = torch.empty(2, 150, 131, dtype=torch.bfloat16, device="cuda")           # rows on odd elements: one channel a lane
    odd[..., 1:65], odd[..., 66:130] = q["x"], q["gate"]
    compare(sa, torch, dict(q, x=odd[..., 1:65], gate=odd[..., 66:130]), "log", True, "bfloat16")
    compare(sa, torch, dict(q, gate=q["gate"][:1, :1].expand(2, 150, 64)), "log", True, "bfloat16")
    compare(sa, torch, dict(q, x=q["x"].transpose(1, 2).contiguous().transpose(1, 2)), "log", True, "bfloat16")   # time next to time: copied


def test_no_start_no_cotangents_and_partial_gradients(sa, torch):
    q = inputs(torch, 12, (2, 140, 20), 2, "sigmoid", "float32")
    compare(sa, torch, q, "sigmoid", False, "float32", h0=False)
    sol = sa.recurrence_solve(q["x"], q["gate"], q["h0"], form="sigmoid")
    full = sa.recurrence_adjoint(sol, q["dh"], torch.zeros_like(q["dhf"]))
    only = sa.recurrence_adjoint(sol, q["dh"], need=(False, True, False))
    assert only[0] is None and only[2] is None and torch.equal(only[1], full[1])
    a = sa.recurrence_adjoint(sol, None, q["dhf"]); b = sa.recurrence_adjoint(sol, torch.zeros_like(q["dh"]), q["dhf"])
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert torch.equal(sa.recurrence_solve(q["x"], q["gate"], q["h0"], form="sigmoid", adjoint=False).h, sol.h)
    with pytest.raises(ValueError, match="adjoint=False"):
        sa.recurrence_adjoint(sa.recurrence_solve(q["x"], q["gate"], adjoint=False), q["dh"])


def test_results_do_not_depend_on_the_order_of_the_workgroups(sa, torch):
    q = inputs(torch, 13, (2, 3000, 200), 2, "sigmoid", "bfloat16")
    def once():
        sol = sa.recurrence_solve(q["x"], q["gate"], q["h0"], form="sigmoid", coupled=True)
        return [sol.h, sol.h_final, *sa.recurrence_adjoint(sol, q["dh"], q["dhf"])]
    first = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_autograd_against_the_oracle_and_differences(sa, torch):
    q = inputs(torch, 14, (2, 90, 5), 2, "log", "float64")
    x, g, h0 = (q[k].clone().requires_grad_() for k in ("x", "gate", "h0"))
    h, hf = sa.gated_recurrence(x, g, h0, form="log", coupled=True)
    ((h * q["dh"]).sum() + (hf * q["dhf"]).sum()).backward()
    sol = sa.recurrence_solve(q["x"], q["gate"], q["h0"], form="log", coupled=True)
    for got, want in zip((x.grad, g.grad, h0.grad), sa.recurrence_adjoint(sol, q["dh"], q["dhf"])):
        assert torch.equal(got, want)
    # central differences in 64 bits: step 1e-6, truncation ~1e-12 and cancellation ~1e-9 of a loss of order 100
    def loss(x, g, h0):
        h, hf = sa.gated_recurrence(x, g, h0, form="log", coupled=True)
        return float((h * q["dh"]).sum() + (hf * q["dhf"]).sum())
    for k, grad in (("x", x.grad), ("gate", g.grad), ("h0", h0.grad)):
        step = torch.randn(q[k].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(5)).cuda()
        up, down = ({**q, k: q[k] + s * 1e-6 * step} for s in (1, -1))
        diff = (loss(up["x"], up["gate"], up["h0"]) - loss(down["x"], down["gate"], down["h0"])) / 2e-6
        assert abs(diff - float((grad * step).sum())) < 1e-5 * max(1.0, abs(diff))


def test_autograd_of_broadcast_gates_and_changed_inputs(sa, torch):
    q = inputs(torch, 15, (2, 40, 6), 2, "sigmoid", "float64")
    g = q["gate"][0, 0].clone().requires_grad_()
    h, _ = sa.gated_recurrence(q["x"], g.expand(2, 40, 6), form="sigmoid")
    (h * q["dh"]).sum().backward()
    full = q["gate"][:1, :1].expand(2, 40, 6).clone().requires_grad_()
    h, _ = sa.gated_recurrence(q["x"], full, form="sigmoid")
    (h * q["dh"]).sum().backward()
    assert torch.allclose(g.grad, full.grad.sum((0, 1)), rtol=1e-12, atol=1e-12)
    x = q["x"].clone().requires_grad_()
    y = x * 1.0
    h, _ = sa.gated_recurrence(y, q["gate"], form="sigmoid")
    with torch.no_grad():
        y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("channels", [1, 64, 130, 1027])
def test_single_steps_continue_a_solve(sa, torch, dtype, channels):
    q = inputs(torch, 16, (3, 20, channels), 3, "log", dtype)
    want = O.whole(host(q["x"]), host(q["gate"]), host(q["h0"]), "log", True, unit(dtype), None)
    sol = sa.recurrence_solve(q["x"][:, :15], q["gate"][:, :15], q["h0"], form="log", coupled=True, adjoint=False)
    state = sol.h_final
    for t in range(15, 20):
        h = sa.gated_recurrence_step(q["x"][:, t], q["gate"][:, t], state, form="log", coupled=True)
        near(h, (want["h"][0][:, t], want["h"][1][:, t]), dtype, f"step {t}")
    near(state, want["h_final"], "float64" if dtype == "float64" else "float32", "state")


@pytest.mark.parametrize("bits", [32, 64])
def test_steps_by_slot(sa, torch, bits):
    """Scattered states, padding rows, and rows of one state in a row: consecutive steps."""
    rng = np.random.default_rng(17)
    q = inputs(torch, 17, (9, 70), 12, "sigmoid", "float32")
    slots = [4, -1, 7, 4, 0, 12, 4, 11, 7]
    state = q["h0"].clone()
    h = sa.gated_recurrence_step(q["x"], q["gate"], state, form="sigmoid", slots=torch.tensor(slots, dtype=torch.int32 if bits == 32 else torch.int64, device="cuda"))
    want, hw = O.LD(host(q["h0"])), np.zeros((9, 70), O.LD)
    a, _ = O.decay("sigmoid", O.LD(host(q["gate"])))
    for i, s in enumerate(slots):
        if 0 <= s < 12:
            want[s] = a[i] * want[s] + O.LD(host(q["x"]))[i]
            hw[i] = want[s]
    near(h, (hw, 3 * O.K * 2.0 ** -24 * (np.abs(hw) + 8)), "float32", "h")            # at most three steps of values below 8
    near(state, (want, 3 * O.K * 2.0 ** -24 * (np.abs(want) + 8)), "float32", "state")
    untouched = [s for s in range(12) if s not in slots]
    assert torch.equal(state[untouched], q["h0"][untouched])


def test_step_on_strided_states_and_empty_batches(sa, torch):
    q = inputs(torch, 18, (4, 33), 4, "decay", "bfloat16")
    pool = torch.zeros(4, 2, 33, device="cuda"); pool[:, 1] = q["h0"]
    dense = q["h0"].clone()
    a = sa.gated_recurrence_step(q["x"], q["gate"], dense, form="decay")
    b = sa.gated_recurrence_step(q["x"], q["gate"], pool[:, 1], form="decay")
    assert torch.equal(a, b) and torch.equal(pool[:, 1], dense) and not pool[:, 0].any()
    assert sa.gated_recurrence_step(q["x"][:0], q["gate"][:0], dense).shape == (0, 33)


def test_captured_replays_and_other_streams(sa, torch):
    """Captured once, replayed with new inputs and eager work between: every replay equals the eager result.  Two calls at once on two streams do not disturb each other."""
    q = inputs(torch, 19, (2, 700, 130), 2, "log", "bfloat16")
    x, g, state = q["x"].clone(), q["gate"].clone(), q["h0"].clone()
    def work():
        sol = sa.recurrence_solve(x, g, q["h0"], form="log", coupled=True)
        return [sol.h, sol.h_final, *sa.recurrence_adjoint(sol, q["dh"], q["dhf"]), sa.gated_recurrence_step(x[:, 0], g[:, 0], state, coupled=True)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = work()
        graphs.append((gr, outs))
    for i in range(4):
        x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)))
        for gr, outs in graphs:
            state.copy_(q["h0"])
            gr.replay()
            got = [t.clone() for t in outs]
            torch.cuda.synchronize()
            state.copy_(q["h0"])
            assert all(torch.equal(a, b) for a, b in zip(got, work())), i
    want = work()[:5]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                sol = sa.recurrence_solve(x, g, q["h0"], form="log", coupled=True)
                results.append([sol.h, sol.h_final, *sa.recurrence_adjoint(sol, q["dh"], q["dhf"])])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in results for a, b in zip(r, want))


def test_training_step_captured_into_a_graph(sa, torch):
    """Forward and backward of torch's autograd in one graph, dense and packed: every replay, with eager work between, leaves the gradients of the adjoint itself."""
    q = inputs(torch, 29, (300, 70), 3, "log", "bfloat16")
    off = torch.tensor([2, 100, 230, 290], dtype=torch.int32, device="cuda")
    leaves = [q[k].clone().requires_grad_() for k in ("x", "gate", "h0")]
    def dense(x, g, h0): return sa.gated_recurrence(x[None], g[None], h0[:1], coupled=True)
    def packed(x, g, h0): return sa.gated_recurrence(x, g, h0, coupled=True, offsets=off)
    def step():
        out = []
        for f in (dense, packed):
            h, last = f(*leaves)
            out += torch.autograd.grad([h, last], leaves, [q["dh"].reshape(h.shape), q["dhf"][:last.shape[0]]])
        return out
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(q["x"].shape, device="cuda", generator=torch.Generator("cuda").manual_seed(i)))
        graph.replay()
        x, g, h0 = (t.detach() for t in leaves)
        a = sa.recurrence_adjoint(sa.recurrence_solve(x[None], g[None], h0[:1], coupled=True), q["dh"][None], q["dhf"][:1])
        b = sa.recurrence_adjoint(sa.recurrence_solve(x, g, h0, coupled=True, offsets=off), q["dh"], q["dhf"])
        torch.cuda.synchronize()
        assert torch.equal(got[0], a[0][0]) and torch.equal(got[1], a[1][0]) and torch.equal(got[2][:1], a[2]) and not got[2][1:].any(), i
        assert all(torch.equal(u, v) for u, v in zip(got[3:], b)), i


def test_offsets_past_32_bits(sa, torch):
    """Rows 2^31 elements apart: the addresses of the second batch row do not fit 32 bits."""
    far = torch.empty(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    q = inputs(torch, 20, (2, 30, 16), 2, "log", "bfloat16")
    view = far.as_strided((2, 30, 16), (2 ** 31, 16, 1))
    view.copy_(q["x"])
    compare(sa, torch, dict(q, x=view), "log", True, "bfloat16")

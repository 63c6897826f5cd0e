"""The adjoint of the gated linear recurrence behind strong decays (`-m gpu`): every gradient carries the decay itself, however small it is next to one."""
import numpy as np
import pytest

import recurrence_oracle as O
from test_gpu_recurrence import host, inputs, near, unit

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def compare(sa, torch, q, form, coupled, dtype, offsets, gate_dtype, with_dh):
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device="cuda")
    sol = sa.recurrence_solve(q["x"], q["gate"], q["h0"], form=form, coupled=coupled, offsets=off)
    dx, dg, d0 = sa.recurrence_adjoint(sol, q["dh"] if with_dh else None, q["dhf"])
    as3 = (lambda t: host(t)[None]) if offsets is not None else host
    dh = as3(q["dh"]) if with_dh else np.zeros_like(as3(q["x"]))
    want = O.whole(as3(q["x"]), as3(q["gate"]), host(q["h0"]), form, coupled, unit(dtype), offsets, dh, host(q["dhf"]))
    # Products of many strong decays leave the range of normal numbers, where the oracle's relative bound ends: a result there is off by up to 2^-149 (half a step, or flushed to zero).  A row
    # forms its cotangent (state) from the one behind (before) it, and a map's product of decays, rounded there, is multiplied by a cotangent (state) of at most 8: at most 9 such errors are
    # added a row, and what was added before is multiplied by the decay; dgate multiplies it by |h - x| <= 16 at most and rounds three times.
    least = 2.0 ** -149
    with np.errstate(all="ignore"):
        a = np.abs(O.decay(form, O.LD(as3(q["gate"])))[0])
    back, ahead = np.zeros_like(a), np.zeros_like(a)
    for t in range(a.shape[1]):
        u = a.shape[1] - 1 - t
        ahead[:, t] = 9 * least + (a[:, t] * ahead[:, t - 1] if t else 0)
        back[:, u] = 9 * least + (a[:, u + 1] * back[:, u + 1] if t else 0)
    for name, extra in (("h", ahead), ("dx", back), ("dgate", 16 * back + 3 * least), ("h_final", ahead.max()), ("dh0", back.max() + least)):
        want[name][1] += extra
    state = "float64" if dtype == "float64" else "float32"
    for name, got, t in (("h", sol.h, dtype), ("h_final", sol.h_final, state), ("dx", dx, dtype), ("dgate", dg, gate_dtype), ("dh0", d0, state)):
        near(got, want[name], t, f"{name} {dtype} {form}")


def strong(torch, q, form, low, high, rows=slice(None)):
    """Gates of the given rows between two log-decays."""
    shape = q["gate"][..., rows, :].shape
    g = low + (high - low) * torch.rand(shape, dtype=torch.float64, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    if form == "decay":
        g = g.exp()
    q["gate"][..., rows, :] = g.to(q["gate"].dtype)


@pytest.mark.parametrize("with_dh", [True, False])
@pytest.mark.parametrize("offsets", [None, [0, 40, 41, 150]], ids=["dense", "packed"])
@pytest.mark.parametrize("coupled", [False, True])
@pytest.mark.parametrize("form", ["decay", "log", "sigmoid"])
@pytest.mark.parametrize("dtype,gate_dtype", [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float32"), ("float32", "float32")])
def test_gradients_of_strong_decays(sa, torch, dtype, gate_dtype, form, coupled, offsets, with_dh):
    """Decays from exp(-30) to one in every row: dgate is a small factor times ordinary ones, not a difference from one."""
    shape = (150, 70) if offsets else (2, 150, 70)
    q = inputs(torch, 31, shape, 3 if offsets else 2, form, dtype, gate_dtype)
    strong(torch, q, form, -30.0, 0.0)
    compare(sa, torch, q, form, coupled, dtype, offsets, gate_dtype, with_dh)


@pytest.mark.parametrize("rows", [2, 9, 17])
@pytest.mark.parametrize("coupled", [False, True])
@pytest.mark.parametrize("form", ["log", "sigmoid"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
def test_several_strong_decays_in_a_row(sa, torch, dtype, form, coupled, rows):
    """Only the last state has a cotangent: what reaches the rows before is the product of the decays, each with its own digits, on both sides of a piece of rows."""
    for low, high in ((-9.0, -8.9), (-14.0, -13.0)):
        q = inputs(torch, 32, (1, 80, 34), 1, form, dtype)
        strong(torch, q, form, low, high, slice(60 - rows, 60))
        q["x"][:, 55:] = 0.0
        compare(sa, torch, q, form, coupled, dtype, None, dtype, False)


@pytest.mark.parametrize("form", ["log", "sigmoid"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_decays_next_to_one_and_above(sa, torch, dtype, form):
    """The other side: what is kept there is 1 - a with its own digits, for log gates above zero too."""
    q = inputs(torch, 33, (1, 150, 70), 1, form, dtype)
    g = 10.0 ** (-4.0 + 3.5 * torch.rand(1, 150, 70, device="cuda", generator=torch.Generator("cuda").manual_seed(4)))
    q["gate"] = ((g - 0.05) if form == "log" else -torch.log(torch.expm1(g))).to(q["gate"].dtype)
    compare(sa, torch, q, form, True, dtype, None, dtype, True)
    compare(sa, torch, q, form, False, dtype, None, dtype, True)

"""Gates far from zero in the gated linear recurrence (`-m gpu`): decays that overflow, that are tiny, and that stand alone because nothing else reaches a row."""
import numpy as np
import pytest

import recurrence_oracle as O
from test_gpu_recurrence import host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("dtype", ["float32", "float64", "bfloat16", "float16"])
def test_an_exponential_that_overflows_is_infinite(sa, torch, dtype):
    """Log gates above the largest exponent: infinite decays, with their sign from the state, not NaN; below, numbers."""
    g = torch.linspace(89.0, 400.0, 1500, dtype=torch.float64).to(getattr(torch, dtype)).cuda()
    if dtype == "float64":
        g = g + 650.0
    h0 = torch.ones(1, 1500, dtype=torch.float64 if dtype == "float64" else torch.float32, device="cuda")
    h0[0, ::2] = -1.0
    x = torch.zeros(1, 1, 1500, dtype=g.dtype, device="cuda")
    last = sa.recurrence_solve(x, g[None, None], h0, form="log").h_final
    assert torch.equal(last, h0 * float("inf"))
    state = h0.clone()
    sa.gated_recurrence_step(x[0], g[None], state, form="log")
    assert torch.equal(state, h0 * float("inf"))
    finite = sa.recurrence_solve(x, torch.full_like(g, 700.0 if dtype == "float64" else 88.0)[None, None], h0, form="log").h_final
    assert torch.isfinite(finite).all()


@pytest.mark.parametrize("form", ["log", "sigmoid"])
@pytest.mark.parametrize("dtype,gate_dtype", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float32")])
def test_strong_decays_keep_their_digits_in_the_states(sa, torch, dtype, gate_dtype, form):
    """One row and nothing added: h_final is the decay times the start and dh0 the decay times the last cotangent, in 32 bits also for 16-bit data, each within the 4 units of a decay and
    the product's half."""
    g = torch.linspace(-80.0, 0.0, 4001, dtype=torch.float64).to(getattr(torch, gate_dtype)).cuda()
    x = torch.zeros(1, 1, 4001, dtype=getattr(torch, dtype), device="cuda")
    h0 = torch.full((1, 4001), 1.5, device="cuda")
    sol = sa.recurrence_solve(x, g[None, None], h0, form=form)
    _, dg, d0 = sa.recurrence_adjoint(sol, None, h0)
    want = 1.5 * O.decay(form, O.LD(host(g)))[0]
    for got in (sol.h_final, d0):
        assert np.abs(host(got)[0] / want - 1).max() <= 4.5 * 2.0 ** -23
    state = h0.clone()
    sa.gated_recurrence_step(x[0], g[None], state, form=form)
    assert np.abs(host(state)[0] / want - 1).max() <= 4.5 * 2.0 ** -23

"""Maps that are handed from tile to tile of the gated linear recurrence (`-m gpu`): what a long axis may not add to a state, and what becomes of states and decays that are not finite or
whose products are not."""
import numpy as np
import pytest

import recurrence_oracle as O
from test_gpu_recurrence import compare, host, inputs, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


# one chain, three and many (groups of 32, 16 and 8 tiles); whole groups and one row more
@pytest.mark.parametrize("channels", [3, 200, 700])
@pytest.mark.parametrize("length", [8192, 65537])
@pytest.mark.parametrize("dtype,form,coupled", [("float32", "log", False), ("float32", "decay", True), ("bfloat16", "log", True), ("float64", "decay", False)])
def test_a_held_state_stays_what_it_is(sa, torch, dtype, form, coupled, length, channels):
    """A decay of exactly one and nothing added: the last state is the first one and the gradient of the first state the last one's, bit for bit, however many tiles lie between."""
    wide = torch.float64 if dtype == "float64" else torch.float32
    gen = torch.Generator("cuda").manual_seed(channels)
    h0, dhf = (torch.randn(1, channels, dtype=wide, device="cuda", generator=gen) for _ in range(2))
    x = torch.zeros(1, length, channels, dtype=getattr(torch, dtype), device="cuda")
    gate = torch.full_like(x, 1.0 if form == "decay" else 0.0)
    sol = sa.recurrence_solve(x, gate, h0, form=form, coupled=coupled)
    dx, dg, d0 = sa.recurrence_adjoint(sol, None, dhf)
    assert torch.equal(sol.h_final, h0) and torch.equal(sol.h[0], h0.to(x.dtype).expand(length, channels))
    assert torch.equal(d0, dhf) and torch.equal(dx[0], (dhf * (0.0 if coupled else 1.0)).to(x.dtype).expand(length, channels))


def test_a_state_that_has_overflowed_stays_infinite(sa, torch):
    """Decays of four from a small state: infinite from the row on where a row-by-row evaluation is, not the largest number times a state below one."""
    x = torch.zeros(1, 1500, 70, device="cuda")
    h0 = torch.full((1, 70), 1e-3, device="cuda")
    sol = sa.recurrence_solve(x, torch.full_like(x, 4.0), h0, form="decay")
    first = int(np.ceil((128 - np.log2(1e-3)) / 2))      # 1e-3 times 4 ** (first + 1) is above 2 ** 128
    rows = torch.isinf(sol.h[0])
    assert rows[first:].all() and not rows[:first - 2].any() and torch.isinf(sol.h_final).all()
    assert not torch.isnan(sol.h).any()


@pytest.mark.parametrize("rate", [0.5, 1.0, 3.0])
def test_an_infinite_state_decays_to_no_number(sa, torch, rate):
    """Infinity times a decay above zero is infinity, also where the decays' product over a tile is below the smallest number; only a decay of zero makes it NaN, and finite states are not
    touched by any of it."""
    x = torch.zeros(1, 3000, 6, device="cuda")
    gate = torch.full_like(x, -rate)
    gate[0, 2000:, 4] = -float("inf")
    h0 = torch.tensor([[float("inf"), -float("inf"), 1.0, 0.0, float("inf"), 1e30]], device="cuda")
    sol = sa.recurrence_solve(x, gate, h0, form="log")
    h = sol.h[0]
    assert (h[:, 0] == float("inf")).all() and (h[:, 1] == -float("inf")).all() and (h[:, 3] == 0).all()
    assert (h[:2000, 4] == float("inf")).all() and torch.isnan(h[2000:, 4]).all()
    assert (h[1000:, [2, 5]] == 0).all()

"""Gates far from zero in the gated linear recurrence (`-m gpu`): decays that overflow, that are tiny, and that stand alone because nothing else reaches a row."""
import pytest

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


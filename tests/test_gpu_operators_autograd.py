"""What torch's autograd sees of the operators (`-m gpu`): tensors that are written in place, hooks on saved tensors, grad mode."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def rows(torch, *shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(len(shape)))


def test_a_state_that_a_step_has_changed_is_an_error_in_the_backward_pass(sa, torch):
    x, pool = rows(torch, 3, 20, 8).requires_grad_(), rows(torch, 3, 8)
    h, _ = sa.gated_recurrence(x, -x.detach().abs(), pool)
    sa.gated_recurrence_step(x[:, 0].detach(), -x[:, 0].detach().abs(), pool)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        h.sum().backward()


def test_a_matrix_that_an_update_has_changed_is_an_error_in_the_backward_pass(sa, torch):
    for changed in ("momentum", "out"):
        w, v = rows(torch, 30, 40).requires_grad_(), rows(torch, 30, 40)
        loss = (w * v).sum()
        sa.orthogonalized_update(w.detach().clone(), **{changed: v})
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


def test_tensors_that_require_grad_are_not_written_in_grad_mode(sa, torch):
    x = rows(torch, 4, 8)
    for leaf in (True, False):
        state, m, out = (rows(torch, 4, 8).requires_grad_() for _ in range(3))
        if not leaf:
            state, m, out = state * 1, m * 1, out * 1
        for name, t, call in (("state", state, lambda: sa.gated_recurrence_step(x, x, state)), ("momentum", m, lambda: sa.orthogonalized_update(x, m)),
                              ("out", out, lambda: sa.orthogonalized_update(x, out=out))):
            before, version = t.detach().clone(), t._version
            with pytest.raises(ValueError, match=f"{name} requires grad"):
                call()
            assert torch.equal(t, before) and t._version == version
            with torch.no_grad():
                call()
            assert t._version > version and not torch.equal(t, before)


def test_inference_tensors_are_written(sa, torch):
    with torch.inference_mode():
        state = rows(torch, 4, 8)
        before = state.clone()
        sa.gated_recurrence_step(before, -before.abs(), state)
        assert not torch.equal(state, before)


def test_the_step_of_a_chain_takes_a_gradient_that_requires_grad(sa, torch):
    fun = sa.WideDeviceFunction.dense_chain("update_chain_autograd", (2, 50, 2), input_power=3)
    dp = torch.randn(fun.np, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    got = fun.orthogonalized_update(dp.clone().requires_grad_())
    assert not got.requires_grad and torch.equal(got, fun.orthogonalized_update(dp))

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


@pytest.mark.parametrize("packed", [False, True])
def test_saved_tensors_that_come_back_in_another_layout(sa, torch, packed):
    """Hooks that move saved tensors to the host and back, or hand out copies with other strides: slices and broadcast gates come back dense, offsets at another address."""
    both = rows(torch, 2, 90, 24).requires_grad_()
    gate = rows(torch, 12).requires_grad_()
    h0 = rows(torch, 4 if packed else 2, 12).requires_grad_()
    off = torch.tensor([0, 20, 20, 61, 85], dtype=torch.int32, device="cuda")
    dh = rows(torch, 2, 90, 12)

    def grads(broadcast):
        x, g = both[..., :12], (-gate.abs()).expand(2, 90, 12) if broadcast else -both[..., 12:].abs()
        kw, d = {}, dh
        if packed:
            x, g, d, kw = x[0], g[0], dh[0], dict(offsets=off.clone())
        h, last = sa.gated_recurrence(x, g, h0, coupled=True, **kw)
        kw.clear()
        torch.full((5,), 1 << 20, dtype=torch.int32, device="cuda")          # what a freed copy of the offsets would hold
        return torch.autograd.grad((h * d).sum() + last.sum(), [both, gate, h0] if broadcast else [both, h0])
    for broadcast in (False, True):
        want = grads(broadcast)
        with torch.autograd.graph.save_on_cpu():
            assert all(torch.equal(a, b) for a, b in zip(grads(broadcast), want))
        for pack, unpack in ((lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)), (lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t)):
            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                assert all(torch.equal(a, b) for a, b in zip(grads(broadcast), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.double() if t.is_floating_point() else t), pytest.raises(ValueError, match="came back as"):
        h, _ = sa.gated_recurrence(rows(torch, 1, 9, 4).requires_grad_(), -rows(torch, 1, 9, 4).abs())
        h.sum().backward()


def test_no_checkpoints_where_no_gradient_can_follow(sa, torch, monkeypatch):
    """Parameters require grad, but not under no_grad: only the forward pass's own bytes are written."""
    from scimlsensitivity_jl_amd import operators
    asked, solve = [], operators.recurrence_solve
    monkeypatch.setattr(operators, "recurrence_solve", lambda *a, **kw: (asked.append(kw["adjoint"]), solve(*a, **kw))[1])
    x = rows(torch, 2, 200, 8).requires_grad_()
    h, _ = operators.gated_recurrence(x, -x.abs())
    with torch.no_grad():
        again, _ = operators.gated_recurrence(x, -x.abs())
    with torch.inference_mode():
        operators.gated_recurrence(x, -x.abs())
    operators.gated_recurrence(x.detach(), -x.detach().abs())
    assert asked == [True, False, False, False] and torch.equal(h, again) and h.requires_grad and not again.requires_grad

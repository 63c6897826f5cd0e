"""Inputs of the gated linear recurrence whose rows overlap or lie in other orders (`-m gpu`): results as for their copies."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("length,channels", [(8, 64), (70, 64), (150, 200), (1, 3)])
def test_sliding_windows(sa, torch, dtype, length, channels):
    """Row t is the signal from t on: neighbouring rows share all but one element, and there may be fewer of them than channels."""
    gen = torch.Generator("cuda").manual_seed(1)
    signal = torch.randn(3 * length + channels, device="cuda", generator=gen).to(getattr(torch, dtype))
    gate = -torch.rand(3, length, channels, device="cuda", generator=gen).to(signal.dtype)
    packed = signal.unfold(0, channels, 1)[:length]
    batched = signal.as_strided((3, length, channels), (1, channels, 1)) if signal.numel() >= length * channels + 2 else signal.as_strided((3, length, channels), (length, 1, 1))
    off = torch.tensor([0, length // 2, length], device="cuda")
    for x, g, kw in ((packed, gate[0], dict(offsets=off)), (packed[None], gate[:1], {}), (batched, gate, {})):
        got, want = (sa.recurrence_solve(v, g, form="log", **kw) for v in (x, x.clone(memory_format=torch.contiguous_format)))
        assert torch.equal(got.h, want.h) and torch.equal(got.h_final, want.h_final)
        dh = torch.randn(x.shape, device="cuda", generator=gen).to(x.dtype)
        assert all(torch.equal(a, b) for a, b in zip(sa.recurrence_adjoint(got, dh), sa.recurrence_adjoint(want, dh)))
        window = sa.recurrence_solve(dh, -x.abs(), form="log", **kw), sa.recurrence_solve(dh, -x.abs().clone(), form="log", **kw)
        assert torch.equal(window[0].h, window[1].h)


def test_results_keep_the_order_of_batch_and_time(sa, torch):
    """[length][batch][channels] in memory: h has the same order, as before."""
    x = torch.randn(40, 3, 16, device="cuda").transpose(0, 1)
    sol = sa.recurrence_solve(x, -x.abs(), form="log")
    assert sol.h.stride() == x.stride() and torch.equal(sol.h, sa.recurrence_solve(x.contiguous(), -x.abs().contiguous(), form="log").h)


def test_views_whose_sign_is_yet_to_be_turned(sa, torch):
    """The imaginary part of a conjugate is a view of the other sign: one channel, where its stride does not ask for a copy, and several."""
    gen = torch.Generator("cuda").manual_seed(5)
    for channels in (1, 4):
        parts = [torch.complex(*torch.randn(2, 1, 30, channels, device="cuda", generator=gen)).conj().imag for _ in range(3)]
        starts = [torch.complex(*torch.randn(2, 1, channels, device="cuda", generator=gen)).conj().imag for _ in range(2)]
        assert all(t.is_neg() for t in parts + starts)
        results = []
        for turn in (lambda t: t, lambda t: t.resolve_neg().clone()):
            x, g, dh, h0, last = (turn(t) for t in parts + starts)
            sol = sa.recurrence_solve(x, g, h0, form="sigmoid", coupled=True)
            results.append([sol.h, sol.h_final, *sa.recurrence_adjoint(sol, dh, last), sa.gated_recurrence_step(x[0], g[0], torch.ones(30, channels, device="cuda"), form="sigmoid"),
                            sa.orthogonalized_update(x), sa.orthogonalized_update(x.transpose(1, 2))])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        # (with several channels these views have strides of two, for which they are refused before their sign)
        with pytest.raises(ValueError, match="sign is yet" if channels == 1 else "neighbouring channels"):
            sa.gated_recurrence_step(parts[0][0], parts[1][0], parts[2][0])
        with pytest.raises(ValueError, match="sign is yet" if channels == 1 else "row-major"):
            sa.orthogonalized_update(parts[0].resolve_neg(), out=parts[1])

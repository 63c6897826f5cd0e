"""The operators on streams other than the one a solution was made on (`-m gpu`)."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def busy(torch, n=40):
    """Some milliseconds of work on the current stream."""
    a = torch.ones(4096, 4096, device="cuda")
    for _ in range(n):
        a = a @ a * 1e-4
    return a


@pytest.mark.parametrize("packed", [False, True])
def test_a_solution_dropped_while_its_adjoint_waits_on_another_stream(sa, torch, packed):
    """What the solution holds of its own (checkpoints, copies of inputs) is not handed out again before the other stream has read it."""
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(700, 64, 4, device="cuda", generator=gen).transpose(0, 2)         # channels apart: copied
    gate, dh = -torch.rand(4, 64, 700, device="cuda", generator=gen), torch.randn(4, 64, 700, device="cuda", generator=gen)
    kw = {}
    if packed:
        x, gate, dh = x[:, 0], gate[:, 0], dh[:, 0]
        kw = dict(offsets=torch.tensor([0, 3, 4], device="cuda").repeat_interleave(2)[::2])
    want = sa.recurrence_adjoint(sa.recurrence_solve(x, gate, **kw), dh)
    side = torch.cuda.Stream()
    busy(torch)
    torch.cuda.synchronize()
    for _ in range(3):
        sol = sa.recurrence_solve(x, gate, **kw)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            busy(torch)
            got = sa.recurrence_adjoint(sol, dh)
        sizes = [t.numel() * t.element_size() for t in (sol._checkpoints, sol.x, sol.gate)]
        del sol
        over = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
        torch.cuda.current_stream().synchronize()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del over


@pytest.mark.parametrize("packed", [False, True])
def test_an_adjoint_captured_of_an_eager_solution(sa, torch, packed):
    """The solution belongs to the default stream, its adjoint to a captured graph: every replay gives the eager gradients, also after new cotangents, with eager work between."""
    gen = torch.Generator("cuda").manual_seed(6)
    x, gate, dh = (torch.randn(2, 300, 40, device="cuda", generator=gen) for _ in range(3))
    kw = {}
    if packed:
        x, gate, dh, kw = x[0], gate[0], dh[0], dict(offsets=torch.tensor([0, 100, 290], device="cuda"))
    sol = sa.recurrence_solve(x, gate, form="sigmoid", **kw)
    sa.recurrence_adjoint(sol, dh)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sa.recurrence_adjoint(sol, dh)
    for i in range(4):
        dh.copy_(torch.randn(dh.shape, device="cuda", generator=gen))
        graph.replay()
        want = sa.recurrence_adjoint(sol, dh)
        busy(torch, 2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i

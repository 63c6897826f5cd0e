"""Which layouts the orthogonalised update takes for what it writes in place: none where two elements share a place (the check against all places, without a device, and the refusals
on one)."""
import itertools

import pytest
import torch

from scimlsensitivity_jl_amd import operators


def test_disjoint_against_all_places():
    seen = set()
    for batch, rows, cols in itertools.product((1, 2, 3), (1, 2, 4), (1, 2, 3)):
        for sb, sr, turned in itertools.product(range(14), range(8), (False, True)):
            store = torch.empty(200)
            t = store.as_strided((batch, rows, cols), (sb, sr, 1))
            places = {b * sb + r * sr + c for b in range(batch) for r in range(rows) for c in range(cols)}
            t = t.transpose(-1, -2) if turned else t
            want = len(places) == batch * rows * cols
            assert operators._disjoint(t) == want, (t.shape, t.stride())
            seen.add(want)
    assert seen == {True, False}
    assert operators._disjoint(torch.empty(0, 3, 4)) and operators._disjoint(torch.empty(6, 5, 7)[:, 1:4, 2:6])


@pytest.mark.gpu
def test_overlapping_rows_are_refused(sa):
    z = lambda *s: torch.zeros(*s, device="cuda")                              # noqa: E731
    g = z(2, 5, 4)
    for bad in (z(40).as_strided((2, 5, 4), (20, 1, 1)), z(40).as_strided((2, 5, 4), (4, 4, 1)), z(60).unfold(0, 4, 2)[:10].view(2, 5, 4)):
        for kw in (dict(momentum=bad), dict(out=bad)):
            with pytest.raises(ValueError, match="not overlap"):
                sa.orthogonalized_update(g, **kw)
    with pytest.raises(ValueError, match="both be row-major"):                 # neither columns nor rows next to each other: refused for that
        sa.orthogonalized_update(g, out=z(2, 5, 8)[..., ::2])
    heads = z(5, 2, 4).transpose(0, 1)                                         # matrices side by side
    assert sa.orthogonalized_update(g, out=heads) is heads and sa.orthogonalized_update(z(2, 4, 5).transpose(1, 2), z(2, 4, 5).transpose(1, 2)).shape == g.shape


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 5, 4), (200, 150)])
def test_momentum_in_the_place_of_another_argument_is_refused(sa, shape):
    g = torch.randn(*shape, device="cuda")
    m = torch.randn(*shape, device="cuda")
    before = g.clone(), m.clone()
    for call in (lambda: sa.orthogonalized_update(g, g), lambda: sa.orthogonalized_update(g, m, out=m), lambda: sa.orthogonalized_update(g.transpose(-1, -2), g.transpose(-1, -2))):
        with pytest.raises(ValueError, match="momentum is written in place"):
            call()
    assert torch.equal(g, before[0]) and torch.equal(m, before[1])
    want = sa.orthogonalized_update(g.clone(), m.clone())
    assert torch.equal(sa.orthogonalized_update(g, m, out=g), want) and torch.equal(g, want)

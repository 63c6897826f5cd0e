"""WideDeviceFunction.orthogonalized_update (`-m gpu`): how a gradient may lie in memory, and which coefficients are taken."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def chain(sa):
    return sa.WideDeviceFunction.dense_chain("update_chain_layouts", (2, 50, 2), input_power=3)


def gradient(chain):
    import torch
    return torch.randn(chain.np, device="cuda", generator=torch.Generator("cuda").manual_seed(2))


def test_a_gradient_that_is_a_column_of_a_batch(chain):
    """dp of one trajectory among others: a column of [np, N], in 32 and 64 bits."""
    import torch
    dp = gradient(chain)
    many = torch.stack([dp, 2 * dp, -dp], dim=1)
    for t in (torch.float32, torch.float64):
        got = chain.orthogonalized_update(many[:, 0].to(t) if t == torch.float32 else many.double()[:, 0])
        assert got.dtype == t and torch.equal(got.float(), chain.orthogonalized_update(dp))


def test_coefficients_in_arrays(sa, chain):
    """Lists, tuples and numpy arrays of any float type, once for all steps or for each."""
    dp = gradient(chain)
    import torch
    one = (2.0, -1.5, 0.5)
    want = chain.orthogonalized_update(dp, steps=3, coefficients=one)
    g = dp[:100].view(2, 50)
    direct = sa.orthogonalized_update(g, steps=3, coefficients=one)
    for c in (list(one), np.array(one), np.array(one, np.float32), [one] * 3, np.array([one] * 3, np.float32), [np.array(one)] * 3):
        assert torch.equal(chain.orthogonalized_update(dp, steps=3, coefficients=c), want) and torch.equal(sa.orthogonalized_update(g, steps=3, coefficients=c), direct)
    for bad in ((), (1.0, 2.0), [one] * 2, np.zeros(4)):
        with pytest.raises(ValueError, match="three numbers"):
            sa.orthogonalized_update(g, steps=3, coefficients=bad)

"""The orthogonalised update on the device (`-m gpu`) against its definition in 64 bits (tests/orthogonal_oracle.py).

Factors are rounded to two F16 terms (22 bits; with the F32 accumulation 2^-20 a factor is allowed), or to one (2^-11) for bfloat16 with both sides of at least 256; the output adds
half a step of its type."""
import numpy as np
import pytest

import orthogonal_oracle as O

pytestmark = pytest.mark.gpu
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def gradient(torch, seed, shape, dtype, factor=1e-3):
    rng = np.random.default_rng(seed)
    k = max(1, min(shape[-2:]) // 8)
    g = rng.standard_normal((*shape[:-1], k)) @ rng.standard_normal((*shape[:-2], k, shape[-1])) / k ** 0.5 + 0.3 * rng.standard_normal(shape)
    return torch.tensor(g * factor).to(getattr(torch, dtype)).cuda()


def host(t):
    return t.detach().double().cpu().numpy()


def near(got, u, dtype, one_term=False, **kw):
    """got against the iteration from u."""
    want = O.iterate(u, kw.get("steps", 5), kw.get("coefficients", O.C), kw.get("scale", 1.0))
    norm, most = O.allowance(u, 2.0 ** -11 if one_term else 2.0 ** -20, **kw)
    d = host(got) - want
    half = HALF[dtype]
    assert np.linalg.norm(d) <= norm + half * np.linalg.norm(want), (np.linalg.norm(d), norm, np.linalg.norm(want))
    assert np.abs(d).max() <= most + half * np.abs(want).max(), (np.abs(d).max(), most)


# sides of one, below, at and above the padding of 128, squares, wide and tall ones
SHAPES = [(1, 1), (1, 7), (9, 1), (2, 2), (50, 2), (2, 50), (16, 33), (64, 64), (127, 128), (128, 128), (129, 127), (130, 300), (333, 500), (500, 333), (257, 1030)]


@pytest.mark.parametrize("shape", SHAPES, ids=[f"{a}x{b}" for a, b in SHAPES])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_shapes_and_types(sa, torch, shape, dtype):
    g = gradient(torch, 1, shape, dtype)
    before = g.clone()
    got = sa.orthogonalized_update(g)
    assert got.dtype == g.dtype and got.shape == g.shape and torch.equal(g, before)
    near(got, host(g), dtype, one_term=dtype == "bfloat16" and min(shape) >= 256)


# few rows and long ones: X X' is summed in parts
@pytest.mark.parametrize("shape,dtype", [((200, 2900), "float32"), ((2900, 200), "bfloat16"), ((256, 4200), "bfloat16"), ((2, 300, 5000), "float16"), ((9000, 130), "float32"),
                                         ((3, 16400, 256), "bfloat16")])
def test_long_rows(sa, torch, shape, dtype):
    g = gradient(torch, 3, shape, dtype)
    got, again = sa.orthogonalized_update(g), sa.orthogonalized_update(g)
    assert torch.equal(got, again)
    for a, b in zip(got.reshape(-1, *shape[-2:]), g.reshape(-1, *shape[-2:])):
        near(a, host(b), dtype, one_term=dtype == "bfloat16" and min(shape[-2:]) >= 256)


@pytest.mark.parametrize("shape", [(256, 256), (700, 300), (384, 1500), (1024, 1024)])
def test_one_term_products(sa, torch, shape):
    g = gradient(torch, 2, shape, "bfloat16")
    got = sa.orthogonalized_update(g)
    near(got, host(g), "bfloat16", one_term=True)
    want = O.iterate(host(g), 5, O.C, 1.0)
    # what the choice of one term promises: together with the output's rounding (rms 0.41 of half a step, 1.65e-3 of the norm) at most 1.5 times the rounding alone
    assert np.linalg.norm(host(got) - want) < 1.5 * 1.66e-3 * np.linalg.norm(want)


@pytest.mark.parametrize("nesterov", [True, False])
def test_momentum(sa, torch, nesterov):
    g = gradient(torch, 3, (3, 70, 40), "float32")
    m = gradient(torch, 4, (3, 70, 40), "float32")
    before = host(m)
    got = sa.orthogonalized_update(g, m, beta=0.9, nesterov=nesterov)
    for b in range(3):
        _, want_m, u = O.update(host(g)[b], before[b], beta=0.9, nesterov=nesterov)
        size = np.abs(0.9 * before[b]) + np.abs(host(g)[b])
        assert np.all(np.abs(host(m)[b] - want_m) <= 3 * 2.0 ** -24 * size)
        near(got[b], u, "float32")
    second = sa.orthogonalized_update(g, m, beta=0.9, nesterov=nesterov)
    assert not torch.equal(second, got)


def test_batches_heads_and_strides(sa, torch):
    g = gradient(torch, 5, (2, 3, 48, 80), "bfloat16")
    got = sa.orthogonalized_update(g)
    for i in range(2):
        for j in range(3):
            one = sa.orthogonalized_update(g[i, j].contiguous())
            assert torch.equal(one, got[i, j])
    wide = torch.zeros(2, 3, 48, 200, dtype=torch.bfloat16, device="cuda")
    wide[..., 60:140] = g
    assert torch.equal(sa.orthogonalized_update(wide[..., 60:140]), got)
    assert torch.equal(sa.orthogonalized_update(g.transpose(0, 1)), got.transpose(0, 1))
    out = torch.full((2, 3, 50, 90), 7.0, dtype=torch.bfloat16, device="cuda")
    back = sa.orthogonalized_update(g[:, 0], out=out[:, 0, 1:49, 5:85])
    assert back.data_ptr() == out[:, 0, 1:49, 5:85].data_ptr() and torch.equal(back, got[:, 0])
    rest = out.clone(); rest[:, 0, 1:49, 5:85] = 7.0
    assert (rest == 7.0).all()


def test_transposes_and_in_place(sa, torch):
    g = gradient(torch, 6, (90, 60), "float32")
    got = sa.orthogonalized_update(g)
    flipped = sa.orthogonalized_update(g.t())                          # column-major input, column-major result
    assert torch.equal(flipped, got.t()) and flipped.stride() == (1, 60)
    m = gradient(torch, 7, (90, 60), "float32")
    mt = m.clone().t()
    a = sa.orthogonalized_update(g, m)
    b = sa.orthogonalized_update(g.t(), mt)
    assert torch.equal(a, b.t()) and torch.equal(m, mt.t())
    same = g.clone()
    assert sa.orthogonalized_update(same, out=same) is same and torch.equal(same, got)


def test_steps_coefficients_and_scale(sa, torch):
    g = gradient(torch, 8, (40, 60), "float32")
    for steps, co in ((1, O.C), (2, O.C), (3, (2.0, -1.5, 0.5))):
        got = sa.orthogonalized_update(g, steps=steps, coefficients=co, scale=0.25)
        near(got, host(g), "float32", steps=steps, coefficients=co, scale=0.25)
    # these let singular values grow past what the factors' type holds (in 64 bits: to 1e4): refused
    with pytest.raises(sa.HipadjError, match="can grow"):
        sa.orthogonalized_update(g, steps=4, coefficients=[(4.0, -6.0, 3.0), (3.4445, -4.775, 2.0315), (2.0, -1.5, 0.5), (1.875, -1.25, 0.375)])
    # 1.875, -1.25, 0.375 converges: the result is the orthogonal factor
    u, _, vt = np.linalg.svd(host(g), full_matrices=False)
    got = sa.orthogonalized_update(g, steps=14, coefficients=[O.C] * 4 + [(1.875, -1.25, 0.375)] * 10)
    assert np.abs(host(got) - u @ vt).max() < 1e-5


@pytest.mark.parametrize("factor", [1e-30, 1e-12, 1e12, 1e30])
def test_size_of_the_gradient_does_not_matter(sa, torch, factor):
    """Except through the 1e-7 next to the norm: a gradient of 1e-12 is far below it."""
    g = gradient(torch, 9, (64, 96), "float32", factor)
    near(sa.orthogonalized_update(g), host(g), "float32")


def test_zero_one_direction_and_not_finite(sa, torch):
    assert not sa.orthogonalized_update(torch.zeros(30, 20, device="cuda")).any()
    g = torch.zeros(300, 260, device="cuda", dtype=torch.bfloat16)
    g[17, 200] = 3.0                                                   # one entry: rank one, the largest entry an X can have
    got = host(sa.orthogonalized_update(g))
    x = 3.0 / (3.0 + 1e-7)
    for _ in range(5):
        x = O.C[0] * x + O.C[1] * x ** 3 + O.C[2] * x ** 5
    # one entry: each of the 3 products and roundings of a step within 2^-11, and a gain of at most 1.6 a step near one
    assert abs(got[17, 200] - x) < 2.0 ** -8 * x + 5 * 1.6 ** 4 * 3 * 2.0 ** -11 * 4.8 and np.count_nonzero(got) == 1
    for bad in (float("nan"), float("inf")):
        g = gradient(torch, 10, (2, 40, 30), "float32")
        g[0, 3, 5] = bad
        got = sa.orthogonalized_update(g)
        assert torch.isnan(got[0]).all() and torch.equal(got[1], sa.orthogonalized_update(g[1:].clone())[0])


def test_empty(sa, torch):
    for shape in ((0, 5, 4), (3, 0, 4), (3, 5, 0)):
        assert sa.orthogonalized_update(torch.empty(shape, device="cuda")).shape == shape


def test_same_result_every_time_captured_and_on_other_streams(sa, torch):
    g = gradient(torch, 11, (300, 700), "bfloat16"); m0 = gradient(torch, 12, (300, 700), "float32"); small = gradient(torch, 13, (2, 60, 50), "float32")
    m = m0.clone()
    work = lambda: [sa.orthogonalized_update(g, m), sa.orthogonalized_update(small)]      # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = work()
        graphs.append((gr, outs))
    for i in range(4):
        g.copy_(gradient(torch, 20 + i, (300, 700), "bfloat16"))
        for gr, outs in graphs:
            m.copy_(m0)
            gr.replay()
            got, mom = [t.clone() for t in outs], m.clone()
            torch.cuda.synchronize()
            m.copy_(m0)
            assert all(torch.equal(a, b) for a, b in zip(got, work())) and torch.equal(mom, m)
    want = sa.orthogonalized_update(small)
    streams, results = [torch.cuda.Stream() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(sa.orthogonalized_update(small))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)

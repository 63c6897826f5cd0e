"""The operators without a handle (recurrence, orthogonalised update) where there is no device: what the C entry points refuse before they touch one, the sizes they report,
that there is no CPU fallback, and the oracles of the device tests against closed forms."""
import ctypes as C

import numpy as np
import pytest

import orthogonal_oracle as OO
import recurrence_oracle as RO


@pytest.fixture()
def lib(sa):
    from scimlsensitivity_jl_amd import _lib
    return _lib, _lib.load()


def recurrence(_lib, **kw):
    r = _lib.HipadjRecurrence()
    r.struct_size, r.dtype, r.gate_dtype, r.gate, r.batch, r.length, r.channels = C.sizeof(r), 1, 1, 1, 2, 300, 70
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def orthogonal(_lib, coefficients=OO.C, **kw):
    o = _lib.HipadjOrthogonal()
    o.struct_size, o.dtype, o.steps, o.batch, o.rows, o.cols, o.beta, o.scale = C.sizeof(o), 1, 5, 1, 40, 60, 0.9, 1.0
    o._co = (C.c_double * 15)(*(list(coefficients) * 5))
    o.coefficients = C.cast(o._co, C.POINTER(C.c_double))
    for k, v in kw.items():
        setattr(o, k, v)
    return o


@pytest.mark.parametrize("kw,status,text", [
    (dict(struct_size=8), -1, "struct_size"), (dict(dtype=2, gate_dtype=3), -6, "gate of x's type"), (dict(dtype=0, gate_dtype=1), -6, "gate of x's type"), (dict(dtype=9), -6, "F64, F32"),
    (dict(gate=3), -1, "hipadj_gate"), (dict(length=-1), -1, "negative"), (dict(nseq=2), -1, "batch = 1"), (dict(nseq=2, batch=1), -1, "offsets"),
    (dict(nseq=2, batch=1, offsets=64, offsets_bits=16), -1, "32 or 64"), (dict(batch=1 << 30, length=1 << 20), -6, "tiles")])
def test_recurrence_refusals(lib, kw, status, text):
    _lib, L = lib
    r = recurrence(_lib, **kw)
    assert L.hipadj_recurrence_sizes(C.byref(r), None, None) == status and text in L.hipadj_last_error(None).decode()
    assert L.hipadj_recurrence_forward_dev(C.byref(r), *[256] * 9) == status
    assert L.hipadj_recurrence_adjoint_dev(C.byref(r), *[256] * 12) == status


def test_recurrence_arguments_and_sizes(lib):
    _lib, L = lib
    r = recurrence(_lib)
    ck, ws = C.c_int64(), C.c_int64()
    assert L.hipadj_recurrence_sizes(C.byref(r), C.byref(ck), C.byref(ws)) == 0
    assert ck.value == 2 * 5 * 70 * 4 and ws.value > 0                       # a checkpoint every 64 rows
    short = recurrence(_lib, length=64)
    assert L.hipadj_recurrence_sizes(C.byref(short), None, C.byref(ws)) == 0 and ws.value == 0
    assert L.hipadj_recurrence_forward_dev(C.byref(r), None, 256, None, 256, 256, None, 256, ws.value, None) == -1
    assert L.hipadj_recurrence_adjoint_dev(C.byref(r), 256, 256, None, None, None, None, 256, 256, 256, 256, 0, None) == -1 and b"checkpoints" in L.hipadj_last_error(None)
    assert L.hipadj_recurrence_forward_dev(C.byref(recurrence(_lib, batch=0)), *[None] * 7, 0, None) == 0
    step = lambda **k: L.hipadj_recurrence_step_dev(*{**dict(device=0, dtype=1, gate_dtype=1, gate=1, coupled=0, batch=2, channels=4, x=256, xs=4, g=256, gs=4, st=256, ss=4, n=2,     # noqa: E731
                                                              slots=None, bits=32, h=256, hs=4, stream=None), **k}.values())
    assert step(n=1) == -1 and step(gate=5) == -1 and step(dtype=2, gate_dtype=0) == -6 and step(x=None) == -1 and step(slots=256, bits=8) == -1 and step(batch=-1) == -1
    assert step(batch=0) == 0


def test_recurrence_launch_limits(lib):
    """A launch has 2^32 - 1 threads: more tiles of 512 or more step rows of 256 are refused by name, the largest that fit get as far as the device."""
    _lib, L = lib
    most = (2 ** 32 - 1) // 512
    r = lambda b: C.byref(recurrence(_lib, batch=b, length=1, channels=64, device=1 << 20))                                                     # noqa: E731
    for b, refused in ((most + 1, True), (most, False)):
        for status in (L.hipadj_recurrence_forward_dev(r(b), *[256] * 7, 0, None), L.hipadj_recurrence_adjoint_dev(r(b), *[256] * 10, 0, None)):
            assert (status == -6) == refused and status != 0 and (b"at a time" in L.hipadj_last_error(None)) == refused
    most = (2 ** 32 - 1) // 256
    for b, refused in ((most + 1, True), (most, False), (most // 2 + 1, False)):
        status = L.hipadj_recurrence_step_dev(1 << 20, 1, 1, 1, 0, b, 4, 256, 4, 256, 4, 256, 4, b, None, 32, 256, 4, None)
        assert (status == -6) == refused and status != 0 and (b"at most" in L.hipadj_last_error(None)) == refused


@pytest.mark.parametrize("kw,status,text", [
    (dict(struct_size=4), -1, "struct_size"), (dict(dtype=0), -6, "F32, BF16 or F16"), (dict(rows=-1), -1, "negative"), (dict(steps=0), -1, "steps"), (dict(steps=65), -1, "steps"),
    (dict(beta=float("nan")), -1, "finite"), (dict(rows=70000, cols=70000), -6, "at most"), (dict(batch=65536), -6, "at most"), (dict(coefficients=(33.0, 0.0, 0.0)), -1, "within"),
    (dict(coefficients=(float("nan"), 0.0, 0.0)), -1, "within"), (dict(coefficients=(4.0, 0.0, 0.0)), -6, "grow"), (dict(coefficients=(2.0, -1.5, 0.5), steps=5), 0, "")])
def test_orthogonal_refusals(lib, kw, status, text):
    _lib, L = lib
    o = orthogonal(_lib, **kw)
    ws = C.c_int64()
    assert L.hipadj_orthogonalized_update_size(C.byref(o), C.byref(ws)) == status
    if status:
        assert text in L.hipadj_last_error(None).decode()
        assert L.hipadj_orthogonalized_update_dev(C.byref(o), *[256] * 4, 0, None) == status


def test_orthogonal_arguments(lib):
    _lib, L = lib
    o = orthogonal(_lib)
    assert L.hipadj_orthogonalized_update_dev(C.byref(o), None, None, 256, 256, 0, None) == -1
    large = orthogonal(_lib, rows=400)
    assert L.hipadj_orthogonalized_update_dev(C.byref(large), 256, None, 256, 128, 1 << 40, None) == -1 and b"aligned" in L.hipadj_last_error(None)
    assert L.hipadj_orthogonalized_update_dev(C.byref(large), 256, None, 256, 256, 1000, None) == -1
    assert L.hipadj_orthogonalized_update_dev(C.byref(orthogonal(_lib, rows=0)), None, None, None, None, 0, None) == 0


def test_no_cpu_fallback(sa):
    import torch
    x = torch.zeros(2, 5, 4)
    with pytest.raises(ValueError, match="no CPU fallback"):
        sa.recurrence_solve(x, x)
    with pytest.raises(ValueError, match="no CPU fallback"):
        sa.gated_recurrence(x, x)
    with pytest.raises(ValueError, match="no CPU fallback"):
        sa.gated_recurrence_step(x[0], x[0], x[0])
    with pytest.raises(ValueError, match="no CPU fallback"):
        sa.orthogonalized_update(x)
    with pytest.raises(ValueError, match=r"\[rows\]\[channels\]"):
        sa.recurrence_solve(x, x, offsets=torch.tensor([0, 5]))


def test_recurrence_oracle_against_closed_forms():
    """Constant decay and input: h_t = a^t h_0 + b (1 - a^t) / (1 - a); its gradients by differences of the oracle itself."""
    L, a, b, h0 = 40, 0.8, 0.3, 2.0
    one = np.ones((L, 1))
    (h, _), _ = RO.solve(b * one, a * one, np.array([h0]), "decay", False, 0)
    t = np.arange(1, L + 1)
    assert np.allclose(np.float64(h[:, 0]), a ** t * h0 + b * (1 - a ** t) / (1 - a), rtol=1e-14)
    for form in ("decay", "log", "sigmoid"):
        g = {"decay": a, "log": np.log(a), "sigmoid": np.log(a / (1 - a))}[form]
        (q, _), _ = RO.solve(b * one, g * one, np.array([h0]), form, True, 0)
        assert np.allclose(np.float64(q[:, 0]), a ** t * h0 + b * (1 - a ** t), rtol=1e-13)       # coupled: towards x
    rng = np.random.default_rng(0)
    x, g, h0 = rng.standard_normal((12, 3)), -np.exp(rng.standard_normal((12, 3))), rng.standard_normal(3)
    dh, dhf = rng.standard_normal((12, 3)), rng.standard_normal(3)
    for form, coupled in (("log", True), ("log", False), ("sigmoid", True), ("decay", True)):
        def loss(x, g, h0):
            (h, _), (hf, _) = RO.solve(x, g, h0, form, coupled, 0)
            return np.sum(h * dh) + np.sum(hf * dhf)
        grads = RO.adjoint(x, g, h0, form, coupled, 0, dh, dhf)
        for k in range(3):
            at = [x, g, h0]
            d = rng.standard_normal(at[k].shape)
            e = RO.LD(1e-6)                                     # 80 bits: truncation 1e-12, cancellation 1e-13
            up, down = list(at), list(at)
            up[k], down[k] = at[k] + e * d, at[k] - e * d
            assert abs((loss(*up) - loss(*down)) / (2 * e) - np.sum(grads[k][0] * d)) < 1e-8 * max(1, abs(loss(x, g, h0)))


def test_orthogonal_oracle_against_singular_values():
    """The iteration acts on the singular values alone."""
    rng = np.random.default_rng(1)
    for shape in ((6, 9), (9, 6), (5, 5), (1, 4)):
        g = rng.standard_normal(shape)
        u, s, vt = np.linalg.svd(g, full_matrices=False)
        s = s / (np.linalg.norm(g) + 1e-7)
        for _ in range(5):
            s = OO.C[0] * s + OO.C[1] * s ** 3 + OO.C[2] * s ** 5
        assert np.allclose(OO.iterate(g, 5, OO.C, 2.0), 2 * (u * s) @ vt, atol=1e-12)
        m = rng.standard_normal(shape)
        out, new, v = OO.update(g, m, beta=0.5)
        assert np.allclose(new, 0.5 * m + g) and np.allclose(v, g + 0.5 * new) and np.allclose(out, OO.iterate(v, 5, OO.C, 1.0))

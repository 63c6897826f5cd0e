"""What the recurrence reads and writes (`-m gpu`), through its C entry points on slices of larger buffers: outputs are surrounded by a sentinel that has to stay, inputs by NaN that may not be
read into a result.  Offsets that do not ascend, or lie outside the rows, give unspecified results, and these come from inside too."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

GUARD, SENTINEL = 3, 1234.5


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def guarded(torch, shape, dtype, fill, inside=None):
    """A slice of a larger buffer: GUARD rows before, behind and between batch rows, 2 channels on both sides."""
    big = torch.full((*shape[:-2], shape[-2] + 2 * GUARD, shape[-1] + 4), fill, dtype=dtype, device="cuda")
    view = big[..., GUARD:GUARD + shape[-2], 2:2 + shape[-1]]
    if inside is not None:
        view.copy_(inside)
    return big, view


def framed(torch, shape, dtype, fill, inside=None):
    """As above for what has no strides: GUARD rows before and behind."""
    big = torch.full((shape[0] + 2 * GUARD, shape[1]), fill, dtype=dtype, device="cuda")
    if inside is not None:
        big[GUARD:-GUARD].copy_(inside)
    return big, big[GUARD:GUARD + shape[0]]


BAD = [[5, 3, 9, 1], [0, 100, 50, 20], [7, 7, 300, 2], [-5, 4, -1, 8], [20, 0, 0, 20], [2 ** 31 - 1] * 4, [-2 ** 31, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [300, 299, 0, -1]]


@pytest.mark.parametrize("length,channels", [(20, 66), (300, 34), (1, 5)])
@pytest.mark.parametrize("offsets", [[0, 0, 10, 20]] + BAD, ids=[str(i) for i in range(len(BAD) + 1)])
@pytest.mark.parametrize("dtype,bits", [("float32", 32), ("bfloat16", 64)])
def test_nothing_outside_is_read_or_written(sa, torch, dtype, bits, offsets, length, channels):
    from scimlsensitivity_jl_amd import _lib
    L, t, f32, nseq = _lib.load(), getattr(torch, dtype), torch.float32, 3
    gen = torch.Generator("cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)             # noqa: E731
    nan = float("nan")
    rows = (length, channels)
    ins = {k: guarded(torch, rows, t, nan, v) for k, v in dict(x=rnd(*rows), gate=-rnd(*rows).abs(), dh=rnd(*rows)).items()}
    outs = {k: guarded(torch, rows, t, SENTINEL) for k in ("h", "dx", "dgate")}
    state_in = {k: framed(torch, (nseq, channels), f32, nan, rnd(nseq, channels)) for k in ("h0", "dh_final")}
    state_out = {k: framed(torch, (nseq, channels), f32, SENTINEL) for k in ("h_final", "dh0")}
    off = torch.tensor(offsets, dtype=torch.int64 if bits == 64 else torch.int32, device="cuda")
    around = torch.full((off.numel() + 2 * 8,), -7, dtype=off.dtype, device="cuda")
    around[8:-8] = off
    r = _lib.HipadjRecurrence()
    r.struct_size, r.device, r.dtype, r.gate_dtype, r.gate, r.coupled = C.sizeof(r), 0, {"float32": 1, "bfloat16": 2}[dtype], {"float32": 1, "bfloat16": 2}[dtype], 1, 1
    r.batch, r.length, r.channels, r.nseq, r.offsets, r.offsets_bits = 1, length, channels, nseq, around[8:].data_ptr(), bits
    for name, (_, v) in {**ins, **outs}.items():
        getattr(r, name + "_stride")[:] = (0, v.stride(0))
    ck, ws = C.c_int64(), C.c_int64()
    assert L.hipadj_recurrence_sizes(C.byref(r), C.byref(ck), C.byref(ws)) == 0
    checkpoints, ckpt = framed(torch, (1, ck.value // 4), f32, SENTINEL)
    work = torch.full((ws.value // 8 + 16,), -1, dtype=torch.int64, device="cuda")
    p = lambda d, k: d[k][1].data_ptr()                                        # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    assert L.hipadj_recurrence_forward_dev(C.byref(r), p(ins, "x"), p(ins, "gate"), p(state_in, "h0"), p(outs, "h"), p(state_out, "h_final"), ckpt.data_ptr(), work[8:].data_ptr(), ws.value,
                                           stream) == 0
    assert L.hipadj_recurrence_adjoint_dev(C.byref(r), p(ins, "x"), p(ins, "gate"), p(state_in, "h0"), ckpt.data_ptr(), p(ins, "dh"), p(state_in, "dh_final"), p(outs, "dx"), p(outs, "dgate"),
                                           p(state_out, "dh0"), work[8:].data_ptr(), ws.value, stream) == 0
    torch.cuda.synchronize()
    for name, (big, view) in outs.items():
        assert torch.isfinite(view).all(), name
        view.fill_(SENTINEL)
        assert (big == big.flatten()[0]).all() and float(big.flatten()[0]) == float(torch.tensor(SENTINEL).to(t)), name
    for name, (big, view) in state_out.items():
        assert torch.isfinite(view).all(), name                               # (rows of no sequence keep the sentinel)
        assert (big[:GUARD] == SENTINEL).all() and (big[-GUARD:] == SENTINEL).all(), name
    assert torch.isfinite(ckpt).all() and (checkpoints[:GUARD] == SENTINEL).all() and (checkpoints[-GUARD:] == SENTINEL).all()
    assert (work[:8] == -1).all() and (work[8 + ws.value // 8:] == -1).all() and (around[:8] == -7).all() and (around[-8:] == -7).all()


@pytest.mark.parametrize("batch,length,channels", [(2, 130, 66), (3, 1, 1), (1, 65, 130)])
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_dense_rows_too(sa, torch, dtype, batch, length, channels):
    """Dense: inputs as slices through the package's own call, where only they can have neighbours."""
    t = getattr(torch, dtype)
    gen = torch.Generator("cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=gen)             # noqa: E731
    shape = (batch, length, channels)
    clean = {k: v.to(t) for k, v in dict(x=rnd(*shape), gate=-rnd(*shape).abs(), dh=rnd(*shape)).items()}
    slices = {k: guarded(torch, shape, t, float("nan"), v)[1] for k, v in clean.items()}
    a, b = (sa.recurrence_solve(q["x"], q["gate"], form="log", coupled=True) for q in (clean, slices))
    assert torch.equal(a.h, b.h) and torch.equal(a.h_final, b.h_final)
    assert all(torch.equal(u, v) for u, v in zip(sa.recurrence_adjoint(a, clean["dh"]), sa.recurrence_adjoint(b, slices["dh"])))

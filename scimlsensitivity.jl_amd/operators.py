"""Operators of sequence models on torch device tensors, next to the solves: the gated linear recurrence with its adjoint and its single step, and the
orthogonalised update of weight matrices (include/hipadj.h: hipadj_recurrence*, hipadj_orthogonalized_update*).

torch is used for device memory and streams only: a call runs on torch's current stream of its tensors' device, its workspace comes from torch's allocator on that
stream, nothing is kept between calls, and nothing waits for the device (so every call can be captured into a graph)."""
import ctypes as C

from . import _lib
from ._lib import HipadjError, HipadjOrthogonal, HipadjRecurrence

GATES = {"decay": 0, "log": 1, "sigmoid": 2}
_DTYPES = None


def _torch():
    global _DTYPES
    import torch
    if _DTYPES is None:
        _DTYPES = {torch.float64: 0, torch.float32: 1, torch.bfloat16: 2, torch.float16: 3}
    return torch


def _check(rc):
    if rc != _lib.OK:
        raise HipadjError(rc, _lib.load().hipadj_last_error(None).decode())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream(torch, device):
    """The hipStream_t of torch's current stream (as torch.cuda.current_stream(device).cuda_stream, without the Stream object: 0.1 of 2 us)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _on(name, t, like, dtype=None, shape=None):
    if t.device != like.device:
        raise ValueError(f"{name} lives on {t.device}, x on {like.device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _adjacent(t):
    return t.dim() == 0 or t.shape[-1] <= 1 or t.stride(-1) == 1


def _rows(t):
    """t with channels next to each other: as it is, or a copy; a view whose sign torch has yet to turn (the imaginary part of a conjugate) with its sign turned."""
    t = t.resolve_neg()
    return t if _adjacent(t) else t.contiguous()


def _gate_types(torch, x, gate, form):
    if not x.is_cuda:
        raise ValueError("x must be a GPU tensor: there is no CPU fallback")
    if form not in GATES:
        raise ValueError(f"form must be one of {sorted(GATES)}, got {form!r}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be float64, float32, bfloat16 or float16, got {x.dtype}")
    if gate.dtype != x.dtype and not (gate.dtype == torch.float32 and x.dtype in (torch.bfloat16, torch.float16)):
        raise ValueError(f"gate must have x's type ({x.dtype}), or float32 next to bfloat16 / float16; got {gate.dtype}")
    _on("gate", gate, x, shape=x.shape)
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def _written(torch, name, t):
    """Before a call writes t in place, outside of what autograd records: refused where that would make a recorded gradient wrong, and counted as a change of t, so that a graph that has
    saved t says so."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad and is written in place, which has no gradient: call under torch.no_grad(), or pass {name}.detach()")
    if t.is_neg():
        raise ValueError(f"{name} is a view whose sign is yet to be turned (the imaginary part of a conjugate) and cannot be written in place: pass {name}.resolve_neg()")
    torch.autograd.graph.increment_version(t)


class RecurrenceSolution:
    """What recurrence_solve returns: h [like x], h_final [rows][channels], and what recurrence_adjoint needs of the forward pass (x, the gate and h0 by
    reference — they must not change before the adjoint — and the states at the checkpoints)."""
    __slots__ = ("h", "h_final", "x", "gate", "h0", "offsets", "form", "coupled", "_checkpoints", "_config", "_workspace_bytes", "_state_type", "_final_shape", "_stream")


def _strides(t, packed):
    """(batch, time) strides; a batch of one has none."""
    if packed:
        return (0, t.stride(0))
    return (t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0)


def recurrence_solve(x, gate, h0=None, *, form="log", coupled=False, offsets=None, adjoint=True):
    """The gated linear recurrence h_t = a_t h_{t-1} + b_t of every channel: a = gate ("decay"), exp(gate) ("log") or sigmoid(gate) ("sigmoid"); b = x, or
    (1 - a) x when coupled — with form="log" and gate = -r dt that is the diagonal system h' = r (x - h) stepped exactly.

    x, gate [batch][length][channels] (any batch and time strides), h0 [batch][channels] (None: zeros); or packed sequences: x, gate [rows][channels] and offsets
    [nseq + 1] (int32 / int64 on the same device, ascending), h0 [nseq][channels].  Types: float64, float32, bfloat16, float16; the gate may be float32 next to the
    16-bit ones; h0 and h_final are float64 for float64 and float32 otherwise.  Rows of no sequence get h = 0.
    adjoint=False leaves out the checkpoints that recurrence_adjoint reads.  Returns a RecurrenceSolution."""
    torch = _torch()
    packed = offsets is not None
    if x.dim() != (2 if packed else 3):
        raise ValueError(f"x must be {'[rows][channels]' if packed else '[batch][length][channels]'}, got shape {tuple(x.shape)}")
    wide = _gate_types(torch, x, gate, form)
    x, gate = _rows(x), _rows(gate)
    batch, length, channels = (1, *x.shape) if packed else x.shape
    nseq = 0
    if packed:
        _on("offsets", offsets, x)
        if offsets.dim() != 1 or offsets.numel() < 2 or offsets.dtype not in (torch.int32, torch.int64):
            raise ValueError("offsets must be int32 or int64 [nseq + 1] with at least one sequence")
        offsets = offsets.contiguous()
        nseq = offsets.numel() - 1
    rows = nseq or batch
    if h0 is not None:
        h0 = _on("h0", h0, x, wide, (rows, channels)).resolve_neg().contiguous()
    r = HipadjRecurrence()
    r.struct_size, r.device, r.dtype, r.gate_dtype = C.sizeof(HipadjRecurrence), x.device.index, _DTYPES[x.dtype], _DTYPES[gate.dtype]
    r.gate, r.coupled, r.batch, r.length, r.channels, r.nseq = GATES[form], int(bool(coupled)), batch, length, channels, nseq
    if packed:
        r.offsets, r.offsets_bits = offsets.data_ptr(), 64 if offsets.dtype == torch.int64 else 32
    h = torch.empty_like(x)                                  # in x's order of batch and time, where its channels lie next to each other (not so for windows that overlap)
    if not _adjacent(h):
        h = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    r.x_stride[:], r.gate_stride[:], r.h_stride[:] = _strides(x, packed), _strides(gate, packed), _strides(h, packed)
    L = _lib.load()
    ck, ws = C.c_int64(), C.c_int64()
    _check(L.hipadj_recurrence_sizes(C.byref(r), C.byref(ck), C.byref(ws)))
    sol = RecurrenceSolution()
    sol.h, sol.h_final = h, torch.empty((rows, channels), dtype=wide, device=x.device)
    sol._checkpoints = torch.empty(ck.value, dtype=torch.uint8, device=x.device) if adjoint else None
    work = torch.empty(ws.value, dtype=torch.uint8, device=x.device) if ws.value else None
    sol._stream = _stream(torch, x.device)
    _check(L.hipadj_recurrence_forward_dev(C.byref(r), _ptr(x), _ptr(gate), _ptr(h0), _ptr(h), _ptr(sol.h_final), _ptr(sol._checkpoints), _ptr(work), ws.value, sol._stream))
    sol.x, sol.gate, sol.h0, sol.offsets, sol.form, sol.coupled = x, gate, h0, offsets, form, bool(coupled)
    sol._config, sol._workspace_bytes, sol._state_type, sol._final_shape = r, ws.value, wide, (rows, channels)
    return sol


def recurrence_adjoint(sol, dh=None, dh_final=None, *, need=(True, True, True)):
    """(dx, dgate, dh0): the gradients of sum(dh * h) + sum(dh_final * h_final) with respect to x, gate and h0 (also for h0=None: of the zeros), each of its
    argument's type; dh [like h], dh_final [like h_final], None = zeros.  need: which of the three to compute (the others are None).  On a stream other than the solution's, that stream
    has to wait for the solution's first, as for any tensor."""
    torch = _torch()
    if sol._checkpoints is None:
        raise ValueError("the solution was computed with adjoint=False: it has no checkpoints")
    x, gate, packed = sol.x, sol.gate, sol.offsets is not None
    r = HipadjRecurrence.from_buffer_copy(sol._config)
    r.x_stride[:], r.gate_stride[:] = _strides(x, packed), _strides(gate, packed)      # of the tensors as they are now: hooks on saved tensors may have laid them out anew
    if packed:
        r.offsets = sol.offsets.data_ptr()
    if dh is not None:
        dh = _rows(_on("dh", dh, x, x.dtype, x.shape))
        r.dh_stride[:] = _strides(dh, packed)
    if dh_final is not None:
        dh_final = _on("dh_final", dh_final, x, sol._state_type, sol._final_shape).resolve_neg().contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
    dgate = torch.empty(gate.shape, dtype=gate.dtype, device=x.device) if need[1] else None
    dh0 = torch.empty(sol._final_shape, dtype=sol._state_type, device=x.device) if need[2] else None
    if dx is not None:
        r.dx_stride[:] = _strides(dx, packed)
    if dgate is not None:
        r.dgate_stride[:] = _strides(dgate, packed)
    stream = _stream(torch, x.device)
    if stream != sol._stream:                                # what the solution holds of its own is not to be handed out again before this stream has read it
        for t in (x, gate, sol.h0, sol.offsets, sol._checkpoints):
            if t is not None:
                t.record_stream(torch.cuda.current_stream(x.device))
    work = torch.empty(sol._workspace_bytes, dtype=torch.uint8, device=x.device) if sol._workspace_bytes else None
    _check(_lib.load().hipadj_recurrence_adjoint_dev(C.byref(r), _ptr(x), _ptr(gate), _ptr(sol.h0), _ptr(sol._checkpoints), _ptr(dh), _ptr(dh_final), _ptr(dx), _ptr(dgate), _ptr(dh0),
                                                     _ptr(work), sol._workspace_bytes, stream))
    return dx, dgate, dh0


_function = None


def gated_recurrence(x, gate, h0=None, *, form="log", coupled=False, offsets=None):
    """(h, h_final) of the gated linear recurrence (recurrence_solve), differentiable by torch's autograd with respect to x, gate and h0; first derivatives.
    Forward and backward can be captured into a graph; as with any function of torch's autograd, no eager result of the same leaves may be alive at the capture (the engine would
    wait for the eager pass's stream inside it)."""
    global _function
    torch = _torch()
    if _function is None:
        class GatedRecurrence(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, gate, h0, form, coupled, offsets, graph):
                want = graph and any(ctx.needs_input_grad[:3])      # (the latter are set under no_grad too)
                sol = recurrence_solve(x, gate, h0, form=form, coupled=coupled, offsets=offsets, adjoint=want)
                if want:
                    saved = (sol.x, sol.gate, sol.h0, sol.offsets, sol._checkpoints)
                    ctx.save_for_backward(*saved)            # versions are checked: a changed input is an error, not a wrong gradient
                    ctx.kinds = [(None, None, None) if t is None else (t.dtype, t.shape, t.device) for t in saved]
                    ctx.rest = (sol.form, sol.coupled, sol._config, sol._workspace_bytes, sol._state_type, sol._final_shape, sol._stream)
                    ctx.set_materialize_grads(False)
                return sol.h, sol.h_final

            @staticmethod
            @torch.autograd.function.once_differentiable
            def backward(ctx, dh, dh_final):
                sol = RecurrenceSolution()
                saved = []
                for name, t, (dtype, shape, device) in zip(("x", "gate", "h0", "offsets", "the checkpoints"), ctx.saved_tensors, ctx.kinds):
                    if t is not None and (t.dtype, t.shape, t.device) != (dtype, shape, device):
                        raise ValueError(f"{name} was saved as {dtype} {tuple(shape)} on {device} and came back as {t.dtype} {tuple(t.shape)} on {t.device}")
                    saved.append(t if t is None else _rows(t) if name in ("x", "gate") else t.resolve_neg().contiguous())
                sol.x, sol.gate, sol.h0, sol.offsets, sol._checkpoints = saved
                sol.form, sol.coupled, sol._config, sol._workspace_bytes, sol._state_type, sol._final_shape, sol._stream = ctx.rest
                dx, dgate, dh0 = recurrence_adjoint(sol, dh, dh_final, need=ctx.needs_input_grad[:3])
                return dx, dgate, dh0, None, None, None, None
        _function = GatedRecurrence
    return _function.apply(x, gate, h0, form, coupled, offsets, torch.is_grad_enabled())


def gated_recurrence_step(x, gate, state, *, form="log", coupled=False, slots=None):
    """One step of running sequences: state[slots[i]] <- a state[slots[i]] + b in place, and h[i] = the new state in x's type.  x, gate [batch][channels]; state
    [nslots][channels] float32 (float64 for float64); slots int32 / int64 [batch] or None (row i has state i).  A slot outside the states (-1) pads the batch: h[i] = 0.
    Rows with the same slot are consecutive steps of that state in row order.  No gradients: gated_recurrence over one row has them; a state that requires grad is refused in grad mode.  x and gate may not
    lie in state."""
    torch = _torch()
    if x.dim() != 2:
        raise ValueError(f"x must be [batch][channels], got shape {tuple(x.shape)}")
    wide = _gate_types(torch, x, gate, form)
    if state.device != x.device or state.dtype != wide or state.dim() != 2 or state.shape[1] != x.shape[1] or (state.shape[1] > 1 and state.stride(1) != 1):
        raise ValueError(f"state must be {wide} [nslots][{x.shape[1]}] on {x.device} with neighbouring channels, got {state.dtype} {tuple(state.shape)} on {state.device}")
    if state.shape[0] > 1 and abs(state.stride(0)) < state.shape[1]:
        raise ValueError("the rows of state overlap")
    if slots is not None:
        if slots.device != x.device or slots.dtype not in (torch.int32, torch.int64) or tuple(slots.shape) != (x.shape[0],):
            raise ValueError(f"slots must be int32 or int64 [{x.shape[0]}] on {x.device}")
        slots = slots.contiguous()
    elif state.shape[0] < x.shape[0]:
        raise ValueError(f"{x.shape[0]} rows without slots need as many states, got {state.shape[0]}")
    x, gate = _rows(x), _rows(gate)
    _written(torch, "state", state)
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    _check(_lib.load().hipadj_recurrence_step_dev(x.device.index, _DTYPES[x.dtype], _DTYPES[gate.dtype], GATES[form], bool(coupled), x.shape[0], x.shape[1], x.data_ptr(), x.stride(0),
                                                  gate.data_ptr(), gate.stride(0), state.data_ptr(), state.stride(0), state.shape[0], _ptr(slots),
                                                  64 if slots is not None and slots.dtype == torch.int64 else 32, h.data_ptr(), h.stride(0), _stream(torch, x.device)))
    return h


def _disjoint(t):
    """Whether no two elements of t [batch, rows, cols] share a place, for a t with columns or rows next to each other (others are refused for that)."""
    if t.numel() == 0:
        return True
    t = t if _adjacent(t) else t.transpose(-1, -2)
    if not _adjacent(t):
        return True
    (batch, rows, cols), (sb, sr, _) = t.shape, t.stride()
    if rows > 1 and sr < cols:
        return False
    if batch == 1 or sb > (rows - 1) * sr + cols - 1 or (sb >= cols and sr > (batch - 1) * sb + cols - 1):      # one behind the other, or side by side
        return True
    # matrix k starts k sb behind the first: not within cols of one of its rows
    return all(k * sb - r * sr >= cols and (r + 1 >= rows or (r + 1) * sr - k * sb >= cols) for k in range(1, batch) for r in (min(rows - 1, k * sb // max(sr, 1)),))


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)      # the usual quintic: steep at zero, singular values end in 0.7 ... 1.2 (K. Jordan, Muon, 2024)


def orthogonalized_update(grad, momentum=None, *, beta=0.95, nesterov=True, steps=5, coefficients=NEWTON_SCHULZ, scale=1.0, out=None):
    """The orthogonalised update of weight matrices: momentum <- beta momentum + grad (in place, float32, like grad; None: no momentum), u = grad + beta momentum
    (nesterov) or momentum, X = u / (|u| + 1e-7), `steps` times X <- c0 X + c1 A X + c2 A A X with A = X X', and scale X is returned in grad's type.

    grad [..., rows, cols] float32, bfloat16 or float16: every matrix of the leading dimensions by itself (heads, layers); row-major or its transpose.
    coefficients: three numbers, or three for each step.  out: where to write (like grad; grad itself is allowed); momentum may overlap
    neither, and neither momentum nor out may require grad in grad mode.  For weights W [out, in] the usual step is
    W -= lr * orthogonalized_update(dW, m, scale=max(1, out / in) ** 0.5)."""
    torch = _torch()
    if not grad.is_cuda:
        raise ValueError("grad must be a GPU tensor: there is no CPU fallback")
    if grad.dim() < 2:
        raise ValueError(f"grad must be [..., rows, cols], got shape {tuple(grad.shape)}")
    if grad.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"grad must be float32, bfloat16 or float16, got {grad.dtype}")
    for name, t, dt in (("momentum", momentum, torch.float32), ("out", out, grad.dtype)):
        if t is not None:
            _on(name, t, grad, dt, grad.shape)
    try:
        co = [float(c) for c in coefficients] * int(steps)
    except TypeError:                                        # rows of three
        co = [float(c) for row in coefficients for c in row]
    if len(co) != 3 * int(steps):
        raise ValueError(f"coefficients: three numbers, or three for each of the {steps} steps")

    def matrices(t):       # [batch, rows, cols] with one stride between matrices; None where t's memory does not allow it
        if t.dim() == 2:
            return t.unsqueeze(0)
        try:
            return t.view(-1, *t.shape[-2:]) if t.dim() > 3 else t
        except RuntimeError:
            return None

    given_out, grad = out, grad.resolve_neg()
    if out is None:
        out = torch.empty(grad.shape, dtype=grad.dtype, device=grad.device) if grad.stride(-1) == 1 or grad.stride(-2) != 1 else \
            torch.empty((*grad.shape[:-2], grad.shape[-1], grad.shape[-2]), dtype=grad.dtype, device=grad.device).transpose(-1, -2)
    g, m, o = matrices(grad), None if momentum is None else matrices(momentum), matrices(out)
    if g is None:
        g = matrices(grad.contiguous())
    if (momentum is not None and (m is None or not _disjoint(m))) or o is None or not _disjoint(o):
        raise ValueError("momentum and out are written in place: their matrices must lie at one stride from each other and not overlap")
    # one order for all: columns next to each other, or the transposes (the iteration commutes with transposition)
    row_major = lambda t: t.shape[-1] <= 1 or t.stride(-1) == 1       # noqa: E731
    written = [t for t in (m, o) if t is not None]
    if not all(row_major(t) for t in written):
        if not all(row_major(t.transpose(-1, -2)) for t in written):
            raise ValueError("momentum and out must both be row-major or both be column-major")
        g, o, m = g.transpose(-1, -2), o.transpose(-1, -2), None if m is None else m.transpose(-1, -2)
    if not row_major(g):
        g = g.contiguous()
    q = HipadjOrthogonal()
    q.struct_size, q.device, q.dtype, q.steps, q.nesterov = C.sizeof(HipadjOrthogonal), grad.device.index, _DTYPES[grad.dtype], int(steps), int(bool(nesterov))
    q.batch, q.rows, q.cols = g.shape
    q.grad_stride[:], q.out_stride[:] = (g.stride(0), g.stride(1)), (o.stride(0), o.stride(1))
    if m is not None:
        q.momentum_stride[:] = (m.stride(0), m.stride(1))
    q.beta, q.scale = float(beta), float(scale)
    co = (C.c_double * len(co))(*co)
    q.coefficients = C.cast(co, C.POINTER(C.c_double))
    L = _lib.load()
    ws = C.c_int64()
    _check(L.hipadj_orthogonalized_update_size(C.byref(q), C.byref(ws)))
    if m is not None and m.numel() and m.data_ptr() in (g.data_ptr(), o.data_ptr()):
        raise ValueError("momentum is written in place and may not be grad or out")
    for name, t in (("momentum", momentum), ("out", given_out)):
        if t is not None:
            _written(torch, name, t)
    work = torch.empty(ws.value, dtype=torch.uint8, device=grad.device) if ws.value else None
    _check(L.hipadj_orthogonalized_update_dev(C.byref(q), _ptr(g), _ptr(m), _ptr(o), _ptr(work), ws.value, _stream(torch, grad.device)))
    return given_out if given_out is not None else out

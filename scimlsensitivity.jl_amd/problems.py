"""Problem / solver / loss descriptors of the host API (names follow SciMLBase / OrdinaryDiffEq)."""
from dataclasses import dataclass, field
import numpy as np
np_ = np   # DeviceFunction's constructor takes `np` (the parameter count, as the C ABI names it)

from . import _lib


@dataclass(frozen=True)
class RK4:
    """Fixed-step classic Runge-Kutta 4 (the `alg` handed to solve / adjoint_sensitivities)."""


@dataclass(frozen=True)
class Tsit5:
    """Adaptive Tsitouras 5(4) with PI step control and its own 4th-order interpolant — the stepper of the
    reference's own tests (test/Core3/adjoint.jl:31-43).  Per-trajectory step sequences on the device."""


@dataclass(frozen=True)
class Rosenbrock23:
    """Adaptive Rosenbrock23 (ode23s as OrdinaryDiffEq ships it) — the stiff stepper of the lane-per-trajectory models (include/hipadj.h
    HIPADJ_STEPPER_ROSENBROCK23_ADAPTIVE; the solver of test/Core2/stiff_adjoints.jl:53-75).  Forward AND reverse solve run with it (the adjoint takes the forward solve's alg,
    src/sensitivity_interface.jl:487-491): W = I - d h J factored per lane in registers, J from the model's VJP.  Interpolating-, Gauss-, GaussKronrod- and QuadratureAdjoint;
    `abstol` / `reltol` as for Tsit5()."""


@dataclass(frozen=True)
class ETDRK4:
    """Fixed-step exponential Runge-Kutta 4 (Cox & Matthews 2002; OrdinaryDiffEq's ETDRK4 for SplitODEProblems): the stiff linear part of a semilinear problem is integrated
    exactly, the step is bound by the nonlinear part only.  Offered for the PDE family ("bruss": the periodic diffusion operator is diagonal in the 2-D DFT basis,
    csrc/hipadj_field_etd.hpp) with Interpolating- and QuadratureAdjoint — the stepper for the horizon the reference's Brusselator example documents with FBDF
    (docs/src/examples/pde/brusselator.md:115)."""


class DeviceFunction:
    """ODEFunction(f!; vjp, vjp_p) for the device (src/derivative_wrappers.jl:284-359, test/Core3/user_vjp.jl:77):
    the three function BODIES as HIP C++ text over `du`/`out`, `u`, `p`, `lam`, `t` (all double), compiled at solve time
    with hiprtc for gfx950.  Usable wherever a registered model name is: ODEProblem(DeviceFunction(...), u0, tspan, p).
    With vjp = vjp_p = None the VJPs are generated by forward-mode dual numbers (the reference's autojacvec = true); the body
    of `f` must then declare its locals as `real` (or `auto`)."""

    def __init__(self, name, n, np, f, vjp=None, vjp_p=None, check=False, mass_matrix=None):
        self.name, self.n, self.np = name, int(n), int(np)
        self.id = _lib.register_model(name, n, np, f, vjp, vjp_p, check=False)
        self.mass_matrix = None
        self.affect = None
        if mass_matrix is not None:
            self.set_mass_matrix(mass_matrix)
        if check:
            _lib.check_model(self.id)

    @classmethod
    def from_callable(cls, name, f, n, np, auto_vjp=False, check=False, mass_matrix=None, bundle=False):
        """ODEFunction(f!) from a host-language function: `f(du, u, p, t)` is traced once (trace.py), its expression graph is
        differentiated in reverse mode, and f, (df/du)^T lam, (df/dp)^T lam are emitted as C text — the path from a user's `f` to the
        device that the Julia glue takes with Symbolics (julia/HIPAdj/ext/HIPAdjSymbolicsExt.jl).  auto_vjp = True emits f alone and
        leaves both VJPs to forward-mode dual numbers on the device (autojacvec = true).  bundle = True writes the VJP temporaries as `auto`, which lets
        segment lanes push all adjoint columns through the bodies at once (column bundles)."""
        from . import trace
        fb, vu, vp = trace.bodies(f, n, np, auto_vjp=auto_vjp, bundle=bundle)
        fun = cls(name, n, np, fb, vu, vp, check=check, mass_matrix=mass_matrix)
        fun.source = dict(f=fb, vjp=vu, vjp_p=vp)
        return fun

    def set_mass_matrix(self, M):
        """ODEFunction(f; mass_matrix = M): M u' = f with a constant non-singular matrix (test/Core3/adjoint.jl:1315-1376).  The
        adjoint follows the reference's convention: dp is the gradient, du0 is lam(t0) of M' lam' = -J' lam (src/sensitivity_interface.jl:500),
        i.e. dG/du0 = M' du0.  A SINGULAR M of the semi-explicit form [Md 0; 0 0] (zero rows that are also zero columns: algebraic variables, src/adjoint_common.jl:116-135) makes
        the model a DAE: `Rosenbrock23()` integrates it in mass-matrix form from a consistent state (the algebraic variables of u0 are solved for, BrownFullBasicInit) with
        Interpolating-, Gauss-, GaussKronrod- and QuadratureAdjoint (test/Core3/adjoint.jl:1434-1530); every other stepper refuses such a model.  None removes the matrix."""
        _lib.set_model_mass_matrix(self.id, self.n, M)
        self.mass_matrix = None if M is None else np_.array(M, dtype=np_.float64)
        return self

    def set_affect(self, body):
        """The affect! of a DiscreteCallback as device text (test/Callbacks1/discrete_callbacks.jl:260-330): `body` edits `un` — which starts
        as a copy of `u` — from `u`, `p`, `t` (locals `real`), e.g. "un[0] += 2.0;" or "for (int i = 0; i < N; ++i) un[i] += p[1] / 8.0 * sin(u[i]);".
        Used by solve(..., callback=PresetTimeCallback(times)).  None removes it."""
        _lib.set_model_affect(self.id, body)
        self.affect = body
        return self

    def set_continuous_callback(self, condition, affect=None, max_events=0, ncond=1, direction=0):
        """ContinuousCallback(condition, affect!; save_positions = (false, false)) as device text (test/Callbacks2/continuous_callbacks.jl; src/callback_tracking.jl:232-479):
        `condition` assigns `c` from `u`, `p`, `t` — the event is its zero crossing, in either direction —, `affect` edits `un` (a copy of `u`; `terminate = true;` in it is
        terminate!(integrator)); e.g. the bouncing ball:
        condition="c = u[0];", affect="un[1] = -p[1] * u[1];".  Every later solve of the model with Tsit5() / Rosenbrock23() locates the events per trajectory on the dense
        output; every sensealg differentiates through them, event times included (checkpointing=True included).  `max_events` bounds the events of one trajectory (0 = 64).
        `ncond` > 1: a VectorContinuousCallback — `condition` assigns `out[0 .. ncond)`, `affect` also sees `idx`, the component that fired
        (test/Callbacks2/vector_continuous_callbacks.jl), e.g. condition="out[0] = u[0]; out[1] = (u[2] - 10.0) * u[2];".  condition=None removes the callback."""
        _lib.set_model_continuous_callback(self.id, condition, affect, max_events, ncond)
        if condition is not None and direction:      # +1: only upcrossings fire (ContinuousCallback(condition, affect!, nothing)); -1: only downcrossings
            _lib.set_model_callback_direction(self.id, direction)
        self.continuous_callback = None if condition is None else (condition, affect)
        from . import interface
        interface._attached_callbacks.pop(self.id, None)
        return self

    def set_discrete_loss(self, dgdu=None, dgdp=None, l=None, body=None, value=False):
        """Attach a discrete loss that stays on the device — the `dgdu_discrete` / `dgdp_discrete` keywords of adjoint_sensitivities
        (src/sensitivity_interface.jl:373-526; evaluated by ReverseLossCallback, src/adjoint_common.jl:771-779) as HIP C++ bodies writing `out` from
        `u`, `p`, `t`, `i` (0-based index of the loss time) and `d` (the data column of this trajectory and time), e.g. dgdu="for (int j = 0; j < N; ++j) out[j] = 2.0 * (u[j] - d[j]);".
        Alternatively l="l = u[0]*u[0] + p[0];" gives the loss itself (gradients by dual numbers; `real` locals) and lets the device return its value.
        l may also be a host-language callable l(u, p, t, i, d) -> scalar: it is traced once (trace.discrete_loss_bodies) like the right-hand side of from_callable and
        its gradients are emitted as explicit bodies; value=True hands the loss itself over instead (gradients by dual numbers), so that the device can also return its value.
        A WideDeviceFunction takes one SPMD `body` instead (include/hipadj.h hipadj_wmodel_set_discrete_loss).  Select with dgdu_discrete=ModelLoss(data)."""
        if callable(l):
            from . import trace
            gu, gp, lb = trace.discrete_loss_bodies(l, self.n, self.np)
            self.discrete_loss_source = dict(dgdu=gu, dgdp=gp, l=lb)
            if value:
                _lib.set_model_discrete_loss(self.id, None, None, lb)
            else:
                _lib.set_model_discrete_loss(self.id, gu, gp, None)
            return self
        _lib.set_model_discrete_loss(self.id, dgdu, dgdp, l, wide=body)
        return self

    def set_cost(self, dgdu=None, dgdp=None, g=None):
        """Attach a continuous cost through its gradients — the `dgdu_continuous` / `dgdp_continuous` keywords of
        adjoint_sensitivities (src/sensitivity_interface.jl:373-526) as HIP C++ bodies writing `out` from `u`, `p`, `t`.
        Alternatively g="g = u[0]*u[0] + p[0];" gives the cost itself and its gradients come from dual numbers.
        Select it with solve(..., g=ModelCost())."""
        _lib.set_model_cost(self.id, dgdu, dgdp, g)
        return self

    def __repr__(self):
        return f"DeviceFunction({self.name!r}, n={self.n}, np={self.np}, id={self.id})"


DENSE_CHAINS = {}            # model name -> (widths, input_power) of WideDeviceFunction.dense_chain models (declared to the library, which selects their kernel family)
WIDE_MASS_MATRICES = {}      # model name -> M of traced wide models registered with a mass matrix (WideDeviceFunction.from_callable): engine.py maps du0 with it


class WideDeviceFunction(DeviceFunction):
    """A right-hand side for the workgroup-per-trajectory family (csrc/hipadj_wide.hpp; include/hipadj.h `hipadj_wmodel_register`): more than
    8 states or more than 32 parameters, up to n = 4096.  One workgroup of `threads` threads integrates one trajectory; `f` and `vjp` are SPMD
    bodies of HIP C++ run by every thread (work split with HIPADJ_W_FOR(i, count), phases separated by wg_sync(), `ws` = `lds_doubles` of LDS
    scratch).  `vjp` is the joint product of the reference's vecjacobian! (src/derivative_wrappers.jl:256-267): dlam = (df/du)' lam and, under
    `if (WP)`, `gp[j] += w * ...` for gradient entries owned by one thread or `acc[q] += w * ...` for the `nacc` parameters
    [acc_first, acc_first + nacc) that every component feeds.  The emitters below write these bodies for common structured models."""

    def __init__(self, name, n, np, f, vjp, threads=0, lds_doubles=0, nacc=0, acc_first=0, check=False):
        self.name, self.n, self.np = name, int(n), int(np)
        self.id = _lib.register_wide_model(name, n, np, f, vjp, threads, lds_doubles, nacc, acc_first, check=False)
        WIDE_MASS_MATRICES.pop(name, None)      # a name registered again starts without the mass matrix of its predecessor (from_callable sets it below)
        DENSE_CHAINS.pop(name, None)            # ... and is a dense chain only if dense_chain registers it again
        self.mass_matrix, self.affect = None, None
        self.source = dict(f=f, vjp=vjp, lds_doubles=int(lds_doubles), nacc=int(nacc), acc_first=int(acc_first), threads=int(threads))
        if check:
            _lib.check_model(self.id)

    @classmethod
    def dense_chain(cls, name, widths, input_power=1, threads=0, check=False):
        """Lux.Chain(x -> x.^input_power, Dense(w0, w1, tanh), ..., Dense(w_{L-1}, w_L)) as a right-hand side u' = chain(u): tanh on every layer
        but the last, parameters in Lux's flattening order (per layer: weight [out x in] column-major, then bias).  widths = (2, 50, 2) with
        input_power = 3 is the neural ODE of docs/src/Benchmark.md:62."""
        w = [int(x) for x in widths]
        if len(w) < 2 or w[0] != w[-1]:
            raise ValueError("dense_chain: widths = (n, ..., n) with at least one layer")
        L = len(w) - 1
        Woff, Boff, off = [0], [0], 0
        for l in range(1, L + 1):
            Woff.append(off); off += w[l] * w[l - 1]
            Boff.append(off); off += w[l]
        npar = off
        A = [0]                                   # activations a_0 .. a_{L-1} in ws
        for l in range(1, L):
            A.append(A[-1] + w[l - 1])
        G0 = A[-1] + w[L - 1]                      # backward vectors g_{L-1} .. g_0 after them
        G = {}
        o = G0
        for l in range(L - 1, -1, -1):
            G[l] = o; o += w[l]
        nw = o
        inp = "u[i]" if input_power == 1 else " * ".join(["u[i]"] * int(input_power))
        dinp = "1.0" if input_power == 1 else f"{float(input_power)} * " + " * ".join(["u[j]"] * (int(input_power) - 1))
        NARROW = 8      # a contraction with at most this many outputs over at least 16 inputs runs lanes-over-inputs + wg_sum (shuffle butterfly) per output

        def matvec(out_expr, n_out, n_in, coef, vec, bias=None, post="s"):
            """out_expr(i) = post(bias_i + sum_j coef(i, j) * vec(j)): lanes over the outputs with a serial loop over the inputs, or — few outputs, many inputs —
            lanes over the inputs and one workgroup sum per output"""
            if n_out <= NARROW and n_in >= 16:
                lines = []
                for i in range(n_out):
                    b = f"{bias(i)} + " if bias else ""
                    lines.append(f"{{ double part = 0.0; HIPADJ_W_FOR(j, {n_in}) part += {coef(str(i), 'j')} * {vec('j')}; const double s = {b}wg_sum(part); if (tid == 0) {out_expr(str(i))} = {post.replace('IDX', str(i))}; }}")
                return lines
            b = bias("i") if bias else "0.0"
            return [f"HIPADJ_W_FOR(i, {n_out}) {{ double s = {b}; for (int j = 0; j < {n_in}; ++j) s += {coef('i', 'j')} * {vec('j')}; {out_expr('i')} = {post.replace('IDX', 'i')}; }}"]

        if L == 2 and w[0] <= NARROW:
            # ONE hidden layer between few inputs / outputs (the published 2-50-2 net): everything a hidden unit needs or produces stays in the registers of the
            # thread that owns it — input powers recomputed per thread, activation, its back-propagated value, its five gradient entries — with no LDS
            # publication and no barrier; only the d outputs (f) / the d entries of dlam (vjp) cross lanes, in pairs (wg_sum2: two wavefront sums for 27 instructions).  (Round 3's form published
            # every layer to `ws`, walked the weight gradients with e % w / e / w loops of two masked iterations and needed three barriers: ~250 instructions per
            # joint VJP against ~130 here.)
            d, H = w[0], w[1]
            W1, B1, W2, B2 = Woff[1], Boff[1], Woff[2], Boff[2]
            xs = [f"const double x{k} = " + (" * ".join([f"u[{k}]"] * int(input_power))) + ";" for k in range(d)]
            # every multiply-add is an explicit fma(): a sum of two products can be contracted either way round, and the dense and the checkpointed sweep (two kernels,
            # compared bit for bit by the tests) must not depend on which way the compiler picked in each
            hid = (f"double s = p[{B1} + i]; " + " ".join(f"s = fma(p[{W1} + i + {k * H}], x{k}, s);" for k in range(d)) + " const double h = tanh(s);")
            fb = "\n".join(xs + [" ".join(f"double part{m} = 0.0;" for m in range(d)),
                                 f"HIPADJ_W_FOR(i, {H}) {{ {hid} " + " ".join(f"part{m} = fma(p[{W2} + {m} + i * {d}], h, part{m});" for m in range(d)) + " }"] +
                           [(f"{{ double s{m}, s{m + 1}; wg_sum2(part{m}, part{m + 1}, s{m}, s{m + 1}); if (tid >= {m} && tid < {m + 2}) du[tid] = p[{B2} + tid] + (tid == {m} ? s{m} : s{m + 1}); }}"
                             if m + 1 < d else f"{{ const double s = p[{B2} + {m}] + wg_sum(part{m}); if (tid == {m}) du[{m}] = s; }}") for m in range(0, d, 2)])
            dx = [("1.0" if input_power == 1 else f"{float(input_power)} * " + " * ".join([f"u[{k}]"] * (int(input_power) - 1))) for k in range(d)]
            dxt = "1.0" if input_power == 1 else f"{float(input_power)} * " + " * ".join(["u[tid]"] * (int(input_power) - 1))      # the same, for the thread that owns entry tid
            vb = "\n".join(xs + [" ".join(f"const double l{m} = lam[{m}];" for m in range(d)), " ".join(f"double part{k} = 0.0;" for k in range(d)),
                                 f"HIPADJ_W_FOR(i, {H}) {{ {hid}",
                                 f"  double gh = p[{W2} + 0 + i * {d}] * l0; " + " ".join(f"gh = fma(p[{W2} + {m} + i * {d}], l{m}, gh);" for m in range(1, d)),
                                 "  if (WP) { const double wh = w * h; " + " ".join(f"gp[{W2} + {m} + i * {d}] = fma(l{m}, wh, gp[{W2} + {m} + i * {d}]);" for m in range(d)) + " }",
                                 "  gh *= 1.0 - h * h;",
                                 "  if (WP) { const double wg = w * gh; " + " ".join(f"gp[{W1} + i + {k * H}] = fma(wg, x{k}, gp[{W1} + i + {k * H}]);" for k in range(d)) + f" gp[{B1} + i] += wg; }}",
                                 "  " + " ".join(f"part{k} = fma(p[{W1} + i + {k * H}], gh, part{k});" for k in range(d)) + " }",
                                 f"if (WP) {{ HIPADJ_W_FOR(m, {d}) gp[{B2} + m] = fma(w, lam[m], gp[{B2} + m]); }}"] +
                           [(f"{{ double s{k}, s{k + 1}; wg_sum2(part{k}, part{k + 1}, s{k}, s{k + 1}); if (tid >= {k} && tid < {k + 2}) dlam[tid] = (tid == {k} ? s{k} : s{k + 1}) * {dxt}; }}"
                             if k + 1 < d else f"{{ const double s = wg_sum(part{k}); if (tid == {k}) dlam[{k}] = s * {dx[k]}; }}") for k in range(0, d, 2)])
            fun = cls(name, w[0], npar, fb, vb, threads=threads, lds_doubles=1, check=check)
            fun.chain = (tuple(w), int(input_power)); DENSE_CHAINS[name] = fun.chain
            _lib.declare_dense_chain(fun.id, w, input_power)      # the library selects the kernel family from the structure (hipadj_wmodel_declare_dense_chain, ABI 109)
            return fun
        fwd = [f"HIPADJ_W_FOR(i, {w[0]}) ws[{A[0]} + i] = {inp};", "wg_sync();"]
        for l in range(1, L):
            fwd += matvec(lambda i, l=l: f"ws[{A[l]} + {i}]", w[l], w[l - 1], lambda i, j, l=l: f"p[{Woff[l]} + {i} + {j} * {w[l]}]", lambda j, l=l: f"ws[{A[l - 1]} + {j}]",
                          bias=lambda i, l=l: f"p[{Boff[l]} + {i}]", post="tanh(s)") + ["wg_sync();"]
        fb = "\n".join(fwd + matvec(lambda i: f"du[{i}]", w[L], w[L - 1], lambda i, j: f"p[{Woff[L]} + {i} + {j} * {w[L]}]", lambda j: f"ws[{A[L - 1]} + {j}]",
                                    bias=lambda i: f"p[{Boff[L]} + {i}]"))
        vb = list(fwd)
        for l in range(L, 0, -1):
            gl = "lam" if l == L else f"(ws + {G[l]})"
            # derivative of the activation that produced a_{l-1} (tanh, or the input map for l = 1), as a function of the output index IDX of this product
            dact = dinp.replace("u[j]", "u[IDX]") if l == 1 else f"(1.0 - ws[{A[l - 1]} + IDX] * ws[{A[l - 1]} + IDX])"
            vb += [f"if (WP) {{ HIPADJ_W_FOR(e, {w[l] * w[l - 1]}) gp[{Woff[l]} + e] += w * {gl}[e % {w[l]}] * ws[{A[l - 1]} + e / {w[l]}]; HIPADJ_W_FOR(i, {w[l]}) gp[{Boff[l]} + i] += w * {gl}[i]; }}"]
            # g_{l-1}[j] = (sum_i W_l[i, j] g_l[i]) * dact_j : the transposed product (output index j, input index i)
            vb += matvec((lambda j: f"dlam[{j}]") if l == 1 else (lambda j, l=l: f"ws[{G[l - 1]} + {j}]"), w[l - 1], w[l],
                         lambda j, i, l=l: f"p[{Woff[l]} + {i} + {j} * {w[l]}]", lambda i, gl=gl: f"{gl}[{i}]", post=f"s * {dact}")
            if l > 1:
                vb.append("wg_sync();")
        fun = cls(name, w[0], npar, fb, "\n".join(vb), threads=threads, lds_doubles=nw, check=check)
        fun.chain = (tuple(w), int(input_power)); DENSE_CHAINS[name] = fun.chain
        _lib.declare_dense_chain(fun.id, w, input_power)      # hipadj_create routes (2, H, H, 2) chains with H in {32, 64, 128} to the FP64-MFMA family (csrc/hipadj_route.hpp)
        return fun

    def weight_blocks(self):
        """[(offset, out, in)] of the weights of a dense_chain model in its parameter vector: each the [out x in] matrix column-major, followed by its `out` biases."""
        if getattr(self, "chain", None) is None:
            raise ValueError(f"{self.name} is not a dense_chain model: its parameters are not known to be weight matrices")
        blocks, off = [], 0
        for inp, out in zip(self.chain[0][:-1], self.chain[0][1:]):
            blocks.append((off, out, inp))
            off += out * inp + out
        return blocks

    def orthogonalized_update(self, dp, momentum=None, *, beta=0.95, nesterov=True, steps=5, coefficients=None, device=0):
        """The step of a dense_chain model's parameters after a gradient `dp` [np] of a loss (adjoint_sensitivities, Engine.adjoint_dev): every weight matrix's part is the
        orthogonalised update (operators.orthogonalized_update) of its gradient, times max(1, out / in) ** 0.5; the biases' parts are the plain ones.  p -= lr * the result.
        dp: a numpy array (the result is one, computed on cuda:`device`) or a GPU tensor.  momentum: float32 GPU tensor [np], updated in place (None: no momentum).
        The weights' parts are computed in 32 bits."""
        import torch
        from . import operators
        blocks = self.weight_blocks()
        host = not isinstance(dp, torch.Tensor)
        g = torch.as_tensor(np_.ascontiguousarray(dp), device=f"cuda:{int(device)}") if host else dp.detach()
        if tuple(g.shape) != (self.np,):
            raise ValueError(f"dp must have shape ({self.np},), got {tuple(g.shape)}")
        if momentum is not None and (tuple(momentum.shape) != (self.np,) or momentum.dtype != torch.float32 or momentum.device != g.device or not momentum.is_contiguous()):
            raise ValueError(f"momentum must be a contiguous float32 tensor ({self.np},) on {g.device}")
        g32, out = g.float().contiguous(), torch.empty(self.np, dtype=torch.float32, device=g.device)
        for off, rows, cols in blocks:                       # column-major [rows x cols] is row-major [cols x rows], and the iteration commutes with transposition
            at, b = slice(off, off + rows * cols), slice(off + rows * cols, off + rows * cols + rows)
            view = lambda t: t[at].view(cols, rows)          # noqa: B023, E731
            operators.orthogonalized_update(view(g32), None if momentum is None else view(momentum), beta=beta, nesterov=nesterov, steps=steps,
                                            coefficients=operators.NEWTON_SCHULZ if coefficients is None else coefficients, scale=max(1.0, rows / cols) ** 0.5, out=view(out))
            if momentum is None:
                out[b] = g32[b]
            else:
                momentum[b].mul_(beta).add_(g32[b])
                out[b] = g32[b] + beta * momentum[b] if nesterov else momentum[b]
        out = out.to(g.dtype)
        return out.cpu().numpy() if host else out

    @classmethod
    def from_callable(cls, name, fn, n, np, threads=0, check=False, cost=None, mass_matrix=None):
        """A wide model from a host-language right-hand side written with array operations: `fn(u, p, t, ops) -> du` is traced once (wtrace.py), the recorded
        graph is differentiated in reverse mode and BOTH SPMD bodies are emitted — the automatic counterpart of the reference's AD-generated `vecjacobian!`
        (src/derivative_wrappers.jl:649-1145) for models beyond the lane family's 8 states.  See wtrace.py for the operations.
        cost = g(u, p, t, ops) -> scalar: a continuous cost traced the same way (select it with solve(..., g=ModelCost())).
        mass_matrix = M (constant, non-singular, n x n): ODEFunction(f; mass_matrix = M), M u' = f (test/Core3/adjoint.jl:1315-1376).  The C ABI refuses a mass matrix on a
        wide model; a traced model takes it at trace level instead: the device integrates u' = F(u) = M^{-1} f(u) (ops.matvec_const) and the adjoint nu of THAT system with the
        plain jumps nu += g_u; nu = M' lam with lam the reference's adjoint, so dp is unchanged and the host-pointer entry points map du0 = lam(t0) = M^{-T} nu(t0) (engine.py)."""
        from . import wtrace
        Minv = None
        if mass_matrix is not None:
            M = np_.array(mass_matrix, dtype=np_.float64)
            if M.shape != (int(n), int(n)) or abs(np_.linalg.det(M)) < 1e-13 * max(1.0, np_.abs(M).max()) ** int(n):
                raise ValueError("mass_matrix: a constant NON-SINGULAR n x n matrix for the wide family (a semi-explicit DAE is a lane-family model on Rosenbrock23: DeviceFunction(..., mass_matrix=M))")
            Minv = np_.linalg.inv(M)
            f0 = fn
            fn = lambda u, p, t, ops: ops.matvec_const(Minv, f0(u, p, t, ops))      # noqa: E731
        fb, vb, nw, nacc, acc0 = wtrace.bodies(fn, int(n), int(np))
        cb = None
        if cost is not None:
            cb, cw, _, _ = wtrace.cost_body(cost, int(n), int(np))
            nw = max(nw, cw)
        fun = cls(name, n, np, fb, vb, threads=threads, lds_doubles=nw, nacc=nacc, acc_first=acc0, check=False)
        fun.traced = True
        if Minv is not None:
            fun.mass_matrix = np_.array(mass_matrix, dtype=np_.float64)
            WIDE_MASS_MATRICES[name] = fun.mass_matrix
        if cb is not None:
            fun.set_cost(body=cb)
        if check:
            _lib.check_model(fun.id)
        return fun

    def with_mass_matrix(self, M, name=None):
        """ODEFunction(f; mass_matrix = M) for a wide model with HAND-WRITTEN bodies (test/Core3/adjoint.jl:1315-1376; the C ABI's hipadj_model_set_mass_matrix serves the
        lane family, a traced model takes M in from_callable): registers a NEW model (`name`, default "<this name>_mm") whose bodies wrap this model's text — the device
        integrates u' = F(u) = M^{-1} f(u) and the adjoint nu = M' lam of THAT system:
            f'    runs f into an LDS row behind the model's scratch and applies M^{-1} (a constant table in the code object) on the way to `du`
            vjp'  forms M^{-T} lam in that row and hands it to the model's joint VJP as `lam`:  F_u' nu = f_u' (M^{-T} nu),  F_p' nu = f_p' (M^{-T} nu)
        Loss jumps stay nu += g_u, dp is unchanged, and the host entry points map du0 = lam(t0) = M^{-T} nu(t0) like for traced models (engine.py).  n <= 256."""
        n = self.n
        M = np_.array(M, dtype=np_.float64)
        if M.shape != (n, n) or abs(np_.linalg.det(M)) < 1e-13 * max(1.0, np_.abs(M).max()) ** n:
            raise ValueError("mass_matrix: a constant NON-SINGULAR n x n matrix for the wide family (a semi-explicit DAE is a lane-family model on Rosenbrock23: DeviceFunction(..., mass_matrix=M))")
        if n > 256 or getattr(self, "traced", False) or self.mass_matrix is not None:
            raise ValueError("with_mass_matrix: hand-written wide bodies with n <= 256 and no mass matrix yet (a traced model takes mass_matrix in from_callable)")
        Minv = np_.linalg.inv(M)
        table = ", ".join(float(x).hex() for x in Minv.ravel())           # row-major, exact
        src = self.source
        nw = int(src["lds_doubles"])
        head = f"static constexpr double MINV_[{n * n}] = {{{table}}};\ndouble* const mm_row_ = ws + {nw};\n"
        fb = (head + "double* const mm_du_ = du;\n{ double* const du = mm_row_;\n" + src["f"] + "\n}\nwg_sync();\n"
              f"HIPADJ_W_FOR(i, {n}) {{ double s = 0.0; for (int j = 0; j < {n}; ++j) s = fma(MINV_[i * {n} + j], mm_row_[j], s); mm_du_[i] = s; }}")
        vb = (head + f"HIPADJ_W_FOR(j, {n}) {{ double s = 0.0; for (int i = 0; i < {n}; ++i) s = fma(MINV_[i * {n} + j], lam[i], s); mm_row_[j] = s; }}\nwg_sync();\n"
              "{ const double* const lam = mm_row_;\n" + src["vjp"] + "\n}")
        fun = WideDeviceFunction(name or self.name + "_mm", n, self.np, fb, vb, threads=src["threads"], lds_doubles=nw + n, nacc=src["nacc"], acc_first=src["acc_first"], check=False)
        fun.mass_matrix = M
        WIDE_MASS_MATRICES[fun.name] = M
        if src.get("cost"):
            fun.set_cost(body=src["cost"])
        return fun

    def set_affect(self, body, vjp=""):
        """The affect! of a DiscreteCallback on a wide model (include/hipadj.h hipadj_wmodel_set_affect): `body` edits `un` / `pn` (copies of u / p) from u, p, t as SERIAL code
        over plain arrays; `vjp` edits `lo` / `go` (copies of lam / gp) into the reverse callback lo = (dun/du)' lam + (dpn/du)' gp, go = (dun/dp)' lam + (dpn/dp)' gp
        ("" = the affect's Jacobian is the identity, e.g. a constant dose).  Used by solve(..., callback=PresetTimeCallback(times)).  None removes it."""
        _lib.set_wide_model_affect(self.id, body, None if body is None else vjp)
        self.affect = body
        return self

    def set_cost(self, body=None, dgdu=None, dgdp=None, g=None):
        """The continuous cost of a wide model (include/hipadj.h hipadj_wmodel_set_cost): ONE SPMD body that adds dg/du into `dlam` and, under `if (WP)`, `w * dg/dp` into
        `gp` / `acc` — the `dgdu_continuous` / `dgdp_continuous` keywords of adjoint_sensitivities.  Traced costs: from_callable(..., cost=g).  None removes it."""
        if dgdu is not None or dgdp is not None or g is not None:
            raise ValueError("a wide model takes its cost as one SPMD body (set_cost(body=...)) or traced (from_callable(..., cost=g))")
        L = _lib.load()
        rc = L.hipadj_wmodel_set_cost(int(self.id), None if body is None else body.encode())
        if rc != _lib.OK:
            raise _lib.HipadjError(rc, L.hipadj_last_error(None).decode())
        self.source["cost"] = body
        return self

    @classmethod
    def dense_linear(cls, name, n, threads=0, check=False):
        """u' = A u with A = reshape(p, n, n) (column-major): every parameter is an entry of a dense linear map (np = n^2)."""
        n = int(n)
        fb = f"HIPADJ_W_FOR(i, {n}) {{ double s = 0.0; for (int j = 0; j < {n}; ++j) s += p[i + j * {n}] * u[j]; du[i] = s; }}"
        vb = (f"HIPADJ_W_FOR(j, {n}) {{ double s = 0.0; for (int i = 0; i < {n}; ++i) s += p[i + j * {n}] * lam[i]; dlam[j] = s; }}\n"
              f"if (WP) {{ HIPADJ_W_FOR(e, {n * n}) gp[e] += w * lam[e % {n}] * u[e / {n}]; }}")
        return cls(name, n, n * n, fb, vb, threads=threads, check=check)

    @classmethod
    def index_affine(cls, name, rows, cols, threads=0, check=False):
        """The matrix-state right-hand side of the reference's size test, df[i, j] = p[1] i + p[2] j on a rows x cols state
        (test/Core5/size_handling_adjoint.jl:41-48; 1-based i, j; column-major): both parameters are fed by every component, so their
        gradient is accumulated as per-thread partials (`acc`) and summed over the workgroup once per sweep."""
        R, Cc = int(rows), int(cols)
        fb = f"HIPADJ_W_FOR(c, {R * Cc}) du[c] = p[0] * (double)(c % {R} + 1) + p[1] * (double)(c / {R} + 1);"
        vb = (f"HIPADJ_W_FOR(c, {R * Cc}) dlam[c] = 0.0;\n"
              f"if (WP) {{ HIPADJ_W_FOR(c, {R * Cc}) {{ acc[0] += w * (double)(c % {R} + 1) * lam[c]; acc[1] += w * (double)(c / {R} + 1) * lam[c]; }} }}")
        return cls(name, R * Cc, 2, fb, vb, threads=threads, nacc=2, acc_first=0, check=check)

    def __repr__(self):
        return f"WideDeviceFunction({self.name!r}, n={self.n}, np={self.np}, id={self.id})"


@dataclass
class ODEProblem:
    """ODEProblem(f, u0, tspan, p) with `f` a name from the device model registry (include/hipadj.h)."""
    f: str
    u0: np.ndarray
    tspan: tuple
    p: np.ndarray
    dims: tuple = (0, 0, 0, 0)

    def __post_init__(self):
        if isinstance(self.f, DeviceFunction):
            self.f = self.f.name
        if self.f not in _lib.MODEL:
            raise ValueError(f"unknown model {self.f!r}; registered: {sorted(_lib.MODEL)}")
        self.u0 = np.ascontiguousarray(self.u0, dtype=np.float64)
        self.p = np.ascontiguousarray(self.p, dtype=np.float64)
        self.tspan = (float(self.tspan[0]), float(self.tspan[1]))


@dataclass
class EnsembleProblem:
    """EnsembleProblem(prob; prob_func): N independent trajectories that differ in u0 (and optionally p)
    (test/Core4/ensembles.jl:13-31).  u0: [N][n]; p: [np] shared or [N][np]."""
    prob: ODEProblem
    u0: np.ndarray
    p: np.ndarray = None

    def __post_init__(self):
        self.u0 = np.ascontiguousarray(self.u0, dtype=np.float64)
        if self.u0.ndim != 2:
            raise ValueError("EnsembleProblem u0 must be [N][n]")
        self.p = self.prob.p if self.p is None else np.ascontiguousarray(self.p, dtype=np.float64)


@dataclass(frozen=True)
class PresetTimeCallback:
    """DiscreteCallback(condition = t in times, affect!) with the affect attached to the DeviceFunction (set_affect) and the times as
    tstops (test/Callbacks1/discrete_callbacks.jl).  save_positions = (false, false): a save time that coincides with an event time holds
    the RIGHT limit (the state after the affect)."""
    times: tuple

    def __post_init__(self):
        object.__setattr__(self, "times", tuple(float(x) for x in self.times))


@dataclass(frozen=True)
class ContinuousCallback:
    """ContinuousCallback(condition, affect!; save_positions = (false, false)) (test/Callbacks2/continuous_callbacks.jl): `condition` assigns `c` from `u`, `p`, `t`, `affect`
    edits `un` (a copy of `u`), both as device text — solve(..., callback=ContinuousCallback("c = u[0];", "un[1] = -p[1] * u[1];")) attaches them to the problem's
    DeviceFunction (DeviceFunction.set_continuous_callback; it stays attached) and solves with per-trajectory event detection (include/hipadj.h
    hipadj_model_set_continuous_callback).  `sol.engine.event_counts()` returns the events of each trajectory."""
    condition: str
    affect: str = None
    max_events: int = 0
    direction: int = 0       # +1: only upcrossings fire (affect_neg! = nothing), -1: only downcrossings, 0: both
    ncond: int = 1           # > 1: VectorContinuousCallback(condition, affect!, ncond) — `out[k]` in the condition, `idx` in the affect


@dataclass(frozen=True)
class LsqShift:
    """dgdu_discrete(out, u, p, t, i) = u - shift  (test/Core3/adjoint.jl:49-51: `out .= -2.0 .+ u`),
    evaluated inside the reverse kernel."""
    shift: float = 0.0


class LsqData:
    """dgdu_discrete(out, u, p, t, i) = scale * (u - data[:, i]) with the data block [N][M][n] resident on the device — scale = 2 is the gradient of
    `sum(abs2, sol .- data)`, the loss of the reference's tutorials (docs/src/Benchmark.md:80, docs/src/tutorials/parameter_estimation_ode.md:43).
    Evaluated inside the reverse kernels (HIPADJ_LOSS_LSQ_DATA); `value(sol)` = scale / 2 * sum |u - data|^2 from the device as well."""

    def __init__(self, data, scale=2.0):
        self.data = np.ascontiguousarray(data, dtype=np.float64)
        self.scale = float(scale)

    def __eq__(self, other):
        return isinstance(other, LsqData) and self.scale == other.scale and self.data.shape == other.data.shape and np.array_equal(self.data, other.data)

    def __hash__(self):
        return hash((self.scale, self.data.shape))

    def __repr__(self):
        return f"LsqData(data{self.data.shape}, scale={self.scale})"


class ModelLoss:
    """The discrete loss attached to a DeviceFunction with set_discrete_loss(...) — its dgdu_discrete / dgdp_discrete bodies run inside the reverse
    kernels at every loss time (HIPADJ_LOSS_MODEL; src/adjoint_common.jl:771-779).  `data` [N][M][n] (optional) is what the bodies see as `d`."""

    def __init__(self, data=None):
        self.data = None if data is None else np.ascontiguousarray(data, dtype=np.float64)

    def __eq__(self, other):
        return isinstance(other, ModelLoss) and ((self.data is None and other.data is None) or (self.data is not None and other.data is not None and np.array_equal(self.data, other.data)))

    def __hash__(self):
        return hash(("ModelLoss", None if self.data is None else self.data.shape))

    def __repr__(self):
        return "ModelLoss()" if self.data is None else f"ModelLoss(data{self.data.shape})"


@dataclass(frozen=True)
class HalfSquaredSum:
    """Continuous cost g(u, p, t) = (sum(u))^2 / 2 with dgdu_continuous = sum(u) in every component
    (the `g`/`dg` pair of test/Core3/adjoint.jl:913-919); evaluated inside the reverse kernels
    (accumulate_cost!, src/derivative_wrappers.jl:1411-1442)."""


@dataclass(frozen=True)
class FirstStateSquaredPlusFirstParam:
    """Continuous cost g(u, p, t) = u[1]^2 + p[1] with dgdu_continuous = [2 u1, 0, ...] and dgdp_continuous = [1, 0, ...]
    (test/Core7/mixed_costs.jl:46-57): the registered cost with a parameter term."""


@dataclass(frozen=True)
class ModelCost:
    """The continuous cost attached to a DeviceFunction with set_cost(dgdu, dgdp)."""


@dataclass
class EnsembleSolution:
    """What the reverse pass needs from the forward solve: the handle owning the device-resident interpolant
    tiles / checkpoints, plus the primal output at the save times."""
    engine: object
    u: np.ndarray                # [N][M][n] = sol(ts)
    t: np.ndarray                # [M]
    prob: object
    alg: object
    dt: float
    dense: bool = True
    retcode: str = "Success"
    extra: dict = field(default_factory=dict)

    def loss_value(self):
        """The loss of a device-resident discrete loss (LsqShift / LsqData / a ModelLoss given as the loss itself), summed over the ensemble, evaluated on the
        device from the saved states (include/hipadj.h hipadj_loss_value)."""
        if self.u is None:
            raise ValueError("loss_value needs the saved states (solve(..., want_out=True))")
        return self.engine.loss_value(self.u)

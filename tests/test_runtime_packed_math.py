"""Runtime models are compiled like the library itself: without the packed 32-bit arithmetic instructions, some forms of which have given wrong results on this hardware.  Read off the
code objects that are handed out (no device needed)."""
import ctypes as C
import glob
import os
import re
import subprocess

import pytest

import emu as E
from test_isa_lint import isa_lint

pytestmark = pytest.mark.skipif(not os.path.exists(isa_lint.OBJDUMP), reason="llvm-objdump of the ROCm toolchain not found")

# two states in 32-bit arithmetic, side by side: what the compiler packs when it may
F = "const float a = (float)u[0], b = (float)u[1], c = (float)p[0], d = (float)p[1]; const float q0 = a * c + b * 0.5f, q1 = b * c + a * 0.5f; du[0] = (double)(q0 * a + d); du[1] = (double)(q1 * b + d);"
VJP = ("const float a = (float)u[0], b = (float)u[1], c = (float)p[0], l = (float)lam[0], m = (float)lam[1];"
       "out[0] = (double)((2.0f * a * c + b * 0.5f) * l + 0.5f * b * m); out[1] = (double)(0.5f * a * l + (2.0f * b * c + a * 0.5f) * m);")
VJP_P = "const float a = (float)u[0], b = (float)u[1], l = (float)lam[0], m = (float)lam[1]; out[0] = (double)(a * a * l + b * b * m); out[1] = (double)(l + m);"


@pytest.mark.parametrize("stepper", [0, 1])
def test_runtime_models_have_no_packed_32_bit_arithmetic(sa, tmp_path, monkeypatch, stepper):
    from scimlsensitivity_jl_amd import _lib
    name = f"float_model_{stepper}"
    _lib.register_model(name, 2, 2, F, VJP, VJP_P)
    monkeypatch.setenv("HIPADJ_RTC_DUMP", str(tmp_path))
    cfg = E.make_config(name, "interpolating", 200, 0.0, 0.5, 0.0 if stepper else 0.01, [], loss_kind=1, stepper=stepper, abstol=1e-6, reltol=1e-6, checkpointing=False)
    L = _lib.load()
    assert L.hipadj_model_check_config(C.byref(cfg)) == _lib.OK, L.hipadj_last_error(None)
    objs = glob.glob(str(tmp_path / "*.hsaco"))
    assert objs
    for o in objs:
        text = subprocess.run([isa_lint.OBJDUMP, "-d", o], capture_output=True, text=True, check=True).stdout
        assert "v_fma" in text and not re.findall(r"v_pk_(?:add|mul|fma)_f32", text)

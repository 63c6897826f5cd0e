"""Errors of the HIP runtime around the operators (`-m gpu`): an earlier one of the host program is neither taken for the call's own nor taken away."""
import ctypes as C
import re

import pytest

pytestmark = pytest.mark.gpu


def runtime():
    """The HIP runtime that this process has loaded."""
    with open("/proc/self/maps") as f:
        paths = sorted(set(re.findall(r"(/\S*libamdhip64\.so\S*)", f.read())))
    assert len(paths) == 1, paths
    return C.CDLL(paths[0])


def test_a_pending_error_of_the_host_program_stays(sa):
    import torch
    hip = runtime()
    x = torch.randn(3, 200, 64, device="cuda")
    pool, small, large = torch.zeros(3, 64, device="cuda"), torch.randn(40, 50, device="cuda"), torch.randn(200, 150, device="cuda")
    def calls():
        yield "solve", lambda: sa.recurrence_solve(x, x, form="sigmoid").h
        yield "step", lambda: sa.gated_recurrence_step(x[:, 0], x[:, 0], pool.zero_(), form="sigmoid")
        yield "no rows", lambda: sa.recurrence_solve(x[:, :0], x[:, :0], pool.zero_()).h_final
        yield "small", lambda: sa.orthogonalized_update(small)
        yield "large", lambda: sa.orthogonalized_update(large)
    want = {name: call() for name, call in calls()}
    torch.cuda.synchronize()
    for name, call in calls():
        # the launches themselves, without torch's own calls between: torch reports a pending error as its next one's
        from scimlsensitivity_jl_amd import _lib
        L, seen = _lib.load(), []
        entries = ("hipadj_recurrence_forward_dev", "hipadj_recurrence_step_dev", "hipadj_orthogonalized_update_dev")

        class Wrapped:
            def __getattr__(self, entry):
                f = getattr(L, entry)
                if entry not in entries:
                    return f
                def g(*a):
                    assert hip.hipSetDevice(4096) == 101              # hipErrorInvalidDevice
                    pending = hip.hipPeekAtLastError()
                    rc = f(*a)
                    seen.append((pending, rc, hip.hipGetLastError()))
                    return rc
                return g
        with pytest.MonkeyPatch.context() as m:
            m.setattr(_lib, "load", lambda: Wrapped())
            got = call()
        torch.cuda.synchronize()
        assert seen and all(s == (101, 0, 101) for s in seen), (name, seen)
        assert torch.equal(got, want[name])

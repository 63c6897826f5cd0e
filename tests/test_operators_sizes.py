"""Sizes at the end of their type's range, where there is no device: refused, not taken for small ones after an overflow."""
import ctypes as C

import pytest

from test_operators_host import lib, recurrence                      # noqa: F401

MOST = 2 ** 63 - 1


@pytest.mark.parametrize("kw", [dict(batch=1, length=MOST), dict(batch=1, length=MOST - 62, channels=1), dict(batch=1, length=1, channels=MOST), dict(batch=1, length=1, channels=MOST - 61),
                                dict(batch=MOST, length=1, channels=1), dict(batch=1, nseq=3, offsets=256, offsets_bits=32, length=MOST)])
def test_recurrence_sizes_that_do_not_fit(lib, kw):                 # noqa: F811
    _lib, L = lib
    r = recurrence(_lib, device=1 << 20, **kw)
    ck, ws = C.c_int64(7), C.c_int64(7)
    assert L.hipadj_recurrence_sizes(C.byref(r), C.byref(ck), C.byref(ws)) == -6 and b"tiles" in L.hipadj_last_error(None) and (ck.value, ws.value) == (7, 7)
    assert L.hipadj_recurrence_forward_dev(C.byref(r), *[256] * 7, MOST, None) == -6
    assert L.hipadj_recurrence_adjoint_dev(C.byref(r), *[256] * 10, MOST, None) == -6


@pytest.mark.parametrize("kw", [dict(channels=MOST), dict(channels=MOST - 254), dict(batch=MOST, n=MOST), dict(batch=MOST, slots=256)])
def test_step_sizes_that_do_not_fit(lib, kw):                       # noqa: F811
    _lib, L = lib
    a = {**dict(device=1 << 20, dtype=1, gate_dtype=1, gate=1, coupled=0, batch=1, channels=4, x=256, xs=4, g=256, gs=4, st=256, ss=4, n=1, slots=None, bits=32, h=256, hs=4, stream=None), **kw}
    assert L.hipadj_recurrence_step_dev(*a.values()) == -6 and b"at most" in L.hipadj_last_error(None)

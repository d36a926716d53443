"""The check of pow that the driver asks can fail (CPU): the library's pow is held against the interpreter's, which is what the
reference's arithmetic runs on (memory.py:301,308,341-342,376-377)."""
import ctypes as C

import numpy as np
import pytest

from sam_tf_amd import _lib, ops


@pytest.fixture(autouse=True)
def _asked_anew(monkeypatch):
    monkeypatch.setattr(ops, '_POW_OK', None)


def test_this_machines_pow():
    assert ops.pow_matches_host(20000)


class _OtherPow(object):
    """The library with a pow that is one step of the last place off in one of the values it is asked for."""

    def __getattr__(self, name):
        f = getattr(_lib.lib(), name)
        if name != 'samx_pow_host':
            return f

        def wrong(x, y, n, out):
            rc = f(x, y, n, out)
            a = np.ctypeslib.as_array(C.cast(out, C.POINTER(C.c_double)), (n,))
            a[n // 2] = np.nextafter(a[n // 2], np.inf)
            return rc
        return wrong


def test_a_pow_with_another_last_bit(monkeypatch):
    monkeypatch.setattr(ops, '_L', _OtherPow)
    assert not ops.pow_matches_host(20000)


def test_selfcheck_counts():
    L = _lib.lib()
    assert L.samx_pow_selfcheck(1000) == 0 and L.samx_pow_selfcheck(0) == 0

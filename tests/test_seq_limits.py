"""Sizes at the limits of the sequence-policy entry points: what is refused (CPU)."""
import ctypes as C

import pytest

from sam_tf_amd import _lib
from tests.test_seq_refusals import P, _refused, _shape


@pytest.mark.parametrize('B', [1 << 62, (1 << 62) + 1, 1 << 32, (1 << 63) - 1])
def test_so_many_sequences_that_their_heads_are_no_64_bit_number(B):
    L = _lib.lib()
    s = _shape(B=B)
    _refused(L.samx_linattn(C.byref(s), P, P, P, P, 1.0, None, None, P, P, P, 1 << 40, None))
    _refused(L.samx_linattn_grad(C.byref(s), P, P, P, P, P, 1.0, None, None, None, P, P, P, P, P, 1 << 40, None))
    _refused(L.samx_linattn_step(C.byref(s), P, P, P, P, 1.0, P, P, None))
    assert L.samx_linattn_ws_bytes(C.byref(s)) == 0 and L.samx_linattn_grad_ws_bytes(C.byref(s)) == 0


def test_as_many_heads_as_the_launches_take():
    L = _lib.lib()
    for B, H, ok in ((16384, 4, True), (4096, 16, True), (32768, 4, True), (32769, 4, False), (131072, 1, True), (131073, 1, False)):
        s = _shape(B=B, H=H, HK=1)
        assert (L.samx_linattn_ws_bytes(C.byref(s)) > 0) == ok and (L.samx_linattn_grad_ws_bytes(C.byref(s)) > 0) == ok

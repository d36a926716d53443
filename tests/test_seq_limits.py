"""Sizes at the limits of the sequence-policy entry points: what is refused (CPU)."""
import ctypes as C
import os
import subprocess
import sys

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


def test_a_torch_without_its_private_stream_calls():
    """ops loads, and the sequence wrappers still refuse what is not on a GPU, where torch._C has neither of the names."""
    code = ('import torch\n'
            'for n in ("_cuda_getCurrentRawStream", "_cuda_getDevice"):\n'
            '    if hasattr(torch._C, n): delattr(torch._C, n)\n'
            'from sam_tf_amd import ops\n'
            'x, w = torch.zeros(4, 8), torch.ones(8)\n'
            'try: ops.block_norm(x, x, w, w)\n'
            'except TypeError as e: print("refused:", e)\n')
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, '-c', code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and 'refused: y must be a CUDA tensor' in r.stdout, r.stderr

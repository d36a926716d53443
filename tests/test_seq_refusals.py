"""What the sequence-policy entry points refuse before they touch a GPU (no GPU in this tier)."""
import ctypes as C
import math

import pytest
import torch

from sam_tf_amd import _lib, ops

ARG, WORKSPACE = -1, -3
P = C.c_void_p(0x1000)    # some address: a refused call does not look behind it


def _refused(rc, code=ARG, text=None):
    assert rc == code, _lib.lib().samx_last_error()
    if text:
        assert text in _lib.lib().samx_last_error().decode()


def _shape(**kw):
    s = _lib.LinattnShape(1, 4, 2, 32, 48, 0, 2, 100)
    s.q[:] = (100 * 128, 128, 32)
    s.k[:] = (100 * 64, 64, 32)
    s.v[:] = (100 * 96, 96, 48)
    s.o[:] = (100 * 192, 192, 48)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


BAD_SHAPES = [dict(dtype=3), dict(dtype=-1), dict(B=-1), dict(T=-1), dict(T=1 << 31), dict(H=0), dict(HK=0), dict(H=3),
              dict(D=0), dict(D=129), dict(DV=0), dict(DV=129), dict(B=40000)]


@pytest.mark.parametrize('bad', BAD_SHAPES)
def test_linattn_shapes(bad):
    L = _lib.lib()
    s = _shape(**bad)
    _refused(L.samx_linattn(C.byref(s), P, P, P, P, 1.0, None, None, P, P, P, 1 << 40, None))
    _refused(L.samx_linattn_grad(C.byref(s), P, P, P, P, P, 1.0, None, None, None, P, P, P, P, P, 1 << 40, None))
    _refused(L.samx_linattn_step(C.byref(s), P, P, P, P, 1.0, P, P, None))
    assert L.samx_linattn_ws_bytes(C.byref(s)) == 0 and L.samx_linattn_grad_ws_bytes(C.byref(s)) == 0


def test_linattn_pointers_scale_and_workspace():
    L = _lib.lib()
    s = _shape()
    for i in (0, 1, 2, 3, 6, 7):
        a = [P, P, P, P, 1.0, None, P, P]
        a = a[:4] + [1.0, None, None, P, P]
        at = {0: 0, 1: 1, 2: 2, 3: 3, 6: 7, 7: 8}[i]
        a[at] = None
        _refused(L.samx_linattn(C.byref(s), *a, P, 1 << 40, None), text='null')
    for x in (math.inf, math.nan):
        _refused(L.samx_linattn(C.byref(s), P, P, P, P, x, None, None, P, P, P, 1 << 40, None), text='scale')
        _refused(L.samx_linattn_step(C.byref(s), P, P, P, P, x, P, P, None), text='scale')
    _refused(L.samx_linattn(None, P, P, P, P, 1.0, None, None, P, P, P, 0, None), text='null')
    # shared heads need room for each head's part of the gradient
    _refused(L.samx_linattn_grad(C.byref(s), P, P, P, P, P, 1.0, None, None, None, P, P, P, P, P, 100, None), WORKSPACE)
    _refused(L.samx_linattn_grad(C.byref(s), P, P, P, P, P, 1.0, None, None, None, P, P, P, P, None, 1 << 40, None), WORKSPACE)
    odd = C.c_void_p(0x1008)
    _refused(L.samx_linattn_grad(C.byref(s), P, P, P, P, P, 1.0, None, None, None, P, P, P, P, odd, 1 << 40, None), text='aligned')
    _refused(L.samx_linattn(C.byref(_shape(T=5000)), P, P, P, P, 1.0, None, None, P, P, odd, 1 << 40, None), text='aligned')
    long = _shape(T=5000)
    assert L.samx_linattn_ws_bytes(C.byref(long)) > 4096
    _refused(L.samx_linattn(C.byref(long), P, P, P, P, 1.0, None, None, P, P, P, 16, None), WORKSPACE)


def test_nothing_to_do():
    L = _lib.lib()
    s = _shape(B=0)
    assert L.samx_linattn(C.byref(s), None, None, None, None, 1.0, None, None, None, None, None, 0, None) == 0
    assert L.samx_linattn_grad(C.byref(s), None, None, None, None, None, 1.0, None, None, None, None, None, None, None, None,
                               0, None) == 0
    assert L.samx_linattn_step(C.byref(s), None, None, None, None, 1.0, None, None, None) == 0
    assert L.samx_block_norm(None, None, 0, 0, 64, None, None, 0, None, None, None, 1.0, 0, 1e-6, None, None, None) == 0
    assert L.samx_distill_loss(None, 64, 0, 0, 64, None, None, 4, 1.0, None, None, None, None) == 0


def test_block_norm():
    L = _lib.lib()
    ok = dict(dtype=1, N=8, D=64, post_b=None, gate_kind=0, gate=None, pre_b=None, res=1.0, kind=0, eps=1e-6, x=P, u=P)

    def call(**kw):
        a = dict(ok, **kw)
        return L.samx_block_norm(a['x'], P, a['dtype'], a['N'], a['D'], P, a['post_b'], a['gate_kind'], a['gate'], P,
                                 a['pre_b'], a['res'], a['kind'], a['eps'], C.c_void_p(0x2000), a['u'], None)
    for bad in (dict(dtype=3), dict(N=-1), dict(D=0), dict(D=16385), dict(dtype=0, D=8193), dict(kind=2), dict(gate_kind=3),
                dict(gate_kind=-1), dict(res=math.inf), dict(eps=-1e-9), dict(eps=math.nan), dict(x=None), dict(u=None),
                dict(gate_kind=1), dict(gate_kind=2), dict(kind=1), dict(kind=1, post_b=P), dict(u=C.c_void_p(0x2000))):
        _refused(call(**bad))
    g = lambda **kw: L.samx_block_norm_grad(P, P, P, P, kw.get('dtype', 1), 8, 64, P, kw.get('post_b'), kw.get('gk', 0),
                                            kw.get('gate'), P, 1.0, kw.get('kind', 0), 1e-6, P, P, kw.get('dgate'), P,
                                            kw.get('dpost_b'), P, kw.get('dpre_b'), kw.get('ws', P), kw.get('n', 1 << 40), None)
    _refused(g(dtype=9))
    _refused(g(gk=1, gate=P), text='gate')
    _refused(g(kind=1, post_b=P, dpost_b=P), text='LayerNorm')
    _refused(g(ws=None))
    _refused(g(ws=C.c_void_p(0x1008)), text='aligned')
    _refused(g(n=64), WORKSPACE)
    assert L.samx_block_norm_grad_ws_bytes(1, 8, 0) == 0 and L.samx_block_norm_grad_ws_bytes(5, 8, 64) == 0


def test_distill():
    L = _lib.lib()

    def call(ld=64, dtype=1, N=8, V=64, K=4, tau=1.0, scale=1.0, ldg=64, grad=C.c_void_p(0x9000), z=P, idx=P, loss=P):
        return L.samx_distill_grad(z, ld, dtype, N, V, idx, P, K, tau, None, None, scale, loss, grad, ldg, None)
    for bad in (dict(ld=63), dict(ldg=63), dict(dtype=3), dict(N=-1), dict(V=0), dict(V=(1 << 31) - 64, ld=1 << 31, ldg=1 << 31),
                dict(K=0), dict(K=1025), dict(tau=0.0), dict(tau=-1.0), dict(tau=1e-7), dict(tau=math.nan), dict(tau=math.inf),
                dict(scale=math.nan), dict(grad=None), dict(z=None), dict(idx=None), dict(loss=None),
                dict(grad=P, ld=64, ldg=70)):
        _refused(call(**bad))


def test_tensors_have_to_be_on_a_gpu():
    x = torch.zeros(4, 8)
    w = torch.ones(8)
    with pytest.raises(TypeError):
        ops.block_norm(x, x, w, w)
    with pytest.raises(TypeError):
        ops.block_norm_grad(x, x, x, x, w, w)
    with pytest.raises(TypeError):
        ops.distill_loss(x, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))
    with pytest.raises(TypeError):
        ops.distill_grad(x, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))
    q = torch.zeros(1, 4, 2, 8)
    with pytest.raises(TypeError):
        ops.linattn(q, q, q, w[:2])
    with pytest.raises(TypeError):
        ops.linattn_grad(q, q, q, w[:2], q)
    with pytest.raises(TypeError):
        ops.linattn_step(q[:, 0], q[:, 0], q[:, 0], w[:2], torch.zeros(1, 2, 8, 8))


def test_reference_gradients_are_those_of_differentiation():
    """The plain forms that the GPU tests compare with, against automatic differentiation (float64)."""
    from tests import seq_ref as R
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    B, T, H, HK, D, DV = 2, 7, 4, 2, 3, 5
    leaf = [r(B, T, H, D), r(B, T, HK, D), r(B, T, HK, DV), r(B, H, D, DV)]
    decay, lengths, do, dS = -torch.rand(H, generator=g, dtype=torch.float64), torch.tensor([7, 4]), r(B, T, H, DV), r(B, H, D, DV)
    for t in leaf:
        t.requires_grad_(True)
    outs, states = [], []
    for b in range(B):
        S = leaf[3][b]
        row = []
        for t in range(int(lengths[b])):
            k, v = (leaf[i][b, t].repeat_interleave(H // HK, 0) for i in (1, 2))
            S = torch.exp(decay)[:, None, None] * S + k[:, :, None] * v[:, None, :]
            row.append(0.3 * (leaf[0][b, t][:, None, :] @ S)[:, 0])
        outs.append(row)
        states.append(S)
    loss = sum((o * do[b, t]).sum() for b, row in enumerate(outs) for t, o in enumerate(row)) + (torch.stack(states) * dS).sum()
    want = torch.autograd.grad(loss, leaf)
    with torch.no_grad():
        got = R.linattn_grad(leaf[0], leaf[1], leaf[2], decay, do, 0.3, leaf[3], dS, lengths)
        out, S = R.linattn(leaf[0], leaf[1], leaf[2], decay, 0.3, leaf[3], lengths)
    assert all(torch.allclose(a, b, rtol=1e-12, atol=1e-12) for a, b in zip(got, want))
    assert torch.allclose(S, torch.stack(states), rtol=1e-12) and bool((out[1, 4:] == 0).all())

    for kind in ('rms', 'layer'):
        for gate in (None, r(6), r(4, 6)):
            x, y, dh, du = r(4, 6), r(4, 6), r(4, 6), r(4, 6)
            p = dict(post_w=r(6), pre_w=r(6), post_b=r(6) if kind == 'layer' else None, pre_b=r(6) if kind == 'layer' else None)
            v = dict(x=x, y=y, gate=gate, **p)
            names = [n for n in v if v[n] is not None]
            for n in names:
                v[n].requires_grad_(True)
            h, u = R.block(v['x'], v['y'], v['post_w'], v['pre_w'], v['post_b'], v['pre_b'], v['gate'], 0.7, kind, 1e-5)
            want = dict(zip(names, torch.autograd.grad((h * dh).sum() + (u * du).sum(), [v[n] for n in names])))
            with torch.no_grad():
                got = R.block_grad(y, h, dh, du, v['post_w'], v['pre_w'], v['post_b'], v['pre_b'], v['gate'], 0.7, kind, 1e-5)
            assert all(torch.allclose(got[n], want[n], rtol=1e-10, atol=1e-12) for n in names)
            assert all(got[n] is None for n in got if n not in names)

    z, idx, t = r(3, 9), torch.tensor([[1, 4, 4], [0, -1, 9], [8, 2, 3]]), r(3, 3)
    w, lse = torch.rand(3, generator=g, dtype=torch.float64), torch.logsumexp(t / 2, 1) + 0.3
    z.requires_grad_(True)
    logq = torch.log_softmax(z / 2, 1)
    loss = 0.0
    for i in range(3):
        for k in range(3):
            if 0 <= int(idx[i, k]) < 9:
                x = t[i, k] / 2 - lse[i]
                loss = loss + w[i] * x.exp() * (x - logq[i, idx[i, k]])
    want, = torch.autograd.grad(0.4 * loss, z)
    with torch.no_grad():
        ls, got, _ = R.distill(z, idx, t, 2.0, lse, w, 0.4)
    assert torch.allclose(got, want, rtol=1e-12, atol=1e-14) and torch.allclose(ls.sum(), loss.detach(), rtol=1e-12)

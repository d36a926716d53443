"""The sequence-policy operators in one run, as a policy that reads trajectories uses them: projection, linear attention, the
norms around the block, a head, imitation of a teacher's top logits, and all the way back."""
import math

import pytest
import torch

from tests import seq_ref as R

pytestmark = pytest.mark.gpu

B, T, OBS, H, HK, D, DV, C, V, K = 3, 70, 11, 4, 2, 16, 24, 48, 18, 4
WIDTH = H * D + HK * D + HK * DV      # q, k and v of one joint projection
LENGTHS = [70, 1, 37]
SCALE, RES, EPS, TAU = D ** -0.5, 0.8, 1e-6, 1.5


def _problem(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    p = dict(Wx=r(OBS, C) / OBS ** 0.5, Wj=r(C, WIDTH) / C ** 0.5, Wo=r(H * DV, C) / (H * DV) ** 0.5, Wh=r(C, V) / C ** 0.5,
             post_w=1 + 0.2 * r(C), post_b=0.1 * r(C), pre_w=1 + 0.2 * r(C), pre_b=0.1 * r(C), gate=1 + 0.3 * r(C))
    live = (torch.arange(T)[None] < torch.tensor(LENGTHS)[:, None]).reshape(-1)
    d = dict(obs=r(B * T, OBS), decay=-torch.rand(H, generator=g) * 0.3, S0=0.3 * r(B, H, D, DV),
             idx=torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(B * T)]).to(torch.int32),
             t=2 * r(B * T, K), weight=live.float() / live.sum())
    return p, d


def _linear(x, w, tx=False, tw=False):
    """x w with the framework's own product; tx, tw: of the transpose."""
    from sam_tf_amd import ops
    x, w = x.contiguous(), w.contiguous()
    (R_, M), (M2, N) = (x.shape[::-1] if tx else x.shape), (w.shape[::-1] if tw else w.shape)
    assert M == M2
    return ops.gemm_f32(x, (1, x.shape[1]) if tx else (x.shape[1], 1), w, (1, w.shape[1]) if tw else (w.shape[1], 1), R_, N, M)


def _views(j):
    j = j.view(B, T, WIDTH)
    a, b = H * D, H * D + HK * D
    return j[..., :a].unflatten(-1, (H, D)), j[..., a:b].unflatten(-1, (HK, D)), j[..., b:].unflatten(-1, (HK, DV))


def _own(p, d, lengths):
    """(loss of each row, logits, the state behind, every gradient) by the framework's kernels."""
    from sam_tf_amd import ops
    x = _linear(d['obs'], p['Wx'])
    j = _linear(x, p['Wj'])
    q, k, v = _views(j)
    o, S = ops.linattn(q, k, v, d['decay'], SCALE, d['S0'], lengths)
    y = _linear(o.view(B * T, H * DV), p['Wo'])
    norm = dict(post_b=p['post_b'], pre_b=p['pre_b'], gate=p['gate'], res_scale=RES, kind='layer', eps=EPS)
    h, u = ops.block_norm(x, y, p['post_w'], p['pre_w'], **norm)
    z = _linear(u, p['Wh'])
    loss, dz = ops.distill_grad(z, d['idx'], d['t'], tau=TAU, weight=d['weight'])
    g = dict(Wh=_linear(u, dz, tx=True))
    b = ops.block_norm_grad(y, h, torch.zeros_like(h), _linear(dz, p['Wh'], tw=True), p['post_w'], p['pre_w'], **norm)
    g.update((n, b[n]) for n in ('post_w', 'post_b', 'pre_w', 'pre_b', 'gate'))
    g['Wo'] = _linear(o.view(B * T, H * DV), b['y'], tx=True)
    do = _linear(b['y'], p['Wo'], tw=True).view(B, T, H, DV)
    dq, dk, dv, g['S0'] = ops.linattn_grad(q, k, v, d['decay'], do, SCALE, d['S0'], None, lengths)
    dj = torch.cat([t.reshape(B * T, -1) for t in (dq, dk, dv)], 1)
    g['Wj'] = _linear(x, dj, tx=True)
    dx = b['x'] + _linear(dj, p['Wj'], tw=True)
    g['Wx'] = _linear(d['obs'], dx, tx=True)
    return loss, z, S, g


def _plain(p, d):
    """The same in float64 with the plain forms: (loss of each row, logits, state)."""
    x = d['obs'] @ p['Wx']
    q, k, v = _views(x @ p['Wj'])
    out, S = [], []
    for b, n in enumerate(LENGTHS):
        s, row = d['S0'][b], []
        for t in range(T):
            if t < n:
                s = torch.exp(d['decay'])[:, None, None] * s + (k[b, t][:, :, None] * v[b, t][:, None, :]).repeat_interleave(H // HK, 0)
                row.append(SCALE * (q[b, t][:, None, :] @ s)[:, 0])
            else:
                row.append(torch.zeros(H, DV, dtype=torch.float64))
        out.append(torch.stack(row))
        S.append(s)
    y = torch.stack(out).reshape(B * T, H * DV) @ p['Wo']
    h, u = R.block(x, y, p['post_w'], p['pre_w'], p['post_b'], p['pre_b'], p['gate'], RES, 'layer', EPS)
    z = u @ p['Wh']
    logp = torch.log_softmax(d['t'] / TAU, 1)
    logq = torch.log_softmax(z / TAU, 1).gather(1, d['idx'].long())
    return d['weight'] * (logp.exp() * (logp - logq)).sum(1), z, torch.stack(S)


def _gpu(t):
    return {n: x.cuda() for n, x in t.items()}


# Every stage is a product or a sum of at most B T = 210 terms behind a factor that does not enlarge its input's relative
# error more than fourfold (weights of norm about 1, norms of rows with a spread of about 1, a softmax): 14 stages there and
# back, 256 U32 and 4 each, are 14 * 4 * 256 * 2^-24 = 8.5e-4 of a gradient's norm.
CLOSE = 1e-3


def _near(a, b, what):
    a, b = a.detach().cpu().double(), b.detach().double()
    assert a.shape == b.shape and bool(torch.isfinite(a).all()), what
    off = float((a - b).norm() / b.norm())
    assert off < CLOSE, '%s is off by %.2g of its norm' % (what, off)


def test_training_step():
    p, d = _problem()
    loss, z, S, g = _own(_gpu(p), _gpu(d), torch.tensor(LENGTHS, dtype=torch.int32, device='cuda'))
    q = {n: x.double().requires_grad_(True) for n, x in p.items()}
    e = {n: x.double() for n, x in d.items()}
    e['S0'].requires_grad_(True)
    wl, wz, wS = _plain(q, e)
    leaves = dict(q, S0=e['S0'])
    want = dict(zip(leaves, torch.autograd.grad(wl.sum(), list(leaves.values()))))
    _near(loss, wl, 'loss')
    _near(z, wz, 'logits')
    _near(S, wS, 'state')
    assert set(g) == set(want)
    for n in want:
        _near(g[n], want[n], n)


def test_gradient_against_differences():
    p, d = _problem(1)
    g = _own(_gpu(p), _gpu(d), torch.tensor(LENGTHS, dtype=torch.int32, device='cuda'))[3]
    gen = torch.Generator().manual_seed(2)
    p64, d64 = {n: x.double() for n, x in p.items()}, {n: x.double() for n, x in d.items()}
    step = 1e-4          # its square is what the quotient loses of a loss whose third differences are about 1
    for n in list(p) + ['S0']:
        way = torch.randn(g[n].shape, generator=gen).double()
        way /= way.norm()
        at = []
        for s in (step, -step):
            if n == 'S0':
                at.append(float(_plain(p64, dict(d64, S0=d64['S0'] + s * way))[0].sum()))
            else:
                at.append(float(_plain(dict(p64, **{n: p64[n] + s * way}), d64)[0].sum()))
        slope = (at[0] - at[1]) / (2 * step)
        own = g[n].cpu().double()
        assert abs(slope - float((own * way).sum())) < CLOSE * float(own.norm()) + 1e-6, n


def test_acting_is_reading():
    """Row by row with the recurrent step, the same logits and the same state as over the whole trajectory."""
    from sam_tf_amd import ops
    p, d = _problem(3)
    P, E = _gpu(p), _gpu(d)
    z, S = _own(P, E, None)[1:3]
    state = E['S0'].clone()
    obs = E['obs'].view(B, T, OBS)
    for t in range(T):
        x = _linear(obs[:, t], P['Wx'])
        j = _linear(x, P['Wj'])
        a, b = H * D, H * D + HK * D
        o = ops.linattn_step(j[:, :a].unflatten(-1, (H, D)), j[:, a:b].unflatten(-1, (HK, D)),
                             j[:, b:].unflatten(-1, (HK, DV)), E['decay'], state, SCALE)
        u = ops.block_norm(x, _linear(o.view(B, H * DV), P['Wo']), P['post_w'], P['pre_w'], post_b=P['post_b'],
                           pre_b=P['pre_b'], gate=P['gate'], res_scale=RES, kind='layer', eps=EPS)[1]
        _near(_linear(u, P['Wh']), z.view(B, T, V)[:, t].cpu(), 'row %d' % t)
    _near(state, S.cpu(), 'state')


def test_captured_step():
    """The whole training step in a graph, replayed with new inputs and other work between the replays."""
    p, d = _problem(4)
    P, E = _gpu(p), _gpu(d)
    lengths = torch.tensor(LENGTHS, dtype=torch.int32, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _own(P, E, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, z, S, g = _own(P, E, lengths)
    for seed in range(5, 9):
        p2, d2 = _problem(seed)
        for n in P:
            P[n].copy_(p2[n])
        for n in E:
            E[n].copy_(d2[n])
        lengths.copy_(torch.tensor([(seed * 13) % (T + 1), T, 0], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [loss.clone(), z.clone(), S.clone()] + [g[n].clone() for n in sorted(g)]
        el, ez, eS, eg = _own(P, E, lengths)
        for a, b in zip(got, [el, ez, eS] + [eg[n] for n in sorted(eg)]):
            assert torch.equal(a, b)

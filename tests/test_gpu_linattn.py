"""samx_linattn, its gradient and its step against the float64 recurrence (tests/seq_ref.py)."""
import math

import pytest
import torch

from tests import seq_ref as R
from tests.seq_ref import U32, half_step, smallest, within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _case(B, T, H, HK, D, DV, dtype, seed=0, state=True, lengths=None, decay=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    c = dict(q=r(B, T, H, D), k=r(B, T, HK, D), v=r(B, T, HK, DV), dout=r(B, T, H, DV))
    c = {n: t.to(dtype) for n, t in c.items()}
    c['decay'] = -torch.exp2(-(8.0 * torch.arange(H) / H)) if decay is None else torch.tensor(decay)
    c['state'] = r(B, H, D, DV) if state else None
    c['dstate'] = r(B, H, D, DV) if state else None
    c['lengths'] = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return c


def _gpu(c):
    return {n: None if t is None else t.cuda() for n, t in c.items()}


def _d(c):
    return {n: t if t is None or n == 'lengths' else t.double() for n, t in c.items()}


def _abs(c):
    return {n: t if t is None or n in ('lengths', 'decay') else t.abs() for n, t in c.items()}


def _errors(dtype, T, D, DV):
    """(relative to the sum of magnitudes: of an output, of a state).  float32: dot products of D or DV terms and of a
    chunk's 64 (their roundings at most one for each), four for each chunk that a state goes through, and the powers: l^n
    has 2 U32 and its argument U32 |g n| (|g n| l^n is below 1, and at most two powers meet a term), 64 together.  16-bit
    types: the scores' and the state's rounding where they meet the values (half a step each), and the second half of a
    split number's (half a step squared)."""
    f = (max(D, DV) + 64 + 4 * (T // 64 + 1) + 64) * U32
    if dtype == F32:
        return f, f
    h = half_step(dtype)
    return f + 2.1 * h, f + 1.1 * h * h


def _check(c, scale, dtype, grad=True, what=''):
    from sam_tf_amd import ops
    g, d = _gpu(c), _d(c)
    B, T, H, D = c['q'].shape
    DV = c['v'].shape[3]
    eo, es = _errors(dtype, T, D, DV)
    h = 1.01 * half_step(dtype)
    tiny = smallest(dtype)
    # half precision's second halves may be below its normal range: so much for each row and key
    low = (T + 1) * smallest(dtype) * 2 * max(float(t.double().abs().max()) if t.numel() else 0.0 for t in (c['q'], c['k'], c['v'], c['dout']))
    a = _abs(d)
    out, S = ops.linattn(g['q'], g['k'], g['v'], g['decay'], scale=scale, state=g['state'], lengths=g['lengths'])
    wo, wS = R.linattn(d['q'], d['k'], d['v'], d['decay'], scale, d['state'], d['lengths'])
    mo, mS = R.linattn(a['q'], a['k'], a['v'], d['decay'], scale, a['state'], d['lengths'])
    within(out, wo, eo * mo + h * wo.abs() + tiny + low, what + ' out')
    within(S, wS, es * mS + low, what + ' state')
    if not grad:
        return
    got = ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], scale=scale, state=g['state'],
                           dstate=g['dstate'], lengths=g['lengths'])
    args = lambda x: (x['q'], x['k'], x['v'], d['decay'], x['dout'], scale, x['state'], x['dstate'], d['lengths'])
    want, size = R.linattn_grad(*args(d)), R.linattn_grad(*args(a))
    for n, x, w, m in zip(('dq', 'dk', 'dv'), got, want, size):
        within(x, w, (eo + (H + 2) * U32) * m + h * w.abs() + tiny + low * D, what + ' ' + n)
    within(got[3], want[3], es * size[3] + low, what + ' dstate')


SHAPES = [  # B, T, H, HK, D, DV
    (1, 1, 1, 1, 1, 1), (2, 2, 2, 1, 8, 8), (1, 3, 3, 3, 16, 5), (2, 63, 2, 2, 33, 64), (1, 64, 2, 2, 64, 64),
    (3, 65, 1, 1, 64, 17), (1, 129, 4, 2, 72, 88), (2, 100, 2, 2, 128, 128), (1, 200, 3, 1, 127, 66)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('shape', SHAPES)
def test_shapes(shape, dtype):
    B, T, H, HK, D, DV = shape
    for state in (True, False):
        _check(_case(B, T, H, HK, D, DV, dtype, seed=T, state=state), D ** -0.5, dtype, what='state %s' % state)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('T,D', [(512, 32), (777, 40), (1300, 128)])
def test_time_in_segments(T, D, dtype):
    """Few heads and many rows: the segments, their joined states, lengths that end in any of them."""
    _check(_case(1, T, 2, 2, D, D, dtype, seed=1), D ** -0.5, dtype, what='whole')
    _check(_case(3, T, 2, 1, D, 24, dtype, seed=2, lengths=[T // 3, T, T // 2 + 1]), D ** -0.5, dtype, what='ragged')


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_lengths(dtype):
    T = 150
    c = _case(9, T, 2, 2, 24, 40, dtype, seed=3, lengths=[0, 1, 63, 64, 65, 128, 149, 150, 1000])
    _check(c, 0.3, dtype)
    c = _case(2, T, 2, 2, 24, 40, dtype, seed=4, lengths=[-3, 5], state=False)
    _check(c, 0.3, dtype)


def test_rows_behind_the_end_are_not_read():
    from sam_tf_amd import ops
    c = _case(2, 700, 2, 2, 64, 64, BF16, seed=5, lengths=[300, 70])
    g = _gpu(c)
    kw = dict(scale=0.125, state=g['state'], lengths=g['lengths'])
    one = ops.linattn(g['q'], g['k'], g['v'], g['decay'], **kw) + \
        ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], dstate=g['dstate'], **kw)
    for n in ('q', 'k', 'v', 'dout'):
        for b, e in enumerate((300, 70)):
            g[n][b, e:] = float('nan')
    two = ops.linattn(g['q'], g['k'], g['v'], g['decay'], **kw) + \
        ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], dstate=g['dstate'], **kw)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    assert all(bool((t[1, 70:] == 0).all()) for i, t in enumerate(two) if t.dim() == 4 and t.shape[1] == 700)


def test_no_rows_and_no_sequences():
    from sam_tf_amd import ops
    g = _gpu(_case(2, 0, 2, 2, 16, 24, BF16))
    out, S = ops.linattn(g['q'], g['k'], g['v'], g['decay'], state=g['state'])
    assert out.shape == (2, 0, 2, 24) and torch.equal(S, g['state'])
    *_, dS = ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], state=g['state'], dstate=g['dstate'])
    assert torch.equal(dS, g['dstate'])
    g = _gpu(_case(0, 9, 2, 2, 16, 24, BF16))
    assert ops.linattn(g['q'], g['k'], g['v'], g['decay'])[0].shape == (0, 9, 2, 24)
    assert ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'])[1].shape == (0, 9, 2, 16)


@pytest.mark.parametrize('decay', [[0.0, -math.inf], [-100.0, -1e-7], [-0.5, -20.0]])
def test_decays(decay):
    """No decay at all, no memory, and what is next to them."""
    _check(_case(2, 190, 2, 2, 20, 20, F32, decay=decay), 1.0, F32)
    _check(_case(1, 600, 2, 2, 20, 20, BF16, decay=decay), 1.0, BF16)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_strides(dtype):
    """Views of one projection, of odd widths and at odd places; heads before rows; sequences that share one."""
    from sam_tf_amd import ops
    B, T, H, D, DV = 2, 90, 3, 21, 35
    c = _case(B, T, H, H, D, DV, dtype, seed=6)
    g = _gpu(c)
    kw = dict(scale=0.2, state=g['state'])
    want = ops.linattn(g['q'], g['k'], g['v'], g['decay'], **kw) + \
        ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], dstate=g['dstate'], **kw)
    row = torch.zeros(B, T, 1 + H * (2 * D + 2 * DV), dtype=dtype, device='cuda')
    at, v = 1, {}
    for n in ('q', 'k', 'v', 'dout'):
        w = g[n].shape[-1]
        v[n] = row[..., at:at + H * w].unflatten(-1, (H, w))
        v[n].copy_(g[n])
        at += H * w
    got = ops.linattn(v['q'], v['k'], v['v'], g['decay'], **kw) + \
        ops.linattn_grad(v['q'], v['k'], v['v'], g['decay'], v['dout'], dstate=g['dstate'], **kw)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    t = {n: g[n].transpose(1, 2).contiguous().transpose(1, 2) for n in v}
    got = ops.linattn(t['q'], t['k'], t['v'], g['decay'], **kw) + \
        ops.linattn_grad(t['q'], t['k'], t['v'], g['decay'], t['dout'], dstate=g['dstate'], **kw)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    k = g['k'][:1].expand(B, T, H, D)
    got = ops.linattn(g['q'], k, g['v'], g['decay'], **kw)
    want = ops.linattn(g['q'], k.contiguous(), g['v'], g['decay'], **kw)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('B,H,HK,D,DV', [(1, 1, 1, 1, 1), (3, 4, 2, 24, 7), (2, 3, 3, 128, 128), (70, 2, 1, 65, 34), (1, 8, 8, 64, 64)])
def test_step(B, H, HK, D, DV, dtype):
    """Four steps in place; float32 throughout: D terms, one more rounding a step, and the output's own."""
    from sam_tf_amd import ops
    c = _case(B, 4, H, HK, D, DV, dtype, seed=7)
    g, d = _gpu(c), _d(c)
    S = g['state'].clone()
    e = (D + 16 + 4 * 4) * U32
    for t in range(4):
        o = ops.linattn_step(g['q'][:, t], g['k'][:, t], g['v'][:, t], g['decay'], S, scale=0.3)
        part = lambda x: (x['q'][:, :t + 1], x['k'][:, :t + 1], x['v'][:, :t + 1], d['decay'], 0.3, x['state'], None)
        wo, wS = R.linattn(*part(d))
        mo, mS = R.linattn(*part(_abs(d)))
        within(o, wo[:, t], e * mo[:, t] + 1.01 * half_step(dtype) * wo[:, t].abs() + smallest(dtype), 'out')
        within(S, wS, e * mS, 'state')


def test_steps_are_the_rows_of_the_whole():
    """Acting row by row and reading the trajectory give one state (float32: within both their errors)."""
    from sam_tf_amd import ops
    c = _case(2, 130, 2, 2, 48, 48, F32, seed=8)
    g = _gpu(c)
    out, S = ops.linattn(g['q'], g['k'], g['v'], g['decay'], scale=0.2, state=g['state'])
    s = g['state'].clone()
    rows = [ops.linattn_step(g['q'][:, t], g['k'][:, t], g['v'][:, t], g['decay'], s, scale=0.2) for t in range(130)]
    a = _abs(_d(c))
    mo, mS = R.linattn(a['q'], a['k'], a['v'], a['decay'], 0.2, a['state'], None)
    e = _errors(F32, 130, 48, 48)[0] + (48 + 16 + 4 * 130) * U32
    within(torch.stack(rows, 1), out, e * mo, 'out')
    within(s, S, e * mS, 'state')


def test_pieces_carry_the_state():
    """A trajectory in three calls, and its gradient in three calls backwards."""
    from sam_tf_amd import ops
    c = _case(2, 210, 2, 1, 32, 48, F32, seed=9)
    g = _gpu(c)
    cuts = [0, 70, 71, 210]
    s, states, outs = g['state'], [], []
    for a, b in zip(cuts, cuts[1:]):
        states.append(s)
        o, s = ops.linattn(g['q'][:, a:b], g['k'][:, a:b], g['v'][:, a:b], g['decay'], scale=0.2, state=s)
        outs.append(o)
    d = _d(c)
    wo, wS = R.linattn(d['q'], d['k'], d['v'], d['decay'], 0.2, d['state'], None)
    m = _abs(d)
    mo, mS = R.linattn(m['q'], m['k'], m['v'], d['decay'], 0.2, m['state'], None)
    e = 2 * _errors(F32, 210, 32, 48)[0]
    within(torch.cat(outs, 1), wo, e * mo, 'out')
    within(s, wS, e * mS, 'state')
    ds, parts = g['dstate'], []
    for i in reversed(range(3)):
        a, b = cuts[i], cuts[i + 1]
        *p, ds = ops.linattn_grad(g['q'][:, a:b], g['k'][:, a:b], g['v'][:, a:b], g['decay'], g['dout'][:, a:b], scale=0.2,
                                  state=states[i], dstate=ds)
        parts.insert(0, p)
    want = R.linattn_grad(d['q'], d['k'], d['v'], d['decay'], d['dout'], 0.2, d['state'], d['dstate'], None)
    size = R.linattn_grad(m['q'], m['k'], m['v'], d['decay'], m['dout'], 0.2, m['state'], m['dstate'], None)
    for j, n in enumerate(('dq', 'dk', 'dv')):
        within(torch.cat([p[j] for p in parts], 1), want[j], e * size[j], n)
    within(ds, want[3], e * size[3], 'dstate')


def test_gradient_against_differences():
    """The loss is linear in each of q, k, v and the state: central differences are exact but for rounding, U32 times the
    outputs' magnitudes over the step."""
    from sam_tf_amd import ops
    c = _gpu(_case(2, 75, 2, 1, 12, 20, F32, seed=10))

    def loss(x):
        o, S = ops.linattn(x['q'], x['k'], x['v'], x['decay'], scale=0.3, state=x['state'])
        return float((o.double() * x['dout'].double()).sum() + (S.double() * x['dstate'].double()).sum())
    got = ops.linattn_grad(c['q'], c['k'], c['v'], c['decay'], c['dout'], scale=0.3, state=c['state'], dstate=c['dstate'])
    gen = torch.Generator().manual_seed(0)
    for n, x in zip(('q', 'k', 'v', 'state'), got):
        d = torch.randn(x.shape, generator=gen).cuda()
        up, down = (loss(dict(c, **{n: c[n] + s * d})) for s in (1.0, -1.0))
        want = float((x.double() * d.double()).sum())
        size = float((x.double().abs() * d.double().abs()).sum())
        assert abs((up - down) / 2 - want) < 1e-4 * size, n


def test_same_twice_and_many_heads():
    from sam_tf_amd import ops
    g = _gpu(_case(40, 70, 16, 4, 32, 32, BF16, seed=11))
    kw = dict(scale=0.2, state=g['state'])
    a = ops.linattn(g['q'], g['k'], g['v'], g['decay'], **kw) + \
        ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], dstate=g['dstate'], **kw)
    b = ops.linattn(g['q'], g['k'], g['v'], g['decay'], **kw) + \
        ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], dstate=g['dstate'], **kw)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = {n: t if t is None or n == 'decay' else t[17:18].contiguous() for n, t in g.items()}
    o, S = ops.linattn(one['q'], one['k'], one['v'], one['decay'], scale=0.2, state=one['state'])
    assert torch.equal(o[0], a[0][17]) and torch.equal(S[0], a[1][17])


def test_captured_and_replayed():
    from sam_tf_amd import ops
    g = _gpu(_case(2, 600, 2, 1, 64, 64, BF16, seed=12, lengths=[600, 333]))
    kw = dict(scale=0.125, state=g['state'], lengths=g['lengths'])
    acting = g['state'].clone()

    def step():
        r = list(ops.linattn(g['q'], g['k'], g['v'], g['decay'], **kw))
        r += ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], dstate=g['dstate'], **kw)
        r.append(ops.linattn_step(g['q'][:, 0], g['k'][:, 0], g['v'][:, 0], g['decay'], acting))
        return r
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for n in ('q', 'k', 'v', 'dout'):
            g[n].copy_(torch.randn(g[n].shape, generator=torch.Generator().manual_seed(9 * i + len(n))))
        g['lengths'].copy_(torch.tensor([600 - 130 * i, 70 * i], dtype=torch.int32))
        start = g['state'] * (i + 1)
        acting.copy_(start)
        want = step()
        s = acting.clone()
        acting.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(s, acting)


@pytest.mark.parametrize('what', ['q', 'k', 'v', 'dout'])
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('dtype,D,DV', [(F32, 24, 40), (BF16, 40, 24), (F16, 64, 64), (BF16, 128, 128), (F32, 100, 128)])
def test_what_is_not_finite_stays_with_its_rows(dtype, D, DV, bad, what):
    """Row 75 of sequence 1, key head 0 or query head 1: rows and heads that do not meet it are as they were: bit for bit
    outside of its chunk, in it the same products in another order (each order within _errors of the sum of magnitudes,
    rounded once each)."""
    from sam_tf_amd import ops
    B, T, H, HK, at = 2, 150, 4, 2, 75
    c0 = _case(B, T, H, HK, D, DV, dtype, seed=5)
    a = _abs(_d(c0))
    most = (R.linattn(a['q'], a['k'], a['v'], a['decay'], 0.5, a['state'], None)[0],) + R.linattn_grad(
        a['q'], a['k'], a['v'], a['decay'], a['dout'], 0.5, a['state'], a['dstate'], None)[:3]
    e, h = _errors(dtype, T, D, DV)[0], 1.01 * half_step(dtype)
    c = _gpu(c0)
    run = lambda: (ops.linattn(c['q'], c['k'], c['v'], c['decay'], 0.5, c['state']) +
                   ops.linattn_grad(c['q'], c['k'], c['v'], c['decay'], c['dout'], 0.5, c['state'], c['dstate']))
    want = run()
    head = 1 if what in ('q', 'dout') else 0
    c[what][1, at, head, 3] = bad
    got = run()
    heads = [1] if what in ('q', 'dout') else [0, 1]               # query heads that meet it
    behind, upto, only, none = slice(at, None), slice(None, at + 1), slice(at, at + 1), slice(0, 0)
    # rows of (out, dq, dk, dv) that may change, and whether the state behind and the gradient of the one before may
    rows, ends = {'q': ((only, none, upto, upto), (False, True)), 'dout': ((none, only, upto, upto), (False, True)),
                  'k': ((behind, behind, none, only), (True, False)), 'v': ((behind, behind, only, none), (True, False))}[what]
    for x, w, r, m, name in zip((got[0], got[2], got[3], got[4]), (want[0], want[2], want[3], want[4]), rows, most, ('out', 'dq', 'dk', 'dv')):
        touched = torch.zeros(x.shape[:3], dtype=torch.bool, device='cuda')
        for h in heads if name in ('out', 'dq') else sorted({h * HK // H for h in heads}):
            touched[1, r, h] = True
        same = ~touched.cpu()
        within(x.cpu()[same], w.cpu()[same], (2 * e * m + 2 * h * w.cpu().double().abs() + 2 * smallest(dtype))[same], name)
        assert torch.equal(x[0], w[0]), name
        far = slice(0, 64) if name in ('out', 'dq') else slice(T - 64, T)       # chunks are counted from either end
        if not bool(touched[1, far].any()):
            assert torch.equal(x[1, far], w[1, far]), name
        if bool(touched.any()):
            assert not bool(torch.isfinite(x[touched]).all(-1).any()), name
    for x, w, may in ((got[1], want[1], ends[0]), (got[5], want[5], ends[1])):
        touched = torch.zeros(x.shape[:2], dtype=torch.bool, device='cuda')
        touched[1, heads] = may
        assert torch.equal(x[~touched], w[~touched])
        if may:
            assert not bool(torch.isfinite(x[touched].flatten(1)).all(-1).any())


@pytest.mark.parametrize('dtype,D,DV', [(BF16, 72, 100), (F16, 128, 128), (BF16, 40, 88), (F16, 96, 61), (F32, 72, 100), (F32, 128, 33)])
def test_more_heads_than_units(dtype, D, DV):
    """Enough of them that a workgroup has all columns of a head (fewer: two workgroups share them)."""
    _check(_case(66, 66, 4, 2, D, DV, dtype, seed=9, lengths=[(7 * b) % 67 for b in range(66)]), 0.5, dtype)


@pytest.mark.parametrize('dtype,D,DV', [(BF16, 128, 128), (BF16, 100, 61), (F16, 72, 120), (BF16, 128, 40), (F16, 24, 128), (F32, 100, 72),
                                        (F32, 65, 127)])
def test_two_workgroups_of_a_head(dtype, D, DV):
    """Few heads of more than 64 columns: ragged, of no rows, with and without a state, in segments."""
    _check(_case(6, 150, 2, 1, D, DV, dtype, seed=6, lengths=[0, 1, 64, 65, 128, 150]), 0.3, dtype)
    _check(_case(2, 20, 2, 2, D, DV, dtype, seed=7, lengths=[0, 20], state=False), 0.3, dtype)
    _check(_case(1, 700, 2, 2, D, DV, dtype, seed=8), 0.1, dtype)


def test_two_streams_at_once():
    """Calls that overlap on two streams, each with its own workspace, and one after the other: the same numbers."""
    from sam_tf_amd import ops
    cs = [_gpu(_case(2, 1500, 3, 3, 128, 128, BF16, seed=s)) for s in (20, 21)]
    run = lambda c: (ops.linattn(c['q'], c['k'], c['v'], c['decay'], 0.1, c['state']) +
                     ops.linattn_grad(c['q'], c['k'], c['v'], c['decay'], c['dout'], 0.1, c['state'], c['dstate']))
    want = [run(c) for c in cs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for c, st in zip(cs, streams):
            with torch.cuda.stream(st):
                got.append(run(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_rows_far_apart():
    """Rows 2^31 bytes from each other: offsets of 64 bits, and the same numbers."""
    from sam_tf_amd import ops
    B, T, H, D, DV = 1, 3, 2, 16, 24
    c = _gpu(_case(B, T, H, H, D, DV, BF16))
    want = ops.linattn(c['q'], c['k'], c['v'], c['decay'], 0.5, c['state'])
    gwant = ops.linattn_grad(c['q'], c['k'], c['v'], c['decay'], c['dout'], 0.5, c['state'], c['dstate'])
    step = 2 ** 30
    room = torch.empty((T - 1) * step + 1024, dtype=BF16, device='cuda')
    far, at = {}, 0
    for n in ('q', 'k', 'v', 'dout'):
        d = c[n].shape[-1]
        far[n] = room.as_strided((B, T, H, d), (T * step, step, d, 1), at)
        far[n].copy_(c[n])
        at += H * d
    got = ops.linattn(far['q'], far['k'], far['v'], c['decay'], 0.5, c['state'])
    ggot = ops.linattn_grad(far['q'], far['k'], far['v'], c['decay'], far['dout'], 0.5, c['state'], c['dstate'])
    assert all(torch.equal(a, b) for a, b in zip(want + gwant, got + ggot))


def test_outputs_apart_from_inputs():
    from sam_tf_amd import ops
    g = _gpu(_case(2, 8, 4, 4, 16, 16, F32))
    with pytest.raises(ValueError):
        ops.linattn(g['q'], g['k'], g['v'], g['decay'], out=g['q'])
    with pytest.raises(ValueError):
        ops.linattn_step(g['q'][:, 0], g['k'][:, 0], g['v'][:, 0], g['decay'], g['state'], out=g['v'].view(-1)[:2 * 4 * 16].view(2, 4, 16))
    from tests.test_gpu_block_norm import _case as norms, _gpu as to
    c = to(norms(9, 64, F32, 'rms', 'full'))
    room = torch.empty(10, 64, device='cuda')
    room[:9] = c['x']
    with pytest.raises(ValueError):
        ops.block_norm(room[:9], c['y'], c['post_w'], c['pre_w'], gate=c['gate'], kind='rms', h=room[1:])
    with pytest.raises(ValueError):
        ops.block_norm(c['x'], c['y'], c['post_w'], c['pre_w'], gate=c['gate'], kind='rms', u=c['gate'])
    h, u = ops.block_norm(c['x'], c['y'], c['post_w'], c['pre_w'], gate=c['gate'], kind='rms', h=c['y'], u=c['x'])
    assert h is c['y'] and u is c['x']


def test_refusals():
    from sam_tf_amd import ops
    from sam_tf_amd._lib import SamxError
    g = _gpu(_case(2, 8, 4, 2, 16, 24, F32))
    a = (g['q'], g['k'], g['v'], g['decay'])
    with pytest.raises(TypeError):
        ops.linattn(g['q'].double(), *a[1:])
    with pytest.raises(TypeError):
        ops.linattn(g['q'], g['k'].bfloat16(), *a[2:])
    with pytest.raises(ValueError):
        ops.linattn(g['q'][0], *a[1:])
    with pytest.raises(ValueError):
        ops.linattn(g['q'], g['k'][:, :5], *a[2:])
    with pytest.raises(ValueError):
        ops.linattn(g['q'].transpose(2, 3).contiguous().transpose(2, 3), *a[1:])
    with pytest.raises(ValueError):
        ops.linattn(*a[:3], g['decay'][:2])
    with pytest.raises(ValueError):
        ops.linattn(*a, state=g['state'][:1])
    with pytest.raises(ValueError):
        ops.linattn(*a, state=g['state'], state_out=g['state'])
    with pytest.raises(TypeError):
        ops.linattn(*a, lengths=torch.ones(2, dtype=torch.int64, device='cuda'))
    with pytest.raises(SamxError):
        ops.linattn(g['q'][:, :, :3], *a[1:3], g['decay'][:3].contiguous())
    with pytest.raises(SamxError):
        ops.linattn(*a, scale=float('inf'))
    wide = torch.zeros(1, 2, 1, 129, device='cuda')
    with pytest.raises(SamxError):
        ops.linattn(wide, wide, wide, g['decay'][:1].contiguous())
    long = torch.zeros(1, 1024, 1, 16, device='cuda')
    with pytest.raises(SamxError):
        ops.linattn(long, long, long, g['decay'][:1].contiguous(), ws=torch.empty(8, dtype=torch.uint8, device='cuda'))
    with pytest.raises(ValueError):
        ops.linattn_step(*a, g['state'])

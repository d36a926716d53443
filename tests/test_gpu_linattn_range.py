"""Linear attention of float16 near both ends of the type's range, and float32 states whatever the operands' type: against the
float64 recurrence (tests/seq_ref.py)."""
import pytest
import torch

from tests import seq_ref as R
from tests.seq_ref import U32, half_step, smallest, within
from tests.test_gpu_linattn import BF16, F16, F32, _abs, _case, _d, _errors, _gpu

pytestmark = pytest.mark.gpu

# factors of (q, k, v, dout, state, dstate), scale
ENDS = {
    'small gradient': ((1, 1, 1, 1e-3, 1, 1e-3), 0.125),
    'smaller gradient': ((1, 1, 1, 1e-5, 1, 1e-5), 0.125),
    'smallest gradient': ((1, 1, 1, 1e-6, 1, 0), 0.125),
    'small values': ((1, 1, 1e-3, 1, 1e-3, 1), 0.125),
    'smaller values': ((1, 1, 1e-5, 1, 1e-5, 1), 0.125),
    'small queries and keys': ((1e-4, 1e-4, 100, 1, 1e-4, 1), 10.0),
    'large state': ((1e-3, 1, 1, 1e-3, 1e6, 1), 0.01),
    'large state gradient': ((1, 1e-3, 1e-3, 1, 1, 1e6), 0.01),
    'large scores': ((300, 300, 1e-4, 1e-4, 1e-3, 1e-3), 0.02),
    'large scale': ((1e-2, 1e-2, 1e-2, 100, 1e-3, 1), 1000.0),
    'large everywhere': ((1000, 1000, 1000, 1000, 1e6, 1), 1e-9),
}


def _scaled(c, factors, dtype):
    for n, f in zip(('q', 'k', 'v', 'dout', 'state', 'dstate'), factors):
        c[n] = (c[n].float() * f).to(F32 if 'state' in n else dtype)
    return c


def _most(t):
    return float(t.double().abs().max())


def _hold(c, scale, dtype, what=''):
    """States are float32: the bound is that of float32 operands.  Outputs: a step of the type where scores and state meet the
    values, relative, and one for the output itself.  The last term of both: of a column (or a row of scores) whose largest
    value is m, float16 keeps what is above 2^-39 m; T rows and two such products meet."""
    from sam_tf_amd import ops
    g, d = _gpu(c), _d(c)
    a = _abs(d)
    B, T, H, D = c['q'].shape
    DV = c['v'].shape[3]
    es, eo, h = _errors(F32, T, D, DV)[0], _errors(dtype, T, D, DV)[0], 1.01 * half_step(dtype)
    q, k, v, o = (_most(c[n]) for n in ('q', 'k', 'v', 'dout'))
    dim, low = max(D, DV), 2.0 ** -38 * (T + 64)
    S, G = _most(c['state']) + T * k * v, _most(c['dstate']) + T * scale * q * o
    run = lambda x: (R.linattn(x['q'], x['k'], x['v'], d['decay'], scale, x['state'], d['lengths']) +
                     R.linattn_grad(x['q'], x['k'], x['v'], d['decay'], x['dout'], scale, x['state'], x['dstate'], d['lengths']))
    want, size = run(d), run(a)
    assert all(_most(want[i]) < 65504 for i in (0, 2, 3, 4)), 'the case itself is beyond float16'
    got = (ops.linattn(g['q'], g['k'], g['v'], g['decay'], scale=scale, state=g['state'], lengths=g['lengths']) +
           ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], scale=scale, state=g['state'], dstate=g['dstate'],
                            lengths=g['lengths']))
    rep = H // c['k'].shape[2]
    lows = [low * x for x in (scale * q * dim * S, k * v, scale * o * dim * S, rep * v * dim * G, rep * k * dim * G, scale * q * o)]
    for i, n in enumerate(('out', 'state', 'dq', 'dk', 'dv', 'dstate')):
        e, r, t = (es, 0.0, 0.0) if 'state' in n else (eo + (H + 2) * U32, h, smallest(dtype))
        within(got[i], want[i], e * size[i] + r * want[i].abs() + t + lows[i], what + ' ' + n)


@pytest.mark.parametrize('D,DV,HK', [(64, 64, 2), (128, 128, 2), (40, 100, 1), (77, 33, 2)])
@pytest.mark.parametrize('end', sorted(ENDS))
def test_float16_at_the_ends_of_its_range(end, D, DV, HK):
    f, scale = ENDS[end]
    _hold(_scaled(_case(2, 150, 2, HK, D, DV, F16, seed=31, lengths=[150, 97]), f, F16), scale, F16)


@pytest.mark.parametrize('end', ['smaller gradient', 'small values', 'large state', 'large scores', 'large scale'])
def test_float16_at_the_ends_in_segments(end):
    f, scale = ENDS[end]
    _hold(_scaled(_case(1, 1100, 2, 2, 72, 64, F16, seed=32), f, F16), scale, F16)


@pytest.mark.parametrize('end', ['smaller gradient', 'large state', 'large scores'])
def test_float16_at_the_ends_of_more_heads_than_units(end):
    f, scale = ENDS[end]
    _hold(_scaled(_case(66, 70, 4, 4, 72, 100, F16, seed=33, lengths=[70 - b for b in range(66)]), f, F16), scale, F16)


@pytest.mark.parametrize('dtype', [BF16, F16])
def test_columns_of_different_size(dtype):
    """Each column of v and dout by its own power of two, from 2^-14 to 2^8: the small ones' states as exact as the large ones'."""
    c = _case(2, 200, 2, 2, 48, 46, dtype, seed=34)
    p = 2.0 ** torch.linspace(-14, 8, 46).round()
    for n in ('v', 'dout'):
        c[n] = (c[n].float() * p).to(dtype)
    from sam_tf_amd import ops
    g, d = _gpu(c), _d(c)
    a = _abs(d)
    S = ops.linattn(g['q'], g['k'], g['v'], g['decay'], scale=0.1)[1]
    dS = ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], scale=0.1)[3]
    f = lambda x: (R.linattn(x['q'], x['k'], x['v'], d['decay'], 0.1, None, None)[1],
                   R.linattn_grad(x['q'], x['k'], x['v'], d['decay'], x['dout'], 0.1, None, None, None)[3])
    e = _errors(F32, 200, 48, 46)[0]
    for x, w, m, n in zip((S, dS), f(d), f(a), ('state', 'dstate')):
        most = m.amax((0, 1, 2))               # of a column
        within(x, w, e * m + 2.0 ** -38 * 264 * most, n)


@pytest.mark.parametrize('what', ['q', 'k', 'v', 'dout'])
@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
@pytest.mark.parametrize('dtype,D,DV', [(F32, 24, 40), (BF16, 40, 24), (F16, 64, 64), (F16, 100, 128), (BF16, 128, 128)])
def test_rows_beside_one_that_is_not_finite(dtype, D, DV, bad, what):
    """Row 75 of sequence 1 has a value that is not finite.  Rows that do not meet it, those of its own chunk among them, are as
    they were: the same products in another order, each order within _errors of the sum of magnitudes, rounded once each."""
    from sam_tf_amd import ops
    T, H, HK, at, scale = 150, 4, 2, 75, 0.5
    c0 = _case(2, T, H, HK, D, DV, dtype, seed=35)
    a = _abs(_d(c0))
    size = R.linattn(a['q'], a['k'], a['v'], a['decay'], scale, a['state'], None)[:1] + R.linattn_grad(
        a['q'], a['k'], a['v'], a['decay'], a['dout'], scale, a['state'], a['dstate'], None)[:3]
    error, step = _errors(dtype, T, D, DV)[0], 1.01 * half_step(dtype)
    c = _gpu(c0)

    def run():
        o = ops.linattn(c['q'], c['k'], c['v'], c['decay'], scale, c['state'])[:1]
        return o + ops.linattn_grad(c['q'], c['k'], c['v'], c['decay'], c['dout'], scale, c['state'], c['dstate'])[:3]
    want = run()
    c[what][1, at, 1 if what in ('q', 'dout') else 0, 3] = bad
    got = run()
    meets = [1] if what in ('q', 'dout') else [0, 1]               # query heads that meet it; their key head is 0
    none, only, behind, upto = slice(0, 0), slice(at, at + 1), slice(at, None), slice(None, at + 1)
    rows = {'q': (only, none, upto, upto), 'dout': (none, only, upto, upto),
            'k': (behind, behind, none, only), 'v': (behind, behind, only, none)}[what]
    q, k, v, o, S, dS = (_most(c0[n]) for n in ('q', 'k', 'v', 'dout', 'state', 'dstate'))
    S, G = S + T * k * v, dS + T * scale * q * o
    low = 2.0 ** -38 * (T + 64) * max(D, DV) * max(scale * q * S, scale * o * S, 2 * v * G, 2 * k * G)      # (as in _hold)
    for x, w, r, m, n in zip(got, want, rows, size, ('out', 'dq', 'dk', 'dv')):
        same = torch.ones(x.shape[:3], dtype=torch.bool)
        same[1, r, meets if n in ('out', 'dq') else [0]] = False
        x, w = x.cpu().double(), w.cpu().double()
        tol = 2 * (error + (H + 2) * U32) * m + 2 * step * w.abs() + 2 * smallest(dtype) + low
        within(x[same], w[same], tol[same], n)
        if not bool(same.all()):
            assert not bool(torch.isfinite(x[~same]).all(-1).any()), n


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('B,T,H,HK,D,DV,lengths', [(2, 200, 2, 2, 64, 64, None), (3, 150, 4, 2, 128, 128, [150, 64, 97]), (2, 130, 2, 1, 45, 100, None),
                                                   (1, 1100, 2, 2, 128, 72, None), (66, 70, 4, 4, 96, 128, [70 - b for b in range(66)])])
def test_outputs_of_16_bits_are_rounded_once(B, T, H, HK, D, DV, lengths, dtype):
    """Scores and the state's copy meet the values as two numbers each, so half a step squared is lost there (twice, and once
    more where the state's terms are split); the output's own rounding is the only one of half a step."""
    from sam_tf_amd import ops
    scale = D ** -0.5
    c = _case(B, T, H, HK, D, DV, dtype, seed=36, lengths=lengths)
    g, d = _gpu(c), _d(c)
    a = _abs(d)
    step, f = half_step(dtype), _errors(F32, T, D, DV)[0]
    run = lambda x: (R.linattn(x['q'], x['k'], x['v'], d['decay'], scale, x['state'], d['lengths'])[:1] +
                     R.linattn_grad(x['q'], x['k'], x['v'], d['decay'], x['dout'], scale, x['state'], x['dstate'], d['lengths'])[:3])
    kw = dict(scale=scale, state=g['state'], lengths=g['lengths'])
    got = ops.linattn(g['q'], g['k'], g['v'], g['decay'], **kw)[:1] + \
        ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], dstate=g['dstate'], **kw)[:3]
    q, k, v, o, S, dS = (_most(c[n]) for n in ('q', 'k', 'v', 'dout', 'state', 'dstate'))
    S, G = S + T * k * v, dS + T * scale * q * o
    low = 0.0 if dtype == BF16 else 2.0 ** -38 * (T + 64) * max(D, DV) * max(scale * q * S, scale * o * S, 2 * v * G, 2 * k * G)  # (as in _hold)
    for x, w, m, n in zip(got, run(d), run(a), ('out', 'dq', 'dk', 'dv')):
        within(x, w, (f + (H + 2) * U32 + 3.3 * step * step) * m + step * (1 + step) * w.abs() + smallest(dtype) + low, n)


@pytest.mark.parametrize('bad', [float('inf'), float('nan')])
@pytest.mark.parametrize('dtype,D,DV', [(F32, 24, 40), (BF16, 40, 24), (F16, 64, 64), (F16, 100, 128), (BF16, 128, 128)])
def test_a_state_that_is_not_finite_in_one_place(dtype, D, DV, bad):
    """Element (3, 5) of one head's state meets column 5 of out and element 3 of dq; of its gradient, element 3 of dk and
    column 5 of dv.  Everything else has the same bits."""
    from sam_tf_amd import ops
    c = _gpu(_case(2, 150, 2, 2, D, DV, dtype, seed=37))

    def run(state, dstate):
        return (ops.linattn(c['q'], c['k'], c['v'], c['decay'], 0.2, state) +
                ops.linattn_grad(c['q'], c['k'], c['v'], c['decay'], c['dout'], 0.2, state, dstate))
    want = run(c['state'], c['dstate'])
    s, d = c['state'].clone(), c['dstate'].clone()
    s[1, 1, 3, 5] = bad
    d[1, 0, 3, 5] = bad
    got = run(s, d)
    meets = [torch.zeros(w.shape, dtype=torch.bool, device='cuda') for w in want]
    out, state, dq, dk, dv, dstate = meets
    out[1, :, 1, 5] = state[1, 1, 3, 5] = dq[1, :, 1, 3] = dk[1, :, 0, 3] = dv[1, :, 0, 5] = dstate[1, 0, 3, 5] = True
    for x, w, m, n in zip(got, want, meets, ('out', 'state', 'dq', 'dk', 'dv', 'dstate')):
        assert torch.equal(x[~m], w[~m]), n
        assert not bool(torch.isfinite(x[m]).any()), n


def test_float16_captured_and_replayed():
    from sam_tf_amd import ops
    g = _gpu(_case(3, 700, 2, 1, 128, 72, F16, seed=38, lengths=[700, 333, 64]))

    def step():
        return (ops.linattn(g['q'], g['k'], g['v'], g['decay'], 0.1, g['state'], g['lengths']) +
                ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], 0.1, g['state'], g['dstate'], g['lengths']))
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
            g[n].copy_(torch.randn(g[n].shape, generator=torch.Generator().manual_seed(9 * i + len(n))) * 10.0 ** (1 - i))
        g['lengths'].copy_(torch.tensor([700 - 150 * i, 90 * i, 64 + i], dtype=torch.int32))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_rows_of_zeros_meet_a_huge_state(dtype):
    """0 times a state of 1e30 is 0, also where the row's scores are zeros."""
    from sam_tf_amd import ops
    c = _case(2, 100, 2, 2, 72, 80, dtype, seed=39)
    c['state'] *= 1e30
    c['dstate'] *= 1e30
    for n in ('q', 'k', 'v', 'dout'):
        c[n][:, 30:71] = 0
    g = _gpu(c)
    out = ops.linattn(g['q'], g['k'], g['v'], g['decay'], scale=0.5, state=g['state'])[0]
    got = ops.linattn_grad(g['q'], g['k'], g['v'], g['decay'], g['dout'], scale=0.5, state=g['state'], dstate=g['dstate'])[:3]
    for x in (out,) + got:
        assert bool((x[:, 30:71] == 0).all())

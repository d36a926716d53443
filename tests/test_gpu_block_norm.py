"""samx_block_norm / samx_block_norm_grad against the float64 formulas (tests/seq_ref.py)."""
import pytest
import torch

from tests import seq_ref as R
from tests.seq_ref import U32, half_step, smallest, within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _case(N, D, dtype, kind, gate, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    c = dict(x=r(N, D), y=r(N, D) + shift, h=r(N, D) * 1.3 + shift, dh=r(N, D), du=r(N, D))
    c = {k: v.to(dtype) for k, v in c.items()}
    c['post_w'], c['pre_w'] = 1 + 0.1 * r(D), 1 + 0.1 * r(D)
    c['post_b'], c['pre_b'] = (0.1 * r(D), 0.1 * r(D)) if kind == 'layer' else (None, None)
    c['gate'] = None if gate == 'none' else r(D) if gate == 'channel' else r(N, D).to(dtype)
    return c


def _gpu(c):
    return {k: None if v is None else v.cuda() for k, v in c.items()}


def _d(c):
    return {k: None if v is None else v.double() for k, v in c.items()}


def _spread(x, kind, eps):
    """(1 / spread, the largest value of a row): what the error of a mean costs the normalised row."""
    m = x.mean(-1, keepdim=True) if kind == 'layer' else 0.0
    return 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps), x.abs().amax(-1, keepdim=True)


# A sum of a row's D values in float32: at most 16 values of a thread one after the other, 6 steps over the lanes, at
# most 16 waves: 38 roundings, 38 U32 of the sum of magnitudes; a product, a square root and a quotient behind it: 48.
C = 48 * U32


def _tol_forward(c, res, kind, eps, dtype):
    d = _d(c)
    s, top = _spread(d['y'], kind, eps)
    yh, _, n = R.norm(d['y'], d['post_w'], d['post_b'], kind, eps)
    g = 1.0 if d['gate'] is None else d['gate'].abs()
    # the mean's error, C of the largest value, times s; the spread's, C relative (twice with the mean's in it)
    off_h = g * (2 * C * (yh.abs() + top * s) * d['post_w'].abs() + 4 * U32 * n.abs()) + 4 * U32 * (res * d['x']).abs()
    h, u = R.block(d['x'], d['y'], d['post_w'], d['pre_w'], d['post_b'], d['pre_b'], d['gate'], res, kind, eps)
    s2, top2 = _spread(h, kind, eps)
    hh = R.norm(h, d['pre_w'], d['pre_b'], kind, eps)[0]
    worst = off_h.amax(-1, keepdim=True)
    off_u = (2 * C * (hh.abs() + top2 * s2) + s2 * (off_h + worst * (1 + hh.abs()))) * d['pre_w'].abs() + 4 * U32 * u.abs()
    r = half_step(dtype) * 1.01
    return h, u, off_h + r * h.abs() + smallest(dtype), off_u + r * u.abs() + smallest(dtype)


SHAPES = [(1, 1), (3, 2), (1, 7), (5, 64), (33, 65), (9, 100), (70, 128), (7, 513), (1025, 96), (4, 1000), (2, 2048),
          (600, 4096), (3, 4100), (2, 8192)]
LONG = [(300, 8195), (3, 16384)]      # rows of 16 bits of which a thread holds two pieces


@pytest.mark.parametrize('gate', ['none', 'channel', 'full'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_forward(dtype, kind, gate):
    from sam_tf_amd import ops
    for N, D in SHAPES + (LONG if dtype != F32 else []):
        eps = 1e-6
        c = _case(N, D, dtype, kind, gate, seed=N + D)
        k = _gpu(c)
        h, u = ops.block_norm(k['x'], k['y'], k['post_w'], k['pre_w'], post_b=k['post_b'], pre_b=k['pre_b'],
                              gate=k['gate'], res_scale=0.75, kind=kind, eps=eps)
        wh, wu, th, tu = _tol_forward(c, 0.75, kind, eps, dtype)
        if D == 1 and kind == 'layer':      # a row of one value has no spread: its normalised value is 0
            tu, th = tu + 1.0, th + 1.0
        within(h, wh, th, 'h %d x %d' % (N, D))
        within(u, wu, tu, 'u %d x %d' % (N, D))


@pytest.mark.parametrize('gate', ['none', 'channel', 'full'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_gradient(dtype, kind, gate):
    from sam_tf_amd import ops
    for N, D in [s for s in SHAPES if s[1] > 1] + (LONG if dtype != F32 else []):
        eps, res = 1e-6, 0.75
        c = _case(N, D, dtype, kind, gate, seed=N + 7 * D)
        k, d = _gpu(c), _d(c)
        got = ops.block_norm_grad(k['y'], k['h'], k['dh'], k['du'], k['post_w'], k['pre_w'], post_b=k['post_b'],
                                  pre_b=k['pre_b'], gate=k['gate'], res_scale=res, kind=kind, eps=eps)
        a = (d['y'], d['h'], d['dh'], d['du'], d['post_w'], d['pre_w'], d['post_b'], d['pre_b'], d['gate'], res, kind, eps)
        want = R.block_grad(*a)
        # Each row's error is a few C of the magnitudes that go into it (six reductions, each with C; the mean's error
        # through `top * s`); of the sums over N rows, N more roundings at most (one group adds them all).
        s, top = _spread(d['h'], kind, eps)
        sy, topy = _spread(d['y'], kind, eps)
        hh, yh = R.norm(d['h'], d['pre_w'], None, kind, eps)[0].abs(), R.norm(d['y'], d['post_w'], None, kind, eps)[0].abs()
        hx, yx = hh + top * s, yh + topy * sy           # what their errors, times C, are of
        kk = (d['du'] * d['pre_w']).abs()
        mk = (kk * hx).mean(-1, keepdim=True)
        et = 8 * C * (s * (kk + hx * mk + kk.mean(-1, keepdim=True)) + d['dh'].abs())
        t = s * (kk + hh * mk + kk.mean(-1, keepdim=True)) + d['dh'].abs()
        g = torch.ones(()) if d['gate'] is None else d['gate'].abs()
        ek, kt = g * d['post_w'].abs() * et, g * d['post_w'].abs() * t
        ey = sy * (ek + 8 * C * (kt + yx * (kt * yx).mean(-1, keepdim=True) + kt.mean(-1, keepdim=True)) +
                   yx * (ek * yx).mean(-1, keepdim=True) + ek.mean(-1, keepdim=True))
        n = yx * d['post_w'].abs() + (d['post_b'].abs() if d['post_b'] is not None else 0.0)
        r = half_step(dtype) * 1.01
        within(got['x'], want['x'], res * et + r * want['x'].abs() + smallest(dtype), 'dx %d x %d' % (N, D))
        within(got['y'], want['y'], ey + r * want['y'].abs() + smallest(dtype), 'dy %d x %d' % (N, D))
        rows = (N + 64) * U32
        within(got['post_w'], want['post_w'], (g * (et * yx + t * yx * (8 * C + rows))).sum(0), 'dpost_w')
        within(got['pre_w'], want['pre_w'], (d['du'].abs() * hx * (8 * C + rows)).sum(0), 'dpre_w')
        if kind == 'layer':
            within(got['post_b'], want['post_b'], (g * (et + t * rows)).sum(0), 'dpost_b')
            within(got['pre_b'], want['pre_b'], (d['du'].abs() * rows).sum(0), 'dpre_b')
        else:
            assert got['post_b'] is None and got['pre_b'] is None
        if gate == 'channel':
            within(got['gate'], want['gate'], (et * n + t * n * (8 * C + rows)).sum(0), 'dgate')
        elif gate == 'full':
            within(got['gate'], want['gate'], et * n + t * n * 8 * C + r * want['gate'].abs() + smallest(dtype), 'dgate')
        else:
            assert got['gate'] is None


def test_rows_far_from_zero_keep_their_spread():
    """LayerNorm of rows whose mean is a thousand times their spread: the variance is that of the differences."""
    from sam_tf_amd import ops
    c = _case(40, 700, F32, 'layer', 'channel', shift=1000.0)
    k = _gpu(c)
    h, u = ops.block_norm(k['x'], k['y'], k['post_w'], k['pre_w'], post_b=k['post_b'], pre_b=k['pre_b'], gate=k['gate'],
                          kind='layer', eps=1e-6)
    wh, wu, th, tu = _tol_forward(c, 1.0, 'layer', 1e-6, F32)
    within(h, wh, th, 'h')
    within(u, wu, tu, 'u')


def test_outputs_over_their_inputs_and_equal_twice():
    from sam_tf_amd import ops
    c = _gpu(_case(777, 515, BF16, 'rms', 'full'))
    args = dict(gate=c['gate'], kind='rms')
    h, u = ops.block_norm(c['x'], c['y'], c['post_w'], c['pre_w'], **args)
    x, y = c['x'].clone(), c['y'].clone()
    h2, u2 = ops.block_norm(x, y, c['post_w'], c['pre_w'], h=x, u=y, **args)
    assert h2 is x and u2 is y and torch.equal(h, h2) and torch.equal(u, u2)
    a = ops.block_norm_grad(c['y'], h, c['dh'], c['du'], c['post_w'], c['pre_w'], **args)
    b = ops.block_norm_grad(c['y'], h, c['dh'], c['du'], c['post_w'], c['pre_w'], **args)
    assert all(a[n] is b[n] is None or torch.equal(a[n], b[n]) for n in a)


def test_no_rows():
    from sam_tf_amd import ops
    c = _gpu(_case(0, 48, BF16, 'layer', 'channel'))
    kw = dict(post_b=c['post_b'], pre_b=c['pre_b'], gate=c['gate'], kind='layer')
    h, u = ops.block_norm(c['x'], c['y'], c['post_w'], c['pre_w'], **kw)
    g = ops.block_norm_grad(c['y'], h, c['dh'], c['du'], c['post_w'], c['pre_w'], **kw)
    assert h.shape == u.shape == (0, 48) and g['x'].shape == (0, 48)
    assert all(bool((g[n] == 0).all()) for n in ('gate', 'post_w', 'post_b', 'pre_w', 'pre_b'))


def test_a_bad_row_stays_a_row():
    """A row of infinities and NaN spoils its own outputs only."""
    from sam_tf_amd import ops
    c = _gpu(_case(9, 300, F32, 'layer', 'none'))
    kw = dict(post_b=c['post_b'], pre_b=c['pre_b'], kind='layer')
    h, u = ops.block_norm(c['x'], c['y'], c['post_w'], c['pre_w'], **kw)
    y = c['y'].clone()
    y[4] = float('nan')
    y[6, 3] = float('inf')
    h2, u2 = ops.block_norm(c['x'], y, c['post_w'], c['pre_w'], **kw)
    keep = [i for i in range(9) if i not in (4, 6)]
    assert torch.equal(h[keep], h2[keep]) and torch.equal(u[keep], u2[keep]) and bool(torch.isnan(u2[4]).all())


def test_gradient_against_differences():
    """The kernel's gradient along random directions against central differences of the kernel's forward pass
    (float32).  Step e: the cut-off is e^2 / 6 of a third derivative that is of the order of the loss's first ones here
    (values of order one), the noise U32 sqrt(values) / e: both far below 2e-3 of the sum of magnitudes at e = 1e-2."""
    from sam_tf_amd import ops
    N, D, e = 6, 40, 1e-2
    c = _gpu(_case(N, D, F32, 'layer', 'full', seed=5))
    names = ('x', 'y', 'gate', 'post_w', 'post_b', 'pre_w', 'pre_b')

    def loss(v):
        h, u = ops.block_norm(v['x'], v['y'], v['post_w'], v['pre_w'], post_b=v['post_b'], pre_b=v['pre_b'], gate=v['gate'],
                              res_scale=0.8, kind='layer', eps=1e-3)
        return float((h.double() * c['dh'].double()).sum() + (u.double() * c['du'].double()).sum()), h
    h = loss(c)[1]
    g = ops.block_norm_grad(c['y'], h, c['dh'], c['du'], c['post_w'], c['pre_w'], post_b=c['post_b'], pre_b=c['pre_b'],
                            gate=c['gate'], res_scale=0.8, kind='layer', eps=1e-3)
    gen = torch.Generator().manual_seed(1)
    for n in names:
        d = torch.randn(c[n].shape, generator=gen).cuda()
        d /= d.norm()
        up, down = (loss(dict(c, **{n: c[n] + s * e * d}))[0] for s in (1, -1))
        want = float((g[n].double() * d.double()).sum())
        size = float((g[n].double() * d.double()).abs().sum()) + 1.0
        assert abs((up - down) / (2 * e) - want) < 2e-3 * size, n


def test_captured_and_replayed():
    from sam_tf_amd import ops
    c = _gpu(_case(300, 256, BF16, 'layer', 'channel'))
    kw = dict(post_b=c['post_b'], pre_b=c['pre_b'], gate=c['gate'], kind='layer')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        h, u = ops.block_norm(c['x'], c['y'], c['post_w'], c['pre_w'], **kw)
        return [h, u] + list(ops.block_norm_grad(c['y'], h, c['dh'], c['du'], c['post_w'], c['pre_w'], **kw).values())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for n in ('x', 'y', 'dh', 'du'):
            c[n].copy_(torch.randn(c[n].shape, generator=torch.Generator().manual_seed(50 * i + len(n))))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    from sam_tf_amd import ops
    from sam_tf_amd._lib import SamxError
    c = _gpu(_case(8, 32, F32, 'rms', 'channel'))
    ok = (c['x'], c['y'], c['post_w'], c['pre_w'])
    with pytest.raises(TypeError):
        ops.block_norm(c['x'].double(), c['y'].double(), c['post_w'], c['pre_w'])
    with pytest.raises(TypeError):
        ops.block_norm(c['x'].bfloat16(), c['y'], c['post_w'], c['pre_w'])
    with pytest.raises(ValueError):
        ops.block_norm(c['x'][:4], c['y'], c['post_w'], c['pre_w'])
    with pytest.raises(ValueError):
        ops.block_norm(*ok, kind='batch')
    with pytest.raises(ValueError):
        ops.block_norm(*ok, post_b=c['post_w'])
    with pytest.raises(ValueError):
        ops.block_norm(*ok, gate=c['gate'][:5])
    with pytest.raises(ValueError):
        ops.block_norm(c['x'].t().contiguous().t(), c['y'], c['post_w'], c['pre_w'])
    both = torch.empty_like(c['x'])
    with pytest.raises(ValueError):
        ops.block_norm(*ok, h=both, u=both)
    with pytest.raises(SamxError):
        ops.block_norm(*ok, eps=-1.0)
    with pytest.raises(SamxError):
        ops.block_norm(*ok, res_scale=float('nan'))
    wide = torch.zeros(1, 8193, device='cuda')
    with pytest.raises(SamxError):
        ops.block_norm(wide, wide, wide[0], wide[0])
    with pytest.raises(SamxError):
        ops.block_norm_grad(c['y'], c['h'], c['dh'], c['du'], c['post_w'], c['pre_w'],
                            ws=torch.empty(16, dtype=torch.uint8, device='cuda'))

"""samx_distill_loss / samx_distill_grad against the float64 definition (tests/seq_ref.py)."""
import math

import pytest
import torch

from tests import seq_ref as R
from tests.seq_ref import U32, half_step, smallest, within

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _case(N, V, K, dtype, seed=0, pad=0, lse=False, tau=1.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.full((N, V + pad), 7.0)
    z[:, :V] = torch.randn(N, V, generator=g) * 2
    z = z.to(dtype)
    idx = torch.stack([torch.randperm(V, generator=g)[torch.arange(K) % V] for _ in range(N)]).to(torch.int32)
    t = torch.randn(N, K, generator=g) * 2
    w = torch.rand(N, generator=g) + 0.5
    norm = torch.logsumexp(t / tau, 1) + torch.rand(N, generator=g) if lse else None
    return dict(full=z, z=z[:, :V], idx=idx, t=t, w=w, lse=norm)


def _run(c, tau, scale, **kw):
    from sam_tf_amd import ops
    V = c['z'].shape[1]
    full = c['full'].cuda()
    dev = lambda x: None if x is None else x.cuda()
    a = (full[:, :V], dev(c['idx']), dev(c['t']))
    loss, grad = ops.distill_grad(*a, tau=tau, lse=dev(c['lse']), weight=dev(c['w']), scale=scale, **kw)
    alone = ops.distill_loss(*a, tau=tau, lse=dev(c['lse']), weight=dev(c['w']))
    assert torch.equal(torch.nan_to_num(loss, nan=12345.0), torch.nan_to_num(alone, nan=12345.0))
    return loss, grad


def _check(c, tau, scale, dtype, what=''):
    loss, grad = _run(c, tau, scale)
    z = c['z'].double()
    wl, wg, mass = R.distill(z, c['idx'], c['t'].double(), tau, c['lse'], c['w'], scale)
    # An exponent's argument a carries 3 U32 |a|, its result 2 U32 more; terms of size e^a with |a| e^a below 1 make the
    # sums 8 U32 off, and their at most V / G + 16 additions of one thread and the tree's 22 another (m + 40) U32 at most.
    m = 160
    top = torch.nan_to_num((z / tau).abs(), posinf=0.0).amax(1) + torch.nan_to_num((c['t'].double() / tau).abs(), posinf=0.0).amax(1) + math.log(z.shape[1])
    w = c['w'].double() if c['w'] is not None else torch.ones(z.shape[0], dtype=torch.float64)
    e = (m + 48 + 8 * top) * U32
    # each of the K terms: p's error times the bracket (at most 2 top + its own), the bracket's U32 m
    within(loss, wl, w * (mass.clamp(min=1e-30) * (4 * top + 4) * e + 1e-30) + U32 * wl.abs().nan_to_num(posinf=0.0), what + ' loss')
    f = scale / tau * w
    want = wg
    p_err = e[:, None] * (want.abs() + 2 * f[:, None] * mass[:, None] * torch.softmax(torch.nan_to_num(z / tau, neginf=-1e30), 1))
    dup = torch.zeros_like(z)
    dup.scatter_add_(1, c['idx'].clamp(0, z.shape[1] - 1).long(), torch.ones_like(c['t'].double()))
    p_err = p_err + (dup > 0) * (f * e * mass * 2)[:, None]
    within(grad, want, p_err + 1.01 * half_step(dtype) * want.abs() + smallest(dtype), what + ' grad')


# (V, K): every form of the kernel (one wave a row up to rows read twice) and the borders between them
SIZES = [(1, 1), (2, 3), (7, 2), (18, 4), (255, 16), (513, 5), (1025, 8), (2049, 64), (4097, 33), (8193, 20), (16385, 7)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('V,K', SIZES)
def test_sizes(V, K, dtype):
    for N, pad, lse, tau, scale in ((1, 0, False, 1.0, 1.0), (5, 3, True, 2.0, 0.25), (6, 61, False, 0.7, 3.0)):
        _check(_case(N, V, K, dtype, seed=V + N, pad=pad, lse=lse, tau=tau), tau, scale, dtype, 'N %d' % N)


@pytest.mark.parametrize('V,dtype', [(32769, BF16), (65537, F32), (131073, BF16), (131073, F16), (65543, BF16), (65544, BF16), (131073, F32)])
def test_wide_rows(V, dtype):
    _check(_case(3, V, 70, dtype, seed=1, lse=True), 1.0, 1.0, dtype)


@pytest.mark.parametrize('V', [50, 3000, 40000, 140000])
def test_entries_that_do_not_count_and_entries_that_stand_twice(V):
    c = _case(6, V, 12, F32, seed=3)
    c['idx'][0] = -1                                         # nothing is known of the row
    c['idx'][1, 3:] = -1
    c['idx'][2, 4], c['idx'][2, 5], c['idx'][2, 6] = V, -7, 2 ** 31 - 1
    c['idx'][3, 1:6] = c['idx'][3, 0]                        # the same index six times
    c['idx'][4] = V - 1
    c['w'][5] = 0.0
    c['full'][5] = math.nan                                  # a padding row may hold anything
    _check(c, 1.0, 1.0, F32)
    loss, grad = _run(c, 1.0, 1.0)
    assert float(loss[0]) == 0.0 and bool((grad[0] == 0).all())
    assert float(loss[5]) == 0.0 and bool((grad[5] == 0).all())


@pytest.mark.parametrize('V', [40, 9000, 70000, 140000])
def test_masked_logits(V):
    c = _case(6, V, 6, F32, seed=4)
    c['idx'] = torch.stack([torch.arange(6) * 5 for _ in range(6)]).to(torch.int32)
    c['full'][0, 31:V] = -math.inf                          # masked, none of the teacher's
    c['full'][1, :V] = torch.finfo(F32).min                 # a mask of the lowest value, one entry left
    c['full'][1, 5] = 1.0
    c['full'][2, 10] = -math.inf                            # the teacher has mass where the student has none
    c['full'][3, :V] = -math.inf                            # nothing left
    c['t'][4, 2] = -math.inf                                # the teacher's own mask
    c['full'][4, 10] = -math.inf
    c['full'][5, 3] = math.nan
    loss, grad = _run(c, 1.0, 1.0)
    assert float(loss[2]) == math.inf and float(loss[3]) == math.inf and math.isnan(float(loss[5]))
    assert bool(torch.isfinite(grad[:5]).all()) and bool(torch.isnan(grad[5]).all())
    assert bool((grad[0, 31:] == 0).all())
    keep = [0, 2, 3, 4]
    part = {k: None if v is None else v[keep] for k, v in c.items()}
    _check(part, 1.0, 1.0, F32)


def test_all_rows_of_a_launch():
    """Many rows, more than the device holds at once: each as it is alone."""
    c = _case(1, 700, 9, BF16)
    n = 5000
    from sam_tf_amd import ops
    g = torch.Generator().manual_seed(9)
    z = torch.randn(n, 700, generator=g).to(BF16).cuda()
    idx, t = torch.randint(0, 700, (n, 9), generator=g).to(torch.int32).cuda(), torch.randn(n, 9, generator=g).cuda()
    loss, grad = ops.distill_grad(z, idx, t)
    for i in (0, 1, 63, 1024, 4097, n - 1):
        a, b = ops.distill_grad(z[i:i + 1].contiguous(), idx[i:i + 1].contiguous(), t[i:i + 1].contiguous())
        assert torch.equal(a[0], loss[i]) and torch.equal(b[0], grad[i])


@pytest.mark.parametrize('V', [90, 5001, 140000])
def test_in_place_and_behind_the_columns(V):
    c = _case(7, V, 10, BF16, pad=5)
    loss, grad = _run(c, 1.0, 1.0)
    from sam_tf_amd import ops
    full = c['full'].cuda()
    z = full[:, :V]
    l2, g2 = ops.distill_grad(z, c['idx'].cuda(), c['t'].cuda(), weight=c['w'].cuda(), grad=z)
    assert g2 is z and torch.equal(l2, loss) and torch.equal(g2, grad)
    assert bool((full[:, V:] == 7.0).all())


def test_gradient_against_differences():
    """Central differences of the float64-summed kernel losses (float32): noise U32 * loss * sqrt(N) / e, cut-off e^2."""
    from sam_tf_amd import ops
    c = _case(8, 300, 12, F32, seed=2, lse=True, tau=2.0)
    z, idx, t, w, lse = (c[k].cuda() for k in ('z', 'idx', 't', 'w', 'lse'))
    z = z.contiguous()
    kw = dict(tau=2.0, lse=lse, weight=w)
    g = ops.distill_grad(z, idx, t, scale=0.5, **kw)[1]
    gen = torch.Generator().manual_seed(0)
    for _ in range(4):
        d = torch.randn(z.shape, generator=gen).cuda()
        d /= d.norm()
        e = 3e-2
        up, down = (0.5 * float(ops.distill_loss(z + s * e * d, idx, t, **kw).double().sum()) for s in (1, -1))
        assert abs((up - down) / (2 * e) - float((g.double() * d.double()).sum())) < 5e-4


def test_captured_and_replayed():
    from sam_tf_amd import ops
    c = _case(64, 4000, 16, BF16, seed=8)
    z, idx, t, w = (c[k].cuda() for k in ('z', 'idx', 't', 'w'))
    z = z.contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.distill_grad(z, idx, t, weight=w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, grad = ops.distill_grad(z, idx, t, weight=w)
    for i in range(4):
        z.copy_(torch.randn(z.shape, generator=torch.Generator().manual_seed(i)))
        a, b = ops.distill_grad(z, idx, t, weight=w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, a) and torch.equal(grad, b)


def test_rows_far_apart():
    """Rows 2^32 bytes from each other: offsets of 64 bits, and the same numbers."""
    from sam_tf_amd import ops
    c = _case(3, 100, 5, F32, seed=3)
    z, idx, t = c['z'].contiguous().cuda(), c['idx'].cuda(), c['t'].cuda()
    want = ops.distill_grad(z, idx, t)
    room = torch.empty(2 * 2 ** 30 + 100, device='cuda')
    far = room.as_strided((3, 100), (2 ** 30, 1))
    far.copy_(z)
    loss, grad = ops.distill_grad(far, idx, t, grad=far)
    assert grad is far and torch.equal(loss, want[0]) and torch.equal(far, want[1])


def test_refusals():
    from sam_tf_amd import ops
    from sam_tf_amd._lib import SamxError
    c = _case(4, 64, 4, F32)
    z, idx, t = c['z'].contiguous().cuda(), c['idx'].cuda(), c['t'].cuda()
    with pytest.raises(TypeError):
        ops.distill_loss(z.double(), idx, t)
    with pytest.raises(TypeError):
        ops.distill_loss(z, idx.long(), t)
    with pytest.raises(ValueError):
        ops.distill_loss(z, idx[:2], t)
    with pytest.raises(ValueError):
        ops.distill_loss(z.t(), idx, t)
    with pytest.raises(ValueError):
        ops.distill_loss(z, idx, t, weight=torch.ones(3, device='cuda'))
    with pytest.raises(ValueError):
        ops.distill_grad(z, idx, t, grad=torch.empty(4, 63, device='cuda'))
    big = torch.zeros(5, 64, device='cuda')
    with pytest.raises(ValueError):
        ops.distill_grad(big[:4], idx, t, grad=big[1:])
    for tau in (0.0, -1.0, float('nan'), float('inf')):
        with pytest.raises(SamxError):
            ops.distill_loss(z, idx, t, tau=tau)
    many = torch.zeros(4, 1025, dtype=torch.int32, device='cuda')
    with pytest.raises(SamxError):
        ops.distill_loss(z, many, many.float())
    with pytest.raises(SamxError):
        ops.distill_loss(z[:1].expand(4, 64), idx, t)
    a, b = ops.distill_grad(z[:0], idx[:0], t[:0])
    assert a.shape == (0,) and b.shape == (0, 64)

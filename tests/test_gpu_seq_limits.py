"""The sequence-policy operators at the sizes that they take at most."""
import pytest
import torch

from tests import seq_ref as R
from tests.seq_ref import U32, half_step, smallest, within
from tests.test_gpu_linattn import BF16, F32, _abs, _case, _check, _d, _gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_step_of_65536_heads(dtype):
    """4096 environments of 16 heads: D terms, and a rounding of each product and sum."""
    from sam_tf_amd import ops
    B, H, HK, D, DV = 4096, 16, 4, 8, 12
    c = _case(B, 1, H, HK, D, DV, dtype, seed=41)
    g, d = _gpu(c), _d(c)
    S = g['state'].clone()
    o = ops.linattn_step(g['q'][:, 0], g['k'][:, 0], g['v'][:, 0], g['decay'], S, scale=0.3)

    def formula(x):
        k, v = (x[n][:, 0].repeat_interleave(H // HK, 1) for n in ('k', 'v'))
        s = torch.exp(d['decay'])[:, None, None] * x['state'] + k[..., None] * v[..., None, :]
        return 0.3 * (x['q'][:, 0][..., None] * s).sum(-2), s
    (wo, ws), (mo, ms), e = formula(d), formula(_abs(d)), (D + 20) * U32
    within(o, wo, e * mo + 1.01 * half_step(dtype) * wo.abs() + smallest(dtype), 'out')
    within(S, ws, e * ms, 'state')


def test_sequences_of_131072_heads():
    _check(_case(4096, 2, 32, 16, 4, 4, BF16, seed=42, lengths=[(b + 2) % 3 for b in range(4096)]), 0.5, BF16)


def test_distillation_of_more_rows_than_a_launch_takes():
    """2^26 rows and some of 64 threads each.  Exponents' arguments have two roundings relative to at most 12, sums a few more:
    64 U32 of a probability, of a logarithm absolute."""
    from sam_tf_amd import ops
    N, V = 2 ** 26 + 7, 2
    g = torch.Generator(device='cuda').manual_seed(43)
    z = torch.randn(N, V, device='cuda', generator=g)
    idx = torch.randint(0, V, (N, 1), device='cuda', generator=g, dtype=torch.int32)
    teacher = torch.zeros(N, 1, device='cuda')
    weight = torch.rand(N, device='cuda', generator=g)
    loss, grad = ops.distill_grad(z, idx, teacher, weight=weight, scale=0.5)
    alone = ops.distill_loss(z, idx, teacher, weight=weight)
    for a in range(0, N, 2 ** 24):
        s = slice(a, a + 2 ** 24)
        q = torch.log_softmax(z[s].double(), 1)
        w, i = weight[s].double(), idx[s].long()
        want = -w * q.gather(1, i)[:, 0]
        for x in (loss, alone):
            assert float(((x[s].double() - want).abs() / (w * (1 + want.abs()) + 1e-30)).max()) < 64 * U32
        dense = q.exp().scatter_add(1, i, -torch.ones_like(q[:, :1]))
        assert float((grad[s].double() - 0.5 * w[:, None] * dense).abs().max()) < 64 * U32


def test_shared_heads_gradient_of_more_elements_than_a_launch_takes():
    """2^32 elements and some of dk.  All rows alike (one row, stride 0): the gradient's state is a geometric sum, and both
    gradients are known."""
    from sam_tf_amd import ops
    H, D, DV, T, scale = 2, 128, 8, 2 ** 25 + 3, 0.25
    c = _case(1, 1, H, 1, D, DV, BF16, seed=44, state=False, decay=[-1.0, -2.0])
    row = {n: c[n].double()[0, 0] for n in ('q', 'k', 'v', 'dout')}
    g = _gpu(c)
    q, k, v, o = (g[n].expand(1, T, -1, -1) for n in ('q', 'k', 'v', 'dout'))
    got = ops.linattn_grad(q, k, v, g['decay'], o, scale=scale)
    left = T - torch.arange(T - 64, T, dtype=torch.float64)                # rows from each of the last 64 on to the end
    lam = torch.exp(c['decay'].double())
    many = scale * (1 - lam ** left[:, None]) / (1 - lam)                  # [64, H]
    b = lambda t: t.abs()
    f = lambda q, o, k, v: (((o * v).sum(-1)[:, None] * q * many[..., None]).sum(1), ((q * k).sum(-1)[:, None] * o * many[..., None]).sum(1))
    want, size = f(row['q'], row['dout'], row['k'], row['v']), f(b(row['q']), b(row['dout']), b(row['k']), b(row['v']))
    h = half_step(BF16)
    for x, w, m in zip(got[1:3], want, size):
        x = x[0, :, 0]
        tol = (3.2 * h + 300 * U32) * m
        within(x[-64:], w, tol)
        far, most = w[0].cuda(), tol[0].cuda()
        for a in range(0, T - 64, 2 ** 22):
            assert bool(((x[a:min(T - 64, a + 2 ** 22)].double() - far).abs() <= most).all()), a

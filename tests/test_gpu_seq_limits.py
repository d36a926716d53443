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

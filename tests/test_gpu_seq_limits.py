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

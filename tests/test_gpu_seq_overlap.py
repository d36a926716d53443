"""Outputs of the distillation that are given: apart from every input, and from each other."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_distillation_outputs_over_inputs_are_refused():
    from sam_tf_amd import ops
    N, V, K = 8, 32, 4
    g = torch.Generator().manual_seed(1)
    room = torch.zeros(4096, device='cuda')
    part = lambda at, *s: room[at:at + torch.Size(s).numel()].view(*s)
    z, t, lse, w, loss = part(0, N, V), part(512, N, K), part(1024, N), part(1100, N), part(1200, N)
    z.copy_(torch.randn(N, V, generator=g))
    t.copy_(torch.randn(N, K, generator=g))
    w.fill_(1.0)
    idx = torch.randint(0, V, (N, K), generator=g, dtype=torch.int32).cuda()
    over = dict(logits=part(V * N - 3, N), teacher=part(512 + 5, N), lse=part(1024, N), weight=part(1100 - 7, N),
                idx=idx.view(-1).view(torch.float32)[:N])
    for f in (ops.distill_loss, ops.distill_grad):
        for n, x in over.items():
            with pytest.raises(ValueError, match=n):
                f(z, idx, t, lse=lse, weight=w, loss=x)
        f(z, idx, t, lse=lse, weight=w, loss=loss)
    for n, x in dict(teacher=part(600 - 250, N, V), lse=part(1031, N, V), weight=part(1107, N, V), loss=part(1200, N, V)).items():
        with pytest.raises(ValueError, match=n):
            ops.distill_grad(z, idx, t, lse=lse if n != 'weight' else None, weight=w, loss=loss, grad=x)
    wide = torch.zeros(N, 48, device='cuda')
    with pytest.raises(ValueError, match='loss'):
        ops.distill_grad(z, idx, t, loss=wide.view(-1)[-40:-32], grad=wide[:, :V])
    want = ops.distill_grad(z, idx, t, lse=lse, weight=w)
    got = ops.distill_grad(z, idx, t, lse=lse, weight=w, loss=loss, grad=z)
    assert got[1] is z and all(torch.equal(a, b) for a, b in zip(want, got))

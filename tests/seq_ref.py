"""Plain float64 forms of the sequence-policy operators (CPU), and the error a float32 computation may have."""
import math

import torch

U32 = 2.0 ** -24                      # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """What rounding to a type can lose of a value below its normal range."""
    return {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]


def within(got, want, tol, what=''):
    """|got - want| <= tol everywhere; infinities and NaN in the same places."""
    got, want = got.detach().cpu().double(), want.detach().cpu().double()
    tol = torch.as_tensor(tol, dtype=torch.float64).cpu().expand_as(want)
    assert got.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ': NaN'
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), what + ': infinities'
    off = (got - want).abs()[fine]
    bad = off > tol[fine]
    assert not bool(bad.any()), '%s: %d of %d beyond the tolerance, worst %.3g of it (off %.3g)' % (
        what, int(bad.sum()), bad.numel(), float((off / tol[fine].clamp(min=1e-300)).max()), float(off.max()))


# ------------------------------------------------------------------ block norms

def norm(x, w, b, kind, eps):
    m = x.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros((), dtype=x.dtype)
    s = 1.0 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    xh = (x - m) * s
    return xh, s, xh * w + (b if b is not None else 0.0)


def block(x, y, post_w, pre_w, post_b, pre_b, gate, res, kind, eps):
    n = norm(y, post_w, post_b, kind, eps)[2]
    h = res * x + (n if gate is None else gate * n)
    return h, norm(h, pre_w, pre_b, kind, eps)[2]


def block_grad(y, h, dh, du, post_w, pre_w, post_b, pre_b, gate, res, kind, eps):
    """By the formulas; None where there is no such gradient."""
    hh, sh, _ = norm(h, pre_w, pre_b, kind, eps)
    yh, sy, n = norm(y, post_w, post_b, kind, eps)

    def back(k, xh, s):
        r = k - xh * (k * xh).mean(-1, keepdim=True)
        if kind == 'layer':
            r = r - k.mean(-1, keepdim=True)
        return r * s
    t = dh + back(du * pre_w, hh, sh)
    dn = t if gate is None else t * gate
    dgate = None if gate is None else (t * n).sum(0) if gate.dim() == 1 else t * n
    lay = kind == 'layer'
    return dict(x=res * t, y=back(dn * post_w, yh, sy), gate=dgate, post_w=(dn * yh).sum(0),
                post_b=dn.sum(0) if lay else None, pre_w=(du * hh).sum(0), pre_b=du.sum(0) if lay else None)


# ------------------------------------------------------------------ distillation

def distill(z, idx, t, tau, lse, weight, scale):
    """(loss, gradient of scale * sum(loss), P): row by row from the definition."""
    N, V = z.shape
    loss, grad, mass = torch.zeros(N, dtype=torch.float64), torch.zeros_like(z), torch.zeros(N, dtype=torch.float64)
    for i in range(N):
        w = 1.0 if weight is None else float(weight[i])
        if w == 0.0:
            continue
        ks = [k for k in range(idx.shape[1]) if 0 <= int(idx[i, k]) < V]
        if bool((z[i] == -math.inf).all()):
            logq = torch.full((V,), -math.inf, dtype=torch.float64)
        else:
            logq = torch.log_softmax(z[i] / tau, 0)
        x = torch.tensor([float(t[i, k]) / tau for k in ks], dtype=torch.float64)
        if lse is not None:
            x = x - float(lse[i])
        elif len(ks):
            x = x - torch.logsumexp(x, 0)
        p = x.exp()
        dense = torch.zeros(V, dtype=torch.float64)
        total = 0.0
        for j, k in enumerate(ks):
            dense[int(idx[i, k])] += p[j]
            if float(p[j]) > 0.0:
                total += float(p[j]) * (float(x[j]) - float(logq[int(idx[i, k])]))
        mass[i] = p.sum()
        loss[i] = w * total
        grad[i] = scale / tau * w * (mass[i] * logq.exp() - dense)
    return loss, grad, mass


# ------------------------------------------------------------------ linear attention

def _spans(lengths, B, T):
    return [T if lengths is None else max(0, min(T, int(lengths[b]))) for b in range(B)]


def linattn(q, k, v, decay, scale, state, lengths):
    """The recurrence: (out, state behind the last row)."""
    B, T, H, D = q.shape
    HK, DV = k.shape[2], v.shape[3]
    out = torch.zeros(B, T, H, DV, dtype=torch.float64)
    S = torch.zeros(B, H, D, DV, dtype=torch.float64) if state is None else state.clone()
    lam = torch.exp(decay)[:, None, None]
    head = torch.arange(H) // (H // HK)
    for b, n in enumerate(_spans(lengths, B, T)):
        for t in range(n):
            S[b] = lam * S[b] + k[b, t, head][:, :, None] * v[b, t, head][:, None, :]
            out[b, t] = scale * (q[b, t][:, None, :] @ S[b])[:, 0]
    return out, S


def linattn_grad(q, k, v, decay, dout, scale, state, dstate, lengths):
    """By the formulas: (dq, dk, dv, gradient of the state before the first row)."""
    B, T, H, D = q.shape
    HK, DV = k.shape[2], v.shape[3]
    dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64) for t in (q, k, v))
    S = torch.zeros(B, H, D, DV, dtype=torch.float64) if state is None else state.clone()
    G = torch.zeros(B, H, D, DV, dtype=torch.float64) if dstate is None else dstate.clone()
    lam = torch.exp(decay)[:, None, None]
    head, rep = torch.arange(H) // (H // HK), H // HK
    for b, n in enumerate(_spans(lengths, B, T)):
        for t in range(n):
            S[b] = lam * S[b] + k[b, t, head][:, :, None] * v[b, t, head][:, None, :]
            dq[b, t] = scale * (S[b] @ dout[b, t][:, :, None])[:, :, 0]
        for t in reversed(range(n)):
            g = G[b] + scale * q[b, t][:, :, None] * dout[b, t][:, None, :]
            dk[b, t] = (g @ v[b, t, head][:, :, None])[:, :, 0].reshape(HK, rep, D).sum(1)
            dv[b, t] = (k[b, t, head][:, None, :] @ g)[:, 0].reshape(HK, rep, DV).sum(1)
            G[b] = lam * g
    return dq, dk, dv, G

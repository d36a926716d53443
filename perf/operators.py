"""Sequence-policy operators: what is measured, in plain torch operations and as the library's kernels.

Three operators, the parts of one training or acting step of a policy that reads a sequence:

  mix      linear attention with a decay for each head: the chunked form for whole trajectories ("mix_fwd", its
           gradient "mix_grad") and the recurrent form for one new step per environment ("mix_step")
  block    the norm behind a block, its gate, the scaled residual and the norm in front of the next block, in one
           pass ("block_fwd") and its gradient ("block_grad")
  distill  imitation of a teacher's top logits: the loss of each row ("distill_loss"), and the loss with the gradient
           of the student's logits ("distill_grad")

`own` False: `run` computes the plain form.  `own` True: `run` calls sam_tf_amd.ops.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
DEV = 'cuda'


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one environment acting: a small recurrent policy, latency is all
        dict(name='mix step, one env', op='mix_step', dtype='bf16', B=1, H=8, HK=8, D=64, DV=64),
        # a rollout server that steps many environments at once
        dict(name='mix step, 192 envs', op='mix_step', dtype='bf16', B=192, H=16, HK=16, D=128, DV=128),
        # a batch of long trajectories read in one go
        dict(name='mix forward, long', op='mix_fwd', dtype='bf16', B=2, T=4096, H=16, HK=16, D=128, DV=128,
             state=True, ragged=False),
        # odd sizes in full precision, trajectories of different lengths, key heads shared by two query heads
        dict(name='mix forward, odd f32', op='mix_fwd', dtype='f32', B=3, T=1531, H=6, HK=3, D=72, DV=88,
             state=True, ragged=True),
        # the training pass over a replayed batch of trajectories
        dict(name='mix gradient', op='mix_grad', dtype='bf16', B=4, T=2048, H=16, HK=16, D=128, DV=128,
             state=True, ragged=True),
        # one token of an acting policy between two blocks
        dict(name='block forward, one row', op='block_fwd', dtype='bf16', N=1, D=2048, kind='rms', gate='channel'),
        # odd width in full precision, the LayerNorm kind, a gate for each row and channel
        dict(name='block forward, odd f32', op='block_fwd', dtype='f32', N=4099, D=1000, kind='layer', gate='full'),
        # the training pass: 16k tokens of a wide policy
        dict(name='block gradient', op='block_grad', dtype='bf16', N=16384, D=4096, kind='rms', gate='channel'),
        # a small discrete action set
        dict(name='distill loss, 18 actions', op='distill_loss', dtype='f32', N=256, V=18, K=4, tau=1.0, lse=False),
        # an odd vocabulary inside padded rows
        dict(name='distill gradient, odd', op='distill_grad', dtype='f32', N=1021, V=10007, K=20, tau=2.0, lse=True),
        # an ordinary vocabulary
        dict(name='distill gradient', op='distill_grad', dtype='bf16', N=4096, V=32000, K=64, tau=1.0, lse=True),
        # the largest: a wide vocabulary
        dict(name='distill gradient, wide', op='distill_grad', dtype='bf16', N=4096, V=128000, K=128, tau=2.0,
             lse=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['mix_step', 'mix_fwd', 'mix_fwd', 'mix_grad', 'block_fwd', 'block_grad', 'distill_loss',
                     'distill_grad', 'distill_grad'])
    dtype = rng.choice(['bf16', 'bf16', 'f32', 'f16'])
    if op.startswith('mix'):
        hk = rng.choice([1, 2, 3, 4, 8])
        c = dict(op=op, dtype=dtype, H=hk * rng.choice([1, 1, 2]), HK=hk, D=rng.randint(8, 128), DV=rng.randint(8, 128))
        if rng.random() < 0.4:
            c['D'] = c['DV'] = rng.choice([32, 64, 128])
        if op == 'mix_step':
            c['B'] = _log_int(rng, 1, 192)
        else:
            c['T'] = _log_int(rng, 16, 4096)
            most = max(1, min(16, (4 << 26) // (c['H'] * c['T'] * c['T'])))
            c['B'] = _log_int(rng, 1, most)
            c['state'], c['ragged'] = rng.random() < 0.5, rng.random() < 0.5
        return c
    if op.startswith('block'):
        d = rng.choice([64, 256, 512, 1024, 2048, 4096]) if rng.random() < 0.5 else _log_int(rng, 24, 5000)
        return dict(op=op, dtype=dtype, N=_log_int(rng, 1, max(2, min(16384, (1 << 25) // d))), D=d,
                    kind=rng.choice(['rms', 'layer']), gate=rng.choice(['none', 'channel', 'full']))
    v = _log_int(rng, 16, 128000)
    return dict(op=op, dtype=dtype, N=_log_int(rng, 1, max(2, min(4096, (1 << 27) // v))), V=v,
                K=min(v, _log_int(rng, 1, 256)), tau=rng.choice([1.0, 2.0, 0.7]), lse=rng.random() < 0.5)


def work(c):
    e = torch.empty(0, dtype=TYPES[c['dtype']]).element_size()
    if c['op'].startswith('mix'):
        B, H, HK, D, DV = c['B'], c['H'], c['HK'], c['D'], c['DV']
        S = B * H * D * DV
        if c['op'] == 'mix_step':
            return dict(bytes=e * B * (H * D + HK * (D + DV) + H * DV) + 8 * S, flops=5 * S)
        rows = _rows_total(c)
        state_in = 4 * S if c['state'] else 0
        if c['op'] == 'mix_fwd':
            return dict(bytes=e * (rows * (H * D + HK * (D + DV)) + B * c['T'] * H * DV) + state_in + 4 * S,
                        flops=4.0 * rows * H * D * DV)
        return dict(bytes=e * (rows * (H * D + HK * (D + DV) + H * DV) + B * c['T'] * (H * D + HK * (D + DV))) +
                    2 * state_in + 4 * S, flops=10.0 * rows * H * D * DV)
    if c['op'].startswith('block'):
        n = c['N'] * c['D']
        full = n if c['gate'] == 'full' else 0
        if c['op'] == 'block_fwd':
            return dict(bytes=e * (4 * n + full) + 4 * c['D'] * (2 + (c['kind'] == 'layer') * 2 + (c['gate'] == 'channel')),
                        flops=12.0 * n)
        return dict(bytes=e * (6 * n + 2 * full) + 8 * c['D'] * (2 + (c['kind'] == 'layer') * 2 + (c['gate'] == 'channel')),
                    flops=30.0 * n)
    n = c['N'] * c['V']
    rows = 4 * c['N'] * (2 + 2 * c['K'] + (1 if c['lse'] else 0))
    return dict(bytes=e * n * (2 if c['op'] == 'distill_grad' else 1) + rows, flops=(6.0 if c['op'] == 'distill_grad' else 4.0) * n)


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _lengths(c):
    """Rows of each trajectory: the first is whole, the others end anywhere (a length of one among them)."""
    B, T = c['B'], c['T']
    if not c['ragged']:
        return [T] * B
    return [T if b == 0 else 1 + (T - 1) * ((b * 5 + 1) % 8) // 8 for b in range(B)]


def _rows_total(c):
    return sum(_lengths(c))


def prepare(c, seed):
    g = _gen(seed)
    dt = TYPES[c['dtype']]

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)

    s = dict(case=c)
    if c['op'].startswith('mix'):
        B, H, HK, D, DV = c['B'], c['H'], c['HK'], c['D'], c['DV']
        s['scale'] = D ** -0.5
        # memory lengths from about two steps to about five hundred
        s['decay'] = -torch.exp2(-(1.0 + 8.0 * torch.arange(H, device=DEV, dtype=torch.float32) / H))
        if c['op'] == 'mix_step':
            s['q'], s['k'], s['v'] = randn(B, H, D, dtype=dt), randn(B, HK, D, dtype=dt), randn(B, HK, DV, dtype=dt)
            s['state'] = randn(B, H, D, DV)
            return s
        T = c['T']
        # what a projection of the sequence gives: q, k and v side by side in one row
        row = randn(B, T, H * D + HK * D + HK * DV, dtype=dt)
        s['q'] = row[..., :H * D].unflatten(-1, (H, D))
        s['k'] = row[..., H * D:H * D + HK * D].unflatten(-1, (HK, D))
        s['v'] = row[..., H * D + HK * D:].unflatten(-1, (HK, DV))
        s['lengths'] = torch.tensor(_lengths(c), dtype=torch.int32, device=DEV) if c['ragged'] else None
        s['state'] = randn(B, H, D, DV) if c['state'] else None
        if c['op'] == 'mix_grad':
            s['dout'] = randn(B, T, H, DV, dtype=dt)
            s['dstate'] = randn(B, H, D, DV) if c['state'] else None
        return s
    if c['op'].startswith('block'):
        N, D = c['N'], c['D']
        s['y'] = randn(N, D, dtype=dt)
        s['post_w'], s['pre_w'] = 1.0 + randn(D, scale=0.1), 1.0 + randn(D, scale=0.1)
        s['post_b'], s['pre_b'] = (randn(D, scale=0.1), randn(D, scale=0.1)) if c['kind'] == 'layer' else (None, None)
        s['gate'] = {'none': lambda: None, 'channel': lambda: randn(D, scale=0.5),
                     'full': lambda: randn(N, D, dtype=dt, scale=0.5)}[c['gate']]()
        s['res_scale'], s['eps'] = 0.9, 1e-6
        if c['op'] == 'block_fwd':
            s['x'] = randn(N, D, dtype=dt)
        else:  # the residual stream as the forward pass left it, and what the layers above send back
            s['h'] = randn(N, D, dtype=dt, scale=1.3)
            s['dh'], s['du'] = randn(N, D, dtype=dt), randn(N, D, dtype=dt)
        return s
    N, V, K = c['N'], c['V'], c['K']
    width = (V + 63) // 64 * 64   # rows padded to a multiple of 64, as a head's product writes them
    s['logits'] = randn(N, width, dtype=dt, scale=2.0)[:, :V]
    # K different entries of each row, in no order; a few rows have fewer
    start = torch.randint(0, V, (N, 1), device=DEV, generator=g)
    step = max(1, V // K)
    s['idx'] = ((start + torch.arange(K, device=DEV) * step) % V).to(torch.int32)
    s['teacher'] = randn(N, K, scale=3.0)
    if K > 1:
        s['idx'][3::7, K // 2:] = -1
    # the teacher's own normaliser: above its top logits' (so its top probabilities sum to less than one)
    s['lse'] = (torch.logsumexp(s['teacher'] / c['tau'], 1) + torch.rand(N, device=DEV, generator=g)) if c['lse'] else None
    w = torch.rand(N, device=DEV, generator=g) + 0.5
    w[5::16] = 0.0   # rows of padding
    s['weight'] = w
    s['scale'] = (4096.0 if c['dtype'] == 'f16' else 1.0) / N   # half precision trains with a scaled loss
    return s


# ------------------------------------------------------------------ one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from sam_tf_amd import ops
    c = s['case']
    if c['op'] == 'mix_step':
        return ops.linattn_step(s['q'], s['k'], s['v'], s['decay'], s['state'], scale=s['scale']), s['state']
    if c['op'] == 'mix_fwd':
        return ops.linattn(s['q'], s['k'], s['v'], s['decay'], scale=s['scale'], state=s['state'], lengths=s['lengths'])
    if c['op'] == 'mix_grad':
        return ops.linattn_grad(s['q'], s['k'], s['v'], s['decay'], s['dout'], scale=s['scale'], state=s['state'],
                                dstate=s['dstate'], lengths=s['lengths'])
    if c['op'] == 'block_fwd':
        return ops.block_norm(s['x'], s['y'], s['post_w'], s['pre_w'], post_b=s['post_b'], pre_b=s['pre_b'],
                              gate=s['gate'], res_scale=s['res_scale'], kind=c['kind'], eps=s['eps'])
    if c['op'] == 'block_grad':
        return ops.block_norm_grad(s['y'], s['h'], s['dh'], s['du'], s['post_w'], s['pre_w'], post_b=s['post_b'],
                                   pre_b=s['pre_b'], gate=s['gate'], res_scale=s['res_scale'], kind=c['kind'],
                                   eps=s['eps'])
    if c['op'] == 'distill_loss':
        return ops.distill_loss(s['logits'], s['idx'], s['teacher'], tau=c['tau'], lse=s['lse'], weight=s['weight'])
    return ops.distill_grad(s['logits'], s['idx'], s['teacher'], tau=c['tau'], lse=s['lse'], weight=s['weight'],
                            scale=s['scale'])


def _run_plain(s):
    op = s['case']['op']
    return {'mix_step': _plain_step, 'mix_fwd': _plain_mix, 'mix_grad': _plain_mix_grad, 'block_fwd': _plain_block,
            'block_grad': _plain_block_grad, 'distill_loss': _plain_distill, 'distill_grad': _plain_distill}[op](s)


def _plain_step(s):
    """S <- e^decay S + k v^T ;  out = scale q S   (S is updated in place: it is the caller's)"""
    q, k, v = s['q'].float(), s['k'].float(), s['v'].float()
    rep = q.shape[1] // k.shape[1]
    if rep > 1:
        k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    S = s['state']
    S.mul_(torch.exp(s['decay'])[None, :, None, None]).add_(k[..., :, None] * v[..., None, :])
    out = (q[..., None, :] @ S)[..., 0, :] * s['scale']
    return out.to(s['q'].dtype), S


def _heads(x, H, valid):
    """[B, T, h, d] -> float32 [B, H, T, d]; rows behind a trajectory's end count as zeros."""
    x = x.float().transpose(1, 2)
    if valid is not None:
        x = torch.where(valid, x, torch.zeros((), device=x.device))
    if x.shape[1] != H:
        x = x.repeat_interleave(H // x.shape[1], 1)
    return x.contiguous()


def _mix_parts(s):
    B, T, H, _ = s['q'].shape
    t = torch.arange(T, device=DEV)
    n = t[:, None] - t[None, :]
    mask = torch.where(n >= 0, torch.exp(s['decay'][:, None, None] * n.clamp(min=0)), torch.zeros((), device=DEV))
    valid = None
    left = (T - 1 - t).expand(B, T)          # rows between a row and its trajectory's last one
    total = torch.full((B,), T, device=DEV)
    if s['lengths'] is not None:
        total = s['lengths'].long()
        valid = (t[None] < total[:, None])[:, None, :, None]
        left = (total[:, None] - 1 - t[None]).clamp(min=0)
    q, k, v = (_heads(s[x], H, valid) for x in 'qkv')
    d = s['decay']
    since = torch.exp(d[:, None] * (t + 1))[None, :, :, None]           # e^{decay (t+1)}  [1, H, T, 1]
    until = torch.exp(d[None, :, None] * left[:, None, :])[..., None]   # e^{decay left}   [B, H, T, 1]
    whole = torch.exp(d[None, :] * total[:, None])[..., None, None]     # e^{decay length} [B, H, 1, 1]
    return q, k, v, mask, valid, since, until, whole


def _plain_mix(s):
    """out_t = scale sum_{s<=t} e^{decay (t-s)} (q_t . k_s) v_s  (+ the state before the first row)"""
    q, k, v, mask, _, since, until, whole = _mix_parts(s)
    p = q @ k.transpose(-1, -2)
    p *= mask
    out = p @ v
    S = (k * until).transpose(-1, -2) @ v
    if s['state'] is not None:
        out += since * (q @ s['state'])
        S += whole * s['state']
    return (out * s['scale']).transpose(1, 2).to(s['q'].dtype).contiguous(), S


def _plain_mix_grad(s):
    q, k, v, mask, valid, since, until, whole = _mix_parts(s)
    H, dt, scale = s['q'].shape[2], s['q'].dtype, s['scale']
    do = _heads(s['dout'], H, valid)
    e = do @ v.transpose(-1, -2)
    e *= mask
    dq = e @ k
    dk = e.transpose(-1, -2) @ q
    del e
    p = q @ k.transpose(-1, -2)
    p *= mask
    dv = p.transpose(-1, -2) @ do
    del p
    dS = scale * ((q * since).transpose(-1, -2) @ do)
    dk, dv = dk * scale, dv * scale
    if s['state'] is not None:
        dq += since * (do @ s['state'].transpose(-1, -2))
    if s['dstate'] is not None:
        dk += until * (v @ s['dstate'].transpose(-1, -2))
        dv += until * (k @ s['dstate'])
        dS += whole * s['dstate']
    out = []
    for x, n in ((dq * scale, H), (dk, s['k'].shape[2]), (dv, s['k'].shape[2])):
        if valid is not None:
            x = torch.where(valid, x, torch.zeros((), device=x.device))
        if n != H:
            x = x.unflatten(1, (n, H // n)).sum(2)
        out.append(x.transpose(1, 2).to(dt).contiguous())
    return out[0], out[1], out[2], dS


def _norm(x, w, b, kind, eps):
    """(the normalised rows, one over their spread, weight times them plus bias)"""
    if kind == 'layer':
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    xh = x * r
    y = xh * w
    return xh, r, y if b is None else y + b


def _norm_back(dy, xh, r, w, kind):
    """(gradient of the rows, of the weight, of the bias)"""
    g = dy * w
    m = (g * xh).mean(-1, keepdim=True)
    dx = g - xh * m
    if kind == 'layer':
        dx = dx - g.mean(-1, keepdim=True)
    return dx * r, (dy * xh).sum(0), dy.sum(0) if kind == 'layer' else None


def _plain_block(s):
    """h = res_scale x + gate * norm(y) ;  u = norm(h)"""
    c = s['case']
    x, y = s['x'].float(), s['y'].float()
    n = _norm(y, s['post_w'], s['post_b'], c['kind'], s['eps'])[2]
    if s['gate'] is not None:
        n = n * s['gate'].float()
    h = s['res_scale'] * x + n
    u = _norm(h, s['pre_w'], s['pre_b'], c['kind'], s['eps'])[2]
    return h.to(s['x'].dtype), u.to(s['x'].dtype)


def _plain_block_grad(s):
    c, dt = s['case'], s['y'].dtype
    hh, rh, _ = _norm(s['h'].float(), s['pre_w'], s['pre_b'], c['kind'], s['eps'])
    dh, dpre_w, dpre_b = _norm_back(s['du'].float(), hh, rh, s['pre_w'], c['kind'])
    dh = dh + s['dh'].float()
    yh, ry, n = _norm(s['y'].float(), s['post_w'], s['post_b'], c['kind'], s['eps'])
    dgate, dn = None, dh
    if s['gate'] is not None:
        dgate = dh * n
        dgate = dgate.sum(0) if s['gate'].dim() == 1 else dgate.to(dt)
        dn = dh * s['gate'].float()
    dy, dpost_w, dpost_b = _norm_back(dn, yh, ry, s['post_w'], c['kind'])
    return dict(x=(s['res_scale'] * dh).to(dt), y=dy.to(dt), gate=dgate, post_w=dpost_w, post_b=dpost_b,
                pre_w=dpre_w, pre_b=dpre_b)


def _plain_distill(s):
    """loss_i = weight_i sum_k p_k (log p_k - log softmax(z / tau)[idx_k]);  gradient of scale sum_i loss_i"""
    c = s['case']
    tau = c['tau']
    z = s['logits'].float() / tau
    there = s['idx'] >= 0
    at = s['idx'].clamp(min=0).long()
    t = torch.where(there, s['teacher'] / tau, torch.full((), -math.inf, device=DEV))
    norm = s['lse'] if s['lse'] is not None else torch.logsumexp(t, 1)
    logp = t - norm[:, None]
    p = torch.exp(logp)
    zmax = z.max(1, keepdim=True).values
    ez = torch.exp(z - zmax)
    total = ez.sum(1, keepdim=True)
    logq = torch.gather(z, 1, at) - zmax - torch.log(total)
    loss = torch.where(p > 0, p * (logp - logq), torch.zeros((), device=DEV)).sum(1) * s['weight']
    if c['op'] == 'distill_loss':
        return loss
    grad = ez.mul_(p.sum(1, keepdim=True) / total)
    grad.scatter_add_(1, at, -p)
    grad.mul_((s['weight'] * (s['scale'] / tau))[:, None])
    return loss, grad.to(s['logits'].dtype)


# ------------------------------------------------------------------ the definitions, in 64 bits

def exact(c, seed):
    s = prepare(c, seed)
    op = c['op']
    if op.startswith('mix'):
        return _exact_mix(c, s)
    if op.startswith('block'):
        return _exact_block(c, s)
    return _exact_distill(c, s)


def _exact_mix(c, s):
    """The recurrence, one row after the other."""
    H, HK, scale = c['H'], c['HK'], s['scale']
    lam = torch.exp(s['decay'].double())[None, :, None, None]
    group = torch.arange(H, device=DEV) // (H // HK)
    q, k, v = s['q'].double(), s['k'].double(), s['v'].double()
    if c['op'] == 'mix_step':
        S = lam * s['state'].double() + torch.einsum('bhd,bhe->bhde', k[:, group], v[:, group])
        return torch.einsum('bhd,bhde->bhe', q, S) * scale, S
    B, T, D, DV = c['B'], c['T'], c['D'], c['DV']
    zero = torch.zeros(B, H, D, DV, dtype=torch.float64, device=DEV)
    first = zero if s['state'] is None else s['state'].double()
    length = torch.tensor(_lengths(c), device=DEV)
    out = torch.zeros(B, T, H, DV, dtype=torch.float64, device=DEV)
    dq = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV)
    do = s['dout'].double() if c['op'] == 'mix_grad' else None
    S = first.clone()
    for t in range(T):
        on = (t < length)[:, None, None]
        S = torch.where(on[..., None], lam * S + k[:, t, group][..., :, None] * v[:, t, group][..., None, :], S)
        if do is None:
            out[:, t] = torch.where(on, (q[:, t][..., None, :] @ S)[..., 0, :] * scale, 0.0)
        else:
            dq[:, t] = torch.where(on, (S @ do[:, t][..., :, None])[..., 0] * scale, 0.0)
    if do is None:
        return out, S
    dk = torch.zeros(B, T, HK, D, dtype=torch.float64, device=DEV)
    dv = torch.zeros(B, T, HK, DV, dtype=torch.float64, device=DEV)
    G = zero.clone() if s['dstate'] is None else s['dstate'].double()   # the gradient of the state behind row t
    for t in reversed(range(T)):
        on = (t < length)[:, None, None]
        Gt = G + scale * q[:, t][..., :, None] * do[:, t][..., None, :]
        a = (Gt @ v[:, t, group][..., :, None])[..., 0]
        b = (k[:, t, group][..., None, :] @ Gt)[..., 0, :]
        dk[:, t] = torch.where(on, a.reshape(B, HK, H // HK, D).sum(2), 0.0)
        dv[:, t] = torch.where(on, b.reshape(B, HK, H // HK, DV).sum(2), 0.0)
        G = torch.where(on[..., None], lam * Gt, G)
    return dq, dk, dv, G


def _exact_block(c, s):
    """The gradient by automatic differentiation of the forward formula."""
    layer = c['kind'] == 'layer'
    names = ['y', 'post_w', 'pre_w'] + (['post_b', 'pre_b'] if layer else []) + (['gate'] if s['gate'] is not None else [])
    leaf = {n: s[n].double() for n in names}

    def normed(x, w, b):
        if layer:
            return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, s['eps'])
        return x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + s['eps']) * w

    if c['op'] == 'block_fwd':
        h = s['res_scale'] * s['x'].double() + leaf.get('gate', 1.0) * normed(leaf['y'], leaf['post_w'], leaf.get('post_b'))
        return h, normed(h, leaf['pre_w'], leaf.get('pre_b'))
    for v in leaf.values():
        v.requires_grad_(True)
    h = s['h'].double().requires_grad_(True)
    u = normed(h, leaf['pre_w'], leaf.get('pre_b'))
    pre = [n for n in names if n.startswith('pre')]
    got = torch.autograd.grad(u, [h] + [leaf[n] for n in pre], s['du'].double())
    dh = got[0] + s['dh'].double()
    res = dict(zip(pre, got[1:]), x=s['res_scale'] * dh)
    n = leaf.get('gate', 1.0) * normed(leaf['y'], leaf['post_w'], leaf.get('post_b'))
    rest = [m for m in names if not m.startswith('pre')]
    res.update(zip(rest, torch.autograd.grad(n, [leaf[m] for m in rest], dh)))
    return {n: res.get(n) for n in ('x', 'y', 'gate', 'post_w', 'post_b', 'pre_w', 'pre_b')}


def _exact_distill(c, s):
    N, V, tau = c['N'], c['V'], c['tau']
    losses = torch.empty(N, dtype=torch.float64, device=DEV)
    grad = torch.empty(N, V, dtype=torch.float64, device=DEV) if c['op'] == 'distill_grad' else None
    for lo in range(0, N, 512):
        r = slice(lo, min(N, lo + 512))
        logq = torch.log_softmax(s['logits'][r].double() / tau, 1)
        idx, w = s['idx'][r].long(), s['weight'][r].double()
        t = (s['teacher'][r].double() / tau).masked_fill(idx < 0, -math.inf)
        logp = t - (s['lse'][r].double()[:, None] if s['lse'] is not None else torch.logsumexp(t, 1, keepdim=True))
        p = logp.exp()
        dense = torch.zeros(idx.shape[0], V + 1, dtype=torch.float64, device=DEV)
        dense.scatter_add_(1, torch.where(idx < 0, V, idx), p)
        dense = dense[:, :V]
        entropy = torch.where(p > 0, p * logp, 0.0).sum(1)
        losses[r] = w * (entropy - (dense * logq).sum(1))
        if grad is not None:
            grad[r] = (s['scale'] / tau * w)[:, None] * (dense.sum(1, keepdim=True) * logq.exp() - dense)
    return losses if grad is None else (losses, grad)

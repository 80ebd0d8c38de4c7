"""The fine-tuning operators as measured cases: log probabilities through the tied head, the preference and the clipped
policy loss, and the MLP whose activations are kept in 8 bits, each with its gradients.

`own` false: the operators in elementary torch operations, in 32 bits, rounded once at the end. `own` true: the calls a
user makes of asrn_b200. Sizes are those of this repository's models: V = 256, d = 64 (the small byte model), d = 256,
d = 512, and V = 50304, d = 768, feed-forward width 2 d.
"""
import math

import torch

own = False

BLOCK = 32                       # activations kept in 8 bits share a power-of-two scale by blocks of 32


def listed():
    return [
        # a unit-test sized byte model: three short lines, nothing to hide the launches behind
        dict(name='head small', op='head', rows=48, V=256, d=64, seq=48, prompt=0, tau=1.0),
        # ragged on every side: odd vocabulary and row count, sampling temperature, prompts left out of the loss
        dict(name='head ragged', op='head', rows=1003, V=5003, d=200, seq=59, prompt=23, tau=0.8),
        # one device batch of preference pairs on the 50304-token model: 2 x 2 sequences of 1024, half of each a prompt
        dict(name='head pairs', op='head', rows=4096, V=50304, d=768, seq=1024, prompt=512, tau=1.0),
        # a full policy batch: 16 sequences of 1024 tokens, every position counted
        dict(name='head batch', op='head', rows=16384, V=50304, d=768, seq=1024, prompt=0, tau=1.0),
        # a few pairs of short answers: one device's micro batch
        dict(name='pref small', op='pref', P=4, L=256, kind='sigmoid', beta=0.1, smoothing=0.0),
        # many long pairs, length-normalised
        dict(name='pref large', op='pref', P=512, L=4096, kind='ipo', beta=0.1, smoothing=0.0),
        # one group of answers to one prompt, an advantage for each answer
        dict(name='policy small', op='policy', B=8, L=512, per_token=False, ref=True, per='token', kl=0.04),
        # odd sizes, no reference model
        dict(name='policy ragged', op='policy', B=37, L=1111, per_token=True, ref=False, per='token', kl=0.0),
        # a rollout batch of long answers, an advantage for each token, sequences weighted alike
        dict(name='policy large', op='policy', B=512, L=8192, per_token=True, ref=True, per='sequence', kl=0.04),
        # the small byte model's MLP on one short batch
        dict(name='mlp small', op='mlp', rows=64, d=64, ff=128),
        # odd row count at the width of the 256-wide layer
        dict(name='mlp ragged', op='mlp', rows=3001, d=256, ff=520),
        # one block of the 768-wide model on 4 sequences of 8192
        dict(name='mlp large', op='mlp', rows=32768, d=768, ff=1536),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['head', 'pref', 'policy', 'mlp'])
    if op == 'head':
        while True:
            rows, V, d = _log(rng, 1, 16384), _log(rng, 200, 65536), 8 * _log(rng, 4, 128)
            if rows * V * d <= 16384 * 50304 * 768:
                break
        seq = _log(rng, 8, 2048)
        return dict(op=op, rows=rows, V=V, d=d, seq=seq, prompt=min(seq, rows) // rng.choice([2, 3, 1 << 20]),
                    tau=rng.choice([1.0, 0.8, 1.3]))
    if op == 'pref':
        while True:
            P, L = _log(rng, 1, 2048), _log(rng, 1, 8192)
            if P * L <= 512 * 4096:
                break
        return dict(op=op, P=P, L=L, kind=rng.choice(['sigmoid', 'ipo']), beta=rng.choice([0.05, 0.1, 0.5]),
                    smoothing=rng.choice([0.0, 0.1]))
    if op == 'policy':
        while True:
            B, L = _log(rng, 1, 4096), _log(rng, 1, 16384)
            if B * L <= 512 * 8192:
                break
        ref = rng.random() < 0.7
        return dict(op=op, B=B, L=L, per_token=rng.random() < 0.5, ref=ref, per=rng.choice(['token', 'sequence']),
                    kl=rng.choice([0.02, 0.04, 0.1]) if ref else 0.0)
    while True:
        rows, d = _log(rng, 1, 32768), 8 * _log(rng, 4, 128)
        ff = 8 * rng.randint(d // 8, d // 2)
        if rows * d * ff <= 32768 * 768 * 1536:
            break
    return dict(op=op, rows=rows, d=d, ff=ff)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _ranges(B, L, g):
    """Per row the answer's first and one-past-last position: a prompt, an answer, padding; every 16th row is empty."""
    start = (torch.rand(B, generator=g, device='cuda') * 0.5 * L).long()
    end = (start + 1 + (torch.rand(B, generator=g, device='cuda') * (L - start)).long()).clamp(max=L)
    empty = (torch.arange(B, device='cuda') % 16) == 15
    t = torch.arange(L, device='cuda')
    return (t >= start[:, None]) & (t < end[:, None]) & ~empty[:, None]


def prepare(case, seed):
    g = torch.Generator('cuda').manual_seed(int(seed))
    rn = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    op = case['op']
    if op == 'head':
        N, V, d = case['rows'], case['V'], case['d']
        w = (rn(V, d) * 0.06).bfloat16()
        y = torch.randint(0, V, (N,), generator=g, device='cuda')
        # half of the positions predict their token well, as a trained model's do
        h = rn(N, d)
        sure = torch.rand(N, generator=g, device='cuda') < 0.5
        h = (h + sure[:, None] * (8.0 / (0.06 ** 2 * d)) * w[y].float()).bfloat16()
        y = torch.where(torch.arange(N, device='cuda') % case['seq'] < case['prompt'], -1, y)
        grad = rn(N) / N
        return dict(case=case, h=h.requires_grad_(), w=w.requires_grad_(), y=y, g=grad)
    if op == 'pref':
        P, L = case['P'], case['L']
        ref = -torch.rand(2, P, L, generator=g, device='cuda') * 5
        logp = ref + 0.1 * rn(2, P, L) + torch.tensor([0.01, -0.01], device='cuda')[:, None, None]
        mask = torch.stack([_ranges(P, L, g), _ranges(P, L, g)])
        return dict(case=case, logp=logp * mask, ref=ref * mask, mask=mask)
    if op == 'policy':
        B, L = case['B'], case['L']
        old = -torch.rand(B, L, generator=g, device='cuda') * 5
        logp = old + 0.15 * rn(B, L)
        mask = _ranges(B, L, g)
        adv = rn(B, L) if case['per_token'] else rn(B)
        ref = (old + 0.3 * rn(B, L)) * mask if case['ref'] else None
        return dict(case=case, logp=logp * mask, old=old * mask, adv=adv, mask=mask, ref=ref)
    N, d, ff = case['rows'], case['d'], case['ff']
    s = dict(x=rn(N, d).bfloat16(), w1=(rn(ff, d) / d ** 0.5).bfloat16(), b1=(0.1 * rn(ff)).bfloat16(),
             w2=(rn(d, ff) / ff ** 0.5).bfloat16(), b2=(0.1 * rn(d)).bfloat16())
    s = {k: v.requires_grad_() for k, v in s.items()}
    return dict(case=case, dy=(rn(N, d) / N).bfloat16(), **s)


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    op = s['case']['op']
    if own:
        return _own(s['case'], s)
    return {'head': _head, 'pref': _pref, 'policy': _policy, 'mlp': _mlp}[op](s['case'], s)


def _own(c, s):
    import asrn_b200 as asrn
    if c['op'] == 'head':
        logp = asrn.head_logprobs(s['h'], s['w'], s['y'], temperatura=c['tau'])
        dh, dw = torch.autograd.grad(logp, (s['h'], s['w']), s['g'])
        return dict(logp=logp, dh=dh, dw=dw)
    if c['op'] == 'pref':
        r = asrn.preference_loss(s['logp'], s['ref'], s['mask'], beta=c['beta'], smoothing=c['smoothing'],
                                 kind=c['kind'])
        return dict(loss=r.loss, grad=r.grad, chosen=r.chosen, rejected=r.rejected)
    if c['op'] == 'policy':
        r = asrn.policy_loss(s['logp'], s['old'], s['adv'], s['mask'], ref_logp=s['ref'], kl=c['kl'], per=c['per'])
        return dict(loss=r.loss, grad=r.grad, kl=r.kl, clipped=r.clipped)
    y = asrn.mlp8(s['x'], s['w1'], s['b1'], s['w2'], s['b2'])
    dx, dw1, db1, dw2, db2 = torch.autograd.grad(y, (s['x'], s['w1'], s['b1'], s['w2'], s['b2']), s['dy'])
    return dict(y=y, dx=dx, dw1=dw1, db1=db1, dw2=dw2, db2=db2)


@torch.no_grad()
def _head(c, s):
    h, w, y, tau = s['h'].float(), s['w'].float(), s['y'], c['tau']
    on = y >= 0
    at = y.clamp(min=0)[:, None]
    z = h @ w.t() / tau
    top = z.amax(1, keepdim=True)
    own_z = z.gather(1, at)
    e = torch.exp(z - top)
    tot = e.sum(1, keepdim=True)
    logp = torch.where(on, (own_z - top - torch.log(tot))[:, 0], 0.0)
    g = torch.where(on, s['g'], 0.0)[:, None] / tau
    dz = e * (-g / tot)
    dz.scatter_add_(1, at, g)
    return dict(logp=logp, dh=(dz @ w).bfloat16(), dw=(dz.t() @ h).bfloat16())


@torch.no_grad()
def _pref(c, s):
    beta, eps = c['beta'], c['smoothing']
    diff = torch.where(s['mask'], s['logp'] - s['ref'], 0.0)
    n = s['mask'].sum(2)                                            # (2, P) tokens of each answer
    tot = diff.sum(2)
    on = (n > 0).all(0)
    pairs = on.sum().clamp(min=1)
    if c['kind'] == 'ipo':
        den = n.clamp(min=1).float()
        gap = tot[0] / den[0] - tot[1] / den[1] - 1 / (2 * beta)
        each, slope = gap * gap, 2 * gap / den
    else:
        x = beta * (tot[0] - tot[1])
        low, soft = x.clamp(max=0), torch.log(1 + torch.exp(-x.abs()))
        each = (1 - eps) * (soft - low) + eps * (soft + x - low)    # -(1-e) log sigma(x) - e log sigma(-x)
        up = 1 / (1 + torch.exp(x))                                 # sigma(-x)
        slope = (beta * (eps - up)).expand(2, -1)
    loss = torch.where(on, each, 0.0).sum() / pairs
    slope = torch.where(on, slope, 0.0) / pairs
    sign = torch.tensor([1.0, -1.0], device=slope.device)[:, None]
    grad = (slope * sign)[:, :, None] * s['mask']
    return dict(loss=loss, grad=grad, chosen=beta * tot[0], rejected=beta * tot[1])


@torch.no_grad()
def _policy(c, s):
    m = s['mask']
    adv = s['adv'] if c['per_token'] else s['adv'][:, None]
    lr = torch.where(m, s['logp'] - s['old'], 0.0).clamp(-20, 20)
    r = torch.exp(lr)
    low, high = math.log1p(-0.2), math.log1p(0.2)
    cut = ((adv > 0) & (lr > high)) | ((adv < 0) & (lr < low))
    kept = torch.where(cut, torch.exp(lr.clamp(low, high)), r) * adv
    each, slope = -kept, torch.where(cut, 0.0, -r * adv)
    if c['ref']:
        q = torch.where(m, s['ref'] - s['logp'], 0.0).clamp(-20, 20)
        k3 = torch.exp(q) - q - 1
        each, slope = each + c['kl'] * k3, slope + c['kl'] * (1 - torch.exp(q))
    else:
        k3 = torch.zeros_like(lr)
    n = m.sum(1)
    if c['per'] == 'sequence':
        weight = torch.where(n > 0, 1 / n.clamp(min=1), 0.0)[:, None] / (n > 0).sum().clamp(min=1)
    else:
        weight = 1 / n.sum().clamp(min=1)
    total = n.sum().clamp(min=1)
    return dict(loss=torch.where(m, each * weight, 0.0).sum(), grad=torch.where(m, slope * weight, 0.0),
                kl=torch.where(m, k3, 0.0).sum() / total, clipped=(cut & m).sum() / total)


def _kept(v):
    """The values that 8-bit blocks of 32 with a power-of-two scale stand for."""
    n, f = v.shape
    pad = -f % BLOCK
    b = torch.nn.functional.pad(v, (0, pad)).view(n, -1, BLOCK)
    top = b.abs().amax(2, keepdim=True)
    _, e = torch.frexp(top)
    e = e - 7                                                       # 2^(e-1) <= top < 2^e: top 2^(7-e) < 128
    e = e + (torch.ldexp(top, -e) > 127)
    return torch.ldexp(torch.round(torch.ldexp(b, -e)), e).reshape(n, f + pad)[:, :f]


_SQRT2, _SQRT2PI = math.sqrt(2.0), math.sqrt(2 * math.pi)


@torch.no_grad()
def _mlp(c, s):
    x, w1, b1, w2, b2, dy = (s[k].float() for k in ('x', 'w1', 'b1', 'w2', 'b2', 'dy'))
    a = x @ w1.t() + b1
    y = (a * (0.5 + 0.5 * torch.erf(a / _SQRT2))) @ w2.t() + b2
    ak, xk = _kept(a), _kept(x)
    cdf = 0.5 + 0.5 * torch.erf(ak / _SQRT2)
    da = (dy @ w2) * (cdf + ak * torch.exp(-0.5 * ak * ak) / _SQRT2PI)
    out = dict(y=y, dx=da @ w1, dw1=da.t() @ xk, db1=da.sum(0), dw2=dy.t() @ (ak * cdf), db2=dy.sum(0))
    return {k: v.bfloat16() for k, v in out.items()}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    return {'head': _exact_head, 'pref': _exact_pref, 'policy': _exact_policy, 'mlp': _exact_mlp}[case['op']](case, s)


def _exact_head(c, s):
    logp, dh, dw = [], [], torch.zeros_like(s['w'])
    for i in range(0, c['rows'], 2048):                             # rows do not touch one another
        h, y, g = s['h'][i:i + 2048], s['y'][i:i + 2048], s['g'][i:i + 2048]
        on = (y >= 0).double()
        lp = torch.log_softmax(h @ s['w'].t() / c['tau'], 1)
        pick = torch.zeros_like(lp)
        pick[torch.arange(len(y), device=y.device), y.clamp(min=0)] = on
        logp.append((lp * pick).sum(1))
        dz = (pick - on[:, None] * lp.exp()) * (g / c['tau'])[:, None]
        dh.append(dz @ s['w'])
        dw += dz.t() @ h
    return dict(logp=torch.cat(logp), dh=torch.cat(dh), dw=dw)


def _exact_pref(c, s):
    logp = s['logp'].requires_grad_()
    m = s['mask'].double()
    n = m.sum(2)
    R = ((logp - s['ref']) * m).sum(2)
    on = (n[0] > 0) & (n[1] > 0)
    if c['kind'] == 'ipo':
        means = R / n.clamp(min=1)
        each = (means[0] - means[1] - 0.5 / c['beta']) ** 2
    else:
        x = c['beta'] * (R[0] - R[1])
        each = -(1 - c['smoothing']) * torch.nn.functional.logsigmoid(x) \
            - c['smoothing'] * torch.nn.functional.logsigmoid(-x)
    loss = each[on].sum() / max(1, int(on.sum()))
    grad, = torch.autograd.grad(loss, logp)
    return dict(loss=loss, grad=grad, chosen=c['beta'] * R[0].detach(), rejected=c['beta'] * R[1].detach())


def _exact_policy(c, s):
    m = s['mask']
    logp = s['logp'].requires_grad_()
    A = (s['adv'] if c['per_token'] else s['adv'][:, None].expand(c['B'], c['L']))[m]
    r = torch.exp((logp - s['old'])[m])
    clip = r.clamp(0.8, 1.2)
    each = -torch.minimum(r * A, clip * A)
    k3 = torch.zeros_like(each)
    if c['ref']:
        q = (s['ref'] - logp)[m]
        k3 = torch.expm1(q) - q
        each = each + c['kl'] * k3
    n = m.sum(1)
    if c['per'] == 'sequence':
        weight = (1.0 / n.clamp(min=1).double() / max(1, int((n > 0).sum())))[:, None].expand(c['B'], c['L'])[m]
    else:
        weight = 1.0 / max(1, int(n.sum()))
    loss = (each * weight).sum()
    grad, = torch.autograd.grad(loss, logp)
    total = max(1, int(n.sum()))
    return dict(loss=loss, grad=grad, kl=k3.detach().sum() / total,
                clipped=((clip * A < r * A).double().sum() / total))


def _exact_mlp(c, s):
    def eight(v):
        n, f = v.shape
        blocks = torch.nn.functional.pad(v, (0, -f % 32)).unflatten(1, (-1, 32))
        top = blocks.abs().amax(2, keepdim=True)
        scale = torch.exp2(torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 127)))
        scale = torch.where(127 * scale < top, 2 * scale, scale)
        return (torch.round(blocks / scale) * scale).flatten(1)[:, :f]
    gelu = torch.nn.functional.gelu
    a = torch.addmm(s['b1'], s['x'], s['w1'].t())
    y = torch.addmm(s['b2'], gelu(a), s['w2'].t())
    ak, xk = eight(a).requires_grad_(), eight(s['x'])
    gk = gelu(ak)
    da, = torch.autograd.grad(gk, ak, s['dy'] @ s['w2'])
    return dict(y=y, dx=da @ s['w1'], dw1=da.t() @ xk, db1=da.sum(0), dw2=s['dy'].t() @ gk.detach(),
                db2=s['dy'].sum(0))


# ---- what one pass cannot do without --------------------------------------------------------------------------------

def work(case):
    c = case
    if c['op'] == 'head':
        N, V, d = c['rows'], c['V'], c['d']
        active = sum(1 for i in range(N) if i % c['seq'] >= c['prompt'])
        return {'bytes': 4 * N * d + 4 * V * d + 16 * N, 'flops': 6 * active * V * d}
    if c['op'] == 'pref':
        n = 2 * c['P'] * c['L']
        return {'bytes': 13 * n + 8 * c['P'], 'flops': 4 * n}
    if c['op'] == 'policy':
        n = c['B'] * c['L']
        return {'bytes': n * (13 + 4 * bool(c['ref']) + 4 * bool(c['per_token'])) + 4 * c['B'], 'flops': 16 * n}
    N, d, ff = c['rows'], c['d'], c['ff']
    return {'bytes': 2 * (4 * N * d + 4 * d * ff + 2 * (d + ff)), 'flops': 12 * N * d * ff}

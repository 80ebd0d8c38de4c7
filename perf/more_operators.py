"""More operators of the model's training and answering as measured cases: layer norm with the residual sum before it, the
matrix product with bias, activation and residual in its epilogue, and log probabilities through the tied head with the
distribution's entropy and its likeliest tokens. With gradients where a training step calls them, without where a step of
generation does.

`own` false: the operators in elementary torch operations, in 32 bits, rounded once at the end (scores of the likeliest
tokens, which stand next to one another, in 64). `own` true: the calls a user makes of asrn_b200. Sizes are those of this
repository's models: V = 256, d = 64 (the small byte model), d = 256, d = 512, and V = 50304, d = 768, feed-forward width
2 d; batches of 64 sequences in generation, 4 x 8192 tokens in training.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}


def listed():
    return [
        # one generation step of 64 sequences: the local block's sum of stream and branch, and the norm before the MLP
        dict(name='norm step', op='norm', rows=64, d=768, x='bf16', res='f32', y='bf16', bias=True, grad=False),
        # odd width and row count, no sum before it: the norm of a short fp32 batch
        dict(name='norm ragged', op='norm', rows=3001, d=257, x='f32', res='none', y='f32', bias=True, grad=True),
        # a norm whose rows are wider than the model, bf16 stream, no bias
        dict(name='norm wide', op='norm', rows=1500, d=5000, x='bf16', res='bf16', y='bf16', bias=False, grad=True),
        # one block's second norm in a training step of 4 sequences of 8192
        dict(name='norm large', op='norm', rows=32768, d=768, x='bf16', res='f32', y='bf16', bias=True, grad=True),
        # the MLP's first product for a single token
        dict(name='linear token', op='linear', rows=1, d=768, n=1536, act='gelu', res='none', bias=True, grad=False),
        # the MLP's second product in a generation step of 64 sequences
        dict(name='linear step', op='linear', rows=64, d=1536, n=768, act='none', res='f32', bias=True, grad=False),
        # ragged on every side, another activation, no bias
        dict(name='linear ragged', op='linear', rows=1003, d=200, n=520, act='silu', res='bf16', bias=False, grad=True),
        # the MLP's two products in a training step of 4 sequences of 8192
        dict(name='linear up', op='linear', rows=32768, d=768, n=1536, act='gelu', res='none', bias=True, grad=True),
        dict(name='linear down', op='linear', rows=32768, d=1536, n=768, act='none', res='f32', bias=True, grad=True),
        # answers of 8 sequences that show each token's alternatives: one step, no targets
        dict(name='stats step', op='stats', rows=8, V=50304, d=768, seq=1, prompt=0, tau=1.0, top=5, targets=False,
             grad=False),
        # odd vocabulary, prompts left out, entropy in the loss
        dict(name='stats ragged', op='stats', rows=1003, V=5003, d=200, seq=59, prompt=23, tau=0.8, top=3, targets=True,
             grad=True),
        # a full policy batch with an entropy bonus and a log of the alternatives: 16 sequences of 1024 tokens
        dict(name='stats batch', op='stats', rows=16384, V=50304, d=768, seq=1024, prompt=0, tau=1.0, top=8, targets=True,
             grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['norm', 'linear', 'stats'])
    if op == 'norm':
        while True:
            rows, d = _log(rng, 1, 65536), _log(rng, 2, 8192)
            if rows * d <= 32768 * 768:
                break
        return dict(op=op, rows=rows, d=d, x=rng.choice(['f32', 'bf16']), res=rng.choice(['none', 'f32', 'bf16']),
                    y=rng.choice(['f32', 'bf16']), bias=rng.random() < 0.7, grad=rng.random() < 0.7)
    if op == 'linear':
        while True:
            rows, d, n = _log(rng, 1, 32768), 8 * _log(rng, 4, 256), 8 * _log(rng, 4, 256)
            if rows * d * n <= 32768 * 768 * 1536:
                break
        return dict(op=op, rows=rows, d=d, n=n, act=rng.choice(['none', 'gelu', 'silu', 'relu']),
                    res=rng.choice(['none', 'f32', 'bf16']), bias=rng.random() < 0.7, grad=rng.random() < 0.6)
    while True:
        rows, V, d = _log(rng, 1, 16384), _log(rng, 200, 65536), 8 * _log(rng, 4, 128)
        if rows * V * d <= 16384 * 50304 * 768:
            break
    seq, targets = _log(rng, 8, 2048), rng.random() < 0.7
    prompt = min(seq, rows) // rng.choice([2, 3, 1 << 20]) if targets else 0
    return dict(op=op, rows=rows, V=V, d=d, seq=seq, prompt=prompt, tau=rng.choice([1.0, 0.8, 1.3]),
                top=rng.choice([0, 1, 5, 8, 20]), targets=targets, grad=rng.random() < 0.6)


# ---- inputs ---------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator('cuda').manual_seed(int(seed))
    rn = lambda *s: torch.randn(*s, generator=g, device='cuda')  # noqa: E731
    c, op = case, case['op']
    leaf = lambda t, kind='bf16': t.to(TYPES[kind]).requires_grad_(c['grad'])  # noqa: E731
    if op == 'norm':
        N, d = c['rows'], c['d']
        # a stream as deep models have it: every channel with its own mean and size, some of them large
        size = torch.exp(0.5 * rn(d)) * torch.where(torch.rand(d, generator=g, device='cuda') < 0.01, 20.0, 1.0)
        stream = rn(N, d) * size + 0.3 * rn(d)
        s = dict(case=c, w=leaf(1 + 0.2 * rn(d), 'f32'), b=leaf(0.1 * rn(d), 'f32') if c['bias'] else None)
        if c['res'] == 'none':
            s.update(x=leaf(stream, c['x']), res=None)
        else:
            s.update(x=leaf(0.3 * rn(N, d), c['x']), res=leaf(stream, c['res']))
        if c['grad']:
            s.update(dy=(rn(N, d) / N).to(TYPES[c['y']]),
                     ds=(rn(N, d) / N).to(TYPES[c['res']]) if c['res'] != 'none' else None)
        return s
    if op == 'linear':
        N, d, n = c['rows'], c['d'], c['n']
        s = dict(case=c, x=leaf(rn(N, d)), w=leaf(rn(n, d) / d ** 0.5), b=leaf(0.1 * rn(n)) if c['bias'] else None,
                 res=leaf(rn(N, n), c['res']) if c['res'] != 'none' else None)
        if c['grad']:
            s['dy'] = (rn(N, n) / N).to(TYPES['bf16' if c['res'] == 'none' else c['res']])
        return s
    N, V, d = c['rows'], c['V'], c['d']
    w = (rn(V, d) * 0.06).bfloat16()
    y = torch.randint(0, V, (N,), generator=g, device='cuda')
    # half of the positions predict a token well, as a trained model's do
    sure = torch.rand(N, generator=g, device='cuda') < 0.5
    h = (rn(N, d) + sure[:, None] * (8.0 / (0.06 ** 2 * d)) * w[y].float()).bfloat16()
    y = torch.where(torch.arange(N, device='cuda') % c['seq'] < c['prompt'], -1, y) if c['targets'] else None
    s = dict(case=c, h=leaf(h), w=leaf(w), y=y)
    if c['grad']:
        s.update(g=rn(N) / N if c['targets'] else None, gh=0.05 * rn(N) / N)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s['case'], s)
    return {'norm': _norm, 'linear': _linear, 'stats': _stats}[s['case']['op']](s['case'], s)


def _given(**tensors):
    return {k: v for k, v in tensors.items() if v is not None}


def _own(c, s):
    import asrn_b200 as asrn
    if c['op'] == 'norm':
        r = asrn.layer_norm(s['x'], s['w'], s['b'], residual=s['res'], eps=EPS, dtype=TYPES[c['y']])
        out = dict(y=r) if s['res'] is None else dict(y=r[0], s=r[1])
        into = _given(dx=s['x'], dres=s['res'], dw=s['w'], db=s['b'])
        up = None if not c['grad'] else (s['dy'],) if s['res'] is None else (s['dy'], s['ds'])
    elif c['op'] == 'linear':
        act = None if c['act'] == 'none' else c['act']
        out = dict(y=asrn.linear(s['x'], s['w'], s['b'], activation=act, residual=s['res']))
        into = _given(dx=s['x'], dw=s['w'], db=s['b'], dres=s['res'])
        up = (s['dy'],) if c['grad'] else None
    else:
        r = asrn.head_stats(s['h'], s['w'], s['y'], temperatura=c['tau'], top=c['top'])
        out = _given(entropy=r.entropy, logp=r.logp)
        into = dict(dh=s['h'], dw=s['w'])
        if c['grad']:
            grads = torch.autograd.grad(tuple(out.values()), tuple(into.values()),
                                        (s['gh'],) if s['y'] is None else (s['gh'], s['g']))
            out.update(zip(into, grads))
        if c['top']:
            out.update(top_logp=r.top_logp, top_tokens=r.top_tokens)
        return out
    if c['grad']:
        out.update(zip(into, torch.autograd.grad(tuple(out.values()), tuple(into.values()), up)))
    return out


@torch.no_grad()
def _norm(c, s):
    x, w = s['x'].float(), s['w'].float()
    out = {}
    if s['res'] is not None:
        sent = (x + s['res'].float()).to(s['res'].dtype)
        out['s'] = sent
        x = sent.float()
    mid = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((mid * mid).mean(1, keepdim=True) + EPS)
    hat = mid * rstd
    y = hat * w
    if s['b'] is not None:
        y = y + s['b'].float()
    out['y'] = y.to(TYPES[c['y']])
    if c['grad']:
        dy = s['dy'].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
        if s['res'] is not None:
            dx = dx + s['ds'].float()
            out['dres'] = dx.to(s['res'].dtype)
        out.update(dx=dx.to(s['x'].dtype), dw=(dy * hat).sum(0))
        if s['b'] is not None:
            out['db'] = dy.sum(0)
    return out


_SQRT2, _SQRT2PI = math.sqrt(2.0), math.sqrt(2 * math.pi)


def _act(kind, a):
    """The activation and its slope."""
    if kind == 'gelu':
        cdf = 0.5 + 0.5 * torch.erf(a / _SQRT2)
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / _SQRT2PI
    if kind == 'silu':
        p = 1 / (1 + torch.exp(-a))
        return a * p, p * (1 + a * (1 - p))
    if kind == 'relu':
        return a.clamp(min=0), (a > 0).float()
    return a, None


@torch.no_grad()
def _linear(c, s):
    x, w = s['x'].float(), s['w'].float()
    a = x @ w.t()
    if s['b'] is not None:
        a = a + s['b'].float()
    y, slope = _act(c['act'], a)
    if s['res'] is not None:
        y = y + s['res'].float()
    out = dict(y=y.to(torch.bfloat16 if s['res'] is None else s['res'].dtype))
    if c['grad']:
        da = s['dy'].float()
        if s['res'] is not None:
            out['dres'] = s['dy']
        if slope is not None:
            da = da * slope
        out.update(dx=(da @ w).bfloat16(), dw=(da.t() @ x).bfloat16())
        if s['b'] is not None:
            out['db'] = da.sum(0).bfloat16()
    return out


@torch.no_grad()
def _stats(c, s):
    h, w, y, tau, V = s['h'].float(), s['w'].float(), s['y'], c['tau'], c['V']
    on = torch.ones(len(h), dtype=torch.bool, device=h.device) if y is None else y >= 0
    z = h @ w.t() / tau
    top = z.amax(1, keepdim=True)
    out = {}
    if c['top']:
        # the likeliest few by the fp32 scores, then in the order of their scores in 64 bits, equal ones by their number
        few = z.topk(min(V, c['top'] + 8), 1).indices.sort(dim=1).values
        exact = torch.cat([(w[f].double() * r.double()[:, None]).sum(2)
                           for f, r in zip(few.split(2048), h.split(2048))]) / tau
        best, at = exact.sort(dim=1, descending=True, stable=True)
        best, tokens = best[:, :c['top']], few.gather(1, at)[:, :c['top']]
    e = torch.exp(z - top)
    tot = e.sum(1, keepdim=True)
    lp = z - top - torch.log(tot)
    p = e / tot
    H = -(p * lp).sum(1, keepdim=True)
    out['entropy'] = torch.where(on, H[:, 0], 0.0)
    if c['top']:
        best = (best - top.double() - torch.log(tot).double()).float()
        out['top_logp'] = torch.where(on[:, None], best, 0.0)
        out['top_tokens'] = torch.where(on[:, None], tokens, -1)
    if y is not None:
        at = y.clamp(min=0)[:, None]
        out['logp'] = torch.where(on, lp.gather(1, at)[:, 0], 0.0)
    if c['grad']:
        gh = (torch.where(on, s['gh'], 0.0) / tau)[:, None]
        dz = -gh * p * (lp + H)
        if y is not None:
            g = (torch.where(on, s['g'], 0.0) / tau)[:, None]
            dz = dz - g * p
            dz.scatter_add_(1, at, g)
        out.update(dh=(dz @ w).bfloat16(), dw=(dz.t() @ h).bfloat16())
    return out


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach().double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    return {'norm': _exact_norm, 'linear': _exact_linear, 'stats': _exact_stats}[case['op']](case, s)


def _exact_norm(c, s):
    leaves = {k: s[k].requires_grad_() for k in ('x', 'res', 'w', 'b') if s[k] is not None}
    total = s['x'] if s['res'] is None else s['x'] + s['res']
    # what is normalised is the sum as it is handed on
    held = total if c['res'] != 'bf16' else total + (total.detach().float().bfloat16().double() - total.detach())
    y = torch.nn.functional.layer_norm(held, (c['d'],), s['w'], s['b'], EPS)
    out = dict(y=y.detach()) if s['res'] is None else dict(y=y.detach(), s=total.detach())
    if c['grad']:
        loss = (y * s['dy']).sum() if s['res'] is None else (y * s['dy']).sum() + (held * s['ds']).sum()
        names = dict(x='dx', res='dres', w='dw', b='db')
        for (k, _), grad in zip(leaves.items(), torch.autograd.grad(loss, tuple(leaves.values()))):
            out[names[k]] = grad
    return out


def _exact_linear(c, s):
    F = torch.nn.functional
    a = F.linear(s['x'], s['w'], s['b']).requires_grad_()
    act = {'none': lambda t: t * 1.0, 'gelu': F.gelu, 'silu': F.silu, 'relu': F.relu}[c['act']]
    f = act(a)
    out = dict(y=f.detach() if s['res'] is None else f.detach() + s['res'])
    if c['grad']:
        da, = torch.autograd.grad(f, a, s['dy'])
        out.update(dx=da @ s['w'], dw=da.t() @ s['x'])
        if s['b'] is not None:
            out['db'] = da.sum(0)
        if s['res'] is not None:
            out['dres'] = s['dy']
    return out


def _exact_stats(c, s):
    k, tau, y = c['top'], c['tau'], s['y']
    parts, dw = [], torch.zeros_like(s['w'])
    for i in range(0, c['rows'], 2048):                             # rows do not touch one another
        h = s['h'][i:i + 2048]
        on = torch.ones(len(h), device=h.device).double() if y is None else (y[i:i + 2048] >= 0).double()
        z = h @ s['w'].t()
        lp = torch.log_softmax(z / tau, 1)
        p = lp.exp()
        H = -(p * lp).sum(1)
        part = dict(entropy=H * on)
        if k:
            left, found = z.clone(), []
            for _ in range(k):                                      # the first of equal ones each time
                found.append(left.argmax(1, keepdim=True))
                left.scatter_(1, found[-1], -math.inf)
            found = torch.cat(found, 1)
            part.update(top_logp=lp.gather(1, found) * on[:, None], top_tokens=torch.where(on[:, None] > 0, found, -1))
        dz = torch.zeros_like(z)
        if c['grad']:
            dz -= (s['gh'][i:i + 2048] * on)[:, None] * p * (lp + H[:, None])
        if y is not None:
            pick = torch.zeros_like(lp)
            pick[torch.arange(len(h), device=h.device), y[i:i + 2048].clamp(min=0)] = on
            part['logp'] = (lp * pick).sum(1)
            if c['grad']:
                dz += s['g'][i:i + 2048, None] * (pick - on[:, None] * p)
        if c['grad']:
            part['dh'] = dz @ s['w'] / tau
            dw += dz.t() @ h / tau
        parts.append(part)
    out = {key: torch.cat([p[key] for p in parts]) for key in parts[0]}
    if c['grad']:
        out['dw'] = dw
    return out


# ---- what one pass cannot do without --------------------------------------------------------------------------------

def work(case):
    c, grad = case, case['grad']
    size = {'f32': 4, 'bf16': 2, 'none': 0}
    if c['op'] == 'norm':
        e, params = c['rows'] * c['d'], 4 * c['d'] * (1 + c['bias'])
        b = e * (size[c['x']] + 2 * size[c['res']] + size[c['y']]) + params
        if grad:                                 # reads dy and ds; writes dx, dres, dw, db
            b += e * (size[c['y']] + size[c['x']] + 2 * size[c['res']]) + params
        return {'bytes': b, 'flops': e * (20 if grad else 8)}
    if c['op'] == 'linear':
        N, d, n = c['rows'], c['d'], c['n']
        y = size[c['res']] or 2
        b = 2 * (N * d + n * d + n * c['bias']) + N * n * (y + size[c['res']])
        if grad:                                 # reads dy; writes dx, dw, db (the residual's gradient is dy itself)
            b += N * n * y + 2 * (N * d + n * d + n * c['bias'])
        return {'bytes': b, 'flops': (6 if grad else 2) * N * d * n}
    N, V, d = c['rows'], c['V'], c['d']
    active = sum(1 for i in range(N) if i % c['seq'] >= c['prompt']) if c['targets'] else N
    b = 2 * N * d + 2 * V * d + N * (4 + 12 * c['targets'] + 12 * c['top'])
    if grad:
        b += 2 * N * d + 2 * V * d + N * (4 + 4 * c['targets'])
    return {'bytes': b, 'flops': (6 if grad else 2) * active * V * d}

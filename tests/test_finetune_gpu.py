"""The fine-tuning operators (asrn_b200.finetune) against plain implementations in 64 bits, at the sizes and masks where
they can go wrong. Bounds, with u = 2^-8 the unit roundoff of bf16 (8 bits of significand) and e = 2^-24 that of fp32:
  scores      d products summed in fp32, 16 at a time, truncated: at most (d / 16 + 2) 2 e sum|h w|, twice that for a
              score and the log of the sum; exp2's and the logarithm's own errors a few e of 1 + |logp|
  products    of one operand rounded to bf16, result rounded to bf16: u (|result| + sum |a b|); the fp32 sums' and the
              second-order terms are far below what separates this worst case from what rounding errors do
  losses      fp64 sums of fp32 terms: a few e relative to the largest term"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -24


def rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


# ---- head ---------------------------------------------------------------------------------------------------------------

def head_reference(h, w, y, g, tau):
    h, w, g = h.double(), w.double(), g.double()
    lp = torch.log_softmax(h @ w.t() / tau, 1)
    on = (y >= 0)
    pick = torch.nn.functional.one_hot(y.clamp(min=0), w.shape[0]).double() * on[:, None]
    other = lp.exp() * (1 - pick) * on[:, None]                # 1 - p_y as the others' sum: 1 - exp would cancel
    ds = (pick * other.sum(1, keepdim=True) - other) * (g / tau)[:, None]
    size = (h.abs() @ w.abs().t()).amax() / tau
    return (lp * pick).sum(1), ds, ds @ w, ds.t() @ h, float(size)


def check_head(h, w, y, g, tau=1.0):
    import asrn_b200 as asrn
    h, w = h.detach().requires_grad_(), w.detach().requires_grad_()
    logp = asrn.head_logprobs(h, w, y, temperatura=tau)
    dh, dw = torch.autograd.grad(logp, (h, w), g)
    ref, ds, rh, rw, size = head_reference(h.detach(), w.detach(), y, g, tau)
    d = h.shape[1]
    tol = 4 * E * (d / 16 + 2) * size + 16 * E * (1 + ref.abs())
    assert ((logp.double() - ref).abs() <= tol).all(), (logp.double() - ref).abs().max()
    assert (logp[y < 0] == 0).all() and (dh[y < 0] == 0).all()
    tiny = 1e-30
    assert ((dh.double() - rh).abs() <= U * (rh.abs() + ds.abs() @ w.double().abs()) + tiny).all()
    assert ((dw.double() - rw).abs() <= U * (rw.abs() + ds.abs().t() @ h.double().abs()) + tiny).all()
    return logp, dh, dw


@pytest.mark.parametrize('N,V,d,skip', [
    (1, 1, 8, 0), (1, 200, 32, 0), (2, 3, 64, 0), (7, 257, 64, 3), (48, 256, 64, 0), (127, 129, 72, 2),
    (128, 512, 128, 0), (129, 1000, 200, 5), (256, 255, 768, 0), (257, 5003, 96, 2), (600, 513, 1024, 7),
    (1100, 70001, 64, 3), (1025, 777, 40, 2), (3000, 256, 256, 0)])
def test_head_sizes(cuda, N, V, d, skip):
    h, w = rand((N, d), 1), rand((V, d), 2, 0.1)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(3)).cuda()
    if skip:
        y[torch.arange(N, device='cuda') % skip == skip - 1] = -100
    check_head(h, w, y, rand((N,), 4, dtype=torch.float32))


@pytest.mark.parametrize('tau', [0.25, 0.8, 3.0])
def test_head_temperature_and_peaked_scores(cuda, tau):
    """Scores of a trained model: the target's probability near 1, and others far below."""
    N, V, d = 300, 3001, 128
    w = rand((V, d), 5, 0.3)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(6)).cuda()
    h = (rand((N, d), 7, dtype=torch.float32) + 3 * w[y].float()).bfloat16()
    check_head(h, w, y, rand((N,), 8, dtype=torch.float32), tau)


@pytest.mark.parametrize('which', ['all', 'first', 'last', 'one'])
def test_head_rows_without_a_target(cuda, which):
    N, V, d = 400, 300, 64
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(9)).cuda()
    keep = torch.zeros(N, dtype=torch.bool, device='cuda')
    if which == 'first':
        keep[:130] = True
    elif which == 'last':
        keep[-1:] = True
    elif which == 'one':
        keep[200] = True
    y[~keep] = -1
    h = rand((N, d), 10)
    h[~keep] = float('nan')                   # what an ignored row holds reaches nothing
    import asrn_b200 as asrn
    w = rand((V, d), 11, 0.1)
    g = rand((N,), 12, dtype=torch.float32)
    g[~keep] = float('inf')
    hh, ww = h.requires_grad_(), w.requires_grad_()
    logp = asrn.head_logprobs(hh, ww, y)
    dh, dw = torch.autograd.grad(logp, (hh, ww), g)
    assert (logp[~keep] == 0).all() and (dh[~keep] == 0).all()
    if which == 'all':
        assert (dw == 0).all()
        return
    lk, hk, wk = check_head(h.detach()[keep], w, y[keep], g[keep])
    assert torch.equal(lk, logp[keep]) and torch.equal(hk, dh[keep])
    assert (dw.float() - wk.float()).abs().max() <= 2 * U * wk.float().abs().max()


def test_head_more_rows_than_one_count(cuda):
    """Past 32768 positions the targets are counted by blocks first; nearly all of them ignored here."""
    N, V, d = 70001, 130, 16
    y = torch.full((N,), -1, dtype=torch.int64)
    at = torch.randperm(N, generator=torch.Generator().manual_seed(13))[:999]
    y[at] = torch.randint(0, V, (999,), generator=torch.Generator().manual_seed(14))
    check_head(rand((N, d), 15), rand((V, d), 16, 0.2), y.cuda(), rand((N,), 17, dtype=torch.float32))


def test_head_several_chunks_of_rows(cuda):
    """A vocabulary so wide that dS of all rows is over a gigabyte: dW adds up over the chunks."""
    N, V, d = 700, 1 << 20, 8
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(18)).cuda()
    y[::3] = -1
    check_head(rand((N, d), 19), rand((V, d), 20, 0.3), y, rand((N,), 21, dtype=torch.float32))


def test_head_layouts_shapes_and_repeats(cuda):
    """Leading dimensions, strided and unaligned operands, and bit-equal repeats."""
    import asrn_b200 as asrn
    B, L, V, d = 3, 50, 400, 48
    h, w = rand((B, L, d), 22), rand((V, d), 23, 0.1)
    y = torch.randint(-1, V, (B, L), generator=torch.Generator().manual_seed(24)).cuda()
    base = asrn.head_logprobs(h, w, y)
    assert base.shape == (B, L) and base.dtype == torch.float32
    strided = rand((B, d, L), 25)
    strided.copy_(h.transpose(1, 2))
    wide = torch.empty(V * d + 1, dtype=torch.bfloat16, device='cuda')[1:].view(V, d)
    wide.copy_(w)
    yt = y.t().contiguous().t()
    assert torch.equal(asrn.head_logprobs(strided.transpose(1, 2), wide, yt), base)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        h32, w32 = h.float().requires_grad_(), w.float().requires_grad_()
        out = asrn.head_logprobs(h32, w32, y)
    assert torch.equal(out, base)
    out.sum().backward()
    assert h32.grad.dtype == torch.float32 and w32.grad.dtype == torch.float32
    h1, w1 = h.clone().requires_grad_(), w.clone().requires_grad_()
    a = torch.autograd.grad(asrn.head_logprobs(h1, w1, y).sum(), (h1, w1))
    b = torch.autograd.grad(asrn.head_logprobs(h1, w1, y).sum(), (h1, w1))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert torch.equal(a[0].float(), h32.grad.to(torch.bfloat16).float())
    only_w = torch.autograd.grad(asrn.head_logprobs(h, w1, y).sum(), w1)[0]
    assert torch.equal(only_w, a[1])
    empty = asrn.head_logprobs(h[:, :0].clone().requires_grad_(), w1, y[:, :0])
    assert empty.shape == (B, 0)
    assert (torch.autograd.grad(empty.sum(), w1)[0] == 0).all()


def test_head_token_outside_the_vocabulary_gives_nan(cuda):
    import asrn_b200 as asrn
    h, w = rand((5, 16), 26), rand((9, 16), 27)
    out = asrn.head_logprobs(h, w, torch.tensor([0, 8, 9, 1 << 40, -5], device='cuda'))
    assert out.isnan().tolist() == [False, False, True, True, False]


@pytest.mark.parametrize('N,V,d', [(1, 40000, 64), (3, 300, 256), (48, 256, 64), (300, 1000, 128), (512, 777, 96)])
def test_head_few_rows_are_off_by_their_own_rounding(cuda, N, V, d):
    """Up to 512 rows dS goes into the products with its remainder: what is left is the result's rounding, u, and the
    scores' fp32 error in each term, 2^-17 of it at most for scores below 32."""
    h, w = rand((N, d), 32), rand((V, d), 33, 0.1)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(34)).cuda()
    g = rand((N,), 35, dtype=torch.float32)
    _, dh, dw = check_head(h, w, y, g)
    _, ds, rh, rw, size = head_reference(h, w, y, g, 1.0)
    assert size < 32
    fine = 2.0 ** -16
    assert ((dh.double() - rh).abs() <= U * rh.abs() * (1 + fine) + fine * (ds.abs() @ w.double().abs())).all()
    assert ((dw.double() - rw).abs() <= U * rw.abs() * (1 + fine) + fine * (ds.abs().t() @ h.double().abs())).all()


def test_head_gradient_against_differences(cuda):
    """Central differences of the kernel's own logp along a direction in h: the step is a power of two that bf16 h
    takes exactly; what is left is the scores' fp32 error over the step and the third derivative."""
    import asrn_b200 as asrn
    N, V, d, step = 64, 500, 64, 2.0 ** -5
    h = (torch.randint(-8, 9, (N, d), generator=torch.Generator().manual_seed(28)) / 8).bfloat16().cuda()
    w = rand((V, d), 29, 0.2)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(30)).cuda()
    dirn = (torch.randint(0, 2, (N, d), generator=torch.Generator().manual_seed(31)) * 2 - 1).bfloat16().cuda()
    hh = h.clone().requires_grad_()
    dh, = torch.autograd.grad(asrn.head_logprobs(hh, w, y).sum(), hh)
    up = asrn.head_logprobs((h + step * dirn).bfloat16(), w, y)
    down = asrn.head_logprobs((h - step * dirn).bfloat16(), w, y)
    slope = (up.double() - down.double()) / (2 * step)
    got = (dh.double() * dirn.double()).sum(1)
    s = (dirn.double() @ w.double().t()).abs().amax()                     # third derivative: at most 8 s^3
    size = float((h.double().abs() @ w.double().abs().t()).amax())
    tol = 8 * s ** 3 * step ** 2 / 6 + 4 * E * (d / 16 + 2) * (size + 1) / step + 2 * U * w.double().abs().sum(1).max()
    assert ((slope - got).abs() <= tol).all()


# ---- losses -------------------------------------------------------------------------------------------------------------

def lengths_mask(rows, L, seed, empty=()):
    g = torch.Generator().manual_seed(seed)
    a = (torch.rand(rows, generator=g) * L * 0.5).long()
    b = a + 1 + (torch.rand(rows, generator=g) * (L - a)).long()
    t = torch.arange(L)
    m = (t >= a[:, None]) & (t < b[:, None])
    for r in empty:
        m[r] = False
    return m.cuda()


def pref_reference(logp, ref, mask, beta, eps, kind):
    lp = torch.where(mask, logp, 0).double().requires_grad_()
    rf = torch.where(mask, ref, 0).double()
    n = mask.sum(2).double()
    R = ((lp - rf) * mask).sum(2)
    on = (n[0] > 0) & (n[1] > 0)
    if kind == 'ipo':
        M = R / n.clamp(min=1)
        each = (M[0] - M[1] - 0.5 / beta) ** 2
    else:
        x = beta * (R[0] - R[1])
        ls = torch.nn.functional.logsigmoid
        each = -(1 - eps) * ls(x) - eps * ls(-x)
    loss = torch.where(on, each, 0).sum() / max(1, int(on.sum()))
    grad, = torch.autograd.grad(loss, lp)
    return loss.detach(), grad, beta * R.detach()


@pytest.mark.parametrize('P,L', [(1, 1), (1, 2), (2, 1), (3, 7), (4, 256), (5, 2049), (40, 333), (513, 3), (600, 17),
                                 (700, 40), (2, 20000)])
@pytest.mark.parametrize('kind,eps', [('sigmoid', 0.0), ('sigmoid', 0.2), ('ipo', 0.0), ('ipo', 0.2)])
def test_preference_sizes(cuda, P, L, kind, eps):
    import asrn_b200 as asrn
    ref = -rand((2, P, L), 40, dtype=torch.float32).abs()
    logp = ref + rand((2, P, L), 41, 0.2, torch.float32)
    mask = torch.stack([lengths_mask(P, L, 42, range(7, P, 9)), lengths_mask(P, L, 43, range(3, P, 11))])
    logp = torch.where(mask, logp, float('nan'))         # outside the mask nothing is used
    ref = torch.where(mask, ref, float('inf'))
    r = asrn.preference_loss(logp, ref, mask, beta=0.3, smoothing=eps, kind=kind)
    loss, grad, rew = pref_reference(logp, ref, mask, 0.3, eps, kind)
    assert abs(float(r.loss) - float(loss)) <= 4 * E * max(1.0, abs(float(loss)))
    assert (r.grad.double() - grad).abs().max() <= 4 * E * max(float(grad.abs().max()), 1e-30)
    assert (r.grad[~mask] == 0).all()
    got = torch.stack([r.chosen, r.rejected]).double()
    assert (got - rew).abs().max() <= 4 * E * max(float(rew.abs().max()), 1e-30)


def test_preference_no_pair_counts(cuda):
    import asrn_b200 as asrn
    z = torch.zeros(2, 4, 9, device='cuda')
    m = torch.zeros(2, 4, 9, dtype=torch.bool, device='cuda')
    m[0] = True                                          # the chosen answers only
    r = asrn.preference_loss(z + 1, z, m)
    assert float(r.loss) == 0 and (r.grad == 0).all() and (r.chosen - 0.9).abs().max() < 1e-6
    for shape in ((2, 0, 5), (2, 3, 0)):
        e = torch.zeros(shape, device='cuda')
        r = asrn.preference_loss(e, e, e.bool())
        assert float(r.loss) == 0 and r.grad.shape == shape and (r.chosen == 0).all()


def test_preference_far_apart_answers(cuda):
    """Margins where the exponential under- and overflows in either direction."""
    import asrn_b200 as asrn
    lp = torch.zeros(2, 4, 1, device='cuda')
    lp[0, :, 0] = torch.tensor([1e4, -1e4, 3e38, -3e38])
    m = torch.ones_like(lp, dtype=torch.bool)
    r = asrn.preference_loss(lp[:, :2], torch.zeros_like(lp)[:, :2], m[:, :2], beta=1.0)
    assert abs(float(r.loss) - 5e3) <= 4 * E * 5e3
    assert r.grad[0, :, 0].tolist() == [0.0, -0.5]
    r = asrn.preference_loss(lp, torch.zeros_like(lp), m, beta=1.0)
    assert r.grad[0, :, 0].tolist() == [0.0, -0.25, 0.0, -0.25]


def policy_reference(logp, old, adv, mask, ref, clip, kl, per):
    A = (adv if adv.dim() == 2 else adv[:, None].expand_as(logp)).double()
    lp = torch.where(mask, logp, 0).double().requires_grad_()
    lr = (lp - torch.where(mask, old, 0).double()).clamp(-20, 20)
    r = lr.exp()
    lo, hi = math.log1p(-clip[0]), math.log1p(clip[1])
    cut = ((A > 0) & (lr > hi)) | ((A < 0) & (lr < lo))
    each = -torch.where(cut, r.detach().clamp(1 - clip[0], 1 + clip[1]), r) * A
    k3 = torch.zeros_like(each)
    if ref is not None:
        q = (torch.where(mask, ref, 0).double() - lp).clamp(-20, 20)
        k3 = torch.expm1(q) - q
        each = each + kl * k3
    n = mask.sum(1)
    m = mask.double()
    if per == 'sequence':
        w = m / n.clamp(min=1)[:, None] / max(1, int((n > 0).sum()))
    else:
        w = m / max(1, int(n.sum()))
    loss = torch.where(mask, each * w, 0).sum()
    grad, = torch.autograd.grad(loss, lp)
    tot = max(1, int(n.sum()))
    return loss.detach(), grad, torch.where(mask, k3, 0).sum().detach() / tot, (cut & mask).sum().double() / tot


@pytest.mark.parametrize('B,L', [(1, 1), (2, 1), (1, 3), (8, 512), (37, 1111), (3, 2048), (3, 2049), (1025, 5),
                                 (1, 40000), (300, 100)])
@pytest.mark.parametrize('per', ['token', 'sequence'])
@pytest.mark.parametrize('per_token,with_ref', [(False, True), (True, False), (True, True)])
def test_policy_sizes(cuda, B, L, per, per_token, with_ref):
    import asrn_b200 as asrn
    old = -rand((B, L), 50, dtype=torch.float32).abs() * 3
    logp = old + rand((B, L), 51, 0.3, torch.float32)
    ref = old + rand((B, L), 52, 0.3, torch.float32) if with_ref else None
    adv = rand((B, L) if per_token else (B,), 53, dtype=torch.float32)
    mask = lengths_mask(B, L, 54, range(5, B, 6))
    bad = torch.full_like(logp, float('nan'))
    logp, old = torch.where(mask, logp, bad), torch.where(mask, old, bad)
    ref = None if ref is None else torch.where(mask, ref, bad)
    adv = torch.where(mask, adv, bad) if per_token else adv
    kl = 0.1 if with_ref else 0.0
    r = asrn.policy_loss(logp, old, adv, mask, ref_logp=ref, clip=(0.2, 0.3), kl=kl, per=per)
    a = torch.where(mask, adv, torch.zeros_like(adv)) if per_token else adv
    loss, grad, k3, cut = policy_reference(logp, old, a, mask, ref, (0.2, 0.3), kl, per)
    # each term is off by a few e of itself; the terms reach a few times the largest advantage
    size = 8 * float(a.abs().max()) + 1
    assert abs(float(r.loss) - float(loss)) <= 8 * E * size
    assert (r.grad.double() - grad).abs().max() <= 16 * E * max(float(grad.abs().max()), 1e-30)
    assert (r.grad[~mask] == 0).all()
    assert abs(float(r.kl) - float(k3)) <= 8 * E * max(1.0, float(k3)) and abs(float(r.clipped) - float(cut)) <= 2 * E


def test_policy_empty_masks_and_sizes(cuda):
    import asrn_b200 as asrn
    z = torch.full((4, 30), float('nan'), device='cuda')
    r = asrn.policy_loss(z, z, z, torch.zeros(4, 30, dtype=torch.uint8, device='cuda'), ref_logp=z, kl=1.0)
    assert float(r.loss) == 0 and (r.grad == 0).all() and float(r.kl) == 0 and float(r.clipped) == 0
    for shape in ((0, 5), (5, 0)):
        e = torch.zeros(shape, device='cuda')
        r = asrn.policy_loss(e, e, torch.zeros(shape[0], device='cuda'), e.bool(), per='sequence')
        assert float(r.loss) == 0 and r.grad.shape == shape


def test_policy_far_ratios_and_nan(cuda):
    """Held at 20 nats with no gradient beyond; a NaN under the mask shows in the loss."""
    import asrn_b200 as asrn
    lp = torch.tensor([[30.0, -30.0, 30.0, -30.0]], device='cuda')
    adv = torch.tensor([[1.0, 1.0, -1.0, -1.0]], device='cuda')
    m = torch.ones(1, 4, dtype=torch.bool, device='cuda')
    r = asrn.policy_loss(lp, torch.zeros_like(lp), adv, m)
    want = (-1.2 - math.exp(-20) + math.exp(20) + 0.8) / 4
    assert abs(float(r.loss) - want) <= 8 * E * want and (r.grad == 0).all()
    assert float(r.clipped) == 0.5
    r = asrn.policy_loss(torch.full((1, 4), float('nan'), device='cuda'), lp, adv, m)
    assert math.isnan(float(r.loss)) and r.grad.isnan().all()


@pytest.mark.parametrize('which', ['sigmoid', 'ipo', 'policy'])
def test_loss_gradients_against_differences_and_autograd(cuda, which):
    """Central differences of the loss itself: its fp32 rounding over the step, and the third derivative (kinks kept
    away by ratios that no step carries across a bound)."""
    import asrn_b200 as asrn
    step = 2.0 ** -6
    if which == 'policy':
        old = -rand((6, 50), 60, dtype=torch.float32).abs()
        ratio = torch.tensor([0.5, 0.9, 1.05, 1.6], device='cuda').log()
        logp = old + ratio[torch.arange(300, device='cuda').view(6, 50) % 4]
        adv, mask = rand((6,), 61, dtype=torch.float32), lengths_mask(6, 50, 62, [2])
        f = lambda x: asrn.policy_loss(x, old, adv, mask, ref_logp=old, kl=0.1)  # noqa: E731
    else:
        logp = rand((2, 5, 20), 63, 0.3, torch.float32)
        ref, mask = rand((2, 5, 20), 64, 0.3, torch.float32), torch.stack([lengths_mask(5, 20, 65, [1]),
                                                                           lengths_mask(5, 20, 66)])
        f = lambda x: asrn.preference_loss(x, ref, mask, beta=0.2, kind=which)  # noqa: E731
    dirn = torch.sign(rand(logp.shape, 67, dtype=torch.float32))
    r = f(logp)
    got = float((r.grad.double() * dirn.double()).sum())
    up, down = f(logp + step * dirn).loss.double(), f(logp - step * dirn).loss.double()
    slope = float(up - down) / (2 * step)
    third = 40.0                                          # of terms like r A and beta^3 20^3 / 10, all below this
    size = abs(float(r.loss)) + 1
    assert abs(slope - got) <= third * step ** 2 / 6 + 4 * E * size / step
    x = logp.clone().requires_grad_()
    out = f(x)
    (out.loss * 3).backward()
    assert torch.equal(x.grad, out.grad * 3) and torch.equal(out.loss.detach(), r.loss)
    assert all(torch.equal(a, b) for a, b in zip(f(logp), r))


# ---- 8 bits -------------------------------------------------------------------------------------------------------------

def packed(x):
    """codes and exponents by the definition, in 64 bits."""
    rows, f = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -f % 32)).view(rows, -1, 32)
    top = b.abs().amax(2)
    e = torch.full(top.shape, -120, dtype=torch.int64, device=x.device)
    ok = top.isfinite()
    for _ in range(300):
        e = torch.where(ok & (top > 127 * torch.exp2(e.double())), e + 1, e)
    codes = torch.round(b * torch.exp2(-e.double())[:, :, None])
    codes = torch.where(ok[:, :, None], codes, 0.0).reshape(rows, -1)[:, :f]
    return codes.to(torch.int8), torch.where(ok, e, -128).to(torch.int8)


@pytest.mark.parametrize('rows,f', [(1, 8), (3, 24), (5, 32), (7, 40), (130, 264), (33, 1536)])
def test_pack8_is_the_definition(cuda, rows, f):
    from asrn_b200 import finetune as ft
    x = rand((rows, f), 70, dtype=torch.float32) * torch.exp2(torch.linspace(-126, 120, rows * f).view(rows, f)).cuda()
    x = x.bfloat16()
    x[0, 0] = 127.0
    x[-1, -8:] = 0
    p = ft.pack8(x)
    codes, e = packed(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.exps, e)
    want = codes.double() * torch.exp2(e.double()).repeat_interleave(32, 1)[:, :f]
    assert torch.equal(ft.unpack8(p).double(), want)


def test_pack8_edges(cuda):
    from asrn_b200 import finetune as ft
    x = torch.zeros(1, 8 * 32, dtype=torch.bfloat16, device='cuda')
    x[0, 5] = 127.0                                      # the largest value of its scale
    x[0, 32] = 127.5                                     # bf16 128 would be next: over 127, so the next scale
    x[0, 64], x[0, 65] = 64.0, 0.25                      # ties to even: 0.25 2^1 -> 0, 0.75 2^1 -> 2
    x[0, 66] = 0.75
    x[0, 96] = float('inf')
    x[0, 128] = float('nan')
    x[0, 160] = 3.3e38
    x[0, 192] = 1e-40                                    # below the least scale
    p = ft.pack8(x)
    codes, e = packed(x)
    assert torch.equal(p.codes, codes) and torch.equal(p.exps, e)
    y = ft.unpack8(p)
    assert y[0, 96:160].isnan().all() and not y[0, :96].isnan().any() and not y[0, 160:].isnan().any()
    assert (y[0, 224:] == 0).all()
    big = rand((4, 3, 64), 71)
    q = ft.pack8(big.transpose(0, 1))
    assert ft.unpack8(q).shape == (3, 4, 64)
    assert (ft.unpack8(q).float() - big.transpose(0, 1).float()).abs().max() <= big.abs().max() / 64 / 2
    assert ft.unpack8(ft.pack8(torch.zeros(0, 8, dtype=torch.bfloat16, device='cuda'))).shape == (0, 8)


def mlp_reference(x, w1, b1, w2, b2, dy):
    x, w1, b1, w2, b2, dy = (t.double() for t in (x, w1, b1, w2, b2, dy))
    a = x @ w1.t() + b1
    g = torch.nn.functional.gelu(a)
    y = g @ w2.t() + b2

    def kept(v):
        c, e = packed_double(v)
        return c * torch.exp2(e.double()).repeat_interleave(32, 1)[:, :v.shape[1]]
    ak, xk = kept(a).requires_grad_(), kept(x)
    gk = torch.nn.functional.gelu(ak)
    slope, = torch.autograd.grad(gk.sum(), ak)
    gk = gk.detach()
    dg = dy @ w2
    da = dg * slope
    res = dict(y=y, dx=da @ w1, dw1=da.t() @ xk, db1=da.sum(0), dw2=dy.t() @ gk, db2=dy.sum(0))
    size = dict(y=g.abs() @ w2.abs().t() + b2.abs(), dx=da.abs() @ w1.abs(), dw1=da.abs().t() @ xk.abs(),
                db1=da.abs().sum(0), dw2=dy.abs().t() @ gk.abs(), db2=dy.abs().sum(0))
    return res, size


def packed_double(v):
    rows, f = v.shape
    b = torch.nn.functional.pad(v, (0, -f % 32)).view(rows, -1, 32)
    top = b.abs().amax(2)
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 127))
    e = torch.where(127 * torch.exp2(e) < top, e + 1, torch.where(127 * torch.exp2(e - 1) >= top, e - 1, e))
    return torch.round(b * torch.exp2(-e)[:, :, None]).reshape(rows, -1)[:, :f], e


def run_mlp(x, w1, b1, w2, b2, dy):
    import asrn_b200 as asrn
    ins = [t.detach().requires_grad_() for t in (x, w1, b1, w2, b2)]
    y = asrn.mlp8(*ins)
    grads = torch.autograd.grad(y, ins, dy)
    return dict(zip(('y', 'dx', 'dw1', 'db1', 'dw2', 'db2'), (y.detach(), *grads)))


MLP_SIZES = [(1, 8, 8, 8), (1, 64, 128, 64), (3, 40, 24, 72), (64, 64, 128, 64), (127, 96, 200, 96), (129, 256, 520, 128),
             (300, 264, 512, 8), (1000, 768, 1536, 768), (5000, 64, 128, 64)]


@pytest.mark.parametrize('N,d,ff,dout', MLP_SIZES)
def test_mlp8_on_exact_sums(cuda, N, d, ff, dout):
    """Integers over powers of two: x w1^T + b1 is exact in any order, so the 8-bit codes are the definition's to the
    last one, and only the operands' and results' roundings are left."""
    g = torch.Generator().manual_seed(80)
    ints = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).float()  # noqa: E731
    x, w1, b1 = ints(-4, 4, N, d) / 4, ints(-2, 2, ff, d) / 8, ints(-8, 8, ff) / 8
    w2, b2, dy = ints(-4, 4, dout, ff) / 16, ints(-4, 4, dout) / 4, ints(-8, 8, N, dout) / 64
    ts = [t.bfloat16().cuda() for t in (x, w1, b1, w2, b2, dy)]
    got = run_mlp(*ts)
    want, size = mlp_reference(*ts)
    for k in want:
        err = (got[k].double() - want[k]).abs()
        assert (err <= U * (want[k].abs() + size[k]) + 1e-30).all(), (k, float((err / (size[k] + 1e-30)).max()))


@pytest.mark.parametrize('N,d,ff,dout', [(1, 8, 8, 8), (33, 96, 200, 40), (127, 64, 128, 64), (512, 256, 520, 128)])
def test_mlp8_few_rows_are_off_by_their_own_rounding(cuda, N, d, ff, dout):
    """Up to 512 rows gelu(a) and dA go into the products with their remainders: what is left is the result's rounding, u,
    and of each term 2^-18 of the remainder's rounding and a few 2^-21 of the normal tail's formula."""
    g = torch.Generator().manual_seed(79)
    ints = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).float()  # noqa: E731
    x, w1, b1 = ints(-4, 4, N, d) / 4, ints(-2, 2, ff, d) / 8, ints(-8, 8, ff) / 8
    w2, b2, dy = ints(-4, 4, dout, ff) / 16, ints(-4, 4, dout) / 4, ints(-8, 8, N, dout) / 64
    ts = [t.bfloat16().cuda() for t in (x, w1, b1, w2, b2, dy)]
    got = run_mlp(*ts)
    want, size = mlp_reference(*ts)
    fine = 2.0 ** -16
    # where gelu or gelu' is small against a the formula's absolute error, 2^-23 |a|, is what counts: |a| is below 32
    a = 2.0 ** -18
    floor = dict(y=a * ts[3].double().abs().sum(1), dx=a * ((ts[5].double() @ ts[3].double()).abs() @ ts[1].double().abs()),
                 dw1=a * ((ts[5].double() @ ts[3].double()).abs().t() @ ts[0].double().abs()),
                 db1=a * (ts[5].double() @ ts[3].double()).abs().sum(0),
                 dw2=a * ts[5].double().abs().sum(0)[:, None], db2=0.0)
    for k in want:
        err = (got[k].double() - want[k]).abs()
        assert (err <= U * want[k].abs() * (1 + fine) + fine * size[k] + floor[k]).all(), k


@pytest.mark.parametrize('N,d,ff', [(257, 256, 520), (4096, 768, 1536)])
def test_mlp8_on_ordinary_values(cuda, N, d, ff):
    """Two roundings to bf16 of the terms' size each, uniform in the last place: 1.7e-3 each in 2-norm, 2.4e-3 together;
    a code that falls on the other side of a tie (a few in 10^5) moves a value by 1/64 of its block's largest."""
    x, w1, b1 = rand((N, d), 81), rand((ff, d), 82, d ** -0.5), rand((ff,), 83, 0.1)
    w2, b2, dy = rand((d, ff), 84, ff ** -0.5), rand((d,), 85, 0.1), rand((N, d), 86)
    got = run_mlp(x, w1, b1, w2, b2, dy)
    want, _ = mlp_reference(x, w1, b1, w2, b2, dy)
    for k in want:
        assert float((got[k].double() - want[k]).norm() / want[k].norm()) <= 3e-3, k
    again = run_mlp(x, w1, b1, w2, b2, dy)
    assert all(torch.equal(got[k], again[k]) for k in got)


def test_mlp8_near_full_precision_gradients(cuda):
    """The 8-bit values stay within 1/127 of their blocks' largest: the gradients within 2 % of the unrounded ones'."""
    N, d, ff = 512, 256, 512
    x, w1, b1 = rand((N, d), 87), rand((ff, d), 88, d ** -0.5), rand((ff,), 89, 0.1)
    w2, b2, dy = rand((d, ff), 90, ff ** -0.5), rand((d,), 91, 0.1), rand((N, d), 92)
    got = run_mlp(x, w1, b1, w2, b2, dy)
    ins = [t.double().requires_grad_() for t in (x, w1, b1, w2, b2)]
    y = torch.nn.functional.gelu(ins[0] @ ins[1].t() + ins[2]) @ ins[3].t() + ins[4]
    for k, ref in zip(('dx', 'dw1', 'db1', 'dw2', 'db2'), torch.autograd.grad(y, ins, dy.double())):
        assert float((got[k].double() - ref).norm() / ref.norm()) <= 2e-2, k


def test_mlp8_shapes_and_what_it_keeps(cuda):
    import asrn_b200 as asrn
    x, w1, b1, w2, b2 = rand((2, 33, 64), 93), rand((128, 64), 94, 0.1), rand((128,), 95), rand((64, 128), 96, 0.1), \
        rand((64,), 97)
    with torch.no_grad():
        y = asrn.mlp8(x, w1, b1, w2, b2)
    assert y.shape == x.shape and not y.requires_grad
    xs = torch.empty(2, 64, 33, dtype=torch.bfloat16, device='cuda')
    xs.copy_(x.transpose(1, 2))
    assert torch.equal(asrn.mlp8(xs.transpose(1, 2), w1, b1, w2, b2), y)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        assert torch.equal(asrn.mlp8(x.float(), w1.float(), b1.float(), w2.float(), b2.float()), y)
    w = w1.clone().requires_grad_()
    torch.cuda.synchronize()
    with torch.no_grad():                                # nothing is kept where no gradient is wanted
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = asrn.mlp8(x, w, b1, w2, b2)
        peak = torch.cuda.max_memory_allocated() - before
    assert torch.equal(out, y) and peak <= y.nbytes + 2 * 96 * 128 * 2 + 2 * 512
    only, = torch.autograd.grad(asrn.mlp8(x, w, b1, w2, b2).sum(), w)
    full = run_mlp(x, w1, b1, w2, b2, torch.ones_like(y))
    assert torch.equal(only, full['dw1'])
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.nbytes) or t, lambda t: t):
        asrn.mlp8(x, w, b1, w2, b2)
    assert sum(kept) <= w1.nbytes + w2.nbytes + 66 * (64 + 128) * 33 // 32 + 4 * 256
    e = asrn.mlp8(x[:, :0].clone().requires_grad_(), w, b1, w2, b2)
    assert e.shape == (2, 0, 64) and (torch.autograd.grad(e.sum(), w)[0] == 0).all()


def test_nan_and_infinity_reach_only_their_rows(cuda):
    x, w1, b1, w2, b2 = rand((40, 64), 98), rand((128, 64), 99, 0.1), rand((128,), 100), rand((64, 128), 101, 0.1), \
        rand((64,), 102)
    x[7, 3], x[21, 60] = float('nan'), float('inf')
    got = run_mlp(x, w1, b1, w2, b2, rand((40, 64), 103))
    bad = got['y'].isnan().any(1)
    assert bad.nonzero().flatten().tolist() == [7, 21]
    assert got['dx'].isnan().any(1).nonzero().flatten().tolist() == [7, 21]


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------------

def test_on_another_stream_and_in_a_graph(cuda):
    import asrn_b200 as asrn
    from asrn_b200 import finetune as ft
    h, w = rand((200, 64), 110), rand((500, 64), 111, 0.1)
    y = torch.randint(-1, 500, (200,), generator=torch.Generator().manual_seed(112)).cuda()
    x, w1, b1, w2, b2 = rand((200, 64), 113), rand((128, 64), 114, 0.1), rand((128,), 115), rand((64, 128), 116, 0.1), \
        rand((64,), 117)
    want = asrn.head_logprobs(h, w, y), asrn.mlp8(x, w1, b1, w2, b2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = asrn.head_logprobs(h, w, y), asrn.mlp8(x, w1, b1, w2, b2)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        got = asrn.head_logprobs(h, w, y), asrn.mlp8(x, w1, b1, w2, b2)
    h.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], asrn.head_logprobs(h, w, y)) and torch.equal(got[1], want[1])
    assert ft.status() == 0


@pytest.mark.parametrize('rows,L', [(4, 100), (40, 3000), (700, 4096)])
def test_losses_in_a_graph_and_on_another_stream(cuda, rows, L):
    """One block, one cooperative launch, two overlapping launches: each captured and replayed on other values."""
    import asrn_b200 as asrn
    lp, ref = rand((2, rows, L), 140, 0.2, torch.float32), rand((2, rows, L), 141, 0.2, torch.float32)
    m = torch.stack([lengths_mask(rows, L, 142), lengths_mask(rows, L, 143)])
    adv = rand((rows,), 144, dtype=torch.float32)

    def both():
        return (*asrn.preference_loss(lp, ref, m), *asrn.policy_loss(lp[0], ref[0], adv, m[0], ref_logp=ref[1], kl=0.1))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    want = both()
    with torch.cuda.stream(s):
        got = both()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    lp.mul_(-0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(both(), got))


def test_refusals(cuda):
    import asrn_b200 as asrn
    from asrn_b200 import finetune as ft
    h, w, y = rand((4, 16), 120), rand((9, 16), 121), torch.zeros(4, dtype=torch.int64, device='cuda')
    with pytest.raises(ValueError):
        asrn.head_logprobs(h, w, y[:3])
    with pytest.raises(ValueError):
        asrn.head_logprobs(h, w, y, temperatura=0.0)
    with pytest.raises(TypeError):
        asrn.head_logprobs(h, w, y.int())
    with pytest.raises(NotImplementedError):
        asrn.head_logprobs(h[:, :12], w[:, :12], y)
    with pytest.raises(NotImplementedError):
        asrn.head_logprobs(h.float(), w.float(), y)
    z = torch.zeros(2, 3, 4, device='cuda')
    with pytest.raises(ValueError):
        asrn.preference_loss(z, z[:, :2], z.bool())
    with pytest.raises(ValueError):
        asrn.preference_loss(z, z, z)
    with pytest.raises(ValueError):
        asrn.preference_loss(z, z, z.bool(), beta=0.0)
    with pytest.raises(ValueError):
        asrn.preference_loss(z, z, z.bool(), kind='hinge')
    z = z[0]
    with pytest.raises(ValueError):
        asrn.policy_loss(z, z, z[:, 0], z.bool(), kl=0.1)
    with pytest.raises(ValueError):
        asrn.policy_loss(z, z, z[0], z.bool())
    with pytest.raises(ValueError):
        asrn.policy_loss(z, z, z, z.bool(), clip=(1.0, 0.2))
    with pytest.raises(ValueError):
        asrn.policy_loss(z, z, z, z.bool(), per='batch')
    with pytest.raises(RuntimeError, match='CUDA'):
        asrn.policy_loss(z.cpu(), z.cpu(), z.cpu(), z.cpu().bool())
    with pytest.raises(NotImplementedError):
        asrn.mlp8(h, rand((12, 16), 122), rand((12,), 123), rand((16, 12), 124), rand((16,), 125))
    with pytest.raises(ValueError):
        asrn.mlp8(h, rand((8, 24), 126), rand((8,), 127), rand((16, 8), 128), rand((16,), 129))
    with pytest.raises(NotImplementedError):
        ft.pack8(rand((2, 12), 130))
    with pytest.raises(TypeError):
        ft.pack8(h.float())


@pytest.mark.parametrize('mode', [torch.no_grad, torch.inference_mode])
def test_forward_without_gradients_is_the_same(cuda, mode):
    import asrn_b200 as asrn
    g = torch.Generator(cuda).manual_seed(3)
    rand = lambda *s: torch.randn(*s, device=cuda, generator=g).bfloat16()  # noqa: E731
    h, w, y = rand(33, 64), rand(97, 64).requires_grad_(), torch.arange(33, device=cuda)
    u, b, v = rand(48, 64), rand(48), rand(64, 48)
    lp, out = asrn.head_logprobs(h, w, y), asrn.mlp8(h, u.requires_grad_(), b, v, h[0])
    with mode():
        lp2, out2 = asrn.head_logprobs(h, w, y), asrn.mlp8(h, u, b, v, h[0])
    assert not lp2.requires_grad and not out2.requires_grad and lp.requires_grad and out.requires_grad
    assert torch.equal(lp, lp2) and torch.equal(out, out2)


def test_a_weight_changed_in_place_is_noticed(cuda):
    import asrn_b200 as asrn
    w = torch.ones(8, 8, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    lp = asrn.head_logprobs(w[:3].detach(), w, torch.zeros(3, dtype=torch.int64, device=cuda))
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match='modified'):
        lp.sum().backward()

"""head_stats against a plain implementation in 64 bits. Bounds, with U = 2^-8 and E = 2^-24 the unit roundoffs of bf16 and fp32:
  scores     d products summed in fp32, 16 at a time, truncated: A = (d / 16 + 2) 2 E max sum|h w| / tau; the exponents'
             scaling and offset 4 E max|s|
  logp       twice a score's error, and a few E of 1 + |logp|
  entropy    dH = - sum p (log p + H) ds, so the scores' error times sum p |log p + H|, and the logarithms' own 64 E (1 + H)
  tokens     ranked by their exact scores: equal to the ranking in 64 bits
  gradients  dS rounded to bf16 as an operand, results rounded to bf16: U (|result| + sum |dS| |other|)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -24


def rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def targets(N, V, seed, skip=0):
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(seed)).cuda()
    if skip:
        y[torch.arange(N, device='cuda') % skip == skip - 1] = -100
    return y


def check(h, w, y=None, tau=1.0, top=0, grads=True):
    import asrn_b200 as asrn
    h, w = h.detach().requires_grad_(grads), w.detach().requires_grad_(grads)
    r = asrn.head_stats(h, w, y, temperatura=tau, top=top)
    (V, d), N = w.shape, h.shape[0]
    h64, w64 = h.detach().double(), w.detach().double()
    z = h64 @ w64.t()
    lp = torch.log_softmax(z / tau, 1)
    p = lp.exp()
    plp = torch.where(p > 0, p * lp, 0.0)
    H = -plp.sum(1)
    on = torch.ones(N, dtype=torch.bool, device='cuda') if y is None else y >= 0
    size = float((h64.abs() @ w64.abs().t())[on].amax()) / tau if on.any() else 0.0
    A = (d / 16 + 2) * 2 * E * size + 4 * E * size
    spread = torch.where(p > 0, p * (lp + H[:, None]).abs(), 0.0).sum(1)
    got = r.entropy.detach().double()
    tol = A * spread + 64 * E * (1 + H)
    assert ((got - H).abs()[on] <= tol[on]).all(), ((got - H).abs() / tol)[on].max()
    assert (r.entropy[~on] == 0).all()
    if y is None:
        assert r.logp is None
    else:
        ref = lp.gather(1, y.clamp(min=0)[:, None])[:, 0]
        assert ((r.logp.detach().double() - ref).abs()[on] <= (2 * A + 16 * E * (1 + ref.abs()))[on]).all()
        assert (r.logp[~on] == 0).all()
    if top:
        order = z.sort(dim=1, descending=True, stable=True)
        tokens = torch.where(on[:, None], order.indices[:, :top], -1)
        assert torch.equal(r.top_tokens, tokens), (r.top_tokens != tokens).nonzero()[:5]
        best = lp.gather(1, order.indices[:, :top])
        tol = 2 * A + 16 * E * (1 + best.abs())
        assert ((r.top_logp.detach().double() - best).abs() <= tol)[on].all() and (r.top_logp[~on] == 0).all()
        assert not r.top_logp.requires_grad
    else:
        assert r.top_logp is None and r.top_tokens is None
    if not grads:
        return r
    g, gh = rand((N,), 90, dtype=torch.float32), rand((N,), 91, dtype=torch.float32)
    out, up = ((r.entropy,), (gh,)) if y is None else ((r.entropy, r.logp), (gh, g))
    dh, dw = torch.autograd.grad(out, (h, w), up)
    g64, gh64 = torch.where(on, g.double(), 0.0)[:, None], torch.where(on, gh.double(), 0.0)[:, None]
    ds = -gh64 * torch.where(p > 0, p * (lp + H[:, None]), 0.0)
    if y is not None:
        pick = torch.nn.functional.one_hot(y.clamp(min=0), V).double() * on[:, None]
        other = p * (1 - pick)                                  # 1 - p_y as the others' sum: 1 - exp would cancel
        ds = ds + g64 * (pick * other.sum(1, keepdim=True) - other * on[:, None])
    ds = ds / tau
    # dS itself: p is off by A of itself, log p + H by the scores' and the entropy's errors
    off = (A + 8 * E) * ds.abs() + p * (gh64.abs() * (2 * A + 64 * E * (1 + H[:, None]))) / tau
    rh, rw = ds @ w64, ds.t() @ h64
    assert ((dh.double() - rh).abs() <= U * (rh.abs() + ds.abs() @ w64.abs()) + 2 * off @ w64.abs() + 1e-30).all()
    assert ((dw.double() - rw).abs() <= U * (rw.abs() + ds.abs().t() @ h64.abs()) + 2 * off.t() @ h64.abs() + 1e-30).all()
    assert (dh[~on] == 0).all()
    return r


@pytest.mark.parametrize('N,V,d,skip,top', [
    (1, 1, 8, 0, 1), (1, 200, 32, 0, 5), (2, 3, 64, 0, 3), (7, 257, 64, 3, 4), (48, 256, 64, 0, 32), (127, 129, 72, 2, 1),
    (128, 512, 128, 0, 5), (129, 1000, 200, 5, 20), (256, 255, 768, 0, 2), (257, 5003, 96, 2, 7), (600, 513, 1024, 7, 8),
    (1100, 70001, 64, 3, 5), (1025, 777, 40, 2, 0), (3000, 256, 256, 0, 3), (5000, 130, 16, 0, 0)])
@pytest.mark.parametrize('given', [True, False])
def test_sizes(cuda, N, V, d, skip, top, given):
    check(rand((N, d), 1), rand((V, d), 2, 0.1), targets(N, V, 3, skip) if given else None, top=top)


@pytest.mark.parametrize('tau', [0.25, 0.8, 3.0])
def test_temperature_and_peaked_scores(cuda, tau):
    N, V, d = 300, 3001, 128
    w = rand((V, d), 5, 0.3)
    y = targets(N, V, 6)
    h = (rand((N, d), 7, dtype=torch.float32) + 3 * w[y].float()).bfloat16()
    check(h, w, y, tau, 5)
    check(h, w, (y + 1) % V, tau, 5)                      # another token than the one that is all but sure
    check(h, w, None, tau, 5)


def test_one_token_all_but_sure(cuda):
    """Entropies far below 1: what is left of them is the other tokens' own sum."""
    N, V, d = 64, 500, 64
    w = rand((V, d), 8, 0.3)
    y = targets(N, V, 9)
    h = (6 * w[y].float()).bfloat16()
    r = check(h, w, y, 0.5, 3)
    lp = torch.log_softmax(h.double() @ w.double().t() / 0.5, 1)
    H = -(lp.exp() * lp).sum(1)
    assert (H < 1e-4).any()
    assert (r.entropy.double() - H).abs().max() <= 1e-3 * H.max() + 1e-9


@pytest.mark.parametrize('which', ['all', 'first', 'last', 'one'])
def test_rows_without_a_target(cuda, which):
    import asrn_b200 as asrn
    N, V, d = 400, 300, 64
    y = targets(N, V, 10)
    keep = torch.zeros(N, dtype=torch.bool, device='cuda')
    keep[{'all': slice(0, 0), 'first': slice(0, 130), 'last': slice(399, 400), 'one': slice(200, 201)}[which]] = True
    y[~keep] = -1
    h, w = rand((N, d), 11), rand((V, d), 12, 0.1)
    h[~keep] = float('nan')                               # what an ignored row holds reaches nothing
    hh, ww = h.requires_grad_(), w.requires_grad_()
    r = asrn.head_stats(hh, ww, y, top=4)
    g = rand((2, N), 13, dtype=torch.float32)
    g[:, ~keep] = float('inf')
    dh, dw = torch.autograd.grad((r.entropy, r.logp), (hh, ww), tuple(g))
    for t in (r.entropy, r.logp, r.top_logp, dh):
        assert (t[~keep] == 0).all()
    assert (r.top_tokens[~keep] == -1).all()
    if which == 'all':
        assert (dw == 0).all()
        return
    # calls of up to 64 rows sum in another order: bit for bit only among calls of one kind
    check(h.detach()[keep], w, y[keep], top=4)
    k = check(torch.where(keep[:, None], h.detach(), 0), w, y, top=4)
    assert torch.equal(k.logp, r.logp) and torch.equal(k.top_tokens, r.top_tokens)
    assert torch.equal(k.entropy, r.entropy) and torch.equal(k.top_logp, r.top_logp)


def test_more_rows_than_one_count_and_several_chunks(cuda):
    N, V, d = 70001, 130, 16
    y = torch.full((N,), -1, dtype=torch.int64)
    at = torch.randperm(N, generator=torch.Generator().manual_seed(14))[:999]
    y[at] = torch.randint(0, V, (999,), generator=torch.Generator().manual_seed(15))
    check(rand((N, d), 16), rand((V, d), 17, 0.2), y.cuda(), top=3)
    check(rand((N, d), 18), rand((V, d), 19, 0.2), None, top=2, grads=False)
    check(rand((700, 8), 20), rand((1 << 20, 8), 21, 0.3), targets(700, 1 << 20, 22, 3), top=6)


@pytest.mark.parametrize('given', [True, False])
def test_equal_scores_come_in_the_order_of_their_numbers(cuda, given):
    V, d = 1500, 32
    w = rand((V, d), 23, 0.3)
    w[700:] = w[:800].clone()                                # most tokens have a twin
    w[3] = w[4] = w[1400]
    h = rand((60, d), 24)
    h[5] = 0                                              # all scores equal
    h[6] = w[3] * 8
    y = targets(60, V, 25) if given else None
    r = check(h, w, y, top=32)
    assert torch.equal(r.top_tokens[5], torch.arange(32, device='cuda'))
    assert r.top_tokens[6, :3].tolist() == [3, 4, 704] or r.top_tokens[6, 0] == 3


def test_scores_that_fp32_sums_cannot_tell_apart(cuda):
    """Rows of W that differ in one small coordinate behind large ones that cancel: exact scores decide, within a group of 128
    and across groups."""
    V, d = 2000, 256
    g = torch.Generator().manual_seed(26)
    base = torch.randn(d, generator=g) * 4
    w = base.bfloat16().repeat(V, 1)
    w[:, 17] = (torch.randn(V, generator=g) * 2.0 ** -12).bfloat16()
    h = (torch.randn(20, d, generator=g) * 8).bfloat16()
    h[:, 17] = 2.0 ** -3
    check(h.cuda(), w.cuda(), None, top=8, grads=False)
    check(h.cuda(), w.cuda(), targets(20, V, 27), top=32, grads=False)


@pytest.mark.parametrize('V', [220, 1500, 5003, 33001, 70001])
@pytest.mark.parametrize('N', [3, 100, 700])
@pytest.mark.parametrize('top', [1, 6, 20, 32])
def test_rankings_of_every_kind(cuda, V, N, top):
    """Every way the notes are kept and the rows are ranked: plain scores, twins, near twins, several of a group, rows of zeros."""
    d = 72
    w = rand((V, d), 60, 0.2)
    w[V // 2:V // 2 + 40] *= 4                            # neighbours that are likely
    w[-30:] = w[V // 2:V // 2 + 30].clone()               # and their twins
    w[-60:-30] = w[V // 2:V // 2 + 30].clone()
    w[-60:-30, 3] += 2.0 ** -8 * w[-60:-30, 3]            # near twins: one coordinate's last bit or two
    h = rand((N, d), 61)
    h[::5] = 0
    h[1::5, 3] = 2.0 ** -9                                # where that coordinate hardly counts
    check(h, w, targets(N, V, 62, 7), top=top, grads=False)
    check(h, w, None, tau=0.7, top=top, grads=False)


@pytest.mark.parametrize('N,V,d', [(1500, 5003, 768), (2500, 5003, 136), (9000, 2100, 72), (6000, 900, 520)])
def test_rankings_of_many_rows(cuda, N, V, d):
    """Among so many some stand nearer their neighbours than the products round; rows of the weight of several sizes."""
    h, w = rand((N, d), 63), rand((V, d), 64, 0.05)
    w = w * (1 + torch.arange(V, device='cuda') % 4)[:, None].to(w.dtype)
    for top, given in ((32, True), (9, False)):
        check(h, w, targets(N, V, 65, 11) if given else None, top=top, grads=False)


@pytest.mark.parametrize('N', [5, 900])
def test_many_near_the_last_one_that_counts(cuda, N):
    """Tokens of one group and of others whose scores differ by less than fp32 sums tell, more of them than are asked for: which of
    them come first is a matter of the sums in 64 bits."""
    V, d = 5003, 256
    w = rand((V, d), 67, 0.05)
    base = rand((d,), 68)
    for i in range(12):                                  # six in one group of 32, six in groups of their own
        w[320 + 3 * i if i < 6 else 400 * (i - 4)] = base
    rows = torch.tensor([320 + 3 * i if i < 6 else 400 * (i - 4) for i in range(12)], device='cuda')
    w[rows, 7] = (torch.randn(12, generator=torch.Generator().manual_seed(69)) * 2.0 ** -10).bfloat16().cuda()
    h = base.repeat(N, 1) * rand((N, 1), 70).abs().clamp(min=0.1)
    h[:, 7] = 2.0 ** -5 * torch.where(torch.arange(N, device='cuda') % 2 == 0, 1.0, -1.0).bfloat16()
    for top in (2, 5, 9, 14):
        check(h, w, None, top=top, grads=False)
        check(h, w, targets(N, V, 71, 4), top=top, grads=False)


def test_weights_of_zeros(cuda):
    """All tokens are as likely: the first ones, whatever the hidden state."""
    import asrn_b200 as asrn
    for N, V in ((700, 5003), (6, 50304), (600, 1000)):
        h, w = rand((N, 64), 63), torch.zeros(V, 64, dtype=torch.bfloat16, device='cuda')
        r = check(h, w, targets(N, V, 64), top=20, grads=False)
        assert torch.equal(r.top_tokens, torch.arange(20, device='cuda').expand(N, 20))
        w[V // 3:] = rand((V - V // 3, 64), 65, 0.1)      # and where a part of them is
        check(h, w, None, top=20, grads=False)
        check(-h.abs(), w.abs(), targets(N, V, 66), top=20, grads=False)


def test_likeliest_tokens_in_one_group(cuda):
    """Common tokens have neighbouring numbers: all of the likeliest stand in one group of 128, or in two."""
    V, d = 4000, 64
    w = rand((V, d), 28, 0.1)
    h = rand((90, d), 29)
    for first in (0, 64, 128, 3900, 3990):
        v = w.clone()
        v[first:first + 40] *= 6
        check(h, v, targets(90, V, 30), top=32, grads=False)
        check(h, v, None, top=5, grads=False)


def test_minus_infinity_bad_rows_and_targets_outside(cuda):
    import asrn_b200 as asrn
    N, V, d = 40, 300, 64
    h, w = rand((N, d), 31).abs(), rand((V, d), 32, 0.1)
    w[::2] = -float('inf')                                # a vocabulary of which half is ruled out
    y = targets(N, V, 33) // 2 * 2 + 1
    r = check(h, w, y, top=5, grads=False)
    assert (r.top_tokens % 2 == 1).all()
    y[3] = 4                                              # a target that is ruled out
    r = asrn.head_stats(h, w, y, top=2)
    assert r.logp[3] == -float('inf') and torch.isfinite(r.entropy).all()
    few = asrn.head_stats(h[:, :8].contiguous(), w[:7, :8].contiguous(), None, top=7)     # 3 scores are finite
    assert (few.top_tokens.sort(1).values == torch.arange(7, device='cuda')).all()
    assert torch.equal(few.top_tokens[:, 3:], torch.tensor([0, 2, 4, 6], device='cuda').expand(N, 4))
    assert torch.isinf(few.top_logp[:, 3:]).all() and torch.isfinite(few.top_logp[:, :3]).all()
    w = rand((V, d), 34, 0.1)
    y = targets(N, V, 35)
    good = asrn.head_stats(h, w, y, top=3)
    hh = h.clone()
    hh[4, 2], hh[5, 3], hh[6, 1] = float('nan'), float('inf'), -float('inf')
    y[7], y[8] = V, 1 << 40
    r = asrn.head_stats(hh, w, y, top=3)
    bad = torch.zeros(N, dtype=torch.bool, device='cuda')
    bad[4:9] = True
    for t in (r.logp, r.entropy, r.top_logp):
        assert torch.isnan(t[bad]).all()
    assert (r.top_tokens[bad] == -1).all()
    for p, q in zip(r, good):
        assert torch.equal(p[~bad], q[~bad])


def test_logp_agrees_with_head_logprobs(cuda):
    import asrn_b200 as asrn
    N, V, d = 700, 5003, 200
    h, w, y = rand((N, d), 36).requires_grad_(), rand((V, d), 37, 0.1).requires_grad_(), targets(N, V, 38, 4)
    g = rand((N,), 39, dtype=torch.float32)
    a, b = asrn.head_logprobs(h, w, y, 0.7), asrn.head_stats(h, w, y, 0.7).logp
    assert (a - b).abs().max() <= 16 * E * (1 + a.abs().max())
    for p, q in zip(torch.autograd.grad(a, (h, w), g), torch.autograd.grad(b, (h, w), g)):
        assert (p.float() - q.float()).abs().max() <= 2 * U * p.float().abs().max()


@pytest.mark.parametrize('N,V', [(1, 50304), (9, 5003), (64, 700), (130, 5003), (900, 40000)])
def test_without_targets_and_gradients(cuda, N, V):
    """Nothing is gathered then: the values are those of the call that keeps them."""
    import asrn_b200 as asrn
    h, w = rand((N, 136), 70), rand((V, 136), 71, 0.1)
    a = check(h, w, None, top=7, grads=False)
    b = check(h, w, None, top=7)
    assert torch.equal(a.entropy, b.entropy) and torch.equal(a.top_tokens, b.top_tokens) and torch.equal(a.top_logp, b.top_logp)
    h[N // 2] = float('nan')
    c = asrn.head_stats(h, w, top=7)
    ok = torch.arange(N, device='cuda') != N // 2
    assert torch.equal(c.entropy[ok], a.entropy[ok]) and c.entropy[N // 2].isnan() and (c.top_tokens[N // 2] == -1).all()


def test_shapes_views_streams_autocast_and_empty(cuda):
    import asrn_b200 as asrn
    big, w, y = rand((6, 50, 100), 40), rand((321, 64), 41, 0.1), targets(300, 321, 42).view(6, 50)
    v = big[:, :, 9:73]
    r = asrn.head_stats(v, w, y, top=3)
    flat = check(v.reshape(300, 64), w, y.flatten(), top=3)
    assert r.logp.shape == (6, 50) and r.top_tokens.shape == (6, 50, 3)
    assert torch.equal(r.logp.flatten(), flat.logp) and torch.equal(r.top_logp.flatten(0, 1), flat.top_logp)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check(v.reshape(300, 64), w, y.flatten(), top=3)
    s.synchronize()
    one = asrn.head_stats(v[0, 0], w, top=2)               # a single position has no dimensions
    assert one.entropy.shape == () and one.top_tokens.shape == (2,) and one.logp is None
    assert torch.equal(one.top_tokens, asrn.head_stats(v[0, :1], w, top=2).top_tokens[0])
    h32, w32 = v.float().requires_grad_(), w.float().requires_grad_()
    with torch.autocast('cuda', dtype=torch.bfloat16):
        a = asrn.head_stats(h32, w32, y)
    assert torch.equal(a.entropy, r.entropy)
    assert all(t.dtype == torch.float32 for t in torch.autograd.grad(a.entropy.sum(), (h32, w32)))
    x = torch.empty(0, 64, dtype=torch.bfloat16, device='cuda').requires_grad_()
    ww = w.clone().requires_grad_()
    e = asrn.head_stats(x, ww, torch.empty(0, dtype=torch.int64, device='cuda'), top=2)
    assert e.logp.shape == (0,) and e.top_tokens.shape == (0, 2)
    dx, dw = torch.autograd.grad(e.entropy.sum(), (x, ww))
    assert (dw == 0).all() and dx.shape == (0, 64)


def test_repeats_bit_for_bit_and_in_a_graph(cuda):
    import asrn_b200 as asrn
    N, V, d = 700, 3001, 128
    h, w, y = rand((N, d), 43).requires_grad_(), rand((V, d), 44, 0.1).requires_grad_(), targets(N, V, 45, 5)
    g = tuple(rand((2, N), 46, dtype=torch.float32))

    def step():
        r = asrn.head_stats(h, w, y, 0.9, 6)
        return (*(t.detach() for t in r), *torch.autograd.grad((r.entropy, r.logp), (h, w), g))
    assert all(torch.equal(p, q) for p, q in zip(step(), step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        h.copy_(rand((N, d), 47))
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(step(), held))


def test_entropy_gradient_against_differences(cuda):
    """Along a direction of h and of W, by central differences of the entropy in 64 bits."""
    import asrn_b200 as asrn
    N, V, d = 30, 200, 64
    h, w = rand((N, d), 48).requires_grad_(), rand((V, d), 49, 0.2).requires_grad_()
    c = rand((N,), 50, dtype=torch.float32)
    dh, dw = torch.autograd.grad(asrn.head_stats(h, w, None, 0.8).entropy, (h, w), c)

    def value(h, w):
        lp = torch.log_softmax(h @ w.t() / 0.8, 1)
        return (-(lp.exp() * lp).sum(1) * c.double()).sum()
    for grad, leaf, f in ((dh, h, lambda t: value(t, w.detach().double())), (dw, w, lambda t: value(h.detach().double(), t))):
        u = rand(leaf.shape, 51, dtype=torch.float64)
        t = 1e-4
        diff = (f(leaf.detach().double() + t * u) - f(leaf.detach().double() - t * u)) / (2 * t)
        # gradients in bf16 (U each) from a dS whose remainder is multiplied too
        assert (diff - (grad.double() * u).sum()).abs() <= 2 * U * (grad.double() * u).abs().sum()


def test_refusals(cuda):
    import asrn_b200 as asrn
    h, w, y = rand((4, 64), 52), rand((30, 64), 53), torch.zeros(4, dtype=torch.int64, device='cuda')
    for error, call in [
            (ValueError, lambda: asrn.head_stats(h, w, y[:3])), (ValueError, lambda: asrn.head_stats(h, w[:, :32], y)),
            (TypeError, lambda: asrn.head_stats(h, w, y.int())), (ValueError, lambda: asrn.head_stats(h, w, y, 0.0)),
            (ValueError, lambda: asrn.head_stats(h, w, y, top=31)), (ValueError, lambda: asrn.head_stats(h, w, y, top=-1)),
            (ValueError, lambda: asrn.head_stats(h, torch.cat([w, w]), y, top=33)),
            (NotImplementedError, lambda: asrn.head_stats(h.float(), w.float(), y)),
            (NotImplementedError, lambda: asrn.head_stats(h[:, :12].contiguous(), w[:, :12].contiguous(), y)),
            (RuntimeError, lambda: asrn.head_stats(h.cpu(), w.cpu(), y.cpu())), (RuntimeError, lambda: asrn.head_stats(h, w, y.cpu()))]:
        with pytest.raises(error):
            call()

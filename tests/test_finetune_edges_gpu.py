"""The fine-tuning operators (asrn_b200.finetune) at their edges: sizes, values and calls that the tests by operator
(test_finetune_gpu.py, whose references and bounds these use) do not reach."""
import ctypes
import math

import pytest
import torch

from test_finetune_gpu import E, U, lengths_mask, mlp_reference, policy_reference, pref_reference, rand, run_mlp

pytestmark = pytest.mark.gpu


# ---- head ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('V,bad', [(2, 1), (129, 128), (257, 256), (300, 256), (257, 0), (1000, 700)])
def test_head_a_nan_in_the_weight_reaches_every_target(cuda, V, bad):
    """Each row's sum runs over all of the vocabulary, the row of `weight` that holds a NaN too."""
    import asrn_b200 as asrn
    N, d = 40, 64
    h, w = rand((N, d), 200), rand((V, d), 201, 0.1)
    y = torch.arange(N, device='cuda') % V
    clean = asrn.head_logprobs(h, w, y)
    assert clean.isfinite().all()
    w[bad, 5] = float('nan')
    if V > 256:
        w[256:] = w[bad]                                     # a part of the vocabulary that holds nothing else
    assert asrn.head_logprobs(h, w, y).isnan().all()
    y[3] = -1
    assert asrn.head_logprobs(h, w, y).isnan().tolist() == [i != 3 for i in range(N)]


def head_by_rows(h, w, y, g):
    """head_reference's logp, dh, dw and bounds' sums, some rows at a time."""
    w = w.double()
    lp, dh, sh = [], [], []
    dw, sw, size = torch.zeros_like(w), torch.zeros_like(w), 0.0
    for i in range(0, h.shape[0], 128):
        hi, yi, gi = h[i:i + 128].double(), y[i:i + 128], g[i:i + 128].double()
        z = hi @ w.t()
        on = (yi >= 0).double()
        logz = torch.log_softmax(z, 1)
        at = yi.clamp(min=0)[:, None]
        own = logz.gather(1, at)[:, 0]
        ds = -logz.exp() * (on * gi)[:, None]
        others = ds.sum(1) - ds.gather(1, at)[:, 0]
        ds.scatter_(1, at, -others[:, None])
        lp.append(own * on)
        dh.append(ds @ w)
        sh.append(ds.abs() @ w.abs())
        dw += ds.t() @ hi
        sw += ds.abs().t() @ hi.abs()
        size = max(size, float((hi.abs() @ w.abs().t()).amax()))
    return torch.cat(lp), torch.cat(dh), dw, torch.cat(sh), sw, size


@pytest.mark.parametrize('N,V,d,left', [(1500, 1 << 20, 8, 'third'), (1025, 1 << 20, 16, 'none'), (6000, 200003, 64, 'third'),
                                        (6000, 200003, 64, 'first'), (6000, 200003, 64, 'edge'),
                                        (6000, 200003, 64, 'all')])
def test_head_rows_in_several_chunks(cuda, N, V, d, left):
    """dS of all rows is over two gigabytes: it is made by chunks of rows, dW adding up over them; targets in every
    chunk, in the first one only, up to the second one's very start, and none at all."""
    import asrn_b200 as asrn
    from asrn_b200 import _lib
    pad, pitch = (N + 255) // 256 * 256, (V + 63) // 64 * 64
    assert _lib.lib().asrn_head_workspace_bytes(N, V, d, 1) < 0.9 * 2 * pad * pitch
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(210)).cuda()
    if left == 'third':
        y[::3] = -1
    elif left == 'first':
        y[500:] = -1
    elif left == 'edge':
        y[3072:] = -1                                        # the first chunk's rows: half of them, in blocks of 256
    elif left == 'all':
        y[:] = -1
    h, w = rand((N, d), 211).requires_grad_(), rand((V, d), 212, 0.1).requires_grad_()
    g = rand((N,), 213, dtype=torch.float32)
    logp = asrn.head_logprobs(h, w, y)
    dh, dw = torch.autograd.grad(logp, (h, w), g)
    ref, rh, rw, sh, sw, size = head_by_rows(h.detach(), w.detach(), y, g)
    tol = 4 * E * (d / 16 + 2) * size + 16 * E * (1 + ref.abs())
    assert ((logp.double() - ref).abs() <= tol).all()
    assert (logp[y < 0] == 0).all() and (dh[y < 0] == 0).all()
    assert ((dh.double() - rh).abs() <= U * (rh.abs() + sh) + 1e-30).all()
    assert ((dw.double() - rw).abs() <= U * (rw.abs() + sw) + 1e-30).all()


# ---- losses -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('rows', [1024, 1025, 2000])
def test_losses_of_many_sequences_without_positions(cuda, rows):
    """More rows than one block keeps, and no positions at all: zeros."""
    import asrn_b200 as asrn
    e = torch.zeros(rows, 0, device='cuda')
    for adv in (torch.ones(rows, device='cuda'), e):
        for per in ('token', 'sequence'):
            for ref in (None, e):
                r = asrn.policy_loss(e, e, adv, e.bool(), ref_logp=ref, kl=0.0 if ref is None else 0.1, per=per)
                assert r.grad.shape == (rows, 0)
                assert float(r.loss) == 0 and float(r.kl) == 0 and float(r.clipped) == 0
    e = torch.zeros(2, rows, 0, device='cuda')
    r = asrn.preference_loss(e, e, e.bool())
    assert float(r.loss) == 0 and r.grad.shape == e.shape and (r.chosen == 0).all() and (r.rejected == 0).all()


def test_policy_without_sequences_and_with_a_reference(cuda):
    """An empty batch has no log probabilities of the reference model in memory either: not an error."""
    import asrn_b200 as asrn
    e = torch.zeros(0, 5, device='cuda')
    r = asrn.policy_loss(e, e, e[:, 0], e.bool(), ref_logp=e, kl=0.1)
    assert float(r.loss) == 0 and float(r.kl) == 0 and r.grad.shape == (0, 5)


@pytest.mark.parametrize('eps', [0.0, 0.25])
def test_preference_infinite_margins(cuda, eps):
    """A token that the reference model holds impossible: the margin is infinite, and the loss what its formula gives
    there, 0 where the pair is on the right side and nothing is smoothed."""
    import asrn_b200 as asrn
    inf = float('inf')
    lp = torch.zeros(2, 2, 3, device='cuda')
    m = torch.ones_like(lp, dtype=torch.bool)
    for side, want, slope in ((0, inf if eps else 0.0, eps), (1, inf, eps - 1.0)):
        ref = lp.clone()
        ref[side, 1, 1] = -inf                               # R is +inf in that answer; the other pair's margin is 0
        r = asrn.preference_loss(lp, ref, m, beta=0.5, smoothing=eps)
        assert float(r.loss) == pytest.approx(want if want else math.log(2) / 2, rel=4 * E)
        assert r.grad[0, 1].tolist() == [0.25 * slope] * 3 and r.grad[1, 1].tolist() == [-0.25 * slope] * 3


@pytest.mark.parametrize('P,L', [(700, 2049), (300, 4096), (300, 20001), (300, 20000)])
@pytest.mark.parametrize('kind,eps', [('sigmoid', 0.2), ('ipo', 0.0)])
def test_preference_two_launches(cuda, P, L, kind, eps):
    """More than 2^21 tokens; from 16 chunks of 1024 in a row's part on the masks are read again."""
    import asrn_b200 as asrn
    assert 2 * P * L > 1 << 21
    ref = -rand((2, P, L), 240, dtype=torch.float32).abs()
    logp = ref + rand((2, P, L), 241, 0.02, torch.float32)
    mask = torch.stack([lengths_mask(P, L, 242, range(7, P, 9)), lengths_mask(P, L, 243, range(3, P, 11))])
    logp = torch.where(mask, logp, float('nan'))
    ref = torch.where(mask, ref, float('inf'))
    r = asrn.preference_loss(logp, ref, mask, beta=0.3, smoothing=eps, kind=kind)
    loss, grad, rew = pref_reference(logp, ref, mask, 0.3, eps, kind)
    assert abs(float(r.loss) - float(loss)) <= 4 * E * max(1.0, abs(float(loss)))
    assert (r.grad.double() - grad).abs().max() <= 4 * E * max(float(grad.abs().max()), 1e-30)
    assert (r.grad[~mask] == 0).all()
    got = torch.stack([r.chosen, r.rejected]).double()
    assert (got - rew).abs().max() <= 4 * E * max(float(rew.abs().max()), 1e-30)


@pytest.mark.parametrize('B,L', [(300, 1111), (129, 4096), (20, 40001)])
@pytest.mark.parametrize('per', ['token', 'sequence'])
@pytest.mark.parametrize('per_token,with_ref', [(False, True), (False, False), (True, True)])
def test_policy_two_launches(cuda, B, L, per, per_token, with_ref):
    """More than 2^18 tokens."""
    import asrn_b200 as asrn
    assert B * L > 1 << 18
    old = -rand((B, L), 250, dtype=torch.float32).abs() * 3
    logp = old + rand((B, L), 251, 0.3, torch.float32)
    ref = old + rand((B, L), 252, 0.3, torch.float32) if with_ref else None
    adv = rand((B, L) if per_token else (B,), 253, dtype=torch.float32)
    mask = lengths_mask(B, L, 254, range(5, B, 6))
    bad = torch.full_like(logp, float('nan'))
    logp, old = torch.where(mask, logp, bad), torch.where(mask, old, bad)
    ref = None if ref is None else torch.where(mask, ref, bad)
    adv = torch.where(mask, adv, bad) if per_token else adv
    kl = 0.1 if with_ref else 0.0
    r = asrn.policy_loss(logp, old, adv, mask, ref_logp=ref, clip=(0.2, 0.3), kl=kl, per=per)
    a = torch.where(mask, adv, torch.zeros_like(adv)) if per_token else adv
    loss, grad, k3, cut = policy_reference(logp, old, a, mask, ref, (0.2, 0.3), kl, per)
    size = 8 * float(a.abs().max()) + 1
    assert abs(float(r.loss) - float(loss)) <= 8 * E * size
    assert (r.grad.double() - grad).abs().max() <= 16 * E * max(float(grad.abs().max()), 1e-30)
    assert (r.grad[~mask] == 0).all()
    assert abs(float(r.kl) - float(k3)) <= 8 * E * max(1.0, float(k3)) and abs(float(r.clipped) - float(cut)) <= 2 * E


def test_policy_ratio_against_exp(cuda):
    """With an advantage of 1, no upper bound and 2^12 tokens the gradient is -exp(logp - old_logp) / 2^12: the
    exponential by itself. ex2.approx is off by 2^-22 of its result at most, the product's rounding is made up for to the
    first order (the second is below 2^-40), and the last addition rounds once: 2^-24."""
    import asrn_b200 as asrn
    d = torch.cat([torch.linspace(-20, 20, 3000), torch.linspace(-0.01, 0.01, 1090),
                   torch.tensor([20.0, -20.0, 0.0, -0.0, 1e-30, 2.0 ** -24])]).view(1, -1).cuda()
    assert d.numel() == 4096
    m = torch.ones_like(d, dtype=torch.bool)
    r = asrn.policy_loss(d, torch.zeros_like(d), torch.ones(1, device='cuda'), m, clip=(0.2, 1e30))
    got, want = -r.grad.double() * 4096, d.double().exp()
    assert float(r.clipped) == 0 and ((got - want).abs() <= (2.0 ** -22 + 2.0 ** -24) * 1.01 * want).all()


# ---- 8 bits -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('N', [600, 2051])
def test_mlp8_exponents_outside_the_table(cuda, N):
    """More than 512 rows, and columns whose x w1^T + b1 is above 254 or below 0.004 all over: gelu and its derivative
    of those blocks are computed, not looked up. Exact sums, as in test_mlp8_on_exact_sums, and its bound."""
    from asrn_b200 import finetune as ft
    d, ff, dout = 64, 160, 64
    g = torch.Generator().manual_seed(220)
    ints = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).float()  # noqa: E731
    x, w1, b1 = ints(-4, 4, N, d) / 4, ints(-2, 2, ff, d) / 8, ints(-8, 8, ff) / 8
    scale = torch.tensor([1.0, 2.0 ** 10, 2.0 ** -12, 1.0, 2.0 ** 20]).repeat_interleave(32)
    w1, b1 = w1 * scale[:, None], b1 * scale
    w2, b2, dy = ints(-4, 4, dout, ff) / 16, ints(-4, 4, dout) / 4, ints(-8, 8, N, dout) / 64
    ts = [t.bfloat16().cuda() for t in (x, w1, b1, w2, b2, dy)]
    e = ft.pack8((ts[0].float() @ ts[1].float().t() + ts[2].float()).bfloat16()).exps
    assert (e[:, 0] >= -14).all() and (e[:, 1] > 1).any() and (e[:, 2] < -14).all() and (e[:, 4] > 1).all()
    got = run_mlp(*ts)
    want, size = mlp_reference(*ts)
    for k in want:
        err = (got[k].double() - want[k]).abs()
        assert (err <= U * (want[k].abs() + size[k]) + 1e-30).all(), (k, float((err / (size[k] + 1e-30)).max()))


# ---- derivatives --------------------------------------------------------------------------------------------------------

def penalty_calls():
    import asrn_b200 as asrn
    h, w, y = rand((5, 16), 230), rand((9, 16), 231, 0.3), torch.arange(5, device='cuda')
    u, v, b = rand((8, 16), 232, 0.3), rand((16, 8), 233, 0.3), rand((8,), 234)
    z, m = torch.zeros(2, 3, 4, device='cuda'), torch.ones(2, 3, 4, dtype=torch.bool, device='cuda')
    return {'head': (h, lambda x: asrn.head_logprobs(x, w, y).sum()),
            'mlp8': (h, lambda x: asrn.mlp8(x, u, b, v, h[0]).float().square().sum()),
            'preference': (z.clone(), lambda x: asrn.preference_loss(x, z, m).loss),
            'policy': (z[0].clone(), lambda x: asrn.policy_loss(x, z[0], z[0, :, 0] + 1, m[0]).loss)}


@pytest.mark.parametrize('which', ['head', 'mlp8', 'preference', 'policy'])
def test_second_derivatives_are_refused(cuda, which):
    x, f = penalty_calls()[which]
    x.requires_grad_()
    first, = torch.autograd.grad(f(x), x)
    d, = torch.autograd.grad(f(x), x, create_graph=True)
    assert torch.equal(d, first)                             # the first derivative is there as ever
    penalty = d.float().square().sum() + x.float().square().sum()      # another term keeps the graph alive
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(penalty, x)
    d, = torch.autograd.grad(f(x), x, create_graph=True)
    with pytest.raises(RuntimeError, match='second derivative'):
        (d.float().square().sum() + x.float().square().sum()).backward()


def test_loss_scaled_by_a_parameter_that_learns(cuda):
    """The gradient is linear in what the loss is multiplied by, and that derivative is there."""
    import asrn_b200 as asrn
    z, m = torch.zeros(2, 3, 4, device='cuda'), torch.ones(2, 3, 4, dtype=torch.bool, device='cuda')
    x, s = z.clone().requires_grad_(), torch.tensor(3.0, device='cuda', requires_grad=True)
    r = asrn.preference_loss(x, z, m)
    d, = torch.autograd.grad(r.loss * s, x, create_graph=True)
    ds, = torch.autograd.grad(d.sum() + d[0].sum(), s)
    assert torch.allclose(ds, r.grad.sum() + r.grad[0].sum())


@pytest.mark.parametrize('which', ['head', 'mlp8', 'preference', 'policy'])
def test_forward_mode_is_refused(cuda, which):
    import torch.autograd.forward_ad as fwd
    x, f = penalty_calls()[which]
    with fwd.dual_level(), pytest.raises(NotImplementedError if which in ('preference', 'policy') else RuntimeError):
        f(fwd.make_dual(x, torch.ones_like(x)))


# ---- bounded waits ------------------------------------------------------------------------------------------------------

TIMEOUT = 5


def test_a_recorded_timeout_is_raised_until_it_is_cleared(cuda):
    """The word is written here as a kernel whose wait gives up writes it: no call goes on as if nothing had happened,
    forward or backward, and all do once it is cleared."""
    import asrn_b200 as asrn
    from asrn_b200 import _lib
    from asrn_b200 import finetune as ft
    h, w, y = rand((40, 64), 300), rand((99, 64), 301, 0.1).requires_grad_(), torch.arange(40, device='cuda')
    u, b, v, c = rand((48, 64), 302, 0.1), rand((48,), 303), rand((64, 48), 304), rand((64,), 305)
    calls = [lambda: asrn.head_logprobs(h, w, y), lambda: asrn.mlp8(w, u, b, v, c)]
    outs = [f() for f in calls]
    want = [torch.autograd.grad(o.float().sum(), w, retain_graph=True)[0] for o in outs]
    assert ft.status() == 0
    word = ctypes.c_int.from_address(_lib.finetune().status_address(0))
    word.value = TIMEOUT
    try:
        for f in calls + [lambda o=o: torch.autograd.grad(o.float().sum(), w, retain_graph=True) for o in outs]:
            with pytest.raises(RuntimeError, match='bounded wait'):
                f()
        assert ft.status() == TIMEOUT and ft.status() == TIMEOUT
        assert ft.status(reset=True) == TIMEOUT and ft.status() == 0
    finally:
        word.value = 0
    assert all(torch.equal(f(), o) for f, o in zip(calls, outs))
    assert all(torch.equal(torch.autograd.grad(o.float().sum(), w)[0], a) for o, a in zip(outs, want))
    with pytest.raises(ValueError):
        ft.status('cpu')


def test_an_earlier_calls_timeout_stops_no_later_call(cuda):
    """The C entries with a status word that already holds a timeout: the products wait for their operands all the same."""
    from asrn_b200 import _lib
    L, P, s = _lib.lib(), _lib.ptr, _lib.stream_ptr(cuda)
    N, V, d, ff = 600, 5003, 256, 512
    h, w = rand((N, d), 310), rand((V, d), 311, 0.1)
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(312)).cuda()
    u, b, v, c = rand((ff, d), 313, 0.1), rand((ff,), 314), rand((d, ff), 315, 0.1), rand((d,), 316)
    buf = lambda n: torch.empty(n, dtype=torch.uint8, device='cuda')  # noqa: E731
    nb = [L.asrn_head_saved_bytes(N, d), L.asrn_head_workspace_bytes(N, V, d, 0), L.asrn_mlp8_workspace_bytes(N, d, ff, d, 0)]
    mem = [buf(n) for n in nb]
    out = []
    for before in (0, TIMEOUT):
        word = torch.full((1,), before, dtype=torch.int32, device='cuda')
        lp, z = torch.full((N,), 7.0, device='cuda'), torch.full((N, d), 7.0, dtype=torch.bfloat16, device='cuda')
        assert L.asrn_head_forward(N, V, d, P(h), P(w), P(y), 1.0, P(lp), P(mem[0]), nb[0], P(mem[1]), nb[1], P(word), s) == 0
        assert L.asrn_mlp8_forward(N, d, ff, d, P(h), P(u), P(b), P(v), P(c), P(z), None, 0, P(mem[2]), nb[2], P(word), s) == 0
        assert int(word) == before
        out.append((lp, z))
    assert all(torch.equal(a, b) for a, b in zip(*out))


# ---- the model's blocks --------------------------------------------------------------------------------------------------

def block8(d=64):
    import asrn_b200 as asrn
    m = asrn.create_model(V=64, d=d, n_capas=2, semilla=0, checkpoint='8bits').cuda().train()
    return m.bloques[0], torch.randn(2, 33, d, generator=torch.Generator().manual_seed(1)).cuda()


@pytest.mark.parametrize('how', ['hook', 'pre-hook', 'backward hook', 'other linear', 'activation', 'no bias', 'forward'])
def test_8bit_blocks_call_the_mlps_own_modules_where_they_do_more(cuda, how):
    blq, h = block8()
    seen = []
    lin, act = blq.ff[0], blq.ff[1]
    if how == 'hook':
        lin.register_forward_hook(lambda m, i, o: seen.append(1) or o * 2)
    elif how == 'pre-hook':
        blq.ff.register_forward_pre_hook(lambda m, i: seen.append(1))
    elif how == 'backward hook':
        act.register_full_backward_hook(lambda m, i, o: seen.append(1))
    elif how == 'other linear':
        class Twice(torch.nn.Linear):
            def forward(self, x):
                seen.append(1)
                return 2 * super().forward(x)
        new = Twice(lin.in_features, lin.out_features).cuda()
        new.load_state_dict(lin.state_dict())
        blq.ff[0] = new
    elif how == 'activation':
        class Relu(torch.nn.ReLU):
            def forward(self, x):
                seen.append(1)
                return super().forward(x)
        blq.ff[1] = Relu()
    elif how == 'no bias':
        blq.ff[0].bias = None
        seen.append(1)
    else:
        own = lin.forward
        lin.forward = lambda x: seen.append(1) or own(x)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        out = blq(h)
        out.sum().backward()
        assert seen
        blq.activaciones_8bits = False
        assert torch.equal(blq(h), out)


@pytest.mark.parametrize('how', ['hook', 'bias', 'other class'])
def test_logprobs_call_the_head_where_it_does_more(cuda, how):
    """A head that is more than its weight (a hook, a bias, a class of its own) is called, in bf16 too."""
    import asrn_b200 as asrn
    m = asrn.create_model(V=64, d=64, n_capas=2, semilla=0).cuda()
    x = torch.randint(0, 64, (2, 33), generator=torch.Generator().manual_seed(2)).cuda()
    if how == 'hook':
        m.head.register_forward_hook(lambda _, i, o: o * 3)
    else:
        class Shifted(torch.nn.Linear):
            def forward(self, h):
                return 3 * super().forward(h)
        new = (Shifted if how == 'other class' else torch.nn.Linear)(64, 64, bias=how == 'bias').cuda()
        m.head = new
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        h = m.estado(x)
        m.estado = lambda x: h
        want = torch.log_softmax(m(x).float(), -1)[:, :-1].gather(-1, x[:, 1:, None])[..., 0]
        assert torch.equal(m.logprobs(x)[:, :-1], want)

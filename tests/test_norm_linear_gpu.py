"""layer_norm and linear against plain implementations in 64 bits. Bounds, with U = 2^-8 the unit roundoff of bf16 and
E = 2^-24 that of fp32 (a sum of n terms in fp32 by parts: at most its longest chain of additions times E sum|terms|):
  norm       a row's sums: chains of at most 32 additions a thread, 5 in a warp, 16 over warps: 64 E mean|s| for the mean, which
             moves (s - m) k by DH = 64 E mean|s| k; 64 E relative for 1 / sqrt(var) and the products after it
  columns    dw, db: chains of at most rows / 128 + 64 additions
  products   d products summed in fp32, 16 at a time, truncated: (d / 16 + 2) 2 E sum|x w|
  act        gelu and silu are off by 4e-7 max(1, |a|), their slopes by 5e-7; a slope kept in fp16 (11 bits of
             significand: half a step is 2^-11 of the value) by 2^-11 of itself or 2^-25
  roundings  a result in bf16: U of itself; dA as an operand: U of itself above 512 rows, U^2 up to there"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def rand(shape, seed, scale=1.0, dtype=BF16, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).cuda()


def unit(dtype):
    return U if dtype == BF16 else E


def close(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs().max()),
                           float(((got.double() - want).abs() / tol.clamp(min=1e-300)).max()))


# ---- layer norm -----------------------------------------------------------------------------------------------------

def check_norm(x, w, b, res=None, dtype=None, eps=1e-5, grads=True):
    import asrn_b200 as asrn
    N, d = x.numel() // x.shape[-1], x.shape[-1]
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, res)]
    x, w, b, res = leaves
    out = asrn.layer_norm(x, w, b, residual=res, eps=eps, dtype=dtype)
    y, s = (out, x) if res is None else out
    dtype = dtype or x.dtype
    assert y.dtype == dtype and y.shape == x.shape
    if res is not None:
        want = (x.detach().float() + res.detach().float()).to(res.dtype)
        assert torch.equal(s.detach(), want) and s.dtype == res.dtype
    s64, w64 = s.detach().double().view(N, d), w.detach().double()
    m, v = s64.mean(1, keepdim=True), s64.var(1, unbiased=False, keepdim=True)
    k = (v + eps).rsqrt()
    h = (s64 - m) * k
    ref = h * w64 + (b.detach().double() if b is not None else 0)
    DH = 64 * E * s64.abs().mean(1, keepdim=True) * k + 64 * E * h.abs()
    close(y.detach().view(N, d), ref, DH * w64.abs() + 4 * E * (ref.abs() + (h * w64).abs()) + unit(dtype) * ref.abs() + 1e-38,
          'y')
    if not grads:
        return
    dy = rand(x.shape, 90, dtype=dtype)
    ds = rand(x.shape, 91, dtype=res.dtype) if res is not None else None
    into = [t for t in leaves if t is not None]
    got = dict(zip([n for n, t in zip(('x', 'w', 'b', 'res'), leaves) if t is not None],
                   torch.autograd.grad(out, into, dy if res is None else (dy, ds))))
    dy64 = dy.double().view(N, d)
    g = dy64 * w64
    gm, hm = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = k * (g - gm - h * hm)
    ga, ha = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    tol = k * (128 * E * (g.abs() + ga + h.abs() * ha) + DH * ha + h.abs() * (g.abs() * DH).mean(1, keepdim=True))
    if ds is not None:
        dx = dx + ds.double().view(N, d)
    tol = tol + 4 * E * (dx.abs() + (ds.double().abs().view(N, d) if ds is not None else 0))
    close(got['x'].view(N, d), dx, tol + unit(x.dtype) * dx.abs() + 1e-38, 'dx')
    if res is not None:
        close(got['res'].view(N, d), dx, tol + unit(res.dtype) * dx.abs() + 1e-38, 'dres')
    depth = (N / 128 + 64) * E
    dw = (dy64 * h).sum(0)
    close(got['w'], dw, (dy64.abs() * DH).sum(0) + depth * (dy64 * h).abs().sum(0) + unit(w.dtype) * dw.abs() + 1e-38, 'dw')
    if b is not None:
        close(got['b'], dy64.sum(0), depth * dy64.abs().sum(0) + unit(b.dtype) * dy64.sum(0).abs() + 1e-38, 'db')
    return got


@pytest.mark.parametrize('N,d', [(1, 1), (3, 2), (1, 8), (5, 7), (33, 64), (129, 256), (130, 257), (65, 264), (700, 512), (40, 513),
                                 (601, 768), (64, 1000), (33, 1024), (9, 1025), (21, 1032), (17, 2048), (31, 2056),
                                 (12, 4096), (7, 4104), (9, 5001), (5, 8192), (4, 8200), (3, 8193), (3, 16384), (2, 16383),
                                 (2500, 96), (5003, 40)])
def test_norm_sizes(cuda, N, d):
    check_norm(rand((N, d), 1, dtype=F32, shift=0.5), rand((d,), 2, 0.3, F32, 1.0), rand((d,), 3, dtype=F32))


@pytest.mark.parametrize('x', [F32, BF16])
@pytest.mark.parametrize('res', [None, F32, BF16])
@pytest.mark.parametrize('y', [F32, BF16])
@pytest.mark.parametrize('d', [72, 300, 768, 1536, 77])
def test_norm_types(cuda, x, res, y, d):
    N = 150
    check_norm(rand((3, N // 3, d), 4, dtype=x), rand((d,), 5, 0.3, F32, 1.0), rand((d,), 6, dtype=F32),
               None if res is None else rand((3, N // 3, d), 7, 2.0, res, 0.3), y)
    check_norm(rand((N, d), 8, dtype=x), rand((d,), 9, 0.3, BF16, 1.0), None,
               None if res is None else rand((N, d), 10, dtype=res), y)


def test_norm_rows_with_a_large_mean_and_constant_rows(cuda):
    d = 768
    x = rand((64, d), 11, dtype=F32)
    x[::4] += 1000.0
    x[1::4] = 3.0
    x[2::4] = 0.0
    x[3::4, 5] = 1e6
    check_norm(x, rand((d,), 12, 0.3, F32, 1.0), rand((d,), 13, dtype=F32))


def test_norm_bad_values_stay_in_their_rows(cuda):
    import asrn_b200 as asrn
    d = 256
    x = rand((40, d), 14, dtype=F32)
    w, b = rand((d,), 15, dtype=F32), rand((d,), 16, dtype=F32)
    good = asrn.layer_norm(x, w, b)
    x[3, 7], x[11, 0], x[12, 9] = float('nan'), float('inf'), -float('inf')
    y = asrn.layer_norm(x, w, b)
    bad = torch.zeros(40, dtype=torch.bool, device='cuda')
    bad[[3, 11, 12]] = True
    assert torch.isnan(y[bad]).any(1).all() and torch.equal(y[~bad], good[~bad])


def test_norm_views_streams_and_empty(cuda):
    """Rows that are slices, misaligned, transposed; a stream of their own; no rows; only some gradients; no gradient of the sum."""
    import asrn_b200 as asrn
    big = rand((70, 900), 17, dtype=F32)
    w, b = rand((768,), 18, dtype=F32), rand((768,), 19, dtype=F32)
    for v in (big[:, 3:771], big[:, 8:776], big[::2, 100:868], rand((768, 50), 20, dtype=F32).t(),
              big.flatten()[1:1 + 768 * 60].view(60, 768)):
        assert torch.equal(asrn.layer_norm(v, w, b), asrn.layer_norm(v.contiguous().clone(), w, b)) or \
            v.is_contiguous()
        check_norm(v, w, b)
    check_norm(rand((10, 256), 21, dtype=F32), big.flatten()[3:259], big.flatten()[301:557])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check_norm(big[:, :768], w, b)
    s.synchronize()
    x = torch.empty(0, 768, device='cuda', requires_grad=True)
    ww = w.clone().requires_grad_()
    y = asrn.layer_norm(x, ww, b)
    assert y.shape == (0, 768)
    dx, dw = torch.autograd.grad(y.sum(), (x, ww))
    assert dx.shape == x.shape and (dw == 0).all()
    x = big[:, :768].contiguous().requires_grad_()
    r = rand((70, 768), 22, dtype=F32).requires_grad_()
    y, t = asrn.layer_norm(x, w, b, residual=r)
    assert not w.requires_grad
    gx, gr = torch.autograd.grad(t.sum(), (x, r), retain_graph=True)       # y has no part
    assert (gx == 1).all() and (gr == 1).all()
    gx, = torch.autograd.grad(y, (x,), torch.ones_like(y), retain_graph=True)
    gr, = torch.autograd.grad(y, (r,), torch.ones_like(y))
    assert torch.equal(gx, gr)


@pytest.mark.parametrize('d', [768, 333])
@pytest.mark.parametrize('x,res', [(BF16, F32), (F32, F32), (F32, None)])
def test_norm_one_gradient_at_a_time_and_shared_inputs(cuda, d, x, res):
    import asrn_b200 as asrn
    t = dict(x=rand((90, d), 100, dtype=x), w=rand((d,), 101, dtype=F32), b=rand((d,), 102, dtype=F32),
             res=None if res is None else rand((90, d), 103, dtype=res))
    t = {k: v for k, v in t.items() if v is not None}
    dy = rand((90, d), 104, dtype=x)
    call = lambda q: asrn.layer_norm(q['x'], q['w'], q['b'], residual=q.get('res'))  # noqa: E731
    first = lambda r: r if res is None else r[0]  # noqa: E731
    every = {k: v.clone().requires_grad_() for k, v in t.items()}
    want = dict(zip(every, torch.autograd.grad(first(call(every)), tuple(every.values()), dy)))
    for need in t:
        one = {k: v.clone().requires_grad_(k == need) for k, v in t.items()}
        got, = torch.autograd.grad(first(call(one)), (one[need],), dy)
        assert torch.equal(got, want[need]), need
    if x == res:                                          # the same tensor as both summands
        both = t['x'].clone().requires_grad_()
        y, s = asrn.layer_norm(both, t['w'], t['b'], residual=both)
        got, = torch.autograd.grad(y, (both,), dy)
        two = t['x'].clone().requires_grad_()
        want, = torch.autograd.grad(asrn.layer_norm(2 * two, t['w'], t['b']), (two,), dy)
        assert torch.equal(s, 2 * both) and torch.equal(got, want)


def test_norm_rows_at_the_end_of_their_memory(cuda):
    """Odd widths are read by whole vectors: what lies before and behind the rows reaches nothing and is left alone."""
    import asrn_b200 as asrn
    for N, d in ((1, 3), (2, 7), (5, 77), (9, 130), (7, 333), (3, 1021), (3, 2051), (3, 5001)):
        room = torch.full((N * d + 64,), float('nan'), device='cuda')
        x = room[32:32 + N * d].view(N, d)                # 128 bytes in: aligned, NaN on both sides
        x.copy_(rand((N, d), 105, dtype=F32))
        w, b = rand((d,), 106, dtype=F32), rand((d,), 107, dtype=F32)
        check_norm(x, w, b)
        assert torch.equal(asrn.layer_norm(x, w, b), asrn.layer_norm(x.clone(), w, b))
        assert room[:32].isnan().all() and room[32 + N * d:].isnan().all()


def test_norm_repeats_bit_for_bit_and_in_a_graph(cuda):
    import asrn_b200 as asrn
    x, w, b = rand((3001, 520), 23, dtype=F32), rand((520,), 24, dtype=F32), rand((520,), 25, dtype=F32)
    r, dy = rand((3001, 520), 26), rand((3001, 520), 27, dtype=F32)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]

    def step():
        y, s = asrn.layer_norm(x, w, b, residual=r)
        return (y.detach(), s.detach(), *torch.autograd.grad((y, s), leaves, (dy, s.detach())))
    one, two = step(), step()                            # of detached results: no eager graph may live under a capture
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        x.copy_(rand((3001, 520), 28, dtype=F32))
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(step(), held))


# ---- product with bias, activation and residual -----------------------------------------------------------------------

ACTS = [None, 'gelu', 'silu', 'relu']


def act64(kind, a):
    if kind == 'gelu':
        cdf = 0.5 * torch.erfc(-a / 2 ** 0.5)
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / (2 * torch.pi) ** 0.5
    if kind == 'silu':
        p = torch.sigmoid(a)
        return a * p, p * (1 + a * (1 - p))
    if kind == 'relu':
        return a.clamp(min=0), (a > 0).double()
    return a, torch.ones_like(a)


def check_linear(x, w, b=None, act=None, res=None, grads=True):
    import asrn_b200 as asrn
    n, d = w.shape
    N = x.numel() // d
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, res)]
    x, w, b, res = leaves
    y = asrn.linear(x, w, b, activation=act, residual=res)
    dtype = BF16 if res is None else res.dtype
    assert y.dtype == dtype and y.shape == (*x.shape[:-1], n)
    x64, w64 = x.detach().double().view(N, d), w.detach().double()
    a = x64 @ w64.t()
    acc = (d / 16 + 2) * 2 * E * (x64.abs() @ w64.abs().t()) + 2 * E * a.abs()
    if b is not None:
        a = a + b.detach().double()
        acc = acc + E * a.abs()
    f, slope = act64(act, a)
    off = 1.2 * acc + (4e-7 * a.abs().clamp(min=1) if act else 0)
    ref = f if res is None else f + res.detach().double().view(N, n)
    close(y.detach().view(N, n), ref, off + 4 * E * (ref.abs() + f.abs()) + unit(dtype) * ref.abs() + 1e-38, 'y')
    if not grads:
        return
    dy = rand(y.shape, 92, dtype=dtype)
    into = [t for t in leaves if t is not None]
    got = dict(zip([k for k, t in zip(('x', 'w', 'b', 'res'), leaves) if t is not None], torch.autograd.grad(y, into, dy)))
    dy64 = dy.double().view(N, n)
    da = dy64 * slope
    dda = 0 * da
    if act:
        dda = dy64.abs() * (2.0 ** -11 * slope.abs() + 2.0 ** -25 + 5e-7 + acc)
        if act == 'relu':
            dda = dda + dy64.abs() * (a.abs() <= acc)
    exact = act is None and dtype == BF16
    cut = 0 if exact else U if N > 512 else U * U
    daw = dda + cut * (da.abs() + dda) + E * da.abs()
    dx = da @ w64
    close(got['x'].view(N, d), dx, U * dx.abs() + 1.01 * daw @ w64.abs() + (2 * n / 16 + 2) * 2 * E * (da.abs() @ w64.abs())
          + 1e-38, 'dx')
    dw = da.t() @ x64
    close(got['w'], dw, U * dw.abs() + 1.01 * daw.t() @ x64.abs() + (2 * N / 16 + 40) * 2 * E * (da.abs().t() @ x64.abs())
          + 1e-38, 'dw')
    if b is not None:
        db = da.sum(0)
        close(got['b'], db, U * db.abs() + dda.sum(0) + (N / 64 + 64) * E * da.abs().sum(0) + 1e-38, 'db')
    if res is not None:
        assert torch.equal(got['res'], dy)
    return got


@pytest.mark.parametrize('N,d,n', [(1, 8, 8), (1, 768, 1536), (2, 16, 24), (7, 40, 72), (8, 64, 128), (9, 72, 8), (16, 256, 520),
                                   (17, 200, 264), (32, 1536, 768), (33, 128, 16), (63, 264, 248), (64, 768, 1536), (65, 64, 128),
                                   (127, 96, 40), (128, 520, 256), (129, 72, 264), (300, 8, 1024), (512, 256, 512),
                                   (513, 256, 520), (1003, 200, 520), (1500, 1032, 8), (2049, 64, 2056), (70, 64, 50304)])
@pytest.mark.parametrize('act', ['gelu', None])
def test_linear_sizes(cuda, N, d, n, act):
    check_linear(rand((N, d), 30), rand((n, d), 31, d ** -0.5), rand((n,), 32, 0.3), act, grads=n < 5000)


@pytest.mark.parametrize('N', [5, 13, 30, 64, 200, 700])
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('res', [None, F32, BF16])
@pytest.mark.parametrize('bias', [True, False])
def test_linear_kinds(cuda, N, act, res, bias):
    d, n = 136, 328
    check_linear(rand((N, d), 33), rand((n, d), 34, 0.2), rand((n,), 35) if bias else None, act,
                 None if res is None else rand((N, n), 36, dtype=res))


@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('N', [3, 700])
def test_linear_activations_over_their_range(cuda, act, N):
    """Arguments from tiny to large of both signs, through a product that passes them on."""
    d = n = 64
    x = torch.zeros(N, d)
    x[:, :] = torch.randn(N, d, generator=torch.Generator().manual_seed(37)) * torch.logspace(-6, 2.3, d)
    check_linear(x.bfloat16().cuda(), torch.eye(n).bfloat16().cuda(), None, act, rand((N, n), 38, 1e-3, F32))


@pytest.mark.parametrize('N', [4, 300])
@pytest.mark.parametrize('act', ACTS)
def test_linear_infinities_and_nan(cuda, N, act):
    """Sums past bf16's range and NaN in a row: the limits, and NaN in that row alone."""
    import asrn_b200 as asrn
    d, n = 64, 72
    x, w = rand((N, d), 39), rand((n, d), 40, 0.2)
    good = asrn.linear(x, w, None, act)
    x[1], w2 = 0, w.clone()
    x[1, 0], w2[:, 0] = 3e38, 0
    w2[0, 0], w2[1, 0] = 1e5, -1e5                       # +inf and -inf in fp32
    x[2, 5] = float('nan')
    y = asrn.linear(x, w2, None, act).float()
    assert y[1, 0] == float('inf') and y[1, 1] == (-float('inf') if act is None else 0) and (y[1, 2:] == 0).all()
    assert torch.isnan(y[2]).all() and not torch.isnan(y[3]).any()
    x[1], x[2] = 0, 0
    assert torch.equal(asrn.linear(x, w, None, act)[3], good[3])


@pytest.mark.parametrize('N,d,n', [(4096, 72, 64), (4100, 72, 64), (1025, 40, 256), (200, 1000, 1312), (5000, 264, 56), (16, 64, 65536),
                                   (17, 64, 15424), (96, 2056, 136), (320, 136, 816), (321, 136, 824),
                                   (6144, 72, 64), (6145, 72, 64), (48, 264, 8192), (49, 264, 8192), (16, 72, 50304), (17, 72, 50304),
                                   (1200, 264, 328), (3000, 1000, 136), (700, 1544, 600)])
@pytest.mark.parametrize('act', ['silu', None])
def test_linear_sizes_on_both_sides_of_the_rule(cuda, N, d, n, act):
    check_linear(rand((N, d), 130), rand((n, d), 131, d ** -0.5), rand((n,), 132, 0.3), act, rand((N, n), 133), grads=n < 5000)


@pytest.mark.parametrize('N,n', [(900, 328), (270, 1000), (1300, 328), (400, 1000)])
@pytest.mark.parametrize('act', ACTS)
@pytest.mark.parametrize('res', [None, F32, BF16])
@pytest.mark.parametrize('bias', [True, False])
def test_linear_kinds_of_larger_products(cuda, N, n, act, res, bias):
    check_linear(rand((N, 136), 134), rand((n, 136), 135, 0.2), rand((n,), 136) if bias else None, act,
                 None if res is None else rand((N, n), 137, dtype=res))


@pytest.mark.parametrize('act', ACTS)
def test_larger_products_over_the_range_and_with_infinities(cuda, act):
    test_linear_activations_over_their_range(cuda, act, 4200)
    test_linear_infinities_and_nan(cuda, 3700, act)
    test_linear_activations_over_their_range(cuda, act, 6200)
    test_linear_infinities_and_nan(cuda, 5600, act)


@pytest.mark.parametrize('N,n', [(130, 96), (5000, 96)])
def test_linear_rows_do_not_meet(cuda, N, n):
    """A row's result is its own: other rows changed, and rows behind the last one of the memory, change nothing."""
    import asrn_b200 as asrn
    x, w, r = rand((N + 70, 200), 138), rand((n, 200), 139, 0.1), rand((N + 70, n), 140, dtype=F32)
    x[N:], r[N:] = float('nan'), float('nan')
    y = asrn.linear(x[:N], w, None, 'gelu', r[:N])
    assert y.isfinite().all()
    x[1::2], r[1::2] = float('nan'), float('nan')
    z = asrn.linear(x[:N], w, None, 'gelu', r[:N])
    assert torch.equal(z[::2], y[::2]) and z[1::2].isnan().all()


@pytest.mark.parametrize('N', [30, 900])
@pytest.mark.parametrize('res', [F32, BF16])
def test_linear_one_gradient_at_a_time_and_broadcast_inputs(cuda, N, res):
    import asrn_b200 as asrn
    t = dict(x=rand((N, 72), 141), w=rand((520, 72), 142, 0.2), b=rand((520,), 143), r=rand((N, 520), 144, dtype=res))
    dy = rand((N, 520), 145, dtype=res)
    call = lambda q: asrn.linear(q['x'], q['w'], q['b'], 'gelu', q['r'])  # noqa: E731
    every = {k: v.clone().requires_grad_() for k, v in t.items()}
    want = dict(zip(every, torch.autograd.grad(call(every), tuple(every.values()), dy)))
    assert torch.equal(want['r'], dy)
    for need in t:
        one = {k: v.clone().requires_grad_(k == need) for k, v in t.items()}
        got, = torch.autograd.grad(call(one), (one[need],), dy)
        assert torch.equal(got, want[need]), need
    # inputs that are a row given to every row: their gradients are the rows' sums
    row, rrow = t['x'][:1].clone().requires_grad_(), t['r'][:1].clone().requires_grad_()
    q = dict(every, x=row.expand(N, 72), r=rrow.expand(N, 520))
    got = torch.autograd.grad(call(q), (row, rrow), dy)
    full = dict(every, x=t['x'][:1].repeat(N, 1).requires_grad_(), r=t['r'][:1].repeat(N, 1).requires_grad_())
    dx, dr = torch.autograd.grad(call(full), (full['x'], full['r']), dy)
    assert torch.equal(got[0], dx.sum(0, keepdim=True)) and torch.equal(got[1], dr.sum(0, keepdim=True))
    # a scalar's backward pass: a gradient without strides of its own
    dx, = torch.autograd.grad(call(every).sum(), (every['x'],))
    assert torch.equal(dx, torch.autograd.grad(call(every), (every['x'],), torch.ones_like(dy))[0])


def test_linear_views_streams_and_empty(cuda):
    import asrn_b200 as asrn
    big = rand((300, 400), 41)
    w, b = rand((96, 128), 42, 0.1), rand((96,), 43)
    for v in (big[:, 5:133], big[::3, 8:136], rand((128, 90), 44).t(), big[:130, :384].view(130, 3, 128)):
        assert torch.equal(asrn.linear(v, w, b, 'silu'), asrn.linear(v.contiguous(), w, b, 'silu'))
        check_linear(v, w, b, 'silu')
    check_linear(big[:70, :128], rand((128, 96), 45, 0.1).t(), big.flatten()[3:99], 'gelu', rand((96, 70), 46, dtype=F32).t())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check_linear(big[:, :128], w, b, 'gelu')
        check_linear(big[:9, :128], w, b, 'gelu')
    s.synchronize()
    x, ww, bb = torch.empty(0, 5, 128, dtype=BF16, device='cuda').requires_grad_(), w.clone().requires_grad_(), \
        b.clone().requires_grad_()
    y = asrn.linear(x, ww, bb, 'relu')
    assert y.shape == (0, 5, 96)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, ww, bb))
    assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
    for need in ('x', 'w', 'b', 'res'):                  # one gradient at a time
        t = dict(x=big[:, :128].clone(), w=w.clone(), b=b.clone(), res=rand((300, 96), 47, dtype=F32))
        t[need].requires_grad_()
        y = asrn.linear(t['x'], t['w'], t['b'], 'gelu', t['res'])
        dy = rand(y.shape, 48, dtype=F32)
        one, = torch.autograd.grad(y, (t[need],), dy)
        every = {k: v.detach().requires_grad_() for k, v in t.items()}
        y = asrn.linear(every['x'], every['w'], every['b'], 'gelu', every['res'])
        assert torch.equal(one, torch.autograd.grad(y, tuple(every.values()), dy)[list(every).index(need)])


def test_linear_under_autocast_casts_as_a_linear_layer_does(cuda):
    import asrn_b200 as asrn
    x, w, b = (t.requires_grad_() for t in (rand((90, 64), 49, dtype=F32), rand((40, 64), 50, 0.2, F32), rand((40,), 51, dtype=F32)))
    with pytest.raises(NotImplementedError):
        asrn.linear(x, w, b)
    with torch.autocast('cuda', dtype=BF16):
        y = asrn.linear(x, w, b, 'gelu', x[:, :40])
    assert y.dtype == F32
    z = asrn.linear(x.bfloat16(), w.bfloat16(), b.bfloat16(), 'gelu', x[:, :40])
    assert torch.equal(y, z)
    for p, q in zip(torch.autograd.grad(y.sum(), (x, w, b)), torch.autograd.grad(z.sum(), (x, w, b))):
        assert p.dtype == F32 and torch.equal(p, q)


@pytest.mark.parametrize('N', [40, 900])
def test_linear_repeats_bit_for_bit_and_in_a_graph(cuda, N):
    import asrn_b200 as asrn
    x, w, b, r = (t.requires_grad_() for t in (rand((N, 264), 52), rand((520, 264), 53, 0.1), rand((520,), 54),
                                               rand((N, 520), 55, dtype=F32)))
    dy = rand((N, 520), 56, dtype=F32)

    def step():
        y = asrn.linear(x, w, b, 'gelu', r)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b, r), dy))
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
        x.copy_(rand((N, 264), 57))
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(step(), held))


def test_linear_gradient_against_differences(cuda):
    """The loss along a direction of each leaf, by central differences of the operator's own fp32 output."""
    import asrn_b200 as asrn
    N, d, n = 100, 64, 48
    x, w, b, r = rand((N, d), 58), rand((n, d), 59, 0.2), rand((n,), 60), rand((N, n), 61, dtype=F32)
    dy = rand((N, n), 62, dtype=F32)
    for act in ('gelu', 'silu'):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        grads = torch.autograd.grad(asrn.linear(*leaves[:3], act, leaves[3]), leaves, dy)
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            # steps that bf16 holds: a power of two of each value's own size
            step = (leaf.detach() * 2.0 ** -4 * torch.sign(rand(leaf.shape, 63 + i, dtype=F32))).to(leaf.dtype)
            args = lambda sign: [t.detach() if j != i else (t.detach() + sign * step) for j, t in enumerate(leaves)]  # noqa: E731
            lo, hi = args(-1), args(1)
            moved = (hi[i].double() - lo[i].double())
            f = lambda a: (asrn.linear(*a[:3], act, a[3]).double() * dy.double()).sum()  # noqa: E731
            diff, along = f(hi) - f(lo), (grad.double() * moved).sum()
            # the third derivative's part, steps of 1/16 of values of about 1: 1/24 (1/16 2)^3 of sum|dy| at the most; the
            # gradients' roundings U of sum|grad step|
            tol = (dy.double().abs().sum() / 24 * (2 / 16) ** 3) + 2 * U * (grad.double() * moved).abs().sum()
            assert (diff - along).abs() <= tol, (act, i, float(diff), float(along))


def test_what_is_kept_for_the_backward_pass_may_not_be_overwritten(cuda):
    import asrn_b200 as asrn
    x, r = rand((40, 64), 110).requires_grad_(), rand((40, 64), 111, dtype=F32).requires_grad_()
    w, ww = rand((64,), 112, dtype=F32).requires_grad_(), rand((64, 64), 113, 0.1)
    y, s = asrn.layer_norm(x, w, residual=r)
    s.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.float().sum().backward()
    c = x.detach() * 1
    y = asrn.linear(c, ww.requires_grad_(), activation='gelu')
    y.mul_(2)                                            # the result is not kept
    torch.autograd.grad(y.float().sum(), (ww,), retain_graph=True)
    c.zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.float().sum().backward()
    y, s = asrn.layer_norm(x, w, residual=r)
    first = torch.autograd.grad((y, s), (x, r, w), (torch.ones_like(y), torch.ones_like(s)), retain_graph=True)
    again = torch.autograd.grad((y, s), (x, r, w), (torch.ones_like(y), torch.ones_like(s)))
    assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_inference_mode_and_saved_tensor_hooks(cuda):
    import asrn_b200 as asrn
    x, r, w = rand((70, 64), 114), rand((70, 64), 115, dtype=F32), rand((64, 64), 116, 0.1)
    want = (*asrn.layer_norm(x, r[0], residual=r), asrn.linear(x, w, activation='silu', residual=r), *asrn.head_stats(x, w, top=3)[1:])
    with torch.inference_mode():
        got = (*asrn.layer_norm(x, r[0], residual=r), asrn.linear(x, w, activation='silu', residual=r), *asrn.head_stats(x, w, top=3)[1:])
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]

    def loss():
        y, s = asrn.layer_norm(leaves[0], leaves[1][0], residual=leaves[1])
        return asrn.head_stats(asrn.linear(y, leaves[2], activation='silu', residual=s).bfloat16(), leaves[2]).entropy.sum()
    want = [g.clone() for g in torch.autograd.grad(loss(), leaves)]
    with torch.autograd.graph.save_on_cpu():
        held = loss()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(held, leaves), want))


@pytest.mark.parametrize('N', [1, 40, 700])
def test_two_streams_at_once(cuda, N):
    import asrn_b200 as asrn
    t = [(rand((N, 768), 120 + i), rand((N, 768), 122 + i, dtype=F32), rand((1536, 768), 124 + i, 0.03), rand((5003, 768), 126 + i, 0.03))
         for i in range(2)]

    def chain(x, r, w, head):
        y, s = asrn.layer_norm(x, r[0], residual=r)
        a = asrn.linear(y, w, activation='gelu')
        b = asrn.linear(a, w.t().contiguous(), residual=s)
        return (b, *asrn.head_stats(b.bfloat16(), head, top=4)[1:])
    with torch.no_grad():
        want = [chain(*q) for q in t]
        streams = [torch.cuda.Stream() for _ in t]
        torch.cuda.synchronize()
        got = [None, None]
        for _ in range(20):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[i] = chain(*t[i])
        torch.cuda.synchronize()
    for g, q in zip(got, want):
        assert all(torch.equal(p, o) for p, o in zip(g, q))


def test_second_and_forward_mode_derivatives_are_refused(cuda):
    import asrn_b200 as asrn
    x, w = rand((20, 64), 70).requires_grad_(), rand((64, 64), 71, 0.1).requires_grad_()
    for f in (lambda: asrn.linear(x, w, None, 'gelu'), lambda: asrn.layer_norm(x, w[0]),
              lambda: asrn.head_stats(x, w).entropy):
        g, = torch.autograd.grad(f().float().square().sum(), (x,), create_graph=True)
        with pytest.raises(RuntimeError, match='second derivative'):
            g.float().square().sum().backward()
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), torch.no_grad():
        t = fw.make_dual(x.detach(), torch.ones_like(x))
        for f in (lambda: asrn.linear(t, w), lambda: asrn.layer_norm(t, w[0]), lambda: asrn.head_stats(t, w)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                f()


def test_refusals(cuda):
    import asrn_b200 as asrn
    x, w, b = rand((4, 64), 80), rand((32, 64), 81), rand((32,), 82)
    for error, call in [
            (ValueError, lambda: asrn.linear(x, w, b, 'tanh')), (ValueError, lambda: asrn.linear(x, w.t(), b)),
            (ValueError, lambda: asrn.linear(x, w, b[:8])), (ValueError, lambda: asrn.linear(x, w, b, residual=x)),
            (TypeError, lambda: asrn.linear(x, w, b, residual=rand((4, 32), 83, dtype=torch.float16))),
            (NotImplementedError, lambda: asrn.linear(x[:, :12].contiguous(), w[:, :12].contiguous())),
            (NotImplementedError, lambda: asrn.linear(x.half(), w.half())),
            (RuntimeError, lambda: asrn.linear(x, w.cpu())), (RuntimeError, lambda: asrn.linear(x, w, b, residual=b.cpu().expand(4, 32))),
            (ValueError, lambda: asrn.layer_norm(x, b)), (ValueError, lambda: asrn.layer_norm(x, w[0], b)),
            (ValueError, lambda: asrn.layer_norm(x, w[0], residual=x[:2])), (ValueError, lambda: asrn.layer_norm(x, w[0], eps=-1.0)),
            (TypeError, lambda: asrn.layer_norm(x.half(), w[0])), (TypeError, lambda: asrn.layer_norm(x, w[0], dtype=torch.float16)),
            (TypeError, lambda: asrn.layer_norm(x, w[0], w[1].float())), (TypeError, lambda: asrn.layer_norm(x, w[0], dtype=3)),
            (NotImplementedError, lambda: asrn.layer_norm(rand((1, 16392), 84), rand((16392,), 85))),
            (RuntimeError, lambda: asrn.layer_norm(x, w[0].cpu()))]:
        with pytest.raises(error):
            call()

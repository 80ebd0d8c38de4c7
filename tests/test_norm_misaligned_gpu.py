"""layer_norm's C entries on buffers that start between two 16-byte boundaries, which go value by value (the package hands its
kernels aligned copies), against the formulas in 64 bits; and the package on such views. Bounds, with U = 2^-8 and E = 2^-24 the unit
roundoffs of bf16 and fp32: a row's sums are chains of at most 32 additions a thread, 5 in a warp and 16 over warps, so the mean is off
by 64 E mean|s|, which moves (s - m) k by DH = 64 E mean|s| k, and 1 / sqrt(var) and the products after it by 64 E of themselves; columns'
sums are chains of at most rows / 128 + 64."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U, E = 2.0 ** -8, 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
EPS = 1e-5


def rand(shape, seed, scale=1.0, dtype=F32, shift=0.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale + shift).to(dtype).cuda()


def close(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(((got.double() - want).abs() / tol.clamp(min=1e-300)).max()))


class Room:
    """Buffers between guards, those named in `odd` one element off a 512-byte boundary."""
    def __init__(self, odd):
        self.odd, self.all = odd, []

    def __call__(self, name, shape, dtype, values=None):
        n = torch.empty(shape, dtype=dtype, device='meta')
        size, at = n.numel() * n.element_size(), 512 + (n.element_size() if name in self.odd else 0)
        raw = torch.full((size + 1024 + 16,), 0xA5, dtype=torch.uint8, device='cuda')
        self.all.append((raw, at, size))
        t = raw[at:at + size].view(dtype).view(shape)
        if values is not None:
            t.copy_(values)
        return t

    def check(self):
        for raw, at, size in self.all:
            assert (raw[:at] == 0xA5).all() and (raw[at + size:] == 0xA5).all()


def run(N, d, xt, rt, yt, wt, odd, seed=0):
    from asrn_b200 import _lib
    L, P, stream = _lib.lib(), _lib.ptr, _lib.stream_ptr(torch.device('cuda:0'))
    code = lambda t: 1 if t == BF16 else 0  # noqa: E731
    unit = lambda t: U if t == BF16 else E  # noqa: E731
    room = Room(odd)
    x = room('x', (N, d), xt, rand((N, d), seed + 1, shift=0.3))
    w, b = room('w', (d,), wt, rand((d,), seed + 2, 0.3, shift=1.0)), room('b', (d,), wt, rand((d,), seed + 3))
    r = None if rt is None else room('r', (N, d), rt, rand((N, d), seed + 4, 2.0))
    s = None if rt is None else room('s', (N, d), rt)
    y, stats = room('y', (N, d), yt), room('stats', (N, 2), F32)
    assert L.asrn_layer_norm(N, d, P(x), code(xt), P(r), code(rt), P(w), P(b), code(wt), EPS, P(s), P(y), code(yt), P(stats), stream) == 0
    read, st = (x, xt) if rt is None else (s, rt)
    if rt is not None:
        assert torch.equal(s, (x.float() + r.float()).to(rt))
    s64, w64 = read.double(), w.double()
    m, v = s64.mean(1, keepdim=True), s64.var(1, unbiased=False, keepdim=True)
    k = (v + EPS).rsqrt()
    h = (s64 - m) * k
    DH = 64 * E * s64.abs().mean(1, keepdim=True) * k + 64 * E * h.abs()
    ref = h * w64 + b.double()
    close(y, ref, DH * w64.abs() + 4 * E * (ref.abs() + (h * w64).abs()) + unit(yt) * ref.abs() + 1e-38, 'y')
    dy = room('dy', (N, d), yt, rand((N, d), seed + 5))
    ds = None if rt is None else room('ds', (N, d), st, rand((N, d), seed + 6))
    ot = BF16 if st == F32 else F32
    out, other = room('out', (N, d), st), room('other', (N, d), ot)
    dw, db = room('dw', (d,), wt), room('db', (d,), wt)
    nb = L.asrn_layer_norm_workspace_bytes(N, d)
    ws = room('ws', (nb,), torch.uint8)
    assert L.asrn_layer_norm_backward(N, d, P(read), code(st), P(stats), P(dy), code(yt), P(ds), P(w), code(wt), P(out), P(other), P(dw),
                                      P(db), P(ws), nb, stream) == 0
    dy64 = dy.double()
    g = dy64 * w64
    ga, ha = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    dx = k * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    tol = k * (128 * E * (g.abs() + ga + h.abs() * ha) + DH * ha + h.abs() * (g.abs() * DH).mean(1, keepdim=True))
    if ds is not None:
        dx = dx + ds.double()
        tol = tol + 4 * E * ds.double().abs()
    tol = tol + 4 * E * dx.abs()
    close(out, dx, tol + unit(st) * dx.abs() + 1e-38, 'out')
    close(other, dx, tol + unit(ot) * dx.abs() + 1e-38, 'other')
    depth = (N / 128 + 64) * E
    close(dw, (dy64 * h).sum(0), (dy64.abs() * DH).sum(0) + depth * (dy64 * h).abs().sum(0) + unit(wt) * (dy64 * h).sum(0).abs() + 1e-38, 'dw')
    close(db, dy64.sum(0), depth * dy64.abs().sum(0) + unit(wt) * dy64.sum(0).abs() + 1e-38, 'db')
    room.check()


ALL = ('x', 'r', 's', 'w', 'b', 'y', 'dy', 'ds', 'out', 'other', 'dw', 'db')


@pytest.mark.parametrize('N,d', [(1, 1), (9, 2), (3500, 5), (700, 96), (130, 255), (61, 256), (61, 257), (40, 700), (33, 1024), (33, 1025),
                                 (9, 3000), (310, 2056), (5, 8192), (5, 8200), (3, 16384), (300, 8201)])
@pytest.mark.parametrize('xt,rt,yt,wt', [(F32, None, F32, F32), (BF16, F32, BF16, F32), (BF16, BF16, F32, BF16), (F32, F32, BF16, F32)])
def test_sizes(cuda, N, d, xt, rt, yt, wt):
    run(N, d, xt, rt, yt, wt, ALL)


@pytest.mark.parametrize('odd', ALL)
@pytest.mark.parametrize('d', [77, 1032])
def test_one_buffer_at_a_time(cuda, odd, d):
    run(20, d, BF16, F32, BF16, F32, (odd,))
    run(20, d, F32, BF16, F32, BF16, (odd,))


def test_views_of_the_package(cuda):
    import asrn_b200 as asrn
    big, w, b = rand((70 * 768 + 64,), 7), rand((768,), 8), rand((768,), 9)
    for at in (0, 1, 2, 3, 4):
        v = big[at:at + 768 * 60].view(60, 768)
        assert v.is_contiguous()
        assert torch.equal(asrn.layer_norm(v, w, b), asrn.layer_norm(v.clone(), w, b))

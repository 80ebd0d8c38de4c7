"""The C entries of layer_norm, linear and head_stats: exactly the room that they ask for, nothing written around it or where
nothing is wanted, the package's results; and the status word's errors in the package's calls."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TIMEOUT = 5


def rand(shape, seed, scale=1.0, dtype=BF16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


class Room:
    """Buffers between guards."""
    def __init__(self):
        self.all = []

    def __call__(self, shape, dtype=torch.uint8):
        n = torch.empty(shape, dtype=dtype, device='meta')
        size = n.numel() * n.element_size()
        raw = torch.full((size + 1024,), 0xA5, dtype=torch.uint8, device='cuda')
        self.all.append((raw, size))
        return raw[512:512 + size].view(dtype).view(shape)

    def check(self):
        for raw, size in self.all:
            assert (raw[:512] == 0xA5).all() and (raw[512 + size:] == 0xA5).all()

    @staticmethod
    def untouched(t):
        return bool((t.contiguous().view(torch.uint8) == 0xA5).all())


def code(dtype):
    return 1 if dtype == BF16 else 0


@pytest.mark.parametrize('N,d', [(1, 8), (3, 5), (33, 64), (700, 333), (50, 768), (9, 2050), (5, 6000)])
@pytest.mark.parametrize('x,res', [(BF16, F32), (F32, None), (BF16, BF16)])
def test_layer_norm(cuda, N, d, x, res):
    import asrn_b200 as asrn
    from asrn_b200 import _lib
    L, P, s = _lib.lib(), _lib.ptr, _lib.stream_ptr(cuda)
    a, w, b, dy = rand((N, d), 1, dtype=x), rand((d,), 2, dtype=F32), rand((d,), 3, dtype=F32), rand((N, d), 4, dtype=x)
    r = None if res is None else rand((N, d), 5, dtype=res)
    leaves = [t.requires_grad_() for t in (a, w, b) + (() if r is None else (r,))]
    out = asrn.layer_norm(a, w, b, residual=r)
    y_want = (out if r is None else out[0]).detach()
    want = torch.autograd.grad(out if r is None else out[0], leaves, dy)
    room = Room()
    y, stats, total = room((N, d), x), room((N, 2), F32), None if r is None else room((N, d), res)
    norm = lambda st: L.asrn_layer_norm(N, d, P(a), code(x), P(r), code(res), P(w), P(b), 0, 1e-5, P(total), P(y), code(x), P(st), s)  # noqa: E731,E501
    assert norm(None) == 0 and torch.equal(y, y_want)
    y.zero_()
    assert norm(stats) == 0 and torch.equal(y, y_want)
    read = a if r is None else total
    of, other = (read.dtype, x) if r is not None else (x, BF16 if x == F32 else F32)
    nb = L.asrn_layer_norm_workspace_bytes(N, d)
    back = lambda o, q, dw, db, ws: L.asrn_layer_norm_backward(  # noqa: E731
        N, d, P(read), code(of), P(stats), P(dy), code(x), None, P(w), 0, P(o), P(q), P(dw), P(db), P(ws), 0 if ws is None else nb, s)
    o, dw, db, ws = room((N, d), of), room((d,), F32), room((d,), F32), room((nb,))
    assert back(o, None, dw, db, ws) == 0
    assert torch.equal(o, want[3] if r is not None else want[0]) and torch.equal(dw, want[1]) and torch.equal(db, want[2])
    dw.fill_(0), ws.fill_(0xA5), o.fill_(0)
    assert back(None, None, dw, None, ws) == 0 and torch.equal(dw, want[1])
    assert back(o, None, None, None, None) == 0 and torch.equal(o, want[3] if r is not None else want[0])
    if other != of:
        q = room((N, d), other)
        assert back(None, q, None, None, None) == 0
        assert r is None or torch.equal(q, want[0])
    assert back(None, None, None, None, None) == 0
    assert back(None, None, dw, None, None) != 0                  # no workspace
    room.check()


@pytest.mark.parametrize('N,d,n', [(1, 8, 8), (7, 64, 40), (64, 200, 24), (65, 72, 520), (513, 64, 128), (1500, 136, 264)])
@pytest.mark.parametrize('act,res', [(0, None), (1, F32), (2, BF16), (0, F32)])
def test_linear(cuda, N, d, n, act, res):
    import asrn_b200 as asrn
    from asrn_b200 import _lib
    L, P, s = _lib.lib(), _lib.ptr, _lib.stream_ptr(cuda)
    x, w, b = rand((N, d), 10), rand((n, d), 11, 0.2), rand((n,), 12)
    r = None if res is None else rand((N, n), 13, dtype=res)
    of = res or BF16
    dy = rand((N, n), 14, dtype=of)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    kept = asrn.linear(*leaves, activation=(None, 'gelu', 'silu')[act], residual=r)
    y_want = kept.detach()
    want = torch.autograd.grad(kept, leaves, dy)
    room, word = Room(), torch.zeros(1, dtype=torch.int32, device='cuda')
    y, slope = room((N, n), of), room((N, n), torch.float16)
    forward = lambda sl: L.asrn_linear_forward(N, d, n, P(x), P(w), P(b), act, P(r), code(of), P(y), P(sl), P(word), s)  # noqa: E731
    assert forward(None) == 0 and torch.equal(y, y_want)
    y.zero_()
    assert forward(slope) == 0 and torch.equal(y, y_want) and (act or Room.untouched(slope))
    nb = L.asrn_linear_workspace_bytes(N, d, n, act, code(of))
    dx, dw, db, ws = room((N, d), BF16), room((n, d), BF16), room((n,), BF16), room((nb,))
    back = lambda a, c, e: L.asrn_linear_backward(N, d, n, P(dy), code(of), P(x), P(w), act, P(slope) if act else None, P(a), P(c), P(e),  # noqa: E731,E501
                                                  P(ws), nb, P(word), s)
    assert back(dx, dw, db) == 0 and all(torch.equal(p, q) for p, q in zip((dx, dw, db), want))
    for i in range(3):
        one = [torch.zeros_like(t) if k == i else None for k, t in enumerate((dx, dw, db))]
        ws.fill_(0xA5)
        assert back(*one) == 0 and torch.equal(one[i], want[i])
    assert back(None, None, None) == 0 and int(word) == 0
    room.check()


@pytest.mark.parametrize('N,V,d', [(1, 40, 8), (8, 5003, 72), (30, 300, 64), (33, 300, 64), (300, 2100, 136), (600, 33001, 64)])
@pytest.mark.parametrize('top', [0, 4, 32])
def test_head_stats(cuda, N, V, d, top):
    import asrn_b200 as asrn
    from asrn_b200 import _lib
    L, P, s = _lib.lib(), _lib.ptr, _lib.stream_ptr(cuda)
    h, w = rand((N, d), 20).requires_grad_(), rand((V, d), 21, 0.2).requires_grad_()
    y = torch.randint(0, V, (N,), generator=torch.Generator().manual_seed(22)).cuda()
    y[1::3] = -1
    g, gh = rand((N,), 23, dtype=F32), rand((N,), 24, dtype=F32)
    room, word = Room(), torch.zeros(1, dtype=torch.int32, device='cuda')
    ns, nf, nb = (L.asrn_head_stats_saved_bytes(N, d), L.asrn_head_stats_workspace_bytes(N, V, d, top, 0),
                  L.asrn_head_stats_workspace_bytes(N, V, d, 0, 1))
    for tok in (y, None):
        r = asrn.head_stats(h, w, tok, temperatura=0.9, top=top)
        up = (r.entropy,) if tok is None else (r.entropy, r.logp)
        dh_want, dw_want = torch.autograd.grad(up, (h, w), (gh, g)[:len(up)])
        lp, en, tl, tt = room((N,), F32), room((N,), F32), room((N, max(top, 1)), F32), room((N, max(top, 1)), torch.int64)
        saved, wf, wb = room((ns,)), room((nf,)), room((nb,))
        forward = lambda sv: L.asrn_head_stats_forward(N, V, d, P(h), P(w), P(tok), 0.9, top, P(lp), P(en), P(tl), P(tt), P(sv),  # noqa: E731,E501
                                                       0 if sv is None else ns, P(wf), nf, P(word), s)
        for sv in (saved,) if tok is not None else (None, saved):
            en.fill_(7)
            assert forward(sv) == 0 and torch.equal(en, r.entropy)
            assert torch.equal(lp, r.logp) if tok is not None else Room.untouched(lp)
            if top:
                assert torch.equal(tl, r.top_logp) and torch.equal(tt, r.top_tokens)
            else:
                assert Room.untouched(tl) and Room.untouched(tt)
        dh, dw = room((N, d), BF16), room((V, d), BF16)
        back = lambda a, c: L.asrn_head_stats_backward(N, V, d, P(w), P(saved), ns, 0.9, P(g) if tok is not None else None, P(gh), P(a), P(c),  # noqa: E731,E501
                                                       P(wb), nb, P(word), s)
        assert back(dh, dw) == 0 and torch.equal(dh, dh_want) and torch.equal(dw, dw_want)
        dh.zero_(), dw.zero_()
        assert back(dh, None) == 0 and torch.equal(dh, dh_want)
        assert back(None, dw) == 0 and torch.equal(dw, dw_want)
    assert int(word) == 0
    room.check()


def test_a_recorded_timeout_is_raised_until_it_is_cleared(cuda):
    """The word is written here as a kernel whose wait gives up writes it. layer_norm waits for nothing and goes on."""
    import asrn_b200 as asrn
    from asrn_b200 import _lib
    from asrn_b200 import finetune as ft
    x, w = rand((40, 64), 30), rand((96, 64), 31, 0.1).requires_grad_()
    calls = [lambda: asrn.linear(x, w, activation='gelu'), lambda: asrn.head_stats(x, w, top=2).entropy]
    outs = [f() for f in calls]
    want = [torch.autograd.grad(o.float().sum(), w, retain_graph=True)[0] for o in outs]
    assert ft.status() == 0
    word = ctypes.c_int.from_address(_lib.finetune().status_address(0))
    word.value = TIMEOUT
    try:
        for f in calls + [lambda o=o: torch.autograd.grad(o.float().sum(), w, retain_graph=True) for o in outs]:
            with pytest.raises(RuntimeError, match='bounded wait'):
                f()
        asrn.layer_norm(x, w[0])
        assert ft.status(reset=True) == TIMEOUT
    finally:
        word.value = 0
    assert all(torch.equal(f(), o) for f, o in zip(calls, outs))
    assert all(torch.equal(torch.autograd.grad(o.float().sum(), w)[0], a) for o, a in zip(outs, want))

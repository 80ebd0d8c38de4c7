"""Host-side checks of layer_norm, linear and head_stats that need no GPU: what the C entry points refuse and how much room they
ask for, the package's errors, and that there is no CPU path."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p
ARG, UNSUPPORTED, WORKSPACE = 1, 2, 3


@pytest.fixture(scope='module')
def lib():
    from asrn_b200 import _lib
    return _lib.lib()


@pytest.fixture(scope='module')
def at():
    buf = ctypes.create_string_buffer(8192)
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    return lambda off=0, keep=buf: P(base + off)


def test_norm_refusals(lib, at):
    ok, odd = at(), at(1)
    f = lambda N=4, d=16, x=ok, xt=0, r=None, rt=0, w=ok, b=ok, wt=0, eps=1e-5, s=None, y=ok, yt=0, st=None: lib.asrn_layer_norm(  # noqa: E731,E501
        N, d, x, xt, r, rt, w, b, wt, eps, s, y, yt, st, None)
    assert f(N=-1) == ARG and f(d=0) == ARG and f(d=16385) == UNSUPPORTED and f(N=1 << 31) == UNSUPPORTED
    assert f(xt=2) == ARG and f(wt=-1) == ARG and f(yt=3) == ARG and f(r=ok, s=ok, rt=2) == ARG
    assert f(x=None) == ARG and f(w=None) == ARG and f(y=None) == ARG and f(r=ok) == ARG
    assert f(x=odd) == ARG and f(x=at(2)) == ARG and f(b=odd) == ARG and f(y=odd) == ARG and f(st=at(4)) == ARG
    assert f(r=at(2), s=ok) == ARG and f(r=ok, s=at(2)) == ARG
    assert f(eps=-1.0) == ARG and f(eps=float('nan')) == ARG and f(N=0, x=None) == 0
    g = lambda N=4, d=16, s=ok, st=0, stats=ok, dy=ok, yt=0, ds=None, w=ok, wt=0, out=ok, other=None, dw=ok, db=None, ws=ok, nb=1 << 30: lib.asrn_layer_norm_backward(  # noqa: E731,E501
        N, d, s, st, stats, dy, yt, ds, w, wt, out, other, dw, db, ws, nb, None)
    assert g(N=-1) == ARG and g(d=16385) == UNSUPPORTED and g(st=2) == ARG and g(yt=2) == ARG and g(wt=2) == ARG
    assert g(s=None) == ARG and g(stats=None) == ARG and g(dy=None) == ARG and g(w=None) == ARG
    assert g(out=odd) == ARG and g(other=odd) == ARG and g(dw=odd) == ARG and g(ds=odd) == ARG
    assert g(ws=None) == WORKSPACE and g(nb=64) == WORKSPACE and g(ws=at(8)) == WORKSPACE
    assert g(out=None, dw=None) == 0                      # nothing wanted
    assert lib.asrn_layer_norm_workspace_bytes(0, 16) == 0 and lib.asrn_layer_norm_workspace_bytes(4, 1 << 15) == 0
    assert lib.asrn_layer_norm_workspace_bytes(1, 768) == 2 * 768 * 4
    assert lib.asrn_layer_norm_workspace_bytes(1 << 20, 768) < 16 << 20


def test_linear_refusals(lib, at):
    ok, odd = at(), at(2)
    f = lambda N=4, d=16, n=32, x=ok, w=ok, b=ok, act=1, r=None, rt=0, y=ok, sl=None: lib.asrn_linear_forward(  # noqa: E731
        N, d, n, x, w, b, act, r, rt, y, sl, None, None)
    assert f(N=-1) == ARG and f(d=0) == ARG and f(n=0) == ARG and f(d=12) == UNSUPPORTED and f(n=36) == UNSUPPORTED
    assert f(d=1 << 17) == UNSUPPORTED and f(N=1 << 27) == UNSUPPORTED and f(n=1 << 21) == UNSUPPORTED
    assert f(act=4) == ARG and f(act=-1) == ARG and f(r=ok, rt=2) == ARG
    assert f(x=None) == ARG and f(w=None) == ARG and f(y=None) == ARG
    assert f(x=odd) == ARG and f(w=odd) == ARG and f(b=odd) == ARG and f(y=odd) == ARG and f(r=odd) == ARG and f(sl=odd) == ARG
    assert f(N=0, x=None) == 0
    g = lambda N=4, d=16, n=32, dy=ok, yt=1, x=ok, w=ok, act=1, sl=ok, dx=ok, dw=ok, db=ok, ws=ok, nb=1 << 40: lib.asrn_linear_backward(  # noqa: E731,E501
        N, d, n, dy, yt, x, w, act, sl, dx, dw, db, ws, nb, None, None)
    assert g(N=-1) == ARG and g(d=20) == UNSUPPORTED and g(yt=2) == ARG and g(act=5) == ARG
    assert g(dy=None) == ARG and g(x=None) == ARG and g(w=None) == ARG and g(sl=None) == ARG
    assert g(dy=odd) == ARG and g(dx=odd) == ARG and g(dw=odd) == ARG and g(db=at(1)) == ARG
    assert g(ws=None) == WORKSPACE and g(nb=8) == WORKSPACE and g(ws=odd) == WORKSPACE
    size = lib.asrn_linear_workspace_bytes
    assert size(0, 768, 1536, 1, 1) == 0 and size(4, 12, 16, 0, 1) == 0
    assert size(32768, 768, 1536, 1, 1) >= 32768 * 1536 * 2       # dA
    assert size(32768, 768, 1536, 0, 1) < 32768 * 1536 * 2        # dA is dY
    assert size(100, 768, 1536, 0, 0) >= 2 * 128 * 1536 * 2       # dA and its remainder


def test_stats_refusals(lib, at):
    ok, odd = at(), at(2)
    f = lambda N=4, V=9, d=16, h=ok, w=ok, tok=ok, tau=1.0, top=2, lp=ok, en=ok, tl=ok, tt=ok, sv=ok, ns=1 << 40, ws=ok, nw=1 << 40: lib.asrn_head_stats_forward(  # noqa: E731,E501
        N, V, d, h, w, tok, tau, top, lp, en, tl, tt, sv, ns, ws, nw, None, None)
    assert f(N=-1) == ARG and f(V=0) == ARG and f(d=12) == UNSUPPORTED and f(V=1 << 25) == UNSUPPORTED
    assert f(tau=0.0) == ARG and f(tau=float('nan')) == ARG and f(top=-1) == ARG and f(top=10) == ARG
    assert f(V=99, top=33) == UNSUPPORTED and f(h=None) == ARG and f(w=odd) == ARG and f(en=None) == ARG
    assert f(lp=None) == ARG and f(tl=None) == ARG and f(tt=None) == ARG
    assert f(sv=None) == WORKSPACE and f(tok=None, sv=None, nw=8) == WORKSPACE and f(ns=8) == WORKSPACE and f(nw=8) == WORKSPACE and f(ws=odd) == WORKSPACE
    assert f(N=0) == 0
    g = lambda N=4, w=ok, tau=1.0, sv=ok, ns=1 << 40, dh=ok, ws=ok, nw=1 << 40: lib.asrn_head_stats_backward(  # noqa: E731
        N, 9, 16, w, sv, ns, tau, None, None, dh, ok, ws, nw, None, None)
    assert g(w=None) == ARG and g(tau=-1.0) == ARG and g(dh=odd) == ARG and g(sv=None) == WORKSPACE and g(nw=8) == WORKSPACE
    room = lib.asrn_head_stats_workspace_bytes
    assert room(1000, 50304, 768, 5, 0) > room(1000, 50304, 768, 0, 0) > 1000 * 50304 // 128 * 12
    assert room(1000, 50304, 768, 0, 1) == lib.asrn_head_workspace_bytes(1000, 50304, 768, 1)
    assert lib.asrn_head_stats_saved_bytes(1000, 768) > lib.asrn_head_saved_bytes(1000, 768)
    assert lib.asrn_head_stats_saved_bytes(1000, 100) == 0


def test_the_packages_errors_and_no_cpu_path():
    import asrn_b200 as asrn
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    i = torch.zeros(3, dtype=torch.int64)
    for error, call in [
            (RuntimeError, lambda: asrn.layer_norm(b(3, 8), b(8))), (RuntimeError, lambda: asrn.linear(b(3, 8), b(16, 8))),
            (RuntimeError, lambda: asrn.head_stats(b(3, 8), b(5, 8), i)),
            (ValueError, lambda: asrn.layer_norm(b(3, 8), b(9))), (ValueError, lambda: asrn.layer_norm(b(3, 8), b(8), b(4))),
            (ValueError, lambda: asrn.layer_norm(b(3, 8), b(8), residual=b(3, 9))),
            (ValueError, lambda: asrn.layer_norm(b(3, 8), b(8), eps=float('nan'))),
            (TypeError, lambda: asrn.layer_norm(b(3, 8).double(), b(8))), (TypeError, lambda: asrn.layer_norm(b(3, 8), b(8), dtype='f')),
            (ValueError, lambda: asrn.linear(b(3, 8), b(16, 9))), (ValueError, lambda: asrn.linear(b(3, 8), b(16, 8), b(8))),
            (ValueError, lambda: asrn.linear(b(3, 8), b(16, 8), activation='GELU')),
            (ValueError, lambda: asrn.linear(b(3, 8), b(16, 8), residual=b(3, 8))),
            (ValueError, lambda: asrn.linear(b(3, 8), b(16, 8), residual=b(1, 16))),
            (TypeError, lambda: asrn.linear(b(3, 8), b(16, 8), residual=torch.zeros(3, 16, dtype=torch.int64))),
            (ValueError, lambda: asrn.head_stats(b(3, 8), b(5, 16))), (ValueError, lambda: asrn.head_stats(b(3, 8), b(5, 8), i[:2])),
            (TypeError, lambda: asrn.head_stats(b(3, 8), b(5, 8), i.int())), (ValueError, lambda: asrn.head_stats(b(3, 8), b(5, 8), top=6)),
            (ValueError, lambda: asrn.head_stats(b(3, 8), b(5, 8), temperatura=-1.0))]:
        with pytest.raises(error):
            call()


def test_the_models_option():
    import asrn_b200 as asrn
    m = asrn.create_model(V=32, d=16, n_capas=2, fundido=True)
    assert m.fundido and all(b.fundido for b in m.bloques) and 'fundido' not in m.config
    n = asrn.create_model(V=32, d=16, n_capas=2)
    assert not n.fundido and not any(b.fundido for b in n.bloques)
    del m.bloques[0].__dict__['fundido'], m.__dict__['fundido']      # as blocks and models pickled before the option was there
    assert m.bloques[0].fundido is False and m.fundido is False

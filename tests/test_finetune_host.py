"""Host-side checks of the fine-tuning operators that need no GPU: what the C entry points refuse and how much room they
ask for, and that there is no CPU path."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p
ARG, UNSUPPORTED, WORKSPACE = 1, 2, 3


@pytest.fixture(scope='module')
def lib():
    from asrn_b200 import _lib
    return _lib.lib()


def test_sizes(lib):
    assert lib.asrn_head_saved_bytes(1000, 768) >= 1024 * 768 * 2 + 5 * 4 * 1000
    assert lib.asrn_head_saved_bytes(1000, 100) == 0 and lib.asrn_head_saved_bytes(-1, 64) == 0
    # dS of a chunk of rows at most: two gigabytes, whatever the number of rows
    big = lib.asrn_head_workspace_bytes(1 << 20, 50304, 768, 1)
    assert 1 << 31 <= big + (1 << 28) and big < 3 << 30
    assert lib.asrn_head_workspace_bytes(48, 256, 64, 1) < 1 << 20
    assert lib.asrn_mlp8_saved_bytes(4096, 768, 1536) <= 4096 * (768 + 1536) * 33 // 32 + 1024
    assert lib.asrn_mlp8_saved_bytes(4096, 768, 1532) == 0
    assert lib.asrn_preference_workspace_bytes(4, 256) == 0 and lib.asrn_preference_workspace_bytes(512, 4096) > 0
    assert lib.asrn_policy_workspace_bytes(-1, 5) == 0


def test_refusals(lib):
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    ok, odd = P(at), P(at + 2)
    head = lambda N=4, V=9, d=16, h=ok, w=ok, tau=1.0, saved=ok, nb=1 << 40, ws=ok, nw=1 << 40: lib.asrn_head_forward(  # noqa: E731,E501
        N, V, d, h, w, ok, tau, ok, saved, nb, ws, nw, None, None)
    assert head(N=-1) == ARG and head(V=0) == ARG and head(tau=0.0) == ARG and head(tau=float('nan')) == ARG
    assert head(h=None) == ARG and head(h=odd) == ARG and head(w=odd) == ARG
    assert head(d=12) == UNSUPPORTED and head(V=1 << 25) == UNSUPPORTED and head(N=1 << 25) == UNSUPPORTED
    assert head(N=1 << 24, V=1 << 24) == UNSUPPORTED
    assert head(saved=None) == WORKSPACE and head(nb=16) == WORKSPACE and head(nw=16) == WORKSPACE
    assert head(saved=odd) == WORKSPACE and head(N=0) == 0
    back = lambda d=16, g=ok, tau=1.0, nb=1 << 40, nw=1 << 40: lib.asrn_head_backward(  # noqa: E731
        4, 9, d, ok, ok, nb, tau, g, ok, ok, ok, nw, None, None)
    assert back(d=4) == UNSUPPORTED and back(g=None) == ARG and back(tau=-1.0) == ARG
    assert back(nb=0) == WORKSPACE and back(nw=0) == WORKSPACE
    pref = lambda Pn=600, L=600, kind=0, beta=0.1, eps=0.0, lp=ok, loss=ok, ws=ok, nw=1 << 40: lib.asrn_preference_loss(  # noqa: E731,E501
        Pn, L, lp, ok, ok, kind, beta, eps, loss, None, ok, ws, nw, None)
    assert pref(Pn=-1) == ARG and pref(kind=2) == ARG and pref(beta=0.0) == ARG and pref(eps=0.5) == ARG
    assert pref(beta=float('nan')) == ARG and pref(lp=None) == ARG and pref(loss=None) == ARG
    assert pref(ws=None) == WORKSPACE and pref(nw=8) == WORKSPACE and pref(L=1 << 40) == UNSUPPORTED
    pol = lambda B=600, L=600, lo=0.2, hi=0.2, kl=0.0, ref=None, adv=ok, nw=1 << 40: lib.asrn_policy_loss(  # noqa: E731
        B, L, ok, ok, ref, adv, 0, ok, lo, hi, kl, 0, ok, None, ok, ok, nw, None)
    assert pol(B=-1) == ARG and pol(lo=1.0) == ARG and pol(hi=-0.1) == ARG and pol(kl=0.1) == ARG and pol(kl=-1.0) == ARG
    assert pol(adv=None) == ARG and pol(nw=8) == WORKSPACE
    mlp = lambda N=4, d=16, ff=32, do=16, x=ok, nw=1 << 40, sv=None, ns=0, b=ok: lib.asrn_mlp8_forward(  # noqa: E731
        N, d, ff, do, x, ok, b, ok, ok, ok, sv, ns, ok, nw, None, None)
    assert mlp(N=-1) == ARG and mlp(ff=0) == ARG and mlp(d=12) == UNSUPPORTED and mlp(do=4) == UNSUPPORTED
    assert mlp(b=odd) == ARG and mlp(x=odd) == ARG and mlp(x=None) == ARG and mlp(nw=0) == WORKSPACE and mlp(sv=ok, ns=8) == WORKSPACE
    assert mlp(N=0) == 0
    assert lib.asrn_mlp8_backward(4, 16, 32, 16, ok, ok, ok, None, 0, *[ok] * 6, 1 << 40, None, None) == WORKSPACE
    assert lib.asrn_mlp8_backward(4, 16, 32, 16, odd, ok, ok, ok, 1 << 40, *[ok] * 6, 1 << 40, None, None) == ARG
    assert lib.asrn_pack8(2, 12, ok, ok, ok, None) == UNSUPPORTED and lib.asrn_pack8(-1, 8, ok, ok, ok, None) == ARG
    assert lib.asrn_pack8(2, 8, odd, ok, ok, None) == ARG and lib.asrn_unpack8(2, 8, ok, None, ok, None) == ARG
    assert lib.asrn_pack8(0, 8, None, None, None, None) == 0


def test_no_cpu_path():
    import asrn_b200 as asrn
    h, w = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='CUDA'):
        asrn.head_logprobs(h, w, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match='CUDA'):
        asrn.mlp8(h, w[:, :8].repeat(2, 1)[:8], w[0], w[0].expand(8, 8).contiguous(), w[0])
    z = torch.zeros(2, 3, 4)
    with pytest.raises(RuntimeError, match='CUDA'):
        asrn.preference_loss(z, z, z.bool())
    m = asrn.create_model(V=32, d=16, n_capas=2, checkpoint='8bits')
    assert all(b.activaciones_8bits for b in m.bloques)
    assert not any(b.activaciones_8bits for b in asrn.create_model(V=32, d=16, n_capas=2, checkpoint=True).bloques)


def test_errors_are_the_packages_own():
    import asrn_b200 as asrn
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    z, i = torch.zeros(2, 3, 4), torch.zeros(3, dtype=torch.int64)
    for error, call in [
            (ValueError, lambda: asrn.head_logprobs(b(3, 8), b(5, 16), i)),
            (TypeError, lambda: asrn.head_logprobs(b(3, 8), b(5, 8), i.int())),
            (ValueError, lambda: asrn.head_logprobs(b(3, 8), b(5, 8), i, temperatura=0.0)),
            (ValueError, lambda: asrn.head_logprobs(b(3, 8), b(5, 8), i, temperatura=float('nan'))),
            (ValueError, lambda: asrn.preference_loss(z, z, z.bool(), kind='hinge')),
            (ValueError, lambda: asrn.preference_loss(z, z, z.bool(), beta=0.0)),
            (ValueError, lambda: asrn.preference_loss(z, z[:, :2], z.bool())),
            (ValueError, lambda: asrn.policy_loss(z[0], z[0], z[0, :2], z[0].bool())),
            (ValueError, lambda: asrn.policy_loss(z[0], z[0], z[0], z[0].bool(), kl=0.1)),
            (ValueError, lambda: asrn.policy_loss(z[0], z[0], z[0], z[0].bool(), clip=(1.0, 0.2))),
            (ValueError, lambda: asrn.mlp8(b(3, 8), b(8, 16), b(8), b(8, 8), b(8))),
            (TypeError, lambda: asrn.finetune.pack8(torch.zeros(3, 8)))]:
        with pytest.raises(error):
            call()

"""Fine-tuning on the device: log probabilities through the tied head, losses on them, and an MLP whose activations are
kept in 8 bits (the C ABI's asrn_head_*, asrn_preference_loss, asrn_policy_loss, asrn_mlp8_*, asrn_pack8).

    head_logprobs    log softmax(h W^T / temperatura)[token] and its gradients, without the (tokens, V) logits in memory
    preference_loss  logistic or squared (IPO) loss of pairs of a chosen and a rejected answer
    policy_loss      clipped policy loss with an advantage per answer or token and a KL term against a reference model
    mlp8             gelu(x W1^T + b1) W2^T + b2 that keeps x and x W1^T + b1 in 8 bits for its backward pass
    pack8, unpack8   the 8-bit form by itself

The losses return their gradient with the loss (one pass over the tokens makes both), so a step is

    logp = model.logprobs(x, targets)
    r = preference_loss(logp.detach(), ref_logp, mask)
    logp.backward(r.grad)

and r.loss.backward() works as well when logp requires a gradient. Everything runs on CUDA tensors, on the current
stream, and repeats bit for bit; there is no counterpart in the reference.
"""
from collections import namedtuple
from functools import lru_cache

import torch

from . import _lib

_status = {}


def _p(t):
    return None if t is None else t.data_ptr()


def _status_word(dev):
    """The device's status word of these kernels' bounded waits (none while a graph that would own it is captured)."""
    w = _status.get(dev)
    if w is None:
        if torch.cuda.is_current_stream_capturing():
            return None
        w = _status[dev] = torch.zeros(1, dtype=torch.int32, device=dev)
    return w.data_ptr()


def status(device=None, reset=False):
    """0, or the first error these kernels recorded on the device (ASRN_ERR_TIMEOUT: a bounded wait gave up and that
    call's results are void). Synchronises."""
    dev = torch.device('cuda', torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.index is None:
        dev = torch.device('cuda', torch.cuda.current_device())
    w = _status.get(dev)
    if w is None:
        return 0
    v = int(w.item())
    if reset:
        w.zero_()
    return v


def _stream(dev):
    """The current stream's handle on dev, an int (a call that takes about 10 us in all feels a Stream object's 2)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _need_cuda(what, first, *ts):
    """The tensors' device; they all have to be on the same GPU."""
    at = first.get_device()
    for t in ts:
        if t is not None and t.get_device() != at:
            raise (ValueError if at >= 0 and t.is_cuda else RuntimeError)(
                f'asrn_b200.{what} runs on CUDA tensors of one device; got {first.device} and {t.device}')
    if at < 0:
        raise RuntimeError(f'asrn_b200.{what} runs on CUDA tensors only (there is no CPU implementation)')
    return first.device


def _rows(t):
    """Contiguous and 16-byte aligned (a view into a larger buffer may be neither); read through its address only."""
    if not t.is_contiguous():
        t = t.detach().contiguous()
    return t if t.data_ptr() % 16 == 0 else t.detach().clone()


@lru_cache(1024)
def _bytes(name, *sizes):
    """A size query of the library (a pure function of the sizes)."""
    return getattr(_lib.lib(), name)(*sizes)


def _scratch(nbytes, dev):
    return torch.empty(nbytes or 256, dtype=torch.uint8, device=dev)


# ---- head -------------------------------------------------------------------------------------------------------------

class _HeadLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, tokens, tau):
        V, d = w.shape
        N, dev, lib = tokens.numel(), h.device, _lib.lib()
        hr, wr, tok = _rows(h), _rows(w), tokens.contiguous()
        out = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        nb_saved, nb = _bytes('asrn_head_saved_bytes', N, d), _bytes('asrn_head_workspace_bytes', N, V, d, 0)
        saved, ws = _scratch(nb_saved, dev), _scratch(nb, dev)
        _lib.check(lib.asrn_head_forward(N, V, d, hr.data_ptr(), wr.data_ptr(), tok.data_ptr(), tau, out.data_ptr(),
                                         saved.data_ptr(), nb_saved, ws.data_ptr(), nb, _status_word(dev),
                                         _stream(dev)), 'asrn_head_forward')
        ctx.save_for_backward(wr, saved)
        ctx.meta = (h.shape, N, V, d, tau, dev, nb_saved)
        return out

    @staticmethod
    def backward(ctx, g):
        w, saved = ctx.saved_tensors
        shape, N, V, d, tau, dev, nb_saved = ctx.meta
        lib = _lib.lib()
        need = ctx.needs_input_grad
        dh = w.new_empty(shape) if need[0] else None
        dw = torch.empty_like(w) if need[1] else None
        g32 = _f32(g)
        nb = _bytes('asrn_head_workspace_bytes', N, V, d, 1)
        ws = _scratch(nb, dev)
        _lib.check(lib.asrn_head_backward(N, V, d, w.data_ptr(), saved.data_ptr(), nb_saved, tau, g32.data_ptr(),
                                          _p(dh), _p(dw), ws.data_ptr(), nb, _status_word(dev), _stream(dev)),
                   'asrn_head_backward')
        return dh, dw, None, None


def _autocast_bf16():
    return torch.is_autocast_enabled('cuda') and torch.get_autocast_dtype('cuda') == torch.bfloat16


def _bf16(what, *ts):
    """The operands in bf16: as they are, or cast as autocast casts a linear layer's operands."""
    for t in ts:
        if t.dtype is not torch.bfloat16:
            break
    else:
        return ts
    if not _autocast_bf16():
        raise NotImplementedError(f'{what} computes in bfloat16: pass bfloat16 tensors or call it under '
                                  "torch.autocast('cuda', dtype=torch.bfloat16)")
    if any(t.dtype not in (torch.bfloat16, torch.float32) for t in ts):
        raise TypeError(f'{what} takes float32 or bfloat16 tensors')
    return tuple(t.to(torch.bfloat16) for t in ts)


def head_logprobs(h, weight, tokens, temperatura=1.0):
    """log softmax(h weight^T / temperatura) at tokens: h (..., d), weight (V, d) bfloat16 (or float32 under bf16
    autocast), tokens (...) int64 -> float32 (...), differentiable in h and weight. A negative token leaves its
    position out (0, no gradient, none of the work); a token >= V gives NaN. d has to be a multiple of 8."""
    sh, sw = h.shape, weight.shape
    if not sh or len(sw) != 2 or sh[-1] != sw[1] or tokens.shape != sh[:-1]:
        raise ValueError(f'head_logprobs: h (..., d), weight (V, d) and tokens (...) do not fit: {tuple(h.shape)}, '
                         f'{tuple(weight.shape)}, {tuple(tokens.shape)}')
    if tokens.dtype is not torch.int64:
        raise TypeError('head_logprobs: tokens are int64')
    if not 0 < temperatura <= 1e30:
        raise ValueError('head_logprobs: temperatura has to be positive')
    _need_cuda('head_logprobs', h, weight, tokens)
    h, weight = _bf16('head_logprobs', h, weight)
    if sh[-1] % 8:
        raise NotImplementedError(f'head_logprobs: the width ({sh[-1]}) has to be a multiple of 8')
    return _HeadLogprobs.apply(h, weight, tokens, float(temperatura))


# ---- losses -----------------------------------------------------------------------------------------------------------

class _WithGrad(torch.autograd.Function):
    """A loss whose gradient is known: backward scales it."""

    @staticmethod
    def forward(ctx, logp, loss, grad):
        ctx.save_for_backward(grad)
        ctx.dtype = logp.dtype
        return loss.clone()

    @staticmethod
    def backward(ctx, g):
        grad, = ctx.saved_tensors
        return (grad * g).to(ctx.dtype), None, None


def _f32(t):
    """float32 and contiguous; read through its address only."""
    if t.dtype is torch.float32 and t.is_contiguous():
        return t
    return t.detach().to(torch.float32).contiguous()


def _mask(m, shape, what):
    if m.shape != shape or (m.dtype is not torch.bool and m.dtype is not torch.uint8):
        raise ValueError(f'{what}: mask has to be bool or uint8 of shape {tuple(shape)}; got {m.dtype} {tuple(m.shape)}')
    return m if m.is_contiguous() else m.contiguous()


PreferenceLoss = namedtuple('PreferenceLoss', 'loss grad chosen rejected')
PolicyLoss = namedtuple('PolicyLoss', 'loss grad kl clipped')

_KINDS = {'sigmoid': 0, 'ipo': 1}
_PER = {'token': 0, 'sequence': 1}


def preference_loss(logp, ref_logp, mask, beta=0.1, smoothing=0.0, kind='sigmoid'):
    """Loss of P pairs of answers, logp and ref_logp (2, P, L) per-token log probabilities under the model and the
    reference model ([0] the chosen answers, [1] the rejected ones), mask (2, P, L) the answers' tokens. With R the sum
    over the mask of logp - ref_logp and D = R_chosen - R_rejected:
      'sigmoid'  -(1 - smoothing) log sigma(beta D) - smoothing log sigma(-beta D)
      'ipo'      (D - 1 / (2 beta))^2 with R the mean over the answer's tokens (smoothing has no part in it)
    Mean over the pairs whose two answers both have tokens (other pairs get no gradient; 0 without any). Returns
    PreferenceLoss(loss, grad = dloss/dlogp (2, P, L), chosen and rejected = the rewards beta R (P)), float32."""
    sh = logp.shape
    if len(sh) != 3 or sh[0] != 2 or ref_logp.shape != sh:
        raise ValueError(f'preference_loss: logp and ref_logp are (2, P, L); got {tuple(sh)} and '
                         f'{tuple(ref_logp.shape)}')
    if kind not in _KINDS:
        raise ValueError(f'preference_loss: kind is one of {sorted(_KINDS)}')
    if not beta > 0 or not 0 <= smoothing < 0.5:
        raise ValueError('preference_loss: beta > 0 and 0 <= smoothing < 0.5')
    dev, lib = _need_cuda('preference_loss', logp, ref_logp, mask), _lib.lib()
    m = _mask(mask, sh, 'preference_loss')
    _, P, L = sh
    lp, rf = _f32(logp), _f32(ref_logp)
    nb = _bytes('asrn_preference_workspace_bytes', P, L)
    loss, rewards, grad = lp.new_empty(()), lp.new_empty((2, P)), torch.empty_like(lp)
    ws = _scratch(nb, dev) if nb else None
    _lib.check(lib.asrn_preference_loss(P, L, lp.data_ptr(), rf.data_ptr(), m.data_ptr(), _KINDS[kind], beta, smoothing,
                                        loss.data_ptr(), grad.data_ptr(), rewards.data_ptr(), _p(ws), nb,
                                        _stream(dev)), 'asrn_preference_loss')
    if logp.requires_grad and torch.is_grad_enabled():
        loss = _WithGrad.apply(logp, loss, grad)
    return PreferenceLoss(loss, grad, *rewards.unbind())


def policy_loss(logp, old_logp, advantages, mask, ref_logp=None, clip=(0.2, 0.2), kl=0.0, per='token'):
    """Clipped policy loss of B sequences of L positions: logp, old_logp, ref_logp (B, L) per-token log probabilities
    under the model, the model that wrote the answers and a reference model; advantages (B, L) or (B); mask (B, L).
    With r = exp(logp - old_logp) and q = ref_logp - logp (both differences held to [-20, 20], without gradient beyond)
      l = -min(r A, clip(r, 1 - clip[0], 1 + clip[1]) A) + kl (exp(q) - q - 1)
    per 'token': the mean over the mask's tokens; 'sequence': over each sequence's tokens, then over the sequences that
    have one. Returns PolicyLoss(loss, grad = dloss/dlogp (B, L), kl = the mean of exp(q) - q - 1, clipped = the share
    of tokens whose ratio was clipped), float32."""
    sh, sa = logp.shape, advantages.shape
    if len(sh) != 2 or old_logp.shape != sh or (ref_logp is not None and ref_logp.shape != sh):
        raise ValueError('policy_loss: logp, old_logp and ref_logp are (B, L); got ' + ', '.join(
            str(tuple(t.shape)) for t in (logp, old_logp, ref_logp) if t is not None))
    B, L = sh
    if sa != sh and (len(sa) != 1 or sa[0] != B):
        raise ValueError(f'policy_loss: advantages are (B, L) or (B); got {tuple(sa)}')
    if per not in _PER:
        raise ValueError(f'policy_loss: per is one of {sorted(_PER)}')
    low, high = clip
    if not 0 <= low < 1 or not high >= 0 or not kl >= 0:
        raise ValueError('policy_loss: 0 <= clip[0] < 1, clip[1] >= 0 and kl >= 0')
    if kl > 0 and ref_logp is None:
        raise ValueError('policy_loss: a KL term needs ref_logp')
    dev, lib = _need_cuda('policy_loss', logp, old_logp, advantages, mask, ref_logp), _lib.lib()
    m = _mask(mask, sh, 'policy_loss')
    lp, old, adv = _f32(logp), _f32(old_logp), _f32(advantages)
    ref = None if ref_logp is None else _f32(ref_logp)
    out, grad = lp.new_empty(3), torch.empty_like(lp)
    nb = _bytes('asrn_policy_workspace_bytes', B, L)
    ws = _scratch(nb, dev) if nb else None
    base = out.data_ptr()
    _lib.check(lib.asrn_policy_loss(B, L, lp.data_ptr(), old.data_ptr(), _p(ref), adv.data_ptr(), len(sa) == 2,
                                    m.data_ptr(), low, high, kl, _PER[per], base, grad.data_ptr(), base + 4, _p(ws), nb,
                                    _stream(dev)), 'asrn_policy_loss')
    loss, k3, clipped = out.unbind()
    if logp.requires_grad and torch.is_grad_enabled():
        loss = _WithGrad.apply(logp, loss, grad)
    return PolicyLoss(loss, grad, k3, clipped)


# ---- activations in 8 bits ----------------------------------------------------------------------------------------------

Packed8 = namedtuple('Packed8', 'codes exps shape')


def pack8(x):
    """x (..., f) bfloat16 in 8 bits: int8 codes and an exponent byte per block of 32 along the last dimension (value =
    code 2^e, e the least with max|x| <= 127 2^e). A block with an infinity or a NaN reads back as NaN. f has to be a
    multiple of 8."""
    if x.dim() < 1 or x.dtype != torch.bfloat16:
        raise TypeError('pack8 takes a bfloat16 tensor (..., f)')
    _need_cuda('pack8', x)
    f = x.shape[-1]
    if f % 8 or f == 0:
        raise NotImplementedError(f'pack8: the last dimension ({f}) has to be a multiple of 8')
    rows, dev = x.numel() // f, x.device
    xr = _rows(x.detach())
    codes = torch.empty(rows, f, dtype=torch.int8, device=dev)
    exps = torch.empty(rows, (f + 31) // 32, dtype=torch.int8, device=dev)
    _lib.check(_lib.lib().asrn_pack8(rows, f, _p(xr), _p(codes), _p(exps), _lib.stream_ptr(dev)), 'asrn_pack8')
    return Packed8(codes, exps, x.shape)


def unpack8(p):
    """The bfloat16 tensor that pack8's result stands for."""
    _need_cuda('unpack8', p.codes, p.exps)
    rows, f = p.codes.shape
    x = torch.empty(p.shape, dtype=torch.bfloat16, device=p.codes.device)
    _lib.check(_lib.lib().asrn_unpack8(rows, f, _p(p.codes), _p(p.exps), _p(x), _lib.stream_ptr(x.device)),
               'asrn_unpack8')
    return x


class _Mlp8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, grad):
        d, ff, dout = x.shape[-1], w1.shape[0], w2.shape[0]
        N, dev, lib = x.numel() // d, x.device, _lib.lib()
        xr, w1, b1, w2, b2 = _rows(x), _rows(w1), _rows(b1), _rows(w2), _rows(b2)
        y = xr.new_empty((*x.shape[:-1], dout))
        keep = grad and any(ctx.needs_input_grad)
        nb_saved = _bytes('asrn_mlp8_saved_bytes', N, d, ff) if keep else 0
        nb = _bytes('asrn_mlp8_workspace_bytes', N, d, ff, dout, 0)
        saved = _scratch(nb_saved, dev) if keep else None
        ws = _scratch(nb, dev)
        _lib.check(lib.asrn_mlp8_forward(N, d, ff, dout, xr.data_ptr(), w1.data_ptr(), b1.data_ptr(), w2.data_ptr(),
                                         b2.data_ptr(), y.data_ptr(), _p(saved), nb_saved, ws.data_ptr(), nb,
                                         _status_word(dev), _stream(dev)), 'asrn_mlp8_forward')
        if keep:
            ctx.save_for_backward(w1, w2, saved)
            ctx.meta = (x.shape, N, d, ff, dout, dev, nb_saved)
        return y

    @staticmethod
    def backward(ctx, dy):
        w1, w2, saved = ctx.saved_tensors
        shape, N, d, ff, dout, dev, nb_saved = ctx.meta
        lib = _lib.lib()
        sizes = (shape, (ff, d), (ff,), (dout, ff), (dout,))
        out = [w1.new_empty(s) if n else None for s, n in zip(sizes, ctx.needs_input_grad)]
        dyr = _rows(dy)
        nb = _bytes('asrn_mlp8_workspace_bytes', N, d, ff, dout, 1)
        ws = _scratch(nb, dev)
        _lib.check(lib.asrn_mlp8_backward(N, d, ff, dout, dyr.data_ptr(), w1.data_ptr(), w2.data_ptr(),
                                          saved.data_ptr(), nb_saved, *[_p(t) for t in out], ws.data_ptr(), nb,
                                          _status_word(dev), _stream(dev)), 'asrn_mlp8_backward')
        return (*out, None)


def mlp8(x, w1, b1, w2, b2):
    """gelu(x w1^T + b1) w2^T + b2 with x (..., d), w1 (ff, d), b1 (ff), w2 (dout, ff), b2 (dout) bfloat16 (or float32
    under bf16 autocast) -> bfloat16 (..., dout). For the backward pass it keeps x and x w1^T + b1 in 8 bits (pack8's
    form: (d + ff) 33 / 32 bytes a row), and the gradients are those of the values so kept. d, ff and dout have to be
    multiples of 8."""
    sx, s1, s2 = x.shape, w1.shape, w2.shape
    if not sx or len(s1) != 2 or len(s2) != 2 or s1[1] != sx[-1] or b1.shape != s1[:1] or s2[1] != s1[0] or \
            b2.shape != s2[:1]:
        raise ValueError('mlp8: x (..., d), w1 (ff, d), b1 (ff), w2 (dout, ff), b2 (dout) do not fit: ' + ', '.join(
            str(tuple(t.shape)) for t in (x, w1, b1, w2, b2)))
    _need_cuda('mlp8', x, w1, b1, w2, b2)
    if s1[0] % 8 or s1[1] % 8 or s2[0] % 8 or not s1[0] * s1[1] * s2[0]:
        raise NotImplementedError(f'mlp8: the widths ({s1[1]}, {s1[0]}, {s2[0]}) have to be multiples of 8')
    return _Mlp8.apply(*_bf16('mlp8', x, w1, b1, w2, b2), torch.is_grad_enabled())

"""Fine-tuning on the device: log probabilities through the tied head, losses on them, an MLP whose activations are
kept in 8 bits, and the norm, the product and the head's statistics that training and answering share (the C ABI's
asrn_head_*, asrn_preference_loss, asrn_policy_loss, asrn_mlp8_*, asrn_pack8, asrn_layer_norm*, asrn_linear_*).

    head_logprobs    log softmax(h W^T / temperatura)[token] and its gradients; the (tokens, V) logits are not kept
    preference_loss  logistic or squared (IPO) loss of pairs of a chosen and a rejected answer
    policy_loss      clipped policy loss with an advantage per answer or token and a KL term against a reference model
    mlp8             gelu(x W1^T + b1) W2^T + b2 that keeps x and x W1^T + b1 in 8 bits for its backward pass
    pack8, unpack8   the 8-bit form by itself
    layer_norm       layer norm with the residual sum before it
    linear           activation(x W^T + b) + residual
    head_stats       head_logprobs with the distribution's entropy and its likeliest tokens

The losses return their gradient with the loss (one pass over the tokens makes both), so a step is

    logp = model.logprobs(x, targets)
    r = preference_loss(logp.detach(), ref_logp, mask)
    logp.backward(r.grad)

and r.loss.backward() works as well when logp requires a gradient. The losses are functions of logp: their other inputs
are constants. Everything runs on CUDA tensors, on the current stream, and repeats bit for bit; second derivatives and
forward-mode ones are refused. There is no counterpart in the reference.

What head_logprobs and mlp8 round to bf16 besides their results: the head dL/dscores, mlp8 gelu and dL/d(x w1^T + b1), once
each, as operands of the next products (and gelu' to fp16). In calls of up to 512 rows, left-out ones counted (the head:
and rows x V x d up to 2^34), the remainders are multiplied too, and gelu' is not rounded: a weight's gradient from few rows
would else hold little but those roundings. So a row's y, dx and dh differ in their last bits with the number of rows in the
call: against 64 bits they are off by 2.3e-3 to 2.5e-3 of themselves in the 2-norm above 512, by 1.7e-3 up to there.
linear and head_stats follow the same rules (linear: up to 512 rows; it keeps the slope in fp16 in any call), and small
calls (linear up to 3 2^17 results, 2^20 of up to 16 rows, head_stats up to 16 rows, 32 of small vocabularies) take a kernel
that sums in another order. layer_norm rounds its results only. Products are summed in fp32 as the tensor cores sum,
truncated: a result in fp32 (linear with a residual in fp32) is off by 1e-6 of itself at d = 1536.
"""
from collections import namedtuple

import torch

from . import _lib


def status(device=None, reset=False):
    """0, or the error that these kernels recorded on the device (ASRN_ERR_TIMEOUT: a bounded wait gave up, and the
    results since then are void). Synchronises. While an error stands head_logprobs, head_stats, linear, mlp8 and their backward
    passes raise RuntimeError as soon as the host sees it; reset=True clears it and allows new calls."""
    dev = torch.device('cuda', torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.type != 'cuda':
        raise ValueError(f'status: {dev} is not a CUDA device')
    index = torch.cuda.current_device() if dev.index is None else dev.index
    return _lib.finetune().status(index, reset)


def head_logprobs(h, weight, tokens, temperatura=1.0):
    """log softmax(h weight^T / temperatura) at tokens: h (..., d), weight (V, d) bfloat16 (or float32 under bf16
    autocast), tokens (...) int64 -> float32 (...), differentiable in h and weight. A negative token leaves its
    position out (0, no gradient, none of the work); a token >= V gives NaN. d has to be a multiple of 8. The backward pass
    forms the scores again and holds their gradient, (counted tokens, V) in bf16, by chunks of rows of up to 2 GiB (more
    where 256 rows are more)."""
    return _lib.finetune().head_logprobs(h, weight, tokens, temperatura)


PreferenceLoss = namedtuple('PreferenceLoss', 'loss grad chosen rejected')
PolicyLoss = namedtuple('PolicyLoss', 'loss grad kl clipped')

_KINDS = {'sigmoid': 0, 'ipo': 1}
_PER = {'token': 0, 'sequence': 1}


def preference_loss(logp, ref_logp, mask, beta=0.1, smoothing=0.0, kind='sigmoid'):
    """Loss of P pairs of answers, logp and ref_logp (2, P, L) per-token log probabilities under the model and the
    reference model ([0] the chosen answers, [1] the rejected ones), mask (2, P, L) the answers' tokens. With R the sum
    over the mask of logp - ref_logp, n the answer's tokens and D = R_chosen - R_rejected:
      'sigmoid'  -(1 - smoothing) log sigma(beta D) - smoothing log sigma(-beta D)
      'ipo'      (R_chosen / n_chosen - R_rejected / n_rejected - 1 / (2 beta))^2 (smoothing has no part in it)
    Mean over the pairs whose two answers both have tokens (other pairs get no gradient; 0 without any). Returns
    PreferenceLoss(loss, grad = dloss/dlogp (2, P, L), chosen and rejected = the rewards beta R (P), sums
    in both kinds), float32."""
    if kind not in _KINDS:
        raise ValueError(f'preference_loss: kind is one of {sorted(_KINDS)}')
    loss, grad, chosen, rejected = _lib.finetune().preference_loss(logp, ref_logp, mask, _KINDS[kind], beta, smoothing)
    if logp.requires_grad and torch.is_grad_enabled():
        loss = _lib.finetune().known_gradient(logp, loss, grad)
    return PreferenceLoss(loss, grad, chosen, rejected)


def policy_loss(logp, old_logp, advantages, mask, ref_logp=None, clip=(0.2, 0.2), kl=0.0, per='token'):
    """Clipped policy loss of B sequences of L positions: logp, old_logp, ref_logp (B, L) per-token log probabilities
    under the model, the model that wrote the answers and a reference model; advantages (B, L) or (B); mask (B, L).
    With r = exp(logp - old_logp) and q = ref_logp - logp (both differences held to [-20, 20], without gradient beyond)
      l = -min(r A, clip(r, 1 - clip[0], 1 + clip[1]) A) + kl (exp(q) - q - 1)
    per 'token': the mean over the mask's tokens; 'sequence': over each sequence's tokens, then over the sequences that
    have one. Returns PolicyLoss(loss, grad = dloss/dlogp (B, L), kl = the mean of exp(q) - q - 1, clipped = the share
    of tokens whose ratio was clipped), float32."""
    if per not in _PER:
        raise ValueError(f'policy_loss: per is one of {sorted(_PER)}')
    low, high = clip
    loss, grad, k3, clipped = _lib.finetune().policy_loss(logp, old_logp, advantages, mask, ref_logp, low, high, kl,
                                                          _PER[per])
    if logp.requires_grad and torch.is_grad_enabled():
        loss = _lib.finetune().known_gradient(logp, loss, grad)
    return PolicyLoss(loss, grad, k3, clipped)


Packed8 = namedtuple('Packed8', 'codes exps shape')


def pack8(x):
    """x (..., f) bfloat16 in 8 bits: int8 codes and an exponent byte per block of 32 along the last dimension (value =
    code 2^e, e the least with max|x| <= 127 2^e). A block with an infinity or a NaN reads back as NaN. f has to be a
    multiple of 8."""
    return Packed8(*_lib.finetune().pack8(x), x.shape)


def unpack8(p):
    """The bfloat16 tensor that pack8's result stands for."""
    return _lib.finetune().unpack8(p.codes, p.exps, p.shape)


def mlp8(x, w1, b1, w2, b2):
    """gelu(x w1^T + b1) w2^T + b2 with x (..., d), w1 (ff, d), b1 (ff), w2 (dout, ff), b2 (dout) bfloat16 (or float32
    under bf16 autocast) -> bfloat16 (..., dout). For the backward pass it keeps x and x w1^T + b1 in 8 bits (pack8's
    form: (d + ff) 33 / 32 bytes a row), and the gradients are those of the values so kept. d, ff and dout have to be
    multiples of 8."""
    return _lib.finetune().mlp8(x, w1, b1, w2, b2)


def layer_norm(x, weight, bias=None, residual=None, eps=1e-5, dtype=None):
    """Layer norm over the last dimension, x (..., d), weight and bias (d), d up to 16384, each float32 or bfloat16 ->
    y of type `dtype` (default: x's). With residual (..., d) the sum s = x + residual, rounded to the residual's type, is
    normalised and handed on: returns (y, s), one pass over memory for both. Sums and statistics in fp32. Differentiable
    in x, weight, bias and residual; the weight's gradient is summed in fp32, in a fixed order."""
    y, s = _lib.finetune().layer_norm(x, weight, bias, residual, eps, dtype)
    return y if residual is None else (y, s)


_ACTIVATIONS = {None: 0, 'gelu': 1, 'silu': 2, 'relu': 3}


def linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight^T + bias) + residual in one product: x (..., d), weight (n, d), bias (n) bfloat16 (or float32
    under bf16 autocast), activation None, 'gelu' (erf), 'silu' or 'relu', residual (..., n) float32 or bfloat16 -> (..., n)
    of the residual's type, bfloat16 without one. d and n have to be multiples of 8. For the backward pass it keeps x and
    the activation's slope in fp16. Small calls (up to 3 2^17 results, 2^20 of up to 16 rows) take a kernel that spreads
    the weight over the whole GPU."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"linear: activation is None, 'gelu', 'silu' or 'relu'; got {activation!r}")
    return _lib.finetune().linear(x, weight, bias, _ACTIVATIONS[activation], residual)


HeadStats = namedtuple('HeadStats', 'logp entropy top_logp top_tokens')


def head_stats(h, weight, tokens=None, temperatura=1.0, top=0):
    """The distribution p = softmax(h weight^T / temperatura) by its statistics, without its (tokens, V) logits: h (..., d),
    weight (V, d) bfloat16 (or float32 under bf16 autocast), tokens (...) int64 or None. Returns HeadStats:
      logp        log p[token] (None without tokens), float32, head_logprobs' values
      entropy     - sum p log p, float32
      top_logp, top_tokens   (..., top) the `top` (up to 32) likeliest tokens and their log probabilities, the likeliest first,
                  equal ones by their number (None without top). Scores nearer one another than sums in fp32 tell are ranked
                  by sums in 64 bits
    Differentiable in h and weight through logp and entropy. A negative token leaves its position out (0, tokens -1, no
    gradient, none of the work); a token >= V, and scores whose exponentials have no finite sum, give NaN and tokens -1. d has
    to be a multiple of 8. The call takes V / 4 bytes of workspace a position; with top as much again (V / 8 above 32768 tokens), or
    4 V in vocabularies of up to 2048 tokens where top^2 is more than V^2 / (24 d). The backward pass holds what head_logprobs'
    does."""
    return HeadStats(*_lib.finetune().head_stats(h, weight, tokens, temperatura, top))

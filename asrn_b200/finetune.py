"""Fine-tuning on the device: log probabilities through the tied head, losses on them, and an MLP whose activations are
kept in 8 bits (the C ABI's asrn_head_*, asrn_preference_loss, asrn_policy_loss, asrn_mlp8_*, asrn_pack8).

    head_logprobs    log softmax(h W^T / temperatura)[token] and its gradients; the (tokens, V) logits are not kept
    preference_loss  logistic or squared (IPO) loss of pairs of a chosen and a rejected answer
    policy_loss      clipped policy loss with an advantage per answer or token and a KL term against a reference model
    mlp8             gelu(x W1^T + b1) W2^T + b2 that keeps x and x W1^T + b1 in 8 bits for its backward pass
    pack8, unpack8   the 8-bit form by itself

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
"""
from collections import namedtuple

import torch

from . import _lib


def status(device=None, reset=False):
    """0, or the error that these kernels recorded on the device (ASRN_ERR_TIMEOUT: a bounded wait gave up, and the
    results since then are void). Synchronises. While an error stands head_logprobs, mlp8 and their backward passes raise
    RuntimeError as soon as the host sees it; reset=True clears it and allows new calls."""
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

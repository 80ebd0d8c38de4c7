"""The fine-tuning operators where the model uses them: model.logprobs against the model's own logits, local blocks with
8-bit activations against the same blocks without, and the example that runs everything together."""
import os
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def make(cuda, V=600, d=64, **kw):
    import asrn_b200 as asrn
    m = asrn.create_model(V=V, d=d, n_capas=4, semilla=3, **kw).to(cuda)
    x = torch.randint(0, V, (3, 70), generator=torch.Generator().manual_seed(5)).to(cuda)
    return m, x


def test_logprobs_of_the_logits(cuda):
    """Under autocast the logits are rounded to bf16 (unit roundoff 2^-8) and head_logprobs' scores are not: the two differ
    by that much of the largest logit, twice (the target's and the sum's)."""
    m, x = make(cuda)
    y = torch.nn.functional.pad(x[:, 1:], (0, 1), value=-1)
    y[0, :40] = -1
    m.eval()
    with torch.no_grad():
        # the layers' sums over the tables vary from run to run in their last bits: one state for both sides
        h = m.estado(x)
        m.estado = lambda x: h
        lg = m(x)
        ref = torch.log_softmax(lg, -1).gather(-1, y.clamp(min=0)[..., None])[..., 0] * (y >= 0)
        assert torch.equal(m.logprobs(x, y), ref)                        # the fp32 model
        with torch.autocast('cuda', dtype=torch.bfloat16):
            lg = m(x).float()
            got = m.logprobs(x, y)
            ref = torch.log_softmax(lg, -1).gather(-1, y.clamp(min=0)[..., None])[..., 0] * (y >= 0)
    assert got.dtype == torch.float32
    assert float((got - ref).abs().max()) <= 2 * 2.0 ** -8 * float(lg.abs().max()) + 1e-6
    assert (got[y < 0] == 0).all()
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        assert torch.equal(m.logprobs(x)[1:], got[1:])                   # the default targets: each next token
    with pytest.raises(ValueError):
        m.logprobs(x, y[:, :-1])


def grads(m, x, loss):
    m.zero_grad(set_to_none=True)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        loss(m, x).backward()
    return {k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None}


def test_logprobs_gradients_are_the_cross_entropys(cuda):
    """mean(-logprobs) is the cross entropy of the logits; the paths differ by bf16 roundings of logits and gradients
    (2^-8 each at most, on a few of them), through four blocks and two ASRN layers."""
    m, x = make(cuda)
    m.train()

    def ce(m, x):
        lg = m(x)[:, :-1].float()
        return torch.nn.functional.cross_entropy(lg.reshape(-1, lg.shape[-1]), x[:, 1:].reshape(-1))
    a = grads(m, x, ce)
    b = grads(m, x, lambda m, x: -m.logprobs(x).sum() / (x.shape[0] * (x.shape[1] - 1)))
    assert set(a) == set(b)
    for k in ('emb.weight', 'ln_f.weight', 'bloques.3.ff.2.weight', 'bloques.0.conv.weight'):
        assert float((a[k] - b[k]).norm() / a[k].norm()) <= 2e-2, k


def test_blocks_with_8bit_activations(cuda):
    """The forward pass is the unfused block's but for the bf16 rounding of x W1 + b1 that mlp8 leaves out; gradients stay
    within the 8-bit values' error (1/127 of a block's largest, a few of them along the way)."""
    import asrn_b200 as asrn
    m, x = make(cuda)
    m8 = asrn.create_model(V=600, d=64, n_capas=4, semilla=3, checkpoint='8bits').to(cuda)
    assert not m.bloques[0].activaciones_8bits and m8.bloques[0].activaciones_8bits
    assert m.config == m8.config and m.state_dict().keys() == m8.state_dict().keys()
    m.train(), m8.train()
    loss = lambda m, x: -m.logprobs(x).mean()  # noqa: E731
    a, b = grads(m, x, loss), grads(m8, x, loss)
    for k in ('emb.weight', 'bloques.0.ff.0.weight', 'bloques.0.ff.0.bias', 'bloques.1.ff.2.weight', 'bloques.3.ff.2.bias'):
        assert b[k].dtype == torch.float32
        assert float((a[k] - b[k]).norm() / a[k].norm()) <= 6e-2, k
    h = torch.randn(2, 50, 64, generator=torch.Generator().manual_seed(6)).to(cuda)
    with torch.no_grad():                                                # inference, and the fp32 block: as before
        assert torch.equal(m.bloques[0](h), m8.bloques[0](h))
        with torch.autocast('cuda', dtype=torch.bfloat16):
            assert torch.equal(m.bloques[0](h), m8.bloques[0](h))
    assert torch.equal(m.bloques[0](h), m8.bloques[0](h))


def test_8bit_activations_take_less_memory(cuda):
    import asrn_b200 as asrn
    kept = {}
    for how in (False, '8bits'):
        blq = asrn.create_model(V=64, d=256, n_capas=2, semilla=0, checkpoint=how).to(cuda).train().bloques[0]
        h = torch.randn(2, 2048, 256, device=cuda, requires_grad=True)
        sizes = {}

        def keep(t):
            sizes[t.untyped_storage().data_ptr()] = t.untyped_storage().nbytes()
            return t
        with torch.autocast('cuda', dtype=torch.bfloat16), torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            blq(h)
        kept[how] = sum(sizes.values())
    # the MLP's x, x W1 + b1 and gelu of it in bf16 (d + 2 ff) against (d + ff) bytes and a scale for every 32
    n, d, ff = 4096, 256, 512
    assert kept[False] - kept['8bits'] >= 0.9 * (2 * n * (d + 2 * ff) - n * (d + ff) * 33 // 32)


def test_the_example_learns(cuda):
    sys.path.insert(0, os.path.join(ROOT, 'examples'))
    try:
        import preference_tuning
    finally:
        sys.path.pop(0)
    pref, policy = preference_tuning.main(['--pairs', '6', '--length', '65', '--steps', '12'])
    assert abs(pref[0] - 0.6931) < 1e-3 and pref[-1] < 0.6 and policy[-1] < policy[0] + 1e-6

"""layer_norm, linear and head_stats where the model uses them: local blocks with fundido=True against the same blocks without,
model.stats against the model's own logits, and a policy step with an entropy term that runs all of them together."""
import os
import sys

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


def make(cuda, V=600, d=64, **kw):
    import asrn_b200 as asrn
    m = asrn.create_model(V=V, d=d, n_capas=4, semilla=3, **kw).to(cuda)
    x = torch.randint(0, V, (3, 70), generator=torch.Generator().manual_seed(5)).to(cuda)
    return m, x


def grads(m, x, loss):
    m.zero_grad(set_to_none=True)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        loss(m, x).backward()
    return {k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None}


@pytest.mark.parametrize('d,ff', [(64, None), (200, 304)])
def test_block_forward(cuda, d, ff):
    """Both paths round to bf16 the norms' results, x W1 + b1 or gelu of it, and the MLP's result; the norms' may fall to either
    side where fp32 sums differ in their last bits: 2 U of each operand through the products that follow."""
    m, _ = make(cuda, d=d, ff=ff)
    f, _ = make(cuda, d=d, ff=ff, fundido=True)
    h = torch.randn(2, 90, d, generator=torch.Generator().manual_seed(6)).to(cuda)
    a, b = m.bloques[1], f.bloques[1]
    assert b.fundido and not a.fundido
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        if not a._fused_ok(h):
            one, two = a(h), b(h)
        else:
            one, two = a._fused(h), b._fundido(h)
    z = a.ln1(h)
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        c = torch.nn.functional.gelu(a.conv(torch.nn.functional.pad(z.transpose(1, 2), (a.k - 1, 0))).transpose(1, 2))
    with torch.no_grad():
        w1, w2 = a.ff[0].weight.double().abs(), a.ff[2].weight.double().abs()
        u = a.ln2(h + c).double()
        p = u @ a.ff[0].weight.double().t() + a.ff[0].bias.double()
        g = torch.nn.functional.gelu(p)
        dp = 2 * U * u.abs() @ w1.t() + U * p.abs()
        out = (g @ a.ff[2].weight.double().t() + a.ff[2].bias.double()).abs()
        tol = 2 * (1.2 * dp + U * g.abs()) @ w2.t() + 2 * U * out
        # the first norm's flips, through the conv: at most one unit of its result's
        conv = torch.nn.functional.conv1d(torch.nn.functional.pad(2 * U * z.double().abs().transpose(1, 2), (a.k - 1, 0)),
                                          a.conv.weight.double().abs()).transpose(1, 2)
        tol = tol + conv + 2 * U * c.double().abs()
        # and from there through norm and MLP: a change of the state as large moves the norm by at most twice it over its spread
        spread = (h + c).double().std(-1, unbiased=False, keepdim=True)
        tol = tol + ((2 * (conv + 2 * U * c.double().abs()) / spread) @ w1.t() * 1.2) @ w2.t()
    assert one.dtype == two.dtype == torch.float32
    assert ((one.double() - two.double()).abs() <= tol).all(), float(((one - two).abs() / tol).max())


@pytest.mark.parametrize('kw', [{}, dict(checkpoint='8bits')])
def test_training_gradients(cuda, kw):
    """The same loss through both paths: they differ by bf16 roundings (2^-8 each at most, on a few of them) of operands and
    gradients through four blocks and two ASRN layers."""
    m, x = make(cuda, **kw)
    f, _ = make(cuda, fundido=True, **kw)
    assert m.config == f.config and m.state_dict().keys() == f.state_dict().keys()
    m.train(), f.train()
    loss = lambda m, x: -m.logprobs(x).mean()  # noqa: E731
    a, b = grads(m, x, loss), grads(f, x, loss)
    assert set(a) == set(b)
    for k in ('emb.weight', 'ln_f.weight', 'ln_f.bias', 'bloques.0.ln1.weight', 'bloques.1.ln2.bias', 'bloques.3.ff.2.weight',
              'bloques.0.ff.0.weight', 'bloques.2.ff.0.bias', 'bloques.0.conv.weight'):
        assert b[k].dtype == torch.float32
        assert float((a[k] - b[k]).norm() / a[k].norm()) <= (6e-2 if kw else 3e-2), k


def test_what_is_not_as_built_is_called(cuda):
    f, x = make(cuda, fundido=True)
    blq = f.bloques[0]
    h = torch.randn(2, 30, 64, generator=torch.Generator().manual_seed(7)).to(cuda)
    seen = []
    with torch.autocast('cuda', dtype=torch.bfloat16):
        assert blq._fundido_ok(h)
        hook = blq.ln2.register_forward_hook(lambda *a: seen.append(1))
        blq(h)
        assert seen == [1]
        hook.remove()
        blq.ff[1].forward = lambda t: seen.append(2) or torch.relu(t)
        blq(h)
        assert seen == [1, 2]
        del blq.ff[1].forward
        old, blq.ff[0] = blq.ff[0], torch.nn.Linear(64, 128, bias=False).to(cuda)
        assert not blq._fundido_ok(h)
        blq.ff[0] = old
        assert not blq._fundido_ok(h.half()) and not blq._fundido_ok(h.double())
    assert not blq._fundido_ok(h)                          # the fp32 model keeps PyTorch's operations
    g, _ = make(cuda)
    assert torch.equal(g.bloques[0](h), blq(h))
    # dropout at work: the same mask falls on the same branch
    blq.drop.p = 0.5
    f.train()
    with torch.autocast('cuda', dtype=torch.bfloat16):
        torch.manual_seed(0)
        one = blq(h)
        torch.manual_seed(0)
        assert torch.equal(blq(h), one)
        blq.eval()
        assert not torch.equal(blq(h), one)


def test_dropout_goes_by_its_own_mode_and_is_called_where_it_has_hooks(cuda):
    f, _ = make(cuda, fundido=True)
    blq = f.bloques[0]
    h = torch.randn(2, 30, 64, generator=torch.Generator().manual_seed(8)).to(cuda)
    seen = []
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        f.eval()
        plain = blq._fundido(h)
        hook = blq.drop.register_forward_hook(lambda *a: seen.append(1))
        blq._fundido(h)
        assert len(seen) == 2                              # after the conv and after the MLP
        hook.remove()
        blq.drop.p = 0.5
        assert torch.equal(blq._fundido(h), plain)         # not in training
        blq.drop.train()
        assert not torch.equal(blq._fundido(h), plain)     # the module alone is
        blq.drop = torch.nn.Identity()
        assert (blq._fundido(h) - plain).abs().max() <= 2 * U * plain.abs().max()


def test_recomputed_blocks_give_the_same_gradients(cuda):
    """checkpoint=True runs a block's forward pass again in the backward pass: the kernels repeat bit for bit. What is not
    bitwise the same is what PyTorch's own operations (the embedding's sum) add up in any order."""
    f, x = make(cuda, fundido=True)
    g, _ = make(cuda, fundido=True, checkpoint=True)
    f.train(), g.train()
    loss = lambda m, x: -m.logprobs(x).mean()  # noqa: E731
    a, b = grads(f, x, loss), grads(g, x, loss)
    assert torch.equal(a['ln_f.weight'], b['ln_f.weight']) and torch.equal(a['bloques.3.ff.2.weight'], b['bloques.3.ff.2.weight'])
    assert torch.equal(a['bloques.3.ln2.weight'], b['bloques.3.ln2.weight'])


def test_saved_models_load_either_way(cuda, tmp_path):
    import asrn_b200 as asrn
    f, x = make(cuda, fundido=True)
    asrn.save(f, str(tmp_path / 'm.pt'))
    g, h = asrn.load(str(tmp_path / 'm.pt'), fundido=True), asrn.load(str(tmp_path / 'm.pt'))
    assert g.fundido and g.bloques[2].fundido and not h.fundido and not h.bloques[2].fundido
    assert all(torch.equal(a, b) for a, b in zip(g.state_dict().values(), f.state_dict().values()))


@pytest.mark.parametrize('fundido', [False, True])
def test_stats_of_the_logits(cuda, fundido):
    """Under autocast the logits are rounded to bf16 and head_stats' scores are not: 2^-8 of the largest logit, twice."""
    m, x = make(cuda, fundido=fundido)
    y = torch.nn.functional.pad(x[:, 1:], (0, 1), value=-1)
    y[0, :40] = -1
    y[1, 3] = 600
    m.eval()
    with torch.no_grad():
        h = m.estado(x)                                   # one state for both sides (its last bits vary from run to run)
        m.estado = lambda x: h
        lp = torch.log_softmax(m(x), -1)
        H = -(lp.exp() * lp).sum(-1)
        on, out = y >= 0, y >= 600
        r = m.stats(x, y, top=4)                          # the fp32 model
        for t in r[:3]:
            assert t.dtype == torch.float32 and (t[~on] == 0).all() and t[out].isnan().all()
        good = on & ~out
        assert torch.equal(r.logp[good], lp.gather(-1, y.clamp(0, 599)[..., None])[..., 0][good])
        assert (r.entropy - H)[good].abs().max() <= 1e-5 and (r.top_tokens[~good] == -1).all()
        assert torch.equal(r.top_tokens[good], lp.sort(dim=-1, descending=True, stable=True).indices[good][:, :4])
        assert torch.equal(m.logprobs(x, y)[good], r.logp[good])
        free = m.stats(x, top=1)
        assert free.logp is None and torch.equal(free.top_tokens[..., 0], lp.argmax(-1))
        with torch.autocast('cuda', dtype=torch.bfloat16):
            q = m.stats(x, y, top=4)
            big = float(m(x).float().abs().max())
        assert (q.logp - r.logp)[good].abs().max() <= 4 * U * big and (q.entropy - r.entropy)[good].abs().max() <= 8 * U * big
        assert (q.top_tokens[~good] == -1).all() and q.entropy[out].isnan().all() and (q.top_logp[~on] == 0).all()
        assert (q.top_logp - r.top_logp)[good].abs().max() <= 4 * U * big
    for kw in (dict(top=33), dict(top=-1), dict(temperatura=0.0), dict(objetivos=y[:, 1:])):
        with pytest.raises(ValueError):
            m.stats(x, **kw)
    m.head.register_forward_hook(lambda *a: None)         # a head with hooks is called
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        assert m.stats(x, y).logp.shape == y.shape


def test_stats_of_a_padded_batch(cuda):
    """What stands behind a sequence's end changes nothing before it, in either direction, and gets nothing itself."""
    f, x = make(cuda, fundido=True)
    f.eval()
    y = torch.nn.functional.pad(x[:, 1:], (0, 1), value=-1)
    end = torch.tensor([70, 41, 1], device=cuda)
    y = torch.where(torch.arange(70, device=cuda) < end[:, None], y, -1)
    keep = f.estado
    with torch.autocast('cuda', dtype=torch.bfloat16):
        with torch.no_grad():
            h = keep(x).detach()
        junk = torch.where((torch.arange(70, device=cuda) < end[:, None])[..., None], h, torch.full_like(h, float('nan')))
        got = []
        for state in (h, junk):
            state = state.clone().requires_grad_()
            f.estado = lambda x, state=state: state
            r = f.stats(x, y, top=3)
            w, = (p for n, p in f.named_parameters() if n == 'emb.weight' or n == 'head.weight')
            got.append((*(t.detach() for t in r), *torch.autograd.grad(r.logp.sum() + r.entropy.sum(), (state, w))))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    off = y < 0
    assert (got[0][0][off] == 0).all() and (got[0][3][off] == -1).all() and (got[0][4][off] == 0).all()


def test_a_policy_step_with_an_entropy_term(cuda):
    """norms, products, head statistics and policy loss in one step, against the same loss by torch's operations on the logits."""
    import asrn_b200 as asrn
    f, x = make(cuda, fundido=True)
    m, _ = make(cuda)
    y = torch.nn.functional.pad(x[:, 1:], (0, 1), value=-1)
    y[:, :20] = -1
    mask = y >= 0
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        old = f.logprobs(x, y) + 0.05 * torch.randn(y.shape, generator=torch.Generator().manual_seed(8)).to(cuda) * mask
    adv = torch.tensor([1.0, -0.5, 0.3], device=cuda)
    c = 0.02
    f.train(), m.train()
    f.zero_grad(set_to_none=True)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        r = f.stats(x, y, top=3)
    p = asrn.policy_loss(r.logp.detach(), old, adv, mask)
    torch.autograd.backward((r.logp, r.entropy), (p.grad, -c * mask / mask.sum()))
    got = {k: q.grad for k, q in f.named_parameters() if q.grad is not None}

    def loss(m, x):
        lp = torch.log_softmax(m(x).float(), -1)
        H = -(lp.exp() * lp).sum(-1)
        ratio = (lp.gather(-1, y.clamp(min=0)[..., None])[..., 0] - old)[mask].exp()
        A = adv[:, None].expand(mask.shape)[mask]
        return -torch.minimum(ratio * A, ratio.clamp(0.8, 1.2) * A).mean() - c * H[mask].mean()
    want = grads(m, x, loss)
    for k in ('emb.weight', 'ln_f.weight', 'bloques.3.ff.2.weight', 'bloques.0.ff.0.weight', 'bloques.1.ln2.weight'):
        assert float((got[k] - want[k]).norm() / want[k].norm()) <= 5e-2, k
    assert r.top_tokens.shape == (*y.shape, 3) and (r.top_logp[mask] <= 0).all()


def test_the_example_runs_with_all_of_them(cuda):
    sys.path.insert(0, os.path.join(ROOT, 'examples'))
    try:
        import preference_tuning
    finally:
        sys.path.pop(0)
    pref, policy = preference_tuning.main(['--pairs', '4', '--length', '65', '--steps', '3', '--fused', '--entropy', '0.01'])
    assert len(pref) == len(policy) == 3 and all(v == v for v in pref + policy)

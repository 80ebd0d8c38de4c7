"""First derivatives recorded with create_graph where an output has no gradient: the values of the call that does not record, and
the refusal of the second derivative."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def calls():
    import asrn_b200 as asrn
    x, r, w, b = rand((9, 64), 1), rand((9, 64), 2, dtype=torch.float32), rand((64,), 3, dtype=torch.float32), rand((64,), 4, dtype=torch.float32)
    head, y = rand((40, 64), 5, 0.2), torch.arange(9, device='cuda')
    norm = lambda x, r, w, b: asrn.layer_norm(x, w, b, residual=r)  # noqa: E731
    stats = lambda top, t: lambda h, w: asrn.head_stats(h, w, t, top=top)  # noqa: E731
    return {'norm y': ((x, r, w, b), lambda *t: norm(*t)[0]), 'norm sum': ((x, r, w, b), lambda *t: norm(*t)[1]),
            'norm both': ((x, r, w, b), lambda *t: norm(*t)[0].float() + norm(*t)[1]),
            'logp': ((x, head), lambda *t: stats(0, y)(*t).logp), 'entropy': ((x, head), lambda *t: stats(0, y)(*t).entropy),
            'logp and tokens': ((x, head), lambda *t: stats(3, y)(*t).logp),
            'entropy and tokens': ((x, head), lambda *t: stats(3, None)(*t).entropy)}


@pytest.mark.parametrize('which', ['norm y', 'norm sum', 'norm both', 'logp', 'entropy', 'logp and tokens', 'entropy and tokens'])
def test_recorded_first_derivatives(cuda, which):
    leaves, f = calls()[which]
    leaves = [t.requires_grad_() for t in leaves]
    grads = lambda **k: torch.autograd.grad(f(*leaves).float().square().sum(), leaves, allow_unused=True, **k)  # noqa: E731
    want, got = grads(), grads(create_graph=True)
    for p, q in zip(want, got):
        assert (p is None and q is None) or torch.equal(p, q)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(got[0].float().sum(), leaves[0])

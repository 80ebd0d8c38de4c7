"""linear's gradients from a dY that holds infinities: dA = dY act'(a), dx = dA W, dW = dA^T x as these products give them, the same for few
rows (whose roundings are multiplied, too) and many."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rand(shape, seed, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


@pytest.mark.parametrize('N', [3, 100, 512, 600])
@pytest.mark.parametrize('residual', [True, False])
@pytest.mark.parametrize('act', [None, 'gelu', 'relu'])
def test_an_infinite_gradient(cuda, N, residual, act):
    import asrn_b200 as asrn
    d, n = 64, 40
    x, w = rand((N, d), 1), rand((n, d), 2, 0.1)
    x[0, 0], w[5, 0] = 40, 40                             # a at (0, 5) is large: act' = 1
    w[5] = torch.where(w[5] == 0, 0.5, w[5])
    x[0] = torch.where(x[0] == 0, 0.5, x[0])
    r = rand((N, n), 3, dtype=torch.float32) if residual else None
    leaves = x.requires_grad_(), w.requires_grad_()
    y = asrn.linear(*leaves, activation=act, residual=r)
    dy = rand((N, n), 4, dtype=y.dtype)
    dy[0, 5] = float('inf')
    dx, dw = torch.autograd.grad(y, leaves, dy)
    assert torch.equal(dx[0].float(), w.detach()[5].float().sign() * float('inf')) and torch.isfinite(dx[1:]).all()
    rest = torch.arange(n, device='cuda') != 5
    assert torch.equal(dw[5].float(), x.detach()[0].float().sign() * float('inf')) and torch.isfinite(dw[rest]).all()


@pytest.mark.parametrize('N', [3, 100, 600])
@pytest.mark.parametrize('bad', [float('inf'), -float('inf'), float('nan')])
def test_what_relu_left_out_takes_no_part(cuda, N, bad):
    import asrn_b200 as asrn
    d, n = 64, 40
    x, w, b = rand((N, d), 5).requires_grad_(), rand((n, d), 6, 0.1).requires_grad_(), rand((n,), 7).requires_grad_()
    y = asrn.linear(x, w, b, activation='relu')
    off = y.detach() == 0
    dy = rand((N, n), 8)
    want = torch.autograd.grad(y, (x, w, b), torch.where(off, 0.0, dy), retain_graph=True)
    got = torch.autograd.grad(y, (x, w, b), torch.where(off, bad, dy))
    assert off.any() and all(torch.equal(p, q) for p, q in zip(want, got))

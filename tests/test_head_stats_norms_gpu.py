"""The likeliest tokens of head_stats where rows of the weight differ much in size: a token's score in fp32 is off by as much as its own
products are large, not by those of the likeliest one. The order is that of the exact scores; 64 bits hold the sums here with 2^-53 of
their magnitudes."""
import math

import pytest
import torch

from test_head_stats_gpu import check, rand, targets

pytestmark = pytest.mark.gpu


def weight(V, d, large, seed):
    """Small rows, whose scores with a state of ones (but for its last two values) are up to about 1.2; and at `large` rows that begin with a
    large value B, take it back at the end, and hold values s between, each below 2^-25 B, which a sum in fp32 that has B in it
    loses whole. Their scores are 1 to 4, some 2^-8 apart, and the last coordinate's part."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, d, generator=g) * 0.3 / d ** 0.5
    n = len(large)
    assert n <= 128
    s = (1 + torch.randperm(128, generator=g)[:n].float() / 128) * 2.0 ** math.floor(math.log2(1.4 / (d - 4)) + 0.5)     # exact in bf16
    rows = s[:, None].repeat(1, d)
    rows[:, 0] = 2.0 ** 25 * 2.0 ** math.ceil(math.log2(2.8 / (d - 4)) + 0.5)
    rows[:, -3] = -rows[:, 0]
    rows[:, -2:] = 0
    w[large] = rows
    return w.bfloat16().cuda()


def states(N, d, seed):
    h = torch.ones(N, d)
    h[:, -1] = 0.25 * (1 + torch.arange(N) % 3)
    h[:, -2] = torch.randn(N, generator=torch.Generator().manual_seed(seed))
    return h.bfloat16().cuda()


@pytest.mark.parametrize('N', [3, 20, 300, 1500])
@pytest.mark.parametrize('V,d', [(300, 64), (1500, 264), (5003, 768), (33001, 256), (50304, 768)])
def test_large_rows_that_cancel(cuda, N, V, d):
    large = torch.arange(0, V, max(1, V // 100))[:100]
    w, h = weight(V, d, large, 1), states(N, d, 2)
    for top in (1, 5, 20):
        check(h, w, None, top=top, grads=False)
        check(h, w, targets(N, V, 3, 5), tau=0.8, top=top, grads=False)


@pytest.mark.parametrize('N', [4, 40, 700])
def test_one_large_row(cuda, N):
    """Where most rows answer from the scores as they are, one row that the sums know least of."""
    V, d = 5003, 768
    for at in (0, 31, 2500, V - 1):
        w, h = weight(V, d, torch.tensor([at]), 4), states(N, d, 5)
        for value in (0.0, 0.5, -1.0, -8.0, 8.0):
            w[at, -1] = value
            check(h, w, None, top=8, grads=False)
            check(h, w, torch.full((N,), at, device='cuda'), top=8, grads=False)


def test_values_out_of_the_range_of_squares(cuda):
    """Sizes whose squares fp32 does not hold, rows of infinities beside them, states of zeros."""
    V, d = 1200, 72
    for N in (5, 200):
        for big, small in ((2.0 ** 70, 2.0 ** -70), (2.0 ** -80, 2.0 ** 60), (2.0 ** 65, 2.0 ** -66), (2.0 ** -75, 2.0 ** -40)):
            h, w = rand((N, d), 6, small), rand((V, d), 7, big)
            w[600:640] = 0
            h[0] = 0
            check(h, w, None, top=6, grads=False)
        h, w = rand((N, d), 8).abs(), rand((V, d), 9, 0.1)
        keep = torch.arange(V, device='cuda') % 3 > 0
        w[~keep] = -float('inf')                                # ruled out
        import asrn_b200 as asrn
        r = asrn.head_stats(h, w, top=9)
        want = (h.double() @ torch.where(keep[:, None], w, 0).double().t()).masked_fill(~keep, -float('inf'))
        assert torch.equal(r.top_tokens, want.sort(dim=1, descending=True, stable=True).indices[:, :9])

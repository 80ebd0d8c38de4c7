"""layer_norm at widths below a vector of eight, whose rows share vectors with several neighbours, and linear at the ends of its
widths. The bounds are those of test_norm_linear_gpu.py."""
import pytest
import torch

from test_norm_linear_gpu import BF16, F32, check_linear, check_norm, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('d', range(1, 16))
@pytest.mark.parametrize('N', [1, 2, 3, 8, 119, 5001])
def test_narrow_rows(cuda, N, d):
    for x, res in ((F32, None), (BF16, None), (BF16, F32), (F32, BF16)):
        check_norm(rand((N, d), 1, dtype=x, shift=0.5), rand((d,), 2, 0.3, F32, 1.0), rand((d,), 3, dtype=F32),
                   None if res is None else rand((N, d), 4, 2.0, res), BF16 if res else F32)


@pytest.mark.parametrize('N,d,n', [(1, 65536, 8), (40, 65536, 16), (600, 32768, 8), (1, 8, 1 << 20), (20, 8, 1 << 18), (70001, 8, 8),
                                   (513, 8, 4104)])
def test_widths_at_the_ends(cuda, N, d, n):
    for act, res in ((None, F32), ('gelu', None)):
        check_linear(rand((N, d), 5), rand((n, d), 6, d ** -0.5), rand((n,), 7), act,
                     None if res is None else rand((N, n), 8, dtype=res))

"""Which operators the tuning example trains with: with --fused linear, without it the MLP that keeps its activations in 8 bits."""
import os

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('fused', [True, False])
def test_operators_of_the_example(cuda, fused, monkeypatch):
    import torch
    import asrn_b200.model as model
    monkeypatch.syspath_prepend(os.path.join(ROOT, 'examples'))
    import preference_tuning
    calls = dict(linear=0, mlp8=0, layer_norm=0)

    def counted(name):
        f = getattr(model, name)

        def call(x, *args, **options):
            y = f(x, *args, **options)
            calls[name] += (y[0] if isinstance(y, tuple) else y).requires_grad and torch.is_grad_enabled()
            return y
        monkeypatch.setattr(model, name, call)
    for name in calls:
        counted(name)
    preference_tuning.main(['--pairs', '2', '--length', '33', '--steps', '2'] + ['--fused'] * fused)
    assert (calls['linear'] > 0) == (calls['layer_norm'] > 0) == fused and (calls['mlp8'] > 0) == (not fused)

"""The fine-tuning operators (asrn_b200.finetune) at their edges: sizes, values and calls that the tests by operator
(test_finetune_gpu.py, whose references and bounds these use) do not reach."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# ---- losses -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('rows', [1024, 1025, 2000])
def test_losses_of_many_sequences_without_positions(cuda, rows):
    """More rows than one block keeps, and no positions at all: zeros."""
    import asrn_b200 as asrn
    e = torch.zeros(rows, 0, device='cuda')
    for adv in (torch.ones(rows, device='cuda'), e):
        for per in ('token', 'sequence'):
            for ref in (None, e):
                r = asrn.policy_loss(e, e, adv, e.bool(), ref_logp=ref, kl=0.0 if ref is None else 0.1, per=per)
                assert r.grad.shape == (rows, 0)
                assert float(r.loss) == 0 and float(r.kl) == 0 and float(r.clipped) == 0
    e = torch.zeros(2, rows, 0, device='cuda')
    r = asrn.preference_loss(e, e, e.bool())
    assert float(r.loss) == 0 and r.grad.shape == e.shape and (r.chosen == 0).all() and (r.rejected == 0).all()


def test_policy_without_sequences_and_with_a_reference(cuda):
    """An empty batch has no log probabilities of the reference model in memory either: not an error."""
    import asrn_b200 as asrn
    e = torch.zeros(0, 5, device='cuda')
    r = asrn.policy_loss(e, e, e[:, 0], e.bool(), ref_logp=e, kl=0.1)
    assert float(r.loss) == 0 and float(r.kl) == 0 and r.grad.shape == (0, 5)

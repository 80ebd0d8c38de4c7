"""The fine-tuning operators at the model's edges, as far as they need no GPU."""
import pytest
import torch


def model(V=11, d=16):
    """A model whose state is given: what the fp32 log probabilities make of it."""
    import asrn_b200 as asrn
    m = asrn.create_model(V=V, d=d, n_capas=2, semilla=0)
    h = torch.randn(2, 5, d, generator=torch.Generator().manual_seed(1)).requires_grad_()
    m.estado = lambda x: h
    return m, h, torch.zeros(2, 5, dtype=torch.int64)


def test_fp32_logprobs_of_a_token_outside_the_vocabulary():
    """NaN, with a NaN gradient, as in bf16: torch's gather would fail on the host and stop the context on a GPU."""
    m, h, x = model()
    y = torch.tensor([[3, 10, 11, -1, 0], [1 << 40, -100, 2, 5, 9]])
    lp = m.logprobs(x, y)
    assert lp.isnan().tolist() == [[False, False, True, False, False], [True, False, False, False, False]]
    assert (lp[y < 0] == 0).all()
    want = torch.log_softmax(m.head(h), -1)
    for at in ((0, 0), (0, 1), (1, 4)):
        assert lp[at] == want[at][y[at]]
    lp.sum().backward()
    assert h.grad.isnan().any(-1).tolist() == lp.isnan().tolist()
    assert (h.grad[0, 3] == 0).all()


@pytest.mark.parametrize('tau', [0.0, -1.0, float('nan'), float('inf')])
def test_fp32_logprobs_refuse_what_bf16_refuses(tau):
    m, _, x = model()
    with pytest.raises(ValueError, match='temperatura'):
        m.logprobs(x, temperatura=tau)
    assert m.logprobs(x, temperatura=0.5).shape == x.shape


def test_checkpoint_takes_no_other_text():
    """A mistyped '8bits' turned nothing on and said nothing."""
    import asrn_b200 as asrn
    for text in ('8bit', '8 bits', 'fp8', ''):
        with pytest.raises(ValueError, match='checkpoint'):
            asrn.create_model(V=11, d=16, n_capas=2, checkpoint=text)
    for value in (False, True, None, 0, 1):
        assert asrn.create_model(V=11, d=16, n_capas=2, checkpoint=value).checkpoint is value


def test_a_loaded_model_can_keep_activations_in_8_bits(tmp_path):
    import asrn_b200 as asrn
    m = asrn.create_model(V=11, d=16, n_capas=2, semilla=0, checkpoint='8bits')
    asrn.save(m, str(tmp_path / 'm.pt'))
    load = lambda **kw: asrn.load(str(tmp_path / 'm.pt'), dispositivo='cpu', **kw)  # noqa: E731
    assert not any(b.activaciones_8bits for b in load().bloques)         # the file does not say
    back = load(checkpoint='8bits')
    assert back.checkpoint == '8bits' and all(b.activaciones_8bits for b in back.bloques)
    assert all(torch.equal(a, b) for a, b in zip(m.state_dict().values(), back.state_dict().values()))
    with pytest.raises(ValueError):
        load(checkpoint='8')


def test_a_block_pickled_without_the_8bit_setting_still_runs():
    import asrn_b200 as asrn
    blq = asrn.create_model(V=11, d=16, n_capas=2, semilla=0).bloques[0]
    h = torch.randn(2, 5, 16, generator=torch.Generator().manual_seed(3))
    want = blq(h)
    vars(blq).pop('activaciones_8bits', None)
    assert torch.equal(blq(h), want)

"""ModeloASRN.stats where it goes by the logits (fp32 models, heads that were replaced), on the CPU with given states: the ranking
goes by the scores."""
import torch


def model(h, weight):
    import asrn_b200 as asrn
    m = asrn.create_model(V=weight.shape[0], d=weight.shape[1], n_capas=2)
    m.head = torch.nn.Linear(weight.shape[1], weight.shape[0], bias=False)
    with torch.no_grad():
        m.head.weight.copy_(weight)
    m.estado = lambda x: h
    return m


def rand(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def test_scores_whose_log_probabilities_round_to_one_value():
    """At a high temperature all log probabilities are all but equal; and score differences below an ulp of the log probability."""
    x, h, w = torch.zeros(2, 3, dtype=torch.int64), rand(2, 3, 16, seed=1), rand(200, 16, seed=2)
    for scale, tau in ((1.0, 1e7), (1.0, 1e30), (1e-5, 1.0)):
        m = model(h * scale, w)
        with torch.no_grad():
            z = m.head(h * scale)
            r = m.stats(x, temperatura=tau, top=20)
        want = z.sort(dim=-1, descending=True, stable=True).indices[..., :20]
        lp = torch.log_softmax(z / tau, -1)
        assert len(lp[0, 0].unique()) < 200                     # some are equal
        assert torch.equal(r.top_tokens, want)
        assert torch.equal(r.top_logp, lp.gather(-1, want))


def test_equal_scores_come_in_the_order_of_their_numbers():
    h, w = rand(1, 2, 16, seed=3), rand(50, 16, seed=4)
    w[25:] = w[:25]
    r = model(h, w).stats(torch.zeros(1, 2, dtype=torch.int64), top=8)
    assert (r.top_tokens[..., 1::2] == r.top_tokens[..., ::2] + 25).all()

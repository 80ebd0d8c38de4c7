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


def test_positions_left_out_reach_no_gradient():
    """A state that is not finite, at a position without a target."""
    h, w, y = rand(2, 3, 16, seed=5), rand(40, 16, seed=6), torch.arange(6).view(2, 3)
    y[0, 1] = -1
    grads = []
    for bad in (0.0, float('nan'), float('inf')):
        t = h.clone()
        t[0, 1, 3] = bad
        t.requires_grad_()
        m = model(t, w)
        r = m.stats(torch.zeros(2, 3, dtype=torch.int64), y, temperatura=0.7, top=2)
        assert r.logp[0, 1] == 0 and r.entropy[0, 1] == 0 and (r.top_tokens[0, 1] == -1).all() and (r.top_logp[0, 1] == 0).all()
        grads.append(torch.autograd.grad((r.logp.sum() + r.entropy.square().sum()), (t, m.head.weight)))
    for dh, dw in grads[1:]:
        assert torch.equal(dh, grads[0][0]) and torch.equal(dw, grads[0][1]) and (dh[0, 1] == 0).all()

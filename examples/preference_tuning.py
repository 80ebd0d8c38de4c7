"""Preference tuning, then policy tuning, of a small ASRN model on synthetic answers, with everything asrn_b200 has for
it: log probabilities through the tied head (model.logprobs), the preference and the clipped policy loss, and local
blocks that keep their activations in 8 bits (checkpoint='8bits').

    python examples/preference_tuning.py [--V 256 --d 64 --pairs 8 --length 128 --steps 20]

The prompts are random; a chosen answer repeats its prompt, a rejected one is random. In the second part answers are
drawn from the model itself and rewarded for each token that the prompt holds.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), '..'))
import asrn_b200 as asrn  # noqa: E402


def pairs(P, L, V, seed):
    """Token rows (2 P, L), the chosen answers first, and the targets: each position's next token within the answer."""
    g = torch.Generator().manual_seed(seed)
    prompt = torch.randint(0, V, (P, L // 2), generator=g)
    other = torch.randint(0, V, (P, L - L // 2), generator=g)
    chosen = torch.cat([prompt, prompt[:, :1].expand(-1, L % 2), prompt], 1)[:, :L]
    x = torch.cat([chosen, torch.cat([prompt, other], 1)]).cuda()
    targets = torch.nn.functional.pad(x[:, 1:], (0, 1), value=-1)
    targets[:, :L // 2 - 1] = -1
    return x, targets


def preference_steps(model, optimiser, x, targets, steps):
    mask = (targets >= 0).view(2, -1, x.shape[1])
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        ref = model.logprobs(x, targets).view(mask.shape)
    losses = []
    for _ in range(steps):
        with torch.autocast('cuda', dtype=torch.bfloat16):
            logp = model.logprobs(x, targets).view(mask.shape)
        r = asrn.preference_loss(logp.detach(), ref, mask, beta=0.1)
        optimiser.zero_grad(set_to_none=True)
        logp.backward(r.grad)
        optimiser.step()
        losses.append(r.loss)
    return torch.stack(losses).tolist(), float((r.chosen - r.rejected).mean())


def policy_steps(model, optimiser, prompt, answers, steps):
    """One rollout, `steps` updates on it: the reward is the share of the answer's tokens that the prompt holds."""
    L0 = prompt.shape[1]
    model.eval()
    with torch.autocast('cuda', dtype=torch.bfloat16):
        rows, _ = asrn.generate(model, prompt, n_nuevos=answers, temperatura=1.0, top_k=0, conservar_cita=False,
                                devolver_logits=False)
    model.train()
    x = rows.cuda()
    reward = (x[:, L0:, None] == x[:, None, :L0]).any(2).float().mean(1)
    advantages = (reward - reward.mean()) / (reward.std() + 1e-6)
    targets = torch.nn.functional.pad(x[:, 1:], (0, 1), value=-1)
    targets[:, :L0 - 1] = -1
    mask = targets >= 0
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        old = model.logprobs(x, targets)
    losses = []
    for _ in range(steps):
        with torch.autocast('cuda', dtype=torch.bfloat16):
            logp = model.logprobs(x, targets)
        r = asrn.policy_loss(logp.detach(), old, advantages, mask, ref_logp=old, kl=0.04)
        optimiser.zero_grad(set_to_none=True)
        logp.backward(r.grad)
        optimiser.step()
        losses.append(r.loss)
    return torch.stack(losses).tolist(), float(r.kl)


def main(argv=None):
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument('--V', type=int, default=256)
    a.add_argument('--d', type=int, default=64)
    a.add_argument('--layers', type=int, default=4)
    a.add_argument('--pairs', type=int, default=8)
    a.add_argument('--length', type=int, default=128)
    a.add_argument('--steps', type=int, default=20)
    a = a.parse_args(argv)
    model = asrn.create_model(V=a.V, d=a.d, n_capas=a.layers, semilla=0, checkpoint='8bits').cuda().train()
    optimiser = torch.optim.Adam(model.parameters(), lr=1e-3)
    x, targets = pairs(a.pairs, a.length, a.V, seed=0)
    pref, margin = preference_steps(model, optimiser, x, targets, a.steps)
    print(f'preference loss {pref[0]:.4f} -> {pref[-1]:.4f}, reward margin {margin:.3f}')
    policy, kl = policy_steps(model, optimiser, x[:a.pairs, :a.length // 2], a.length // 2, a.steps)
    print(f'policy loss {policy[0]:.4f} -> {policy[-1]:.4f}, KL {kl:.4f}')
    return pref, policy


if __name__ == '__main__':
    main()

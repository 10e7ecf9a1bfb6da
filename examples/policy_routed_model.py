"""A model with routed experts learns by policy gradient.

Each token's features go to the k best of its experts (device.top_entries on the router's scores); device.group_entries, gated_experts and
combine_experts are the experts' feed-forward blocks and the sum of their outputs; device.log_probs scores the answers that were
sampled and gives the entropies.  log_probs_grad, combine_experts_grad and gated_experts_grad are the way back; what lies between them are
ordinary products.  An answer is rewarded if it is the features' own token.

    python examples/policy_routed_model.py [steps]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from comet_b200 import device  # noqa: E402


def parameters(width, inner, experts, vocabulary, generator, kind=torch.bfloat16):
    normal = lambda *shape: torch.randn(shape, generator=generator, device="cuda")              # noqa: E731
    return {"router": normal(width, experts) * width ** -0.5, "w": (normal(experts, 2 * inner, width) * width ** -0.5).to(kind),
            "v": (normal(experts, width, inner) * 0.5 * inner ** -0.5).to(kind), "head": (normal(vocabulary, width) * 0.5 * width ** -0.5).to(kind)}


def forward(p, x, chosen):
    """The logits, and what the way back takes."""
    scores = x.float() @ p["router"]
    choices, _ = device.top_entries(scores, chosen)
    gate = torch.softmax(scores.gather(1, choices.crd.view(-1, chosen)), 1)
    groups = device.group_entries(device.DeviceCSR(choices.nrows, choices.ncols, choices.pos, choices.crd, gate.reshape(-1)))
    h = device.gated_experts(groups, x, p["w"])
    hidden = x + device.combine_experts(groups, h, p["v"])
    return hidden @ p["head"].t(), (gate, groups, h, hidden)


def gradients(p, x, kept, logits, answers, advantage, bonus, scale=1.0):
    """Of scale times the mean over tokens of -(advantage * log probability of the answer) - bonus * entropy.  The logits are overwritten."""
    gate, groups, h, hidden = kept
    n = x.shape[0]
    given = device.DeviceCSR(n, logits.shape[1], torch.arange(n + 1, device="cuda"), answers, None)
    values, sums, entropy, _ = device.log_probs(given, logits, entropy=True)
    d_logits = device.log_probs_grad(given, logits, sums, advantage * (-scale / n), entropy=entropy, d_entropy=torch.full_like(entropy, -bonus * scale / n), grad=logits)
    d_hidden = d_logits @ p["head"]
    d_h, d_v, d_gate = device.combine_experts_grad(groups, h, p["v"], d_hidden)
    _, d_w = device.gated_experts_grad(groups, x, p["w"], d_h, grad_x=False)
    d_gate = d_gate.view_as(gate)
    d_chosen = gate * (d_gate - (gate * d_gate).sum(1, keepdim=True))
    d_scores = torch.zeros(n, groups.S.ncols, device="cuda").scatter_(1, groups.S.crd.view_as(gate), d_chosen)
    return {"router": x.float().t() @ d_scores, "w": d_w, "v": d_v, "head": d_logits.t() @ hidden}, values, entropy


def train(steps=80, tokens=512, width=64, inner=64, vocabulary=40, experts=8, chosen=2, rate=0.4, bonus=0.01, seed=0):
    """The mean reward and the mean entropy of each step."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    p = parameters(width, inner, experts, vocabulary, g)
    features = torch.randn(vocabulary, width, generator=g, device="cuda")
    history = []
    for _ in range(steps):
        wanted = torch.randint(vocabulary, (tokens,), generator=g, device="cuda")
        x = (features[wanted] + 0.3 * torch.randn(tokens, width, generator=g, device="cuda")).bfloat16()
        logits, kept = forward(p, x, chosen)
        answers = torch.multinomial(torch.softmax(logits.float(), 1), 1, generator=g).view(-1)
        reward = (answers == wanted).float()
        d, _, entropy = gradients(p, x, kept, logits, answers, reward - reward.mean(), bonus)
        for name in p:
            step = d[name].float()
            p[name] = (p[name].float() - rate * step / (step.norm() + 1e-6)).to(p[name].dtype)
        kept[1].check()
        history.append((float(reward.mean()), float(entropy.mean())))
    return history


if __name__ == "__main__":
    history = train(int(sys.argv[1]) if len(sys.argv) > 1 else 80)
    for i, (reward, entropy) in list(enumerate(history))[::10] + [(len(history) - 1, history[-1])]:
        print("step %3d  reward %.3f  entropy %.3f" % (i, reward, entropy))

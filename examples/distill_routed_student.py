"""A student with routed experts learns from a teacher's top logits.

The teacher is a fixed linear map to a vocabulary; device.top_entries keeps the largest of its logits as a CSR matrix, with the sum that
they are a part of.  The student sends each token to the k best of its experts (device.top_entries again, on the router's logits),
device.distill_loss compares its logits with the teacher's list, device.balance_loss keeps the experts in use; both give
gradients of the logits, from which the layers' own are ordinary products.

    python examples/distill_routed_student.py [steps]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from comet_b200 import device  # noqa: E402


def train(steps=60, tokens=512, width=64, vocabulary=1031, experts=8, chosen=2, listed=16, rate=5.0, seed=0):
    """The losses of each step as (distillation, balance) and the last step's tokens per expert."""
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")          # noqa: E731
    teacher = normal(width, vocabulary) * (3 / width ** 0.5)
    router = (normal(width, experts) * 0.1).requires_grad_()
    expert = (normal(experts, width, width) / width ** 0.5).requires_grad_()
    head = torch.zeros(width, vocabulary, device="cuda", requires_grad=True)
    x = normal(tokens, width)
    lists, lse = device.top_entries(x @ teacher, listed, lse=True)
    history = []
    for _ in range(steps):
        scores = x @ router
        choices, _ = device.top_entries(scores.detach(), chosen)
        column = choices.crd.view(tokens, chosen)
        gate = torch.softmax(scores.gather(1, column), 1)
        hidden = torch.einsum("tk,tkd->td", gate, torch.einsum("ti,tkid->tkd", x, expert[column]))
        logits = hidden @ head
        loss, _, d_logits = device.distill_loss(lists, logits.detach(), lse=lse, scale=1 / tokens)
        balance, counts, d_scores = device.balance_loss(choices, scores.detach(), scale=0.01)
        torch.autograd.backward([logits, scores], [d_logits, d_scores])
        with torch.no_grad():
            for p in (router, expert, head):
                p -= rate * p.grad
                p.grad = None
        history.append((float(loss), float(balance)))
    return history, counts[0].tolist()


if __name__ == "__main__":
    history, counts = train(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
    for i, (loss, balance) in list(enumerate(history))[::10] + [(len(history) - 1, history[-1])]:
        print("step %3d  distillation %.4f  balance %.5f" % (i, loss, balance))
    print("tokens per expert:", counts)

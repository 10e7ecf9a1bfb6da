"""The operators together, as examples/policy_routed_model.py uses them: router, experts' blocks, log probabilities, and all the way back."""
import importlib.util
import math
import os

import pytest

pytestmark = pytest.mark.gpu


def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "policy_routed_model.py")
    spec = importlib.util.spec_from_file_location("policy_routed_model", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("tokens,chosen", [(1, 2), (37, 2), (900, 3)])
def test_gradients_of_the_whole_model(tokens, chosen):
    """Against automatic differentiation in 64 bits of the same model, with the choices that were made.

    In f16 a rounding is off by 2^-11 of a value.  On the way to any gradient there are at most twelve of them (H, Y, hidden, logits; the gradients of the logits,
    of hidden, of H, dz, val H, and the results), each of a tensor whose own share in the gradient's norm is not above three times the gradient's (products with
    matrices of independent entries keep norms; the residual path and the softmax's difference of two terms give the factor): 12 x 3 x 2^-11 = 1.8e-2 of the norm."""
    import torch
    e = example()
    g = torch.Generator("cuda")
    g.manual_seed(tokens)
    width, inner, experts, vocabulary, bonus, scale = 72, 56, 6, 1009, 0.05, 4096.0
    p = e.parameters(width, inner, experts, vocabulary, g, kind=torch.float16)
    x = torch.randn(tokens, width, generator=g, device="cuda").half()
    answers = torch.randint(vocabulary, (tokens,), generator=g, device="cuda")
    advantage = torch.randn(tokens, generator=g, device="cuda")
    logits, kept = e.forward(p, x, chosen)
    column = kept[1].S.crd.view(tokens, chosen)
    want = {k: v.double().requires_grad_() for k, v in p.items()}
    xd = x.double()
    gate = torch.softmax((xd @ want["router"]).gather(1, column), 1)
    z = torch.einsum("nd,nkfd->nkf", xd, want["w"][column])
    h = torch.nn.functional.silu(z[..., :inner]) * z[..., inner:]
    hidden = xd + torch.einsum("nk,nkf,nkdf->nd", gate, h, want["v"][column])
    logq = torch.log_softmax(hidden @ want["head"].t(), 1)
    entropy = -(logq.exp() * logq).sum(1)
    value = logq.gather(1, answers[:, None])[:, 0]
    (scale * (-(advantage.double() * value) - bonus * entropy).mean()).backward()
    assert float((logits.double() - hidden @ want["head"].t()).norm() / (hidden @ want["head"].t()).norm()) < 12 * 3 * 2.0 ** -11
    got, values, ent = e.gradients(p, x, kept, logits, answers, advantage, bonus, scale)
    # absolute errors of logits of a few units, 2^-11 each
    assert float((values.double() - value).abs().max()) < 0.05 and float((ent.double() - entropy).abs().max()) < 0.05
    for name, d in got.items():
        assert float((d.double() - want[name].grad).norm() / want[name].grad.norm()) < 12 * 3 * 2.0 ** -11, name
    kept[1].check()


def test_the_example_runs():
    history = example().train(steps=3, tokens=64)
    assert len(history) == 3 and all(math.isfinite(v) for h in history for v in h)

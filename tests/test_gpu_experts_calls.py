"""Calls of a router's experts at the ends of what is allowed, against the definitions in 64 bits (tests/test_gpu_experts.py has the oracle and its bounds)."""
import numpy as np
import pytest

from tests.test_gpu_experts import Oracle, close, matrix

pytestmark = pytest.mark.gpu


def test_one_expert_with_half_a_billion_entries():
    """A sum over an expert's tokens that takes longer than any other wait may: 7.8 million steps in one tile.  All but a few entries have a gradient of 0."""
    import torch
    from comet_b200 import device
    n, few = 500_000_000, [0, 1, 250_000_000, 499_999_900, 499_999_999]
    rng = np.random.default_rng(1)
    W, x, d = matrix(rng, "bf16", 1, 16, 8), matrix(rng, "bf16", len(few), 8), matrix(rng, "bf16", len(few), 8)
    at = torch.tensor(few, device="cuda")
    X, dH = torch.ones((n, 8), dtype=torch.bfloat16, device="cuda"), torch.zeros((n, 8), dtype=torch.bfloat16, device="cuda")
    X[at], dH[at] = x, d
    S = device.DeviceCSR(n, 1, torch.arange(n + 1, device="cuda"), torch.zeros(n, dtype=torch.int64, device="cuda"), None)
    G = device.group_entries(S)
    dX, dW = device.gated_experts_grad(G, X, W, dH, grad_x=False)
    G.check()
    small = device.DeviceCSR(len(few), 1, torch.arange(len(few) + 1), torch.zeros(len(few), dtype=torch.int64), torch.ones(len(few)))
    _, _, dw, ow = Oracle(small, None, np.zeros(len(few), np.int64), np.arange(len(few)), "bf16").gated_grad(x, W, d)
    assert dX is None
    close(dW, dw, ow, "bf16")
    del X, dH, S, G
    torch.cuda.empty_cache()

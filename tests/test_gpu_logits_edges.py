"""Operators on rows of logits at the ends of their ranges: logits and temperatures whose quotient is large, lists that leave nothing or
claim too much, sums of infinity, float64 teachers, gradients in place.  Tolerances and the 64-bit definitions are those of
test_gpu_logits.py; where a test has one of its own, it says what it is made of.
"""
import math

import numpy as np
import pytest

from tests.test_gpu_logits import TOL, csr, distill, log_sum_exp, logits, teacher

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tau", [1.0, 0.7, 2.0])
@pytest.mark.parametrize("near", [8.0, 30.0])
def test_distill_probabilities_beside_a_large_sum(near, tau):
    """64 entries around `near` that leave 1e-4 of the sum.  Where the student gives the listed columns nothing, a gradient there is -p: the
    exponential's two units in the last place (2^-22), its argument's residue, two products and a difference (2^-24 each) are 2^-21 of it
    at most.  The sum of 64 p adds eight roundings: 2^-22 + 8 2^-24 < 2^-20 for the rest that is left, and for each term of a loss."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(int(near * 10 + tau * 100))
    n, cols, k = 200, 3001, 64
    S, pos, crd, val = teacher(rng, n, cols, k, False)
    val = (val - 6 + near).astype(np.float32).astype(np.float64)
    S, pos = csr(n, cols, np.full(n, k), crd, val)
    lse = np.array([log_sum_exp(val[a:b] / tau) for a, b in zip(pos, pos[1:])]) - math.log(1 - 1e-4)
    lse = lse.astype(np.float32)
    x = torch.from_numpy(rng.normal(0, 1, (n, cols)).astype(np.float32))
    x[torch.arange(n).repeat_interleave(k), torch.from_numpy(crd)] = -60.0 * tau
    x64 = x.double().numpy()
    _, rows, grad = device.distill_loss(S, x.cuda(), temperature=tau, lse=torch.from_numpy(lse).cuda(), scale=tau)
    p = np.exp(val / tau - np.repeat(lse.astype(np.float64), k))
    got = -grad.double().cpu().numpy()[np.repeat(np.arange(n), k), crd]
    assert (np.abs(got - p) <= 2.0 ** -21 * p + 1e-20).all()
    wrows, _, _, _, roff = distill(pos, crd, val, x64, tau, lse)
    assert (np.abs(rows.double().cpu().numpy() - wrows) <= 2.0 ** -20 / TOL * roff).all()

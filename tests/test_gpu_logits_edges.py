"""Operators on rows of logits at the ends of their ranges: logits and temperatures whose quotient is large, lists that leave nothing or
claim too much, sums of infinity, float64 teachers, gradients in place.  Tolerances and the 64-bit definitions are those of
test_gpu_logits.py; where a test has one of its own, it says what it is made of.
"""
import math

import numpy as np
import pytest

from tests.test_gpu_logits import TOL, close_gradient, csr, distill, log_sum_exp, logits, teacher

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


def test_distill_float64_teachers_keep_their_digits():
    """Values whose differences are lost in f32, and values beyond it.  Gradients are scaled by the temperature: a q below 2^-126 is 0, and LEAST is
    of that size."""
    rng = np.random.default_rng(21)
    x, x64 = logits(rng, 40, 3001, "f32")
    S, pos, crd, val = teacher(rng, 40, 3001, 20, True, np.float64)
    for shift, tau in ((1e8, 1.0), (-1e8, 0.5), (1e12, 0.01), (1e8, 1e-3)):
        more = np.round((val + shift) * 2 ** 10) / 2 ** 10
        S, pos = csr(40, 3001, np.diff(pos), crd, more, np.float64)
        less = more - shift                                            # exact: the shift is no part of the probabilities
        wrows, _, wgrad, off, roff = distill(pos, crd, less, x64, tau, scale=tau)
        check_float64(S, x, tau, wrows, wgrad, off, roff)
    S, pos = csr(2, 3001, [3, 2], [5, 6, 9, 0, 3000], [1e300, 1e300, 5e299, -1e300, -2e300], np.float64)
    wrows, _, wgrad, off, roff = distill(pos, np.array([5, 6, 9, 0, 3000]), np.array([0.0, 0.0, -1e30, 0.0, -1e30]), x64[:2])
    check_float64(S, x[:2], 1.0, wrows, wgrad, off, roff)


def check_float64(S, x, tau, wrows, wgrad, off, roff):
    from comet_b200 import device
    _, rows, grad = device.distill_loss(S, x, temperature=tau, scale=tau)
    assert (np.abs(rows.double().cpu().numpy() - wrows) <= roff).all()
    close_gradient(grad, wgrad, off, "f32")

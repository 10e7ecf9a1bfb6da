"""Operators on rows of logits at the ends of their ranges: logits and temperatures whose quotient is large, lists that leave nothing or
claim too much, sums of infinity, float64 teachers, gradients in place.  Tolerances and the 64-bit definitions are those of
test_gpu_logits.py; where a test has one of its own, it says what it is made of.
"""
import math

import numpy as np
import pytest

from tests.test_gpu_logits import (TOL, TYPES, check_balance, check_top, choices, close_gradient, csr, distill, log_softmax, log_sum_exp, logits,
                                   teacher, torch_type)

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


def large_quotients(kind, cols):
    """Rows of one large value, of one above all, of two values, and of neighbours of 18.125: (CUDA tensor, the same values in f64)."""
    import torch
    rng = np.random.default_rng(cols)
    most = {"bf16": 1e20, "f32": 1e20, "f16": 6e4}[kind]
    rows = [np.full(cols, s * v) for v in (1e9, 1e10, 1e20) if v <= most for s in (1, -1)]
    rows += [np.where(np.arange(cols) == cols // 2, b, 1.5 * b if b < 0 else 0.5 * b) for b in (-most / 2, most / 2)]
    rows += [np.where(rng.random(cols) < 0.5, b, 1.5 * b if b < 0 else 0.5 * b) for b in (-most / 2, most / 2, 18.125, -18.125)]
    unit = {"bf16": 2.0 ** -3, "f16": 2.0 ** -6, "f32": 2.0 ** -19}[kind]               # the spacing of the type at 18
    rows += [18.125 + unit * rng.integers(0, 4, cols), -18.125 - unit * rng.integers(0, 4, cols),
             18.125 + unit * (np.arange(cols) * 8 // cols)]                             # each CTA's part has a maximum of its own
    x = torch.from_numpy(np.array(rows, np.float64)).float().to(torch_type(kind))
    return x.cuda(), x.double().numpy()


# 18.125 log2(e) over the temperature lies at 2^22 and on both sides of it
BESIDE = [v * math.log2(math.e) / 2 ** 22 for v in (18.125, 18.126, 18.124)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [300, 9001, 131072])
def test_distill_large_quotients(cols, kind):
    x, x64 = large_quotients(kind, cols)
    rng = np.random.default_rng(cols + 1)
    S, pos, crd, val = teacher(rng, len(x64), cols, 12, False)
    for tau in [1.0, 1e-7, 1e-9] + BESIDE:
        check_quotients(S, pos, crd, val, x, x64, kind, tau)
    for tau in [1.0] + BESIDE:                                         # a sum of 10^8 has no digits behind the point
        check_quotients(S, pos, crd, val, x, x64, kind, tau, np.array([log_sum_exp(val[a:b] / tau) + 0.3 for a, b in zip(pos, pos[1:])], np.float32))


def check_quotients(S, pos, crd, val, x, x64, kind, tau, lse=None):
    """As check_distill.  Where what is not listed is below f32's range, a loss with a sum is infinite: more than 0.2 (87 - 1) it has to be."""
    import torch
    from comet_b200 import device
    _, rows, grad = device.distill_loss(S, x, temperature=tau, lse=None if lse is None else torch.from_numpy(lse).cuda(), scale=tau)
    wrows, _, wgrad, off, roff = distill(pos, crd, val, x64, tau, lse, None, tau)
    got = rows.double().cpu().numpy()
    assert not np.isnan(got).any() and not grad.isnan().any()
    far = np.isposinf(got)
    assert (wrows[far] > 17).all() and not (far.any() and lse is None)
    assert (np.abs(got - wrows)[~far] <= roff[~far]).all()
    close_gradient(grad[torch.from_numpy(~far).cuda()], wgrad[~far], off[~far], kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [300, 9001, 131072])
def test_top_entries_sums_of_large_quotients(cols, kind):
    x, x64 = large_quotients(kind, cols)
    for tau in [1.0, 1e-7, 1e-9] + BESIDE:
        check_top(x, x64, 5, tau)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols,k,near", [(1, 1, 0.0), (64, 64, 0.0), (64, 64, 30.0), (700, 700, -20.0), (1024, 1024, 5.0), (5000, 40, 10.0)])
@pytest.mark.parametrize("tau", [1.0, 0.7])
def test_distill_complete_lists(cols, k, near, tau, kind):
    """The teacher lists all that it gives any probability, and the student has none elsewhere: what the list's sum lacks of 1 is rounding.  The sum is
    off by less than TOL, and so is each p beside the teacher's own: twice the tolerance of a list without a sum."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(cols + k)
    n = 300
    t, t64 = logits(rng, n, cols, "f32")
    t += near
    x, _ = logits(rng, n, cols, kind)
    if k < cols:
        hidden = torch.ones((n, cols), dtype=torch.bool)
        hidden.scatter_(1, torch.from_numpy(np.argsort(rng.random((n, cols)), 1)[:, :k].copy()), False)
        t[hidden.cuda()] = -math.inf
        x[hidden.cuda()] = -math.inf
    S, lse = device.top_entries(t, k, temperature=tau, lse=True)
    loss, rows, grad = device.distill_loss(S, x, temperature=tau, lse=lse)
    crd, val = S.crd.cpu().numpy(), S.val.double().cpu().numpy()
    wrows, wloss, wgrad, off, roff = distill(np.arange(n + 1) * k, crd, val, x.double().cpu().numpy(), tau)
    assert (np.abs(rows.double().cpu().numpy() - wrows) <= 2 * roff).all()
    assert math.isfinite(float(loss))
    close_gradient(grad, wgrad, 2 * off, kind)


def test_distill_a_rest_that_the_student_cannot_have():
    """A complete list whose sum lacks more than rounding: the rest has a probability, and the student gives it none."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(22)
    x, x64 = logits(rng, 3, 40, "f32")
    S, lse = device.top_entries(x + 1, 40, lse=True)
    lse += torch.tensor([0.0, 0.001, 0.4], device="cuda")
    loss, rows, grad = device.distill_loss(S, x, lse=lse)
    assert abs(float(rows[0])) < TOL * 30 and rows[1] == math.inf and rows[2] == math.inf and loss == math.inf
    assert not grad.isnan().any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols,less", [(40, 0.3), (9001, 0.01), (131072, 2.0)])
def test_distill_lists_above_their_sum(cols, less, kind):
    """A list whose probabilities add up to more than 1: nothing is left, and the gradient is that of sum p (log p - log q), (sum p) q - p."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(cols)
    x, x64 = logits(rng, 6, cols, kind)
    S, pos, crd, val = teacher(rng, 6, cols, 9, False)
    for tau in (1.0, 2.0):
        lse = np.array([log_sum_exp(val[a:b] / tau) - less for a, b in zip(pos, pos[1:])], np.float32)
        loss, rows, grad = device.distill_loss(S, x, temperature=tau, lse=torch.from_numpy(lse).cuda(), scale=64.0)
        wrows, wgrad, off, roff = np.zeros(6), np.zeros_like(x64), np.zeros_like(x64), np.zeros(6)
        for t in range(6):
            at = slice(pos[t], pos[t + 1])
            logq = log_softmax(x64[t] / tau)
            logp = val[at] / tau - float(lse[t])
            p = np.exp(logp)
            wrows[t] = (p * (logp - logq[crd[at]])).sum()
            roff[t] = TOL * p.sum() * (1 + np.abs(logp).max() + np.abs(logq[crd[at]]).max())
            wgrad[t], off[t] = p.sum() * np.exp(logq), 2 * p.sum() * np.exp(logq)      # the sum is off by TOL too
            wgrad[t, crd[at]] -= p
            off[t, crd[at]] += p
        assert (np.abs(rows.double().cpu().numpy() - wrows) <= roff).all()
        close_gradient(grad, wgrad * 64 / tau, TOL * off * 64 / tau, kind)


@pytest.mark.parametrize("listed", [7, 40])
def test_distill_gradient_of_lists_above_their_sum_against_differences(listed):
    """Central differences with h = 1/16: the third derivative of (sum p) log sum exp is below 0.1 e^0.4, so h^2 / 6 times it is below 1e-4; two losses below
    12 within 1e-6 of themselves, over 2 h, add 2e-4."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(23)
    x, _ = logits(rng, 1, 40, "f32", 1.0)
    S, pos, crd, val = teacher(rng, 1, 40, listed, False)
    lse = torch.tensor([log_sum_exp(val) - 0.4], dtype=torch.float32, device="cuda")
    grad = device.distill_loss(S, x, lse=lse)[2]
    h = 1 / 16
    for j in list(crd[:4]) + [0, 39, 20]:
        at = []
        for d in (h, -h):
            y = x.clone()
            y[0, j] += d
            at.append(float(device.distill_loss(S, y, lse=lse, grad=False)[0]))
        assert abs((at[0] - at[1]) / (2 * h) - float(grad[0, j])) < 3e-4


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols,k", [(5, 2), (64, 8), (300, 40), (900, 9), (9001, 20), (9001, 600), (131072, 8)])
def test_top_entries_sum_of_infinity(cols, k, kind):
    """The sum of a row with +inf is +inf, with NaN NaN."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(cols)
    x, _ = logits(rng, 8, cols, kind)
    for t, at in enumerate([(0,), (cols - 1,), (cols // 2, 1), (0, cols - 1), (3,)]):
        x[t, list(at)] = math.inf
    x[3, 1] = -math.inf
    x[4, 4 % cols] = math.nan
    x[5, :] = math.inf
    x[6, :] = -math.inf
    got = device.top_entries(x, k, lse=True)[1].cpu()
    assert (got[[0, 1, 2, 3, 5]] == math.inf).all() and got[4].isnan() and got[6] == -math.inf and got[7].isfinite()


def test_temperatures_that_are_refused():
    """1 / temperature has to be an f32 number; without a sum the entries' temperature is checked all the same."""
    import torch
    from comet_b200 import _lib, device
    x = torch.zeros((4, 9), device="cuda")
    S, _ = csr(4, 9, [1, 1, 1, 1], [0, 1, 2, 3], [1, 1, 1, 1])
    for bad in (0.0, -1.0, math.nan, math.inf, 1e-39, 1e31):
        for call in (lambda: device.distill_loss(S, x, temperature=bad), lambda: device.top_entries(x, 2, temperature=bad, lse=True),
                     lambda: device.top_entries(x, 2, temperature=bad)):
            with pytest.raises(_lib.CometB200Error, match="temperature"):
                call()
    for good in (1e-37, 1e30):
        assert abs(float(device.distill_loss(S, x, temperature=good, scale=0.25)[0]) - math.log(9)) < TOL * 4
        assert abs(float(device.top_entries(x, 2, temperature=good, lse=True)[1][0]) - math.log(9)) < TOL * 4


def test_entry_points_without_a_temperature():
    """The C entry of top_entries takes no temperature where it gives no sum, and refuses its absence where it does."""
    import torch
    from comet_b200 import _lib, device
    x = torch.randn((3, 40), device="cuda")
    pos, crd = torch.empty(4, dtype=torch.int64, device="cuda"), torch.empty(6, dtype=torch.int64, device="cuda")
    val, lse = torch.empty(6, device="cuda"), torch.empty(3, device="cuda")
    call = lambda sums: device._call("comet_b200_dev_top_entries_f32_i64", 3, 40, x.data_ptr(), 40, 2, 0, pos.data_ptr(), crd.data_ptr(),  # noqa: E731
                                     val.data_ptr(), sums, device._stream())
    call(0)
    assert torch.equal(val.view(3, 2).sort(1).values, x.topk(2, 1).values.sort(1).values)
    with pytest.raises(_lib.CometB200Error, match="temperature"):
        call(lse.data_ptr())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols", [(9000, 8), (9000, 64), (3000, 256), (700, 1024), (9000, 9), (2000, 100)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_balance_in_place_beyond_one_cluster(rows, cols, scores, kind):
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows + cols)
    x, x64 = logits(rng, rows, cols, kind)
    S, pos, crd = choices(rng, rows, cols, min(cols, 4), True)
    seq = torch.tensor([0, rows // 3, rows // 3, rows], device="cuda")
    apart = device.balance_loss(S, x, seq=seq, scores=scores, scale=64.0)
    check_balance(S, pos, crd, x.clone(), x64, kind, seq.tolist(), None, scores, 64.0)
    loss, counts, grad = device.balance_loss(S, x, seq=seq, scores=scores, scale=64.0, grad=x)
    assert grad is x
    for a, b in zip(apart, (loss, counts, x)):
        assert torch.equal(a, b)


def test_gradients_in_place_are_seen_by_autograd():
    """Logits that a graph has saved and that a call overwrites: the backward pass refuses them, as after any operation in place."""
    import torch
    from comet_b200 import device
    S, _ = csr(4, 9, [1, 1, 1, 1], [0, 1, 2, 3], [1, 1, 1, 1])
    for op in (device.distill_loss, device.balance_loss):
        w = torch.randn((4, 9), device="cuda", requires_grad=True)
        y = w * 2
        z = (y * y).sum()
        op(S, y.detach(), grad=y.detach())
        with pytest.raises(RuntimeError, match="inplace"):
            z.backward()
        y = w * 2
        z = (y * y).sum()
        op(S, y.detach())                                              # a gradient of its own disturbs nothing
        z.backward()

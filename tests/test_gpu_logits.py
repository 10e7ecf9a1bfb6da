"""Operators on rows of logits beside a CSR matrix (device.top_entries, distill_loss, balance_loss) against their definitions
in 64 bits.

Tolerances.  The kernels work in f32: exp2 of an argument a has a relative error of about 2^-22 + |a| 2^-23, so with the
arguments here (below 60 in magnitude where the result is not lost in a sum) a softmax entry is within 1.2e-5 of itself,
TOL = 2e-5.  A loss is a sum of probabilities times logarithms: absolute error TOL times (1 + the largest logarithm).
A gradient is rounded once more to its type.  Rounding keeps the order, so it lies between the rounded ends of the interval
that the f32 value lies in.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = 2e-5
LEAST = {"bf16": 1e-38, "f16": 2.0 ** -25, "f32": 1e-37}            # below it a type's results are 0 or subnormal
TYPES = ["bf16", "f16", "f32"]


def torch_type(kind):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[kind]


def logits(rng, rows, cols, kind, spread=3.0):
    """(CUDA tensor, the same values in f64)."""
    import torch
    x = torch.from_numpy(rng.normal(0, spread, (rows, cols)).astype(np.float32)).to(torch_type(kind))
    return x.cuda(), x.double().numpy()


def csr(rows, cols, counts, crd, val, dtype=np.float32):
    import torch
    from comet_b200 import device
    pos = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()                     # noqa: E731
    return device.DeviceCSR(rows, cols, up(pos), up(np.asarray(crd, np.int64)), up(np.asarray(val, dtype))), pos


def teacher(rng, rows, cols, k, ragged, dtype=np.float32):
    counts = rng.integers(0, k + 1, rows) if ragged else np.full(rows, k)
    crd = np.concatenate([np.sort(rng.choice(cols, c, replace=False)) for c in counts] + [np.zeros(0, np.int64)])
    val = rng.normal(6, 2, len(crd)).astype(dtype)
    S, pos = csr(rows, cols, counts, crd, val, dtype)
    return S, pos, crd.astype(np.int64), val.astype(np.float64)


def log_sum_exp(v):
    m = v.max(initial=-np.inf)
    return m if not np.isfinite(m) else m + math.log(np.exp(v - m).sum())


def log_softmax(v):
    """v - log_sum_exp(v), where the logarithm would be lost beside the maximum too."""
    m = v.max()
    return v - m - math.log(np.exp(v - m).sum())


def distill(pos, crd, val, x, tau=1.0, lse=None, weight=None, scale=1.0):
    """The definition, a row at a time: rows' losses, loss, gradient, and for each gradient how far it may be off before it is rounded."""
    rows, grad, off, large = np.zeros(len(x)), np.zeros_like(x), np.zeros_like(x), np.zeros(len(x))
    for t, (lo, hi) in enumerate(zip(pos, pos[1:])):
        w = 1.0 if weight is None else float(weight[t])
        z = val[lo:hi] / tau
        if hi == lo or w == 0 or z.max() == -np.inf:
            continue
        u = x[t] / tau
        logq = log_softmax(u)
        q = np.exp(logq)
        logp = log_softmax(z) if lse is None else z - float(lse[t])
        p = np.exp(logp)
        on = p > 0
        dense = np.zeros(x.shape[1])
        np.add.at(dense, crd[lo:hi], p)
        rows[t] = (p[on] * (logp[on] - logq[crd[lo:hi]][on])).sum()
        large[t] = 1 + np.abs(logp[on]).max() + np.abs(logq[crd[lo:hi]][on]).max()
        g, o = q - dense, q + dense
        if lse is not None:
            left = max(0.0, 1 - p.sum())
            others = np.ones(x.shape[1], bool)
            others[crd[lo:hi]] = False
            rest = q[others].sum()
            if left > 0:
                rows[t] += left * (math.log(left) - (math.log(rest) if rest > 0 else -np.inf))
                large[t] += abs(math.log(left)) + (abs(math.log(rest)) if rest > 0 else 0)
            g[others] = q[others] * (1 - (left / rest if rest > 0 else 0))
            # left is 1 minus a sum of f32 probabilities, each off by TOL of itself
            o[others] = q[others] * (1 + (1 + left) / rest if rest > 0 else 1)
        grad[t], off[t] = g * scale * w / tau, np.abs(o * scale * w / tau)
    weights = np.ones(len(x)) if weight is None else np.asarray(weight, np.float64)
    return rows, scale * (rows * weights)[weights != 0].sum(), grad, TOL * off, TOL * large


def close_gradient(got, want, off, kind):
    """Within `off` before it was rounded to its type."""
    import torch
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    end = lambda v: torch.from_numpy(v).float().to(torch_type(kind)).double().numpy()     # noqa: E731
    assert (end(want - off - LEAST[kind]) <= got)[fine].all() and (got <= end(want + off + LEAST[kind]))[fine].all()


def check_distill(S, pos, crd, val, x, x64, kind, tau=1.0, lse=None, weight=None, scale=1.0, **more):
    import torch
    from comet_b200 import device
    up = lambda a: None if a is None else torch.from_numpy(np.asarray(a, np.float32)).cuda()   # noqa: E731
    loss, rows, grad = device.distill_loss(S, x, temperature=tau, lse=up(lse), weight=up(weight), scale=scale, **more)
    wrows, wloss, wgrad, off, roff = distill(pos, crd, val, x64, tau, None if lse is None else np.asarray(lse, np.float32), weight, scale)
    got = rows.double().cpu().numpy()
    fine = np.isfinite(wrows)
    assert np.array_equal(got[~fine], wrows[~fine])
    assert (np.abs(got - wrows)[fine] <= roff[fine]).all()
    if fine.all():
        w = np.ones(len(wrows)) if weight is None else np.abs(weight)
        assert abs(float(loss) - wloss) <= abs(scale) * (roff * w).sum() + 1e-6 * abs(wloss)
    if grad is not None:
        close_gradient(grad, wgrad, off, kind)
    return grad


SHAPES = [(1, 1, 1), (1, 2, 1), (2, 7, 3), (3, 17, 4), (40, 33, 5), (7, 1000, 8), (5, 4099, 33), (300, 1025, 6), (2, 50021, 64), (3, 131072, 16), (1, 20000, 700),
          # many rows, and rows of several CTAs; more entries than a CTA has threads; the longest rows
          (1300, 9, 4), (700, 700, 700), (600, 4096, 9), (200, 24001, 200), (160, 60007, 300), (90, 140001, 64), (1, 390000, 8)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,k", SHAPES)
def test_distill(rows, cols, k, kind):
    rng = np.random.default_rng(rows * 1000003 + cols)
    x, x64 = logits(rng, rows, cols, kind)
    for ragged, rest, tau, weighted in [(False, False, 1.0, False), (True, True, 2.0, True), (False, True, 0.7, False)]:
        S, pos, crd, val = teacher(rng, rows, cols, k, ragged)
        lse = weight = None
        if rest:
            lse = [log_sum_exp(val[a:b] / tau) + rng.uniform(0.05, 1.0) for a, b in zip(pos, pos[1:])]
            lse = np.where(np.isfinite(lse), lse, 0.0)
        if weighted:
            weight = np.where(rng.random(rows) < 0.3, 0.0, rng.uniform(0.5, 1.5, rows)).astype(np.float32)
        check_distill(S, pos, crd, val, x, x64, kind, tau, lse, weight, scale=4096.0 / rows)
        check_distill(S, pos, crd, val, x, x64, kind, tau, lse, weight, grad=False)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [1, 6, 250, 4097, 33333])
def test_distill_strides_alignments_and_in_place(cols, kind):
    """Slices of wider matrices at odd places, gradients at other alignments than the logits, and in place of them."""
    import torch
    rng = np.random.default_rng(cols)
    rows = 5
    S, pos, crd, val = teacher(rng, rows, cols, min(cols, 9), True)
    for before, behind in [(0, 0), (1, 0), (3, 2), (8, 5)]:
        wide, wide64 = logits(rng, rows, before + cols + behind, kind)
        kept = wide.clone()
        x, x64 = wide[:, before:before + cols], wide64[:, before:before + cols]
        check_distill(S, pos, crd, val, x, x64, kind, scale=512.0)
        for shift in (0, 1, 4):
            room = torch.full((rows, cols + 9), 7.0, dtype=x.dtype, device="cuda")
            check_distill(S, pos, crd, val, x, x64, kind, scale=512.0, grad=room[:, shift:shift + cols])
            assert (room[:, :shift] == 7).all() and (room[:, shift + cols:] == 7).all()      # nothing beside it is written
        assert torch.equal(wide, kept)
        check_distill(S, pos, crd, val, x, x64, kind, scale=512.0, grad=x)                   # in place
        assert torch.equal(wide[:, :before], kept[:, :before]) and torch.equal(wide[:, before + cols:], kept[:, before + cols:])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [50, 9000])
def test_distill_masked_logits(cols, kind):
    """-inf and the type's lowest value in masked places, rows of nothing else, and a teacher's -inf."""
    import torch
    rng = np.random.default_rng(5)
    low = torch.finfo(torch_type(kind)).min
    x, _ = logits(rng, 6, cols, kind)
    S, pos, crd, val = teacher(rng, 6, cols, 4, False)
    val[1], val[4:8] = -np.inf, -np.inf                                # one entry of row 0, all of row 1
    S, pos = csr(6, cols, np.full(6, 4), crd, val)
    x[0, :] = torch.where(torch.rand(cols, device="cuda") < 0.5, x[0], torch.tensor(-math.inf, dtype=x.dtype, device="cuda"))
    x[2, cols // 2:] = low
    x[3, :] = low
    for r in (0, 2):                                                   # what the teacher lists is not masked
        x[r, torch.from_numpy(crd[4 * r:4 * r + 4]).cuda()] = 1.0
    x[4, :] = -math.inf
    x[5, crd[20]] = -math.inf                                          # the student cannot say what the teacher does
    x64 = x.double().cpu().numpy()
    loss, rows, grad = __import__("comet_b200.device", fromlist=["x"]).distill_loss(S, x)
    keep = [0, 1, 2, 3]
    wrows, _, wgrad, off, roff = distill(pos[:5], crd, val, x64[:4])
    assert (np.abs(rows.double().cpu().numpy()[keep] - wrows) <= roff).all()
    close_gradient(grad[:4], wgrad, off, kind)
    assert wrows[1] == 0 and not wgrad[1].any()
    assert rows[4] == math.inf and rows[5] == math.inf and loss == math.inf
    assert not grad.isnan().any()
    want = torch.zeros(cols, dtype=torch.float64)                      # softmax of nothing is 0: the gradient is -p
    p = np.exp(val[16:20] - log_sum_exp(val[16:20]))
    want[torch.from_numpy(crd[16:20])] = torch.from_numpy(-p)
    close_gradient(grad[4:5], want[None].numpy(), np.full((1, cols), TOL), kind)


def test_distill_nan_and_infinity_stay_in_their_rows():
    from comet_b200 import device
    rng = np.random.default_rng(6)
    x, x64 = logits(rng, 4, 5000, "f32")
    S, pos, crd, val = teacher(rng, 4, 5000, 6, False)
    x[1, 77], x[2, 4999] = math.nan, math.inf
    _, rows, grad = device.distill_loss(S, x)
    assert rows[1].isnan() and rows[2].isnan() and grad[1].isnan().all() and grad[2].isnan().all()
    wrows, _, wgrad, off, roff = distill(pos, crd, val, x64)
    for r in (0, 3):
        assert abs(float(rows[r]) - wrows[r]) <= roff[r]
        close_gradient(grad[r:r + 1], wgrad[r:r + 1], off[r:r + 1], "f32")
    val[0] = math.nan
    S, _ = csr(4, 5000, np.full(4, 6), crd, val)
    assert device.distill_loss(S, x)[1][0].isnan()


def test_distill_repeated_and_impossible_columns():
    from comet_b200 import device
    rng = np.random.default_rng(7)
    x, x64 = logits(rng, 3, 700, "f32")
    crd = np.array([5, 5, 9, 600, 600, 600, 0, 699, 3, 700])
    val = rng.normal(0, 1, 10).astype(np.float32).astype(np.float64)
    S, pos = csr(3, 700, [6, 2, 2], crd, val)
    _, rows, grad = device.distill_loss(S, x)
    wrows, _, wgrad, off, roff = distill(pos[:3], crd, val, x64[:2])
    assert (np.abs(rows.double().cpu().numpy()[:2] - wrows) <= roff).all()
    close_gradient(grad[:2], wgrad, off, "f32")
    assert rows[2].isnan()                                             # column 700 of 700
    lse = np.array([log_sum_exp(val[a:b]) + 0.3 for a, b in zip(pos, pos[1:])], np.float32)
    import torch
    _, rows, grad = device.distill_loss(S, x, lse=torch.from_numpy(lse).cuda())
    wrows, _, wgrad, off, roff = distill(pos[:3], crd, val, x64[:2], lse=lse)
    assert (np.abs(rows.double().cpu().numpy()[:2] - wrows) <= roff).all()
    close_gradient(grad[:2], wgrad, off, "f32")


def test_distill_teacher_in_f64_and_cross_entropy():
    """A CSR matrix as to_device brings it (f64 values), and one entry a row: the cross entropy."""
    import scipy.sparse as sp
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(8)
    x, x64 = logits(rng, 50, 3001, "f32")
    labels = rng.integers(0, 3001, 50)
    S = device.to_device(sp.csr_matrix((np.ones(50), labels, np.arange(51)), shape=(50, 3001)))
    assert S.val.dtype == torch.float64
    loss, rows, grad = device.distill_loss(S, x, scale=1 / 50)
    check_distill(S, np.arange(51), labels, np.ones(50), x, x64, "f32", scale=1 / 50)
    want = np.array([log_sum_exp(r) - r[l] for r, l in zip(x64, labels)])
    assert np.abs(rows.double().cpu().numpy() - want).max() <= TOL * (1 + want.max())


@pytest.mark.parametrize("rest", [False, True])
def test_distill_gradient_against_differences(rest):
    """Central differences of the loss with h = 1/16: the third derivative of log sum exp is below 0.1 and that of the rest's term below
    0.5, so h^2 / 6 times it is below 4e-4; two losses below 8 within 1e-6 of themselves, over 2 h, add 1.3e-4."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(9)
    x, x64 = logits(rng, 1, 40, "f32", 1.0)
    S, pos, crd, val = teacher(rng, 1, 40, 7, False)
    lse = torch.tensor([log_sum_exp(val) + 0.4], dtype=torch.float32, device="cuda") if rest else None
    grad = device.distill_loss(S, x, lse=lse)[2]
    h = 1 / 16
    for j in list(crd[:4]) + [0, 39, 20]:
        at = []
        for d in (h, -h):
            y = x.clone()
            y[0, j] += d
            at.append(float(device.distill_loss(S, y, lse=lse, grad=False)[0]))
        assert abs((at[0] - at[1]) / (2 * h) - float(grad[0, j])) < 6e-4


def test_distill_far_rows():
    """Rows more than 2^32 bytes apart."""
    import torch
    rng = np.random.default_rng(10)
    cols = 1000
    x, x64 = logits(rng, 2, cols, "bf16")
    room = torch.empty((1 << 31) + 2000, dtype=torch.bfloat16, device="cuda")
    far = room.as_strided((2, cols), ((1 << 31) + 5, 1))
    far.copy_(x)
    S, pos, crd, val = teacher(rng, 2, cols, 5, False)
    check_distill(S, pos, crd, val, far, x64, "bf16")
    check_distill(S, pos, crd, val, far, x64, "bf16", grad=far)


def test_distill_on_another_stream_and_again():
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(11)
    x, x64 = logits(rng, 64, 9999, "bf16")
    S, pos, crd, val = teacher(rng, 64, 9999, 20, True)
    first = device.distill_loss(S, x)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    with torch.cuda.stream(other):
        y = x.clone()
        second = device.distill_loss(S, y)
    other.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)                                       # the same bits, every time


def test_distill_no_rows_and_no_entries():
    import torch
    from comet_b200 import device
    S, _ = csr(0, 12, [], [], [])
    loss, rows, grad = device.distill_loss(S, torch.empty((0, 12), device="cuda"))
    assert float(loss) == 0 and rows.shape == (0,) and grad.shape == (0, 12)
    S, _ = csr(3, 12, [0, 0, 0], [], [])
    loss, rows, grad = device.distill_loss(S, torch.full((3, 12), math.nan, device="cuda"))
    assert float(loss) == 0 and not rows.any() and not grad.any()


def top(x64, k):
    """Columns of the k largest of each row: NaN above all, equal ones by column."""
    v = np.where(np.isnan(x64), np.inf, x64)
    order = np.lexsort((np.broadcast_to(np.arange(x64.shape[1]), x64.shape), -v, ~np.isnan(x64)))
    return np.sort(order[:, :k], axis=1)


def check_top(x, x64, k, tau=1.0, lse=True):
    from comet_b200 import device
    got, sums = device.top_entries(x, k, temperature=tau, lse=lse)
    rows, cols = x64.shape
    want = top(x64, k)
    assert got.pos.tolist() == [k * t for t in range(rows + 1)]
    assert np.array_equal(got.crd.cpu().numpy().reshape(rows, k), want)
    val = got.val.double().cpu().numpy().reshape(rows, k)
    assert np.array_equal(val, np.take_along_axis(x64, want, 1), equal_nan=True)
    if lse:
        for t in range(rows):
            if not np.isnan(x64[t]).any() and not (x64[t] == np.inf).any():
                w = log_sum_exp(x64[t] / tau)
                assert float(sums[t]) == w if w == -np.inf else abs(float(sums[t]) - w) <= TOL * (1 + abs(w))
    else:
        assert sums is None


TOP_SHAPES = [(1, 1, 1), (3, 5, 2), (40, 8, 2), (33, 64, 8), (70, 61, 61), (9, 100, 33), (65, 256, 8), (5, 511, 16), (4, 513, 40), (6, 1000, 1000), (2, 3000, 1024),
              (3, 20011, 50), (1, 131072, 64), (2, 131072, 1024), (400, 9000, 12), (37, 700, 20), (9, 1024, 32), (9, 1025, 32), (6, 1000, 33)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,k", TOP_SHAPES)
def test_top_entries(rows, cols, k, kind):
    rng = np.random.default_rng(rows * 999983 + cols)
    x, x64 = logits(rng, rows, cols, kind)
    check_top(x, x64, k)
    check_top(x, x64, k, lse=False)
    wide, wide64 = logits(rng, rows, cols + 6, kind)                   # rows at odd places
    check_top(wide[:, 3:3 + cols], wide64[:, 3:3 + cols], k, tau=1.7)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols,k", [(8, 3), (60, 8), (250, 9), (700, 40), (9000, 1), (40000, 100), (40000, 1024), (100003, 300)])
def test_top_entries_of_hard_rows(cols, k, kind):
    """Rows in order, of few values, of one, of zeros of both signs, of -inf and NaN."""
    import torch
    rng = np.random.default_rng(cols + k)
    rows = [np.sort(rng.normal(0, 3, cols)), -np.sort(rng.normal(0, 3, cols)), rng.integers(0, 3, cols).astype(float), np.full(cols, 1.5),
            np.full(cols, -np.inf), np.where(rng.random(cols) < 0.5, 0.0, -0.0), np.where(rng.random(cols) < 2 / cols, 1.0, -np.inf),
            np.where(rng.random(cols) < 3 / cols, np.nan, rng.normal(0, 1, cols)), np.full(cols, np.nan),
            np.where(rng.random(cols) < 1.5 * k / cols, np.inf, rng.normal(0, 1, cols)), np.where(rng.random(cols) < 0.6 * k / cols, 2.0, -3.0),
            np.full(cols, torch.finfo(torch_type(kind)).min)]
    x = torch.from_numpy(np.array(rows, np.float32)).to(torch_type(kind))
    check_top(x.cuda(), x.double().numpy(), k)


def test_top_entries_far_rows_and_streams():
    import torch
    rng = np.random.default_rng(12)
    for cols, k in [(40, 4), (3000, 20)]:
        x, x64 = logits(rng, 2, cols, "f16")
        room = torch.empty((1 << 31) + 5000, dtype=torch.float16, device="cuda")
        far = room.as_strided((2, cols), ((1 << 31) + 5, 1))
        far.copy_(x)
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            check_top(far, x64, k)
    from comet_b200 import device
    got, sums = device.top_entries(torch.empty((0, 9), device="cuda"), 3, lse=True)
    assert got.pos.tolist() == [0] and got.nnz == 0 and sums.shape == (0,)


def balance(pos, crd, x, seq=None, mask=None, scores="softmax", scale=1.0):
    """The definition: loss, counts, gradient, and how far the gradient may be off before it is rounded."""
    rows, E = x.shape
    seq = [0, rows] if seq is None else seq
    counts, grad, off, loss = np.zeros((len(seq) - 1, E), np.int64), np.zeros_like(x), np.zeros_like(x), 0.0
    active = np.diff(pos) > 0 if mask is None else (np.diff(pos) > 0) & mask
    used = [s for s, (a, b) in enumerate(zip(seq, seq[1:])) if active[a:b].any()]
    for s in used:
        these = [t for t in range(seq[s], seq[s + 1]) if active[t]]
        for t in these:
            np.add.at(counts[s], crd[pos[t]:pos[t + 1]], 1)
        K = counts[s].sum()
        g = (counts[s] * E - K) / (K * E)                              # f - 1 / E, from whole numbers
        for t in these:
            u = x[t] if scores == "softmax" else np.minimum(x[t], 0) - np.log1p(np.exp(-np.abs(x[t])))
            p = np.exp(log_softmax(u)) if u.max() > -np.inf else np.zeros(E)
            by = scale * E / len(used) / len(these)
            slope = 1.0 if scores == "softmax" else np.exp(np.minimum(-x[t], 0) - np.log1p(np.exp(-np.abs(x[t]))))
            loss += by * (p.sum() / E + g @ p)
            grad[t] = by * p * (g - g @ p) * slope
            off[t] = abs(by) * p * (np.abs(g) + np.abs(g) @ p) * slope
    return loss, counts, grad, 3 * TOL * off


def choices(rng, rows, cols, k, ragged):
    counts = rng.integers(0, k + 1, rows) if ragged else np.full(rows, k)
    crd = np.concatenate([np.sort(rng.choice(cols, c, replace=False)) for c in counts] + [np.zeros(0, np.int64)]).astype(np.int64)
    S, pos = csr(rows, cols, counts, crd, np.zeros(len(crd)))
    return S, pos, crd


def check_balance(S, pos, crd, x, x64, kind, seq=None, mask=None, scores="softmax", scale=1.0, **more):
    import torch
    from comet_b200 import device
    up = lambda a, t: None if a is None else torch.from_numpy(np.asarray(a, t)).cuda()    # noqa: E731
    loss, counts, grad = device.balance_loss(S, x, seq=up(seq, np.int64), mask=up(mask, bool), scores=scores, scale=scale, **more)
    wloss, wcounts, wgrad, off = balance(pos, crd, x64, seq, mask, scores, scale)
    assert np.array_equal(counts.cpu().numpy(), wcounts)
    assert abs(float(loss) - wloss) <= TOL * abs(wloss)
    if grad is not None:
        close_gradient(grad, wgrad, off, kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (1, 8, 2), (5, 3, 3), (128, 8, 2), (300, 64, 8), (77, 61, 5), (1000, 256, 8), (40, 257, 3), (33, 1000, 16), (20, 1024, 1),
                                         (3000, 30, 1), (9000, 16, 2)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_balance(rows, cols, k, scores, kind):
    rng = np.random.default_rng(rows * 31 + cols)
    x, x64 = logits(rng, rows, cols, kind, 2.0)
    S, pos, crd = choices(rng, rows, cols, k, False)
    check_balance(S, pos, crd, x, x64, kind, scores=scores, scale=64.0)
    S, pos, crd = choices(rng, rows, cols, k, True)
    mask = rng.random(rows) < 0.8
    for sequences in (1, 3, min(rows, 50)):
        seq = np.concatenate([[0], np.sort(rng.integers(0, rows + 1, sequences - 1)), [rows]])
        check_balance(S, pos, crd, x, x64, kind, seq, mask, scores, scale=64.0)
    check_balance(S, pos, crd, x, x64, kind, np.arange(rows + 1), None, scores, scale=64.0)      # a sequence per row
    check_balance(S, pos, crd, x, x64, kind, None, mask, scores, grad=False)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [7, 64, 200])
def test_balance_strides_in_place_and_masked_experts(cols, kind):
    import torch
    rng = np.random.default_rng(cols)
    rows = 37
    S, pos, crd = choices(rng, rows, cols, 3, True)
    for before, behind in [(0, 0), (1, 0), (3, 2), (8, 5)]:
        wide, _ = logits(rng, rows, before + cols + behind, kind)
        x = wide[:, before:before + cols]
        x[2:9, ::2] = -math.inf
        x[9:12, 1:] = torch.finfo(x.dtype).min
        x[12, :] = torch.finfo(x.dtype).min
        x[13, :] = -math.inf
        kept, x64 = wide.clone(), x.double().cpu().numpy()
        for shift in (0, 1, 4):
            room = torch.full((rows, cols + 9), 7.0, dtype=x.dtype, device="cuda")
            check_balance(S, pos, crd, x, x64, kind, scale=64.0, grad=room[:, shift:shift + cols])
            assert (room[:, :shift] == 7).all() and (room[:, shift + cols:] == 7).all()
        assert torch.equal(wide.nan_to_num(), kept.nan_to_num())
        check_balance(S, pos, crd, x, x64, kind, scores="sigmoid", scale=64.0)
        check_balance(S, pos, crd, x, x64, kind, scale=64.0, grad=x)
        assert torch.equal(wide[:, :before], kept[:, :before]) and torch.equal(wide[:, before + cols:], kept[:, before + cols:])


def test_balance_sigmoid_of_very_low_logits():
    """Every sigmoid of a row is below f32's range: the scores' shares are still what they are."""
    rng = np.random.default_rng(13)
    x, _ = logits(rng, 40, 16, "f32")
    x -= 300
    S, pos, crd = choices(rng, 40, 16, 2, False)
    check_balance(S, pos, crd, x, x.double().cpu().numpy(), "f32", scores="sigmoid")


def test_balance_nothing_active():
    import torch
    from comet_b200 import device
    S, _ = csr(0, 12, [], [], [])
    loss, counts, grad = device.balance_loss(S, torch.empty((0, 12), device="cuda"))
    assert float(loss) == 0 and not counts.any() and grad.shape == (0, 12)
    S, pos, crd = choices(np.random.default_rng(1), 30, 12, 2, False)
    loss, counts, grad = device.balance_loss(S, torch.full((30, 12), math.nan, device="cuda"), mask=torch.zeros(30, dtype=torch.bool, device="cuda"))
    assert float(loss) == 0 and not counts.any() and not grad.any()


def test_balance_impossible_column_and_nan():
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(14)
    x, x64 = logits(rng, 3, 6, "f32")
    S, pos = csr(3, 6, [1, 1, 1], [0, 6, 2], [0, 0, 0])
    assert device.balance_loss(S, x)[0].isnan()
    S, pos = csr(3, 6, [1, 1, 1], [0, 5, 2], [0, 0, 0])
    assert not device.balance_loss(S, x)[0].isnan()                    # and the call before leaves nothing behind
    x[1, 1] = math.nan
    loss, counts, grad = device.balance_loss(S, x)
    assert loss.isnan() and grad[1].isnan().all() and not grad[0].isnan().any() and not grad[2].isnan().any()


def test_balance_gradient_against_differences():
    """Central differences with h = 1/32: third derivatives of E f p are below E / 2 = 3 over 5 rows, so h^2 / 6 times them is below 1e-4; two
    losses near 1 within 1e-6 over 2 h add 3.2e-5."""
    from comet_b200 import device
    rng = np.random.default_rng(15)
    for scores in ("softmax", "sigmoid"):
        x, _ = logits(rng, 5, 6, "f32", 1.0)
        S, pos, crd = choices(rng, 5, 6, 2, False)
        grad = device.balance_loss(S, x, scores=scores)[2]
        h = 1 / 32
        for t, e in [(0, 0), (1, 5), (4, 3), (2, 2)]:
            at = []
            for d in (h, -h):
                y = x.clone()
                y[t, e] += d
                at.append(float(device.balance_loss(S, y, scores=scores, grad=False)[0]))
            assert abs((at[0] - at[1]) / (2 * h) - float(grad[t, e])) < 2e-4


def test_same_bits_every_time():
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(16)
    x, _ = logits(rng, 20000, 64, "bf16")
    S, pos, crd = choices(rng, 20000, 64, 4, True)
    first = device.balance_loss(S, x)
    for _ in range(5):
        for a, b in zip(first, device.balance_loss(S, x)):
            assert torch.equal(a, b)


def test_refusals():
    import torch
    from comet_b200 import _lib, device
    x = torch.zeros((4, 9), device="cuda")
    S, _ = csr(4, 9, [1, 1, 1, 1], [0, 1, 2, 3], [1, 1, 1, 1])
    other, _ = csr(4, 8, [1, 1, 1, 1], [0, 1, 2, 3], [1, 1, 1, 1])
    dcsr = device.DeviceCSR(4, 9, S.pos, S.crd, S.val, row_ids=S.crd)
    half = torch.zeros(4, dtype=torch.float16, device="cuda")
    for call in (lambda: device.top_entries(x, 0), lambda: device.top_entries(x, 10), lambda: device.top_entries(torch.zeros((1, 5000), device="cuda"), 1025),
                 lambda: device.top_entries(x.double(), 2), lambda: device.top_entries(x.cpu(), 2), lambda: device.top_entries(x.t(), 2),
                 lambda: device.top_entries(x[0], 2), lambda: device.top_entries(x[:, :0], 1), lambda: device.top_entries(x[:1].expand(4, 9), 2),
                 lambda: device.distill_loss(other, x), lambda: device.distill_loss(dcsr, x), lambda: device.distill_loss(S, x, lse=half),
                 lambda: device.distill_loss(S, x, weight=half), lambda: device.distill_loss(S, x, weight=torch.zeros(3, device="cuda")),
                 lambda: device.distill_loss(S, x, grad=x.half()), lambda: device.distill_loss(S, x, grad=x[:, :8]),
                 lambda: device.distill_loss(device.DeviceCSR(4, 9, S.pos, S.crd, S.val.half()), x),
                 lambda: device.distill_loss(device.DeviceCSR(4, 9, S.pos.int(), S.crd, S.val), x),
                 lambda: device.balance_loss(other, x), lambda: device.balance_loss(dcsr, x), lambda: device.balance_loss(S, x, scores="tanh"),
                 lambda: device.balance_loss(S, x, seq=torch.zeros(1, dtype=torch.int64, device="cuda")),
                 lambda: device.balance_loss(S, x, seq=torch.zeros(3, device="cuda")), lambda: device.balance_loss(S, x, mask=half.bool()[:3]),
                 lambda: device.balance_loss(S, x, mask=half)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: device.distill_loss(S, x, temperature=0.0), lambda: device.distill_loss(S, x, temperature=-1.0),
                 lambda: device.distill_loss(S, x, temperature=math.nan), lambda: device.top_entries(x, 2, temperature=0.0, lse=True)):
        with pytest.raises(_lib.CometB200Error, match="temperature"):
            call()
    wide = torch.zeros((1, 800000), device="cuda")
    S, _ = csr(1, 800000, [1], [5], [1])
    with pytest.raises(_lib.CometB200Error, match="do not fit"):
        device.distill_loss(S, wide)
    S, _ = csr(1, 1025, [1], [5], [1])
    with pytest.raises(ValueError, match="experts"):
        device.balance_loss(S, wide[:, :1025])
    assert float(device.top_entries(x, 2)[0].val.sum()) == 0           # and the library goes on


def test_a_routed_student_learns():
    """The example: its distillation loss falls to less than half."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "distill_routed_student.py")
    spec = importlib.util.spec_from_file_location("distill_routed_student", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    history, counts = example.train(steps=40)
    assert sum(counts) == 512 * 2
    losses = [loss for loss, _ in history]
    assert all(math.isfinite(v) for v in losses) and losses[-1] < losses[0] / 2

"""Log probabilities of given columns (device.log_probs) and their gradient against their definitions in 64 bits.

Tolerances.  exp2 of an f32 argument d is off by 2^-22 + |d| 2^-24 of itself (the instruction's two units, and the argument's own rounding, doubled).  A
sum of n terms per thread, 256 threads and two sums each, is off by (n / 512 + 32) 2^-24 of itself at most, so log s is off by
    rel = 2^-20 + mean|d| 2^-23 + (n / 512 + 32) 2^-24,
mean under the row's probabilities, which the oracle has; a value is a rounded difference of that and (x - m) / temperature.  The entropy is log s minus the mean
of d: the terms of that sum carry rel and their argument's rounding, mean(d^2) 2^-23.  A gradient's q is off by 2^-20 + 2^-22 (|log q| + log s) of itself; it
is rounded once more to its type.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TYPES = ["bf16", "f16", "f32"]


def torch_type(kind):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[kind]


def given(rng, rows, cols, k, ragged=True, repeat=False):
    import torch
    from comet_b200 import device
    counts = rng.integers(0, k + 1, rows) if ragged else np.full(rows, k)
    crd = np.concatenate([np.zeros(0, np.int64)] + [np.sort(rng.choice(cols, c, replace=repeat)) for c in counts]).astype(np.int64)
    pos = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    up = lambda a: torch.from_numpy(a).cuda()                                                  # noqa: E731
    return device.DeviceCSR(rows, cols, up(pos), up(crd), None), up(np.repeat(np.arange(rows), counts))


def logits(rng, rows, cols, kind, spread=3.0):
    import torch
    return torch.from_numpy(rng.normal(0, spread, (rows, cols)).astype(np.float32)).to(torch_type(kind)).cuda()


class Oracle:
    def __init__(self, x, tau):
        import torch
        u = x.double() / tau
        self.m = u.amax(1, keepdim=True)
        d = u - self.m
        e = d.exp()
        s = e.sum(1, keepdim=True)
        self.log = s.log()
        self.logq = d - self.log
        self.q = e / s
        self.entropy = torch.where(self.q > 0, -self.q * self.logq, torch.zeros_like(self.q)).sum(1)
        far = torch.where(self.q > 0, d.abs() / math.log(2), torch.zeros_like(d))
        mean, square = (self.q * far).sum(1), (self.q * far * far).sum(1)
        self.rel = 2.0 ** -20 + mean * 2.0 ** -23 + (x.shape[1] / 512 + 32) * 2.0 ** -24
        self.off_entropy = self.rel * (2 + mean) + square * 2.0 ** -23 + (self.log[:, 0].abs() + self.entropy) * 2.0 ** -22
        self.tau, self.shape = tau, x.shape

    def off_value(self, logq, row):
        return self.rel[row] + 2.0 ** -22 * (2 * logq.abs() + self.log[row, 0].abs())

    def grad(self, S, row, d, h):
        import torch
        came = torch.zeros(self.shape, dtype=torch.float64, device="cuda").index_put_((row, S.crd), d.double(), accumulate=True)
        size = torch.zeros(self.shape, dtype=torch.float64, device="cuda").index_put_((row, S.crd), d.double().abs(), accumulate=True)
        n = S.pos.diff()[:, None] + 4
        g = came - self.q * came.sum(1, keepdim=True)
        relq = 2.0 ** -20 + 2.0 ** -22 * (torch.where(self.q > 0, self.logq.abs(), torch.zeros_like(self.q)) + self.log)
        off = size * 2.0 ** -22 * n + self.q * (came.sum(1, keepdim=True).abs() * relq + size.sum(1, keepdim=True) * n * 2.0 ** -23)
        if h is not None:
            w = h.double()[:, None].abs()
            inner = torch.where(self.q > 0, self.logq, torch.zeros_like(self.q)) + self.entropy[:, None]
            big = inner.abs() + 2 * self.entropy[:, None]
            g = g - h.double()[:, None] * self.q * inner
            off = off + w * self.q * (big * (relq + 2.0 ** -22) + self.off_entropy[:, None] + self.rel[:, None] + relq)
        return g / self.tau, off / self.tau


def within(got, want, off):
    import torch
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].double().nan_to_num(7), want[~fine].nan_to_num(7))
    over = ((got.double() - want).abs() - off)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, "off by %g more than it may" % float(over.max())


def rounded(got, want, off):
    import torch
    info = torch.finfo(got.dtype)
    # What rounds beyond the type's largest number, max (1 + eps / 4) being half a step above it, is infinite.
    over = want.abs() - off > info.max * (1 + info.eps / 4)
    assert torch.equal(got[over].double(), torch.sign(want[over]) * math.inf)
    got, want, off = got[~over], want[~over], off[~over]
    # f32 results below the least normal number are 0
    least = info.smallest_normal * (1 if got.dtype == torch.float32 else info.eps / 2)
    within(got, want, off + (want.abs() + off) * info.eps / 2 + least)


def check(S, row, x, tau, top=0):
    from comet_b200 import device
    o = Oracle(x, tau)
    values, sums, entropy, best = device.log_probs(S, x, temperature=tau, entropy=True, top=top)
    want = o.logq[row, S.crd]
    within(values, want, o.off_value(want.nan_to_num(0, 0, 0), row))
    within(sums[:, 1], o.log[:, 0], o.rel + 2.0 ** -22 * o.log[:, 0].abs())
    assert (sums[:, 0] == x.float().amax(1)).all()
    within(entropy, o.entropy, o.off_entropy)
    assert device.log_probs(S, x, temperature=tau, top=top)[2] is None
    if top:
        T, _ = device.top_entries(x, top)
        assert (T.pos == best.pos).all() and (T.crd == best.crd).all()
        at = np.repeat(np.arange(x.shape[0]), top)
        want = o.logq[at, best.crd]
        within(best.val, want, o.off_value(want.nan_to_num(0, 0, 0), at))
    return o, sums, entropy


SHAPES = [(1, 1, 1), (1, 2, 1), (2, 7, 3), (3, 17, 4), (40, 33, 5), (7, 250, 4), (129, 256, 2), (7, 1000, 8), (33, 1024, 3), (9, 1025, 2), (300, 2041, 6), (300, 2048, 6),
          (5, 2049, 3), (5, 4099, 33), (2, 50021, 64), (3, 131072, 16), (700, 4096, 9), (1300, 9, 4), (160, 60007, 300), (90, 140001, 8), (1, 390000, 8), (1, 20000, 700)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,k", SHAPES)
def test_values_and_gradient(rows, cols, k, kind):
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows * 1009 + cols)
    x = logits(rng, rows, cols, kind)
    for tau, top in [(1.0, 0), (0.7, min(cols, 20)), (2.0, min(cols, 300))]:
        S, row = given(rng, rows, cols, min(k, cols), ragged=tau != 1.0)
        o, sums, entropy = check(S, row, x, tau, top)
        d = torch.from_numpy(rng.standard_normal(S.nnz).astype(np.float32)).cuda()
        for h in (None, torch.from_numpy(rng.uniform(-1, 1, rows).astype(np.float32)).cuda()):
            g = device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h, temperature=tau)
            rounded(g, *o.grad(S, row, d, h))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [40, 1500, 9001])
def test_masked_columns(cols, kind):
    """Columns of -inf and of the type's lowest value; rows of nothing else."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(cols)
    x = logits(rng, 12, cols, kind)
    low = torch.finfo(x.dtype).min
    x[1, ::2] = -math.inf
    x[2, 1:] = -math.inf
    x[3, 3:] = low
    x[4, :] = low
    x[5, ::3] = low
    x[6, 1::2] = -math.inf
    x[6, ::2] = low
    S, row = given(rng, 12, cols, 4, ragged=False)
    for top in (0, 3):
        o, sums, entropy = check(S, row, x, 1.0, top)
    d = torch.from_numpy(rng.standard_normal(S.nnz).astype(np.float32)).cuda()
    h = torch.ones(12, device="cuda")
    rounded(device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h), *o.grad(S, row, d, h))
    rounded(device.log_probs_grad(S, x, sums, d), *o.grad(S, row, d, None))
    # a row of nothing, of NaN, of +inf
    x[7] = -math.inf
    x[8, cols // 2] = math.nan
    x[9, cols // 3] = math.inf
    for top in (0, 3):
        values, sums, entropy, best = device.log_probs(S, x, entropy=True, top=top)
        of = values.view(12, 4)
        assert (of[7] == -math.inf).all() and sums[7].tolist() == [-math.inf, 0.0] and float(entropy[7]) == 0.0
        assert torch.isnan(of[8:10]).all() and torch.isnan(entropy[8:10]).all() and torch.isfinite(entropy[:8]).all()
        if top:
            assert (best.val.view(12, 3)[7] == -math.inf).all()
    g = device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h)
    assert (g[7] == 0).all() and torch.isnan(g[8]).any() and not torch.isnan(g[:7]).any() and not torch.isnan(g[10:]).any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("tau", [1e-3, 1e4])
def test_temperatures_and_large_logits(tau, kind):
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(5)
    x = logits(rng, 9, 6001, kind, spread=tau if tau < 1 else 3)
    if tau < 1:
        x += 500                                           # exact differences of large logits over a small temperature
    S, row = given(rng, 9, 6001, 4, ragged=False)
    o, sums, entropy = check(S, row, x, tau, 5)
    d, h = torch.randn(S.nnz, device="cuda"), torch.randn(9, device="cuda")
    rounded(device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h, temperature=tau), *o.grad(S, row, d, h))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [50, 1999, 20011])
def test_views_repeats_and_gradients_in_place(cols, kind):
    """Rows at every alignment, repeated columns, a gradient in the logits' place, and what lies around the view stays."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(cols)
    for shift in (0, 1, 3, 8):
        wide = logits(rng, 7, cols + 21, kind)
        x = wide[:, shift:shift + cols]
        S, row = given(rng, 7, cols, 5, ragged=True, repeat=True)
        o, sums, entropy = check(S, row, x, 1.5)
        d, h = torch.randn(S.nnz, device="cuda"), torch.randn(7, device="cuda")
        want, off = o.grad(S, row, d, h)
        other = torch.full((7, cols + 5), 9.0, dtype=x.dtype, device="cuda")
        got = device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h, temperature=1.5, grad=other[:, 2:2 + cols])
        rounded(got, want, off)
        assert (other[:, :2] == 9).all() and (other[:, 2 + cols:] == 9).all()
        before, version = wide.clone(), x._version
        assert device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h, temperature=1.5, grad=x) is x
        rounded(x, want, off)
        assert x._version > version
        assert torch.equal(wide[:, :shift], before[:, :shift]) and torch.equal(wide[:, shift + cols:], before[:, shift + cols:])


def test_gradient_by_differences():
    """Of sum d values + h entropy, in f32."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(1)
    x = logits(rng, 3, 37, "f32")
    S, row = given(rng, 3, 37, 4, ragged=False)
    d, h = torch.randn(S.nnz, device="cuda").double(), torch.randn(3, device="cuda").double()
    _, sums, entropy, _ = device.log_probs(S, x, temperature=1.3, entropy=True)
    g = device.log_probs_grad(S, x, sums, d.float(), entropy=entropy, d_entropy=h.float(), temperature=1.3).double()

    def loss(v):
        o = Oracle(v, 1.3)
        return float((d.float().double() * o.logq[row, S.crd]).sum() + (h.float().double() * o.entropy).sum())

    step = 1e-5
    for _ in range(40):
        i, j = int(rng.integers(3)), int(rng.integers(37))
        up, down = x.double().clone(), x.double().clone()
        up[i, j] += step
        down[i, j] -= step
        # the differences' own error: step^2 times a third derivative (below 10), and 2^-52 of the losses (below 100) over the step
        assert abs((loss(up) - loss(down)) / (2 * step) - float(g[i, j])) < 1e-8 + 1e-5


def test_columns_outside_and_any_order():
    import torch
    from comet_b200 import device
    x = logits(np.random.default_rng(0), 2, 3000, "bf16")
    S = device.DeviceCSR(2, 3000, torch.tensor([0, 4, 6]).cuda(), torch.tensor([2999, -1, 0, 3000, 7, 7]).cuda(), None)
    o = Oracle(x, 1.0)
    for top in (0, 4):
        v = device.log_probs(S, x, top=top)[0]
        assert torch.isnan(v[[1, 3]]).all()
        at, row = torch.tensor([2999, 0, 7, 7]).cuda(), torch.tensor([0, 0, 1, 1]).cuda()
        want = o.logq[row, at]
        within(v[[0, 2, 4, 5]], want, o.off_value(want, row))


def test_empty_batches():
    import torch
    from comet_b200 import device
    x = torch.empty((0, 100), device="cuda")
    S = device.DeviceCSR(0, 100, torch.zeros(1, dtype=torch.int64).cuda(), torch.zeros(0, dtype=torch.int64).cuda(), None)
    values, sums, entropy, best = device.log_probs(S, x, entropy=True, top=3)
    assert values.shape == (0,) and sums.shape == (0, 2) and entropy.shape == (0,) and best.pos.tolist() == [0]
    assert device.log_probs_grad(S, x, sums, values).shape == (0, 100)
    # rows without tokens
    x = torch.randn(3, 5000, device="cuda")
    S = device.DeviceCSR(3, 5000, torch.zeros(4, dtype=torch.int64).cuda(), torch.zeros(0, dtype=torch.int64).cuda(), None)
    values, sums, entropy, _ = device.log_probs(S, x, entropy=True)
    within(entropy, Oracle(x, 1.0).entropy, Oracle(x, 1.0).off_entropy)
    assert (device.log_probs_grad(S, x, sums, values) == 0).all()


def test_same_bits_streams_and_graphs():
    """Calls on another stream and captured ones give the same bits as eager ones, and follow their inputs."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(3)
    x = logits(rng, 50, 30011, "bf16")
    S, _ = given(rng, 50, 30011, 3)
    d = torch.randn(S.nnz, device="cuda")

    def both():
        values, sums, entropy, best = device.log_probs(S, x, entropy=True, top=5)
        plain = device.log_probs(S, x, entropy=True)
        return [values, sums, entropy, best.crd, best.val, plain[0], plain[2], device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=entropy)]

    want = both()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for a, b in zip(want, both()):
            assert torch.equal(a, b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = both()
    x.copy_(logits(rng, 50, 30011, "bf16"))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(both(), held):
        assert torch.equal(a, b)


def test_refusals():
    import torch
    from comet_b200 import device
    x = torch.randn(4, 50, device="cuda")
    S, _ = given(np.random.default_rng(0), 4, 50, 2)
    sums, d = device.log_probs(S, x)[1], torch.zeros(S.nnz, device="cuda")
    bad = device.DeviceCSR(4, 51, S.pos, S.crd, None)
    for call in (lambda: device.log_probs(bad, x), lambda: device.log_probs(S, x, top=51), lambda: device.log_probs(S, x, top=-1),
                 lambda: device.log_probs(S, x.double()), lambda: device.log_probs(S, x.t()), lambda: device.log_probs(S, x.cpu()),
                 lambda: device.log_probs(device.DeviceCSR(4, 50, S.pos.int(), S.crd, None), x),
                 lambda: device.log_probs_grad(S, x, sums, d.double()), lambda: device.log_probs_grad(S, x, sums[:3], d),
                 lambda: device.log_probs_grad(S, x, sums, d, d_entropy=torch.zeros(4, device="cuda")),
                 lambda: device.log_probs_grad(S, x, sums, d, grad=None), lambda: device.log_probs_grad(S, x, sums, d, grad=x.half())):
        with pytest.raises(ValueError):
            call()
    for tau in (0.0, -1.0, math.nan, math.inf, 1e-39):
        with pytest.raises(RuntimeError, match="temperature"):
            device.log_probs(S, x, temperature=tau)
        with pytest.raises(RuntimeError, match="temperature"):
            device.log_probs_grad(S, x, sums, d, temperature=tau)


@pytest.mark.parametrize("kind,cols", [("bf16", 131072), ("f32", 1201)])
def test_offsets_beyond_32_bits(kind, cols):
    """More than 2^31 logits: the last rows are what they are alone, the gradient in the logits' place too."""
    import torch
    from comet_b200 import device
    rows, last = (1 << 31) // cols + 100, 50
    x = torch.empty((rows, cols), dtype=torch_type(kind), device="cuda")
    x[-2 * last:] = torch.randn((2 * last, cols), device="cuda").to(x.dtype)
    x[:-2 * last] = 0
    S = device.DeviceCSR(rows, cols, torch.arange(rows + 1, device="cuda"), torch.arange(rows, device="cuda") % cols, None)
    part = device.DeviceCSR(last, cols, torch.arange(last + 1, device="cuda"), S.crd[-last:].clone(), None)
    d, h = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
    own = x[-last:].clone()
    want = device.log_probs(part, own, entropy=True, top=3)
    for top in (0, 3):
        values, sums, entropy, best = device.log_probs(S, x, entropy=True, top=top)
        # alone the rows may be cut into parts: the same but for the order of sums
        assert float((values[-last:] - want[0]).abs().max()) < 1e-5 and float((entropy[-last:] - want[2]).abs().max()) < 1e-5
        assert float((sums[-last:] - want[1]).abs().max()) < 1e-5
        if top:
            assert torch.equal(best.crd[-3 * last:], want[3].crd) and float((best.val[-3 * last:] - want[3].val).abs().max()) < 1e-5
    want = device.log_probs_grad(part, own, sums[-last:].clone(), d[-last:].clone(), entropy=entropy[-last:].clone(), d_entropy=h[-last:].clone())
    device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h, grad=x)
    assert torch.equal(x[-last:], want)


@pytest.mark.parametrize("kind", TYPES)
def test_products_beyond_what_is_exact(kind):
    """Logits over the temperature beyond 2^22: differences to the largest one are taken first."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(8)
    x = logits(rng, 5, 4500, kind, spread=1.0) + 300
    x[1:3] += 1000
    x[2, 7] = 2000
    S, row = given(rng, 5, 4500, 4, ragged=False)
    for tau in (1e-5, 3e-4):
        o, sums, entropy = check(S, row, x, tau, 4)
        d, h = torch.randn(S.nnz, device="cuda"), torch.randn(5, device="cuda")
        rounded(device.log_probs_grad(S, x, sums, d, entropy=entropy, d_entropy=h, temperature=tau), *o.grad(S, row, d, h))

"""A router's experts (device.group_entries, gated_experts, combine_experts and their gradients) against their definitions in 64 bits.

Tolerances.  A product of two 16-bit numbers is exact in f32; a sum of K of them is off by at most K 2^-23 of the sum of their magnitudes (one
unit in the last place an addition, whatever the order), which the oracle computes beside each result.  The logistic function is off by 2^-20 of
itself (exp2 of an argument below 60 with a relative error of 2^-22 + 60 x 2^-23 / 2, a quotient).  What is computed from sums carries their bounds to first
order, doubled for the rest.  Rounding to T bits costs eps / 2 of the value; where gradients are rounded before they are multiplied again, that of each.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
TYPES = ["bf16", "f16"]


def torch_type(kind):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16}[kind]


def half_step(kind):
    import torch
    return torch.finfo(torch_type(kind)).eps / 2


def routes(rng, rows, experts, counts, columns=None):
    """A DeviceCSR of choices with weights, and (pos, crd, row of each entry) on the host."""
    import torch
    from comet_b200 import device
    pos = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    if columns is None:
        columns = [np.sort(rng.choice(experts, c, replace=False)) for c in counts]
    crd = np.concatenate([np.zeros(0, np.int64)] + list(columns)).astype(np.int64)
    val = rng.uniform(0.05, 1.0, len(crd)).astype(np.float32)
    up = lambda a: torch.from_numpy(a).cuda()                                                  # noqa: E731
    return device.DeviceCSR(rows, experts, up(pos), up(crd), up(val)), pos, crd, np.repeat(np.arange(rows), counts)


def matrix(rng, kind, *shape, scale=1.0):
    import torch
    return torch.from_numpy((rng.standard_normal(shape) * scale).astype(np.float32)).to(torch_type(kind)).cuda()


def activation(g, kind):
    """act(g) and its slope, in 64 bits."""
    import torch
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    a, b = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(a * (g + b * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * b * g * g)


class Oracle:
    """All results in 64 bits with what each may be off by; a loop over experts."""

    def __init__(self, S, pos, crd, row, kind, act="silu"):
        import torch
        self.torch, self.S, self.row, self.kind, self.act = torch, S, torch.from_numpy(row).cuda(), kind, act
        self.crd = torch.from_numpy(crd).cuda()
        self.e = half_step(kind)
        info = torch.finfo(torch_type(kind))
        self.least = info.smallest_normal * info.eps / 2       # a subnormal result is a multiple of twice that, so off by no more than it

    def zeros(self, *shape):
        return self.torch.zeros(shape, dtype=self.torch.float64, device="cuda")

    def experts(self):
        for j in range(self.S.ncols):
            yield j, (self.crd == j).nonzero().reshape(-1)

    def products(self, X, w):
        """Gate and up with their bounds."""
        n = w.shape[0] // 2
        z, off = X @ w.T, X.abs() @ w.abs().T * (w.shape[1] * 2.0 ** -23)
        return z[:, :n], z[:, n:], off[:, :n], off[:, n:]

    def gated(self, X, W):
        h, off = self.zeros(len(self.crd), W.shape[1] // 2), self.zeros(len(self.crd), W.shape[1] // 2)
        for j, at in self.experts():
            g, u, og, ou = self.products(X[self.row[at]].double(), W[j].double())
            a, slope = activation(g, self.act)
            h[at] = a * u
            off[at] = 2 * (og * (slope.abs() + og) * u.abs() + a.abs() * ou + (a * u).abs() * 2.0 ** -20)
        return h, off + self.e * h.abs()

    def gated_grad(self, X, W, dH):
        n, width = W.shape[1] // 2, W.shape[2]
        dx, ox, dw, ow = self.zeros(self.S.nrows, width), self.zeros(self.S.nrows, width), self.zeros(*W.shape), self.zeros(*W.shape)
        for j, at in self.experts():
            x, w, d = X[self.row[at]].double(), W[j].double(), dH[at].double()
            g, u, og, ou = self.products(x, w)
            a, slope = activation(g, self.act)
            dz = self.torch.cat([d * u * slope, d * a], 1)
            # the second derivatives of both activations are below 1.3 in magnitude
            oz = 2 * self.torch.cat([d.abs() * (ou * slope.abs() + u.abs() * (1.3 * og + 2.0 ** -18)), d.abs() * (og * slope.abs() + og * og + a.abs() * 2.0 ** -20)], 1)
            oz = oz + self.e * dz.abs() + self.least
            dx.index_add_(0, self.row[at], dz @ w)
            ox.index_add_(0, self.row[at], oz @ w.abs() + dz.abs() @ w.abs() * (2 * n * 2.0 ** -23 + 2.0 ** -20))
            dw[j] = dz.T @ x
            ow[j] = oz.T @ x.abs() + dz.abs().T @ x.abs() * (len(at) * 2.0 ** -23)
        return dx, ox + self.e * (dx.abs() + ox), dw, ow + self.e * (dw.abs() + ow)

    def combine(self, H, V):
        val = self.S.val.double()
        y, off = self.zeros(self.S.nrows, V.shape[1]), self.zeros(self.S.nrows, V.shape[1])
        for j, at in self.experts():
            h, v, w = H[at].double(), V[j].double(), val[at][:, None]
            y.index_add_(0, self.row[at], w * (h @ v.T))
            off.index_add_(0, self.row[at], w * (h.abs() @ v.abs().T) * ((V.shape[2] + 16) * 2.0 ** -23))
        return y, off + self.e * (y.abs() + off)

    def combine_grad(self, H, V, dY):
        val = self.S.val.double()
        dh, oh, dv, ov = self.zeros(*H.shape), self.zeros(*H.shape), self.zeros(*V.shape), self.zeros(*V.shape)
        dval, oval = self.zeros(len(self.crd)), self.zeros(len(self.crd))
        for j, at in self.experts():
            h, v, w, d = H[at].double(), V[j].double(), val[at][:, None], dY[self.row[at]].double()
            back, o = d @ v, d.abs() @ v.abs() * (V.shape[1] * 2.0 ** -23)
            dh[at], oh[at] = w * back, w * (o + back.abs() * 2.0 ** -23)
            dval[at], oval[at] = (back * h).sum(1), (o * h.abs()).sum(1) + (back * h).abs().sum(1) * (V.shape[2] * 2.0 ** -23)
            dv[j] = d.T @ (w * h)
            ov[j] = d.abs().T @ (w * h.abs() * (self.e + 2.0 ** -23 + len(at) * 2.0 ** -23) + self.least)
        return dh, oh + self.e * (dh.abs() + oh), dv, ov + self.e * (dv.abs() + ov), dval, oval


def close(got, want, off, kind):
    """Within its bound, and half the least step of its type."""
    import torch
    least = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    over = (got.double() - want).abs() - off - least
    assert got.shape == want.shape and not torch.isnan(got).any()
    assert float(over.max() if over.numel() else 0) <= 0, "off by %g more than %g at most" % (float(over.max()), float(off.max()))


def run_block(rng, rows, experts, counts, width, inner, act, kind, columns=None):
    """All operators in a row, each against the oracle."""
    from comet_b200 import device
    S, pos, crd, row = routes(rng, rows, experts, counts, columns)
    O = Oracle(S, pos, crd, row, kind, act)
    X, W = matrix(rng, kind, rows, width), matrix(rng, kind, experts, 2 * inner, width, scale=width ** -0.5)
    V, dY = matrix(rng, kind, experts, width, inner, scale=inner ** -0.5), matrix(rng, kind, rows, width)
    G = device.group_entries(S)
    H = device.gated_experts(G, X, W, activation=act)
    close(H, *O.gated(X, W), kind)
    dH = matrix(rng, kind, len(crd), inner)
    dX, dW = device.gated_experts_grad(G, X, W, dH, activation=act)
    dx, ox, dw, ow = O.gated_grad(X, W, dH)
    close(dX, dx, ox, kind)
    close(dW, dw, ow, kind)
    close(device.combine_experts(G, H, V), *O.combine(H, V), kind)
    dH2, dV, dval = device.combine_experts_grad(G, H, V, dY)
    dh, oh, dv, ov, dvalue, oval = O.combine_grad(H, V, dY)
    close(dH2, dh, oh, kind)
    close(dV, dv, ov, kind)
    close(dval, dvalue, oval + 1e-7 * dvalue.abs(), kind)
    G.check()


SHAPES = [
    # rows, experts, chosen, width, inner
    (1, 1, 1, 8, 8), (1, 8, 2, 64, 64), (1, 64, 8, 256, 128), (2, 3, 3, 72, 40), (5, 4, 1, 136, 264), (128, 1, 1, 64, 128), (129, 2, 1, 200, 136),
    (300, 5, 2, 256, 512), (777, 10, 3, 1000, 712), (1500, 64, 6, 128, 96), (4099, 7, 2, 64, 72), (64, 1000, 5, 72, 24),
    # one token with many experts, and with rows too long for the kernels of one token
    (1, 64, 20, 264, 136), (1, 1000, 300, 72, 40), (1, 3, 2, 8200, 40), (1, 2, 2, 64, 2056),
]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,experts,chosen,width,inner", SHAPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_block(rows, experts, chosen, width, inner, ragged, kind):
    rng = np.random.default_rng(rows * 31 + experts * 7 + width + ragged)
    counts = rng.integers(0, chosen + 1, rows) if ragged else np.full(rows, chosen)
    run_block(rng, rows, experts, counts, width, inner, "gelu" if ragged else "silu", kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,experts,chosen,width,inner", [(700, 1, 1, 264, 200), (2000, 3, 2, 320, 384), (5000, 4, 1, 72, 1032)])
def test_many_entries_an_expert(rows, experts, chosen, width, inner, kind):
    """Tiles by pairs: even and odd numbers of them, an expert without any and one with few."""
    rng = np.random.default_rng(rows)
    weight = np.linspace(3, 0.2, experts) if experts < 4 else np.array([5, 0, 0.02, 2])
    columns = [np.sort(rng.choice(experts, chosen, replace=False, p=weight / weight.sum())) for _ in range(rows)]
    run_block(rng, rows, experts, np.full(rows, chosen), width, inner, "silu", kind, columns)


def listed_slots(G):
    """(column, entry, token) of each filled slot in order, and the numbers of entries without a column, from a plan as csrc/groups.cuh lays it out."""
    p, n, nnz = G.plan.cpu().numpy(), G.S.ncols, G.S.nnz
    tiles = nnz // 128 + min(nnz, n) + 1
    counts = p[16:16 + n]
    first = p[16 + (n + 3) // 4 * 4:][:n + 1]
    column = p[16 + (n + 3) // 4 * 4 + (n + 4) // 4 * 4:][:tiles]
    slots = tiles * 128
    order, token = p[-2 * slots:-slots], p[-slots:]
    assert p[0] == first[n] and p[2] == 0
    used = np.arange(p[0] * 128)
    got = order[used] >= 0
    assert (column[:p[0]] == np.repeat(np.arange(n), np.diff(first))).all() and (np.diff(first) == -(-counts // 128)).all()
    assert (token[used][~got] == -1).all()
    return column[used[got] // 128], order[used[got]], token[used[got]], sorted(order[slots - p[1]:])


@pytest.mark.parametrize("rows,experts,most,bad", [(1, 64, 8, 0), (1, 1, 1, 0), (3, 1024, 60, 2), (40, 5, 5, 0), (256, 3, 1, 0), (257, 3, 1, 3), (1000, 700, 3, 0), (1025, 64, 8, 5),
                                                   (9000, 64, 8, 0), (9000, 1024, 8, 7), (40000, 16, 8, 0), (30000, 1000, 9, 1)])
def test_groups(rows, experts, most, bad):
    """Entries in the order of columns, and inside a column in their own; by one CTA, by clusters, with and without room to sort in."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows + experts)
    counts = rng.integers(0, most + 1, rows)
    counts[rng.integers(rows)] = most
    pos = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    # some columns are asked for much more often; repeated ones in a row, and those in any order, are allowed
    crd = np.minimum((rng.random(pos[-1]) ** 2 * experts).astype(np.int64), experts - 1)
    wrong = rng.choice(pos[-1], min(bad, int(pos[-1])), replace=False)
    crd[wrong] = rng.choice([-1, experts, 1 << 40], len(wrong))
    up = lambda a: torch.from_numpy(a).cuda()                                                  # noqa: E731
    column, order, token, left = listed_slots(device.group_entries(device.DeviceCSR(rows, experts, up(pos), up(crd), None)))
    good = np.flatnonzero((crd >= 0) & (crd < experts))
    want = good[np.argsort(crd[good], kind="stable")]
    assert (order == want).all() and (column == crd[want]).all() and (token == np.repeat(np.arange(rows), counts)[want]).all()
    assert left == sorted(wrong)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows", [1, 5, 700])
def test_repeated_columns(rows, kind):
    """A token that has an expert more than once, and columns in any order."""
    rng = np.random.default_rng(rows)
    columns = [rng.integers(0, 3, 5) for _ in range(rows)]
    run_block(rng, rows, 3, np.full(rows, 5), 136, 72, "gelu", kind, columns)


@pytest.mark.parametrize("rows", [1, 40, 900])
def test_columns_outside(rows):
    """An entry whose column is no expert's makes its own results NaN, and those of its token; the experts' gradients leave it out."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows)
    S, pos, crd, row = routes(rng, rows, 4, np.full(rows, 2))
    bad = [0, len(crd) - 1] if rows > 1 else [1]
    S.crd[bad[0]] = -1
    S.crd[bad[-1]] = 4
    O = Oracle(S, pos, S.crd.cpu().numpy(), row, "bf16")
    X, W, V = matrix(rng, "bf16", rows, 64), matrix(rng, "bf16", 4, 96, 64, scale=0.1), matrix(rng, "bf16", 4, 64, 48, scale=0.1)
    G = device.group_entries(S)
    fine = torch.ones(len(crd), dtype=torch.bool, device="cuda")
    fine[bad] = False
    tokens = torch.ones(rows, dtype=torch.bool, device="cuda")
    tokens[row[bad]] = False
    H = device.gated_experts(G, X, W)
    assert torch.isnan(H[~fine]).all()
    want, off = O.gated(X, W)
    close(H[fine], want[fine], off[fine], "bf16")
    H = matrix(rng, "bf16", len(crd), 48)
    Y = device.combine_experts(G, H, V)
    want, off = O.combine(H, V)
    assert torch.isnan(Y[~tokens]).all()
    close(Y[tokens], want[tokens], off[tokens], "bf16")
    dX, dW = device.gated_experts_grad(G, X, W, H)
    dx, ox, dw, ow = O.gated_grad(X, W, H)
    assert torch.isnan(dX[~tokens]).all()
    close(dX[tokens], dx[tokens], ox[tokens], "bf16")
    close(dW, dw, ow, "bf16")
    dH, dV, dval = device.combine_experts_grad(G, H, V, X)
    dh, oh, dv, ov, dvalue, oval = O.combine_grad(H, V, X)
    assert torch.isnan(dH[~fine]).all() and torch.isnan(dval[~fine]).all()
    close(dH[fine], dh[fine], oh[fine], "bf16")
    close(dV, dv, ov, "bf16")
    close(dval[fine], dvalue[fine], oval[fine] + 1e-7 * dvalue[fine].abs(), "bf16")


@pytest.mark.parametrize("rows", [0, 3])
def test_nothing_stored(rows):
    import torch
    from comet_b200 import device
    S = device.DeviceCSR(rows, 4, torch.zeros(rows + 1, dtype=torch.int64).cuda(), torch.zeros(0, dtype=torch.int64).cuda(), torch.zeros(0).cuda())
    G = device.group_entries(S)
    new = lambda *shape: torch.randn(shape, device="cuda").bfloat16()                           # noqa: E731
    X, W, H, V = new(rows, 16), new(4, 32, 16), new(0, 16), new(4, 16, 16)
    assert device.gated_experts(G, X, W).shape == (0, 16)
    dX, dW = device.gated_experts_grad(G, X, W, H)
    assert dX.shape == X.shape and not dX.any() and not dW.any()
    assert torch.equal(device.combine_experts(G, H, V), torch.zeros_like(X))
    dH, dV, dval = device.combine_experts_grad(G, H, V, X)
    assert dH.shape == (0, 16) and not dV.any() and dval.shape == (0,)
    G.check()


@pytest.mark.parametrize("rows", [1, 6, 500])
def test_rows_with_a_stride(rows):
    """Tokens' rows in a wider matrix, and no more gradients than are asked for."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows)
    S, pos, crd, row = routes(rng, rows, 5, np.full(rows, 2))
    wide, W = matrix(rng, "f16", rows, 200), matrix(rng, "f16", 5, 160, 104, scale=0.1)
    X, V, dY = wide[:, 16:120], matrix(rng, "f16", 5, 104, 80, scale=0.1), wide[:, 88:192]
    G = device.group_entries(S)
    H = device.gated_experts(G, X, W)
    assert torch.equal(H, device.gated_experts(G, X.contiguous(), W))
    dH = matrix(rng, "f16", len(crd), 80)
    dX, dW = device.gated_experts_grad(G, X.contiguous(), W, dH)
    for x, w in [(True, True), (True, False), (False, True)]:
        got = device.gated_experts_grad(G, X, W, dH, grad_x=x, grad_w=w)
        assert (got[0] is None) == (not x) and (got[1] is None) == (not w)
        assert not x or torch.equal(got[0], dX)
        assert not w or torch.equal(got[1], dW)
    want = device.combine_experts_grad(G, H, V, dY.contiguous())
    for a, b in zip(device.combine_experts_grad(G, H, V, dY), want):
        assert torch.equal(a, b)
    got = device.combine_experts_grad(G, H, V, dY, grad_v=False)
    assert torch.equal(got[0], want[0]) and got[1] is None and torch.equal(got[2], want[2])


def test_infinities_stay_with_their_expert():
    """A token of infinities and a weight of NaN: other tokens' and experts' results are what they were."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(4)
    S, pos, crd, row = routes(rng, 300, 6, np.full(300, 2))
    X, W, V = matrix(rng, "bf16", 300, 64), matrix(rng, "bf16", 6, 64, 64, scale=0.1), matrix(rng, "bf16", 6, 64, 32, scale=0.1)
    G = device.group_entries(S)
    d = matrix(rng, "bf16", len(crd), 32)
    H, dW, Y, dV = device.gated_experts(G, X, W), device.gated_experts_grad(G, X, W, d)[1], device.combine_experts(G, d, V), device.combine_experts_grad(G, d, V, X)[1]
    X[7], W[2], V[2] = math.inf, math.nan, math.nan
    entry = torch.from_numpy((row != 7) & (crd != 2)).cuda()
    token = torch.tensor([t != 7 and 2 not in crd[pos[t]:pos[t + 1]] for t in range(300)]).cuda()
    expert = torch.tensor([j != 2 and j not in crd[pos[7]:pos[8]] for j in range(6)]).cuda()
    without = torch.tensor([2 not in crd[pos[t]:pos[t + 1]] for t in range(300)]).cuda()
    assert torch.equal(device.gated_experts(G, X, W)[entry], H[entry])
    assert torch.equal(device.gated_experts_grad(G, X, W, d)[1][expert], dW[expert])
    assert torch.equal(device.combine_experts(G, d, V)[without], Y[without]) and token.any()
    assert torch.equal(device.combine_experts_grad(G, d, V, X)[1][expert], dV[expert])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,chosen", [(60, 2), (900, 2)])
def test_gradients_by_differences(rows, chosen, kind):
    """Along a direction: the difference quotient of the block in 64 bits against the kernels' gradients times the direction."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows)
    S, pos, crd, row = routes(rng, rows, 3, np.full(rows, chosen))
    O = Oracle(S, pos, crd, row, kind, "gelu")
    X, W = matrix(rng, kind, rows, 40), matrix(rng, kind, 3, 48, 40, scale=0.3)
    H, V = matrix(rng, kind, len(crd), 24), matrix(rng, kind, 3, 40, 24, scale=0.3)
    dH, dY = matrix(rng, kind, len(crd), 24), matrix(rng, kind, rows, 40)
    G = device.group_entries(S)
    to = lambda t: torch.from_numpy(rng.standard_normal(t.shape)).cuda()                         # noqa: E731
    vx, vw, vh, vv, vs = to(X), to(W), to(H), to(V), to(S.val)

    def gated(s):
        return float((O.gated(X.double() + s * vx, W.double() + s * vw)[0] * dH.double()).sum())

    def combine(s):
        O.S = device.DeviceCSR(S.nrows, S.ncols, S.pos, S.crd, S.val.double() + s * vs)
        y = O.combine(H.double() + s * vh, V.double() + s * vv)[0]
        O.S = S
        return float((y * dY.double()).sum())

    step = 1e-4
    dX, dW = device.gated_experts_grad(G, X, W, dH, activation="gelu")
    _, ox, _, ow = O.gated_grad(X, W, dH)
    got = float((dX.double() * vx).sum() + (dW.double() * vw).sum())
    off = float((ox * vx.abs()).sum() + (ow * vw.abs()).sum())
    # the quotient's own error, step^2 times a third derivative, is that of the same quotient with twice the step, divided by three
    quotient = lambda f, s: (f(s) - f(-s)) / (2 * s)                                             # noqa: E731
    own = abs(quotient(gated, 2 * step) - quotient(gated, step)) + 1e-6
    assert abs(got - quotient(gated, step)) <= off + own and off < 0.2 * float((dX.double() * vx).abs().sum())
    dh, dV, dval = device.combine_experts_grad(G, H, V, dY)
    _, oh, _, ov, _, oval = O.combine_grad(H, V, dY)
    got = float((dh.double() * vh).sum() + (dV.double() * vv).sum() + (dval.double() * vs).sum())
    off = float((oh * vh.abs()).sum() + (ov * vv.abs()).sum() + (oval * vs.abs()).sum())
    own = abs(quotient(combine, 2 * step) - quotient(combine, step)) + 1e-6
    assert abs(got - quotient(combine, step)) <= off + own


@pytest.mark.parametrize("rows", [1, 30, 2000])
def test_same_bits_streams_and_graphs(rows):
    """Calls on another stream, two at once, and captured ones give an eager call's bits, and follow their inputs; so does a graph that holds all of them."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows)
    S, pos, crd, row = routes(rng, rows, 4, np.full(rows, 2))
    X, W, V = matrix(rng, "bf16", rows, 264), matrix(rng, "bf16", 4, 400, 264, scale=0.1), matrix(rng, "bf16", 4, 264, 200, scale=0.1)
    d = matrix(rng, "bf16", len(crd), 200)

    def everything():
        G = device.group_entries(S)
        H = device.gated_experts(G, X, W)
        return [H, device.combine_experts(G, H, V), *device.gated_experts_grad(G, X, W, d), *device.combine_experts_grad(G, H, V, X), G.plan[2:3]]

    want = everything()
    for a, b in zip(want, everything()):
        assert torch.equal(a, b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(everything())
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(want, g):
            assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        held = everything()
    other = np.concatenate([np.sort(rng.choice(4, 2, replace=False)) for _ in range(rows)])
    S.crd.copy_(torch.from_numpy(other))
    X.copy_(matrix(rng, "bf16", rows, 264))
    torch.cuda.synchronize()
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(everything(), held):
        assert torch.equal(a, b)


def test_refusals():
    import torch
    from comet_b200 import _lib, device
    rng = np.random.default_rng(0)
    S, pos, crd, row = routes(rng, 6, 4, np.full(6, 2))
    G = device.group_entries(S)
    X, W, H, V = matrix(rng, "bf16", 6, 64), matrix(rng, "bf16", 4, 96, 64), matrix(rng, "bf16", 12, 48), matrix(rng, "bf16", 4, 64, 48)
    wide = matrix(rng, "bf16", 6, 80)
    csr = lambda **k: device.DeviceCSR(**{**dict(nrows=6, ncols=4, pos=S.pos, crd=S.crd, val=S.val), **k})          # noqa: E731
    no_values, doubles = device.group_entries(csr(val=None)), device.group_entries(csr(val=S.val.double()))
    for call in (lambda: device.group_entries(csr(ncols=0)), lambda: device.group_entries(csr(ncols=1025)), lambda: device.group_entries(csr(pos=S.pos.int())),
                 lambda: device.group_entries(csr(crd=S.crd.int())), lambda: device.group_entries(csr(nrows=7)), lambda: device.group_entries(csr(pos=S.pos.cpu())),
                 lambda: device.group_entries(csr(row_ids=S.pos[:6])),
                 lambda: device.gated_experts(G, X.float(), W.float()), lambda: device.gated_experts(G, X.half(), W), lambda: device.gated_experts(G, X[:5], W),
                 lambda: device.gated_experts(G, X, W[:3]), lambda: device.gated_experts(G, X, W[:, :, :32]), lambda: device.gated_experts(G, X, W[:, :88].contiguous()),
                 lambda: device.gated_experts(G, X, W, activation="relu"), lambda: device.gated_experts(G, wide[:, 1:65], W), lambda: device.gated_experts(G, X.t(), W),
                 lambda: device.gated_experts(G, X.cpu(), W), lambda: device.gated_experts(G, X, W.transpose(1, 2)),
                 lambda: device.gated_experts(G, wide[:, :68], matrix(rng, "bf16", 4, 96, 68)),
                 lambda: device.gated_experts_grad(G, X, W, H[:11]), lambda: device.gated_experts_grad(G, X, W, H.half()), lambda: device.gated_experts_grad(G, X, W, H[:, :40]),
                 lambda: device.combine_experts(G, H, V.half()), lambda: device.combine_experts(G, H[:11], V), lambda: device.combine_experts(G, H, V[:, :60].contiguous()),
                 lambda: device.combine_experts(no_values, H, V), lambda: device.combine_experts(doubles, H, V),
                 lambda: device.combine_experts_grad(G, H, V, X.half()), lambda: device.combine_experts_grad(G, H, V, wide), lambda: device.combine_experts_grad(G, H, V, X[:3])):
        with pytest.raises(ValueError):
            call()
    # the C entries themselves
    at = [t.data_ptr() for t in (G.plan, X, W, H)]
    for sizes, ldx, plan in [((6, 4, 12, 60, 48), 64, at[0]), ((6, 4, 12, 64, 44), 64, at[0]), ((6, 4, 12, 64, 48), 60, at[0]), ((6, 4, 12, 64, 48), 68, at[0]),
                             ((6, 0, 12, 64, 48), 64, at[0]), ((6, 1025, 12, 64, 48), 64, at[0]), ((-1, 4, 12, 64, 48), 64, at[0]), ((6, 4, -1, 64, 48), 64, at[0])]:
        with pytest.raises(_lib.CometB200Error, match="gated_experts"):
            device._call("comet_b200_dev_gated_experts_bf16_i64", *sizes, 0, plan, at[1], ldx, at[2], at[3], device._stream())
    with pytest.raises(_lib.CometB200Error, match="16 bytes"):
        device._call("comet_b200_dev_gated_experts_bf16_i64", 6, 4, 12, 64, 48, 0, at[0], at[1] + 2, 64, at[2], at[3], device._stream())
    torch.cuda.synchronize()
    G.check()
    G.plan[2] = 1                                                          # what a kernel leaves that gave up waiting
    with pytest.raises(_lib.CometB200Error, match="wait"):
        G.check()


@pytest.mark.parametrize("width,inner", [(64, 1024), (1024, 64)])
def test_offsets_beyond_32_bits(width, inner):
    """2.4 million entries: more than 2^31 elements of H, of dz and of the rows that are summed.  The last tokens are what they are alone."""
    import torch
    from comet_b200 import device
    rows, experts, chosen, last = 300000, 8, 8, 200
    g = torch.Generator("cuda")
    g.manual_seed(3)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda").bfloat16()           # noqa: E731
    pos = torch.arange(rows + 1, device="cuda") * chosen
    crd = torch.arange(experts, device="cuda").repeat(rows)
    val = torch.rand(rows * chosen, generator=g, device="cuda")
    X, W, V = normal(rows, width), normal(experts, 2 * inner, width) * width ** -0.5, normal(experts, width, inner) * inner ** -0.5
    S = device.DeviceCSR(rows, experts, pos, crd, val)
    G = device.group_entries(S)
    H = device.gated_experts(G, X, W)
    assert H.numel() * (1 if inner > width else width // inner) > 2 ** 31
    Y = device.combine_experts(G, H, V)
    dH, _, dval = device.combine_experts_grad(G, H, V, X, grad_v=False)
    dX, _ = device.gated_experts_grad(G, X, W, H, grad_w=False)
    torch.cuda.synchronize()
    G.check()
    few = slice(-last * chosen, None)
    g2 = device.group_entries(device.DeviceCSR(last, experts, pos[:last + 1], crd[few], val[few]))
    x, h = X[-last:].contiguous(), H[few].contiguous()
    assert torch.equal(device.gated_experts(g2, x, W), h)
    assert torch.equal(device.combine_experts(g2, h, V), Y[-last:])
    dh, _, dv = device.combine_experts_grad(g2, h, V, x, grad_v=False)
    assert torch.equal(dh, dH[few]) and float((dv - dval[few]).abs().max()) <= 1e-5 * float(dv.abs().max())
    assert torch.equal(device.gated_experts_grad(g2, x, W, h, grad_w=False)[0], dX[-last:])


@pytest.mark.parametrize("rows,experts,width,inner", [(128 * 74, 1, 264, 264), (128 * 149, 1, 256, 200), (128 * 100, 2, 1032, 520), (128 * 30 + 1, 1, 2568, 1288)])
def test_last_rounds(rows, experts, width, inner):
    """Numbers of tiles around the number of SMs: rounds that end with few tiles, whose columns are halved."""
    rng = np.random.default_rng(width)
    run_block(rng, rows, experts, np.full(rows, 1), width, inner, "silu", "bf16")

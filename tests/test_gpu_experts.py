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

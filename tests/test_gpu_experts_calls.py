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


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("rows", [1, 700])
def test_gates_whose_square_is_infinite(act, rows):
    """Gates of 1e20 and -1e20: the activation's slope is 1 and 0 there, though the cube inside gelu is infinite in f32."""
    import torch
    from comet_b200 import device
    width, inner = 64, 16
    crd = torch.arange(rows, device="cuda") % 2
    S = device.DeviceCSR(rows, 2, torch.arange(rows + 1, device="cuda"), crd, None)
    X = torch.zeros((rows, width), device="cuda")
    X[:, 0] = 1e10
    X[:, 1] = 1.0
    W = torch.zeros((2, 2 * inner, width), device="cuda")
    W[0, :inner, 0], W[1, :inner, 0] = 1e10, -1e10
    W[:, inner:, 1] = 2.0
    X, W = X.bfloat16(), W.bfloat16()
    G = device.group_entries(S)
    H = device.gated_experts(G, X, W, activation=act)
    big = X[0, 0].double() * W[0, 0, 0].double()
    want = torch.where(crd == 0, 2 * big, 0.0)[:, None].expand(-1, inner)
    assert float((H.double() - want).abs().max()) <= 2.0 ** -8 * 2 * float(big)
    d = torch.full((rows, inner), 0.5, device="cuda").bfloat16()
    dX, dW = device.gated_experts_grad(G, X, W, d, activation=act)
    # d_gate = 0.5 * 2 * slope, d_up = 0.5 * act(gate); the products of 0 with other columns' weights are 0
    assert not torch.isnan(dX).any() and not torch.isnan(dW).any()
    n0, n1 = (rows + 1) // 2, rows // 2
    x0 = X[0, 0].double()
    want = torch.stack([torch.full((inner,), float(n0 * x0), device="cuda"), torch.zeros(inner, device="cuda")])
    off = (dW[:, :inner, 0].double() - want).abs()
    assert n1 <= n0 and float(off.max()) <= 2.0 ** -7 * n0 * float(x0)
    assert float(dW[1, :inner].abs().max()) == 0
    # column 0: 16 gate rows of weight 1e10 with a gradient of 1 each, and nothing from up rows
    want = torch.where(crd == 0, inner * W[0, 0, 0].double(), 0.0)
    assert float((dX[:, 0].double() - want).abs().max()) <= 2.0 ** -8 * inner * float(W[0, 0, 0])
    G.check()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows,width,inner", [(40, 2048, 64), (700, 2048, 1024), (700, 8192, 512), (60, 32768, 128)])
def test_gradients_of_values_have_f32s_digits(rows, width, inner, kind):
    """However long the sums are.  The tensor cores cut off what is below a unit in the last place of the sum so far, 32 times in the 512 terms that they add up.  A unit is
    0.72 x 2^-23 of a sum on average, half of it is lost: 4.3e-8 of the sum, always towards zero.  Of sums of random signs, which grow with the root of the number of their terms,
    the 32 losses are 32 / sqrt(3) of that: 8e-7 of the norm.  Beyond 512 terms sums are rounded to the nearest: 2^-24 of the sum, of random signs, 64 times for the
    longest here, and as often in the sum with h: 4e-7 at most."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(width)
    S = device.DeviceCSR(rows, 2, torch.arange(rows + 1, device="cuda"), torch.arange(rows, device="cuda") % 2, torch.ones(rows, device="cuda"))
    H, V, dY = matrix(rng, kind, rows, inner), matrix(rng, kind, 2, width, inner, scale=inner ** -0.5), matrix(rng, kind, rows, width)
    G = device.group_entries(S)
    got = device.combine_experts_grad(G, H, V, dY, grad_v=False)[2].double()
    want = torch.cat([((dY[j::2].double() @ V[j].double()) * H[j::2].double()).sum(1, keepdim=True) for j in range(2)])
    order = torch.argsort(torch.cat([torch.arange(j, rows, 2) for j in range(2)])).cuda()
    want = want.reshape(-1)[order]
    assert float((got - want).norm() / want.norm()) < 1.2e-6
    G.check()


def test_two_host_threads():
    """Calls from two threads at once, on a stream each and at temperatures of their own, give what each of them gives alone."""
    import threading

    import torch
    from comet_b200 import device
    torch.cuda.init()
    wrong, work = [], []
    for t, (rows, kind) in enumerate([(1, "bf16"), (300, "f16")]):
        rng = np.random.default_rng(t)
        crd = torch.from_numpy(np.concatenate([np.sort(rng.choice(6, 2, replace=False)) for _ in range(rows)])).cuda()
        S = device.DeviceCSR(rows, 6, torch.arange(0, 2 * rows + 1, 2, device="cuda"), crd, torch.rand(2 * rows, device="cuda"))
        X, W, V = matrix(rng, kind, rows, 136), matrix(rng, kind, 6, 80, 136, scale=0.1), matrix(rng, kind, 6, 136, 40, scale=0.1)
        L = torch.randn(rows, 5000, device="cuda")
        given = device.DeviceCSR(rows, 5000, torch.arange(rows + 1, device="cuda"), torch.arange(rows, device="cuda") * 7, None)

        def everything(tau, S=S, X=X, W=W, V=V, L=L, given=given):
            G = device.group_entries(S)
            H = device.gated_experts(G, X, W)
            values, sums, entropy, best = device.log_probs(given, L, temperature=tau, entropy=True, top=3)
            return [H, device.combine_experts(G, H, V), *device.gated_experts_grad(G, X, W, H), *device.combine_experts_grad(G, H, V, X), values, entropy, best.val,
                    device.log_probs_grad(given, L, sums, values, temperature=tau), G.plan[2:3]]

        taus = [0.5 + 0.01 * i + 10 * t for i in range(200)]
        work.append((everything, taus, [everything(tau) for tau in taus[::40]]))
    torch.cuda.synchronize()

    def go(everything, taus, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for i, tau in enumerate(taus):
                    got = everything(tau)
                    if i % 40 == 0 and not all(torch.equal(a, b) for a, b in zip(got, want[i // 40])):
                        wrong.append((tau, [k for k, (a, b) in enumerate(zip(got, want[i // 40])) if not torch.equal(a, b)]))
        except Exception as e:                                             # noqa: BLE001 - told by the main thread
            wrong.append(e)

    threads = [threading.Thread(target=go, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong


@pytest.mark.parametrize("rows,part", [(40, slice(7, 8)), (40, slice(3, 30)), (100, slice(0, 99)), (3000, slice(100, 101)), (3000, slice(100, 140)), (3000, slice(500, 2500))])
def test_some_rows_of_a_larger_matrix(rows, part):
    """pos of some rows beside crd and values of all: the other rows' entries are no token's here.  What belongs to the rows is what it is without them, and the experts'
    gradients leave them out."""
    import torch
    from comet_b200 import device
    rng = np.random.default_rng(rows)
    crd = np.concatenate([np.sort(rng.choice(5, 2, replace=False)) for _ in range(rows)])
    crd[[0, -1]] = [-1, 5]                                                 # of rows that are left out, or not
    crd, val, pos = torch.from_numpy(crd).cuda(), torch.rand(2 * rows, device="cuda"), torch.arange(0, 2 * rows + 1, 2, device="cuda")
    n, of = part.stop - part.start, slice(2 * part.start, 2 * part.stop)
    X, W, V = matrix(rng, "bf16", n, 72), matrix(rng, "bf16", 5, 80, 72, scale=0.1), matrix(rng, "bf16", 5, 72, 40, scale=0.1)
    d = torch.full((2 * rows, 40), float("nan"), device="cuda").bfloat16()
    d[of] = matrix(rng, "bf16", 2 * n, 40)
    S, alone = device.DeviceCSR(n, 5, pos[part.start:part.stop + 1], crd, val), device.DeviceCSR(n, 5, pos[:n + 1].clone(), crd[of].clone(), val[of].clone())
    G, A = device.group_entries(S), device.group_entries(alone)
    equal = lambda a, b: torch.equal(a.float().nan_to_num(7.0), b.float().nan_to_num(7.0))        # noqa: E731
    assert equal(device.gated_experts(G, X, W)[of], device.gated_experts(A, X, W))
    assert equal(device.combine_experts(G, d, V), device.combine_experts(A, d[of].clone(), V))
    for a, b in zip(device.gated_experts_grad(G, X, W, d), device.gated_experts_grad(A, X, W, d[of].clone())):
        assert equal(a, b)
    a, b = device.combine_experts_grad(G, d, V, X), device.combine_experts_grad(A, d[of].clone(), V, X)
    assert equal(a[0][of], b[0]) and equal(a[1], b[1]) and not torch.isnan(a[1]).any()
    # the sums of parts of a row of h, whose width goes by the number of all entries, in f32
    values, want = a[2][of], b[2]
    assert torch.equal(torch.isnan(values), torch.isnan(want)) and float((values - want).nan_to_num(0.0).abs().max()) <= 1e-5 * float(want.nan_to_num(0.0).abs().max())
    G.check()

"""Operators on rows of logits that have a sparse side: the largest entries of dense rows as a CSR matrix, distillation from
a teacher's top logits (a CSR matrix) with its gradient, and a router's balance loss with its counts and gradient.

The operands are in GPU memory.  Logits are what the last product of a model gives: normal with a spread of 2 to 3 in
bf16, f16 or f32, a few columns of each row well above the rest.  A teacher stores the k largest of its own logits, in
f32, columns ascending; a router's choices are the k largest of its logits.
"""
import math

import torch

own = False

TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST = 4096 * 131072                     # elements of the largest matrix of logits


def listed():
    return [
        # Distillation of one token, as a student that learns while it serves does it: latency.
        {"name": "distill_one_token", "op": "distill", "rows": 1, "cols": 32768, "k": 32, "type": "bf16", "temperature": 1.0, "rest": False,
         "ragged": False, "weight": False, "grad": True},
        # A short batch in f32, an odd vocabulary (rows at every alignment), ragged top lists, a third of the tokens masked by weight.
        {"name": "distill_odd_f32", "op": "distill", "rows": 509, "cols": 50021, "k": 17, "type": "f32", "temperature": 2.0, "rest": True,
         "ragged": True, "weight": True, "grad": True},
        # The training step of a micro-batch of 4096 tokens with a large vocabulary; what the teacher does not list counts as one outcome.
        {"name": "distill_train", "op": "distill", "rows": 4096, "cols": 131072, "k": 64, "type": "bf16", "temperature": 1.0, "rest": True,
         "ragged": False, "weight": False, "grad": True},
        # Evaluation: the loss alone, f16 logits, long top lists with prompts' rows empty.
        {"name": "distill_eval", "op": "distill", "rows": 4096, "cols": 65536, "k": 256, "type": "f16", "temperature": 1.0, "rest": False,
         "ragged": True, "weight": False, "grad": False},
        # The teacher's side of a single token.
        {"name": "top_one_token", "op": "top", "rows": 1, "cols": 131072, "k": 50, "type": "f32", "temperature": 1.0, "lse": True},
        # The teacher's side of a micro-batch: its top 64 logits and the sum that they are a part of.
        {"name": "top_teacher", "op": "top", "rows": 4096, "cols": 131072, "k": 64, "type": "bf16", "temperature": 1.0, "lse": True},
        # Odd sizes, a long list, no sum.
        {"name": "top_odd_f16", "op": "top", "rows": 777, "cols": 50021, "k": 200, "type": "f16", "temperature": 1.0, "lse": False},
        # A router of 64 experts, 8 a token.
        {"name": "top_router", "op": "top", "rows": 16384, "cols": 64, "k": 8, "type": "f32", "temperature": 1.0, "lse": False},
        # A router of 256 experts over a long batch.
        {"name": "top_wide_router", "op": "top", "rows": 65536, "cols": 256, "k": 8, "type": "bf16", "temperature": 1.0, "lse": False},
        # The balance loss of a small batch and 8 experts: launches count.
        {"name": "balance_small", "op": "balance", "rows": 128, "cols": 8, "k": 2, "type": "f32", "sequences": 1, "mask": False, "scores": "softmax"},
        # The balance loss of a micro-batch as one group.
        {"name": "balance_step", "op": "balance", "rows": 16384, "cols": 64, "k": 8, "type": "f32", "sequences": 1, "mask": False,
         "scores": "softmax"},
        # The same per sequence, sigmoid scores, padding masked, many experts.
        {"name": "balance_sequences", "op": "balance", "rows": 65536, "cols": 256, "k": 8, "type": "bf16", "sequences": 32, "mask": True,
         "scores": "sigmoid"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: from one token to a micro-batch, vocabularies and numbers of experts over their range."""
    op = rng.choice(["distill", "distill", "top", "balance"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "balance":
        cols = _log(rng, 8, 512)
        rows = _log(rng, 1, 65536 if cols <= 256 else 32768)
        return {"op": op, "rows": rows, "cols": cols, "k": rng.randint(1, min(16, cols // 2)), "type": kind,
                "sequences": rng.choice([1, _log(rng, 1, 64)]), "mask": rng.random() < 0.5, "scores": rng.choice(["softmax", "sigmoid"])}
    if op == "top" and rng.random() < 0.5:
        cols = _log(rng, 8, 512)
        return {"op": op, "rows": _log(rng, 1, 65536 if cols <= 256 else 32768), "cols": cols, "k": rng.randint(1, min(16, cols // 2)),
                "type": kind, "temperature": 1.0, "lse": rng.random() < 0.3}
    cols = _log(rng, 4096, 160000)
    rows = _log(rng, 1, max(1, min(8192, MOST // (cols * (2 if kind == "f32" else 1)))))
    c = {"op": op, "rows": rows, "cols": cols, "k": _log(rng, 1, 256), "type": kind, "temperature": rng.choice([1.0, 1.0, 0.7, 2.0, 4.0])}
    if op == "top":
        return dict(c, lse=rng.random() < 0.6)
    return dict(c, rest=rng.random() < 0.5, ragged=rng.random() < 0.5, weight=rng.random() < 0.3, grad=rng.random() < 0.75)


def _scale(case):
    """Losses are means over the batch; f16 gradients are scaled up, as training in f16 does."""
    return (65536.0 if case["type"] == "f16" else 1.0) / case["rows"]


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    rows, cols, k, kind = case["rows"], case["cols"], case["k"], TYPE[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")          # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=g, device="cuda")          # noqa: E731

    x = torch.empty((rows, cols), dtype=kind, device="cuda")
    step = max(1, (1 << 26) // cols)
    for r in range(0, rows, step):                                                   # in pieces: f32 normals of all of it would be large
        x[r:r + step] = normal(min(step, rows - r), cols) * 2.5
    s = {"case": case, "x": x}
    if case["op"] == "top":
        n = max(1, cols // 1024)                                                     # a column in each of n equal stretches: distinct
        hot = ((torch.arange(n, device="cuda") + uniform(rows, n)).double() * (cols / n)).to(torch.int64).clamp_(max=cols - 1)
        x.scatter_(1, hot, (normal(rows, n) * 3 + 4).to(kind))
        return s

    if case["op"] == "balance":
        x += (normal(cols) * 0.7).to(kind)                                           # some experts are liked better
        crd = torch.topk(x.float() + 1e-3 * uniform(rows, cols), k, dim=1).indices.sort(dim=1).values
        counts = torch.full((rows,), k, device="cuda")
        s["mask"] = uniform(rows) < 0.9 if case["mask"] else None
        s["seq"] = None
        if case["sequences"] > 1:                                                    # ragged lengths
            cuts = (uniform(case["sequences"] - 1) * (rows + 1)).to(torch.int64).clamp_(0, rows).sort().values
            s["seq"] = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), rows)])
        val = x.float().gather(1, crd)
        keep = None
    else:
        # columns of a row: one in each of k equal stretches of the vocabulary, so ascending and distinct
        at = torch.arange(k, device="cuda") + uniform(rows, k)
        crd = (at.double() * (cols / k)).to(torch.int64).clamp_(max=cols - 1)
        val = normal(rows, k) * 2 + 8
        top = (val + normal(rows, k) * (0.5 + 2.0 * uniform(rows, 1))).to(kind)      # the student has learnt some of it
        x.scatter_(1, crd, top)
        counts = torch.full((rows,), k, device="cuda")
        if case["ragged"]:                                                           # fewer than k stored; one row in eight is a prompt's
            counts = (uniform(rows) * k).to(torch.int64) + 1
            counts = torch.where(uniform(rows) < 0.125, torch.zeros_like(counts), counts)
        keep = torch.arange(k, device="cuda")[None, :] < counts[:, None]
        s["weight"] = None
        if case["weight"]:
            s["weight"] = torch.where(uniform(rows) < 1 / 3, torch.zeros(rows, device="cuda"), 0.5 + uniform(rows))
        s["lse"] = None
        if case["rest"]:                                                             # 1 to 30 % of the teacher's mass is not listed
            z = torch.where(keep, val / case["temperature"], torch.full_like(val, -math.inf))
            z = torch.where(counts[:, None] > 0, z, torch.zeros_like(z))
            s["lse"] = torch.logsumexp(z.double(), 1).sub(torch.log(0.7 + 0.29 * uniform(rows).double())).float()
    s["pos"] = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
    s["pos"][1:] = torch.cumsum(counts, 0)
    s["crd"], s["val"] = (crd.reshape(-1), val.reshape(-1)) if keep is None else (crd[keep], val[keep])
    return s


def run(state):
    c = state["case"]
    if own:
        from comet_b200 import device
        if c["op"] == "top":
            got, lse = device.top_entries(state["x"], c["k"], temperature=c["temperature"], lse=c["lse"])
            return {"pos": got.pos, "crd": got.crd, "val": got.val, "lse": lse}
        s = device.DeviceCSR(c["rows"], c["cols"], state["pos"], state["crd"], state["val"])
        if c["op"] == "balance":
            loss, counts, grad = device.balance_loss(s, state["x"], seq=state["seq"], mask=state["mask"], scores=c["scores"], scale=_scale(c))
            return {"loss": loss, "counts": counts, "grad": grad}
        loss, rows, grad = device.distill_loss(s, state["x"], temperature=c["temperature"], lse=state["lse"], weight=state["weight"],
                                               scale=_scale(c), grad=c["grad"])
        return {"loss": loss, "rows": rows, "grad": grad}
    return {"top": _plain_top, "distill": _plain_distill, "balance": _plain_balance}[c["op"]](state)


def _plain_top(state):
    c = state["case"]
    x = state["x"].float()
    crd = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["k"]].sort(dim=1).values
    out = {"pos": torch.arange(c["rows"] + 1, device=x.device) * c["k"], "crd": crd.reshape(-1), "val": x.gather(1, crd).reshape(-1), "lse": None}
    if c["lse"]:
        u = x / c["temperature"]
        m = u.amax(1, keepdim=True)
        out["lse"] = (m + (u - m).exp().sum(1, keepdim=True).log()).reshape(-1)
    return out


def _plain_distill(state):
    c = state["case"]
    x, pos, crd, tau = state["x"], state["pos"], state["crd"], c["temperature"]
    t, v = x.shape
    n = pos[1:] - pos[:-1]
    row = torch.repeat_interleave(torch.arange(t, device=x.device), n, output_size=crd.shape[0])
    weight = torch.ones(t, device=x.device) if state["weight"] is None else state["weight"]
    weight = torch.where(n > 0, weight, torch.zeros_like(weight))
    counted = weight != 0
    # teacher
    z = state["val"].float() / tau
    if c["rest"]:
        logp = z - state["lse"][row]
        p = logp.exp()
        left = (1 - torch.zeros(t, device=x.device).index_add_(0, row, p)).clamp_(min=0)
    else:
        top = torch.full((t,), -math.inf, device=x.device).scatter_reduce_(0, row, z, "amax")
        logp = z - top[row]
        logp = logp - torch.zeros(t, device=x.device).index_add_(0, row, logp.exp()).log()[row]
        p = logp.exp()
    # student
    u = x.float() / tau
    m = u.amax(1, keepdim=True)
    e = (u - m).exp()
    total = e.sum(1)
    at = row * v + crd
    logq = u.reshape(-1)[at] - m.reshape(-1)[row] - total.log()[row]
    rows = torch.zeros(t, device=x.device).index_add_(0, row, p * (logp - logq))
    if c["rest"]:
        q_at = e.reshape(-1)[at] / total[row]
        e.reshape(-1)[at] = 0
        others = e.sum(1)
        rows = rows + torch.where(left > 0, left * (left.log() - (others / total).log()), torch.zeros_like(left))
    rows = torch.where(counted, rows, torch.zeros_like(rows))
    out = {"loss": (rows * weight).sum() * _scale(c), "rows": rows, "grad": None}
    if c["grad"]:
        by = torch.where(counted, weight * (_scale(c) / tau), torch.zeros_like(weight))
        if c["rest"]:
            grad = e * (by * (1 / total - left / others))[:, None]
            grad.reshape(-1)[at] = (q_at - p) * by[row]
        else:
            grad = e * (by / total)[:, None]
            grad.reshape(-1).index_add_(0, at, -p * by[row])
        out["grad"] = grad.to(x.dtype)
    return out


def _plain_balance(state):
    c = state["case"]
    x, pos, crd = state["x"], state["pos"], state["crd"]
    t, e = x.shape
    n = pos[1:] - pos[:-1]
    row = torch.repeat_interleave(torch.arange(t, device=x.device), n, output_size=crd.shape[0])
    active = n > 0
    if state["mask"] is not None:
        active = active & state["mask"]
    seq = state["seq"] if state["seq"] is not None else torch.tensor([0, t], device=x.device)
    sequences = seq.shape[0] - 1
    of = (torch.arange(t, device=x.device)[:, None] >= seq[None, 1:-1]).sum(1)
    counts = torch.zeros(sequences * e, dtype=torch.int64, device=x.device)
    counts = counts.index_add_(0, of[row] * e + crd, active[row].to(torch.int64)).reshape(sequences, e)
    tokens = torch.zeros(sequences, device=x.device).index_add_(0, of, active.float())
    f = counts.float() / counts.sum(1, keepdim=True).clamp(min=1).float()
    r = x.float()
    if c["scores"] == "sigmoid":
        s = 1 / (1 + (-r).exp())
        p = s / s.sum(1, keepdim=True)
    else:
        p = (r - r.amax(1, keepdim=True)).exp()
        p = p / p.sum(1, keepdim=True)
    by = torch.where(active, (_scale(c) * e / (tokens > 0).sum() / tokens.clamp(min=1))[of], torch.zeros(t, device=x.device))
    dot = (f[of] * p).sum(1, keepdim=True)
    grad = by[:, None] * p * (f[of] - dot)
    if c["scores"] == "sigmoid":
        grad = grad * (1 - s)
    return {"loss": (by * dot.reshape(-1)).sum(), "counts": counts, "grad": grad.to(x.dtype)}


def work(case):
    rows, cols, k = case["rows"], case["cols"], case["k"]
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["type"]]
    n = rows * cols
    if case["op"] == "top":
        return {"bytes": n * size + rows * k * 12 + rows * (12 if case["lse"] else 8) + 8, "flops": n * (4 if case["lse"] else 1)}
    if case["op"] == "balance":
        got = case["sequences"] * cols * 8 + 4
        return {"bytes": 2 * n * size + rows * k * 8 + rows * (9 if case["mask"] else 8) + got, "flops": 10 * n}
    stored, read = (rows * (7 / 16) * (k + 1), rows * 7 / 8) if case["ragged"] else (rows * k, rows)
    if case["weight"]:                                                               # a row that is not counted need not be read
        stored, read = stored * 2 / 3, read * 2 / 3
    return {"bytes": read * cols * size + (n * size if case["grad"] else 0) + stored * 12 + rows * (20 if case["rest"] else 16),
            "flops": read * cols * (8 if case["grad"] else 4)}


def exact(case, seed):
    s = prepare(case, seed)
    x, rows, cols = s["x"], case["rows"], case["cols"]
    if case["op"] == "top":
        val, lse = [], []
        for part in x.split(max(1, (1 << 26) // cols)):
            u = part.double()
            least = torch.topk(u, case["k"], dim=1).values[:, -1:]                   # the value of the last one that is taken
            more = u > least
            same = (u == least) & (torch.cumsum(u == least, 1) <= case["k"] - more.sum(1, keepdim=True))
            val.append(u[more | same])
            if case["lse"]:
                lse.append(torch.logsumexp(u / case["temperature"], 1))
        return {"pos": None, "crd": None, "val": torch.cat(val), "lse": torch.cat(lse) if lse else None}
    pos, crd = s["pos"].cpu(), s["crd"]
    step = max(1, (1 << 26) // cols)
    if case["op"] == "balance":
        seq = [0, rows] if s["seq"] is None else s["seq"].tolist()
        chosen = torch.zeros((rows, cols), dtype=torch.float64, device="cuda")
        of = torch.repeat_interleave(torch.arange(rows, device="cuda"), s["pos"].diff())
        chosen[of, crd] = 1
        if s["mask"] is not None:
            chosen *= s["mask"][:, None]
        active = (chosen.sum(1) > 0).double()
        r = x.double()
        used = [(a, b) for a, b in zip(seq, seq[1:]) if b > a and float(active[a:b].sum()) > 0]
        loss, grad = torch.zeros((), dtype=torch.float64, device="cuda"), torch.zeros_like(r)
        for a, b in used:
            score = torch.softmax(r[a:b], 1) if case["scores"] == "softmax" else torch.sigmoid(r[a:b]) / torch.sigmoid(r[a:b]).sum(1, keepdim=True)
            share = chosen[a:b].sum(0) / chosen[a:b].sum()
            by = _scale(case) * cols / len(used) / active[a:b].sum() * active[a:b]
            inner = score @ share
            loss += by @ inner
            slope = share[None, :] - inner[:, None]
            if case["scores"] == "sigmoid":
                slope = slope * torch.sigmoid(-r[a:b])
            grad[a:b] = by[:, None] * score * slope
        return {"loss": loss, "counts": None, "grad": grad}

    tau = case["temperature"]
    losses, grads = [], []
    for a in range(0, rows, step):
        b = min(rows, a + step)
        lo, hi = int(pos[a]), int(pos[b])
        of = torch.repeat_interleave(torch.arange(b - a, device="cuda"), s["pos"][a:b + 1].diff())
        teacher = torch.full((b - a, cols), -math.inf, dtype=torch.float64, device="cuda")
        teacher[of, crd[lo:hi]] = s["val"][lo:hi].double() / tau
        stored = torch.isfinite(teacher)
        has = stored.any(1)
        logq = torch.log_softmax(x[a:b].double() / tau, 1)
        norm = s["lse"][a:b].double() if case["rest"] else torch.where(has, torch.logsumexp(teacher, 1), torch.zeros(b - a, dtype=torch.float64, device="cuda"))
        logp = teacher - norm[:, None]
        p = logp.exp()
        loss = torch.where(stored, p * (logp - logq), torch.zeros_like(p)).sum(1)
        grad = logq.exp() - p
        if case["rest"]:
            left = (1 - p.sum(1)).clamp(min=0)
            q_left = torch.where(stored, torch.zeros_like(p), logq.exp()).sum(1)
            loss = loss + torch.where(left > 0, left * (left / q_left).log(), torch.zeros_like(left))
            grad = torch.where(stored, grad, logq.exp() * (1 - left / q_left)[:, None])
        weight = has.double() if s["weight"] is None else has * s["weight"][a:b].double()
        losses.append(torch.where(weight != 0, loss, torch.zeros_like(loss)))
        if case["grad"]:
            grads.append(grad * (weight * _scale(case) / tau)[:, None])
    losses = torch.cat(losses)
    weight = torch.ones_like(losses) if s["weight"] is None else s["weight"].double()
    return {"loss": (losses * weight).sum() * _scale(case), "rows": losses, "grad": torch.cat(grads) if case["grad"] else None}

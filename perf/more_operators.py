"""Operators of a language model with routed experts, around a CSR matrix: log probabilities of given tokens with entropy and the
best alternatives, and their gradient; the gated feed-forward block of the experts that a router has chosen, the sum of
their outputs for each token, and the gradients of both.

The operands are in GPU memory.  Logits are what the last product of a model gives (normal, spread 2.5, a few columns of each
row well above the rest); the given tokens are a CSR matrix of the logits' shape, of which only the columns count.  A router's
choices are a CSR matrix too (rows tokens, columns experts, values the weights of the experts' outputs); some experts are
liked better than others, and padding stores nothing.
"""
import math

import torch

own = False

TYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_LOGITS = 4096 * 131072              # elements of the largest matrix of logits
MOST_PRODUCT = 65536 * 2048 * 1024       # entries x width x inner of the largest experts


def listed():
    return [
        # The answer's next token, as a server reports it: its log probability and the 20 best alternatives.  Latency.
        {"name": "logp_one_token", "op": "logp", "rows": 1, "cols": 131072, "given": 1, "ragged": False, "type": "bf16", "temperature": 1.0,
         "entropy": False, "top": 20},
        # A micro-batch of sampled answers, scored for a policy gradient: log probability of each token and the row's entropy.
        {"name": "logp_rollout", "op": "logp", "rows": 4096, "cols": 131072, "given": 1, "ragged": False, "type": "bf16", "temperature": 1.0,
         "entropy": True, "top": 0},
        # Scoring with alternatives: an odd vocabulary (rows at every alignment), prompts' rows without a token, candidates of several tokens.
        {"name": "logp_alternatives", "op": "logp", "rows": 1021, "cols": 50021, "given": 5, "ragged": True, "type": "f16", "temperature": 0.7,
         "entropy": True, "top": 20},
        # The gradient of a policy loss with an entropy bonus.
        {"name": "logp_grad_step", "op": "logp_grad", "rows": 4096, "cols": 131072, "given": 1, "ragged": False, "type": "bf16", "temperature": 1.0,
         "entropy": True},
        # The same in f32, with an odd vocabulary and several candidates a row.
        {"name": "logp_grad_odd_f32", "op": "logp_grad", "rows": 509, "cols": 50021, "given": 5, "ragged": True, "type": "f32", "temperature": 2.0,
         "entropy": False},
        # One new token through 8 of 64 experts: the weights are read, latency counts.
        {"name": "gated_one_token", "op": "gated", "rows": 1, "experts": 64, "chosen": 8, "width": 2048, "inner": 1024, "type": "bf16",
         "ragged": False, "activation": "silu"},
        # A long batch through the same experts.
        {"name": "gated_batch", "op": "gated", "rows": 8192, "experts": 64, "chosen": 8, "width": 2048, "inner": 1024, "type": "bf16",
         "ragged": False, "activation": "silu"},
        # Few experts of odd widths, f16, a part of the tokens padding.
        {"name": "gated_odd_f16", "op": "gated", "rows": 777, "experts": 10, "chosen": 3, "width": 1000, "inner": 712, "type": "f16",
         "ragged": True, "activation": "gelu"},
        # The backward pass of a micro-batch.
        {"name": "gated_grad_step", "op": "gated_grad", "rows": 4096, "experts": 32, "chosen": 4, "width": 2048, "inner": 1024, "type": "bf16",
         "ragged": True, "activation": "silu"},
        # The outputs of one token's experts, summed with the router's weights.
        {"name": "combine_one_token", "op": "combine", "rows": 1, "experts": 64, "chosen": 8, "width": 2048, "inner": 1024, "type": "bf16",
         "ragged": False},
        # The same for the long batch.
        {"name": "combine_batch", "op": "combine", "rows": 8192, "experts": 64, "chosen": 8, "width": 2048, "inner": 1024, "type": "bf16",
         "ragged": False},
        # Its backward pass for a micro-batch: the inner rows, the experts' weights and the router's.
        {"name": "combine_grad_step", "op": "combine_grad", "rows": 4096, "experts": 32, "chosen": 4, "width": 2048, "inner": 1024, "type": "bf16",
         "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: from one token to a micro-batch; vocabularies, experts and widths over their range."""
    op = rng.choice(["logp", "logp", "logp_grad", "gated", "gated_grad", "combine", "combine_grad"])
    if op.startswith("logp"):
        kind = rng.choice(["bf16", "bf16", "f16", "f32"])
        short = rng.random() < 0.2                                                   # a router's scores or a classifier's
        cols = _log(rng, 8, 2048) if short else _log(rng, 4096, 160000)
        rows = _log(rng, 1, 32768 if short else max(1, min(8192, MOST_LOGITS // (cols * (2 if kind == "f32" else 1)))))
        c = {"op": op, "rows": rows, "cols": cols, "given": rng.choice([1, 1, rng.randint(1, 8)]), "ragged": rng.random() < 0.4, "type": kind,
             "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]), "entropy": rng.random() < 0.5}
        if op == "logp":
            c["top"] = rng.choice([0, 0, rng.randint(1, 20)]) if cols >= 32 else 0
            if c["top"] and rows * cols > 1 << 26:                                   # the plain form sorts whole rows
                c["rows"] = max(1, (1 << 26) // cols)
        return c
    experts = _log(rng, 1, 128)
    chosen = rng.randint(1, min(8, experts))
    width, inner = 8 * _log(rng, 8, 512), 8 * _log(rng, 8, 256)
    experts = max(chosen, min(experts, (64 * 2048 * 1024) // (width * inner)))
    most = MOST_PRODUCT // (1 if op in ("gated", "combine") else 4)
    rows = _log(rng, 1, max(1, min(8192, most // (chosen * width * inner))))
    c = {"op": op, "rows": rows, "experts": experts, "chosen": chosen, "width": width, "inner": inner, "type": rng.choice(["bf16", "bf16", "f16"]),
         "ragged": rows > 8 and rng.random() < 0.5}
    if op.startswith("gated"):
        c["activation"] = rng.choice(["silu", "silu", "gelu"])
    return c


def _scale(case):
    """Losses are means over the batch; f16 gradients are scaled up, as training in f16 does."""
    return (4096.0 if case["type"] == "f16" else 1.0) / case["rows"]


def _counts(case, k, uniform):
    """How many entries each row stores.  Ragged: a case's counts are always the same ones (so results have one shape), in an order of the seed's: one row in
    eight stores nothing (a prompt's, padding), and of the others some have fewer than k (candidates: any number; choices: a tenth were dropped)."""
    rows = case["rows"]
    i = torch.arange(rows, device="cuda")
    counts = torch.full((rows,), k, device="cuda")
    if case["ragged"]:
        fewer = 1 + i // 8 * 5 % k if case["op"].startswith("logp") else torch.where(i // 8 % 10 == 9, i // 80 % k, counts)
        counts = torch.where(i % 8 == 7, torch.zeros_like(counts), fewer)[uniform(rows).argsort()]
    return counts


def _csr(counts, columns):
    """pos and crd of a matrix that stores the first counts[t] of columns[t], columns ascending."""
    rows, k = columns.shape
    pos = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
    pos[1:] = torch.cumsum(counts, 0)
    keep = torch.arange(k, device="cuda")[None, :] < counts[:, None]
    return pos, torch.where(keep, columns, torch.full_like(columns, 1 << 40)).sort(dim=1).values[keep]


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    rows, kind = case["rows"], TYPE[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")          # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=g, device="cuda")          # noqa: E731
    s = {"case": case}
    if case["op"].startswith("logp"):
        cols, k = case["cols"], case["given"]
        x = s["x"] = torch.empty((rows, cols), dtype=kind, device="cuda")
        step = max(1, (1 << 26) // cols)
        for r in range(0, rows, step):                                               # in pieces: f32 normals of all of it would be large
            x[r:r + step] = normal(min(step, rows - r), cols) * 2.5
        k = min(k, cols)
        # the given tokens and a few others are likely ones: a column in each of n equal stretches, so distinct
        n = min(cols, max(k, cols // 4096))
        hot = ((torch.arange(n, device="cuda") + uniform(rows, n)).double() * (cols / n)).to(torch.int64).clamp_(max=cols - 1)
        x.scatter_(1, hot, (normal(rows, n) * 3 + 5).to(kind))
        given = hot.gather(1, uniform(rows, n).argsort(dim=1)[:, :k])
        s["pos"], s["crd"] = _csr(_counts(case, k, uniform), given)
        if case["op"] == "logp_grad":                                                # what the forward pass has kept, and the gradients that come in
            sums, entropy = [], []
            for r in range(0, rows, step):
                u = x[r:r + step].double() / case["temperature"]
                m = u.amax(1, keepdim=True)
                e = (u - m).exp()
                total = e.sum(1)
                sums.append(torch.stack([x[r:r + step].amax(1).float(), total.log().float()], 1))
                entropy.append((total.log() - (e * (u - m)).sum(1) / total).float())
            s["sums"], s["entropy"] = torch.cat(sums), torch.cat(entropy)
            s["d_values"] = normal(s["crd"].shape[0]) * _scale(case)
            s["d_entropy"] = (0.2 + 0.1 * uniform(rows)) * _scale(case) if case["entropy"] else None
        return s

    experts, chosen, width, inner = case["experts"], case["chosen"], case["width"], case["inner"]
    scores = normal(rows, experts) + 0.5 * normal(experts)
    best = torch.topk(scores, chosen, dim=1).indices
    s["pos"], s["crd"] = _csr(_counts(case, chosen, uniform), best)
    entries = s["crd"].shape[0]
    s["val"] = 0.05 + uniform(entries) / chosen
    # rows for the fullest expert, as a program that pads its batches knows it
    s["room"] = int(torch.bincount(s["crd"], minlength=experts).max())
    make = lambda scale, *shape: (normal(*shape) * scale).to(kind)                  # noqa: E731
    if case["op"].startswith("gated"):
        s["x"] = make(1.0, rows, width)
        s["w"] = torch.empty((experts, 2 * inner, width), dtype=kind, device="cuda")
        for e in range(experts):
            s["w"][e] = normal(2 * inner, width) * width ** -0.5
        if case["op"] == "gated_grad":
            s["d_h"] = make(_scale(case), entries, inner)
    else:
        s["h"] = make(0.5, entries, inner)
        s["v"] = torch.empty((experts, width, inner), dtype=kind, device="cuda")
        for e in range(experts):
            s["v"][e] = normal(width, inner) * inner ** -0.5
        if case["op"] == "combine_grad":
            s["d_y"] = make(_scale(case), rows, width)
    return s


def run(state):
    c = state["case"]
    if own:
        return _own(state, c)
    return {"logp": _plain_logp, "logp_grad": _plain_logp_grad, "gated": _plain_gated, "gated_grad": _plain_gated_grad, "combine": _plain_combine,
            "combine_grad": _plain_combine_grad}[c["op"]](state, c)


def _own(s, c):
    from comet_b200 import device
    if c["op"].startswith("logp"):
        given = device.DeviceCSR(c["rows"], c["cols"], s["pos"], s["crd"], None)
        if c["op"] == "logp_grad":
            return {"grad": device.log_probs_grad(given, s["x"], s["sums"], s["d_values"], entropy=s["entropy"], d_entropy=s["d_entropy"],
                                                  temperature=c["temperature"])}
        values, sums, entropy, best = device.log_probs(given, s["x"], temperature=c["temperature"], entropy=c["entropy"], top=c["top"])
        return {"values": values, "sums": sums, "entropy": entropy, "crd": best.crd if best else None, "best": best.val if best else None}
    groups = device.group_entries(device.DeviceCSR(c["rows"], c["experts"], s["pos"], s["crd"], s["val"]))
    if c["op"] == "gated":
        return {"h": device.gated_experts(groups, s["x"], s["w"], activation=c["activation"])}
    if c["op"] == "gated_grad":
        d_x, d_w = device.gated_experts_grad(groups, s["x"], s["w"], s["d_h"], activation=c["activation"])
        return {"d_x": d_x, "d_w": d_w}
    if c["op"] == "combine":
        return {"y": device.combine_experts(groups, s["h"], s["v"])}
    d_h, d_v, d_values = device.combine_experts_grad(groups, s["h"], s["v"], s["d_y"])
    return {"d_h": d_h, "d_v": d_v, "d_values": d_values}


def _row_of(s, rows):
    return torch.repeat_interleave(torch.arange(rows, device="cuda"), s["pos"][1:] - s["pos"][:-1], output_size=s["crd"].shape[0])


def _plain_logp(s, c):
    x, tau = s["x"].float(), c["temperature"]
    m = x.amax(1)
    u = (x - m[:, None]) / tau
    e = u.exp()
    total = e.sum(1)
    log = total.log()
    row = _row_of(s, c["rows"])
    out = {"values": u.reshape(-1)[row * c["cols"] + s["crd"]] - log[row], "sums": torch.stack([m, log], 1),
           "entropy": log - (e * u).sum(1) / total if c["entropy"] else None, "crd": None, "best": None}
    if c["top"]:
        crd = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["top"]].sort(dim=1).values
        out["crd"], out["best"] = crd.reshape(-1), (u.gather(1, crd) - log[:, None]).reshape(-1)
    return out


def _plain_logp_grad(s, c):
    tau, row = c["temperature"], _row_of(s, c["rows"])
    logq = (s["x"].float() - s["sums"][:, :1]) / tau - s["sums"][:, 1:]
    q = logq.exp()
    given = torch.zeros(c["rows"], device="cuda").index_add_(0, row, s["d_values"])
    grad = -q * given[:, None]
    grad.reshape(-1)[row * c["cols"] + s["crd"]] += s["d_values"]
    if c["entropy"]:
        grad -= s["d_entropy"][:, None] * q * (logq + s["entropy"][:, None])
    return {"grad": (grad / tau).to(s["x"].dtype)}


def _places(s, c):
    """For the entries in the experts' order: entry, its token, its place in a batch of the experts' padded rows."""
    column, order = torch.sort(s["crd"], stable=True)
    counts = torch.zeros(c["experts"], dtype=torch.int64, device="cuda").index_add_(0, column, torch.ones_like(column))
    first = torch.cumsum(counts, 0) - counts
    place = column * s["room"] + torch.arange(column.shape[0], device="cuda") - first[column]
    return order, _row_of(s, c["rows"])[order], place


def _padded(s, c, place, rows):
    out = torch.zeros((c["experts"] * s["room"], rows.shape[1]), device="cuda")
    out[place] = rows.float()
    return out.view(c["experts"], s["room"], -1)


def _in_order(order, rows, kind):
    out = torch.empty(rows.shape, dtype=kind, device="cuda")
    out[order] = rows.to(kind)
    return out


def _activation(g, kind):
    """The activation and its slope."""
    if kind == "silu":
        t = 1 / (1 + (-g).exp())
        return g * t, t * (1 + g * (1 - t))
    a, b = math.sqrt(2 / math.pi), 0.044715
    t = torch.tanh(a * (g + b * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * b * g * g)


def _plain_gated(s, c):
    order, token, place = _places(s, c)
    z = torch.bmm(_padded(s, c, place, s["x"][token]), s["w"].float().transpose(1, 2)).view(-1, 2 * c["inner"])[place]
    h = _activation(z[:, :c["inner"]], c["activation"])[0] * z[:, c["inner"]:]
    return {"h": _in_order(order, h, s["x"].dtype)}


def _plain_gated_grad(s, c):
    order, token, place = _places(s, c)
    x, w = _padded(s, c, place, s["x"][token]), s["w"].float()
    z = torch.bmm(x, w.transpose(1, 2)).view(-1, 2 * c["inner"])[place]
    act, slope = _activation(z[:, :c["inner"]], c["activation"])
    d_h = s["d_h"][order].float()
    d_z = _padded(s, c, place, torch.cat([d_h * z[:, c["inner"]:] * slope, d_h * act], 1))
    d_x = torch.zeros((c["rows"], c["width"]), device="cuda").index_add_(0, token, torch.bmm(d_z, w).view(-1, c["width"])[place])
    return {"d_x": d_x.to(s["x"].dtype), "d_w": torch.bmm(d_z.transpose(1, 2), x).to(s["x"].dtype)}


def _plain_combine(s, c):
    order, token, place = _places(s, c)
    out = torch.bmm(_padded(s, c, place, s["h"][order]), s["v"].float().transpose(1, 2)).view(-1, c["width"])[place]
    y = torch.zeros((c["rows"], c["width"]), device="cuda").index_add_(0, token, s["val"][order][:, None] * out)
    return {"y": y.to(s["h"].dtype)}


def _plain_combine_grad(s, c):
    order, token, place = _places(s, c)
    weight = s["val"][order][:, None]
    d_y, h = s["d_y"][token].float(), s["h"][order].float()
    back = torch.bmm(_padded(s, c, place, d_y), s["v"].float()).view(-1, c["inner"])[place]
    d_v = torch.bmm(_padded(s, c, place, d_y * weight).transpose(1, 2), _padded(s, c, place, h))
    return {"d_h": _in_order(order, back * weight, s["h"].dtype), "d_v": d_v.to(s["h"].dtype),
            "d_values": _in_order(order, (back * h).sum(1, keepdim=True), torch.float32).reshape(-1)}


def work(case):
    size = 4 if case["type"] == "f32" else 2
    rows, op = case["rows"], case["op"]
    if op.startswith("logp"):
        n, k = rows * case["cols"], min(case["given"], case["cols"])
        stored = rows * (7 / 16) * (k + 1) if case["ragged"] else rows * k
        if op == "logp":
            return {"bytes": n * size + stored * 12 + rows * (20 if case["entropy"] else 16) + rows * case["top"] * 12,
                    "flops": n * (6 if case["entropy"] else 4)}
        return {"bytes": 2 * n * size + stored * 12 + rows * (24 if case["entropy"] else 16), "flops": n * (6 if case["entropy"] else 3)}
    experts, width, inner = case["experts"], case["width"], case["inner"]
    entries = rows * case["chosen"] * (7 / 8 * 0.95 if case["ragged"] else 1)
    used = experts * (1 - (1 - 1 / experts) ** entries)                              # experts with a token
    each = used * width * inner * size                                               # the bytes of one matrix of them
    routes = entries * 8 + rows * 8
    product = 2 * entries * width * inner
    if op == "gated":
        return {"bytes": routes + rows * width * size + 2 * each + entries * inner * size, "flops": 2 * product}
    if op == "gated_grad":
        return {"bytes": routes + 2 * rows * width * size + 2 * each + 2 * experts * width * inner * size + entries * inner * size,
                "flops": 6 * product}
    if op == "combine":
        return {"bytes": routes + entries * 4 + entries * inner * size + each + rows * width * size, "flops": product}
    return {"bytes": routes + entries * 8 + rows * width * size + 2 * entries * inner * size + each + experts * width * inner * size,
            "flops": 2 * product}


def _exact_logp(case, s):
    x, tau, cols = s["x"], case["temperature"], case["cols"]
    pos = s["pos"].cpu()
    found = {"values": [], "sums": [], "entropy": [], "best": [], "grad": []}
    step = max(1, (1 << 26) // cols)
    for a in range(0, case["rows"], step):
        b = min(case["rows"], a + step)
        lo, hi = int(pos[a]), int(pos[b])
        of = torch.repeat_interleave(torch.arange(b - a, device="cuda"), s["pos"][a:b + 1].diff())
        part = x[a:b].double()
        logq = torch.log_softmax(part / tau, 1)
        entropy = torch.special.entr(logq.exp()).sum(1)
        if case["op"] == "logp":
            found["values"].append(logq[of, s["crd"][lo:hi]])
            found["sums"].append(torch.stack([part.amax(1), torch.logsumexp((part - part.amax(1, keepdim=True)) / tau, 1)], 1))
            found["entropy"].append(entropy)
            if case["top"]:
                least = torch.topk(part, case["top"], dim=1).values[:, -1:]          # the value of the last one that is taken
                more, same = part > least, part == least
                same &= torch.cumsum(same, 1) <= case["top"] - more.sum(1, keepdim=True)
                found["best"].append(logq[more | same])
            continue
        came = torch.zeros_like(logq)
        came[of, s["crd"][lo:hi]] = s["d_values"][lo:hi].double()
        grad = came - logq.exp() * came.sum(1, keepdim=True)
        if case["entropy"]:
            grad -= s["d_entropy"][a:b, None].double() * logq.exp() * (logq + entropy[:, None])
        found["grad"].append(grad / tau)
    if case["op"] == "logp_grad":
        return {"grad": torch.cat(found["grad"])}
    return {"values": torch.cat(found["values"]), "sums": torch.cat(found["sums"]), "entropy": torch.cat(found["entropy"]) if case["entropy"] else None,
            "crd": None, "best": torch.cat(found["best"]) if case["top"] else None}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("logp"):
        return _exact_logp(case, s)
    pos = s["pos"]
    token = torch.searchsorted(pos, torch.arange(s["crd"].shape[0], device="cuda"), right=True) - 1
    inner, width, rows = case["inner"], case["width"], case["rows"]
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.float64, device="cuda")    # noqa: E731
    entries = token.shape[0]
    out = {"gated": lambda: {"h": zeros(entries, inner)}, "gated_grad": lambda: {"d_x": zeros(rows, width), "d_w": zeros(*s["w"].shape)},
           "combine": lambda: {"y": zeros(rows, width)},
           "combine_grad": lambda: {"d_h": zeros(entries, inner), "d_v": zeros(*s["v"].shape), "d_values": zeros(entries)}}[case["op"]]()
    for e in range(case["experts"]):
        at = (s["crd"] == e).nonzero().reshape(-1)
        if not at.shape[0]:
            continue
        t = token[at]
        if case["op"].startswith("gated"):
            x, w = s["x"][t].double(), s["w"][e].double()
            gate, up = x @ w[:inner].T, x @ w[inner:].T
            gate.requires_grad_()
            with torch.enable_grad():
                act = torch.nn.functional.silu(gate) if case["activation"] == "silu" else torch.nn.functional.gelu(gate, approximate="tanh")
                h = act * up
            if case["op"] == "gated":
                out["h"][at] = h.detach()
                continue
            d_h = s["d_h"][at].double()
            d_gate, = torch.autograd.grad(h, gate, d_h)
            d_up = d_h * act.detach()
            out["d_x"][t] += d_gate @ w[:inner] + d_up @ w[inner:]                   # a token has an expert once
            out["d_w"][e] = torch.cat([d_gate.T @ x, d_up.T @ x])
            continue
        h, v, weight = s["h"][at].double(), s["v"][e].double(), s["val"][at].double()[:, None]
        if case["op"] == "combine":
            out["y"][t] += weight * (h @ v.T)
            continue
        d_y = s["d_y"][t].double()
        out["d_h"][at] = weight * (d_y @ v)
        out["d_v"][e] = (weight * d_y).T @ h
        out["d_values"][at] = (d_y * (h @ v.T)).sum(1)
    return out

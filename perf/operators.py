"""Cases of the token operators (``ebr_b200.token_ops``): the scaled embedding with its gradient, tokens sorted by expert
and back, and the distillation loss on a teacher's top logits.

``listed`` gives the fixed cases, ``draw`` more of the same ranges, ``prepare`` a case's inputs on the GPU, ``run`` one
pass (the plain torch form, or the framework's calls where ``own`` is true), ``exact`` the same in float64 from the
definitions, and ``work`` the bytes and operations that a pass cannot do without.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
MOST_BYTES = 1.6e9  # a drawn case's pass moves no more than this (the largest listed one moves 2.1e9)


def listed():
    return [
        # One 9 x 9 board embedded for inference: a call that is all latency.
        {"name": "embed_one_board", "op": "embed", "n": 81, "vocab": 10, "dim": 512, "wtype": "fp32", "otype": "bf16",
         "ids": "board", "train": False},
        # The training batch of the sudoku network: 768 boards, every gradient row falls on one of ten table rows.
        {"name": "embed_boards_train", "op": "embed", "n": 62208, "vocab": 10, "dim": 512, "wtype": "fp32",
         "otype": "bf16", "ids": "board", "train": True},
        # A batch of text over a large vocabulary, word frequencies, padding ids: the table's gradient is the traffic.
        {"name": "embed_text_train", "op": "embed", "n": 16384, "vocab": 131072, "dim": 2048, "wtype": "bf16",
         "otype": "bf16", "ids": "zipf", "train": True},
        # Odd sizes: rows that are no multiple of 16 bytes, few repeats.
        {"name": "embed_odd_train", "op": "embed", "n": 5003, "vocab": 50021, "dim": 771, "wtype": "fp16",
         "otype": "fp16", "ids": "uniform", "train": True},
        # One board through a sparse MLP's routing at inference: latency.
        {"name": "experts_one_board", "op": "experts", "tokens": 81, "experts": 8, "topk": 2, "dim": 512,
         "type": "bf16", "capacity": 0, "train": False},
        # The sudoku training batch through eight experts, two per token, forward and backward.
        {"name": "experts_boards_train", "op": "experts", "tokens": 62208, "experts": 8, "topk": 2, "dim": 512,
         "type": "bf16", "capacity": 0, "train": True},
        # Many small experts and eight per token, as wide sparse layers have them; forward.
        {"name": "experts_wide", "op": "experts", "tokens": 16384, "experts": 64, "topk": 8, "dim": 2048,
         "type": "bf16", "capacity": 0, "train": False},
        # Odd sizes with a fixed capacity per expert, slots over it dropped, float32.
        {"name": "experts_odd_capacity_train", "op": "experts", "tokens": 3001, "experts": 60, "topk": 6, "dim": 999,
         "type": "fp32", "capacity": 320, "train": True},
        # The sudoku training batch's decoded logits: many rows of ten; a loss for each row, and its backward.
        {"name": "distill_boards_rows", "op": "distill", "rows": 62208, "vocab": 10, "topk": 4, "type": "bf16",
         "tau": 1.0, "mode": "rows", "empty": 0.3, "masked": False},
        # Text tokens of a training step over a large vocabulary, the stored 64 best of a teacher, prompts left out.
        {"name": "distill_text_train", "op": "distill", "rows": 4096, "vocab": 131072, "topk": 64, "type": "bf16",
         "tau": 2.0, "mode": "mean", "empty": 0.1, "masked": False},
        # Odd vocabulary, float32 logits, a vocabulary mask of -inf, row weights.
        {"name": "distill_odd_train", "op": "distill", "rows": 777, "vocab": 50021, "topk": 20, "type": "fp32",
         "tau": 1.5, "mode": "weighted", "empty": 0.1, "masked": True},
        # A few positions scored without a gradient: few rows, a long axis.
        {"name": "distill_few_rows", "op": "distill", "rows": 12, "vocab": 151665, "topk": 32, "type": "fp16",
         "tau": 1.0, "mode": "eval", "empty": 0.0, "masked": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "experts", "distill"])
    if op == "embed":
        vocab = _log_int(rng, 2, 140000)
        c = {"op": op, "n": _log_int(rng, 1, 200000), "vocab": vocab, "dim": _log_int(rng, 16, 4100),
             "wtype": rng.choice(["fp32", "bf16", "fp16"]), "ids": rng.choice(["board", "zipf", "uniform"]),
             "train": rng.random() < 0.7}
        c["otype"] = c["wtype"] if rng.random() < 0.5 else rng.choice(["bf16", "fp32"])
        if rng.random() < 0.6:
            c["dim"] = max(16, c["dim"] // 64 * 64)
        most, key, least = MOST_BYTES, "n", 1
        if work(dict(c, n=1))["bytes"] > most:
            c["vocab"] = max(2, vocab // 4)
    elif op == "experts":
        experts = _log_int(rng, 2, 500)
        topk = min(experts, _log_int(rng, 1, 10))
        c = {"op": op, "tokens": _log_int(rng, 1, 80000), "experts": experts, "topk": topk,
             "dim": _log_int(rng, 16, 4100), "type": rng.choice(["fp32", "bf16", "bf16", "fp16"]), "capacity": 0,
             "train": rng.random() < 0.6}
        if rng.random() < 0.6:
            c["dim"] = max(16, c["dim"] // 64 * 64)
        if rng.random() < 0.4:
            c["capacity"] = -1  # set below, from the final number of tokens
        most, key, least = MOST_BYTES, "tokens", 1
    else:
        vocab = _log_int(rng, 2, 152000)
        c = {"op": op, "rows": _log_int(rng, 1, 70000), "vocab": vocab, "topk": min(vocab, _log_int(rng, 1, 128)),
             "type": rng.choice(["bf16", "bf16", "fp32", "fp16"]), "tau": rng.choice([1.0, 1.3, 2.0, 4.0]),
             "mode": rng.choice(["mean", "rows", "weighted", "eval"]), "empty": rng.choice([0.0, 0.1, 0.5]),
             "masked": rng.random() < 0.3}
        if c["rows"] < 64:  # a few rows: none of them without an entry
            c["empty"], c["masked"] = 0.0, False
        if c["type"] == "fp16" and c["mode"] == "mean":
            c["mode"] = "rows"  # a mean over many rows leaves float16's range without a loss scale
        most, key, least = MOST_BYTES, "rows", 64
    spent = work(dict(c, capacity=0) if c.get("capacity") else c)["bytes"]
    if spent > most:
        c[key] = max(least, int(c[key] * most / spent * 0.9))
    if c.get("capacity"):
        mean = c["tokens"] * c["topk"] / c["experts"]
        c["capacity"] = max(1, int(mean * rng.uniform(0.8, 1.5)))
    return c


# ------------------------------------------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _draw_ids(kind, n, vocab, g):
    """Token ids: board cells (mostly the blank, id 0), word frequencies, or even; -1 pads one in twenty of the latter."""
    u = torch.rand(n, generator=g, device=DEV)
    if kind == "board":
        other = torch.randint(1, max(2, vocab), (n,), generator=g, device=DEV).clamp_(max=vocab - 1)
        return torch.where(u < 0.7, torch.zeros_like(other), other)
    ids = (vocab ** u - 1).long() if kind == "zipf" else (u * vocab).long()  # density ~ 1 / (id + 1), or even
    ids = ids.clamp_(0, vocab - 1)
    pad = torch.rand(n, generator=g, device=DEV) < 0.05
    pad[0] = False
    return torch.where(pad, torch.full_like(ids, -1), ids)


def prepare(case, seed):
    g = _gen(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    st = {"case": case}
    if case["op"] == "embed":
        st["tokens"] = _draw_ids(case["ids"], case["n"], case["vocab"], g)
        st["scale"] = math.sqrt(case["dim"])
        w = randn(case["vocab"], case["dim"]) * case["dim"] ** -0.5
        st["weight"] = w.to(TYPES[case["wtype"]]).requires_grad_(case["train"])
        if case["train"]:
            st["gout"] = randn(case["n"], case["dim"]).to(TYPES[case["otype"]])
    elif case["op"] == "experts":
        t, e, k, c, dt = (case[x] for x in ("tokens", "experts", "topk", "dim", "type"))
        dt = TYPES[dt]
        # a router's scores: some experts are liked more than others
        score = randn(t, e) + 0.7 * randn(1, e)
        top, ids = score.topk(k, dim=1)
        dropped = torch.rand(t, k, generator=g, device=DEV) < 0.02
        dropped[0, 0] = False
        st["ids"] = torch.where(dropped, torch.full_like(ids, -1), ids)
        st["weights"] = top.softmax(dim=1).requires_grad_(case["train"])
        st["x"] = randn(t, c).to(dt).requires_grad_(case["train"])
        rows = e * case["capacity"] if case["capacity"] else t * k
        st["y"] = randn(rows, c).to(dt).requires_grad_(case["train"])  # what the experts made of their rows
        if case["train"]:
            st["grows"] = randn(rows, c).to(dt)
            st["gout"] = randn(t, c).to(dt)
    else:
        n, v, k, dt = case["rows"], case["vocab"], case["topk"], TYPES[case["type"]]
        # k distinct ids a row: a random start and random steps that add up to less than the vocabulary
        step = max(1, v // k)
        steps = torch.randint(1, step + 1, (n, k), generator=g, device=DEV)
        start = torch.randint(0, v, (n, 1), generator=g, device=DEV)
        ids = (start + steps.cumsum(1) - steps[:, :1]) % v
        top = (randn(n, k) * 3 + 4).sort(dim=1, descending=True).values
        logits = randn(n, v) * 1.5
        logits.scatter_add_(1, ids, 0.8 * top)
        if case["masked"]:  # a part of the vocabulary that the student may not use
            logits[:, torch.rand(v, generator=g, device=DEV) < 0.1] = float("-inf")
            keep = torch.isfinite(logits.gather(1, ids))
            ids = torch.where(keep, ids, torch.full_like(ids, -1))
        empty = torch.rand(n, 1, generator=g, device=DEV) < case["empty"]
        short = torch.arange(k, device=DEV) >= torch.randint(1, 2 * k + 1, (n, 1), generator=g, device=DEV)
        st["ids"] = torch.where(empty | short, torch.full_like(ids, -1), ids)
        st["top"] = top.to(dt)
        st["logits"] = logits.to(dt).requires_grad_(case["mode"] != "eval")
        if case["mode"] == "rows":
            st["gout"] = torch.rand(n, generator=g, device=DEV) + 0.5
        if case["mode"] == "weighted":
            st["row_weight"] = torch.rand(n, generator=g, device=DEV) + 0.5
    return st


# ------------------------------------------------------------------------------------------------------- plain forms


def _plain_embed(st):
    case, w, ids = st["case"], st["weight"].detach(), st["tokens"]
    v = case["vocab"]
    ok = (ids >= 0) & (ids < v)
    at = torch.where(ok, ids, torch.zeros_like(ids))
    out = w[at].float() * st["scale"] * ok.unsqueeze(1)
    out = out.to(TYPES[case["otype"]])
    if not case["train"]:
        return [out]
    dw = torch.zeros(v, case["dim"], device=DEV)
    dw.index_add_(0, at, st["gout"].float() * ok.unsqueeze(1))
    return [out, (dw * st["scale"]).to(w.dtype)]


def _plain_experts(st):
    case, x, y, w, ids = st["case"], st["x"].detach(), st["y"].detach(), st["weights"].detach(), st["ids"]
    t, k, e, cap = case["tokens"], case["topk"], case["experts"], case["capacity"]
    flat = ids.reshape(-1)
    ok = (flat >= 0) & (flat < e)
    key = torch.where(ok, flat, torch.full_like(flat, e))
    order = key.sort(stable=True).indices
    counts = torch.zeros(e + 1, dtype=torch.int64, device=DEV).index_add_(0, key, torch.ones_like(key))
    offsets = torch.zeros(e + 1, dtype=torch.int64, device=DEV)
    offsets[1:] = counts[:e].cumsum(0)
    place = torch.empty_like(order)
    place[order] = torch.arange(t * k, device=DEV)
    if cap:
        rank = place - offsets[key]
        ok = ok & (rank < cap)
        place = key * cap + rank
        rows = e * cap
    else:
        rows = t * k
    row_of = torch.where(ok, place, torch.full_like(place, -1))
    at = row_of.clamp(min=0)
    token = torch.arange(t, device=DEV).repeat_interleave(k)
    live = ok.unsqueeze(1)

    def spread(per_slot):  # rows of slots -> rows of experts; rows of no slot are zeros
        out = torch.zeros(rows + 1, case["dim"], device=DEV)
        out[torch.where(ok, place, torch.full_like(place, rows))] = per_slot
        return out[:rows]

    sent = spread(x.float()[token]).to(x.dtype)
    got = y[at].float() * live
    back = (got * w.reshape(-1, 1)).view(t, k, -1).sum(1).to(x.dtype)
    outs = [row_of.view(t, k).int(), offsets.int(), sent, back]
    if case["train"]:
        gout = st["gout"].float()
        dx = (st["grows"][at].float() * live).view(t, k, -1).sum(1).to(x.dtype)
        dy = spread(gout[token] * w.reshape(-1, 1)).to(y.dtype)
        dw = (got.view(t, k, -1) * gout.unsqueeze(1)).sum(2)
        outs += [dx, dy, dw]
    return outs


def _plain_distill(st):
    case, s, ids, tau = st["case"], st["logits"].detach().float(), st["ids"], st["case"]["tau"]
    n, v = s.shape
    ok = (ids >= 0) & (ids < v)
    any_ok = ok.any(1)
    at = torch.where(ok, ids, torch.zeros_like(ids))
    t = torch.where(ok, st["top"].float() / tau, torch.full_like(s[:1, :1], float("-inf")))
    tmax = torch.where(any_ok, t.max(1).values, torch.zeros_like(t[:, 0])).unsqueeze(1)
    num = (t - tmax).exp() * ok
    total = torch.where(any_ok, num.sum(1), torch.ones_like(num[:, 0])).unsqueeze(1)
    p = num / total
    logp = t - tmax - total.log()
    smax = s.max(1, keepdim=True).values
    ex = ((s - smax) / tau).exp()
    sums = ex.sum(1, keepdim=True)
    logq = (s.gather(1, at) - smax) / tau - sums.log()
    terms = torch.where(p > 0, p * (logp - logq), torch.zeros_like(p))
    rows = tau * tau * terms.sum(1)
    if case["mode"] == "eval":
        return [rows]
    if case["mode"] == "rows":
        g, loss = st["gout"], rows
    elif case["mode"] == "weighted":
        g = st["row_weight"]
        loss = (rows * g).sum()
    else:
        g = torch.full((n,), 1.0 / n, device=DEV)
        loss = rows.mean()
    coef = (g * tau * any_ok).unsqueeze(1)
    grad = torch.where(any_ok.unsqueeze(1), ex * (coef / sums), torch.zeros_like(ex))
    grad.scatter_add_(1, at, -coef * p)
    return [loss, grad.to(st["logits"].dtype)]


# ------------------------------------------------------------------------------------------------------- the framework's calls


def _own_embed(st):
    from ebr_b200.token_ops import scaled_embedding

    case, w = st["case"], st["weight"]
    out = scaled_embedding(st["tokens"], w, st["scale"], TYPES[case["otype"]])
    if not case["train"]:
        return [out]
    (dw,) = torch.autograd.grad(out, w, st["gout"])
    return [out, dw]


def _own_experts(st):
    from ebr_b200.token_ops import expert_combine, expert_dispatch, expert_route

    case, x, y, w = st["case"], st["x"], st["y"], st["weights"]
    route = expert_route(st["ids"], case["experts"], case["capacity"] or None)
    sent = expert_dispatch(x, route)
    back = expert_combine(y, route, w)
    outs = [route.row_of, route.offsets, sent, back]
    if case["train"]:
        outs += torch.autograd.grad([sent, back], [x, y, w], [st["grows"], st["gout"]])
    return outs


def _own_distill(st):
    from ebr_b200.token_ops import topk_distill_loss

    case, s, mode = st["case"], st["logits"], st["case"]["mode"]
    how = {"eval": "none", "rows": "none", "weighted": "sum", "mean": "mean"}[mode]
    loss = topk_distill_loss(s, st["ids"], st["top"], case["tau"], row_weight=st.get("row_weight"), reduction=how)
    if mode == "eval":
        return [loss]
    (grad,) = torch.autograd.grad(loss, s, st.get("gout"))
    return [loss, grad]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"embed": _own_embed, "experts": _own_experts, "distill": _own_distill}[op](state)
    with torch.no_grad():
        return {"embed": _plain_embed, "experts": _plain_experts, "distill": _plain_distill}[op](state)


# ------------------------------------------------------------------------------------------------------- float64


def _exact_embed(st):
    case, ids = st["case"], st["tokens"]
    table = torch.cat([st["weight"].detach().double(), torch.zeros(1, case["dim"], device=DEV, dtype=torch.float64)])
    at = ids.masked_fill((ids < 0) | (ids >= case["vocab"]), case["vocab"])
    out = torch.nn.functional.embedding(at, table) * st["scale"]
    if not case["train"]:
        return [out]
    # sums over sorted tokens: differences of segment-wise sums, one id's tokens at a time through a sparse product
    one = torch.sparse_coo_tensor(torch.stack([at, torch.arange(case["n"], device=DEV)]),
                                  torch.ones(case["n"], device=DEV, dtype=torch.float64),
                                  (case["vocab"] + 1, case["n"]), check_invariants=False)  # fmt: skip
    dw = torch.sparse.mm(one, st["gout"].double()) * st["scale"]
    return [out, dw[: case["vocab"]]]


def _exact_experts(st):
    case, ids = st["case"], st["ids"].cpu()
    t, k, e, cap, c = (case[x] for x in ("tokens", "topk", "experts", "capacity", "dim"))
    flat = ids.reshape(-1)
    row_of = torch.full((t * k,), -1, dtype=torch.int64)
    offsets, begin = [0], 0
    for expert in range(e):  # each expert's slots in their own order
        mine = (flat == expert).nonzero().squeeze(1)
        kept = mine[:cap] if cap else mine
        row_of[kept] = torch.arange(len(kept)) + (expert * cap if cap else begin)
        begin += len(mine)
        offsets.append(begin)
    rows = e * cap if cap else t * k
    row_of = row_of.view(t, k).to(DEV)
    d = lambda a: a.detach().double()  # noqa: E731
    x, y, w = d(st["x"]), d(st["y"]), d(st["weights"])
    sent = torch.zeros(rows + 1, c, device=DEV, dtype=torch.float64)
    back = torch.zeros(t, c, device=DEV, dtype=torch.float64)
    pad = torch.cat([y, torch.zeros(1, c, device=DEV, dtype=torch.float64)])
    for j in range(k):
        sent.index_copy_(0, row_of[:, j].masked_fill(row_of[:, j] < 0, rows), x)
        back.addcmul_(pad[row_of[:, j]], w[:, j : j + 1])
    outs = [None, None, sent[:rows], back]
    if case["train"]:
        gout = d(st["gout"])
        gpad = torch.cat([d(st["grows"]), torch.zeros(1, c, device=DEV, dtype=torch.float64)])
        dx, dy = torch.zeros_like(x), torch.zeros(rows + 1, c, device=DEV, dtype=torch.float64)
        dw = torch.zeros_like(w)
        for j in range(k):
            dx += gpad[row_of[:, j]]
            dy.index_copy_(0, row_of[:, j].masked_fill(row_of[:, j] < 0, rows), gout * w[:, j : j + 1])
            dw[:, j] = torch.einsum("tc,tc->t", pad[row_of[:, j]], gout)
        outs += [dx, dy[:rows], dw]
    return outs


def _exact_distill(st):
    case, ids, tau = st["case"], st["ids"], st["case"]["tau"]
    n, v = case["rows"], case["vocab"]
    mode = case["mode"]
    g = {"rows": st.get("gout"), "weighted": st.get("row_weight"), "mean": torch.full((n,), 1.0 / n, device=DEV),
         "eval": None}[mode]  # fmt: skip
    grad = None if mode == "eval" else torch.empty(n, v, device=DEV, dtype=torch.float64)
    losses = torch.empty(n, device=DEV, dtype=torch.float64)
    size = max(1, int(1.5e8) // v)
    for a in range(0, n, size):
        b = min(n, a + size)
        logq = torch.log_softmax(st["logits"][a:b].detach().double() / tau, dim=1)
        valid = ids[a:b] >= 0
        t = (st["top"][a:b].double() / tau).masked_fill(~valid, float("-inf"))
        logp = (t - torch.logsumexp(t, dim=1, keepdim=True)).masked_fill(~valid, 0.0)
        p = logp.exp().masked_fill(~valid, 0.0)
        mine = torch.gather(logq, 1, ids[a:b].clamp(min=0)).masked_fill(~valid, 0.0)
        losses[a:b] = tau**2 * (p * (logp - mine)).sum(1)
        if grad is not None:
            part = logq.exp().masked_fill(~valid.any(1, keepdim=True), 0.0)
            part.scatter_add_(1, ids[a:b].clamp(min=0), -p)
            grad[a:b] = part * (tau * g[a:b].double().unsqueeze(1))
    if mode == "eval":
        return [losses]
    if mode == "rows":
        return [losses, grad]
    return [(losses * g.double()).sum(), grad]


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    return {"embed": _exact_embed, "experts": _exact_experts, "distill": _exact_distill}[case["op"]](st)


# ------------------------------------------------------------------------------------------------------- work


def work(case):
    if case["op"] == "embed":
        n, v, c = case["n"], case["vocab"], case["dim"]
        ws, os_ = SIZE[case["wtype"]], SIZE[case["otype"]]
        total = 8 * n + min(n, v) * c * ws + n * c * os_
        flops = n * c
        if case["train"]:
            total += n * c * os_ + v * c * ws
            flops += 2 * n * c
        return {"bytes": total, "flops": flops}
    if case["op"] == "experts":
        t, k, c, e = case["tokens"], case["topk"], case["dim"], case["experts"]
        size = SIZE[case["type"]]
        rows = e * case["capacity"] if case["capacity"] else t * k
        live = min(rows, t * k)
        # ids, weights, the row numbers and offsets; x once and its rows; the rows once and their sums
        total = 16 * t * k + 4 * e + (2 * t + rows + live) * c * size
        flops = 2 * t * k * c
        if case["train"]:
            # rows' gradient -> dx; dout and the rows -> the rows' gradient and the weights'
            total += 8 * t * k + (2 * t + 2 * live + rows) * c * size
            flops += 4 * t * k * c
        return {"bytes": total, "flops": flops}
    n, v, k, size = case["rows"], case["vocab"], case["topk"], SIZE[case["type"]]
    read = (1 - case["empty"]) * n * v * size  # a row without a teacher's entry needs no logits
    total, flops = read + n * k * (8 + size) + 4 * n, 4 * n * v
    if case["mode"] != "eval":
        total, flops = total + n * v * size, flops + 2 * n * v
    return {"bytes": total, "flops": flops}

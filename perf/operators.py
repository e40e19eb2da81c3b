"""Cases of the operators whose rows choose their own weights: rows sorted by group and back (`group_rows`,
`gather_rows_`, `combine_rows_` and the gradients), products of row groups (`gemm_grouped_` and its gradients), and
low-rank adapters of many requests beside a shared projection (`gemm_lora_`).

`run` makes the calls of the library where `own` is true; otherwise it computes the same in elementary torch
operations in 32 bits.  `exact` is a third form in 64 bits."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One decoding step of a few requests through a layer of many small experts: launches and latency.
        {"name": "rows_step", "op": "rows", "tokens": 16, "choices": 8, "groups": 128, "width": 2048, "type": "bf16", "dropped": 0.0, "train": False},
        # A batch of prompts through the same layer: one read and eight writes of every token, and back.
        {"name": "rows_prompts", "op": "rows", "tokens": 16384, "choices": 8, "groups": 128, "width": 2048, "type": "bf16", "dropped": 0.0, "train": False},
        # A training step of a layer with few wide experts: there and back, and both gradients.
        {"name": "rows_training", "op": "rows", "tokens": 8192, "choices": 2, "groups": 8, "width": 4096, "type": "bf16", "dropped": 0.0, "train": True},
        # Odd sizes, rows that no 16-byte access fits, and choices that capacity has dropped.
        {"name": "rows_odd", "op": "rows", "tokens": 2039, "choices": 3, "groups": 17, "width": 1001, "type": "f32", "dropped": 0.1, "train": True},
        # The experts' products of a decoding step: one or two rows a group, every weight is streamed once.
        {"name": "grouped_step", "op": "grouped", "rows": 128, "groups": 64, "n": 2048, "k": 2048, "type": "bf16", "out": "bf16", "empty": 0.1, "train": False},
        # The experts' products of a batch of prompts, routed unevenly: bound by the tensor cores.
        {"name": "grouped_prompts", "op": "grouped", "rows": 32768, "groups": 32, "n": 4096, "k": 2048, "type": "bf16", "out": "bf16", "empty": 0.0, "train": False},
        # Their gradients in training, with respect to the rows and to every group's weight.
        {"name": "grouped_training", "op": "grouped", "rows": 16384, "groups": 8, "n": 4096, "k": 4096, "type": "bf16", "out": "bf16", "empty": 0.0, "train": True},
        # Ragged groups, some of them empty, sizes that fill no tile, Float32 outputs and weight gradients.
        {"name": "grouped_odd", "op": "grouped", "rows": 1537, "groups": 13, "n": 1000, "k": 1336, "type": "f16", "out": "f32", "empty": 0.3, "train": True},
        # One token of one request beside a projection: latency alone.
        {"name": "lora_token", "op": "lora", "tokens": 1, "requests": 1, "adapters": 4, "rank": 16, "n": 4096, "k": 4096, "type": "bf16", "out": "bf16"},
        # A decoding step of many requests that use many adapters.
        {"name": "lora_step", "op": "lora", "tokens": 128, "requests": 128, "adapters": 64, "rank": 16, "n": 4096, "k": 4096, "type": "bf16", "out": "bf16"},
        # Prompts of several requests: bound by reading the rows and adding to the projection's output.
        {"name": "lora_prompts", "op": "lora", "tokens": 16384, "requests": 24, "adapters": 12, "rank": 64, "n": 4096, "k": 4096, "type": "bf16", "out": "bf16"},
        # Single tokens beside short prompts, sizes that fill no tile, a Float32 output.
        {"name": "lora_odd", "op": "lora", "tokens": 777, "requests": 37, "adapters": 9, "rank": 24, "n": 2056, "k": 1000, "type": "f16", "out": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["f16", "bf16"])
    op = rng.choice(["rows", "grouped", "lora"])
    if op == "rows":
        choices, width = rng.randint(1, 8), _log(rng, 64, 8192)
        tokens = _log(rng, 1, max(1, min(16384, (1 << 27) // (choices * width))))
        return {"op": "rows", "tokens": tokens, "choices": choices, "groups": _log(rng, max(choices, 2), 256), "width": width,
                "type": rng.choice(["f32", "f16", "bf16"]), "dropped": rng.choice([0.0, 0.0, 0.25]), "train": rng.random() < 0.5}
    if op == "grouped":
        groups, n, k = _log(rng, 1, 64), 8 * _log(rng, 8, 512), 8 * _log(rng, 8, 512)
        while groups * n * k > 1 << 28:
            groups = max(1, groups // 2)
        rows = _log(rng, 1, max(1, min(32768, (1 << 37) // (n * k))))
        return {"op": "grouped", "rows": rows, "groups": groups, "n": n, "k": k, "type": kind,
                "out": rng.choice([kind, "f32"]), "empty": rng.choice([0.0, 0.2]), "train": rng.random() < 0.5}
    tokens = _log(rng, 1, 12000)
    return {"op": "lora", "tokens": tokens, "requests": _log(rng, 1, min(tokens, 128)), "adapters": _log(rng, 1, 64),
            "rank": 8 * rng.randint(1, 8), "n": 8 * _log(rng, 16, 640), "k": 8 * _log(rng, 16, 640), "type": kind, "out": rng.choice([kind, "f32"])}


# ---------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _offsets(counts):
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    dt = TYPES[case["type"]]
    if case["op"] == "rows":
        t, c, e, h = case["tokens"], case["choices"], case["groups"], case["width"]
        # a router's choices: some groups are liked more than others; a token's choices differ
        logits = torch.randn(t, e, generator=gen, device="cuda") + torch.randn(e, generator=gen, device="cuda")
        top, ids = logits.topk(c, dim=1)
        s["weights"] = torch.softmax(top, dim=1)
        s["ids"] = torch.where(torch.rand(t, c, generator=gen, device="cuda") < case["dropped"], -1, ids)
        s["x"] = _randn(gen, t, h, dtype=dt)
        s["ys"] = _randn(gen, t * c, h, dtype=dt)
        s["gathered"] = torch.zeros(t * c, h, dtype=dt, device="cuda")
        s["combined"] = torch.empty(t, h, dtype=dt, device="cuda")
        if case["train"]:
            s["d_combined"] = _randn(gen, t, h, dtype=dt)
            s["d_gathered"] = _randn(gen, t * c, h, dtype=dt)
            s["d_ys"] = torch.zeros(t * c, h, dtype=dt, device="cuda")
            s["d_weights"] = torch.empty(t, c, device="cuda")
            s["d_x"] = torch.empty(t, h, dtype=dt, device="cuda")
    elif case["op"] == "grouped":
        r, g, n, k = case["rows"], case["groups"], case["n"], case["k"]
        out = TYPES[case["out"]]
        liked = torch.randn(g, generator=gen, device="cuda") * 0.7
        gone = torch.rand(g, generator=gen, device="cuda") < case["empty"]
        liked = torch.where(gone & ~gone.all(), torch.full_like(liked, -math.inf), liked)
        to = torch.multinomial(torch.softmax(liked, 0), r, replacement=True, generator=gen)
        counts = torch.zeros(g, dtype=torch.int64, device="cuda").index_add_(0, to, torch.ones_like(to))
        s["offsets"], s["longest"] = _offsets(counts), int(counts.max())
        s["b"] = _randn(gen, g, n, k, dtype=dt, scale=1 / math.sqrt(k))
        s["a"] = _randn(gen, r, k, dtype=dt)
        if case["train"]:
            s["d"] = _randn(gen, r, n, dtype=dt)
            s["d_a"] = torch.zeros(r, k, dtype=out, device="cuda")
            s["d_b"] = torch.zeros(g, n, k, dtype=out, device="cuda")
        else:
            s["d"] = torch.zeros(r, n, dtype=out, device="cuda")
    else:
        t, q, n, k, rank = case["tokens"], case["requests"], case["n"], case["k"], case["rank"]
        cuts = torch.randperm(t - 1, generator=gen, device="cuda")[: q - 1].sort().values + 1 if q > 1 else torch.zeros(0, dtype=torch.int64, device="cuda")
        edges = torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), t)])
        s["offsets"], s["longest"] = edges.to(torch.int32), int((edges[1:] - edges[:-1]).max())
        # one request in eight, but never the first, has no adapter
        which = torch.randint(0, case["adapters"], (q,), generator=gen, device="cuda", dtype=torch.int32)
        none = (torch.rand(q, generator=gen, device="cuda") < 0.125) & (torch.arange(q, device="cuda") > 0)
        s["which"] = torch.where(none, torch.full_like(which, -1), which)
        s["scales"] = torch.rand(case["adapters"], generator=gen, device="cuda") + 0.5
        s["x"] = _randn(gen, t, k, dtype=dt)
        s["a"] = _randn(gen, case["adapters"], rank, k, dtype=dt, scale=1 / math.sqrt(k))
        s["b"] = _randn(gen, case["adapters"], n, rank, dtype=dt, scale=1 / math.sqrt(rank))
        s["c"] = _randn(gen, t, n, dtype=TYPES[case["out"]])
        s["d"] = torch.empty(t, n, dtype=TYPES[case["out"]], device="cuda")
    return s


# ---------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    return {"rows": _plain_rows, "grouped": _plain_grouped, "lora": _plain_lora}[s["op"]](s)


def _own(s):
    from __graft_entry__ import load_package
    mb = load_package()
    if s["op"] == "rows":
        plan = mb.group_rows(s["ids"], s["groups"])
        mb.gather_rows_(s["gathered"], s["x"], plan)
        mb.combine_rows_(s["combined"], s["ys"], plan, s["weights"])
        out = {"order": plan.order, "offsets": plan.offsets, "inverse": plan.inverse, "gathered": s["gathered"], "combined": s["combined"]}
        if s["train"]:
            mb.combine_rows_grad_(s["d_ys"], s["d_weights"], s["d_combined"], s["ys"], plan, s["weights"])
            mb.combine_rows_(s["d_x"], s["d_gathered"], plan)
            out.update(d_ys=s["d_ys"], d_weights=s["d_weights"], d_x=s["d_x"])
        return out
    if s["op"] == "grouped":
        if not s["train"]:
            return {"d": mb.gemm_grouped_(s["d"], s["a"], s["b"], s["offsets"])}
        mb.gemm_grouped_(s["d_a"], s["d"], s["b"].transpose(1, 2), s["offsets"])
        mb.gemm_grouped_grad_(s["d_b"], s["d"], s["a"], s["offsets"])
        return {"d_a": s["d_a"], "d_b": s["d_b"]}
    if s["c"].dtype == torch.float32:  # a Float32 sum is added to in place, as the plain form does
        return {"d": mb.gemm_lora_(s["c"], s["x"], s["a"], s["b"], s["which"], s["offsets"], scales=s["scales"])}
    return {"d": mb.gemm_lora_(s["d"], s["x"], s["a"], s["b"], s["which"], s["offsets"], scales=s["scales"], C=s["c"])}


def _plain_rows(s):
    ids, e, dt = s["ids"], s["groups"], s["x"].dtype
    t, c = ids.shape
    flat = ids.reshape(-1)
    kept = (flat >= 0) & (flat < e)
    key = torch.where(kept, flat, torch.full_like(flat, e))
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(e + 1, dtype=torch.int64, device="cuda").index_add_(0, key, torch.ones_like(key))
    offsets = _offsets(counts[:e])
    place = torch.empty_like(order)
    place[order] = torch.arange(t * c, device="cuda")
    live = torch.arange(t * c, device="cuda") < offsets[e]
    gathered = torch.where(live[:, None], s["x"][order // c], torch.zeros((), dtype=dt, device="cuda"))
    w = torch.where(kept.view(t, c), s["weights"], torch.zeros((), device="cuda"))
    mine = s["ys"].float()[place].view(t, c, -1)
    out = {"order": torch.where(live, order, -1).to(torch.int32), "offsets": offsets, "inverse": torch.where(kept, place, -1).to(torch.int32).view(t, c),
           "gathered": gathered, "combined": (mine * w[:, :, None]).sum(1).to(dt)}
    if s["train"]:
        dy = s["d_combined"].float()
        d_ys = torch.where(live[:, None], dy[order // c] * w.reshape(-1)[order][:, None], torch.zeros((), device="cuda"))
        d_w = torch.where(kept.view(t, c), (mine * dy[:, None, :]).sum(2), torch.zeros((), device="cuda"))
        d_x = (s["d_gathered"].float()[place].view(t, c, -1) * kept.view(t, c, 1)).sum(1)
        out.update(d_ys=d_ys.to(dt), d_weights=d_w, d_x=d_x.to(dt))
    return out


def _padded(offsets, longest):
    """Row numbers of every group beside one another, and which of them are the group's own."""
    at = torch.arange(longest, device="cuda")[None, :]
    own_row = at < (offsets[1:] - offsets[:-1])[:, None]
    return torch.where(own_row, offsets[:-1, None] + at, torch.zeros_like(at)).long(), own_row


def _pick(x, at, own_row):
    return x.float()[at] * own_row[:, :, None]


def _plain_grouped(s):
    at, own_row = _padded(s["offsets"], s["longest"])
    w = s["b"].float()
    if not s["train"]:
        d = torch.zeros(s["rows"], s["n"], device="cuda")
        d[at[own_row]] = torch.bmm(_pick(s["a"], at, own_row), w.transpose(1, 2))[own_row]
        return {"d": d.to(s["d"].dtype)}
    dd = _pick(s["d"], at, own_row)
    d_a = torch.zeros(s["rows"], s["k"], device="cuda")
    d_a[at[own_row]] = torch.bmm(dd, w)[own_row]
    d_b = torch.bmm(dd.transpose(1, 2), _pick(s["a"], at, own_row))
    return {"d_a": d_a.to(s["d_a"].dtype), "d_b": d_b.to(s["d_b"].dtype)}


def _plain_lora(s):
    at, own_row = _padded(s["offsets"], s["longest"])
    which = s["which"].long()
    has = own_row & (which >= 0)[:, None]
    w = which.clamp(min=0)
    v = torch.bmm(_pick(s["x"], at, own_row), s["a"].float()[w].transpose(1, 2))
    u = torch.bmm(v, s["b"].float()[w].transpose(1, 2)) * s["scales"][w][:, None, None]
    d = s["c"].float()
    d[at[has]] += u[has]
    return {"d": d.to(s["d"].dtype)}


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    b = BYTES[case["type"]]
    if case["op"] == "rows":
        t, c, e, h = case["tokens"], case["choices"], case["groups"], case["width"]
        n = t * c
        kept = n * (1 - case["dropped"])
        bytes_ = n * 8 + n * 4 * 2 + (e + 1) * 4 + (t + kept) * h * b + n * 4 + (kept + t) * h * b
        flops = 2 * kept * h
        if case["train"]:
            bytes_ += (t + 2 * kept) * h * b + n * 8 + (kept + t) * h * b
            flops += 4 * kept * h
        return {"bytes": bytes_, "flops": flops}
    if case["op"] == "grouped":
        r, g, n, k = case["rows"], case["groups"], case["n"], case["k"]
        o = BYTES[case["out"]]
        live = max(1.0, g * (1 - case["empty"]))
        used = live * (1 - (1 - 1 / live) ** r)  # weights that some row asks for
        if not case["train"]:
            return {"bytes": r * k * b + used * n * k * b + r * n * o, "flops": 2.0 * r * n * k}
        return {"bytes": r * (n + k) * b + used * n * k * b + r * k * o + g * n * k * o, "flops": 4.0 * r * n * k}
    t, q, n, k, rank = case["tokens"], case["requests"], case["n"], case["k"], case["rank"]
    o = BYTES[case["out"]]
    share = 1 - 0.125 * (q - 1) / q
    used = case["adapters"] * (1 - (1 - 1 / case["adapters"]) ** (q * share))
    return {"bytes": t * share * k * b + used * rank * (n + k) * b + 2 * t * n * o, "flops": 2.0 * t * share * rank * (n + k)}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        return _exact_rows(s)
    edge = s["offsets"].tolist()
    if case["op"] == "grouped":
        if s["train"]:
            d_a = torch.zeros(s["rows"], s["k"], dtype=torch.float64, device="cuda")
            d_b = torch.zeros(s["groups"], s["n"], s["k"], dtype=torch.float64, device="cuda")
            for g in range(s["groups"]):
                lo, hi = edge[g], edge[g + 1]
                d_a[lo:hi] = s["d"][lo:hi].double() @ s["b"][g].double()
                d_b[g] = s["d"][lo:hi].double().T @ s["a"][lo:hi].double()
            return {"d_a": d_a, "d_b": d_b}
        d = torch.zeros(s["rows"], s["n"], dtype=torch.float64, device="cuda")
        for g in range(s["groups"]):
            d[edge[g]:edge[g + 1]] = s["a"][edge[g]:edge[g + 1]].double() @ s["b"][g].double().T
        return {"d": d}
    d = s["c"].double()
    for q, which in enumerate(s["which"].tolist()):
        if which >= 0:
            lo, hi = edge[q], edge[q + 1]
            d[lo:hi] += s["scales"][which].double() * ((s["x"][lo:hi].double() @ s["a"][which].double().T) @ s["b"][which].double().T)
    return {"d": d}


def _exact_rows(s):
    ids, e = s["ids"].cpu(), s["groups"]
    t, c = ids.shape
    flat = ids.reshape(-1).tolist()
    order, edge = [], [0]
    members = [[] for _ in range(e)]
    for i, g in enumerate(flat):
        if 0 <= g < e:
            members[g].append(i)
    for m in members:
        order += m
        edge.append(len(order))
    n = len(order)
    at = torch.tensor(order, dtype=torch.int64, device="cuda")
    inverse = torch.full((t * c,), -1, dtype=torch.int64, device="cuda")
    inverse[at] = torch.arange(n, device="cuda")
    h = s["width"]
    gathered = torch.zeros(t * c, h, dtype=torch.float64, device="cuda")
    gathered[:n] = s["x"].double()[at // c]
    combined = torch.zeros(t, h, dtype=torch.float64, device="cuda")
    w = s["weights"].double().reshape(-1)
    ys, inv = s["ys"], inverse.view(t, c)
    out = {"order": torch.cat([at, at.new_full((t * c - n,), -1)]), "offsets": torch.tensor(edge), "inverse": inv, "gathered": gathered, "combined": combined}
    if s["train"]:
        dy = s["d_combined"].double()
        out["d_ys"] = torch.zeros(t * c, h, dtype=torch.float64, device="cuda")
        out["d_ys"][:n] = dy[at // c] * w[at][:, None]
        out["d_weights"] = torch.zeros(t, c, dtype=torch.float64, device="cuda")
        out["d_x"] = torch.zeros(t, h, dtype=torch.float64, device="cuda")
    for j in range(c):
        has = inv[:, j] >= 0
        rows = inv[has, j]
        combined[has] += ys[rows].double() * s["weights"][has, j].double()[:, None]
        if s["train"]:
            out["d_weights"][has, j] = (ys[rows].double() * dy[has]).sum(1)
            out["d_x"][has] += s["d_gathered"][rows].double()
    return out

"""Cases that measure the serving operators: the page planner, the cache writer, the rotary positions and the
attention of new tokens over a paged cache.

``run`` computes each operator either in its plain form (elementary torch operations in 32 bits, 64 for angles) or,
with ``own`` set, through this package's public calls.  A case is a dict of plain values; request lengths and draft
trees follow from the case itself (its ``mix``), values from the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1}
E4M3_MAX = 448.0


def listed():
    return [
        # One decode step of a serving batch: every request grows by a token, some into a new page.
        {"name": "plan decode b64", "op": "plan", "B": 64, "tokens": 64, "page": 16, "held": 4096, "mix": 1},
        # Admission of prompts next to requests that finish and give their pages back.
        {"name": "plan prompts b500", "op": "plan", "B": 500, "tokens": 65536, "page": 64, "held": 2048, "mix": 2},
        # The decode step's keys and values into the pages.
        {"name": "append decode bf16 t64", "op": "append", "tokens": 64, "Hkv": 8, "D": 128, "page": 16, "pages": 4096,
         "type": "bf16", "cache": "bf16", "rows": False},
        # A long prompt's keys and values quantised into an e4m3 cache, by accepted rows.
        {"name": "append prompt e4m3 t16384", "op": "append", "tokens": 16384, "Hkv": 8, "D": 128, "page": 64,
         "pages": 300, "type": "bf16", "cache": "e4m3", "rows": True},
        # Decode step of a model with time, height and width positions.
        {"name": "rotary decode 3 axes t64", "op": "rotary", "B": 0, "N": 64, "Hq": 32, "Hkv": 8, "D": 128, "dim": 128,
         "axes": 3, "type": "bf16", "interleaved": False, "neighbours": False, "grad": False, "far": 100000},
        # Long-sequence training step, forward and backward, on the package's longest workload.
        {"name": "rotary train n16384", "op": "rotary", "B": 1, "N": 16384, "Hq": 32, "Hkv": 32, "D": 128, "dim": 128,
         "axes": 3, "type": "bf16", "interleaved": True, "neighbours": False, "grad": True, "far": 16384},
        # One user, one token: latency counts.
        {"name": "decode b1 n1000", "op": "tree", "B": 1, "held": 1000, "new": 1, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 16, "type": "bf16", "cache": "bf16", "tree": False, "lse": False, "mix": 3},
        # Decode of a ragged serving batch.
        {"name": "decode b64 n8192", "op": "tree", "B": 64, "held": 8192, "new": 1, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 64, "type": "bf16", "cache": "bf16", "tree": False, "lse": False, "mix": 4},
        # Decode over an 8-bit cache.
        {"name": "decode e4m3 b100 n8192", "op": "tree", "B": 100, "held": 8192, "new": 1, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 64, "type": "bf16", "cache": "e4m3", "tree": False, "lse": False, "mix": 5},
        # Drafted trees, a head of keys for each head of queries.
        {"name": "tree48 f16 d64 b16", "op": "tree", "B": 16, "held": 4096, "new": 48, "Hq": 16, "Hkv": 16, "D": 64,
         "page": 32, "type": "f16", "cache": "f16", "tree": True, "lse": True, "mix": 6},
        # Drafted trees, grouped heads, long requests.
        {"name": "tree64 b8 n16384", "op": "tree", "B": 8, "held": 16384, "new": 64, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 64, "type": "bf16", "cache": "bf16", "tree": True, "lse": False, "mix": 7},
        # A chunk of a long prompt behind what is cached of it.
        {"name": "chunk2048 b2 n8192", "op": "tree", "B": 2, "held": 8192, "new": 2048, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 128, "type": "bf16", "cache": "bf16", "tree": False, "lse": False, "mix": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "rotary", "tree", "tree", "tree"])
    mix = rng.randrange(1 << 30)
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        return {"op": op, "B": _log(rng, 1, 500), "tokens": _log(rng, 500, 65536), "page": page,
                "held": _log(rng, 100, 4096), "mix": mix}
    if op == "append":
        tokens = _log(rng, 1, 16384)
        kind = rng.choice(["bf16", "f16"])
        return {"op": op, "tokens": tokens, "Hkv": rng.choice([1, 2, 4, 5, 8]), "D": rng.choice([64, 128]), "page": page,
                "pages": tokens // page + 1 + _log(rng, 4, 100), "type": kind, "cache": rng.choice([kind, "e4m3"]),
                "rows": rng.random() < 0.5}
    if op == "rotary":
        d = rng.choice([64, 128])
        return {"op": op, "B": rng.choice([0, 1, 2]), "N": _log(rng, 1, 8000), "Hq": rng.choice([8, 12, 16, 32]),
                "Hkv": rng.choice([1, 2, 4, 8]), "D": d, "dim": rng.choice([d, d // 2]), "axes": rng.choice([1, 2, 3]),
                "type": rng.choice(["bf16", "f16", "f32"]), "interleaved": rng.random() < 0.5,
                "neighbours": rng.random() < 0.5, "grad": rng.random() < 0.5, "far": _log(rng, 1000, 1000000)}
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
    d, new = rng.choice([64, 128]), rng.choice([1, 1, 1, _log(rng, 2, 64), _log(rng, 2, 64), _log(rng, 65, 1500)])
    kind = rng.choice(["bf16", "f16"])
    held = _log(rng, 50, 16384)
    most = int(1.0e9 / (held + new) / max(hkv * d * 8, new * hkv * group))
    return {"op": op, "B": min(100, _log(rng, 1, max(2, most))), "held": held, "new": new, "Hq": hkv * group, "Hkv": hkv,
            "D": d, "page": page, "type": kind, "cache": rng.choice([kind, kind, "e4m3"]) if d == 128 else kind,
            "tree": 1 < new <= 64 and rng.random() < 0.7, "lse": rng.random() < 0.5, "mix": mix}


# ---------------------------------------------------------------- what a case fixes beside its values
def _plan_lengths(c):
    """(held, wanted) tokens of each request: decode steps where there is a token a request, else finishing requests
    beside prompts that share the step's tokens."""
    rng = random.Random(c["mix"])
    B, tokens = c["B"], c["tokens"]
    held = [rng.randrange(0, c["held"] + 1) for _ in range(B)]
    if tokens == B:
        return held, [n + 1 for n in held]
    want, left = [], tokens
    for b, n in enumerate(held):
        kind = rng.random()
        if kind < 0.2:
            want.append(rng.choice([0, n // 2]))  # finished, or cut back
        else:
            most = left if b == B - 1 else min(left, 2 * tokens // B)
            new = rng.randrange(0, most + 1)
            left -= new
            want.append(n + new)
    return held, want


def _tree_lengths(c):
    """(cached, new) tokens of each request, ragged; the first request is the longest."""
    rng = random.Random(c["mix"])
    held = [c["held"]] + [rng.randrange(c["held"] // 8, c["held"] + 1) for _ in range(c["B"] - 1)]
    new = [c["new"]] + [rng.randrange(max(1, c["new"] // 2), c["new"] + 1) for _ in range(c["B"] - 1)]
    return held, new


def _ancestors(c, new):
    """Of each request, the list of each node's visible nodes: itself and its ancestors in a random draft tree."""
    rng = random.Random(c["mix"] + 1)
    seen = []
    for n in new:
        rows = []
        for j in range(n):
            parent = rng.randrange(max(-1, j - 8), j) if j else -1
            rows.append((rows[parent] if parent >= 0 else []) + [j])
        seen.append(rows)
    return seen


def _sections(c):
    """Frequency pairs of each axis."""
    half, axes = c["dim"] // 2, c["axes"]
    first = half - (axes - 1) * (half * 3 // (4 * axes))
    return [first] + [half * 3 // (4 * axes)] * (axes - 1)


def _pages(n, page):
    return (n + page - 1) // page


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = random.Random(seed)

    def normal(*shape, kind="bf16"):
        return torch.randn(shape, generator=g, device="cuda").to(DTYPES[kind])

    def ints(values, kind=torch.int32):
        return torch.tensor(values, dtype=kind, device="cuda")

    s = {"case": c}
    if c["op"] == "plan":
        held, want = _plan_lengths(c)
        page = c["page"]
        width = max(_pages(max(a, b), page) for a, b in zip(held, want)) + 3
        used = sum(_pages(n, page) for n in held)
        grown = sum(max(0, _pages(b, page) - _pages(a, page)) for a, b in zip(held, want))
        pages = used + grown + 17
        order = list(range(pages))
        rng.shuffle(order)
        table, at = [], 0
        for n in held:
            k = _pages(n, page)
            table.append(order[at:at + k] + [-1] * (width - k))
            at += k
        s["held"], s["want"], s["table"] = ints(held), ints(want), ints(table)
        s["free"], s["count"] = ints(order[used:] + [-1] * used), ints([pages - used])
        s["held_out"], s["count_out"] = torch.empty_like(s["held"]), torch.empty_like(s["count"])
    elif c["op"] == "append":
        T, H, D = c["tokens"], c["Hkv"], c["D"]
        n_slots = c["pages"] * c["page"]
        slots = torch.randperm(n_slots, generator=g, device="cuda")[:T]
        keep = torch.rand(T, generator=g, device="cuda") > 0.1  # a tenth of the rows go nowhere
        s["slots"] = torch.where(keep, slots, torch.full_like(slots, -1))
        s["k"], s["v"] = normal(T, H, D, kind=c["type"]), normal(T, H, D, kind=c["type"])
        s["rows"] = torch.randperm(T, generator=g, device="cuda").to(torch.int32) if c["rows"] else None
        shape = (c["pages"], H, c["page"], D)
        s["k_cache"], s["v_cache"] = normal(*shape, kind=c["cache"]), normal(*shape, kind=c["cache"])
        s["k_descale"], s["v_descale"] = (0.02, 0.015) if c["cache"] == "e4m3" else (1.0, 1.0)
    elif c["op"] == "rotary":
        lead = (c["N"],) if c["B"] == 0 else (c["B"], c["N"])
        q_shape = (c["N"], c["Hq"], c["D"]) if c["B"] == 0 else (c["B"], c["Hq"], c["N"], c["D"])
        k_shape = (c["N"], c["Hkv"], c["D"]) if c["B"] == 0 else (c["B"], c["Hkv"], c["N"], c["D"])
        s["q"], s["k"] = normal(*q_shape, kind=c["type"]), normal(*k_shape, kind=c["type"])
        s["positions"] = torch.randint(0, c["far"], (c["axes"], *lead), generator=g, device="cuda", dtype=torch.int32)
        if c["grad"]:
            s["gq"], s["gk"] = normal(*q_shape, kind=c["type"]), normal(*k_shape, kind=c["type"])
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
        # The table that a program lays out once: frequency and axis of each pair.
        s["freqs"] = 10000.0 ** (-torch.arange(c["dim"] // 2, dtype=torch.float64, device="cuda") * 2 / c["dim"])
        s["axes"] = ints(_axis_of_pair(c))
    else:
        held, new = _tree_lengths(c)
        page, H, D = c["page"], c["Hkv"], c["D"]
        counts = [_pages(n, page) for n in held]
        pages, width = sum(counts) + 5, max(counts) + 1
        order = list(range(pages))
        rng.shuffle(order)
        table, at = [], 0
        for k in counts:
            table.append(order[at:at + k] + [-1] * (width - k))
            at += k
        T = sum(new)
        s["table"], s["held"] = ints(table), ints(held)
        s["starts"] = ints([sum(new[:b]) for b in range(len(new) + 1)])
        s["q"] = normal(T, c["Hq"], D, kind=c["type"])
        s["k"], s["v"] = normal(T, H, D, kind=c["type"]), normal(T, H, D, kind=c["type"])
        s["k_cache"], s["v_cache"] = normal(pages, H, page, D, kind=c["cache"]), normal(pages, H, page, D, kind=c["cache"])
        s["k_descale"], s["v_descale"] = (0.9, 1.1) if c["cache"] == "e4m3" else (1.0, 1.0)
        s["scale"] = 1.0 / math.sqrt(D)
        s["mask"] = None
        if c["tree"]:
            mask = torch.ones(T, c["new"], dtype=torch.bool)
            t = 0
            for rows in _ancestors(c, new):
                for seen in rows:
                    mask[t, seen] = False
                    t += 1
            s["mask"] = mask.cuda()
    return s


def _package():
    import __graft_entry__
    return __graft_entry__.package()


# ---------------------------------------------------------------- one pass
def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(_package(), s, c)
    return {"plan": _plain_plan, "append": _plain_append, "rotary": _plain_rotary, "tree": _plain_tree}[c["op"]](s, c)


def _run_own(p, s, c):
    if c["op"] == "plan":
        r = p.cache_plan(s["held"], s["want"], s["table"], s["free"], s["count"], c["page"], c["tokens"],
                         lengths_out=s["held_out"], free_count_out=s["count_out"])
        return {"slots": r.slots, "positions": r.positions, "starts": r.starts, "lengths": r.lengths,
                "free_count": r.free_count, "table": s["table"], "free": s["free"]}
    if c["op"] == "append":
        p.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], rows=s["rows"],
                       k_descale=s["k_descale"], v_descale=s["v_descale"])
        return {"k": s["k_cache"], "v": s["v_cache"]}
    if c["op"] == "rotary":
        q, k = p.rotary(s["q"], s["k"], s["positions"], s["freqs"], s["axes"], neighbours=c["neighbours"])
        if not c["grad"]:
            return {"q": q, "k": k}
        gq, gk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return {"q": q.detach(), "k": k.detach(), "gq": gq, "gk": gk}
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda") if c["lse"] else None
    o = p.fused_tree(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["held"], s["starts"], s["scale"],
                     mask=s["mask"], max_new=c["new"], lse=lse, k_descale=s["k_descale"], v_descale=s["v_descale"])
    return {"o": o, "lse": lse} if c["lse"] else {"o": o}


def _plain_plan(s, c):
    held, want, table, free, page = s["held"].long(), s["want"].long(), s["table"].long(), s["free"].long(), c["page"]
    count, width, n_pages, dev = s["count"].long(), table.shape[1], free.shape[0], table.device
    old, new = (held + page - 1) // page, (want + page - 1) // page
    col = torch.arange(width, device=dev)
    dropped = (col >= new[:, None]) & (col < old[:, None])
    grown = (col >= old[:, None]) & (col < new[:, None])
    n_dropped, n_grown = dropped.sum(), grown.sum()
    # The stack with the released pages on top; one place more takes what belongs nowhere.
    rank = torch.cumsum(dropped.flatten(), 0) - 1
    at = torch.where(dropped.flatten(), count + rank, n_pages)
    stack = torch.cat([free, free.new_zeros(1)])
    stack[at.clamp(max=n_pages)] = table.flatten()
    left = count + n_dropped - n_grown
    ok = (left >= 0) & (new.max() <= width) & ((want - held).clamp(min=0).sum() <= c["tokens"])
    pop = (count + n_dropped - torch.cumsum(grown.flatten(), 0)).clamp(0, n_pages)
    table2 = torch.where(grown & ok, stack[pop].view_as(table), table)
    place = torch.arange(n_pages, device=dev)
    free2 = torch.where((place < left) & ok, stack[:n_pages], free)
    starts = torch.cat([held.new_zeros(1), torch.cumsum((want - held).clamp(min=0), 0)]) * ok
    i = torch.arange(c["tokens"], device=dev)
    b = torch.searchsorted(starts[1:].contiguous(), i, right=True).clamp(max=len(held) - 1)
    valid = i < starts[-1]
    pos = torch.where(valid, held[b] + i - starts[b], 0)
    slots = torch.where(valid, table2[b, pos // page] * page + pos % page, -1)
    return {"slots": slots, "positions": pos.int(), "starts": starts.int(), "lengths": torch.where(ok, want, held).int(),
            "free_count": torch.where(ok, left, count).int(), "table": table2.int(), "free": free2.int()}


def _plain_append(s, c):
    page = c["page"]
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    rows = s["rows"][keep].long() if s["rows"] is not None else keep.nonzero().flatten()
    p, o = slots // page, slots % page

    def put(cache, x, descale):
        x = x[rows].float() / descale
        if c["cache"] == "e4m3":
            x = x.clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
            cache.view(torch.uint8)[p, :, o] = x.view(torch.uint8)
        else:
            cache[p, :, o] = x.to(cache.dtype)

    put(s["k_cache"], s["k"], s["k_descale"])
    put(s["v_cache"], s["v"], s["v_descale"])
    return {"k": s["k_cache"], "v": s["v_cache"]}


def _axis_of_pair(c):
    """Axis whose position turns each pair: the sections one after another, or dealt in turn while they last."""
    sections = _sections(c)
    if not c["interleaved"]:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, axes, a = list(sections), [], 0
    while sum(left):
        if left[a]:
            axes.append(a)
            left[a] -= 1
        a = (a + 1) % len(sections)
    return axes


def _angles(s, c):
    angle = s["positions"].double()[s["axes"].long()].movedim(0, -1) * s["freqs"]  # [..., N, dim / 2]
    return angle[:, None, :] if c["B"] == 0 else angle[:, None]  # beside the heads


def _turned(x, cos, sin, c):
    """x with its first `dim` values turned pair by pair."""
    half, dim = c["dim"] // 2, c["dim"]
    a, b = (x[..., 0:dim:2], x[..., 1:dim:2]) if c["neighbours"] else (x[..., :half], x[..., half:dim])
    u, v = a * cos - b * sin, a * sin + b * cos
    pair = torch.stack([u, v], -1).flatten(-2) if c["neighbours"] else torch.cat([u, v], -1)
    return torch.cat([pair, x[..., dim:]], -1)


def _plain_rotary(s, c):
    angle = _angles(s, c)
    cos, sin = angle.cos().float(), angle.sin().float()
    r = {"q": _turned(s["q"].detach().float(), cos, sin, c).to(s["q"].dtype),
         "k": _turned(s["k"].detach().float(), cos, sin, c).to(s["k"].dtype)}
    if c["grad"]:  # the transpose of a turn is the turn back
        r["gq"] = _turned(s["gq"].float(), cos, -sin, c).to(s["q"].dtype)
        r["gk"] = _turned(s["gk"].float(), cos, -sin, c).to(s["k"].dtype)
    return r


def _plain_tree(s, c):
    B, H, D, page, M = c["B"], c["Hkv"], c["D"], c["page"], c["new"]
    group, T, dev = c["Hq"] // H, s["q"].shape[0], s["q"].device
    starts, held = s["starts"].long(), s["held"].long()
    new = starts[1:] - starts[:-1]
    node = torch.arange(M, device=dev)
    at = (starts[:-1, None] + node).clamp(max=T - 1)  # [B, M] rows of the ragged operands

    def cached(cache, descale):
        x = cache[s["table"].long().clamp(min=0)].float() * descale  # [B, W, H, page, D]
        x = x.transpose(1, 2).reshape(B, H, -1, D)
        lives = torch.arange(x.shape[2], device=dev) < held[:, None]
        return torch.where(lives[:, None, :, None], x, 0.0), lives

    def fresh(x):
        return x[at].float().transpose(1, 2)  # [B, H, M, D]

    (k0, lives), (v0, _) = cached(s["k_cache"], s["k_descale"]), cached(s["v_cache"], s["v_descale"])
    k, v = torch.cat([k0, fresh(s["k"])], 2), torch.cat([v0, fresh(s["v"])], 2)
    q = s["q"][at].float().reshape(B, M, H, group, D).permute(0, 2, 3, 1, 4)
    score = (q.reshape(B, H, group * M, D) @ k.transpose(2, 3)).view(B, H, group, M, -1) * s["scale"]
    hidden = (node[None, :] > node[:, None]).expand(B, M, M) if s["mask"] is None else s["mask"][at]
    hidden = hidden | (node >= new[:, None])[:, None, :]
    hidden = torch.cat([~lives[:, None, :].expand(B, M, lives.shape[1]), hidden], 2)
    score = score.masked_fill(hidden[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    o = (weight.view(B, H, group * M, -1) @ v).view(B, H, group, M, D) / total
    lse = (top + total.log()).squeeze(-1)
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    m = t - starts[b]
    r = {"o": o.permute(0, 3, 1, 2, 4)[b, m].reshape(T, c["Hq"], D).to(s["q"].dtype)}
    if c["lse"]:
        r["lse"] = lse.permute(0, 3, 1, 2)[b, m].reshape(T, c["Hq"])
    return r


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "plan":
        held, want = _plan_lengths(c)
        grown = sum(max(0, _pages(b, c["page"]) - _pages(a, c["page"])) for a, b in zip(held, want))
        return {"bytes": 4 * (4 * c["B"] + 1) + 8 * grown + 12 * c["tokens"], "flops": 0}
    if c["op"] == "append":
        values = c["tokens"] * c["Hkv"] * c["D"] * 0.9
        return {"bytes": 2 * values * (BYTES[c["type"]] + BYTES[c["cache"]]) + 8 * c["tokens"] + 4 * c["tokens"] * c["rows"],
                "flops": 2 * values if c["cache"] == "e4m3" else 0}
    if c["op"] == "rotary":
        tokens = max(1, c["B"]) * c["N"]
        values = tokens * (c["Hq"] + c["Hkv"]) * c["D"] * (2 if c["grad"] else 1)
        return {"bytes": 2 * values * BYTES[c["type"]] + 4 * c["axes"] * tokens, "flops": 3 * values}
    held, new = _tree_lengths(c)
    T = sum(new)
    if c["tree"]:
        pairs = sum(len(seen) for rows in _ancestors(c, new) for seen in rows)
    else:
        pairs = sum(n * (n + 1) // 2 for n in new)
    pairs += sum(a * b for a, b in zip(held, new))
    bytes_ = 2 * sum(held) * c["Hkv"] * c["D"] * BYTES[c["cache"]] + 2 * T * (c["Hq"] + c["Hkv"]) * c["D"] * 2
    bytes_ += 4 * sum(_pages(n, c["page"]) for n in held) + 8 * c["B"]
    bytes_ += (T * c["new"] if c["tree"] else 0) + (4 * T * c["Hq"] if c["lse"] else 0)
    return {"bytes": bytes_, "flops": 4 * c["D"] * c["Hq"] * pairs}


# ---------------------------------------------------------------- the same from the definitions, in 64 bits
def exact(case, seed):
    c = case
    if c["op"] == "plan":
        return None  # whole numbers: compared as they are
    s = prepare(c, seed)
    if c["op"] == "append":
        out = {}
        for name in ("k", "v"):
            cache, x = s[name + "_cache"].double(), s[name].double()
            slots = s["slots"].cpu()
            src = torch.arange(len(slots)) if s["rows"] is None else s["rows"].cpu().long()
            to, src = slots[slots >= 0].cuda(), src[slots >= 0].cuda()
            flat = cache.transpose(1, 2).reshape(-1, c["Hkv"], c["D"])
            value = x.index_select(0, src) / s[name + "_descale"]
            flat[to] = value.clamp(-E4M3_MAX, E4M3_MAX) if c["cache"] == "e4m3" else value
            out[name] = flat.view(c["pages"], c["page"], c["Hkv"], c["D"]).transpose(1, 2).contiguous()
        return out
    if c["op"] == "rotary":
        dim, half, pos = c["dim"], c["dim"] // 2, s["positions"].double()
        owner = []
        sections = _sections(c)
        if c["interleaved"]:
            for turn in range(half):
                owner += [a for a in range(c["axes"]) if turn < sections[a]]
        else:
            for a in range(c["axes"]):
                owner += [a] * sections[a]

        def turn(x, sign):
            out = x.detach().double().clone()
            for i in range(half):
                angle = sign * pos[owner[i]] / 10000.0 ** (2.0 * i / dim)
                angle = angle[:, None] if c["B"] == 0 else angle[:, None, :]
                e, f = (2 * i, 2 * i + 1) if c["neighbours"] else (i, i + half)
                a, b = x[..., e].detach().double(), x[..., f].detach().double()
                out[..., e] = a * torch.cos(angle) - b * torch.sin(angle)
                out[..., f] = b * torch.cos(angle) + a * torch.sin(angle)
            return out

        out = {"q": turn(s["q"], 1.0), "k": turn(s["k"], 1.0)}
        if c["grad"]:
            out["gq"], out["gk"] = turn(s["gq"], -1.0), turn(s["gk"], -1.0)
        return out
    held, new = _tree_lengths(c)
    group = c["Hq"] // c["Hkv"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    t = 0
    for b, (length, n) in enumerate(zip(held, new)):
        ids = s["table"][b, :_pages(length, c["page"])].long()
        if s["mask"] is None:
            seen = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        else:
            seen = ~s["mask"][t:t + n, :n]
        seen = torch.cat([torch.ones(n, length, dtype=torch.bool, device="cuda"), seen], 1)
        for h in range(c["Hkv"]):
            k = torch.cat([s["k_cache"][ids, h].double().flatten(0, 1)[:length] * s["k_descale"], s["k"][t:t + n, h].double()])
            v = torch.cat([s["v_cache"][ids, h].double().flatten(0, 1)[:length] * s["v_descale"], s["v"][t:t + n, h].double()])
            for x in range(h * group, (h + 1) * group):
                z = (s["q"][t:t + n, x].double() @ k.T * s["scale"]).masked_fill(~seen, -math.inf)
                lse[t:t + n, x] = torch.logsumexp(z, 1)
                o[t:t + n, x] = torch.softmax(z, 1) @ v
        t += n
    return {"o": o, "lse": lse} if c["lse"] else {"o": o}

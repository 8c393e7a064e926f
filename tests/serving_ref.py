"""Plain 64-bit statements of the serving operators, on CPU tensors and Python lists, for the tests."""
import math

import torch


def plan(lengths, targets, table, free, count, page, tokens):
    """cache_plan on Python lists; returns (slots, positions, starts, lengths, table, free, count, ok)."""
    def pages(n):
        return -(-n // page)

    table, stack = [list(r) for r in table], list(free[:count])
    width = len(table[0]) if table else 0
    valid = all(0 <= n <= width * page for n in lengths) and min(targets, default=0) >= 0
    fits = all(pages(t) <= width for t in targets)
    if valid and fits:
        for b, (n, t) in enumerate(zip(lengths, targets)):
            stack += table[b][pages(t):pages(n)]
        need = sum(max(0, pages(t) - pages(n)) for n, t in zip(lengths, targets))
        new = [max(0, t - n) for n, t in zip(lengths, targets)]
        if need <= len(stack) and sum(new) <= tokens:
            for b, (n, t) in enumerate(zip(lengths, targets)):
                for j in range(pages(n), pages(t)):
                    table[b][j] = stack.pop()
            slots, positions = [], []
            for b, (n, t) in enumerate(zip(lengths, targets)):
                for i in range(n, t):
                    slots.append(table[b][i // page] * page + i % page)
                    positions.append(i)
            pad = tokens - len(slots)
            starts = [sum(new[:b]) for b in range(len(new) + 1)]
            left = len(stack)
            return (slots + [-1] * pad, positions + [0] * pad, starts, list(targets), table,
                    stack[:left] + list(free[left:]), left, True)
    return ([-1] * tokens, [0] * tokens, [0] * (len(lengths) + 1), list(lengths), [list(r) for r in table], list(free),
            count, False)


def rotary(x, positions, freqs, axes, neighbours=False, inverse=False):
    """x [T, H, D] turned by positions [A, T] in 64 bits."""
    out, x = x.double().clone(), x.double()
    half = len(freqs)
    for i in range(half):
        angle = positions[axes[i]].double() * float(freqs[i]) * (-1 if inverse else 1)
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., a] * s + x[..., b] * c
    return out


def tree(q, k_new, v_new, k_cache, v_cache, table, lengths, starts, scale, mask=None, kd=1.0, vd=1.0):
    """(O, LSE, A) in 64 bits, A = sum_j p_j |v_j|: what roundings of the weights are measured by.
    kd, vd: numbers or one value per key head."""
    T, Hq, D = q.shape
    H, page = k_cache.shape[1], k_cache.shape[2]
    g = Hq // H
    kds, vds = ([x] * H if isinstance(x, (int, float)) else [float(y) for y in x] for x in (kd, vd))
    o = torch.zeros(T, Hq, D, dtype=torch.float64)
    a = torch.zeros(T, Hq, D, dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    for b in range(len(lengths)):
        n, t0, t1 = lengths[b], starts[b], starts[b + 1]
        if t1 == t0:
            continue
        ids = table[b][:-(-n // page)].long() if n else torch.zeros(0, dtype=torch.long)
        seen = torch.ones(t1 - t0, t1 - t0, dtype=torch.bool).tril() if mask is None else ~mask[t0:t1, :t1 - t0].bool()
        seen = torch.cat([torch.ones(t1 - t0, n, dtype=torch.bool), seen], 1)
        for h in range(H):
            kc = k_cache[ids, h].double().flatten(0, 1)[:n] * kds[h]
            vc = v_cache[ids, h].double().flatten(0, 1)[:n] * vds[h]
            k, v = torch.cat([kc, k_new[t0:t1, h].double()]), torch.cat([vc, v_new[t0:t1, h].double()])
            for x in range(h * g, (h + 1) * g):
                s = (q[t0:t1, x].double() @ k.T * scale).masked_fill(~seen, -math.inf)
                z = torch.logsumexp(s, 1)
                p = torch.exp(s - z[:, None]).nan_to_num(0.0)
                o[t0:t1, x], a[t0:t1, x], lse[t0:t1, x] = p @ v, p @ v.abs(), z
    return o, lse, a

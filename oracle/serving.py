"""Float64 restatement of the serving operators: page bookkeeping in Python integers and
softmax attention of one (request, head) at a time over the keys that a row sees."""

from __future__ import annotations

import numpy as np


def map_step(cached, new, held, tables, free, num_free, page, num_tokens):
    """Expected outputs of kvcache.map_step; ``tables`` (a list of lists) is updated in place."""
    used, slots, positions, cu, counts = 0, [], [], [0], []
    have = min(max(num_free, 0), len(free))
    for r, (c, n, h) in enumerate(zip(cached, new, held)):
        c, n, h = max(c, 0), max(n, 0), min(max(h, 0), len(tables[r]))
        need = min(-(-(c + n) // page), len(tables[r]))
        old = list(tables[r])
        for j in range(h, max(need, h)):
            at = have - 1 - used
            old[j] = tables[r][j] = free[at] if at >= 0 else -1
            used += 1
        counts.append(max(need, h))
        for i in range(n):
            p = c + i
            where = old[p // page] if p // page < counts[-1] else -1
            slots.append(where * page + p % page if where >= 0 else -1)
            positions.append(p)
        cu.append(min(cu[-1] + n, num_tokens))
    slots = (slots + [-1] * num_tokens)[:num_tokens]
    positions = (positions + [0] * num_tokens)[:num_tokens]
    return {"slots": slots, "positions": positions, "cu_seqlens": cu,
            "seq_lens": [max(c, 0) + max(n, 0) for c, n in zip(cached, new)],
            "page_counts": counts, "num_free": [have - used]}


def attend(q, k, v, seen, scale, unit):
    """One head: q (rows, D), k and v (keys, D) float64, seen (rows, keys) booleans.

    Returns (o, lse, tol, lse_tol). Only seen keys are touched, so what the others hold
    does not matter. The tolerances bound what a kernel with fp32 sums that rounds the
    weights p and the output to a 16-bit type with unit roundoff ``unit`` may be off:
      scores   e = D 2^-24 sum|q||k| s + 2^-22 max|score| + 2^-20   (fp32 dot, scale, exp2)
      weights  unit |p_j| each, in fp16 also 2^-25 (subnormals; the largest p is >= 1)
      output   unit |o| + 2^-25 (fp16 subnormals)
    """
    rows, dim = q.shape
    o = np.zeros((rows, v.shape[1]))
    tol = np.zeros_like(o)
    lse = np.full(rows, -np.inf)
    lse_tol = np.zeros(rows)
    fp16 = unit < 2.0 ** -10
    for i in range(rows):
        idx = np.flatnonzero(seen[i])
        if idx.size == 0:
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = k[idx] @ q[i] * scale
            top = s.max()
            p = np.exp(s - top)
            total = p.sum()
            p /= total
            o[i] = p @ v[idx]
            lse[i] = top + np.log(total)
            e = (dim * 2.0 ** -24 * (np.abs(k[idx]) @ np.abs(q[i])).max() * scale
                 + 2.0 ** -22 * np.abs(s).max() + 2.0 ** -20)
            mass = p @ np.abs(v[idx])
            tol[i] = unit * (np.abs(o[i]) + mass) + 2 * e * mass
            if fp16:
                tol[i] += 2.0 ** -25 * (1 + idx.size * np.abs(v[idx]).max())
            lse_tol[i] = e + 2.0 ** -21 * (1 + abs(lse[i]))
    return o, lse, tol, lse_tol


def causal(n):
    return np.tril(np.ones((n, n), dtype=bool))


def tree_seen(keys, new, words=None):
    """seen (new, keys) of a request's ``new`` last tokens; words[i] an int bit mask or None."""
    seen = np.zeros((new, keys), dtype=bool)
    ctx = keys - new
    for i in range(new):
        for j in range(keys):
            rank = j - ctx
            seen[i, j] = rank < 0 or (rank <= i if words is None else bool(words[i] >> rank & 1))
    return seen

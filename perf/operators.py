"""What the serving operators are measured on: paged key/value caches and the attention over them.

Four operators that one serving step runs in this order:

  slots    kvcache.map_step            pages and cache slots of a step's new tokens, from request lengths
  write    kvcache.write_kv            the new tokens' keys and values into their slots
  prefill  attention.attention_prefill causal attention over packed prompts with grouped heads
  tree     attention.attention_tree    attention of drafted tokens (or one token) over the paged cache

A case's lengths follow from its own values (``draw`` of them is the field "mix"), so that the work
of a case is known; the tensors' contents follow from the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ cases --
def listed():
    return [
        # the bookkeeping of one decode step of a few requests: launch latency is all there is
        {"name": "slots step 6", "op": "slots", "requests": 6, "page": 16, "kind": "step",
         "longest": 1500, "mix": 1},
        # a full server's step that mixes whole prompts, drafts and single tokens
        {"name": "slots mixed 384", "op": "slots", "requests": 384, "page": 64, "kind": "mixed",
         "longest": 2000, "mix": 2},
        # the new tokens of a decode step with drafts
        {"name": "write step 45", "op": "write", "tokens": 45, "heads": 4, "dim": 64, "page": 16,
         "dtype": "fp16", "packed": True, "mix": 3},
        # the keys and values of a batch of prompts
        {"name": "write prompts 16384", "op": "write", "tokens": 16384, "heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "packed": False, "mix": 4},
        # one short chat turn
        {"name": "prefill one 61", "op": "prefill", "prompts": 1, "longest": 61, "hq": 8, "hk": 2,
         "dim": 64, "dtype": "fp16", "mix": 5},
        # a batch of ordinary prompts of uneven lengths
        {"name": "prefill 24 uneven", "op": "prefill", "prompts": 24, "longest": 1100, "hq": 32,
         "hk": 8, "dim": 128, "dtype": "bf16", "mix": 6},
        # many short prompts, every one with a ragged end, heads not grouped
        {"name": "prefill 96 short", "op": "prefill", "prompts": 96, "longest": 300, "hq": 24,
         "hk": 24, "dim": 64, "dtype": "fp16", "mix": 7},
        # one long document: the matrix products are what it costs
        {"name": "prefill long 12031", "op": "prefill", "prompts": 1, "longest": 12031, "hq": 32,
         "hk": 8, "dim": 128, "dtype": "bf16", "mix": 8},
        # one user, one token: latency
        {"name": "tree single token", "op": "tree", "requests": 1, "drafts": 1, "longest": 777,
         "hq": 16, "hk": 2, "dim": 128, "page": 16, "dtype": "bf16", "mask": False, "mix": 9},
        # plain decoding of a full batch: reading the cache once is the floor
        {"name": "tree decode 64x8192", "op": "tree", "requests": 64, "drafts": 1, "longest": 8192,
         "hq": 32, "hk": 8, "dim": 128, "page": 64, "dtype": "bf16", "mask": False, "mix": 10},
        # speculative decoding: trees of up to 64 drafts over caches of uneven lengths
        {"name": "tree 16 drafted", "op": "tree", "requests": 16, "drafts": 64, "longest": 5000,
         "hq": 32, "hk": 8, "dim": 128, "page": 16, "dtype": "bf16", "mask": True, "mix": 11},
        # a small tree over two very long caches: the work is in one long axis
        {"name": "tree long 100003", "op": "tree", "requests": 2, "drafts": 12, "longest": 100003,
         "hq": 16, "hk": 2, "dim": 128, "page": 128, "dtype": "fp16", "mask": True, "mix": 12},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]; 3072 is left to nobody."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(max(v, lo), hi)
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["slots", "write", "prefill", "prefill", "tree", "tree"])
    mix = rng.randrange(1, 1 << 20)
    dtype = rng.choice(["fp16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "slots":
        return {"op": op, "requests": _log(rng, 1, 384), "page": page,
                "kind": rng.choice(["step", "mixed"]), "longest": _log(rng, 30, 2000), "mix": mix}
    hk = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128])
    if op == "write":
        return {"op": op, "tokens": _log(rng, 1, 16384), "heads": hk, "dim": dim, "page": page,
                "dtype": dtype, "packed": rng.random() < 0.5, "mix": mix}
    hq = hk * rng.choice([1, 2, 4, 5, 8] if hk < 8 else [1, 2, 4])
    if op == "prefill":
        prompts = _log(rng, 1, 96)
        longest = _log(rng, 1, max(1, min(12000, int(math.sqrt(4.2e9 / (hq * prompts))))))
        return {"op": op, "prompts": prompts, "longest": longest, "hq": hq, "hk": hk, "dim": dim,
                "dtype": dtype, "mix": mix}
    requests = _log(rng, 1, 64)
    drafts = rng.choice([1, _log(rng, 2, 64)])
    most = min(100000, 64 * 8192 * 8 // (requests * hk))
    most = min(most, int(2e9 / (requests * hq * drafts)))  # the plain form's scores
    longest = _log(rng, 70, max(71, most))
    return {"op": op, "requests": requests, "drafts": drafts, "longest": longest, "hq": hq,
            "hk": hk, "dim": dim, "page": page, "dtype": dtype,
            "mask": drafts > 1 and rng.random() < 0.7, "mix": mix}


def _lengths(case):
    """The case's lengths, from its own values alone: (cached, new) per request, or prompt lengths."""
    rng = random.Random(case["mix"])
    top = case.get("longest", 1)
    if case["op"] == "slots":
        cached, new = [], []
        for _ in range(case["requests"]):
            if case["kind"] == "step":
                cached.append(rng.randint(top // 3, top))
                new.append(1)
            else:
                kind = rng.random()
                cached.append(0 if kind < 0.1 else rng.randint(1, top))
                new.append(rng.randint(1, max(1, top // 2)) if kind < 0.1
                           else rng.randint(2, 32) if kind < 0.6 else 1)
        return cached, new
    if case["op"] == "prefill":
        lens = [max(1, int(top * rng.random() ** 1.5)) for _ in range(case["prompts"])]
        lens[rng.randrange(len(lens))] = top
        return lens
    n = case["requests"]
    lens = [max(case["drafts"], rng.randint(top // 2, top)) for _ in range(n)]
    lens[rng.randrange(n)] = max(case["drafts"], top)
    most = case["drafts"]
    new = [most if most == 1 else rng.randint(max(1, most // 3), most) for _ in range(n)]
    new[rng.randrange(n)] = most
    return [length - t for length, t in zip(lens, new)], new


def work(case):
    if case["op"] == "slots":
        cached, new = _lengths(case)
        page, r, total = case["page"], case["requests"], sum(new)
        pages = sum(-(-(c + t) // page) - -(-c // page) for c, t in zip(cached, new))
        # read: both lengths, page counts, a free page for each new one; written: the table's new
        # entries, a slot and a position per token, lengths, counts and offsets
        return {"bytes": 12 * r + 4 * pages + 4 * pages + 12 * total + 12 * r + 12, "flops": 0}
    if case["op"] == "write":
        row = case["heads"] * case["dim"] * 2
        return {"bytes": case["tokens"] * (2 * 2 * row + 8), "flops": 0}
    hq, hk, dim = case["hq"], case["hk"], case["dim"]
    if case["op"] == "prefill":
        lens = _lengths(case)
        t = sum(lens)
        return {"bytes": t * dim * 2 * (2 * hq + 2 * hk) + t * hq * 4 + 4 * len(lens) + 4,
                "flops": sum(4 * dim * hq * (n * (n + 1) // 2) for n in lens)}
    cached, new = _lengths(case)
    keys, t = sum(cached) + sum(new), sum(new)
    size = 2 * keys * hk * dim * 2 + 2 * t * hq * dim * 2 + t * hq * 4
    size += sum(-(-(c + n) // case["page"]) for c, n in zip(cached, new)) * 4
    if case["mask"]:
        size += 8 * t
    return {"bytes": size, "flops": sum(4 * dim * hq * n * (c + (n + 1) / 2)
                                        for c, n in zip(cached, new))}


# ----------------------------------------------------------------- inputs --
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _normal(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _keys(g, *shape, dtype):
    """Keys (..., heads, dim) whose channels differ in size, as a trained projection's do."""
    size = torch.exp(0.4 * torch.randn((shape[-2], shape[-1]), generator=g, device="cuda"))
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * size).to(dtype)


def _trees(new, rng):
    """Ancestor words of every drafted token: bit j of a token's word says that it sees the
    request's j-th drafted token (its ancestors and itself)."""
    words = []
    for n in new:
        mine = []
        for i in range(n):
            up = 0 if i == 0 else mine[rng.randrange(max(0, i - 8), i)]
            mine.append(up | (1 << i))
        words += mine
    return [w - (1 << 64) if w >> 63 else w for w in words]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "slots":
        cached, new = _lengths(case)
        page = case["page"]
        held = [-(-c // page) for c in cached]
        most = max(-(-(c + n) // page) for c, n in zip(cached, new))
        need = sum(-(-(c + n) // page) for c, n in zip(cached, new))
        pages = torch.randperm(need + need // 4 + 8, generator=g, device="cuda").to(torch.int32)
        used = sum(held)
        at = torch.arange(most, device="cuda")
        filled = at[None, :] < _ints(held)[:, None]
        tables = torch.zeros((case["requests"], most), dtype=torch.int32, device="cuda")
        tables[filled] = pages[:used]
        return {"op": op, "cached": _ints(cached), "new": _ints(new), "counts": _ints(held),
                "tables": tables, "free": pages[used:].contiguous(),
                "num_free": _ints([pages.numel() - used]), "page": page, "tokens": sum(new)}
    dtype, dim = DTYPES[case["dtype"]], case["dim"]
    if op == "write":
        t, h, page = case["tokens"], case["heads"], case["page"]
        n_pages = -(-t // page) + 3
        if case["packed"]:  # keys and values where a fused projection leaves them
            both = _normal(g, t, 2 * h, dim, dtype=dtype)
            k, v = both[:, :h], both[:, h:]
        else:
            k, v = _normal(g, t, h, dim, dtype=dtype), _normal(g, t, h, dim, dtype=dtype)
        k_cache = torch.zeros((n_pages, page, h, dim), dtype=dtype, device="cuda")
        order = torch.randperm(n_pages, generator=g, device="cuda")
        at = torch.arange(t, device="cuda")
        slots = order[at // page] * page + at % page
        return {"op": op, "k": k, "v": v, "k_cache": k_cache, "v_cache": torch.zeros_like(k_cache),
                "slots": slots}
    hq, hk = case["hq"], case["hk"]
    scale = dim ** -0.5
    if op == "prefill":
        lens = _lengths(case)
        t = sum(lens)
        return {"op": op, "q": _normal(g, t, hq, dim, dtype=dtype),
                "k": _keys(g, t, hk, dim, dtype=dtype), "v": _normal(g, t, hk, dim, dtype=dtype),
                "cu": _ints(_offsets(lens)), "scale": scale, "longest": max(lens),
                "lse": torch.empty((hq, t), dtype=torch.float32, device="cuda")}
    cached, new = _lengths(case)
    page, t = case["page"], sum(new)
    lens = [c + n for c, n in zip(cached, new)]
    need = [-(-n // page) for n in lens]
    pages = torch.randperm(sum(need) + 5, generator=g, device="cuda").to(torch.int32)
    filled = torch.arange(max(need), device="cuda")[None, :] < _ints(need)[:, None]
    tables = torch.zeros((len(lens), max(need)), dtype=torch.int32, device="cuda")
    tables[filled] = pages[: sum(need)]
    mask = None
    if case["mask"]:
        words = _trees(new, random.Random(seed))
        mask = torch.tensor(words, dtype=torch.int64, device="cuda").view(t, 1)
    n_pages = pages.numel()
    return {"op": op, "q": _normal(g, t, hq, dim, dtype=dtype),
            "k_cache": _keys(g, n_pages, page, hk, dim, dtype=dtype),
            "v_cache": _normal(g, n_pages, page, hk, dim, dtype=dtype), "tables": tables,
            "lens": _ints(lens), "cu": _ints(_offsets(new)), "mask": mask, "scale": scale,
            "drafts": max(new), "lse": torch.empty((hq, t), dtype=torch.float32, device="cuda")}


# ------------------------------------------------------------- plain forms --
def _plain_slots(s):
    cached, new, held, page = s["cached"].long(), s["new"].long(), s["counts"].long(), s["page"]
    tables, free, num_free = s["tables"], s["free"], s["num_free"].long()
    need = (cached + new + page - 1) // page
    fresh = (need - held).clamp(min=0)
    first = torch.cumsum(fresh, 0) - fresh
    ends = torch.cumsum(new, 0)

    at = torch.arange(tables.shape[1], device=tables.device)
    k = first[:, None] + at[None, :] - held[:, None]
    taken = num_free - 1 - k
    value = torch.where(taken >= 0, free[taken.clamp(0, free.numel() - 1)].long(), -1)
    is_new = (at[None, :] >= held[:, None]) & (at[None, :] < need[:, None])
    tables.copy_(torch.where(is_new, value, tables.long()))

    token = torch.arange(s["tokens"], device=tables.device)
    r = torch.searchsorted(ends, token, right=True).clamp(max=cached.numel() - 1)
    position = cached[r] + token - (ends - new)[r]
    there = tables.long()[r, position // page]
    slots = torch.where(there >= 0, there * page + position % page, -1)
    cu = torch.cat([torch.zeros_like(ends[:1]), ends]).int()
    return {"tables": tables, "slots": slots, "positions": position.int(), "cu_seqlens": cu,
            "seq_lens": (cached + new).int(), "page_counts": (held + fresh).int(),
            "num_free": (num_free - fresh.sum()).int()}


def _plain_write(s):
    _, page, h, dim = s["k_cache"].shape
    keep = s["slots"] >= 0
    where = s["slots"][keep]
    s["k_cache"].view(-1, h, dim)[where] = s["k"][keep]
    s["v_cache"].view(-1, h, dim)[where] = s["v"][keep]
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attention(q, k, v, seen, scale):
    """Rows of q (batch, hk, rows, dim) over k, v (batch, hk, keys, dim) where `seen`
    (batch, 1 or hk, rows, keys): outputs and the scores' log-sum-exp, in 32 bits."""
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = scores.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out, (top + total.log()).squeeze(-1)


def _plain_prefill(s):
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"].long()
    t, hq, dim = q.shape
    hk, b, longest = k.shape[1], cu.numel() - 1, s["longest"]
    group = hq // hk
    at = torch.arange(longest, device=q.device)
    inside = at[None, :] < (cu[1:] - cu[:-1])[:, None]
    row = (cu[:-1, None] + at[None, :]).clamp(max=t - 1)
    qp = q[row].float().view(b, longest, hk, group, dim).permute(0, 2, 3, 1, 4)
    kp = k[row].float().permute(0, 2, 1, 3)
    vp = v[row].float().permute(0, 2, 1, 3)
    seen = (at[None, :] <= at[:, None])[None] & inside[:, None, :]
    seen = seen[:, None, None].expand(b, 1, group, longest, longest)
    out, lse = _plain_attention(qp.reshape(b, hk, group * longest, dim), kp, vp,
                                seen.reshape(b, 1, group * longest, longest), s["scale"])
    out = out.view(b, hk, group, longest, dim).permute(0, 3, 1, 2, 4).reshape(b, longest, hq, dim)
    lse = lse.view(b, hk, group, longest).permute(0, 3, 1, 2).reshape(b, longest, hq)
    return {"o": out[inside].to(q.dtype), "lse": lse[inside].t().contiguous()}


def _plain_tree(s):
    q, cu, lens, tables = s["q"], s["cu"].long(), s["lens"].long(), s["tables"].long()
    t, hq, dim = q.shape
    _, page, hk, _ = s["k_cache"].shape
    r, keys, drafts, group = lens.numel(), tables.shape[1] * page, s["drafts"], hq // hk
    new = cu[1:] - cu[:-1]
    at = torch.arange(drafts, device=q.device)
    row = (cu[:-1, None] + at[None, :]).clamp(max=t - 1)
    qp = q[row].float().view(r, drafts, hk, group, dim).permute(0, 2, 3, 1, 4)
    kp = s["k_cache"][tables].view(r, keys, hk, dim).permute(0, 2, 1, 3).float()
    vp = s["v_cache"][tables].view(r, keys, hk, dim).permute(0, 2, 1, 3).float()
    key = torch.arange(keys, device=q.device)
    rank = key[None, None, :] - (lens - new)[:, None, None]  # among the request's drafted tokens
    if s["mask"] is None:
        seen = rank <= at[None, :, None]
    else:
        bit = (s["mask"][row, 0][:, :, None] >> rank.clamp(0, 63)) & 1
        seen = (rank < 0) | ((rank < 64) & (bit == 1))
    seen = seen & (key[None, None, :] < lens[:, None, None])
    seen = seen[:, None, None].expand(r, 1, group, drafts, keys)
    out, lse = _plain_attention(qp.reshape(r, hk, group * drafts, dim), kp, vp,
                                seen.reshape(r, 1, group * drafts, keys), s["scale"])
    out = out.view(r, hk, group, drafts, dim).permute(0, 3, 1, 2, 4).reshape(r, drafts, hq, dim)
    lse = lse.view(r, hk, group, drafts).permute(0, 3, 1, 2).reshape(r, drafts, hq)
    mine = at[None, :] < new[:, None]
    return {"o": out[mine].to(q.dtype), "lse": lse[mine].t().contiguous()}


# -------------------------------------------------------------------- run --
def run(s):
    op = s["op"]
    if not own:
        return {"slots": _plain_slots, "write": _plain_write, "prefill": _plain_prefill,
                "tree": _plain_tree}[op](s)
    from gfx950_gluon_tutorials_b200 import attention, kvcache
    if op == "slots":
        m = kvcache.map_step(s["cached"], s["new"], s["counts"], s["tables"], s["free"],
                             s["num_free"], page_size=s["page"], num_tokens=s["tokens"])
        return {"tables": s["tables"], "slots": m.slots, "positions": m.positions,
                "cu_seqlens": m.cu_seqlens, "seq_lens": m.seq_lens,
                "page_counts": m.page_counts, "num_free": m.num_free}
    if op == "write":
        kvcache.write_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "prefill":
        o = attention.attention_prefill(s["q"], s["k"], s["v"], s["cu"], sm_scale=s["scale"],
                                        lse=s["lse"])
        return {"o": o, "lse": s["lse"]}
    o = attention.attention_tree(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"],
                                 s["cu"], s["mask"], sm_scale=s["scale"], lse=s["lse"])
    return {"o": o, "lse": s["lse"]}


# ------------------------------------------------------------------ exact --
def _exact_head(q, k, v, seen, scale):
    s = (q @ k.T) * scale
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    return p @ v, lse


def exact(case, seed):
    """Softmax attention of one head of one request at a time, in 64 bits; the written caches page
    row by page row. The maps hold whole numbers only: None."""
    op = case["op"]
    if op == "slots":
        return None
    s = prepare(case, seed)
    if op == "write":
        out = {}
        for name in ("k", "v"):
            rows = s[name + "_cache"].double().flatten(0, 1)
            rows[s["slots"]] = s[name].double()
            out[name + "_cache"] = rows.view(s["k_cache"].shape)
        return out
    q = s["q"].double()
    t, hq, dim = q.shape
    o = torch.empty((t, hq, dim), dtype=torch.float64, device="cuda")
    lse = torch.empty((hq, t), dtype=torch.float64, device="cuda")
    if op == "prefill":
        lens, group = _lengths(case), hq // case["hk"]
        begin = 0
        for n in lens:
            rows = slice(begin, begin + n)
            at = torch.arange(n, device="cuda")
            seen = at[:, None] >= at[None, :]
            for h in range(hq):
                o[rows, h], lse[h, rows] = _exact_head(
                    q[rows, h], s["k"][rows, h // group].double(),
                    s["v"][rows, h // group].double(), seen, s["scale"])
            begin += n
        return {"o": o, "lse": lse}
    cached, new = _lengths(case)
    group, page = hq // case["hk"], case["page"]
    words = None if s["mask"] is None else [w % (1 << 64) for w in s["mask"][:, 0].tolist()]
    begin = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        pages = s["tables"][r, : -(-(c + n) // page)].long()
        k = s["k_cache"][pages].reshape(-1, case["hk"], dim)[: c + n].double()
        v = s["v_cache"][pages].reshape(-1, case["hk"], dim)[: c + n].double()
        seen = torch.ones((n, c + n), dtype=torch.bool)
        for i in range(n):
            seen[i, c:] = torch.tensor([j <= i if words is None else bool(words[begin + i] >> j & 1)
                                        for j in range(n)])
        seen = seen.cuda()
        rows = slice(begin, begin + n)
        for h in range(hq):
            o[rows, h], lse[h, rows] = _exact_head(q[rows, h], k[:, h // group], v[:, h // group],
                                                   seen, s["scale"])
        begin += n
    return {"o": o, "lse": lse}

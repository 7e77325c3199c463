"""Causal packed prefill and tree attention over a paged cache on the B200, against softmax
attention in float64. Tolerances are the error bounds that oracle.serving.attend derives per
element from the inputs: fp32 sums, weights and outputs rounded to the 16-bit type."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

from gfx950_gluon_tutorials_b200 import _lib, attention, kvcache, ops
from oracle import serving

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half the spacing at 1
DTYPES = [torch.float16, torch.bfloat16]


def _np(t):
    return t.double().cpu().numpy()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _cu(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _close(o, lse, ref, where=""):
    want, want_lse, tol, lse_tol = ref
    bad = ~(np.abs(o - want) <= tol) & ~(np.isnan(o) & np.isnan(want)) & ~(o == want)
    assert not bad.any(), f"{where}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(o - want)):.3e}"
    if lse is not None:
        ok = (np.abs(lse - want_lse) <= lse_tol) | (lse == want_lse) | (np.isnan(lse) & np.isnan(want_lse))
        assert ok.all(), f"{where}: lse {lse[~ok][:4]} for {want_lse[~ok][:4]}"


def _rows_of(n, limit=24):
    """Row indices to check of n: all, or the ends, tile borders and a few others."""
    if n <= limit:
        return np.arange(n)
    pick = {0, 1, 31, 32, 63, 64, 126, 127, 128, 129, 255, 256, 257, n // 2, n - 130, n - 129, n - 128, n - 2, n - 1}
    return np.array(sorted(i for i in pick if 0 <= i < n))


# ---------------------------------------------------------------- prefill --
def _check_prefill(q, k, v, lens, o, lse, scale, skip=()):
    begin, group = 0, q.shape[1] // k.shape[1]
    for b, n in enumerate(lens):
        if n and b not in skip:
            rows = _rows_of(n)
            seen = serving.causal(n)[rows]
            for h in sorted({0, q.shape[1] // 2, q.shape[1] - 1}):
                ref = serving.attend(_np(q[begin:begin + n, h])[rows], _np(k[begin:begin + n, h // group]),
                                     _np(v[begin:begin + n, h // group]), seen, scale, UNIT[q.dtype])
                _close(_np(o[begin:begin + n, h])[rows], _np(lse[h, begin:begin + n])[rows], ref,
                       f"prompt {b} head {h}")
        begin += n


def _prefill(q, k, v, lens, scale=None, o=None):
    lse = torch.full((q.shape[1], q.shape[0]), float("nan"), device="cuda")
    o = torch.full_like(q, float("nan")) if o is None else o
    attention.attention_prefill(q, k, v, _cu(lens), o, sm_scale=scale, lse=lse)
    ops.check_status()
    return o, lse


PROMPTS = [
    # lens, HQ, HK, D
    ([1], 1, 1, 64), ([1], 8, 2, 128), ([77], 4, 1, 64), ([128], 2, 2, 128), ([129], 2, 1, 128),
    ([256, 1, 0, 255], 4, 2, 64), ([3, 130, 257, 0, 0, 64, 1], 10, 2, 128), ([1000], 5, 1, 128),
    ([513, 40, 300], 6, 6, 64), ([2049], 2, 1, 128), ([0, 0, 5], 2, 2, 128), ([384, 640], 16, 1, 128),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: f"{'_'.join(map(str, c[0]))}-{c[1]}-{c[2]}-{c[3]}")
def test_prefill(cuda_device, case, dtype):
    lens, hq, hk, d = case
    g, t = _gen(sum(lens) + hq), sum(lens)
    q, k, v = _rand(g, t, hq, d, dtype=dtype), _rand(g, t, hk, d, dtype=dtype), _rand(g, t, hk, d, dtype=dtype)
    o, lse = _prefill(q, k, v, lens)
    _check_prefill(q, k, v, lens, o, lse, d ** -0.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp16", "bf16"])
def test_prefill_many_prompts(cuda_device, dtype):
    """More work items than SMs, of every length from 0 to a few tiles."""
    rng = random.Random(4)
    lens = [rng.choice([0, 1, 2, 127, 128, 129, 256, 300, 400]) for _ in range(150)]
    g, t = _gen(4), sum(lens)
    q, k, v = (_rand(g, t, h, 64, dtype=dtype) for h in (4, 2, 2))
    o, lse = _prefill(q, k, v, lens)
    _check_prefill(q, k, v, lens, o, lse, 0.125)


def test_prefill_moving_max(cuda_device):
    """Scores that grow along the keys by hundreds of powers of two: the running maximum moves
    in every tile."""
    g, n = _gen(11), 1100
    q, k, v = (_rand(g, n, h, 128, dtype=torch.bfloat16) for h in (2, 1, 1))
    k = (k.float() * torch.linspace(0.2, 3.0, n, device="cuda").view(n, 1, 1)).bfloat16()
    o, lse = _prefill(q, k, v, [n], scale=1.0)
    _check_prefill(q, k, v, [n], o, lse, 1.0)


def test_prefill_fused_projection_and_strided_output(cuda_device):
    g, lens = _gen(9), [200, 61]
    qkv = _rand(g, 261, 4 + 2 + 2, 64, dtype=torch.float16)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    big = torch.zeros((261, 4, 128), dtype=torch.float16, device="cuda")
    o, lse = _prefill(q, k, v, lens, o=big[..., 64:])
    _check_prefill(q, k, v, lens, o, lse, 0.125)
    assert bool((big[..., :64] == 0).all()), "wrote outside the output view"


@pytest.mark.parametrize("how", ["odd base", "dim stride", "heads first", "odd output", "one broadcast head"])
def test_prefill_other_layouts(cuda_device, how):
    """Addresses that the kernel cannot read in place are copied; the answer is the same."""
    g, lens, d = _gen(10), [70, 131], 64
    t = sum(lens)
    q, k, v = (_rand(g, t, h, d, dtype=torch.float16) for h in (4, 2, 2))
    o = None
    if how == "odd base":
        q = torch.cat([torch.zeros(1, device="cuda").half(), q.flatten()])[1:].view(q.shape)
    elif how == "dim stride":
        k = k.transpose(1, 2).contiguous().transpose(1, 2)
    elif how == "heads first":
        q, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, v))
    elif how == "odd output":
        o = torch.full((t * 4 * d + 1,), float("nan"), device="cuda").half()[1:].view(t, 4, d)
    else:
        k, v = k[:, :1].expand(-1, 2, -1), v[:, :1].expand(-1, 2, -1)
    o, lse = _prefill(q, k, v, lens, o=o)
    _check_prefill(q, k, v, lens, o, lse, 0.125)


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp16", "bf16"])
def test_prefill_what_is_masked_does_not_count(cuda_device, dtype, what):
    """A prompt of NaN or infinities between two others, and padding rows after the last prompt,
    leave the others as they are."""
    g, lens = _gen(21), [150, 90, 300]
    t = sum(lens) + 60
    q, k, v = (_rand(g, t, h, 128, dtype=dtype) for h in (4, 2, 2))
    for x in (k, v):
        x[150:240] = what
        x[540:] = what
    o = torch.full_like(q, 7.0)
    o, lse = _prefill(q, k, v, lens, o=o)
    _check_prefill(q, k, v, lens, o, lse, 128 ** -0.5, skip={1})
    assert bool((o[540:] == 7.0).all()) and bool(lse[:, 540:].isnan().all())


@pytest.mark.parametrize("which", ["k", "v", "v infinite"])
def test_prefill_nan_in_a_later_token(cuda_device, which):
    """Tokens before a NaN or infinite one do not see it; those from it on do."""
    g, n, at = _gen(22), 400, 333
    q, k, v = (_rand(g, n, h, 64, dtype=torch.bfloat16) for h in (4, 2, 2))
    (k if which == "k" else v)[at, :, 5] = float("inf") if which == "v infinite" else float("nan")
    o, _ = _prefill(q, k, v, [n])
    clean = v.clone()
    clean[at] = 0
    kc = k.clone()
    kc[at] = 0
    want, _ = _prefill(q, kc, clean, [n])
    assert torch.equal(o[:at], want[:at])
    after = o[at:].float()
    if which == "k":
        assert bool(after.isnan().all())
    else:
        assert bool((after[..., 5] == float("inf")).all() if which != "v" else after[..., 5].isnan().all())
        after[..., 5] = 0
        assert bool(after.isfinite().all())


def test_prefill_bad_offsets(cuda_device):
    """Offsets that decrease or pass the end are clamped and reported; nothing is read outside."""
    q, k, v = (_rand(_gen(1), 40, h, 64, dtype=torch.float16) for h in (2, 1, 1))
    for cu in ([0, 50, 60], [0, 30, 20, 40], [5, 40], [-3, 40]):
        attention.attention_prefill(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        if cu == [5, 40]:
            ops.check_status()
            continue
        with pytest.raises(_lib.B2GError) as e:
            ops.check_status()
        assert e.value.code == _lib.STATUS_TOKENS


def test_prefill_deterministic_on_any_stream(cuda_device):
    lens = [700, 33, 260]
    q, k, v = (_rand(_gen(5), sum(lens), h, 128, dtype=torch.bfloat16) for h in (8, 2, 2))
    a, la = _prefill(q, k, v, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = _prefill(q, k, v, lens)
        graph = torch.cuda.CUDAGraph()
        cu, c = _cu(lens), torch.empty_like(q)
        with torch.cuda.graph(graph, stream=side):
            attention.attention_prefill(q, k, v, cu, c)
        graph.replay()
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and torch.equal(la, lb) and torch.equal(a, c)


def test_prefill_refusals(cuda_device):
    q, k = (_rand(_gen(2), 10, h, 64, dtype=torch.float16) for h in (4, 2))
    cu = _cu([10])
    for args in ((q, k, k[:9], cu), (q, k[:9], k[:9], cu), (q, k.bfloat16(), k, cu), (q.float(), k, k, cu),
                 (q, k, k, cu.long()), (q, k, k, cu[:0]), (q[:, :3], k, k, cu), (q[0], k, k, cu),
                 (q[..., :32], k[..., :32], k[..., :32], cu), (q, k, k, cu, q[:9]), (q, k, k, cu, q.bfloat16())):
        with pytest.raises(ValueError):
            attention.attention_prefill(*args)
    for lse in (torch.empty((4, 9), device="cuda"), torch.empty((10, 4), device="cuda").t()):
        with pytest.raises(ValueError):
            attention.attention_prefill(q, k, k, cu, lse=lse)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(_lib.B2GError):
            attention.attention_prefill(q, k, k, cu, sm_scale=scale)
    assert attention.attention_prefill(q[:0], k[:0], k[:0], _cu([0])).shape == (0, 4, 64)


# ------------------------------------------------------------------- tree --
def _words(new, rng, wide=1):
    out = []
    for n in new:
        mine = []
        for i in range(n):
            mine.append((mine[rng.randrange(i)] if i else 0) | 1 << i)
        out += mine
    return out


def _mask(words, wide):
    rows = [[(w >> 64 * j) & (1 << 64) - 1 for j in range(wide)] for w in words]
    rows = [[x - (1 << 64) if x >> 63 else x for x in r] for r in rows]
    return torch.tensor(rows, dtype=torch.int64, device="cuda")


class Tree:
    """A batch over a paged cache: lens keys in all, the last new of them the step's tokens.
    Slots that hold no key of a request are NaN."""

    def __init__(self, lens, new, hq, hk, d, page, dtype, seed, layout="slots", masked=True, spare=3):
        g, rng = _gen(seed), random.Random(seed)
        self.lens, self.new, self.hq, self.hk, self.d, self.page = lens, new, hq, hk, d, page
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        shape = (pages, hk, page, d) if layout == "heads" else (pages, page, hk, d)
        self.kc, self.vc = (torch.full(shape, float("nan"), device="cuda", dtype=dtype) for _ in range(2))
        if layout == "heads":
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        ids = list(range(pages))
        rng.shuffle(ids)
        table, self.k, self.v = [], [], []
        for n, m in zip(lens, need):
            mine = [ids.pop() for _ in range(m)]
            table.append(mine + [-1] * (max(need + [1]) - m))
            self.k.append(_rand(g, n, hk, d, dtype=dtype))
            self.v.append(_rand(g, n, hk, d, dtype=dtype))
            if n:
                at = torch.arange(n, device="cuda")
                where = torch.tensor(mine, device="cuda")[at // page]
                self.kc[where, at % page], self.vc[where, at % page] = self.k[-1], self.v[-1]
        self.table = torch.tensor(table, dtype=torch.int32, device="cuda")
        self.q = _rand(g, sum(new), hq, d, dtype=dtype)
        self.words = _words(new, rng) if masked else None
        wide = max(1, -(-max(new + [1]) // 64))
        self.mask = _mask(self.words, wide) if masked and sum(new) else None

    def run(self, scale=None, o=None):
        lse = torch.full((self.hq, sum(self.new)), float("nan"), device="cuda")
        o = torch.full_like(self.q, float("nan")) if o is None else o
        lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        attention.attention_tree(self.q, self.kc, self.vc, self.table, lens, _cu(self.new), self.mask, o,
                                 sm_scale=scale, lse=lse)
        ops.check_status()
        return o, lse

    def check(self, o, lse, scale=None, heads=None, requests=None):
        scale, group, begin = scale or self.d ** -0.5, self.hq // self.hk, 0
        for r, (keys, n) in enumerate(zip(self.lens, self.new)):
            if n and (requests is None or r in requests):
                rows = _rows_of(n)
                words = None if self.words is None else self.words[begin:begin + n]
                seen = serving.tree_seen(keys, n, words)[rows]
                for h in heads or sorted({0, group - 1, self.hq // 2, self.hq - 1}):
                    ref = serving.attend(_np(self.q[begin:begin + n, h])[rows], _np(self.k[r][:, h // group]),
                                         _np(self.v[r][:, h // group]), seen, scale, UNIT[self.q.dtype])
                    _close(_np(o[begin:begin + n, h])[rows], _np(lse[h, begin:begin + n])[rows], ref,
                           f"request {r} head {h}")
            begin += n


TREES = [
    # lens, new, HQ, HK, D, page, layout, masked
    ([1], [1], 1, 1, 64, 16, "slots", False),
    ([777], [1], 16, 2, 128, 16, "slots", False),
    ([128, 129, 127, 1], [1, 1, 1, 1], 8, 8, 64, 16, "slots", False),
    ([5000], [1], 4, 1, 128, 64, "heads", False),
    ([300, 20, 130], [12, 20, 1], 8, 2, 128, 16, "slots", True),
    ([400, 65], [64, 65], 8, 1, 128, 32, "slots", True),       # 512 rows, two mask words
    ([300, 1000], [33, 7], 10, 2, 64, 8, "heads", True),        # groups of five
    ([129, 257, 64], [3, 2, 64], 32, 2, 128, 128, "slots", True),
    ([700], [40], 4, 4, 128, 256, "slots", True),
    ([2000, 900], [300, 129], 4, 2, 128, 64, "slots", False),   # chunks of prompts
    ([130], [130], 3, 1, 64, 16, "slots", True),                # no context, three mask words
    ([0, 50, 0, 9], [0, 2, 0, 1], 4, 2, 128, 16, "slots", True),
    ([260, 260], [17, 16], 8, 1, 64, 64, "slots", True),        # 136 and 128 rows
    ([1300] * 3, [5, 4, 6], 40, 8, 128, 16, "heads", True),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp16", "bf16"])
@pytest.mark.parametrize("case", TREES, ids=lambda c: "-".join(str(x).replace(", ", "_") for x in c))
def test_tree(cuda_device, case, dtype):
    lens, new, hq, hk, d, page, layout, masked = case
    t = Tree(lens, new, hq, hk, d, page, dtype, seed=sum(lens) + hq, layout=layout, masked=masked)
    o, lse = t.run()
    t.check(o, lse)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp16", "bf16"])
def test_tree_full_batch(cuda_device, dtype):
    """Many requests of uneven lengths: shares of work that begin and end anywhere."""
    rng = random.Random(6)
    lens = [rng.choice([1, 16, 128, 200, 1000, 3000]) for _ in range(90)]
    new = [min(n, rng.choice([1, 1, 3, 9])) for n in lens]
    t = Tree(lens, new, 8, 2, 128, 16, dtype, seed=6)
    o, lse = t.run()
    t.check(o, lse, heads=[0, 7])


@pytest.mark.parametrize("new", [1, 6])
def test_tree_long_axis(cuda_device, new):
    """One request, a long cache: its keys are split over the whole GPU and joined."""
    t = Tree([40001], [new], 8, 1, 128, 16, torch.bfloat16, seed=7)
    o, lse = t.run()
    t.check(o, lse, heads=[0, 7])


def test_tree_moving_max(cuda_device):
    t = Tree([3001, 500], [4, 70], 4, 1, 128, 32, torch.bfloat16, seed=8)
    for r, n in enumerate(t.lens):
        size = torch.linspace(0.2, 3.0, n, device="cuda").view(n, 1, 1)
        t.k[r] = (t.k[r].float() * size).bfloat16()
        at = torch.arange(n, device="cuda")
        t.kc[t.table[r].long()[at // t.page], at % t.page] = t.k[r]
    o, lse = t.run(scale=1.0)
    t.check(o, lse, scale=1.0)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_tree_masked_drafts_do_not_count(cuda_device, what):
    """A draft of NaN or infinities is seen by its descendants only."""
    lens, new = [150, 400], [10, 40]
    t = Tree(lens, new, 8, 2, 128, 16, torch.bfloat16, seed=9)
    bad, r = 3, 1
    at = lens[r] - new[r] + bad
    page, slot = int(t.table[r, at // 16]), at % 16
    t.vc[page, slot] = what
    o, lse = t.run()
    rows = slice(10, 50)
    sees = torch.tensor([bool(w >> bad & 1) for w in t.words[rows]], device="cuda")
    assert 0 < int(sees.sum()) < 40
    t.vc[page, slot] = 0
    t.kc[page, slot] = what  # a masked key is not looked at either
    o2, lse2 = t.run()
    assert torch.equal(o[:10], o2[:10])
    assert torch.equal(o[rows][~sees], o2[rows][~sees]) and torch.equal(lse[:, rows][:, ~sees], lse2[:, rows][:, ~sees])
    assert bool(o[rows][~sees].isfinite().all())
    got = o[rows][sees].float()
    assert bool(got.isnan().all() if math.isnan(what) else (got == what).all())


def test_tree_rows_that_see_nothing(cuda_device):
    """Empty masks, requests without keys, and lengths shorter than the new tokens."""
    t = Tree([20, 0, 0], [20, 0, 0], 4, 2, 64, 16, torch.float16, seed=10)
    t.words[4] = t.words[19] = 0
    t.mask = _mask(t.words, 1)
    o, lse = t.run()
    t.check(o, lse)
    assert bool((o[4] == 0).all()) and bool((lse[:, 19] == float("-inf")).all())
    t.lens, t.new, t.mask = [3, 0, 0], [5, 4, 0], None  # rows 0, 1 and 5 .. 8 lie before the first key
    t.q = t.q[:9].contiguous()
    o, lse = t.run()
    assert bool((o[:2] == 0).all()) and bool((o[5:] == 0).all()) and bool((lse[:, :2] == float("-inf")).all())
    assert bool(o[2:5].isfinite().all()) and bool(lse[:, 2:5].isfinite().all())


def test_tree_bad_pages(cuda_device):
    """Pages outside the cache and tables that are too short are reported, not read."""
    for page in (-1, 10 ** 6):
        t = Tree([100], [2], 4, 2, 64, 16, torch.float16, seed=12)
        t.table[0, 2] = page
        with pytest.raises(_lib.B2GError) as e:
            t.run()
        assert e.value.code == _lib.STATUS_PAGE_TABLE
    t = Tree([100], [2], 4, 2, 64, 16, torch.float16, seed=12)
    t.table = t.table[:, :4].contiguous()
    with pytest.raises(_lib.B2GError) as e:
        t.run()
    assert e.value.code == _lib.STATUS_PAGE_TABLE


def test_tree_strided_tensors(cuda_device):
    """A table with spare columns, one layer of a shared cache, q and o as slices."""
    t = Tree([200, 333], [4, 9], 8, 2, 64, 16, torch.float16, seed=13)
    wide = torch.full((2, 2 * t.table.shape[1]), -5, dtype=torch.int32, device="cuda")
    wide[:, :t.table.shape[1]] = t.table
    t.table = wide[:, :t.table.shape[1]]
    for name in ("kc", "vc"):
        x = getattr(t, name)
        both = torch.zeros((x.shape[0], 2, *x.shape[1:]), dtype=x.dtype, device="cuda")
        both[:, 1] = x
        setattr(t, name, both[:, 1])
    q = torch.zeros((13, 12, 64), dtype=torch.float16, device="cuda")
    q[:, 4:] = t.q
    t.q = q[:, 4:]
    big = torch.zeros((13, 8, 128), dtype=torch.float16, device="cuda")
    o, lse = t.run(o=big[..., :64])
    t.check(o, lse)
    assert bool((big[..., 64:] == 0).all())


def test_tree_large_offsets(cuda_device):
    """Pages past 2^31 elements into the cache."""
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 20 GB")
    t = Tree([260, 40], [3, 1], 8, 8, 128, 128, torch.bfloat16, seed=14)
    kc, vc = (torch.empty((16400, 128, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for r in range(2):
        for j in range(t.table.shape[1]):
            p = int(t.table[r, j])
            if p >= 0:
                far = 16399 - p
                kc[far], vc[far] = t.kc[p], t.vc[p]
                t.table[r, j] = far
    t.kc, t.vc = kc, vc
    o, lse = t.run()
    t.check(o, lse)


def test_tree_deterministic_on_any_stream(cuda_device):
    t = Tree([9000, 70, 700], [3, 1, 30], 8, 2, 128, 16, torch.bfloat16, seed=15)
    a, la = t.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = t.run()
        lens, cu, c = torch.tensor(t.lens, dtype=torch.int32, device="cuda"), _cu(t.new), torch.empty_like(t.q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attention.attention_tree(t.q, t.kc, t.vc, t.table, lens, cu, t.mask, c)
        graph.replay()
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b) and torch.equal(la, lb) and torch.equal(a, c)


def test_tree_refusals(cuda_device):
    t = Tree([100], [4], 4, 2, 64, 16, torch.float16, seed=16)
    lens, cu = torch.tensor([100], dtype=torch.int32, device="cuda"), _cu([4])
    good = dict(q=t.q, k_cache=t.kc, v_cache=t.vc, block_tables=t.table, seq_lens=lens, cu_seqlens=cu,
                tree_mask=t.mask)
    attention.attention_tree(**good)
    for kw in (dict(q=t.q.bfloat16()), dict(q=t.q[..., :32]), dict(q=t.q[:, :3]), dict(q=t.q[0]),
               dict(k_cache=t.kc[:1]), dict(k_cache=t.kc.bfloat16(), v_cache=t.vc.bfloat16()),
               dict(block_tables=t.table.long()), dict(block_tables=t.table[0]), dict(seq_lens=lens.long()),
               dict(cu_seqlens=cu[:1]), dict(tree_mask=t.mask.int()), dict(tree_mask=t.mask[:3]),
               dict(tree_mask=t.mask[:, :0]), dict(lse=torch.empty((4, 3), device="cuda"))):
        with pytest.raises(ValueError):
            attention.attention_tree(**{**good, **kw})
    odd = torch.zeros((4, 24, 2, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(_lib.B2GError):  # a page size that tiles cannot be made of
        attention.attention_tree(**{**good, "k_cache": odd, "v_cache": odd})


# ---------------------------------------------------------------- together --
def test_a_step_of_serving(cuda_device):
    """Prompts prefilled and written, then a tree of drafts over the cache: the drafted path that
    is one chain equals the same tokens prefilled as part of their prompt."""
    hq, hk, d, page, dtype = 8, 2, 64, 16, torch.bfloat16
    lens, drafts = [37, 150, 4], 6
    g = _gen(30)
    whole = [n + drafts for n in lens]
    q, k, v = (_rand(g, sum(whole), h, d, dtype=dtype) for h in (hq, hk, hk))
    full = attention.attention_prefill(q, k, v, _cu(whole))
    at = np.cumsum([0] + whole)
    is_new = np.concatenate([[i >= n for i in range(n + drafts)] for n in lens])
    old, fresh = (torch.tensor(np.flatnonzero(x), device="cuda") for x in (~is_new, is_new))
    kc, vc = (torch.full((40, page, hk, d), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    table = torch.zeros((3, 12), dtype=torch.int32, device="cuda")
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    free = torch.randperm(40, generator=g, device="cuda").int()
    m = kvcache.map_step(ints([0] * 3), ints(lens), ints([0] * 3), table, free, ints([40]),
                         page_size=page, num_tokens=sum(lens))
    kvcache.write_kv(k[old], v[old], kc, vc, m.slots)
    m = kvcache.map_step(m.seq_lens, ints([drafts] * 3), m.page_counts, table, free, m.num_free,
                         page_size=page, num_tokens=3 * drafts)
    kvcache.write_kv(k[fresh], v[fresh], kc, vc, m.slots)
    words = [(1 << i + 1) - 1 for i in range(drafts)] * 3
    for mask in (None, _mask(words, 1)):
        o = attention.attention_tree(q[fresh], kc, vc, table, m.seq_lens, m.cu_seqlens, mask)
        ops.check_status()
        assert int(m.num_free) == 40 - sum(-(-n // page) for n in whole)
        # two roundings of the output and of the weights apart
        diff = (o.float() - full[fresh].float()).abs()
        size = v.float().abs().max()
        assert float(diff.max()) <= 4 * 2.0 ** -8 * float(size)
        assert at[-1] == sum(whole)


def test_graph_outlives_a_larger_call(cuda_device):
    """A captured call keeps its workspace when a larger one on the same stream needs more."""
    small, big = (Tree(n, new, 8, 2, 128, 16, torch.bfloat16, seed=17) for n, new in
                  (([3000], [1]), ([500] * 9, [40] * 9)))
    side = torch.cuda.Stream()  # a stream that has no workspace yet
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, _ = small.run()
        lens, cu, o = torch.tensor(small.lens, dtype=torch.int32, device="cuda"), _cu([1]), torch.empty_like(small.q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attention.attention_tree(small.q, small.kc, small.vc, small.table, lens, cu, small.mask, o)
        before = ops.workspace(0, side.device)
        big.run()
        assert ops.workspace(0, side.device) is not before and any(x is before for x in ops._outgrown)
        torch.cuda.empty_cache()
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    ops.check_status()
    assert torch.equal(o, want)


def test_example_serves(cuda_device):
    """The example's last tokens equal a prefill of the accepted sequences up to two roundings
    of the weights and of the output, and the projections' own (values of a few units)."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(__file__), "..", "examples", "serve_step.py")
    spec = importlib.util.spec_from_file_location("serve_step", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    assert example.main() <= 4 * 2.0 ** -8 * 6.0  # 6: above any of the normal values of V


def test_tree_join_that_never_comes(cuda_device):
    """Parts that nobody publishes: every wait runs out, the kernel ends with a status, and the
    next call is right again."""
    t = Tree([9000, 70], [3, 1], 8, 2, 128, 16, torch.bfloat16, seed=18)
    want, _ = t.run()
    limit = _lib.get_option(_lib.OPT_TIMEOUT_MS)
    try:
        _lib.set_option(_lib.OPT_TIMEOUT_MS, 20)
        _lib.set_option(_lib.OPT_INJECT_FLAG_TIMEOUT, 1)
        with pytest.raises(_lib.B2GError) as e:
            t.run()
        assert e.value.code == _lib.STATUS_TIMEOUT | _lib.SITE_FLAG
    finally:
        _lib.set_option(_lib.OPT_INJECT_FLAG_TIMEOUT, 0)
        _lib.set_option(_lib.OPT_TIMEOUT_MS, limit)
    o, lse = t.run()
    t.check(o, lse)
    assert torch.equal(o, want)


@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("new", [1, 12, 25, 70], ids=["four copies", "two copies", "one", "two row tiles"])
def test_tree_odd_value_in_the_context(cuda_device, new, what):
    """A value of an older token that is not finite comes out in its dim of every row, as itself,
    and changes no other dim."""
    t = Tree([900 + new], [new], 8, 2, 128, 16, torch.bfloat16, seed=19, masked=False)
    want, _ = t.run()
    page, slot = int(t.table[0, 517 // 16]), 517 % 16
    t.vc[page, slot, :, 7] = what
    o, _ = t.run()
    got = o[..., 7].float()
    assert bool(got.isnan().all() if math.isnan(what) else (got == what).all())
    keep = torch.arange(128, device="cuda") != 7
    assert torch.equal(o[..., keep], want[..., keep])

"""Page bookkeeping and cache stores on the GPU: whole values, compared for equality."""

from __future__ import annotations

import random

import pytest
import torch

from gfx950_gluon_tutorials_b200 import _lib, kvcache, ops
from oracle import serving

pytestmark = pytest.mark.gpu


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _map(cached, new, held, tables, free, num_free, page, num_tokens):
    dev = _ints(tables) if tables else torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    m = kvcache.map_step(_ints(cached), _ints(new), _ints(held), dev, _ints(free),
                         _ints([num_free]), page_size=page, num_tokens=num_tokens)
    return m, dev


def _problem(requests, page, top, seed, spare=4):
    rng = random.Random(seed)
    cached = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, top)]) for _ in range(requests)]
    new = [rng.choice([0, 1, page, rng.randint(0, top)]) for _ in range(requests)]
    held = [-(-c // page) + rng.choice([0, 0, 1]) for c in cached]
    width = max(max(-(-(c + n) // page), h) for c, n, h in zip(cached, new, held)) + 1
    need = sum(max(0, -(-(c + n) // page) - h) for c, n, h in zip(cached, new, held))
    ids = list(range(sum(held) + need + spare))
    rng.shuffle(ids)
    tables = []
    for h in held:
        tables.append([ids.pop() for _ in range(h)] + [-7] * (width - h))
    return cached, new, held, tables, ids, len(ids)


def _same(m, dev, want, tables):
    torch.cuda.synchronize()
    assert dev.tolist() == tables
    for name in ("slots", "positions", "cu_seqlens", "seq_lens", "page_counts", "num_free"):
        assert getattr(m, name).tolist() == want[name], name


@pytest.mark.parametrize("requests,page,top", [(1, 16, 40), (7, 16, 200), (33, 8, 50), (130, 64, 700),
                                               (512, 1, 9), (513, 32, 60), (1500, 128, 300), (8192, 16, 20)])
def test_map_step(cuda_device, requests, page, top):
    args = _problem(requests, page, top, seed=requests + page)
    total = sum(args[1])
    m, dev = _map(*args, page, total + 5)  # five rows of padding
    want = serving.map_step(*args[:3], args[3], *args[4:], page, total + 5)
    _same(m, dev, want, args[3])
    ops.check_status()


def test_map_step_twice_is_the_same(cuda_device):
    cached, new, held, tables, free, n = _problem(20, 16, 90, seed=3)
    dev = _ints(tables)
    args = [_ints(x) for x in (cached, new, held)] + [dev, _ints(free), _ints([n])]
    a = kvcache.map_step(*args, page_size=16, num_tokens=sum(new))
    first = dev.clone()
    b = kvcache.map_step(*args, page_size=16, num_tokens=sum(new))
    assert torch.equal(first, dev) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_map_step_when_pages_run_out(cuda_device):
    args = _problem(40, 16, 100, seed=5)
    short = list(args)
    short[5] = 9  # of the free pages only nine are left
    m, dev = _map(*short, 16, sum(args[1]))
    want = serving.map_step(*short[:3], short[3], *short[4:], 16, sum(args[1]))
    assert want["num_free"][0] < 0 and -1 in want["slots"]
    _same(m, dev, want, short[3])
    ops.check_status()


def test_map_step_empty(cuda_device):
    m, _ = _map([], [], [], [], [4], 1, 16, 3)
    assert m.slots.tolist() == [-1] * 3 and m.cu_seqlens.tolist() == [0] and m.num_free.tolist() == [1]
    m, dev = _map([5], [0], [1], [[2]], [], 0, 16, 0)
    assert m.cu_seqlens.tolist() == [0, 0] and m.seq_lens.tolist() == [5] and dev.tolist() == [[2]]
    ops.check_status()


def test_map_step_reports_small_tables_and_token_counts(cuda_device):
    m, dev = _map([0], [40], [0], [[-7, -7]], [3, 1, 0], 3, 16, 40)
    with pytest.raises(_lib.B2GError) as e:
        ops.check_status()
    assert e.value.code == _lib.STATUS_PAGE_TABLE
    assert dev.tolist() == [[0, 1]] and m.slots.tolist()[32:] == [-1] * 8
    assert m.slots.tolist()[:32] == list(range(32)) and m.num_free.tolist() == [1]
    m, _ = _map([0, 0], [5, 9], [0, 0], [[0], [0]], [3, 1], 2, 16, 8)
    with pytest.raises(_lib.B2GError) as e:
        ops.check_status()
    assert e.value.code == _lib.STATUS_TOKENS and m.cu_seqlens.tolist() == [0, 5, 8]


def test_map_step_strided_table(cuda_device):
    cached, new, held, tables, free, n = _problem(6, 16, 90, seed=8)
    wide = torch.full((6, 2 * len(tables[0])), -9, dtype=torch.int32, device="cuda")
    view = wide[:, :len(tables[0])]
    view.copy_(_ints(tables))
    m = kvcache.map_step(_ints(cached), _ints(new), _ints(held), view, _ints(free), _ints([n]),
                         page_size=16, num_tokens=sum(new))
    want = serving.map_step(cached, new, held, tables, free, n, 16, sum(new))
    _same(m, view, want, tables)
    assert bool((wide[:, len(tables[0]):] == -9).all())


# (tokens, heads, dim, page, layout of the cache, how k and v lie)
WRITES = [(1, 1, 64, 16, "slots", "plain"), (45, 4, 64, 16, "slots", "fused"),
          (300, 8, 128, 64, "heads", "plain"), (77, 3, 128, 128, "heads", "fused"),
          (130, 5, 96, 8, "slots", "plain"), (33, 2, 7, 5, "slots", "plain"),
          (33, 2, 12, 16, "heads", "fused"), (40, 2, 64, 16, "slots", "odd"),
          (2000, 8, 128, 32, "layers", "fused")]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", WRITES, ids=lambda c: "-".join(map(str, c)))
def test_write_kv(cuda_device, case, dtype):
    tokens, heads, dim, page, layout, lie = case
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    pages = -(-tokens // page) + 2

    def rand(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    if lie == "fused":
        both = rand(tokens, 3 * heads, dim)
        k, v = both[:, heads:2 * heads], both[:, 2 * heads:]
    elif lie == "odd":  # rows that start at odd addresses
        both = rand(tokens, 2, heads, dim + 1)
        k, v = both[:, 0, :, 1:], both[:, 1, :, 1:]
    else:
        k, v = rand(tokens, heads, dim), rand(tokens, heads, dim)
    if layout == "heads":
        kc, vc = (rand(pages, heads, page, dim).transpose(1, 2) for _ in range(2))
    elif layout == "layers":
        kc, vc = rand(pages, 2, page, heads, dim)[:, 1], rand(pages, 3, page, heads, dim)[:, 2]
    else:
        kc, vc = rand(pages, page, heads, dim), rand(pages, page, heads, dim)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[tokens // 2] = -1  # padding
    want_k, want_v = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            want_k[s // page, s % page], want_v[s // page, s % page] = k[t], v[t]
    kvcache.write_kv(k, v, kc, vc, slots)
    ops.check_status()
    for a, b in ((kc, want_k), (vc, want_v)):
        assert torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


def test_write_kv_slot_past_the_cache(cuda_device):
    k = torch.ones((3, 1, 64), dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros((2, 16, 1, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    kvcache.write_kv(k, k, kc, vc, torch.tensor([0, 32, 31], device="cuda"))
    with pytest.raises(_lib.B2GError) as e:
        ops.check_status()
    assert e.value.code == _lib.STATUS_SLOT
    assert kc.view(32, 64).any(1).nonzero().flatten().tolist() == [0, 31]
    kvcache.write_kv(k[:0], k[:0], kc, vc, torch.zeros(0, dtype=torch.int64, device="cuda"))
    ops.check_status()


def test_write_kv_refusals(cuda_device):
    k = torch.ones((3, 1, 64), dtype=torch.float16, device="cuda")
    kc = torch.zeros((2, 16, 1, 64), dtype=torch.float16, device="cuda")
    s = torch.zeros(3, dtype=torch.int64, device="cuda")
    for args in ((k, k[:2], kc, kc, s), (k, k, kc, kc, s.int()), (k, k, kc, kc, s[:2]),
                 (k.bfloat16(), k, kc, kc, s), (k, k, kc.float(), kc.float(), s),
                 (k[:, :, :32], k[:, :, :32], kc, kc, s), (k.float(), k.float(), kc, kc, s),
                 (k, k, kc, kc[:1], s), (k, k, kc.transpose(2, 3), kc.transpose(2, 3), s)):
        with pytest.raises(ValueError):
            kvcache.write_kv(*args)


def test_large_offsets(cuda_device):
    """Slots past 2^31 elements into a cache of 9 GB."""
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 20 GB")
    kc, vc = (torch.empty((16400, 128, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k = torch.randn((4, 8, 128), device="cuda").bfloat16()
    slots = torch.tensor([16399 * 128 + 127, 0, 16399 * 128, 9000 * 128 + 5], device="cuda")
    kvcache.write_kv(k, -k, kc, vc, slots)
    ops.check_status()
    assert torch.equal(kc.view(-1, 8, 128)[slots], k) and torch.equal(vc.view(-1, 8, 128)[slots], -k)


def test_another_stream_and_graph(cuda_device):
    """Runs where the caller's stream is, and can be captured and replayed."""
    cached, new, held, tables, free, n = _problem(9, 16, 60, seed=12)
    args = [_ints(cached), _ints(new), _ints(held), _ints(tables), _ints(free), _ints([n])]
    want = serving.map_step(cached, new, held, tables, free, n, 16, sum(new))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m = kvcache.map_step(*args, page_size=16, num_tokens=sum(new))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            m2 = kvcache.map_step(*args, page_size=16, num_tokens=sum(new))
        m2.slots.zero_()
        graph.replay()
    torch.cuda.current_stream().wait_stream(side)
    _same(m, args[3], want, tables)
    assert m2.slots.tolist() == want["slots"]

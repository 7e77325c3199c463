"""Edges of the serving attention that the tests of single cases pass by: how shares of work are
found, rows of NaN, sums after late maxima, graphs captured on streams that never ran before, and
batches large enough for every way of planning the work. Against float64, as there."""

from __future__ import annotations

import os
import random
import subprocess
import sys

import pytest
import torch

from gfx950_gluon_tutorials_b200 import _lib, attention, ops
from oracle import serving
from test_attention_serving_gpu import (DTYPES, UNIT, Tree, _check_prefill, _close, _cu, _gen, _np,
                                        _prefill, _rand)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp16", "bf16"])
@pytest.mark.parametrize("lens,new", [([200], [1]), ([5, 90, 1], [1, 2, 1]),
                                      ([3000, 40, 0, 700, 129, 2500, 64], [3, 1, 0, 2, 9, 1, 30])],
                         ids=["fewer tiles than SMs", "short", "uneven"])
def test_tree_finds_its_shares_every_time(cuda_device, lens, new, dtype):
    """Calls in a row, nothing between them, all give the first one's bits: no share is lost."""
    t = Tree(lens, new, 8, 2, 128, 16, dtype, seed=40)
    o, lse = t.run()
    t.check(o, lse)
    runs = [t.run() for _ in range(50)]
    assert all(torch.equal(o, a) and torch.equal(lse, b) for a, b in runs)


ARRANGEMENTS = pytest.mark.parametrize(
    "new", [1, 12, 25, 70], ids=["four copies", "two copies", "one", "two row tiles"])


@ARRANGEMENTS
@pytest.mark.parametrize("keys,requests", [(90, 1), (777, 1), (9000, 1), (300, 150)],
                         ids=["one tile", "few tiles", "split", "whole blocks"])
def test_tree_query_of_nan(cuda_device, keys, requests, new):
    """A query row that holds a NaN comes out as NaN, sums too, however its keys are split; the
    other rows keep their bits."""
    t = Tree([keys + new] * requests, [new] * requests, 8, 2, 128, 16, torch.bfloat16, seed=41)
    want, want_lse = t.run()
    bad = torch.zeros((requests * new, 8), dtype=torch.bool, device="cuda")
    bad[new // 2::7, 3] = True
    bad[new - 1, 6] = True
    t.q[bad, 5] = float("nan")
    o, lse = t.run()
    assert bool(o[bad].isnan().all()) and bool(lse.t()[bad].isnan().all())
    assert torch.equal(o[~bad], want[~bad]) and torch.equal(lse.t()[~bad], want_lse.t()[~bad])


@ARRANGEMENTS
def test_tree_keys_of_nan_fill_a_share(cuda_device, new):
    """Keys of NaN that are all that some CTAs see of a long context reach every row."""
    t = Tree([9000 + new], [new], 8, 2, 128, 16, torch.bfloat16, seed=42, masked=False)
    at = torch.arange(30 * 128, 33 * 128, device="cuda")
    t.kc[t.table[0].long()[at // 16], at % 16] = float("nan")
    o, lse = t.run()
    assert bool(o.isnan().all()) and bool(lse.isnan().all())


def _fresh_stream(keep):
    """A stream without a workspace, and its key."""
    stream = torch.cuda.Stream()
    key = (stream.device.index, stream.cuda_stream)
    torch.cuda.synchronize()
    keep.append(ops._workspaces.pop(key, None))  # an earlier test's graph may still hold it
    return stream, key


def _capture(t, stream):
    """A graph of one call on t, captured on ``stream``, and the call's output."""
    lens, cu, o = torch.tensor(t.lens, dtype=torch.int32, device="cuda"), _cu(t.new), torch.empty_like(t.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        attention.attention_tree(t.q, t.kc, t.vc, t.table, lens, cu, t.mask, o)
    return graph, o, (lens, cu)


def test_graphs_captured_on_a_stream_that_never_ran(cuda_device):
    """Two graphs on one such stream, the second with a larger workspace and replayed first; what
    they wait on is zero before any of them runs, whatever the memory held."""
    small, big = (Tree(n, new, 8, 2, 128, 16, torch.bfloat16, seed=45) for n, new in
                  (([3000], [1]), ([500] * 9, [40] * 9)))
    want = [t.run()[0] for t in (small, big)]
    dirt = [torch.full((n << 20,), 255, dtype=torch.uint8, device="cuda") for n in (1, 2, 8, 64, 200)]
    del dirt
    keep = []
    stream, key = _fresh_stream(keep)
    first, o1, hold1 = _capture(small, stream)
    assert not bool(ops._workspaces[key].any())
    second, o2, hold2 = _capture(big, stream)
    assert not bool(ops._workspaces[key].any())
    for graph, o, expected in ((second, o2, want[1]), (first, o1, want[0]), (second, o2, want[1])):
        o.fill_(float("nan"))
        graph.replay()
        assert torch.equal(o, expected)
    ops.check_status()


def test_a_replay_clears_nothing(cuda_device):
    """The workspace's clearing is no part of a graph that was captured on a fresh stream."""
    t = Tree([3000], [1], 8, 2, 128, 16, torch.bfloat16, seed=46)
    want, _ = t.run()
    keep = []
    stream, key = _fresh_stream(keep)
    lens, cu, o = torch.tensor(t.lens, dtype=torch.int32, device="cuda"), _cu(t.new), torch.empty_like(t.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ws = ops.workspace(96 << 20, cuda_device)  # more than the call takes
        attention.attention_tree(t.q, t.kc, t.vc, t.table, lens, cu, t.mask, o)
    assert ops._workspaces[key] is ws and not bool(ws.any())
    ws[-1] = 7
    graph.replay()
    assert torch.equal(o, want) and int(ws[-1]) == 7
    ws[-1] = 0
    ops.check_status()


FIRST_CALL = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from gfx950_gluon_tutorials_b200 import attention, ops
q, k, v = (torch.randn((50, h, 64), device="cuda").half() for h in (4, 2, 2))
cu, o = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda"), torch.empty_like(q)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    attention.attention_prefill(q, k, v, cu, o)
ops.check_status()
ops.status_tensor(q.device).fill_(0x5000)  # as a kernel of another graph reports
graph.replay()
try:
    ops.check_status()
    raise SystemExit("the replay cleared the status word")
except ops.B2GError as e:
    assert e.code == 0x5000
assert torch.equal(o, attention.attention_prefill(q, k, v, cu))
ops.check_status()
print("as expected")
"""


def test_first_call_of_a_process_is_captured(cuda_device):
    """The status word too is there and clear before the first replay, and no replay clears it."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", FIRST_CALL, root], capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "as expected" in out.stdout, out.stdout + out.stderr


# Many keys of score 0, then one 8 to 9.4 powers of two above: the maximum moves once, and what
# was summed before still is most of the sum. A head for each of 16 such scores.
LATE = dict(start=5.6, end=6.5, steps=16)


def test_prefill_sum_before_a_late_maximum(cuda_device):
    n, hq, d = 12001, 16, 64
    q, k = (torch.zeros((n, h, d), dtype=torch.float16, device="cuda") for h in (hq, 1))
    v = _rand(_gen(43), n, 1, d, dtype=torch.float16)
    q[..., 0] = torch.linspace(**LATE, device="cuda").half()
    k[-1, :, 0] = 1.0
    o, lse = _prefill(q, k, v, [n], scale=1.0)
    for h in range(hq):
        ref = serving.attend(_np(q[-1:, h]), _np(k[:, 0]), _np(v[:, 0]), serving.causal(n)[-1:], 1.0,
                             UNIT[q.dtype])
        _close(_np(o[-1:, h]), _np(lse[h, -1:]), ref, f"head {h}")


def test_tree_sum_before_a_late_maximum(cuda_device):
    """Enough requests that a CTA holds most of a request's keys."""
    keys, requests, new, hq, d, at = 3009, 150, 9, 16, 64, 2990
    t = Tree([keys] * requests, [new] * requests, hq, 1, d, 64, torch.float16, seed=44, masked=False)
    t.kc.zero_()
    t.q.zero_()
    t.q[..., 0] = torch.linspace(**LATE, device="cuda").half()
    for r in range(requests):
        t.k[r].zero_()
        t.k[r][at, 0, 0] = 1.0
        t.kc[t.table[r, at // 64], at % 64, 0, 0] = 1.0
    o, lse = t.run(scale=1.0)
    t.check(o, lse, scale=1.0, heads=range(hq), requests=[0, 1, 2, 74, 75, 149])


def test_prefill_offsets_that_ask_for_too_much(cuda_device):
    """Offsets that go back and forth over a million tokens until the blocks that they name pass
    2^31 are reported, and no block of them is run; the next call is right."""
    tokens, prompts = 1 << 20, (1 << 19) + 1024
    cu = torch.zeros(prompts + 1, dtype=torch.int32, device="cuda")
    cu[1::2] = tokens
    assert (prompts // 2) * (tokens // 128) > 2 ** 31
    q = torch.zeros((tokens, 2, 64), dtype=torch.float16, device="cuda")
    k = torch.zeros((tokens, 1, 64), dtype=torch.float16, device="cuda")
    o = torch.full_like(q, 7.0)
    attention.attention_prefill(q, k, k, cu, o)
    with pytest.raises(ops.B2GError) as e:
        ops.check_status()
    assert e.value.code == _lib.STATUS_TOKENS and bool((o == 7.0).all())
    lens = [300] * 400  # enough blocks for the planning kernel
    g = _gen(47)
    q, k, v = (_rand(g, sum(lens), h, 64, dtype=torch.float16) for h in (2, 1, 1))
    o, lse = _prefill(q, k, v, lens)
    _check_prefill(q, k, v, lens, o, lse, 0.125, skip=range(3, 398))


def test_tree_offsets_that_ask_for_too_much(cuda_device):
    """Offsets that decrease are reported; those that name every row for every second of many
    requests are not run at all. The next call is right."""
    tokens, requests = 4096, 4096
    t = Tree([100], [3], 2, 2, 64, 16, torch.float16, seed=48)
    q = torch.zeros((tokens, 2, 64), dtype=torch.float16, device="cuda")
    lens = torch.full((requests,), 100, dtype=torch.int32, device="cuda")
    table = t.table.expand(requests, -1).contiguous()
    for cu, run in ((torch.arange(requests + 1, device="cuda").int(), True),
                    (torch.arange(requests + 1, device="cuda").int() % 2 * tokens, False)):
        o = torch.full_like(q, 7.0)
        attention.attention_tree(q, t.kc, t.vc, table, lens, cu, None, o)
        if run:
            ops.check_status()
            assert not bool((o == 7.0).all(-1).any())
        else:
            with pytest.raises(ops.B2GError) as e:
                ops.check_status()
            assert e.value.code == _lib.STATUS_TOKENS and bool((o == 7.0).all())
    o, lse = t.run()
    t.check(o, lse)


@pytest.mark.parametrize("requests,hq,hk,d", [(321, 4, 2, 64), (700, 4, 2, 64), (1000, 8, 1, 128)])
def test_tree_more_requests_than_threads(cuda_device, requests, hq, hk, d):
    """More requests than a CTA has threads: shares are found in several rounds, across runs of
    requests without new tokens that span the rounds' borders."""
    rng = random.Random(requests)
    lens = [rng.choice([1, 5, 64, 129, 300]) for _ in range(requests)]
    new = [min(n, rng.choice([0, 1, 1, 3, 9])) for n in lens]
    for r in (*range(300, min(340, requests - 1)), *range(630, min(660, requests - 1))):
        new[r] = 0
    lens[-1] = new[-1] = 1
    t = Tree(lens, new, hq, hk, d, 16, torch.bfloat16, seed=requests)
    o, lse = t.run()
    t.check(o, lse, heads=[0, hq - 1])


def test_tree_no_request_but_the_last(cuda_device):
    """Rounds of requests without any work before the one that has some."""
    t = Tree([0] * 650 + [2000], [0] * 650 + [5], 4, 2, 64, 16, torch.float16, seed=49)
    o, lse = t.run()
    t.check(o, lse)


@pytest.mark.parametrize("hq,hk,d", [(3, 3, 64), (10, 2, 128), (1, 1, 128), (4, 2, 64)])
def test_prefill_planned_blocks(cuda_device, hq, hk, d):
    """Enough blocks for the planning kernel, where an odd number of query heads per key/value
    head takes two row tiles at a time and a ragged one by pairs of heads."""
    rng = random.Random(hq)
    lens = [rng.choice([1, 100, 128, 129, 255, 256, 257, 400, 513, 700]) for _ in range(180)]
    g, t = _gen(hq), sum(lens)
    block = 256 if hq // hk % 2 else 128
    assert sum(-(-n // block) for n in lens) > 256
    q, k, v = (_rand(g, t, h, d, dtype=torch.bfloat16) for h in (hq, hk, hk))
    o, lse = _prefill(q, k, v, lens)
    _check_prefill(q, k, v, lens, o, lse, d ** -0.5, skip=[b for b in range(180) if b % 6])


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 2)])
def test_prefill_more_prompts_than_threads(cuda_device, hq, hk):
    """Hundreds of prompts, nearly all of them empty."""
    lens = [0] * 500
    for b, n in ((0, 3), (7, 300), (319, 1), (320, 129), (321, 256), (498, 40)):
        lens[b] = n
    g, t = _gen(50), sum(lens)
    q, k, v = (_rand(g, t, h, 64, dtype=torch.float16) for h in (hq, hk, hk))
    o, lse = _prefill(q, k, v, lens)
    _check_prefill(q, k, v, lens, o, lse, 0.125)

"""Edges of the serving attention that the tests of single cases pass by: how shares of work are
found, rows of NaN, sums after late maxima, graphs captured on streams that never ran before, and
batches large enough for every way of planning the work. Against float64, as there."""

from __future__ import annotations

import pytest
import torch

from test_attention_serving_gpu import DTYPES, Tree

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

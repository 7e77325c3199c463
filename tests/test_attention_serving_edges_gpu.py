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

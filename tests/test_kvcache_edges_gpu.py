"""Edges of the page bookkeeping that depend on what the process did before."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

COUNTS = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from gfx950_gluon_tutorials_b200 import kvcache, ops
from oracle import serving

def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")

for n in (6112, 6113, 6144, 6145):
    cached, new, held = [r % 5 for r in range(n)], [r % 3 for r in range(n)], [0] * n
    tables, free = [[-7] for _ in range(n)], list(range(n))
    dev = ints(tables)
    m = kvcache.map_step(ints(cached), ints(new), ints(held), dev, ints(free), ints([n]),
                         page_size=16, num_tokens=sum(new))
    want = serving.map_step(cached, new, held, tables, free, n, 16, sum(new))
    ops.check_status()
    assert dev.tolist() == tables, n
    for name in want:
        assert getattr(m, name).tolist() == want[name], (n, name)
print("as expected")
"""


def test_map_step_request_counts_around_48_kb(cuda_device):
    """Request counts whose sums take just under and just over 48 KB of shared memory, in a
    process that has made no larger call yet."""
    out = subprocess.run([sys.executable, "-c", COUNTS, ROOT], capture_output=True, text=True,
                         timeout=300)
    assert out.returncode == 0 and "as expected" in out.stdout, out.stdout + out.stderr

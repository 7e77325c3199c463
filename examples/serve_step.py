"""One attention layer served with a paged cache: prompts, a tree of drafts, single tokens.

    python examples/serve_step.py

A batch of prompts is projected with the framework's GEMM, gets pages and slots from
``kvcache.map_step``, is stored with ``kvcache.write_kv`` and attended with
``attention.attention_prefill``. Then every request drafts a small tree of tokens that
``attention.attention_tree`` attends over the cache in one call; one path of each tree is
accepted, its keys and values move to the front of the drafts' slots, and the accepted
tokens count as cached from then on. Single tokens follow. At the end the last tokens'
outputs are compared with a prefill of the whole accepted sequences.
"""

from __future__ import annotations

import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from gfx950_gluon_tutorials_b200 import a16w16, attention, kvcache, ops  # noqa: E402

WIDTH, HQ, HK, D, PAGE = 1024, 8, 2, 128, 16
# drafted token i's parent in its tree (-1: the last accepted token), and an accepted path
PARENTS, PATH = [-1, 0, 0, 1, 2, 2], [0, 2, 5]


def ancestor_words(parents: list[int]) -> list[int]:
    """Bit j of word i: token i sees token j (its ancestors and itself)."""
    words: list[int] = []
    for i, up in enumerate(parents):
        words.append((words[up] if up >= 0 else 0) | 1 << i)
    return words


class Layer:
    """Projection weights, the layer's cache and the bookkeeping of a batch of requests."""

    def __init__(self, requests: int, pages: int, max_pages: int, seed: int = 0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.w = (torch.randn(((HQ + 2 * HK) * D, WIDTH), generator=g, device="cuda")
                  * WIDTH ** -0.5).bfloat16()
        self.k_cache, self.v_cache = (torch.empty((pages, PAGE, HK, D), dtype=torch.bfloat16,
                                                  device="cuda") for _ in range(2))
        self.tables = torch.zeros((requests, max_pages), dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=g, device="cuda").int()
        self.num_free = torch.tensor([pages], dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.pages_held = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def project(self, x: torch.Tensor):
        """q (tokens, HQ, D), k and v (tokens, HK, D) as views of one product."""
        qkv = a16w16.matmul(x, self.w.T).view(-1, HQ + 2 * HK, D)
        return qkv[:, :HQ], qkv[:, HQ:HQ + HK], qkv[:, HQ + HK:]

    def append(self, k: torch.Tensor, v: torch.Tensor, new: list[int]) -> kvcache.StepMaps:
        """Pages and slots for ``new`` tokens per request, and their keys and values in them."""
        m = kvcache.map_step(self.lens, torch.tensor(new, dtype=torch.int32, device="cuda"),
                             self.pages_held, self.tables, self.free, self.num_free,
                             page_size=PAGE, num_tokens=sum(new))
        kvcache.write_kv(k, v, self.k_cache, self.v_cache, m.slots)
        self.pages_held, self.num_free = m.page_counts, m.num_free
        return m

    def attend(self, q: torch.Tensor, m: kvcache.StepMaps, mask: torch.Tensor | None = None):
        return attention.attention_tree(q, self.k_cache, self.v_cache, self.tables, m.seq_lens,
                                        m.cu_seqlens, mask)


def main() -> float:
    lens = [37, 260, 5]
    n, t = len(lens), len(PARENTS)
    g = torch.Generator(device="cuda").manual_seed(1)
    layer = Layer(n, pages=64, max_pages=24)

    def tokens(count: int) -> torch.Tensor:
        return torch.randn((count, WIDTH), generator=g, device="cuda").bfloat16()

    # the prompts
    x = tokens(sum(lens))
    q, k, v = layer.project(x)
    m = layer.append(k, v, lens)
    layer.lens = m.seq_lens
    attention.attention_prefill(q, k, v, m.cu_seqlens)

    # a tree of drafts per request, all of them in one call
    drafts = tokens(n * t)
    q, k, v = layer.project(drafts)
    m = layer.append(k, v, [t] * n)
    mask = torch.tensor(ancestor_words(PARENTS) * n, dtype=torch.int64, device="cuda").view(-1, 1)
    layer.attend(q, m, mask)

    # the accepted path moves to the front of the drafts' slots
    rows = torch.arange(n, device="cuda")[:, None] * t
    kept = (rows + torch.tensor(PATH, device="cuda")).flatten()
    front = (rows + torch.arange(len(PATH), device="cuda")).flatten()
    kvcache.write_kv(k[kept], v[kept], layer.k_cache, layer.v_cache, m.slots[front])
    layer.lens = layer.lens + len(PATH)

    # one token per request
    last = tokens(n)
    q, k, v = layer.project(last)
    m = layer.append(k, v, [1] * n)
    o = layer.attend(q, m)
    ops.check_status()

    # the same sequences in one go
    whole, ends, at = [], [], 0
    for r, length in enumerate(lens):
        whole += [x[at:at + length], drafts[kept[r * len(PATH):(r + 1) * len(PATH)]], last[r:r + 1]]
        at += length
        ends.append(length + len(PATH) + 1)
    q, k, v = layer.project(torch.cat(whole))
    cu = torch.tensor([0] + ends, dtype=torch.int32, device="cuda").cumsum(0).int()
    want = attention.attention_prefill(q, k, v, cu)[cu[1:].long() - 1]
    ops.check_status()
    diff = float((o.float() - want.float()).abs().max())
    print(f"{n} requests, {int(layer.num_free)} of {layer.free.numel()} pages free, last tokens "
          f"differ from a prefill of the whole sequences by at most {diff:.2e}")
    return diff


if __name__ == "__main__":
    main()

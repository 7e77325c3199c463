"""Refusals of the paged-cache and serving-attention entry points, before anything touches a GPU,
and the integer restatement of the page bookkeeping on a case worked out by hand."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gfx950_gluon_tutorials_b200 import _lib, attention, kvcache
from oracle import serving


def _st(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_oracle_by_hand():
    # pages of 4; request 0 holds page 7 with 3 tokens and gets 6 more, request 1 is new
    tables = [[7, 0, 0], [0, 0, 0]]
    out = serving.map_step([3, 0], [6, 1], [1, 0], tables, [5, 9, 2, 8], 4, 4, 8)
    assert tables == [[7, 8, 2], [9, 0, 0]]
    assert out["slots"] == [31, 32, 33, 34, 35, 8, 36, -1]
    assert out["positions"] == [3, 4, 5, 6, 7, 8, 0, 0]
    assert out["cu_seqlens"] == [0, 6, 7] and out["seq_lens"] == [9, 1]
    assert out["page_counts"] == [3, 1] and out["num_free"] == [1]


MAP = dict(cached=16, new=16, counts=16, tables=16, stride=8, requests=2, max_pages=8, free=16,
           cap=4, num_free=16, page=16, tokens=4, slots=16, positions=16, cu=16, seq=16,
           counts_out=16, num_free_out=16, status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(requests=-1), _lib.ESHAPE), (dict(page=0), _lib.ESHAPE), (dict(tokens=-1), _lib.ESHAPE),
    (dict(tokens=2 ** 31), _lib.ESHAPE), (dict(requests=8193), _lib.ECAPACITY),
    (dict(cached=None), _lib.EINVAL), (dict(tables=None), _lib.EINVAL),
    (dict(cu=None), _lib.EINVAL), (dict(slots=None), _lib.EINVAL), (dict(free=None), _lib.EINVAL),
    (dict(stride=7), _lib.ESTRIDE), (dict(slots=20), _lib.EALIGN),
])
def test_map_step_refusals(kw, code):
    assert _lib.lib().b2g_kv_map_step(*{**MAP, **kw}.values()) == code


WRITE = dict(k=16, v=16, kc=16, vc=16, st=_st(512, 64, 512, 64, 8192, 512, 64, 8192, 512, 64),
             slots=16, tokens=4, heads=8, dim=64, pages=4, page=16, dtype=0, status=None,
             stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), _lib.EINVAL), (dict(st=None), _lib.EINVAL), (dict(k=None), _lib.EINVAL),
    (dict(slots=None), _lib.EINVAL), (dict(heads=0), _lib.ESHAPE), (dict(tokens=-1), _lib.ESHAPE),
    (dict(page=0), _lib.ESHAPE), (dict(slots=12), _lib.EALIGN), (dict(tokens=0), _lib.OK),
])
def test_write_refusals(kw, code):
    assert _lib.lib().b2g_kv_write(*{**WRITE, **kw}.values()) == code


PREFILL = dict(q=16, k=16, v=16, o=16, st=_st(512, 128, 256, 128, 256, 128, 512, 128), cu=16,
               prompts=2, tokens=8, hq=4, hk=2, dim=128, dtype=1, scale=1.0, lse=None, ws=256,
               wsb=1 << 30, status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.EINVAL), (dict(cu=None), _lib.EINVAL), (dict(st=None), _lib.EINVAL),
    (dict(dtype=2), _lib.EINVAL), (dict(scale=0.0), _lib.EINVAL),
    (dict(scale=float("nan")), _lib.EINVAL), (dict(scale=float("inf")), _lib.EINVAL),
    (dict(dim=96), _lib.ESHAPE), (dict(hk=3), _lib.ESHAPE), (dict(hq=0), _lib.ESHAPE),
    (dict(tokens=-1), _lib.ESHAPE), (dict(prompts=-1), _lib.ESHAPE), (dict(k=24), _lib.EALIGN),
    (dict(st=_st(512, 128, 256, 0, 256, 128, 512, 128)), _lib.ESTRIDE),
    (dict(st=_st(512, 128, 256, 132, 256, 128, 512, 128)), _lib.EALIGN),
    (dict(tokens=0), _lib.OK), (dict(prompts=0), _lib.OK),
])
def test_prefill_refusals(kw, code):
    assert _lib.lib().b2g_attention_prefill(*{**PREFILL, **kw}.values()) == code


TREE = dict(q=16, kc=16, vc=16, o=16,
            st=_st(512, 128, 4096, 256, 128, 4096, 256, 128, 512, 128), tables=16, stride=8,
            max_pages=8, lens=16, cu=16, mask=None, words=0, requests=2, tokens=8, hq=4, hk=2,
            dim=128, pages=4, page=16, dtype=1, scale=1.0, lse=None, ws=256, wsb=1 << 30,
            status=None, stream=None)


@pytest.mark.parametrize("kw,code", [
    (dict(kc=None), _lib.EINVAL), (dict(tables=None), _lib.EINVAL), (dict(lens=None), _lib.EINVAL),
    (dict(cu=None), _lib.EINVAL), (dict(mask=16), _lib.EINVAL), (dict(dtype=3), _lib.EINVAL),
    (dict(page=24), _lib.ESHAPE), (dict(page=4), _lib.ESHAPE), (dict(page=192), _lib.ESHAPE),
    (dict(dim=32), _lib.ESHAPE), (dict(hk=3), _lib.ESHAPE), (dict(pages=0), _lib.ESHAPE),
    (dict(stride=7), _lib.ESTRIDE), (dict(kc=24), _lib.EALIGN), (dict(mask=20, words=1), _lib.EALIGN),
    (dict(st=_st(512, 128, 4096, 256, 0, 4096, 256, 128, 512, 128)), _lib.ESTRIDE),
    (dict(st=_st(512, 128, 4096, 260, 128, 4096, 256, 128, 512, 128)), _lib.EALIGN),
    (dict(tokens=0), _lib.OK), (dict(requests=0), _lib.OK),
])
def test_tree_refusals(kw, code):
    assert _lib.lib().b2g_attention_tree(*{**TREE, **kw}.values()) == code


def test_status_texts():
    for code in (_lib.STATUS_PAGE_TABLE, _lib.STATUS_SLOT, _lib.STATUS_TOKENS):
        assert "unknown" not in _lib.strerror(code) and "CUDA" not in _lib.strerror(code)


def test_python_wants_cuda_tensors():
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros((1, 1, 64), dtype=torch.float16)
    c = torch.zeros((1, 16, 1, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        kvcache.map_step(i, i, i, i.view(1, 1), i, i, page_size=16, num_tokens=1)
    with pytest.raises(ValueError, match="CUDA"):
        kvcache.write_kv(x, x, c, c, i.long())
    with pytest.raises(ValueError, match="CUDA"):
        attention.attention_prefill(x, x, x, torch.tensor([0, 1], dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        attention.attention_tree(x, c, c, i.view(1, 1), i, torch.tensor([0, 1], dtype=torch.int32))

"""Refusals of the paged-cache and serving-attention entry points, before anything touches a GPU,
and the integer restatement of the page bookkeeping on a case worked out by hand."""

from __future__ import annotations

import ctypes

import numpy as np
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


@pytest.mark.parametrize("unit", [2.0 ** -8, 2.0 ** -11])
def test_oracle_attention(unit):
    """The float64 restatement against a softmax written out, rows that see nothing, masked NaN,
    and its tolerances against attention whose weights and output are rounded by ``unit``."""
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((5, 16)), rng.standard_normal((9, 16)), rng.standard_normal((9, 16))
    seen = serving.tree_seen(9, 5, [1, 0b11, 0b101, 0b1011, 0b10011])
    assert seen[:, :4].all() and seen[3, 4:].tolist() == [True, True, False, True, False]
    assert (serving.tree_seen(9, 9) == serving.causal(9)).all()
    seen[2] = False
    k[8], v[8] = np.nan, np.inf  # the last draft is seen by the last row alone
    o, lse, tol, lse_tol = serving.attend(q, k, v, seen, 0.25, unit)
    assert (o[2] == 0).all() and lse[2] == -np.inf and not np.isfinite(o[4]).any()
    for i in (0, 1, 3):
        idx = np.flatnonzero(seen[i])
        w = np.exp(0.25 * (k[idx] @ q[i]))
        np.testing.assert_allclose(o[i], (w[:, None] * v[idx]).sum(0) / w.sum(), rtol=1e-12)
        np.testing.assert_allclose(lse[i], np.log(w.sum()), rtol=1e-12)
        w /= w.max()
        rounded = w * (1 + unit * rng.choice([-1, 1], w.shape))
        off = (rounded[:, None] * v[idx]).sum(0) / w.sum() * (1 + unit * rng.choice([-1, 1], 16))
        assert (np.abs(off - o[i]) <= tol[i] * (1 + unit)).all() and lse_tol[i] > 0


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

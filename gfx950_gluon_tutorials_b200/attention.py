"""Drop-in for the reference's FMHA forward launcher.

Mirrors ``run_gluon_attention(q, k, v, o, metadata, scale_on_q=True)`` of
kernels/attention/fmha_v4.py:761-790 and the host helpers it reads from
kernels/attention/common.py (``MetaData`` :58-69, ``get_shape_from_layout``
:72-81, ``get_strides_from_layout`` :84-92, ``input_helper`` :95-112,
``compute_flops`` :177-184): same argument meaning, the same ``bhsd`` / ``bshd``
layouts, output written into ``o`` on the current stream. The work runs in
the sm_100a flash-attention kernel of libb2g.so (``b2g_attention_fwd``).

Differences from the reference launcher, all widenings: Q and K lengths may
differ and need not be multiples of 64 (rows and keys past the ends are
masked), and the softmax log-sum-exp can be returned. ``scale_on_q`` is
accepted for signature compatibility; the kernel always applies the scale to
the fp32 scores, which is the more accurate of the reference's two choices.
Causal masking is not supported there, as in the reference tutorial kernel.

``attention_prefill`` (causal, packed prompts) and ``attention_tree`` (drafted or
single tokens over a paged cache, see ``kvcache``) are a serving step's
attention; the reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .kvcache import _int_vector, check_caches
from .ops import _require_cuda, _stream_handle, status_tensor, workspace

_DT = {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}
HEAD_DIMS = (64, 128)
BLOCK_M, BLOCK_N = 128, 128   # query rows per CTA, keys per tile
KERNEL_NAME = "fmha_fwd_kernel"
_I64x8, _I64x10 = ctypes.c_int64 * 8, ctypes.c_int64 * 10


class MetaData:
    """Host-side descriptor of one attention problem (fields of common.py:58-69)."""

    causal = False
    layout = None
    max_seqlens_q = 0
    max_seqlens_k = 0

    def __init__(self, sm_scale: float = 1.0):
        self.sm_scale = sm_scale


def get_shape_from_layout(q: torch.Tensor, k: torch.Tensor, metadata: MetaData):
    """(batch, heads_q, heads_k, head_dim) of a ``bhsd`` or ``bshd`` problem."""
    if metadata.layout == "bhsd":
        return q.shape[0], q.shape[1], k.shape[1], q.shape[3]
    if metadata.layout == "bshd":
        return q.shape[0], q.shape[2], k.shape[2], q.shape[3]
    raise ValueError(f"Unsupported layout: {metadata.layout}")


def _axis_order(layout: str) -> tuple[int, int, int, int]:
    if layout == "bhsd":
        return (0, 1, 2, 3)
    if layout == "bshd":
        return (0, 2, 1, 3)
    raise ValueError(f"Unsupported layout: {layout}")


def get_strides_from_layout(q, k, v, o, metadata: MetaData):
    """Each tensor's strides in (batch, head, sequence, dim) order."""
    order = _axis_order(metadata.layout)
    return tuple(tuple(t.stride(i) for i in order) for t in (q, k, v, o))


def input_helper(Z, HQ, HK, N_CTX_Q, N_CTX_K, D_HEAD, dtype, layout, requires_grad=False,
                 device="cuda"):
    """Seeded standard-normal q, k, v in ``layout`` and their MetaData, the
    problem recipe of the reference's bench (seed 20, sm_scale = D ** -0.5)."""
    if layout not in ("bhsd", "bshd"):
        raise ValueError(f"Unsupported layout: {layout}")
    torch.manual_seed(20)

    def rand(heads, n_ctx):
        shape = (Z, heads, n_ctx, D_HEAD) if layout == "bhsd" else (Z, n_ctx, heads, D_HEAD)
        return torch.randn(shape, dtype=dtype, device=device, requires_grad=requires_grad)

    q = rand(HQ, N_CTX_Q)
    k = rand(HK, N_CTX_K)
    v = rand(HK, N_CTX_K)
    md = MetaData(sm_scale=D_HEAD ** -0.5)
    md.max_seqlens_q = N_CTX_Q
    md.max_seqlens_k = N_CTX_K
    md.layout = layout
    return q, k, v, md


def compute_flops(B, HQ, M, N, D, causal=False):
    """FLOPs of the forward pass: the QK^T and PV products, 2*B*HQ*M*N*D each."""
    if causal:
        valid = ((N ** 2 + N) / 2) if M > N else (M * N - ((M ** 2 - M) / 2))
        per_matmul = 2.0 * B * HQ * valid * D
    else:
        per_matmul = 2.0 * B * HQ * M * N * D
    return 2 * per_matmul


def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  o: torch.Tensor | None = None, *, sm_scale: float | None = None,
                  layout: str = "bhsd", lse: torch.Tensor | None = None) -> torch.Tensor:
    """O = softmax(Q K^T * sm_scale) V per (batch, query head), GQA by head groups.

    ``q`` is (B, HQ, Sq, D) for ``bhsd`` or (B, Sq, HQ, D) for ``bshd``; ``k`` and
    ``v`` likewise with HK heads and Sk keys; ``o`` takes q's shape and dtype.
    ``lse``, if given, is a float32 (B, HQ, Sq) tensor that receives the
    natural-log log-sum-exp of each row's scaled scores. Asynchronous on the
    current stream; kernel timeouts are reported by ``ops.check_status``.
    """
    dev = _require_cuda(q, k, v, o, lse)
    order = _axis_order(layout)
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share one dtype, float16 or bfloat16")
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be 4-D")
    B, HQ, Sq, D = (q.shape[i] for i in order)
    Bk, HK, Sk, Dk = (k.shape[i] for i in order)
    if (Bk, Dk) != (B, D) or tuple(v.shape) != tuple(k.shape):
        raise ValueError(f"k/v shapes {tuple(k.shape)}/{tuple(v.shape)} do not match q {tuple(q.shape)}")
    if o is None:
        o = torch.empty_like(q)
    if tuple(o.shape) != tuple(q.shape) or o.dtype != q.dtype:
        raise ValueError("o must have q's shape and dtype")
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != (B, HQ, Sq)
                            or not lse.is_contiguous()):
        raise ValueError(f"lse must be a contiguous float32 ({B}, {HQ}, {Sq}) tensor")
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)

    ts = []
    for t in (q, k, v):
        if t.stride(order[3]) != 1 or any((t.stride(i) * 2) % 16 for i in order[:3]) \
                or t.data_ptr() % 16:
            t = t.contiguous()
        ts.append(t)
    o_run = o
    if o.stride(order[3]) != 1 or any((o.stride(i) * 2) % 16 for i in order[:3]) \
            or o.data_ptr() % 16:
        o_run = torch.empty_like(q, memory_format=torch.contiguous_format)
    strides = (ctypes.c_int64 * 16)(*[t.stride(i) for t in (*ts, o_run) for i in order])
    st = status_tensor(dev)
    rc = _lib.lib().b2g_attention_fwd(
        ts[0].data_ptr(), ts[1].data_ptr(), ts[2].data_ptr(), o_run.data_ptr(), strides,
        B, HQ, HK, Sq, Sk, D, _DT[q.dtype], float(sm_scale),
        None if lse is None else lse.data_ptr(), st.data_ptr(), _stream_handle(dev))
    _lib.check(rc)
    if o_run is not o:
        o.copy_(o_run)
    return o


def run_gluon_attention(q, k, v, o, metadata: MetaData, scale_on_q: bool = True):
    """Runs the forward pass on ``q, k, v`` and writes the result into ``o``.

    Same contract as the reference launcher: non-causal only, ``metadata.layout``
    ``bhsd`` or ``bshd``, ``metadata.sm_scale`` the softmax scale. Head dims 64
    and 128 (the reference takes any power of two).
    """
    assert not metadata.causal, "the FMHA forward kernel supports non-causal attention only"
    batch, nheads_q, nheads_k, head_size = get_shape_from_layout(q, k, metadata)
    assert head_size & (head_size - 1) == 0, "head dim must be a power of two"
    assert head_size in HEAD_DIMS, f"head dim must be one of {HEAD_DIMS}"
    assert nheads_q % nheads_k == 0, "query heads must be a multiple of key/value heads"
    del scale_on_q  # the scale is always applied to the fp32 scores
    return attention_fwd(q, k, v, o, sm_scale=metadata.sm_scale, layout=metadata.layout)


def _packed(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """A (tokens, heads, dim) tensor and its token and head strides, copied unless it can be
    read where it lies: unit dim stride, 16-byte aligned base and rows."""
    s0, s1, s2 = t.stride()
    if s2 == 1 and s0 > 0 < s1 and not ((s0 | s1) & 7 or t.data_ptr() & 15):
        return t, s0, s1
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride(0), t.stride(1)


def _check_packed(q: torch.Tensor, hk: int, o, lse) -> tuple:
    """(tokens, HQ, D, the code of q's dtype) of valid packed queries with their o and lse."""
    dtype = _DT.get(q.dtype)
    if dtype is None:
        raise ValueError("q must be float16 or bfloat16")
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("q must be (tokens, heads, head_dim)")
    tokens, hq, dim = shape
    if dim not in HEAD_DIMS:
        raise ValueError(f"head dim must be one of {HEAD_DIMS}, got {dim}")
    if hk < 1 or hq % hk:
        raise ValueError("query heads must be a multiple of key/value heads")
    if o is not None and (o.shape != shape or o.dtype is not q.dtype):
        raise ValueError("o must have q's shape and dtype")
    if lse is not None and (lse.dtype is not torch.float32 or lse.shape != (hq, tokens)
                            or not lse.is_contiguous()):
        raise ValueError(f"lse must be a contiguous float32 ({hq}, {tokens}) tensor")
    return tokens, hq, dim, dtype


def _run_packed(call, nbytes, dev, q, o, lse, args) -> torch.Tensor:
    """``call(*args(out, its strides, lse), workspace, its size, status, stream)`` into o (a new
    tensor if it is None) with the stream's workspace as it is; asks ``nbytes`` how large that has
    to be only when the call finds it too small."""
    if o is None:
        out = o = q.new_empty(q.shape)
        o_token, o_head, _ = o.stride()
    else:
        out, o_token, o_head = _packed(o)  # a copy keeps the rows past the last sequence
    args = args(out.data_ptr(), o_token, o_head, None if lse is None else lse.data_ptr())
    ws, status, stream = workspace(0, dev), status_tensor(dev).data_ptr(), _stream_handle(dev)
    rc = call(*args, ws.data_ptr(), ws.numel(), status, stream)
    if rc == _lib.EWORKSPACE:
        ws = workspace(nbytes(), dev)
        rc = call(*args, ws.data_ptr(), ws.numel(), status, stream)
    if rc != _lib.OK:
        _lib.check(rc, call.__name__)
    if out is not o:
        o.copy_(out)
    return o


def attention_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                      o: torch.Tensor | None = None, *, sm_scale: float | None = None,
                      lse: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention over packed prompts: token i of a prompt sees its tokens 0 .. i.

    ``q`` (tokens, HQ, D), ``k`` and ``v`` (tokens, HK, D) hold the prompts back to
    back, prompt b in rows cu_seqlens[b] .. cu_seqlens[b + 1] (int32, on the GPU;
    empty prompts are fine). Rows past the last prompt are not written. ``lse``, if
    given, is a float32 (HQ, tokens) tensor that receives the natural-log
    log-sum-exp of each row's scaled scores. D is 64 or 128. Asynchronous on the
    current stream; offsets that decrease or pass ``tokens`` and kernel timeouts
    are reported by ``ops.check_status``.
    """
    dev = _require_cuda(q, k, v, cu_seqlens, o, lse)
    kv_shape = k.shape
    if len(kv_shape) != 3 or kv_shape != v.shape:
        raise ValueError("q, k and v must be (tokens, heads, head_dim), k and v of one shape")
    tokens, hq, dim, dtype = _check_packed(q, kv_shape[1], o, lse)
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise ValueError("q, k and v must share one dtype, float16 or bfloat16")
    if kv_shape[0] != tokens or kv_shape[2] != dim:
        raise ValueError(f"k/v shape {tuple(kv_shape)} does not match q {tuple(q.shape)}")
    cu_seqlens = _int_vector(cu_seqlens, None, torch.int32, "cu_seqlens")
    prompts = cu_seqlens.shape[0] - 1
    if prompts < 0:
        raise ValueError("cu_seqlens needs at least one entry")
    if tokens == 0 or prompts == 0:
        return torch.empty_like(q) if o is None else o
    (q, q_token, q_head), (k, k_token, k_head), (v, v_token, v_head) = _packed(q), _packed(k), _packed(v)
    handle = _lib.lib()
    return _run_packed(
        handle.b2g_attention_prefill,
        lambda: handle.b2g_attention_prefill_workspace_bytes(prompts, tokens, hq), dev, q, o, lse,
        lambda out, o_token, o_head, lse_ptr: (
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out,
            _I64x8(q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head),
            cu_seqlens.data_ptr(), prompts, tokens, hq, kv_shape[1], dim, dtype,
            dim ** -0.5 if sm_scale is None else sm_scale, lse_ptr))


def attention_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_tables: torch.Tensor, seq_lens: torch.Tensor, cu_seqlens: torch.Tensor,
                   tree_mask: torch.Tensor | None = None, o: torch.Tensor | None = None, *,
                   sm_scale: float | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's new tokens over a paged cache that already holds them.

    ``q`` (tokens, HQ, D) packs the requests' new tokens, request r's in rows
    cu_seqlens[r] .. cu_seqlens[r + 1]; they are the last tokens of the seq_lens[r]
    that the cache holds for it in the pages of row r of ``block_tables``. A new
    token sees every older token of its request, and of the new ones those whose
    bit is set in its row of ``tree_mask`` (int64 (tokens, words); bit j % 64 of
    word j // 64 is the request's new token j, and a token sets its own bit too).
    Without a mask the new tokens are a chain, each seeing the ones before it: one
    token per request is plain decoding, many are a chunk of a prompt. A token that
    sees nothing gets zeros and an lse of -inf.

    The caches are (pages, page_size, HK, D) with unit dim stride, 16-byte aligned
    rows and a page_size of 8, 16, 32, 64 or a multiple of 128; they are never
    copied. ``block_tables`` is int32 (requests, max_pages), ``seq_lens`` and
    ``cu_seqlens`` int32, ``lse`` as for ``attention_prefill``. Asynchronous on the
    current stream; bad pages and lengths are reported by ``ops.check_status``.
    """
    dev = _require_cuda(q, k_cache, v_cache, block_tables, seq_lens, cu_seqlens, tree_mask, o, lse)
    check_caches(k_cache, v_cache, q.dtype)
    pages, page, hk, cache_dim = k_cache.shape
    tokens, hq, dim, dtype = _check_packed(q, hk, o, lse)
    if cache_dim != dim:
        raise ValueError(f"q has heads of {dim}, the cache of {cache_dim}")
    if block_tables.dtype is not torch.int32 or len(block_tables.shape) != 2:
        raise ValueError("block_tables must be a 2-D int32 tensor")
    requests, max_pages = block_tables.shape
    table_stride, column_stride = block_tables.stride()
    if max_pages > 1 and column_stride != 1:
        block_tables = block_tables.contiguous()
        table_stride = max_pages
    seq_lens = _int_vector(seq_lens, requests, torch.int32, "seq_lens")
    cu_seqlens = _int_vector(cu_seqlens, requests + 1, torch.int32, "cu_seqlens")
    mask_ptr, words = None, 0
    if tree_mask is not None:
        if tree_mask.dtype is not torch.int64 or tree_mask.dim() != 2 or tree_mask.shape[0] != tokens:
            raise ValueError(f"tree_mask must be an int64 ({tokens}, words) tensor")
        words = tree_mask.shape[1]
        if words < 1:
            raise ValueError("tree_mask needs at least one word per token")
        tree_mask = tree_mask.contiguous()
        mask_ptr = tree_mask.data_ptr()
    if tokens == 0 or requests == 0:
        return torch.empty_like(q) if o is None else o
    q, q_token, q_head = _packed(q)
    handle = _lib.lib()
    return _run_packed(
        handle.b2g_attention_tree,
        lambda: handle.b2g_attention_tree_workspace_bytes(requests, tokens, hq, hk, dim), dev, q, o,
        lse,
        lambda out, o_token, o_head, lse_ptr: (
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out,
            _I64x10(q_token, q_head, *k_cache.stride()[:3], *v_cache.stride()[:3], o_token, o_head),
            block_tables.data_ptr(), table_stride, max_pages, seq_lens.data_ptr(),
            cu_seqlens.data_ptr(), mask_ptr, words, requests, tokens, hq, hk, dim, pages, page,
            dtype, dim ** -0.5 if sm_scale is None else sm_scale, lse_ptr))


def main(argv=None) -> None:
    """Times the forward pass on one problem, with the reference FMHA bench's
    flags and defaults (kernels/attention/bench.py:103-155): seeded inputs,
    CUDA-event timing on the current stream, TFLOPS from compute_flops."""
    import argparse

    ap = argparse.ArgumentParser(description="B200 FMHA forward timing")
    ap.add_argument("--dtype", choices=["fp16", "bf16"], default="bf16")
    ap.add_argument("--layout", choices=["bhsd", "bshd"], default="bhsd")
    ap.add_argument("--batch", type=int, default=1)
    ap.add_argument("--hq", type=int, default=64)
    ap.add_argument("--hk", type=int, default=64)
    ap.add_argument("--d", type=int, default=128)
    ap.add_argument("--seqlen", type=int, default=8192)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--iters", type=int, default=10)
    args = ap.parse_args(argv)
    from .ops import check_status

    dt = torch.bfloat16 if args.dtype == "bf16" else torch.float16
    q, k, v, md = input_helper(args.batch, args.hq, args.hk, args.seqlen, args.seqlen, args.d, dt,
                               args.layout)
    o = torch.empty_like(q)
    for _ in range(args.warmup):
        run_gluon_attention(q, k, v, o, md)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(args.iters):
        run_gluon_attention(q, k, v, o, md)
    end.record()
    torch.cuda.synchronize()
    check_status()
    ms = start.elapsed_time(end) / max(args.iters, 1)
    flops = compute_flops(args.batch, args.hq, args.seqlen, args.seqlen, args.d, False)
    print(f"FMHA B={args.batch} HQ={args.hq} HK={args.hk} S={args.seqlen} D={args.d} "
          f"{args.dtype} {args.layout}: {ms * 1e3:.1f} us, {flops / ms / 1e9:.1f} TFLOPS")


if __name__ == "__main__":
    main()

"""Attention of single tokens over a paged cache and of packed prompts.

No counterpart in the reference, whose layer bench calls torch's attention
(fast_route/benchmarks/fused_route/transformerLayer_bench.py:66-95).
"""
from __future__ import annotations

import struct

import torch

from .. import _native as N

_FLOATS = (torch.float16, torch.bfloat16)
_PACKED = struct.Struct("@26qd")  # fr_attention_args
_PAGED = struct.Struct("@30qd")  # fr_paged_args


def _workspace(buf: torch.Tensor | None, nbytes: int, device) -> torch.Tensor | None:
    if buf is None:
        return torch.empty((nbytes,), dtype=torch.uint8, device=device) if nbytes else None
    assert buf.dtype == torch.uint8 and buf.is_contiguous() and buf.device == device, \
        "workspace_buf must be a contiguous uint8 tensor on the operands' device"
    return buf


def _check_rows(x: torch.Tensor, what: str) -> None:
    assert x.dim() == 3 and x.dtype in _FLOATS, "%s must be [tokens, heads, head size] in float16 or bfloat16" % what
    assert x.stride(2) == 1, "%s must be contiguous along a head" % what


def _output(out: torch.Tensor | None, q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must be like q"
    assert out.stride(2) == 1, "out must be contiguous along a head"
    return out


def attention_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor | None = None,
                     causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None,
                     workspace_buf: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed sequences: q [tokens, heads, head size], k and v [keys, kv heads, head size] in f16/bf16 (parts of a joint
    projection's result, for instance), sequence b's rows from cu_seqlens_q[b] to cu_seqlens_q[b + 1] and its keys from cu_seqlens_k[b] on
    (int32 [sequences + 1]; without cu_seqlens_k the same).  heads a multiple of kv heads, consecutive ones share a key head; `scale`
    (head size ** -0.5) on the products.  causal: the last row of a sequence sees all its keys, each row before it one less - a chunk of a
    prompt brings the keys in front of it along.  Scores, softmax and sums in fp32, the softmax's terms rounded to q's type for the product with the values.

    A row that sees no key is zeros.  What a row does not see does not reach it, NaN included.  Rows behind the last sequence: zeros, in an `out` given
    left as they were (out may be q).  Head size a multiple of 8 up to 256; strides (but 1 along a head) multiples of 8 elements, 16-byte aligned.  Forward only."""
    cu_k = cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k
    N.require_cuda(q, k, v, cu_seqlens_q, cu_k)
    _check_rows(q, "q")
    rows, heads, dim = q.shape
    dev, dtype = q.device, q.dtype
    assert k.dim() == 3 and k.shape == v.shape and k.shape[2] == dim, "k and v must be [keys, kv heads, head size]"
    assert k.dtype == dtype and v.dtype == dtype, "q, k and v differ in type"
    (q_row, q_head, _), (k_row, k_head, k1), (v_row, v_head, v1) = q.stride(), k.stride(), v.stride()
    assert k1 == 1 and v1 == 1, "k and v must be contiguous along a head"
    for cu in (cu_seqlens_q, cu_k):
        assert cu.dim() == 1 and cu.dtype == torch.int32 and cu.is_contiguous() and cu.shape[0] >= 1, "cu_seqlens must be contiguous int32 [sequences + 1]"
    assert cu_k.shape == cu_seqlens_q.shape, "cu_seqlens_q and cu_seqlens_k differ in length"
    assert k.device == dev and v.device == dev and cu_seqlens_q.device == dev and cu_k.device == dev, "operands on different devices"
    fill = out is None
    out = _output(out, q)
    B, (keys, kv_heads, _), lib = cu_seqlens_q.shape[0] - 1, k.shape, N.lib()
    need = lib.fr_attention_workspace_bytes(B, rows, keys, heads, kv_heads, dim)
    assert need >= 0, lib.fr_last_error_string().decode()
    ws = _workspace(workspace_buf, need, dev)
    args = _PACKED.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(),
                        0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), B, rows, keys, heads, kv_heads, dim,
                        q_row, q_head, k_row, k_head, v_row, v_head, out.stride(0), out.stride(1), N.dtype_code(dtype), int(bool(causal)), int(fill), 0,
                        float(dim ** -0.5 if scale is None else scale))
    with N.on(dev):
        N.check(lib.fr_attention(args, N.stream_ptr(dev)))
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    scale: float | None = None, out: torch.Tensor | None = None, workspace_buf: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one token per sequence: q [B, heads, head size] over the first seq_lens[b] (int32 [B]) keys of its sequence, held in pages
    k_cache, v_cache [pages, page size, kv heads, head size] (as rotary_to_cache fills them) in the order of block_table
    (int32 [B, pages of a sequence at most]).  f16/bf16; heads a multiple of kv heads, consecutive ones share a key head; `scale`
    (head size ** -0.5) on the products.  Scores, softmax and sums in fp32, the softmax's terms rounded to q's type for the product with the values.

    A row without keys is zeros; a length behind the table's end is the table's end; keys in a page outside the cache take no part; what lies
    behind a length, NaN included, is not read.  Head size a multiple of 8 up to 256; strides (but 1 along a head) multiples of 8 elements, 16-byte aligned;
    page sizes of multiples of 16 are the fast case."""
    N.require_cuda(q, k_cache, v_cache, block_table, seq_lens)
    _check_rows(q, "q")
    B, heads, dim = q.shape
    dev, dtype = q.device, q.dtype
    assert k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] == dim, \
        "k_cache and v_cache must be [pages, page size, kv heads, head size]"
    pages, page_size, kv_heads, _ = k_cache.shape
    (kp, ks, kh, k1), (vp, vs, vh, v1) = k_cache.stride(), v_cache.stride()
    assert k_cache.dtype == dtype and v_cache.dtype == dtype, "q and the cache differ in type"
    assert k1 == 1 and v1 == 1, "the cache must be contiguous along a head"
    assert block_table.dim() == 2 and block_table.shape[0] == B and block_table.dtype == torch.int32, "block_table must be int32 [B, pages]"
    assert block_table.shape[1] <= 1 or block_table.stride(1) == 1, "block_table must be contiguous along its rows"
    assert seq_lens.shape == (B,) and seq_lens.dtype == torch.int32 and seq_lens.is_contiguous(), "seq_lens must be contiguous int32 [B]"
    assert k_cache.device == dev and v_cache.device == dev and block_table.device == dev and seq_lens.device == dev, "operands on different devices"
    out = _output(out, q)
    if B == 0:
        return out
    table_pages, lib = block_table.shape[1], N.lib()
    need = lib.fr_paged_attention_workspace_bytes(B, heads, kv_heads, dim, table_pages * page_size)
    assert need >= 0, lib.fr_last_error_string().decode()
    ws = _workspace(workspace_buf, need, dev)
    args = _PAGED.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
                       0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), B, heads, kv_heads, dim, pages, page_size, table_pages,
                       block_table.stride(0), q.stride(0), q.stride(1), out.stride(0), out.stride(1), kp, ks, kh, vp, vs, vh,
                       N.dtype_code(dtype), 0, 0, 0, float(dim ** -0.5 if scale is None else scale))
    with N.on(dev):
        N.check(lib.fr_paged_attention(args, N.stream_ptr(dev)))
    return out

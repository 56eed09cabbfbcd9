"""Attention of single tokens over a paged cache and of packed prompts.

No counterpart in the reference, whose layer bench calls torch's attention
(fast_route/benchmarks/fused_route/transformerLayer_bench.py:66-95).
"""
from __future__ import annotations

import struct

import torch

from .. import _native as N

_FLOATS = (torch.float16, torch.bfloat16)
_PACKED = struct.Struct("@26qdq")  # fr_attention_args
_PAGED = struct.Struct("@30qdq")  # fr_paged_args


def _workspace(buf: torch.Tensor | None, nbytes: int, device) -> torch.Tensor | None:
    if buf is None:
        return torch.empty((nbytes,), dtype=torch.uint8, device=device) if nbytes else None
    assert buf.dtype == torch.uint8 and buf.is_contiguous() and buf.device == device, \
        "workspace_buf must be a contiguous uint8 tensor on the operands' device"
    return buf


def _rows(x: torch.Tensor, what: str):
    """Shape and strides of [tokens, heads, head size]."""
    shape, strides = x.shape, x.stride()
    assert len(shape) == 3 and strides[2] == 1, "%s must be [tokens, heads, head size], contiguous along a head" % what
    return shape, strides


def _output(out: torch.Tensor | None, q: torch.Tensor):
    """The result and its strides: a new tensor or the caller's."""
    if out is None:
        out = q.new_empty(q.shape)
        return out, out.stride()
    assert out.shape == q.shape and out.dtype == q.dtype and out.device == q.device, "out must be like q"
    strides = out.stride()
    assert strides[2] == 1, "out must be contiguous along a head"
    return out, strides


def attention_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor | None = None,
                     causal: bool = True, scale: float | None = None, out: torch.Tensor | None = None,
                     workspace_buf: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed sequences: q [tokens, heads, head size], k and v [keys, kv heads, head size] in f16/bf16 (parts of a joint
    projection's result, for instance), sequence b's rows from cu_seqlens_q[b] to cu_seqlens_q[b + 1] and its keys from cu_seqlens_k[b] on
    (int32 [sequences + 1]; without cu_seqlens_k the same).  heads a multiple of kv heads, consecutive ones share a key head; `scale`
    (head size ** -0.5) on the products.  causal: the last row of a sequence sees all its keys, each row before it one less - a chunk of a
    prompt brings the keys in front of it along.  Scores, softmax and sums in fp32, the softmax's terms rounded to q's type for the product with the values.

    A row that sees no key is zeros.  What a row does not see does not reach it, NaN included.  Rows of no sequence, in front of the first or behind the last: zeros, in an
    `out` given left as they were (out may be q, of the same strides, and lies beside q, k and v otherwise).  Head size a multiple of 8 up to 256; strides (but 1 along a head) multiples of 8 elements, 16-byte aligned.  Forward only."""
    cu_k = cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k
    dev, dtype = N.device_of(q, k, v, cu_seqlens_q, cu_k), q.dtype
    ((rows, heads, dim), q_strides), (k_shape, k_strides), (v_shape, v_strides) = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    assert dtype in _FLOATS, "q must be float16 or bfloat16"
    assert k_shape == v_shape and k_shape[2] == dim, "k and v must be [keys, kv heads, head size]"
    assert k.dtype == dtype and v.dtype == dtype, "q, k and v differ in type"
    for cu in (cu_seqlens_q, cu_k):
        assert cu.dim() == 1 and cu.dtype == torch.int32 and cu.is_contiguous(), "cu_seqlens must be contiguous int32 [sequences + 1]"
    B, keys, kv_heads, lib = cu_seqlens_q.shape[0] - 1, k_shape[0], k_shape[1], N.lib()
    assert B >= 0 and cu_k.shape[0] == B + 1, "cu_seqlens_q and cu_seqlens_k differ in length, or are empty"
    fill = out is None
    out, out_strides = _output(out, q)
    need = lib.fr_attention_workspace_bytes(B, rows, keys, heads, kv_heads, dim)
    assert need >= 0, lib.fr_last_error_string().decode()
    ws_ptr = ws_bytes = 0
    if need or workspace_buf is not None:
        ws = _workspace(workspace_buf, need, q.device)
        ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
    args = _PACKED.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(), ws_ptr, ws_bytes,
                        B, rows, keys, heads, kv_heads, dim, q_strides[0], q_strides[1], k_strides[0], k_strides[1], v_strides[0], v_strides[1],
                        out_strides[0], out_strides[1], N.dtype_code(dtype), bool(causal), fill, 0, float(dim ** -0.5 if scale is None else scale), 0)
    N.run(dev, lib.fr_attention, args)
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    scale: float | None = None, out: torch.Tensor | None = None, workspace_buf: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one token per sequence: q [B, heads, head size] over the first seq_lens[b] (int32 [B]) keys of its sequence, held in pages
    k_cache, v_cache [pages, page size, kv heads, head size] (as rotary_to_cache fills them) in the order of block_table
    (int32 [B, pages of a sequence at most]).  f16/bf16; heads a multiple of kv heads, consecutive ones share a key head; `scale`
    (head size ** -0.5) on the products.  Scores, softmax and sums in fp32, the softmax's terms rounded to q's type for the product with the values.

    `out` may be q, of the same strides, and lies beside q and the cache otherwise.  A row without keys is zeros; a length behind the table's end is the table's end; keys in a page outside the cache take no part; what lies
    behind a length, NaN included, is not read.  Head size a multiple of 8 up to 256; strides (but 1 along a head) multiples of 8 elements, 16-byte aligned;
    page sizes of multiples of 16 are the fast case."""
    dev, dtype = N.device_of(q, k_cache, v_cache, block_table, seq_lens), q.dtype
    ((B, heads, dim), q_strides), shape, kc, vc = _rows(q, "q"), k_cache.shape, k_cache.stride(), v_cache.stride()
    assert dtype in _FLOATS, "q must be float16 or bfloat16"
    assert len(shape) == 4 and v_cache.shape == shape and shape[3] == dim, "k_cache and v_cache must be [pages, page size, kv heads, head size]"
    assert k_cache.dtype == dtype and v_cache.dtype == dtype, "q and the cache differ in type"
    assert kc[3] == 1 and vc[3] == 1, "the cache must be contiguous along a head"
    table, table_strides = block_table.shape, block_table.stride()
    assert len(table) == 2 and table[0] == B and block_table.dtype == torch.int32, "block_table must be int32 [B, pages]"
    assert table[1] <= 1 or table_strides[1] == 1, "block_table must be contiguous along its rows"
    assert seq_lens.shape == (B,) and seq_lens.dtype == torch.int32 and seq_lens.is_contiguous(), "seq_lens must be contiguous int32 [B]"
    out, out_strides = _output(out, q)
    if B == 0:
        return out
    (pages, page_size, kv_heads, _), lib = shape, N.lib()
    need = lib.fr_paged_attention_workspace_bytes(B, heads, kv_heads, dim, table[1] * page_size)
    assert need >= 0, lib.fr_last_error_string().decode()
    ws_ptr = ws_bytes = 0
    if need or workspace_buf is not None:
        ws = _workspace(workspace_buf, need, q.device)
        ws_ptr, ws_bytes = ws.data_ptr(), ws.numel()
    args = _PAGED.pack(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(),
                       ws_ptr, ws_bytes, B, heads, kv_heads, dim, pages, page_size, table[1], table_strides[0], q_strides[0], q_strides[1],
                       out_strides[0], out_strides[1], kc[0], kc[1], kc[2], vc[0], vc[1], vc[2], N.dtype_code(dtype), 0, 0, 0,
                       float(dim ** -0.5 if scale is None else scale), 0)
    N.run(dev, lib.fr_paged_attention, args)
    return out

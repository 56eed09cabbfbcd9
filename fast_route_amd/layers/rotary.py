"""Rotary positions of queries and keys, alone or together with the keys' and values' way into a paged cache.

No counterpart in the reference, whose layer bench has no positions
(fast_route/benchmarks/fused_route/transformerLayer_bench.py:66-95).
"""
from __future__ import annotations

import math
import struct
from typing import NamedTuple

import torch

from .. import _native as N

_FLOATS = (torch.float16, torch.bfloat16)
_INTS = (torch.int32, torch.int64)
_ARGS = struct.Struct("@37qd")  # fr_rotary_args


class Rotary(NamedTuple):
    """Frequencies as prepare_rotary lays them out: 2^-64 turn per position."""
    turns: torch.Tensor
    interleaved: bool
    factor: float


def rotary_frequencies(turned: int, base: float = 10000.0, scale: float = 1.0, original: int = 0, slow_turns: float = 1.0,
                       fast_turns: float = 4.0) -> torch.Tensor:
    """Radians per position of the pairs of `turned` dimensions, fp64 [turned / 2]: base^(-2 i / turned).

    For contexts `scale` times longer than a model was trained for: with original == 0 every frequency is divided by scale; with the
    original length, those that make up to `slow_turns` turns in it are, those that make `fast_turns` or more stay, and in between the two
    are mixed, linearly in the turns."""
    assert turned >= 0 and turned % 2 == 0, "an even number of dimensions is turned"
    assert base > 0 and scale > 0 and 0 <= slow_turns < fast_turns, "base and scale must be positive, slow_turns below fast_turns"
    i = torch.arange(turned // 2, dtype=torch.float64)
    freq = float(base) ** (-2.0 * i / max(turned, 1))
    if not original:
        return freq / scale
    keep = ((freq * original / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
    return freq * keep + freq / scale * (1.0 - keep)


def prepare_rotary(frequencies: torch.Tensor, interleaved: bool = False, factor: float = 1.0, device=None) -> Rotary:
    """The handle that rotary_embed and rotary_to_cache take, made once: frequencies in radians per position (fp64 or fp32, one per
    pair, of less than half a turn each, for instance from rotary_frequencies), pairs (2 i, 2 i + 1) if interleaved, else (i, i + n), a factor on what is turned.
    On the frequencies' device, or `device`."""
    assert frequencies.dim() == 1 and frequencies.dtype in (torch.float64, torch.float32), "frequencies must be 1-D float64 or float32"
    assert frequencies.numel() <= 256, "at most 512 dimensions are turned"
    values = frequencies.detach().double().cpu()
    assert bool((values.abs() < math.pi).all()), "a frequency is below half a turn (pi) per position"
    device = frequencies.device if device is None else torch.device(device)
    # 2^64 / (2 pi), below 2^63 in magnitude: rounded to 53 bits, like the frequencies
    turns = torch.round(values * (2.0 ** 63 / math.pi)).clamp(-2.0 ** 63 + 1024, 2.0 ** 63 - 1024).to(torch.int64)
    return Rotary(turns.to(device), bool(interleaved), float(factor))


def _check_heads(x: torch.Tensor, what: str) -> None:
    assert x.dim() == 3 and x.dtype in _FLOATS, "%s must be [tokens, heads, head size] in float16 or bfloat16" % what
    assert x.shape[2] == 1 or x.stride(2) == 1, "%s must be contiguous along a head" % what


def _check_cache(cache: torch.Tensor, like: torch.Tensor, what: str) -> None:
    assert cache.dim() == 4 and cache.dtype == like.dtype and cache.device == like.device, \
        "%s must be [pages, page size, heads, head size], in the keys' type and on their device" % what
    assert cache.shape[2:] == like.shape[1:], "%s: other heads than the keys" % what
    assert cache.shape[3] == 1 or cache.stride(3) == 1, "%s must be contiguous along a head" % what
    assert 0 not in cache.stride(), "%s: places that share memory" % what


def _call(q, k, positions, rotary: Rotary, inplace: bool, cached=None):
    N.require_cuda(q, k, positions)
    _check_heads(q, "q")
    _check_heads(k, "k")
    T, heads, dim = q.shape
    kv_heads, dev, turned = k.shape[1], q.device, 2 * rotary.turns.numel()
    assert k.shape == (T, kv_heads, dim) and k.dtype == q.dtype, "q and k differ in tokens, head size or type"
    assert turned <= dim, "more dimensions are turned than a head has"
    assert positions.shape == (T,) and positions.dtype in _INTS and positions.is_contiguous(), "positions must be contiguous int32 or int64 [tokens]"
    assert k.device == dev and positions.device == dev and rotary.turns.device == dev, "operands on different devices"
    v_ptr = kc_ptr = vc_ptr = slots_ptr = pages = slots_i64 = v_token = v_head = 0
    page_size, cache_strides = 1, (0, 0, 0, 0, 0, 0)
    if cached is not None:
        v, k_cache, v_cache, slots = cached
        _check_heads(v, "v")
        assert v.shape == k.shape and v.dtype == k.dtype and v.device == dev, "v must be like k"
        _check_cache(k_cache, k, "k_cache")
        _check_cache(v_cache, k, "v_cache")
        assert k_cache.shape == v_cache.shape, "k_cache and v_cache differ in shape"
        assert slots.shape == (T,) and slots.dtype in _INTS and slots.is_contiguous() and slots.device == dev, \
            "slots must be contiguous int32 or int64 [tokens]"
        v_ptr, kc_ptr, vc_ptr, slots_ptr = v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr()
        (v_token, v_head, _), (pages, page_size, _, _) = v.stride(), k_cache.shape
        cache_strides = k_cache.stride()[:3] + v_cache.stride()[:3]
        slots_i64 = int(slots.dtype == torch.int64)
    if inplace:
        assert 0 not in q.stride() and 0 not in k.stride(), "inplace: rows that share memory"
        q_out, k_out = q, k
    else:
        q_out, k_out = (torch.empty((T, h, dim), dtype=q.dtype, device=dev) for h in (heads, kv_heads))
    if T == 0:
        return q_out, k_out
    args = _ARGS.pack(q.data_ptr(), k.data_ptr(), v_ptr, q_out.data_ptr(), k_out.data_ptr(), kc_ptr, vc_ptr, positions.data_ptr(), slots_ptr,
                      rotary.turns.data_ptr(), T, heads, kv_heads, dim, turned, pages, page_size, *q.stride()[:2], *k.stride()[:2], v_token, v_head,
                      *q_out.stride()[:2], *k_out.stride()[:2], *cache_strides, N.dtype_code(q.dtype), int(rotary.interleaved),
                      int(positions.dtype == torch.int64), slots_i64, rotary.factor)
    with N.on(dev):
        N.check(N.lib().fr_rotary(args, N.stream_ptr(dev)))
    return q_out, k_out


def rotary_embed(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary, inplace: bool = False):
    """Queries q [tokens, heads, head size] and keys k [tokens, kv heads, head size] (f16/bf16, any strides but 1 along a head, such as
    parts of a joint projection's result) turned by their positions (int32/int64 [tokens], any value): new tensors, or with inplace q and k themselves.
    Computed in fp32, angles in 64-bit integers, rounded once."""
    return _call(q, k, positions, rotary, inplace)


def rotary_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, rotary: Rotary, k_cache: torch.Tensor,
                    v_cache: torch.Tensor, slots: torch.Tensor, inplace: bool = False):
    """rotary_embed, and in the same pass the turned keys and the values v [tokens, kv heads, head size] into a paged cache k_cache, v_cache
    [pages, page size, kv heads, head size] (any strides but 1 along a head): token t's into place slots[t] % page size of page
    slots[t] // page size.  A token whose slot (int32/int64) is negative or behind the last page is not kept.  Slots are of one token each: one that two
    tokens name ends up with pieces of either.  The cache holds what paged_attention reads."""
    return _call(q, k, positions, rotary, inplace, (v, k_cache, v_cache, slots))

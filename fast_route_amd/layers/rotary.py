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


def _pi(bits: int) -> int:
    """pi * 2^bits, to a few units: 16 arctan(1/5) - 4 arctan(1/239) (Machin 1706) in whole numbers."""
    def arctan(x):
        term, total, n = (1 << bits + 16) // x, 0, 1
        while term:
            total += term // n if n % 4 == 1 else -(term // n)
            term, n = term // (x * x), n + 2
        return total
    return (16 * arctan(5) - 4 * arctan(239)) >> 16


_TURN_BITS = 160
_TURN = (1 << _TURN_BITS + 199) // _pi(200)  # 2^_TURN_BITS / (2 pi)


def _turn(frequency: float) -> int:
    """frequency / (2 pi) * 2^64, rounded: in whole numbers, since 64 bits are more than a product of floats has."""
    digits, exponent = math.frexp(frequency)
    behind = _TURN_BITS + 53 - 64 - exponent  # binary places of the product below 2^-64 turn
    return (int(digits * 2.0 ** 53) * _TURN + (1 << behind - 1)) >> behind


def prepare_rotary(frequencies: torch.Tensor, interleaved: bool = False, factor: float = 1.0, device=None) -> Rotary:
    """The handle that rotary_embed and rotary_to_cache take, made once: frequencies in radians per position (fp64 or fp32, one per
    pair, of less than half a turn each, for instance from rotary_frequencies), pairs (2 i, 2 i + 1) if interleaved, else (i, i + n), a factor on what is turned.
    On the frequencies' device, or `device`."""
    assert frequencies.dim() == 1 and frequencies.dtype in (torch.float64, torch.float32), "frequencies must be 1-D float64 or float32"
    assert frequencies.numel() <= 256, "at most 512 dimensions are turned"
    values = frequencies.detach().double().cpu()
    assert bool((values.abs() < math.pi).all()), "a frequency is below half a turn (pi) per position"
    device = frequencies.device if device is None else torch.device(device)
    turns = torch.tensor([_turn(f) for f in values.tolist()], dtype=torch.int64)  # below half a turn, 2^63, in magnitude
    return Rotary(turns.to(device), bool(interleaved), float(factor))


def _heads(x: torch.Tensor, what: str):
    """Shape and strides of [tokens, heads, head size]."""
    shape, strides = x.shape, x.stride()
    assert len(shape) == 3 and (strides[2] == 1 or shape[2] == 1), "%s must be [tokens, heads, head size], contiguous along a head" % what
    return shape, strides


def _cache(cache: torch.Tensor, dtype: torch.dtype, heads: int, dim: int, what: str):
    shape, strides = cache.shape, cache.stride()
    assert len(shape) == 4 and cache.dtype == dtype, "%s must be [pages, page size, heads, head size] in the keys' type" % what
    assert shape[2] == heads and shape[3] == dim, "%s: other heads than the keys" % what
    assert strides[3] == 1 or dim == 1, "%s must be contiguous along a head" % what
    return shape, strides


def _call(q, k, positions, rotary: Rotary, inplace: bool, cached=None):
    turns, interleaved, factor = rotary
    assert turns.dtype == torch.int64 and turns.dim() == 1 and turns.is_contiguous(), "rotary: turns must be as prepare_rotary lays them out, contiguous int64"
    ((T, heads, dim), q_strides), (k_shape, k_strides), dtype = _heads(q, "q"), _heads(k, "k"), q.dtype
    kv_heads, turned, at_type = k_shape[1], 2 * turns.shape[0], positions.dtype
    assert dtype in _FLOATS, "q must be float16 or bfloat16"
    assert k_shape[0] == T and k_shape[2] == dim and k.dtype == dtype, "q and k differ in tokens, head size or type"
    assert turned <= dim, "more dimensions are turned than a head has"
    assert positions.shape == (T,) and at_type in _INTS and positions.is_contiguous(), "positions must be contiguous int32 or int64 [tokens]"
    if cached is None:
        dev = N.device_of(q, k, positions, turns)
        v_ptr = kc_ptr = vc_ptr = slots_ptr = pages = slots_i64 = v_token = v_head = 0
        page_size, cache_strides = 1, (0, 0, 0, 0, 0, 0)
    else:
        v, k_cache, v_cache, slots = cached
        dev, slot_type = N.device_of(q, k, positions, turns, v, k_cache, v_cache, slots), slots.dtype
        v_shape, (v_token, v_head, _) = _heads(v, "v")
        assert v_shape == k_shape and v.dtype == dtype, "v must be like k"
        (shape, kc), (v_cache_shape, vc) = _cache(k_cache, dtype, kv_heads, dim, "k_cache"), _cache(v_cache, dtype, kv_heads, dim, "v_cache")
        assert shape == v_cache_shape, "k_cache and v_cache differ in shape"
        assert slots.shape == (T,) and slot_type in _INTS and slots.is_contiguous(), "slots must be contiguous int32 or int64 [tokens]"
        v_ptr, kc_ptr, vc_ptr, slots_ptr = v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr()
        pages, page_size, cache_strides, slots_i64 = shape[0], shape[1], kc[:3] + vc[:3], int(slot_type == torch.int64)
    if inplace:
        q_out, k_out, out_strides = q, k, q_strides[:2] + k_strides[:2]
    else:
        q_out, k_out = q.new_empty((T, heads, dim)), k.new_empty(k_shape)
        out_strides = (heads * dim, dim, kv_heads * dim, dim)
    if T == 0:
        return q_out, k_out
    args = _ARGS.pack(q.data_ptr(), k.data_ptr(), v_ptr, q_out.data_ptr(), k_out.data_ptr(), kc_ptr, vc_ptr, positions.data_ptr(), slots_ptr,
                      turns.data_ptr(), T, heads, kv_heads, dim, turned, pages, page_size, q_strides[0], q_strides[1], k_strides[0], k_strides[1],
                      v_token, v_head, *out_strides, *cache_strides, N.dtype_code(dtype), interleaved, at_type == torch.int64, slots_i64, factor)
    N.run(dev, N.lib().fr_rotary, args)
    return q_out, k_out


def rotary_embed(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary, inplace: bool = False):
    """Queries q [tokens, heads, head size] and keys k [tokens, kv heads, head size] (f16/bf16, any strides but 1 along a head, such as
    parts of a joint projection's result) turned by their positions (int32/int64 [tokens], any value): new tensors, or with inplace q and k themselves,
    which share no memory then (parts of the same rows do not).  Computed in fp32, rounded once; angles in 64-bit integers, off by |position| * 2^-65 turn at
    most and by 2^-25 turn."""
    return _call(q, k, positions, rotary, inplace)


def rotary_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, rotary: Rotary, k_cache: torch.Tensor,
                    v_cache: torch.Tensor, slots: torch.Tensor, inplace: bool = False):
    """rotary_embed, and in the same pass the turned keys and the values v [tokens, kv heads, head size] into a paged cache k_cache, v_cache
    [pages, page size, kv heads, head size] (any strides but 1 along a head): token t's into place slots[t] % page size of page
    slots[t] // page size.  A token whose slot (int32/int64) is negative or behind the last page is not kept.  Slots are of one token each: one that two
    tokens name ends up with pieces of either.  The cache holds what paged_attention reads; k_cache and v_cache share no memory with each other nor with q, k
    and v; inplace, q and k share none with each other nor with v."""
    return _call(q, k, positions, rotary, inplace, (v, k_cache, v_cache, slots))

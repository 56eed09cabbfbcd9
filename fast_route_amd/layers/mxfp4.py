"""MXFP4 operators: rows in 4-bit floats with a power-of-two scale per 32 elements (OCP microscaling), their matrix
product, and the fused MoE layer on expert weights in this format.

No counterpart in the reference.  Weights are quantised once (or come from a checkpoint in the format) and laid out
once; activations are quantised on the way, the activated rows of the layer from their fp32 values; products
accumulate in fp32 and results are rounded once, to the activations' type.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch

from .. import _native as N

BLOCK = 32  # elements that share a scale
_FLOATS = (torch.float16, torch.bfloat16)


class MXFP4Weight(NamedTuple):
    """A weight matrix [N, K] as prepare_linear_mxfp4 lays it out."""
    data: torch.Tensor
    N: int
    K: int


class MXFP4Experts(NamedTuple):
    """Expert weights w1 [E, 2F, H] and w2 [E, H, F] as prepare_weights_mxfp4 lays them out."""
    w1: torch.Tensor
    w2: torch.Tensor
    E: int
    H: int
    F: int


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """The device of a call's tensors as the current one, where it is another."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _check_rows(x: torch.Tensor, what: str):
    """Rows, row length and row stride of a 2-D tensor that the kernels read row by row."""
    N.require_cuda(x)
    assert x.dim() == 2 and x.dtype in _FLOATS, "%s must be a 2-D float16 or bfloat16 tensor" % what
    rows, K = x.shape
    ld, step = x.stride()
    assert K > 0 and K % BLOCK == 0, "%s: row length must be a positive multiple of 32" % what
    assert step == 1, "%s must be contiguous along its rows" % what
    if rows <= 1:
        return rows, K, K
    assert ld >= K and ld % 8 == 0, "%s: rows must not overlap and lie a multiple of 8 elements apart" % what
    return rows, K, ld


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, what: str) -> None:
    N.require_cuda(codes, scales)
    assert codes.device == scales.device, "%s: codes and scales on different devices" % what
    assert codes.dtype == torch.uint8 and scales.dtype == torch.uint8, "%s: codes and scales must be uint8" % what
    assert codes.is_contiguous() and scales.is_contiguous(), "%s: codes and scales must be contiguous" % what
    *lead, half = codes.shape
    assert lead and half > 0 and half % (BLOCK // 2) == 0 and scales.shape == (*lead, half // (BLOCK // 2)), \
        "%s: codes must be [.., K / 2] and scales [.., K / 32]" % what


def quantize_rows_mxfp4(x: torch.Tensor):
    """Rows of a [rows, K] f16/bf16 tensor in MXFP4: (codes uint8 [rows, K / 2], scales uint8 [rows, K / 32]).

    A block of 32 elements has the scale 2^(b - 127), b = floor(log2(max|x|)) - 2 + 127 (127 where all are zero);
    elements are rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 units, ties to the even code, and what exceeds 6
    becomes 6.  The even element of a pair is in the low half of its byte.  A block that holds an infinity or a NaN has b = 255
    and zero codes: all of it reads back as NaN."""
    rows, K, ld = _check_rows(x, "x")
    dev = x.device
    codes = torch.empty((rows, K // 2), dtype=torch.uint8, device=dev)
    scales = codes.new_empty((rows, K // BLOCK))
    with _on(dev):
        N.check(N.lib().fr_quant_mxfp4_rows(x.data_ptr(), N.dtype_code(x.dtype), rows, K, ld, codes.data_ptr(), scales.data_ptr(),
                                            N.stream_ptr(dev)))
    return codes, scales


def dequantize_rows_mxfp4(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [.., K] that codes [.., K / 2] and scales [.., K / 32] stand for, in f16 (what exceeds its range becomes
    infinite), bf16 or f32."""
    _check_codes(codes, scales, "dequantize_rows_mxfp4")
    assert dtype in _FLOATS or dtype == torch.float32, "dtype must be float16, bfloat16 or float32"
    K = codes.shape[-1] * 2
    out = torch.empty(codes.shape[:-1] + (K,), dtype=dtype, device=codes.device)
    with _on(codes.device):
        N.check(N.lib().fr_dequant_mxfp4_rows(codes.data_ptr(), scales.data_ptr(), out.numel() // K, K, N.dtype_code(dtype),
                                              out.data_ptr(), N.stream_ptr(codes.device)))
    return out


def _tiled(codes: torch.Tensor, scales: torch.Tensor, gate_up: bool) -> torch.Tensor:
    matrices, rows, K = codes.shape[0], codes.shape[1], codes.shape[2] * 2
    nbytes = N.lib().fr_mxfp4_tiled_bytes(matrices, rows, K)
    assert nbytes >= 0, "weights of %d x %d x %d are too large" % (matrices, rows, K)
    out = torch.empty((nbytes,), dtype=torch.uint8, device=codes.device)
    with _on(codes.device):
        N.check(N.lib().fr_mxfp4_tile_weights(codes.data_ptr(), scales.data_ptr(), matrices, rows, K, int(gate_up), out.data_ptr(),
                                              N.stream_ptr(codes.device)))
    return out


def _check_tiled(data: torch.Tensor, matrices: int, rows: int, K: int, device: torch.device, what: str) -> None:
    """A prepared weight's data are what its sizes say: the kernels read all of it by these sizes."""
    assert data.device == device, "%s on another device than the rows" % what
    units = matrices * ((rows + 31) // 32) * ((K + 255) // 256)  # of 32 rows x 256 elements
    assert data.dtype == torch.uint8 and data.is_contiguous() and data.numel() == units * 4352, \
        "%s: not the data of a prepared weight of these sizes" % what


def prepare_linear_mxfp4(codes: torch.Tensor, scales: torch.Tensor) -> MXFP4Weight:
    """One-off layout of a weight matrix [N, K] in MXFP4 (codes uint8 [N, K / 2], scales uint8 [N, K / 32], as
    quantize_rows_mxfp4 returns them) for linear_mxfp4.  The originals may be freed afterwards."""
    _check_codes(codes, scales, "prepare_linear_mxfp4")
    assert codes.dim() == 2 and codes.shape[0] >= 1, "prepare_linear_mxfp4: codes must be [N, K / 2]"
    return MXFP4Weight(_tiled(codes[None], scales[None], False), codes.shape[0], codes.shape[1] * 2)


def linear_mxfp4(x: torch.Tensor, weight: MXFP4Weight, workspace_buf: torch.Tensor | None = None) -> torch.Tensor:
    """x [M, K] (f16/bf16, rows a multiple of 8 elements apart) times the transpose of a prepared weight matrix [N, K]: x is
    quantised to MXFP4 row by row, the product accumulates in fp32, the result [M, N] has x's type.  Any N; for more than 128 rows a
    multiple of 8 is the fast case."""
    M, K, ld = _check_rows(x, "x")
    dev = x.device
    assert K == weight.K, "Incompatible dimensions"
    _check_tiled(weight.data, 1, weight.N, K, dev, "weight")
    out = torch.empty((M, weight.N), dtype=x.dtype, device=dev)
    if M == 0:
        return out
    need = N.lib().fr_linear_mxfp4_workspace_bytes(M, weight.N, K)
    assert need >= 0, "linear_mxfp4: %d rows of %d elements are too large" % (M, K)
    ws = _workspace(workspace_buf, need, dev)
    with _on(dev):
        N.check(N.lib().fr_linear_mxfp4(x.data_ptr(), N.dtype_code(x.dtype), M, K, ld, weight.data.data_ptr(), weight.N, out.data_ptr(),
                                        0 if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), N.stream_ptr(dev)))
    return out


def _workspace(buf: torch.Tensor | None, nbytes: int, device) -> torch.Tensor | None:
    if buf is None:
        return torch.empty((nbytes,), dtype=torch.uint8, device=device) if nbytes else None
    assert buf.dtype == torch.uint8 and buf.is_contiguous() and buf.device == device, \
        "workspace_buf must be a contiguous uint8 tensor on the operands' device"
    return buf


def prepare_weights_mxfp4(w1: torch.Tensor, w1_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor) -> MXFP4Experts:
    """One-off layout of expert weights in MXFP4 for fused_moe_mxfp4: w1 [E, 2F, H] (gate rows first) and w2 [E, H, F] as codes
    (uint8, [.., K / 2]) and scales (uint8, [.., K / 32]), for instance from quantize_rows_mxfp4 on w1.view(E * 2F, H) and
    w2.view(E * H, F).  H and F are multiples of 32.  The originals may be freed afterwards."""
    _check_codes(w1, w1_scale, "w1")
    _check_codes(w2, w2_scale, "w2")
    assert w1.device == w2.device, "w1 and w2 on different devices"
    assert w1.dim() == 3 and w2.dim() == 3, "w1 must be [E, 2F, H / 2] and w2 [E, H, F / 2]"
    E, F2, H = w1.shape[0], w1.shape[1], w1.shape[2] * 2
    assert E >= 1 and F2 % 64 == 0 and w2.shape == (E, H, F2 // 4), "w1 must be [E, 2F, H / 2] and w2 [E, H, F / 2]"
    return MXFP4Experts(_tiled(w1, w1_scale, True), _tiled(w2, w2_scale, False), E, H, F2 // 2)


def fused_moe_mxfp4(hidden_states: torch.Tensor, weights: MXFP4Experts, gating_output: torch.Tensor, topk: int,
                    renormalize: bool = True, inplace: bool = False, workspace_buf: torch.Tensor | None = None):
    """Whole layer with expert weights in MXFP4: f16/bf16 hidden_states [M, H], router logits [M, E], weights from
    prepare_weights_mxfp4.  Gating and routing as in fused_moe; hidden states and activated rows are quantised to MXFP4 on the
    way (the latter from their fp32 values), everything is summed in fp32 and rounded once."""
    N.require_cuda(hidden_states, gating_output)
    assert hidden_states.dim() == 2 and hidden_states.shape[1] == weights.H, "Incompatible dimensions"
    assert hidden_states.is_contiguous(), "Hidden_states must be contiguous"
    assert hidden_states.dtype in _FLOATS, "hidden_states must be float16 or bfloat16"
    M, H = hidden_states.shape
    assert gating_output.shape == (M, weights.E), "Number of tokens mismatch"
    assert gating_output.is_contiguous(), "gating_output must be contiguous"
    dev = hidden_states.device
    assert gating_output.device == dev, "operands on different devices"
    _check_tiled(weights.w1, weights.E, 2 * weights.F, H, dev, "w1")
    _check_tiled(weights.w2, weights.E, H, weights.F, dev, "w2")
    topk = int(topk)
    need = N.lib().fr_moe_mxfp4_workspace_bytes(M, H, weights.F, weights.E, topk)
    assert need >= 0, N.lib().fr_last_error_string().decode()
    out = hidden_states if inplace else torch.empty_like(hidden_states)
    if M == 0:
        return out
    ws = _workspace(workspace_buf, need, dev)
    with _on(dev):
        N.check(N.lib().fr_fused_moe_mxfp4(hidden_states.data_ptr(), N.dtype_code(hidden_states.dtype), weights.w1.data_ptr(),
                                           weights.w2.data_ptr(), gating_output.data_ptr(), N.dtype_code(gating_output.dtype), M, H,
                                           weights.F, weights.E, topk, int(bool(renormalize)), out.data_ptr(), ws.data_ptr(),
                                           ws.numel(), N.stream_ptr(dev)))
    return out

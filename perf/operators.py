"""Performance cases of the MXFP4 operators: rows held as 4-bit floats with a power-of-two scale for each 32 elements.

Kinds
  quant   quantize_rows_mxfp4, then dequantize_rows_mxfp4: rows of activations or weights to codes and back to values
  linear  linear_mxfp4: activations times a weight matrix in MXFP4, the activations quantised on the way
  layer   fused_moe_mxfp4: the whole mixture-of-experts layer from hidden states and router logits, expert weights in
          MXFP4, hidden states and activated rows quantised on the way; a few tokens up to a long prefill

Format (OCP microscaling, MXFP4): an element is e2m1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives; nearest value,
ties to the even code, magnitudes above 6 become 6), two to a byte, the even element in the low half; 32 consecutive
elements share a scale 2^(b - 127) with b = floor(log2(largest magnitude)) - 2 + 127, held in a byte (a block of zeros: b = 127).
"""
from __future__ import annotations

import math

import torch

own = False

SHAPES = {
    # 8 wide experts, near-uniform load
    "mixtral": dict(H=4096, F=14336, E=8, topk=2, zipf=False),
    "mixtral22b": dict(H=6144, F=16384, E=8, topk=2, zipf=False),
    # 64 narrow experts, Zipf-skewed load
    "fine": dict(H=2048, F=1408, E=64, topk=6, zipf=True),
    # one small layer: everything but the weight stream is launches and latency
    "small": dict(H=1024, F=3584, E=8, topk=2, zipf=False),
    # the layer of the reference's benchmark protocol
    "protocol": dict(H=4096, F=8192, E=16, topk=2, zipf=False),
    # widths that are multiples of 32 and of nothing more
    "ragged": dict(H=1056, F=1120, E=12, topk=3, zipf=True),
}


def _quant(rows, width, dtype, name=None):
    return _named({"kind": "quant", "rows": int(rows), "width": int(width), "dtype": dtype}, name)


def _linear(tokens, outs, width, dtype, name=None):
    return _named({"kind": "linear", "tokens": int(tokens), "outs": int(outs), "width": int(width), "dtype": dtype}, name)


def _layer(shape, tokens, dtype, name=None):
    return _named({"kind": "layer", "shape": shape, "tokens": int(tokens), "dtype": dtype}, name)


def _named(case, name):
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the hidden states of a few decoding sequences
        _quant(4, 4096, "bf16", "quant_rows_4"),
        # one expert's gate and up weights, as a checkpoint holds them
        _quant(28672, 4096, "fp16", "quant_weights_28672"),
        # the attention's fused query/key/value projection: one decoding sequence, a chunk, a prefill
        _linear(1, 12288, 4096, "bf16", "linear_decode_1"),
        _linear(509, 12288, 4096, "fp16", "linear_chunk_509"),
        _linear(8192, 12288, 4096, "bf16", "linear_prefill_8192"),
        # one sequence decoding: two experts' weights streamed once, launch latency next to it
        _layer("mixtral", 1, "bf16", "mixtral_decode_1"),
        # continuous batching at decode: all experts hit by a few tokens each
        _layer("mixtral", 24, "bf16", "mixtral_decode_24"),
        # a small chunk of prefill, or a large decode batch
        _layer("mixtral", 1031, "bf16", "mixtral_chunk_1031"),
        # a long prefill
        _layer("mixtral", 16384, "bf16", "mixtral_prefill_16384"),
        # many narrow experts: a decode batch and a prefill
        _layer("fine", 32, "bf16", "fine_decode_32"),
        _layer("fine", 8192, "fp16", "fine_prefill_8192"),
        # a handful of sequences on a small layer: launches
        _layer("small", 5, "fp16", "small_decode_5"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    pick, dtype = rng.random(), rng.choice(("bf16", "bf16", "fp16"))
    if pick < 0.15:
        width = 32 * _log_uniform(rng, 1, 512)
        return _quant(_log_uniform(rng, 1, min(65536, 28672 * 4096 // width)), width, dtype)
    if pick < 0.40:
        return _linear(_log_uniform(rng, 1, 8192), _log_uniform(rng, 64, 12288), 32 * _log_uniform(rng, 8, 128), dtype)
    shape, most = rng.choice((("mixtral", 16384), ("mixtral", 16384), ("mixtral22b", 4096), ("fine", 16384), ("fine", 16384),
                              ("small", 16384), ("protocol", 8192), ("ragged", 8192)))
    return _layer(shape, _log_uniform(rng, 1, most), dtype)


def _type(case):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]


# ---- the format, in elementary operations -----------------------------------------------------------------

def _quantised(x):
    """Codes and scale bytes of rows x [rows, K] in 32 bits."""
    blocks = x.reshape(x.shape[0], -1, 32)
    amax = blocks.abs().amax(dim=2)
    exponent = (torch.frexp(amax).exponent - 3).clamp(-127, 127)
    exponent = torch.where(amax > 0, exponent, torch.zeros_like(exponent))
    v = torch.ldexp(blocks.double(), -exponent[:, :, None]).float()  # a power of two: nothing is rounded
    a = v.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5.0).byte() + 8 * (v < 0).byte())
    code = code.reshape(x.shape[0], -1, 2)
    return code[:, :, 0] + 16 * code[:, :, 1], (exponent + 127).byte()


def _values(codes, scales):
    """What codes [rows, K / 2] and scale bytes [rows, K / 32] stand for, in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([table, -table])
    pairs = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], dim=2)
    scale = (scales.int().clamp(min=1) << 23).view(torch.float32)
    scale = torch.where(scales == 0, torch.full_like(scale, 2.0 ** -127), scale)
    return (pairs.reshape(codes.shape[0], -1, 32) * scale[:, :, None]).reshape(codes.shape[0], -1)


# ---- inputs ------------------------------------------------------------------------------------------------

def _logits(gen, M, E, zipf):
    noise = torch.randn(M, E, generator=gen, device=gen.device)
    if not zipf:
        return noise
    # log of a Zipf(1.2) law over the experts, in an order of the seed's own
    p = (torch.randperm(E, generator=gen, device=gen.device) + 1).double().pow(-1.2)
    return (torch.log(p / p.sum()).float()[None, :] + noise).contiguous()


def _weights(gen, matrices, rows, width):
    """Weights of a checkpoint in MXFP4: codes [matrices, rows, width / 2] and scale bytes [matrices, rows, width / 32]."""
    codes = torch.empty((matrices, rows, width // 2), dtype=torch.uint8, device=gen.device)
    scales = torch.empty((matrices, rows, width // 32), dtype=torch.uint8, device=gen.device)
    for m in range(matrices):
        codes[m], scales[m] = _quantised(torch.empty((rows, width), device=gen.device).normal_(0.0, 0.02, generator=gen))
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    dtype, st = _type(case), {"kind": case["kind"]}
    if case["kind"] == "quant":
        st["x"] = torch.empty((case["rows"], case["width"]), dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=gen)
        return st
    if case["kind"] == "linear":
        st["x"] = torch.empty((case["tokens"], case["width"]), dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=gen)
        codes, scales = _weights(gen, 1, case["outs"], case["width"])
        st["w"], st["ws"] = codes[0], scales[0]
        if own:  # weights laid out once, as a serving program keeps them
            from fast_route_amd import prepare_linear_mxfp4
            st["weight"] = prepare_linear_mxfp4(st["w"], st["ws"])
        return st
    s = SHAPES[case["shape"]]
    st["x"] = torch.empty((case["tokens"], s["H"]), dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=gen)
    st["logits"] = _logits(gen, case["tokens"], s["E"], s["zipf"])
    st["topk"] = s["topk"]
    st["w1"], st["w1s"] = _weights(gen, s["E"], 2 * s["F"], s["H"])
    st["w2"], st["w2s"] = _weights(gen, s["E"], s["H"], s["F"])
    if own:
        from fast_route_amd import prepare_weights_mxfp4
        st["weights"] = prepare_weights_mxfp4(st["w1"], st["w1s"], st["w2"], st["w2s"])
    return st


# ---- one pass ----------------------------------------------------------------------------------------------

def run(st):
    x, kind = st["x"], st["kind"]
    if own:
        from fast_route_amd import dequantize_rows_mxfp4, fused_moe_mxfp4, linear_mxfp4, quantize_rows_mxfp4
        if kind == "quant":
            return dequantize_rows_mxfp4(*quantize_rows_mxfp4(x), dtype=x.dtype)
        if kind == "linear":
            return linear_mxfp4(x, st["weight"])
        return fused_moe_mxfp4(x, st["weights"], st["logits"], st["topk"], renormalize=True)
    xv = _values(*_quantised(x.float()))
    if kind == "quant":
        return xv.to(x.dtype)
    if kind == "linear":
        return (xv @ _values(st["w"], st["ws"]).t()).to(x.dtype)
    top, ids = torch.sort(st["logits"], dim=1, descending=True, stable=True)
    top, ids = top[:, : st["topk"]], ids[:, : st["topk"]]
    weights = torch.exp(top - top[:, :1])
    weights = weights / weights.sum(dim=1, keepdim=True)
    out = torch.zeros_like(xv)
    for e in range(st["w1"].shape[0]):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        gate, up = (xv[token] @ _values(st["w1"][e], st["w1s"][e]).t()).chunk(2, dim=1)
        act = _values(*_quantised(gate / (1.0 + torch.exp(-gate)) * up))
        rows = act @ _values(st["w2"][e], st["w2s"][e]).t()
        out.index_add_(0, token, rows * weights[token, slot][:, None])
    return out.to(x.dtype)


# ---- from the definition, in 64 bits -----------------------------------------------------------------------

def _held(x):
    """Rows x [rows, K] as MXFP4 holds them, in 64 bits."""
    x = x.double()
    blocks = x.view(x.shape[0], x.shape[1] // 32, 32)
    top = blocks.abs().amax(dim=2, keepdim=True)
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -900))) - 2).clamp(min=2.0 ** -127)
    # the logarithm of a value just below a power of two may come out as the power's
    unit = torch.where(top < 4 * unit, (unit / 2).clamp(min=2.0 ** -127), unit)
    unit = torch.where(top >= 8 * unit, unit * 2, unit)
    v = blocks / unit
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return ((torch.round(v / step) * step).clamp(-6, 6) * unit).reshape(x.shape)


def _held_weights(codes, scales):
    """Codes [rows, K / 2] and scale bytes [rows, K / 32] in 64 bits, from sign, exponent and mantissa."""
    nibble = torch.stack([codes % 16, codes // 16], dim=2).reshape(codes.shape[0], -1, 32).long()
    sign, exponent, mantissa = 1 - 2 * (nibble // 8), nibble // 2 % 4, nibble % 2
    value = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * 2.0 ** (exponent - 1).double())
    return (sign * value * 2.0 ** (scales.double() - 127)[:, :, None]).reshape(codes.shape[0], -1)


def exact(case, seed):
    st = prepare(case, seed)
    x = _held(st["x"])
    if case["kind"] == "quant":
        return x
    if case["kind"] == "linear":
        return x @ _held_weights(st["w"], st["ws"]).t()
    chosen, ids = torch.sort(st["logits"].double(), dim=1, descending=True, stable=True)
    share = torch.softmax(chosen[:, : st["topk"]], dim=1)
    ids = ids[:, : st["topk"]]
    out = torch.zeros_like(x)
    for e in range(st["w1"].shape[0]):
        mine = ids == e
        token = mine.any(dim=1).nonzero()[:, 0]
        if token.numel() == 0:
            continue
        both = x[token] @ _held_weights(st["w1"][e], st["w1s"][e]).t()
        gate, up = both[:, : both.shape[1] // 2], both[:, both.shape[1] // 2:]
        act = _held(gate * torch.sigmoid(gate) * up)
        out[token] += (act @ _held_weights(st["w2"][e], st["w2s"][e]).t()) * (share * mine).sum(dim=1)[token][:, None]
    return out


def _active_experts(M, E, topk, zipf):
    """Experts that a batch of M tokens hits, from one sample of the case's logits."""
    logits = _logits(torch.Generator(device="cpu").manual_seed(1), min(M, 4096), E, zipf)
    return int(torch.unique(torch.topk(logits, topk, dim=1).indices).numel())


def work(case):
    held = 0.5 + 1 / 32  # bytes of an element in MXFP4
    if case["kind"] == "quant":
        # values in, codes and scales out; these in again, values out
        n = case["rows"] * case["width"]
        return {"bytes": n * (2 + held + held + 2), "flops": 4 * n}
    if case["kind"] == "linear":
        M, N, K = case["tokens"], case["outs"], case["width"]
        return {"bytes": N * K * held + 2 * M * (K + N), "flops": 2 * M * N * K}
    s = SHAPES[case["shape"]]
    M, H, F, E, topk = case["tokens"], s["H"], s["F"], s["E"], s["topk"]
    # weights of the experts hit, tokens and router logits in, rows out
    nbytes = _active_experts(M, E, topk, s["zipf"]) * 3 * H * F * held + 2 * M * H * 2 + 4 * M * E
    return {"bytes": nbytes, "flops": 6 * M * topk * H * F}

"""GPU parity of the MXFP4 operators with the format's definition in 64 bits (oracle/mxfp4_oracle.py)."""
import numpy as np
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _say(msg):
    print("[case] " + msg, flush=True)


def _same_codes(codes, scales, x):
    """Codes and scales of rows x are the definition's; the sign of a zero is not significant."""
    rc, rs = oracle.mxfp4_quant_rows(x)
    codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
    assert codes.shape == rc.shape and scales.shape == rs.shape
    assert np.array_equal(scales, rs), "scales differ"
    for got, ref in ((codes & 15, rc & 15), (codes >> 4, rc >> 4)):
        zero = (ref & 7) == 0
        assert np.array_equal(got[~zero], ref[~zero]) and ((got[zero] & 7) == 0).all(), "codes differ"


def _rows(rows, K, dtype, seed, std=1.0):
    return (torch.randn(rows, K, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (37, 1024), (5, 5024), (130, 4096), (1031, 160), (2, 32 * 1001)])
def test_quantisation_is_the_definition(native, rows, K, dtype):
    from fast_route_amd import dequantize_rows_mxfp4, quantize_rows_mxfp4
    _say(f"quant {rows}x{K} {dtype}")
    x = _rows(rows, K, dtype, rows + K)
    if rows > 2:
        x[1].zero_()
        x[2, :32] *= 2.0 ** -10
    codes, scales = quantize_rows_mxfp4(x.cuda())
    _same_codes(codes, scales, x)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        ref = torch.from_numpy(oracle.mxfp4_held(x))
        got = dequantize_rows_mxfp4(codes, scales, dtype=out).cpu()
        assert got.dtype == out and torch.equal(got.double(), ref.to(out).double())


def test_every_pattern_of_a_bf16_and_an_fp16(native):
    """All 65536 patterns, each once as the largest of its block and once among larger ones."""
    from fast_route_amd import quantize_rows_mxfp4
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    for dtype in TYPES:
        v = bits.view(dtype)
        alone = torch.zeros(1 << 16, 32, dtype=dtype)
        alone[:, 7] = v
        _same_codes(*quantize_rows_mxfp4(alone.cuda()), alone)
        together = v.view(-1, 32)
        _same_codes(*quantize_rows_mxfp4(together.cuda()), together)
        spread = v.view(32, -1).t().contiguous()  # a block spans the exponents
        _same_codes(*quantize_rows_mxfp4(spread.cuda()), spread)


def test_borders_between_levels(native):
    from fast_route_amd import quantize_rows_mxfp4
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875])
    row = torch.cat([base, base * (1 + 2.0 ** -7), base * (1 - 2.0 ** -7), torch.tensor([4.0, 0.0])])
    for shift in (-30, 0, 40):
        x = torch.stack([row, -row]) * 2.0 ** shift
        x = x.bfloat16()
        _same_codes(*quantize_rows_mxfp4(x.cuda()), x)


def test_rows_apart_and_empty(native):
    from fast_route_amd import dequantize_rows_mxfp4, quantize_rows_mxfp4
    wide = _rows(33, 512, torch.bfloat16, 5).cuda()
    part = wide[:, 64:64 + 96]
    codes, scales = quantize_rows_mxfp4(part)
    _same_codes(codes, scales, part.cpu())
    one = wide[3:4, :32].t().contiguous().t()  # one row: its stride says nothing
    _same_codes(*quantize_rows_mxfp4(one), one.cpu())
    codes, scales = quantize_rows_mxfp4(wide[:0])
    assert codes.shape == (0, 256) and scales.shape == (0, 16)
    assert dequantize_rows_mxfp4(codes, scales).shape == (0, 512)
    back = dequantize_rows_mxfp4(*quantize_rows_mxfp4(wide)).view(3, 11, 512)
    c, s = quantize_rows_mxfp4(wide)
    assert torch.equal(dequantize_rows_mxfp4(c.view(3, 11, 256), s.view(3, 11, 16)), back)


def test_values_of_all_codes_and_scales(native):
    """256 scale bytes x 16 codes to every type: subnormal and overflowing values, NaN for scale 255."""
    from fast_route_amd import dequantize_rows_mxfp4
    codes = (torch.arange(16, dtype=torch.uint8) * 17).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(256, 1)
    ref = torch.from_numpy(oracle.mxfp4_values(codes.numpy(), scales.numpy()))
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = dequantize_rows_mxfp4(codes.cuda(), scales.cuda(), dtype=dtype).cpu()
        want = ref.to(torch.float32).to(dtype)  # the values are exact in 32 bits but for overflow
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0, 1e30, -1e30), want.nan_to_num(0.0, 1e30, -1e30))


def _weight(N_, K, seed, std=0.05):
    return oracle.mxfp4_quant_rows(_rows(N_, K, torch.float32, seed, std))


def _sum_error(terms, K):
    """What 32-bit sums of K products may be off by: at most one rounding or truncation (2^-23) per 16 products."""
    return max(1.0, K / 16) * 2.0 ** -23 * terms


LINEAR = [(1, 1, 32), (1, 64, 256), (3, 33, 96), (32, 512, 512), (33, 300, 1024), (65, 257, 544), (130, 1000, 2048), (257, 72, 288),
          (300, 4096, 512), (1000, 128, 256), (2049, 31, 64), (513, 770, 1056)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N_,K", LINEAR)
def test_linear(native, M, N_, K, dtype):
    """Rounding to the output type is half a step; the sums are of exact products."""
    from fast_route_amd import linear_mxfp4, prepare_linear_mxfp4
    _say(f"linear {M}x{N_}x{K} {dtype}")
    x, (codes, scales) = _rows(M, K, dtype, M + N_), _weight(N_, K, K)
    weight = prepare_linear_mxfp4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())
    got = linear_mxfp4(x.cuda(), weight)
    assert got.shape == (M, N_) and got.dtype == dtype and got.is_contiguous()
    xv, wv = oracle.mxfp4_held(x), oracle.mxfp4_values(codes, scales)
    ref, terms = xv @ wv.T, np.abs(xv) @ np.abs(wv).T
    off = np.abs(got.double().cpu().numpy() - ref)
    bound = torch.finfo(dtype).eps / 2 * np.abs(ref) + _sum_error(terms, K) * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).smallest_normal * 2.0 ** -8
    assert (off <= bound).all(), f"{(off / bound).max():.2f} of the bound"


def test_linear_on_rows_apart_and_none(native):
    from fast_route_amd import linear_mxfp4, prepare_linear_mxfp4
    codes, scales = _weight(200, 96, 8)
    weight = prepare_linear_mxfp4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())
    wide = _rows(70, 512, torch.bfloat16, 6).cuda()
    assert torch.equal(linear_mxfp4(wide[:, 32:128], weight), linear_mxfp4(wide[:, 32:128].contiguous(), weight))
    assert linear_mxfp4(wide[:0, :96], weight).shape == (0, 200)


@pytest.mark.parametrize("M", [5, 40, 300])
def test_linear_keeps_a_bad_row_to_itself(native, M):
    """A NaN or an infinity in a token row makes that row NaN and no other; a NaN scale of a weight row its column."""
    from fast_route_amd import linear_mxfp4, prepare_linear_mxfp4
    x, (codes, scales) = _rows(M, 320, torch.bfloat16, M), _weight(100, 320, 4)
    good = linear_mxfp4(x.cuda(), prepare_linear_mxfp4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()))
    x[2, 300], x[4, 0] = float("nan"), float("inf")
    scales[7, 3] = 255
    got = linear_mxfp4(x.cuda(), prepare_linear_mxfp4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()))
    bad = torch.zeros(M, 100, dtype=torch.bool, device="cuda")
    bad[2], bad[4], bad[:, 7] = True, True, True
    assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], good[~bad])


def _layer_inputs(M, H, F, E, dtype, seed, zipf=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, H, generator=g).to(dtype)
    logits = oracle.zipf_logits(M, E, seed) if zipf else torch.randn(M, E, generator=g)
    w1 = torch.randn(E * 2 * F, H, generator=g) * (1.5 / H ** 0.5)
    w2 = torch.randn(E * H, F, generator=g) * (1.0 / F ** 0.5)
    (c1, s1), (c2, s2) = oracle.mxfp4_quant_rows(w1), oracle.mxfp4_quant_rows(w2)
    return x, logits, (c1.reshape(E, 2 * F, -1), s1.reshape(E, 2 * F, -1), c2.reshape(E, H, -1), s2.reshape(E, H, -1))


def _prepared(q):
    from fast_route_amd import prepare_weights_mxfp4
    return prepare_weights_mxfp4(*(torch.from_numpy(t).cuda() for t in q))


def _check_layer(got, x, logits, q, topk, renormalize, dtype):
    """Bound: half a step of the output type, the oracle's doubt (activated rows next to a border of the quantisation), the
    down sum's 32-bit error as in test_linear, and 2^-20 for the routed weights' exponential, quotient and products."""
    ref, doubt = oracle.fused_moe_mxfp4(x, *q, logits, topk, renormalize)
    F = q[2].shape[2] * 2
    eps = torch.finfo(dtype).eps
    terms = np.abs(ref).max()  # of a sum of F products, F^(1/2) times its own size on these inputs at most
    bound = eps / 2 * np.abs(ref) + doubt * (1 + eps) + (_sum_error(terms * F ** 0.5, F) + 2.0 ** -20 * terms) + torch.finfo(dtype).smallest_normal * 2.0 ** -8
    off = np.abs(got.double().cpu().numpy() - ref)
    assert np.isfinite(ref).all() and (off <= bound).all(), f"{(off / bound).max():.2f} of the bound"
    assert doubt.mean() < 0.02 * np.abs(ref).mean()  # the bound says something


LAYERS = [  # M, H, F, E, topk, zipf
    (1, 256, 256, 8, 2, False), (1, 512, 1408, 64, 6, True), (2, 1056, 1120, 12, 3, True), (3, 64, 32, 1, 1, False), (4, 32, 64, 3, 3, False),
    (7, 1024, 512, 8, 2, False), (15, 320, 288, 16, 4, True), (16, 256, 768, 4, 1, False), (17, 512, 256, 8, 2, False),
    (24, 512, 1024, 8, 2, False), (60, 256, 512, 2, 2, False), (100, 288, 352, 5, 2, True), (130, 512, 256, 8, 2, False),
    (333, 256, 512, 8, 2, False), (700, 512, 256, 8, 2, True), (1500, 256, 320, 4, 2, False), (513, 128, 1408, 64, 6, True),
    (2100, 64, 96, 200, 8, False), (300, 96, 64, 1, 1, False), (1025, 320, 288, 3, 2, True),
    # the last and first sizes on either side of the forms for few tokens, and of 256 and 128 weight rows per workgroup
    (31, 256, 288, 16, 8, False), (32, 256, 288, 16, 8, True), (33, 256, 288, 16, 8, False), (32, 96, 160, 40, 9, False), (1, 64, 64, 256, 256, False),
    (4, 1024, 256, 8, 2, False), (5, 1024, 256, 8, 2, False), (1200, 800, 128, 64, 6, True), (2000, 2080, 64, 64, 2, False)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H,F,E,topk,zipf", LAYERS)
def test_layer(native, M, H, F, E, topk, zipf, dtype):
    from fast_route_amd import fused_moe_mxfp4
    _say(f"layer M={M} H={H} F={F} E={E} topk={topk} {dtype}")
    x, logits, q = _layer_inputs(M, H, F, E, dtype, M + H, zipf)
    weights = _prepared(q)
    for renormalize in (True, False) if M < 50 else (True,):
        got = fused_moe_mxfp4(x.cuda(), weights, logits.cuda(), topk, renormalize=renormalize)
        assert got.shape == x.shape and got.dtype == dtype
        _check_layer(got, x, logits, q, topk, renormalize, dtype)


@pytest.mark.parametrize("M", [1, 6, 40, 400])
def test_layer_is_the_same_every_time_in_place_and_in_a_given_workspace(native, M):
    from fast_route_amd import fused_moe_mxfp4
    H, F, E, k = 512, 768, 8, 2
    x, logits, q = _layer_inputs(M, H, F, E, torch.bfloat16, 9)
    weights, xg, lg = _prepared(q), x.cuda(), logits.cuda()
    first = fused_moe_mxfp4(xg, weights, lg, k)
    nbytes = native.fr_moe_mxfp4_workspace_bytes(M, H, F, E, k)
    for fill in (0x00, 0xFF, 0x5A):  # what the workspace held does not matter
        ws = torch.full((nbytes,), fill, dtype=torch.uint8, device="cuda")
        assert torch.equal(fused_moe_mxfp4(xg, weights, lg, k, workspace_buf=ws), first)
    for lt in (torch.bfloat16, torch.float16):
        rounded = lg.to(lt)
        assert torch.equal(fused_moe_mxfp4(xg, weights, rounded, k), fused_moe_mxfp4(xg, weights, rounded.float(), k))
    assert torch.equal(xg.cpu(), x)
    given = xg.clone()
    assert fused_moe_mxfp4(given, weights, lg, k, inplace=True) is given and torch.equal(given, first)


@pytest.mark.parametrize("M", [3, 20, 300])
def test_layer_with_bad_tokens(native, M):
    """A token row with a NaN comes out NaN, the others as without it; a token whose logits are all NaN has no expert
    or those that gating gives it, and nobody else's row changes."""
    from fast_route_amd import fused_moe_mxfp4
    x, logits, q = _layer_inputs(M, 256, 512, 8, torch.bfloat16, 31)
    weights = _prepared(q)
    good = fused_moe_mxfp4(x.cuda(), weights, logits.cuda(), 2)
    x2, l2 = x.clone(), logits.clone()
    x2[1, 100] = float("nan")
    got = fused_moe_mxfp4(x2.cuda(), weights, l2.cuda(), 2)
    assert got[1].isnan().all()
    rest = torch.arange(M, device="cuda") != 1
    assert torch.equal(got[rest], good[rest])
    l2[1] = float("nan")
    got = fused_moe_mxfp4(x.cuda(), weights, l2.cuda(), 2)
    assert torch.equal(got[rest], good[rest])
    l2[1] = float("-inf")
    got = fused_moe_mxfp4(x.cuda(), weights, l2.cuda(), 2)
    assert torch.equal(got[rest], good[rest])


def test_layer_of_no_tokens(native):
    from fast_route_amd import fused_moe_mxfp4
    x, logits, q = _layer_inputs(4, 64, 64, 4, torch.bfloat16, 2)
    out = fused_moe_mxfp4(x.cuda()[:0], _prepared(q), logits.cuda()[:0], 2)
    assert out.shape == (0, 64)


def test_all_tokens_on_one_expert(native):
    from fast_route_amd import fused_moe_mxfp4
    for M in (12, 70, 600):
        x, logits, q = _layer_inputs(M, 256, 288, 8, torch.float16, 12)
        logits[:, 5] += 50
        got = fused_moe_mxfp4(x.cuda(), _prepared(q), logits.cuda(), 1)
        _check_layer(got, x, logits, q, 1, True, torch.float16)


@pytest.mark.parametrize("M", [1, 9, 50, 500])
def test_captured_and_replayed(native, M):
    """The first calls of a set of sizes may be the captured ones; replays see new inputs, eager work lies between them."""
    from fast_route_amd import dequantize_rows_mxfp4, fused_moe_mxfp4, linear_mxfp4, prepare_linear_mxfp4, quantize_rows_mxfp4
    H, F, E, k = 512, 384, 8, 2
    x, logits, q = _layer_inputs(M, H, F, E, torch.bfloat16, 77)
    weights = _prepared(q)
    lin = prepare_linear_mxfp4(*(torch.from_numpy(t).cuda() for t in _weight(320, H, 3)))
    sx, sl = x.cuda(), logits.cuda()

    def step():
        h = dequantize_rows_mxfp4(*quantize_rows_mxfp4(sx), dtype=torch.bfloat16)
        return fused_moe_mxfp4(h, weights, sl, k), linear_mxfp4(h, lin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        sx.copy_(torch.randn(M, H, generator=g))
        sl.copy_(torch.randn(M, E, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(kept, eager):
            assert torch.equal(a, b), f"replay {i}"


def test_two_streams_at_once(native):
    from fast_route_amd import fused_moe_mxfp4
    weights, calls = None, []
    for i, M in enumerate((300, 6)):
        x, logits, q = _layer_inputs(M, 512, 384, 8, torch.bfloat16, 50 + i)
        weights = weights or _prepared(q)
        calls.append((x.cuda(), logits.cuda()))
    want = [fused_moe_mxfp4(x, weights, l, 2) for x, l in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(fused_moe_mxfp4(calls[i][0], weights, calls[i][1], 2))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals(native):
    import fast_route_amd as fr
    x = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    codes, scales = fr.quantize_rows_mxfp4(x)
    weight = fr.prepare_linear_mxfp4(codes, scales)
    w1, s1 = codes.view(1, 8, 32).repeat(1, 16, 1), scales.view(1, 8, 2).repeat(1, 16, 1)
    w2, s2 = codes.view(1, 8, 32).repeat(1, 8, 1), scales.view(1, 8, 2).repeat(1, 8, 1)
    experts = fr.prepare_weights_mxfp4(w1, s1, w2, s2)
    logits = torch.zeros(8, 1, device="cuda")
    assert fr.fused_moe_mxfp4(x, experts, logits, 1).abs().max() == 0
    bad = [
        lambda: fr.quantize_rows_mxfp4(x.float()), lambda: fr.quantize_rows_mxfp4(x[:, :33]), lambda: fr.quantize_rows_mxfp4(x[:, 1:33]),
        lambda: fr.quantize_rows_mxfp4(x.t()), lambda: fr.quantize_rows_mxfp4(x.view(2, 4, 64)), lambda: fr.quantize_rows_mxfp4(x[:1].expand(8, 64)),
        lambda: fr.dequantize_rows_mxfp4(codes, scales[:4]), lambda: fr.dequantize_rows_mxfp4(codes.int(), scales),
        lambda: fr.dequantize_rows_mxfp4(codes, scales, dtype=torch.float64), lambda: fr.dequantize_rows_mxfp4(codes[:, ::2], scales),
        lambda: fr.prepare_linear_mxfp4(codes[:0], scales[:0]), lambda: fr.prepare_linear_mxfp4(w1, s1),
        lambda: fr.linear_mxfp4(x[:, :32], weight), lambda: fr.linear_mxfp4(x.float(), weight),
        lambda: fr.linear_mxfp4(x.repeat(5, 1), weight, workspace_buf=torch.empty(16, dtype=torch.uint8, device="cuda")),
        lambda: fr.linear_mxfp4(x, weight, workspace_buf=torch.empty(1 << 20, dtype=torch.uint8)),
        lambda: fr.prepare_weights_mxfp4(w1, s1, w2[:, :32], s2[:, :32]), lambda: fr.prepare_weights_mxfp4(w1[:, :96], s1[:, :96], w2, s2),
        lambda: fr.fused_moe_mxfp4(x, experts, logits, 2), lambda: fr.fused_moe_mxfp4(x, experts, logits, 0),
        lambda: fr.fused_moe_mxfp4(x, experts, logits[:4], 1), lambda: fr.fused_moe_mxfp4(x.float(), experts, logits, 1),
        lambda: fr.fused_moe_mxfp4(x[:, :32].contiguous(), experts, logits, 1), lambda: fr.fused_moe_mxfp4(x, experts, logits.double(), 1),
        lambda: fr.fused_moe_mxfp4(x, experts, logits, 1, workspace_buf=torch.empty(256, dtype=torch.uint8, device="cuda")),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("case", i, "was not refused", flush=True)
    torch.cuda.synchronize()


def test_transformer_layer_runs_on_mxfp4_weights(native):
    """Projections, attention and experts together, as the bench's --mxfp4 calls them, against the same layer step by step in
    64 bits from the operators' own inputs: the projections' result is what the attention gets, its sum what the experts get."""
    from fast_route_amd import transformer_layer_bench as tb
    hidden, n_head, head_dim, F, E, topk = 256, 4, 64, 320, 8, 2
    torch.manual_seed(5)
    attn = tb.Attention(hidden, n_head, head_dim, torch.float16).to("cuda")
    attn4 = tb.AttentionMXFP4(attn)
    g = torch.Generator(device="cuda").manual_seed(6)
    gate, w1, w2 = (torch.randn(s, device="cuda", dtype=torch.float16, generator=g) / d
                    for s, d in (((hidden, E), 16), ((E, 2 * F, hidden), 12), ((E, hidden, F), 18)))
    experts = tb.quantize_experts_mxfp4(w1, w2)
    q1 = [t.reshape(E, 2 * F, -1) for t in oracle.mxfp4_quant_rows(w1.cpu().view(-1, hidden))]
    q2 = [t.reshape(E, hidden, -1) for t in oracle.mxfp4_quant_rows(w2.cpu().view(-1, F))]
    for b, s in ((1, 1), (2, 33), (1, 300)):
        x = torch.randn((b, s, hidden), device="cuda", dtype=torch.float16, generator=g)
        with torch.no_grad():
            h = (attn4(x) + x).view(-1, hidden)
            logits = h @ gate
            out = tb.transformer_layer_mxfp4(attn4, x, gate, experts, topk)
            qkv = attn4.qkv
            got = tb.linear_mxfp4(x.view(-1, hidden), qkv)
        wq = oracle.mxfp4_held(attn.qkv.weight.detach().cpu())
        xv = oracle.mxfp4_held(x.cpu().view(-1, hidden))
        ref, terms = xv @ wq.T, np.abs(xv) @ np.abs(wq).T
        bound = 2.0 ** -11 * np.abs(ref) + _sum_error(terms, hidden) * 1.001 + 2.0 ** -22
        assert (np.abs(got.double().cpu().numpy() - ref) <= bound).all()
        _check_layer(out, h.cpu(), logits.cpu(), (*q1, *q2), topk, True, torch.float16)


def test_first_calls_of_a_process_under_capture(native):
    """Nothing has run before: the captured calls are the kernels' first, replays equal the eager calls that follow."""
    import subprocess
    import sys
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch, fast_route_amd as fr
g = torch.Generator(device="cuda").manual_seed(1)
E, H, F, k = 8, 512, 384, 2
held = []
for shape in ((E, 2 * F, H), (E, H, F)):
    c, s = fr.quantize_rows_mxfp4(torch.randn(shape, device="cuda", generator=g).bfloat16().view(-1, shape[2]) / 16)
    held += [c.view(shape[0], shape[1], -1), s.view(shape[0], shape[1], -1)]
weights = fr.prepare_weights_mxfp4(*held)
lin = fr.prepare_linear_mxfp4(*fr.quantize_rows_mxfp4(torch.randn((640, H), device="cuda", generator=g).bfloat16()))
calls = []
for M in (1, 20, 300):
    x = torch.randn((M, H), device="cuda", generator=g).bfloat16()
    l = torch.randn((M, E), device="cuda", generator=g)
    calls.append((x, l))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = [(fr.fused_moe_mxfp4(x, weights, l, k), fr.linear_mxfp4(x, lin)) for x, l in calls]
for i in range(3):
    for x, l in calls:
        x.normal_(generator=g)
        l.normal_(generator=g)
    graph.replay()
    torch.cuda.synchronize()
    for (x, l), (a, b) in zip(calls, outs):
        assert torch.equal(a, fr.fused_moe_mxfp4(x, weights, l, k)) and torch.equal(b, fr.linear_mxfp4(x, lin)), i
print("captured first calls ok")
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=110)
    assert run.returncode == 0 and "captured first calls ok" in run.stdout, run.stderr[-2000:]


def _values64(codes, scales):
    """What codes and scales on the GPU stand for, in 64 bits."""
    from fast_route_amd import dequantize_rows_mxfp4
    return dequantize_rows_mxfp4(codes, scales, dtype=torch.float32).double()


def _held64(x):
    """Rows [rows, K] on the GPU as the format holds them, in 64 bits."""
    blocks = x.double().view(x.shape[0], -1, 32)
    top = blocks.abs().amax(dim=2, keepdim=True)
    unit = torch.ldexp(torch.ones_like(top), torch.frexp(top).exponent - 3)
    v = blocks / torch.where(top > 0, unit, torch.ones_like(unit))
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return ((torch.round(v / step) * step).clamp(-6, 6) * unit).reshape(x.shape)


def _random_weights(shape, seed):
    from fast_route_amd import quantize_rows_mxfp4
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(0, 0.02, generator=g)
    codes, scales = quantize_rows_mxfp4(w.view(-1, shape[-1]))
    return codes.view(*shape[:-1], -1), scales.view(*shape[:-1], -1)


@pytest.mark.parametrize("M", [2, 20, 100, 140, 600])
def test_linear_on_weights_larger_than_the_caches_keep(native, M):
    from fast_route_amd import linear_mxfp4, prepare_linear_mxfp4
    N_, K = 70000, 4096
    codes, scales = _random_weights((N_, K), 3)
    x = _rows(M, K, torch.bfloat16, M).cuda()
    got = linear_mxfp4(x, prepare_linear_mxfp4(codes, scales)).double()
    xv = _held64(x)
    for at in range(0, N_, 14000):
        w = _values64(codes[at:at + 14000], scales[at:at + 14000])
        ref, terms = xv @ w.t(), xv.abs() @ w.abs().t()
        assert ((got[:, at:at + 14000] - ref).abs() <= 2.0 ** -8 * ref.abs() + _sum_error(terms, K) * 1.01).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("apart", [0, 8])
def test_rows_larger_than_the_caches_keep(native, dtype, apart):
    """Codes, scales and values are those of the same rows in calls of 1000."""
    from fast_route_amd import dequantize_rows_mxfp4, quantize_rows_mxfp4
    rows, K = 17001, 4096
    x = torch.randn((rows, K + apart), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).to(dtype)[:, :K]
    x[16000, 33] = float("nan")
    codes, scales = quantize_rows_mxfp4(x)
    values = [dequantize_rows_mxfp4(codes, scales, dtype=t) for t in (torch.float16, torch.bfloat16, torch.float32)]
    for at in range(0, rows, 1000):
        c, s = quantize_rows_mxfp4(x[at:at + 1000].contiguous())
        assert torch.equal(codes[at:at + 1000], c) and torch.equal(scales[at:at + 1000], s)
        for v in values:
            assert torch.equal(v[at:at + 1000].nan_to_num(7e4), dequantize_rows_mxfp4(c, s, dtype=v.dtype).nan_to_num(7e4))
    _same_codes(codes[-1001:], scales[-1001:], x[-1001:].cpu())


@pytest.mark.parametrize("apart,K,N_", [(0, 2080, 6176), (8, 2080, 6176), (0, 2080, 8264), (0, 2080, 8260)])
def test_linear_of_rows_larger_than_the_caches_keep(native, apart, K, N_):
    from fast_route_amd import linear_mxfp4, prepare_linear_mxfp4
    M = 8205
    codes, scales = _random_weights((N_, K), 9)
    x = torch.randn((M, K + apart), device="cuda", generator=torch.Generator(device="cuda").manual_seed(10)).bfloat16()[:, :K]
    x[8200, K - 1] = float("inf")
    got = linear_mxfp4(x, prepare_linear_mxfp4(codes, scales)).double()
    assert got[8200].isnan().all()
    got[8200] = 0
    w = _values64(codes, scales)
    for at in range(0, M, 1641):
        xv = _held64(x[at:at + 1641].contiguous()).nan_to_num(0.0)
        if at <= 8200 < at + 1641:
            xv[8200 - at] = 0
        ref, terms = xv @ w.t(), xv.abs() @ w.abs().t()
        assert ((got[at:at + 1641] - ref).abs() <= 2.0 ** -8 * ref.abs() + _sum_error(terms, K) * 1.01).all()


@pytest.mark.parametrize("M", [1, 6, 30, 45, 200, 700])
def test_layer_on_weights_larger_than_the_caches_keep(native, M):
    """Norm of the difference: half a step of bf16 in every value, 2^-8, and as much again for activated rows that rounded the other way
    (test_layer bounds those one by one)."""
    from fast_route_amd import fused_moe_mxfp4, prepare_weights_mxfp4
    E, H, F, topk = 8, 4096, 8192, 2
    w1, s1 = _random_weights((E, 2 * F, H), 5)
    w2, s2 = _random_weights((E, H, F), 6)
    g = torch.Generator(device="cuda").manual_seed(M)
    x = torch.randn((M, H), device="cuda", generator=g).bfloat16()
    logits = torch.randn((M, E), device="cuda", generator=g)
    got = fused_moe_mxfp4(x, prepare_weights_mxfp4(w1, s1, w2, s2), logits, topk).double()
    top, ids = torch.topk(logits.double(), topk, dim=1)
    share, xv, ref = torch.softmax(top, dim=1), _held64(x), torch.zeros((M, H), dtype=torch.float64, device="cuda")
    for e in range(E):
        token, slot = (ids == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        both = xv[token] @ _values64(w1[e], s1[e]).t()
        act = _held64(both[:, :F] * torch.sigmoid(both[:, :F]) * both[:, F:])
        ref[token] += (act @ _values64(w2[e], s2[e]).t()) * share[token, slot][:, None]
    assert (got - ref).norm() <= 2.0 ** -7 * ref.norm()
    assert (got - ref).norm(dim=1).max() <= 2.0 ** -6 * ref.norm(dim=1).max()


@pytest.mark.parametrize("M", [3, 100])
def test_bad_weights_stay_in_their_expert(native, M):
    """A NaN scale in w2 makes one output feature NaN, and only for tokens of that expert; one in w1 their whole rows."""
    from fast_route_amd import fused_moe_mxfp4
    E, H, F, k = 4, 256, 288, 2
    x, logits, q = _layer_inputs(M, H, F, E, torch.bfloat16, 71)
    good = fused_moe_mxfp4(x.cuda(), _prepared(q), logits.cuda(), k)
    hit = (torch.topk(logits, k, dim=1).indices == 2).any(dim=1).cuda()
    bad = [t.copy() for t in q]
    bad[3][2, 33, 4] = 255
    got = fused_moe_mxfp4(x.cuda(), _prepared(bad), logits.cuda(), k)
    want = torch.zeros(M, H, dtype=torch.bool, device="cuda")
    want[:, 33] = hit
    assert torch.equal(got.isnan(), want) and torch.equal(got[~want], good[~want])
    bad = [t.copy() for t in q]
    bad[1][2, 100, 0] = 255
    got = fused_moe_mxfp4(x.cuda(), _prepared(bad), logits.cuda(), k)
    assert torch.equal(got.isnan(), hit[:, None].expand(M, H)) and torch.equal(got[~hit], good[~hit])


def test_launches_of_a_few_tokens(native, kernels_of):
    """Up to four tokens the whole layer is two launches, up to 32 three; a product of up to four rows is one."""
    from fast_route_amd import fused_moe_mxfp4, linear_mxfp4, prepare_linear_mxfp4
    x, logits, q = _layer_inputs(32, 256, 288, 8, torch.bfloat16, 5)
    weights, x, logits = _prepared(q), x.cuda(), logits.cuda()
    lin = prepare_linear_mxfp4(*(torch.from_numpy(t).cuda() for t in _weight(96, 256, 3)))
    for M, layer, product in ((1, 2, 1), (4, 2, 1), (5, 3, 2), (32, 3, 2)):
        for call, want in ((lambda: fused_moe_mxfp4(x[:M], weights, logits[:M], 2), layer), (lambda: linear_mxfp4(x[:M], lin), product)):
            call()
            torch.cuda.synchronize()
            names = [n for n in kernels_of(call)[1] if "mx_" in n]
            assert len(names) == want, names

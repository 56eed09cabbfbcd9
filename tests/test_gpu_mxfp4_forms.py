"""The forms of the MXFP4 layer and product that sizes choose between: values that no form may lose, and each form's own
tails, repeats, captures and streams."""
import json
import os
import tempfile

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _say(msg):
    print("[case] " + msg, flush=True)


def _weights(E, H, F, seed):
    """Codes and scales of w1 [E, 2F, H] and w2 [E, H, F], on the GPU."""
    from fast_route_amd import quantize_rows_mxfp4
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = []
    for shape, std in (((E, 2 * F, H), 1.5 / H ** 0.5), ((E, H, F), F ** -0.5)):
        w = torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).bfloat16()
        codes, scales = quantize_rows_mxfp4(w.view(-1, shape[2]))
        held += [codes.view(*shape[:2], -1), scales.view(*shape[:2], -1)]
    return held


def _tokens(M, H, E, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((M, H), device="cuda", generator=g).to(dtype), torch.randn((M, E), device="cuda", generator=g)


# M, H, F, E, topk: few tokens, whole tiles of 64 and of 32 weight rows per wavefront, a last partial one, K slices
FORMS = [(3, 256, 512, 8, 2), (20, 256, 512, 8, 2), (40, 4096, 512, 8, 2), (300, 256, 512, 8, 2), (1200, 800, 128, 64, 6),
         (2000, 2080, 64, 64, 2), (50, 1024, 3584, 8, 2), (40, 1056, 2336, 12, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H,F,E,topk", FORMS)
def test_a_feature_does_not_depend_on_its_neighbours(native, M, H, F, E, topk, dtype):
    """One output feature in sixteen 2^10 (fp16: 2^6) times larger: all others keep their bits, at every batch size, as sums in fp32
    do; the large ones are scaled by a power of two exactly, but where the type rounded them as subnormals."""
    from fast_route_amd import fused_moe_mxfp4, prepare_weights_mxfp4
    _say(f"neighbours M={M} H={H} F={F} E={E} topk={topk} {dtype}")
    w1, s1, w2, s2 = _weights(E, H, F, M + H)
    x, logits = _tokens(M, H, E, dtype, M)
    plain = fused_moe_mxfp4(x, prepare_weights_mxfp4(w1, s1, w2, s2), logits, topk)
    shift = 10 if dtype == torch.bfloat16 else 6
    s2[:, 5::16] += shift  # scale bytes; far from 255 here
    got = fused_moe_mxfp4(x, prepare_weights_mxfp4(w1, s1, w2, s2), logits, topk)
    large = torch.zeros(H, dtype=torch.bool, device="cuda")
    large[5::16] = True
    assert torch.equal(got[:, ~large], plain[:, ~large])
    was, now = plain[:, large].double(), got[:, large].double()
    normal = was.abs() >= torch.finfo(dtype).smallest_normal
    assert normal.double().mean() > 0.99 and torch.equal(now[normal], was[normal] * 2.0 ** shift)


def test_handles_whose_data_are_others_are_refused(native):
    """Nothing is launched on a prepared weight whose data do not match its sizes or lie elsewhere."""
    import fast_route_amd as fr
    w1, s1, w2, s2 = _weights(4, 64, 96, 1)
    experts = fr.prepare_weights_mxfp4(w1, s1, w2, s2)
    lin = fr.prepare_linear_mxfp4(w1[0], s1[0])
    x, logits = _tokens(40, 64, 4, torch.bfloat16, 2)
    assert fr.linear_mxfp4(x, lin).shape == (40, 192) and fr.fused_moe_mxfp4(x, experts, logits, 2).shape == x.shape
    wide = torch.cat([logits, logits], dim=1)
    bad = [
        lambda: fr.linear_mxfp4(x, lin._replace(N=4096)), lambda: fr.linear_mxfp4(x, lin._replace(data=lin.data[:4352])),
        lambda: fr.linear_mxfp4(x, lin._replace(data=lin.data.cpu())), lambda: fr.linear_mxfp4(x, lin._replace(data=lin.data.to(torch.int32))),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(w2=experts.w2.cpu()), logits, 2),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(w1=experts.w1.cpu()), logits, 2),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(F=128), logits, 2), lambda: fr.fused_moe_mxfp4(x, experts._replace(w2=experts.w2[4352:]), logits, 2),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(E=8), wide, 2),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("case", i, "was not refused", flush=True)
    torch.cuda.synchronize()


# ---- inputs on which every sum is exact --------------------------------------------------------------------------
# Elements are levels of the format times powers of two that cancel between the operands, gate sums are 32 exactly (silu(32) is 32 in
# 32 bits: 1 + exp(-32) rounds to 1), up sums a level, so activated rows are 32 times a level and are held exactly, and the down
# sums are whole numbers of 1/4 times powers of two, below 2^24 of them; routed weights are 1, 1/2 or 1/4.  The result is the exact one rounded
# once: there is no tolerance, and one wrong element fails.

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
ONE, FOUR = 2, 6  # codes


def _levels():
    half = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    return torch.cat([half, -half])


def _packed(codes):
    return (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8)


def _values(packed, scales):
    """Packed codes [rows, K / 2] and scale bytes [rows, K / 32] in 64 bits."""
    codes = torch.stack([packed & 15, packed >> 4], dim=2).reshape(packed.shape[0], -1).int()
    return _levels()[codes] * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=1)


class ExactLayer:
    def __init__(self, H, F, E, seed=0):
        from fast_route_amd import prepare_weights_mxfp4
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.H, self.F, self.E, self.gen = H, F, E, g
        self.shift = torch.randint(-3, 4, (H // 32,), device="cuda", generator=g)  # of a block of x; the weights' is the opposite
        some = min(8, 1 << ((H // 16).bit_length() - 1))  # columns 0, 16, .. of x are 4: so many of them make a gate sum of 32
        w1 = torch.zeros((E, 2 * F, H), dtype=torch.uint8, device="cuda")

        def fixed(count):
            return 16 * torch.rand((E, F, H // 16), device="cuda", generator=g).topk(count, dim=2).indices
        w1[:, :F].scatter_(2, fixed(some), {8: ONE, 4: 4, 2: FOUR}[some])  # 8 x 1, 4 x 2, 2 x 4
        pair = fixed(2)  # 4 and -4 cancel in an up sum
        w1[:, F:].scatter_(2, pair[..., :1], ONE).scatter_(2, pair[..., 1:], 8 | ONE)
        column = 16 * torch.randint(0, H // 16, (E, F, 1), device="cuda", generator=g) + torch.randint(1, 16, (E, F, 1), device="cuda", generator=g)
        w1[:, F:].scatter_(2, column, (ONE + 8 * torch.randint(0, 2, (E, F, 1), device="cuda", generator=g)).to(torch.uint8))
        self.w1, self.s1 = _packed(w1), (127 - self.shift).to(torch.uint8).expand(E, 2 * F, H // 32).contiguous()
        self.w2 = _packed(torch.randint(0, 16, (E, H, F), dtype=torch.uint8, device="cuda", generator=g))
        self.s2 = torch.randint(117, 119, (E, H, F // 32), device="cuda", generator=g).to(torch.uint8)
        self.experts = prepare_weights_mxfp4(self.w1, self.s1, self.w2, self.s2)

    def tokens(self, M, topk, dtype):
        """Hidden states, logits and the layer's result."""
        assert topk in (1, 2, 4) and self.F * 36 * 2 * 4 * topk < 1 << 24
        codes = torch.randint(0, 16, (M, self.H), device="cuda", generator=self.gen)
        codes[:, ::16] = FOUR
        x = (_levels()[codes] * torch.exp2(self.shift.double()).repeat_interleave(32)).to(dtype)
        ids = torch.rand((M, self.E), device="cuda", generator=self.gen).topk(topk, dim=1).indices
        logits = torch.full((M, self.E), -100.0, device="cuda").scatter_(1, ids, 0.0)
        out = torch.zeros((M, self.H), dtype=torch.float64, device="cuda")
        for e in range(self.E):
            token = (ids == e).any(dim=1).nonzero()[:, 0]
            if token.numel():
                both = x[token].double() @ _values(self.w1[e], self.s1[e]).t()
                assert (both[:, :self.F] == 32).all() and both.abs().max() <= 32
                out[token] += 32 * both[:, self.F:] @ _values(self.w2[e], self.s2[e]).t() / topk
        return x, logits, out.float().to(dtype)


def _grids(call):
    """What a call returns and its kernels of this path in order: (name, grid)."""
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as prof:
        out = call()
        torch.cuda.synchronize()
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "trace.json")
        prof.export_chrome_trace(path)
        with open(path) as f:
            events = [e for e in json.load(f)["traceEvents"] if e.get("cat") == "kernel" and "mx_" in e["name"]]
    return out, [(e["name"], tuple(e["args"]["grid"])) for e in sorted(events, key=lambda e: e["ts"])]


def _form(M, H, F, E, topk, kernels):
    """The form that a layer's launches show: few tokens ("route": two launches, "alone": a feature block per wavefront of the gate/up product, "shared":
    per workgroup; parts of the down product), or the products by tiles (K slices of the down product, weight row groups of a wavefront)."""
    n = M * topk
    experts, act_tiles = min(n, E), -(-F // 256)
    by_name = {k: [g for name, g in kernels if k in name] for k in ("few_front", "few_gateup", "few_down", "gemm")}
    if by_name["few_down"]:
        (gateup,), (down,) = by_name["few_gateup"], by_name["few_down"]
        assert gateup[1] == experts and down[0] == H // 32
        kind = "route" if not by_name["few_front"] else {act_tiles * 2: "alone", act_tiles * 8: "shared"}[gateup[0]]
        return kind, down[1]
    down = by_name["gemm"][1]
    tiles = min(n, (n + 31 * E) // 32) // 4 + experts
    wide = {8 * -(-tiles * -(-(H // 32) // (4 * j)) // 8): j for j in (1, 2)}
    return "tiles", down[1], wide[down[0]]


# M, H, F, E, topk, form
EXACT = [(1, 1024, 3584, 8, 2, ("route", 1)), (4, 1024, 3584, 8, 2, ("route", 3)), (5, 1024, 3584, 8, 2, ("alone", 3)),
         (32, 2048, 1408, 64, 4, ("alone", 4)), (6, 256, 2048, 8, 2, ("alone", 2)), (6, 256, 2016, 8, 2, ("shared", 2)),
         (6, 2048, 2048, 8, 1, ("shared", 1)), (9, 2048, 2048, 8, 1, ("alone", 2)), (9, 2080, 2048, 8, 1, ("shared", 2)),
         (24, 4096, 8192, 8, 2, ("shared", 2)), (32, 512, 1408, 64, 4, ("alone", 8)), (2, 4096, 8192, 8, 2, ("route", 2)),
         (50, 1024, 3584, 8, 2, ("tiles", 3, 2)), (40, 1056, 2336, 12, 4, ("tiles", 2, 2)), (45, 4096, 8192, 8, 2, ("tiles", 4, 2)),
         (200, 4096, 8192, 8, 2, ("tiles", 1, 1)), (700, 4096, 8192, 8, 2, ("tiles", 1, 2)), (1200, 800, 128, 64, 4, ("tiles", 1, 2)),
         (2000, 2080, 64, 64, 2, ("tiles", 1, 2)), (300, 320, 1120, 12, 4, ("tiles", 1, 1)), (8192, 1056, 96, 3, 1, ("tiles", 1, 2))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H,F,E,topk,form", EXACT)
def test_exact_layer(native, M, H, F, E, topk, form, dtype):
    """The exact result, by the form that the sizes were chosen for."""
    from fast_route_amd import fused_moe_mxfp4
    _say(f"exact layer M={M} H={H} F={F} E={E} topk={topk} {form} {dtype}")
    layer = ExactLayer(H, F, E, seed=M)
    x, logits, want = layer.tokens(M, topk, dtype)
    assert want.isfinite().all()
    got = fused_moe_mxfp4(x, layer.experts, logits, topk)
    assert torch.equal(got, want)
    got, kernels = _grids(lambda: fused_moe_mxfp4(x, layer.experts, logits, topk))
    assert torch.equal(got, want) and _form(M, H, F, E, topk, kernels) == form


# forms whose workgroups meet through memory: parts of the few-token down product, K slices of the other
JOINED = [(4, 1024, 3584, 8, 2), (5, 1024, 3584, 8, 2), (32, 2048, 1408, 64, 4), (24, 4096, 2048, 8, 2), (50, 1024, 3584, 8, 2), (40, 1056, 2336, 12, 4)]


@pytest.mark.parametrize("M,H,F,E,topk", JOINED)
def test_joined_parts_in_one_workspace(native, M, H, F, E, topk):
    """Call after call in one workspace, other inputs each time, whatever it held before: no part and no count of an earlier call is
    taken for the present one's."""
    from fast_route_amd import fused_moe_mxfp4
    _say(f"joined M={M} H={H} F={F} E={E} topk={topk}")
    layer = ExactLayer(H, F, E, seed=1)
    calls = [layer.tokens(M, topk, torch.bfloat16) for _ in range(3)]
    ws = torch.empty(native.fr_moe_mxfp4_workspace_bytes(M, H, F, E, topk), dtype=torch.uint8, device="cuda")
    for fill in (0x00, 0xFF, 0x5A, None):
        if fill is not None:
            ws.fill_(fill)
        outs = [fused_moe_mxfp4(x, layer.experts, logits, topk, workspace_buf=ws) for x, logits, _ in calls * 4]
        for i, got in enumerate(outs):
            assert torch.equal(got, calls[i % 3][2]), f"fill {fill}, call {i}"
    x, logits, want = calls[0]
    given = x.clone()
    assert fused_moe_mxfp4(given, layer.experts, logits, topk, inplace=True, workspace_buf=ws) is given and torch.equal(given, want)


@pytest.mark.parametrize("M,H,F,E,topk", JOINED)
def test_joined_parts_captured_and_replayed(native, M, H, F, E, topk):
    """A graph of two calls in one workspace, replayed on other inputs with eager calls and synchronizations between the replays."""
    from fast_route_amd import fused_moe_mxfp4
    _say(f"joined captured M={M} H={H} F={F} E={E} topk={topk}")
    layer = ExactLayer(H, F, E, seed=2)
    calls = [layer.tokens(M, topk, torch.bfloat16) for _ in range(4)]
    sx, sl = [calls[0][0].clone() for _ in range(2)], [calls[0][1].clone() for _ in range(2)]
    ws = torch.full((native.fr_moe_mxfp4_workspace_bytes(M, H, F, E, topk),), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [fused_moe_mxfp4(sx[i], layer.experts, sl[i], topk, workspace_buf=ws) for i in range(2)]
    for replay in range(5):
        use = [calls[replay % 4], calls[(replay + 1) % 4]]
        for i in range(2):
            sx[i].copy_(use[i][0])
            sl[i].copy_(use[i][1])
        graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], use[i][2]), f"replay {replay}, call {i}"
        x, logits, want = calls[(replay + 2) % 4]
        assert torch.equal(fused_moe_mxfp4(x, layer.experts, logits, topk, workspace_buf=ws), want)


def test_joined_parts_on_two_streams(native):
    """Both joined forms at once on streams of their own, workspaces from the allocator, other inputs in turn."""
    from fast_route_amd import fused_moe_mxfp4
    H, F, E, topk = 1024, 3584, 8, 2
    layer = ExactLayer(H, F, E, seed=3)
    calls = [[layer.tokens(M, topk, torch.bfloat16) for _ in range(2)] for M in (5, 50)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for r in range(12):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, logits, _ = calls[i][r % 2]
                got[i].append(fused_moe_mxfp4(x, layer.experts, logits, topk))
    torch.cuda.synchronize()
    for i in range(2):
        for r, g in enumerate(got[i]):
            assert torch.equal(g, calls[i][r % 2][2]), f"stream {i}, call {r}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H,F,E,topk", JOINED + [(9, 2048, 2048, 8, 1), (300, 320, 1120, 12, 4), (1200, 800, 128, 64, 4)])
def test_bad_values_stay_where_they_are(native, M, H, F, E, topk, dtype):
    """An infinity in a token row makes that row NaN; a token of NaN logits changes nobody else's row; a NaN scale in w2 makes one
    feature of its expert's tokens NaN, one in w1 their rows."""
    from fast_route_amd import fused_moe_mxfp4, prepare_weights_mxfp4
    _say(f"bad values M={M} H={H} F={F} E={E} topk={topk} {dtype}")
    layer = ExactLayer(H, F, E, seed=4)
    x, logits, want = layer.tokens(M, topk, dtype)
    row = torch.arange(M, device="cuda")
    bad = x.clone()
    bad[M - 1, H - 1] = float("inf")
    got = fused_moe_mxfp4(bad, layer.experts, logits, topk)
    assert got[M - 1].isnan().all() and torch.equal(got[row != M - 1], want[row != M - 1])
    for value in (float("nan"), float("-inf")):
        odd = logits.clone()
        odd[1] = value
        assert torch.equal(fused_moe_mxfp4(x, layer.experts, odd, topk)[row != 1], want[row != 1])
    expert = int(logits[0].argmax())
    hit = logits[:, expert] == 0
    s2 = layer.s2.clone()
    s2[expert, H - 3, F // 32 - 1] = 255
    got = fused_moe_mxfp4(x, prepare_weights_mxfp4(layer.w1, layer.s1, layer.w2, s2), logits, topk)
    nan = torch.zeros((M, H), dtype=torch.bool, device="cuda")
    nan[:, H - 3] = hit
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], want[~nan])
    s1 = layer.s1.clone()
    s1[expert, 2 * F - 1, H // 32 - 1] = 255
    got = fused_moe_mxfp4(x, prepare_weights_mxfp4(layer.w1, s1, layer.w2, layer.s2), logits, topk)
    assert got[hit].isnan().all() and torch.equal(got[~hit], want[~hit])


def test_logits_anywhere_in_memory(native):
    """Rows of logits need no alignment: a dense slice that begins at any element."""
    from fast_route_amd import fused_moe_mxfp4
    for M, E, topk in ((3, 3, 2), (20, 7, 2), (60, 5, 2), (900, 33, 4)):
        layer = ExactLayer(64, 64, E, seed=5)
        x, logits, want = layer.tokens(M, topk, torch.bfloat16)
        for dtype in (torch.float32, torch.bfloat16):
            held = torch.zeros(M * E + 1, device="cuda", dtype=dtype)
            held[1:] = logits.view(-1)
            assert torch.equal(fused_moe_mxfp4(x, layer.experts, held[1:].view(M, E), topk), want), (M, E, dtype)


LINEAR = [(M, 4096, K) for M in (1, 4, 5, 32, 33, 60, 100, 129, 512) for K in (4096, 14336)] + [
    (4, 96, 99 * 256), (4, 96, 100 * 256), (300, 1031, 4096), (600, 12287, 1024), (130, 72, 12288), (2000, 520, 288)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N_,K", LINEAR)
def test_exact_linear(native, M, N_, K, dtype):
    """Levels times powers of two that cancel: sums are whole numbers of 1/4 below 2^24 of them, the result the exact one rounded once."""
    from fast_route_amd import linear_mxfp4, prepare_linear_mxfp4
    _say(f"exact linear {M}x{N_}x{K} {dtype}")
    assert K * 36 * 2 * 4 < 1 << 24
    g = torch.Generator(device="cuda").manual_seed(M + N_ + K)
    shift = torch.randint(-3, 4, (K // 32,), device="cuda", generator=g)
    codes = torch.randint(0, 16, (M, K), device="cuda", generator=g)
    codes[:, ::32] = FOUR
    x = (_levels()[codes] * torch.exp2(shift.double()).repeat_interleave(32)).to(dtype)
    w = _packed(torch.randint(0, 16, (N_, K), dtype=torch.uint8, device="cuda", generator=g))
    scales = (torch.randint(120, 122, (N_, K // 32), device="cuda", generator=g) - shift).to(torch.uint8)
    got, kernels = _grids(lambda: linear_mxfp4(x, prepare_linear_mxfp4(w, scales)))
    assert torch.equal(got, (x.double() @ _values(w, scales).t()).float().to(dtype))
    names = [name for name, _ in kernels if "tile_weights" not in name]
    assert len(names) == (1 if M <= 4 and K < 25600 else 2)  # up to four rows that fit in LDS are quantised inside the product


def test_offsets_beyond_32_bits(native):
    """More than 2^31 elements of rows: the same 4096 rows again and again, every block the first one's result."""
    from fast_route_amd import dequantize_rows_mxfp4, fused_moe_mxfp4, linear_mxfp4, prepare_linear_mxfp4, quantize_rows_mxfp4
    H, block, times = 4096, 4096, 129
    layer = ExactLayer(H, 64, 3, seed=6)
    x, logits, want = layer.tokens(block, 1, torch.bfloat16)
    many, many_logits = x.repeat(times, 1), logits.repeat(times, 1)
    assert many.numel() > 1 << 31
    _say("beyond 32 bits: layer")
    got = fused_moe_mxfp4(many, layer.experts, many_logits, 1).view(times, block, H)
    assert all(torch.equal(got[i], want) for i in range(times))
    del got
    _say("beyond 32 bits: linear")
    narrow = x[:, :64].contiguous()
    weight = prepare_linear_mxfp4(*quantize_rows_mxfp4(x[:, :64]))  # [4096, 64]: as many output features as rows
    first = linear_mxfp4(narrow, weight)
    got = linear_mxfp4(many[:, :64], weight).view(times, block, H)  # rows 8 KB apart
    assert all(torch.equal(got[i], first) for i in range(times))
    del got
    _say("beyond 32 bits: quantisation")
    codes, scales = quantize_rows_mxfp4(many)
    back = dequantize_rows_mxfp4(codes, scales).view(times, block, H)
    assert all(torch.equal(back[i], x) for i in range(times))

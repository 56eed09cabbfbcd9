"""rotary_embed and rotary_to_cache against their definition in 64 bits (oracle/serving_oracle.py)."""
import math

import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _say(msg):
    print("[case] " + msg, flush=True)


def _close(got, x, positions, freq, interleaved, factor=1.0, seen=None):
    """The result's own rounding, and the angle's (its 32-bit part of a turn 2^-25 turn, its frequency 2^-56 turn a position), sine's and cosine's and
    three fp32 operations': together below 2^-20 of the pair's size at positions up to 2^31."""
    ref = oracle.rotary(x, positions, freq, interleaved, factor)
    n = 2 * freq.numel()
    size = torch.zeros_like(ref)
    first, second = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    pair = (x.double()[..., first].abs() + x.double()[..., second].abs()) * abs(factor)
    size[..., first], size[..., second] = pair, pair
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps  # half a step of the subnormal ones, twice
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -10) + 2.0 ** -20 * size + tiny
    bad = (got.cpu().double() - ref).abs() > tol
    assert not bad.any(), "worst %g of the bound" % ((got.cpu().double() - ref).abs() / tol).max().item()


def _inputs(T, H, G, D, dtype, seed, farthest=10000):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, H + 2 * G, D, generator=g).to(dtype)
    return qkv, torch.randint(0, farthest, (T,), generator=g)


SHAPES = [(1, 1, 1, 2, 2), (3, 4, 2, 16, 16), (7, 8, 8, 64, 32), (2, 32, 8, 128, 128), (37, 12, 4, 80, 80), (130, 16, 2, 96, 40), (5, 2, 1, 512, 512), (9, 3, 3, 7, 6),
          (6, 5, 1, 1024, 512), (4, 4, 4, 24, 0), (4099, 4, 2, 64, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,G,D,turned", SHAPES)
def test_turned(native, T, H, G, D, turned, interleaved, dtype):
    from fast_route_amd import prepare_rotary, rotary_embed, rotary_frequencies
    _say(f"T={T} H={H} G={G} D={D} turned={turned} {interleaved} {dtype}")
    qkv, positions = _inputs(T, H, G, D, dtype, T + D)
    freq = rotary_frequencies(turned)
    rotary = prepare_rotary(freq, interleaved, device="cuda")
    held = qkv.cuda()
    q, k = held[:, :H], held[:, H:H + G]
    for at in (positions, positions.int()):
        q2, k2 = rotary_embed(q, k, at.cuda(), rotary)
        _close(q2, qkv[:, :H], positions, freq, interleaved)
        _close(k2, qkv[:, H:H + G], positions, freq, interleaved)
    assert torch.equal(held.cpu(), qkv)
    back = rotary_embed(q, k, positions.cuda(), rotary, inplace=True)
    assert back[0].data_ptr() == q.data_ptr() and torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(held[:, H + G:].cpu(), qkv[:, H + G:])


def test_far_and_negative_positions(native):
    from fast_route_amd import prepare_rotary, rotary_embed, rotary_frequencies
    _say("far positions")
    positions = torch.tensor([0, 1, 8191, 131072, 999999, 10 ** 7 + 1, 2 ** 31 - 1, -1, -4096, -(2 ** 31)])
    qkv, _ = _inputs(len(positions), 4, 2, 128, torch.float16, 5)
    for freq in (rotary_frequencies(128), rotary_frequencies(128, base=500000.0, scale=8.0, original=8192), rotary_frequencies(128, scale=4.0)):
        rotary = prepare_rotary(freq, device="cuda")
        q2, k2 = rotary_embed(qkv[:, :4].cuda(), qkv[:, 4:].cuda(), positions.cuda(), rotary)
        _close(q2, qkv[:, :4], positions, freq, False)
        _close(k2, qkv[:, 4:], positions, freq, False)


def test_factor_and_frequencies(native):
    from fast_route_amd import prepare_rotary, rotary_embed, rotary_frequencies
    _say("factor")
    qkv, positions = _inputs(11, 4, 2, 64, torch.bfloat16, 6)
    freq = torch.linspace(-3.0, 3.0, 32, dtype=torch.float64)
    rotary = prepare_rotary(freq.cuda(), factor=1.2079)
    assert rotary.turns.is_cuda
    q2, k2 = rotary_embed(qkv[:, :4].cuda(), qkv[:, 4:6].cuda(), positions.cuda(), rotary)
    _close(q2, qkv[:, :4], positions, freq, False, 1.2079)
    mixed = rotary_frequencies(64, scale=8.0, original=8192, slow_turns=1.0, fast_turns=4.0)
    plain = rotary_frequencies(64)
    turns = plain * 8192 / (2 * math.pi)
    assert torch.equal(mixed[turns >= 4], plain[turns >= 4]) and torch.allclose(mixed[turns <= 1], plain[turns <= 1] / 8)
    between = (turns > 1) & (turns < 4)
    assert between.any() and (mixed[between] < plain[between]).all() and (mixed[between] > plain[between] / 8).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H,G,D,turned,page,interleaved", [(1, 4, 1, 64, 64, 16, False), (5, 8, 2, 128, 64, 16, True), (67, 6, 3, 80, 48, 8, False),
                                                             (29, 3, 1, 18, 10, 5, True), (4100, 2, 1, 64, 64, 64, False)])
def test_into_the_cache(native, T, H, G, D, turned, page, interleaved, dtype):
    from fast_route_amd import prepare_rotary, rotary_embed, rotary_frequencies, rotary_to_cache
    _say(f"cache T={T} D={D} page={page} {dtype}")
    qkv, positions = _inputs(T, H, G, D, dtype, T)
    rotary = prepare_rotary(rotary_frequencies(turned), interleaved, device="cuda")
    held = qkv.cuda()
    q, k, v = held[:, :H], held[:, H:H + G], held[:, H + G:]
    q2, k2 = rotary_embed(q, k, positions.cuda(), rotary)
    pages = -(-T // page) + 3
    g = torch.Generator().manual_seed(T)
    slots = torch.randperm(pages * page, generator=g)[:T]
    lost = torch.zeros(T, dtype=torch.bool)
    if T > 3:
        slots[1], slots[3] = -1, pages * page  # not kept
        lost[[1, 3]] = True
    for order in ("pages first", "heads first"):
        if order == "pages first":
            kc, vc = (torch.full((pages, page, G, D), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        else:
            kc, vc = (torch.full((pages, G, page, D), 7.0, dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2))
        for kind in (torch.int64, torch.int32):
            q3, k3 = rotary_to_cache(q, k, v, positions.cuda(), rotary, kc, vc, slots.to(kind).cuda())
            assert torch.equal(q3, q2) and torch.equal(k3, k2)
            for cache, rows in ((kc, k2), (vc, v)):
                want = torch.full((pages * page, G, D), 7.0, dtype=dtype)
                want[slots[~lost]] = rows.cpu()[~lost]
                assert torch.equal(cache.reshape(pages * page, G, D).cpu(), want)
    kc.fill_(7.0), vc.fill_(7.0)
    rotary_to_cache(q, k, v, positions.cuda(), rotary, kc, vc, slots.cuda(), inplace=True)
    want = torch.full((pages * page, G, D), 7.0, dtype=dtype)
    want[slots[~lost]] = k2.cpu()[~lost]
    assert torch.equal(kc.reshape(pages * page, G, D).cpu(), want) and torch.equal(q, q2) and torch.equal(k, k2)


def test_odd_addresses_and_strides(native):
    """Rows that 16-byte accesses cannot read give the same values."""
    from fast_route_amd import prepare_rotary, rotary_embed, rotary_frequencies
    _say("odd addresses")
    T, H, D = 9, 4, 64
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    positions = torch.arange(T).cuda()
    for interleaved in (False, True):
        rotary = prepare_rotary(rotary_frequencies(D), interleaved, device="cuda")
        q2, k2 = rotary_embed(x, x[:, :2], positions, rotary)
        odd = torch.empty(T * H * D + 1, dtype=x.dtype, device="cuda")[1:].view(T, H, D).copy_(x)
        apart = torch.empty(T, H + 1, D + 3, dtype=x.dtype, device="cuda")[:, 1:, 3:].copy_(x)
        heads_first = x.transpose(0, 1).contiguous().transpose(0, 1)
        for q in (odd, apart, heads_first):
            a, b = rotary_embed(q, q[:, :2], positions, rotary)
            assert torch.equal(a, q2) and torch.equal(b, k2)


def test_no_tokens(native):
    from fast_route_amd import prepare_rotary, rotary_embed, rotary_frequencies
    _say("no tokens")
    rotary = prepare_rotary(rotary_frequencies(64), device="cuda")
    q, k = rotary_embed(torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda"),
                        torch.empty(0, dtype=torch.int64, device="cuda"), rotary)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)


def test_refusals(native):
    from fast_route_amd import prepare_rotary, rotary_embed, rotary_frequencies, rotary_to_cache
    _say("refusals")
    rotary = prepare_rotary(rotary_frequencies(64), device="cuda")
    q, k = torch.zeros(4, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    at, slots = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    kc, vc = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16, device="cuda")
    calls = [lambda: rotary_embed(q.cpu(), k, at, rotary), lambda: rotary_embed(q.float(), k, at, rotary), lambda: rotary_embed(q, k.half(), at, rotary),
             lambda: rotary_embed(q, k[:3], at, rotary), lambda: rotary_embed(q, k, at[:3], rotary), lambda: rotary_embed(q, k, at.float(), rotary),
             lambda: rotary_embed(q[..., :32], k[..., :32], at, rotary), lambda: rotary_embed(q[..., ::2], k[..., ::2], at, prepare_rotary(rotary_frequencies(32), device="cuda")),
             lambda: rotary_embed(q, k, at, prepare_rotary(rotary_frequencies(64))), lambda: rotary_embed(q, k[:, :1].expand(4, 2, 64), at, rotary, inplace=True),
             lambda: rotary_to_cache(q, k, k, at, rotary, kc, vc[:1], slots), lambda: rotary_to_cache(q, k, k, at, rotary, kc[:, :, :1], vc[:, :, :1], slots),
             lambda: rotary_to_cache(q, k, k, at, rotary, kc.half(), vc, slots), lambda: rotary_to_cache(q, k, k[:, :1], at, rotary, kc, vc, slots),
             lambda: rotary_to_cache(q, k, k, at, rotary, kc, vc, slots[:2]), lambda: rotary_to_cache(q, k, k, at, rotary, kc, vc.cpu(), slots),
             lambda: prepare_rotary(torch.tensor([4.0], dtype=torch.float64)), lambda: prepare_rotary(torch.zeros(257)), lambda: rotary_frequencies(7)]
    for i, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
            print("call %d was taken" % i)

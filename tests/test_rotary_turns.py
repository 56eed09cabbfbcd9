"""The handle of rotary frequencies holds them to half a unit of 2^-64 turn, so that angles keep their meaning at far positions."""
import math
from fractions import Fraction

import pytest
import torch

PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


def _frequencies():
    from fast_route_amd import rotary_frequencies
    g = torch.Generator().manual_seed(1)
    return {"plain": rotary_frequencies(128), "long": rotary_frequencies(64, base=500000.0, scale=8.0, original=8192),
            "any": torch.cat([(torch.rand(200, generator=g, dtype=torch.float64) * 2 - 1) * 3.1415926, torch.tensor([0.0, -0.0, 1e-30, 5e-324, -1.0], dtype=torch.float64)]),
            "ends": torch.tensor([math.nextafter(math.pi, 0.0), -math.nextafter(math.pi, 0.0)], dtype=torch.float64), "single": rotary_frequencies(32).float()}


def test_turns_are_exact():
    from fast_route_amd import prepare_rotary
    for name, freq in _frequencies().items():
        turns = prepare_rotary(freq).turns
        for f, t in zip(freq.tolist(), turns.tolist()):
            assert abs(Fraction(f) * 2 ** 63 / PI - t) <= Fraction(1, 2) + Fraction(1, 1000), (name, f, t)


def test_handle_of_another_kind():
    """The kernel reads 64-bit whole numbers, one after the other: a handle that was cast or sliced is refused, before the tensors' device is asked for."""
    from fast_route_amd import Rotary, prepare_rotary, rotary_embed, rotary_frequencies
    x, at, whole = torch.zeros(4, 2, 64, dtype=torch.half), torch.arange(4), prepare_rotary(rotary_frequencies(64))
    for turns in (whole.turns.int(), whole.turns.double(), whole.turns.float(), whole.turns[::2], whole.turns[None], whole.turns[0], torch.zeros(1, dtype=torch.int64).expand(32)):
        with pytest.raises(AssertionError, match="turns"):
            rotary_embed(x, x, at, Rotary(turns, False, 1.0))
    with pytest.raises(AssertionError, match="MI355X"):
        rotary_embed(x, x, at, whole)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(native, interleaved):
    """Angle: position times half a unit of 2^-64 turn, its 32-bit part 2^-25 turn; sine, cosine and three operations below 2^-21 of the pair's size; the result's rounding."""
    from fast_route_amd import prepare_rotary, rotary_embed
    print("[case] far positions", flush=True)
    at = [2 ** 31, 2 ** 40 + 1, 2 ** 44 - 1, -(2 ** 44) + 5, 10 ** 13 + 7, -(10 ** 12), 123456789012, 3]
    for name, freq in _frequencies().items():
        n = freq.numel()
        x = torch.randn(len(at), 2, 2 * n, generator=torch.Generator().manual_seed(n)).half()
        angle = torch.tensor([[float((Fraction(f) * p / (2 * PI)) % 1) * 2 * math.pi for f in freq.tolist()] for p in at], dtype=torch.float64)[:, None]
        first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
        a, b, ref = x.double()[..., first], x.double()[..., second], x.double().clone()
        ref[..., first], ref[..., second] = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
        off = 2 * math.pi * (torch.tensor(at, dtype=torch.float64).abs() * 2.0 ** -65 + 2.0 ** -25)[:, None, None] + 2.0 ** -21
        size = torch.zeros_like(ref)
        size[..., first] = size[..., second] = a.abs() + b.abs()
        tol = off * size + 2.0 ** -11 * (ref.abs() + off * size) + 2.0 ** -24
        q, k = rotary_embed(x.cuda(), x[:, :1].cuda(), torch.tensor(at).cuda(), prepare_rotary(freq, interleaved, device="cuda"))
        assert ((q.cpu().double() - ref).abs() <= tol).all() and ((k.cpu().double() - ref[:, :1]).abs() <= tol[:, :1]).all(), name

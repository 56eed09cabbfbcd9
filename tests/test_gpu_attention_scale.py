"""Attention with scales that make scores of any size."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _say(msg):
    print("[case] " + msg, flush=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-20, 1e4, 1e6, 1e8, 1e12, 1e20])
def test_any_scale(native, scale, dtype):
    """Whole numbers, so that scores are exact and their order is the definition's: with large scales a row is the mean of the values of its largest score, with the
    smallest one of all it sees.  Off by the terms' rounding (none for terms of 1), 32-bit sums and the result's own; at 1e-20 the terms are 1 to 2^-50."""
    from fast_route_amd import attention_varlen, paged_attention
    _say(f"scale {scale} {dtype}")
    for n, m, H, G, D in ((90, 90, 4, 2, 64), (5, 3000, 4, 2, 128), (1, 700, 8, 4, 64), (1, 700, 4, 2, 64), (1, 700, 3, 3, 64), (1, 40, 4, 4, 64), (1, 40, 2, 1, 192)):
        g = torch.Generator().manual_seed(n + m)
        q, (k, v) = torch.randint(-4, 5, (n, H, D), generator=g), (torch.randint(-4, 5, (m, G, D), generator=g) for _ in range(2))
        seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
        want = torch.zeros(n, H, D, dtype=torch.float64)
        for h in range(H):
            s = (q[:, h] @ k[:, h // (H // G)].t()).masked_fill(~seen, -1 << 40)
            p = (seen if scale < 1 else s == s.amax(dim=1, keepdim=True)).double()
            want[:, h] = p @ v[:, h // (H // G)].double() / p.sum(dim=1, keepdim=True)
        tol = 4 * 2.0 ** -18 + torch.finfo(dtype).eps / 2 * want.abs()
        q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
        cu = [torch.tensor([0, c], dtype=torch.int32).cuda() for c in (n, m)]
        got = attention_varlen(q, k, v, *cu, scale=scale)
        assert ((got.cpu().double() - want).abs() <= tol).all(), (n, m, H, G, D)
        if n == 1:
            pages = -(-m // 16)
            kc, vc = (torch.cat([t, t[:pages * 16 - m]]).view(pages, 16, G, D) for t in (k, v))
            got = paged_attention(q, kc, vc, torch.arange(pages, dtype=torch.int32)[None].cuda(), cu[1][1:], scale=scale)
            assert ((got.cpu().double() - want).abs() <= tol).all(), ("paged", m, H, G, D)

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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_parts_of_different_kinds(native, dtype):
    """Keys split along their length, where some parts are done row by row - a value that is not finite among keys that the tile's first rows do not see, or scores far from
    zero in some of the parts only - and the others are not: they are joined as if all were of one kind."""
    import oracle
    from fast_route_amd import attention_varlen
    _say(f"parts {dtype}")
    n, m, H, G, D = 20, 3000, 4, 2, 64
    g = torch.Generator().manual_seed(2)
    q, (k, v) = torch.randn(n, H, D, generator=g).to(dtype), (torch.randn(m, G, D, generator=g).to(dtype) for _ in range(2))
    cu = [torch.tensor([0, c], dtype=torch.int32).cuda() for c in (n, m)]
    assert native.fr_attention_workspace_bytes(1, n, m, H, G, D) > 0
    seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)
    ref, error = oracle.attention(q, k, v, seen, 0.125)
    tol = error + torch.finfo(dtype).eps / 2 * (ref.abs() + error) + 2.0 ** -24
    bad = v.clone()
    bad[-1] = float("inf")  # the last row alone sees it
    got = attention_varlen(q.cuda(), k.cuda(), bad.cuda(), *cu).cpu()
    assert ((got[:-1].double() - ref[:-1]).abs() <= tol[:-1]).all() and not got[-1].isfinite().any()
    # whole numbers: scores are exact.  The first keys' scores are up to 4096 times the others', at a scale that makes these alone too large for one product.
    q = torch.randint(1, 5, (n, H, D), generator=g)
    k, v = torch.randint(-4, 5, (m, G, D), generator=g), torch.randint(-4, 5, (m, G, D), generator=g)
    for sign in (1, -1):
        far = k.clone()
        far[:300] = sign * 512 * torch.randint(4, 9, (300, G, D), generator=g)
        want = torch.zeros(n, H, D, dtype=torch.float64)
        for h in range(H):
            s = (q[:, h] @ far[:, h // 2].t()).masked_fill(~seen, -1 << 40)
            p = (s == s.amax(dim=1, keepdim=True)).double()
            want[:, h] = p @ v[:, h // 2].double() / p.sum(dim=1, keepdim=True)
        got = attention_varlen(*(t.to(dtype).cuda() for t in (q, far, v)), *cu, scale=64.0).cpu()
        assert ((got.double() - want).abs() <= 4 * 2.0 ** -18 + torch.finfo(dtype).eps / 2 * want.abs()).all(), sign

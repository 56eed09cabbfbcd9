"""Sizes that are taken can be launched; others are refused with the sizes' error, before anything is launched."""
import pytest
import torch


def test_sizes_of_a_launch():
    """A launch has fewer than 2^32 threads, 256 to a workgroup."""
    from fast_route_amd import _native
    lib = _native.lib()
    whole, paged = lib.fr_attention_workspace_bytes, lib.fr_paged_attention_workspace_bytes
    # sequences times key heads and rows times heads / 128: B + 1 tiles of a key head for B sequences that may be empty, and what the rows fill
    for B, rows, heads, kv, good in ((1 << 20, 0, 16, 16, False), (1 << 20, 0, 15, 15, True), ((1 << 20) + 1, 0, 1, 1, False), (1, (1 << 26) - 65536, 32, 32, True),
                                     (1, (1 << 26) - 300, 32, 32, False), (1, (1 << 26) - 1500, 32, 1, True), (1, 1 << 26, 32, 1, False), (65535, (1 << 25), 32, 32, True),
                                     (1 << 18, (1 << 25), 32, 32, False)):
        blocks = (-(-rows * (heads // kv) // 128) + B + 1) * kv
        if good:
            assert blocks < 1 << 24 and whole(B, rows, 100, heads, kv, 64) >= 0, (B, rows, heads, kv)
        else:
            assert whole(B, rows, 100, heads, kv, 64) == -1 and b"2^" in lib.fr_last_error_string(), (B, rows, heads, kv)
    # four heads of 256 dimensions to a workgroup of the joining launch
    assert paged(1 << 20, 63, 1, 256, 600) > 0 and paged(1 << 20, 64, 1, 256, 600) == -1 and paged(16777215, 4, 1, 256, 64) == -1
    assert paged((1 << 20) - 1, 64, 1, 256, 600) > 0 and -(-((1 << 20) - 1) * 64 // 4) < 1 << 24


@pytest.mark.gpu
def test_more_tokens_than_a_launch_takes(native):
    """2^26 + 7 tokens, four to a workgroup, two dimensions: against the definition by groups of positions."""
    from fast_route_amd import prepare_rotary, rotary_to_cache
    print("[case] 2^26 tokens", flush=True)
    T, page = (1 << 26) + 7, 64
    assert (T + 3) // 4 > (1 << 24) - 1
    g = torch.Generator("cuda").manual_seed(1)
    q, k, v = (torch.empty(T, 1, 2, dtype=torch.half, device="cuda").normal_(generator=g) for _ in range(3))
    at = torch.arange(T, dtype=torch.int32, device="cuda") % 1000
    slots = (torch.arange(T, dtype=torch.int32, device="cuda") + 5) % T
    kc, vc = (torch.zeros(T // page + 1, page, 1, 2, dtype=torch.half, device="cuda") for _ in range(2))
    q2, k2 = rotary_to_cache(q, k, v, at, prepare_rotary(torch.tensor([0.37], dtype=torch.float64), device="cuda"), kc, vc, slots)
    for lo in (0, (1 << 25) - 99, T - (1 << 20)):  # the middle, and on either side of the second launch
        part = slice(lo, lo + (1 << 20))
        angle = at[part].double() * 0.37
        cos, sin = angle.cos(), angle.sin()
        for x, y in ((q, q2), (k, k2)):
            a, b = x[part, 0, 0].double(), x[part, 0, 1].double()
            for got, want in ((y[part, 0, 0], a * cos - b * sin), (y[part, 0, 1], b * cos + a * sin)):
                # the result's rounding, and the angle's, sine's and cosine's and three operations' together: 2^-20 of the pair's size
                tol = 2.0 ** -11 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -20 * (a.abs() + b.abs()) + 2.0 ** -24
                assert ((got.double() - want).abs() <= tol).all()
        assert torch.equal(kc.view(-1, 1, 2)[slots[part].long()], k2[part]) and torch.equal(vc.view(-1, 1, 2)[slots[part].long()], v[part])
    # every token, by what a turn leaves: a pair's length
    for x, y in ((q, q2), (k, k2)):
        for part in torch.arange(0, T, 1 << 24).tolist():
            a, b = (t[part:part + (1 << 24), 0].float().norm(dim=1) for t in (x, y))
            assert ((a - b).abs() <= 2.0 ** -9 * a + 2.0 ** -20).all(), part
    assert torch.equal(vc.view(-1, 1, 2)[5:T], v[:T - 5]) and torch.equal(kc.view(-1, 1, 2)[5:T], k2[:T - 5])


def test_pages_of_any_size():
    """A page of more than 2^20 keys is one: what stops this call is the address behind it."""
    import struct
    from fast_route_amd import _native
    lib = _native.lib()

    def call(page_size, table_pages):
        return lib.fr_paged_attention(struct.pack("@30qdq", 16, 24, 16, 16, 16, 16, 0, 0, 2, 4, 2, 64, 4, page_size, table_pages, 2, 256, 64, 256, 64, 2048, 128, 64, 2048, 128, 64, 1,
                                                  0, 0, 0, 1.0, 0), None)
    assert call(16, 2) == -4
    for page_size, table_pages in ((1 << 20, 3), ((1 << 20) + 1, 3), (1 << 21, 1), (1 << 30, 1)):
        assert call(page_size, table_pages) == -4, lib.fr_last_error_string()
    assert call(1 << 30, 2) == -2 and call((1 << 30) + 1, 1) == -2 and call(0, 1) == -2


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1 << 21, (1 << 21) - 5])
def test_one_large_page(native, page):
    import oracle
    from fast_route_amd import paged_attention
    print("[case] page of", page, flush=True)
    g = torch.Generator().manual_seed(page)
    kc, vc = (torch.randn(2, page, 1, 8, generator=g).bfloat16() for _ in range(2))
    q, lengths = torch.randn(3, 2, 8, generator=g).bfloat16(), [2 * page - 70, 5, page + 33]
    got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), torch.tensor([[1, 0]] * 3, dtype=torch.int32).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()).cpu()
    k, v = (torch.cat([c[1], c[0]]) for c in (kc, vc))
    for b, n in enumerate(lengths):
        ref, error = oracle.attention(q[b:b + 1], k[:n], v[:n], torch.ones(1, n, dtype=torch.bool), 8 ** -0.5)
        tol = error + 2.0 ** -8 * (ref.abs() + error)
        assert ((got[b:b + 1].double() - ref).abs() <= tol).all()


def test_workspace_holds_the_heads_that_there_are():
    """A place of a key head of up to 16 query heads: a row for each of them, and two numbers, whole 16 bytes together."""
    from fast_route_amd import _native
    need = _native.lib().fr_paged_attention_workspace_bytes
    for B, heads, kv, dim, most in ((256, 32, 32, 128, 2048), (2048, 32, 32, 128, 2048), (64, 32, 8, 128, 16384), (3, 12, 4, 64, 131072), (5, 7, 7, 80, 3000)):
        share, padded = heads // kv, 64 if dim <= 64 else 128
        plan = 0 if B <= 256 else -(-(B + 2) * 4 // 16) * 16
        of_place = lambda share: kv * (share * padded + -(-2 * share // 4) * 4) * 4
        places, rest = divmod(need(B, heads, kv, dim, most) - plan, of_place(share))
        assert rest == 0 and places > B and need(B, heads * 16 // share, kv, dim, most) - plan == places * of_place(16), (B, heads, kv)
    assert need(256, 32, 32, 128, 2048) < 16 << 20


@pytest.mark.gpu
@pytest.mark.parametrize("H,G,D", [(7, 7, 64), (12, 4, 64), (5, 1, 80), (34, 2, 64), (3, 1, 128), (32, 32, 128), (40, 2, 192)])
def test_workspace_of_any_share(native, H, G, D):
    """Exactly as many bytes as are asked for, with what lies on either side of them."""
    import oracle
    from fast_route_amd import paged_attention
    print("[case] workspace", H, G, D, flush=True)
    g = torch.Generator().manual_seed(H + D)
    lengths, page = [900, 33, 1500], 16
    pages = [-(-n // page) for n in lengths]
    table = torch.zeros(3, max(pages), dtype=torch.int32)
    order = torch.randperm(sum(pages), generator=g).to(torch.int32).split(pages)
    for b, o in enumerate(order):
        table[b, :len(o)] = o
    kc, vc = (torch.randn(sum(pages), page, G, D, generator=g).half() for _ in range(2))
    q, need = torch.randn(3, H, D, generator=g).half(), native.fr_paged_attention_workspace_bytes(3, H, G, D, table.shape[1] * page)
    assert need > 0
    held = torch.full((256 + need + 4096,), 0xA5, dtype=torch.uint8, device="cuda")
    got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), workspace_buf=held[256:256 + need]).cpu()
    assert (held[:256] == 0xA5).all() and (held[256 + need:] == 0xA5).all()
    for b, n in enumerate(lengths):
        at = torch.arange(n)
        where = table[b].long()[at // page]
        ref, error = oracle.attention(q[b:b + 1], kc[where, at % page], vc[where, at % page], torch.ones(1, n, dtype=torch.bool), D ** -0.5)
        tol = error + 2.0 ** -11 * (ref.abs() + error) + 2.0 ** -24
        assert ((got[b:b + 1].double() - ref).abs() <= tol).all(), b

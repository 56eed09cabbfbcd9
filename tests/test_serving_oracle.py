"""CPU-only: the serving oracle against torch in 64 bits, the entry points' refusals (which come before anything is launched), the handles."""
import math
import struct

import pytest
import torch

import oracle


def test_attention_is_softmax():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 16, generator=g, dtype=torch.float64) for n, h in ((9, 4), (12, 2), (12, 2)))
    seen = torch.ones(9, 12, dtype=torch.bool).tril(3)
    out, error = oracle.attention(q, k, v, seen, 0.25)
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(0, 1), k.transpose(0, 1).repeat_interleave(2, 0), v.transpose(0, 1).repeat_interleave(2, 0),
                                                            attn_mask=seen, scale=0.25).transpose(0, 1)
    assert torch.allclose(out, want, rtol=1e-12, atol=1e-14) and (error > 0).all()
    none, _ = oracle.attention(q, k, v, torch.zeros(9, 12, dtype=torch.bool), 0.25)
    assert (none == 0).all()


def test_rotary_keeps_lengths_and_differences():
    g = torch.Generator().manual_seed(2)
    x, y = (torch.randn(5, 2, 8, generator=g, dtype=torch.float64) for _ in range(2))
    freq = 10000.0 ** (-torch.arange(4, dtype=torch.float64) / 4)
    at = torch.tensor([0, 1, 7, 100, 12345])
    for interleaved in (False, True):
        a, b = oracle.rotary(x, at, freq, interleaved), oracle.rotary(y, at + 3, freq, interleaved)
        assert torch.allclose(a.norm(dim=2), x.norm(dim=2), rtol=1e-12)
        c, d = oracle.rotary(x, at * 0, freq, interleaved), oracle.rotary(y, at * 0 + 3, freq, interleaved)
        assert torch.allclose((a * b).sum(dim=2), (c * d).sum(dim=2), rtol=1e-9, atol=1e-9)
        assert torch.equal(c, x)
    head = oracle.rotary(x, at, freq[:2], True)
    assert torch.equal(head[..., 4:], x[..., 4:])


def test_routing_without_groups_is_topk():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(20, 12, generator=g)
    w, ids = oracle.grouped_topk(x, 4)
    top = torch.topk(x.double(), 4, dim=1)
    assert torch.equal(ids.long(), top.indices) and torch.allclose(w, torch.softmax(top.values, dim=1))
    w, ids = oracle.grouped_topk(x, 2, 3, 1, "sigmoid", torch.zeros(12), False, 2.0)
    best = torch.sigmoid(x.double()).view(20, 3, 4).topk(2, dim=2)
    group = best.values.sum(dim=2).argmax(dim=1)
    assert torch.equal(ids // 4, group[:, None].expand(-1, 2).int())
    assert torch.allclose(w, 2.0 * best.values[torch.arange(20), group])


def test_frequencies_and_their_handle():
    from fast_route_amd import prepare_rotary, rotary_frequencies
    freq = rotary_frequencies(64)
    assert freq.dtype == torch.float64 and freq[0] == 1.0 and torch.equal(rotary_frequencies(64, scale=2.0), freq / 2)
    rotary = prepare_rotary(freq, factor=1.5)
    assert rotary.turns.dtype == torch.int64 and rotary.factor == 1.5 and not rotary.interleaved
    assert torch.allclose(rotary.turns.double() / 2.0 ** 64 * 2 * math.pi, freq, rtol=2.0 ** -52)
    for call in (lambda: rotary_frequencies(7), lambda: rotary_frequencies(8, base=0.0), lambda: rotary_frequencies(8, slow_turns=4.0, fast_turns=4.0),
                 lambda: prepare_rotary(torch.tensor([4.0])), lambda: prepare_rotary(torch.zeros(2, 2)), lambda: prepare_rotary(torch.zeros(2).half()),
                 lambda: prepare_rotary(torch.tensor([float("nan")]))):
        with pytest.raises(AssertionError):
            call()


def test_no_cpu_path():
    from fast_route_amd import attention_varlen, grouped_topk, paged_attention, prepare_rotary, rotary_embed, rotary_frequencies
    x, cu = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    cache = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: grouped_topk(torch.zeros(4, 8), 2), lambda: attention_varlen(x, x, x, cu), lambda: paged_attention(x, cache, cache, cu[None].expand(4, 2), cu[:1].expand(4)),
                 lambda: rotary_embed(x, x, torch.arange(4), prepare_rotary(rotary_frequencies(64)))):
        with pytest.raises(AssertionError, match="MI355X"):
            call()


def _rotary(**change):
    f = dict(q=16, k=16, v=16, q_out=16, k_out=16, k_cache=16, v_cache=16, positions=16, slots=0, turns=16, T=2, heads=4, kv_heads=2, dim=64, turned=64, pages=1, page_size=16,
             q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, q_out_token=256, q_out_head=64, k_out_token=128, k_out_head=64, k_cache_page=2048,
             k_cache_slot=128, k_cache_head=64, v_cache_page=2048, v_cache_slot=128, v_cache_head=64, dtype=1, interleaved=0, positions_i64=1, slots_i64=1)
    f.update(change)
    return struct.pack("@37qd", *f.values(), 1.0)


def _attention(scale=1.0, **change):
    f = dict(q=16, k=16, v=16, cu_q=16, cu_k=16, out=16, workspace=0, workspace_bytes=0, B=1, rows=4, keys=4, heads=4, kv_heads=2, dim=64, q_row=256, q_head=64, k_row=128, k_head=64,
             v_row=128, v_head=64, out_row=256, out_head=64, dtype=1, causal=1, fill=0, parts=0)
    f.update(change)
    return struct.pack("@26qdq", *f.values(), scale, 0)


def _paged(scale=1.0, **change):
    f = dict(q=16, k_cache=16, v_cache=16, table=16, lengths=16, out=16, workspace=0, workspace_bytes=0, B=2, heads=4, kv_heads=2, dim=64, pages=4, page_size=16, table_pages=2,
             table_row=2, q_row=256, q_head=64, out_row=256, out_head=64, k_cache_page=2048, k_cache_slot=128, k_cache_head=64, v_cache_page=2048, v_cache_slot=128,
             v_cache_head=64, dtype=1, slots=0, least=0, page_shift=0)
    f.update(change)
    return struct.pack("@30qdq", *f.values(), scale, 0)


def test_refusals_come_before_any_launch():
    """Codes and messages, never aborts; no call here is one that would be launched."""
    from fast_route_amd import _native
    lib = _native.lib()
    gate = lambda *a: lib.fr_gating_grouped(*a)
    good = [16, 2, 4, 64, 64, None, 8, 4, 6, 0, 1, 1.0, 16, 16, None]
    for at, value, code in ((0, None, -1), (1, 4, -3), (2, -1, -2), (3, 0, -2), (3, 1025, -2), (4, 63, -2), (6, 0, -2), (6, 7, -2), (6, 65, -2), (7, 9, -2), (7, 0, -2), (8, 0, -2), (8, 33, -2),
                            (9, 2, -2), (12, None, -1), (13, None, -1)):
        a = list(good)
        a[at] = value
        assert gate(*a) == code, (at, value)
        assert lib.fr_last_error_string()
    assert gate(None, 2, 0, 64, 64, None, 8, 4, 6, 0, 1, 1.0, None, None, None) == 0
    for change, code in ((dict(T=-1), -2), (dict(heads=0), -2), (dict(kv_heads=5000), -2), (dict(dim=0), -2), (dict(dim=1025), -2), (dict(turned=65), -2), (dict(turned=66), -2),
                         (dict(turned=-2), -2), (dict(dim=1024, turned=514), -2), (dict(dtype=2), -3), (dict(q=0), -1), (dict(k_out=0), -1), (dict(positions=0), -1), (dict(turns=0), -1),
                         (dict(slots=16, v=0), -1), (dict(slots=16, k_cache=0), -1), (dict(slots=16, page_size=0), -2), (dict(slots=16, pages=-1), -2)):
        assert lib.fr_rotary(_rotary(**change), None) == code, change
    assert lib.fr_rotary(_rotary(T=0, q=0), None) == 0 and lib.fr_rotary(None, None) == -1
    for change, code in ((dict(heads=3), -2), (dict(kv_heads=0), -2), (dict(dim=60), -2), (dict(dim=264), -2), (dict(dim=0), -2), (dict(rows=-1), -2), (dict(keys=1 << 30), -2), (dict(B=-1), -2),
                         (dict(rows=1 << 29), -2), (dict(dtype=2), -3), (dict(scale=0.0), -2), (dict(scale=-1.0), -2), (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2),
                         (dict(q=0), -1), (dict(out=0), -1), (dict(cu_k=0), -1), (dict(k=0), -1), (dict(q=8), -4), (dict(v=24), -4), (dict(k_row=132), -4), (dict(out_head=4), -4), (dict(k_row=1 << 23), -2),
                         (dict(keys=100000), -5), (dict(keys=100000, workspace=16, workspace_bytes=64), -5)):
        assert lib.fr_attention(_attention(**change), None) == code, change
    assert lib.fr_attention(_attention(rows=0, q=0), None) == 0 and lib.fr_attention(None, None) == -1
    for change, code in ((dict(heads=3), -2), (dict(kv_heads=0), -2), (dict(dim=4), -2), (dict(dim=264), -2), (dict(page_size=0), -2), (dict(table_pages=-1), -2), (dict(pages=-1), -2),
                         (dict(table_pages=1 << 27), -2), (dict(B=1 << 20, table_pages=1 << 20), -2), (dict(dtype=2), -3), (dict(scale=0.0), -2), (dict(scale=float("nan")), -2), (dict(q=0), -1),
                         (dict(lengths=0), -1), (dict(table=0), -1), (dict(k_cache=0), -1), (dict(out=8), -4), (dict(q_row=4), -4), (dict(v_cache_slot=12), -4), (dict(table_pages=4096), -5)):
        assert lib.fr_paged_attention(_paged(**change), None) == code, change
    assert lib.fr_paged_attention(_paged(B=0, q=0), None) == 0 and lib.fr_paged_attention(None, None) == -1


def test_workspace_sizes():
    """None where nothing is split, -1 outside the limits, 16 heads' rows and two sums per place otherwise; growing rows and keys never need more
    than the limits of the places."""
    from fast_route_amd import _native
    lib = _native.lib()
    paged = lib.fr_paged_attention_workspace_bytes
    assert paged(4, 8, 2, 128, 64) == 0 and paged(1024, 32, 8, 128, 512) == 0 and paged(1, 8, 3, 128, 64) == -1 and paged(1, 8, 2, 300, 64) == -1
    for B, heads, kv, dim, most in ((1, 32, 8, 128, 1024), (3, 16, 4, 64, 131072), (64, 32, 8, 128, 16384), (700, 32, 8, 128, 16384), (16, 66, 2, 256, 5000)):
        n = paged(B, heads, kv, dim, most)
        padded = 64 if dim <= 64 else 128 if dim <= 128 else 192 if dim <= 192 else 256
        plan = 0 if B <= 256 else -(-(B + 2) * 4 // 16) * 16
        assert 0 < n < 1 << 30 and (n - plan) % (16 * (padded + 2) * 4) == 0
    whole = lib.fr_attention_workspace_bytes
    assert whole(1, 16384, 16384, 32, 8, 128) == 0 and whole(1, 37, 37, 32, 8, 128) == 0 and whole(1, 37, 37, 32, 5, 128) == -1
    assert whole(1, 509, 8192, 16, 2, 64) == 8 * 509 * 16 * 66 * 4 and whole(254, 4000, 4000, 8, 2, 64) == 0 and whole(256, 4000, 4000, 8, 2, 64) == 259 * 4 + 4

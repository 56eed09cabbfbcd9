"""Results over memory that other workgroups still read, or write, are refused; results beside it are not, also where both are parts of the same rows."""
import random
import struct

import pytest
import torch


def _fields(base, change):
    assert set(change) <= set(base), change
    return {**base, **change}.values()


ROTARY = dict(q=1 << 30, k=2 << 30, v=3 << 30, q_out=4 << 30, k_out=5 << 30, k_cache=6 << 30, v_cache=7 << 30, positions=8 << 30, slots=9 << 30, turns=10 << 30, T=20, heads=4,
              kv_heads=2, dim=64, turned=64, pages=8, page_size=16, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64, q_out_token=256, q_out_head=64,
              k_out_token=128, k_out_head=64, k_cache_page=2048, k_cache_slot=128, k_cache_head=64, v_cache_page=2048, v_cache_slot=128, v_cache_head=64, dtype=1, interleaved=0,
              positions_i64=1, slots_i64=1)
ATTENTION = dict(q=1 << 30, k=2 << 30, v=3 << 30, cu_q=8 << 30, cu_k=9 << 30, out=4 << 30, workspace=0, workspace_bytes=0, B=1, rows=20, keys=20, heads=4, kv_heads=2, dim=64,
                 q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, out_row=256, out_head=64, dtype=1, causal=1, fill=0, parts=0)
PAGED = dict(q=1 << 30, k_cache=2 << 30, v_cache=3 << 30, table=8 << 30, lengths=9 << 30, out=4 << 30, workspace=0, workspace_bytes=0, B=20, heads=4, kv_heads=2, dim=64, pages=4,
             page_size=16, table_pages=2, table_row=2, q_row=256, q_head=64, out_row=256, out_head=64, k_cache_page=2048, k_cache_slot=128, k_cache_head=64, v_cache_page=2048,
             v_cache_slot=128, v_cache_head=64, dtype=1, slots=0, least=0, page_shift=0)
Q, K, V, C = ROTARY["q"], ROTARY["k"], ROTARY["v"], ROTARY["k_cache"]
INPLACE = dict(q_out=Q, k_out=K)
# every one of them would be launched but for the memory that it shares
REFUSED_ROTARY = [
    dict(INPLACE, k=Q, k_out=Q), dict(INPLACE, k=Q + 2 * 128, k_out=Q + 2 * 128), dict(INPLACE, v=K), dict(INPLACE, v=Q + 2 * 64), dict(q_out=Q, q_out_token=264),
    dict(q_out=Q + 16), dict(q_out=Q, q_out_head=128, q_out_token=512), dict(k_out=K, k_out_head=128, k_out_token=256), dict(q_out=K), dict(k_out=Q), dict(q_out=V + 2 * 128 * 19),
    dict(k_out=V), dict(k_out=ROTARY["q_out"] + 2 * 300), dict(v_cache=C), dict(v_cache=C + 2 * 2048 * 7), dict(v_cache=C - 2 * 2048 * 7), dict(k_cache=V - 64), dict(v_cache=V),
    dict(v_cache=Q), dict(k_cache=K), dict(q_out=C + 2048), dict(k_out=ROTARY["v_cache"]), dict(INPLACE, q_token=0, q_out_token=0), dict(INPLACE, k_head=0, k_out_head=0),
    dict(q_out_token=248), dict(q_out_head=32), dict(k_out_token=64), dict(k_cache_page=0), dict(k_cache_slot=0), dict(v_cache_head=8), dict(v_cache_page=2040),
    # heads of a joint row: keys begin inside the queries'
    dict(INPLACE, q_token=512, q_out_token=512, k_token=512, k_out_token=512, k=Q + 2 * 192, k_out=Q + 2 * 192)]
REFUSED_ATTENTION = [dict(out=2 << 30), dict(out=3 << 30), dict(out=(2 << 30) + 2 * 128 * 5), dict(out=(3 << 30) - 2 * 256 * 19), dict(out=(1 << 30) + 16), dict(out=(1 << 30) - 16),
                     dict(out=1 << 30, out_row=264), dict(out=1 << 30, q_row=512), dict(out_row=0), dict(out_head=0), dict(out_row=248), dict(out_head=56), dict(out=1 << 30, k=1 << 30),
                     dict(out=(1 << 30) + 2 * 64, q_row=512, out_row=512), dict(fill=1, out=2 << 30)]
REFUSED_PAGED = [dict(out=2 << 30), dict(out=3 << 30), dict(out=(2 << 30) + 2 * 2048 * 3 + 2 * 1984), dict(out=(1 << 30) + 16), dict(out=1 << 30, out_row=264), dict(out_row=0), dict(out_head=0),
                 dict(out_row=200), dict(out=(1 << 30) + 2 * 64, q_row=512, out_row=512), dict(out=1 << 30, out_head=64, q_head=72, q_row=288, out_row=288)]


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="addresses that there are not: where nothing can be launched")
def test_refused():
    """Every call ends at the check."""
    from fast_route_amd import _native
    lib = _native.lib()
    for entry, base, pack, refused in (
            (lib.fr_rotary, ROTARY, lambda f: struct.pack("@37qd", *f, 1.0), REFUSED_ROTARY), (lib.fr_attention, ATTENTION, lambda f: struct.pack("@26qdq", *f, 1.0, 0), REFUSED_ATTENTION),
            (lib.fr_paged_attention, PAGED, lambda f: struct.pack("@30qdq", *f, 1.0, 0), REFUSED_PAGED)):
        for change in refused:
            assert entry(pack(_fields(base, change)), None) == -2 and b"memory" in lib.fr_last_error_string(), (change, lib.fr_last_error_string())


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="addresses that there are not: where nothing can be launched")
def test_layouts_of_all_kinds():
    """Small arrays of any strides in and near each other: refused where an element of a result is met twice, or in what is read, launched (which fails here) where not."""
    from fast_route_amd import _native
    lib, rng, seen = _native.lib(), random.Random(5), {-2: 0, -6: 0}

    def elements(at, T, token, heads, head, dim):
        return [at + 2 * (t * token + h * head + d) + b for t in range(T) for h in range(heads) for d in range(dim) for b in range(2)]
    for _ in range(6000):
        T, heads, kv, dim = (rng.randint(1, 4) for _ in range(4))
        f = dict(ROTARY, slots=0, v=0, k_cache=0, v_cache=0, T=T, heads=heads, kv_heads=kv, dim=dim, turned=0, turns=0)
        names, base = ("q", "k", "q_out", "k_out"), 1 << 20
        joint = rng.choice((None, rng.randint(1, 40)))
        for n in names:
            f[n] = base + rng.choice((0, 2, 1)) * rng.randint(0, 60)
            f[n + "_token"] = joint if joint and rng.random() < 0.8 else rng.choice((dim * heads, rng.randint(-12, 40), dim))
            f[n + "_head"] = rng.choice((dim, dim, rng.randint(-6, 20), T * dim))
        for n in "qk":
            if rng.random() < 0.4:
                f[n + "_out"], f[n + "_out_token"], f[n + "_out_head"] = f[n], f[n + "_token"], f[n + "_head"]
        if rng.random() < 0.5:  # apart, but for one pair
            for i, n in enumerate(rng.sample(names, 3)):
                f[n] += (i + 1) << 12
        held = {n: elements(f[n], T, f[n + "_token"], heads if n[0] == "q" else kv, f[n + "_head"], dim) for n in names}
        same = {n: all(f[n + s] == f[n + "_out" + s] for s, c in (("", 2), ("_token", T), ("_head", heads if n == "q" else kv)) if c > 1) for n in "qk"}
        bad = any(len(set(held[n])) < len(held[n]) for n in ("q_out", "k_out")) or bool(set(held["q_out"]) & set(held["k_out"]))
        for n in "qk":
            bad = bad or any(not (n == m and same[n]) and set(held[n + "_out"]) & set(held[m]) for m in "qk")
        rc = lib.fr_rotary(struct.pack("@37qd", *f.values(), 1.0), None)
        assert rc == (-2 if bad else -6), (rc, bad, {k: f[k] for k in f if k[0] in "qk" or k in ("T", "heads", "dim")})
        seen[rc] += 1
    assert min(seen.values()) > 1000, seen


def _joint(heads, T=9, D=64, order="heads"):
    """Parts of `heads` heads each of joint rows, one after the other ("heads") or head by head in turn ("turns")."""
    if order == "heads":
        x = torch.randn(T, sum(heads), D, generator=torch.Generator().manual_seed(1)).half().cuda()
        return x, x.split(heads, dim=1)
    x = torch.randn(T, heads[0], len(heads), D, generator=torch.Generator().manual_seed(1)).half().cuda()
    return x, x.unbind(2)


@pytest.mark.gpu
def test_shared_memory_through_the_package(native):
    from fast_route_amd import attention_varlen, paged_attention, prepare_rotary, rotary_embed, rotary_frequencies, rotary_to_cache
    print("[case] refused", flush=True)
    rotary, T = prepare_rotary(rotary_frequencies(64), device="cuda"), 9
    at, slots = torch.arange(T).cuda(), torch.arange(T).cuda()
    x, (q, k, v) = _joint((8, 2, 2))
    before = x.clone()
    kc, vc = (torch.zeros(2, 16, 2, 64, dtype=torch.half, device="cuda") for _ in range(2))
    cu = torch.tensor([0, T], dtype=torch.int32).cuda()
    n, table = torch.full((T,), 5, dtype=torch.int32).cuda(), torch.zeros(T, 1, dtype=torch.int32).cuda()
    compact = x.view(-1)[:T * 8 * 64].view(T, 8, 64)  # over the joint rows, with strides of its own
    calls = [lambda: rotary_embed(x[:, :8], x[:, 6:8], at, rotary, inplace=True), lambda: rotary_embed(x[:, :8], x[:, 7:], at, rotary, inplace=True),
             lambda: rotary_to_cache(q, k, k, at, rotary, kc, vc, slots, inplace=True), lambda: rotary_to_cache(q, k, q[:, :2], at, rotary, kc, vc, slots, inplace=True),
             lambda: rotary_to_cache(q, k, v, at, rotary, kc, kc, slots), lambda: rotary_to_cache(q, k, vc.view(-1, 2, 64)[:T], at, rotary, kc, vc, slots),
             lambda: rotary_to_cache(q, kc.view(-1, 2, 64)[:T], v, at, rotary, kc, vc, slots), lambda: rotary_embed(q[:1].expand(T, 8, 64), k, at, rotary, inplace=True),
             lambda: attention_varlen(q, k, v, cu, out=compact), lambda: attention_varlen(q, k, v, cu, out=x[:, 1:9]), lambda: attention_varlen(q, k, v, cu, out=x[:, 4:]),
             lambda: attention_varlen(q, k, v, cu, out=torch.zeros(T * 8 * 64, device="cuda").half().as_strided((T, 8, 64), (256, 64, 1))),
             lambda: paged_attention(q, kc, vc, table, n, out=compact), lambda: paged_attention(q, kc, vc, table, n, out=x[:, 1:9]),
             lambda: paged_attention(q[:4], kc, vc, table[:4], n[:4], out=kc.view(4, 16, 64)[:, :8])]
    for i, call in enumerate(calls):
        with pytest.raises(AssertionError, match="memory"):
            call()
            print("call %d was taken" % i)
    torch.cuda.synchronize()
    assert torch.equal(x, before) and (kc == 0).all() and (vc == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["heads", "turns"])
def test_parts_of_joint_rows_are_taken(native, order):
    """Results into the queries' own place, or beside queries, keys and values in the same rows; caches that are parts of one tensor."""
    from fast_route_amd import attention_varlen, paged_attention, prepare_rotary, rotary_embed, rotary_frequencies, rotary_to_cache
    print("[case] taken", order, flush=True)
    rotary, T = prepare_rotary(rotary_frequencies(64), device="cuda"), 9
    at, slots, cu = torch.arange(T).cuda(), torch.arange(T).cuda() * 3 - 3, torch.tensor([0, T], dtype=torch.int32).cuda()
    n, table = torch.tensor([5, 16, 17, 1, 0, 24, 30, 32, 8], dtype=torch.int32).cuda(), torch.tensor([[1, 0]] * T, dtype=torch.int32).cuda()
    heads = (8, 2, 2, 8) if order == "heads" else (4, 4, 4, 4)
    G = heads[1]
    _, (q, k, v, _) = _joint(heads, order=order)
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    want_q, want_k = rotary_embed(q0, k0, at, rotary)
    want = attention_varlen(want_q, want_k, v0, cu)
    caches = [torch.zeros(2, 16, G, 64, dtype=torch.half, device="cuda") for _ in range(2)]
    rotary_to_cache(q0, k0, v0, at, rotary, *caches, slots)
    want_paged = paged_attention(want_q, *caches, table, n)
    for dim in (0, 1, 2, 3):  # where keys and values lie beside each other in a tensor of both
        _, (q, k, v, out) = _joint(heads, order=order)
        shape = [2, 16, G, 64]
        shape.insert(dim, 2)
        kc, vc = torch.zeros(shape, dtype=torch.half, device="cuda").unbind(dim)
        got = rotary_to_cache(q, k, v, at, rotary, kc, vc, slots, inplace=True)
        assert got[0].data_ptr() == q.data_ptr() and torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(v, v0)
        assert torch.equal(kc, caches[0]) and torch.equal(vc, caches[1])
        attention_varlen(q, k, v, cu, out=out)
        assert torch.equal(out, want) and torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(v, v0)
        paged_attention(q, kc, vc, table, n, out=out)
        assert torch.equal(out, want_paged)
        paged_attention(q, kc, vc, table, n, out=q)
        assert torch.equal(q, want_paged)
        q.copy_(want_q)
        attention_varlen(q, k, v, cu, out=q)
        assert torch.equal(q, want) and torch.equal(k, want_k) and torch.equal(v, v0)
    rotary_to_cache(q0, k0, k0, at, rotary, *caches, slots)  # read twice, written nowhere
    one = want_q[:1, :1]
    out = torch.zeros(1, 1, 64, dtype=torch.half, device="cuda").as_strided((1, 1, 64), (0, 0, 1))  # strides of a single row and head mean nothing
    attention_varlen(one, want_k[:, :1], v0[:, :1], cu[:2] // T, cu, out=out)
    assert torch.isfinite(out).all() and (out != 0).any()

"""attention_varlen and paged_attention against their definition in 64 bits (oracle/serving_oracle.py)."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")


def _say(msg):
    print("[case] " + msg, flush=True)


def _close(got, ref, error, where=""):
    """`error` and the result's own rounding (half a step; subnormal ones' too)."""
    info = torch.finfo(got.dtype)
    tol = error + info.eps / 2 * (ref.abs() + error) + info.tiny * info.eps
    off = (got.cpu().double() - ref).abs()
    assert not (off > tol).any() and not got.isnan().any(), "%s worst %g of the bound" % (where, (off / tol).max().item())


def _seen(n, m, causal):
    i, j = torch.arange(n)[:, None], torch.arange(m)[None, :]
    return j <= i + (m - n) if causal else torch.ones(n, m, dtype=torch.bool)


def _cu(lengths, first=0):
    return torch.tensor([first] + list(lengths)).cumsum(0).to(torch.int32)


def _packed(lengths, keys, H, G, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return tuple((torch.randn(n, h, D, generator=g) * std).to(dtype) for n, h in ((sum(lengths), H), (sum(keys), G), (sum(keys), G)))


def _want(q, k, v, lengths, keys, causal, scale):
    out, error, r, c = [], [], 0, 0
    for n, m in zip(lengths, keys):
        o, e = oracle.attention(q[r:r + n], k[c:c + m], v[c:c + m], _seen(n, m, causal), scale)
        out.append(o), error.append(e)
        r, c = r + n, c + m
    return torch.cat(out), torch.cat(error)


PACKED = [([1], [1], 1, 1, 8), ([37], [37], 8, 2, 128), ([1, 2, 3, 64, 65], None, 4, 4, 64), ([128, 0, 5], None, 2, 1, 128), ([33, 7], [200, 7], 6, 2, 80),
          ([5, 40], [3, 10], 4, 2, 64), ([3], [700], 16, 1, 128), ([130], None, 3, 1, 96), ([70, 20], [90, 64], 4, 2, 192), ([66], [130], 2, 2, 256),
          ([10, 0, 0, 9], [0, 4, 0, 9], 2, 2, 24), ([300], None, 1, 1, 64), ([17] * 70, None, 2, 1, 64)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,keys,H,G,D", PACKED)
def test_packed(native, lengths, keys, H, G, D, causal):
    from fast_route_amd import attention_varlen
    for dtype in TYPES:
        _say(f"packed {lengths[:5]} {keys} H={H} G={G} D={D} {causal} {dtype}")
        m = keys or lengths
        q, k, v = _packed(lengths, m, H, G, D, dtype, sum(lengths) + D)
        got = attention_varlen(q.cuda(), k.cuda(), v.cuda(), _cu(lengths).cuda(), None if keys is None else _cu(m).cuda(), causal)
        _close(got, *_want(q, k, v, lengths, m, causal, D ** -0.5))


def test_large_scores_and_other_scales(native):
    """Scores of several hundreds, rising and falling along the keys, so that the maximum moves late."""
    from fast_route_amd import attention_varlen
    _say("large scores")
    for dtype in TYPES:
        for scale, std in ((0.5, 3.0), (0.01, 1.0), (4.0, 0.5)):
            q, k, v = _packed([150], [150], 2, 1, 64, dtype, 4, std)
            ramp = torch.linspace(0.1, 2.0, 150)[:, None, None]
            for kk in (k * ramp, k * ramp.flip(0)):
                kk = kk.to(dtype)
                got = attention_varlen(q.cuda(), kk.cuda(), v.cuda(), _cu([150]).cuda(), causal=True, scale=scale)
                _close(got, *_want(q, kk, v, [150], [150], True, scale))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_what_a_row_does_not_see_does_not_reach_it(native, bad, D):
    """Values and keys that are not finite: behind the sequences, in other sequences, behind a row of the same sequence."""
    from fast_route_amd import attention_varlen
    _say(f"bad {bad} D={D}")
    lengths, H, G = [75, 40, 90], 4, 2
    q, k, v = _packed(lengths, lengths, H, G, D, torch.bfloat16, 9)
    ref, error = _want(q, k, v, lengths, lengths, True, D ** -0.5)
    k2, v2 = torch.cat([k, torch.full_like(k[:50], bad)]), torch.cat([v, torch.full_like(v[:50], bad)])
    k2[75 + 30], v2[75 + 30] = bad, bad  # key 30 of the second sequence
    v2[115 + 70, :, 5] = bad  # one value of key 70 of the third
    got = attention_varlen(q.cuda(), k2.cuda(), v2.cuda(), _cu(lengths).cuda(), _cu(lengths).cuda()).cpu()
    clean = torch.ones(sum(lengths), dtype=torch.bool)
    clean[75 + 30:115] = False
    clean[115 + 70:] = False
    _close(got[clean], ref[clean], error[clean])
    assert not got[75 + 30:115].isfinite().all(dim=2).any()
    other = torch.arange(D) != 5
    _close(got[115 + 70:][:, :, other], ref[115 + 70:][:, :, other], error[115 + 70:][:, :, other])
    assert not got[115 + 70:, :, 5].isfinite().any()


def test_rows_without_keys_and_rows_behind(native):
    from fast_route_amd import attention_varlen
    _say("rows without keys")
    q, k, v = _packed([60], [60], 4, 2, 64, torch.bfloat16, 1)
    cu_q, cu_k = _cu([20, 20], 3).cuda(), _cu([5, 0], 2).cuda()
    ref, error = _want(q[3:43], k[2:7], v[2:7], [20, 20], [5, 0], True, 0.125)
    got = attention_varlen(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k)
    _close(got[3:43], ref, error)
    assert (got[3:18] == 0).all() and (got[23:43] == 0).all() and (got[43:] == 0).all()
    out = torch.full_like(q, 5.0).cuda()
    assert attention_varlen(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k, out=out) is out
    assert torch.equal(out[3:43], got[3:43]) and (out[:3] == 5).all() and (out[43:] == 5).all()
    held = q.cuda()
    attention_varlen(held, k.cuda(), v.cuda(), cu_q, cu_k, out=held)  # in place
    assert torch.equal(held[3:43], got[3:43]) and torch.equal(held[43:].cpu(), q[43:])
    none = attention_varlen(q.cuda(), k[:0].cuda(), v[:0].cuda(), cu_q, torch.zeros(3, dtype=torch.int32, device="cuda"), causal=False)
    assert (none[3:] == 0).all()
    assert attention_varlen(q[:0].cuda(), k.cuda(), v.cuda(), cu_q, cu_k).shape == (0, 4, 64)
    assert (attention_varlen(q.cuda(), k.cuda(), v.cuda(), cu_q[:1], cu_k[:1])[3:] == 0).all()


def test_cumulative_lengths_outside_the_rows(native):
    """Taken inside the rows and keys there are: nothing else is read or written."""
    from fast_route_amd import attention_varlen
    _say("cumulative lengths outside")
    q, k, v = (t.cuda() for t in _packed([50], [50], 2, 1, 64, torch.bfloat16, 2))
    want = attention_varlen(q, k, v, _cu([50]).cuda())
    assert torch.equal(attention_varlen(q, k, v, torch.tensor([-7, 1000], dtype=torch.int32, device="cuda")), want)
    guard = torch.full((60, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    out = guard[5:55]
    for wrong in ([0, 50, 20], [90, 120, 300], [-30, -20, 25], [0, 50, 0, 50, 0, 50, 0, 50]):
        attention_varlen(q, k, v, torch.tensor(wrong, dtype=torch.int32, device="cuda"), out=out)
        torch.cuda.synchronize()
        assert (guard[:5] == 5).all() and (guard[55:] == 5).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_parts_of_a_joint_projection(native, dtype):
    """Strides as they come: heads within a token's row, heads first, and results into such places."""
    from fast_route_amd import attention_varlen
    _say("strides")
    n, H, G, D = 77, 8, 2, 128
    qkv = torch.randn(n, H + 2 * G, D, generator=torch.Generator().manual_seed(3)).to(dtype)
    ref, error = _want(qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], [50, 27], [50, 27], True, D ** -0.5)
    held = qkv.cuda()
    q, k, v = held[:, :H], held[:, H:H + G], held[:, H + G:]
    got = attention_varlen(q, k, v, _cu([50, 27]).cuda())
    _close(got, ref, error)
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    out = torch.zeros(n, H + 1, D, dtype=dtype, device="cuda")
    attention_varlen(*swapped, _cu([50, 27]).cuda(), out=out[:, 1:])
    assert torch.equal(out[:, 1:], got) and (out[:, 0] == 0).all()
    shared = attention_varlen(q, k[:, :1].expand(n, G, D), v[:, :1].expand(n, G, D), _cu([50, 27]).cuda())
    assert torch.equal(shared, attention_varlen(q, k[:, :1], v[:, :1], _cu([50, 27]).cuda()))


@pytest.mark.parametrize("causal", [True, False])
def test_keys_split_along_their_length(native, causal):
    """Few rows over many keys: parts that are joined, values that are not finite among the last ones, rows behind the sequences, a workspace's end."""
    from fast_route_amd import attention_varlen
    for lengths, keys, H, G, D in (([40], [3000], 8, 2, 128), ([3, 0, 9], [1500, 20, 2900], 4, 1, 64), ([1], [5000], 28, 4, 96), ([20], [2000], 2, 2, 256)):
        _say(f"split {lengths} {keys} {causal}")
        q, k, v = _packed(lengths, keys, H, G, D, torch.bfloat16, sum(keys))
        ref, error = _want(q, k, v, lengths, keys, causal, D ** -0.5)
        rows = torch.cat([q, q[:2]])
        need = native.fr_attention_workspace_bytes(len(lengths), len(rows), sum(keys), H, G, D)
        assert need > 0
        guard = torch.full((need + 256,), 0xA5, dtype=torch.uint8, device="cuda")
        args = rows.cuda(), k.cuda(), v.cuda(), _cu(lengths).cuda(), _cu(keys).cuda()
        got = attention_varlen(*args, causal=causal, workspace_buf=guard[:need])
        _close(got[:len(q)], ref, error)
        assert (got[len(q):] == 0).all() and (guard[need:] == 0xA5).all()
        out = torch.full_like(args[0], 5.0)
        attention_varlen(*args, causal=causal, out=out)
        assert torch.equal(out[:len(q)], got[:len(q)]) and (out[len(q):] == 5).all()
        with pytest.raises(AssertionError):
            attention_varlen(*args, causal=causal, workspace_buf=guard[:need - 1])
        if causal and lengths[-1] > 1:
            bad = v.clone()
            bad[-1] = NAN  # the last row alone sees it
            got = attention_varlen(args[0][:len(q)], args[1], bad.cuda(), *args[3:])
            _close(got[:-1], ref[:-1], error[:-1])
            assert got[-1].isnan().all()


@pytest.mark.parametrize("count", [65, 300, 1100])
def test_many_sequences(native, count):
    """More sequences than a wavefront holds the lengths of."""
    from fast_route_amd import attention_varlen, paged_attention
    _say(f"{count} sequences")
    g = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 9, (count,), generator=g).tolist()
    lengths[count // 2], lengths[-1] = 150, 70
    q, k, v = _packed(lengths, lengths, 2, 1, 64, torch.bfloat16, count)
    ref, error = _want(q, k, v, lengths, lengths, True, 0.125)
    _close(attention_varlen(q.cuda(), k.cuda(), v.cuda(), _cu(lengths).cuda()), ref, error)
    lengths[3] = 1300
    for page in (16, 6):
        q, kc, vc, table, n = _paged(lengths, 2, 1, 64, page, torch.bfloat16, count)
        _close(paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda()), *_want_paged(q, kc, vc, table, n, 0.125))


def test_long_prompt_and_chunks_of_it(native):
    """A prompt of several thousand rows against fp32 on the GPU, and the same one in chunks with the keys in front of them."""
    from fast_route_amd import attention_varlen
    for dtype, D, H, G in ((torch.bfloat16, 128, 8, 2), (torch.float16, 64, 4, 4)):
        _say(f"long prompt {dtype} {D}")
        n = 4099
        q, k, v = (t.cuda() for t in _packed([n], [n], H, G, D, dtype, 11))
        got = attention_varlen(q, k, v, _cu([n]).cuda())
        u = torch.finfo(dtype).eps / 2
        mask = ~_seen(n, n, True).cuda()
        for h in range(H):
            p = (q[:, h].double() @ k[:, h // (H // G)].double().t() * D ** -0.5).masked_fill_(mask, -INF)
            p = torch.softmax(p, dim=1)
            vh = v[:, h // (H // G)].double()
            # 2^-13 for 32-bit sums: scores' 2 * 2^-23 * 12 * 64, terms' 2^-22 * (n / 16 + 4)
            tol = p @ vh.abs() * (u + 2.0 ** -13) * (1 + u) + u * (p @ vh).abs()
            assert ((got[:, h].double() - p @ vh).abs() <= tol).all()
        r = 0
        for c in (1, 63, 64, 700, 129, n - 957):
            part = attention_varlen(q[r:r + c], k[:r + c], v[:r + c], _cu([c]).cuda(), _cu([r + c]).cuda())
            assert torch.allclose(part.double(), got[r:r + c].double(), rtol=4 * u, atol=16 * u)
            r += c


# ---- pages --------------------------------------------------------------------------------------------------

def _paged(lengths, H, G, D, page, dtype, seed, spare=2, std=1.0):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(counts + [1]) + 1), -5, dtype=torch.int32)  # behind a length: not looked at
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    kc, vc = ((torch.randn(pages, page, G, D, generator=g) * std).to(dtype) for _ in range(2))
    q = torch.randn(len(lengths), H, D, generator=g).to(dtype)
    return q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32)


def _want_paged(q, kc, vc, table, lengths, scale):
    page, out, error = kc.shape[1], [], []
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(max(n, 0))
        where = table[b].long()[at // page]
        there = (where >= 0) & (where < kc.shape[0])
        where = where.clamp(0, kc.shape[0] - 1)
        o, e = oracle.attention(q[b:b + 1], kc[where, at % page], vc[where, at % page], there[None, :], scale)
        out.append(o), error.append(e)
    return torch.cat(out), torch.cat(error)


PAGED = [([1], 1, 1, 8, 16), ([0, 1, 2, 127, 128, 129], 8, 2, 128, 16), ([1000], 32, 8, 128, 64), ([33, 260, 5], 6, 6, 64, 32), ([70, 300], 28, 4, 80, 128), ([515, 16], 16, 1, 64, 48),
         ([400, 31], 40, 2, 128, 16), ([299], 4, 2, 192, 16), ([140, 90], 8, 2, 256, 32), ([77, 200], 4, 2, 128, 1), ([50, 130], 8, 2, 64, 5), ([600, 3], 8, 4, 96, 24),
         ([9] * 130, 2, 1, 64, 16), ([3000, 0, 40], 12, 4, 64, 256), ([100], 66, 2, 64, 8)]


@pytest.mark.parametrize("lengths,H,G,D,page", PAGED)
def test_paged(native, lengths, H, G, D, page):
    from fast_route_amd import paged_attention
    for dtype in TYPES:
        _say(f"paged {lengths[:6]} H={H} G={G} D={D} page={page} {dtype}")
        q, kc, vc, table, n = _paged(lengths, H, G, D, page, dtype, sum(lengths) + D)
        got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda())
        _close(got, *_want_paged(q, kc, vc, table, n, D ** -0.5))


def test_paged_large_scores(native):
    from fast_route_amd import paged_attention
    _say("paged large scores")
    for dtype in TYPES:
        for scale, std in ((1.0, 3.0), (0.01, 1.0)):
            q, kc, vc, table, n = _paged([700, 90], 8, 2, 64, 16, dtype, 6, std=std)
            got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(), scale=scale)
            _close(got, *_want_paged(q, kc, vc, table, n, scale))


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("page", [16, 6])
def test_pages_that_end_inside_a_run(native, page, bad):
    """What lies behind a length, in its last page and in others, is not read; nor are pages behind it."""
    from fast_route_amd import paged_attention
    _say(f"stale pages {page}")
    lengths = [5, 37, 130, 250]
    q, kc, vc, table, n = _paged(lengths, 8, 2, 128, page, torch.bfloat16, 4)
    ref, error = _want_paged(q, kc, vc, table, n, 128 ** -0.5)
    used = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b, m in enumerate(lengths):
        at = torch.arange(m)
        used[table[b].long()[at // page], at % page] = True
    kc[~used], vc[~used] = bad, bad
    _close(paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda()), ref, error)


@pytest.mark.parametrize("page", [16, 64, 7])
def test_pages_and_lengths_that_there_are_not(native, page):
    """Keys in pages outside the cache take no part; lengths are taken inside the table.  The kernel compares page numbers before it forms an address."""
    from fast_route_amd import paged_attention
    _say(f"bad pages {page}")
    lengths = [300, 200, 150, 40]
    q, kc, vc, table, n = _paged(lengths, 4, 2, 64, page, torch.bfloat16, 8)
    table[0, 1], table[1, 0], table[2, 2] = -1, kc.shape[0], 2 ** 31 - 1
    table[3] = -(2 ** 31)  # no key at all
    ref, error = _want_paged(q, kc, vc, table, n, 0.125)
    got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda())
    _close(got, ref, error)
    assert (got[3] == 0).all()
    good = table.clone()
    good[:] = torch.arange(table.shape[1], dtype=torch.int32) % kc.shape[0]
    most = table.shape[1] * page
    got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), good.cuda(), torch.tensor([2 ** 31 - 1, most, -1, -(2 ** 31)], dtype=torch.int32).cuda())
    ref, error = _want_paged(q, kc, vc, good, torch.tensor([most, most, 0, 0]), 0.125)
    _close(got, ref, error)
    empty = paged_attention(q.cuda(), kc[:0].cuda(), vc[:0].cuda(), good.cuda(), n.cuda())
    assert (empty == 0).all()
    assert (paged_attention(q.cuda(), kc.cuda(), vc.cuda(), good[:, :0].cuda(), n.cuda()) == 0).all()


def test_paged_strides_outputs_and_shared_pages(native):
    from fast_route_amd import paged_attention
    _say("paged strides")
    q, kc, vc, table, n = (t.cuda() for t in _paged([500, 77, 260], 8, 2, 64, 16, torch.float16, 12))
    want = paged_attention(q, kc, vc, table, n)
    heads_first = [c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc)]
    both = torch.stack([kc, vc], dim=1)  # keys and values of a page together
    out = torch.full((3, 9, 64), 5.0, dtype=torch.float16, device="cuda")
    wide = torch.cat([table, table], dim=1)[:, : table.shape[1]]
    rows = torch.cat([q, q], dim=1)[:, :8]
    assert torch.equal(paged_attention(rows, *heads_first, wide, n, out=out[:, 1:]), want)
    assert torch.equal(out[:, 1:], want) and (out[:, 0] == 5).all()
    assert torch.equal(paged_attention(q, both[:, 0], both[:, 1], table, n), want)
    same = paged_attention(q, kc, vc, table[:1].expand(3, -1), n[:1].expand(3).contiguous())  # one prefix for all
    assert torch.equal(same[0], want[0]) or torch.allclose(same[0].float(), want[0].float(), rtol=2 ** -9, atol=2 ** -9)
    held = q.clone()
    assert torch.equal(paged_attention(held, kc, vc, table, n, out=held), want)


def test_paged_workspace(native):
    from fast_route_amd import paged_attention
    _say("paged workspace")
    q, kc, vc, table, n = (t.cuda() for t in _paged([900, 1300], 8, 2, 64, 16, torch.bfloat16, 13))
    need = native.fr_paged_attention_workspace_bytes(2, 8, 2, 64, table.shape[1] * 16)
    assert need > 0
    guard = torch.full((need + 256,), 0xA5, dtype=torch.uint8, device="cuda")
    want = paged_attention(q, kc, vc, table, n)
    assert torch.equal(paged_attention(q, kc, vc, table, n, workspace_buf=guard[:need]), want)
    assert (guard[need:] == 0xA5).all()
    with pytest.raises(AssertionError):
        paged_attention(q, kc, vc, table, n, workspace_buf=guard[:need - 1])


def test_long_cache(native):
    """More than 2^31 elements: pages at its end."""
    from fast_route_amd import paged_attention
    _say("long cache")
    G, D, page = 8, 128, 64
    pages = (2 ** 31) // (page * G * D) + 40
    g = torch.Generator(device="cuda").manual_seed(1)
    kc = torch.empty(pages, page, G, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    table = torch.tensor([[pages - 1, 0, pages - 2, pages - 33, 1]], dtype=torch.int32)
    for p in table[0].tolist():
        kc[p].normal_(generator=g), vc[p].normal_(generator=g)
    q, n = torch.randn(1, 16, D, generator=torch.Generator().manual_seed(2)).bfloat16(), torch.tensor([5 * page - 3], dtype=torch.int32)
    got = paged_attention(q.cuda(), kc, vc, table.cuda(), n.cuda())
    near_k, near_v = kc[table[0].long()].cpu(), vc[table[0].long()].cpu()
    _close(got, *_want_paged(q, near_k, near_v, torch.arange(5, dtype=torch.int32)[None], n, D ** -0.5))


def test_captured_and_replayed(native):
    """Both attentions in one graph, lengths changing between replays, against eager calls."""
    from fast_route_amd import attention_varlen, paged_attention
    _say("graph")
    q, kc, vc, table, n = (t.cuda() for t in _paged([700, 300, 90], 8, 2, 64, 16, torch.bfloat16, 14))
    table = table.clamp(min=0)
    pq, pk, pv = (t.cuda() for t in _packed([200], [200], 8, 2, 64, torch.bfloat16, 15))
    cu = _cu([60, 100]).cuda()

    def step():
        return paged_attention(q, kc, vc, table, n), attention_varlen(pq, pk, pv, cu)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i, (lengths, parts) in enumerate((([700, 300, 90], [60, 100]), ([1, 0, 700], [200, 0]), ([701, 500, 64], [1, 7]), ([16, 16, 16], [150, 50]))):
        n.copy_(torch.tensor(lengths)), cu.copy_(_cu(parts))
        pq.normal_(generator=torch.Generator(device="cuda").manual_seed(i))
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager)), i


def test_two_streams_at_once(native):
    from fast_route_amd import attention_varlen, paged_attention
    _say("streams")
    calls = []
    for seed in (16, 17):
        paged = [t.cuda() for t in _paged([900 + seed, 40], 8, 2, 128, 16, torch.bfloat16, seed)]
        packed = [t.cuda() for t in _packed([300 + seed], [300 + seed], 8, 2, 128, torch.bfloat16, seed)] + [_cu([300 + seed]).cuda()]
        calls.append((paged, packed))
    want = [(paged_attention(*a), attention_varlen(*b)) for a, b in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((paged_attention(*calls[i][0]), attention_varlen(*calls[i][1])))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for pair in got[i] for a, b in zip(pair, want[i]))


def test_refusals(native):
    from fast_route_amd import attention_varlen, paged_attention
    _say("refusals")
    q, k, v = (t.cuda() for t in _packed([20], [20], 4, 2, 64, torch.bfloat16, 1))
    cu = _cu([20]).cuda()
    odd = torch.zeros(20 * 2 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(20, 2, 64)
    calls = [lambda: attention_varlen(q.cpu(), k, v, cu), lambda: attention_varlen(q.float(), k, v, cu), lambda: attention_varlen(q, k.half(), v, cu),
             lambda: attention_varlen(q, k[:10], v, cu), lambda: attention_varlen(q[:, :3], k, v, cu), lambda: attention_varlen(q, k, v, cu.long()),
             lambda: attention_varlen(q, k, v, cu.cpu()), lambda: attention_varlen(q, k, v, cu, cu[:1]), lambda: attention_varlen(q, odd, v, cu),
             lambda: attention_varlen(q[..., :60], k[..., :60], v[..., :60], cu), lambda: attention_varlen(q[..., ::2], k[..., ::2], v[..., ::2], cu),
             lambda: attention_varlen(q, k, v, cu, scale=0.0), lambda: attention_varlen(q, k, v, cu, scale=-1.0), lambda: attention_varlen(q, k, v, cu, scale=NAN),
             lambda: attention_varlen(q, k, v, cu, out=q[:10]), lambda: attention_varlen(q, k, v, cu, out=torch.empty_like(q, dtype=torch.float16)),
             lambda: attention_varlen(q, k, v, cu[:0])]
    big = torch.zeros(4, 2, 264, dtype=torch.bfloat16, device="cuda")
    calls += [lambda: attention_varlen(big, big, big, cu)]
    pq, kc, vc, table, n = (t.cuda() for t in _paged([40, 20], 4, 2, 64, 16, torch.bfloat16, 1))
    calls += [lambda: paged_attention(pq.cpu(), kc, vc, table, n), lambda: paged_attention(pq, kc.half(), vc, table, n), lambda: paged_attention(pq, kc, vc[:2], table, n),
              lambda: paged_attention(pq[:, :3], kc, vc, table, n), lambda: paged_attention(pq, kc, vc, table.long(), n), lambda: paged_attention(pq, kc, vc, table[:1], n),
              lambda: paged_attention(pq, kc, vc, table, n.long()), lambda: paged_attention(pq, kc, vc, table, n[:1]), lambda: paged_attention(pq, kc, vc, table.t().contiguous().t(), n),
              lambda: paged_attention(pq, kc, vc, table, n, scale=0.0), lambda: paged_attention(pq[..., :60], kc[..., :60], vc[..., :60], table, n),
              lambda: paged_attention(pq, kc, vc, table, n, out=pq.half()), lambda: paged_attention(pq, kc, vc, table.cpu(), n),
              lambda: paged_attention(pq, kc, vc, table, n, workspace_buf=torch.empty(1 << 20, device="cuda"))]
    for i, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
            print("call %d was taken" % i)

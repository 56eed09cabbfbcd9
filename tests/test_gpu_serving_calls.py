"""The attention, rotary and routing operators called in other ways than one after the other: replayed from graphs that share a workspace, on two
streams, over more sequences than a wavefront's lanes hold, over rows far apart."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu


def _say(msg):
    print("[case] " + msg, flush=True)


def _cu(lengths, first=0):
    return torch.tensor([first] + list(lengths)).cumsum(0).to(torch.int32)


def _close(got, ref, error):
    """`error` and the result's own rounding (half a step; subnormal ones' too)."""
    info = torch.finfo(got.dtype)
    tol = error + info.eps / 2 * (ref.abs() + error) + info.tiny * info.eps
    off = (got.cpu().double() - ref).abs()
    assert not (off > tol).any() and not got.isnan().any(), "worst %g of the bound" % (off / tol).max().item()


def _seen(n, m):
    return torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n)


def _pool(rows, pages, page, G, D, H, seed, each):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(rows, H, D, generator=g).bfloat16()
    kc, vc = (torch.randn(pages, page, G, D, generator=g).bfloat16() for _ in range(2))
    return q, kc, vc, torch.randint(0, pages, (rows, each), generator=g).to(torch.int32)


@pytest.mark.parametrize("count", [1, 3, 253, 254, 255, 256, 257, 700])
def test_rows_of_no_sequence(native, count):
    """In front of the first sequence and behind the last: zeros in a new result, as they were in the caller's."""
    from fast_route_amd import attention_varlen
    _say(f"outside {count}")
    g = torch.Generator().manual_seed(count)
    lengths, front, behind = torch.randint(0, 6, (count,), generator=g).tolist(), 150, 70
    n = sum(lengths)
    q = torch.randn(front + n + behind, 4, 64, generator=g).bfloat16()
    k, v = (torch.randn(5 + n, 2, 64, generator=g).bfloat16() for _ in range(2))
    refs, r = [], 0
    for l in lengths:
        refs.append(oracle.attention(q[front + r:front + r + l], k[5 + r:5 + r + l], v[5 + r:5 + r + l], _seen(l, l), 0.125))
        r += l
    ref, error = torch.cat([x[0] for x in refs]), torch.cat([x[1] for x in refs])
    call = q.cuda(), k.cuda(), v.cuda(), _cu(lengths, front).cuda(), _cu(lengths, 5).cuda()
    junk = torch.full((1 << 22,), 0xA5, dtype=torch.uint8, device="cuda")
    del junk  # what a new result's memory holds, most likely
    got = attention_varlen(*call)
    _close(got[front:front + n], ref, error)
    assert (got[:front] == 0).all() and (got[front + n:] == 0).all()
    out = torch.full_like(got, 5.0)
    attention_varlen(*call, out=out)
    assert torch.equal(out[front:front + n], got[front:front + n]) and (out[:front] == 5).all() and (out[front + n:] == 5).all()


def test_rows_of_no_sequence_where_keys_are_split(native):
    from fast_route_amd import attention_varlen
    _say("outside, split")
    g = torch.Generator().manual_seed(1)
    for rows, heads in ((40, 8), (700, 16)):  # a head to a workgroup of the join, and several
        q, (k, v) = torch.randn(rows, heads, 64, generator=g).bfloat16(), (torch.randn(4000, 2, 64, generator=g).bfloat16() for _ in range(2))
        assert native.fr_attention_workspace_bytes(1, rows, 4000, heads, 2, 64) > 0
        got = attention_varlen(q.cuda(), k.cuda(), v.cuda(), _cu([20], 9).cuda(), _cu([4000]).cuda())
        _close(got[9:29], *oracle.attention(q[9:29], k, v, _seen(20, 4000), 0.125))
        assert (got[:9] == 0).all() and (got[29:] == 0).all()


def test_many_sequences_in_graphs_that_share_a_workspace(native):
    """Lengths change between replays, the two graphs' too, with eager calls on the same workspace between them."""
    from fast_route_amd import attention_varlen, paged_attention
    _say("graphs, one workspace")
    rows = 300
    q, kc, vc, table = (t.cuda() for t in _pool(rows, 200, 16, 1, 64, 2, 3, 60))
    n = torch.zeros(rows, dtype=torch.int32, device="cuda")
    pq, pk = torch.empty(900, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(900, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu = torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    need = max(native.fr_paged_attention_workspace_bytes(rows, 2, 1, 64, 960), native.fr_attention_workspace_bytes(rows, 900, 900, 4, 2, 64))
    assert need > 0
    work = torch.empty(need, dtype=torch.uint8, device="cuda")

    def decode():
        return paged_attention(q, kc, vc, table, n, workspace_buf=work)

    def prompt():
        return attention_varlen(pq, pk, pk, cu, workspace_buf=work)
    decode(), prompt()
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, call in zip(graphs, (decode, prompt)):
        with torch.cuda.graph(graph):
            outs.append(call())
    for i in range(4):
        g = torch.Generator().manual_seed(i)
        lengths = torch.randint(0, 900 if i % 2 else 30, (rows,), generator=g)
        n.copy_(lengths), cu.copy_(_cu(torch.randint(0, 4, (rows,), generator=g).tolist()).clamp(max=900))
        pq.normal_(generator=torch.Generator("cuda").manual_seed(i)), pk.normal_(generator=torch.Generator("cuda").manual_seed(i + 9))
        for j in ((0, 1), (1, 0))[i % 2]:
            graphs[j].replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        eager = decode(), prompt()
        torch.cuda.synchronize()
        assert torch.equal(kept[0], eager[0]) and torch.equal(kept[1], eager[1]), i
        at = torch.arange(960)
        for b in (0, 137, 255, 256, 299):
            where = table[b].cpu().long()[at // 16]
            m = int(lengths[b])
            _close(eager[0][b:b + 1], *oracle.attention(q[b:b + 1].cpu(), kc.cpu()[where, at % 16][:m], vc.cpu()[where, at % 16][:m], torch.ones(1, m, dtype=torch.bool), 0.125))


def test_rotary_and_routing_captured_and_replayed(native):
    from fast_route_amd import grouped_topk, prepare_rotary, rotary_frequencies, rotary_to_cache
    _say("rotary in a graph")
    rotary = prepare_rotary(rotary_frequencies(64), device="cuda")
    qkv = torch.empty(19, 8, 64, dtype=torch.float16, device="cuda")
    at, slots = torch.zeros(19, dtype=torch.int64, device="cuda"), torch.arange(19, device="cuda")
    logits, bias = torch.empty(19, 64, device="cuda"), torch.zeros(64, device="cuda")
    kc, vc = (torch.zeros(4, 16, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))

    def step():
        return (*rotary_to_cache(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], at, rotary, kc, vc, slots),
                *grouped_topk(logits, 6, num_groups=8, topk_groups=3, scoring="sigmoid", bias=bias))
    qkv.normal_(), logits.normal_()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        g = torch.Generator("cuda").manual_seed(i)
        qkv.normal_(generator=g), logits.normal_(generator=g), bias.normal_(generator=g)
        at.copy_(torch.randint(0, 5000, (19,), generator=torch.Generator().manual_seed(i)))
        slots.copy_(torch.randperm(70, generator=torch.Generator().manual_seed(i))[:19] - 3)
        kc.zero_(), vc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in (*out, kc, vc)]
        kc.zero_(), vc.zero_()
        eager = (*step(), kc, vc)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager)), i


def test_rotary_and_routing_on_two_streams(native):
    from fast_route_amd import grouped_topk, prepare_rotary, rotary_embed, rotary_frequencies
    _say("two streams")
    rotary = prepare_rotary(rotary_frequencies(128), True, device="cuda")
    g = torch.Generator("cuda").manual_seed(5)
    calls = [(torch.randn(301, 6, 128, generator=g, device="cuda").bfloat16(), torch.randint(0, 9999, (301,), generator=g, device="cuda"),
              torch.randn(301, 256, generator=g, device="cuda"), torch.randn(256, generator=g, device="cuda")) for _ in range(2)]

    def step(x, at, logits, bias):
        return (*rotary_embed(x[:, :4], x[:, 4:], at, rotary), *grouped_topk(logits, 8, num_groups=8, topk_groups=4, scoring="softmax", bias=bias))
    want = [step(*c) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(*calls[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for out in got[i] for a, b in zip(out, want[i]))


def test_keys_and_rows_far_apart(native):
    """Keys whose offsets pass 32 bits, as parts of a joint projection with long rows."""
    from fast_route_amd import attention_varlen
    _say("far apart")
    keys, pitch = 70000, 40000
    held = torch.empty(keys, pitch, dtype=torch.bfloat16, device="cuda")  # 5.6 GB
    g = torch.Generator("cuda").manual_seed(6)
    k, v, q = held[:, 64:128].unflatten(1, (1, 64)), held[:, 8000:8064].unflatten(1, (1, 64)), held[:, 20000:20128].unflatten(1, (2, 64))
    for part in (k, v, q):
        part.normal_(generator=g)
    assert k.stride(0) == pitch and (keys - 300) * pitch > 2 ** 31
    first = keys - 300  # the last 300 keys, and all of them for the last row
    kk, vv, qq = (t[first:].cpu() for t in (k, v, q))
    got = attention_varlen(q, k, v, torch.tensor([first, keys], dtype=torch.int32, device="cuda"), out=q)
    assert got.data_ptr() == q.data_ptr()
    _close(got[first:], *oracle.attention(qq, kk, vv, _seen(300, 300), 0.125))
    last = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(7)).bfloat16()
    got = attention_varlen(last.cuda(), k, v, _cu([1]).cuda(), _cu([keys]).cuda())
    _close(got, *oracle.attention(last, k.cpu(), v.cpu(), torch.ones(1, keys, dtype=torch.bool), 0.125))


def test_no_tables_and_no_pages(native):
    from fast_route_amd import paged_attention
    _say("no pages")
    q, kc, vc, table = (t.cuda() for t in _pool(5, 3, 16, 2, 64, 4, 8, 2))
    n = torch.full((5,), 20, dtype=torch.int32, device="cuda")
    for call in ((q, kc, vc, table[:, :0], n), (q, kc[:0], vc[:0], table, n), (q, kc, vc, torch.full_like(table, 7), n), (q, kc, vc, table, n * 0), (q, kc, vc, table, n - 100)):
        out = torch.full_like(q, 5.0)
        assert paged_attention(*call, out=out) is out and (out == 0).all()
    assert paged_attention(q[:0], kc, vc, table[:0], n[:0]).shape == (0, 4, 64)


def test_results_over_what_is_still_read(native):
    from fast_route_amd import attention_varlen, prepare_rotary, rotary_embed, rotary_frequencies
    _say("shared memory")
    rotary = prepare_rotary(rotary_frequencies(64), device="cuda")
    x, other, at = torch.zeros(9, 2, 64, device="cuda").half(), torch.zeros(9, 2, 64, device="cuda").half(), torch.arange(9, device="cuda")
    cu = _cu([9]).cuda()
    for call in (lambda: rotary_embed(x, x, at, rotary, inplace=True), lambda: attention_varlen(x, other, x, cu, out=x), lambda: attention_varlen(x, other, x.clone(), cu, out=other),
                 lambda: attention_varlen(x, x, x, cu, out=x)):
        with pytest.raises(AssertionError, match="memory"):
            call()
    rotary_embed(x, x, at, rotary), attention_varlen(x, x, x, cu)
    rotary_embed(x[:0], x[:0], at[:0], rotary, inplace=True), attention_varlen(x[:0], x[:0], x[:0], cu, out=x[:0])

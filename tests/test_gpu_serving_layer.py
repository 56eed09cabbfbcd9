"""A layer that serves: rotary_to_cache, attention_varlen, paged_attention, grouped_topk and fused_experts one after the other, as the layer
bench runs them, against the same steps in 64 bits on the CPU."""
import json
import subprocess
import sys

import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

K, FFN, E, TOPK, H, G, D, PAGE = 256, 128, 16, 4, 8, 2, 64, 16
ROUTING = {"scoring": "sigmoid", "num_groups": 4, "topk_groups": 2}


def _layer(dtype):
    from fast_route_amd.transformer_layer_bench import ServingAttention
    torch.manual_seed(3)
    attn = ServingAttention(K, H, G, D, dtype)
    gate, w1, w2 = (torch.randn(s, device="cuda").to(dtype) / 10 for s in ((K, E), (E, 2 * FFN, K), (E, K, FFN)))
    return attn, gate, w1, w2


def _plain_attention(attn, x):
    """Rows x [n, K] of one sequence from its start, every product in 64 bits."""
    n = x.shape[0]
    freq = 10000.0 ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)
    qkv = (x.double() @ attn.qkv.weight.detach().cpu().double().t()).view(n, H + 2 * G, D)
    at = torch.arange(n)
    q, k = (oracle.rotary(t, at, freq) for t in (qkv[:, :H], qkv[:, H:H + G]))
    seen = torch.ones(n, n, dtype=torch.bool).tril()
    out, _ = oracle.attention(q, k, qkv[:, H + G:], seen, D ** -0.5)
    return out.view(n, H * D) @ attn.proj.weight.detach().cpu().double().t()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prefill_and_decode(native, dtype):
    """Prompts prefilled in two packed chunks, then tokens one by one: every row is the whole sequence's attention.  Bound: five roundings to the type (projection,
    rotary, softmax terms, attention, projection) of sums whose terms are 10 times the result at most."""
    from fast_route_amd.transformer_layer_bench import PagedCache, serving_experts
    print(f"[case] serving layer {dtype}", flush=True)
    attn, gate, w1, w2 = _layer(dtype)
    lengths, steps = [37, 5, 90], 4
    g = torch.Generator().manual_seed(1)
    rows = [torch.randn(n + steps, K, generator=g).to(dtype) for n in lengths]
    cache = PagedCache(3, max(lengths) + steps, PAGE, G, D, dtype)
    cache.table = cache.table.flip(0).contiguous()
    with torch.no_grad():
        x = torch.cat([r[:n] for r, n in zip(rows, lengths)]).cuda()
        seq = torch.cat([torch.full((n,), b) for b, n in enumerate(lengths)]).cuda()
        at = torch.cat([torch.arange(n) for n in lengths]).cuda()
        cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
        got = [list(t.split(lengths)) for t in [attn.prefill(x, cu, at, cache, cache.slots(seq, at))]][0]
        for s in range(steps):
            pos = torch.tensor([n + s for n in lengths]).cuda()
            step = attn.decode(torch.stack([r[n + s] for r, n in zip(rows, lengths)]).cuda(), pos, cache, cache.slots(torch.arange(3).cuda(), pos),
                               (pos + 1).int())
            got = [torch.cat([a, step[b:b + 1]]) for b, a in enumerate(got)]
        u = torch.finfo(dtype).eps / 2
        for b in range(3):
            want = _plain_attention(attn, rows[b])
            assert (got[b].cpu().double() - want).norm() <= 5 * 10 * u * want.norm()
        h = torch.cat(got) + torch.cat(rows).cuda()
        out = serving_experts(h, gate, w1, w2, TOPK, ROUTING)
        logits = (h @ gate).cpu()
        weights, ids = oracle.grouped_topk(logits, TOPK, 4, 2, "sigmoid")
        want = torch.zeros(h.shape, dtype=torch.float64)
        for t in range(h.shape[0]):
            for j in range(TOPK):
                e = int(ids[t, j])
                a, c = (h[t].cpu().double() @ w1[e].cpu().double().t()).chunk(2)
                want[t] += weights[t, j] * ((torch.nn.functional.silu(a) * c) @ w2[e].cpu().double().t())
        assert (out.cpu().double() - want).norm() <= 4 * u * 4 * want.norm()


def test_decode_steps_captured(native):
    """A decode step in a graph, positions and lengths moved on between replays, against eager steps on a cache of its own."""
    from fast_route_amd.transformer_layer_bench import PagedCache, serving_experts
    print("[case] captured decode", flush=True)
    dtype = torch.bfloat16
    attn, gate, w1, w2 = _layer(dtype)
    caches = [PagedCache(2, 40, PAGE, G, D, dtype) for _ in range(2)]
    x, pos, rows = torch.empty(2, K, dtype=dtype, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.arange(2, device="cuda")

    def step(cache):
        h = attn.decode(x, pos, cache, cache.slots(rows, pos), (pos + 1).int()) + x
        return serving_experts(h, gate, w1, w2, TOPK, ROUTING)
    with torch.no_grad():
        x.normal_()
        for c in caches:
            step(c)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(caches[0])
        for i in range(33):
            x.normal_(generator=torch.Generator(device="cuda").manual_seed(i))
            pos.fill_(i)
            graph.replay()
            torch.cuda.synchronize()
            kept = out.clone()
            assert torch.equal(kept, step(caches[1])), i
    assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)


def test_bench_command(native):
    print("[case] bench --serve", flush=True)
    run = subprocess.run([sys.executable, "-m", "fast_route_amd.transformer_layer_bench", "--serve", "-n", "128", "-k", "256", "-e", "16", "--topk", "4", "-b", "2", "--n_head", "8",
                          "--n_kv_head", "2", "--head_dim", "64", "--seqs", "33,64", "--scoring", "sigmoid", "--groups", "4", "--topk_groups", "2"],
                         capture_output=True, text=True, timeout=110)
    assert run.returncode == 0, run.stderr[-1500:]
    lines = [json.loads(l) for l in run.stdout.splitlines() if l.startswith("{")]
    assert [l["seq"] for l in lines] == [33, 64] and all(l["prefill_ms"] > 0 and l["decode_ms"] > 0 for l in lines)

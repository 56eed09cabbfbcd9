"""The layer's attention, prompts and then single tokens, step by step and element by element: each step against its definition in 64 bits on what the step before it gave,
so that the bounds are a rounding's and a key that is left out or a position off by one is beyond them."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

K, H, G, D, PAGE = 256, 8, 2, 64, 16


def _product(x, weight, got):
    """Rows x times weight^T, rounded once: half a step, and 512 sums in 32 bits of terms with one rounding each."""
    want, size = x.double() @ weight.double().t(), x.double().abs() @ weight.double().abs().t()
    assert ((got.double() - want).abs() <= torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -14 * size).all()


def _turned(x, positions, got):
    """The result's rounding; angle, sine, cosine and three operations: 2^-20 of the pair's size."""
    freq = 10000.0 ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)
    want = oracle.rotary(x, positions, freq)
    size = x.double().abs().view(*x.shape[:2], 2, D // 2).sum(dim=2).repeat(1, 1, 2)
    info = torch.finfo(got.dtype)
    assert ((got.double() - want).abs() <= info.eps / 2 * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -20 * size + info.tiny * info.eps).all()


def _beyond(got, q, k, v, seen):
    """Elements of an attention's result off by more than the oracle's error and half a step."""
    want, error = oracle.attention(q, k, v, seen, D ** -0.5)
    info = torch.finfo(got.dtype)
    return (got.double() - want).abs() > error + info.eps / 2 * (want.abs() + error) + info.tiny * info.eps


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_row_of_prefill_and_decode(native, dtype, monkeypatch):
    from fast_route_amd import transformer_layer_bench as bench
    print(f"[case] rows {dtype}", flush=True)
    torch.manual_seed(3)
    attn = bench.ServingAttention(K, H, G, D, dtype)
    qkv_weight, proj_weight = attn.qkv.weight.detach().cpu(), attn.proj.weight.detach().cpu()
    seen = {}

    def recorded(name, pick):
        call = getattr(bench, name)

        def run(*args, **kwargs):
            out = call(*args, **kwargs)
            seen[name] = [t.detach().cpu().clone() for t in pick(out, args)]
            return out
        monkeypatch.setattr(bench, name, run)
    recorded("rotary_to_cache", lambda out, args: [*out, args[2]])
    recorded("attention_varlen", lambda out, args: [out])
    recorded("paged_attention", lambda out, args: [out])
    attn.qkv.register_forward_hook(lambda module, args, out: seen.update(qkv=[out.detach().cpu().clone()]))

    def kept(x, at):
        """The step's queries, keys and values, checked."""
        raw = seen["qkv"][0]
        _product(x, qkv_weight, raw)
        q, k, v = raw.view(-1, H + 2 * G, D).split((H, G, G), dim=1)
        turned_q, turned_k, same_v = seen["rotary_to_cache"]
        _turned(q, at, turned_q), _turned(k, at, turned_k)
        assert torch.equal(v, same_v)
        return turned_q, turned_k, v
    lengths, steps = [37, 5, 90, 1], 5
    g = torch.Generator().manual_seed(1)
    rows = [torch.randn(n + steps, K, generator=g).to(dtype) for n in lengths]
    count = len(rows)
    cache = bench.PagedCache(count, max(lengths) + steps, PAGE, G, D, dtype)
    cache.table = cache.table.flip(0).contiguous()
    with torch.no_grad():
        x = torch.cat([r[:n] for r, n in zip(rows, lengths)])
        sequence, at = torch.repeat_interleave(torch.arange(count), torch.tensor(lengths)), torch.cat([torch.arange(n) for n in lengths])
        cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
        got = attn.prefill(x.cuda(), cu.cuda(), at.cuda(), cache, cache.slots(sequence.cuda(), at.cuda())).cpu()
        q, k, v = kept(x, at)
        out = seen["attention_varlen"][0]
        _product(out.view(-1, H * D), proj_weight, got)
        keys, values = list(k.split(lengths)), list(v.split(lengths))
        for b, n in enumerate(lengths):
            assert not _beyond(out[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]], keys[b], values[b], torch.ones(n, n, dtype=torch.bool).tril()).any(), b
        for s in range(steps):
            at = torch.tensor(lengths) + s
            x = torch.stack([r[n + s] for r, n in zip(rows, lengths)])
            got = attn.decode(x.cuda(), at.cuda(), cache, cache.slots(torch.arange(count).cuda(), at.cuda()), (at + 1).int().cuda()).cpu()
            q, k, v = kept(x, at)
            out = seen["paged_attention"][0]
            _product(out.view(-1, H * D), proj_weight, got)
            for b in range(count):
                keys[b], values[b] = torch.cat([keys[b], k[b:b + 1]]), torch.cat([values[b], v[b:b + 1]])
                whole = torch.ones(1, len(keys[b]), dtype=torch.bool)
                assert not _beyond(out[b:b + 1], q[b:b + 1], keys[b], values[b], whole).any(), (b, s)
                whole[0, -1] = False  # what the check is worth: without the newest key most heads are beyond it
                assert _beyond(out[b:b + 1], q[b:b + 1], keys[b], values[b], whole).any(dim=2).sum() > H // 2, (b, s)

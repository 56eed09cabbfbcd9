"""Attention whose softmax terms span many octaves: a key far above many others, which half precision holds as subnormals."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu


def _say(msg):
    print("[case] " + msg, flush=True)


def _tail(octaves, keys, dtype, seed):
    """Four heads of 64 dimensions over one key head of `keys` keys: the first scores about `octaves` factors of 2 above the others and is worth nothing, so that the
    others are the whole result.  With it the result from the definition and how far it may be off: the oracle's error, and for the terms that fp16 holds as subnormals half
    of their step, 2^-25 where the largest term is at least 2^7, so 2^-32 of that: for the values' sum, and for the terms' sum times the result."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = torch.zeros(1, 4, 64), torch.zeros(keys, 1, 64), 1.0 + torch.rand(keys, 1, 64, generator=g)
    q[..., 0], q[..., 1:5] = 8.0, torch.randn(1, 4, 4, generator=g) * 0.2
    k[0, 0, 0], v[0] = octaves * 0.6931, 0.0
    k[1:, 0, 1:5] = torch.randn(keys - 1, 4, generator=g)
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    out, error = oracle.attention(q, k, v, torch.ones(1, keys, dtype=torch.bool), 0.125)
    if dtype == torch.float16:
        s = 0.125 * (k[:, 0].double() @ q[0].double().t())
        total = torch.exp(s - s.amax(dim=0)).sum(dim=0)[None, :, None]
        error = error + 2.0 ** -32 * (v.double().abs().sum(dim=0)[None] + keys * out.abs()) / total
    return q, k, v, out, error


def _close(got, ref, error):
    info = torch.finfo(got.dtype)
    tol = error + info.eps / 2 * (ref.abs() + error) + info.tiny * info.eps
    off = (got.cpu().double() - ref).abs()
    assert not (off > tol).any() and not got.isnan().any(), "worst %g of the bound" % (off / tol).max().item()


TAILS = [(o, t) for t in (torch.float16, torch.bfloat16) for o in (15, 21, 25, 26.5)]


@pytest.mark.parametrize("octaves,dtype", TAILS)
def test_tail_of_a_prompt(native, octaves, dtype):
    """512 key heads, the same one each: nothing is split."""
    from fast_route_amd import attention_varlen
    _say(f"tail {octaves} {dtype}")
    keys, G = 131072, 512
    q, k, v, ref, error = _tail(octaves, keys, dtype, int(octaves))
    cu = [torch.tensor([0, n], dtype=torch.int32).cuda() for n in (1, keys)]
    assert native.fr_attention_workspace_bytes(1, 1, keys, G, G, 64) == 0
    got = attention_varlen(q.repeat(1, G // 4, 1).cuda(), k.cuda().expand(-1, G, -1), v.cuda().expand(-1, G, -1), *cu)
    _close(got.view(G // 4, 4, 64), ref.expand(G // 4, 4, 64), error)
    got = attention_varlen(q.cuda(), k.cuda(), v.cuda(), *cu)  # and split
    _close(got, ref, error)


@pytest.mark.parametrize("octaves,dtype", TAILS)
def test_tail_over_pages(native, octaves, dtype):
    """1024 key heads, all of them the same: three parts."""
    from fast_route_amd import paged_attention
    _say(f"paged tail {octaves} {dtype}")
    keys, G, page = 131072, 1024, 64
    q, k, v, ref, error = _tail(octaves, keys, dtype, int(octaves))
    kc, vc = (t.cuda().view(keys // page, page, 1, 64).expand(-1, -1, G, -1) for t in (k, v))
    table, n = torch.arange(keys // page, dtype=torch.int32)[None].cuda(), torch.tensor([keys], dtype=torch.int32).cuda()
    got = paged_attention(q.repeat(1, G // 4, 1).cuda(), kc, vc, table, n)
    _close(got.view(G // 4, 4, 64), ref.expand(G // 4, 4, 64), error)
    got = paged_attention(q.cuda(), kc[:, :, :1], vc[:, :, :1], table, n)  # and many
    _close(got, ref, error)

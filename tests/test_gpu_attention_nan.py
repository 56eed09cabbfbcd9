"""Queries, keys and values that are not numbers, where a row sees them: they reach every result they belong to and no other one, however the keys are cut."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _say(msg):
    print("[case] " + msg, flush=True)


def _close(got, ref, error):
    """`error` and the result's own rounding (half a step; subnormal ones' too)."""
    info = torch.finfo(got.dtype)
    tol = error + info.eps / 2 * (ref.abs() + error) + info.tiny * info.eps
    off = (got.cpu().double() - ref).abs()
    assert not (off > tol).any() and not got.isnan().any(), "worst %g of the bound" % (off / tol).max().item()


def _paged(lengths, H, G, D, page, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    table = torch.zeros((len(lengths), max(counts)), dtype=torch.int32)
    order, at = torch.randperm(sum(counts), generator=g).to(torch.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    kc, vc = (torch.randn(sum(counts), page, G, D, generator=g).to(dtype) for _ in range(2))
    return torch.randn(len(lengths), H, D, generator=g).to(dtype), kc, vc, table, torch.tensor(lengths, dtype=torch.int32)


def _want(q, kc, vc, table, lengths, scale):
    page, out, error = kc.shape[1], [], []
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(n)
        where = table[b].long()[at // page]
        o, e = oracle.attention(q[b:b + 1], kc[where, at % page], vc[where, at % page], torch.ones(1, n, dtype=torch.bool), scale)
        out.append(o), error.append(e)
    return torch.cat(out), torch.cat(error)


# key heads (a workgroup's wavefronts on four, two or one of them), lengths (one part each, several, both)
FORMS = [(G, lengths) for G in (8, 4, 6, 2, 1, 3) for lengths in ([40, 17], [500, 700], [900, 30, 333])]


@pytest.mark.parametrize("G,lengths", FORMS)
def test_query_over_pages(native, G, lengths):
    from fast_route_amd import paged_attention
    for dtype, D in ((torch.bfloat16, 64), (torch.float16, 128)):
        _say(f"query G={G} {lengths} {dtype}")
        H = 2 * G
        q, kc, vc, table, n = _paged(lengths, H, G, D, 16, dtype, G + sum(lengths))
        ref, error = _want(q, kc, vc, table, n, D ** -0.5)
        bad = torch.zeros(len(lengths), H, dtype=torch.bool)
        bad[1, H - 1], bad[0, 0] = True, True
        q[bad] = NAN
        q[0, 0, 1:] = 1.0  # one value of the head is enough
        got = paged_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda()).cpu()
        assert got[bad].isnan().all()
        _close(got[~bad], ref[~bad], error[~bad])


@pytest.mark.parametrize("G,lengths", FORMS)
def test_key_and_value_over_pages(native, G, lengths):
    from fast_route_amd import paged_attention
    _say(f"key G={G} {lengths}")
    H, D, page = 2 * G, 64, 16
    q, kc, vc, table, n = _paged(lengths, H, G, D, page, torch.bfloat16, G + sum(lengths))
    ref, error = _want(q, kc, vc, table, n, D ** -0.5)
    where = lambda b, key: (int(table[b, key // page]), key % page)
    keys, values = kc.clone(), vc.clone()
    keys[where(0, lengths[0] - 1)][0] = NAN   # the first sequence's last key, for its first key head
    values[where(1, 3)][G - 1, 5] = NAN       # a value of the second one's, for its last
    got = paged_attention(q.cuda(), keys.cuda(), values.cuda(), table.cuda(), n.cuda()).cpu()
    bad = torch.zeros(ref.shape, dtype=torch.bool)
    bad[0, :2], bad[1, H - 2:, 5] = True, True
    assert got[bad].isnan().all()
    _close(got[~bad], ref[~bad], error[~bad])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,m", [(70, 90), (9, 4000)])
def test_query_of_a_prompt(native, n, m, causal):
    """A part of the keys each and all in one."""
    from fast_route_amd import attention_varlen
    _say(f"prompt {n} {m} {causal}")
    g = torch.Generator().manual_seed(n)
    q, (k, v) = torch.randn(n, 4, 64, generator=g).bfloat16(), (torch.randn(m, 2, 64, generator=g).bfloat16() for _ in range(2))
    seen = torch.arange(m)[None, :] <= torch.arange(n)[:, None] + (m - n) if causal else torch.ones(n, m, dtype=torch.bool)
    ref, error = oracle.attention(q, k, v, seen, 0.125)
    bad = torch.zeros(n, 4, dtype=torch.bool)
    bad[2, 1], bad[n - 1, 3] = True, True
    q[bad] = NAN
    got = attention_varlen(q.cuda(), k.cuda(), v.cuda(), torch.tensor([0, n], dtype=torch.int32).cuda(), torch.tensor([0, m], dtype=torch.int32).cuda(), causal).cpu()
    assert got[bad].isnan().all()
    _close(got[~bad], ref[~bad], error[~bad])

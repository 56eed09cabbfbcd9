"""grouped_topk against its definition in 64 bits (oracle/serving_oracle.py)."""
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _say(msg):
    print("[case] " + msg, flush=True)


def _check(logits, topk, **kw):
    from fast_route_amd import grouped_topk
    bias = kw.pop("bias", None)
    w, ids = grouped_topk(logits.cuda(), topk, bias=None if bias is None else bias.cuda(), **kw)
    rw, rid = oracle.grouped_topk(logits, topk, bias=bias, **kw)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu(), rid), "ids differ at tokens %s" % (ids.cpu() != rid).any(dim=1).nonzero()[:4, 0].tolist()
    # without a bias scores are fp32: the difference of two logits (2^-24 of it, up to 100) and the exponential 2^-17, sums of up to 1024 of
    # them 2^-14 at worst, a division; with one they are rounded once
    tol = 2.0 ** -23 if bias is not None else 2.0 ** -14
    assert ((w.cpu().double() - rw).abs() <= tol * rw.abs() + 1e-38).all(), (w.cpu().double() - rw).abs().max().item()


SHAPES = [(1, 1, 1, 1, 1), (3, 8, 1, 1, 2), (5, 60, 4, 2, 4), (7, 64, 8, 3, 6), (33, 160, 8, 3, 6), (130, 256, 8, 4, 8), (9, 257, 1, 1, 64),
          (6, 384, 64, 9, 7), (4, 512, 16, 4, 10), (5, 1024, 32, 5, 17), (11, 63, 7, 7, 63), (4, 6, 6, 3, 3), (3, 12, 3, 1, 4)]


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("M,E,groups,kept,topk", SHAPES)
def test_choices_and_weights(native, M, E, groups, kept, topk, scoring, biased):
    for dtype in TYPES:
        _say(f"M={M} E={E} groups={groups} kept={kept} topk={topk} {scoring} {biased} {dtype}")
        g = torch.Generator().manual_seed(M * E + topk)
        logits = (torch.randn(M, E, generator=g) * 2).to(dtype)
        bias = torch.randn(E, generator=g) * 0.1 if biased else None
        _check(logits, topk, num_groups=groups, topk_groups=kept, scoring=scoring, bias=bias)


@pytest.mark.parametrize("biased", [False, True])
def test_ties_go_to_the_lower_index(native, biased):
    _say("ties")
    g = torch.Generator().manual_seed(3)
    logits = torch.randint(-2, 3, (200, 96), generator=g).float()
    logits[0] = 0.0
    logits[1, ::2] = -0.0
    logits[1, 1::2] = 0.0
    bias = torch.randint(-1, 2, (96,), generator=g).float() / 4 if biased else None
    for scoring in ("softmax", "sigmoid"):
        for groups, kept in ((1, 1), (12, 5)):
            _check(logits, 9, num_groups=groups, topk_groups=kept, scoring=scoring, bias=bias)


def test_choices_that_differ_in_their_last_bits(native):
    """Scores near each other beyond 32 bits: logits one step apart under a bias that brings them together."""
    _say("near choices")
    E = 256
    x = 1.0 + torch.arange(E) * 2.0 ** -23
    logits = x[torch.stack([torch.randperm(E, generator=torch.Generator().manual_seed(i)) for i in range(64)])]
    bias = (torch.randn(E, generator=torch.Generator().manual_seed(1)) * 2.0 ** -24).float()
    for scoring in ("softmax", "sigmoid"):
        _check(logits, 16, num_groups=8, topk_groups=4, scoring=scoring, bias=bias)
        _check(logits, 16, scoring=scoring, bias=bias)


@pytest.mark.parametrize("biased", [False, True])
def test_infinite_logits_and_nan(native, biased):
    _say("infinite logits")
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(12, 24, generator=g)
    logits[0] = -inf
    logits[1] = nan
    logits[2, 3:] = -inf
    logits[3, [5, 7]] = inf
    logits[4, 2] = nan
    logits[5, 1:] = torch.finfo(torch.float32).min
    logits[6] = torch.finfo(torch.float32).min
    logits[7] = 90.0 + torch.arange(24)
    logits[8] = -90.0 - torch.arange(24)
    bias = torch.randn(24, generator=g) * 0.1 if biased else None
    for scoring in ("softmax", "sigmoid"):
        if biased:
            b = bias.clone()
            b[[0, 9]] = -inf
            b[[1]] = nan
            b[[2]] = inf
            _check(logits, 5, num_groups=4, topk_groups=2, scoring=scoring, bias=b)
            _check(logits, 24, scoring=scoring, bias=b)
        _check(logits, 5, num_groups=4, topk_groups=2, scoring=scoring, bias=bias)


def test_scale_and_plain_weights(native):
    _say("scale")
    logits = torch.randn(50, 64, generator=torch.Generator().manual_seed(2))
    _check(logits, 6, renormalize=False, scale=2.5)
    _check(logits, 6, scoring="sigmoid", renormalize=False)
    _check(logits, 6, scoring="sigmoid", scale=2.5, bias=torch.linspace(-1, 1, 64))
    _check(torch.full((3, 64), -200.0), 6, scoring="sigmoid")  # scores that are zero in 32 bits


def test_same_as_topk_softmax(native):
    """Without bias and groups the choice is topk_softmax's."""
    from fast_route_amd import grouped_topk, topk_softmax
    _say("beside topk_softmax")
    logits = torch.randn(777, 64, generator=torch.Generator().manual_seed(4)).cuda()
    w, ids = grouped_topk(logits, 6)
    rw, rid = topk_softmax(torch.empty(777, 6, device="cuda"), torch.empty(777, 6, dtype=torch.int32, device="cuda"), None, logits, True)
    assert torch.equal(ids, rid) and torch.allclose(w, rw, rtol=2.0 ** -16, atol=0)


def test_many_tokens_rows_apart_and_odd_addresses(native):
    _say("many tokens")
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(20011, 70, generator=g)
    bias = torch.randn(64, generator=g) * 0.1
    for dtype in TYPES:
        held = wide.to(dtype).cuda()
        from fast_route_amd import grouped_topk
        part = held[:, 3:67]
        w, ids = grouped_topk(part, 6, num_groups=8, topk_groups=4, scoring="sigmoid", bias=bias.cuda())
        pick = torch.cat([torch.arange(100), torch.arange(16300, 16500), torch.arange(19900, 20011)])
        rw, rid = oracle.grouped_topk(part.cpu()[pick], 6, 8, 4, "sigmoid", bias)
        assert torch.equal(ids.cpu()[pick], rid)
        assert ((w.cpu()[pick].double() - rw).abs() <= 2.0 ** -23 * rw).all()
        again = grouped_topk(part.contiguous(), 6, num_groups=8, topk_groups=4, scoring="sigmoid", bias=bias.cuda())
        assert torch.equal(again[0], w) and torch.equal(again[1], ids)


def test_no_tokens_and_one(native):
    from fast_route_amd import grouped_topk
    _say("no tokens")
    w, ids = grouped_topk(torch.empty(0, 64, device="cuda"), 6)
    assert w.shape == (0, 6) and ids.shape == (0, 6)
    row = torch.randn(64, 1, generator=torch.Generator().manual_seed(1))
    one = row.cuda().t().contiguous().as_strided((1, 64), (1, 1))  # one row: its stride says nothing
    assert torch.equal(grouped_topk(one, 6)[1].cpu(), oracle.grouped_topk(row.t(), 6)[1])


@pytest.mark.parametrize("E,groups,kept,topk", [(256, 8, 4, 8), (64, 1, 1, 6), (128, 16, 5, 16), (512, 16, 4, 10), (384, 1, 1, 8)])
def test_order_of_many_tokens(native, E, groups, kept, topk):
    """16384 tokens' choices in the order of 64 bits: random logits, and logits whose choices crowd together around the last place, so that more than topk
    have to be told apart (and for some tokens more than a lane each can)."""
    from fast_route_amd import grouped_topk
    _say(f"order E={E} groups={groups}")
    g = torch.Generator(device="cuda").manual_seed(E)
    M = 16384
    logits = torch.randn(M, E, device="cuda", generator=g) * 1.5
    logits[M // 2:] = 0.5 + 2.0 ** -22 * torch.randint(0, 40, (M // 2, E), device="cuda", generator=g).float()
    logits[M // 2::2, : topk - 1] += 1.0  # the first places clear, the others crowded
    bias = torch.randn(E, device="cuda", generator=g) * 0.1
    near = torch.zeros(E, device="cuda")
    near[::3] = 2.0 ** -24
    for scoring in ("sigmoid", "softmax"):
        for b in (None, bias, near):
            x = logits.double()
            score = torch.sigmoid(x) if scoring == "sigmoid" else torch.softmax(x, dim=1)
            choice = x if b is None else score + b.double()
            # distances that 64-bit sums in another order could turn: none of the tokens that are compared
            if groups > 1:
                best = choice.view(M, groups, -1).topk(2, dim=2).values
                worth = best[:, :, 0] if b is None else best.sum(dim=2)
                top = torch.sort(worth, dim=1, descending=True, stable=True)
                out = torch.ones_like(worth, dtype=torch.bool).scatter_(1, top.indices[:, :kept], False)
                choice = choice.masked_fill(out.repeat_interleave(E // groups, dim=1), float("-inf"))
                edge = top.values[:, kept - 1] - top.values[:, kept]
            order = torch.sort(choice, dim=1, descending=True, stable=True)
            clear = torch.ones(M, dtype=torch.bool, device="cuda")
            if b is not None:
                step = order.values[:, :topk] - order.values[:, 1: topk + 1]
                clear = ((step == 0) & (scoring == "sigmoid") | (step > 1e-14)).all(dim=1)
                if groups > 1:
                    clear &= edge > 1e-14
            assert clear[: M // 2].float().mean() > 0.99
            w, ids = grouped_topk(logits, topk, num_groups=groups, topk_groups=kept, scoring=scoring, bias=b)
            same = (ids == order.indices[:, :topk]).all(dim=1)
            assert same[clear].all(), (scoring, b is None, (~same & clear).nonzero()[:3, 0].tolist())
            want = score.gather(1, ids.long())
            want = want / want.sum(dim=1, keepdim=True)
            assert ((w.double() - want).abs() <= 2.0 ** -14 * want).all()


def test_captured_and_replayed(native):
    from fast_route_amd import grouped_topk
    _say("graph")
    logits, bias = torch.empty(37, 256, device="cuda"), torch.empty(256, device="cuda")

    def step():
        return grouped_topk(logits, 8, num_groups=8, topk_groups=4, scoring="sigmoid", bias=bias)
    logits.normal_(), bias.normal_()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        g = torch.Generator(device="cuda").manual_seed(i)
        logits.normal_(generator=g), bias.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in out]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager)), i


def test_refusals(native):
    from fast_route_amd import grouped_topk
    _say("refusals")
    x = torch.zeros(4, 64, device="cuda")
    for call in (lambda: grouped_topk(x.cpu(), 2), lambda: grouped_topk(x.double(), 2), lambda: grouped_topk(x[0], 2), lambda: grouped_topk(x.t(), 2),
                 lambda: grouped_topk(x, 0), lambda: grouped_topk(x, 65), lambda: grouped_topk(x, 2, num_groups=5),
                 lambda: grouped_topk(x, 2, num_groups=0), lambda: grouped_topk(x, 2, num_groups=4, topk_groups=5),
                 lambda: grouped_topk(x, 17, num_groups=4, topk_groups=1), lambda: grouped_topk(x, 2, num_groups=4, topk_groups=0),
                 lambda: grouped_topk(x, 2, scoring="tanh"), lambda: grouped_topk(x, 2, bias=torch.zeros(63, device="cuda")),
                 lambda: grouped_topk(x, 2, bias=torch.zeros(64)), lambda: grouped_topk(x, 2, bias=torch.zeros(64, device="cuda").half()),
                 lambda: grouped_topk(torch.zeros(2, 1025, device="cuda"), 2)):
        with pytest.raises(AssertionError):
            call()

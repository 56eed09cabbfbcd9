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

"""The forms of the MXFP4 layer and product that sizes choose between: values that no form may lose, and each form's own
tails, repeats, captures and streams."""
import numpy as np
import pytest
import torch

import oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def _say(msg):
    print("[case] " + msg, flush=True)


def _weights(E, H, F, seed):
    """Codes and scales of w1 [E, 2F, H] and w2 [E, H, F], on the GPU."""
    from fast_route_amd import quantize_rows_mxfp4
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = []
    for shape, std in (((E, 2 * F, H), 1.5 / H ** 0.5), ((E, H, F), F ** -0.5)):
        w = torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).bfloat16()
        codes, scales = quantize_rows_mxfp4(w.view(-1, shape[2]))
        held += [codes.view(*shape[:2], -1), scales.view(*shape[:2], -1)]
    return held


def _tokens(M, H, E, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn((M, H), device="cuda", generator=g).to(dtype), torch.randn((M, E), device="cuda", generator=g)


# M, H, F, E, topk: few tokens, whole tiles of 64 and of 32 weight rows per wavefront, a last partial one, K slices
FORMS = [(3, 256, 512, 8, 2), (20, 256, 512, 8, 2), (40, 4096, 512, 8, 2), (300, 256, 512, 8, 2), (1200, 800, 128, 64, 6),
         (2000, 2080, 64, 64, 2), (50, 1024, 3584, 8, 2), (40, 1056, 2336, 12, 3)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,H,F,E,topk", FORMS)
def test_a_feature_does_not_depend_on_its_neighbours(native, M, H, F, E, topk, dtype):
    """One output feature in sixteen 2^10 (fp16: 2^6) times larger: all others keep their bits, at every batch size, as sums in fp32
    do; the large ones are scaled by a power of two exactly, but where the type rounded them as subnormals."""
    from fast_route_amd import fused_moe_mxfp4, prepare_weights_mxfp4
    _say(f"neighbours M={M} H={H} F={F} E={E} topk={topk} {dtype}")
    w1, s1, w2, s2 = _weights(E, H, F, M + H)
    x, logits = _tokens(M, H, E, dtype, M)
    plain = fused_moe_mxfp4(x, prepare_weights_mxfp4(w1, s1, w2, s2), logits, topk)
    shift = 10 if dtype == torch.bfloat16 else 6
    s2[:, 5::16] += shift  # scale bytes; far from 255 here
    got = fused_moe_mxfp4(x, prepare_weights_mxfp4(w1, s1, w2, s2), logits, topk)
    large = torch.zeros(H, dtype=torch.bool, device="cuda")
    large[5::16] = True
    assert torch.equal(got[:, ~large], plain[:, ~large])
    was, now = plain[:, large].double(), got[:, large].double()
    normal = was.abs() >= torch.finfo(dtype).smallest_normal
    assert normal.double().mean() > 0.99 and torch.equal(now[normal], was[normal] * 2.0 ** shift)


def test_handles_whose_data_are_others_are_refused(native):
    """Nothing is launched on a prepared weight whose data do not match its sizes or lie elsewhere."""
    import fast_route_amd as fr
    w1, s1, w2, s2 = _weights(4, 64, 96, 1)
    experts = fr.prepare_weights_mxfp4(w1, s1, w2, s2)
    lin = fr.prepare_linear_mxfp4(w1[0], s1[0])
    x, logits = _tokens(40, 64, 4, torch.bfloat16, 2)
    assert fr.linear_mxfp4(x, lin).shape == (40, 192) and fr.fused_moe_mxfp4(x, experts, logits, 2).shape == x.shape
    wide = torch.cat([logits, logits], dim=1)
    bad = [
        lambda: fr.linear_mxfp4(x, lin._replace(N=4096)), lambda: fr.linear_mxfp4(x, lin._replace(data=lin.data[:4352])),
        lambda: fr.linear_mxfp4(x, lin._replace(data=lin.data.cpu())), lambda: fr.linear_mxfp4(x, lin._replace(data=lin.data.to(torch.int32))),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(w2=experts.w2.cpu()), logits, 2),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(w1=experts.w1.cpu()), logits, 2),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(F=128), logits, 2), lambda: fr.fused_moe_mxfp4(x, experts._replace(w2=experts.w2[4352:]), logits, 2),
        lambda: fr.fused_moe_mxfp4(x, experts._replace(E=8), wide, 2),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(AssertionError):
            call()
            print("case", i, "was not refused", flush=True)
    torch.cuda.synchronize()

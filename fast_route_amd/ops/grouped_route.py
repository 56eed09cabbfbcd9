"""Routing by scores with a bias for balance and groups of experts.  No counterpart in the reference, whose routers take the
largest softmax logits (fast_route/fast_route/layers/vllm_route.py:79-87)."""
from __future__ import annotations

import torch

from .. import _native as N

_SCORES = {"softmax": 0, "sigmoid": 1}
_DTYPES = {t: N.dtype_code(t) for t in (torch.float32, torch.bfloat16, torch.float16)}


def grouped_topk(gating_output: torch.Tensor, topk: int, num_groups: int = 1, topk_groups: int = 1, scoring: str = "softmax",
                 bias: torch.Tensor | None = None, renormalize: bool = True, scale: float = 1.0):
    """Experts of each token from router logits [M, E] (f16/bf16/f32): (topk_weights fp32 [M, topk], topk_ids int32 [M, topk]), as
    fused_experts takes them.

    Scores are the softmax over all experts or the sigmoid of the logits.  An expert is chosen by its score plus its bias (fp32 [E],
    which the weights do not see), without a bias by its logit.  Experts come in `num_groups` groups of equal size, one after the
    other; the `topk_groups` best groups are kept - a group is worth its best choice, with a bias the sum of its best two - and the `topk`
    best of their experts are the result, best first, ties to the lower index.  Weights are the scores, divided by their sum
    with `renormalize`, times `scale`.

    With a bias, scores and choices are computed in 64 bits: the order of two experts does not depend on a rounding.  A NaN counts
    as -infinity.  Limits: E <= 1024, num_groups <= 64, topk <= 64."""
    shape, strides, dtype = gating_output.shape, gating_output.stride(), gating_output.dtype
    assert len(shape) == 2 and dtype in _DTYPES, "gating_output must be [M, E] in float16, bfloat16 or float32"
    M, E = shape
    assert E == 1 or strides[1] == 1, "router logits must be contiguous along experts"
    assert scoring in _SCORES, "scoring must be 'softmax' or 'sigmoid'"
    if bias is None:
        dev, bias_ptr = N.device_of(gating_output), 0
    else:
        dev, bias_ptr = N.device_of(gating_output, bias), bias.data_ptr()
        assert bias.dtype == torch.float32 and bias.shape == (E,) and bias.is_contiguous(), "bias must be contiguous float32 [E]"
    topk = int(topk)
    assert 1 <= topk <= 64, "topk outside [1, 64]"
    topk_weights = gating_output.new_empty((M, topk), dtype=torch.float32)
    topk_ids = gating_output.new_empty((M, topk), dtype=torch.int32)
    N.run(dev, N.lib().fr_gating_grouped, gating_output.data_ptr(), _DTYPES[dtype], M, E, strides[0] if M > 1 else E, bias_ptr, int(num_groups),
          int(topk_groups), topk, _SCORES[scoring], bool(renormalize), float(scale), topk_weights.data_ptr(), topk_ids.data_ptr())
    return topk_weights, topk_ids

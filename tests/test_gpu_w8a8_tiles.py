"""The int8 product where it takes LDS tiles, and on all its kernels what NaN scales become."""
import math

import pytest
import torch

from ftmoe.kernel.fused_w8a8_linear import fused_w8a8_expert_forward
from ftmoe.kernel.fused_w8a8_moe import fused_w8a8_moe
from ftmoe.kernel.w8a8_linear import w8a8_linear
from test_gpu_w8a8 import codes, moe_inputs, scales

pytestmark = pytest.mark.gpu
ACTS = ("silu", "gelu", "relu", "swiglu_oai")


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", [(3, 64, 34), (20, 256, 96), (300, 512, 768), (1000, 256, 2200), (40, 50, 26)])
def test_activation_keeps_a_nan(gpu, act, M, K, N):
    """A token with the scale NaN has NaN results under every activation (a clamp does not
    turn them into its limit), and so has a channel whose gate or up scale is NaN; all
    others are what they are without."""
    q, w = codes((M, K), 40, gpu), codes((N, K), 41, gpu)
    s, ws = scales((M,), 42, gpu) * 0.05, scales((N,), 43, gpu)
    ref = w8a8_linear(q, s, w, ws, activation=act, out_dtype=torch.float32)
    s[M // 2], ws[1], ws[N // 2 + 3] = math.nan, math.nan, math.nan
    got = w8a8_linear(q, s, w, ws, activation=act, out_dtype=torch.float32)
    bad = torch.zeros_like(ref, dtype=torch.bool)
    bad[M // 2], bad[:, 1], bad[:, 3] = True, True, True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], ref[~bad])


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [1, 6, 300])
def test_layers_keep_a_token_that_is_not_finite(gpu, act, T):
    """A token with an infinity or NaN leaves the expert and the expert layer as NaN."""
    x, w1, s1, w2, s2, ids, tw = moe_inputs(gpu, T, 8, 128, 64, 2, torch.bfloat16)
    for v in (math.inf, math.nan):
        x[T // 2, 5] = v
        out = fused_w8a8_moe(x, w1, s1, w2, s2, ids, tw, activation=act)
        one = fused_w8a8_expert_forward(x, w1[0], s1[0], w2[0], s2[0], intermediate=64, activation=act)
        for y in (out, one):
            nan = torch.isnan(y)
            assert nan[T // 2].all() and int(nan.sum()) == y.shape[1]

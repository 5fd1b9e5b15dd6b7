"""The norm, the grouped routing, their gradients and the adapters on the GPU at the edges of what their
description allows: values that are not finite, sums that cancel, scores next to each other at any size, workspaces
larger than a call needs."""
import numpy as np
import pytest
import torch

from test_gpu_expert_ops import blk, floats, say  # noqa: F401
from test_gpu_layer_ops import check_norm, run_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [16, 777, 7168, 9000, 36000])
@pytest.mark.parametrize("zero", [0.0, -0.0])
def test_norm_of_an_infinity_under_a_gain_of_zero(blk, H, zero):
    """The row has no scale, also where the gain takes the infinity out of every product but leaves a NaN."""
    say("norm inf under a zero gain", H, zero)
    rng = np.random.default_rng(H)
    for t in ("f32", "bf16", "f16"):
        x, w = floats(rng, (5, H), t), floats(rng, (H,), t)
        x[1, H // 3], x[3, H - 1] = float("inf"), float("-inf")
        w[H // 3], w[H - 1] = zero, zero
        got = run_norm(blk, x, None, w, t, True)
        assert torch.isnan(got["scale"][[1, 3]]).all() and not got["q"][[1, 3]].any()
        assert torch.isnan(got["y"][1, H // 3]) and torch.isnan(got["y"][3, H - 1])
        ok = [0, 2, 4]
        check_norm({k: v[ok] for k, v in got.items()}, x[ok], None, w)


@pytest.mark.parametrize("H", [24, 5000, 36000])
def test_norm_of_a_sum_past_the_type_under_a_gain_of_zero(blk, H):
    """x + residual is infinite in f16 alone: what is stored is what is normalised."""
    say("norm f16 sum past the type", H)
    rng = np.random.default_rng(H)
    x, res, w = floats(rng, (4, H), "f32"), floats(rng, (4, H), "f16"), floats(rng, (H,), "f16")
    x[2, 5], res[2, 5], w[5] = 40000.0, 40000.0, 0.0
    got = run_norm(blk, x, res, w, None, True)
    assert torch.isinf(got["total"][2, 5]) and torch.isnan(got["scale"][2]) and not got["q"][2].any()
    ok = [0, 1, 3]
    check_norm({k: v[ok] for k, v in got.items()}, x[ok], res[ok], w)

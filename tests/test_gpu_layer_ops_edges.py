"""The norm, the grouped routing, their gradients and the adapters on the GPU at the edges of what their
description allows: values that are not finite, sums that cancel, scores next to each other at any size, workspaces
larger than a call needs."""
import numpy as np
import pytest
import torch

from expert_ref import rounded
from test_gpu_expert_ops import blk, floats, say  # noqa: F401
from test_gpu_layer_ops import check_norm, run_norm, run_route

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


def groups_on_a_tie(rng, T):
    """(logits [T, 4], bias [4]): two groups of two experts with biases next to 64, whose c lie on roundings of f32
    (steps of u = 2^-17) and whose sums lie on roundings again (steps of 2u).  In units of u, n1 odd, n2 and n3
    even, n4 odd, n1 + n2 = n3 + n4 = 1 mod 4: c of n + 1/2 goes to the even neighbour, a hair above or below it to the
    nearer one, so that group 0 can come out two units too large and group 1 two too small."""
    n = np.array([65, 64, 64, 65])
    u = 2.0 ** -17
    m = (rng.uniform((0.5, 0.08, 0.5, 0.08), (0.95, 0.24, 0.95, 0.24)) / u).astype(np.int64)  # the score is (m + 1/2) u or so
    bias = ((2 ** 23 + 4 * n) - m) * u
    base = (bias / u + m).astype(np.int64)
    # parities as above, whatever m is
    for e, want in enumerate((1, 0, 0, 1)):
        if base[e] % 2 != want:
            bias[e] += u
            base[e] += 1
    bias[3] += (base[0] + base[1] - base[2] - base[3]) * u
    base[3] = base[0] + base[1] - base[2]
    if (base[0] + base[1]) % 4 != 1:
        bias[[1, 3]] += 2 * u
        base[[1, 3]] += 2
    assert base[0] % 2 == 1 and base[1] % 2 == 0 and base[2] % 2 == 0 and base[3] % 2 == 1
    assert base[0] + base[1] == base[2] + base[3] and (base[0] + base[1]) % 4 == 1
    assert (bias.astype(np.float32) == bias).all() and (np.abs(bias - 64) < 2).all()
    # the first of each group rounds to the tie from anywhere within half a step of its score, the second past it
    p = (m + 0.5) * u + rng.uniform(-1, 1, (T, 4)) * 2.0 ** -25
    return np.log(p / (1 - p)).astype(np.float32), bias.astype(np.float32)


def test_route_of_groups_on_a_tie_of_their_sums(blk):
    """The sum of two scores is rounded as well: what the comparison in 32 bits allows for has to hold it."""
    say("route group sums")
    rng, other = np.random.default_rng(31), 0
    args = (2, 1, 2, 1, 2, True, 1.0)
    one = np.float32(1)
    for _ in range(40):
        l, bias = groups_on_a_tie(rng, 5000)
        ids, _, _ = run_route(blk, torch.from_numpy(l), bias, *args)
        two = (1 / (1 + np.exp(-l.astype(np.float64))) + bias).reshape(-1, 2, 2).sum(2)
        c32 = (one / (one + np.exp(-l))).astype(np.float32) + bias
        over = c32[:, :2].sum(1) - c32[:, 2:].sum(1)
        other += ((over >= 2.0 ** -15) & (two[:, 0] < two[:, 1])).sum()  # two steps of the sums apart, and the other way round
        clear = np.abs(two[:, 0] - two[:, 1]) > 1e-12
        assert (ids[clear].min(1) // 2 == (two[:, 1] > two[:, 0])[clear]).all()
    assert other

"""The norm, the grouped routing, their gradients and the adapters on the GPU at the edges of what their
description allows: values that are not finite, sums that cancel, scores next to each other at any size, workspaces
larger than a call needs."""
import numpy as np
import pytest
import torch

import layer_ref as ref
from expert_ref import TYPES, U, rounded
from test_gpu_expert_ops import blk, close, dev, floats, say  # noqa: F401
from test_gpu_layer_ops import DEV, EPS, check_norm, run_norm, run_route, zeros

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


def test_a_workspace_serves_every_smaller_call(blk):
    """What a call needs grows with each size, so that one workspace for the largest of them does for all."""
    say("workspaces")
    rng = np.random.default_rng(41)
    most = blk.adapters_scratch
    sizes = sorted(set([1, 2, 16, 63, 64, 65, 128, 1000, 4000, 4064, 4095, 4096, 4097, 8160, 8192, 20000]
                       + rng.integers(1, 20000, 60).tolist()))
    for K in (64, 1000, 7168, 100000):
        for R in (1, 8, 16, 17, 32, 33, 64, 65, 1024):
            need = [most(M, K, R) for M in sizes]
            assert all(a <= b for a, b in zip(need, need[1:])), (K, R)
    for M in sizes:
        need = [most(M, K, 16) for K in (1, 63, 64, 1000, 1024, 1025, 7168, 50000)]
        assert all(a <= b for a, b in zip(need, need[1:])), M
        need = [most(M, 7168, R) for R in (1, 15, 16, 17, 32, 33, 64, 65, 128, 1024)]
        assert all(a <= b for a, b in zip(need, need[1:])), M
    widths = (1, 64, 128, 129, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 40000, 2 ** 30)
    for T in (1, 3, 64, 255, 256, 257, 5000, 10 ** 6):
        need = [blk.rms_norm_grad_scratch(T, H) for H in widths]
        assert all(a <= b for a, b in zip(need, need[1:])), T
    for H in widths:
        need = [blk.rms_norm_grad_scratch(T, H) for T in sizes]
        assert all(a <= b for a, b in zip(need, need[1:])), H


@pytest.mark.parametrize("R", [16, 64])
def test_adapters_of_a_smaller_batch_in_the_largest_ones_workspace(blk, R):
    say("adapters, one workspace", R)
    rng = np.random.default_rng(R)
    K, N, n, top = 7168, 64, 3, 4096
    mid = torch.full((blk.adapters_scratch(top, K, R) + 3,), float("nan"), device=DEV)
    x, base = floats(rng, (top, K), "bf16"), floats(rng, (top, N), "f32")
    a = (torch.from_numpy(rng.standard_normal((n, R, K)).astype(np.float32)) / K ** 0.5).bfloat16()
    b = (torch.from_numpy(rng.standard_normal((n, N, R)).astype(np.float32)) / R ** 0.5).bfloat16()
    xd, ad, bd = dev(x), dev(a), dev(b)
    for M in (4096, 4064, 2049, 2000, 100, 65, 64, 1):
        of = np.sort(rng.integers(0, n, M)).astype(np.int32)
        counts, offsets, perm = zeros(n, dtype=torch.int32), zeros(n + 1, dtype=torch.int32), zeros(M, dtype=torch.int32)
        blk.group(dev(of[:, None]), n, counts, offsets, perm)
        out = zeros(M, N)
        blk.adapters(xd[:M], ad, bd, None, offsets, perm, dev(base[:M]), out, mid[:-3])
        some = sorted(set([0, M // 3, M // 2, M - 1]))
        want, bound = ref.adapters(x[some], a, b, None, torch.from_numpy(of)[some], base[some], torch.float32)
        close(out.cpu()[some], want, bound)
    assert torch.isnan(mid[-3:]).all()


def test_norm_gradients_in_the_largest_ones_workspace(blk):
    say("norm_grad, one workspace")
    rng = np.random.default_rng(43)
    part = torch.full((blk.rms_norm_grad_scratch(300, 20000) + 3,), float("nan"), device=DEV)
    for T, H in ((300, 20000), (300, 16384), (300, 16385), (299, 8192), (40, 9000), (300, 64), (1, 20000)):
        dy, h, w = floats(rng, (T, H), "f32"), floats(rng, (T, H), "f32"), floats(rng, (H,), "f32")
        rstd = ref.norm(h, w, EPS)[1].float()
        dx, dw = zeros(T, H), zeros(H)
        blk.rms_norm_grad(dev(dy), dev(h), dev(w), dev(rstd), dx, dw, part[:-3])
        wx, ww, ex, ew = ref.norm_grad(dy, h, w, rstd, None)
        close(dx, wx, rounded(ex, wx, torch.float32))
        close(dw, ww, ew + 1e-40)
    assert torch.isnan(part[-3:]).all()


def test_gain_gradient_of_long_rows_and_many(blk):
    """Terms of one sign that f32 rounds the same way at each addition: a sum along all the rows would be off by far
    more than one of parts."""
    say("dw of long rows, many rows")
    T, H = 8000, 16392
    v = 1.0 + 2.0 ** -14 - 2.0 ** -20
    dy, h = torch.full((T, H), v, device=DEV), torch.ones((T, H), device=DEV)
    dx, dw = torch.empty((T, H), device=DEV), zeros(H)
    blk.rms_norm_grad(dy, h, torch.ones(H, device=DEV), torch.ones(T, device=DEV), dx, dw,
                      zeros(blk.rms_norm_grad_scratch(T, H)))
    want = torch.full((H,), T * v, dtype=torch.float64)
    close(dw, want, (ref.chain(T) + 3) * U * want)


@pytest.mark.parametrize("T, H", [(700, 16386), (2500, 17001)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_norm_grad_of_long_rows(blk, T, H, kind):
    say("norm_grad long", T, H, kind)
    rng = np.random.default_rng(T)
    dy, h, w = floats(rng, (T, H), kind), floats(rng, (T, H), kind), floats(rng, (H,), "f32")
    rstd = ref.norm(h, w, EPS)[1].float()
    dx, dw = zeros(T, H, dtype=TYPES[kind]), zeros(H)
    blk.rms_norm_grad(dev(dy), dev(h), dev(w), dev(rstd), dx, dw, zeros(blk.rms_norm_grad_scratch(T, H)))
    wx, ww, ex, ew = ref.norm_grad(dy, h, w, rstd, None)
    close(dx, wx, rounded(ex, wx, TYPES[kind]))
    close(dw, ww, ew + 1e-40)


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_route_grad_of_picks_with_a_score_that_is_no_number(blk, mode, what):
    """Weights divided by a sum that is NaN (or by an infinite one) have no gradient: neither has the sum's floor."""
    say("route_grad nan", mode, what)
    rng = np.random.default_rng(51)
    T, E, k = 6, 40, 4
    l, dwts = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, k)).astype(np.float32)
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.int32)
    l[2, ids[2, 1]] = what
    dl = zeros(T, E)
    blk.route_grad(dev(l), dev(ids), dev(dwts), mode, True, 1.5, dl)
    got = dl.cpu().double().numpy()
    with np.errstate(all="ignore"):
        want, bound = ref.route_grad(l, ids, dwts, None, mode, True, 1.5)
    ok = [0, 1, 3, 4, 5]
    close(torch.from_numpy(got[ok]), torch.from_numpy(want[ok]), torch.from_numpy(bound[ok]))
    rest = np.setdiff1d(np.arange(E), ids[2])
    assert (got[2, rest] == 0).all()
    if mode == 1 and what == float("inf"):  # a score of 1
        close(torch.from_numpy(got[2]), torch.from_numpy(want[2]), torch.from_numpy(bound[2]))
    else:
        assert np.isnan(got[2, ids[2]]).all(), got[2, ids[2]]


EXACT = [(40, 24, 2, 40, 3), (17, 100, 5, 33, 4), (300, 64, 24, 200, 2), (2100, 64, 8, 7000, 3), (2100, 64, 64, 7000, 3)]


@pytest.mark.parametrize("M, K, R, N, n", EXACT)
@pytest.mark.parametrize("out", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("x", ["bf16", "f16"])
def test_adapters_whose_products_cancel(blk, M, K, R, N, n, out, x):
    """Pairs of A x that agree to 16 bits and are subtracted by B: what is left is in the last 8 bits of 24.  A x is
    a + b / 2^8 + c / 2^16 with whole numbers below 2^7, exact in f32 in any order."""
    say("adapters cancel", M, K, R, N, n, out, x)
    rng = np.random.default_rng(M + R)
    t, pairs = TYPES[x], R // 2
    xs = torch.zeros((M, K))
    xs[:, 3], xs[:, 9], xs[:, K - 1] = 1.0, 2.0 ** -8, 2.0 ** -16 if x == "bf16" else 2.0 ** -14
    a = torch.zeros((n, R, K))
    head = torch.from_numpy(rng.integers(64, 128, (n, pairs, 2)).astype(np.float32))
    for half in (0, 1):  # rows 0 .. pairs, and pairs .. 2 pairs: the same but for the last numbers
        at = slice(half * pairs, (half + 1) * pairs)
        a[:, at, 3], a[:, at, 9] = head[:, :, 0], head[:, :, 1]
        a[:, at, K - 1] = torch.from_numpy(rng.integers(0, 128, (n, pairs)).astype(np.float32))
    b = torch.zeros((n, N, R))
    sign = torch.from_numpy(rng.choice([-1.0, 1.0], (n, N, pairs)).astype(np.float32))
    b[:, :, :pairs], b[:, :, pairs:2 * pairs] = sign, -sign
    of = np.sort(rng.integers(0, n, M)).astype(np.int32)
    base = torch.zeros((M, N), dtype=TYPES[out])
    counts, offsets, perm = zeros(n, dtype=torch.int32), zeros(n + 1, dtype=torch.int32), zeros(M, dtype=torch.int32)
    blk.group(dev(of[:, None]), n, counts, offsets, perm)
    got = zeros(M, N, dtype=TYPES[out])
    blk.adapters(dev(xs.to(t)), dev(a.to(t)), dev(b.to(t)), None, offsets, perm, dev(base), got,
                 zeros(blk.adapters_scratch(M, K, R)))
    which = torch.from_numpy(of).long()
    mid = torch.stack([a[i].double() @ xs[0].double() for i in range(n)])  # every row of x is the same
    want = torch.stack([b[i].double() @ mid[i] for i in range(n)])[which]
    mag = torch.stack([b[i].double().abs() @ mid[i].abs() for i in range(n)])[which]
    # the sum over R: R + 2 additions
    close(got, want, rounded((R + 2) * U * mag, want, TYPES[out]))


@pytest.mark.parametrize("M, N", [(5, 40), (2100, 7000)])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_adapters_with_products_next_to_the_largest_value(blk, M, N, out):
    """A x within f32 but past the largest value of bf16, times a small B."""
    say("adapters largest", M, N, out)
    K, R = 64, 8
    x, a, b = torch.zeros((M, K)), torch.zeros((1, R, K)), torch.zeros((1, N, R))
    x[:, 1], x[:, 40] = 2.0 ** 64, 2.0 ** 60
    a[0, :, 1], a[0, :, 40] = (2 - 2.0 ** -7) * 2.0 ** 63, 1.5 * 2.0 ** 59
    b[0, :, 5] = 2.0 ** -100
    offsets, perm = torch.tensor([0, M], dtype=torch.int32), torch.arange(M, dtype=torch.int32)
    got = zeros(M, N, dtype=TYPES[out])
    blk.adapters(dev(x.bfloat16()), dev(a.bfloat16()), dev(b.bfloat16()), None, dev(offsets), dev(perm),
                 torch.zeros((M, N), dtype=TYPES[out], device=DEV), got, zeros(blk.adapters_scratch(M, K, R)))
    v = ((2 - 2.0 ** -7) * 2.0 ** 127 + 1.5 * 2.0 ** 119) * 2.0 ** -100
    want = torch.full((M, N), v, dtype=torch.float64)
    close(got, want, rounded((R + 2) * U * want, want, TYPES[out]))


def same(got, want, bound):
    """Numbers within the bound; infinities and NaN the same."""
    got, want = got.double().numpy(), np.asarray(want, np.float64)
    assert (np.isnan(got) == np.isnan(want)).all() and (np.isinf(got) == np.isinf(want)).all()
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all()
    ok = np.isfinite(want)
    assert (np.abs(got - want)[ok] <= np.broadcast_to(bound, want.shape)[ok]).all()


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("n_group, keep, top", [(1, 1, 1), (4, 2, 1), (8, 3, 2), (6, 2, 2)])
@pytest.mark.parametrize("biased", [False, True])
def test_route_of_scores_that_are_no_numbers(blk, mode, n_group, keep, top, biased):
    """NaN, infinities and the largest values among the logits and the biases: every row's picks, weights and scores."""
    say("route not finite", mode, n_group, keep, top, biased)
    rng = np.random.default_rng(61)
    T, E, k = 24, 48, 5
    l = rng.standard_normal((T, E)).astype(np.float32)
    high = np.finfo(np.float32).max
    l[0, 3], l[1, 9], l[2, 1], l[3, 2], l[4] = np.inf, np.nan, high, -high, np.nan
    l[5, :46] = -np.inf
    l[5, 46] = np.nan
    l[6, ::2] = np.nan
    l[7, 5:9] = np.inf
    l[8, 4], l[8, 5] = np.inf, np.nan
    l[9, ::3] = -np.inf
    l[10] = -np.inf
    l[11, 1:] = -high
    l[12, :44] = np.nan  # fewer numbers than picks
    bias = None
    if biased:
        bias = (0.3 * rng.standard_normal(E)).astype(np.float32)
        bias[[7, 20, 33]] = np.nan, -np.inf, -np.inf
        bias[13], bias[40] = np.inf, high
    with np.errstate(all="ignore"):
        args = (k, mode, n_group, keep, top, True, 1.5)
        want_ids, want_w, p = ref.route(l, bias, *args)
        half = ref.score_half_steps(np.clip(l.astype(np.float64), -200, 200), mode)
    ids, wts, sc = run_route(blk, torch.from_numpy(l), bias, *args)
    assert (ids == want_ids).all(), np.nonzero((ids != want_ids).any(1))[0]
    with np.errstate(all="ignore"):
        same(sc, p, half * U * np.abs(p) + 1e-37)
        same(wts, want_w, (2 * half + k + 6) * U * np.abs(want_w) + 1e-37)


@pytest.mark.parametrize("M, K, R, N, n", [(40, 512, 16, 64, 3), (300, 520, 64, 264, 2), (2100, 64, 32, 7000, 3)])
@pytest.mark.parametrize("x, out", [("f16", "f32"), ("bf16", "f32"), ("f16", "bf16"), ("bf16", "f16"), ("f32", "f32")])
def test_adapters_keep_what_f32_keeps(blk, M, K, R, N, n, x, out):
    """Rows of very different size, A x past f16's range: no value is off by more than its own f32 sums are."""
    say("adapters in 24 bits", M, K, R, N, n, x, out)
    rng = np.random.default_rng(M + K)
    t = TYPES[x]
    xs = (floats(rng, (M, K), "f32") * torch.from_numpy(4.0 ** rng.integers(-5, 7, (M, 1))).float()).to(t)
    a = (64 * torch.from_numpy(rng.standard_normal((n, R, K)).astype(np.float32)) / K ** 0.5).to(t)
    b = (torch.from_numpy(rng.standard_normal((n, N, R)).astype(np.float32)) / R ** 0.5 / 1024).to(t)
    of, base = np.sort(rng.integers(0, n, M)).astype(np.int32), floats(rng, (M, N), out)
    counts, offsets, perm = zeros(n, dtype=torch.int32), zeros(n + 1, dtype=torch.int32), zeros(M, dtype=torch.int32)
    blk.group(dev(of[:, None]), n, counts, offsets, perm)
    got = zeros(M, N, dtype=TYPES[out])
    blk.adapters(dev(xs), dev(a), dev(b), None, offsets, perm, dev(base), got, zeros(blk.adapters_scratch(M, K, R)))
    # sums over K as in layer_ref.py, over R R + 10 half steps, nothing for a cutting of A x
    want, bound = base.double(), torch.zeros((M, N), dtype=torch.float64)
    for i in range(n):
        r = torch.from_numpy(np.nonzero(of == i)[0])
        X, A, B = xs[r].double(), a[i].double(), b[i].double()
        mid, err = X @ A.t(), (K / 16 + 40) * U * (X.abs() @ A.abs().t())
        want[r] += mid @ B.t()
        e = err @ B.abs().t() + (R + 10) * U * ((mid.abs() + err) @ B.abs().t())
        bound[r] = e + U * (want[r].abs() + e)
    close(got, want, rounded(bound, want, TYPES[out]))


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("keep, k", [(1, 2), (2, 3), (3, 6)])
def test_route_of_groups_with_the_lowest_value_beside_a_large_one(blk, mode, keep, k):
    """A bias of f32's lowest value is a number, and a sum with it may be any number, or an infinity."""
    say("route lowest value", mode, keep, k)
    rng = np.random.default_rng(71)
    high = np.finfo(np.float32).max
    bias = np.array([1, 1, np.inf, -high, 3e38, -high, -1e38, -1e38], np.float32)
    for order in (range(4), (2, 0, 3, 1), (3, 2, 1, 0)):
        b = bias.reshape(4, 2)[list(order)].reshape(-1)
        l = torch.from_numpy(rng.standard_normal((7, 8)).astype(np.float32))
        args = (k, mode, 4, keep, 2, False, 1.0)
        ids, wts, _ = run_route(blk, l, b, *args)
        want_ids, want_w, p = ref.route(l.numpy(), b, *args)
        assert (ids == want_ids).all()
        w = torch.from_numpy(want_w)
        close(wts, w, torch.from_numpy(ref.score_half_steps(l.double().numpy(), mode)) * U * w + 1e-37)

"""The norm, the grouped routing, their gradients and the adapters on the GPU, against 64-bit
statements of them (layer_ref.py) with the error bounds that f32 arithmetic and the
output's rounding allow."""
import threading

import numpy as np
import pytest
import torch

import expert_ref
import layer_ref as ref
import moe_block as mb
from expert_ref import TYPES, U, rounded
from test_gpu_expert_ops import blk, close, dev, floats, say  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6


def zeros(*shape, dtype=torch.float32):
    return torch.full(shape, 7, dtype=dtype, device=DEV)


# ---- norm --------------------------------------------------------------------------------


def run_norm(blk, x, res, w, y_type=None, i8=False, eps=EPS, in_place=False):
    T, H = x.shape
    xd, wd, rd = dev(x), dev(w), None if res is None else dev(res)
    got = dict(rstd=zeros(T))
    if y_type:
        got["y"] = zeros(T, H, dtype=TYPES[y_type])
    if i8:
        got.update(q=zeros(T, H, dtype=torch.int8), scale=zeros(T))
    if res is not None:
        got["total"] = rd if in_place else zeros(T, H, dtype=res.dtype)
    blk.rms_norm(xd, wd, eps, residual=rd, **got)
    return {k: v.cpu() for k, v in got.items()}


def check_norm(got, x, res, w, eps=EPS):
    h = ref.total(x, res)
    if res is not None:
        assert torch.equal(got["total"], h)
    y, r = ref.norm(h, w, eps)
    close(got["rstd"], r, 1.01 * U * r + 1e-45)
    if "y" in got:
        close(got["y"], y, ref.norm_bound(y, got["y"].dtype))
    if "q" in got:
        q, scale = ref.codes(y)
        assert torch.equal(got["scale"], scale)
        assert torch.equal(got["q"], q)


NORM_SIZES = [(1, 1), (1, 7168), (3, 7), (2, 64), (5, 129), (33, 513), (130, 1000), (4, 2048), (9, 5121), (700, 256),
              (2, 8200), (3, 16385), (2, 40000), (1030, 96), (600, 2049)]


@pytest.mark.parametrize("T, H", NORM_SIZES)
@pytest.mark.parametrize("x, res, w, y, i8", [
    ("f32", None, "f32", "f32", False), ("bf16", "bf16", "bf16", "bf16", False), ("f16", "f16", "f16", "f16", True),
    ("bf16", "f32", "f32", "bf16", True), ("f32", "bf16", "f16", "f16", False), ("bf16", None, "bf16", None, True),
    ("f32", "f32", "f32", None, True), ("f16", None, "f32", "f32", True)])
def test_norm(blk, T, H, x, res, w, y, i8):
    say("norm", T, H, x, res, w, y, i8)
    rng = np.random.default_rng(T + H)
    xs, rs = floats(rng, (T, H), x), None if res is None else floats(rng, (T, H), res)
    ws = (1 + 0.3 * floats(rng, (H,), "f32")).to(TYPES[w])
    check_norm(run_norm(blk, xs, rs, ws, y, i8), xs, rs, ws)


@pytest.mark.parametrize("H", [5, 264, 7168, 33000])
def test_norm_in_place_of_the_residual(blk, H):
    say("norm in place", H)
    rng = np.random.default_rng(H)
    for t in ("f32", "bf16"):
        xs, rs, ws = floats(rng, (6, H), t), floats(rng, (6, H), t), floats(rng, (H,), t)
        check_norm(run_norm(blk, xs, rs, ws, t, True, in_place=True), xs, rs, ws)


@pytest.mark.parametrize("H", [31, 500, 2048, 9000, 34000])
def test_norm_of_rows_at_the_ends_of_the_range(blk, H):
    """Rows of zeros, of the largest and the smallest values, with one value far from the others."""
    say("norm ends", H)
    rng = np.random.default_rng(H)
    x = floats(rng, (8, H), "f32")
    x[0] = 0.0
    x[1] *= 1e37
    x[2] *= 1e-38
    x[3] = 0.0
    x[3, H // 2] = -5.0
    x[4, H - 1] = 1e30
    x[5] *= 1e-41
    x[6] = 3e38
    w = 1 + 0.1 * floats(rng, (H,), "f32")
    for eps in (1e-5, 1.2e-38):
        got = run_norm(blk, x, None, w, "f32", True, eps)
        y, r = ref.norm(x, w, eps)
        # r below 2^-126 keeps 22 bits or more.  Half the step of the smallest values is 2^-150: h * r may be off by
        # it, w times that after the second product, which adds another
        bound = (3.01 * U + 2.0 ** -22) * y.abs() + 2.0 ** -150 * (1 + w.abs().double())
        close(got["y"], y, bound)
        close(got["rstd"], r, 1.01 * U * r + 2.0 ** -149)
        q, scale = ref.codes(y)
        assert torch.equal(got["q"], q) and torch.equal(got["scale"], scale)
    assert not got["q"][0].any() and got["scale"][0] == 0


@pytest.mark.parametrize("H", [16, 777, 7168, 36000])
def test_norm_of_rows_without_a_norm(blk, H):
    """A row with a NaN or an infinity has no scale, and leaves the other rows alone."""
    say("norm nan", H)
    rng = np.random.default_rng(H)
    for t in ("f32", "bf16", "f16"):
        x, w = floats(rng, (5, H), t), floats(rng, (H,), t)
        x[1, H // 3], x[3, H - 1] = float("nan"), float("-inf")
        got = run_norm(blk, x, None, w, t, True)
        assert torch.isnan(got["scale"][[1, 3]]).all() and not got["q"][[1, 3]].any()
        assert torch.isnan(got["y"][1]).all() and torch.isnan(got["y"][3, H - 1])
        ok = [0, 2, 4]
        check_norm({k: v[ok] for k, v in got.items()}, x[ok], None, w)


@pytest.mark.parametrize("H", [16, 777, 7168, 36000])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_norm_with_a_gain_that_is_not_finite(blk, H, what):
    """Every row has such a value, so none has a scale."""
    say("norm gain", H, what)
    rng = np.random.default_rng(H)
    x, w = floats(rng, (5, H), "bf16"), floats(rng, (H,), "f32")
    w[H // 2] = what
    got = run_norm(blk, x, None, w, "f32", True)
    assert torch.isnan(got["scale"]).all() and not got["q"].any()
    ok = [i for i in range(H) if i != H // 2]
    y, _ = ref.norm(x, w, EPS)
    close(got["y"][:, ok], y[:, ok], ref.norm_bound(y[:, ok], torch.float32))
    assert not torch.isfinite(got["y"][:, H // 2]).any()


def test_codes_next_to_a_tie(blk):
    """Values whose quotients lie at a half and next to it: decided as in 64 bits."""
    say("ties")
    rng = np.random.default_rng(3)
    for H in (254, 2032, 8128):
        k = torch.from_numpy(rng.integers(-127, 127, (16, H)).astype(np.float64)) + 0.5
        x = (k * torch.from_numpy(1 + rng.integers(-2, 3, (16, H)) * 2.0 ** -23)).float()
        x[:, 0] = 127.0
        w = torch.ones(H)
        got = run_norm(blk, x, None, w, None, True)
        y, _ = ref.norm(x, w, EPS)
        q, scale = ref.codes(y)
        assert torch.equal(got["scale"], scale) and torch.equal(got["q"], q)


@pytest.mark.parametrize("off", [1, 3])
def test_norm_at_odd_addresses(blk, off):
    say("norm odd", off)
    rng = np.random.default_rng(off)
    T, H = 5, 333
    for t in ("bf16", "f32"):
        xs, rs, ws = (floats(rng, s, t) for s in ((T, H), (T, H), (H,)))

        def at(v):
            buf = torch.zeros(v.numel() + off, dtype=v.dtype, device=DEV)[off:]
            buf.copy_(v.reshape(-1))
            return buf.view(v.shape)

        got = dict(total=at(torch.zeros(T, H, dtype=TYPES[t])), y=at(torch.zeros(T, H, dtype=TYPES[t])),
                   q=at(torch.zeros(T, H, dtype=torch.int8)), scale=at(torch.zeros(T)), rstd=at(torch.zeros(T)))
        blk.rms_norm(at(xs), at(ws), EPS, residual=at(rs), **got)
        check_norm({k: v.cpu() for k, v in got.items()}, xs, rs, ws)


GRAD_SIZES = [(1, 1), (1, 7168), (3, 7), (33, 513), (130, 1000), (257, 2048), (9, 5121), (700, 256), (4100, 64), (3, 9000),
              (5, 16390), (2, 33000), (1030, 97), (2500, 24), (66, 4096)]


def run_norm_grad(blk, dy, h, w, rstd, dres, dx_type, in_place=False):
    T, H = dy.shape
    dx = dev(dres) if in_place else zeros(T, H, dtype=TYPES[dx_type])
    dw, part = zeros(H), torch.full((blk.rms_norm_grad_scratch(T, H) + 3,), float("nan"), device=DEV)
    d = dx if in_place else None if dres is None else dev(dres)
    blk.rms_norm_grad(dev(dy), dev(h), dev(w), dev(rstd), dx, dw, part[:-3], dres=d)
    assert torch.isnan(part[-3:]).all()  # nothing past the workspace
    return dx, dw


@pytest.mark.parametrize("T, H", GRAD_SIZES)
@pytest.mark.parametrize("dy, h, w, dx, dres", [
    ("f32", "f32", "f32", "f32", False), ("bf16", "bf16", "bf16", "bf16", True), ("f16", "f32", "f32", "f16", True),
    ("f32", "bf16", "f16", "f32", True), ("bf16", "f16", "bf16", "f32", False)])
def test_norm_grad(blk, T, H, dy, h, w, dx, dres):
    say("norm_grad", T, H, dy, h, w, dx, dres)
    rng = np.random.default_rng(T + 3 * H)
    dys, hs = floats(rng, (T, H), dy), floats(rng, (T, H), h)
    ws = (1 + 0.3 * floats(rng, (H,), "f32")).to(TYPES[w])
    rs = floats(rng, (T, H), dx) if dres else None
    rstd = ref.norm(hs, ws, EPS)[1].float()
    wx, ww, ex, ew = ref.norm_grad(dys, hs, ws, rstd, rs)
    for in_place in ([False, True] if dres else [False]):
        gx, gw = run_norm_grad(blk, dys, hs, ws, rstd, rs, dx, in_place)
        close(gx, wx, rounded(ex, wx, TYPES[dx]))
        close(gw, ww, ew + 1e-40)


def test_norm_grad_is_the_same_each_time(blk):
    say("norm_grad again")
    rng = np.random.default_rng(8)
    T, H = 1500, 768
    dy, h, w = floats(rng, (T, H), "f32"), floats(rng, (T, H), "f32"), floats(rng, (H,), "f32")
    rstd = ref.norm(h, w, EPS)[1].float()
    first = run_norm_grad(blk, dy, h, w, rstd, None, "f32")
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run_norm_grad(blk, dy, h, w, rstd, None, "f32")))


@pytest.mark.parametrize("T, H", [(4, 24), (3, 300)])
def test_norm_gradient_is_that_of_differences(blk, T, H):
    """The kernel's loss along a direction, a step to either side, against the gradient's product with it: off by
    what the same difference is off in 64 bits (the curvature), and by the roundings of the two losses over the step."""
    say("norm differences", T, H)
    rng = np.random.default_rng(H)
    h, w, dout, dh, dw = (floats(rng, s, "f32") for s in ((T, H), (H,), (T, H), (T, H), (H,)))
    step = 2.0 ** -7

    def loss(sign, kernel):
        hh, ww = h + sign * step * dh, w + sign * step * dw
        y = run_norm(blk, hh, None, ww, "f32")["y"].double() if kernel else ref.norm(hh, ww, EPS)[0]
        return (y * dout.double()).sum()

    rstd = ref.norm(h, w, EPS)[1].float()
    gx, gw = run_norm_grad(blk, dout, h, w, rstd, None, "f32")
    got = (gx.cpu().double() * dh.double()).sum() + (gw.cpu().double() * dw.double()).sum()
    by_kernel, in_64 = ((loss(1, k) - loss(-1, k)) / (2 * step) for k in (True, False))
    wx, ww, ex, ew = ref.norm_grad(dout, h, w, rstd, None)
    exact = (wx * dh.double()).sum() + (ww * dw.double()).sum()
    y = ref.norm(h, w, EPS)[0]
    # y changes by a few steps between the two sides: twice its size at the middle covers them
    noise = 2 * 2 * (3.01 * U * y.abs() * dout.abs().double()).sum() / (2 * step)
    grad_err = (ex * dh.abs().double()).sum() + (ew * dw.abs().double()).sum()
    assert abs(by_kernel - got) <= abs(in_64 - exact) + noise + grad_err


# ---- routing -------------------------------------------------------------------------------


def logits_of(rng, T, E, kind, masked):
    l = torch.from_numpy((2 * rng.standard_normal((T, E))).astype(np.float32))
    if masked:
        l[torch.from_numpy(rng.random((T, E)) < masked)] = float("-inf")
        l[T // 2] = float("-inf")
    return l.to(TYPES[kind])


def run_route(blk, l, bias, k, mode, n_group, keep, top, norm, scale):
    T, E = l.shape
    ids, wts, sc = zeros(T, k, dtype=torch.int32), zeros(T, k), zeros(T, E)
    blk.route_groups(dev(l), k, mode, norm, scale, ids, wts, bias=None if bias is None else dev(bias), n_group=n_group,
                     keep=keep, top=top, scores=sc)
    again = zeros(T, k, dtype=torch.int32), zeros(T, k)
    blk.route_groups(dev(l), k, mode, norm, scale, *again, bias=None if bias is None else dev(bias), n_group=n_group,
                     keep=keep, top=top)
    # with and without the scores
    assert torch.equal(again[0], ids) and torch.equal(again[1].nan_to_num(nan=-9.0), wts.nan_to_num(nan=-9.0))
    return ids.cpu().numpy(), wts.cpu(), sc.cpu()


def check_route(got, l, bias, k, mode, n_group, keep, top, norm, scale):
    ids, wts, sc = got
    L = l.float().numpy()
    want_ids, want_w, p = ref.route(L, bias, k, mode, n_group, keep, top, norm, scale)
    assert (ids == want_ids).all(), np.nonzero((ids != want_ids).any(1))[0][:5]
    half = torch.from_numpy(ref.score_half_steps(L.astype(np.float64), mode))
    close(sc, torch.from_numpy(p), half * U * torch.from_numpy(p) + 1e-37)
    w = torch.from_numpy(want_w)
    close(wts, w, (2 * half + k + 6) * U * w.abs() + 1e-37)


ROUTE = [(1, 256, 8, 8, 4), (1, 1, 1, 1, 1), (3, 7, 7, 1, 1), (37, 32, 4, 1, 1), (300, 256, 8, 8, 4), (50, 160, 6, 8, 3),
         (20, 160, 20, 8, 1), (40, 60, 3, 12, 5), (9, 384, 6, 1, 1), (11, 1024, 10, 16, 4), (5, 1000, 64, 4, 4), (33, 64, 8, 64, 8),
         (33, 65, 5, 5, 2), (70, 96, 8, 3, 2), (64, 130, 5, 2, 1), (6, 256, 2, 32, 32), (10, 513, 64, 1, 1)]


@pytest.mark.parametrize("T, E, k, n_group, keep", ROUTE)
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kind, bias, top, norm, scale, masked", [
    ("f32", True, 2, True, 2.5, 0.0), ("bf16", False, 1, True, 1.0, 0.0), ("f16", True, 1, False, 0.0, 0.3),
    ("f32", False, 2, True, 1.0, 0.8), ("bf16", True, 2, True, -0.5, 0.5)])
def test_route(blk, T, E, k, n_group, keep, mode, kind, bias, top, norm, scale, masked):
    say("route", T, E, k, n_group, keep, mode, kind, bias, top, norm, scale, masked)
    rng = np.random.default_rng(T + E + mode)
    l = logits_of(rng, T, E, kind, masked)
    b = (0.2 * rng.standard_normal(E)).astype(np.float32) if bias else None
    args = (k, mode, n_group, keep, top, norm, scale)
    check_route(run_route(blk, l, b, *args), l, b, *args)


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("n_group, keep, top", [(1, 1, 1), (8, 3, 2), (4, 2, 1)])
def test_route_ties_go_to_the_lowest_index(blk, mode, n_group, keep, top):
    say("route ties", mode, n_group)
    rng = np.random.default_rng(n_group)
    for E in (32, 256, 640):
        l = torch.from_numpy(rng.integers(-2, 3, (40, E)).astype(np.float32))
        l[0] = 0.0
        b = rng.integers(0, 2, E).astype(np.float32)
        for bias in (None, b):
            args = (8, mode, n_group, keep, top, True, 1.0)
            check_route(run_route(blk, l, bias, *args), l, bias, *args)


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("n_group, keep, top", [(1, 1, 1), (8, 3, 2), (8, 3, 1), (5, 2, 2)])
@pytest.mark.parametrize("alike", [2, 5, 20, 160])
def test_route_of_scores_closer_than_32_bits_tell(blk, mode, n_group, keep, top, alike):
    """Biases that bring some experts' scores within a rounding of each other: the order in 32 bits is another than
    in 64 for some tokens (which the test checks of its inputs), and the one in 64 holds."""
    say("route close", mode, n_group, keep, top, alike)
    rng = np.random.default_rng(alike + mode)
    E, args = 160, (8, mode, n_group, keep, top, True, 1.0)
    other = 0
    for _ in range(6):
        l = rng.standard_normal((1, E)).astype(np.float32)
        p = ref.scores(l.astype(np.float64), mode)[0]
        bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
        some = rng.permutation(E)[:alike]
        bias[some] = (2.0 - p[some]).astype(np.float32)
        check_route(run_route(blk, torch.from_numpy(l), bias, *args), torch.from_numpy(l), bias, *args)
        c32 = p[some].astype(np.float32) + bias[some]
        other += (np.argsort(-c32, kind="stable") != np.argsort(-(p[some] + bias[some].astype(np.float64)), kind="stable")).any()
    assert other


def test_route_where_the_last_pick_is_close_to_the_next(blk):
    """Of 100 experts well apart, the k-th and the next within a rounding; as many picks as a wave has lanes, and fewer."""
    say("route last pick")
    rng = np.random.default_rng(21)
    for k in (1, 5, 63, 64):
        other = 0
        for _ in range(12):
            l = rng.standard_normal((1, 100)).astype(np.float32)
            p = ref.scores(l.astype(np.float64), 1)[0]
            place = rng.permutation(100)
            target = 2.0 - 0.01 * place
            target[place == k] = target[place == k - 1]  # the expert after the k-th
            bias = (target - p).astype(np.float32)
            args = (k, 1, 1, 1, 1, True, 1.0)
            check_route(run_route(blk, torch.from_numpy(l), bias, *args), torch.from_numpy(l), bias, *args)
            c = p + bias.astype(np.float64)
            other += (np.argsort(-c, kind="stable") != np.argsort(-(p.astype(np.float32) + bias), kind="stable")).any()
        assert other


def test_route_takes_the_two_zeros_as_equal(blk):
    say("route zeros")
    rng = np.random.default_rng(22)
    for n_group, keep in ((1, 1), (4, 2)):
        l = torch.from_numpy(rng.choice([-0.0, 0.0, -1.0], (30, 64)).astype(np.float32))
        for bias in (None, rng.choice([-0.5, -0.0, 0.0], 64).astype(np.float32)):
            for mode in (0, 1, 2):
                args = (6, mode, n_group, keep, 1, False, 1.0)
                check_route(run_route(blk, l, bias, *args), l, bias, *args)


def test_route_of_groups_closer_than_32_bits_tell(blk):
    """Groups whose two best scores sum to within a rounding of the same."""
    say("route groups close")
    rng = np.random.default_rng(11)
    E, G, args = 64, 8, (4, 1, 8, 3, 2, True, 1.0)
    other = 0
    for _ in range(12):
        l = rng.standard_normal((1, E)).astype(np.float32)
        p = ref.scores(l.astype(np.float64), 1)[0]
        bias = np.full(E, -1.0, np.float32)
        for g in range(G):
            a, b = g * 8 + rng.permutation(8)[:2]
            bias[a] = 0.25 + 0.1 * g
            bias[b] = np.float32(3.0 - p[b] - p[a] - np.float64(bias[a]))
        check_route(run_route(blk, torch.from_numpy(l), bias, *args), torch.from_numpy(l), bias, *args)
        c = p + bias.astype(np.float64)
        two = np.sort(c.reshape(G, 8), 1)[:, -2:].sum(1)
        two32 = np.sort((p.astype(np.float32) + bias).reshape(G, 8), 1)[:, -2:].sum(1)
        other += set(np.argsort(-two, kind="stable")[:3]) != set(np.argsort(-two32, kind="stable")[:3])
    assert other


def test_route_of_extreme_logits(blk):
    """The type's lowest and highest values, saturated scores, infinities and NaN."""
    say("route extremes")
    rng = np.random.default_rng(4)
    for mode in (0, 1, 2):
        for n_group, keep in ((1, 1), (4, 2)):
            l = torch.from_numpy(rng.standard_normal((12, 64)).astype(np.float32))
            low, high = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
            l[0, 5:] = low          # masked by the type's lowest value
            l[1] = low
            l[2, :60] = float("-inf")
            l[3, 7] = 80.0
            l[4] = -90.0 - l[4].abs()  # scores next to 0
            args = (4, mode, n_group, keep, 1, True, 1.0)
            got = run_route(blk, l[:5], None, *args)
            want_ids, want_w, p = ref.route(l[:5].numpy(), None, *args)
            assert (got[0] == want_ids).all()
            half = torch.from_numpy(ref.score_half_steps(np.clip(l[:5].numpy().astype(np.float64), -200, 200), mode))
            # scores below f32's smallest normal are off by a step of the smallest values
            close(got[2], torch.from_numpy(p), half * U * torch.from_numpy(p) + 1.2e-38)
            l[5, 3], l[6, 9], l[7, 1] = float("inf"), float("nan"), high
            l[8] = float("nan")
            ids, wts, sc = run_route(blk, l, None, *args)
            assert ((ids >= 0) & (ids < 64)).sum(1).min() >= 0 and (ids[9:] == ref.route(l[9:].numpy(), None, *args)[0]).all()
            for t in range(12):  # different experts, whatever the logits
                there = ids[t][ids[t] >= 0]
                assert len(set(there.tolist())) == len(there)
            if mode == 1:
                assert ids[5, 0] == 3 and 9 not in ids[6] and ids[7, 0] == 1 and torch.isnan(wts[8]).all()


@pytest.mark.parametrize("T, E, k, n_group, keep", ROUTE)
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kind, out, norm, scale, dense, masked", [
    ("f32", "f32", True, 2.5, True, 0.0), ("bf16", "bf16", True, 1.0, False, 0.3), ("f16", "f32", False, 0.0, True, 0.8),
    ("f32", "f16", False, 1.0, False, 0.0)])
def test_route_grad(blk, T, E, k, n_group, keep, mode, kind, out, norm, scale, dense, masked):
    say("route_grad", T, E, k, mode, kind, out, norm, scale, dense, masked)
    rng = np.random.default_rng(T + E + mode)
    l = logits_of(rng, T, E, kind, masked)
    ids = ref.route(l.float().numpy(), None, k, mode, n_group, keep, 1, norm, scale)[0]
    if T > 2:
        ids[1, 0] = E + 5  # outside: takes no part
    dwts = rng.standard_normal((T, k)).astype(np.float32)
    dsc = rng.standard_normal((T, E)).astype(np.float32) if dense else None
    dl = zeros(T, E, dtype=TYPES[out])
    blk.route_grad(dev(l), dev(ids), dev(dwts), mode, norm, scale, dl, dscores=None if dsc is None else dev(dsc))
    want, bound = ref.route_grad(l.float().numpy(), ids, dwts, dsc, mode, norm, scale)
    want, bound = torch.from_numpy(want), torch.from_numpy(bound)
    close(dl, want, rounded(bound, want, TYPES[out]))


def test_route_grad_of_an_expert_named_twice(blk):
    say("route_grad twice")
    rng = np.random.default_rng(6)
    l, dwts = logits_of(rng, 9, 48, "f32", 0.0), rng.standard_normal((9, 6)).astype(np.float32)
    ids = rng.integers(0, 3, (9, 6)).astype(np.int32)
    for mode in (0, 1, 2):
        dl = zeros(9, 48)
        blk.route_grad(dev(l), dev(ids), dev(dwts), mode, True, 1.0, dl)
        want, bound = ref.route_grad(l.numpy(), ids, dwts, None, mode, True, 1.0)
        close(dl, torch.from_numpy(want), torch.from_numpy(bound))


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("norm", [True, False])
def test_route_gradient_is_that_of_differences(blk, mode, norm):
    """As for the norm: central differences of the kernel's weights and scores at fixed picks."""
    say("route differences", mode, norm)
    rng = np.random.default_rng(mode)
    T, E, k, step = 6, 24, 4, 2.0 ** -7
    l = torch.from_numpy(rng.standard_normal((T, E)).astype(np.float32))
    d, dwts, dsc = (rng.standard_normal(s).astype(np.float32) for s in ((T, E), (T, k), (T, E)))
    bias = np.zeros(E, np.float32)
    bias[[2, 9, 10, 23]] = 10.0  # it makes the picks, so that they stay within the step
    base = ref.route(l.numpy(), bias, k, mode, 1, 1, 1, norm, 1.5)[0]

    def loss(sign, kernel):
        at = (l + sign * step * torch.from_numpy(d)).float()
        if kernel:
            ids, wts, p = run_route(blk, at, bias, k, mode, 1, 1, 1, norm, 1.5)
            wts, p = wts.double().numpy(), p.double().numpy()
        else:
            ids, wts, p = ref.route(at.numpy(), bias, k, mode, 1, 1, 1, norm, 1.5)
        assert (np.sort(ids, 1) == np.sort(base, 1)).all()
        w_of = np.zeros((T, E))
        np.put_along_axis(w_of, ids, wts, 1)
        return (np.take_along_axis(w_of, base, 1) * dwts).sum() + (p * dsc).sum()

    dl = zeros(T, E)
    blk.route_grad(dev(l), dev(base), dev(dwts), mode, norm, 1.5, dl, dscores=dev(dsc))
    got = (dl.cpu().double().numpy() * d).sum()
    want, bound = ref.route_grad(l.numpy(), base, dwts, dsc, mode, norm, 1.5)
    by_kernel, in_64 = ((loss(1, c) - loss(-1, c)) / (2 * step) for c in (True, False))
    _, w, p = ref.route(l.numpy(), bias, k, mode, 1, 1, 1, norm, 1.5)
    half = ref.score_half_steps(l.numpy().astype(np.float64), mode)
    noise = 2 * 2 * (((2 * half + k + 6) * U * np.abs(w * dwts)).sum() + (half * U * np.abs(p * dsc)).sum()) / (2 * step)
    assert abs(by_kernel - got) <= abs(in_64 - (want * d).sum()) + noise + (bound * np.abs(d)).sum()


# ---- adapters --------------------------------------------------------------------------------


def adapters_inputs(rng, M, K, R, N, n, x, out, spread, without=0.2):
    of = rng.integers(0, n, M) if spread else np.sort(rng.integers(0, n, M))
    of = np.where(rng.random(M) < without, -1, of).astype(np.int32)
    if M == 1:
        of[0] = n - 1
    t = TYPES[x]
    xs = floats(rng, (M, K), x)
    a = (torch.from_numpy(rng.standard_normal((n, R, K)).astype(np.float32)) / K ** 0.5).to(t)
    b = (torch.from_numpy(rng.standard_normal((n, N, R)).astype(np.float32)) / R ** 0.5).to(t)
    return of, xs, a, b, torch.from_numpy(rng.uniform(-1, 2, n).astype(np.float32)), floats(rng, (M, N), out)


def run_adapters(blk, of, x, a, b, scale, base, in_place):
    M, (n, R, K) = x.shape[0], a.shape
    counts, offsets, perm = (torch.full((m,), -5, dtype=torch.int32, device=DEV) for m in (n, n + 1, M))
    blk.group(dev(of[:, None]), n, counts, offsets, perm)
    bd = dev(base)
    out = bd if in_place else torch.full(base.shape, 3.0, dtype=base.dtype, device=DEV)
    mid = torch.full((blk.adapters_scratch(M, K, R) + 3,), float("nan"), device=DEV)
    blk.adapters(dev(x), dev(a), dev(b), None if scale is None else dev(scale), offsets, perm, bd, out, mid[:-3])
    assert torch.isnan(mid[-3:]).all()
    return out.cpu()


ADAPTERS = [(1, 64, 8, 64, 1), (1, 7168, 16, 512, 3), (2, 7, 1, 3, 2), (16, 256, 16, 128, 16), (17, 100, 5, 33, 4),
            (64, 1024, 32, 256, 3), (130, 520, 64, 96, 7), (300, 96, 8, 200, 40), (33, 2048, 96, 65, 2), (40, 33, 130, 40, 3),
            (9, 4096, 200, 24, 2), (515, 128, 4, 72, 1), (70, 777, 12, 1000, 5), (5, 24, 8, 4099, 1024),
            # rows enough for the staged tiles, of every rank class, over ragged K and N
            (200, 256, 16, 300, 2), (600, 520, 64, 264, 5), (129, 1024, 8, 128, 3), (96, 72, 40, 1000, 1),
            (700, 200, 24, 2056, 4), (150, 64, 128, 136, 2), (2000, 136, 32, 96, 60), (300, 2056, 60, 129, 3),
            (2100, 64, 24, 7945, 3), (2100, 72, 64, 8000, 2), (1000, 64, 8, 7000, 30)]


@pytest.mark.parametrize("M, K, R, N, n", ADAPTERS)
@pytest.mark.parametrize("x, out", [("bf16", "bf16"), ("f16", "f32"), ("f32", "f32"), ("bf16", "f32"), ("f16", "f16"),
                                    ("f32", "bf16")])
@pytest.mark.parametrize("spread", [True, False])
def test_adapters(blk, M, K, R, N, n, x, out, spread):
    say("adapters", M, K, R, N, n, x, out, spread)
    rng = np.random.default_rng(M + K + R)
    of, xs, a, b, scale, base = adapters_inputs(rng, M, K, R, N, n, x, out, spread)
    for sc, in_place in ((scale, True), (None, False)):
        got = run_adapters(blk, of, xs, a, b, sc, base, in_place)
        want, bound = ref.adapters(xs, a, b, sc, torch.from_numpy(of), base, TYPES[out])
        there = torch.from_numpy(of >= 0)
        close(got[there], want[there], bound[there])
        rest = got[~there]  # left as they were
        assert torch.equal(rest, base[~there] if in_place else torch.full_like(rest, 3.0))


def test_adapters_of_no_row_and_rows_of_no_adapter(blk):
    """Every row without an adapter, maps that point outside, offsets outside the rows."""
    say("adapters none")
    rng = np.random.default_rng(0)
    M, K, R, N, n = 20, 72, 8, 40, 3
    of, xs, a, b, scale, base = adapters_inputs(rng, M, K, R, N, n, "bf16", "bf16", True)
    assert torch.equal(run_adapters(blk, np.full(M, -1, np.int32), xs, a, b, scale, base, True), base)
    perm, offsets = np.arange(M, dtype=np.int32), np.array([0, 8, 8, M + 50], np.int32)
    perm[3], perm[12] = -1, M
    out, mid = dev(base), torch.zeros(blk.adapters_scratch(M, K, R), device=DEV)
    blk.adapters(dev(xs), dev(a), dev(b), dev(scale), dev(offsets), dev(perm), out, out, mid)
    of = np.where(np.arange(M) < 8, 0, 2)
    of[[3, 12]] = -1
    want, bound = ref.adapters(xs, a, b, scale, torch.from_numpy(of), base, torch.bfloat16)
    there = torch.from_numpy(of >= 0)
    got = out.cpu()
    close(got[there], want[there], bound[there])
    assert torch.equal(got[~there], base[~there])


def test_adapters_with_large_values(blk):
    """Products of A and x past f16's range, and rows of very different size side by side."""
    say("adapters large")
    rng = np.random.default_rng(1)
    for x, out in (("f16", "f32"), ("bf16", "f32"), ("f16", "bf16")):
        of, xs, a, b, scale, base = adapters_inputs(rng, 40, 512, 16, 64, 3, x, out, True, 0.0)
        xs = (xs.float() * torch.from_numpy(4.0 ** rng.integers(-5, 7, (40, 1))).float()).to(TYPES[x])
        a = (a.float() * 64).to(TYPES[x])
        want, bound = ref.adapters(xs, a, b, scale, torch.from_numpy(of), base, TYPES[out])
        # parts of a row of mid are relative to the row's largest value where the type's range asks for a common factor
        mid = torch.stack([a[i].double() @ r.double() for i, r in zip(of, xs)])
        worst = torch.stack([(b[i].double().abs().sum(1) * abs(float(scale[i])) * m.abs().max()) * 2.0 ** -25
                             for i, m in zip(of, mid)])
        close(run_adapters(blk, of, xs, a, b, scale, base, False), want, bound + worst)


def test_adapters_keep_a_nan_in_its_row(blk):
    say("adapters nan")
    rng = np.random.default_rng(2)
    for x in ("f32", "bf16", "f16"):
        of, xs, a, b, scale, base = adapters_inputs(rng, 37, 136, 8, 48, 2, x, "f32", False, 0.0)
        xs[5, 17] = float("nan")
        xs[20, 3] = float("inf")
        got = run_adapters(blk, of, xs, a, b, scale, base, False)
        assert torch.isnan(got[5]).all() and not torch.isfinite(got[20]).any()
        ok = [i for i in range(37) if i not in (5, 20)]
        want, bound = ref.adapters(xs[ok], a, b, scale, torch.from_numpy(of[ok]), base[ok], torch.float32)
        close(got[ok], want, bound)


# ---- past 4 GiB ------------------------------------------------------------------------------


def test_norm_and_gradient_past_4_gib(blk):
    """Rows whose elements lie past 2^32 bytes, and 2^31 elements, from the buffers' start."""
    say("norm past 4 GiB")
    T, H = 270000, 8192
    x = torch.empty((T, H), dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    w = torch.ones(H, dtype=torch.bfloat16, device=DEV)
    y, q, qs, rstd = torch.empty_like(x), torch.empty((T, H), dtype=torch.int8, device=DEV), zeros(T), zeros(T)
    blk.rms_norm(x, w, EPS, y=y, q=q, scale=qs, rstd=rstd)
    some = [0, 1, 131071, 131072, 262143, 262144, T - 2, T - 1]
    check_norm(dict(y=y[some].cpu(), q=q[some].cpu(), scale=qs[some].cpu(), rstd=rstd[some].cpu()), x[some].cpu(), None, w.cpu())
    dx, dw = torch.empty_like(x), zeros(H)
    blk.rms_norm_grad(y, x, w, rstd, dx, dw, torch.empty(blk.rms_norm_grad_scratch(T, H), device=DEV))
    some = torch.tensor(some)
    ys, xs, rs = y[some.to(DEV)].cpu(), x[some.to(DEV)].cpu(), rstd[some.to(DEV)].cpu()
    wx, _, ex, _ = ref.norm_grad(ys, xs, w.cpu(), rs, None)
    close(dx[some.to(DEV)], wx, rounded(ex, wx, torch.bfloat16))
    want, mag = torch.zeros(H, dtype=torch.float64, device=DEV), torch.zeros(H, dtype=torch.float64, device=DEV)
    for i in range(0, T, 10000):
        term = y[i:i + 10000].double() * (x[i:i + 10000].double() * rstd[i:i + 10000].double()[:, None])
        want += term.sum(0)
        mag += term.abs().sum(0)
    # a workgroup's share is a chain of T / 256 rows and more, the shares a dozen steps
    close(dw, want.cpu(), ((T // 128) * U * mag).cpu())


def test_adapters_past_4_gib(blk):
    say("adapters past 4 GiB")
    M, K, R, N, n = 70000, 32768, 8, 40, 2
    x = torch.empty((M, K), dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(2))
    rng = np.random.default_rng(3)
    _, _, a, b, scale, _ = adapters_inputs(rng, 4, K, R, N, n, "bf16", "f32", True)
    of = np.sort(rng.integers(-1, n, M)).astype(np.int32)
    offsets, perm, _, _ = expert_ref.grouping(of[:, None], n)
    base, out, mid = zeros(M, N), zeros(M, N), torch.empty(blk.adapters_scratch(M, K, R), device=DEV)
    blk.adapters(x, dev(a), dev(b), dev(scale), dev(offsets), dev(perm), base, out, mid)
    some = torch.tensor([0, 1, 30000, 65535, 65536, 66000, M - 2, M - 1])
    xs = x[some.to(DEV)].cpu()
    want, bound = ref.adapters(xs, a, b, scale, torch.from_numpy(of)[some], base.cpu()[some], torch.float32)
    close(out.cpu()[some], want, bound)


# ---- refusals of the library -------------------------------------------------------------------


def refused(status, call, *args, **kw):
    with pytest.raises(mb.MoeError) as e:
        call(*args, **kw)
    assert e.value.status == status, e.value


def test_the_library_refuses(blk):
    say("refusals")
    T, H = 4, 32
    x, w, y = zeros(T, H), zeros(H), zeros(T, H)
    bad = mb.MOE_ERR_INVALID_ARG
    for eps in (0.0, -1.0, float("nan"), float("inf"), 1e-40):
        refused(bad, blk.rms_norm, x, w, eps, y=y)
    refused(bad, blk.rms_norm, x, w, EPS, y=x)
    refused(bad, blk.rms_norm, x, w, EPS, residual=zeros(T, H), total=x, y=y)
    refused(bad, blk.rms_norm, x, w, EPS, y=y, rstd=y.view(-1)[:T])
    n = blk.rms_norm_grad_scratch(T, H)
    g = dict(dy=x, h=zeros(T, H), w=w, rstd=zeros(T), dx=y, dw=zeros(H), part=zeros(max(n, 1)))
    refused(bad, blk.rms_norm_grad, **{**g, "dx": x})
    refused(bad, blk.rms_norm_grad, **{**g, "dw": y.view(-1)[:H]})
    refused(bad, blk.rms_norm_grad, **{**g, "part": x.view(-1)})
    big = blk.rms_norm_grad_scratch(4096, 512)
    if big > 1:
        t = torch.empty((4096, 512), device=DEV)
        refused(bad, blk.rms_norm_grad, t, torch.empty_like(t), zeros(512), zeros(4096), torch.empty_like(t), zeros(512),
                torch.empty(big - 1, device=DEV))
    assert blk.rms_norm_grad_scratch(0, 5) == 0 and blk.rms_norm_grad_scratch(5, 2 ** 30 + 1) == 0
    E, k = 32, 4
    l, ids, wts = zeros(T, E), zeros(T, k, dtype=torch.int32), zeros(T, k)
    r = dict(logits=l, k=k, mode=1, norm=True, scale=1.0, ids=ids, wts=wts)
    for more in (dict(mode=3), dict(mode=-1), dict(n_group=5), dict(n_group=0), dict(n_group=8, keep=9), dict(keep=0),
                 dict(n_group=16, keep=1), dict(top=0), dict(top=3), dict(scores=l), dict(n_group=128, logits=zeros(T, 128))):
        refused(bad, blk.route_groups, **{**r, **more})
    refused(bad, blk.route_groups, zeros(T, 1025), k, 1, True, 1.0, ids, wts)
    refused(bad, blk.route_groups, l, 65, 1, True, 1.0, zeros(T, 65, dtype=torch.int32), zeros(T, 65))
    refused(bad, blk.route_grad, l, ids, wts, 3, True, 1.0, zeros(T, E))
    refused(bad, blk.route_grad, l, ids, wts, 1, True, 1.0, l)
    refused(bad, blk.route_grad, zeros(T, 1025), ids, wts, 1, True, 1.0, zeros(T, 1025))
    a, b, off, perm = zeros(2, 8, H), zeros(2, E, 8), zeros(3, dtype=torch.int32), zeros(T, dtype=torch.int32)
    mid = zeros(blk.adapters_scratch(T, H, 8))
    refused(bad, blk.adapters, x, a, b, None, off, perm, l, x.view(T, E), mid)
    refused(bad, blk.adapters, x, a, b, None, off, perm, l, zeros(T, E), mid[:-1])
    refused(bad, blk.adapters, x, a, b, None, off, perm, l, a.view(-1)[:T * E].view(T, E), mid)
    refused(bad, blk.adapters, x, zeros(2, 1025, H), zeros(2, E, 1025), None, off, perm, l, zeros(T, E), zeros(10 ** 6))
    refused(bad, blk.adapters, x, zeros(1025, 1, H), zeros(1025, E, 1), None, zeros(1026, dtype=torch.int32), perm, l,
            zeros(T, E), mid)
    assert blk.adapters_scratch(1, 8, 1025) == 0 and blk.adapters_scratch(0, 8, 8) == 0


# ---- together ------------------------------------------------------------------------------------


def test_a_training_step_of_the_layer(blk):
    """Norm with residual, router, grouped routing, dispatch, experts that scale their rows, combine; and the way
    back to the input, the gain and the router, against the same step in 64 bits by automatic differentiation."""
    say("step")
    rng = np.random.default_rng(12)
    T, H, E, k, G, keep = 70, 96, 32, 4, 4, 2
    x, res, w = floats(rng, (T, H), "f32"), floats(rng, (T, H), "f32"), 1 + 0.2 * floats(rng, (H,), "f32")
    wr, gain = 0.2 * floats(rng, (E, H), "f32"), 1 + 0.5 * floats(rng, (E,), "f32")
    dout, dtot = floats(rng, (T, H), "f32"), floats(rng, (T, H), "f32")
    bias = 0.1 * floats(rng, (E,), "f32")
    total, y, rstd, logits = zeros(T, H), zeros(T, H), zeros(T), zeros(T, E)
    ids, wts = zeros(T, k, dtype=torch.int32), zeros(T, k)
    counts, off, perm, inv = (zeros(m, dtype=torch.int32) for m in (E, E + 1, T * k, T * k))
    rows, out = zeros(T * k, H), zeros(T, H)
    blk.rms_norm(dev(x), dev(w), EPS, residual=dev(res), total=total, y=y, rstd=rstd)
    blk.router_logits(dev(wr), y, logits)
    blk.route_groups(logits, k, mb.ROUTE_SIGMOID, True, 2.5, ids, wts, bias=dev(bias), n_group=G, keep=keep)
    blk.group(ids, E, counts, off, perm, inv)
    blk.dispatch(y, inv, rows)
    expert = ids.view(-1)[perm.long()].long()
    scaled = rows * dev(gain)[expert, None]
    blk.combine(scaled, wts, inv, out)
    # and back
    drows, dwts, dy1, dlogits = zeros(T * k, H), zeros(T, k), zeros(T, H), zeros(T, E)
    blk.combine_grad(dev(dout), scaled, wts, inv, drows, dwts)
    blk.dispatch_grad(drows * dev(gain)[expert, None], inv, dy1)
    blk.route_grad(logits, ids, dwts, mb.ROUTE_SIGMOID, True, 2.5, dlogits)
    dy = dy1 + dlogits @ dev(wr)
    dx, dw = zeros(T, H), zeros(H)
    blk.rms_norm_grad(dy, total, dev(w), rstd, dx, dw, zeros(blk.rms_norm_grad_scratch(T, H)), dres=dev(dtot))
    # the same step in 64 bits, at the picks that were made
    X, W, R = x.double().requires_grad_(), w.double().requires_grad_(), wr.double()
    h = X + res.double()
    Y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * W
    s = torch.sigmoid(Y @ R.t())
    want_ids = ref.route((Y @ R.t()).detach().numpy(), bias.numpy(), k, 1, G, keep, 2, True, 2.5)[0]
    assert (want_ids == ids.cpu().numpy()).all()
    p = torch.gather(s, 1, torch.from_numpy(want_ids).long())
    p = 2.5 * p / p.sum(1, keepdim=True)
    o = (p * gain.double()[torch.from_numpy(want_ids).long()]).sum(1, keepdim=True) * Y
    ((o * dout.double()).sum() + (h * dtot.double()).sum()).backward()
    # each stage keeps 2^-18 of its values or better; the five between input and gradient, and the sums over H and T, stay
    # within 2^-14 of the largest
    for got, want in ((out, o.detach()), (dx, X.grad), (dw, W.grad)):
        assert (got.cpu().double() - want).abs().max() <= 2.0 ** -14 * want.abs().max()


def test_serving_a_batch_with_adapters(blk):
    """Norm into 8 bits, a shared projection in 8 bits, the requests' adapters added in place, single tokens."""
    say("serving")
    rng = np.random.default_rng(13)
    M, H, N, R, n = 18, 256, 192, 8, 5
    of, x, a, b, scale, _ = adapters_inputs(rng, M, H, R, N, n, "bf16", "bf16", True)
    res, w = floats(rng, (M, H), "bf16"), (1 + 0.2 * floats(rng, (H,), "f32")).to(torch.bfloat16)
    wq = torch.from_numpy(rng.integers(-127, 128, (N, H)).astype(np.int8))
    ws = torch.from_numpy(rng.uniform(0.5, 1, N).astype(np.float32)) / (73 * H ** 0.5)
    total = dev(res)
    y, q, qs, out = zeros(M, H, dtype=torch.bfloat16), zeros(M, H, dtype=torch.int8), zeros(M), zeros(M, N, dtype=torch.bfloat16)
    blk.rms_norm(dev(x), dev(w), EPS, residual=total, total=total, y=y, q=q, scale=qs)
    blk.matmul_i8(q, qs, dev(wq), dev(ws), out)
    shared = out.cpu()
    counts, off, perm = zeros(n, dtype=torch.int32), zeros(n + 1, dtype=torch.int32), zeros(M, dtype=torch.int32)
    blk.group(dev(of[:, None]), n, counts, off, perm)
    blk.adapters(y, dev(a), dev(b), dev(scale), off, perm, out, out, zeros(blk.adapters_scratch(M, H, R)))
    h = ref.total(x, res)
    assert torch.equal(total.cpu(), h)
    yq, _ = ref.norm(h, w, EPS)
    codes, cs = ref.codes(yq)
    assert torch.equal(q.cpu(), codes)
    prod = expert_ref.product(codes, cs, wq, ws)
    close(shared, prod, rounded(expert_ref.product_bound(prod), prod, torch.bfloat16))
    want, bound = ref.adapters(y.cpu(), a, b, scale, torch.from_numpy(of), shared, torch.bfloat16)
    there = torch.from_numpy(of >= 0)
    close(out.cpu()[there], want[there], bound[there])
    assert torch.equal(out.cpu()[~there], shared[~there])


def calls_of(blk, rng, T=40, H=320, E=64, k=4):
    """Every operator as a closure over its own buffers, with its outputs."""
    x, res, w = dev(floats(rng, (T, H), "bf16")), dev(floats(rng, (T, H), "bf16")), dev(floats(rng, (H,), "bf16"))
    b16 = torch.bfloat16
    total, y, q, qs, rstd = zeros(T, H, dtype=b16), zeros(T, H, dtype=b16), zeros(T, H, dtype=torch.int8), zeros(T), zeros(T)
    dx, dw, part = zeros(T, H, dtype=b16), zeros(H), zeros(blk.rms_norm_grad_scratch(T, H))
    l, ids, wts, sc = dev(floats(rng, (T, E), "f32")), zeros(T, k, dtype=torch.int32), zeros(T, k), zeros(T, E)
    dwts, dl = dev(floats(rng, (T, k), "f32")), zeros(T, E)
    n, R, N = 6, 8, 136
    a, b = dev(floats(rng, (n, R, H), "bf16")), dev(floats(rng, (n, N, R), "bf16"))
    offsets, perm, _, _ = expert_ref.grouping(rng.integers(0, n, (T, 1)).astype(np.int32), n)
    off, pm, base, out = dev(offsets), dev(perm), dev(floats(rng, (T, N), "f32")), zeros(T, N)
    mid = zeros(blk.adapters_scratch(T, H, R))

    def run(stream=None):
        blk.rms_norm(x, w, EPS, residual=res, total=total, y=y, q=q, scale=qs, rstd=rstd, stream=stream)
        blk.rms_norm_grad(res, total, w, rstd, dx, dw, part, stream=stream)
        blk.route_groups(l, k, 1, True, 2.5, ids, wts, n_group=8, keep=4, scores=sc, stream=stream)
        blk.route_grad(l, ids, dwts, 0, True, 1.0, dl, dscores=sc, stream=stream)
        blk.adapters(y, a, b, None, off, pm, base, out, mid, stream=stream)

    return run, [total, y, q, qs, rstd, dx, dw, ids, wts, sc, dl, out]


def wipe(outs):
    for o in outs:
        o.fill_(9)


def test_captured_and_replayed(blk):
    say("graphs")
    run, outs = calls_of(blk, np.random.default_rng(1))
    other, more = calls_of(blk, np.random.default_rng(2))
    run()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    graphs = []
    for f in (run, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f()
        graphs.append(g)
    for i in range(4):
        wipe(outs)
        graphs[0].replay()
        graphs[1].replay()
        other()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def test_on_several_streams_and_threads(blk):
    say("streams")
    sets = [calls_of(blk, np.random.default_rng(s)) for s in (1, 2, 3)]
    want = []
    for run, outs in sets:
        run()
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
        wipe(outs)
    torch.cuda.synchronize()
    errors = []

    def work(run):
        try:
            s = torch.cuda.Stream()
            for _ in range(20):
                run(s.cuda_stream)
            s.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(run,)) for run, _ in sets]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not errors
    for (_, outs), w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(outs, w))


def test_through_ctypes_alone_gives_the_same(blk):
    say("ctypes")
    run, outs = calls_of(blk, np.random.default_rng(5))
    run()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    wipe(outs)
    saved = blk._calls
    blk.__dict__["_calls"] = None
    try:
        run()
        torch.cuda.synchronize()
    finally:
        blk.__dict__["_calls"] = saved
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_profiler_names_each_operator(blk):
    say("profiler")
    run, _ = calls_of(blk, np.random.default_rng(7))
    run()
    torch.cuda.synchronize()
    blk.prof_enable(True)
    try:
        blk.prof_read(reset=True)
        run()
        got = blk.prof_read(reset=True)
    finally:
        blk.prof_enable(False)
    assert {m: c for m, (c, _) in got.items()} == {m: 1 for m in ("rms_norm", "rms_norm_grad", "route_groups", "route_grad",
                                                                  "adapters")}

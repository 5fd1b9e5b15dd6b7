"""Dispatch, combine and their gradients, rows in 8 bits and 8-bit products on
the GPU, against 64-bit statements of them (expert_ref.py) with the error
bounds that f32 sums and the output's rounding allow."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import expert_ref as ref
import moe_block as mb
import workloads as wl
from expert_ref import TYPES, U

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def say(*a):
    print("[gpu]", *a, flush=True)


@pytest.fixture(scope="module")
def blk():
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    b = mb.MoeBlock(0)
    yield b
    b.close()


def dev(a):
    return (torch.from_numpy(np.ascontiguousarray(a)) if isinstance(a, np.ndarray) else a).to(DEV)


def floats(rng, shape, kind):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(TYPES[kind])


def close(got, want, bound):
    got, want = got.detach().cpu().double(), want.double()
    off = (got - want).abs()
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all() and (off <= bound).all(), f"off by {worst:.3g} of the bound"


# ---- dispatch and combine ------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 8, 7168), (2, 3, 7), (5, 1, 64), (37, 6, 129), (130, 4, 1000), (3, 64, 72), (700, 8, 256),
         (9, 2, 5121), (2500, 2, 24)]


def setup(T, k, H, dropped, seed):
    rng = np.random.default_rng(seed)
    E = max(8, k)
    ids = ref.ids_of(rng, T, k, E, dropped)
    if T > 1 and dropped:
        ids[T // 2] = -1  # a token without rows
    offsets, perm, inv, kept = ref.grouping(ids, E)
    return rng, ids, E, inv, kept


@pytest.mark.parametrize("T, k, H", SIZES)
@pytest.mark.parametrize("a, b, dropped", [("f32", "f32", 0.0), ("bf16", "bf16", 0.3), ("f16", "f16", 0.3),
                                           ("f32", "bf16", 0.3), ("bf16", "f32", 0.0), ("f16", "bf16", 0.5)])
def test_dispatch(blk, T, k, H, a, b, dropped):
    say("dispatch", T, k, H, a, b, dropped)
    rng, ids, E, inv, kept = setup(T, k, H, dropped, T + H)
    x = floats(rng, (T, H), a)
    rows = torch.full((T * k + 1, H), 7.0, dtype=TYPES[b])
    got = rows.to(DEV)
    blk.dispatch(dev(x), dev(inv), got)
    at = torch.from_numpy(inv.astype(np.int64))
    pair = torch.nonzero(at >= 0).view(-1)
    rows[at[pair]] = x[pair // k].to(TYPES[b])
    assert torch.equal(got.cpu(), rows)  # one rounding, and the rows of no pair as they were


@pytest.mark.parametrize("T, k, H", SIZES)
@pytest.mark.parametrize("a, b, dropped", [("f32", "f32", 0.0), ("bf16", "bf16", 0.3), ("f16", "f32", 0.3),
                                           ("f32", "f16", 0.3), ("bf16", "f16", 0.5)])
def test_combine_and_dispatch_grad(blk, T, k, H, a, b, dropped):
    say("combine", T, k, H, a, b, dropped)
    rng, ids, E, inv, kept = setup(T, k, H, dropped, 2 * T + H)
    rows = floats(rng, (max(kept, 1), H), a)
    wts = torch.from_numpy(rng.uniform(-1, 1, (T, k)).astype(np.float32))
    for w in (wts, None):
        out = torch.full((T, H), float("nan"), dtype=TYPES[b], device=DEV)
        if w is None:
            blk.dispatch_grad(dev(rows), dev(inv), out)
        else:
            blk.combine(dev(rows), dev(w), dev(inv), out)
        want, mag = ref.combine(rows, w, inv, T, k)
        # k fused multiply-adds: each rounds a partial sum of the terms
        close(out, want, ref.rounded((k + 1) * U * mag, want, TYPES[b]))


@pytest.mark.parametrize("T, k, H", SIZES)
@pytest.mark.parametrize("a, b, dropped", [("f32", "f32", 0.3), ("bf16", "bf16", 0.0), ("f16", "f16", 0.3),
                                           ("f32", "bf16", 0.3), ("f16", "f32", 0.5)])
def test_combine_grad(blk, T, k, H, a, b, dropped):
    say("combine_grad", T, k, H, a, b, dropped)
    rng, ids, E, inv, kept = setup(T, k, H, dropped, 3 * T + H)
    R = max(kept, 1) + 1
    dout, rows = floats(rng, (T, H), a), floats(rng, (R, H), b)
    wts = torch.from_numpy(rng.uniform(-1, 1, (T, k)).astype(np.float32))
    drows = torch.full((R, H), 7.0, dtype=TYPES[b], device=DEV)
    dwts = torch.full((T, k), float("nan"), device=DEV)
    blk.combine_grad(dev(dout), dev(rows), dev(wts), dev(inv), drows, dwts)
    at = torch.from_numpy(inv.astype(np.int64))
    pair = torch.nonzero(at >= 0).view(-1)
    want = torch.full((R, H), 7.0, dtype=torch.float64)
    want[at[pair]] = dout[pair // k].double() * wts.view(-1)[pair, None].double()
    close(drows, want, ref.rounded(U * want.abs(), want, TYPES[b]))
    dw, mag = torch.zeros(T * k, dtype=torch.float64), torch.zeros(T * k, dtype=torch.float64)
    prod = dout[pair // k].double() * rows[at[pair]].double()
    dw[pair], mag[pair] = prod.sum(1), prod.abs().sum(1)
    # a lane's chain of FMAs over its share of H, then a sum over lanes of at most 9 steps
    close(dwts, dw.view(T, k), ((H / 64 + 8 + 9) * U * mag + 1e-40).view(T, k))


def test_the_gradients_are_those_of_differences(blk):
    """On small whole numbers every sum is exact, and combine and dispatch are linear in each argument: a difference
    of the forward pass in any direction equals the gradient's product with it."""
    T, k, H = 19, 3, 40
    say("differences", T, k, H)
    rng, ids, E, inv, kept = setup(T, k, H, 0.2, 5)
    whole = lambda *s: dev(rng.integers(-8, 9, s).astype(np.float32))  # noqa: E731
    rows, wts, dout, iv = whole(kept, H), whole(T, k), whole(T, H), dev(inv)

    def combine(r, w):
        out = torch.empty((T, H), device=DEV)
        blk.combine(r, w, iv, out)
        return out.double()

    drows, dwts = torch.empty_like(rows), torch.empty_like(wts)
    blk.combine_grad(dout, rows, wts, iv, drows, dwts)
    d_r, d_w = whole(kept, H), whole(T, k)
    d = dout.double()
    assert ((combine(rows + d_r, wts) - combine(rows, wts)) * d).sum() == (drows.double() * d_r).sum()
    assert ((combine(rows, wts + d_w) - combine(rows, wts)) * d).sum() == (dwts.double() * d_w).sum()
    x, d_x, drows = whole(T, H), whole(T, H), whole(kept, H)

    def dispatch(v):
        out = torch.zeros((kept, H), device=DEV)
        blk.dispatch(v, iv, out)
        return out.double()

    dx = torch.empty_like(x)
    blk.dispatch_grad(drows, iv, dx)
    assert ((dispatch(x + d_x) - dispatch(x)) * drows.double()).sum() == (dx.double() * d_x).sum()


def test_map_entries_outside_the_rows_are_dropped(blk):
    say("map entries outside the rows")
    T, k, H, R = 4, 2, 32, 3
    inv = np.array([0, 3, -7, 2 ** 30, 1, -1, 2, -2 ** 31], np.int32)
    rng = np.random.default_rng(1)
    x, wts, rows = floats(rng, (T, H), "f32"), floats(rng, (T, k), "f32"), floats(rng, (R, H), "f32")
    fine = np.where((inv >= 0) & (inv < R), inv, -1).astype(np.int32)
    got, out = torch.zeros((R, H), device=DEV), torch.empty((T, H), device=DEV)
    blk.dispatch(dev(x), dev(inv), got)
    blk.combine(dev(rows), dev(wts), dev(inv), out)
    want, mag = ref.combine(rows, wts, fine, T, k)
    close(out, want, (k + 1) * U * mag)
    assert torch.equal(got.cpu(), x[[0, 2, 3]])
    drows, dwts = torch.full((R, H), 7.0, device=DEV), torch.empty((T, k), device=DEV)
    blk.combine_grad(dev(x), dev(rows), dev(wts), dev(inv), drows, dwts)
    assert (dwts.cpu().view(-1)[torch.from_numpy(fine) < 0] == 0).all()


def test_infinities_and_nan_stay_in_their_rows(blk):
    say("infinities and NaN")
    T, k, H = 4, 2, 24
    inv = np.array([0, 1, 2, -1, 3, 4, -1, -1], np.int32)
    rows = torch.ones((5, H))
    rows[1, 3], rows[2, 5], rows[4, 0] = float("nan"), float("inf"), -float("inf")
    wts = torch.ones((T, k))
    out = torch.empty((T, H), device=DEV)
    blk.combine(dev(rows), dev(wts), dev(inv), out)
    got = out.cpu()
    want = torch.stack([rows[0] + rows[1], rows[2], rows[3] + rows[4], torch.zeros(H)])
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0.5), want.nan_to_num(0.5))


# ---- rows in 8 bits ------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M, K", [(1, 1), (3, 2), (2, 15), (5, 16), (4, 17), (3, 100), (300, 64), (33, 768), (2, 1000),
                                  (9, 2048), (1, 7168), (5, 7168), (3, 16400), (2, 40001), (1030, 520)])
def test_quantize(blk, M, K, kind):
    say("quantize", M, K, kind)
    rng = np.random.default_rng(M * K)
    x = (floats(rng, (M, K), "f32") * torch.from_numpy(np.exp(rng.uniform(-6, 6, (M, 1))).astype(np.float32))).to(TYPES[kind])
    if M > 2:
        x[1] = 0.0
        x[2, K - 1] = 100.0  # a row whose largest value is its last
    q, s = torch.full((M, K), 99, dtype=torch.int8, device=DEV), torch.full((M,), 99.0, device=DEV)
    blk.quantize_i8(dev(x), q, s)
    wq, ws = ref.quantize(x)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu(), wq)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M, K", [(2100, 700), (2051, 768), (4099, 513), (2049, 8), (700, 256), (515, 255), (600, 1537), (515, 6144),
                                  (600, 5003), (513, 7168)])
def test_quantize_many_rows(blk, M, K, kind):
    test_quantize(blk, M, K, kind)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M, K", [(1, 768), (2100, 700), (600, 248), (9, 7168), (600, 4104)])
def test_quantize_between_two_codes(blk, M, K, kind):
    """Rows whose largest value is 127 units: halves of units are ties, and their neighbours
    the smallest steps beside one."""
    say("quantize between two codes", M, K, kind)
    rng = np.random.default_rng(M + K)
    unit = torch.from_numpy(2.0 ** rng.integers(-8, 8, (M, 1)))
    x = torch.from_numpy((rng.integers(-126, 126, (M, K)) + 0.5)).to(TYPES[kind]).double()
    t = torch.finfo(TYPES[kind])
    step = torch.from_numpy(rng.integers(-1, 2, (M, K))) * t.eps * 2.0 ** torch.floor(torch.log2(x.abs()))
    x = (x + step).clamp(-127, 127)
    x[:, K // 3] = 127.0
    x = (x * unit).to(TYPES[kind])
    q, scale = torch.full((M, K), 99, dtype=torch.int8, device=DEV), torch.full((M,), 7.0, device=DEV)
    blk.quantize_i8(x.to(DEV), q, scale)
    assert torch.equal(scale.cpu().double(), unit[:, 0])
    assert torch.equal(q.cpu().double(), torch.round(x.double() / unit))


@pytest.mark.parametrize("K", [24, 1024, 8192, 33])
def test_quantize_ties_and_extremes(blk, K):
    say("quantize ties and extremes", K)
    rng = np.random.default_rng(K)
    base = rng.integers(-127, 127, K).astype(np.float64) + 0.5
    base[0] = 127.0
    rows = [base * 2.0 ** e for e in (0, -3, 40, 100, -60, -100, -120, -130, -140, -147)]  # every quotient a tie
    rows += [np.full(K, 2.0 ** -149), np.full(K, 3.4e38), np.zeros(K), -np.abs(rng.standard_normal(K)) * 1e-44]
    # quotients one f32 step off a tie on either side
    s = np.float32(np.float32(1.7) / np.float32(127))
    near = ((rng.integers(-100, 100, K) + 0.5) * np.float64(s)).astype(np.float32)
    near = np.where(rng.random(K) < 0.5, np.nextafter(near, np.float32(9)), np.nextafter(near, np.float32(-9)))
    near[0] = 1.7
    rows += [near]
    for bad in (np.nan, np.inf, -np.inf):
        r = rng.standard_normal(K)
        r[K // 2] = bad
        rows += [r]
    x = torch.from_numpy(np.stack(rows).astype(np.float32))
    q, s = torch.full(x.shape, 99, dtype=torch.int8, device=DEV), torch.full((len(rows),), 99.0, device=DEV)
    blk.quantize_i8(dev(x), q, s)
    wq, ws = ref.quantize(x)
    assert torch.equal(s.cpu().isnan(), ws.isnan()) and torch.equal(s.cpu().nan_to_num(0), ws.nan_to_num(0))
    assert torch.equal(q.cpu(), wq)


def test_quantize_at_odd_addresses(blk):
    say("quantize at odd addresses")
    rng = np.random.default_rng(3)
    for kind, K in (("bf16", 776), ("f32", 7168), ("f16", 8)):
        x = floats(rng, (5, K), kind)
        flat = torch.zeros(5 * K + 3, dtype=TYPES[kind], device=DEV)
        xo = flat[3:].view(5, K)
        xo.copy_(x)
        q = torch.zeros(5 * K + 1, dtype=torch.int8, device=DEV)[1:].view(5, K)
        s = torch.zeros(6, device=DEV)[1:]
        blk.quantize_i8(xo, q, s)
        wq, ws = ref.quantize(x)
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


# ---- 8-bit products --------------------------------------------------------------------


def codes(rng, shape):
    return torch.from_numpy(rng.integers(-128, 128, shape, dtype=np.int64).astype(np.int8))


def scales(rng, shape, K):
    return torch.from_numpy(rng.uniform(0.5, 1.5, shape).astype(np.float32) / np.float32(74 * K ** 0.25))


def check_product(got, q, s, w, ws, sw, L, dtype):
    check_against(got, ref.product(q, s, w, ws), sw, L, dtype)


def check_against(got, y, sw, L, dtype):
    if sw:
        h, g = ref.swiglu(y, L)
        close(got, h, ref.rounded(ref.swiglu_bound(h, g), h, dtype))
    else:
        close(got, y, ref.rounded(ref.product_bound(y), y, dtype))


DENSE = [(1, 1, 1), (1, 64, 16), (1, 768, 2048), (2, 130, 7168), (3, 33, 48), (16, 96, 768), (17, 64, 64), (33, 200, 1040),
         (5, 70, 77), (64, 64, 1001), (100, 130, 100), (130, 258, 272), (257, 320, 512), (300, 514, 640), (513, 256, 2064),
         (1, 4098, 256), (4, 31, 131071), (600, 1090, 128), (1100, 770, 336), (65, 2050, 4112)]


@pytest.mark.parametrize("M, N, K", DENSE)
@pytest.mark.parametrize("out, sw, L", [("f32", False, 0.0), ("bf16", True, 0.0), ("f16", False, 0.0), ("f32", True, 1.5)])
def test_dense_product(blk, M, N, K, out, sw, L):
    N = N + N % 2 if sw else N
    say("dense product", M, N, K, out, sw, L)
    rng = np.random.default_rng(M + 7 * N + K)
    q, w, s, ws = codes(rng, (M, K)), codes(rng, (N, K)), scales(rng, M, K), scales(rng, N, K)
    got = torch.full((M, N // 2 if sw else N), float("nan"), dtype=TYPES[out], device=DEV)
    blk.matmul_i8(dev(q), dev(s), dev(w), dev(ws), got, swiglu=sw, clamp=L)
    check_product(got, q, s, w, ws, sw, L, TYPES[out])


def test_the_sum_is_exact_at_its_limit(blk):
    """K = 131071 products of -128 and -128 fill 31 bits; one more is refused."""
    say("sum at its limit")
    K = 131071
    q, w = torch.full((1, K), -128, dtype=torch.int8, device=DEV), torch.full((2, K), -128, dtype=torch.int8, device=DEV)
    one, two, out = torch.ones(1, device=DEV), torch.ones(2, device=DEV), torch.empty((1, 2), device=DEV)
    blk.matmul_i8(q, one, w, two, out)
    assert (out.cpu() == float(np.float32(K * 16384))).all()
    with pytest.raises(mb.MoeError) as ei:
        z = lambda n: torch.zeros((n, K + 1), dtype=torch.int8, device=DEV)  # noqa: E731
        blk.matmul_i8(z(1), one, z(2), two, out)
    assert ei.value.status == mb.MOE_ERR_UNSUPPORTED


def test_products_at_odd_addresses(blk):
    say("products at odd addresses")
    rng = np.random.default_rng(4)
    M, N, K = 40, 72, 256
    q, w, s, ws = codes(rng, (M, K)), codes(rng, (N, K)), scales(rng, M, K), scales(rng, N, K)
    for oq, ow, oo in ((1, 0, 0), (0, 4, 0), (3, 5, 1), (0, 0, 1)):
        put = lambda t, o: torch.cat([torch.zeros(o, dtype=t.dtype), t.view(-1)]).to(DEV)[o:].view(t.shape)  # noqa: E731
        got = torch.full((M * N + 1,), float("nan"), dtype=torch.bfloat16, device=DEV)[oo:M * N + oo].view(M, N)
        blk.matmul_i8(put(q, oq), dev(s), put(w, ow), dev(ws), got)
        check_product(got, q, s, w, ws, False, 0.0, torch.bfloat16)


GROUPED = [  # T, k, E, N, K, dropped, skew
    (1, 1, 1, 2, 16, 0.0, False), (1, 8, 8, 64, 128, 0.0, False), (1, 4, 32, 1536, 2048, 0.0, False),
    (16, 8, 64, 128, 256, 0.0, True), (5, 2, 1024, 34, 48, 0.0, False), (37, 6, 160, 130, 272, 0.25, True),
    (200, 4, 8, 192, 512, 0.1, True), (300, 2, 3, 96, 77, 0.3, False), (64, 3, 7, 66, 144, 1.0, False),
    (700, 4, 16, 256, 768, 0.0, False), (1500, 2, 4, 320, 384, 0.0, True), (1300, 1, 2, 600, 400, 0.2, False),
    (4000, 2, 6, 514, 128, 0.0, True)]


@pytest.mark.parametrize("T, k, E, N, K, dropped, skew", GROUPED)
@pytest.mark.parametrize("out, sw, gather", [("f32", False, False), ("bf16", True, True), ("f32", True, True),
                                             ("f16", False, True)])
def test_grouped_product(blk, T, k, E, N, K, dropped, skew, out, sw, gather):
    say("grouped product", T, k, E, N, K, dropped, skew, out, sw, gather)
    rng = np.random.default_rng(T + E + N + K)
    ids = ref.ids_of(rng, T, k, E, dropped, skew)
    offsets, perm, inv, kept = ref.grouping(ids, E)
    M = T * k
    q, w, s, ws = codes(rng, (T if gather else M, K)), codes(rng, (E, N, K)), scales(rng, T if gather else M, K), scales(rng, (E, N), K)
    got = torch.full((M, N // 2 if sw else N), 7.0, dtype=TYPES[out], device=DEV)
    blk.matmul_i8(dev(q), dev(s), dev(w), dev(ws), got, offsets=dev(offsets), perm=dev(perm) if gather else None,
                  k=k if gather else 1, swiglu=sw, clamp=2.0)
    assert (got[kept:] == 7.0).all()  # rows of no expert as they were
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        if lo < hi:
            at = torch.from_numpy(perm[lo:hi].astype(np.int64) // k) if gather else torch.arange(lo, hi)
            check_product(got[lo:hi], q[at], s[at], w[e], ws[e], sw, 2.0, TYPES[out])


# rows that are few: of one wave's channels to many, K of one lane to several times a
# wave's, weights past the caches; and as many rows more, on narrow tiles
FEW = [(1, 1, 16), (1, 2, 16), (1, 7, 1008), (1, 130, 1024), (1, 258, 1040), (1, 66, 9232), (1, 6, 131056), (2, 2, 16),
       (2, 1030, 64), (2, 4100, 2064), (3, 30, 48), (3, 2730, 272), (4, 2050, 1040), (4, 3000, 4112), (5, 818, 128),
       (5, 820, 528), (8, 1024, 2048), (9, 14, 272), (16, 512, 512), (4096, 2, 32), (3000, 1, 48), (1, 8192, 12304),
       (2, 8190, 12304), (4, 8200, 4096), (5, 4098, 272), (16, 1030, 1040), (7, 7168, 64)]


@pytest.mark.parametrize("M, N, K", FEW)
@pytest.mark.parametrize("out, sw, L", [("f32", False, 0.0), ("bf16", True, 1.5)])
def test_dense_product_of_few_rows(blk, M, N, K, out, sw, L):
    test_dense_product(blk, M, N, K, out, sw, L)


FEW_GROUPED = [  # T, k, E, N, K, dropped, skew
    (1, 8, 64, 130, 1024, 0.0, False), (1, 8, 256, 34, 1040, 0.0, False), (2, 8, 300, 50, 2064, 0.0, False),
    (16, 1, 3, 258, 768, 0.0, True), (16, 1, 1, 66, 1040, 0.0, False), (8, 2, 1024, 18, 16, 0.4, False),
    (1, 8, 16, 2048, 8192, 0.0, False), (17, 1, 3, 66, 768, 0.0, True)]


@pytest.mark.parametrize("T, k, E, N, K, dropped, skew", FEW_GROUPED)
@pytest.mark.parametrize("out, sw, gather", [("f32", False, False), ("bf16", True, True), ("f16", False, True)])
def test_grouped_product_of_few_rows(blk, T, k, E, N, K, dropped, skew, out, sw, gather):
    test_grouped_product(blk, T, k, E, N, K, dropped, skew, out, sw, gather)


# every tile shape that the cost rule knows, at sizes that cut the last tiles
TILES = [(130, 130, 272), (257, 514, 1040), (257, 514, 272), (257, 1794, 272), (130, 6146, 272), (130, 6146, 528), (257, 6146, 528),
         (770, 2562, 1040), (5001, 770, 2064), (4001, 2562, 272), (4097, 1794, 2064)]


@pytest.mark.parametrize("M, N, K", TILES)
@pytest.mark.parametrize("out, sw", [("f32", False), ("bf16", True), ("f16", False)])
def test_dense_product_of_every_tile(blk, M, N, K, out, sw):
    say("dense product of every tile", M, N, K, out, sw)
    rng = np.random.default_rng(M + N + K)
    q, w, s, ws = (dev(t) for t in (codes(rng, (M, K)), codes(rng, (N, K)), scales(rng, M, K), scales(rng, N, K)))
    got = torch.full((M, N // 2 if sw else N), float("nan"), dtype=TYPES[out], device=DEV)
    blk.matmul_i8(q, s, w, ws, got, swiglu=sw, clamp=2.0)
    check_against(got, ref.product(q, s, w, ws).cpu(), sw, 2.0, TYPES[out])


# rows, E, N, K; the second half with weights past the caches: experts with one tile and with more
GROUPED_TILES = [(130, 2, 1026, 272), (130, 2, 1026, 1040), (40, 40, 258, 272), (130, 130, 130, 528), (4001, 2, 258, 528),
                 (130, 130, 130, 272), (4001, 2, 514, 1040), (4001, 2, 1026, 2064), (4001, 2, 2050, 272),
                 (130, 130, 514, 2064), (130, 130, 130, 7184), (4001, 130, 130, 7184), (8003, 130, 130, 7184),
                 (4001, 40, 4098, 1040), (4001, 40, 514, 7184), (4001, 40, 2050, 2064), (8003, 40, 4098, 1040)]


@pytest.mark.parametrize("M, E, N, K", GROUPED_TILES)
@pytest.mark.parametrize("out, sw, gather", [("f32", False, False), ("bf16", True, True)])
def test_grouped_product_of_every_tile(blk, M, E, N, K, out, sw, gather):
    say("grouped product of every tile", M, E, N, K, out, sw, gather)
    rng = np.random.default_rng(M + E + N + K)
    ids = ref.ids_of(rng, M, 1, E, 0.05, M > E)
    offsets, perm, inv, kept = ref.grouping(ids, E)
    g = torch.Generator(device=DEV).manual_seed(M + E)
    w = torch.randint(-128, 128, (E, N, K), dtype=torch.int8, device=DEV, generator=g)
    q, s, ws = dev(codes(rng, (M, K))), dev(scales(rng, M, K)), dev(scales(rng, (E, N), K))
    got = torch.full((M, N // 2 if sw else N), 7.0, dtype=TYPES[out], device=DEV)
    blk.matmul_i8(q, s, w, ws, got, offsets=dev(offsets), perm=dev(perm) if gather else None, swiglu=sw, clamp=2.0)
    assert (got[kept:] == 7.0).all()
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        if lo < hi:
            at = dev(perm[lo:hi].astype(np.int64)) if gather else torch.arange(lo, hi, device=DEV)
            check_against(got[lo:hi], ref.product(q[at], s[at], w[e], ws[e]).cpu(), sw, 2.0, TYPES[out])


def test_row_map_entries_outside_the_sources_are_zero_rows(blk):
    say("row map entries outside the sources")
    rng = np.random.default_rng(8)
    T, k, K, N = 6, 2, 128, 80
    perm = np.array([0, 11, 12, -1, 2 ** 31 - 1, 5, -2 ** 31, 3], np.int32)
    q, w, s, ws = codes(rng, (T, K)), codes(rng, (2, N, K)), scales(rng, T, K), scales(rng, (2, N), K)
    got = torch.full((8, N), float("nan"), device=DEV)
    blk.matmul_i8(dev(q), dev(s), dev(w), dev(ws), got, offsets=dev(np.array([0, 4, 8], np.int32)), perm=dev(perm), k=k)
    got = got.cpu()
    assert (got[[2, 3, 4, 6]] == 0).all()
    for r in (0, 1, 5, 7):
        t = [perm[r] // k]
        check_product(got[[r]], q[t], s[t], w[r // 4], ws[r // 4], False, 0.0, torch.float32)


@pytest.mark.parametrize("K, sw", [(192, False), (192, True), (77, False)])
def test_dense_product_through_a_row_map(blk, K, sw):
    """One matrix, rows taken through perm (the same source more than once)."""
    say("dense product through a row map", K, sw)
    rng = np.random.default_rng(21)
    S, M, N = 9, 150, 72
    perm = rng.integers(0, S * 3, M).astype(np.int32)
    q, w, s, ws = codes(rng, (S, K)), codes(rng, (N, K)), scales(rng, S, K), scales(rng, N, K)
    got = torch.full((M, N // 2 if sw else N), float("nan"), device=DEV)
    blk.matmul_i8(dev(q), dev(s), dev(w), dev(ws), got, perm=dev(perm), k=3, swiglu=sw)
    at = torch.from_numpy(perm.astype(np.int64) // 3)
    check_product(got, q[at], s[at], w, ws, sw, 0.0, torch.float32)


@pytest.mark.parametrize("M, N, K", [(1, 72, 192), (12, 72, 192), (40, 200, 192), (4, 4098, 208)])
@pytest.mark.parametrize("sw", [False, True])
def test_dense_product_of_few_rows_through_a_row_map(blk, M, N, K, sw):
    say("dense product of few rows through a row map", M, N, K, sw)
    rng = np.random.default_rng(M + N)
    S = 9
    perm = rng.integers(0, S * 3, M).astype(np.int32)
    q, w, s, ws = codes(rng, (S, K)), codes(rng, (N, K)), scales(rng, S, K), scales(rng, N, K)
    at = torch.from_numpy(perm.astype(np.int64) // 3)
    y = ref.product(q[at], s[at], w, ws)
    if M > 1:  # a row from outside the sources
        perm[M // 2] = S * 3
        y[M // 2] = 0.0
    got = torch.full((M, N // 2 if sw else N), float("nan"), device=DEV)
    blk.matmul_i8(dev(q), dev(s), dev(w), dev(ws), got, perm=dev(perm), k=3, swiglu=sw)
    check_against(got, y, sw, 0.0, torch.float32)


def test_offsets_past_32_bits(blk):
    """Buffers of more than 4 GiB: the rows at their ends."""
    say("offsets past 32 bits: rows")
    H, R = 4096, 600_000  # 4.9 GB of bf16
    T, k = 4, 2
    inv = np.array([R - 1, 0, 3, R // 2, -1, R - 2, 524_288, 524_289], np.int32)  # 524288 * H * 2 is 2^32
    rng = np.random.default_rng(22)
    x, wts = floats(rng, (T, H), "bf16"), floats(rng, (T, k), "f32")
    rows = torch.zeros((R, H), dtype=torch.bfloat16, device=DEV)
    blk.dispatch(dev(x), dev(inv), rows)
    at = [R - 1, 0, 3, R // 2, R - 2, 524_288, 524_289]
    assert torch.equal(rows[at].cpu(), x[[0, 0, 1, 1, 2, 3, 3]])
    out, dx = torch.empty((T, H), device=DEV), torch.empty((T, H), dtype=torch.bfloat16, device=DEV)
    blk.combine(rows, dev(wts), dev(inv), out)
    there = torch.from_numpy(inv.reshape(T, k) >= 0)
    w = torch.where(there, wts, torch.zeros(()))
    want = x.double() * w.double().sum(1, keepdim=True)
    close(out, want, (k + 1) * U * x.double().abs() * w.double().abs().sum(1, keepdim=True))
    blk.dispatch_grad(rows, dev(inv), dx)
    assert torch.equal(dx.cpu(), (x.float() * there.sum(1, keepdim=True)).to(torch.bfloat16))
    drows, dwts = torch.zeros_like(rows), torch.empty((T, k), device=DEV)
    blk.combine_grad(dev(x), rows, dev(wts), dev(inv), drows, dwts)
    flat = torch.from_numpy(inv.astype(np.int64))
    pair = torch.nonzero(flat >= 0).view(-1)
    v = x[pair // k].double() * wts.view(-1)[pair, None].double()
    close(drows[flat[pair].to(DEV)], v, ref.rounded(U * v.abs(), v, torch.bfloat16))
    del rows, drows
    torch.cuda.empty_cache()
    say("offsets past 32 bits: products")
    for S, K, E, N in ((300_000, 16384, 2, 40), (70, 16384, 70, 4096)):  # 4.9 GB of codes; 4.7 GB of weights
        q = torch.zeros((S, K), dtype=torch.int8, device=DEV)
        w = torch.zeros((E, N, K), dtype=torch.int8, device=DEV)
        M = 70
        src = np.linspace(0, S - 1, M).astype(np.int32)
        src[-1] = S - 1
        qc, wc = codes(rng, (M, K)), codes(rng, (2, N, K))
        q[torch.from_numpy(src.astype(np.int64)).to(DEV)] = dev(qc)
        w[0], w[E - 1] = dev(wc[0]), dev(wc[1])
        s, ws = scales(rng, S, K), scales(rng, (E, N), K)
        offsets = np.full(E + 1, 30, np.int32)
        offsets[0], offsets[E] = 0, M
        got = torch.full((M, N), float("nan"), device=DEV)
        blk.matmul_i8(q, dev(s), w, dev(ws), got, offsets=dev(offsets), perm=dev(src))
        st = s[torch.from_numpy(src.astype(np.int64))]
        check_product(got[:30], qc[:30], st[:30], wc[0], ws[0], False, 0.0, torch.float32)
        check_product(got[30:], qc[30:], st[30:], wc[1], ws[E - 1], False, 0.0, torch.float32)
        del q, w
        torch.cuda.empty_cache()


def test_rows_at_odd_addresses(blk):
    say("dispatch and combine at odd addresses")
    rng = np.random.default_rng(23)
    T, k, H = 5, 3, 520
    inv = np.arange(T * k, dtype=np.int32)[::-1].copy()
    for kind in ("bf16", "f32"):
        put = lambda t, o: torch.cat([torch.zeros(o, dtype=t.dtype), t.view(-1)]).to(DEV)[o:].view(t.shape)  # noqa: E731
        x, wts = floats(rng, (T, H), kind), floats(rng, (T, k), "f32")
        rows = put(torch.zeros((T * k, H), dtype=TYPES[kind]), 3)
        blk.dispatch(put(x, 1), dev(inv), rows)
        assert torch.equal(rows.cpu()[torch.from_numpy(inv.astype(np.int64))], x.repeat_interleave(k, 0))
        out = put(torch.zeros((T, H)), 1)
        blk.combine(rows, put(wts, 1), dev(inv), out)
        want, mag = ref.combine(rows.cpu(), wts, inv, T, k)
        close(out, want, (k + 1) * U * mag)
        drows, dwts = put(torch.zeros((T * k, H), dtype=TYPES[kind]), 1), put(torch.zeros((T, k)), 1)
        blk.combine_grad(put(x, 3), rows, put(wts, 1), dev(inv), drows, dwts)
        v = x.repeat_interleave(k, 0).double() * wts.view(-1, 1).double()
        close(drows[torch.from_numpy(inv.astype(np.int64)).to(DEV)], v, ref.rounded(U * v.abs(), v, TYPES[kind]))


def test_offsets_are_held_to_the_rows(blk):
    """Offsets that leave [0, M] or fall are cut, not followed: the rows inside are right, nothing else is written."""
    say("offsets held to the rows")
    rng = np.random.default_rng(9)
    M, K, N = 20, 64, 32
    q, w, s, ws = codes(rng, (M, K)), codes(rng, (3, N, K)), scales(rng, M, K), scales(rng, (3, N), K)
    got = torch.full((M + 4, N), 7.0, device=DEV)
    blk.matmul_i8(dev(q), dev(s), dev(w), dev(ws), got[:M], offsets=dev(np.array([-5, 8, 3, 900], np.int32)))
    assert (got[M:] == 7.0).all()
    check_product(got[:3], q[:3], s[:3], w[0], ws[0], False, 0.0, torch.float32)


def test_a_row_with_nan_or_infinity_is_nan_and_no_other(blk):
    say("rows with NaN and infinity")
    rng = np.random.default_rng(10)
    M, K, N = 70, 256, 96
    x = floats(rng, (M, K), "f32")
    x[3, 7], x[40, 0] = float("nan"), float("inf")
    q, s = torch.empty((M, K), dtype=torch.int8, device=DEV), torch.empty(M, device=DEV)
    blk.quantize_i8(dev(x), q, s)
    w, ws = codes(rng, (N, K)), scales(rng, N, K)
    for sw, L in ((False, 0.0), (True, 1.0)):
        got = torch.empty((M, N // 2 if sw else N), device=DEV)
        blk.matmul_i8(q, s, dev(w), dev(ws), got, swiglu=sw, clamp=L)
        bad = got.cpu().isnan()
        assert bad[3].all() and bad[40].all() and not bad[[r for r in range(M) if r not in (3, 40)]].any()


# ---- as they are used ------------------------------------------------------------------


def test_training_step_through_the_experts(blk):
    """route -> group -> dispatch -> the caller's expert products -> combine, and back, against torch's own
    gradients of the whole in 64 bits."""
    T, k, E, H = 50, 2, 6, 48
    say("training step", T, k, E, H)
    rng = np.random.default_rng(11)
    x, logits = floats(rng, (T, H), "f32"), floats(rng, (T, E), "f32")
    W = torch.from_numpy(rng.standard_normal((E, H, H)) / H ** 0.5)
    dout = floats(rng, (T, H), "f32")
    ids, wts = torch.empty((T, k), dtype=torch.int32, device=DEV), torch.empty((T, k), device=DEV)
    blk.route(dev(logits), k, mb.ROUTE_SOFTMAX, True, 1.0, ids, wts)
    n = lambda m: torch.empty(m, dtype=torch.int32, device=DEV)  # noqa: E731
    counts, offsets, perm, inv = n(E), n(E + 1), n(T * k), n(T * k)
    blk.group(ids, E, counts, offsets, perm, inv)
    rows, out = torch.empty((T * k, H), device=DEV), torch.empty((T, H), device=DEV)
    blk.dispatch(dev(x), inv, rows)
    off = offsets.cpu().tolist()
    Wd = W.to(DEV)
    y = torch.empty((T * k, H), device=DEV)
    for e in range(E):
        y[off[e]:off[e + 1]] = (rows[off[e]:off[e + 1]].double() @ Wd[e]).float()
    blk.combine(y, wts, inv, out)
    dy, dwts, dx = torch.empty_like(y), torch.empty_like(wts), torch.empty((T, H), device=DEV)
    blk.combine_grad(dev(dout), y, wts, inv, dy, dwts)
    drows = torch.empty_like(rows)
    for e in range(E):
        drows[off[e]:off[e + 1]] = (dy[off[e]:off[e + 1]].double() @ Wd[e].t().contiguous()).float()
    blk.dispatch_grad(drows, inv, dx)
    xr, wr = x.double().requires_grad_(), wts.cpu().double().requires_grad_()
    idc = ids.cpu().long()
    want = sum(wr[:, s, None] * torch.stack([xr[t] @ W[idc[t, s]] for t in range(T)]) for s in range(k))
    want.backward(dout.double())
    # sums of H products of size about 1 and of k rows, and a few f32 roundings: all below 1e-5 of the values' size
    for got, exact in ((out, want.detach()), (dx, xr.grad), (dwts, wr.grad)):
        assert (got.cpu().double() - exact).abs().max() <= 1e-5 * exact.abs().max()


def w8a8(blk, x, ids, wts, gu, dn, k, E, L):
    """The routed experts in 8 bits: (out, h) of tokens x."""
    T, H = x.shape
    F = dn[0].shape[2]
    P = T * k
    n = lambda m: torch.empty(m, dtype=torch.int32, device=DEV)  # noqa: E731
    counts, offsets, perm, inv = n(E), n(E + 1), n(P), n(P)
    blk.group(ids, E, counts, offsets, perm, inv)
    q, s = torch.empty((T, H), dtype=torch.int8, device=DEV), torch.empty(T, device=DEV)
    blk.quantize_i8(x, q, s)
    h = torch.zeros((P, F), dtype=torch.bfloat16, device=DEV)
    blk.matmul_i8(q, s, *gu, h, offsets=offsets, perm=perm, k=k, swiglu=True, clamp=L)
    hq, hs = torch.empty((P, F), dtype=torch.int8, device=DEV), torch.empty(P, device=DEV)
    blk.quantize_i8(h, hq, hs)
    y = torch.zeros((P, H), dtype=torch.bfloat16, device=DEV)
    blk.matmul_i8(hq, hs, *dn, y, offsets=offsets)
    out = torch.empty((T, H), device=DEV)
    blk.combine(y, wts, inv, out)
    return out, h, y, (offsets, perm, inv)


def quantized_weights(blk, rng, E, N, K):
    w = dev(rng.standard_normal((E * N, K)).astype(np.float32) / K ** 0.5)
    q, s = torch.empty((E * N, K), dtype=torch.int8, device=DEV), torch.empty(E * N, device=DEV)
    blk.quantize_i8(w, q, s)
    return q.view(E, N, K), s.view(E, N)


@pytest.mark.parametrize("T, skew", [(1, False), (16, True), (200, True), (2050, False)])
def test_experts_in_8_bits(blk, T, skew):
    """Quantise, gate/up with SwiGLU, quantise, down, combine, at the small layer's shape: every stage against 64 bits
    from the stage before it (so that a code next to a tie is the kernel's own)."""
    H, F, E, k = wl.C1.hidden, wl.C1.ffn, wl.C1.n_expert, wl.C1.n_used
    say("experts in 8 bits", T, skew)
    rng = np.random.default_rng(T)
    gu, dn = quantized_weights(blk, rng, E, 2 * F, H), quantized_weights(blk, rng, E, H, F)
    x = floats(rng, (T, H), "bf16")
    ids = ref.ids_of(rng, T, k, E, 0.1 if T > 1 else 0.0, skew)
    wts = torch.from_numpy(rng.random((T, k)).astype(np.float32))
    out, h, y, (offsets, perm, inv) = w8a8(blk, dev(x), dev(ids), dev(wts), gu, dn, k, E, 2.0)
    ro, rp, ri, kept = ref.grouping(ids, E)
    assert np.array_equal(offsets.cpu().numpy(), ro) and np.array_equal(inv.cpu().numpy(), ri)
    xq, xs = ref.quantize(x)
    hc, yc = h.cpu(), y.cpu()
    hq, hs = ref.quantize(hc)
    for e in np.nonzero(np.diff(ro))[0][:6]:
        r = slice(ro[e], ro[e + 1])
        t = torch.from_numpy(rp[r].astype(np.int64) // k)
        check_product(hc[r], xq[t], xs[t], gu[0][e].cpu(), gu[1][e].cpu(), True, 2.0, torch.bfloat16)
        check_product(yc[r], hq[r], hs[r], dn[0][e].cpu(), dn[1][e].cpu(), False, 0.0, torch.bfloat16)
    want, mag = ref.combine(yc, wts, ri, T, k)
    close(out, want, ref.rounded((k + 1) * U * mag, want, torch.float32))


def test_captured_and_replayed(blk):
    """The 8-bit experts and the gradients captured in a graph of another stream, replayed on new inputs with eager
    work between: every replay equals the eager result bit for bit."""
    T, k, E, H, F = 24, 2, 8, 256, 128
    say("captured and replayed")
    rng = np.random.default_rng(12)
    gu, dn = quantized_weights(blk, rng, E, 2 * F, H), quantized_weights(blk, rng, E, H, F)
    x, ids = dev(floats(rng, (T, H), "bf16")), dev(ref.ids_of(rng, T, k, E, 0.2, True))
    wts, dout = dev(floats(rng, (T, k), "f32")), dev(floats(rng, (T, H), "f32"))

    def step():
        out, h, y, (offsets, perm, inv) = w8a8(blk, x, ids, wts, gu, dn, k, E, 0.0)
        dy, dwts = torch.zeros_like(y), torch.empty_like(wts)
        blk.combine_grad(dout, y, wts, inv, dy, dwts)
        dx = torch.empty((T, H), device=DEV)
        blk.dispatch_grad(dy, inv, dx)
        rows = torch.zeros((T * k, H), device=DEV)
        blk.dispatch(x, inv, rows)
        return out, dwts, dx, rows

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for i in range(4):
        x.copy_(floats(rng, (T, H), "bf16"))
        ids.copy_(torch.from_numpy(ref.ids_of(rng, T, k, E, 0.2, True)))
        dout.copy_(floats(rng, (T, H), "f32"))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b), i


def test_calls_are_the_same_without_the_compiled_comparison(blk):
    """moe_torch and ctypes: the same results, on torch's current stream and on a given one."""
    say("calls without the compiled comparison")
    assert blk._calls, "moe_torch.so was not built for this torch"
    rng = np.random.default_rng(31)
    T, k, E, H, N = 37, 4, 8, 144, 96
    ids = ref.ids_of(rng, T, k, E, 0.2)
    offsets, perm, inv, kept = ref.grouping(ids, E)
    x, rows, y = floats(rng, (T, H), "bf16").to(DEV), floats(rng, (T * k, H), "f16").to(DEV), floats(rng, (T, H), "f32").to(DEV)
    wts = dev(rng.random((T, k)).astype(np.float32))
    q, w, s, ws = dev(codes(rng, (T, H))), dev(codes(rng, (E, N, H))), dev(scales(rng, T, H)), dev(scales(rng, (E, N), H))
    offsets, perm, inv = dev(offsets), dev(perm), dev(inv)

    def every(stream):
        z = lambda shape, t: torch.zeros(shape, dtype=t, device=DEV)  # noqa: E731
        o = [z((T * k, H), torch.float32), z((T, H), torch.bfloat16), z((T, H), torch.float32), z((T * k, H), torch.float16),
             z((T, k), torch.float32), z((T, H), torch.int8), z((T,), torch.float32), z((T * k, N // 2), torch.bfloat16),
             z((T, N), torch.float16)]
        torch.cuda.synchronize()
        blk.dispatch(x, inv, o[0], stream=stream)
        blk.dispatch_grad(rows, inv, o[1], stream=stream)
        blk.combine(rows, wts, inv, o[2], stream=stream)
        blk.combine_grad(y, rows, wts, inv, o[3], o[4], stream=stream)
        blk.quantize_i8(x, o[5], o[6], stream=stream)
        blk.matmul_i8(q, s, w, ws, o[7], offsets=offsets, perm=perm, k=k, swiglu=True, clamp=1.0, stream=stream)
        blk.matmul_i8(q, s, w[2], ws[2], o[8], stream=stream)
        torch.cuda.synchronize()
        return o

    want = every(None)
    calls, other = blk._calls, torch.cuda.Stream()
    got = [every(other.cuda_stream)]
    try:
        blk._calls = None
        got += [every(None), every(other.cuda_stream)]
    finally:
        blk._calls = calls
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(want, o))


def test_two_streams_at_once(blk):
    say("two streams at once")
    rng = np.random.default_rng(13)
    M, N, K = 96, 640, 2048
    w, ws = codes(rng, (N, K)), scales(rng, N, K)
    wd, wsd = dev(w), dev(ws)
    qs = [(codes(rng, (M, K)), scales(rng, M, K)) for _ in range(2)]
    put = [(dev(a), dev(b)) for a, b in qs]
    outs = [torch.empty((M, N), device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(8):
        for (a, b), o, st in zip(put, outs, streams):
            blk.matmul_i8(a, b, wd, wsd, o, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for (a, b), o in zip(qs, outs):
        check_product(o, a, b, w, ws, False, 0.0, torch.float32)


def test_refusals_of_the_library(blk):
    """What the C-ABI itself refuses, with a message, launching nothing."""
    say("refusals")
    lib, h = blk.lib, blk.h
    buf = torch.zeros(4096, device=DEV)
    p, F32 = buf.data_ptr(), mb.GGML_F32
    bad = [
        lib.moe_dispatch(h, p, 99, p, 1, 1, 4, 1, p, F32, None),          # type
        lib.moe_dispatch(h, p + 2, F32, p, 1, 1, 4, 1, p, F32, None),     # alignment
        lib.moe_dispatch(h, None, F32, p, 1, 1, 4, 1, p, F32, None),
        lib.moe_dispatch(h, p, F32, p, 0, 1, 4, 1, p, F32, None),
        lib.moe_dispatch(h, p, F32, p, 1, 65, 4, 1, p, F32, None),
        lib.moe_combine(h, p, F32, 1, None, p, 1, 1, 4, p, F32, None),
        lib.moe_combine_grad(h, p, F32, p, F32, 1, p, p, 1, 1, 4, p, p, None),  # drows is rows
        lib.moe_quantize_i8(h, p, F32, 0, 4, p, p, None),
        lib.moe_quantize_i8(h, p, F32, 1, 2 ** 30 + 1, p, p, None),
        lib.moe_matmul_i8(h, p, p, 1, p, p, 2, None, None, 1, 1, 1, 4, 0, 0.0, p, F32, None),     # E without offsets
        lib.moe_matmul_i8(h, p, p, 1, p, p, 1025, p, None, 1, 1, 1, 4, 0, 0.0, p, F32, None),
        lib.moe_matmul_i8(h, p, p, 1, p, p, 1, None, None, 1, 2, 1, 4, 0, 0.0, p, F32, None),     # fewer sources than rows
        lib.moe_matmul_i8(h, p, p, 1, p, p, 1, None, None, 1, 1, 3, 4, 1, 0.0, p, F32, None),     # SwiGLU of odd channels
        lib.moe_matmul_i8(h, p, p, 1, p, p, 1, None, None, 1, 1, 2, 4, 2, 0.0, p, F32, None),     # unknown flag
        lib.moe_matmul_i8(h, p, p, 1, p, p, 1, None, None, 1, 1, 2, 4, 1, float("nan"), p, F32, None),
    ]
    assert bad == [mb.MOE_ERR_INVALID_ARG] * len(bad)
    # more than a launch takes (checked before anything is read; the addresses are never used)
    far = [p + (i << 44) for i in range(8)]
    big = [
        lib.moe_dispatch(h, far[0], F32, far[1], 2 ** 24, 1, 4, 1, far[2], F32, None),
        lib.moe_combine(h, far[0], F32, 1, far[1], far[2], 2 ** 24, 1, 4, far[3], F32, None),
        lib.moe_dispatch_grad(h, far[0], F32, 1, far[1], 2 ** 24, 1, 4, far[2], F32, None),
        lib.moe_combine_grad(h, far[0], F32, far[1], F32, 1, far[2], far[3], 2 ** 21, 64, 4, far[4], far[5], None),
        lib.moe_quantize_i8(h, far[0], F32, 2 ** 24, 4, far[1], far[2], None),
        lib.moe_matmul_i8(h, far[0], far[1], 2 ** 30, far[2], far[3], 1, None, None, 1, 2 ** 30, 64, 64, 0, 0.0, far[4], F32, None),
        lib.moe_matmul_i8(h, far[0], far[1], 2 ** 30, far[2], far[3], 1, None, None, 1, 2 ** 30, 64, 63, 0, 0.0, far[4], F32, None),
    ]
    assert big == [mb.MOE_ERR_UNSUPPORTED] * len(big)
    assert b"moe_matmul_i8" in lib.moe_ctx_last_error(h)
    torch.cuda.synchronize()
    assert (buf == 0).all()


def test_overlapping_buffers_are_refused(blk):
    say("overlapping buffers")
    H, T, k = 32, 4, 2
    a = torch.zeros((20, H), device=DEV)
    inv, wts = torch.zeros(T * k, dtype=torch.int32, device=DEV), torch.zeros((T, k), device=DEV)
    z8 = torch.zeros((20, H), dtype=torch.int8, device=DEV)
    for call in (lambda: blk.dispatch(a[:T], inv, a[T - 1:12]),
                 lambda: blk.dispatch_grad(a[:8], inv, a[7:7 + T]),
                 lambda: blk.combine(a[:8], wts, inv, a[4:4 + T]),
                 lambda: blk.combine(a[:8], wts, inv, a[8:8 + T]) or blk.combine(a[:8], a[8, :8].view(T, k), inv, a[8:12]),
                 lambda: blk.combine_grad(a[:T], a[4:12], wts, inv, a[4:12], torch.zeros_like(wts)),
                 lambda: blk.combine_grad(a[:T], a[4:12], wts, inv, torch.zeros_like(a[:8]), wts),
                 lambda: blk.quantize_i8(a[:T], z8[:T], a[3, :T]),
                 lambda: blk.quantize_i8(a[:T], a[:1].view(torch.int8).view(T, H), torch.zeros(T, device=DEV)),
                 lambda: blk.matmul_i8(z8[:T], wts[:, 0].contiguous(), z8[4:8], a[0, :4], a[0, :16].view(T, 4))):
        with pytest.raises(mb.MoeError, match="overlaps") as ei:
            call()
        assert ei.value.status == mb.MOE_ERR_INVALID_ARG
    torch.cuda.synchronize()


def test_profiler_counts_the_operators(blk):
    say("profiler")
    blk.prof_enable(True)
    blk.prof_read()
    x, q, s = torch.ones((4, 64), device=DEV), torch.empty((4, 64), dtype=torch.int8, device=DEV), torch.empty(4, device=DEV)
    blk.quantize_i8(x, q, s)
    got = blk.prof_read()
    blk.prof_enable(False)
    assert got["quantize_i8"][0] == 1


def test_a_callers_capture_is_not_timed(blk):
    """With the profiler on, calls that a caller captures record no events into the graph: every replay is right, and
    the profiler still reads and counts the eager calls, and only those."""
    say("a caller's capture with the profiler on")
    T, k, E, H, N = 12, 2, 8, 64, 48
    rng = np.random.default_rng(41)
    x, ids = dev(floats(rng, (T, H), "f32")), dev(ref.ids_of(rng, T, k, E))
    w, ws = dev(codes(rng, (N, H))), dev(scales(rng, N, H))
    n = lambda m: torch.empty(m, dtype=torch.int32, device=DEV)  # noqa: E731
    counts, offsets, perm, inv = n(E), n(E + 1), n(T * k), n(T * k)
    q, s = torch.empty((T, H), dtype=torch.int8, device=DEV), torch.empty(T, device=DEV)
    out, rows = torch.empty((T, N), device=DEV), torch.zeros((T * k, H), device=DEV)

    def step():
        blk.group(ids, E, counts, offsets, perm, inv)
        blk.dispatch(x, inv, rows)
        blk.quantize_i8(x, q, s)
        blk.matmul_i8(q, s, w, ws, out)

    step()
    torch.cuda.synchronize()
    blk.prof_enable(True)
    try:
        blk.prof_read(reset=True)
        step()  # the profiler holds events of its own by now
        names = ("group", "dispatch", "quantize_i8", "matmul_i8")
        assert {m: c for m, (c, _) in blk.prof_read(reset=True).items()} == {m: 1 for m in names}
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        assert blk.prof_read(reset=True) == {}
        for i in range(3):
            x.copy_(floats(rng, (T, H), "f32"))
            g.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in (rows, q, s, out)]
            step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (rows, q, s, out))), i
        assert {m: c for m, (c, _) in blk.prof_read(reset=True).items()} == {m: 3 for m in names}
    finally:
        blk.prof_enable(False)


def test_two_threads_on_one_context(blk):
    """Each on a stream of its own, with the profiler on, good calls between refused ones: every result is right,
    every refusal has one of the messages whole, and every launch is counted once."""
    say("two threads on one context")
    rng = np.random.default_rng(42)
    M, N, K, n, wrong = 24, 80, 208, 150, []
    w, ws = codes(rng, (N, K)), scales(rng, N, K)
    wd, wsd = dev(w), dev(ws)
    sets = [(codes(rng, (M, K)), scales(rng, M, K)) for _ in range(2)]
    put = [(dev(a), dev(b)) for a, b in sets]
    outs = [torch.zeros((n, M, N), device=DEV) for _ in range(2)]
    x = torch.zeros((4, 32), device=DEV)
    inv, clash = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros((4, 32), device=DEV)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    go = threading.Barrier(2)

    def work(i):
        try:
            st = streams[i].cuda_stream
            go.wait(60)
            for j in range(n):
                blk.matmul_i8(*put[i], wd, wsd, outs[i][j], stream=st)
                with pytest.raises(mb.MoeError, match="moe_dispatch: rows overlaps another buffer|"
                                                      "moe_quantize_i8: an output overlaps another buffer"):
                    if i:
                        blk.dispatch(x, inv, x, stream=st)
                    else:
                        blk.quantize_i8(clash, clash.view(-1)[:32].view(torch.int8).view(4, 32), ws4, stream=st)
        except BaseException as e:  # noqa: BLE001 -- a thread's failure is the test's
            wrong.append(e)

    ws4 = torch.zeros(4, device=DEV)
    blk.prof_enable(True)
    try:
        blk.prof_read(reset=True)
        both = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in both:
            t.start()
        for t in both:
            t.join()
        torch.cuda.synchronize()
        stats = blk.prof_read(reset=True)
    finally:
        blk.prof_enable(False)
    assert not wrong, wrong
    assert {m: c for m, (c, _) in stats.items()} == {"matmul_i8": 2 * n}
    for (a, b), o in zip(sets, outs):
        assert (o == o[:1]).all()
        check_product(o[0], a, b, w, ws, False, 0.0, torch.float32)


def whole_numbers(rng, shape, m):
    return torch.from_numpy(rng.integers(-m, m + 1, shape, dtype=np.int64).astype(np.int8))


@pytest.mark.parametrize("E", [0, 1024])
@pytest.mark.parametrize("K", [3, 16])
@pytest.mark.parametrize("M", [65535 * 64 + 1, 2 ** 22 + 65])
def test_rows_past_one_dimension_of_a_grid(blk, M, K, E):
    """More tiles of rows than one grid dimension may hold, by either path: dense, and of 1024 experts.  Scales of 1
    and sums below 2^24: the products are exact."""
    say("rows past one dimension of a grid", M, K, E)
    rng = np.random.default_rng(M + K + E)
    N = 2
    q, w = dev(whole_numbers(rng, (M, K), 127)), dev(whole_numbers(rng, (max(E, 1), N, K), 127))
    one, ones = torch.ones(M, device=DEV), torch.ones((max(E, 1), N), device=DEV)
    got = torch.full((M + 1, N), 7.0, device=DEV)
    if E:
        cuts = np.sort(rng.integers(0, M + 1, E - 1))
        offsets = dev(np.concatenate([[0], cuts, [M]]).astype(np.int32))
        blk.matmul_i8(q, one, w, ones, got[:M], offsets=offsets)
        e = torch.searchsorted(offsets[1:].long(), torch.arange(M, device=DEV), right=True)
    else:
        blk.matmul_i8(q, one, w[0], ones[0], got[:M])
        e = torch.zeros(M, dtype=torch.int64, device=DEV)
    want = torch.stack([(q.int() * w[:, n].int()[e]).sum(1) for n in range(N)], 1)
    assert torch.equal(got[:M], want.float()) and (got[M:] == 7.0).all()


@pytest.mark.parametrize("K", [5, 16])
def test_the_most_rows_of_a_product(blk, K):
    """2^30 - 1 rows of few sources through a row map, by either path (one more is refused, test_refusals_of_the_library)."""
    say("the most rows of a product", K)
    rng = np.random.default_rng(K)
    M, S, N = 2 ** 30 - 1, 61, 1
    q, w = whole_numbers(rng, (S, K), 8), whole_numbers(rng, (N, K), 1)
    perm = torch.arange(M, dtype=torch.int32, device=DEV).remainder_(S)
    got = torch.zeros((M, N), dtype=torch.bfloat16, device=DEV)
    blk.matmul_i8(dev(q), torch.ones(S, device=DEV), dev(w), torch.ones(N, device=DEV), got, perm=perm)
    want = dev((q.int() * w.int()).sum(1).to(torch.bfloat16))  # at most 128: exact
    whole = M // S * S
    assert (got[:whole, 0].view(-1, S) == want).all() and torch.equal(got[whole:, 0], want[:M - whole])
    del got, perm
    torch.cuda.empty_cache()


# ---- buffers past the caches -----------------------------------------------------------

STREAM_BYTES = 96 << 20  # what is moved past the caches from here on (MOE_STREAM_BYTES)


def close_here(got, want, bound):
    """close(), on the device."""
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all() and (off <= bound).all(), f"off by {(off / bound.clamp(min=1e-300)).max().item():.3g} of the bound"


def setup_here(T, k, H, dropped, seed):
    """setup(), with the map on the device too: [T, k] rows, and which pairs have one."""
    rng, ids, E, inv, kept = setup(T, k, H, dropped, seed)
    at = dev(inv.astype(np.int64)).view(T, k)
    return rng, dev(inv), at, at >= 0, kept


def floats_here(g, shape, kind):
    return torch.randn(shape, generator=g, device=DEV).to(TYPES[kind])


# tokens, slots (up to 8 of them in flight, and more), type read, type written, dropped
PAST = [(1500, 8, "f32", "f32", 0.2), (1501, 8, "bf16", "bf16", 0.0), (401, 17, "f32", "f16", 0.3), (400, 17, "bf16", "f32", 0.1),
        (9000, 1, "f16", "f16", 0.0), (5003, 3, "f16", "bf16", 0.25), (36, 9, "bf16", "bf16", 0.2)]


def odd_width(pairs, kind, part=1):
    """The smallest odd H with which so many rows pass STREAM_BYTES / part."""
    size = 4 if kind == "f32" else 2
    return (STREAM_BYTES // part // (pairs * size) + 1) | 1


@pytest.mark.parametrize("T, k, a, b, dropped", PAST)
def test_dispatch_past_the_caches(blk, T, k, a, b, dropped):
    H = odd_width(T * k, b)
    say("dispatch past the caches", T, k, H, a, b, dropped)
    rng, inv, at, there, kept = setup_here(T, k, H, dropped, T + k)
    g = torch.Generator(device=DEV).manual_seed(T)
    x = floats_here(g, (T, H), a)
    got = torch.full((T * k + 1, H), 7.0, dtype=TYPES[b], device=DEV)
    blk.dispatch(x, inv, got)
    want = torch.full_like(got, 7.0)
    t, s = torch.nonzero(there, as_tuple=True)
    want[at[t, s]] = x[t].to(TYPES[b])
    assert torch.equal(got, want)


@pytest.mark.parametrize("T, k, a, b, dropped", PAST)
def test_combine_and_dispatch_grad_past_the_caches(blk, T, k, a, b, dropped):
    H = odd_width(T * k, a)
    say("combine past the caches", T, k, H, a, b, dropped)
    rng, inv, at, there, kept = setup_here(T, k, H, dropped, 2 * T + k)
    g = torch.Generator(device=DEV).manual_seed(T)
    rows, wts = floats_here(g, (kept, H), a), floats_here(g, (T, k), "f32")
    for w in (wts, None):
        out = torch.full((T, H), float("nan"), dtype=TYPES[b], device=DEV)
        if w is None:
            blk.dispatch_grad(rows, inv, out)
        else:
            blk.combine(rows, w, inv, out)
        want = torch.zeros((T, H), dtype=torch.float64, device=DEV)
        mag = torch.zeros_like(want)
        for s in range(k):
            t = torch.nonzero(there[:, s]).view(-1)
            y = rows[at[t, s]].double() * (1.0 if w is None else w[t, s, None].double())
            want[t] += y
            mag[t] += y.abs()
        close_here(out, want, ref.rounded((k + 1) * U * mag, want, TYPES[b]))  # as test_combine_and_dispatch_grad


@pytest.mark.parametrize("T, k, a, b, dropped", PAST)
def test_combine_grad_past_the_caches(blk, T, k, a, b, dropped):
    H = odd_width(T * k, b, 2)
    say("combine_grad past the caches", T, k, H, a, b, dropped)
    rng, inv, at, there, kept = setup_here(T, k, H, dropped, 3 * T + k)
    g = torch.Generator(device=DEV).manual_seed(T)
    R = kept + 1
    dout, rows, wts = floats_here(g, (T, H), a), floats_here(g, (R, H), b), floats_here(g, (T, k), "f32")
    drows = torch.full((R, H), 7.0, dtype=TYPES[b], device=DEV)
    dwts = torch.full((T, k), float("nan"), device=DEV)
    blk.combine_grad(dout, rows, wts, inv, drows, dwts)
    want = torch.full((R, H), 7.0, dtype=torch.float64, device=DEV)
    dw, mag = (torch.zeros((T, k), dtype=torch.float64, device=DEV) for _ in range(2))
    for s in range(k):
        t = torch.nonzero(there[:, s]).view(-1)
        want[at[t, s]] = dout[t].double() * wts[t, s, None].double()
        prod = dout[t].double() * rows[at[t, s]].double()
        dw[t, s], mag[t, s] = prod.sum(1), prod.abs().sum(1)
    close_here(drows, want, ref.rounded(U * want.abs(), want, TYPES[b]))
    close_here(dwts, dw, (H / 64 + 8 + 9) * U * mag + 1e-40)  # as test_combine_grad


# rows, N, K: weights past the caches against few rows and many, on every tile shape that the cost rule takes for them
WIDE = [(16, 65538, 7184), (16, 12290, 8208), (16, 24578, 4112), (65, 12290, 8208), (65, 24578, 4112), (65, 65538, 2064),
        (65, 102402, 1040), (130, 102402, 1040), (130, 12290, 8208), (130, 24578, 4112), (130, 65538, 2064),
        (257, 102402, 1040), (770, 12290, 8208), (4001, 12290, 8208)]


@pytest.mark.parametrize("M, N, K", WIDE)
@pytest.mark.parametrize("out, sw", [("f32", False), ("bf16", True)])
def test_dense_product_with_weights_past_the_caches(blk, M, N, K, out, sw):
    say("dense product with weights past the caches", M, N, K, out, sw)
    rng = np.random.default_rng(M + N + K)
    g = torch.Generator(device=DEV).manual_seed(M + N)
    q, w = (torch.randint(-128, 128, s, dtype=torch.int8, device=DEV, generator=g) for s in ((M, K), (N, K)))
    s, ws = dev(scales(rng, M, K)), dev(scales(rng, N, K))
    got = torch.full((M, N // 2 if sw else N), float("nan"), dtype=TYPES[out], device=DEV)
    blk.matmul_i8(q, s, w, ws, got, swiglu=sw, clamp=2.0)
    y = ref.product(q, s, w, ws)
    if sw:
        h, gate = ref.swiglu(y, 2.0)
        close_here(got, h, ref.rounded(ref.swiglu_bound(h, gate), h, TYPES[out]))
    else:
        close_here(got, y, ref.rounded(ref.product_bound(y), y, TYPES[out]))


# rows, E, N, K: the shapes that GROUPED_TILES leaves out
@pytest.mark.parametrize("M, E, N, K", [(16001, 16, 258, 2064), (130, 3, 2050, 16400), (16001, 130, 130, 7184), (4001, 16, 8194, 1040)])
@pytest.mark.parametrize("out, sw, gather", [("f32", False, False), ("bf16", True, True)])
def test_grouped_product_of_the_other_tiles(blk, M, E, N, K, out, sw, gather):
    test_grouped_product_of_every_tile(blk, M, E, N, K, out, sw, gather)


def microseconds(call, n=20):
    for _ in range(5):
        call()
    best = []
    for _ in range(5):
        a, z = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(n):
            call()
        z.record()
        z.synchronize()
        best.append(a.elapsed_time(z) * 1000 / n)
    return sorted(best)[2]


@pytest.mark.parametrize("M", [2, 8, 16])
def test_rows_of_one_expert_are_the_dense_product(blk, M):
    """The same bits, and about its time (1 to 1.1 times it): the expert's weights are not read again for every row,
    which takes 8 times as long for 16 of them."""
    say("rows of one expert", M)
    rng = np.random.default_rng(M)
    g = torch.Generator(device=DEV).manual_seed(M)
    K = N = 7168
    w = torch.randint(-128, 128, (1, N, K), dtype=torch.int8, device=DEV, generator=g)
    q, s, ws = dev(codes(rng, (M, K))), dev(scales(rng, M, K)), dev(scales(rng, (1, N), K))
    offsets = dev(np.array([0, M], np.int32))
    dense, grouped = (torch.full((M, N), float("nan"), device=DEV) for _ in range(2))
    t_dense = microseconds(lambda: blk.matmul_i8(q, s, w[0], ws[0], dense))
    t_grouped = microseconds(lambda: blk.matmul_i8(q, s, w, ws, grouped, offsets=offsets))
    say(f"dense {t_dense:.1f} us, grouped {t_grouped:.1f} us")
    assert torch.equal(dense, grouped)
    assert t_grouped <= 2 * t_dense


# T, k, E, N, K: experts with one row each and with several, matrices on both sides of the limit of 4 MiB
@pytest.mark.parametrize("T, k, E, N, K", [(16, 1, 4, 258, 768), (8, 2, 4, 130, 1040), (8, 1, 4, 34, 2064), (2, 1, 1, 66, 528),
                                           (4, 1, 2, 4098, 1040), (16, 1, 5, 130, 1024), (16, 1, 3, 2050, 2064), (16, 1, 9, 2050, 2064)])
@pytest.mark.parametrize("out, sw, gather", [("f32", False, False), ("bf16", True, True)])
def test_grouped_product_of_few_rows_and_experts(blk, T, k, E, N, K, out, sw, gather):
    test_grouped_product(blk, T, k, E, N, K, 0.0, False, out, sw, gather)

"""Plain 64-bit statements of the operators around the expert products, on the CPU
(torch), and the error bounds that their f32 arithmetic allows."""
import numpy as np
import torch

U = 2.0 ** -24  # half a step of f32, relative
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """A rounding next to zero is off by at most half the smallest denormal."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rounded(bound, value, dtype):
    """bound on the f32 result, plus the rounding of a value within it to dtype."""
    h = 0.0 if dtype == torch.float32 else half_step(dtype)
    return bound + h * (value.abs() + bound) + tiny(dtype)


def grouping(ids, E):
    """moe_group's offsets, perm, inv and the number of rows, from ids [T, k] (-1: dropped)."""
    flat = ids.reshape(-1).astype(np.int64)
    ok = (flat >= 0) & (flat < E)
    order = np.argsort(np.where(ok, flat, E), kind="stable")
    kept = int(ok.sum())
    inv = np.full(flat.size, -1, np.int32)
    inv[order[:kept]] = np.arange(kept)
    perm = np.zeros(flat.size, np.int32)
    perm[:kept] = order[:kept]
    counts = np.bincount(flat[ok], minlength=E)
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), perm, inv, kept


def ids_of(rng, T, k, E, dropped=0.0, skew=False):
    """[T, k] distinct experts per token, some pairs dropped."""
    lg = rng.standard_normal((T, E))
    if skew:
        lg = lg - 1.5 * np.log(np.arange(E) + 1.0)
    ids = np.argsort(-lg, axis=1)[:, :k].astype(np.int32)
    ids[rng.random((T, k)) < dropped] = -1
    return ids


def combine(rows, wts, inv, T, k):
    """(value, sum of |terms|) of out[t], in f64; wts None: unit weights."""
    inv = torch.from_numpy(inv.astype(np.int64)).view(T, k)
    out = torch.zeros(T, rows.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for s in range(k):
        t = torch.nonzero(inv[:, s] >= 0).view(-1)
        y = rows[inv[t, s]].double() * (1.0 if wts is None else wts[t, s, None].double())
        out[t] += y
        mag[t] += y.abs()
    return out, mag


def quantize(x):
    """(q int8, scale f32) by the definition, in f64."""
    x = x.double()
    bad = ~torch.isfinite(x).all(1)
    amax = torch.where(bad[:, None], 0.0, x).abs().amax(1)
    scale = (amax / 127.0).float()
    s = scale.double()
    q = torch.where(s[:, None] > 0, torch.round(x / torch.where(s > 0, s, 1.0)[:, None]), 0.0)
    q = torch.where(bad[:, None], 0.0, q).clamp(-127, 127)
    scale[bad] = float("nan")
    return q.to(torch.int8), scale


def product(q, scale, w, ws):
    """q [M, K] . w [N, K]^T with its scales, in f64 (the integer sums are exact there)."""
    return (q.double() @ w.double().t().contiguous()) * scale.double()[:, None] * ws.double()[None, :]


def swiglu(y, L):
    F = y.shape[1] // 2
    g, u = y[:, :F], y[:, F:]
    if L > 1e-6:
        g, u = g.clamp(max=L), u.clamp(-L, L)
    return g * torch.sigmoid(g) * u, g


def product_bound(y):
    """The sum is exact; its rounding to f32 and the two products by scales: 3 half steps."""
    return 3.01 * U * y.abs()


def swiglu_bound(h, g):
    """gate and up off by 3 half steps each, and silu moves by (1 + |g|) of gate's error; the exponential by
    2 half steps of its argument |g| and 2 of its own; sum, quotient and product one each."""
    return U * (12 + 6 * g.abs()) * h.abs()

"""Plain 64-bit statements of the norm, the grouped routing, their gradients and the
low-rank adapters, on the CPU, and the error bounds that f32 arithmetic allows."""
import numpy as np
import torch

from expert_ref import U, rounded

FLOOR = 2.0 ** -14


# ---- norm ------------------------------------------------------------------------------


def total(x, res):
    """The rows that are normalised: x + res in f32, rounded to res's type."""
    return x if res is None else (x.float() + res.float()).to(res.dtype)


def norm(h, w, eps):
    """(y, r) in f64."""
    h = h.double()
    r = 1.0 / torch.sqrt((h * h).sum(1) / h.shape[1] + float(np.float32(eps)))
    return h * r[:, None] * w.double(), r


def codes(y):
    """(q, scale) of rows y in f64."""
    bad = ~torch.isfinite(y).all(1)
    amax = torch.where(bad[:, None], 0.0, y).abs().amax(1)
    scale = (amax / 127.0).float()
    s = scale.double()[:, None]
    q = torch.where(s > 0, torch.round(y / torch.where(s > 0, s, 1.0)), 0.0)
    q = torch.where(bad[:, None], 0.0, q).clamp(-127, 127)
    scale[bad] = float("nan")
    return q.to(torch.int8), scale


def norm_bound(y, dtype):
    """r rounded to f32 and two products: 3 half steps; then the output's rounding."""
    return rounded(3.01 * U * y.abs(), y, dtype)


def chain(T):
    """Additions that a sum over T rows has one after the other, at most: rows are dealt to
    64 sums or more, and those sums added up."""
    return min(T, 96 + T // 64) + 16


def norm_grad(dy, h, w, rstd, dres):
    """(dx, dw, |terms| of each for the bounds) in f64; rstd is an input."""
    dy, h, w, r = dy.double(), h.double(), w.double(), rstd.double()[:, None]
    u, g = h * r, dy * w
    c = (g * u).mean(1, keepdim=True)
    cmag = (g * u).abs().mean(1, keepdim=True)
    dx = r * (g - u * c)
    # g and u are off by half a step each, their products and the sum over H (32 a thread, 10 steps over the
    # threads, and a few) by 64 half steps of the sum of |terms|; then two products, a difference, a product
    err = r.abs() * U * (6 * g.abs() + u.abs() * (64 + 6) * cmag)
    if dres is not None:
        dx = dx + dres.double()
        err = err + U * (dx.abs() + err)
    dw = (dy * u).sum(0)
    return dx, dw, err, (chain(dy.shape[0]) + 3) * U * (dy * u).abs().sum(0)


# ---- routing -----------------------------------------------------------------------------


def scores(l, mode):
    """l [T, E] f64 numpy."""
    with np.errstate(all="ignore"):
        if mode == 0:
            top = l.max(1, keepdims=True)
            e = np.exp(l - np.where(top == -np.inf, 0.0, top))
            p = e / e.sum(1, keepdims=True)
        elif mode == 1:
            p = 1.0 / (1.0 + np.exp(-l))
        else:
            p = np.sqrt(np.logaddexp(0.0, l))
    return np.where(l == -np.inf, 0.0, p)


def _order(key, among):
    """Indexes `among`, largest key first, ties to the lower index, NaN last."""
    return sorted(among, key=lambda e: (np.isnan(key[e]), -key[e] if not np.isnan(key[e]) else 0.0, e))


def route(l, bias, k, mode, n_group, keep, top, norm, scale):
    """(ids, wts, p) by the definition, token by token."""
    l = l.astype(np.float64)
    T, E = l.shape
    p = scores(l, mode)
    c = p if bias is None else p + bias.astype(np.float64)
    key = l if bias is None else c  # without a bias the scores are in the logits' order
    group_key = key if top == 1 else c
    per = E // n_group
    ids, wts = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        there = [e for e in range(E) if l[t, e] != -np.inf]
        if n_group > 1:
            order = []
            for g in range(n_group):
                best = _order(group_key[t], [e for e in there if e // per == g and not np.isnan(group_key[t, e])])[:top]
                order.append((not best, -sum(group_key[t, best]) if best else 0.0, g))
            stay = {g for _, _, g in sorted(order)[:keep]}
            there = [e for e in there if e // per in stay]
        pick = _order(key[t], there)[:k]
        ids[t, :len(pick)], wts[t, :len(pick)] = pick, p[t, pick]
    if norm:
        wts = wts / np.maximum(wts.sum(1, keepdims=True), FLOOR)
    return ids, wts * (scale if scale != 0 else 1.0), p


def score_half_steps(l, mode):
    """How many half steps of f32 a score may be off: the exponential by 2 of its own and by 1 of its argument's
    size for softmax's difference (and so its sum), the sum over E by 24 (16 a lane, 6 over the lanes), the
    logarithm by 4, quotient, root and the rounding by 1 each."""
    l = np.where(np.isfinite(l), l, 0.0)
    if mode == 0:
        return 2 * (4 + (l.max(1, keepdims=True) - l.min(1, keepdims=True))) + 24
    return np.full((l.shape[0], 1), 12.0)


def route_grad(l, ids, dwts, dscores, mode, norm, scale):
    """(dl, bound on its f32 error) by the formulas, in f64 (numpy)."""
    l = l.astype(np.float64)
    T, E = l.shape
    p = scores(l, mode)
    masked = l == -np.inf
    dw = dwts.astype(np.float64) * (scale if scale != 0 else 1.0)
    there = (ids >= 0) & (ids < E)
    at = np.where(there, ids, 0)
    dw, w = np.where(there, dw, 0.0), np.where(there, np.take_along_axis(p, at, 1), 0.0)
    mag = np.abs(dw)
    if norm:
        S = w.sum(1, keepdims=True)
        D = np.maximum(S, FLOOR)
        inner, imag = (dw * w).sum(1, keepdims=True) / D, (np.abs(dw) * w).sum(1, keepdims=True) / D
        dw, mag = (dw - np.where(S >= FLOOR, inner, 0.0)) / D, (mag + np.where(S >= FLOOR, imag, 0.0)) / D
    ds = np.zeros((T, E)) if dscores is None else dscores.astype(np.float64).copy()
    dmag = np.abs(ds)
    for j in range(ids.shape[1]):
        t = np.nonzero(there[:, j])[0]
        np.add.at(ds, (t, ids[t, j]), dw[t, j])
        np.add.at(dmag, (t, ids[t, j]), mag[t, j])
    with np.errstate(all="ignore"):
        if mode == 0:
            dl, dmag = p * (ds - (p * ds).sum(1, keepdims=True)), p * (dmag + (p * dmag).sum(1, keepdims=True))
        else:
            sig = 1.0 / (1.0 + np.exp(-l))
            slope = sig * (1.0 / (1.0 + np.exp(l))) if mode == 1 else np.where(p > 0, sig / (2 * p), 0.0)
            dl, dmag = ds * slope, dmag * slope
    # the scores twice (in dp and in the slope), the sums over the slots (64), and a dozen products
    half = 2 * score_half_steps(l, mode) + ids.shape[1] + 40
    return np.where(masked, 0.0, dl), np.where(masked, 0.0, half * U * dmag) + 1e-37


# ---- adapters ----------------------------------------------------------------------------


def adapters(x, a, b, scale, of, base, out_dtype):
    """(out f64, bound) for the rows that have an adapter; `of`: each row's, -1 for none."""
    out, bound = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64)
    K, R = x.shape[1], a.shape[1]
    # what of mid does not fit two parts of a 16-bit type (16-bit output); three: less than half a step of f32
    part = 0.0 if x.dtype == torch.float32 else (torch.finfo(x.dtype).eps / 2) ** (3 if out_dtype == torch.float32 and
                                                                                    x.dtype == torch.bfloat16 else 2)
    for i in sorted(set(of.tolist()) - {-1}):
        r = torch.nonzero(of == i).view(-1)
        s = 1.0 if scale is None else float(scale[i])
        xr, A, B = x[r].double(), a[i].double(), b[i].double()
        mid, mag = xr @ A.t(), xr.abs() @ A.abs().t()
        delta = s * (mid @ B.t())
        # sums over K: chains of K / 16 steps at most, and 40 over lanes, waves and splits; over R: R + 8, and
        # the product by scale
        err_mid = (K / 16 + 40) * U * mag
        err = abs(s) * ((err_mid @ B.abs().t()) + ((R + 10) * U + part) * ((mid.abs() + err_mid) @ B.abs().t()))
        out[r] += delta
        bound[r] = err + U * (out[r].abs() + err)
    return out, rounded(bound, out, out_dtype)

"""The rows' way into the experts and beside them, as timed cases.

norm           h = x + residual, rounded to the residual's type and kept; y = h * r * w with r = (mean h^2 + eps)^-1/2; or
               y in 8 bits, one scale a row (s = amax / 127 in 32 bits, q = y / s to the nearest whole number)
norm_grad      with g = dy * w: dx = r * (g - h * r^2 * mean(g h)) + dres, dw = sum over the rows of dy * h * r
route          scores s of the logits (softmax, sigmoid or sqrt(softplus)), c = s + bias; a group of experts scores the
               sum of its `top` largest c, the `keep` best groups stay, of their experts the k largest c are picked
               (ties: the lowest index), with weights s, divided by their sum if `norm`, times a factor.  An expert whose
               logit is -inf is masked: it is not picked, and a slot that finds no expert has id -1 and weight 0
route_grad     the logits' gradient from the weights' and the scores'
adapters       out[r] = base[r] + scale[a] * B[a] (A[a] x[r]), a the adapter of row r, for the rows that have one; the
               rows grouped by adapter as the experts' rows are (offsets, perm)
"""
import importlib
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MODES = {"softmax": 0, "sigmoid": 1, "sqrt_softplus": 2}
EPS = 1e-6
FLOOR = 2.0 ** -14  # of the sum that weights are divided by
_blocks = {}  # the framework's context, one for the process


def _block():
    if "mb" not in _blocks:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama-sandbox_amd"))
        _blocks["mb"] = importlib.import_module("moe_block").MoeBlock(0)
    return _blocks["mb"]


def _norm_case(T, H, x, res, w, y, i8=False):
    """Types of x, of the residual stream ("": none), of the gain and of the output; i8: the output in 8 bits."""
    return {"op": "norm", "T": T, "H": H, "x": x, "res": res, "w": w, "y": "" if i8 else y, "i8": i8}


def _norm_grad_case(T, H, dy, h, w, dx, dres=True):
    return {"op": "norm_grad", "T": T, "H": H, "dy": dy, "h": h, "w": w, "dx": dx, "dres": dres}


def _route_case(op, T, E, k, mode, x, bias=True, groups=1, keep=1, top=2, norm=True, factor=1.0, scores=False, masked=0.0):
    """scores: the scores are an output too (and have a gradient); masked: the share of masked experts."""
    return {"op": op, "T": T, "E": E, "k": k, "mode": mode, "x": x, "bias": bias, "groups": groups, "keep": keep, "top": top,
            "norm": norm, "factor": factor, "scores": scores, "masked": masked}


def _adapters_case(M, K, R, N, n, x, out, prompts, without=0.1):
    """prompts: rows of one request stand together; else each row is a request's single token.  without: the share of
    requests that have no adapter."""
    return {"op": "adapters", "M": M, "K": K, "R": R, "N": N, "n": n, "x": x, "out": out, "prompts": prompts, "without": without}


def listed():
    return [
        # one token before the router and the experts: the smallest call
        {"name": "norm_decode", **_norm_case(1, 7168, "bf16", "bf16", "bf16", "bf16")},
        # a long prompt chunk
        {"name": "norm_prefill", **_norm_case(4096, 7168, "bf16", "bf16", "bf16", "bf16")},
        # a ragged chunk on a residual stream in 32 bits, for the 8-bit products
        {"name": "norm_i8_509", **_norm_case(509, 5120, "bf16", "f32", "f32", "", True)},
        # the backward pass of a long chunk
        {"name": "norm_grad_prefill", **_norm_grad_case(4096, 7168, "bf16", "bf16", "bf16", "bf16")},
        # a ragged micro-batch of a small layer, in 32 bits
        {"name": "norm_grad_301", **_norm_grad_case(301, 2048, "f32", "f32", "f32", "f32", False)},
        # one token among 256 experts in 8 groups, with a bias for balance
        {"name": "route_decode", **_route_case("route", 1, 256, 8, "sigmoid", "f32", True, 8, 4, 2, True, 2.5)},
        # a long prompt chunk
        {"name": "route_prefill", **_route_case("route", 4096, 256, 8, "sigmoid", "f32", True, 8, 4, 2, True, 2.5)},
        # a training step's chunk, with a loss on the scores
        {"name": "route_grad_prefill", **_route_case("route_grad", 4096, 256, 8, "softmax", "f32", False, scores=True)},
        # a ragged micro-batch from 16-bit logits
        {"name": "route_grad_301", **_route_case("route_grad", 301, 160, 6, "sigmoid", "bf16", True, factor=2.5)},
        # a batch of single tokens, each request with its adapter
        {"name": "adapters_decode", **_adapters_case(16, 7168, 16, 4096, 24, "bf16", "bf16", False)},
        # prompt chunks of several requests beside a large projection
        {"name": "adapters_prefill", **_adapters_case(4096, 7168, 64, 7168, 8, "bf16", "bf16", True)},
        # ragged prompts of a small layer
        {"name": "adapters_517", **_adapters_case(517, 2048, 8, 768, 32, "f16", "f32", True)},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _drawn(rng):
    """A case, or None where the sizes drawn are too large together."""
    types = ["f32", "bf16", "f16"]
    op = rng.choice(["norm", "norm", "norm_grad", "route", "route", "route_grad", "adapters", "adapters"])
    t = [rng.choice(types) for _ in range(4)]
    T = _log(rng, 1, 8191)
    if op in ("norm", "norm_grad"):
        H = rng.randint(100, 8000) if rng.random() < 0.25 else 8 * _log(rng, 16, 1000)
        if op == "norm":
            return _norm_case(T, H, t[0], rng.choice(["", t[1]]), t[2], t[3], rng.random() < 0.4)
        return _norm_grad_case(T, H, *t, rng.random() < 0.6)
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 4, 8, rng.randint(2, 16)])
        E = groups * _log(rng, max(1, 16 // groups), 1024 // groups)
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(10, E // groups * keep))
        case = _route_case(op, T, E, k, rng.choice(list(MODES)), t[0], rng.random() < 0.6, groups, keep, rng.randint(1, 2),
                           rng.random() < 0.7, rng.choice([1.0, 2.5]), rng.random() < 0.4, rng.choice([0.0, 0.0, 0.2, 0.7]))
        return case if T * E <= 2.1e6 else None
    M, n = _log(rng, 1, 4096), _log(rng, 1, 64)
    K, N = 8 * _log(rng, 12, 896), 8 * _log(rng, 12, 896)
    if rng.random() < 0.15:
        K, N = K + rng.randint(1, 7), N + rng.randint(1, 7)
    R = rng.choice([4, 8, 16, 32, 64, rng.randint(1, 96)])
    if M * R * (K + N) > 3e9 or n * R * (K + N) > 64e6 or M * n * R > 64e6:
        return None
    return _adapters_case(M, K, R, N, n, t[0], t[1], rng.random() < 0.5, rng.choice([0.0, 0.1, 0.6]))


def draw(rng):
    while True:
        case = _drawn(rng)
        if case and work(case)["bytes"] <= 170e6:
            return case


# ---- inputs --------------------------------------------------------------------------


def _gen(seed, i):
    return torch.Generator(device=DEV).manual_seed(1000 * int(seed) + i)


def _floats(shape, kind, seed, i):
    """Normal values with a few larger channels, as hidden states are."""
    g = _gen(seed, i)
    gain = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV))
    return (torch.randn(shape, generator=g, device=DEV) * gain).to(TYPES[kind])


def _gain(H, kind, seed, i):
    return (1.0 + 0.2 * torch.randn(H, generator=_gen(seed, i), device=DEV)).to(TYPES[kind])


def _logits(case, seed):
    """[T, E], some masked; where some are, every 16th token has none left (padding)."""
    T, E = case["T"], case["E"]
    l = torch.randn((T, E), generator=_gen(seed, 0), device=DEV) * 1.5
    if case["masked"]:
        gone = torch.rand((T, E), generator=_gen(seed, 1), device=DEV) < case["masked"]
        gone[5::16] = True
        l = l.masked_fill(gone, float("-inf"))
    return l.to(TYPES[case["x"]])


def _rows_of(case, seed):
    """The adapter of each row, -1 for none, and their stable grouping."""
    rng = np.random.default_rng([int(seed), 11])
    M, n = case["M"], case["n"]
    if case["prompts"]:
        cuts = np.sort(rng.integers(0, M + 1, max(1, min(n, M // 8))))
        request = np.searchsorted(cuts, np.arange(M), side="right")
        of = rng.permutation(max(n, request[-1] + 1))[request] % n
    else:
        request, of = np.arange(M), rng.integers(0, n, M)
    of = np.where(rng.random(request[-1] + 1)[request] < case["without"], -1, of).astype(np.int32)
    order = np.argsort(np.where(of < 0, n, of), kind="stable").astype(np.int32)
    counts = np.bincount(of[of >= 0], minlength=n)
    return of, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), order


def prepare(case, seed):
    op, s = case["op"], {"case": case, "blk": _block() if own else None}
    dev = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(DEV)  # noqa: E731
    empty = lambda shape, kind: torch.zeros(shape, dtype=TYPES[kind], device=DEV)  # noqa: E731
    if op == "norm":
        T, H = case["T"], case["H"]
        s.update(x=_floats((T, H), case["x"], seed, 0), w=_gain(H, case["w"], seed, 1), rstd=empty(T, "f32"))
        if case["res"]:
            s.update(res=_floats((T, H), case["res"], seed, 2), total=empty((T, H), case["res"]))
        if case["i8"]:
            s.update(q=torch.zeros((T, H), dtype=torch.int8, device=DEV), scale=empty(T, "f32"))
        else:
            s["y"] = empty((T, H), case["y"])
    elif op == "norm_grad":
        T, H = case["T"], case["H"]
        s.update(dy=_floats((T, H), case["dy"], seed, 0), w=_gain(H, case["w"], seed, 1), h=_floats((T, H), case["h"], seed, 2),
                 dx=empty((T, H), case["dx"]), dw=empty(H, "f32"))
        s["rstd"] = (s["h"].double().square().mean(1) + EPS).rsqrt().float()
        if case["dres"]:
            s["dres"] = _floats((T, H), case["dx"], seed, 3)
        if own:
            s["part"] = empty(s["blk"].rms_norm_grad_scratch(T, H), "f32")
    elif op in ("route", "route_grad"):
        T, E, k = case["T"], case["E"], case["k"]
        s["logits"] = _logits(case, seed)
        if case["bias"]:
            s["bias"] = 0.05 * torch.randn(E, generator=_gen(seed, 2), device=DEV)
        s.update(ids=torch.zeros((T, k), dtype=torch.int32, device=DEV), wts=empty((T, k), "f32"))
        if case["scores"]:
            s["scores"] = empty((T, E), "f32")
        if op == "route_grad":
            s["ids"].copy_(_plain_route(s)["ids"])
            s["dwts"] = torch.randn((T, k), generator=_gen(seed, 3), device=DEV)
            s["dlogits"] = empty((T, E), case["x"])
            if case["scores"]:
                s["dscores"] = torch.randn((T, E), generator=_gen(seed, 4), device=DEV) / E
    else:
        M, K, R, N, n = (case[v] for v in ("M", "K", "R", "N", "n"))
        of, offsets, perm = _rows_of(case, seed)
        s.update(of=dev(of.astype(np.int64)), offsets=dev(offsets), perm=dev(perm), x=_floats((M, K), case["x"], seed, 0))
        s["a"] = (torch.randn((n, R, K), generator=_gen(seed, 1), device=DEV) / K ** 0.5).to(TYPES[case["x"]])
        s["b"] = (torch.randn((n, N, R), generator=_gen(seed, 2), device=DEV) / R ** 0.5).to(TYPES[case["x"]])
        s["scale"] = 0.25 + torch.rand(n, generator=_gen(seed, 3), device=DEV)
        s["base"] = _floats((M, N), case["out"], seed, 4)
        s["out"] = s["base"].clone()  # rows without an adapter stay as they are
        if own:
            s["mid"] = empty(s["blk"].adapters_scratch(M, K, R), "f32")
    return s


# ---- one pass ------------------------------------------------------------------------


def _plain_norm(s):
    case, h = s["case"], s["x"]
    got = {}
    if case["res"]:
        h = got["total"] = (s["x"].float() + s["res"].float()).to(TYPES[case["res"]])
    rstd = torch.rsqrt(h.double().square().mean(1, keepdim=True) + EPS)  # a long sum: in 64 bits
    got["rstd"] = rstd[:, 0].float()
    if not case["i8"]:
        got["y"] = (h.float() * rstd.float() * s["w"].float()).to(TYPES[case["y"]])
        return got
    y = h.double() * s["w"].double() * rstd  # in 64 bits, for the quotients next to a tie
    scale = (y.abs().amax(1, keepdim=True) / 127.0).float()
    q = torch.round(y / torch.where(scale > 0, scale, 1.0).double()).clamp(-127, 127)
    got["y"] = q.float() * scale
    return got


def _plain_norm_grad(s):
    case, dy, h, r = s["case"], s["dy"].float(), s["h"].float(), s["rstd"][:, None]
    g = dy * s["w"].float()
    dx = r * (g - h * ((g * h).mean(1, keepdim=True) * r * r))
    if case["dres"]:
        dx = dx + s["dres"].float()
    return {"dx": dx.to(TYPES[case["dx"]]), "dw": (dy * (h * r)).sum(0)}


def _plain_scores(l, mode):
    if mode == "softmax":
        top = l.amax(1, keepdim=True)
        e = torch.exp(l - torch.where(top == float("-inf"), 0.0, top))
        return e / e.sum(1, keepdim=True).clamp(min=1e-300)
    return 1 / (1 + torch.exp(-l)) if mode == "sigmoid" else torch.sqrt(torch.log1p(torch.exp(l)))


def _plain_route(s):
    """In 64 bits: which experts are picked hangs on the order of scores that are close to each other."""
    case = s["case"]
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    l = s["logits"].double()
    none = float("-inf")
    masked = l == none
    p = _plain_scores(l, case["mode"])
    c = torch.where(masked, none, p + s["bias"] if case["bias"] else p)
    if not case["bias"] and (G == 1 or case["top"] == 1):
        c = l  # the scores are in the logits' order
    if G > 1:
        best = torch.sort(c.view(T, G, E // G), dim=2, descending=True)[0][:, :, :case["top"]]
        score = torch.where(best[:, :, 0] == none, none, torch.where(best == none, 0.0, best).sum(2))
        kept = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :case["keep"]]
        stay = torch.zeros((T, G), dtype=torch.bool, device=DEV).scatter_(1, kept, True)
        c = torch.where(stay.repeat_interleave(E // G, 1), c, none)
    c, ids = torch.sort(c, dim=1, descending=True, stable=True)
    there, ids = c[:, :k] != none, ids[:, :k]
    w = torch.where(there, torch.gather(p, 1, ids), 0.0)
    if case["norm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=FLOOR)
    got = {"ids": torch.where(there, ids, -1).int(), "wts": (w * case["factor"]).float()}
    if case["scores"]:
        got["scores"] = p.float()
    return got


def _plain_route_grad(s):
    case, ids, l = s["case"], s["ids"].long(), s["logits"].float()
    there, at = ids >= 0, ids.clamp(min=0)
    masked = l == float("-inf")
    p = _plain_scores(l.double(), case["mode"]).float() if case["mode"] == "softmax" else _plain_scores(l, case["mode"])
    dw = s["dwts"] * case["factor"]
    if case["norm"]:
        w = torch.where(there, torch.gather(p, 1, at), 0.0)
        total = w.sum(1, keepdim=True)
        d = total.clamp(min=FLOOR)
        dw = (dw - torch.where(total >= FLOOR, (dw * w).sum(1, keepdim=True) / d, 0.0)) / d
    dp = s["dscores"] if case["scores"] else torch.zeros_like(l)
    dp = dp.scatter_add(1, at, torch.where(there, dw, 0.0))
    if case["mode"] == "softmax":
        dl = p * (dp - (p * dp).sum(1, keepdim=True))
    elif case["mode"] == "sigmoid":
        dl = dp * p / (1 + torch.exp(l))
    else:
        dl = dp * torch.where(p > 0, 0.5 / ((1 + torch.exp(-l)) * p.clamp(min=1e-30)), 0.0)
    return {"dlogits": torch.where(masked, 0.0, dl).to(TYPES[case["x"]])}


def _plain_adapters(s):
    """The rows by every adapter's A, those of other adapters taken out, by every B."""
    case, of, M = s["case"], s["of"], s["case"]["M"]
    n, R, N = case["n"], case["R"], case["N"]
    mid = (s["x"].float() @ s["a"].float().view(n * R, -1).T).view(M, n, R)
    mine = torch.arange(n, device=DEV) == of[:, None]
    mid = torch.where(mine[:, :, None], mid * s["scale"][:, None], 0.0).view(M, n * R)
    delta = mid @ s["b"].float().transpose(1, 2).reshape(n * R, N)
    out = torch.where(of[:, None] >= 0, (s["base"].float() + delta).to(TYPES[case["out"]]), s["base"])
    return {"out": out}


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "route": _plain_route, "route_grad": _plain_route_grad,
                "adapters": _plain_adapters}[op](s)
    blk = s["blk"]
    if op == "norm":
        blk.rms_norm(s["x"], s["w"], EPS, residual=s.get("res"), total=s.get("total"), y=s.get("y"), q=s.get("q"),
                     scale=s.get("scale"), rstd=s["rstd"])
        got = {"y": torch.mul(s["q"], s["scale"][:, None]) if case["i8"] else s["y"], "rstd": s["rstd"]}
        return {**got, "total": s["total"]} if case["res"] else got
    if op == "norm_grad":
        blk.rms_norm_grad(s["dy"], s["h"], s["w"], s["rstd"], s["dx"], s["dw"], s["part"], dres=s.get("dres"))
        return {"dx": s["dx"], "dw": s["dw"]}
    if op == "route":
        blk.route_groups(s["logits"], case["k"], MODES[case["mode"]], case["norm"], case["factor"], s["ids"], s["wts"],
                         bias=s.get("bias"), n_group=case["groups"], keep=case["keep"], top=case["top"], scores=s.get("scores"))
        got = {"ids": s["ids"], "wts": s["wts"]}
        return {**got, "scores": s["scores"]} if case["scores"] else got
    if op == "route_grad":
        blk.route_grad(s["logits"], s["ids"], s["dwts"], MODES[case["mode"]], case["norm"], case["factor"], s["dlogits"],
                       dscores=s.get("dscores"))
        return {"dlogits": s["dlogits"]}
    blk.adapters(s["x"], s["a"], s["b"], s["scale"], s["offsets"], s["perm"], s["base"], s["out"], s["mid"])
    return {"out": s["out"]}


def work(case):
    """Each input read once and each output written once; adapters that have rows, a multiply and an add for each of
    their products.  Output in 8 bits is returned as the values it stands for, in 32."""
    size = lambda t: {"": 0, "f32": 4}.get(t, 2)  # noqa: E731
    op = case["op"]
    if op == "norm":
        T, H = case["T"], case["H"]
        row = size(case["x"]) + 2 * size(case["res"]) + (1 + 1 + 4 if case["i8"] else size(case["y"]))
        return {"bytes": T * H * row + H * size(case["w"]) + 4 * T * (2 if case["i8"] else 1), "flops": 5 * T * H}
    if op == "norm_grad":
        T, H = case["T"], case["H"]
        row = size(case["dy"]) + size(case["h"]) + size(case["dx"]) * (2 if case["dres"] else 1)
        return {"bytes": T * H * row + H * (size(case["w"]) + 4) + 4 * T, "flops": 9 * T * H}
    if op in ("route", "route_grad"):
        T, E, k, x = case["T"], case["E"], case["k"], size(case["x"])
        per = (x + 4 * case["scores"]) if op == "route" else 2 * x + 4 * case["scores"]
        return {"bytes": T * E * per + 8 * T * k + 4 * E * case["bias"], "flops": 10 * T * E}
    M, K, R, N = (case[v] for v in ("M", "K", "R", "N"))
    of = _rows_of(case, 1)[0]
    rows, touched, x, o = int((of >= 0).sum()), len(np.unique(of[of >= 0])), size(case["x"]), size(case["out"])
    return {"bytes": max(1, rows * (K * x + 2 * N * o) + touched * R * (K + N) * x + 4 * M), "flops": 2 * rows * R * (K + N)}


# ---- the definitions in 64 bits -------------------------------------------------------


def _exact_scores(l, mode):
    if mode == "sigmoid":
        return torch.sigmoid(l)
    if mode == "softmax":
        return torch.nan_to_num(torch.softmax(l, 1), nan=0.0)  # a row of masked experts alone
    return torch.sqrt(torch.logaddexp(l, torch.zeros_like(l)))


def _exact_route(case, seed):
    """Expert by expert, on the host."""
    l = _logits(case, seed).double()
    p = _exact_scores(l, case["mode"])
    bias = 0.05 * torch.randn(case["E"], generator=_gen(seed, 2), device=DEV) if case["bias"] else None
    c = p if bias is None else p + bias.double()
    L, P, C = l.cpu().numpy(), p.cpu().numpy(), c.cpu().numpy()
    T, E, k, G = case["T"], case["E"], case["k"], case["groups"]
    by_logit = bias is None and (G == 1 or case["top"] == 1)
    ids, wts = np.full((T, k), -1, np.int64), np.zeros((T, k))
    for t in range(T):
        key = L[t] if by_logit else C[t]
        open_ = L[t] > -np.inf
        if G > 1:
            score = []
            for g in range(G):
                e = np.arange(g * (E // G), (g + 1) * (E // G))
                best = np.sort(key[e[open_[e]]])[::-1][:case["top"]]
                score.append(best.sum() if best.size else -np.inf)
            keep = np.argsort(-np.array(score), kind="stable")[:case["keep"]]
            open_ = open_ & np.isin(np.arange(E) // (E // G), keep)
        e = np.nonzero(open_)[0]
        e = e[np.argsort(-key[e], kind="stable")][:k]
        ids[t, :e.size], wts[t, :e.size] = e, P[t, e]
    if case["norm"]:
        wts /= np.maximum(wts.sum(1, keepdims=True), FLOOR)
    return ids, torch.from_numpy(wts * case["factor"]).to(DEV), p, l


def exact(case, seed):
    op = case["op"]
    if op == "norm":
        T, H = case["T"], case["H"]
        h, w = _floats((T, H), case["x"], seed, 0), _gain(H, case["w"], seed, 1).double()
        got = {}
        if case["res"]:
            h = h.float() + _floats((T, H), case["res"], seed, 2).float()
            got["total"] = h = h.to(TYPES[case["res"]]).double()  # the sum is the one rounded value that the norm is of
        h = h.double()
        var = torch.linalg.vector_norm(h, dim=1).square() / H + EPS
        got["rstd"] = 1 / torch.sqrt(var)
        y = h / torch.sqrt(var)[:, None] * w
        if case["i8"]:
            s = (torch.linalg.vector_norm(y, ord=float("inf"), dim=1) / 127).float().double()
            y = torch.round(y / s[:, None]) * s[:, None]
        return {**got, "y": y}
    if op == "norm_grad":
        T, H = case["T"], case["H"]
        h = _floats((T, H), case["h"], seed, 2)
        r = (h.double().square().mean(1) + EPS).rsqrt().float().double()  # an input, in 32 bits
        dy, w, h = _floats((T, H), case["dy"], seed, 0).double(), _gain(H, case["w"], seed, 1).double(), h.double()
        u = h * r[:, None]  # the normalised rows
        g = dy * w
        dx = (g - u * ((g * u).sum(1) / H)[:, None]) * r[:, None]
        dw = (dy * u).sum(0)
        if case["dres"]:
            dx += _floats((T, H), case["dx"], seed, 3).double()
        return {"dx": dx, "dw": dw}
    if op == "route":
        ids, wts, p, _ = _exact_route(case, seed)
        got = {"ids": torch.from_numpy(ids.astype(np.int32)).to(DEV), "wts": wts}
        return {**got, "scores": p} if case["scores"] else got
    if op == "route_grad":
        ids, wts, p, l = _exact_route(case, seed)
        T, E, k = case["T"], case["E"], case["k"]
        dwts = torch.randn((T, k), generator=_gen(seed, 3), device=DEV).double()
        ids = torch.from_numpy(ids).to(DEV)
        masked = l == float("-inf")
        # with respect to a copy of the logits whose masked ones are far down, where every score's slope is 0
        z = torch.where(masked, -700.0, l).requires_grad_()
        s = torch.where(masked, 0.0, _exact_scores(z, case["mode"]))
        w = torch.where(ids >= 0, torch.gather(s, 1, ids.clamp(min=0)), 0.0)
        if case["norm"]:
            w = w / torch.maximum(w.sum(1, keepdim=True), torch.full_like(w[:, :1], FLOOR))
        loss = (w * case["factor"] * dwts).sum()
        if case["scores"]:
            loss = loss + (s * (torch.randn((T, E), generator=_gen(seed, 4), device=DEV) / E).double()).sum()
        return {"dlogits": torch.where(masked, 0.0, torch.autograd.grad(loss, z)[0])}
    M, K, R, N, n = (case[v] for v in ("M", "K", "R", "N", "n"))
    of, offsets, perm = _rows_of(case, seed)
    t = TYPES[case["x"]]
    x = _floats((M, K), case["x"], seed, 0)
    a = (torch.randn((n, R, K), generator=_gen(seed, 1), device=DEV) / K ** 0.5).to(t)
    b = (torch.randn((n, N, R), generator=_gen(seed, 2), device=DEV) / R ** 0.5).to(t)
    scale = 0.25 + torch.rand(n, generator=_gen(seed, 3), device=DEV)
    out = _floats((M, N), case["out"], seed, 4).double()
    for i in np.unique(of[of >= 0]).tolist():
        rows = torch.from_numpy(np.nonzero(of == i)[0]).to(DEV)
        mid = x[rows].double() @ a[i].double().t().contiguous()
        out[rows] += scale[i].double() * (mid @ b[i].double().t().contiguous())
    return {"out": out}

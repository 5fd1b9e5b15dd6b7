"""Operators around the expert products, as timed cases.

dispatch       rows[inv[t, s]] = x[t]: the tokens' rows in expert order; its gradient dx[t] = sum_s drows[inv[t, s]]
combine        out[t] = sum_s wts[t, s] * rows[inv[t, s]]: back in token order; its gradient drows[inv[t, s]] =
               wts[t, s] * dout[t] and dwts[t, s] = <dout[t], rows[inv[t, s]]>
linear,        float rows quantised to 8 bits, one scale a row (s = amax / 127 in 32 bits, q = x / s to the nearest
experts        whole number, ties to even), times 8-bit weights with one scale a channel: y[r, n] = s[r] * ws[n] *
               sum_k q[r, k] * w[n, k].  experts: the rows stand in expert order and each expert has its weights;
               swiglu: the channels are F of gate, then F of up, and silu(gate) * up is written

inv, perm and offsets are the token-to-expert grouping that moe_group makes: pairs (token, slot) stably sorted by
expert.  Pairs without an expert here (id -1: another rank holds it) have no row.
"""
import importlib
import os
import sys

import numpy as np
import torch

own = False
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_blocks = {}  # the framework's context, one for the process


def _block():
    if "mb" not in _blocks:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama-sandbox_amd"))
        _blocks["mb"] = importlib.import_module("moe_block").MoeBlock(0)
    return _blocks["mb"]


def _rows_case(op, T, k, H, a, b, dropped=0.0, E=256):
    """a: the type of what is read, b: of what is written."""
    return {"op": op, "T": T, "k": k, "H": H, "E": E, "a": a, "b": b, "dropped": dropped}


def _linear_case(M, K, N, a, b, swiglu=False, clamp=0.0):
    return {"op": "linear", "T": M, "K": K, "N": N, "a": a, "b": b, "swiglu": swiglu, "clamp": clamp}


def _experts_case(op, T, k, E, K, N, a, b, zipf=False, dropped=0.0, clamp=0.0):
    """op experts_up: x [T, K] through the grouping, N = 2F channels, SwiGLU; experts_down: rows [T * k, K] in
    expert order."""
    return {"op": op, "T": T, "k": k, "E": E, "K": K, "N": N, "a": a, "b": b, "zipf": zipf, "dropped": dropped,
            "swiglu": op == "experts_up", "clamp": clamp}


def listed():
    return [
        # the smallest call: one token to its eight experts
        {"name": "dispatch_decode", **_rows_case("dispatch", 1, 8, 7168, "bf16", "bf16")},
        # a long prompt chunk to its experts
        {"name": "dispatch_prefill", **_rows_case("dispatch", 4096, 8, 7168, "bf16", "bf16")},
        # a training step's rows back to the tokens, a quarter of the pairs on other ranks
        {"name": "dispatch_grad_509", **_rows_case("dispatch_grad", 509, 6, 5120, "f32", "f32", 0.25, 160)},
        # a small batch's expert rows back in token order
        {"name": "combine_37", **_rows_case("combine", 37, 6, 5120, "f16", "f32", 0.0, 160)},
        # a prompt chunk's expert rows, as this block's kernels hold them
        {"name": "combine_prefill", **_rows_case("combine", 2048, 8, 7168, "f32", "f32")},
        # the backward pass of a long chunk's combine
        {"name": "combine_grad_prefill", **_rows_case("combine_grad", 4096, 8, 7168, "bf16", "bf16")},
        # a ragged micro-batch of a small layer, with pairs on other ranks
        {"name": "combine_grad_301", **_rows_case("combine_grad", 301, 4, 2048, "f32", "f32", 0.25, 32)},
        # one token through a shared expert's gate and up
        {"name": "linear_decode", **_linear_case(1, 7168, 4096, "bf16", "bf16", True)},
        # a prompt chunk through a dense layer: the largest product
        {"name": "linear_prefill", **_linear_case(4096, 7168, 7168, "bf16", "bf16")},
        # a few concurrent sequences through the routed experts' gate and up
        {"name": "experts_decode", **_experts_case("experts_up", 16, 8, 256, 7168, 4096, "bf16", "bf16", True)},
        # a prompt chunk through them
        {"name": "experts_prefill", **_experts_case("experts_up", 512, 8, 256, 7168, 4096, "f32", "bf16", False)},
        # a long odd chunk through a small layer's down product
        {"name": "experts_down_8191", **_experts_case("experts_down", 8191, 4, 32, 768, 2048, "bf16", "f32", True)},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    types = ["f32", "bf16", "f16"]
    op = rng.choice(["dispatch", "dispatch_grad", "combine", "combine_grad", "linear", "linear", "experts_up",
                     "experts_down"])
    a, b = rng.choice(types), rng.choice(types)
    dropped = rng.choice([0.0, 0.0, 0.25, 0.6])
    while True:
        k, E = rng.randint(1, 8), _log(rng, 8, 256)
        if op in ("dispatch", "dispatch_grad", "combine", "combine_grad"):
            T, H = _log(rng, 1, 8191), rng.randint(100, 8000) if rng.random() < 0.25 else 8 * rng.randint(16, 1000)
            if T * k * H <= 110e6:
                dropped = dropped if T * k >= 16 else 0.0
                return _rows_case(op, T, k, H, a, a if op == "combine_grad" else b, dropped, E)
        K = rng.randint(100, 2000) if rng.random() < 0.15 else 16 * _log(rng, 8, 448)
        N = _log(rng, 64, 7168) if rng.random() < 0.5 else 64 * _log(rng, 1, 112)
        T = _log(rng, 1, 4096)
        if op == "linear":
            if T * K * N <= 2e11:
                N += N % 2
                return _linear_case(T, K, N, a, b, rng.random() < 0.3, rng.choice([0.0, 2.0, 10.0]))
        elif E * N * K <= 7e9 and T * k * N * K <= 1.1e11 and E * T * (K + N) <= 2e9:
            N += N % 2
            dropped = dropped if T * k >= 16 else 0.0
            return _experts_case(op, T, k, E, K, N, a, b, rng.random() < 0.5, dropped, rng.choice([0.0, 2.0, 10.0]))


# ---- inputs --------------------------------------------------------------------------


def _ids(case, seed):
    """[T, k] experts of the tokens, distinct in a token; -1 where the pair is dropped."""
    rng = np.random.default_rng([int(seed), 7])
    lg = rng.standard_normal((case["T"], case["E"]), dtype=np.float32)
    if case.get("zipf"):
        p = (np.arange(case["E"]) + 1.0) ** -1.1
        lg = lg + np.log(p / p.sum())[rng.permutation(case["E"])].astype(np.float32)
    ids = np.argsort(-lg, axis=1, kind="stable")[:, :case["k"]].astype(np.int32)
    ids[rng.random(ids.shape) < case["dropped"]] = -1
    return ids


def _grouping(ids, E):
    """counts [E], offsets [E + 1], perm (grouped row -> pair), inv (pair -> grouped row, -1: none)."""
    flat = ids.reshape(-1).astype(np.int64)
    order = np.argsort(np.where(flat < 0, E, flat), kind="stable")
    kept = int((flat >= 0).sum())
    counts = np.bincount(flat[flat >= 0], minlength=E)
    perm = np.zeros(flat.size, np.int32)
    perm[:kept] = order[:kept]
    inv = np.full(flat.size, -1, np.int32)
    inv[order[:kept]] = np.arange(kept, dtype=np.int32)
    return counts, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), perm, inv, kept


def _gen(seed, i):
    return torch.Generator(device=DEV).manual_seed(1000 * int(seed) + i)


def _floats(shape, kind, seed, i):
    """Normal values with a few larger channels, as hidden states are."""
    g = _gen(seed, i)
    gain = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV))
    return (torch.randn(shape, generator=g, device=DEV) * gain).to(TYPES[kind])


def _weights(shape, seed, i):
    """8-bit codes of normal weights, and a scale for each channel that gives sums of about 1."""
    g, n = _gen(seed, i), shape[-1]
    w = torch.empty(shape, dtype=torch.int8, device=DEV)
    for m in (w if len(shape) == 3 else w[None]):
        m.copy_(torch.randn(m.shape, generator=g, device=DEV).mul_(36.0).round_().clamp_(-127, 127))
    scale = (0.5 + torch.rand(shape[:-1], generator=g, device=DEV)) / (36.0 * n ** 0.5)
    return w, scale


def prepare(case, seed):
    op, T, s = case["op"], case["T"], {"case": case, "blk": _block() if own else None}
    dev = lambda v: torch.from_numpy(np.ascontiguousarray(v)).to(DEV)  # noqa: E731
    if op != "linear":
        ids = _ids(case, seed)
        counts, offsets, perm, inv, kept = _grouping(ids, case["E"])
        P = ids.size
        s.update(offsets=dev(offsets), perm=dev(perm), inv=dev(inv), cap=max(1, int(counts.max())),
                 kept=dev(np.arange(P) < kept))
    if op in ("dispatch", "dispatch_grad", "combine", "combine_grad"):
        H = case["H"]
        n_in, n_out = {"dispatch": (T, P), "dispatch_grad": (P, T), "combine": (P, T), "combine_grad": (P, P)}[op]
        s["in"] = _floats((n_in, H), case["a"], seed, 0)
        s["out"] = torch.zeros((n_out, H), dtype=TYPES[case["b"]], device=DEV)
        if op in ("combine", "combine_grad"):
            w = torch.rand((T, case["k"]), generator=_gen(seed, 1), device=DEV) + 0.05
            s["wts"] = w / w.sum(1, keepdim=True)
        if op == "combine_grad":
            s["dout"] = _floats((T, H), case["a"], seed, 2)
            s["dwts"] = torch.zeros((T, case["k"]), device=DEV)
        return s
    K, N = case["K"], case["N"]
    M = T if op != "experts_down" else T * case["k"]
    s["in"] = _floats((M, K), case["a"], seed, 0)
    s["q"] = torch.zeros((M, K), dtype=torch.int8, device=DEV)
    s["scale"] = torch.zeros(M, device=DEV)
    s["w"], s["ws"] = _weights((N, K) if op == "linear" else (case["E"], N, K), seed, 1)
    rows = T if op == "linear" else T * case["k"]
    s["out"] = torch.zeros((rows, N // 2 if case["swiglu"] else N), dtype=TYPES[case["b"]], device=DEV)
    return s


# ---- one pass ------------------------------------------------------------------------


def _plain_rows(s, op):
    case = s["case"]
    T, k, H, b = case["T"], case["k"], case["H"], TYPES[case["b"]]
    inv = s["inv"].long()
    there, at = (inv >= 0)[:, None], inv.clamp(min=0)
    if op == "dispatch":
        return {"rows": torch.where(s["kept"][:, None], s["in"][(s["perm"] // k).long()].to(b), 0)}
    if op == "combine_grad":
        token = (s["perm"] // k).long()
        w = s["wts"].reshape(-1)[s["perm"].long()]
        drows = torch.where(s["kept"][:, None], s["dout"][token].float() * w[:, None], 0.0)
        y = torch.where(there, s["in"][at].float(), 0.0).view(T, k, H)
        return {"drows": drows.to(b), "dwts": (y * s["dout"].float()[:, None]).sum(2)}
    y = torch.where(there, s["in"][at].float(), 0.0).view(T, k, H)
    if op == "combine":
        y = y * s["wts"][:, :, None]
    return {"dx" if op == "dispatch_grad" else "out": y.sum(1).to(b)}


def _swiglu(y, L):
    g, u = y.chunk(2, dim=-1)
    if L > 0:
        g, u = torch.clamp(g, max=L), torch.clamp(u, -L, L)
    return g / (1 + torch.exp(-g)) * u


def _codes(x):
    """x [M, K] -> whole numbers and scale [M, 1], both in 32 bits; the quotients in 64, for those next to a tie."""
    scale = x.float().abs().amax(1, keepdim=True) / torch.full((1, 1), 127.0, device=x.device)
    q = torch.round(x.double() / torch.where(scale > 0, scale, 1.0).double())
    return q.clamp(-127, 127).float(), scale


def _plain_product(s):
    case, b = s["case"], TYPES[s["case"]["b"]]
    q, scale = _codes(s["in"])
    if case["op"] == "linear":
        y = q @ s["w"].float().T * scale * s["ws"]
        return {"out": (_swiglu(y, case["clamp"]) if case["swiglu"] else y).to(b)}
    E, cap, P = case["E"], s["cap"], case["T"] * case["k"]
    offsets = s["offsets"].long()
    at = (offsets[:-1, None] + torch.arange(cap, device=DEV)).clamp(max=P - 1)  # [E, cap] rows, those past an expert's idle
    src = s["perm"].long()[at] // case["k"] if case["op"] == "experts_up" else at
    y = torch.bmm(q[src.view(-1)].view(E, cap, -1), s["w"].float().transpose(1, 2))
    y = y * scale[src.view(-1)].view(E, cap, 1) * s["ws"][:, None, :]
    y = _swiglu(y, case["clamp"]) if case["swiglu"] else y
    row = torch.arange(P, device=DEV)
    e = (torch.searchsorted(offsets, row, right=True) - 1).clamp(max=E - 1)
    y = y[e, (row - offsets[e]).clamp(max=cap - 1)]
    return {"out": torch.where(s["kept"][:, None], y, 0.0).to(b)}


def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        return _plain_rows(s, op) if "H" in case else _plain_product(s)
    blk = s["blk"]
    if op == "dispatch":
        blk.dispatch(s["in"], s["inv"], s["out"])
        return {"rows": s["out"]}
    if op == "dispatch_grad":
        blk.dispatch_grad(s["in"], s["inv"], s["out"])
        return {"dx": s["out"]}
    if op == "combine":
        blk.combine(s["in"], s["wts"], s["inv"], s["out"])
        return {"out": s["out"]}
    if op == "combine_grad":
        blk.combine_grad(s["dout"], s["in"], s["wts"], s["inv"], s["out"], s["dwts"])
        return {"drows": s["out"], "dwts": s["dwts"]}
    blk.quantize_i8(s["in"], s["q"], s["scale"])
    if op == "linear":
        blk.matmul_i8(s["q"], s["scale"], s["w"], s["ws"], s["out"], swiglu=case["swiglu"], clamp=case["clamp"])
    elif op == "experts_up":
        blk.matmul_i8(s["q"], s["scale"], s["w"], s["ws"], s["out"], offsets=s["offsets"], perm=s["perm"],
                      k=case["k"], swiglu=True, clamp=case["clamp"])
    else:
        blk.matmul_i8(s["q"], s["scale"], s["w"], s["ws"], s["out"], offsets=s["offsets"])
    return {"out": s["out"]}


def work(case):
    """Each input read once and each output written once; weights of the experts that have rows, a multiply and an
    add for each of their products."""
    a, b = (4 if case[t] == "f32" else 2 for t in ("a", "b"))
    T, op = case["T"], case["op"]
    if op == "linear":
        P = kept = T
        touched = 1
    else:
        ids = _ids(case, 1)
        P, kept, touched = ids.size, int((ids >= 0).sum()), len(np.unique(ids[ids >= 0]))
    if "H" in case:
        H, n = case["H"], 4 * P
        if op == "dispatch":
            return {"bytes": n + T * H * a + kept * H * b, "flops": 0}
        if op == "combine_grad":
            return {"bytes": 3 * n + T * H * a + kept * H * (a + b), "flops": 3 * kept * H}
        return {"bytes": n * (2 if op == "combine" else 1) + kept * H * a + T * H * b, "flops": 2 * kept * H}
    K, N = case["K"], case["N"]
    rows_in = kept if op == "experts_down" else T
    n_out = N // 2 if case["swiglu"] else N
    return {"bytes": rows_in * K * a + touched * N * (K + 4) + kept * n_out * b + (0 if op == "linear" else 4 * P),
            "flops": 2 * kept * K * N}


# ---- the definitions in 64 bits -------------------------------------------------------


def _product64(case, x, w, ws):
    """The quantised product of x [M, K] with one weight matrix, in 64 bits.  A row's scale is a 32-bit number."""
    x = x.double()
    s = (x.abs().amax(1) / 127.0).float().double()
    q = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[:, None]).clamp(-127, 127)
    y = torch.matmul(q, w.double().t().contiguous()) * s[:, None] * ws.double()[None, :]
    if not case["swiglu"]:
        return y
    F, L = case["N"] // 2, case["clamp"]
    g, u = y[:, :F], y[:, F:]
    if L > 0:
        g, u = torch.minimum(g, torch.full_like(g, L)), torch.minimum(torch.maximum(u, torch.full_like(u, -L)), torch.full_like(u, L))
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    op, T = case["op"], case["T"]
    if op == "linear":
        w, ws = _weights((case["N"], case["K"]), seed, 1)
        return {"out": _product64(case, _floats((T, case["K"]), case["a"], seed, 0), w, ws)}
    ids, k = _ids(case, seed), case["k"]
    counts, offsets, perm, inv, kept = _grouping(ids, case["E"])
    P = ids.size
    if "H" not in case:
        up = op == "experts_up"
        x = _floats((T if up else P, case["K"]), case["a"], seed, 0)
        w, ws = _weights((case["E"], case["N"], case["K"]), seed, 1)
        out = torch.zeros((P, case["N"] // 2 if up else case["N"]), dtype=torch.float64, device=DEV)
        for e in np.nonzero(counts)[0].tolist():
            lo, hi = int(offsets[e]), int(offsets[e + 1])
            rows = torch.from_numpy(perm[lo:hi].astype(np.int64) // k).to(DEV) if up else slice(lo, hi)
            out[lo:hi] = _product64(case, x[rows], w[e], ws[e])
        return {"out": out}
    H = case["H"]
    at = torch.from_numpy(inv.astype(np.int64)).to(DEV).view(T, k)
    x = _floats((T if op == "dispatch" else P, H), case["a"], seed, 0)
    if op == "dispatch":
        rows = torch.zeros((P, H), dtype=torch.float64, device=DEV)
        for s in range(k):
            t = torch.nonzero(at[:, s] >= 0).view(-1)
            rows[at[t, s]] = x[t].double()
        return {"rows": rows}
    out = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    wts = None
    if op != "dispatch_grad":
        wts = torch.rand((T, k), generator=_gen(seed, 1), device=DEV) + 0.05
        wts = (wts / wts.sum(1, keepdim=True)).double()
    if op == "combine_grad":
        dout = _floats((T, H), case["a"], seed, 2).double()
        drows, dwts = torch.zeros((P, H), dtype=torch.float64, device=DEV), torch.zeros_like(wts)
        for s in range(k):
            t = torch.nonzero(at[:, s] >= 0).view(-1)
            drows[at[t, s]] = dout[t] * wts[t, s, None]
            dwts[t, s] = (dout[t] * x[at[t, s]].double()).sum(1)
        return {"drows": drows, "dwts": dwts}
    for s in range(k):
        t = torch.nonzero(at[:, s] >= 0).view(-1)
        y = x[at[t, s]].double()
        out[t] += y if wts is None else y * wts[t, s, None]
    return {"dx" if op == "dispatch_grad" else "out": out}

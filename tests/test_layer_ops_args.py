"""The bindings of the norm, the grouped routing, their gradients and the adapters refuse
tensors that would make the kernels read or write out of bounds, before the C-ABI;
and the C-ABI refuses what it can see.  CPU only, on host tensors."""
import ctypes

import pytest
import torch

import moe_block as mb
from test_expert_ops_args import block, f, i32, i8, torch_calls

T, H, E, K_, R, N, n = 3, 64, 16, 2, 4, 24, 5
GOOD = {
    "rms_norm": dict(x=f(T, H), w=f(H), eps=1e-6, residual=f(T, H), total=f(T, H), y=f(T, H), q=i8(T, H), scale=f(T), rstd=f(T)),
    "rms_norm_grad": dict(dy=f(T, H), h=f(T, H), w=f(H), rstd=f(T), dx=f(T, H), dw=f(H), part=f(9), dres=f(T, H)),
    "route_groups": dict(logits=f(T, E), k=K_, mode=1, norm=True, scale=1.0, ids=i32(T, K_), wts=f(T, K_), bias=f(E), n_group=4,
                         keep=2, top=2, scores=f(T, E)),
    "route_grad": dict(logits=f(T, E), ids=i32(T, K_), dwts=f(T, K_), mode=1, norm=True, scale=1.0, dlogits=f(T, E),
                       dscores=f(T, E)),
    "adapters": dict(x=f(T, H), a=f(n, R, H), b=f(n, N, R), scale=f(n), offsets=i32(n + 1), perm=i32(T), base=f(T, N),
                     out=f(T, N), mid=f(9)),
}
half = torch.float16


@pytest.mark.parametrize("op", list(GOOD))
def test_well_formed_host_tensors_are_refused_only_for_the_device(op):
    with pytest.raises(ValueError, match="ROCm device"):
        getattr(block(), op)(**GOOD[op])


@pytest.mark.parametrize("op, left_out", [
    ("rms_norm", dict(residual=None, total=None)), ("rms_norm", dict(y=None)), ("rms_norm", dict(q=None, scale=None)),
    ("rms_norm", dict(rstd=None)), ("rms_norm", dict(x=f(T, H, dtype=half), w=f(H, dtype=half), y=f(T, H, dtype=half))),
    ("rms_norm_grad", dict(dres=None)), ("route_groups", dict(bias=None, scores=None)), ("route_grad", dict(dscores=None)),
    ("adapters", dict(scale=None))])
def test_what_may_be_left_out(op, left_out):
    with pytest.raises(ValueError, match="ROCm device"):
        getattr(block(), op)(**{**GOOD[op], **left_out})


BAD = [
    ("rms_norm", dict(x=f(T, H, dtype=torch.float64)), "dtype"),
    ("rms_norm", dict(x=None), "torch tensor"),
    ("rms_norm", dict(x=f(0, H)), "empty"),
    ("rms_norm", dict(x=f(T, 2 * H)[:, ::2]), "contiguous"),
    ("rms_norm", dict(w=f(H + 1)), "shape"),
    ("rms_norm", dict(w=f(1, H)), "shape"),
    ("rms_norm", dict(w=f(2 * H)[::2]), "contiguous"),
    ("rms_norm", dict(w=i32(H)), "dtype"),
    ("rms_norm", dict(residual=None), "both or neither"),
    ("rms_norm", dict(total=None), "both or neither"),
    ("rms_norm", dict(total=f(T, H, dtype=half)), "dtype"),
    ("rms_norm", dict(residual=f(T + 1, H)), "shape"),
    ("rms_norm", dict(q=None), "both or neither"),
    ("rms_norm", dict(y=None, q=None, scale=None), "at least one"),
    ("rms_norm", dict(y=f(T, H - 1)), "shape"),
    ("rms_norm", dict(q=f(T, H)), "dtype"),
    ("rms_norm", dict(scale=f(T, 1)), "shape"),
    ("rms_norm", dict(rstd=f(T, dtype=half)), "dtype"),
    ("rms_norm_grad", dict(h=f(T, H + 1)), "shape"),
    ("rms_norm_grad", dict(w=f(H - 1)), "shape"),
    ("rms_norm_grad", dict(rstd=f(T + 1)), "shape"),
    ("rms_norm_grad", dict(dx=f(T + 1, H)), "shape"),
    ("rms_norm_grad", dict(dw=f(H, dtype=half)), "dtype"),
    ("rms_norm_grad", dict(part=f(3, 3)), "shape"),
    ("rms_norm_grad", dict(dres=f(T, H, dtype=half)), "dtype"),
    ("rms_norm_grad", dict(dres=f(T, H + 1)), "shape"),
    ("route_groups", dict(logits=f(T, 0)), "empty"),
    ("route_groups", dict(logits=i32(T, E)), "dtype"),
    ("route_groups", dict(ids=i32(T, K_ + 1)), "shape"),
    ("route_groups", dict(ids=torch.zeros((T, K_), dtype=torch.int64)), "dtype"),
    ("route_groups", dict(wts=f(T, K_, dtype=half)), "dtype"),
    ("route_groups", dict(bias=f(E + 1)), "shape"),
    ("route_groups", dict(scores=f(T, E + 1)), "shape"),
    ("route_grad", dict(ids=i32(T * K_)), "shape"),
    ("route_grad", dict(ids=i32(T + 1, K_)), "shape"),
    ("route_grad", dict(dwts=f(T, K_ + 1)), "shape"),
    ("route_grad", dict(dlogits=f(T, E - 1)), "shape"),
    ("route_grad", dict(dscores=f(T, E, dtype=half)), "dtype"),
    ("adapters", dict(a=f(n, R, H + 1)), "shape"),
    ("adapters", dict(a=f(n, R, H, dtype=half)), "dtype"),
    ("adapters", dict(b=f(n + 1, N, R)), "shape"),
    ("adapters", dict(b=f(n, N, R + 1)), "shape"),
    ("adapters", dict(b=f(n, N, R, dtype=torch.bfloat16)), "dtype"),
    ("adapters", dict(a=f(n, 0, H), b=f(n, N, 0)), "empty"),
    ("adapters", dict(scale=f(n + 1)), "shape"),
    ("adapters", dict(offsets=i32(n)), "shape"),
    ("adapters", dict(perm=i32(T + 1)), "shape"),
    ("adapters", dict(out=f(T, N + 1)), "shape"),
    ("adapters", dict(base=f(T, N, dtype=half)), "dtype"),
    ("adapters", dict(mid=f(9, dtype=half)), "dtype"),
]


@pytest.mark.parametrize("op, bad, msg", BAD)
def test_refusals(op, bad, msg):
    with pytest.raises(ValueError, match=msg):
        getattr(block(), op)(**{**GOOD[op], **bad})


def test_null_context_is_refused_by_every_entry_point():
    lib = mb.load_library()
    buf = (ctypes.c_uint8 * 4096)()
    p = ctypes.addressof(buf)
    F, bad = mb.GGML_F32, mb.MOE_ERR_INVALID_ARG
    assert lib.moe_rms_norm(None, p, F, None, None, F, p, F, 1e-6, 1, 4, p, F, None, None, None, None) == bad
    assert lib.moe_rms_norm_grad(None, p, F, p, F, p, F, p, None, 1, 4, p, F, p, p, 64, None) == bad
    assert lib.moe_route_groups(None, p, F, None, 1, 4, 1, 0, 1, 1, 1, 0, 1.0, p, p, None, None) == bad
    assert lib.moe_route_grad(None, p, F, p, p, None, 1, 4, 1, 0, 0, 1.0, p, F, None) == bad
    assert lib.moe_adapters(None, p, p, p, F, None, 1, p, p, 1, 4, 1, 4, p, p, F, p, 64, None) == bad
    assert lib.moe_rms_norm_grad_scratch(None, 1, 4) == 0 and lib.moe_adapters_scratch(None, 1, 4, 1) == 0


@pytest.mark.parametrize("op", list(GOOD))
def test_the_compiled_comparison_says_nothing_of_what_is_not_fine(op):
    calls = torch_calls()
    entries = ctypes.create_string_buffer(8 * 11)  # no entry points: nothing here may get as far as a call
    at, args, call = ctypes.addressof(entries), list(GOOD[op].values()), getattr(calls, op)
    assert call(at, 1, 0, *args, 0) is None  # host tensors
    assert call(at, None, 0, *args, 0) is None and call(at, 1, 0, *args, None) is None
    assert call() is None and call(at, 1, 0, *args) is None and call(at, 1, 0, *args, 0, 0) is None
    for i in range(len(args)):
        for bad in (None, 3, "x", 2 ** 70, torch.zeros(()), torch.zeros(2, 2).to_sparse(), torch.empty((3, 64), device="meta")):
            assert call(at, 1, 0, *args[:i], bad, *args[i + 1:], 0) is None

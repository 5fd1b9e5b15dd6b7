"""The bindings of the operators around the expert products refuse tensors that
would make the kernels read or write out of bounds, before the C-ABI; and the
C-ABI refuses what it can see.  CPU only, on host tensors."""
import ctypes

import pytest
import torch

import moe_block as mb
from test_wrapper_args import _NoLib

H, T, K_, R = 64, 3, 2, 6


def block():
    b = mb.MoeBlock.__new__(mb.MoeBlock)
    b.lib, b.h, b.descs, b.device = _NoLib(), None, {}, 0
    return b


def f(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def i8(*shape):
    return torch.zeros(shape, dtype=torch.int8)


GOOD = {
    "dispatch": dict(x=f(T, H), inv=i32(T * K_), rows=f(R, H)),
    "dispatch_grad": dict(drows=f(R, H), inv=i32(T * K_), dx=f(T, H)),
    "combine": dict(rows=f(R, H), wts=f(T, K_), inv=i32(T * K_), out=f(T, H)),
    "combine_grad": dict(dout=f(T, H), rows=f(R, H), wts=f(T, K_), inv=i32(T * K_), drows=f(R, H), dwts=f(T, K_)),
    "quantize_i8": dict(x=f(T, H), q=i8(T, H), scale=f(T)),
    "matmul_i8": dict(q=i8(T, H), scale=f(T), w=i8(8, H), w_scale=f(8), out=f(T, 8)),
}
GROUPED = dict(q=i8(T, H), scale=f(T), w=i8(4, 8, H), w_scale=f(4, 8), out=f(R, 8), offsets=i32(5), perm=i32(R), k=2)


@pytest.mark.parametrize("op", list(GOOD))
def test_well_formed_host_tensors_are_refused_only_for_the_device(op):
    with pytest.raises(ValueError, match="ROCm device"):
        getattr(block(), op)(**GOOD[op])


def test_well_formed_grouped_product_is_refused_only_for_the_device():
    with pytest.raises(ValueError, match="ROCm device"):
        block().matmul_i8(**GROUPED)
    with pytest.raises(ValueError, match="ROCm device"):
        block().matmul_i8(**{**GROUPED, "swiglu": True, "out": f(R, 4)})


BAD = [
    ("dispatch", dict(x=f(T, H, dtype=torch.float64)), "dtype"),
    ("dispatch", dict(x=None), "torch tensor"),
    ("dispatch", dict(x=f(0, H)), "empty"),
    ("dispatch", dict(x=f(T, 2 * H)[:, ::2]), "contiguous"),
    ("dispatch", dict(rows=f(R, H + 1)), "shape"),
    ("dispatch", dict(rows=f(0, H)), "empty"),
    ("dispatch", dict(inv=i32(T * K_ + 1)), "inv"),
    ("dispatch", dict(inv=i32(0)), "inv"),
    ("dispatch", dict(inv=i32(K_, T)), "inv"),
    ("dispatch", dict(inv=i32(T * 65)), "at most 64"),
    ("dispatch", dict(inv=torch.zeros(T * K_, dtype=torch.int64)), "dtype"),
    ("dispatch_grad", dict(dx=f(T, H - 1)), "shape"),
    ("combine", dict(wts=f(T, K_ + 1)), "shape"),
    ("combine", dict(wts=f(T, K_, dtype=torch.float16)), "dtype"),
    ("combine", dict(out=f(T, H, dtype=torch.int8)), "dtype"),
    ("combine_grad", dict(drows=f(R, H, dtype=torch.float16)), "dtype"),
    ("combine_grad", dict(drows=f(R + 1, H)), "shape"),
    ("combine_grad", dict(dwts=f(T * K_)), "shape"),
    ("quantize_i8", dict(q=i8(T, H + 1)), "shape"),
    ("quantize_i8", dict(q=f(T, H)), "dtype"),
    ("quantize_i8", dict(scale=f(T + 1)), "shape"),
    ("matmul_i8", dict(w=i8(8, H + 1)), "shape"),
    ("matmul_i8", dict(w=i8(1, 8, H)), "shape"),
    ("matmul_i8", dict(w_scale=f(9)), "shape"),
    ("matmul_i8", dict(out=f(T + 1, 8)), "rows"),
    ("matmul_i8", dict(out=f(T, 8, dtype=torch.int32)), "dtype"),
    ("matmul_i8", dict(w=i8(7, H), w_scale=f(7), out=f(T, 3), swiglu=True), "gate and up"),
    ("matmul_i8", dict(swiglu=True), "shape"),
    ("matmul_i8", dict(k=2), "perm"),
    ("matmul_i8", dict(q=i8(T, 0), w=i8(8, 0)), "empty"),
    ("matmul_i8", dict(perm=i32(T + 1)), "shape"),
    ("matmul_i8", dict(offsets=i32(2)), "shape"),
]


@pytest.mark.parametrize("op, bad, msg", BAD)
def test_refusals(op, bad, msg):
    with pytest.raises(ValueError, match=msg):
        getattr(block(), op)(**{**GOOD[op], **bad})


@pytest.mark.parametrize("bad", [dict(offsets=i32(4)), dict(perm=i32(R - 1)), dict(w_scale=f(4, 9)), dict(w=i8(8, H)),
                                 dict(perm=None)])
def test_grouped_refusals(bad):
    with pytest.raises(ValueError):
        block().matmul_i8(**{**GROUPED, **bad})


def test_null_context_is_refused_by_every_entry_point():
    lib = mb.load_library()
    buf = (ctypes.c_uint8 * 4096)()
    p = ctypes.addressof(buf)
    F32 = mb.GGML_F32
    assert lib.moe_dispatch(None, p, F32, p, 1, 1, 4, 1, p, F32, None) == mb.MOE_ERR_INVALID_ARG
    assert lib.moe_dispatch_grad(None, p, F32, 1, p, 1, 1, 4, p, F32, None) == mb.MOE_ERR_INVALID_ARG
    assert lib.moe_combine(None, p, F32, 1, p, p, 1, 1, 4, p, F32, None) == mb.MOE_ERR_INVALID_ARG
    assert lib.moe_combine_grad(None, p, F32, p, F32, 1, p, p, 1, 1, 4, p, p, None) == mb.MOE_ERR_INVALID_ARG
    assert lib.moe_quantize_i8(None, p, F32, 1, 4, p, p, None) == mb.MOE_ERR_INVALID_ARG
    assert lib.moe_matmul_i8(None, p, p, 1, p, p, 1, None, None, 1, 1, 1, 4, 0, 0.0, p, F32, None) == mb.MOE_ERR_INVALID_ARG


def torch_calls():
    mb._know_torch()
    if mb._torch_calls is None:
        pytest.skip("moe_torch.so was not built for this torch")
    return mb._torch_calls


ENTRIES = ctypes.create_string_buffer(8 * 6)  # no entry points: nothing here may get as far as a call


@pytest.mark.parametrize("op", list(GOOD))
def test_the_compiled_comparison_says_nothing_of_what_is_not_fine(op):
    calls, at = torch_calls(), ctypes.addressof(ENTRIES)
    args = list(GOOD[op].values()) + ([None, None, 1, False, 0.0] if op == "matmul_i8" else [])
    call = getattr(calls, op)
    assert call(at, 1, 0, *args, 0) is None  # host tensors
    assert call(at, None, 0, *args, 0) is None and call(at, 1, 0, *args, None) is None
    assert call() is None and call(at, 1, 0, *args) is None and call(at, 1, 0, *args, 0, 0) is None
    assert call(at, 2 ** 70, 0, *args, 0) is None and call(at, 1, 0, *args, "stream") is None
    for i in range(len(args)):
        for bad in (None, 3, "x", torch.zeros(()), torch.zeros(2, 2).to_sparse(), torch.empty((3, 64), device="meta")):
            assert call(at, 1, 0, *args[:i], bad, *args[i + 1:], 0) is None


def test_dimensions_past_32_bits_are_refused():
    """meta tensors: shapes without memory, on the context's device as far as the check can see."""
    class OnDevice:
        def __init__(self, t):
            self.t = t

        def __getattr__(self, name):
            return getattr(self.t, name)

        def get_device(self):
            return 0

    n = 2 ** 31 + T
    x, rows = (OnDevice(torch.empty((m, 1), device="meta")) for m in (n, R))
    inv = OnDevice(torch.empty((n * K_,), dtype=torch.int32, device="meta"))
    with pytest.raises(ValueError, match="at most 2"):
        block().dispatch(x, inv, rows)

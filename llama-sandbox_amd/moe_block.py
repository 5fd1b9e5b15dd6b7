"""Python binding of the gfx950 MoE block (ctypes over libmoe_block.so).

A thin host-side mirror of the C-ABI in include/moe_block.h.  Device
buffers are torch tensors on a ROCm device (torch is only the allocator and
stream owner here); every computation runs in the HIP library.  There is no
CPU fallback in this module: if the library is missing or a call fails, a
MoeError is raised and the caller decides (the reference's backend falls
back to ggml-cpu at that point, moe-serv/src/moe_backend.cpp:436-445).
"""
from __future__ import annotations

import ctypes
import functools
import importlib.util
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmoe_block.so")

MOE_OK = 0
MOE_ERR_INVALID_ARG = -1
MOE_ERR_HIP = -2
MOE_ERR_OUT_OF_BUDGET = -3
MOE_ERR_UNSUPPORTED = -4
MOE_ERR_NOT_RESIDENT = -5
MOE_ERR_NO_DEVICE = -6
MOE_ERR_INJECTED = -7
MOE_ERR_FORMAT = -8

MOE_FWD_PER_SLOT = 1
MOE_FWD_NO_SHARED = 2
MOE_MM_SWIGLU = 1

ROUTE_SOFTMAX, ROUTE_SIGMOID, ROUTE_SQRT_SOFTPLUS = 0, 1, 2
T_GATE, T_UP, T_DOWN = 0, 1, 2

# every entry point include/moe_block.h declares
EXPORTS = (
    "moe_ctx_create", "moe_ctx_destroy", "moe_ctx_last_error", "moe_status_str", "moe_ctx_budget_left",
    "moe_device_memory",
    "moe_ctx_reserve", "moe_layer_upload", "moe_layer_generate", "moe_layer_read_blocks",
    "moe_layer_release", "moe_layer_bytes", "moe_route", "moe_group", "moe_forward", "moe_forward_noalloc",
    "moe_forward_host",
    "moe_route_forward", "moe_graph_capture", "moe_graph_launch", "moe_graph_destroy",
    "moe_prof_enable", "moe_prof_read", "moe_call_stats_read", "moe_debug_set_taps",
    "moe_debug_quantize_q8_0", "moe_debug_wave_sum", "moe_debug_last_h", "moe_debug_set_timeline",
    "moe_debug_read_timeline",
    "moe_gguf_read_layer", "moe_layer_upload_gguf",
    "moe_server_open", "moe_server_close", "moe_server_last_error", "moe_server_handle", "moe_server_listen",
    "moe_server_serve", "moe_router_logits", "moe_node_claimed", "moe_split_parse", "moe_split_compute",
    "moe_dispatch", "moe_dispatch_grad", "moe_combine", "moe_combine_grad", "moe_quantize_i8", "moe_matmul_i8",
    "moe_rms_norm", "moe_rms_norm_grad", "moe_rms_norm_grad_scratch", "moe_route_groups", "moe_route_grad",
    "moe_adapters", "moe_adapters_scratch",
)

# graph nodes of the ggml backend's split (include/moe_block.h, moe_node)
(NODE_NONE, NODE_RESHAPE, NODE_VIEW, NODE_PERMUTE, NODE_TRANSPOSE, NODE_MUL_MAT_ID, NODE_CLAMP, NODE_MUL, NODE_GLU,
 NODE_ADD, NODE_OTHER) = range(11)
GLU_SWIGLU = 2
GGML_F32, GGML_F16, GGML_BF16, GGML_I32, GGML_MXFP4 = 0, 1, 30, 26, 39

# nano-glm moe-server protocol v2 (include/moe_block.h, moe_wire_*)
WIRE_MAGIC, WIRE_VERSION = 0x454F4D4E, 2
WIRE_REQUEST, WIRE_RESPONSE, WIRE_HELLO = 1, 2, 3
WIRE_RET_COMBINED, WIRE_RET_PER_SLOT = 0, 1
WIRE_OK, WIRE_ERR_VERSION, WIRE_ERR_DIMS, WIRE_ERR_LAYER, WIRE_ERR_MODE, WIRE_ERR_INTERNAL = range(6)


class MoeError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"{message} (status {status})")
        self.status = status


class LayerDesc(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int32), ("ffn", ctypes.c_int32), ("n_expert", ctypes.c_int32),
                ("n_used", ctypes.c_int32), ("has_shared", ctypes.c_int32), ("clamp", ctypes.c_float)]

    @classmethod
    def of(cls, shape) -> "LayerDesc":
        return cls(shape.hidden, shape.ffn, shape.n_expert, shape.n_used, int(shape.has_shared),
                   float(shape.clamp))


class GgufLayer(ctypes.Structure):
    """moe_gguf_layer: one MoE layer of a GGUF model (shape and router keys)."""
    _fields_ = [("desc", LayerDesc), ("n_layer", ctypes.c_int32), ("route_mode", ctypes.c_int32),
                ("route_norm", ctypes.c_int32), ("route_scale", ctypes.c_float), ("shared_type", ctypes.c_int32),
                ("arch", ctypes.c_char * 32)]


class WireHelloRequest(ctypes.Structure):
    _fields_ = [("magic", ctypes.c_uint32), ("version", ctypes.c_uint32), ("msg_type", ctypes.c_uint32),
                ("reserved", ctypes.c_uint32), ("payload_bytes", ctypes.c_uint64)]


class WireHelloResponse(ctypes.Structure):
    _fields_ = [("magic", ctypes.c_uint32), ("version", ctypes.c_uint32), ("msg_type", ctypes.c_uint32),
                ("status", ctypes.c_uint32), ("arch", ctypes.c_char * 16), ("n_embd", ctypes.c_uint32),
                ("n_layer", ctypes.c_uint32), ("n_dense_lead", ctypes.c_uint32), ("n_expert", ctypes.c_uint32),
                ("n_expert_used", ctypes.c_uint32), ("n_ff_exp", ctypes.c_uint32), ("expert_scale", ctypes.c_float),
                ("expert_norm", ctypes.c_uint32), ("reserved", ctypes.c_uint32 * 2),
                ("payload_bytes", ctypes.c_uint64)]


class WireRequest(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("magic", "version", "msg_type", "layer", "n_embd", "n_tokens",
                                               "return_mode", "reserved")] + [("payload_bytes", ctypes.c_uint64)]


class WireResponse(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("magic", "version", "msg_type", "status", "n_embd", "n_tokens",
                                               "n_slots", "reserved", "t_parse_us", "t_route_us", "t_compute_us",
                                               "t_serialize_us")] + [("payload_bytes", ctypes.c_uint64)]


class MoeNode(ctypes.Structure):
    pass


MoeNode._fields_ = [("op", ctypes.c_int32), ("type", ctypes.c_int32), ("ne", ctypes.c_int64 * 4),
                    ("contiguous", ctypes.c_int32), ("in_moe_buffer", ctypes.c_int32), ("glu_op", ctypes.c_int32),
                    ("glu_swapped", ctypes.c_int32), ("clamp_min", ctypes.c_float), ("clamp_max", ctypes.c_float),
                    ("src", ctypes.POINTER(MoeNode) * 3), ("view_src", ctypes.POINTER(MoeNode)),
                    ("data", ctypes.c_void_p), ("name", ctypes.c_char_p)]


class MoeSplit(ctypes.Structure):
    _fields_ = [(n, ctypes.POINTER(MoeNode)) for n in ("gate_w", "up_w", "down_w", "x", "ids", "wts", "out")] + \
               [(n, ctypes.c_float) for n in ("gate_min", "gate_max", "up_min", "up_max")] + \
               [(n, ctypes.c_int32) for n in ("layer", "n_slots", "n_tokens", "hidden", "ffn", "n_expert")]


class KernelStat(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char_p), ("launches", ctypes.c_uint64), ("total_us", ctypes.c_double)]


class CallStats(ctypes.Structure):
    """moe_call_stats: engagement and phase counters of the host-boundary calls."""
    _fields_ = [(n, ctypes.c_uint64) for n in ("calls", "refusals", "expert_loads", "timed_calls")] + \
               [(n, ctypes.c_double) for n in ("upload_us", "compute_us", "read_us", "total_us", "last_upload_us",
                                              "last_compute_us", "last_read_us", "last_total_us")] + \
               [(n, ctypes.c_uint32) for n in ("last_experts", "last_tokens", "last_timed")]


_vp = ctypes.c_void_p
_lib = None


def load_library(path: str | None = None):
    """Load libmoe_block.so; raises MoeError if it has not been built."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = path or LIB_PATH
    if not os.path.exists(p):
        raise MoeError(MOE_ERR_NO_DEVICE, f"{p} is not built (run __graft_entry__.build())")
    L = ctypes.CDLL(p)
    st = ctypes.c_int
    L.moe_ctx_create.restype = st
    L.moe_ctx_create.argtypes = [ctypes.c_int, ctypes.c_uint64, ctypes.POINTER(_vp)]
    L.moe_ctx_destroy.restype = None
    L.moe_ctx_destroy.argtypes = [_vp]
    L.moe_ctx_last_error.restype = ctypes.c_char_p
    L.moe_ctx_last_error.argtypes = [_vp]
    L.moe_status_str.restype = ctypes.c_char_p
    L.moe_status_str.argtypes = [st]
    L.moe_ctx_budget_left.restype = ctypes.c_uint64
    L.moe_ctx_budget_left.argtypes = [_vp]
    L.moe_ctx_reserve.restype = st
    L.moe_ctx_reserve.argtypes = [_vp, ctypes.POINTER(LayerDesc), ctypes.c_int]
    L.moe_layer_upload.restype = st
    L.moe_layer_upload.argtypes = [_vp, ctypes.c_int, ctypes.POINTER(LayerDesc)] + [_vp] * 6
    L.moe_layer_generate.restype = st
    L.moe_layer_generate.argtypes = [_vp, ctypes.c_int, ctypes.POINTER(LayerDesc), ctypes.c_uint64,
                                     ctypes.c_int, ctypes.c_int]
    L.moe_layer_read_blocks.restype = st
    L.moe_layer_read_blocks.argtypes = [_vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp]
    L.moe_layer_release.restype = st
    L.moe_layer_release.argtypes = [_vp, ctypes.c_int]
    L.moe_layer_bytes.restype = st
    L.moe_layer_bytes.argtypes = [_vp, ctypes.c_int, ctypes.POINTER(ctypes.c_uint64)]
    L.moe_route.restype = st
    L.moe_route.argtypes = [_vp, _vp, _vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                            ctypes.c_int, ctypes.c_float, _vp, _vp, _vp]
    L.moe_group.restype = st
    L.moe_group.argtypes = [_vp, _vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp, _vp, _vp, _vp, _vp]
    L.moe_forward.restype = st
    L.moe_forward.argtypes = [_vp, ctypes.c_int, _vp, _vp, _vp, ctypes.c_int, _vp, ctypes.c_uint32, _vp]
    L.moe_forward_noalloc.restype = st
    L.moe_forward_noalloc.argtypes = [_vp, ctypes.c_int, _vp, _vp, _vp, ctypes.c_int, _vp, ctypes.c_uint32, _vp]
    L.moe_forward_host.restype = st
    L.moe_forward_host.argtypes = [_vp, ctypes.c_int, _vp, _vp, _vp, ctypes.c_int, _vp, ctypes.c_uint32]
    L.moe_route_forward.restype = st
    L.moe_route_forward.argtypes = [_vp, ctypes.c_int, _vp, _vp, _vp, ctypes.c_int, ctypes.c_int,
                                    ctypes.c_int, ctypes.c_float, _vp, _vp, _vp, ctypes.c_uint32, _vp]
    L.moe_graph_capture.restype = st
    L.moe_graph_capture.argtypes = [_vp, ctypes.c_int, ctypes.POINTER(ctypes.c_int), ctypes.POINTER(_vp),
                                    ctypes.POINTER(_vp), ctypes.POINTER(_vp), ctypes.POINTER(_vp),
                                    ctypes.c_int, ctypes.c_uint32, ctypes.POINTER(_vp)]
    L.moe_graph_launch.restype = st
    L.moe_graph_launch.argtypes = [_vp, _vp]
    L.moe_graph_destroy.restype = None
    L.moe_graph_destroy.argtypes = [_vp]
    L.moe_prof_enable.restype = st
    L.moe_prof_enable.argtypes = [_vp, ctypes.c_int]
    L.moe_prof_read.restype = st
    L.moe_prof_read.argtypes = [_vp, ctypes.POINTER(KernelStat), ctypes.c_int, ctypes.POINTER(ctypes.c_int),
                                ctypes.c_int]
    L.moe_call_stats_read.restype = st
    L.moe_call_stats_read.argtypes = [_vp, ctypes.POINTER(CallStats), ctypes.c_int]
    L.moe_debug_set_taps.restype = st
    L.moe_debug_set_taps.argtypes = [_vp, ctypes.c_int]
    L.moe_debug_quantize_q8_0.restype = st
    L.moe_debug_quantize_q8_0.argtypes = [_vp, _vp, ctypes.c_int, _vp, _vp, _vp]
    L.moe_debug_wave_sum.restype = st
    L.moe_debug_wave_sum.argtypes = [_vp, _vp, ctypes.c_int, _vp, _vp]
    L.moe_debug_last_h.restype = st
    L.moe_debug_last_h.argtypes = [_vp, _vp, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)]
    L.moe_debug_set_timeline.restype = st
    L.moe_debug_set_timeline.argtypes = [_vp, ctypes.c_int]
    L.moe_debug_read_timeline.restype = st
    L.moe_debug_read_timeline.argtypes = [_vp, _vp, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t),
                                          ctypes.POINTER(ctypes.c_size_t)]
    L.moe_gguf_read_layer.restype = st
    L.moe_gguf_read_layer.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(GgufLayer), ctypes.c_char_p,
                                      ctypes.c_size_t]
    L.moe_layer_upload_gguf.restype = st
    L.moe_layer_upload_gguf.argtypes = [_vp, ctypes.c_int, ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(GgufLayer)]
    L.moe_server_open.restype = st
    L.moe_server_open.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_uint64, ctypes.POINTER(_vp),
                                  ctypes.c_char_p, ctypes.c_size_t]
    L.moe_server_close.restype = None
    L.moe_server_close.argtypes = [_vp]
    L.moe_server_last_error.restype = ctypes.c_char_p
    L.moe_server_last_error.argtypes = [_vp]
    L.moe_server_handle.restype = st
    L.moe_server_handle.argtypes = [_vp, _vp, ctypes.c_size_t, _vp, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)]
    L.moe_server_listen.restype = st
    L.moe_server_listen.argtypes = [_vp, ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    L.moe_server_serve.restype = st
    L.moe_server_serve.argtypes = [_vp, ctypes.c_int]
    L.moe_node_claimed.restype = ctypes.c_int
    L.moe_node_claimed.argtypes = [ctypes.POINTER(MoeNode)]
    L.moe_split_parse.restype = st
    L.moe_split_parse.argtypes = [ctypes.POINTER(ctypes.POINTER(MoeNode)), ctypes.c_int, ctypes.POINTER(MoeSplit),
                                  ctypes.c_char_p, ctypes.c_size_t]
    L.moe_split_compute.restype = st
    L.moe_split_compute.argtypes = [_vp, ctypes.POINTER(ctypes.POINTER(MoeNode)), ctypes.c_int]
    L.moe_router_logits.restype = st
    L.moe_router_logits.argtypes = [_vp, _vp, _vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp, _vp]
    ci = ctypes.c_int
    L.moe_dispatch.restype = st
    L.moe_dispatch.argtypes = [_vp, _vp, ci, _vp, ci, ci, ci, ci, _vp, ci, _vp]
    L.moe_dispatch_grad.restype = st
    L.moe_dispatch_grad.argtypes = [_vp, _vp, ci, ci, _vp, ci, ci, ci, _vp, ci, _vp]
    L.moe_combine.restype = st
    L.moe_combine.argtypes = [_vp, _vp, ci, ci, _vp, _vp, ci, ci, ci, _vp, ci, _vp]
    L.moe_combine_grad.restype = st
    L.moe_combine_grad.argtypes = [_vp, _vp, ci, _vp, ci, ci, _vp, _vp, ci, ci, ci, _vp, _vp, _vp]
    L.moe_quantize_i8.restype = st
    L.moe_quantize_i8.argtypes = [_vp, _vp, ci, ci, ci, _vp, _vp, _vp]
    L.moe_matmul_i8.restype = st
    L.moe_matmul_i8.argtypes = [_vp, _vp, _vp, ci, _vp, _vp, ci, _vp, _vp, ci, ci, ci, ci, ctypes.c_uint32,
                                ctypes.c_float, _vp, ci, _vp]
    cf, sz = ctypes.c_float, ctypes.c_size_t
    L.moe_rms_norm.restype = st
    L.moe_rms_norm.argtypes = [_vp, _vp, ci, _vp, _vp, ci, _vp, ci, cf, ci, ci, _vp, ci, _vp, _vp, _vp, _vp]
    L.moe_rms_norm_grad_scratch.restype = sz
    L.moe_rms_norm_grad_scratch.argtypes = [_vp, ci, ci]
    L.moe_rms_norm_grad.restype = st
    L.moe_rms_norm_grad.argtypes = [_vp, _vp, ci, _vp, ci, _vp, ci, _vp, _vp, ci, ci, _vp, ci, _vp, _vp, sz, _vp]
    L.moe_route_groups.restype = st
    L.moe_route_groups.argtypes = [_vp, _vp, ci, _vp, ci, ci, ci, ci, ci, ci, ci, ci, cf, _vp, _vp, _vp, _vp]
    L.moe_route_grad.restype = st
    L.moe_route_grad.argtypes = [_vp, _vp, ci, _vp, _vp, _vp, ci, ci, ci, ci, ci, cf, _vp, ci, _vp]
    L.moe_adapters_scratch.restype = sz
    L.moe_adapters_scratch.argtypes = [_vp, ci, ci, ci]
    L.moe_adapters.restype = st
    L.moe_adapters.argtypes = [_vp, _vp, _vp, _vp, ci, _vp, ci, _vp, _vp, ci, ci, ci, ci, _vp, _vp, ci, _vp, sz, _vp]
    if path is None:
        _lib = L
    return L


def node_list(nodes):
    """A C array of pointers to MoeNode structures (the caller keeps them alive)."""
    arr = (ctypes.POINTER(MoeNode) * len(nodes))()
    for i, nd in enumerate(nodes):
        arr[i] = ctypes.pointer(nd)
    return arr


def node_claimed(node: MoeNode) -> bool:
    return bool(load_library().moe_node_claimed(ctypes.byref(node)))


def split_parse(nodes) -> MoeSplit:
    """Parse the routed-expert split; raises MoeError (MOE_ERR_UNSUPPORTED with the reason)."""
    L = load_library()
    sp = MoeSplit()
    why = ctypes.create_string_buffer(256)
    st = L.moe_split_parse(node_list(nodes), len(nodes), ctypes.byref(sp), why, len(why))
    if st != MOE_OK:
        raise MoeError(st, f"moe_split_parse: {why.value.decode()}")
    return sp


def read_gguf_layer(path: str, layer: int) -> GgufLayer:
    """Shape and router keys of one MoE layer of a GGUF model (no device needed);
    raises MoeError (MOE_ERR_FORMAT for a file that cannot be read as one)."""
    L = load_library()
    info = GgufLayer()
    err = ctypes.create_string_buffer(512)
    st = L.moe_gguf_read_layer(os.fsencode(path), int(layer), ctypes.byref(info), err, len(err))
    if st != MOE_OK:
        raise MoeError(st, f"moe_gguf_read_layer: {err.value.decode(errors='replace')}")
    return info


def _ptr(t) -> int | None:
    """Device pointer of a torch tensor (or None)."""
    return None if t is None else int(t.data_ptr())


# ---- argument checks ---------------------------------------------------------------
# The C-ABI takes raw pointers and sizes: a tensor of the wrong dtype, shape or
# device would make the kernels read or write out of bounds.  Every wrapper
# below checks its tensors before the call and raises ValueError instead.
# The order (dtype, shape, contiguity, device) lets the CPU tests reach each
# refusal with host tensors.

NOALLOC_SCRATCH_BYTES = 64 << 20  # MOE_NOALLOC_SCRATCH_BYTES

_dtypes: dict = {}  # name -> torch dtype, filled at the first use (torch is imported by then)


def _is_fine(t, dtype: str, shape, device: bool) -> bool:
    """Does t pass check_tensor?  A decode call checks four to seven tensors in
    the 15 us that its kernels take, and comparing objects costs a fifth of
    building the names and the messages."""
    try:
        want = _dtypes.get(dtype)
        if want is None:
            import torch
            want = _dtypes[dtype] = getattr(torch, dtype)
        return (t.dtype is want and (shape is None or t.shape == shape) and t.is_contiguous()
                and (not device or t.is_cuda))
    except (AttributeError, ImportError):  # without torch nothing is a tensor
        return False


def check_tensor(t, name: str, dtype: str, shape=None, device: bool = True):
    """t: a torch tensor of `dtype` ("float32", "int32", ...), `shape` (a
    tuple, None entries match anything), contiguous, on a GPU if `device`."""
    if _is_fine(t, dtype, shape, device):
        return
    if t is None or not hasattr(t, "data_ptr"):
        raise ValueError(f"{name}: expected a torch tensor, got {type(t).__name__}")
    if str(t.dtype) != f"torch.{dtype}":
        raise ValueError(f"{name}: dtype {t.dtype}, expected torch.{dtype}")
    if shape is not None:
        if t.dim() != len(shape) or any(want is not None and got != want for got, want in zip(t.shape, shape)):
            raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: not contiguous")
    if device and t.device.type != "cuda":
        raise ValueError(f"{name}: on {t.device}, expected a ROCm device tensor")


_row_types: dict = {}  # torch dtype -> ggml type of a row operand, filled by the first call that takes one
_raw_stream = _torch_calls = None


def _know_torch():
    """What the operators on torch tensors need of torch; nothing where it is not installed."""
    global _raw_stream, _torch_calls
    if not _row_types:
        try:
            import torch
        except ImportError:
            return
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        # csrc/moe_torch.cpp, built against one torch; without it the same calls go through ctypes
        try:
            spec = importlib.util.spec_from_file_location("moe_torch", os.path.join(_HERE, "moe_torch.so"))
            calls = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(calls)
            whole = all(hasattr(calls, n[len("moe_"):]) for n, _ in _Entries._fields_)  # (not one of an earlier build)
            if whole and calls.torch_version == torch.__version__.partition("+")[0] and _raw_stream is not None:
                calls.set_current_stream(_raw_stream)
                _torch_calls = calls
        except ImportError:
            pass
        # last: another thread that finds the types finds the rest too
        _row_types.update({torch.float32: GGML_F32, torch.float16: GGML_F16, torch.bfloat16: GGML_BF16})


class _Entries(ctypes.Structure):
    """The entry points that moe_torch calls, by address."""
    _fields_ = [(n, _vp) for n in ("moe_dispatch", "moe_dispatch_grad", "moe_combine", "moe_combine_grad",
                                   "moe_quantize_i8", "moe_matmul_i8", "moe_rms_norm", "moe_rms_norm_grad",
                                   "moe_route_groups", "moe_route_grad", "moe_adapters")]


def _row_type(t, name: str) -> int:
    """The ggml type of a row operand (float32, float16 or bfloat16)."""
    _know_torch()
    v = _row_types.get(getattr(t, "dtype", None))
    if v is None:
        if not hasattr(t, "data_ptr"):
            raise ValueError(f"{name}: expected a torch tensor, got {type(t).__name__}")
        raise ValueError(f"{name}: dtype {t.dtype}, expected torch.float32, torch.float16 or torch.bfloat16")
    return v


def check_rows(name: str, t, rows=None, cols=None) -> int:
    """t: a contiguous 2-d row operand of [rows, cols] (None: any, at least
    one) of a row type; its ggml type."""
    ty = _row_type(t, name)
    sh = t.shape
    if len(sh) != 2 or (rows is not None and sh[0] != rows) or (cols is not None and sh[1] != cols):
        raise ValueError(f"{name}: shape {tuple(sh)}, expected {(rows, cols)}")
    if sh[0] == 0 or sh[1] == 0:
        raise ValueError(f"{name}: empty")
    if not t.is_contiguous():
        raise ValueError(f"{name}: not contiguous")
    return ty


def check_gain(w, H: int) -> int:
    """w: a contiguous [H] operand of a row type; its ggml type."""
    ty = _row_type(w, "w")
    if w.dim() != 1 or w.shape[0] != H:
        raise ValueError(f"w: shape {tuple(w.shape)}, expected ({H},)")
    if not w.is_contiguous():
        raise ValueError("w: not contiguous")
    return ty


def check_pairs(inv, T: int) -> int:
    """k of a pair map inv, int32 [T * k] (or [T, k]) for T tokens."""
    check_tensor(inv, "inv", "int32", device=False)
    n = inv.numel()
    if n == 0 or n % T or (inv.dim() == 2 and inv.shape[0] != T) or inv.dim() > 2:
        raise ValueError(f"inv: shape {tuple(inv.shape)}, expected (T * k,) or (T, k) with T = {T}")
    if n // T > 64:
        raise ValueError(f"inv: k = {n // T}, at most 64")
    return n // T


def check_forward_args(desc, x, ids, wts, out, flags: int = 0):
    """moe_forward's tensors: x float32 [T, H]; ids int32 / wts float32
    [T, k]; out float32 [T, H], or [T, k, H] with MOE_FWD_PER_SLOT.  desc:
    the layer's LayerDesc (None: the layer is unknown here, the library
    answers MOE_ERR_NOT_RESIDENT; only dtypes and layout are checked)."""
    H = desc.hidden if desc is not None else None
    k = desc.n_used if desc is not None else None
    if desc is not None and getattr(x, "ndim", 0) == 2:
        T = x.shape[0]
        rows = (T, k)
        if (T > 0 and _is_fine(x, "float32", (T, H), True) and _is_fine(ids, "int32", rows, True)
                and _is_fine(wts, "float32", rows, True)
                and _is_fine(out, "float32", (T, k, H) if flags & MOE_FWD_PER_SLOT else (T, H), True)):
            return T
    check_tensor(x, "x", "float32", (None, H), device=False)
    T = int(x.shape[0])
    if T <= 0:
        raise ValueError("x: no tokens")
    check_tensor(ids, "ids", "int32", (T, k), device=False)
    check_tensor(wts, "wts", "float32", (T, k), device=False)
    check_tensor(out, "out", "float32", (T, k, H) if flags & MOE_FWD_PER_SLOT else (T, H), device=False)
    for t, nm in ((x, "x"), (ids, "ids"), (wts, "wts"), (out, "out")):
        if t.device.type != "cuda":
            raise ValueError(f"{nm}: on {t.device}, expected a ROCm device tensor")
    return T


def check_host_forward_args(desc, x, ids, wts):
    """moe_forward_host's numpy arrays: x [T, H], ids / wts [T, k]."""
    if x.ndim != 2 or x.shape[1] != desc.hidden or x.shape[0] <= 0:
        raise ValueError(f"x: shape {x.shape}, expected (T, {desc.hidden})")
    T = x.shape[0]
    for a, nm in ((ids, "ids"), (wts, "wts")):
        if a.shape != (T, desc.n_used):
            raise ValueError(f"{nm}: shape {a.shape}, expected ({T}, {desc.n_used})")
    return T


def _current_stream() -> int:
    """The handle of torch.cuda.current_stream(), without the Stream object
    around it (3 us of a 16 us call) where torch offers that."""
    import torch
    raw, dev = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)
    if raw is None or dev is None or not torch.cuda.is_initialized():
        return int(torch.cuda.current_stream().cuda_stream)
    return int(raw(dev()))


def _stream(stream) -> int | None:
    return _current_stream() if stream is None else int(stream)


def _device_stream(device: int) -> int:
    """The handle of torch's current stream of one device, whichever is current."""
    if _raw_stream is not None:
        return _raw_stream(device)
    import torch
    return int(torch.cuda.current_stream(device).cuda_stream)


class Graph:
    def __init__(self, ctx: "MoeBlock", handle: int, keep):
        self._ctx, self._h, self._keep = ctx, handle, keep

    def launch(self, stream=None):
        self._ctx._check(self._ctx.lib.moe_graph_launch(self._h, _stream(stream)), "moe_graph_launch")

    def close(self):
        if self._h:
            self._ctx.lib.moe_graph_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class MoeBlock:
    """One device context: resident layers plus per-call scratch."""

    def __init__(self, device: int = 0, budget_bytes: int = 2 ** 64 - 1, lib_path: str | None = None):
        self.lib = load_library(lib_path)
        h = _vp()
        st = self.lib.moe_ctx_create(device, budget_bytes, ctypes.byref(h))
        if st != MOE_OK:
            raise MoeError(st, f"moe_ctx_create: {self.lib.moe_status_str(st).decode()}")
        self.h = h.value
        self.device = int(device)
        self.descs: dict[int, LayerDesc] = {}

    @functools.cached_property
    def _calls(self):
        """moe_torch's argument, the address of this context's library's entry points; None: calls go
        through ctypes.  Found at the first call: a context on host arrays needs no torch."""
        if not self.h:
            return None
        _know_torch()
        if _torch_calls is None:
            return None
        self._entries = _Entries(*(ctypes.cast(getattr(self.lib, n), _vp).value for n, _ in _Entries._fields_))
        return ctypes.addressof(self._entries)

    # -- lifecycle --------------------------------------------------------
    def close(self):
        if getattr(self, "h", None):
            self.lib.moe_ctx_destroy(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st: int, what: str):
        if st != MOE_OK:
            msg = self.lib.moe_ctx_last_error(self.h).decode() if self.h else ""
            raise MoeError(st, f"{what}: {self.lib.moe_status_str(st).decode()}: {msg}")

    @property
    def budget_left(self) -> int:
        return int(self.lib.moe_ctx_budget_left(self.h))

    def reserve(self, shape, max_tokens: int):
        d = LayerDesc.of(shape)
        self._check(self.lib.moe_ctx_reserve(self.h, ctypes.byref(d), max_tokens), "moe_ctx_reserve")

    # -- residency ----------------------------------------------------------
    def upload_layer(self, layer: int, shape, gate: np.ndarray, up: np.ndarray, down: np.ndarray,
                     shared=None):
        d = LayerDesc.of(shape)
        arrs = [np.ascontiguousarray(a, np.uint8) for a in (gate, up, down)]
        sh = [np.ascontiguousarray(a, np.uint8) for a in shared] if shared is not None else [None] * 3
        ptrs = [a.ctypes.data if a is not None else None for a in arrs + sh]
        self._check(self.lib.moe_layer_upload(self.h, layer, ctypes.byref(d), *ptrs), "moe_layer_upload")
        self.descs[layer] = d

    def upload_layer_gguf(self, layer: int, path: str, file_layer: int) -> GgufLayer:
        """Make layer `file_layer` of a GGUF model resident as `layer`."""
        info = GgufLayer()
        self._check(self.lib.moe_layer_upload_gguf(self.h, int(layer), os.fsencode(path), int(file_layer),
                                                   ctypes.byref(info)), "moe_layer_upload_gguf")
        self.descs[layer] = info.desc
        return info

    def generate_layer(self, layer: int, shape, seed: int, e_lo: int = 124, e_span: int = 7):
        d = LayerDesc.of(shape)
        self._check(self.lib.moe_layer_generate(self.h, layer, ctypes.byref(d), seed, e_lo, e_span),
                    "moe_layer_generate")
        self.descs[layer] = d

    def read_blocks(self, layer: int, tensor: int, expert: int) -> np.ndarray:
        d = self.descs[layer]
        rows, K = (d.ffn, d.hidden) if tensor in (T_GATE, T_UP) else (d.hidden, d.ffn)
        out = np.empty((rows, K // 32, 17), np.uint8)
        self._check(self.lib.moe_layer_read_blocks(self.h, layer, tensor, expert, out.ctypes.data),
                    "moe_layer_read_blocks")
        return out

    def release_layer(self, layer: int):
        self._check(self.lib.moe_layer_release(self.h, layer), "moe_layer_release")
        self.descs.pop(layer, None)

    def layer_bytes(self, layer: int) -> int:
        v = ctypes.c_uint64()
        self._check(self.lib.moe_layer_bytes(self.h, layer, ctypes.byref(v)), "moe_layer_bytes")
        return int(v.value)

    # -- per call (torch device tensors) ---------------------------------------
    def route(self, logits, k: int, mode: int, norm: bool, scale: float, ids, wts, bias=None, stream=None):
        check_tensor(logits, "logits", "float32", (None, None))
        T, E = logits.shape
        check_tensor(ids, "ids", "int32", (T, k))
        check_tensor(wts, "wts", "float32", (T, k))
        if bias is not None:
            check_tensor(bias, "bias", "float32", (E,))
        self._check(self.lib.moe_route(self.h, _ptr(logits), _ptr(bias), T, E, k, mode, int(norm), scale,
                                       _ptr(ids), _ptr(wts), _stream(stream)), "moe_route")

    def router_logits(self, w, x, logits, w_type: int = 0, stream=None):
        """logits [T][E] = x [T][H] . w [E][H]^T (f32 device tensors); w_type:
        the ggml type w was widened from (GGML_F32 / GGML_F16 / GGML_BF16: x
        is rounded to it first, as ggml-cpu's mul_mat does)."""
        check_tensor(x, "x", "float32", (None, None))
        T, H = x.shape
        check_tensor(w, "w", "float32", (None, H))
        E = w.shape[0]
        check_tensor(logits, "logits", "float32", (T, E))
        self._check(self.lib.moe_router_logits(self.h, _ptr(w), _ptr(x), T, E, H, w_type, _ptr(logits),
                                               _stream(stream)),
                    "moe_router_logits")

    def group(self, ids, E: int, counts, offsets, perm, inv=None, stream=None):
        check_tensor(ids, "ids", "int32", (None, None))
        T, k = ids.shape
        check_tensor(counts, "counts", "int32", (E,))
        check_tensor(offsets, "offsets", "int32", (E + 1,))
        check_tensor(perm, "perm", "int32", (T * k,))
        if inv is not None:
            check_tensor(inv, "inv", "int32", (T * k,))
        self._check(self.lib.moe_group(self.h, _ptr(ids), T, k, E, _ptr(counts), _ptr(offsets), _ptr(perm),
                                       _ptr(inv), _stream(stream)), "moe_group")

    def forward(self, layer: int, x, ids, wts, out, flags: int = 0, stream=None):
        T = check_forward_args(self.descs.get(layer), x, ids, wts, out, flags)
        self._check(self.lib.moe_forward(self.h, layer, _ptr(x), _ptr(ids), _ptr(wts), T, _ptr(out), flags,
                                         _stream(stream)), "moe_forward")

    def forward_noalloc(self, layer: int, x, ids, wts, out, flags: int = 0, stream=None):
        """moe_forward_noalloc: the same block with the per-call buffers in the
        library's file-scope device scratch (no allocation)."""
        T = check_forward_args(self.descs.get(layer), x, ids, wts, out, flags)
        self._check(self.lib.moe_forward_noalloc(self.h, layer, _ptr(x), _ptr(ids), _ptr(wts), T, _ptr(out), flags,
                                                 _stream(stream)), "moe_forward_noalloc")

    def route_forward(self, layer: int, x, logits, ids, wts, out, mode: int, norm: bool = True,
                      scale: float = 1.0, bias=None, flags: int = 0, stream=None):
        d = self.descs.get(layer)
        T = check_forward_args(d, x, ids, wts, out, flags)
        check_tensor(logits, "logits", "float32", (T, d.n_expert) if d is not None else (T, None))
        if bias is not None:
            check_tensor(bias, "bias", "float32", (logits.shape[1],))
        self._check(self.lib.moe_route_forward(self.h, layer, _ptr(x), _ptr(logits), _ptr(bias), T, mode,
                                               int(norm), scale, _ptr(ids), _ptr(wts), _ptr(out), flags,
                                               _stream(stream)), "moe_route_forward")

    # -- around the expert products (torch device tensors) ------------------------
    # moe_torch compares a call's tensors with what it needs and makes it; the checks
    # that name what is wrong run only where it returns None.  Buffers that overlap are
    # refused by the library.
    def _on_device(self, *named):
        for t, name in named:
            if t is not None and t.get_device() != self.device:
                raise ValueError(f"{name}: on {t.device}, expected this context's ROCm device (cuda:{self.device})")
            if t is not None and max(t.shape) > 2 ** 31 - 1:
                raise ValueError(f"{name}: shape {tuple(t.shape)}, at most 2^31 - 1 along each")

    def dispatch(self, x, inv, rows, stream=None):
        """rows[inv[t*k+s]] = x[t]: tokens' rows [T, H] to expert order
        [n_rows, H]; inv from group(); rows no pair names stay as they were."""
        st = self._calls and _torch_calls.dispatch(self._calls, self.h, self.device, x, inv, rows, stream)
        if st is None:
            xt = check_rows("x", x)
            T, H = x.shape
            rt = check_rows("rows", rows, None, H)
            k, R = check_pairs(inv, T), rows.shape[0]
            self._on_device((x, "x"), (inv, "inv"), (rows, "rows"))
            st = self.lib.moe_dispatch(self.h, x.data_ptr(), xt, inv.data_ptr(), T, k, H, R, rows.data_ptr(), rt,
                                       _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_dispatch")

    def dispatch_grad(self, drows, inv, dx, stream=None):
        """dx[t] = sum over s of drows[inv[t*k+s]]."""
        st = self._calls and _torch_calls.dispatch_grad(self._calls, self.h, self.device, drows, inv, dx, stream)
        if st is None:
            xt = check_rows("dx", dx)
            T, H = dx.shape
            rt = check_rows("drows", drows, None, H)
            k, R = check_pairs(inv, T), drows.shape[0]
            self._on_device((drows, "drows"), (inv, "inv"), (dx, "dx"))
            st = self.lib.moe_dispatch_grad(self.h, drows.data_ptr(), rt, R, inv.data_ptr(), T, k, H, dx.data_ptr(), xt,
                                            _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_dispatch_grad")

    def combine(self, rows, wts, inv, out, stream=None):
        """out[t] = sum over s of wts[t, s] * rows[inv[t*k+s]]: expert rows
        [n_rows, H] back in token order [T, H], weighted."""
        st = self._calls and _torch_calls.combine(self._calls, self.h, self.device, rows, wts, inv, out, stream)
        if st is None:
            ot = check_rows("out", out)
            T, H = out.shape
            rt = check_rows("rows", rows, None, H)
            k, R = check_pairs(inv, T), rows.shape[0]
            check_tensor(wts, "wts", "float32", (T, k), device=False)
            self._on_device((rows, "rows"), (wts, "wts"), (inv, "inv"), (out, "out"))
            st = self.lib.moe_combine(self.h, rows.data_ptr(), rt, R, wts.data_ptr(), inv.data_ptr(), T, k, H,
                                      out.data_ptr(), ot,
                                      _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_combine")

    def combine_grad(self, dout, rows, wts, inv, drows, dwts, stream=None):
        """combine's gradient: drows[inv[t*k+s]] = wts[t, s] * dout[t] and
        dwts[t, s] = <dout[t], rows[inv[t*k+s]]> (0 for a dropped pair)."""
        st = self._calls and _torch_calls.combine_grad(self._calls, self.h, self.device, dout, rows, wts, inv, drows, dwts,
                                                       stream)
        if st is None:
            dt = check_rows("dout", dout)
            T, H = dout.shape
            rt = check_rows("rows", rows, None, H)
            R = rows.shape[0]
            if check_rows("drows", drows, R, H) != rt:
                raise ValueError(f"drows: dtype {drows.dtype}, expected rows' {rows.dtype}")
            k = check_pairs(inv, T)
            check_tensor(wts, "wts", "float32", (T, k), device=False)
            check_tensor(dwts, "dwts", "float32", (T, k), device=False)
            self._on_device((dout, "dout"), (rows, "rows"), (wts, "wts"), (inv, "inv"), (drows, "drows"), (dwts, "dwts"))
            st = self.lib.moe_combine_grad(self.h, dout.data_ptr(), dt, rows.data_ptr(), rt, R, wts.data_ptr(),
                                           inv.data_ptr(), T, k, H, drows.data_ptr(), dwts.data_ptr(),
                                           _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_combine_grad")

    def quantize_i8(self, x, q, scale, stream=None):
        """Rows x [M, K] in 8 bits: scale [M] = amax / 127, q [M, K] int8 = x /
        scale to the nearest whole number."""
        st = self._calls and _torch_calls.quantize_i8(self._calls, self.h, self.device, x, q, scale, stream)
        if st is None:
            xt = check_rows("x", x)
            M, K = x.shape
            check_tensor(q, "q", "int8", (M, K), device=False)
            check_tensor(scale, "scale", "float32", (M,), device=False)
            self._on_device((x, "x"), (q, "q"), (scale, "scale"))
            st = self.lib.moe_quantize_i8(self.h, x.data_ptr(), xt, M, K, q.data_ptr(), scale.data_ptr(),
                                          _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_quantize_i8")

    def matmul_i8(self, q, scale, w, w_scale, out, offsets=None, perm=None, k: int = 1, swiglu: bool = False,
                  clamp: float = 0.0, stream=None):
        """out[r, n] = (sum of q[src, i] * w[e, n, i]) * scale[src] * w_scale[e, n].
        Dense: w [N, K], out [M, N] for q [M, K].  Grouped: w [E, N, K], rows
        offsets[e] .. offsets[e+1] are expert e's (offsets [E + 1] and perm from
        group(): row r's codes are those of token perm[r] // k; without perm, of
        row r).  swiglu: the channels are N/2 of gate and N/2 of up, and out
        [M, N/2] is silu(gate) * up, clamped as LayerDesc.clamp says."""
        st = self._calls and _torch_calls.matmul_i8(self._calls, self.h, self.device, q, scale, w, w_scale, out, offsets,
                                                    perm, k, swiglu, clamp, stream)
        if st is None:
            grouped = offsets is not None
            check_tensor(q, "q", "int8", (None, None), device=False)
            S, K = q.shape
            check_tensor(w, "w", "int8", (None, None, K) if grouped else (None, K), device=False)
            E, N = (w.shape[0], w.shape[1]) if grouped else (1, w.shape[0])
            check_tensor(scale, "scale", "float32", (S,), device=False)
            check_tensor(w_scale, "w_scale", "float32", (E, N) if grouped else (N,), device=False)
            if swiglu and N % 2:
                raise ValueError(f"w: {N} channels are not gate and up of one width")
            ot = check_rows("out", out, None, N // 2 if swiglu else N)
            M = out.shape[0]
            if S * K * N * E == 0:
                raise ValueError(f"w: shape {tuple(w.shape)} for q of {tuple(q.shape)}: empty")
            if grouped:
                check_tensor(offsets, "offsets", "int32", (E + 1,), device=False)
            if perm is not None:
                check_tensor(perm, "perm", "int32", (M,), device=False)
            elif k != 1 or S != M:
                raise ValueError(f"out: {M} rows for {S} rows of q without perm (k = {k})")
            self._on_device((q, "q"), (scale, "scale"), (w, "w"), (w_scale, "w_scale"), (out, "out"),
                            (offsets, "offsets"), (perm, "perm"))
            st = self.lib.moe_matmul_i8(self.h, q.data_ptr(), scale.data_ptr(), S, w.data_ptr(), w_scale.data_ptr(), E,
                                        None if offsets is None else offsets.data_ptr(),
                                        None if perm is None else perm.data_ptr(), int(k), M, N, K, 1 if swiglu else 0,
                                        clamp, out.data_ptr(), ot,
                                        _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_matmul_i8")

    # -- on the way into the experts and beside them (torch device tensors) -------
    def rms_norm(self, x, w, eps: float, residual=None, total=None, y=None, q=None, scale=None, rstd=None, stream=None):
        """Norm of rows x [T, H]: y = h * r * w with r = (mean h^2 + eps)^-1/2, w
        [H].  With residual [T, H], h = x + residual, rounded to its type and
        written to total (of that type; residual itself: in place), else h = x.
        q, scale: y in 8 bits as quantize_i8 writes rows (y, q and scale, or
        both); rstd [T] float32 takes r, for the gradient."""
        st = self._calls and _torch_calls.rms_norm(self._calls, self.h, self.device, x, w, eps, residual, total, y, q, scale,
                                                   rstd, stream)
        if st is None:
            xt = check_rows("x", x)
            T, H = x.shape
            wt = check_gain(w, H)
            if (residual is None) != (total is None):
                raise ValueError("residual and total: both or neither")
            if (q is None) != (scale is None):
                raise ValueError("q and scale: both or neither")
            if y is None and q is None:
                raise ValueError("y, or q and scale: at least one output")
            rt = yt = 0
            if residual is not None:
                rt = check_rows("residual", residual, T, H)
                if check_rows("total", total, T, H) != rt:
                    raise ValueError(f"total: dtype {total.dtype}, expected residual's {residual.dtype}")
            if y is not None:
                yt = check_rows("y", y, T, H)
            if q is not None:
                check_tensor(q, "q", "int8", (T, H), device=False)
                check_tensor(scale, "scale", "float32", (T,), device=False)
            if rstd is not None:
                check_tensor(rstd, "rstd", "float32", (T,), device=False)
            self._on_device((x, "x"), (w, "w"), (residual, "residual"), (total, "total"), (y, "y"), (q, "q"),
                            (scale, "scale"), (rstd, "rstd"))
            st = self.lib.moe_rms_norm(self.h, _ptr(x), xt, _ptr(residual), _ptr(total), rt, _ptr(w), wt, eps, T, H,
                                       _ptr(y), yt, _ptr(q), _ptr(scale), _ptr(rstd),
                                       _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_rms_norm")

    def rms_norm_grad_scratch(self, T: int, H: int) -> int:
        """Floats of rms_norm_grad's part for T rows of H and for every smaller call."""
        return int(self.lib.moe_rms_norm_grad_scratch(self.h, T, H))

    def rms_norm_grad(self, dy, h, w, rstd, dx, dw, part, dres=None, stream=None):
        """rms_norm's gradient, h what was normalised (total, or x) and rstd its r:
        with u = h * r and g = dy * w, dx = r * (g - u * mean(g * u)) + dres (the
        gradient of x and of residual; dres, of dx's type, may be dx itself)
        and dw [H] float32 = sum over the rows of dy * u.  part: float32, a
        workspace of rms_norm_grad_scratch(T, H) values."""
        st = self._calls and _torch_calls.rms_norm_grad(self._calls, self.h, self.device, dy, h, w, rstd, dx, dw, part, dres,
                                                        stream)
        if st is None:
            dt = check_rows("dy", dy)
            T, H = dy.shape
            ht, wt, xt = check_rows("h", h, T, H), check_gain(w, H), check_rows("dx", dx, T, H)
            check_tensor(rstd, "rstd", "float32", (T,), device=False)
            check_tensor(dw, "dw", "float32", (H,), device=False)
            check_tensor(part, "part", "float32", (None,), device=False)
            if dres is not None and check_rows("dres", dres, T, H) != xt:
                raise ValueError(f"dres: dtype {dres.dtype}, expected dx's {dx.dtype}")
            self._on_device((dy, "dy"), (h, "h"), (w, "w"), (rstd, "rstd"), (dx, "dx"), (dw, "dw"), (part, "part"),
                            (dres, "dres"))
            st = self.lib.moe_rms_norm_grad(self.h, _ptr(dy), dt, _ptr(h), ht, _ptr(w), wt, _ptr(rstd), _ptr(dres), T, H,
                                            _ptr(dx), xt, _ptr(dw), _ptr(part), part.numel(),
                                            _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_rms_norm_grad")

    def route_groups(self, logits, k: int, mode: int, norm: bool, scale: float, ids, wts, bias=None, n_group: int = 1,
                     keep: int = 1, top: int = 2, scores=None, stream=None):
        """route() for logits [T, E] of any row type, with groups: the experts
        stand in n_group groups of E / n_group, the keep groups stay whose top
        (1 or 2) best experts sum to most, and the k best of theirs are picked.  An
        expert whose logit is -inf is masked: a slot that finds no other
        has id -1 (group() drops the pair) and weight 0.  scores [T, E]
        float32: the scores as well."""
        st = self._calls and _torch_calls.route_groups(self._calls, self.h, self.device, logits, k, mode, norm, scale, ids,
                                                       wts, bias, n_group, keep, top, scores, stream)
        if st is None:
            lt = check_rows("logits", logits)
            T, E = logits.shape
            check_tensor(ids, "ids", "int32", (T, k), device=False)
            check_tensor(wts, "wts", "float32", (T, k), device=False)
            if bias is not None:
                check_tensor(bias, "bias", "float32", (E,), device=False)
            if scores is not None:
                check_tensor(scores, "scores", "float32", (T, E), device=False)
            self._on_device((logits, "logits"), (ids, "ids"), (wts, "wts"), (bias, "bias"), (scores, "scores"))
            st = self.lib.moe_route_groups(self.h, _ptr(logits), lt, _ptr(bias), T, E, int(k), mode, n_group, keep, top,
                                           int(norm), scale, _ptr(ids), _ptr(wts), _ptr(scores),
                                           _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_route_groups")

    def route_grad(self, logits, ids, dwts, mode: int, norm: bool, scale: float, dlogits, dscores=None, stream=None):
        """The logits' gradient dlogits [T, E] of route_groups, from dwts [T, k] (of
        the weights of the experts ids; a slot outside [0, E) takes no part) and
        dscores [T, E] (of the scores; None: 0), both float32."""
        st = self._calls and _torch_calls.route_grad(self._calls, self.h, self.device, logits, ids, dwts, mode, norm, scale,
                                                     dlogits, dscores, stream)
        if st is None:
            lt = check_rows("logits", logits)
            T, E = logits.shape
            dt = check_rows("dlogits", dlogits, T, E)
            check_tensor(ids, "ids", "int32", (T, None), device=False)
            k = ids.shape[1]
            check_tensor(dwts, "dwts", "float32", (T, k), device=False)
            if dscores is not None:
                check_tensor(dscores, "dscores", "float32", (T, E), device=False)
            self._on_device((logits, "logits"), (ids, "ids"), (dwts, "dwts"), (dlogits, "dlogits"), (dscores, "dscores"))
            st = self.lib.moe_route_grad(self.h, _ptr(logits), lt, _ptr(ids), _ptr(dwts), _ptr(dscores), T, E, k, mode,
                                         int(norm), scale, _ptr(dlogits), dt,
                                         _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_route_grad")

    def adapters_scratch(self, M: int, K: int, R: int) -> int:
        """Floats of adapters' mid for M rows of K and rank R and for every smaller call."""
        return int(self.lib.moe_adapters_scratch(self.h, M, K, R))

    def adapters(self, x, a, b, scale, offsets, perm, base, out, mid, stream=None):
        """out[r] = base[r] + scale[i] * b[i] (a[i] x[r]) for the rows r of adapter i:
        x [M, K], a [n, R, K] and b [n, N, R] of one row type, base and out [M, N] of one
        (out may be base), scale [n] float32 or None (1).  offsets [n + 1] and perm [M]
        group the rows by adapter, from group() with the rows' adapters as [M, 1] ids
        (-1: none; such a row of out stays as it was).  mid: float32, a workspace
        of adapters_scratch(M, K, R) values."""
        st = self._calls and _torch_calls.adapters(self._calls, self.h, self.device, x, a, b, scale, offsets, perm, base, out,
                                                   mid, stream)
        if st is None:
            xt = check_rows("x", x)
            M, K = x.shape
            dt = str(x.dtype).replace("torch.", "")
            check_tensor(a, "a", dt, (None, None, K), device=False)
            n, R = a.shape[0], a.shape[1]
            check_tensor(b, "b", dt, (n, None, R), device=False)
            N = b.shape[1]
            if n * R * N == 0:
                raise ValueError(f"a, b: shapes {tuple(a.shape)}, {tuple(b.shape)}: empty")
            ot = check_rows("out", out, M, N)
            if check_rows("base", base, M, N) != ot:
                raise ValueError(f"base: dtype {base.dtype}, expected out's {out.dtype}")
            if scale is not None:
                check_tensor(scale, "scale", "float32", (n,), device=False)
            check_tensor(offsets, "offsets", "int32", (n + 1,), device=False)
            check_tensor(perm, "perm", "int32", (M,), device=False)
            check_tensor(mid, "mid", "float32", (None,), device=False)
            self._on_device((x, "x"), (a, "a"), (b, "b"), (scale, "scale"), (offsets, "offsets"), (perm, "perm"),
                            (base, "base"), (out, "out"), (mid, "mid"))
            st = self.lib.moe_adapters(self.h, _ptr(x), _ptr(a), _ptr(b), xt, _ptr(scale), n, _ptr(offsets), _ptr(perm),
                                       M, K, R, N, _ptr(base), _ptr(out), ot, _ptr(mid), mid.numel(),
                                       _device_stream(self.device) if stream is None else int(stream))
        if st:
            self._check(st, "moe_adapters")

    def split_compute(self, nodes):
        """Compute a parsed split (moe_split_compute) into its MUL node's host data."""
        self._check(self.lib.moe_split_compute(self.h, node_list(nodes), len(nodes)), "moe_split_compute")

    def forward_host(self, layer: int, x: np.ndarray, ids: np.ndarray, wts: np.ndarray,
                     flags: int = 0) -> np.ndarray:
        d = self.descs[layer]
        x = np.ascontiguousarray(x, np.float32)
        ids = np.ascontiguousarray(ids, np.int32)
        wts = np.ascontiguousarray(wts, np.float32)
        T = check_host_forward_args(d, x, ids, wts)
        shape = (T, d.n_used, d.hidden) if flags & MOE_FWD_PER_SLOT else (T, d.hidden)
        out = np.empty(shape, np.float32)
        self._check(self.lib.moe_forward_host(self.h, layer, x.ctypes.data, ids.ctypes.data, wts.ctypes.data,
                                              T, out.ctypes.data, flags), "moe_forward_host")
        return out

    def graph_capture(self, layers, xs, ids, wts, outs, flags: int = 0) -> Graph:
        n = len(layers)
        if n == 0 or not (len(xs) == len(ids) == len(wts) == len(outs) == n):
            raise ValueError("graph_capture: one x/ids/wts/out per layer")
        T = xs[0].shape[0]
        for i in range(n):
            if check_forward_args(self.descs.get(layers[i]), xs[i], ids[i], wts[i], outs[i], flags) != T:
                raise ValueError(f"graph_capture: layer {i} has {xs[i].shape[0]} tokens, expected {T}")
        la = (ctypes.c_int * n)(*layers)
        mk = lambda ts: (_vp * n)(*[_ptr(t) for t in ts])  # noqa: E731
        px, pi, pw, po = mk(xs), mk(ids), mk(wts), mk(outs)
        g = _vp()
        self._check(self.lib.moe_graph_capture(self.h, n, la, px, pi, pw, po, T, flags, ctypes.byref(g)),
                    "moe_graph_capture")
        return Graph(self, g.value, (xs, ids, wts, outs))

    # -- profiling ----------------------------------------------------------------
    def prof_enable(self, on: bool = True):
        self._check(self.lib.moe_prof_enable(self.h, int(on)), "moe_prof_enable")

    def prof_read(self, reset: bool = True) -> dict:
        """{kernel class: (launches, total_us)} since the last reset."""
        cap = 32
        arr = (KernelStat * cap)()
        n = ctypes.c_int()
        self._check(self.lib.moe_prof_read(self.h, arr, cap, ctypes.byref(n), int(reset)), "moe_prof_read")
        return {arr[i].name.decode(): (int(arr[i].launches), float(arr[i].total_us)) for i in range(min(n.value, cap))}

    def call_stats(self, reset: bool = False) -> dict:
        """Engagement and phase counters of the host-boundary calls (moe_call_stats_read)."""
        cs = CallStats()
        self._check(self.lib.moe_call_stats_read(self.h, ctypes.byref(cs), int(reset)), "moe_call_stats_read")
        return {n: getattr(cs, n) for n, _ in CallStats._fields_}

    # -- test hooks -------------------------------------------------------------
    def set_taps(self, on: bool = True):
        self._check(self.lib.moe_debug_set_taps(self.h, int(on)), "moe_debug_set_taps")
    def debug_quantize_q8_0(self, x, qs, d, stream=None):
        check_tensor(x, "x", "float32")
        n = x.numel()
        check_tensor(qs, "qs", "int8", (n,) if qs.dim() == 1 else tuple(x.shape))
        if d.numel() != n // 32 or d.element_size() != 2:
            raise ValueError("d: expected n/32 16-bit scales")
        check_tensor(d, "d", str(d.dtype).replace("torch.", ""))
        self._check(self.lib.moe_debug_quantize_q8_0(self.h, _ptr(x), x.numel(), _ptr(qs), _ptr(d),
                                                     _stream(stream)), "moe_debug_quantize_q8_0")

    def debug_wave_sum(self, x, out, stream=None):
        check_tensor(x, "x", "float32")
        if x.numel() % 64 or out.numel() < x.numel() // 64:
            raise ValueError("debug_wave_sum: x of 64*n floats, out of n")
        check_tensor(out, "out", "float32")
        self._check(self.lib.moe_debug_wave_sum(self.h, _ptr(x), x.numel() // 64, _ptr(out), _stream(stream)),
                    "moe_debug_wave_sum")

    def debug_last_h(self, cap: int) -> np.ndarray:
        buf = np.empty(cap, np.float32)
        n = ctypes.c_size_t()
        self._check(self.lib.moe_debug_last_h(self.h, buf.ctypes.data, cap, ctypes.byref(n)), "moe_debug_last_h")
        return buf[: n.value]

    def set_timeline(self, on: bool = True):
        self._check(self.lib.moe_debug_set_timeline(self.h, int(on)), "moe_debug_set_timeline")

    def read_timeline(self):
        """The last eager decode call's per-wave stamps (100 MHz clock ticks):
        (gate_up [n, 3], down [n, 3]) uint64, columns entry / K-loop end / exit."""
        buf = np.empty(3 * 8192, np.uint64)
        ng, nd = ctypes.c_size_t(), ctypes.c_size_t()
        self._check(self.lib.moe_debug_read_timeline(self.h, buf.ctypes.data, buf.size, ctypes.byref(ng),
                                                     ctypes.byref(nd)), "moe_debug_read_timeline")
        st = buf[: 3 * (ng.value + nd.value)].reshape(-1, 3)
        return st[: ng.value].copy(), st[ng.value:].copy()


class MoeServer:
    """nano-glm moe-server protocol v2 served from the MoE block
    (moe_server_open / handle / listen / serve)."""

    def __init__(self, gguf_path: str, device: int = 0, budget_bytes: int = 2 ** 64 - 1,
                 lib_path: str | None = None):
        self.lib = load_library(lib_path)
        h = _vp()
        err = ctypes.create_string_buffer(512)
        st = self.lib.moe_server_open(os.fsencode(gguf_path), device, budget_bytes, ctypes.byref(h), err, len(err))
        if st != MOE_OK:
            raise MoeError(st, f"moe_server_open: {self.lib.moe_status_str(st).decode()}: "
                               f"{err.value.decode(errors='replace')}")
        self.h = h.value

    def close(self):
        if getattr(self, "h", None):
            self.lib.moe_server_close(self.h)
            self.h = None

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st: int, what: str):
        if st != MOE_OK:
            msg = self.lib.moe_server_last_error(self.h).decode() if self.h else ""
            raise MoeError(st, f"{what}: {self.lib.moe_status_str(st).decode()}: {msg}")

    def handle(self, msg: bytes) -> bytes:
        """One whole message in, the whole response out."""
        n = ctypes.c_size_t()
        cap = 1 << 16
        while True:
            buf = ctypes.create_string_buffer(cap)
            st = self.lib.moe_server_handle(self.h, msg, len(msg), buf, cap, ctypes.byref(n))
            if st == MOE_OK:
                return buf.raw[: n.value]
            if st == MOE_ERR_INVALID_ARG and n.value > cap:
                cap = n.value
                continue
            self._check(st, "moe_server_handle")

    def listen(self, host: str = "127.0.0.1", port: int = 0) -> int:
        """Bind; returns the port (port 0 = any free one)."""
        bound = ctypes.c_int()
        self._check(self.lib.moe_server_listen(self.h, host.encode(), port, ctypes.byref(bound)), "moe_server_listen")
        return bound.value

    def serve(self, max_connections: int = -1):
        """Serve connections one at a time (blocks; ctypes releases the GIL)."""
        self._check(self.lib.moe_server_serve(self.h, max_connections), "moe_server_serve")

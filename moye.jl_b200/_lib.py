"""ctypes binding of libmoye_b200 (the C ABI declared in include/moye_b200.h).

The shared library is built in-tree (``moye.jl_b200/lib/libmoye_b200.so``) by
``build.py``.  There is no CPU fallback: if the library is missing, or no sm_100 device is
visible when a handle is requested, the call raises.
"""
import ctypes
import importlib.machinery
import importlib.util
import os
import struct
import threading

from .build import calls_marker

MAX_RANK = 4
MAX_FLAT_RANK = 12

# moye_dtype_t
F32, F16, BF16, S8, U8, E4M3, S32, U16, U32, U64, U128 = range(11)
DTYPE_BYTES = {F32: 4, F16: 2, BF16: 2, S8: 1, U8: 1, E4M3: 1, S32: 4, U16: 2, U32: 4, U64: 8, U128: 16}

COPY_AUTO, COPY_UNIVERSAL128, COPY_TMA, COPY_TRANSPOSE = 0, 1, 2, 3
COPY_LDSM = 100  # host-side tag of the ldmatrix tiled copy (its own entry point, moye_b200_ldsm_copy)

STATUS_NAMES = {
    0: "OK", -1: "INVALID_ARG", -2: "UNSUPPORTED_DTYPE", -3: "UNSUPPORTED_LAYOUT", -4: "UNSUPPORTED_SHAPE",
    -5: "MISALIGNED", -6: "CUDA", -7: "TIMEOUT", -8: "NO_DEVICE", -9: "TOO_LARGE", -10: "NCCL",
}


class MoyeError(RuntimeError):
    """A non-zero return code from the C ABI (code + the library's message)."""

    def __init__(self, code, message):
        super().__init__(f"libmoye_b200: {STATUS_NAMES.get(code, code)}: {message}")
        self.code = code


class Tensor(ctypes.Structure):
    _fields_ = [("ptr", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("rank", ctypes.c_int32),
                ("shape", ctypes.c_int64 * MAX_RANK), ("stride", ctypes.c_int64 * MAX_RANK)]


class FlatLayout(ctypes.Structure):
    _fields_ = [("rank", ctypes.c_int32), ("reserved", ctypes.c_int32),
                ("shape", ctypes.c_int64 * MAX_FLAT_RANK), ("stride", ctypes.c_int64 * MAX_FLAT_RANK)]


class GemmParams(ctypes.Structure):
    _fields_ = [("alpha", ctypes.c_float), ("beta", ctypes.c_float), ("scale_a", ctypes.c_float),
                ("scale_b", ctypes.c_float), ("tile_n", ctypes.c_int32), ("split_k", ctypes.c_int32),
                ("path", ctypes.c_int32), ("flags", ctypes.c_int32), ("bias", ctypes.c_void_p)]


# fused-epilogue selectors of GemmParams.flags (MOYE_EPI_* in the header)
EPI_ACT = {None: 0, "none": 0, "relu": 1, "gelu": 2, "silu": 3}
EPI_BIAS_COL, EPI_BIAS_ROW = 0x10, 0x20
# kernel-choice bits of GemmParams.flags (MOYE_GEMM_* in the header)
GEMM_TAIL_OFF, GEMM_TAIL_ON, GEMM_ALLOW_TF32 = 0x100, 0x200, 0x400


class CopyParams(ctypes.Structure):
    _fields_ = [("mode", ctypes.c_int32), ("tile_m", ctypes.c_int32), ("tile_n", ctypes.c_int32),
                ("flags", ctypes.c_int32)]


# MOYE_B200_DEBUG=1 selects the debug build of the same library (`build.py --debug`): identical entry points, with
# the kernels' address arithmetic checked on the device (a violation is reported through moye_b200_status).
LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib",
                        "libmoye_b200_debug.so" if os.environ.get("MOYE_B200_DEBUG") == "1" else "libmoye_b200.so")

EXPORTS = {
    "moye_b200_create": (ctypes.c_int, [ctypes.POINTER(ctypes.c_void_p)]),
    "moye_b200_destroy": (ctypes.c_int, [ctypes.c_void_p]),
    "moye_b200_version": (ctypes.c_int, []),
    "moye_b200_last_error": (ctypes.c_char_p, []),
    "moye_b200_status": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int32)]),
    "moye_b200_selftest_bounded_wait": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "moye_b200_selftest_dirty_tickets": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "moye_b200_gemm": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(Tensor), ctypes.POINTER(Tensor),
                                      ctypes.POINTER(Tensor), ctypes.POINTER(Tensor), ctypes.POINTER(GemmParams),
                                      ctypes.c_void_p]),
    "moye_b200_copy": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(Tensor), ctypes.POINTER(Tensor),
                                      ctypes.POINTER(CopyParams), ctypes.c_void_p]),
    "moye_b200_layout_copy": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(FlatLayout),
                                             ctypes.c_void_p, ctypes.POINTER(FlatLayout), ctypes.c_int32,
                                             ctypes.c_void_p]),
    "moye_b200_gemm_skinny_static": (ctypes.c_int, [ctypes.POINTER(Tensor), ctypes.POINTER(Tensor),
                                                    ctypes.POINTER(Tensor), ctypes.c_float, ctypes.c_void_p,
                                                    ctypes.c_void_p]),
    "moye_b200_gemm_skinny_static_status": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_int32)]),
    "moye_b200_axpby": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(Tensor), ctypes.POINTER(Tensor), ctypes.c_float,
                                       ctypes.c_float, ctypes.c_void_p]),
    "moye_b200_comm_unique_id": (ctypes.c_int, [ctypes.c_char_p]),
    "moye_b200_comm_init": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_char_p]),
    "moye_b200_comm_destroy": (ctypes.c_int, [ctypes.c_void_p]),
    "moye_b200_allgather": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(Tensor), ctypes.POINTER(Tensor),
                                           ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p]),
    "moye_b200_bcast": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(Tensor), ctypes.c_int32, ctypes.c_void_p]),
    "moye_b200_ldsm_copy": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32,
                                           ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                           ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(ctypes.c_int32), ctypes.c_void_p]),
    # descriptors of the row-group calls are packed bytes (see pack_tensor), hence plain pointers
    "moye_b200_group_rows": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32] + [ctypes.c_void_p] * 4),
    "moye_b200_gather_rows": (ctypes.c_int, [ctypes.c_void_p] * 4 + [ctypes.c_int32, ctypes.c_void_p]),
    "moye_b200_combine_rows": (ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_int32, ctypes.c_void_p]),
    "moye_b200_combine_rows_grad": (ctypes.c_int, [ctypes.c_void_p] * 7 + [ctypes.c_int32, ctypes.c_void_p]),
    "moye_b200_gemm_grouped": (ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_float, ctypes.c_float, ctypes.c_void_p]),
    "moye_b200_gemm_grouped_grad": (ctypes.c_int, [ctypes.c_void_p] * 5 + [ctypes.c_float, ctypes.c_float, ctypes.c_void_p]),
    "moye_b200_gemm_lora": (ctypes.c_int, [ctypes.c_void_p] * 8 + [ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p]),
    "moye_b200_layout_eval": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(FlatLayout), ctypes.c_int64,
                                             ctypes.c_int64, ctypes.c_void_p, ctypes.c_void_p]),
}

_lib = None
_handles = {}  # (thread, device) -> handle
calls = None  # the compiled module of the row-group calls, bound to the loaded library
_lock = threading.Lock()


def load():
    """dlopen the in-tree library and type its exports.  Raises if it has not been built."""
    global _lib, calls
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise FileNotFoundError(
                    f"{LIB_PATH} is missing: build it with `python moye.jl_b200/build.py` "
                    "(there is no fallback implementation)")
            lib = ctypes.CDLL(LIB_PATH)
            for name, (res, args) in EXPORTS.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            calls = _load_calls(lib)
            _lib = lib
    return _lib


def _load_calls(lib):
    """csrc/calls.cpp, bound to the entry points of `lib`.  None where it was not built, or for another torch, interpreter
    or version of the library than the ones that run: the calls then take the way through ctypes into the same entry
    points, at more of the host's time."""
    path = os.path.join(os.path.dirname(LIB_PATH), "moye_calls.so")
    try:
        with open(path, "rb") as f:
            if calls_marker(lib.moye_b200_version()) not in f.read():
                return None
        import torch  # noqa: F401  the module's own libraries
        loader = importlib.machinery.ExtensionFileLoader("moye_calls", path)
        mod = importlib.util.module_from_spec(importlib.util.spec_from_file_location("moye_calls", path, loader=loader))
        loader.exec_module(mod)
    except (ImportError, OSError):
        return None
    names = ("group_rows", "gather_rows", "combine_rows", "combine_rows_grad", "gemm_grouped", "gemm_grouped_grad", "gemm_lora")
    mod.bind(tuple(ctypes.cast(getattr(lib, "moye_b200_" + n), ctypes.c_void_p).value for n in names), _handles)
    return mod


def check(rc):
    if rc != 0:
        raise MoyeError(rc, load().moye_b200_last_error().decode())


def handle(device=None):
    """The per-(thread, device) library handle, created on first use with `device` current."""
    import torch
    if device is None:
        device = torch.cuda.current_device()
    key = (threading.get_ident(), int(device))
    h = _handles.get(key)
    if h is None:
        lib = load()
        out = ctypes.c_void_p()
        with torch.cuda.device(device):
            check(lib.moye_b200_create(ctypes.byref(out)))
        h = out
        _handles[key] = h
    return h


def make_tensor(ptr, dtype, shape, stride):
    t = Tensor()
    t.ptr = ptr
    t.dtype = dtype
    t.rank = len(shape)
    for i, (s, d) in enumerate(zip(shape, stride)):
        t.shape[i] = s
        t.stride[i] = d
    return t


# one packer per rank: pointer, type, rank, shape and strides, the unused modes zero
TENSOR_PACKERS = [None] + [struct.Struct(f"<Qii{r}q{8 * (MAX_RANK - r)}x{r}q{8 * (MAX_RANK - r)}x") for r in range(1, MAX_RANK + 1)]


def pack_tensor(ptr, dtype, shape, stride):
    """`make_tensor` as the bytes of a moye_tensor_t, which a call takes by pointer: a third of the cost of filling the
    ctypes structure, for entry points whose descriptors are made anew on every call."""
    return TENSOR_PACKERS[len(shape)].pack(ptr, dtype, len(shape), *shape, *stride)


def make_flat_layout(shape, stride):
    l = FlatLayout()
    l.rank = len(shape)
    for i, (s, d) in enumerate(zip(shape, stride)):
        l.shape[i] = s
        l.stride[i] = d
    return l

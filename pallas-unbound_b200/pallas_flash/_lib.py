"""ctypes binding of libpu_attn.so — the C ABI declared in include/pu_attn.h.

This is the Python side of the drop-in boundary: every compute call of the
package goes through these symbols.  There is no fallback: if the library
is missing or cannot load, `lib()` raises.
"""
from __future__ import annotations

import ctypes
import os
import struct
import threading
from pathlib import Path

import torch

PU_OK = 0
PU_ERR_INVALID_ARGUMENT = 1
PU_ERR_UNSUPPORTED = 2
PU_ERR_CUDA = 3
PU_ERR_WORKSPACE = 4
PU_ERR_DEVICE_TIMEOUT = 5

PU_DTYPE_BF16 = 0
PU_DTYPE_F16 = 1
PU_DTYPE_F32 = 2
PU_DTYPE_FP8_E4M3 = 3

PU_COMM_ID_BYTES = 128

_LIB_PATH = Path(__file__).resolve().parent / "_native" / "libpu_attn.so"

_c_void_p = ctypes.c_void_p
_i64 = ctypes.c_int64
_int = ctypes.c_int
_float = ctypes.c_float
_size_t = ctypes.c_size_t

# name -> (restype, argtypes); mirrors include/pu_attn.h
SIGNATURES = {
    "pu_version": (ctypes.c_char_p, []),
    "pu_last_error": (ctypes.c_char_p, []),
    "pu_device_status": (_int, [ctypes.POINTER(_int)]),
    "pu_binary_arch": (_int, [ctypes.POINTER(_int)]),
    "pu_selftest_wait_timeout": (_int, [ctypes.c_uint64, _c_void_p]),
    "pu_attn_fwd": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
                           _i64, _i64, _i64, _i64, _i64, _float, _int, _c_void_p]),
    "pu_attn_bwd_workspace_size": (_size_t, [_i64, _i64, _i64, _i64]),
    "pu_attn_bwd": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
                           _c_void_p, _c_void_p, _c_void_p, _c_void_p, _size_t,
                           _i64, _i64, _i64, _i64, _i64, _float, _int, _c_void_p]),
    "pu_attn_bwd_deterministic": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
                                         _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
                                         _size_t, _i64, _i64, _i64, _i64, _i64, _float, _int,
                                         _c_void_p]),
    "pu_decode_workspace_size": (_size_t, [_i64, _i64, _i64, _i64]),
    "pu_decode_partial": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _i64,
                                 _c_void_p, _c_void_p, _size_t, _i64, _i64, _i64, _i64, _float,
                                 _c_void_p]),
    "pu_decode_combine": (_int, [_c_void_p, _i64, _c_void_p, _c_void_p, _i64, _i64, _i64,
                                 _c_void_p]),
    "pu_decode": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _c_void_p,
                         _c_void_p, _c_void_p, _size_t, _i64, _i64, _i64, _i64, _float,
                         _c_void_p]),
    "pu_decode_noalloc": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p,
                                 _c_void_p, _c_void_p, _i64, _i64, _i64, _i64, _float,
                                 _c_void_p]),
    "pu_decode_gqa_workspace_size": (_size_t, [_i64, _i64, _i64, _i64, _i64]),
    "pu_decode_gqa": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _c_void_p,
                             _c_void_p, _c_void_p, _size_t, _i64, _i64, _i64, _i64, _i64, _float,
                             _float, _float, _c_void_p]),
    "pu_decode_paged_workspace_size": (_size_t, [_i64, _i64, _i64, _i64, _i64]),
    "pu_decode_paged": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _i64,
                               _i64, _i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _size_t,
                               _i64, _i64, _i64, _float, _c_void_p]),
    "pu_peer_alloc": (_int, [_size_t, ctypes.POINTER(_c_void_p), _c_void_p]),
    "pu_peer_free": (_int, [_c_void_p]),
    "pu_peer_open": (_int, [_c_void_p, ctypes.POINTER(_c_void_p)]),
    "pu_peer_close": (_int, [_c_void_p]),
    "pu_decode_exchange_bytes": (_size_t, [_i64, _i64, _i64, _i64]),
    "pu_decode_push": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _i64,
                              _c_void_p, _i64, _i64, ctypes.c_uint32, _c_void_p, _size_t,
                              _i64, _i64, _i64, _i64, _float, _c_void_p]),
    "pu_decode_pull": (_int, [_c_void_p, _i64, ctypes.c_uint32, _c_void_p, _c_void_p, _i64,
                              _i64, _i64, ctypes.c_uint64, _c_void_p]),
    "pu_decode_sharded": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _i64,
                                 _c_void_p, _i64, _i64, ctypes.c_uint32, _c_void_p, _c_void_p,
                                 _c_void_p, _size_t, _i64, _i64, _i64, _i64, _float,
                                 ctypes.c_uint64, _c_void_p]),
    "pu_outproj_exchange_bytes": (_size_t, [_i64, _i64, _i64]),
    "pu_outproj_allreduce": (_int, [_c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64,
                                    ctypes.c_uint32, _i64, _i64, _i64, ctypes.c_uint64, _c_void_p]),
    "pu_comm_unique_id": (_int, [_c_void_p]),
    "pu_comm_init": (_int, [_c_void_p, _i64, _i64, ctypes.POINTER(_c_void_p)]),
    "pu_allgather_partials": (_int, [_c_void_p, _c_void_p, _i64, _i64, _i64, _c_void_p, _c_void_p]),
    "pu_comm_destroy": (_int, [_c_void_p]),
    "pu_decode_paged_gqa_workspace_size": (_size_t, [_i64, _i64, _i64, _i64, _i64, _i64]),
    "pu_decode_paged_gqa": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _i64,
                                   _i64, _i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _size_t,
                                   _i64, _i64, _i64, _i64, _float, _float, _float, _c_void_p]),
    "pu_decode_paged_heads": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _i64,
                                     _i64, _i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _size_t,
                                     _i64, _i64, _i64, _i64, _float, _float, _float, _c_void_p]),
    "pu_decode_paged_shared_workspace_size": (_size_t, [_i64, _i64, _i64, _i64, _i64]),
    "pu_decode_paged_shared": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _int, _c_void_p, _i64,
                                      _i64, _i64, _c_void_p, _c_void_p, _c_void_p, _i64, _c_void_p,
                                      _c_void_p, _c_void_p, _size_t, _i64, _i64, _i64, _i64, _float,
                                      _float, _float, _c_void_p]),
    "pu_page_bounds": (_int, [_c_void_p, _int, _c_void_p, _c_void_p, _i64, _i64, _i64, _i64, _i64,
                              _c_void_p]),
    "pu_select_pages": (_int, [_c_void_p, _int, _c_void_p, _int, _c_void_p, _i64, _i64, _i64, _c_void_p,
                               _c_void_p, _c_void_p, _i64, _i64, _i64, _i64, _i64, _i64, _i64,
                               _c_void_p]),
    # arguments as packed 8-byte words (PAGED_GQA and the like below)
    "pu_call_packed": (_int, [_int, _c_void_p]),
    "pu_page_plan": (_int, [_c_void_p, _c_void_p, _i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p,
                            _c_void_p, _i64, _c_void_p, _c_void_p, _i64, _c_void_p, _c_void_p,
                            _c_void_p, _c_void_p, _i64, _i64, _c_void_p]),
    "pu_page_share": (_int, [_c_void_p, _i64, _i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _i64,
                             _i64, _i64, _c_void_p]),
    "pu_page_plan_shared": (_int, [_c_void_p, _i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64, _c_void_p,
                                   _i64, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _c_void_p, _i64,
                                   _i64, _c_void_p]),
    # the description (pu_qk_rope_desc) is passed as packed bytes
    "pu_qk_norm_rope_fwd": (_int, [_c_void_p] * 6),
    "pu_qk_norm_rope_bwd_workspace_size": (_size_t, [_i64]),
    "pu_qk_norm_rope_bwd": (_int, [_c_void_p] * 10 + [_size_t, _c_void_p]),
    "pu_qk_norm_rope_append": (_int, [_c_void_p] * 8 + [_int, _i64, _i64, _float, _float, _c_void_p]),
    "pu_kv_append": (_int, [_c_void_p, _c_void_p, _int, _c_void_p, _c_void_p, _c_void_p, _i64,
                            _i64, _i64, _c_void_p, _i64, _i64, _i64, _c_void_p]),
}

# entries of pu_call_packed, and their words: whole numbers and pointers, scales as doubles
DECODE_PAGED_GQA, DECODE_PAGED_HEADS, DECODE_PAGED_SHARED, PAGE_BOUNDS, SELECT_PAGES = range(5)
pack_decode = struct.Struct("<18q3dq").pack
pack_shared = struct.Struct("<21q3dq").pack
pack_bounds = struct.Struct("<10q").pack
pack_select = struct.Struct("<19q").pack

_lock = threading.Lock()
_lib = None


class PuError(RuntimeError):
    """A nonzero status from libpu_attn (message from pu_last_error)."""

    def __init__(self, code: int, where: str, message: str):
        super().__init__(f"{where} failed with status {code}: {message}")
        self.code = code


def library_path() -> Path:
    return Path(os.environ.get("PU_ATTN_LIB", _LIB_PATH))


def lib() -> ctypes.CDLL:
    """Load (once) and return the library; raises if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            path = library_path()
            if not path.exists():
                raise RuntimeError(
                    f"libpu_attn.so not found at {path}; build it with "
                    "`python pallas-unbound_b200/build.py` (there is no CPU fallback)")
            handle = ctypes.CDLL(str(path))
            for name, (res, args) in SIGNATURES.items():
                fn = getattr(handle, name)
                fn.restype = res
                fn.argtypes = args
            _lib = handle
    return _lib


def check(code: int, where: str) -> None:
    if code != PU_OK:
        msg = lib().pu_last_error()
        raise PuError(code, where, msg.decode() if msg else "")


# handle of a device's current stream (the public call builds a Stream object
# first, which costs more than a small kernel's launch)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


_empty_strided = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)

# dispatch modes in force
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None) or (lambda: 1)


def empty(shape, strides, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A new tensor on `device`, which is current: a third of torch.empty's time for the outputs of a small call.
    That function goes past the dispatcher, so dispatch modes and the deterministic fill of new memory, which
    act there, get torch.empty_strided."""
    if _empty_strided is not None and not _modes() and not torch._C._get_deterministic_algorithms():
        return _empty_strided(shape, strides, dtype)
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


# the current device's index, without the public call's checks
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class on_device:
    """Makes `device` current where it is not and gives the handle of its
    current stream: `with on_device(t.device) as stream`."""

    __slots__ = ("index", "before")

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self) -> int:
        now = _current_device()
        if now == self.index:
            self.before = None
        else:
            self.before = now
            torch.cuda.set_device(self.index)
        return _raw_stream(self.index)

    def __exit__(self, *exc) -> None:
        if self.before is not None:
            torch.cuda.set_device(self.before)


def device_status() -> tuple[int, int]:
    """Synchronise the current device and read/clear its kernel status word."""
    detail = _int(0)
    code = lib().pu_device_status(ctypes.byref(detail))
    return code, detail.value

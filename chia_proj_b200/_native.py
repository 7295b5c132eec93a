"""ctypes binding of ``libchia_attn.so`` (declared in ``include/chia_attn.h``
and ``include/chia_paged.h``).

The library is built in-tree by ``chia_proj_b200.build`` and loaded from
``chia_proj_b200/_lib/``. There is no fallback: if the library is missing or
fails to load, importing the operators raises.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.metadata
import importlib.util
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_lib", "libchia_attn.so")

ABI_VERSION = 4
WORKSPACE_BYTES = 256
NOALLOC_SCRATCH_BYTES = 256
NOALLOC_MAX_UNITS = 1 << 30

DTYPE_BF16, DTYPE_F16 = 0, 1
NORM_SOFTMAX, NORM_SIGMOID, NORM_RELU = 0, 1, 2
MOD_NONE, MOD_SOFTCAP, MOD_ALIBI, MOD_TEMP = 0, 1, 2, 3

STATUS = {
    0: "CHIA_OK",
    1: "CHIA_ERR_INVALID_ARGUMENT",
    2: "CHIA_ERR_UNSUPPORTED",
    3: "CHIA_ERR_MISALIGNED",
    4: "CHIA_ERR_LAUNCH",
    5: "CHIA_ERR_DEVICE_TIMEOUT",
    6: "CHIA_ERR_NO_DEVICE",
    8: "CHIA_ERR_BAD_INDEX",
    16: "CHIA_ERR_NO_PAGES",
}

EXPORTED_SYMBOLS = (
    "chia_attn_fwd",
    "chia_attn_fwd_noalloc",
    "chia_attn_visible_pairs",
    "chia_attn_tile_plan",
    "chia_attn_status_string",
    "chia_attn_abi_version",
    "chia_attn_decode",
    "chia_attn_decode_workspace_bytes",
    "chia_attn_bwd",
    "chia_attn_bwd_workspace_bytes",
)


class AttnParams(ctypes.Structure):
    """Mirror of ``chia_attn_params_t`` (include/chia_attn.h)."""

    _fields_ = [
        ("abi_version", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("norm", ctypes.c_int32),
        ("mod", ctypes.c_int32),
        ("heads_kv", ctypes.c_int32),
        ("batch", ctypes.c_int64),
        ("heads", ctypes.c_int64),
        ("seqlen_q", ctypes.c_int64),
        ("seqlen_kv", ctypes.c_int64),
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("q_stride", ctypes.c_int64 * 3),
        ("k_stride", ctypes.c_int64 * 3),
        ("v_stride", ctypes.c_int64 * 3),
        ("o_stride", ctypes.c_int64 * 3),
        ("scale", ctypes.c_float),
        ("softcap", ctypes.c_float),
        ("sig_bias", ctypes.c_float),
        ("out_scale", ctypes.c_float),
        ("head_param", ctypes.c_void_p),
        ("win_left", ctypes.c_int64),
        ("win_right", ctypes.c_int64),
        ("block", ctypes.c_int64),
        ("prefix", ctypes.c_int64),
        ("dilation", ctypes.c_int64),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("seq_offsets", ctypes.c_void_p),
        ("num_seqs", ctypes.c_int64),
        ("lse", ctypes.c_void_p),
        ("wait_limit_ns", ctypes.c_uint64),
    ]


class AttnGrads(ctypes.Structure):
    """Mirror of ``chia_attn_grads_t`` (include/chia_attn.h)."""

    _fields_ = [
        ("dout", ctypes.c_void_p),
        ("dout_stride", ctypes.c_int64 * 3),
        ("dq", ctypes.c_void_p),
        ("dk", ctypes.c_void_p),
        ("dv", ctypes.c_void_p),
        ("dq_stride", ctypes.c_int64 * 3),
        ("dk_stride", ctypes.c_int64 * 3),
        ("dv_stride", ctypes.c_int64 * 3),
    ]


# ---- the paged 8-bit K/V cache (include/chia_paged.h)
PAGED_ABI_VERSION = 1

PAGED_SYMBOLS = (
    "chia_page_tables",
    "chia_release_pages",
    "chia_cache_append",
    "chia_paged_attn",
    "chia_paged_attn_workspace_bytes",
    "chia_trim_pages",
)


class TablesParams(ctypes.Structure):
    """Mirror of ``chia_tables_params_t`` (include/chia_paged.h)."""

    _fields_ = [
        ("abi_version", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("batch", ctypes.c_int64),
        ("table_width", ctypes.c_int64),
        ("table_stride", ctypes.c_int64),
        ("ring_size", ctypes.c_int64),
        ("max_tokens", ctypes.c_int64),
        ("seq_lens", ctypes.c_void_p),
        ("new_lens", ctypes.c_void_p),
        ("block_table", ctypes.c_void_p),
        ("free_pages", ctypes.c_void_p),
        ("free_state", ctypes.c_void_p),
        ("slots", ctypes.c_void_p),
        ("positions", ctypes.c_void_p),
        ("cu_q", ctypes.c_void_p),
        ("new_seq_lens", ctypes.c_void_p),
        ("new_free_state", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class AppendParams(ctypes.Structure):
    """Mirror of ``chia_append_params_t`` (include/chia_paged.h)."""

    _fields_ = [
        ("abi_version", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("cache_dtype", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("heads_kv", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("tokens", ctypes.c_int64),
        ("num_pages", ctypes.c_int64),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("k_stride", ctypes.c_int64 * 2),
        ("v_stride", ctypes.c_int64 * 2),
        ("slots", ctypes.c_void_p),
        ("k_cache", ctypes.c_void_p),
        ("v_cache", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("status", ctypes.c_void_p),
    ]


class PagedParams(ctypes.Structure):
    """Mirror of ``chia_paged_params_t`` (include/chia_paged.h)."""

    _fields_ = [
        ("abi_version", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("cache_dtype", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("norm", ctypes.c_int32),
        ("mod", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("heads_kv", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("max_q", ctypes.c_int32),
        ("batch", ctypes.c_int64),
        ("tokens", ctypes.c_int64),
        ("num_pages", ctypes.c_int64),
        ("table_width", ctypes.c_int64),
        ("table_stride", ctypes.c_int64),
        ("q", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("q_stride", ctypes.c_int64 * 2),
        ("o_stride", ctypes.c_int64 * 2),
        ("k_cache", ctypes.c_void_p),
        ("v_cache", ctypes.c_void_p),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("block_table", ctypes.c_void_p),
        ("seq_lens", ctypes.c_void_p),
        ("cu_q", ctypes.c_void_p),
        ("lse", ctypes.c_void_p),
        ("head_param", ctypes.c_void_p),
        ("scale", ctypes.c_float),
        ("softcap", ctypes.c_float),
        ("sig_bias", ctypes.c_float),
        ("out_scale", ctypes.c_float),
        ("win_left", ctypes.c_int64),
        ("win_right", ctypes.c_int64),
        ("block", ctypes.c_int64),
        ("prefix", ctypes.c_int64),
        ("dilation", ctypes.c_int64),
        ("status", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64),
        ("wait_limit_ns", ctypes.c_uint64),
    ]


_binding_module = None


def binding():
    """The compiled argument checks of ``paged.py`` (``csrc/binding.cpp``),
    given the entry points of the library. Raises if it has not been built."""
    global _binding_module
    if _binding_module is not None:
        return _binding_module
    lib = load()
    path = os.path.join(_HERE, "_lib", f"_binding-{importlib.metadata.version('torch')}.so")
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -m chia_proj_b200.build`")
    loader = importlib.machinery.ExtensionFileLoader("_binding", path)
    m = importlib.util.module_from_spec(importlib.util.spec_from_loader("_binding", loader))
    loader.exec_module(m)
    m.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in PAGED_SYMBOLS))
    _binding_module = m
    return m


def status_name(code: int) -> str:
    """Its name; of a status word, where kernels OR their errors, the names of all of them."""
    if code in STATUS:
        return STATUS[code]
    parts = [b for b in (code & 7, code & 8, code & 16) if b]
    if sum(parts) != code or any(p not in STATUS for p in parts):
        return f"status {code}"
    return " | ".join(STATUS[p] for p in parts)


class ChiaError(RuntimeError):
    """A non-zero ``chia_status`` returned by the library."""

    def __init__(self, code: int, what: str = ""):
        self.code = code
        name = status_name(code)
        super().__init__(f"{name}{': ' + what if what else ''}")


_lock = threading.Lock()
_lib = None


def load() -> ctypes.CDLL:
    """Load the native library (once). Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise ImportError(
                    f"{LIB_PATH} is missing: build it with "
                    "`python -m chia_proj_b200.build` (nvcc, sm_100a)")
            lib = ctypes.CDLL(LIB_PATH)
            lib.chia_attn_fwd.argtypes = [ctypes.POINTER(AttnParams), ctypes.c_void_p]
            lib.chia_attn_fwd.restype = ctypes.c_int
            lib.chia_attn_fwd_noalloc.argtypes = [ctypes.POINTER(AttnParams), ctypes.c_void_p]
            lib.chia_attn_fwd_noalloc.restype = ctypes.c_int
            lib.chia_attn_decode.argtypes = [ctypes.POINTER(AttnParams), ctypes.c_void_p,
                                             ctypes.c_int64, ctypes.c_void_p]
            lib.chia_attn_decode.restype = ctypes.c_int
            lib.chia_attn_decode_workspace_bytes.argtypes = [ctypes.POINTER(AttnParams)]
            lib.chia_attn_decode_workspace_bytes.restype = ctypes.c_int64
            lib.chia_attn_bwd.argtypes = [ctypes.POINTER(AttnParams), ctypes.POINTER(AttnGrads),
                                          ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p]
            lib.chia_attn_bwd.restype = ctypes.c_int
            lib.chia_attn_bwd_workspace_bytes.argtypes = [ctypes.POINTER(AttnParams)]
            lib.chia_attn_bwd_workspace_bytes.restype = ctypes.c_int64
            lib.chia_attn_visible_pairs.argtypes = [ctypes.POINTER(AttnParams)]
            lib.chia_attn_visible_pairs.restype = ctypes.c_int64
            lib.chia_attn_tile_plan.argtypes = [
                ctypes.POINTER(AttnParams), ctypes.c_int64, ctypes.c_int32, ctypes.c_int32,
                ctypes.POINTER(ctypes.c_int64), ctypes.POINTER(ctypes.c_int64),
                ctypes.POINTER(ctypes.c_uint64)]
            lib.chia_attn_tile_plan.restype = ctypes.c_int
            lib.chia_attn_status_string.argtypes = [ctypes.c_int]
            lib.chia_attn_status_string.restype = ctypes.c_char_p
            lib.chia_attn_abi_version.argtypes = []
            lib.chia_attn_abi_version.restype = ctypes.c_int
            for name in PAGED_SYMBOLS[:4] + PAGED_SYMBOLS[5:]:  # the parameters as the bytes of their struct
                getattr(lib, name).argtypes = [ctypes.c_char_p, ctypes.c_void_p]
                getattr(lib, name).restype = ctypes.c_int
            lib.chia_paged_attn_workspace_bytes.argtypes = [ctypes.c_char_p]
            lib.chia_paged_attn_workspace_bytes.restype = ctypes.c_int64
            if lib.chia_attn_abi_version() != ABI_VERSION:
                raise ImportError(f"{LIB_PATH}: ABI version mismatch")
            _lib = lib
    return _lib


def check(code: int, what: str = "") -> None:
    if code != 0:
        raise ChiaError(code, what)

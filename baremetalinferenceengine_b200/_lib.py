"""ctypes binding of ``libbm_layer_ops.so`` (the C ABI in ``include/bm_layer_ops.h``).

Loading fails loudly when the library has not been built: there is no CPU or
PyTorch fallback for any op.
"""
from __future__ import annotations

import ctypes
import os
import threading

from .build import BINDING_PATH, LIB_PATH

c_int, c_int32, c_int64, c_float, c_double = (ctypes.c_int, ctypes.c_int32, ctypes.c_int64,
                                              ctypes.c_float, ctypes.c_double)
c_void_p, c_char_p = ctypes.c_void_p, ctypes.c_char_p
P_INT32 = ctypes.POINTER(ctypes.c_int32)

BM_OK = 0
BM_ERR_INVALID_ARGUMENT = 1
BM_ERR_CUDA = 2
BM_ERR_DEVICE = 3

BM_F32 = 0
BM_BF16 = 1

BM_DEVERR_BAD_ID = 0x1
BM_DEVERR_BAD_POSITION = 0x2
BM_DEVERR_BAD_SEQUENCE = 0x4
BM_DEVERR_TIMEOUT = 0x8
BM_DEVERR_BAD_PAGE = 0x10
BM_DEVERR_BAD_PARAMETER = 0x20

BM_ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "bands": 3, "yarn": 4}


class LayerStepC(ctypes.Structure):
    """Mirror of bm_layer_step_t (include/bm_layer_ops.h): one layer step's sizes
    and device buffers."""

    _fields_ = [
        ("rows", c_int64), ("dim", c_int32), ("ffn", c_int32), ("vocab", c_int64),
        ("num_q_heads", c_int32), ("num_kv_heads", c_int32), ("head_dim", c_int32), ("max_seq", c_int32),
        ("num_seqs", c_int32), ("eps", c_float), ("theta", c_double),
        ("ids", c_void_p), ("embed", c_void_p), ("hidden", c_void_p), ("attn_out", c_void_p), ("w_attn", c_void_p),
        ("y_attn", c_void_p), ("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("positions", c_void_p),
        ("seq_ids", c_void_p), ("k_cache", c_void_p), ("v_cache", c_void_p), ("rope_table", c_void_p),
        ("rope_table_len", c_int32), ("ffn_out", c_void_p), ("w_ffn", c_void_p), ("y_ffn", c_void_p),
        ("gate", c_void_p), ("up", c_void_p), ("act", c_void_p),
    ]


class RopeScalingC(ctypes.Structure):
    """Mirror of bm_rope_scaling_t."""

    _fields_ = [("kind", c_int32), ("original_max_pos", c_int32), ("factor", c_double), ("low", c_double),
                ("high", c_double), ("mscale", c_double)]


class PagedKVC(ctypes.Structure):
    """Mirror of bm_paged_kv_t."""

    _fields_ = [("k_pages", c_void_p), ("v_pages", c_void_p), ("page_table", c_void_p), ("num_pages", c_int32),
                ("page_size", c_int32), ("max_pages", c_int32), ("num_seqs", c_int32), ("num_kv_heads", c_int32),
                ("head_dim", c_int32)]


class PagedKV8C(ctypes.Structure):
    """Mirror of bm_paged_kv8_t."""

    _fields_ = [("k_pages", c_void_p), ("v_pages", c_void_p), ("k_scales", c_void_p), ("v_scales", c_void_p),
                ("page_table", c_void_p), ("num_pages", c_int32), ("page_size", c_int32), ("block", c_int32),
                ("max_pages", c_int32), ("num_seqs", c_int32), ("num_kv_heads", c_int32), ("head_dim", c_int32)]


# name -> (restype, argtypes). Every symbol include/bm_layer_ops.h declares.
SIGNATURES = {
    "bm_status_string": (c_char_p, [c_int]),
    "bm_abi_version": (c_int, []),
    "bm_last_error_message": (c_char_p, []),
    "bm_status_read": (c_int, [c_void_p, P_INT32, c_void_p]),
    "bm_embed_gather": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int,
                                c_void_p, c_void_p]),
    "bm_rmsnorm": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_float, c_int64, c_int64, c_int,
                           c_void_p]),
    "bm_add_rmsnorm": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_float, c_int,
                               c_void_p]),
    "bm_add": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int, c_void_p]),
    "bm_swiglu": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int, c_void_p]),
    "bm_rope_table_fill": (c_int, [c_void_p, c_int32, c_int32, c_double, c_void_p]),
    "bm_rope_table_create": (c_int, [c_int32, c_int32, c_double, ctypes.POINTER(c_void_p)]),
    "bm_rope_table_destroy": (c_int, [c_void_p]),
    "bm_rope_kv_store": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p, c_void_p,
                                 c_void_p, c_int32, c_double, c_int64, c_int32, c_int32, c_int32, c_int32, c_int32,
                                 c_int, c_void_p, c_void_p]),
    "bm_rope": (c_int, [c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_int32, c_double, c_int64, c_int32,
                        c_int32, c_int32, c_int, c_void_p, c_void_p]),
    "bm_kv_store": (c_int, [c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_int64, c_int32, c_int32, c_int32,
                            c_int32, c_int, c_void_p, c_void_p]),
    "bm_decode_attention_workspace_size": (c_int, [c_int64, c_int32, c_int32, c_int32, c_int32,
                                                   ctypes.POINTER(ctypes.c_size_t)]),
    "bm_gemm_swiglu": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_int32, c_int, c_void_p,
                               c_void_p]),
    "bm_gemm": (c_int, [c_void_p, c_void_p, c_void_p, c_int64, c_int32, c_int32, c_int, c_void_p, c_void_p]),
    "bm_gemm_shared_a": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int64, c_int32, c_int, c_void_p,
                                 c_void_p]),
    "bm_rmsnorm_gemm": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_void_p, c_void_p,
                                c_void_p, c_int32, c_int32, c_int64, c_int32, c_int, c_void_p, c_void_p]),
    "bm_rope_kv_decode_attention": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32,
                                            c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int64, c_int32, c_int32,
                                            c_int32, c_int32, c_int32, c_float, c_void_p, ctypes.c_size_t, c_int,
                                            c_void_p, c_void_p]),
    "bm_softmax": (c_int, [c_void_p, c_int64, c_int64, c_int64, c_int, c_void_p]),
    "bm_decode_attention": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int64,
                                    c_int32, c_int32, c_int32, c_int32, c_int32, c_float, c_void_p, ctypes.c_size_t,
                                    c_int, c_void_p, c_void_p]),
    "bm_decode_attention_static_scratch": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                                   c_int32, c_int64, c_int32, c_int32, c_int32, c_int32, c_int32,
                                                   c_float, c_int, c_void_p, c_void_p]),
    "bm_kv_cache_create": (c_int, [c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_int,
                                   ctypes.POINTER(c_void_p)]),
    "bm_kv_cache_destroy": (c_int, [c_void_p]),
    "bm_kv_cache_layer": (c_int, [c_void_p, c_int32, ctypes.POINTER(c_void_p), ctypes.POINTER(c_void_p)]),
    "bm_kv_cache_seq_len": (c_int, [c_void_p, c_int32, P_INT32]),
    "bm_kv_cache_reset": (c_int, [c_void_p, c_int32]),
    "bm_kv_cache_append": (c_int, [c_void_p, c_void_p, c_int64, ctypes.POINTER(c_void_p), ctypes.POINTER(c_void_p),
                                   c_void_p]),
    "bm_selftest_bounded_wait": (c_int, [c_int64, c_void_p, c_void_p, c_void_p]),
    "bm_rotary_table_fill": (c_int, [c_void_p, c_int32, c_int32, c_double, ctypes.POINTER(RopeScalingC), c_void_p]),
    "bm_rotary": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_int32, c_int32, c_int32,
                          c_int64, c_int32, c_int32, c_int32, c_int64, c_int64, c_int64, c_int64, c_int, c_void_p,
                          c_void_p]),
    "bm_paged_kv_append": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                   ctypes.POINTER(PagedKVC), c_void_p, c_int32, c_int32, c_int32, c_int64, c_int32,
                                   c_int64, c_int64, c_int64, c_int64, c_int, c_void_p, c_void_p]),
    "bm_paged_tree_attention_workspace_size": (c_int, [c_int64, c_int64, c_int32, c_int32, c_int32, c_int32, c_int32,
                                                       ctypes.POINTER(ctypes.c_size_t)]),
    "bm_paged_tree_attention": (c_int, [c_void_p, c_void_p, ctypes.POINTER(PagedKVC), c_void_p, c_void_p, c_void_p,
                                        c_void_p, c_int32, c_int64, c_int64, c_int32, c_int32, c_int32, c_float,
                                        c_void_p, ctypes.c_size_t, c_int, c_void_p, c_void_p]),
    "bm_qk_norm_rotary": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_float, c_void_p, c_int32,
                                  c_void_p, c_int32, c_int32, c_int32, c_int64, c_int32, c_int32, c_int32, c_int64,
                                  c_int64, c_int64, c_int64, c_int, c_void_p, c_void_p]),
    "bm_paged_kv8_append": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_float, c_void_p,
                                    ctypes.POINTER(PagedKV8C), c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_int32,
                                    c_int32, c_int64, c_int64, c_int32, c_int32, c_int64, c_int64, c_int64, c_int64, c_int,
                                    c_void_p, c_void_p]),
    "bm_paged_kv8_read": (c_int, [c_void_p, c_void_p, ctypes.POINTER(PagedKV8C), c_void_p, c_void_p, c_void_p, c_int64,
                                  c_int64, c_int32, c_int, c_void_p, c_void_p]),
    "bm_paged_kv8_tree_attention_workspace_size": (c_int, [c_int64, c_int64, c_int32, c_int32, c_int32, c_int32, c_int32,
                                                           ctypes.POINTER(ctypes.c_size_t)]),
    "bm_paged_kv8_tree_attention": (c_int, [c_void_p, c_void_p, ctypes.POINTER(PagedKV8C), c_void_p, c_void_p, c_void_p,
                                            c_void_p, c_int32, c_int64, c_int64, c_int32, c_int32, c_int32, c_float,
                                            c_void_p, ctypes.c_size_t, c_int, c_void_p, c_void_p]),
    "bm_sample": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                          c_int64, c_int, c_void_p, c_void_p]),
    "bm_layer_step": (c_int, [ctypes.POINTER(LayerStepC), c_int, c_void_p, c_void_p]),
}

_lock = threading.Lock()
_lib = None


class BMError(RuntimeError):
    """A non-zero bm_status_t from the C ABI, with the library's message."""

    def __init__(self, status: int, message: str):
        super().__init__(f"{message} [{status_name(status)}]")
        self.status = status


def status_name(status: int) -> str:
    return {BM_OK: "BM_OK", BM_ERR_INVALID_ARGUMENT: "BM_ERR_INVALID_ARGUMENT", BM_ERR_CUDA: "BM_ERR_CUDA",
            BM_ERR_DEVICE: "BM_ERR_DEVICE"}.get(status, f"BM_ERR_{status}")


def lib_path() -> str:
    return LIB_PATH


def load() -> ctypes.CDLL:
    """Loads the library once; raises if it is missing (no fallback path)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"{LIB_PATH} is missing: build the sm_100a kernels first "
                    "(python -m baremetalinferenceengine_b200.build)")
            lib = ctypes.CDLL(LIB_PATH)
            for name, (restype, argtypes) in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = restype
                fn.argtypes = argtypes
            _lib = lib
        return _lib


_serving = None


def serving_ops():
    """The CPython module over the paged-cache serving operators (csrc/binding/); raises if
    it is missing (no fallback path)."""
    global _serving
    if _serving is not None:
        return _serving
    load()
    with _lock:
        if _serving is None:
            if not os.path.exists(BINDING_PATH):
                raise RuntimeError(f"{BINDING_PATH} is missing: build it first (python -m baremetalinferenceengine_b200.build)")
            import importlib.machinery
            import importlib.util

            name = __package__ + "._serving_ops"
            spec = importlib.util.spec_from_file_location(
                name, BINDING_PATH, loader=importlib.machinery.ExtensionFileLoader(name, BINDING_PATH))
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
            _serving = module
        return _serving


def check(status: int) -> None:
    if status != BM_OK:
        msg = load().bm_last_error_message()
        raise BMError(status, msg.decode() if msg else "")

"""Loader for libquipsharp_hip.so (the C ABI declared in include/quipsharp_hip.h).

The library is mandatory: every compute entry point of quipsharp_amd goes
through it, and there is no CPU or pure-PyTorch substitute.  A missing or
unloadable library raises immediately.
"""
import contextlib
import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libquipsharp_hip.so")

QS_OK = 0
QS_STAGE_E8P = 0
QS_STAGE_E8_1BIT = 1
QS_DTYPE_F32, QS_DTYPE_F16, QS_DTYPE_BF16 = 0, 1, 2
QS_LAYOUT_ROWMAJOR, QS_LAYOUT_TILED = 0, 1
QS_SIGNS_BITS = 0x100  # layout flag: su / sv are packed sign bits
QS_MAX_STAGES = 4
QS_MAX_KRON = 64
QS_MAX_GROUP = 4
QS_NOALLOC_SCRATCH_BYTES = 32 << 20
QS_PREOP_RMSNORM, QS_PREOP_SILU_MUL = 1, 2
QS_MAX_STATES = 8

_vp = ctypes.c_void_p


class LinearJob(ctypes.Structure):
    """qs_linear_job (include/quipsharp_hip.h)."""
    _fields_ = [("codes0", ctypes.c_void_p), ("codes1", ctypes.c_void_p), ("m", ctypes.c_int64),
                ("su", ctypes.c_void_p), ("sv", ctypes.c_void_p), ("kron_pm", ctypes.c_int),
                ("kron_m", ctypes.c_void_p), ("s0", ctypes.c_float), ("s1", ctypes.c_float),
                ("layer_scale", ctypes.c_float), ("bias", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("ldy", ctypes.c_int64), ("sign_bits", ctypes.c_int)]



class PreOp(ctypes.Structure):
    """qs_preop (include/quipsharp_hip.h)."""
    _fields_ = [("kind", ctypes.c_int), ("x2", ctypes.c_void_p), ("ldx2", ctypes.c_int64),
                ("weight", ctypes.c_void_p), ("h_out", ctypes.c_void_p), ("ldo", ctypes.c_int64),
                ("eps", ctypes.c_float)]


class PagePool(ctypes.Structure):
    """qs_page_pool (include/quipsharp_hip.h)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_page", ctypes.c_int64),
                ("k_head", ctypes.c_int64), ("k_pos", ctypes.c_int64), ("v_page", ctypes.c_int64),
                ("v_head", ctypes.c_int64), ("v_pos", ctypes.c_int64), ("pages", ctypes.c_int64),
                ("page", ctypes.c_int), ("table", ctypes.c_void_p), ("table_ld", ctypes.c_int64),
                ("cols", ctypes.c_int64), ("lengths", ctypes.c_void_p)]


class PageStore(ctypes.Structure):
    """qs_page_store (include/quipsharp_hip.h)."""
    _fields_ = [("data", ctypes.c_void_p), ("planes", ctypes.c_int64), ("pages", ctypes.c_int64),
                ("kv_heads", ctypes.c_int), ("page", ctypes.c_int), ("row_bytes", ctypes.c_int64)]


class AdapterJob(ctypes.Structure):
    """qs_adapter_job (include/quipsharp_hip.h)."""
    _fields_ = [("down", ctypes.c_void_p), ("up", ctypes.c_void_p), ("scale", ctypes.c_void_p),
                ("down_adapter", ctypes.c_int64), ("down_row", ctypes.c_int64), ("up_adapter", ctypes.c_int64),
                ("up_row", ctypes.c_int64), ("rank", ctypes.c_int), ("m", ctypes.c_int64), ("y", ctypes.c_void_p),
                ("ldy", ctypes.c_int64), ("out", ctypes.c_void_p), ("ldo", ctypes.c_int64)]


_i64 = ctypes.c_int64
_int = ctypes.c_int
_f32 = ctypes.c_float
_int_p = ctypes.POINTER(ctypes.c_int)
_f32_p = ctypes.POINTER(ctypes.c_float)
_pool_p = ctypes.POINTER(PagePool)
_store_p = ctypes.POINTER(PageStore)

_SIGNATURES = {
    "qs_last_error": ([], ctypes.c_char_p),
    "qs_abi_version": ([], _int),
    "qs_e8p_abs_table": ([_vp], _int),
    "qs_e81_table": ([_vp], _int),
    "qs_rvq_encode": ([_vp, _i64, _i64, _int, _int_p, _f32_p, _f32, _f32, _vp, _i64, _vp, _int, _i64, _i64,
                       _vp], _int),
    "qs_div_f32": ([_vp, _vp, _i64, _f32, _vp], _int),
    "qs_rvq_decode": ([_vp, _int, _i64, _i64, _int, _int_p, _f32_p, _f32, _vp, _vp], _int),
    "qs_ldlq_step": ([_vp, _i64, _vp, _vp, _vp, _i64, _vp, _i64, _vp, _i64, _i64, _int, _int_p, _f32_p,
                      _vp, _int, _i64, _i64, _vp], _int),
    "qs_ldlq_chunk": ([_vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _int, _int, _i64, _int, _int_p,
                       _f32_p, _vp, _int, _i64, _i64, _vp], _int),
    "qs_rht_f32": ([_vp, _vp, _i64, _i64, _i64, _vp, _vp, _vp, _int, _vp, _vp], _int),
    "qs_pack_codes": ([_vp, _int, _i64, _i64, _int, _int, _vp, _vp], _int),
    "qs_linear_workspace_bytes": ([_i64, _i64, _i64, _int], ctypes.c_size_t),
    "qs_linear_forward": ([_vp, _int, _i64, _i64, _i64, _i64, _vp, _vp, _int, _int, _vp, _vp, _int, _vp,
                           _int, _vp, _f32, _f32, _f32, _vp, _vp, _int, _i64, _vp, ctypes.c_size_t, _vp, _vp,
                           _vp], _int),
    "qs_linear_forward_noalloc": ([_vp, _int, _i64, _i64, _i64, _i64, _vp, _vp, _int, _int, _vp, _vp, _int, _vp,
                                   _int, _vp, _f32, _f32, _f32, _vp, _vp, _int, _i64, _vp], _int),
    "qs_decode_matvec": ([_vp, _int, _i64, _i64, _i64, _i64, _vp, _vp, _int, _int, _f32, _f32, _f32, _vp, _int,
                          _i64, _vp, ctypes.c_size_t, _vp], _int),
    "qs_linear_group_workspace_bytes": ([_i64, _i64, _int, ctypes.POINTER(ctypes.c_int64)], ctypes.c_size_t),
    "qs_linear_forward_group": ([_vp, _int, _i64, _i64, _i64, _int, _vp, _int, ctypes.POINTER(LinearJob), _int,
                                 _vp, ctypes.c_size_t, _vp, _vp, _vp], _int),
    "qs_linear_forward_group_pre": ([_vp, _i64, _i64, _i64, _int, _vp, _int, ctypes.POINTER(LinearJob),
                                     ctypes.POINTER(PreOp), _int, _vp, ctypes.c_size_t, _vp], _int),
    "qs_busy_wait": ([_i64, _vp], _int),
    "qs_dec_rmsnorm": ([_vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _f32, _vp], _int),
    "qs_dec_qk_norm_rope": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _int, _int, _int, _i64,
                             _f32, _vp], _int),
    "qs_dec_attention_workspace_bytes": ([_i64, _int, _i64], _i64),
    "qs_dec_attention": ([_vp, _vp, _vp, _vp, _vp, _i64, _vp, _i64, _i64, _int, _int, _int, _i64, _f32, _vp], _int),
    "qs_dec_attention_rope": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _i64, _i64, _int,
                               _int, _int, _i64, _f32, _f32, _vp], _int),
    "qs_dec_silu_mul": ([_vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _vp], _int),
    "qs_page_append": ([_vp, _vp, _i64, _i64, _int, _int, _i64, _i64, _i64, _i64, _vp, _pool_p, _vp], _int),
    "qs_page_append_over": ([_vp, _vp, _i64, _i64, _int, _int, _i64, _i64, _i64, _i64, _vp, _pool_p, _vp, _vp], _int),
    "qs_page_append_rope": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _i64, _int, _int, _int, _pool_p, _f32,
                             _vp], _int),
    "qs_page_append_rope_over": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i64, _vp, _i64, _int, _int, _int, _pool_p, _vp,
                                  _f32, _vp], _int),
    "qs_attend_token_workspace_bytes": ([_i64, _int, _int, _int, _i64, _int, _int, _int], ctypes.c_size_t),
    "qs_attend_token": ([_vp, _int, _i64, _int, _int, _int, _i64, _i64, _pool_p, _f32, _int, _int, _vp, _i64, _vp,
                         ctypes.c_size_t, _vp], _int),
    "qs_attend_token_over": ([_vp, _int, _i64, _int, _int, _int, _i64, _i64, _pool_p, _vp, _f32, _int, _int, _vp, _i64,
                              _vp, ctypes.c_size_t, _vp], _int),
    "qs_attend_chunk": ([_vp, _int, _i64, _i64, _int, _int, _int, _i64, _i64, _vp, _pool_p, _f32, _int, _int, _vp,
                         _i64, _vp], _int),
    "qs_attend_chunk_workspace_bytes": ([_i64, _i64, _int, _int, _int, _i64, _int, _int, _int], ctypes.c_size_t),
    "qs_attend_chunk_ws": ([_vp, _int, _i64, _i64, _int, _int, _int, _i64, _i64, _vp, _pool_p, _f32, _int, _int, _vp,
                            _i64, _vp, ctypes.c_size_t, _vp], _int),
    "qs_attend_chunk_over": ([_vp, _int, _i64, _i64, _int, _int, _int, _i64, _i64, _vp, _pool_p, _vp, _f32, _int, _int,
                              _vp, _i64, _vp, ctypes.c_size_t, _vp], _int),
    "qs_page_advance_workspace_bytes": ([_i64], ctypes.c_size_t),
    "qs_page_advance": ([_store_p, _vp, _vp, _vp, _vp, _i64, _i64, _int, _vp, _vp, _vp, _vp, _vp, ctypes.c_size_t,
                         _vp], _int),
    "qs_page_advance_rows": ([_store_p, _vp, _vp, _vp, _vp, _i64, _i64, _int, _vp, _vp, _vp, _vp, _vp, _vp,
                              ctypes.c_size_t, _vp], _int),
    "qs_page_advance_over": ([_store_p, _vp, _vp, _vp, _vp, _i64, _i64, _int, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp,
                              ctypes.c_size_t, _vp], _int),
    "qs_page_free": ([_vp, _vp, _vp, _vp, _i64, _i64, _i64, _int, _int, _int, _vp, _vp, _vp, _vp], _int),
    "qs_page_compact_workspace_bytes": ([_i64], ctypes.c_size_t),
    "qs_page_compact": ([_store_p, _vp, _vp, _i64, _i64, _vp, _vp, _vp, ctypes.c_size_t, _vp], _int),
    "qs_page_copy": ([_store_p, _vp, _vp, _i64, _vp], _int),
    "qs_beam_select_workspace_bytes": ([_i64, _int, _i64, _int], ctypes.c_size_t),
    "qs_beam_select": ([_vp, _int, _i64, _i64, _int, _i64, _vp, _vp, _i64, _int, _vp, _vp, _vp, _vp,
                        ctypes.c_size_t, _vp], _int),
    "qs_reorder_states": ([_int, ctypes.POINTER(_vp), ctypes.POINTER(_vp), ctypes.POINTER(_i64),
                           ctypes.POINTER(_i64), _vp, _i64, _i64, _vp], _int),
    "qs_page_append_rotated": ([_vp, _vp, _vp, _int, _i64, _i64, _int, _int, _int, _i64, _i64, _i64, _i64, _i64, _i64,
                                _vp, _pool_p, _vp, _vp, _int, _int, _f32, _vp, _i64, _vp], _int),
    "qs_adapters_workspace_bytes": ([_i64, _i64, _i64, _int, _int_p], ctypes.c_size_t),
    "qs_adapters_plan": ([_i64, _i64, _i64, _int, _int_p, ctypes.POINTER(_i64), _int_p], _int),
    "qs_adapters_add": ([_vp, _int, _i64, _i64, _i64, _vp, _i64, _int, ctypes.POINTER(AdapterJob), _vp,
                         ctypes.c_size_t, _vp], _int),
    "qs_token_logprobs_workspace_bytes": ([_i64, _i64, _int, _int], ctypes.c_size_t),
    "qs_token_logprobs_workspace_most": ([_i64, _i64, _int, _int], ctypes.c_size_t),
    "qs_token_logprobs": ([_vp, _int, _i64, _i64, _i64, _vp, _int, _int, _vp, _vp, _vp, _vp, _vp, _vp,
                           ctypes.c_size_t, _vp], _int),
}

EXPORTED = tuple(_SIGNATURES)

_lib = None


class QuipHipError(RuntimeError):
    """An entry point of libquipsharp_hip.so returned an error."""


def lib():
    """The loaded library (loaded on first use, after torch)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m quipsharp_amd.build` "
                "(quipsharp_amd has no fallback implementation)")
        L = ctypes.CDLL(LIB_PATH)
        for name, (args, res) in _SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        _lib = L
    return _lib


def check(rc):
    if rc != QS_OK:
        raise QuipHipError(lib().qs_last_error().decode(errors="replace") or f"error {rc}")


def ptr(t):
    return None if t is None else _vp(t.data_ptr())


def stream_of(t):
    return _vp(torch._C._cuda_getCurrentRawStream(t.get_device()))  # torch.cuda.current_stream's handle alone


_HERE_ALREADY = contextlib.nullcontext()


def device_of(t):
    """A context in which kernels go to t's device, at no cost where that is the current one."""
    return _HERE_ALREADY if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def require_gpu(*tensors, what="quipsharp_amd"):
    """Every compute path runs on the GPU; CPU tensors are rejected, not emulated."""
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{what} runs on the GPU (MI355X / gfx950); got a tensor on {t.device}")


def no_gradient(what):
    """A call that records nothing for autograd, and was given a tensor that requires a gradient, would lose it."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or detach its inputs")


def int_array(vals):
    arr = (ctypes.c_int * len(vals))(*vals)
    return arr


def float_array(vals):
    return (ctypes.c_float * len(vals))(*vals)


def dtype_code(dt):
    if dt == torch.float32:
        return QS_DTYPE_F32
    if dt == torch.float16:
        return QS_DTYPE_F16
    if dt == torch.bfloat16:
        return QS_DTYPE_BF16
    raise TypeError(f"unsupported dtype {dt} (float32, float16 or bfloat16)")

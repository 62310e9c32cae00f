"""ctypes binding of ``libfused_attn_hip.so`` (the C ABI in ``include/fused_attn_hip.h``).

This module replaces the reference's compiled pybind extension ``fused_attn._C``
(csrc/bindings.cpp:90-96).  It turns torch tensors into the plain pointers,
element strides and sizes of ``fa_fwd_params``, allocates every output and
workspace with the torch caching allocator on the tensors' device, enqueues the
kernels on the current stream and maps ``fa_status`` codes to ``RuntimeError``
(the reference's TORCH_CHECK failures surfaced as RuntimeError too,
csrc/bindings.cpp:35-50).

There is no fallback here: if the library is missing or the device is not a
gfx950 GPU, every entry point raises.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import os
import threading
import warnings
from typing import Optional

import torch

LIB_NAME = "libfused_attn_hip.so"
ABI_VERSION = 6

# fa_dtype codes
F16, BF16, F32, FP8_E4M3, INT4 = 0, 1, 2, 3, 4
_DTYPE_CODE = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}
_FP8 = getattr(torch, "float8_e4m3fn", None)
if _FP8 is not None:
    _DTYPE_CODE[_FP8] = FP8_E4M3

FA_OK, FA_ERR_INVALID_ARGUMENT, FA_ERR_UNSUPPORTED, FA_ERR_WORKSPACE, FA_ERR_HIP = range(5)
_STATUS_NAME = {
    FA_ERR_INVALID_ARGUMENT: "invalid argument",
    FA_ERR_UNSUPPORTED: "unsupported",
    FA_ERR_WORKSPACE: "workspace",
    FA_ERR_HIP: "HIP error",
}

FP8_QBLOCK = 64  # keys per FP8 scale block; split-K partitions are multiples of it


class FwdParams(ctypes.Structure):
    """Mirror of ``fa_fwd_params`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("q_stride_b", ctypes.c_int64),
        ("q_stride_h", ctypes.c_int64),
        ("q_stride_n", ctypes.c_int64),
        ("k_stride_b", ctypes.c_int64),
        ("k_stride_h", ctypes.c_int64),
        ("k_stride_n", ctypes.c_int64),
        ("v_stride_b", ctypes.c_int64),
        ("v_stride_h", ctypes.c_int64),
        ("v_stride_n", ctypes.c_int64),
        ("o_stride_b", ctypes.c_int64),
        ("o_stride_h", ctypes.c_int64),
        ("o_stride_n", ctypes.c_int64),
        ("batch", ctypes.c_int32),
        ("heads_q", ctypes.c_int32),
        ("heads_kv", ctypes.c_int32),
        ("seqlen_q", ctypes.c_int32),
        ("seqlen_k", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("causal", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("kv_dtype", ctypes.c_int32),
        ("cu_seqlens_q", ctypes.c_void_p),
        ("cu_seqlens_k", ctypes.c_void_p),
        ("max_seqlen_q", ctypes.c_int32),
        ("max_seqlen_k", ctypes.c_int32),
        ("lse", ctypes.c_void_p),
        ("lse_stride_b", ctypes.c_int64),
        ("lse_stride_h", ctypes.c_int64),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        ("scale_stride_b", ctypes.c_int64),
        ("scale_stride_h", ctypes.c_int64),
    ]


class QuantParams(ctypes.Structure):
    """Mirror of ``fa_quant_params`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("x", ctypes.c_void_p),
        ("x_stride_b", ctypes.c_int64),
        ("x_stride_h", ctypes.c_int64),
        ("x_stride_n", ctypes.c_int64),
        ("batch", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("seqlen", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("x8", ctypes.c_void_p),
        ("scale", ctypes.c_void_p),
    ]


class PagedKV(ctypes.Structure):
    """Mirror of ``fa_paged_kv`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("block_table", ctypes.c_void_p),
        ("block_table_stride", ctypes.c_int64),
        ("block_table_cols", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("seqlens_k", ctypes.c_void_p),
        ("num_pages", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("k_page_stride", ctypes.c_int64),
        ("v_page_stride", ctypes.c_int64),
    ]


def _int64s(*names: str) -> list:
    return [(n, ctypes.c_int64) for n in names]


class Int4Params(ctypes.Structure):
    """Mirror of ``fa_int4_params`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("x", ctypes.c_void_p),
        *_int64s("x_stride_b", "x_stride_h", "x_stride_n"),
        ("batch", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("seqlen", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("codes", ctypes.c_void_p),
        *_int64s("codes_stride_b", "codes_stride_h", "codes_stride_n"),
        ("scale", ctypes.c_void_p),
        *_int64s("scale_stride_b", "scale_stride_h", "scale_stride_n"),
    ]


class Int4AppendParams(ctypes.Structure):
    """Mirror of ``fa_int4_append_params`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("k", Int4Params),
        ("v", Int4Params),
        ("seqlens_k", ctypes.c_void_p),
        ("capacity", ctypes.c_int64),
        ("block_table", ctypes.c_void_p),
        ("block_table_stride", ctypes.c_int64),
        ("block_table_cols", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


class CacheParams(ctypes.Structure):
    """Mirror of ``fa_cache_params`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        *_int64s("q_stride_b", "q_stride_h", "q_stride_n", "k_stride_b", "k_stride_h", "k_stride_n", "v_stride_b",
                 "v_stride_h", "v_stride_n", "o_stride_b", "o_stride_h", "o_stride_n"),
        ("batch", ctypes.c_int32),
        ("heads_q", ctypes.c_int32),
        ("heads_kv", ctypes.c_int32),
        ("seqlen_q", ctypes.c_int32),
        ("seqlen_k", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("scale", ctypes.c_float),
        ("causal", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("kv_dtype", ctypes.c_int32),
        ("k_scale", ctypes.c_void_p),
        ("v_scale", ctypes.c_void_p),
        *_int64s("k_scale_stride_b", "k_scale_stride_h", "k_scale_stride_n", "v_scale_stride_b", "v_scale_stride_h",
                 "v_scale_stride_n"),
        ("seqlens_k", ctypes.c_void_p),
        ("block_table", ctypes.c_void_p),
        ("block_table_stride", ctypes.c_int64),
        ("block_table_cols", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
        ("lse", ctypes.c_void_p),
        *_int64s("lse_stride_b", "lse_stride_h"),
        ("scores_in", ctypes.c_void_p),
        *_int64s("scores_in_stride_b", "scores_in_stride_h"),
        ("scores_out", ctypes.c_void_p),
        *_int64s("scores_out_stride_b", "scores_out_stride_h"),
    ]


MAX_EVICT_TENSORS = 8  # FA_MAX_EVICT_TENSORS


class EvictTensor(ctypes.Structure):
    """Mirror of ``fa_evict_tensor`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("src", ctypes.c_void_p),
        ("dst", ctypes.c_void_p),
        *_int64s("src_stride_b", "src_stride_h", "src_stride_n", "dst_stride_b", "dst_stride_h", "dst_stride_n",
                 "row_bytes"),
    ]


class EvictParams(ctypes.Structure):
    """Mirror of ``fa_evict_params`` (include/fused_attn_hip.h)."""

    _fields_ = [
        ("scores", ctypes.c_void_p),
        *_int64s("scores_stride_b", "scores_stride_h"),
        ("seqlens_k", ctypes.c_void_p),
        ("batch", ctypes.c_int32),
        ("heads", ctypes.c_int32),
        ("seqlen", ctypes.c_int32),
        ("keep", ctypes.c_int32),
        ("recent", ctypes.c_int32),
        ("num_tensors", ctypes.c_int32),
        ("index", ctypes.c_void_p),
        ("scores_out", ctypes.c_void_p),
        ("seqlens_out", ctypes.c_void_p),
        ("tensors", EvictTensor * MAX_EVICT_TENSORS),
    ]


_lib = None
_lib_error: Optional[str] = None
_lock = threading.Lock()


def library_path() -> str:
    """``$FUSED_ATTN_HIP_LIB`` if set, else the in-tree build next to this file."""
    return os.environ.get("FUSED_ATTN_HIP_LIB") or os.path.join(os.path.dirname(os.path.abspath(__file__)), LIB_NAME)


def _has_fwd_workspace(lib: ctypes.CDLL) -> bool:
    return isinstance(getattr(lib, "fa_attention_fwd_ws", None), lib._FuncPtr)


def _has_int4(lib: ctypes.CDLL) -> bool:
    return isinstance(getattr(lib, "fa_attention_cache", None), lib._FuncPtr)


def _cache_library() -> ctypes.CDLL:
    """The library, if it has the 4-bit cache's functions and eviction (added within this ABI version)."""
    lib = load_library()
    if not _has_int4(lib):
        raise RuntimeError(f"fused_attn HIP backend: {library_path()} is older than the 4-bit cache: build it again")
    return lib


def _bind(lib: ctypes.CDLL) -> None:
    P = ctypes.POINTER(FwdParams)
    lib.fa_attention_fwd.argtypes = [P, ctypes.c_void_p]
    lib.fa_attention_fwd.restype = ctypes.c_int
    if _has_fwd_workspace(lib):
        lib.fa_attention_fwd_workspace_bytes.argtypes = [P]
        lib.fa_attention_fwd_workspace_bytes.restype = ctypes.c_size_t
        lib.fa_attention_fwd_ws.argtypes = [P, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
        lib.fa_attention_fwd_ws.restype = ctypes.c_int
    else:  # a library of this ABI from before the pair was added: no key splits
        lib.fa_attention_fwd_workspace_bytes = lambda p: 0
        lib.fa_attention_fwd_ws = lambda p, ws, nbytes, stream: lib.fa_attention_fwd(p, stream)
    lib.fa_attention_varlen_fwd.argtypes = [P, ctypes.c_void_p]
    lib.fa_attention_varlen_fwd.restype = ctypes.c_int
    lib.fa_splitk_workspace_bytes.argtypes = [ctypes.c_int32] * 5
    lib.fa_splitk_workspace_bytes.restype = ctypes.c_size_t
    lib.fa_attention_splitk.argtypes = [P, ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.fa_attention_splitk.restype = ctypes.c_int
    lib.fa_attention_splitk_noalloc.argtypes = [P, ctypes.c_int32, ctypes.c_void_p]
    lib.fa_attention_splitk_noalloc.restype = ctypes.c_int
    lib.fa_choose_num_splits.argtypes = [ctypes.c_int32] * 5
    lib.fa_choose_num_splits.restype = ctypes.c_int32
    lib.fa_attention_paged_decode.argtypes = [P, ctypes.POINTER(PagedKV), ctypes.c_int32, ctypes.c_void_p,
                                              ctypes.c_size_t, ctypes.c_void_p]
    lib.fa_attention_paged_decode.restype = ctypes.c_int
    lib.fa_quantize_kv_fp8.argtypes = [ctypes.POINTER(QuantParams), ctypes.c_void_p]
    lib.fa_quantize_kv_fp8.restype = ctypes.c_int
    if _has_int4(lib):
        for f in (lib.fa_quantize_kv_int4, lib.fa_dequantize_kv_int4):
            f.argtypes, f.restype = [ctypes.POINTER(Int4Params), ctypes.c_void_p], ctypes.c_int
        lib.fa_append_kv_int4.argtypes = [ctypes.POINTER(Int4AppendParams), ctypes.c_void_p]
        lib.fa_append_kv_int4.restype = ctypes.c_int
        lib.fa_attention_cache_workspace_bytes.argtypes = [ctypes.POINTER(CacheParams), ctypes.c_int32]
        lib.fa_attention_cache_workspace_bytes.restype = ctypes.c_size_t
        lib.fa_attention_cache.argtypes = [ctypes.POINTER(CacheParams), ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t,
                                           ctypes.c_void_p]
        lib.fa_attention_cache.restype = ctypes.c_int
        lib.fa_evict_kv_workspace_bytes.argtypes = [ctypes.POINTER(EvictParams)]
        lib.fa_evict_kv_workspace_bytes.restype = ctypes.c_size_t
        lib.fa_evict_kv.argtypes = [ctypes.POINTER(EvictParams), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
        lib.fa_evict_kv.restype = ctypes.c_int
    lib.fa_device_supported.argtypes = [ctypes.c_int32]
    lib.fa_device_supported.restype = ctypes.c_int32
    lib.fa_last_error.argtypes = []
    lib.fa_last_error.restype = ctypes.c_char_p


def load_library() -> ctypes.CDLL:
    """Load and bind the shared library once; raise RuntimeError if it is unusable."""
    global _lib, _lib_error
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not os.path.exists(path):
            _lib_error = f"{path} not found: build it with `python -c 'import __graft_entry__ as g; g.build()'`"
            raise RuntimeError(f"fused_attn HIP backend unavailable: {_lib_error}")
        try:
            lib = ctypes.CDLL(path)
        except OSError as e:
            _lib_error = str(e)
            raise RuntimeError(f"fused_attn HIP backend unavailable: {e}") from e
        got = lib.fa_abi_version()  # before the rest is bound, which another version need not have
        if got != ABI_VERSION:
            _lib_error = f"ABI version mismatch: library {got}, bindings {ABI_VERSION}"
            raise RuntimeError(f"fused_attn HIP backend unavailable: {_lib_error}")
        _bind(lib)
        _lib = lib
        return lib


def library_loaded() -> bool:
    try:
        load_library()
        return True
    except RuntimeError:
        return False


TORCH_LIB_NAME = "libfused_attn_torch.so"
_native: Optional[ctypes.CDLL] = None
_native_devices: set[int] = set()


def load_native() -> None:
    """Load and register the native dispatcher kernels of ``fused_attn::attention`` (csrc/fa_torch.cpp), if they are
    built for this very torch (there is no stable C++ ABI: another build's symbols may resolve and still read its
    tensors wrongly) and these bindings: they hand every call back to the Python kernels until ``_enable_native``
    names its device."""
    global _native
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), TORCH_LIB_NAME)
    if _native is not None or torch.version.hip is None or not os.path.exists(path):
        return
    want = (f"{torch.__version__} {torch.version.git_version}", ABI_VERSION, ctypes.sizeof(FwdParams))
    try:
        lib = ctypes.CDLL(path)
        lib.fa_torch_built_for.restype = ctypes.c_char_p
        lib.fa_torch_params_size.restype = ctypes.c_size_t
        got = (lib.fa_torch_built_for().decode(), lib.fa_torch_abi_version(), lib.fa_torch_params_size())
        if got != want:
            raise OSError(f"built for torch, ABI version and parameter size {got}, found {want}")
        if not lib.fa_torch_register():
            raise OSError("torch refused its kernels")
    except (OSError, AttributeError) as e:
        warnings.warn(f"fused_attn: {path} does not load, calls take the slower Python path: {e}")
        return
    lib.fa_torch_bind.argtypes = [ctypes.c_void_p] * 5
    lib.fa_torch_bind.restype = None
    lib.fa_torch_enable.argtypes = [ctypes.c_int32]
    lib.fa_torch_enable.restype = None
    lib.fa_torch_route.argtypes = [ctypes.c_int32] + [ctypes.c_int64] * 6
    lib.fa_torch_route.restype = ctypes.c_int64
    _native = lib


def _enable_native(index: int) -> None:
    """Let the native kernels serve device ``index``, which ``device_supported`` has accepted."""
    hip = load_library()
    with _lock:
        if _native is not None and _has_fwd_workspace(hip):
            if not _native_devices:
                _native.fa_torch_bind(*(ctypes.cast(f, ctypes.c_void_p) for f in (
                    hip.fa_attention_fwd_workspace_bytes, hip.fa_attention_fwd_ws, hip.fa_splitk_workspace_bytes,
                    hip.fa_attention_splitk, hip.fa_last_error)))
            _native.fa_torch_enable(index)
        _native_devices.add(index)


_device_ok: dict[int, bool] = {}


def device_supported(device: torch.device | int | None = None) -> bool:
    """True when the library loads and ``device`` is a gfx950 GPU (has_tensor_core_kernel analogue)."""
    if isinstance(device, torch.device) and device.index is not None:
        ok = _device_ok.get(device.index)  # per-call fast path: the answer is fixed per device
        if ok is not None:
            return ok
    if not torch.cuda.is_available():
        return False
    if device is None:
        idx = torch.cuda.current_device()
    elif isinstance(device, int):
        idx = device
    else:
        idx = torch.device(device).index
        idx = torch.cuda.current_device() if idx is None else idx
    if idx not in _device_ok:
        try:
            _device_ok[idx] = bool(load_library().fa_device_supported(idx))
        except RuntimeError:
            _device_ok[idx] = False
    return _device_ok[idx]


def available() -> bool:
    return device_supported()


def _check(status: int, what: str) -> None:
    if status != FA_OK:
        msg = load_library().fa_last_error().decode(errors="replace")
        raise RuntimeError(f"fused_attn HIP {what} failed ({_STATUS_NAME.get(status, status)}): {msg}")


# ----------------------------------------------------------------------------------------------
# tensor preparation
# ----------------------------------------------------------------------------------------------


TOKEN_STRIDE_LIMIT_BYTES = 1 << 24  # the C ABI's bound on K/V token strides


def _aligned_view(t: torch.Tensor, vec_elems: int, base_align: int) -> torch.Tensor:
    """``t`` itself when its D stride is 1 and its pointer/other strides allow the kernels'
    vector accesses, else a contiguous copy (the kernels never see an unaligned view)."""
    # (fast path: a contiguous tensor's strides are multiples of its last size)
    if (t.is_contiguous() and t.dim() >= 3 and t.size(-1) % vec_elems == 0 and t.data_ptr() % base_align == 0
            and t.stride(2 if t.dim() == 4 else 0) * t.element_size() < TOKEN_STRIDE_LIMIT_BYTES):
        return t
    ok = t.stride(-1) == 1 and t.data_ptr() % base_align == 0
    if ok:
        for i in range(t.dim() - 1):
            if t.size(i) > 1 and t.stride(i) % vec_elems != 0:
                ok = False
                break
    # The kernels address up to 128 K/V rows from a tile start with 32-bit byte offsets, and the
    # C ABI rejects token strides of 16 MiB or more: such a view is copied too.  The token dim is
    # 2 of [B, H, N, D] and 0 of a packed [T, H, D].
    tok = 2 if t.dim() == 4 else 0
    if ok and t.dim() >= 3 and t.size(tok) > 1 and t.stride(tok) * t.element_size() >= TOKEN_STRIDE_LIMIT_BYTES:
        ok = False
    # clone, not contiguous(): an already-contiguous view at an unaligned offset must be copied too
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _check_qkv(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, layout: str, kv_fp8: bool = False) -> None:
    """Reject q/k/v that do not describe one attention problem before anything is launched
    (the reference's check_inputs, csrc/bindings.cpp:35-44, and _check, triton_fwd.py:217-222):
    the kernels take head_dim and the batch from q and the K/V dtype, lengths and heads from k,
    so a V of another shape or dtype, or a K of another head_dim, would be read out of bounds.

    layout: "dense" q [B,Hq,Nq,D], k/v [B or 1,Hkv,Nk,D]; "varlen" q [Tq,Hq,D], k/v [Tk,Hkv,D];
    "paged" q [B,Hq,Nq,D], k/v pools [P,Hkv,page,D]."""
    nd = 3 if layout == "varlen" else 4
    if q.dim() != nd or k.dim() != nd or v.dim() != nd:
        raise RuntimeError(f"expected {nd}-D q, k and v for the {layout} layout, got "
                           f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if k.shape != v.shape:
        raise RuntimeError(f"k and v must have the same shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != v.dtype:
        raise RuntimeError(f"k and v must have the same dtype, got {k.dtype} and {v.dtype}")
    if kv_fp8:
        if k.dtype != _FP8:
            raise RuntimeError(f"FP8 K/V must be float8_e4m3fn, got {k.dtype}")
    elif q.dtype != k.dtype:
        raise RuntimeError(f"q/k/v dtypes must match, got {q.dtype} and {k.dtype}")
    if q.shape[-1] != k.shape[-1]:
        raise RuntimeError(f"q and k must have the same head_dim, got {q.shape[-1]} and {k.shape[-1]}")
    hq, hkv = q.shape[-2 if layout == "varlen" else 1], k.shape[-2 if layout == "varlen" else 1]
    if hkv == 0 or hq % hkv != 0:
        raise RuntimeError(f"H_q ({hq}) must be a multiple of H_kv ({hkv})")
    if layout == "dense" and k.shape[0] not in (q.shape[0], 1):
        raise RuntimeError(f"k/v batch ({k.shape[0]}) must equal q's ({q.shape[0]}) or be 1")


def _prep_qkv(q, k, v, kv_fp8: bool = False):
    q = _aligned_view(q, 8, 16)
    kv_vec = 16 if kv_fp8 else 8
    k = _aligned_view(k, kv_vec, 16)
    v = _aligned_view(v, kv_vec, 16)
    return q, k, v


def _new_output(q: torch.Tensor) -> torch.Tensor:
    """A contiguous output of q's shape and dtype, whatever q's strides.

    The custom ops' fake kernels return ``q.new_empty(q.shape)`` (fused_attn/ops.py:102-104), which
    is contiguous, and Inductor checks a custom op's real output against the fake's strides.  The
    reference's ``torch::empty_like`` (csrc/bindings.cpp:56) keeps a ``[B,N,H,D]`` view's strides
    instead, so a compiled graph fed such a view would fail that check; a contiguous output keeps
    eager and compiled calls alike.  The kernels write through the output's strides either way."""
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def _check_out(out: torch.Tensor, q: torch.Tensor) -> None:
    """A caller-provided output must be what the kernels write: q's shape, dtype and device, unit
    D stride, 8-byte aligned with 8-byte strides (the C ABI's rule for o).  Checked before anything
    is launched, since a smaller buffer would be written past its end."""
    if tuple(out.shape) != tuple(q.shape):
        raise RuntimeError(f"out must have q's shape {tuple(q.shape)}, got {tuple(out.shape)}")
    if out.dtype != q.dtype:
        raise RuntimeError(f"out must have q's dtype {q.dtype}, got {out.dtype}")
    if out.device != q.device:
        raise RuntimeError(f"out must be on {q.device}, got {out.device}")
    vec = 8 // out.element_size()
    if out.numel() and (out.stride(-1) != 1 or out.data_ptr() % 8
                        or any(out.size(i) > 1 and out.stride(i) % vec for i in range(out.dim() - 1))):
        raise RuntimeError("out needs a unit D stride, an 8-byte aligned start and strides of whole 8-byte words")


def _check_lse_out(lse: torch.Tensor, shape: tuple, device: torch.device) -> None:
    """A caller-provided LSE: fp32 of the given shape on the device, unit stride along the last dim
    (the kernels write it through its first two strides)."""
    if tuple(lse.shape) != tuple(shape):
        raise RuntimeError(f"lse must have shape {tuple(shape)}, got {tuple(lse.shape)}")
    if lse.dtype != torch.float32:
        raise RuntimeError(f"lse must be float32, got {lse.dtype}")
    if lse.device != device:
        raise RuntimeError(f"lse must be on {device}, got {lse.device}")
    if lse.numel() and (lse.size(-1) > 1 and lse.stride(-1) != 1 or lse.stride(0) < 0 or lse.stride(1) < 0):
        raise RuntimeError("lse needs a unit stride along its last dim")


def _stride(t: torch.Tensor, i: int) -> int:
    # a size-1 dim is never stepped over; its stride is irrelevant and passed as 0
    return t.stride(i) if t.size(i) > 1 else 0


def make_params(q, k, v, o, causal: bool, scale: float, *, kv_dtype=None, lse=None, k_scale=None, v_scale=None,
                cu_seqlens_q=None, cu_seqlens_k=None, max_seqlen_q=0, max_seqlen_k=0) -> FwdParams:
    """Fill ``fa_fwd_params`` from tensors.  Dense: q/o [B,Hq,Nq,D], k/v [B,Hkv,Nk,D].
    Varlen: q/o [Tq,Hq,D], k/v [Tk,Hkv,D] with int32 cu_seqlens of length batch+1."""
    if cu_seqlens_q is None:
        # one positional constructor call (filled in C) instead of a Python attribute set per field
        qz, kz, vz, oz = q.shape, k.shape, v.shape, o.shape
        qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), o.stride()
        p = FwdParams(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
            qs[0] if qz[0] > 1 else 0, qs[1] if qz[1] > 1 else 0, qs[2] if qz[2] > 1 else 0,
            ks[0] if kz[0] > 1 else 0, ks[1] if kz[1] > 1 else 0, ks[2] if kz[2] > 1 else 0,
            vs[0] if vz[0] > 1 else 0, vs[1] if vz[1] > 1 else 0, vs[2] if vz[2] > 1 else 0,
            os_[0] if oz[0] > 1 else 0, os_[1] if oz[1] > 1 else 0, os_[2] if oz[2] > 1 else 0,
            qz[0], qz[1], kz[1], qz[2], kz[2], qz[3])
    else:
        p = FwdParams()
        p.q, p.k, p.v, p.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr()
        p.q_stride_b = p.k_stride_b = p.v_stride_b = p.o_stride_b = 0
        p.q_stride_h, p.q_stride_n = _stride(q, 1), _stride(q, 0)
        p.k_stride_h, p.k_stride_n = _stride(k, 1), _stride(k, 0)
        p.v_stride_h, p.v_stride_n = _stride(v, 1), _stride(v, 0)
        p.o_stride_h, p.o_stride_n = _stride(o, 1), _stride(o, 0)
        p.batch = cu_seqlens_q.numel() - 1
        p.heads_q, p.head_dim = q.shape[1], q.shape[2]
        p.heads_kv = k.shape[1]
        p.seqlen_q, p.seqlen_k = int(max_seqlen_q), int(max_seqlen_k)
        p.cu_seqlens_q, p.cu_seqlens_k = cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr()
        p.max_seqlen_q, p.max_seqlen_k = int(max_seqlen_q), int(max_seqlen_k)
    p.scale = float(scale)
    p.causal = 1 if causal else 0
    p.dtype = _DTYPE_CODE.get(q.dtype, -1)
    p.kv_dtype = _DTYPE_CODE.get(k.dtype if kv_dtype is None else kv_dtype, -1)
    if lse is not None:
        p.lse = lse.data_ptr()
        p.lse_stride_b, p.lse_stride_h = lse.stride(0), lse.stride(1)
    if k_scale is not None:
        p.k_scale, p.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        p.scale_stride_b, p.scale_stride_h = k_scale.stride(0), k_scale.stride(1)
    return p


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(t: torch.Tensor) -> int:
    """Handle of the current stream of t's device: the stream the op's work goes on."""
    if _raw_stream is not None:
        return _raw_stream(t.device.index)
    return torch.cuda.current_stream(t.device).cuda_stream


_SAME_DEVICE = contextlib.nullcontext()


def _on_device(dev: torch.device):
    """``torch.cuda.device(dev)``, or no device switch at all when ``dev`` is already current."""
    return _SAME_DEVICE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _require_gpu(*ts: torch.Tensor) -> None:
    dev = ts[0].device
    if dev.type != "cuda":
        raise RuntimeError("fused_attn HIP backend needs GPU tensors")
    for t in ts[1:]:
        if t.device != dev:
            raise RuntimeError(f"all tensors must be on {dev}, got {t.device}")
    if not device_supported(dev):
        raise RuntimeError(
            f"fused_attn HIP backend unavailable on {dev}: "
            + (_lib_error or "device is not a gfx950 GPU (set FUSED_ATTN_BACKEND=reference to run the unfused path)"))
    if dev.index not in _native_devices:
        _enable_native(dev.index)


# ----------------------------------------------------------------------------------------------
# entry points
# ----------------------------------------------------------------------------------------------


def fwd(q, k, v, causal: bool = False, scale: Optional[float] = None, return_lse: bool = False,
        out: Optional[torch.Tensor] = None):
    """Dense FA2 forward.  q [B,Hq,Nq,D]; k, v [B,Hkv,Nk,D]; returns o (and natural-log LSE [B,Hq,Nq])."""
    _check_qkv(q, k, v, "dense")
    if out is not None:
        _check_out(out, q)
    _require_gpu(q, k, v)
    lib = load_library()
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    q, k, v = _prep_qkv(q, k, v)
    o = _new_output(q) if out is None else out
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
    p = make_params(q, k, v, o, causal, scale, lse=lse)
    need = lib.fa_attention_fwd_workspace_bytes(p)
    ws = torch.empty(need // 4, dtype=torch.float32, device=q.device) if need else None
    with _on_device(q.device):
        _check(lib.fa_attention_fwd_ws(p, ws.data_ptr() if need else None, need, _stream(q)), "attention_fwd")
    return (o, lse) if return_lse else o


def varlen_fwd(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q: int, max_seqlen_k: int, causal: bool = False,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Packed varlen forward.  q [Tq,Hq,D]; k, v [Tk,Hkv,D]; cu_seqlens int32 [nseq+1] on the GPU.

    With ``return_lse`` also returns the natural-log LSE as fp32 [Hq, Tq]; rows of tokens outside every
    sequence are left unwritten (like the output rows)."""
    _check_qkv(q, k, v, "varlen")
    if out is not None:
        _check_out(out, q)
    _require_gpu(q, k, v, cu_seqlens_q, cu_seqlens_k)
    if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_k.dtype != torch.int32:
        raise RuntimeError("cu_seqlens must be int32")
    if cu_seqlens_q.numel() != cu_seqlens_k.numel():
        raise RuntimeError("cu_seqlens_q and cu_seqlens_k must have the same length")
    lib = load_library()
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    q, k, v = _prep_qkv(q, k, v)
    cu_q, cu_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    o = _new_output(q) if out is None else out
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device) if return_lse else None
    p = make_params(q, k, v, o, causal, scale, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=max_seqlen_q,
                    max_seqlen_k=max_seqlen_k)
    if lse is not None:  # [Hq, Tq]: head stride Tq, unit token stride
        p.lse = lse.data_ptr()
        p.lse_stride_b, p.lse_stride_h = 0, lse.stride(0)
    with _on_device(q.device):
        _check(lib.fa_attention_varlen_fwd(ctypes.byref(p), ctypes.c_void_p(_stream(q))), "attention_varlen_fwd")
    return (o, lse) if return_lse else o


def _check_fp8_scales(k: torch.Tensor, k_scale, v_scale) -> None:
    """FP8 block scales must be [B_k, Hkv, ceil(Nk / 64)] floats on k's device
    (fused_attn/fp8.py:31-45): the kernel indexes them by (batch, kv-head, 64-key block)."""
    if k_scale is None or v_scale is None:
        raise RuntimeError("FP8 K/V needs k_scale and v_scale")
    want = (k.shape[0], k.shape[1], -(-k.shape[2] // FP8_QBLOCK))
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if tuple(t.shape) != want:
            raise RuntimeError(f"{name} must have shape {want} (per 64-key block of k), got {tuple(t.shape)}")
        if not t.is_floating_point() or t.dtype == _FP8:
            raise RuntimeError(f"{name} must be a float tensor, got {t.dtype}")
        if t.device != k.device:
            raise RuntimeError(f"{name} must be on {k.device}, got {t.device}")


def _prep_fp8_scales(k: torch.Tensor, k_scale, v_scale):
    """FP8 block scales as the kernel reads them: fp32 with unit stride along the blocks and the
    same strides for both.  Scales of another float dtype are converted: the kernel reads raw
    fp32 words."""
    if k_scale.dtype != torch.float32 or k_scale.stride(-1) != 1:
        k_scale = k_scale.to(torch.float32).contiguous()
    if v_scale.dtype != torch.float32 or v_scale.stride(-1) != 1:
        v_scale = v_scale.to(torch.float32).contiguous()
    if k_scale.stride() != v_scale.stride():
        k_scale, v_scale = k_scale.contiguous(), v_scale.contiguous()
    return k_scale, v_scale


def split_len_for(seqlen_k: int, num_splits: int, block: int = FP8_QBLOCK) -> int:
    """Split length rounded up to whole ``block``-key tiles (triton_splitk.py:153-154)."""
    num_splits = max(1, int(num_splits))
    per = -(-max(seqlen_k, 1) // num_splits)
    return -(-per // block) * block


def splitk(q, k, v, causal: bool = False, scale: Optional[float] = None, split_len: int = 128,
           k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
           workspace: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Split-K flash-decoding + LSE combine.  k/v may be float8_e4m3fn with per-64-key fp32 scales.
    With ``return_lse`` also returns the natural-log LSE, fp32 [B, Hq, Nq] (-inf for rows without keys)."""
    fp8 = _FP8 is not None and k.dtype == _FP8
    _check_qkv(q, k, v, "dense", kv_fp8=fp8)
    if fp8:
        _check_fp8_scales(k, k_scale, v_scale)
    _require_gpu(q, k, v)
    lib = load_library()
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    q, k, v = _prep_qkv(q, k, v, kv_fp8=fp8)
    if fp8:
        k_scale, v_scale = _prep_fp8_scales(k, k_scale, v_scale)
    o = _new_output(q)
    b, hq, nq, d = q.shape
    nk = k.shape[2]
    splits = -(-nk // split_len) if nk > 0 else 1
    need = lib.fa_splitk_workspace_bytes(b, hq, nq, d, splits)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 16) // 4 + 4, dtype=torch.float32, device=q.device)
    lse = torch.empty((b, hq, nq), dtype=torch.float32, device=q.device) if return_lse else None
    p = make_params(q, k, v, o, causal, scale, k_scale=k_scale if fp8 else None, v_scale=v_scale if fp8 else None,
                    lse=lse)
    with _on_device(q.device):
        _check(lib.fa_attention_splitk(ctypes.byref(p), int(split_len), ctypes.c_void_p(workspace.data_ptr()),
                                       workspace.numel() * workspace.element_size(),
                                       ctypes.c_void_p(_stream(q))), "attention_splitk")
    return (o, lse) if return_lse else o


SPLITK_NOALLOC_MAX_BYTES = 64 << 20  # FA_SPLITK_NOALLOC_MAX_BYTES


def splitk_noalloc(q, k, v, causal: bool = False, scale: Optional[float] = None, split_len: int = 128,
                   k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, return_lse: bool = False,
                   lse: Optional[torch.Tensor] = None):
    """``splitk`` through fa_attention_splitk_noalloc: the library uses its own static per-GPU workspace
    (at most SPLITK_NOALLOC_MAX_BYTES) and allocates nothing; calls overlapping on one GPU race.

    A call that must allocate nothing passes ``out`` ([B,Hq,Nq,D] in q's dtype) and, for the LSE,
    ``lse`` (fp32 [B,Hq,Nq], implies ``return_lse``), with q/k/v (and FP8 scales) already in the
    kernels' layout (unit D stride, 16-byte aligned rows), so that nothing is copied either.  Both are
    checked against q before anything is launched.  Without them they are allocated here."""
    fp8 = _FP8 is not None and k.dtype == _FP8
    _check_qkv(q, k, v, "dense", kv_fp8=fp8)
    if out is not None:
        _check_out(out, q)
    if lse is not None:
        _check_lse_out(lse, q.shape[:3], q.device)
        return_lse = True
    if fp8:
        _check_fp8_scales(k, k_scale, v_scale)
    _require_gpu(q, k, v)
    lib = load_library()
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    q, k, v = _prep_qkv(q, k, v, kv_fp8=fp8)
    if fp8:
        k_scale, v_scale = _prep_fp8_scales(k, k_scale, v_scale)
    o = _new_output(q) if out is None else out
    if return_lse and lse is None:
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    p = make_params(q, k, v, o, causal, scale, k_scale=k_scale if fp8 else None, v_scale=v_scale if fp8 else None,
                    lse=lse)
    with _on_device(q.device):
        _check(lib.fa_attention_splitk_noalloc(ctypes.byref(p), int(split_len), ctypes.c_void_p(_stream(q))),
               "attention_splitk_noalloc")
    return (o, lse) if return_lse else o


def _check_paged_fp8_scales(k_cache: torch.Tensor, k_scale, v_scale) -> None:
    """FP8 pools carry 64-key block scales per page, [num_pages, Hkv, page_size / 64] floats on
    the pools' device: the kernel indexes them by (page, kv-head, block inside the page)."""
    if k_scale is None or v_scale is None:
        raise RuntimeError("FP8 pools need k_scale and v_scale")
    if k_cache.shape[2] % FP8_QBLOCK:
        raise RuntimeError(f"FP8 pools need page_size a multiple of {FP8_QBLOCK}, got {k_cache.shape[2]}")
    want = (k_cache.shape[0], k_cache.shape[1], k_cache.shape[2] // FP8_QBLOCK)
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        if tuple(t.shape) != want:
            raise RuntimeError(f"{name} must have shape {want} (per page, kv-head and 64-key block), "
                               f"got {tuple(t.shape)}")
        if not t.is_floating_point() or t.dtype == _FP8:
            raise RuntimeError(f"{name} must be a float tensor, got {t.dtype}")
        if t.device != k_cache.device:
            raise RuntimeError(f"{name} must be on {k_cache.device}, got {t.device}")


def paged_decode(q, k_cache, v_cache, block_table, seqlens_k, max_seqlen_k: int, causal: bool = False,
                 scale: Optional[float] = None, split_len: int = 128, workspace: Optional[torch.Tensor] = None,
                 return_lse: bool = False, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
    """Split-K decode over a paged cache.  q [B,Hq,Nq,D]; k_cache/v_cache [num_pages, Hkv, page_size, D]
    (any strides with unit D stride); block_table int32 [B, cols]; seqlens_k int32 [B], both on the GPU.
    FP8 pools (float8_e4m3fn) take their block scales k_scale/v_scale [num_pages, Hkv, page_size / 64].
    With ``return_lse`` also returns the natural-log LSE, fp32 [B, Hq, Nq]."""
    if k_cache.shape != v_cache.shape or k_cache.dim() != 4:
        raise RuntimeError("k_cache and v_cache must both be [num_pages, Hkv, page_size, D]")
    fp8 = k_cache.dtype == _FP8
    _check_qkv(q, k_cache, v_cache, "paged", kv_fp8=fp8)
    if fp8:
        _check_paged_fp8_scales(k_cache, k_scale, v_scale)
    _require_gpu(q, k_cache, v_cache, block_table, seqlens_k)
    if block_table.dtype != torch.int32 or seqlens_k.dtype != torch.int32:
        raise RuntimeError("block_table and seqlens_k must be int32")
    if block_table.dim() != 2 or seqlens_k.dim() != 1 or block_table.shape[0] != q.shape[0] \
            or seqlens_k.shape[0] != q.shape[0]:
        raise RuntimeError("block_table must be [B, pages] and seqlens_k [B] for q's batch B")
    lib = load_library()
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    q, k_cache, v_cache = _prep_qkv(q, k_cache, v_cache, kv_fp8=fp8)
    if fp8:
        k_scale, v_scale = _prep_fp8_scales(k_cache, k_scale, v_scale)
    bt = block_table if block_table.stride(-1) == 1 else block_table.contiguous()
    sl = seqlens_k.contiguous()
    o = _new_output(q)
    b, hq, nq, d = q.shape
    max_k = int(max_seqlen_k)
    splits = -(-max_k // split_len) if max_k > 0 else 1
    need = lib.fa_splitk_workspace_bytes(b, hq, nq, d, splits)
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(max(need, 16) // 4 + 4, dtype=torch.float32, device=q.device)
    lse = torch.empty((b, hq, nq), dtype=torch.float32, device=q.device) if return_lse else None
    p = make_params(q, k_cache, v_cache, o, causal, scale, lse=lse, k_scale=k_scale if fp8 else None,
                    v_scale=v_scale if fp8 else None)
    p.seqlen_k = max_k
    p.k_stride_b = p.v_stride_b = 0
    kv = PagedKV()
    kv.block_table, kv.block_table_stride, kv.block_table_cols = bt.data_ptr(), bt.stride(0), bt.shape[1]
    kv.page_size, kv.num_pages = k_cache.shape[2], k_cache.shape[0]
    kv.seqlens_k = sl.data_ptr()
    kv.k_page_stride, kv.v_page_stride = _stride(k_cache, 0), _stride(v_cache, 0)
    with _on_device(q.device):
        _check(lib.fa_attention_paged_decode(ctypes.byref(p), ctypes.byref(kv), int(split_len),
                                             ctypes.c_void_p(workspace.data_ptr()),
                                             workspace.numel() * workspace.element_size(),
                                             ctypes.c_void_p(_stream(q))), "attention_paged_decode")
    return (o, lse) if return_lse else o


def choose_num_splits(batch: int, heads: int, seqlen_k: int, seqlen_q: int, num_cus: int) -> int:
    return int(load_library().fa_choose_num_splits(batch, heads, seqlen_k, seqlen_q, num_cus))


def workspace_bytes(batch: int, heads_q: int, seqlen_q: int, head_dim: int, num_splits: int) -> int:
    return int(load_library().fa_splitk_workspace_bytes(batch, heads_q, seqlen_q, head_dim, num_splits))


QUANT_HEAD_DIMS = (16, 32, 64, 128, 256)


def quantize_kv_fp8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Fused FP8 KV quantiser.  x [B,Hkv,N,D] fp32/fp16/bf16 on the GPU -> (float8_e4m3fn
    [B,Hkv,N,D] contiguous, fp32 scales [B,Hkv,ceil(N/64)]), bit-identical to the reference's
    torch chain on the GPU (fused_attn/fp8.py:31-45)."""
    _require_gpu(x)
    if _FP8 is None:
        raise RuntimeError("this torch build has no float8_e4m3fn")
    if x.dim() != 4:
        raise RuntimeError(f"x must be [B, H, N, D], got {tuple(x.shape)}")
    lib = load_library()
    x = _aligned_view(x, 16 // x.element_size(), 16)
    b, h, n, d = x.shape
    nblk = -(-n // FP8_QBLOCK)
    x8 = torch.empty((b, h, n, d), dtype=_FP8, device=x.device)
    scale = torch.empty((b, h, nblk), dtype=torch.float32, device=x.device)
    p = QuantParams()
    p.x, p.x8, p.scale = x.data_ptr(), x8.data_ptr(), scale.data_ptr()
    p.x_stride_b, p.x_stride_h, p.x_stride_n = _stride(x, 0), _stride(x, 1), _stride(x, 2)
    p.batch, p.heads, p.seqlen, p.head_dim = b, h, n, d
    p.dtype = _DTYPE_CODE.get(x.dtype, -1) if x.dtype != _FP8 else -1
    with _on_device(x.device):
        _check(lib.fa_quantize_kv_fp8(ctypes.byref(p), ctypes.c_void_p(_stream(x))), "quantize_kv_fp8")
    return x8, scale


# ----------------------------------------------------------------------------------------------
# 4-bit cache, scored attention, eviction
# ----------------------------------------------------------------------------------------------

INT4_HEAD_DIMS = (64, 128, 256)


def _strides3(t: torch.Tensor, unit: int = 1) -> tuple[int, int, int]:
    z, s = t.shape, t.stride()
    return (s[0] // unit if z[0] > 1 else 0, s[1] // unit if z[1] > 1 else 0, s[2] // unit if z[2] > 1 else 0)


def _aligned_rows(t: torch.Tensor, vec: int) -> torch.Tensor:
    """``_aligned_view`` for rows of whole 16 bytes: a contiguous tensor needs only its start looked at."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else _aligned_view(t, vec, 16)


def _pairs_ok(t: torch.Tensor) -> bool:
    """Whether the kernels can read t's (scale, zero) pairs as 4-byte words."""
    if t.data_ptr() % 4:
        return False
    return t.is_contiguous() or (t.stride(-1) == 1 and all(
        t.size(i) <= 1 or (t.stride(i) >= 0 and t.stride(i) % 2 == 0) for i in range(3)))


def _word_pairs(t: torch.Tensor) -> torch.Tensor:
    ok = _pairs_ok(t) and t.stride(2) * 2 < TOKEN_STRIDE_LIMIT_BYTES
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def check_int4_rows(codes: torch.Tensor, scale: torch.Tensor, name: str, shape=None) -> None:
    """4-bit rows: uint8 codes [B, Hkv, N, D/2] (or a pool of pages) and fp16 pairs [B, Hkv, N, 2]."""
    cs = codes.shape
    if len(cs) != 4 or codes.dtype != torch.uint8:
        raise RuntimeError(f"{name} must be uint8 [B, Hkv, N, D/2], got {codes.dtype} {tuple(cs)}")
    if shape is not None and cs != shape:
        raise RuntimeError(f"{name} must have shape {tuple(shape)}, got {tuple(cs)}")
    ss = scale.shape if isinstance(scale, torch.Tensor) else ()
    if len(ss) != 4 or ss[3] != 2 or ss[:3] != cs[:3] or scale.dtype != torch.float16:
        got = f"{scale.dtype} {tuple(ss)}" if isinstance(scale, torch.Tensor) else scale
        raise RuntimeError(f"the scale of {name} must be float16 {(*cs[:3], 2)}, (scale, zero) a row, got {got}")
    if scale.device != codes.device:
        raise RuntimeError(f"the scale of {name} must be on {codes.device}, got {scale.device}")


def _check_int4_writable(codes: torch.Tensor, scale: torch.Tensor, name: str) -> None:
    """Rows that are written in place cannot be copied into another layout first."""
    sizes = range(3)
    if codes.numel() and (codes.stride(-1) != 1 or codes.data_ptr() % 4
                          or any(codes.size(i) > 1 and (codes.stride(i) <= 0 or codes.stride(i) % 4) for i in sizes)):
        raise RuntimeError(f"{name} needs a unit last stride, a 4-byte aligned start and strides of whole 4-byte words")
    if scale.numel() and not (_pairs_ok(scale) and all(scale.size(i) <= 1 or scale.stride(i) > 0 for i in sizes)):
        raise RuntimeError(f"the scale of {name} needs a unit last stride, a 4-byte aligned start and even strides")


def _int4_params(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor) -> Int4Params:
    return Int4Params(x.data_ptr(), *_strides3(x), *x.shape, _DTYPE_CODE[x.dtype], 0, codes.data_ptr(), *_strides3(codes),
                      scale.data_ptr(), *_strides3(scale, 2))


def _check_float_rows(x: torch.Tensor, name: str = "x") -> None:
    if x.dim() != 4 or x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError(f"{name} must be float32, float16 or bfloat16 [B, Hkv, N, D], got {x.dtype} {tuple(x.shape)}")
    if x.shape[-1] not in INT4_HEAD_DIMS:
        raise RuntimeError(f"head_dim must be one of {INT4_HEAD_DIMS}, got {x.shape[-1]}")


def quantize_kv_int4(x: torch.Tensor, out=None):
    """x [B,Hkv,N,D] -> (codes uint8 [B,Hkv,N,D/2], (scale, zero) fp16 [B,Hkv,N,2]), into ``out`` if given."""
    _check_float_rows(x)
    b, h, n, d = x.shape
    shape = (b, h, n, d // 2)
    if out is not None:
        codes, scale = out
        check_int4_rows(codes, scale, "out", shape)
        _check_int4_writable(codes, scale, "out")
        _require_gpu(x, codes, scale)
    else:
        _require_gpu(x)
        codes = torch.empty(shape, dtype=torch.uint8, device=x.device)
        scale = torch.empty((b, h, n, 2), dtype=torch.float16, device=x.device)
    lib = _cache_library()
    x = _aligned_rows(x, 16 // x.element_size())
    with _on_device(x.device):
        _check(lib.fa_quantize_kv_int4(_int4_params(x, codes, scale), _stream(x)), "quantize_kv_int4")
    return codes, scale


def dequantize_kv_int4(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Values [B,Hkv,N,D] of 4-bit rows."""
    check_int4_rows(codes, scale, "codes")
    _require_gpu(codes, scale)
    x = torch.empty((*codes.shape[:3], 2 * codes.shape[3]), dtype=dtype, device=codes.device)
    _check_float_rows(x, "the result")
    lib = _cache_library()
    codes = _aligned_view(codes, 4, 4)
    scale = _word_pairs(scale)
    with _on_device(codes.device):
        _check(lib.fa_dequantize_kv_int4(_int4_params(x, codes, scale), _stream(codes)), "dequantize_kv_int4")
    return x


def check_append(k, v, k_cache, k_scale, v_cache, v_scale, seqlens_k, block_table) -> None:
    if k.shape != v.shape or k.dtype != v.dtype:
        raise RuntimeError(f"k and v must have the same shape and dtype, got {k.dtype} {tuple(k.shape)} and "
                           f"{v.dtype} {tuple(v.shape)}")
    if k.dim() != 4:
        raise RuntimeError(f"k and v must be [B, Hkv, new tokens, D], got {tuple(k.shape)}")
    b, hkv, _, d = k.shape
    for name, codes, scale in (("k_cache", k_cache, k_scale), ("v_cache", v_cache, v_scale)):
        check_int4_rows(codes, scale, name)
        if codes.shape[1] != hkv or codes.shape[3] * 2 != d or (block_table is None and codes.shape[0] != b):
            raise RuntimeError(f"{name} {tuple(codes.shape)} does not fit k {tuple(k.shape)}")
        _check_int4_writable(codes, scale, name)
    if k_cache.shape != v_cache.shape:
        raise RuntimeError(f"k_cache and v_cache must have the same shape, got {tuple(k_cache.shape)} and "
                           f"{tuple(v_cache.shape)}")
    check_lengths(seqlens_k, b)
    if block_table is not None:
        check_block_table(block_table, b)


def check_lengths(seqlens_k: torch.Tensor, b: int) -> None:
    if seqlens_k.dtype != torch.int32 or tuple(seqlens_k.shape) != (b,):
        raise RuntimeError(f"seqlens_k must be int32 [{b}], got {seqlens_k.dtype} {tuple(seqlens_k.shape)}")


def check_block_table(block_table: torch.Tensor, b: int) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != b:
        raise RuntimeError(f"block_table must be int32 [{b}, pages], got {block_table.dtype} {tuple(block_table.shape)}")


def _plain_table(block_table: torch.Tensor) -> torch.Tensor:
    ok = block_table.stride(-1) == 1 and (block_table.shape[0] <= 1 or block_table.stride(0) >= block_table.shape[1])
    return block_table if ok else block_table.contiguous()


def append_kv_int4(k, v, k_cache, k_scale, v_cache, v_scale, seqlens_k, block_table=None) -> None:
    """New tokens k, v [B,Hkv,n,D] into a 4-bit cache in place, at positions seqlens_k[b] .. + n - 1."""
    check_append(k, v, k_cache, k_scale, v_cache, v_scale, seqlens_k, block_table)
    _check_float_rows(k, "k")
    _require_gpu(k, v, k_cache, k_scale, v_cache, v_scale, seqlens_k, *([] if block_table is None else [block_table]))
    lib = _cache_library()
    vec = 16 // k.element_size()
    k, v = _aligned_rows(k, vec), _aligned_rows(v, vec)
    seqlens_k = seqlens_k.contiguous()
    if k_cache.numel() == 0:
        return
    p = Int4AppendParams(_int4_params(k, k_cache, k_scale), _int4_params(v, v_cache, v_scale), seqlens_k.data_ptr(),
                         k_cache.shape[2])
    if block_table is not None:
        if block_table.shape[1] == 0:
            return
        block_table = _plain_table(block_table)
        p.block_table, p.block_table_stride = block_table.data_ptr(), block_table.stride(0)
        p.block_table_cols, p.page_size, p.num_pages = block_table.shape[1], k_cache.shape[2], k_cache.shape[0]
    with _on_device(k.device):
        _check(lib.fa_append_kv_int4(p, _stream(k)), "append_kv_int4")


def check_cache_attention(q, k, v, k_scale, v_scale, paged: bool = False) -> bool:
    """Whether the K/V are 4-bit; raises for operands that do not describe one attention problem."""
    if q.dim() != 4 or q.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError(f"q must be float16 or bfloat16 [B, Hq, Nq, D], got {q.dtype} {tuple(q.shape)}")
    int4 = k.dtype == torch.uint8
    if not int4:
        _check_qkv(q, k, v, "dense")
        if k_scale is not None or v_scale is not None:
            raise RuntimeError("k_scale and v_scale belong to 4-bit K/V (uint8)")
        return False
    check_int4_rows(k, k_scale, "k")
    check_int4_rows(v, v_scale, "v", k.shape)
    if v.device != k.device:
        raise RuntimeError(f"all tensors must be on {k.device}, got {v.device}")
    if k.shape[3] * 2 != q.shape[3]:
        raise RuntimeError(f"q has head_dim {q.shape[3]}, the 4-bit rows {2 * k.shape[3]}")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1] != 0:
        raise RuntimeError(f"H_q ({q.shape[1]}) must be a multiple of H_kv ({k.shape[1]})")
    if not paged and k.shape[0] not in (q.shape[0], 1):
        raise RuntimeError(f"k/v batch ({k.shape[0]}) must equal q's ({q.shape[0]}) or be 1")
    return True


# Default partitions: workgroups that they make (of up to 32 rows, of 64), the shortest and longest (keys), the most
CACHE_TARGET_WGS = {16: 1024, 32: 1024, 64: 320}
MIN_CACHE_KEYS = 128
MAX_CACHE_KEYS = 4096
MAX_CACHE_SPLITS = 128


def default_cache_split_len(seqlen_q: int, seqlen_k: int, batch: int, heads_kv: int, group: int, head_dim: int) -> int:
    """Keys per partition when the caller does not choose: as long as the grid keeps about CACHE_TARGET_WGS
    workgroups, in whole rounds of a workgroup's four waves of 32 keys.

    A workgroup costs about 4 us before and after its tiles, and more with 64 rows, whose merge moves 64 KiB through LDS
    (8 heads, 128 rows each, 8191 keys, D=128 16-bit: 37 us at 512 keys, 72 at 128).  A lone sequence is cut into 128 at
    most, as long as they are of 4096 keys or fewer: the merge of more costs more than they save (2 x 54738 keys, D=256: 18
    us at 512 keys, 34 at 128).

    The length is made from the longest sequence, so ragged batches and D=64, whose keys are few bytes, would often take
    a shorter one: 48 x 8 heads of up to 8192 keys, D=64 paged, 49 us at the 4096 chosen here and 42 at 2048; 35 x 8 heads
    of 32 rows, D=64, 12618 keys 96 and 84; 1 x 8 heads of 7735 keys, D=256, scored, takes 22 at 128 and 19 at 512."""
    rows = group * seqlen_q
    block = 16 if rows <= 16 else 32 if rows <= 32 or head_dim == 256 else 64  # rows of a workgroup
    items = max(1, batch * heads_kv * -(-rows // block))
    keys = -(-max(seqlen_k, 1) // min(max(1, CACHE_TARGET_WGS[block] // items), MAX_CACHE_SPLITS))
    return int(min(max(-(-keys // 128) * 128, MIN_CACHE_KEYS), MAX_CACHE_KEYS))


def cache_attention(q, k, v, k_scale, v_scale, causal: bool, scale: float, split_len: Optional[int],
                    seqlens_k=None,
                    block_table=None, max_seqlen_k: Optional[int] = None, return_lse: bool = False, scores=None,
                    return_scores: bool = False):
    """Attention over a 4-bit cache (dense, or paged with ``block_table``), or scored attention over a dense cache.
    Returns o, then the LSE and the new scores where asked for."""
    int4 = check_cache_attention(q, k, v, k_scale, v_scale, paged=block_table is not None)
    more = [t for t in (k_scale, v_scale, seqlens_k, block_table, scores) if t is not None]
    _require_gpu(q, k, v, *more)
    (b, hq, nq, d), hkv = q.shape, k.shape[1]
    nk = k.shape[2] if block_table is None else int(max_seqlen_k)
    if block_table is not None:
        check_block_table(block_table, b)
        if nk > block_table.shape[1] * k.shape[2]:  # (a table without columns has no address that the library could see)
            raise RuntimeError(f"block_table {tuple(block_table.shape)} has fewer pages per sequence than max_seqlen_k {nk} needs")
    if seqlens_k is not None:
        check_lengths(seqlens_k, b)
        seqlens_k = seqlens_k.contiguous()
    if scores is not None:
        check_scores(scores, (b, hkv, nk))
        if scores.stride(-1) != 1 and nk > 1:
            scores = scores.contiguous()
    if split_len is None:
        split_len = default_cache_split_len(nq, nk, b, hkv, hq // hkv, d)
        if block_table is not None:  # a partition spans at most 257 pages
            split_len = min(split_len, max(64, 256 * k.shape[2] // 64 * 64))
    split_len = int(split_len)
    lib = _cache_library()
    vec = 16 if int4 else 8
    q, k, v = _aligned_rows(q, 8), _aligned_rows(k, vec), _aligned_rows(v, vec)
    o = _new_output(q)
    if int4:
        k_scale, v_scale = _word_pairs(k_scale), _word_pairs(v_scale)
        pairs = (k_scale.data_ptr(), v_scale.data_ptr(), *_strides3(k_scale, 2), *_strides3(v_scale, 2))
    else:
        pairs = (None, None, 0, 0, 0, 0, 0, 0)
    p = CacheParams(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), *_strides3(q), *_strides3(k), *_strides3(v),
                    *_strides3(o), b, hq, hkv, nq, nk, d, float(scale), int(bool(causal)), _DTYPE_CODE[q.dtype],
                    INT4 if int4 else _DTYPE_CODE[k.dtype], *pairs, None if seqlens_k is None else seqlens_k.data_ptr())
    if block_table is not None:
        block_table = _plain_table(block_table)
        p.block_table, p.block_table_stride = block_table.data_ptr(), block_table.stride(0)
        p.block_table_cols, p.page_size, p.num_pages = block_table.shape[1], k.shape[2], k.shape[0]
    lse = torch.empty((b, hq, nq), dtype=torch.float32, device=q.device) if return_lse else None
    if lse is not None:
        p.lse, p.lse_stride_b, p.lse_stride_h = lse.data_ptr(), lse.stride(0), lse.stride(1)
    new = None
    if return_scores:
        if b * hq * nq == 0:  # no query adds a weight
            new = torch.zeros((b, hkv, nk), dtype=torch.float32, device=q.device) if scores is None else scores.clone()
        else:
            new = torch.empty((b, hkv, nk), dtype=torch.float32, device=q.device)
        # a tensor without scores has no address; the library only looks whether it is asked for them, and writes none
        p.scores_out = new.data_ptr() if new.numel() else 16
        p.scores_out_stride_b, p.scores_out_stride_h = new.stride(0), new.stride(1)
        if scores is not None:
            p.scores_in, p.scores_in_stride_b, p.scores_in_stride_h = scores.data_ptr(), scores.stride(0), scores.stride(1)
    need = lib.fa_attention_cache_workspace_bytes(p, split_len)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    with _on_device(q.device):
        _check(lib.fa_attention_cache(p, split_len, ws.data_ptr(), need, _stream(q)), "attention_cache")
    got = (o,) + ((lse,) if return_lse else ()) + ((new,) if return_scores else ())
    return got if len(got) > 1 else o


def check_scores(scores: torch.Tensor, shape) -> None:
    if scores.dtype != torch.float32 or (shape is not None and tuple(scores.shape) != tuple(shape)):
        want = "float32" if shape is None else f"float32 {tuple(shape)}"
        raise RuntimeError(f"scores must be {want} [B, Hkv, Nk], got {scores.dtype} {tuple(scores.shape)}")


def _row_elems(t: torch.Tensor) -> int:
    n = 1
    for z in t.shape[3:]:
        n *= z
    return n


def _repeated(t: torch.Tensor, cut: int) -> tuple[int, int]:
    """Bytes: (common divisor of the strides of at least ``cut``, extent of what those dims repeat)."""
    size, step, last = t.element_size(), 0, 0
    for n, stride in zip(t.shape, t.stride()):
        if n > 1 and stride * size >= cut:
            step = math.gcd(step, stride * size)
        elif n > 1:
            last += (n - 1) * stride * size
    return step, last + size


def _apart(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether x and y are seen to share no byte: their whole extents are apart, or with the dims of the larger strides
    taken as repetitions at multiples of a common step, what they repeat is (halves of one buffer's rows, or of its
    positions)."""
    a, b = x.data_ptr(), y.data_ptr()
    ea, eb = _repeated(x, 1 << 62)[1], _repeated(y, 1 << 62)[1]
    if a + ea <= b or b + eb <= a:
        return True
    for cut in {s * t.element_size() for t in (x, y) for n, s in zip(t.shape, t.stride()) if n > 1 and s > 0}:
        (ga, ea), (gb, eb) = _repeated(x, cut), _repeated(y, cut)
        step = math.gcd(ga, gb)
        if step and (b - a) % step >= ea and (a - b) % step >= eb:
            return True
    return False


def check_evict(scores, caches, keep: int, recent: int, seqlens_k, out) -> None:
    if scores.dim() != 3:
        raise RuntimeError(f"scores must be float32 [B, Hkv, N], got {tuple(scores.shape)}")
    check_scores(scores, None)
    if not 0 <= recent <= keep:
        raise RuntimeError(f"need 0 <= recent <= keep, got recent {recent}, keep {keep}")
    if len(caches) > MAX_EVICT_TENSORS:
        raise RuntimeError(f"at most {MAX_EVICT_TENSORS} caches, got {len(caches)}")
    rows = min(keep, scores.shape[2])
    for t in caches:
        if t.shape[:3] != scores.shape:
            raise RuntimeError(f"a cache must be [B, Hkv, N, ...] as scores {tuple(scores.shape)}, got {tuple(t.shape)}")
        if _row_elems(t) == 0:
            raise RuntimeError(f"a cache needs rows, got {tuple(t.shape)}")
    if seqlens_k is not None:
        check_lengths(seqlens_k, scores.shape[0])
    if out is not None:
        if len(out) != len(caches):
            raise RuntimeError(f"out must hold one tensor for each of the {len(caches)} caches, got {len(out)}")
        for o, t in zip(out, caches):
            if o.dtype != t.dtype or o.dim() != t.dim() or o.shape[:2] != t.shape[:2] or o.shape[3:] != t.shape[3:] \
                    or o.shape[2] < rows:
                raise RuntimeError(f"out for a cache {t.dtype} {tuple(t.shape)} needs its type and at least {rows} rows, "
                                   f"got {o.dtype} {tuple(o.shape)}")
            if not _rows_contiguous(o) or any(o.size(i) > 1 and o.stride(i) <= 0 for i in range(3)):
                raise RuntimeError("out needs contiguous rows and positive strides")
            end = _row_elems(o)
            for stride, size in sorted((o.stride(i), o.size(i)) for i in range(3) if o.size(i) > 1):
                if stride < end:
                    raise RuntimeError("rows of out overlap")
                end += stride * (size - 1)
        written = [o for o in out if o.numel()]
        for i, o in enumerate(written):
            if not all(_apart(o, t) for t in (scores, *caches, *written[:i]) if t.numel()):
                raise RuntimeError("out must not share memory with the caches, the scores or another out")


def _rows_contiguous(t: torch.Tensor) -> bool:
    if t.is_contiguous():
        return True
    want = 1
    for i in range(t.dim() - 1, 2, -1):
        if t.size(i) > 1 and t.stride(i) != want:
            return False
        want *= t.size(i)
    return True


def evict_kv(scores, caches, keep: int, recent: int, seqlens_k, out):
    check_evict(scores, caches, keep, recent, seqlens_k, out)
    _require_gpu(scores, *caches, *([] if seqlens_k is None else [seqlens_k]), *(out or ()))
    lib = _cache_library()
    b, h, n = scores.shape
    keep, recent = min(keep, n), min(recent, n)
    if n > 1 and scores.stride(-1) != 1:
        scores = scores.contiguous()
    caches = [t if _rows_contiguous(t) else t.contiguous() for t in caches]
    seqlens_k = None if seqlens_k is None else seqlens_k.contiguous()
    dev = scores.device
    index = torch.empty((b, h, keep), dtype=torch.int32, device=dev)
    kept = torch.empty((b, h, keep), dtype=torch.float32, device=dev)
    lens = torch.empty((b,), dtype=torch.int32, device=dev)
    dst = [t.new_empty((b, h, keep, *t.shape[3:])) for t in caches] if out is None else out
    if h == 0:
        lens = torch.full((b,), n, dtype=torch.int32, device=dev) if seqlens_k is None else seqlens_k.clamp(0, n)
        return dst, kept, index, lens.clamp(max=keep)
    p = EvictParams(scores.data_ptr(), _stride(scores, 0), _stride(scores, 1),
                    None if seqlens_k is None else seqlens_k.data_ptr(), b, h, n, keep, recent, len(caches),
                    index.data_ptr(), kept.data_ptr(), lens.data_ptr())
    for i, (s, d) in enumerate(zip(caches, dst)):
        size = s.element_size()
        p.tensors[i] = EvictTensor(s.data_ptr(), d.data_ptr(), *(x * size for x in _strides3(s)),
                                   *(x * size for x in _strides3(d)), _row_elems(s) * size)
    with _on_device(dev):
        need = lib.fa_evict_kv_workspace_bytes(p)
        workspace = torch.empty(need // 4, dtype=torch.float32, device=dev) if need else None
        _check(lib.fa_evict_kv(p, workspace.data_ptr() if need else None, need, _stream(scores)), "evict_kv")
    return dst, kept, index, lens

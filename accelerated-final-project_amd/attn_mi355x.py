"""Python binding of libattn_mi355x.so (the C ABI in include/attn_mi355x.h).

This is a thin ctypes layer for tests, the benchmark and Python callers.
Device memory, streams and events come from hip_rt (ctypes over the same
libamdhip64.so.7 the library links); the compute is the library's HIP
kernels.  There is no fallback: if the shared library is missing, lib()
raises.

Drop-in functions keep the reference names and argument order
(e.g. attention_forward_optimized(Q, K, V, out, batch_sz, num_heads, len_q,
len_k, head_d), final/attention.cu:195-205) and take hip_rt.DeviceArray
objects in place of raw device pointers; like the reference they
synchronize and terminate the process on a HIP error, so the wrappers here
check shapes and dtypes first and raise ValueError instead.
"""
from __future__ import annotations

import ctypes
import os
import re
import subprocess

_PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(_PKG)
LIB_PATH = os.path.join(_PKG, "lib", "libattn_mi355x.so")
HEADER_PATH = os.path.join(ROOT, "include", "attn_mi355x.h")

# status codes (include/attn_mi355x.h)
ATN_OK = 0
ATN_ERR_NULL_POINTER = -1
ATN_ERR_BAD_DIMENSION = -2
ATN_ERR_BAD_ROTARY = -3
ATN_ERR_SIZE_OVERFLOW = -4
ATN_ERR_ALIASING = -5
ATN_ERR_NO_DEVICE = -6
ATN_ERR_HIP = -7
ATN_ERR_WORKSPACE = -8
ATN_ERR_BAD_ARGUMENT = -9
ATN_ERR_MISALIGNED = -10
ATN_ERR_DEVICE_TIMEOUT = -11
ATN_ERR_CAPTURE = -12
ATN_ERR_SCRATCH_LIMIT = -13
ATN_ERR_NOT_PREPARED = -14

ATN_DTYPE_F32 = 0
ATN_DTYPE_BF16 = 1
ATN_PE_NONE = 0
ATN_PE_ROPE = 1
ATN_PE_SINUSOIDAL = 2
ATN_ROPE_INTERLEAVED = 0
ATN_ROPE_HALF = 1
ATN_PATH_FUSED_SMALL = 1
ATN_PATH_SPLIT_D = 2
ATN_PATH_GEMM = 3
ATN_PATH_FLASH = 4


class PeDesc(ctypes.Structure):
    """atn_pe_desc."""
    _fields_ = [
        ("kind", ctypes.c_int),
        ("pairing", ctypes.c_int),
        ("rotary_dim", ctypes.c_int),
        ("apply_q", ctypes.c_int),
        ("apply_k", ctypes.c_int),
        ("base", ctypes.c_float),
        ("table_a", ctypes.c_void_p),
        ("table_b", ctypes.c_void_p),
    ]


class Tuning(ctypes.Structure):
    """atn_tuning (process-wide overrides for measurement and tests)."""
    _fields_ = [(n, ctypes.c_int) for n in (
        "fused_rows", "fused_dc", "fused_exchange", "fused_xcd", "no_fused", "no_flash",
        "gemm_fused_k",
        "workspace_cap_mib", "model_cus", "model_xccs", "preset_status", "flash_form",
        "splitd_tile", "flash_split")]


class FusedPlanInfo(ctypes.Structure):
    """atn_fused_plan_info."""
    _fields_ = [(n, ctypes.c_int) for n in (
        "rows", "dc", "nchunk", "gather1", "xcd", "workgroups", "lds")]


class CallPlanInfo(ctypes.Structure):
    """atn_call_plan_info."""
    _fields_ = [(n, ctypes.c_int) for n in (
        "path", "tiles", "flash_form", "flash_parts", "keys_once", "chunk_heads",
        "chunk_rows")] + [("scratch", ctypes.c_size_t)]


class _KvCacheDesc(ctypes.Structure):
    """atn_kv_cache."""
    _fields_ = [("K", ctypes.c_void_p), ("V", ctypes.c_void_p),
                ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
                ("len", ctypes.c_void_p), ("seen", ctypes.c_void_p),
                ("weight", ctypes.c_void_p), ("pos", ctypes.c_void_p),
                ("dtype", ctypes.c_int), ("batch", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("capacity", ctypes.c_int), ("head_d", ctypes.c_int)]


class _DraftsDesc(ctypes.Structure):
    """atn_drafts."""
    _fields_ = [("Q", ctypes.c_void_p), ("K", ctypes.c_void_p), ("V", ctypes.c_void_p),
                ("q_stride", ctypes.c_int64 * 3), ("k_stride", ctypes.c_int64 * 3),
                ("v_stride", ctypes.c_int64 * 3),
                ("count", ctypes.c_void_p), ("mask", ctypes.c_void_p),
                ("heads", ctypes.c_int), ("tokens", ctypes.c_int)]


class _PagedCacheDesc(ctypes.Structure):
    """atn_paged_cache."""
    _fields_ = [("K", ctypes.c_void_p), ("V", ctypes.c_void_p),
                ("k_stride", ctypes.c_int64 * 3), ("v_stride", ctypes.c_int64 * 3),
                ("table", ctypes.c_void_p), ("len", ctypes.c_void_p),
                ("dtype", ctypes.c_int), ("batch", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("pages", ctypes.c_int), ("page_rows", ctypes.c_int),
                ("table_pages", ctypes.c_int), ("head_d", ctypes.c_int)]


class _RotaryDesc(ctypes.Structure):
    """atn_rotary."""
    _fields_ = [("pairing", ctypes.c_int), ("rotary_dim", ctypes.c_int),
                ("freq", ctypes.c_void_p), ("amplitude", ctypes.c_float)]


class _RotatedDesc(ctypes.Structure):
    """atn_rotated."""
    _fields_ = [("inp", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("in_stride", ctypes.c_int64 * 3), ("out_stride", ctypes.c_int64 * 3),
                ("heads", ctypes.c_int)]


class _SharedPrefixDesc(ctypes.Structure):
    """atn_shared_prefix."""
    _fields_ = [("first", ctypes.c_void_p), ("rows", ctypes.c_void_p), ("groups", ctypes.c_int)]


class _RopeScaling(ctypes.Structure):
    """atn_rope_scaling."""
    _fields_ = [("kind", ctypes.c_int), ("factor", ctypes.c_double), ("original", ctypes.c_int),
                ("low", ctypes.c_double), ("high", ctypes.c_double)]


class AtnError(RuntimeError):
    def __init__(self, status: int, where: str):
        self.status = status
        hip = lib().atn_last_hip_error() if status in (ATN_ERR_HIP, ATN_ERR_NO_DEVICE) else 0
        msg = f"{where}: status {status} ({status_string(status)})"
        if hip:
            msg += f", hip error {hip}"
        super().__init__(msg)


def build(jobs: int = 8) -> None:
    """Compile lib/libattn_mi355x.so for gfx950 (always recompiles)."""
    subprocess.run(["make", "-s", "-B", "-C", _PKG, f"-j{jobs}"], check=True)


_lib = None
_vp = ctypes.c_void_p
_i = ctypes.c_int
_f = ctypes.c_float

_SIGS = {
    "atn_status_string": ([_i], ctypes.c_char_p),
    "atn_last_hip_error": ([], _i),
    "atn_device_count": ([], _i),
    "atn_attention_fwd_ex": ([_i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i,
                              ctypes.POINTER(PeDesc), _vp, ctypes.c_size_t, _vp], _i),
    "atn_attention_fwd_noalloc_ex": ([_i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i,
                                      ctypes.POINTER(PeDesc), _vp], _i),
    "atn_attention_workspace_bytes": ([_i, _i, _i, _i, _i, _i, ctypes.POINTER(PeDesc)],
                                      ctypes.c_size_t),
    "atn_pe_apply_ex": ([_i, _vp, _vp, ctypes.c_long, _i, _i, ctypes.POINTER(PeDesc), _vp], _i),
    "atn_prepare_pe_ex": ([ctypes.POINTER(PeDesc), _i, _i], _i),
    "atn_sync_status_ex": ([_vp, _i, _i, _vp], _i),
    "atn_attention_path_ex": ([_i] * 6 + [ctypes.POINTER(PeDesc)], _i),
    "atn_set_tuning_ex": ([ctypes.POINTER(Tuning)], _i),
    "atn_get_tuning_ex": ([ctypes.POINTER(Tuning)], _i),
    "atn_fused_plan_ex": ([_i] * 6 + [ctypes.POINTER(PeDesc), ctypes.POINTER(FusedPlanInfo)],
                          _i),
    "atn_call_plan_ex": ([_i] * 6 + [ctypes.POINTER(PeDesc), ctypes.c_size_t,
                                     ctypes.POINTER(CallPlanInfo)], _i),
    "atn_tree_attention_ex": ([_vp, _vp, _vp, _vp, _vp, _f, _i, _vp, ctypes.c_size_t, _vp], _i),
    "atn_tree_attention_workspace_bytes": ([_vp, _vp, _i], ctypes.c_size_t),
    "atn_cache_commit_ex": ([_vp, _vp, _vp, _vp, _i, _vp], _i),
    "atn_cache_weigh_ex": ([_vp, _vp, _vp, _vp, _vp, _i, _vp, _f, _i, _vp], _i),
    "atn_cache_evict_ex": ([_vp, _i, _i, _vp, ctypes.c_size_t, _vp], _i),
    "atn_cache_evict_workspace_bytes": ([_vp, _i], ctypes.c_size_t),
    "atn_cache_advance_ex": ([_vp, _vp, _vp, _vp, _i, _i, _vp], _i),
    "atn_rope_frequencies": ([_vp, _i, ctypes.c_double, _vp, _vp], _i),
    "atn_rotary_ex": ([_i, _vp, _vp, _i, _i, _i, _i, _vp, _i, _vp], _i),
    "atn_paged_append_ex": ([_vp, _vp, _vp, _vp, _vp, _vp, _vp], _i),
    "atn_paged_attention_ex": ([_vp, _vp, _vp, _vp, _vp, _vp, _f, _i, _vp, ctypes.c_size_t, _vp],
                               _i),
    "atn_paged_attention_workspace_bytes": ([_vp, _vp, _vp, _i], ctypes.c_size_t),
    "atn_paged_advance_ex": ([_vp, _vp, _vp], _i),
    "atn_rerun_count": ([_i], ctypes.c_long),
    "atn_retained_bytes_ex": ([], ctypes.c_size_t),
    "atn_release_ex": ([], _i),
    "attention_forward_optimized": ([_vp] * 4 + [_i] * 5, None),
    "attention_forward": ([_vp] * 4 + [_i] * 5, None),
    "attention_forward_rope_fused": ([_vp] * 6 + [_i] * 5, None),
    "attention_forward_rope_fused_v7_hybrid": ([_vp] * 4 + [_i] * 6, None),
    "attention_forward_separate_rope": ([_vp] * 8 + [_i] * 6, None),
    "rope_forward": ([_vp] * 4 + [_i] * 4, None),
    "apply_sinusoidal_embeddings": ([_vp] * 4 + [_i] * 3, None),
    "attention_forward_sinusoidal_fused": ([_vp] * 4 + [_i] * 5, None),
    "attention_forward_sinusoidal_hybrid": ([_vp] * 7 + [_i] * 5, None),
    "attention_forward_sinusoidal_separate": ([_vp] * 8 + [_i] * 5, None),
    "attention_forward_bf16": ([_vp] * 4 + [_i] * 5, None),
    "attention_forward_rope_bf16": ([_vp] * 4 + [_i] * 6, None),
    "attention_forward_rope_fused_bf16": ([_vp] * 4 + [_i] * 5, None),
    "attention_forward_sinusoidal_bf16": ([_vp] * 4 + [_i] * 5, None),
    "precompute_rope_cache": ([_vp, _vp, _i, _i, _f], None),
    "precompute_sinusoidal_table": ([_vp, _vp, _i, _i], None),
}


def lib():
    """The loaded library; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with __graft_entry__.build() "
                               "(the HIP library has no CPU fallback)")
        L = ctypes.CDLL(LIB_PATH)
        for name, (args, res) in _SIGS.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        _lib = L
    return _lib


def status_string(status: int) -> str:
    return lib().atn_status_string(status).decode()


def header_functions(path: str = HEADER_PATH) -> list[str]:
    """Names of every function declared in include/attn_mi355x.h."""
    text = open(path).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = re.findall(r"^[A-Za-z_][\w \*]*?\b([a-z_][a-z0-9_]*)\s*\(", text, flags=re.M)
    return [n for n in names if n not in ("defined",)]


def device_count() -> int:
    return lib().atn_device_count()


# ---------------------------------------------------------------- tuning
_EXCHANGE = {None: 0, "gather": 1, "rsag": 2}
_SCOPE = {None: 0, "xcd": 1, "device": 2}
_FUSED_K = {None: 0, "on": 1, "off": 2}


_FLASH_FORM = {None: 0, "4x16": 1, "8x16": 2, "4x32": 3, "8x32": 4}


def set_tuning(fused_rows: int = 0, fused_dc: int = 0, fused_exchange: str | None = None,
               fused_xcd: str | None = None, no_fused: bool = False, no_flash: bool = False,
               gemm_fused_k: str | None = None, workspace_cap_mib: int = 0, model_cus: int = 0,
               model_xccs: int = 0, preset_status: bool = False, flash_form: str | None = None,
               splitd_tile: int = 0, flash_split: int = 0) -> None:
    """atn_set_tuning_ex with named fields (every field not given is reset).
    flash_form: "4x16", "8x16", "4x32" or "8x32" (waves x query rows per
    wave); flash_split: 1 never split the flash kernel's keys, n >= 2 into
    n parts."""
    t = Tuning(fused_rows, fused_dc, _EXCHANGE[fused_exchange], _SCOPE[fused_xcd],
               int(no_fused), int(no_flash), _FUSED_K[gemm_fused_k], workspace_cap_mib,
               model_cus, model_xccs, int(preset_status), _FLASH_FORM[flash_form], splitd_tile,
               flash_split)
    st = lib().atn_set_tuning_ex(ctypes.byref(t))
    if st != ATN_OK:
        raise AtnError(st, "atn_set_tuning_ex")


def get_tuning() -> Tuning:
    t = Tuning()
    lib().atn_get_tuning_ex(ctypes.byref(t))
    return t


class tuning:
    """Context manager: overrides for the block, the previous ones restored
    after it (``with tuning(fused_rows=16): ...``)."""

    def __init__(self, **kw):
        self.kw = kw

    def __enter__(self):
        self.saved = get_tuning()
        set_tuning(**self.kw)
        return self

    def __exit__(self, *exc):
        lib().atn_set_tuning_ex(ctypes.byref(self.saved))
        return False


def fused_plan(dtype_code: int, B, H, Lq, Lk, D, pe: PeDesc | None = None) -> dict | None:
    """The single-launch kernel's plan for the shape (None when the shape
    does not run on it)."""
    info = FusedPlanInfo()
    r = lib().atn_fused_plan_ex(dtype_code, B, H, Lq, Lk, D,
                                ctypes.byref(pe) if pe is not None else None,
                                ctypes.byref(info))
    if r < 0:
        raise AtnError(r, "atn_fused_plan_ex")
    if r == 0:
        return None
    return {n: getattr(info, n) for n, _ in FusedPlanInfo._fields_}


def call_plan(dtype_code: int, B, H, Lq, Lk, D, pe: PeDesc | None = None,
              scratch_bytes: int = 0) -> dict:
    """What a call of the shape runs as with this much scratch (0: the cap of
    the library's own workspace)."""
    info = CallPlanInfo()
    st = lib().atn_call_plan_ex(dtype_code, B, H, Lq, Lk, D,
                                ctypes.byref(pe) if pe is not None else None, scratch_bytes,
                                ctypes.byref(info))
    if st != ATN_OK:
        raise AtnError(st, "atn_call_plan_ex")
    return {n: getattr(info, n) for n, _ in CallPlanInfo._fields_}


def rerun_count(reset: bool = False) -> int:
    return lib().atn_rerun_count(int(reset))


def retained_bytes() -> int:
    return lib().atn_retained_bytes_ex()


def release() -> None:
    st = lib().atn_release_ex()
    if st != ATN_OK:
        raise AtnError(st, "atn_release_ex")


# ---------------------------------------------------------------- array helpers
# Arguments are hip_rt.DeviceArray objects ([B,H,L,D], 'f32' or 'bf16').
def _ptr(t):
    if t is not None and getattr(t, "strides", None) is not None:
        raise ValueError("a strided array where a contiguous one is needed")
    return None if t is None else t.ptr


def _check(t, dtype, shape, name, strided=False):
    from hip_rt import DeviceArray
    if not isinstance(t, DeviceArray):
        raise ValueError(f"{name} must be a hip_rt.DeviceArray")
    if not strided and t.strides is not None:
        raise ValueError(f"{name} must be contiguous")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _dtype_code(t) -> int:
    if t.dtype == "f32":
        return ATN_DTYPE_F32
    if t.dtype == "bf16":
        return ATN_DTYPE_BF16
    raise ValueError(f"unsupported dtype {t.dtype}")


def _stream_handle(stream) -> int | None:
    """A hip_rt.Stream, a hipStream_t as an int, or None (the null stream)."""
    return stream if stream is None or isinstance(stream, int) else stream.handle


def make_pe(kind: str = "none", pairing: str = "interleaved", rotary_dim: int = 0,
            apply_q: bool = True, apply_k: bool = True, base: float = 10000.0,
            table_a=None, table_b=None) -> PeDesc | None:
    """Build an atn_pe_desc.  kind: none | rope | sinusoidal; tables are
    device arrays in the reference's layouts, or None for library tables."""
    if kind == "none":
        return None
    d = PeDesc()
    d.kind = {"rope": ATN_PE_ROPE, "sinusoidal": ATN_PE_SINUSOIDAL}[kind]
    d.pairing = {"interleaved": ATN_ROPE_INTERLEAVED, "half": ATN_ROPE_HALF}[pairing]
    d.rotary_dim = rotary_dim
    d.apply_q = int(apply_q)
    d.apply_k = int(apply_k)
    d.base = base
    d.table_a = _ptr(table_a)
    d.table_b = _ptr(table_b)
    return d


def attention_ex(Q, K, V, out=None, pe: PeDesc | None = None, workspace=None, stream=None):
    """atn_attention_fwd_ex on device arrays [B,H,L,D]; asynchronous on
    `stream` (hip_rt.Stream or None = null stream).  Raises AtnError."""
    from hip_rt import DeviceArray
    B, H, Lq, D = Q.shape
    Lk = K.shape[2]
    _check(Q, Q.dtype, (B, H, Lq, D), "Q")
    _check(K, Q.dtype, (B, H, Lk, D), "K")
    _check(V, Q.dtype, (B, H, Lk, D), "V")
    if out is None:
        out = DeviceArray(Q.shape, Q.dtype)
    _check(out, Q.dtype, (B, H, Lq, D), "out")
    ws_ptr, ws_bytes = (None, 0)
    if workspace is not None:
        ws_ptr, ws_bytes = _ptr(workspace), workspace.nbytes
    st = lib().atn_attention_fwd_ex(_dtype_code(Q), _ptr(Q), _ptr(K), _ptr(V), _ptr(out), B, H,
                                    Lq, Lk, D, ctypes.byref(pe) if pe is not None else None,
                                    ws_ptr, ws_bytes, _stream_handle(stream))
    if st != ATN_OK:
        raise AtnError(st, "atn_attention_fwd_ex")
    return out


def attention_noalloc_ex(Q, K, V, out=None, pe: PeDesc | None = None, stream=None):
    """atn_attention_fwd_noalloc_ex (scratch in the library's per-device
    static array, no allocation); raises AtnError."""
    from hip_rt import DeviceArray
    B, H, Lq, D = Q.shape
    Lk = K.shape[2]
    _check(Q, Q.dtype, (B, H, Lq, D), "Q")
    _check(K, Q.dtype, (B, H, Lk, D), "K")
    _check(V, Q.dtype, (B, H, Lk, D), "V")
    if out is None:
        out = DeviceArray(Q.shape, Q.dtype)
    _check(out, Q.dtype, (B, H, Lq, D), "out")
    st = lib().atn_attention_fwd_noalloc_ex(_dtype_code(Q), _ptr(Q), _ptr(K), _ptr(V), _ptr(out),
                                            B, H, Lq, Lk, D,
                                            ctypes.byref(pe) if pe is not None else None,
                                            _stream_handle(stream))
    if st != ATN_OK:
        raise AtnError(st, "atn_attention_fwd_noalloc_ex")
    return out


def path(dtype_code: int, B, H, Lq, Lk, D, pe: PeDesc | None = None) -> int:
    """ATN_PATH_* that atn_attention_fwd_ex takes for this shape."""
    return lib().atn_attention_path_ex(dtype_code, B, H, Lq, Lk, D,
                                       ctypes.byref(pe) if pe is not None else None)


def sync_status(workspace=None, B: int = 1, H: int = 1, stream=None) -> int:
    """atn_sync_status_ex: ATN_OK or ATN_ERR_DEVICE_TIMEOUT."""
    return lib().atn_sync_status_ex(_ptr(workspace), B, H, _stream_handle(stream))


def workspace_bytes(dtype_code: int, B, H, Lq, Lk, D, pe: PeDesc | None = None) -> int:
    return lib().atn_attention_workspace_bytes(dtype_code, B, H, Lq, Lk, D,
                                               ctypes.byref(pe) if pe is not None else None)


def pe_apply_ex(x, out, seq_len: int, pe: PeDesc, stream=None):
    """atn_pe_apply_ex over the rows of x ([..., D]); position = row % seq_len."""
    D = x.shape[-1]
    n_rows = x.size // D
    st = lib().atn_pe_apply_ex(_dtype_code(x), _ptr(x), _ptr(out), n_rows, seq_len, D,
                               ctypes.byref(pe), _stream_handle(stream))
    if st != ATN_OK:
        raise AtnError(st, "atn_pe_apply_ex")
    return out


def _dropin_check(dtype, Q, K, V, out):
    B, H, Lq, D = Q.shape
    Lk = K.shape[2]
    _check(Q, dtype, (B, H, Lq, D), "Q")
    _check(K, dtype, (B, H, Lk, D), "K")
    _check(V, dtype, (B, H, Lk, D), "V")
    _check(out, dtype, (B, H, Lq, D), "out")
    return B, H, Lq, Lk, D


def _rot_check(rotary_dim, D):
    if rotary_dim < 2 or rotary_dim > D or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and in [2, head_d]")


def attention_forward_optimized(Q, K, V, out):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K, V, out)
    lib().attention_forward_optimized(Q.ptr, K.ptr, V.ptr, out.ptr, B, H, Lq, Lk, D)
    return out


def attention_forward(Q, K, V, out):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K, V, out)
    lib().attention_forward(Q.ptr, K.ptr, V.ptr, out.ptr, B, H, Lq, Lk, D)
    return out


def attention_forward_rope_fused(Q, K, V, out, cos_cache, sin_cache):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K, V, out)
    for n, t in (("cos_cache", cos_cache), ("sin_cache", sin_cache)):
        if t.shape[-1] != D or t.size < max(Lq, Lk) * D:
            raise ValueError(f"{n} must be [>= max(len_q, len_k)][head_d]")
    lib().attention_forward_rope_fused(Q.ptr, K.ptr, V.ptr, out.ptr, _ptr(cos_cache),
                                       _ptr(sin_cache), B, H, Lq, Lk, D)
    return out


def attention_forward_rope_fused_v7_hybrid(Q, K_rotated, V, out, rotary_dim: int):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K_rotated, V, out)
    _rot_check(rotary_dim, D)
    lib().attention_forward_rope_fused_v7_hybrid(Q.ptr, K_rotated.ptr, V.ptr, out.ptr, B, H, Lq,
                                                 Lk, D, rotary_dim)
    return out


def attention_forward_separate_rope(Q, K, V, Q_rope, K_rope, out, cos_cache, sin_cache,
                                    rotary_dim: int):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K, V, out)
    _check(Q_rope, "f32", Q.shape, "Q_rope")
    _check(K_rope, "f32", K.shape, "K_rope")
    _rot_check(rotary_dim, D)
    lib().attention_forward_separate_rope(Q.ptr, K.ptr, V.ptr, Q_rope.ptr, K_rope.ptr, out.ptr,
                                          _ptr(cos_cache), _ptr(sin_cache), B, H, Lq, Lk, D,
                                          rotary_dim)
    return out


def rope_forward(x, out, cos_cache, sin_cache, rotary_dim: int, seq_len: int):
    D = x.shape[-1]
    _rot_check(rotary_dim, D)
    lib().rope_forward(_ptr(x), _ptr(out), _ptr(cos_cache), _ptr(sin_cache), x.size // D, D,
                       rotary_dim, seq_len)
    return out


def apply_sinusoidal_embeddings(x, sin_table, cos_table, out, seqlen: int):
    D = x.shape[-1]
    lib().apply_sinusoidal_embeddings(_ptr(x), _ptr(sin_table), _ptr(cos_table), _ptr(out),
                                      x.size // D,
                                      D, seqlen)
    return out


def attention_forward_sinusoidal_fused(Q, K, V, out):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K, V, out)
    lib().attention_forward_sinusoidal_fused(Q.ptr, K.ptr, V.ptr, out.ptr, B, H, Lq, Lk, D)
    return out


def attention_forward_sinusoidal_hybrid(Q, K, V, sin_table, cos_table, K_emb, out):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K, V, out)
    _check(K_emb, "f32", K.shape, "K_emb")
    lib().attention_forward_sinusoidal_hybrid(Q.ptr, K.ptr, V.ptr, _ptr(sin_table),
                                              _ptr(cos_table), K_emb.ptr, out.ptr, B, H, Lq, Lk, D)
    return out


def attention_forward_sinusoidal_separate(Q, K, V, sin_table, cos_table, Q_emb, K_emb, out):
    B, H, Lq, Lk, D = _dropin_check("f32", Q, K, V, out)
    _check(Q_emb, "f32", Q.shape, "Q_emb")
    _check(K_emb, "f32", K.shape, "K_emb")
    lib().attention_forward_sinusoidal_separate(Q.ptr, K.ptr, V.ptr, _ptr(sin_table),
                                                _ptr(cos_table), Q_emb.ptr, K_emb.ptr, out.ptr, B,
                                                H, Lq, Lk, D)
    return out


def attention_forward_bf16(Q, K, V, out):
    B, H, Lq, Lk, D = _dropin_check("bf16", Q, K, V, out)
    lib().attention_forward_bf16(Q.ptr, K.ptr, V.ptr, out.ptr, B, H, Lq, Lk, D)
    return out


def attention_forward_rope_bf16(Q, K_rotated, V, out, rotary_dim: int):
    B, H, Lq, Lk, D = _dropin_check("bf16", Q, K_rotated, V, out)
    _rot_check(rotary_dim, D)
    lib().attention_forward_rope_bf16(Q.ptr, K_rotated.ptr, V.ptr, out.ptr, B, H, Lq, Lk, D,
                                      rotary_dim)
    return out


def attention_forward_rope_fused_bf16(Q, K, V, out):
    B, H, Lq, Lk, D = _dropin_check("bf16", Q, K, V, out)
    if D % 2:
        raise ValueError("head_d must be even for RoPE")
    lib().attention_forward_rope_fused_bf16(Q.ptr, K.ptr, V.ptr, out.ptr, B, H, Lq, Lk, D)
    return out


def attention_forward_sinusoidal_bf16(Q, K, V, out):
    B, H, Lq, Lk, D = _dropin_check("bf16", Q, K, V, out)
    lib().attention_forward_sinusoidal_bf16(Q.ptr, K.ptr, V.ptr, out.ptr, B, H, Lq, Lk, D)
    return out


# ---------------------------------------------------------------- decoding over a cache
ATN_TREE_MAX_TOKENS = 256
ATN_CACHE_MAX_HEAD_D = 8192


def _strides(t, name):
    """Batch, head and row strides of a [B][heads][rows][D] array (0, 0, 0: contiguous)."""
    if t is None or t.strides is None:
        return (ctypes.c_int64 * 3)(0, 0, 0)
    if t.strides[3] != 1 and t.shape[3] != 1:
        raise ValueError(f"{name}: the elements of a row must be adjacent")
    if not any(t.strides[:3]) and max(t.shape[:3]) > 1:
        raise ValueError(f"{name}: strides 0, 0, 0 mean a contiguous array to the library")
    return (ctypes.c_int64 * 3)(*t.strides[:3])


class KvCache:
    """A key/value cache (atn_kv_cache): K and V [B][kv heads][capacity][D], `length` [B] rows in
    use, and where the calls need them `seen` [B], `weight` and `pos` [B][kv heads][capacity].
    Holds the arrays it is made of."""

    def __init__(self, K, V, length, seen=None, weight=None, pos=None):
        _check(K, K.dtype, K.shape, "K", strided=True)
        if len(K.shape) != 4:
            raise ValueError("K must be [batch][kv heads][capacity][head_d]")
        _check(V, K.dtype, K.shape, "V", strided=True)
        B, G, cap, D = K.shape
        _check(length, "i32", (B,), "length")
        for t, dt, shape, name in ((seen, "i32", (B,), "seen"), (weight, "f32", (B, G, cap), "weight"),
                                   (pos, "i32", (B, G, cap), "pos")):
            if t is not None:
                _check(t, dt, shape, name)
        self.K, self.V, self.length, self.seen, self.weight, self.pos = K, V, length, seen, weight, pos
        self.dtype, self.shape = K.dtype, (B, G, cap, D)
        self.desc = _KvCacheDesc(K.ptr, V.ptr, _strides(K, "K"), _strides(V, "V"), _ptr(length),
                                 _ptr(seen), _ptr(weight), _ptr(pos), _dtype_code(K), B, G, cap, D)


class Drafts:
    """Drafted tokens (atn_drafts): Q [B][heads][T][D], K and V [B][kv heads][T][D], `count` [B]
    tokens of each sequence, `mask` [B][T][ceil(T / 32)] words (tree_mask)."""

    def __init__(self, Q, K=None, V=None, count=None, mask=None):
        if len(Q.shape) != 4:
            raise ValueError("Q must be [batch][heads][tokens][head_d]")
        B, H, T, D = Q.shape
        _check(Q, Q.dtype, Q.shape, "Q", strided=True)
        if (K is None) != (V is None):
            raise ValueError("K and V go together")
        if K is not None:
            _check(K, Q.dtype, (B, K.shape[1], T, D), "K", strided=True)
            _check(V, Q.dtype, K.shape, "V", strided=True)
        if count is not None:
            _check(count, "i32", (B,), "count")
        if mask is not None:
            _check(mask, "i32", (B, T, (T + 31) // 32), "mask")
        self.Q, self.K, self.V, self.count, self.mask = Q, K, V, count, mask
        self.dtype, self.shape = Q.dtype, (B, H, T, D)
        self.desc = _DraftsDesc(Q.ptr, None if K is None else K.ptr, None if V is None else V.ptr,
                                _strides(Q, "Q"), _strides(K, "K"), _strides(V, "V"), _ptr(count),
                                _ptr(mask), H, T)

    def check(self, cache: KvCache) -> None:
        B, G, _, D = cache.shape
        if self.dtype != cache.dtype or self.shape[0] != B or self.shape[3] != D:
            raise ValueError(f"drafts {self.dtype} {self.shape} do not fit a cache "
                             f"{cache.dtype} {cache.shape}")
        if self.shape[1] % G:
            raise ValueError("heads must be a multiple of the cache's kv heads")
        if self.K is not None and self.K.shape[1] != G:
            raise ValueError(f"K must have the cache's {G} kv heads")


def tree_mask(parents):
    """Mask words (int32 numpy [B][T][ceil(T / 32)]) of trees given by parents [B][T]: draft t
    attends itself, its parent parents[b][t] < t and that one's ancestors; -1: none."""
    import numpy as np
    parents = np.asarray(parents)
    B, T = parents.shape
    see = np.zeros((B, T, (T + 31) // 32 * 32), dtype=bool)
    for b in range(B):
        for t in range(T):
            p = int(parents[b, t])
            if not -1 <= p < t:
                raise ValueError(f"parent {p} of draft {t} must be an earlier draft or -1")
            if p >= 0:
                see[b, t] = see[b, p]
            see[b, t, t] = True
    return np.packbits(see, axis=-1, bitorder="little").view("<i4")


class Call:
    """An entry point bound to its arguments: call it with a stream (hip_rt.Stream, hipStream_t as
    an int, or None) as often as its buffers hold new values.  Raises AtnError."""

    def __init__(self, name, args, result, keep):
        self.name, self.fn, self.args, self.result, self._keep = (name, getattr(lib(), name), args,
                                                                  result, keep)

    def __call__(self, stream=None):
        st = self.fn(*self.args, _stream_handle(stream))
        if st != ATN_OK:
            raise AtnError(st, self.name)
        return self.result


def _ref(desc):
    return ctypes.cast(ctypes.pointer(desc), _vp)


def _path_args(cache, path, accepted, tokens):
    B = cache.shape[0]
    n = tokens
    if path is not None:
        n = path.shape[-1]
        _check(path, "i32", (B, n), "path")
    if accepted is not None:
        _check(accepted, "i32", (B,), "accepted")
    return _ptr(path), _ptr(accepted), n


def tree_attention_workspace_bytes(cache: KvCache, drafts: Drafts, max_len: int = 0) -> int:
    return lib().atn_tree_attention_workspace_bytes(_ref(cache.desc), _ref(drafts.desc), max_len)


def tree_attention_call(cache: KvCache, drafts: Drafts, out=None, lse=None, scale: float = 0.0,
                        max_len: int = 0, workspace=None) -> Call:
    """atn_tree_attention_ex bound to its arguments; calling it returns out [B][heads][T][D]."""
    from hip_rt import DeviceArray
    drafts.check(cache)
    if out is None:
        out = DeviceArray(drafts.shape, drafts.dtype)
    _check(out, drafts.dtype, drafts.shape, "out", strided=True)
    if lse is not None:
        _check(lse, "f32", drafts.shape[:3], "lse")
    strides = _strides(out, "out")
    args = (_ref(cache.desc), _ref(drafts.desc), out.ptr, ctypes.cast(strides, _vp), _ptr(lse),
            scale, max_len, _ptr(workspace), workspace.nbytes if workspace is not None else 0)
    return Call("atn_tree_attention_ex", args, out, (cache, drafts, lse, strides, workspace))


def tree_attention_ex(cache, drafts, out=None, lse=None, scale=0.0, max_len=0, workspace=None,
                      stream=None):
    """atn_tree_attention_ex; asynchronous on `stream`.  Raises AtnError."""
    return tree_attention_call(cache, drafts, out, lse, scale, max_len, workspace)(stream)


def cache_commit_call(cache: KvCache, drafts: Drafts, path=None, accepted=None) -> Call:
    drafts.check(cache)
    p, a, n = _path_args(cache, path, accepted, drafts.shape[2])
    return Call("atn_cache_commit_ex", (_ref(cache.desc), _ref(drafts.desc), p, a, n), cache,
                (cache, drafts, path, accepted))


def cache_commit_ex(cache, drafts, path=None, accepted=None, stream=None):
    """atn_cache_commit_ex: accepted drafts become rows of the cache (lengths stay)."""
    return cache_commit_call(cache, drafts, path, accepted)(stream)


def cache_weigh_call(cache: KvCache, drafts: Drafts, lse, path=None, accepted=None, weight_in="own",
                     scale: float = 0.0, max_len: int = 0) -> Call:
    """weight_in: an array, None for zeros, or "own": cache.weight, in place."""
    drafts.check(cache)
    if weight_in == "own":
        weight_in = cache.weight
    _check(lse, "f32", drafts.shape[:3], "lse")
    if weight_in is not None:
        _check(weight_in, "f32", cache.shape[:3], "weight_in")
    p, a, n = _path_args(cache, path, accepted, drafts.shape[2])
    args = (_ref(cache.desc), _ref(drafts.desc), _ptr(lse), p, a, n, _ptr(weight_in), scale, max_len)
    return Call("atn_cache_weigh_ex", args, cache.weight,
                (cache, drafts, lse, path, accepted, weight_in))


def cache_weigh_ex(cache, drafts, lse, path=None, accepted=None, weight_in="own", scale=0.0,
                   max_len=0, stream=None):
    """atn_cache_weigh_ex: the rows gather the accepted drafts' attention weight."""
    return cache_weigh_call(cache, drafts, lse, path, accepted, weight_in, scale, max_len)(stream)


def cache_evict_workspace_bytes(cache: KvCache, budget: int) -> int:
    return lib().atn_cache_evict_workspace_bytes(_ref(cache.desc), budget)


def cache_evict_call(cache: KvCache, budget: int, recent: int = 0, workspace=None) -> Call:
    args = (_ref(cache.desc), budget, recent, _ptr(workspace),
            workspace.nbytes if workspace is not None else 0)
    return Call("atn_cache_evict_ex", args, cache, (cache, workspace))


def cache_evict_ex(cache, budget, recent=0, workspace=None, stream=None):
    """atn_cache_evict_ex: keeps the recent and heaviest `budget` rows of each head (lengths stay)."""
    return cache_evict_call(cache, budget, recent, workspace)(stream)


def cache_advance_call(cache: KvCache, drafts: Drafts | None = None, path=None, accepted=None,
                       limit: int = 0) -> Call:
    p, a, n = None, None, 1
    if drafts is not None:
        drafts.check(cache)
        p, a, n = _path_args(cache, path, accepted, drafts.shape[2])
    return Call("atn_cache_advance_ex",
                (_ref(cache.desc), None if drafts is None else _ref(drafts.desc), p, a, n, limit),
                cache, (cache, drafts, path, accepted))


def cache_advance_ex(cache, drafts=None, path=None, accepted=None, limit=0, stream=None):
    """atn_cache_advance_ex: the lengths take in the committed rows, then come down to `limit`."""
    return cache_advance_call(cache, drafts, path, accepted, limit)(stream)


# ---------------------------------------------------------------- serving from a paged cache
ATN_PAGED_MAX_TOKENS = 65536
_ROPE_SCALE = {None: 0, "linear": 1, "base": 2, "parts": 3}
_PAIRING = {"interleaved": ATN_ROPE_INTERLEAVED, "half": ATN_ROPE_HALF}


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None,
                     factor: float = 1.0, original: int = 0, low: float = 0.0, high: float = 0.0):
    """atn_rope_frequencies: (radians a position, float32 numpy [rotary_dim / 2]; amplitude).
    scaling: None, "linear", "base" or "parts"."""
    import numpy as np
    f = np.zeros(max(rotary_dim, 0) // 2, dtype=np.float32)
    s = _RopeScaling(_ROPE_SCALE[scaling], factor, original, low, high)
    amplitude = ctypes.c_float(0)
    st = lib().atn_rope_frequencies(f.ctypes.data, rotary_dim, base, ctypes.addressof(s),
                                    ctypes.addressof(amplitude))
    if st != ATN_OK:
        raise AtnError(st, "atn_rope_frequencies")
    return f, amplitude.value


class Rotary:
    """Rotation by position (atn_rotary): freq [rotary_dim / 2] fp32 on the device, pairing
    "interleaved" or "half", rotary_dim 0: two dims a frequency."""

    def __init__(self, freq, pairing: str = "interleaved", rotary_dim: int = 0, amplitude: float = 1.0):
        if len(freq.shape) != 1:
            raise ValueError("freq must be [rotary_dim / 2]")
        rotary_dim = rotary_dim or 2 * freq.shape[0]
        _check(freq, "f32", (rotary_dim // 2,), "freq")
        self.freq, self.rotary_dim = freq, rotary_dim
        self.desc = _RotaryDesc(_PAIRING[pairing], rotary_dim, _ptr(freq), amplitude)


def rotary_call(rotary: Rotary, tensors, pos=None, inverse: bool = False) -> Call:
    """atn_rotary_ex bound to its arguments.  tensors: up to three (x, out) of [B][heads][T][D]
    arrays, out may be x; pos [B][T]."""
    if not 1 <= len(tensors) <= 3 or len(tensors[0][0].shape) != 4:
        raise ValueError("tensors: one to three pairs of [batch][heads][tokens][head_d] arrays")
    x0 = tensors[0][0]
    B, _, T, D = x0.shape
    descs = (_RotatedDesc * len(tensors))()
    for i, (x, out) in enumerate(tensors):
        _check(x, x0.dtype, (B, x.shape[1], T, D), f"x{i}", strided=True)
        _check(out, x0.dtype, x.shape, f"out{i}", strided=True)
        descs[i] = _RotatedDesc(x.ptr, out.ptr, _strides(x, f"x{i}"), _strides(out, f"out{i}"),
                                x.shape[1])
    if pos is not None:
        _check(pos, "i32", (B, T), "pos")
    outs = tuple(out for _, out in tensors)
    args = (_dtype_code(x0), _ref(rotary.desc), ctypes.cast(descs, _vp), len(tensors), B, T, D,
            _ptr(pos), int(inverse))
    return Call("atn_rotary_ex", args, outs, (rotary, tuple(tensors), descs, pos))


def rotary_ex(rotary, tensors, pos=None, inverse=False, stream=None):
    """atn_rotary_ex: each x turned by its tokens' positions into its out (inverse: the gradient)."""
    return rotary_call(rotary, tensors, pos, inverse)(stream)


class PagedCache:
    """A paged key/value cache (atn_paged_cache): K and V [pages][kv heads][page rows][D], `table`
    [B][pages of a sequence], `length` [B] rows in use.  Holds the arrays it is made of."""

    def __init__(self, K, V, table, length):
        if len(K.shape) != 4:
            raise ValueError("K must be [pages][kv heads][page rows][head_d]")
        _check(K, K.dtype, K.shape, "K", strided=True)
        _check(V, K.dtype, K.shape, "V", strided=True)
        if len(table.shape) != 2:
            raise ValueError("table must be [batch][pages of a sequence]")
        _check(table, "i32", table.shape, "table")
        B, slots = table.shape
        _check(length, "i32", (B,), "length")
        pages, G, rows, D = K.shape
        self.K, self.V, self.table, self.length = K, V, table, length
        self.dtype, self.batch, self.kv_heads, self.head_d = K.dtype, B, G, D
        self.desc = _PagedCacheDesc(K.ptr, V.ptr, _strides(K, "K"), _strides(V, "V"), _ptr(table),
                                    _ptr(length), _dtype_code(K), B, G, pages, rows, slots, D)

    def check(self, drafts: Drafts) -> None:
        if drafts.dtype != self.dtype or drafts.shape[0] != self.batch or \
                drafts.shape[3] != self.head_d:
            raise ValueError(f"tokens {drafts.dtype} {drafts.shape} do not fit a cache {self.dtype} of "
                             f"{self.batch} sequences, head_d {self.head_d}")
        if drafts.shape[1] % self.kv_heads:
            raise ValueError("heads must be a multiple of the cache's kv heads")
        if drafts.K is not None and drafts.K.shape[1] != self.kv_heads:
            raise ValueError(f"K must have the cache's {self.kv_heads} kv heads")


class SharedPrefix:
    """Groups of sequences that begin with the same rows (atn_shared_prefix): `first` [groups + 1],
    `rows` [groups]."""

    def __init__(self, first, rows):
        if len(rows.shape) != 1:
            raise ValueError("rows must be [groups]")
        _check(rows, "i32", rows.shape, "rows")
        _check(first, "i32", (rows.shape[0] + 1,), "first")
        self.first, self.rows = first, rows
        self.desc = _SharedPrefixDesc(_ptr(first), _ptr(rows), rows.shape[0])


def paged_append_call(cache: PagedCache, drafts: Drafts, rotary: Rotary | None = None, pos=None,
                      q_out=None) -> Call:
    """atn_paged_append_ex bound to its arguments; calling it returns q_out."""
    cache.check(drafts)
    B, H, T, D = drafts.shape
    strides = None
    if q_out is not None:
        _check(q_out, drafts.dtype, drafts.shape, "q_out", strided=True)
        strides = _strides(q_out, "q_out")
    if pos is not None:
        _check(pos, "i32", (B, T), "pos")
    args = (_ref(cache.desc), _ref(drafts.desc), None if rotary is None else _ref(rotary.desc),
            _ptr(pos), None if q_out is None else q_out.ptr,
            None if strides is None else ctypes.cast(strides, _vp))
    return Call("atn_paged_append_ex", args, q_out, (cache, drafts, rotary, pos, strides))


def paged_append_ex(cache, drafts, rotary=None, pos=None, q_out=None, stream=None):
    """atn_paged_append_ex: the tokens' keys and values become rows of the cache (lengths stay)."""
    return paged_append_call(cache, drafts, rotary, pos, q_out)(stream)


def paged_attention_workspace_bytes(cache: PagedCache, drafts: Drafts,
                                    prefix: SharedPrefix | None = None, max_len: int = 0) -> int:
    return lib().atn_paged_attention_workspace_bytes(
        _ref(cache.desc), _ref(drafts.desc), None if prefix is None else _ref(prefix.desc), max_len)


def paged_attention_call(cache: PagedCache, drafts: Drafts, out=None, lse=None,
                         prefix: SharedPrefix | None = None, scale: float = 0.0, max_len: int = 0,
                         workspace=None) -> Call:
    """atn_paged_attention_ex bound to its arguments; calling it returns out [B][heads][T][D]."""
    from hip_rt import DeviceArray
    cache.check(drafts)
    if out is None:
        out = DeviceArray(drafts.shape, drafts.dtype)
    _check(out, drafts.dtype, drafts.shape, "out", strided=True)
    if lse is not None:
        _check(lse, "f32", drafts.shape[:3], "lse")
    strides = _strides(out, "out")
    args = (_ref(cache.desc), _ref(drafts.desc), None if prefix is None else _ref(prefix.desc),
            out.ptr, ctypes.cast(strides, _vp), _ptr(lse), scale, max_len, _ptr(workspace),
            workspace.nbytes if workspace is not None else 0)
    return Call("atn_paged_attention_ex", args, out, (cache, drafts, prefix, lse, strides, workspace))


def paged_attention_ex(cache, drafts, out=None, lse=None, prefix=None, scale=0.0, max_len=0,
                       workspace=None, stream=None):
    """atn_paged_attention_ex; asynchronous on `stream`.  Raises AtnError."""
    return paged_attention_call(cache, drafts, out, lse, prefix, scale, max_len, workspace)(stream)


def paged_advance_call(cache: PagedCache, drafts: Drafts) -> Call:
    cache.check(drafts)
    return Call("atn_paged_advance_ex", (_ref(cache.desc), _ref(drafts.desc)), cache, (cache, drafts))


def paged_advance_ex(cache, drafts, stream=None):
    """atn_paged_advance_ex: the lengths take in the appended rows."""
    return paged_advance_call(cache, drafts)(stream)


def precompute_rope_cache(max_seq_len: int, rotary_dim: int, base: float = 10000.0):
    """Host cos/sin caches [pos][rotary_dim] (final/rope.cu:20-40) as numpy."""
    import numpy as np
    c = np.zeros((max_seq_len, rotary_dim), dtype=np.float32)
    s = np.zeros((max_seq_len, rotary_dim), dtype=np.float32)
    lib().precompute_rope_cache(c.ctypes.data, s.ctypes.data, max_seq_len, rotary_dim, base)
    return c, s


def precompute_sinusoidal_table(seqlen: int, hdim: int):
    """Host sin/cos tables [pos][hdim] (final/sinusoidal.cu:838-855) as numpy."""
    import numpy as np
    s = np.zeros((seqlen, hdim), dtype=np.float32)
    c = np.zeros((seqlen, hdim), dtype=np.float32)
    lib().precompute_sinusoidal_table(s.ctypes.data, c.ctypes.data, seqlen, hdim)
    return s, c

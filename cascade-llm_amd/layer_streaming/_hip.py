"""ctypes binding to libcascade_hip.so, the gfx950 kernels of the decode path.

The C ABI is declared in ``include/cascade_hip.h``.  This module is the only
place that touches the library; everything above it passes torch tensors.
Every wrapper validates device, dtype, contiguity and size before launching,
because a host pointer or a short buffer reaching a kernel would fault the
GPU.  ``torch`` is imported first so the library binds to the HIP runtime
torch already loaded (both carry the same SONAME), which makes torch's
streams and device pointers valid here.

There is no fallback: if the library is missing or fails to load, every
entry point raises :class:`HipLibraryError`.
"""

import contextlib
import ctypes
import operator
import os
import threading
import weakref

import torch

from .w4 import W4Matrix

__all__ = [
    "HipLibraryError",
    "HipCallError",
    "HipEvent",
    "library_path",
    "load",
    "exported_symbols",
]

_PACKAGE_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIBRARY_NAME = "libcascade_hip.so"

_I64 = ctypes.c_int64
_P = ctypes.c_void_p
_F = ctypes.c_float
_D = ctypes.c_double
_INT = ctypes.c_int
_SZ = ctypes.c_size_t
_U64 = ctypes.c_uint64

# name -> (restype, argtypes); mirrors include/cascade_hip.h exactly.
_SIGNATURES = {
    "cascade_abi_version": (_INT, []),
    "cascade_error_string": (ctypes.c_char_p, [_INT]),
    "cascade_rmsnorm_bf16": (_INT, [_P, _P, _P, _I64, _I64, _F, _P]),
    "cascade_gemv_bf16": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "cascade_gemv_residual_bf16": (_INT, [_P, _P, _P, _P, _I64, _I64, _P]),
    "cascade_qkv_rope_bf16": (
        _INT,
        [_P, _P, _P, _I64, _I64, _I64, _I64, _P, _P, _F, _P, _P, _P, _P, _P,
         _I64, _P],
    ),
    "cascade_qkv_rope_at_bf16": (
        _INT,
        [_P, _P, _P, _I64, _I64, _I64, _I64, _P, _P, _F, _P, _P, _P, _P, _P,
         _I64, _P, _I64, _P],
    ),
    "cascade_gate_up_swiglu_bf16": (
        _INT, [_P, _P, _I64, _I64, _P, _P, _F, _P, _P]),
    "cascade_gate_silu_bf16": (_INT, [_P, _I64, _I64, _P, _P, _F, _P, _P]),
    "cascade_up_mul_bf16": (_INT, [_P, _I64, _I64, _P, _P, _F, _P, _P, _P]),
    "cascade_decode_attention_workspace_bytes": (_SZ, [_I64, _I64, _I64, _I64]),
    "cascade_decode_attention_bf16": (
        _INT,
        [_P, _P, _P, _I64, _I64, _I64, _I64, _I64, _F, _P, _P, _SZ, _P],
    ),
    "cascade_decode_attention_at_bf16": (
        _INT,
        [_P, _P, _P, _I64, _P, _I64, _I64, _I64, _I64, _F, _P, _P, _SZ, _P],
    ),
    "cascade_decode_attention_fused_bf16": (
        _INT,
        [_P, _P, _P, _I64, _I64, _I64, _I64, _I64, _F, _P, _P, _SZ, _P, _P, _P],
    ),
    "cascade_decode_attention_fused_at_bf16": (
        _INT,
        [_P, _P, _P, _I64, _P, _I64, _I64, _I64, _I64, _F, _P, _P, _SZ, _P, _P,
         _P],
    ),
    "cascade_decode_attention_noalloc_bf16": (
        _INT, [_P, _P, _P, _I64, _I64, _I64, _I64, _I64, _F, _P, _P]),
    "cascade_gemm_bf16": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "cascade_gemm_residual_bf16": (
        _INT, [_P, _P, _P, _P, _I64, _I64, _I64, _P]),
    "cascade_gemm_f32out_bf16": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "cascade_gate_up_swiglu_gemm_bf16": (
        _INT, [_P, _P, _P, _P, _I64, _I64, _I64, _P]),
    "cascade_gate_silu_gemm_bf16": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "cascade_up_mul_gemm_bf16": (
        _INT, [_P, _P, _P, _P, _I64, _I64, _I64, _P]),
    "cascade_qkv_rope_gemm_bf16": (
        _INT,
        [_P, _I64, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _P, _I64, _I64, _P,
         _P, _P, _I64, _I64, _P],
    ),
    "cascade_prefill_attention_bf16": (
        _INT, [_P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F, _P, _P]),
    "cascade_lm_head_workspace_bytes": (_SZ, [_I64, _I64]),
    "cascade_lm_head_topk_bf16": (
        _INT,
        [_P, _I64, _I64, _I64, _P, _I64, _INT, _P, _P, _SZ, _P, _P, _P],
    ),
    "cascade_topk_f32": (_INT, [_P, _I64, _I64, _P, _SZ, _P, _P, _P]),
    "cascade_gemm_workspace_bytes": (_SZ, [_I64, _I64, _I64]),
    "cascade_gemm_ws_bf16": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P, _SZ, _P]),
    "cascade_gemm_residual_ws_bf16": (
        _INT, [_P, _P, _P, _P, _I64, _I64, _I64, _P, _SZ, _P]),
    "cascade_paged_append_bf16": (
        _INT,
        [_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I64, _I64, _I64, _I64,
         _P, _P, _P, _I64, _I64, _I64, _P, _P, _I64, _I64, _INT, _P, _I64, _I64,
         _P, _P, _I64, _I64, _I64, _I64, _P, _P],
    ),
    "cascade_paged_append_turned_bf16": (
        _INT,
        [_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _I64, _I64, _I64, _I64,
         _P, _P, _P, _P, _I64, _I64, _I64, _P, _P, _I64, _I64, _INT, _P, _I64,
         _I64, _P, _P, _I64, _I64, _I64, _I64, _P, _P],
    ),
    "cascade_paged_attention_workspace_bytes": (
        _SZ, [_I64, _I64, _I64, _I64, _I64]),
    "cascade_paged_decode_attention_bf16": (
        _INT,
        [_P, _I64, _I64, _P, _P, _I64, _I64, _I64, _I64, _P, _I64, _I64, _P, _P,
         _I64, _I64, _I64, _I64, _I64, _F, _P, _I64, _I64, _P, _SZ, _P, _P],
    ),
    "cascade_copy_pages": (
        _INT, [_P, _I64, _I64, _I64, _I64, _P, _I64, _P, _P]),
    "cascade_paged_tree_attention_workspace_bytes": (
        _SZ, [_I64, _I64, _I64, _I64, _I64, _I64]),
    "cascade_paged_tree_attention_bf16": (
        _INT,
        [_P, _I64, _I64, _I64, _P, _P, _I64, _I64, _P, _P, _I64, _I64, _I64,
         _I64, _P, _I64, _I64, _P, _P, _I64, _I64, _I64, _I64, _F, _P, _I64,
         _I64, _P, _SZ, _P, _P],
    ),
    "cascade_paged_tree_accept": (
        _INT,
        [_P, _P, _P, _P, _I64, _I64, _I64, _P, _P, _P, _P, _I64, _I64, _I64,
         _I64, _I64, _I64, _P, _I64, _I64, _I64, _P, _P, _P, _P],
    ),
    "cascade_linear_w4_workspace_bytes": (_SZ, [_I64, _I64, _I64]),
    "cascade_linear_w4_bf16": (
        _INT,
        [_P, _I64, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _I64, _P, _I64, _P,
         _SZ, _P],
    ),
    "cascade_linear_w4_f32out_bf16": (
        _INT,
        [_P, _I64, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _I64, _P, _SZ, _P]),
    "cascade_gate_up_swiglu_w4_bf16": (
        _INT,
        [_P, _I64, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _I64,
         _P]),
    "cascade_sample_workspace_bytes": (_SZ, [_I64, _I64]),
    "cascade_sample_f32": (
        _INT,
        [_P, _I64, _I64, _I64, _P, _P, _D, _P, _I64, _P, _D, _P, _D, _P, _P, _P,
         _SZ, _P],
    ),
    "cascade_embedding_gather_bf16": (
        _INT, [_P, _I64, _I64, _P, _I64, _P, _P, _P]),
    "cascade_decode_step_begin_bf16": (
        _INT, [_P, _I64, _I64, _P, _P, _P, _P, _I64, _P, _P]),
    "cascade_memcpy_h2d_async": (_INT, [_P, _P, _SZ, _P]),
    "cascade_memcpy_d2d_async": (_INT, [_P, _P, _SZ, _P]),
    "cascade_event_create": (_INT, [ctypes.POINTER(_U64), _INT]),
    "cascade_event_destroy": (_INT, [_U64]),
    "cascade_event_record": (_INT, [_U64, _P]),
    "cascade_stream_wait_event": (_INT, [_P, _U64]),
    "cascade_event_synchronize": (_INT, [_U64]),
    "cascade_event_query": (_INT, [_U64]),
    "cascade_event_elapsed_ms": (_INT, [_U64, _U64, ctypes.POINTER(_F)]),
    "cascade_host_copy": (_INT, [_P, _P, _SZ, _INT]),
    "cascade_copy_pool_create": (_INT, [_INT, _INT, ctypes.POINTER(_U64)]),
    "cascade_copy_pool_copy": (_INT, [_U64, _P, _P, _SZ]),
    "cascade_copy_pool_info": (
        _INT, [_U64, ctypes.POINTER(_INT), ctypes.POINTER(_INT)]),
    "cascade_copy_pool_destroy": (_INT, [_U64]),
    "cascade_hbm_read": (_INT, [_P, _SZ, _P, _I64, _P]),
    "cascade_device_copy": (_INT, [_P, _P, _SZ, _P]),
    "cascade_time_next_launch": (_INT, [_U64, _U64]),
}

ABI_VERSION = 7
ESHAPE = 1003  # CASCADE_ESHAPE
# fused decode attention: sync buffer size and the bits it ors into the
# caller's error word (include/cascade_hip.h)
ATTENTION_SYNC_BYTES = 1024
ATTN_EPLACEMENT = 2
ATTN_ETIMEOUT = 4
# or-ed into a paged operator's error word by an index out of range
PAGED_ERANGE = 8
# the fused form needs one KV head per XCD and at least 8 splits of 32 rows
FUSED_ATTENTION_KV_HEADS = 8
FUSED_ATTENTION_MIN_LEN = 225


class HipLibraryError(RuntimeError):
    """libcascade_hip.so is missing, stale or failed to load."""


class HipCallError(RuntimeError):
    """A libcascade_hip entry point returned a non-zero status."""

    def __init__(self, name, code, message):
        super().__init__("{} failed ({}): {}".format(name, code, message))
        self.code = code


_lock = threading.Lock()
_lib = None


def library_path():
    """Absolute path of the in-tree library (``<package>/lib``)."""

    override = os.environ.get("CASCADE_HIP_LIBRARY")
    if override:
        return override
    return os.path.join(_PACKAGE_ROOT, "lib", LIBRARY_NAME)


def exported_symbols():
    """Names every build of the library must export."""

    return tuple(_SIGNATURES)


def load():
    """Load and type the library once; raise HipLibraryError if impossible."""

    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        path = library_path()
        if not os.path.exists(path):
            raise HipLibraryError(
                "{} is missing; build it with "
                "`python -c 'import __graft_entry__ as g; g.build()'` "
                "from the repository root".format(path)
            )
        try:
            lib = ctypes.CDLL(path)
        except OSError as error:
            raise HipLibraryError(
                "cannot load {}: {}".format(path, error)
            ) from error
        for name, (restype, argtypes) in _SIGNATURES.items():
            try:
                fn = getattr(lib, name)
            except AttributeError as error:
                raise HipLibraryError(
                    "{} does not export {}".format(path, name)
                ) from error
            fn.restype = restype
            fn.argtypes = argtypes
        version = lib.cascade_abi_version()
        if version != ABI_VERSION:
            raise HipLibraryError(
                "{} has ABI version {}, expected {}".format(
                    path, version, ABI_VERSION
                )
            )
        _lib = lib
    return _lib


def _check(name, code):
    if code != 0:
        message = load().cascade_error_string(int(code))
        raise HipCallError(
            name, int(code), message.decode() if message else "unknown"
        )


def call(name, *args):
    """Call an entry point by name and raise HipCallError on failure."""

    _check(name, getattr(load(), name)(*args))


def check(name, code):
    """Raise HipCallError when a raw entry-point call returned non-zero."""

    if code != 0:
        _check(name, code)


def bf16_weight(tensor, name, rows=None, k=None):
    """Validate a weight view once (device, dtype, layout, shape) and return
    its (rows, K); the executor then launches on raw pointers."""

    _bf16(tensor, name)
    if tensor.dim() != 2:
        raise ValueError("{} must be 2-D [rows, K]".format(name))
    n, kk = tensor.shape
    if (rows is not None and n != rows) or (k is not None and kk != k):
        raise ValueError("{} has shape {}, expected [{}, {}]".format(
            name, tuple(tensor.shape), rows, k))
    if tensor.data_ptr() % 16 or kk % 8:
        raise ValueError("{} is not 16-byte aligned".format(name))
    return n, kk


def stream_handle(stream=None, device=None):
    """Raw hipStream_t (as int) of a torch stream; default: current stream."""

    if stream is None:
        stream = torch.cuda.current_stream(device)
    return stream.cuda_stream


# --------------------------------------------------------------- validation


def require_device(tensor, name, dtype=None, min_numel=None, contiguous=True):
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("{} must be a torch.Tensor".format(name))
    if tensor.device.type != "cuda":
        raise ValueError(
            "{} must live on the GPU, got {}".format(name, tensor.device)
        )
    if dtype is not None and tensor.dtype != dtype:
        raise TypeError(
            "{} must be {}, got {}".format(name, dtype, tensor.dtype)
        )
    if contiguous and not tensor.is_contiguous():
        raise ValueError("{} must be contiguous".format(name))
    if min_numel is not None and tensor.numel() < min_numel:
        raise ValueError(
            "{} holds {} elements, needs at least {}".format(
                name, tensor.numel(), min_numel
            )
        )
    return tensor


def _bf16(tensor, name, min_numel=None):
    return require_device(tensor, name, torch.bfloat16, min_numel)


def _matrix(tensor, name):
    _bf16(tensor, name)
    if tensor.dim() != 2:
        raise ValueError("{} must be 2-D [rows, K]".format(name))
    return tensor.shape


# ------------------------------------------------------------------ kernels


def rmsnorm(x, weight, out, eps, stream=None):
    """out[r] = rmsnorm(x[r]) for every row of x (last dim = hidden)."""

    n = weight.numel()
    _bf16(weight, "weight")
    _bf16(x, "x")
    if x.numel() % n:
        raise ValueError("x width does not match the norm weight")
    rows = x.numel() // n
    _bf16(out, "out", x.numel())
    call("cascade_rmsnorm_bf16", x.data_ptr(), weight.data_ptr(),
         out.data_ptr(), rows, n, float(eps), stream_handle(stream))
    return out


def gemv(weight, x, out, stream=None):
    n, k = _matrix(weight, "weight")
    _bf16(x, "x", k)
    _bf16(out, "out", n)
    call("cascade_gemv_bf16", weight.data_ptr(), x.data_ptr(),
         out.data_ptr(), n, k, stream_handle(stream))
    return out


def gemv_residual(weight, x, residual, out, stream=None):
    n, k = _matrix(weight, "weight")
    _bf16(x, "x", k)
    _bf16(residual, "residual", n)
    _bf16(out, "out", n)
    call("cascade_gemv_residual_bf16", weight.data_ptr(), x.data_ptr(),
         residual.data_ptr(), out.data_ptr(), n, k, stream_handle(stream))
    return out


def qkv_rope(wq, wk, wv, x, norm_weight, eps, rope_cos, rope_sin, q_out,
             k_out, v_out, kv_head_stride, stream=None):
    """Fused RMSNorm + Q/K/V GEMVs + RoPE + KV write for one token.

    Any of wq / wk / wv may be None (matrix granularity).  rope_cos /
    rope_sin are the 64-entry bf16 rows of this position; k_out / v_out are
    views starting at this position of KV head 0 of the layer's cache.
    """

    k = None
    sizes = []
    for name, w in (("wq", wq), ("wk", wk), ("wv", wv)):
        if w is None:
            sizes.append(0)
            continue
        n, kk = _matrix(w, name)
        if k is not None and kk != k:
            raise ValueError("q/k/v matrices disagree on K")
        k = kk
        sizes.append(n)
    if k is None:
        raise ValueError("at least one of wq, wk, wv is required")
    nq, nk, nv = sizes
    _bf16(x, "x", k)
    if norm_weight is not None:
        _bf16(norm_weight, "norm_weight", k)
    if nq or nk:
        _bf16(rope_cos, "rope_cos", 64)
        _bf16(rope_sin, "rope_sin", 64)
    heads_k = nk // 128
    heads_v = nv // 128
    if nq:
        _bf16(q_out, "q_out", nq)
    for name, buf, heads in (("k_out", k_out, heads_k), ("v_out", v_out, heads_v)):
        if heads:
            require_device(buf, name, torch.bfloat16, contiguous=False)
            if buf.storage_offset() + (heads - 1) * kv_head_stride + 128 > (
                buf.untyped_storage().nbytes() // 2
            ):
                raise ValueError("{} cannot hold {} heads".format(name, heads))

    def ptr(t):
        return 0 if t is None else t.data_ptr()

    call(
        "cascade_qkv_rope_bf16",
        ptr(wq), ptr(wk), ptr(wv), nq, nk, nv, k,
        x.data_ptr(), ptr(norm_weight), float(eps),
        ptr(rope_cos) if (nq or nk) else 0,
        ptr(rope_sin) if (nq or nk) else 0,
        ptr(q_out) if nq else 0,
        ptr(k_out) if nk else 0,
        ptr(v_out) if nv else 0,
        int(kv_head_stride), stream_handle(stream),
    )


def gate_up_swiglu(w_gate, w_up, x, norm_weight, eps, out, stream=None):
    n, k = _matrix(w_gate, "w_gate")
    if tuple(_matrix(w_up, "w_up")) != (n, k):
        raise ValueError("gate and up matrices differ in shape")
    _bf16(x, "x", k)
    if norm_weight is not None:
        _bf16(norm_weight, "norm_weight", k)
    _bf16(out, "out", n)
    call("cascade_gate_up_swiglu_bf16", w_gate.data_ptr(), w_up.data_ptr(),
         n, k, x.data_ptr(),
         0 if norm_weight is None else norm_weight.data_ptr(), float(eps),
         out.data_ptr(), stream_handle(stream))
    return out


def gate_silu(w_gate, x, norm_weight, eps, out, stream=None):
    n, k = _matrix(w_gate, "w_gate")
    _bf16(x, "x", k)
    if norm_weight is not None:
        _bf16(norm_weight, "norm_weight", k)
    _bf16(out, "out", n)
    call("cascade_gate_silu_bf16", w_gate.data_ptr(), n, k, x.data_ptr(),
         0 if norm_weight is None else norm_weight.data_ptr(), float(eps),
         out.data_ptr(), stream_handle(stream))
    return out


def up_mul(w_up, x, norm_weight, eps, gate, out, stream=None):
    n, k = _matrix(w_up, "w_up")
    _bf16(x, "x", k)
    if norm_weight is not None:
        _bf16(norm_weight, "norm_weight", k)
    _bf16(gate, "gate", n)
    _bf16(out, "out", n)
    call("cascade_up_mul_bf16", w_up.data_ptr(), n, k, x.data_ptr(),
         0 if norm_weight is None else norm_weight.data_ptr(), float(eps),
         gate.data_ptr(), out.data_ptr(), stream_handle(stream))
    return out


# ------------------------------------------------------ prefill (M > 1)


def _rows(x, name, k):
    """Validate a token-row operand [.., M, K] and return M."""

    _bf16(x, name)
    if x.numel() % k or x.numel() == 0:
        raise ValueError("{} is not a whole number of {}-wide rows".format(name, k))
    return x.numel() // k


def gemm_workspace_bytes(m, n, k):
    """Workspace bytes of the split-K forms for this shape on the current
    device (0: these shapes run the one-pass GEMM)."""

    return int(load().cascade_gemm_workspace_bytes(int(m), int(n), int(k)))


def _ws(workspace):
    if workspace is None:
        return 0, 0
    require_device(workspace, "workspace", torch.uint8)
    return workspace.data_ptr(), workspace.numel()


def gemm(x, weight, out, stream=None, workspace=None):
    """out[M, N] = bf16(x[M, K] . weight[N, K]^T) on the matrix cores; with
    a workspace (gemm_workspace_bytes) K may be split where the tiles would
    leave CUs idle."""

    n, k = _matrix(weight, "weight")
    m = _rows(x, "x", k)
    _bf16(out, "out", m * n)
    if workspace is None:
        call("cascade_gemm_bf16", x.data_ptr(), weight.data_ptr(), out.data_ptr(),
             m, n, k, stream_handle(stream))
    else:
        ws, ws_bytes = _ws(workspace)
        call("cascade_gemm_ws_bf16", x.data_ptr(), weight.data_ptr(),
             out.data_ptr(), m, n, k, ws, ws_bytes, stream_handle(stream))
    return out


def gemm_residual(x, weight, residual, out, stream=None, workspace=None):
    """out = bf16(residual + bf16(x . weight^T)); out may be residual; with a
    workspace K may be split as in gemm()."""

    n, k = _matrix(weight, "weight")
    m = _rows(x, "x", k)
    _bf16(residual, "residual", m * n)
    _bf16(out, "out", m * n)
    if workspace is None:
        call("cascade_gemm_residual_bf16", x.data_ptr(), weight.data_ptr(),
             residual.data_ptr(), out.data_ptr(), m, n, k, stream_handle(stream))
    else:
        ws, ws_bytes = _ws(workspace)
        call("cascade_gemm_residual_ws_bf16", x.data_ptr(), weight.data_ptr(),
             residual.data_ptr(), out.data_ptr(), m, n, k, ws, ws_bytes,
             stream_handle(stream))
    return out


def gemm_f32out(x, weight, out, stream=None):
    """fp32 out[M, N] = x . weight^T (no rounding; LM-head logits)."""

    n, k = _matrix(weight, "weight")
    m = _rows(x, "x", k)
    require_device(out, "out", torch.float32, m * n)
    call("cascade_gemm_f32out_bf16", x.data_ptr(), weight.data_ptr(),
         out.data_ptr(), m, n, k, stream_handle(stream))
    return out


def gate_up_swiglu_gemm(x, w_gate, w_up, out, stream=None):
    n, k = _matrix(w_gate, "w_gate")
    if tuple(_matrix(w_up, "w_up")) != (n, k):
        raise ValueError("gate and up matrices differ in shape")
    m = _rows(x, "x", k)
    _bf16(out, "out", m * n)
    call("cascade_gate_up_swiglu_gemm_bf16", x.data_ptr(), w_gate.data_ptr(),
         w_up.data_ptr(), out.data_ptr(), m, n, k, stream_handle(stream))
    return out


def gate_silu_gemm(x, w_gate, out, stream=None):
    n, k = _matrix(w_gate, "w_gate")
    m = _rows(x, "x", k)
    _bf16(out, "out", m * n)
    call("cascade_gate_silu_gemm_bf16", x.data_ptr(), w_gate.data_ptr(),
         out.data_ptr(), m, n, k, stream_handle(stream))
    return out


def up_mul_gemm(x, w_up, gate, out, stream=None):
    n, k = _matrix(w_up, "w_up")
    m = _rows(x, "x", k)
    _bf16(gate, "gate", m * n)
    _bf16(out, "out", m * n)
    call("cascade_up_mul_gemm_bf16", x.data_ptr(), w_up.data_ptr(),
         gate.data_ptr(), out.data_ptr(), m, n, k, stream_handle(stream))
    return out


def _kv_span_ok(buf, name, heads, kv_head_stride, end_slot, head_dim=128):
    require_device(buf, name, torch.bfloat16, contiguous=False)
    if kv_head_stride < end_slot * head_dim:
        raise ValueError("{}: slot {} is outside the head stride".format(
            name, end_slot - 1))
    end = buf.storage_offset() + (heads - 1) * kv_head_stride + end_slot * head_dim
    if end > buf.untyped_storage().nbytes() // 2:
        raise ValueError("{} cannot hold {} heads up to slot {}".format(
            name, heads, end_slot))


def qkv_rope_gemm(x, wq, wk, wv, rope_cos, rope_sin, pos0, q_out, k_out,
                  v_out, kv_head_stride, slot0, stream=None):
    """Q/K/V GEMMs of M token rows + RoPE + KV write.

    rope_cos / rope_sin are whole [positions, 64] bf16 tables; row r uses
    position pos0 + r and cache slot slot0 + r; k_out / v_out start at
    position 0 of KV head 0 of the layer's cache.
    """

    k = None
    sizes = []
    for name, w in (("wq", wq), ("wk", wk), ("wv", wv)):
        if w is None:
            sizes.append(0)
            continue
        n, kk = _matrix(w, name)
        if k is not None and kk != k:
            raise ValueError("q/k/v matrices disagree on K")
        k = kk
        sizes.append(n)
    if k is None:
        raise ValueError("at least one of wq, wk, wv is required")
    nq, nk, nv = sizes
    m = _rows(x, "x", k)
    positions = 0
    if nq or nk:
        _bf16(rope_cos, "rope_cos")
        _bf16(rope_sin, "rope_sin", rope_cos.numel())
        positions = rope_cos.numel() // 64
    if nq:
        _bf16(q_out, "q_out", m * nq)
    if nk:
        _kv_span_ok(k_out, "k_out", nk // 128, kv_head_stride, slot0 + m)
    if nv:
        _kv_span_ok(v_out, "v_out", nv // 128, kv_head_stride, slot0 + m)

    def ptr(t, used=True):
        return t.data_ptr() if (used and t is not None) else 0

    call("cascade_qkv_rope_gemm_bf16", x.data_ptr(), m, ptr(wq), ptr(wk),
         ptr(wv), nq, nk, nv, k, ptr(rope_cos, nq or nk),
         ptr(rope_sin, nq or nk), positions, int(pos0), ptr(q_out, nq),
         ptr(k_out, nk), ptr(v_out, nv), int(kv_head_stride), int(slot0),
         stream_handle(stream))


def prefill_attention(q, k_cache, v_cache, kv_head_stride, past, tokens, out,
                      scale, n_q_heads=32, n_kv_heads=8, head_dim=128,
                      stream=None):
    """Causal GQA attention of ``tokens`` query rows at slots past .. past +
    tokens - 1 over a layer cache (views from position 0 of KV head 0)."""

    width = n_q_heads * head_dim
    _bf16(q, "q", tokens * width)
    _bf16(out, "out", tokens * width)
    for name, buf in (("k_cache", k_cache), ("v_cache", v_cache)):
        _kv_span_ok(buf, name, n_kv_heads, kv_head_stride, past + tokens,
                    head_dim)
    call("cascade_prefill_attention_bf16", q.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), int(kv_head_stride), int(past), int(tokens),
         n_q_heads, n_kv_heads, head_dim, float(scale), out.data_ptr(),
         stream_handle(stream))
    return out


def attention_workspace_bytes(max_len, n_q_heads=32, n_kv_heads=8,
                              head_dim=128):
    size = load().cascade_decode_attention_workspace_bytes(
        int(max_len), int(n_q_heads), int(n_kv_heads), int(head_dim)
    )
    if size == 0:
        raise ValueError("unsupported attention shape")
    return int(size)


def decode_attention(q, k_cache, v_cache, kv_head_stride, length, out,
                     workspace, scale, n_q_heads=32, n_kv_heads=8,
                     head_dim=128, stream=None):
    """One-token GQA attention over positions [0, length) of a layer cache.

    k_cache / v_cache are views starting at position 0 of KV head 0.
    """

    _bf16(q, "q", n_q_heads * head_dim)
    _bf16(out, "out", n_q_heads * head_dim)
    for name, buf in (("k_cache", k_cache), ("v_cache", v_cache)):
        require_device(buf, name, torch.bfloat16, contiguous=False)
        end = buf.storage_offset() + (n_kv_heads - 1) * kv_head_stride + (
            length * head_dim
        )
        if end > buf.untyped_storage().nbytes() // 2:
            raise ValueError("{} is too small for length {}".format(name, length))
    require_device(workspace, "workspace", torch.uint8)
    call("cascade_decode_attention_bf16", q.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), int(kv_head_stride), int(length), n_q_heads,
         n_kv_heads, head_dim, float(scale), out.data_ptr(),
         workspace.data_ptr(), workspace.numel(), stream_handle(stream))
    return out


def _length_word(length, capacity):
    require_device(length, "length", torch.int64, 1)
    if int(capacity) <= 0:
        raise ValueError("capacity must be positive")


def qkv_rope_at(wq, wk, wv, x, norm_weight, eps, rope_cos, rope_sin, q_out,
                k_cache, v_cache, kv_head_stride, length, capacity,
                stream=None):
    """q|k|v + RoPE + KV write at the position *length - 1 held on the device.

    rope_cos / rope_sin are the [capacity, 64] tables; k_cache / v_cache are
    views at position 0 of KV head 0 of the layer cache.
    """

    _length_word(length, capacity)
    nq = 0 if wq is None else _matrix(wq, "wq")[0]
    nk = 0 if wk is None else _matrix(wk, "wk")[0]
    nv = 0 if wv is None else _matrix(wv, "wv")[0]
    k = _matrix(next(w for w in (wq, wk, wv) if w is not None), "w")[1]
    _bf16(x, "x", k)
    if norm_weight is not None:
        _bf16(norm_weight, "norm_weight", k)
    if nq or nk:
        _bf16(rope_cos, "rope_cos", capacity * 64)
        _bf16(rope_sin, "rope_sin", capacity * 64)
    if nq:
        _bf16(q_out, "q_out", nq)
    for name, buf, heads in (("k_cache", k_cache, nk // 128),
                             ("v_cache", v_cache, nv // 128)):
        if heads:
            require_device(buf, name, torch.bfloat16, contiguous=False)
            if buf.storage_offset() + (heads - 1) * kv_head_stride + (
                capacity * 128
            ) > buf.untyped_storage().nbytes() // 2:
                raise ValueError("{} cannot hold {} positions".format(name, capacity))

    def ptr(t):
        return 0 if t is None else t.data_ptr()

    call("cascade_qkv_rope_at_bf16", ptr(wq), ptr(wk), ptr(wv), nq, nk, nv, k,
         x.data_ptr(), ptr(norm_weight), float(eps),
         ptr(rope_cos) if (nq or nk) else 0,
         ptr(rope_sin) if (nq or nk) else 0,
         ptr(q_out) if nq else 0, ptr(k_cache) if nk else 0,
         ptr(v_cache) if nv else 0, int(kv_head_stride), length.data_ptr(),
         int(capacity), stream_handle(stream))


def decode_attention_at(q, k_cache, v_cache, kv_head_stride, length, capacity,
                        out, workspace, scale, n_q_heads=32, n_kv_heads=8,
                        head_dim=128, stream=None):
    """decode_attention over positions [0, *length) held on the device; the
    split plan follows ``capacity``."""

    _length_word(length, capacity)
    _bf16(q, "q", n_q_heads * head_dim)
    _bf16(out, "out", n_q_heads * head_dim)
    for name, buf in (("k_cache", k_cache), ("v_cache", v_cache)):
        require_device(buf, name, torch.bfloat16, contiguous=False)
        end = buf.storage_offset() + (n_kv_heads - 1) * kv_head_stride + (
            capacity * head_dim
        )
        if end > buf.untyped_storage().nbytes() // 2:
            raise ValueError("{} is too small for capacity {}".format(name, capacity))
    require_device(workspace, "workspace", torch.uint8)
    call("cascade_decode_attention_at_bf16", q.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), int(kv_head_stride), length.data_ptr(),
         int(capacity), n_q_heads, n_kv_heads, head_dim, float(scale),
         out.data_ptr(), workspace.data_ptr(), workspace.numel(),
         stream_handle(stream))
    return out


def _fused_attention_args(sync, error_flag, n_kv_heads):
    require_device(sync, "sync", torch.uint8, ATTENTION_SYNC_BYTES)
    require_device(error_flag, "error_flag", torch.int32, 1)
    if n_kv_heads != FUSED_ATTENTION_KV_HEADS:
        raise ValueError("the fused attention needs {} KV heads".format(
            FUSED_ATTENTION_KV_HEADS))


def decode_attention_fused(q, k_cache, v_cache, kv_head_stride, length, out,
                           workspace, sync, error_flag, scale, n_q_heads=32,
                           n_kv_heads=8, head_dim=128, stream=None):
    """decode_attention with the split merge inside the attention launch
    (bit-identical results).  ``sync``: ATTENTION_SYNC_BYTES zero-filled
    bytes, left zeroed; ``error_flag``: int32 word that receives
    ATTN_EPLACEMENT / ATTN_ETIMEOUT.  length >= FUSED_ATTENTION_MIN_LEN."""

    if int(length) < FUSED_ATTENTION_MIN_LEN:
        raise ValueError("the fused attention needs length >= {}".format(
            FUSED_ATTENTION_MIN_LEN))
    _fused_attention_args(sync, error_flag, n_kv_heads)
    _bf16(q, "q", n_q_heads * head_dim)
    _bf16(out, "out", n_q_heads * head_dim)
    for name, buf in (("k_cache", k_cache), ("v_cache", v_cache)):
        require_device(buf, name, torch.bfloat16, contiguous=False)
        end = buf.storage_offset() + (n_kv_heads - 1) * kv_head_stride + (
            length * head_dim
        )
        if end > buf.untyped_storage().nbytes() // 2:
            raise ValueError("{} is too small for length {}".format(name, length))
    require_device(workspace, "workspace", torch.uint8)
    call("cascade_decode_attention_fused_bf16", q.data_ptr(), k_cache.data_ptr(),
         v_cache.data_ptr(), int(kv_head_stride), int(length), n_q_heads,
         n_kv_heads, head_dim, float(scale), out.data_ptr(),
         workspace.data_ptr(), workspace.numel(), sync.data_ptr(),
         error_flag.data_ptr(), stream_handle(stream))
    return out


def decode_attention_fused_at(q, k_cache, v_cache, kv_head_stride, length,
                              capacity, out, workspace, sync, error_flag, scale,
                              n_q_heads=32, n_kv_heads=8, head_dim=128,
                              stream=None):
    """decode_attention_at with the split merge inside the attention launch;
    capacity >= FUSED_ATTENTION_MIN_LEN."""

    _length_word(length, capacity)
    if int(capacity) < FUSED_ATTENTION_MIN_LEN:
        raise ValueError("the fused attention needs capacity >= {}".format(
            FUSED_ATTENTION_MIN_LEN))
    _fused_attention_args(sync, error_flag, n_kv_heads)
    _bf16(q, "q", n_q_heads * head_dim)
    _bf16(out, "out", n_q_heads * head_dim)
    for name, buf in (("k_cache", k_cache), ("v_cache", v_cache)):
        require_device(buf, name, torch.bfloat16, contiguous=False)
        end = buf.storage_offset() + (n_kv_heads - 1) * kv_head_stride + (
            capacity * head_dim
        )
        if end > buf.untyped_storage().nbytes() // 2:
            raise ValueError("{} is too small for capacity {}".format(name, capacity))
    require_device(workspace, "workspace", torch.uint8)
    call("cascade_decode_attention_fused_at_bf16", q.data_ptr(),
         k_cache.data_ptr(), v_cache.data_ptr(), int(kv_head_stride),
         length.data_ptr(), int(capacity), n_q_heads, n_kv_heads, head_dim,
         float(scale), out.data_ptr(), workspace.data_ptr(), workspace.numel(),
         sync.data_ptr(), error_flag.data_ptr(), stream_handle(stream))
    return out


def decode_step_begin(table, ids, out, length, history, error_flag=None,
                      stream=None):
    """Gather table[ids[0]] into out, then history[L] = ids[0] and
    *length = L + 1 (L = *length on entry, 0 <= L < history.numel())."""

    vocab, hidden = _matrix(table, "table")
    require_device(ids, "ids", torch.int64, contiguous=False)
    _bf16(out, "out", hidden)
    require_device(history, "history", torch.int64)
    _length_word(length, history.numel())
    if error_flag is not None:
        require_device(error_flag, "error_flag", torch.int32, 1)
    call("cascade_decode_step_begin_bf16", table.data_ptr(), vocab, hidden,
         ids.data_ptr(), out.data_ptr(), length.data_ptr(), history.data_ptr(),
         history.numel(), 0 if error_flag is None else error_flag.data_ptr(),
         stream_handle(stream))
    return out


def lm_head_workspace_bytes(rows, top_k):
    size = load().cascade_lm_head_workspace_bytes(int(rows), int(top_k))
    if size == 0:
        raise ValueError("unsupported LM-head shape (rows={}, top_k={})".format(
            rows, top_k))
    return int(size)


def lm_head_topk(weight, hidden, top_k, row_offset, first_chunk, workspace,
                 out_values, out_indices, logits_out=None, stream=None):
    rows, k = _matrix(weight, "weight")
    _bf16(hidden, "hidden", k)
    require_device(workspace, "workspace", torch.uint8)
    require_device(out_values, "out_values", torch.float32, top_k)
    require_device(out_indices, "out_indices", torch.int64, top_k)
    if logits_out is not None:
        require_device(logits_out, "logits_out", torch.float32, rows)
    call("cascade_lm_head_topk_bf16", weight.data_ptr(), rows, k,
         int(row_offset), hidden.data_ptr(), int(top_k),
         1 if first_chunk else 0,
         0 if logits_out is None else logits_out.data_ptr(),
         workspace.data_ptr(), workspace.numel(), out_values.data_ptr(),
         out_indices.data_ptr(), stream_handle(stream))


def topk_f32(logits, top_k, workspace, out_values, out_indices, stream=None):
    """Exact top-k of one row of fp32 logits already on the device (value
    descending, index ascending; lm_head_topk's order) into out_values /
    out_indices.  workspace: lm_head_workspace_bytes(rows, top_k) bytes."""

    require_device(logits, "logits", torch.float32)
    rows = logits.numel()
    require_device(workspace, "workspace", torch.uint8)
    require_device(out_values, "out_values", torch.float32, top_k)
    require_device(out_indices, "out_indices", torch.int64, top_k)
    call("cascade_topk_f32", logits.data_ptr(), rows, int(top_k),
         workspace.data_ptr(), workspace.numel(), out_values.data_ptr(),
         out_indices.data_ptr(), stream_handle(stream))


def embedding_gather(table, ids, out, error_flag=None, stream=None):
    vocab, hidden = _matrix(table, "table")
    require_device(ids, "ids", torch.int64)
    _bf16(out, "out", ids.numel() * hidden)
    if error_flag is not None:
        require_device(error_flag, "error_flag", torch.int32, 1)
    call("cascade_embedding_gather_bf16", table.data_ptr(), vocab, hidden,
         ids.data_ptr(), ids.numel(), out.data_ptr(),
         0 if error_flag is None else error_flag.data_ptr(),
         stream_handle(stream))
    return out


def hbm_read(src, sink, blocks=0, stream=None):
    require_device(src, "src")
    require_device(sink, "sink", torch.float32, 1)
    call("cascade_hbm_read", src.data_ptr(),
         src.numel() * src.element_size(), sink.data_ptr(), int(blocks),
         stream_handle(stream))


def device_copy(dst, src, stream=None):
    require_device(src, "src")
    require_device(dst, "dst", src.dtype, src.numel())
    call("cascade_device_copy", dst.data_ptr(), src.data_ptr(),
         src.numel() * src.element_size(), stream_handle(stream))


# ------------------------------------------- paged KV cache and sampling
# These operators take strided views, and launch on the current stream of the
# tensors' own device (or on ``stream``).  At a decode step's sizes the checks
# below would cost more than the kernels, so each wrapper first asks, in one
# expression, whether its arguments have the ordinary form; only others go
# through the checks one by one, which refuse them by name or say what the
# strides of a dimension of one stand for.

_BF16, _F32, _I32, _LONG, _U8 = (torch.bfloat16, torch.float32, torch.int32,
                                 torch.int64, torch.uint8)
# the current device, and the current stream's handle by device index, without
# the Python around them (the device is initialised: its tensors are here)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(
    torch._C, "_cuda_getCurrentRawStream") else (
        lambda index: torch.cuda.current_stream(index).cuda_stream)


def _placed(device, name, tensor, dtype, dim=None):
    """A tensor of this device, dtype and number of dimensions."""

    if not isinstance(tensor, torch.Tensor):
        raise TypeError("{} must be a torch.Tensor".format(name))
    if tensor.device != device:
        raise ValueError("{} must live on {}, got {}".format(
            name, device, tensor.device))
    if tensor.dtype != dtype:
        raise TypeError("{} must be {}, got {}".format(name, dtype, tensor.dtype))
    if dim is not None and tensor.dim() != dim:
        raise ValueError("{} must have {} dimensions".format(name, dim))
    return tensor


def _gpu_of(name, tensor):
    if not isinstance(tensor, torch.Tensor):
        raise TypeError("{} must be a torch.Tensor".format(name))
    if tensor.device.type != "cuda":
        raise ValueError("{} must live on the GPU, got {}".format(
            name, tensor.device))
    return tensor.device


def _vector(device, name, tensor, dtype, count):
    """A contiguous vector of ``count`` values."""

    _placed(device, name, tensor, dtype, 1)
    if tensor.shape[0] != count:
        raise ValueError("{} holds {} entries, expected {}".format(
            name, tensor.shape[0], count))
    if count > 1 and tensor.stride(0) != 1:
        raise ValueError("{} must be contiguous".format(name))


def _strides(name, tensor):
    """(outer, inner) strides of a [.., .., dim] view with contiguous dims."""

    outer, inner, last = tensor.stride()
    n_outer, n_inner, dim = tensor.shape
    if dim > 1 and last != 1:
        raise ValueError("{}: the last dimension must be contiguous".format(name))
    # the stride of a dimension of one says nothing
    return outer if n_outer > 1 else 0, inner if n_inner > 1 else 0


def _apart(name, tensor):
    """Refuse an output whose rows share memory (an expanded view)."""

    dim = tensor.shape[-1]
    spans = sorted((stride, size) for stride, size in zip(
        tensor.stride()[:-1], tensor.shape[:-1]) if size > 1)
    for stride, size in spans:
        if stride < dim:
            raise ValueError("{}: rows overlap".format(name))
        dim = stride * (size - 1) + dim


def _check_error_word(device, error_flag):
    if error_flag is not None:
        _placed(device, "error_flag", error_flag, torch.int32)
        if error_flag.numel() < 1:
            raise ValueError("error_flag is empty")


def _page_pools(device, k_pages, v_pages):
    """Check two [pages, kv_heads, page_size, head_dim] pools of one layout
    and return (page stride, head stride)."""

    _placed(device, "k_pages", k_pages, torch.bfloat16, 4)
    _placed(device, "v_pages", v_pages, torch.bfloat16, 4)
    page_stride, head_stride, row, last = k_pages.stride()
    if k_pages.shape != v_pages.shape or k_pages.stride() != v_pages.stride():
        raise ValueError("k_pages and v_pages differ in shape or layout")
    pages, heads, page_size, dim = k_pages.shape
    if (dim > 1 and last != 1) or (page_size > 1 and row != dim):
        raise ValueError("the rows of a page's head must be contiguous")
    if heads == 1:
        head_stride = page_size * dim
    if pages == 1:
        page_stride = heads * head_stride
    return page_stride, head_stride


def _table_stride(device, page_table):
    _placed(device, "page_table", page_table, torch.int32, 2)
    if page_table.shape[1] > 1 and page_table.stride(1) != 1:
        raise ValueError("the rows of page_table must be contiguous")
    sequences, width = page_table.shape
    stride = width if sequences == 1 else page_table.stride(0)
    if stride < width:
        raise ValueError("the rows of page_table overlap")
    return stride


def _check_bytes(device, workspace):
    _placed(device, "workspace", workspace, torch.uint8, 1)
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")


def _call_on(index, stream, name, *args):
    """Call an entry point whose last argument is the stream, with device
    ``index`` current."""

    handle = _current_stream(index) if stream is None else stream.cuda_stream
    fn = getattr(_lib or load(), name)
    if index == _current_device():
        code = fn(*args, handle)
    else:
        with torch.cuda.device(index):
            code = fn(*args, handle)
    if code != 0:
        _check(name, code)


def _check_append(q, k, v, positions, k_pages, v_pages, page_table, rows, rope,
                  q_out, rope_at, error_flag):
    """The checks of paged_append; returns the strides of q, k, v, q_out, the
    pools and the table."""

    device = _gpu_of("k", k)
    _placed(device, "k", k, torch.bfloat16, 3)
    _placed(device, "v", v, torch.bfloat16, 3)
    tokens, kv_heads, dim = k.shape
    if v.shape != k.shape:
        raise ValueError("k and v differ in shape")
    pool = _page_pools(device, k_pages, v_pages)
    if (k_pages.shape[1], k_pages.shape[3]) != (kv_heads, dim):
        raise ValueError("the pools hold {} heads of {}, the rows {} of {}".format(
            k_pages.shape[1], k_pages.shape[3], kv_heads, dim))
    q_strides = out_strides = (0, 0)
    if q is not None:
        _placed(device, "q", q, torch.bfloat16, 3)
        if q.shape != (tokens, q.shape[1], dim):
            raise ValueError("q and k differ in tokens or head size")
        q_strides = _strides("q", q)
        if q_out is not q:
            _placed(device, "q_out", q_out, torch.bfloat16, 3)
            if q_out.shape != q.shape:
                raise ValueError("q_out and q differ in shape")
        _apart("q_out", q_out)
        out_strides = _strides("q_out", q_out)
    elif q_out is not None:
        raise ValueError("q_out without q")
    table_stride = _table_stride(device, page_table)
    _vector(device, "positions", positions, torch.int32, tokens)
    if rows is not None:
        _vector(device, "rows", rows, torch.int32, tokens)
    elif tokens > page_table.shape[0]:
        raise ValueError("more tokens than page table rows (give rows)")
    if rope is not None:
        cos, sin = rope
        _placed(device, "rope cos", cos, torch.bfloat16, 2)
        _placed(device, "rope sin", sin, torch.bfloat16, 2)
        if cos.shape != sin.shape:
            raise ValueError("rope cos and sin differ in shape")
        if not (cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError("the rope tables must be contiguous")
    if rope_at is not None:
        _vector(device, "rope_at", rope_at, torch.int32, tokens)
    _check_error_word(device, error_flag)
    return q_strides, _strides("k", k), _strides("v", v), out_strides, pool, table_stride


def paged_append(q, k, v, positions, k_pages, v_pages, page_table, rows=None,
                 rope=None, interleaved=False, q_out=None, error_flag=None,
                 stream=None, rope_at=None):
    """Rotate projected rows by their positions and write K and V into pages.

    ``q`` [tokens, heads, dim] (or None), ``k`` and ``v`` [tokens, kv_heads,
    dim]: bf16 views with contiguous dims.  Token t sits at ``positions[t]``
    of page table row ``rows[t]`` (row t without ``rows``); a negative position
    or row marks padding, of which nothing is written.  ``rope``: (cos, sin)
    tables, bf16 [positions, r / 2]; the first r dims of a head turn, in pairs
    (i, i + r / 2) or, ``interleaved``, (2 i, 2 i + 1).  None copies the rows
    as they are; ``rope_at`` (int32 [tokens]) gives the tables' rows where they
    are not the positions (a drafted tree's depths).  ``q_out`` (q itself by
    default; none of its rows may be another's q, k or v) receives the rotated
    q rows and is returned.  Pools
    are [pages, kv_heads, page_size, dim] views, ``page_table`` int32
    [sequences, pages of one].  An index out of range leaves its token out
    and ors PAGED_ERANGE into ``error_flag``."""

    if q is not None and q_out is None:
        q_out = q
    q_strides = out_strides = (0, 0)
    q_heads = half = rope_positions = 0
    cos, sin = (None, None) if rope is None else rope
    try:
        index = k.get_device()
        k_strides, v_strides, pool = k.stride(), v.stride(), k_pages.stride()
        table_stride, table_last = page_table.stride()
        tokens, kv_heads, dim = shape = k.shape
        pages, pool_heads, page_size, pool_dim = pool_shape = k_pages.shape
        sequences, max_pages = page_table.shape
        ordinary = (
            tokens > 0 and pages > 1 and index >= 0
            and v.shape == shape and v_pages.shape == pool_shape
            and pool_heads == kv_heads and pool_dim == dim and v_pages.stride() == pool
            and k_strides[2] == v_strides[2] == pool[3] == table_last == 1
            and pool[2] == dim and table_stride >= max_pages
            and k.dtype is _BF16 and v.dtype is _BF16 and k_pages.dtype is _BF16
            and v_pages.dtype is _BF16 and page_table.dtype is _I32
            and positions.dtype is _I32 and index == v.get_device()
            == k_pages.get_device() == v_pages.get_device()
            == page_table.get_device() == positions.get_device()
            and positions.shape == (tokens,) and positions.is_contiguous()
            and (tokens <= sequences if rows is None else (
                rows.dtype is _I32 and rows.get_device() == index
                and rows.shape == (tokens,) and rows.is_contiguous()))
            and (rope_at is None or (
                rope_at.dtype is _I32 and rope_at.get_device() == index
                and rope_at.shape == (tokens,) and rope_at.is_contiguous()))
            and (error_flag is None or (
                error_flag.dtype is _I32 and error_flag.get_device() == index
                and error_flag.numel() > 0)))
        if q is not None:
            q_tokens, q_heads, q_dim = shape = q.shape
            q_strides, out_strides = q.stride(), (q_heads * dim, dim)
            ordinary = (
                ordinary and q_tokens == tokens and q_dim == dim and q_strides[2] == 1
                and q_out.shape == shape and q_out.is_contiguous()
                and q.dtype is _BF16 and q_out.dtype is _BF16
                and index == q.get_device() == q_out.get_device())
        elif q_out is not None:
            ordinary = False
        if rope is not None:
            rope_positions, half = shape = cos.shape
            ordinary = (
                ordinary and sin.shape == shape and cos.is_contiguous()
                and sin.is_contiguous() and cos.dtype is _BF16 and sin.dtype is _BF16
                and index == cos.get_device() == sin.get_device())
    except (AttributeError, IndexError, TypeError, ValueError, RuntimeError):
        ordinary = False
    if ordinary:
        # (the stride of a dimension of one says nothing)
        if tokens == 1:
            k_strides, v_strides = (0, k_strides[1]), (0, v_strides[1])
            q_strides = (0, q_strides[1])
        if kv_heads == 1:
            k_strides, v_strides = (k_strides[0], 0), (v_strides[0], 0)
            pool = (pool[0], page_size * dim)
        if q_heads == 1:
            q_strides = (q_strides[0], 0)
    else:
        q_strides, k_strides, v_strides, out_strides, pool, table_stride = _check_append(
            q, k, v, positions, k_pages, v_pages, page_table, rows, rope, q_out,
            rope_at, error_flag)
        index = k.get_device()
        tokens, kv_heads, dim = k.shape
        pages, _, page_size, _ = k_pages.shape
        sequences, max_pages = page_table.shape
        q_heads = 0 if q is None else q.shape[1]
        rope_positions, half = (0, 0) if rope is None else cos.shape
        if tokens == 0:
            return q_out
    rotated = (
        0 if q is None else q.data_ptr(), q_strides[0], q_strides[1], k.data_ptr(),
        k_strides[0], k_strides[1], v.data_ptr(), v_strides[0], v_strides[1], tokens,
        q_heads, kv_heads, dim, positions.data_ptr())
    placed = (
        0 if rows is None else rows.data_ptr(), page_table.data_ptr(), table_stride,
        sequences, max_pages, 0 if rope is None else cos.data_ptr(),
        0 if rope is None else sin.data_ptr(), rope_positions, 2 * half,
        1 if interleaved else 0, 0 if q is None else q_out.data_ptr(), out_strides[0],
        out_strides[1], k_pages.data_ptr(), v_pages.data_ptr(), pool[0], pool[1], pages,
        page_size, 0 if error_flag is None else error_flag.data_ptr())
    if rope_at is None:
        _call_on(index, stream, "cascade_paged_append_bf16", *rotated, *placed)
    else:
        _call_on(index, stream, "cascade_paged_append_turned_bf16", *rotated,
                 rope_at.data_ptr(), *placed)
    return q_out


def paged_attention_workspace_bytes(batch, n_q_heads, n_kv_heads, head_dim,
                                    max_length):
    """Workspace bytes of paged_decode_attention for up to ``batch`` rows of
    up to ``max_length`` positions."""

    size = load().cascade_paged_attention_workspace_bytes(
        int(batch), int(n_q_heads), int(n_kv_heads), int(head_dim),
        int(max_length))
    if size == 0:
        raise ValueError("unsupported paged attention shape")
    return int(size)


def _check_attention(q, k_pages, v_pages, page_table, lengths, out, workspace,
                     rows, error_flag):
    """The checks of paged_decode_attention; returns the strides of q, out,
    the pools and the table."""

    device = _gpu_of("q", q)
    _placed(device, "q", q, torch.bfloat16, 3)
    batch, _, dim = q.shape
    pool = _page_pools(device, k_pages, v_pages)
    if k_pages.shape[3] != dim:
        raise ValueError("the pools hold heads of {}, q of {}".format(
            k_pages.shape[3], dim))
    _placed(device, "out", out, torch.bfloat16, 3)
    if out.shape != q.shape:
        raise ValueError("out and q differ in shape")
    _apart("out", out)
    table_stride = _table_stride(device, page_table)
    sequences = page_table.shape[0]
    _vector(device, "lengths", lengths, torch.int32, sequences)
    if rows is not None:
        _vector(device, "rows", rows, torch.int32, batch)
    elif batch > sequences:
        raise ValueError("more rows than page table rows (give rows)")
    _check_bytes(device, workspace)
    _check_error_word(device, error_flag)
    return _strides("q", q), _strides("out", out), pool, table_stride


def paged_decode_attention(q, k_pages, v_pages, page_table, lengths, out,
                           workspace, scale, rows=None, max_length=None,
                           error_flag=None, stream=None):
    """One-token GQA attention of every batch row over its sequence's pages.

    ``q`` and ``out`` [batch, heads, dim]; batch row b reads positions
    [0, lengths[r]) of page table row r = ``rows[b]`` (b without ``rows``); a
    negative row is padding, whose output stays as it is.  ``lengths``: int32,
    one a table row, at most ``max_length`` (default: what a table row
    holds).  An empty sequence gives zeros.  Positions on a page outside the
    pool are left out and flagged, as are longer lengths and larger rows
    (PAGED_ERANGE in ``error_flag``).  ``workspace``:
    paged_attention_workspace_bytes(...) uint8, one each for calls that may
    overlap."""

    try:
        index = q.get_device()
        q_strides, pool = q.stride(), k_pages.stride()
        table_stride, table_last = page_table.stride()
        batch, q_heads, dim = shape = q.shape
        pages, kv_heads, page_size, pool_dim = pool_shape = k_pages.shape
        sequences, width = page_table.shape
        ordinary = (
            batch > 0 and pages > 1 and index >= 0
            and v_pages.shape == pool_shape and pool_dim == dim
            and v_pages.stride() == pool and out.shape == shape
            and q_strides[2] == pool[3] == table_last == 1 and pool[2] == dim
            and table_stride >= width
            and q.dtype is _BF16 and k_pages.dtype is _BF16 and v_pages.dtype is _BF16
            and out.dtype is _BF16 and page_table.dtype is _I32
            and lengths.dtype is _I32 and workspace.dtype is _U8
            and index == k_pages.get_device() == v_pages.get_device()
            == out.get_device() == page_table.get_device() == lengths.get_device()
            == workspace.get_device()
            and lengths.shape == (sequences,) and lengths.is_contiguous()
            and (batch <= sequences if rows is None else (
                rows.dtype is _I32 and rows.get_device() == index
                and rows.shape == (batch,) and rows.is_contiguous()))
            and out.is_contiguous()
            and workspace.dim() == 1 and workspace.is_contiguous()
            and (error_flag is None or (
                error_flag.dtype is _I32 and error_flag.get_device() == index
                and error_flag.numel() > 0)))
    except (AttributeError, IndexError, TypeError, ValueError, RuntimeError):
        ordinary = False
    if ordinary:
        # (the stride of a dimension of one says nothing)
        q_strides = (q_strides[0] if batch > 1 else 0, q_strides[1] if q_heads > 1 else 0)
        out_strides = (q_heads * dim, dim)
        if kv_heads == 1:
            pool = (pool[0], page_size * dim)
    else:
        q_strides, out_strides, pool, table_stride = _check_attention(
            q, k_pages, v_pages, page_table, lengths, out, workspace, rows,
            error_flag)
        index = q.get_device()
        batch, q_heads, dim = q.shape
        pages, kv_heads, page_size, _ = k_pages.shape
        sequences, width = page_table.shape
    if max_length is None:
        max_length = width * page_size
    elif not 0 < max_length <= width * page_size:
        raise ValueError("max_length {} is outside the page table's {}".format(
            max_length, width * page_size))
    if batch == 0:
        return out
    _call_on(
        index, stream, "cascade_paged_decode_attention_bf16", q.data_ptr(),
        q_strides[0], q_strides[1], k_pages.data_ptr(), v_pages.data_ptr(), pool[0],
        pool[1], pages, page_size, page_table.data_ptr(), table_stride, sequences,
        lengths.data_ptr(), 0 if rows is None else rows.data_ptr(), batch,
        int(max_length), q_heads, kv_heads, dim, scale, out.data_ptr(),
        out_strides[0], out_strides[1], workspace.data_ptr(), workspace.numel(),
        0 if error_flag is None else error_flag.data_ptr())
    return out


def copy_pages(pages, pairs, error_flag=None, stream=None):
    """Copy page pairs[i, 0] over page pairs[i, 1] in every plane of ``pages``.

    ``pages``: a contiguous pool [layers, 2, pages, ...], or [planes, pages,
    ...] with ``pages.dim()`` 4 or less: one layer's [2, pages, kv_heads,
    page_size, dim] is given as ``pages.flatten(2)``, and a single [pages,
    kv_heads, page_size, dim] as ``pages[None].flatten(2)``.  Five dimensions
    that may be one layer's are refused.  ``pairs``: int32 [n, 2].  The pairs
    are copied in no order: no destination may occur twice or be another
    pair's source.  A negative page marks padding; one outside the pool
    leaves its pair out and flags PAGED_ERANGE.  Returns ``pages``."""

    device = _gpu_of("pages", pages)
    if not pages.is_contiguous():
        raise ValueError("pages must be contiguous")
    shape = pages.shape
    if len(shape) < 3:
        raise ValueError("pages must be [layers, 2, pages, ...] or [planes, pages, ...]")
    if len(shape) >= 5:
        if shape[1] != 2 or (len(shape) == 5 and shape[0] == 2):
            raise ValueError("pages {} are not [layers, 2, pages, ...], or may be one "
                             "layer's [2, pages, ...]: give pages.flatten(2) for those, or "
                             "pages.flatten(0, 1).flatten(2)".format(list(shape)))
        planes, count = shape[0] * shape[1], shape[2]
    else:
        planes, count = shape[0], shape[1]
    _placed(device, "pairs", pairs, torch.int32, 2)
    if pairs.shape[1] != 2 or not pairs.is_contiguous():
        raise ValueError("pairs must be contiguous [n, 2]")
    _check_error_word(device, error_flag)
    if pairs.shape[0] == 0 or pages.numel() == 0:
        return pages
    plane_bytes = pages.numel() * pages.element_size() // planes
    _call_on(device.index, stream, "cascade_copy_pages", pages.data_ptr(), planes,
             plane_bytes, count, plane_bytes // count, pairs.data_ptr(),
             pairs.shape[0], 0 if error_flag is None else error_flag.data_ptr())
    return pages


def _count(name, value, low, high):
    """An integer of a range."""

    value = operator.index(value)
    if not low <= value <= high:
        raise ValueError("{} {} is outside [{}, {}]".format(name, value, low, high))
    return value


def paged_tree_attention_workspace_bytes(trees, max_tree, n_q_heads, n_kv_heads,
                                         head_dim, max_length):
    """Workspace bytes of paged_tree_attention for up to ``trees`` trees of up
    to ``max_tree`` nodes over sequences of up to ``max_length`` positions."""

    size = load().cascade_paged_tree_attention_workspace_bytes(
        int(trees), int(max_tree), int(n_q_heads), int(n_kv_heads), int(head_dim),
        int(max_length))
    if size == 0:
        raise ValueError("unsupported tree attention shape")
    return int(size)


def _check_tree_attention(q, starts, masks, k_pages, v_pages, page_table, lengths,
                          out, workspace, rows, error_flag):
    """The checks of paged_tree_attention; returns the strides of q, out, the
    pools and the table."""

    device = _gpu_of("q", q)
    _placed(device, "q", q, torch.bfloat16, 3)
    tokens, _, dim = q.shape
    _placed(device, "starts", starts, torch.int32, 1)
    trees = starts.shape[0] - 1
    if trees < 0:
        raise ValueError("starts holds one entry more than there are trees")
    _vector(device, "starts", starts, torch.int32, trees + 1)
    _vector(device, "masks", masks, torch.int64, tokens)
    pool = _page_pools(device, k_pages, v_pages)
    if k_pages.shape[3] != dim:
        raise ValueError("the pools hold heads of {}, q of {}".format(
            k_pages.shape[3], dim))
    _placed(device, "out", out, torch.bfloat16, 3)
    if out.shape != q.shape:
        raise ValueError("out and q differ in shape")
    _apart("out", out)
    table_stride = _table_stride(device, page_table)
    sequences = page_table.shape[0]
    _vector(device, "lengths", lengths, torch.int32, sequences)
    if rows is not None:
        _vector(device, "rows", rows, torch.int32, trees)
    elif trees > sequences:
        raise ValueError("more trees than page table rows (give rows)")
    _check_bytes(device, workspace)
    _check_error_word(device, error_flag)
    return _strides("q", q), _strides("out", out), pool, table_stride


def paged_tree_attention(q, starts, masks, k_pages, v_pages, page_table, lengths,
                         out, workspace, scale, rows=None, max_tree=64,
                         max_length=None, error_flag=None, stream=None):
    """GQA attention of drafted trees' nodes over their sequences' pages.

    ``q`` and ``out`` [tokens, heads, dim]; tree b has the rows ``starts[b]``
    .. ``starts[b + 1]`` - 1 (int32 [trees + 1]; up to ``max_tree`` of them, 64
    at most) and is the last of the ``lengths[r]`` positions of page table row
    r = ``rows[b]`` (b without ``rows``; negative: padding).  A node reads
    all positions before its tree, and of the tree the nodes j whose bit j is
    set in its ``masks`` (int64 [tokens], see tree_masks).  A node that sees
    nothing gives zeros; rows of no tree stay as they are.  Lengths count the
    tree's nodes and are at most ``max_length`` (default: what a table row
    holds).  A tree out of range is left out and flagged, as are positions on a
    page outside the pool (PAGED_ERANGE in ``error_flag``).  ``workspace``:
    paged_tree_attention_workspace_bytes(...) uint8, one each for calls that may
    overlap."""

    try:
        index = q.get_device()
        q_strides, pool = q.stride(), k_pages.stride()
        table_stride, table_last = page_table.stride()
        tokens, q_heads, dim = shape = q.shape
        trees = starts.shape[0] - 1
        pages, kv_heads, page_size, pool_dim = pool_shape = k_pages.shape
        sequences, width = page_table.shape
        ordinary = (
            tokens > 0 and trees > 0 and pages > 1 and index >= 0
            and v_pages.shape == pool_shape and pool_dim == dim
            and v_pages.stride() == pool and out.shape == shape
            and q_strides[2] == pool[3] == table_last == 1 and pool[2] == dim
            and table_stride >= width
            and q.dtype is _BF16 and k_pages.dtype is _BF16 and v_pages.dtype is _BF16
            and out.dtype is _BF16 and page_table.dtype is _I32
            and starts.dtype is _I32 and masks.dtype is _LONG
            and lengths.dtype is _I32 and workspace.dtype is _U8
            and index == k_pages.get_device() == v_pages.get_device()
            == out.get_device() == page_table.get_device() == lengths.get_device()
            == workspace.get_device() == starts.get_device() == masks.get_device()
            and starts.dim() == 1 and starts.is_contiguous()
            and masks.shape == (tokens,) and masks.is_contiguous()
            and lengths.shape == (sequences,) and lengths.is_contiguous()
            and (trees <= sequences if rows is None else (
                rows.dtype is _I32 and rows.get_device() == index
                and rows.shape == (trees,) and rows.is_contiguous()))
            and out.is_contiguous()
            and workspace.dim() == 1 and workspace.is_contiguous()
            and (error_flag is None or (
                error_flag.dtype is _I32 and error_flag.get_device() == index
                and error_flag.numel() > 0)))
    except (AttributeError, IndexError, TypeError, ValueError, RuntimeError):
        ordinary = False
    if ordinary:
        # (the stride of a dimension of one says nothing)
        q_strides = (q_strides[0] if tokens > 1 else 0, q_strides[1] if q_heads > 1 else 0)
        out_strides = (q_heads * dim, dim)
        if kv_heads == 1:
            pool = (pool[0], page_size * dim)
    else:
        q_strides, out_strides, pool, table_stride = _check_tree_attention(
            q, starts, masks, k_pages, v_pages, page_table, lengths, out, workspace,
            rows, error_flag)
        index = q.get_device()
        tokens, q_heads, dim = q.shape
        trees = starts.shape[0] - 1
        pages, kv_heads, page_size, _ = k_pages.shape
        sequences, width = page_table.shape
    max_tree = _count("max_tree", max_tree, 1, 64)
    if max_length is None:
        max_length = width * page_size
    elif not 0 < max_length <= width * page_size:
        raise ValueError("max_length {} is outside the page table's {}".format(
            max_length, width * page_size))
    if tokens == 0 or trees == 0:
        return out
    _call_on(
        index, stream, "cascade_paged_tree_attention_bf16", q.data_ptr(),
        q_strides[0], q_strides[1], tokens, starts.data_ptr(), masks.data_ptr(), trees,
        max_tree, k_pages.data_ptr(), v_pages.data_ptr(), pool[0], pool[1], pages,
        page_size, page_table.data_ptr(), table_stride, sequences, lengths.data_ptr(),
        0 if rows is None else rows.data_ptr(), int(max_length), q_heads, kv_heads, dim,
        scale, out.data_ptr(), out_strides[0], out_strides[1], workspace.data_ptr(),
        workspace.numel(), 0 if error_flag is None else error_flag.data_ptr())
    return out


def _check_accept(starts, ids, parents, targets, path, counts, next_ids, pages,
                  page_table, lengths, rows, error_flag):
    """The checks of paged_tree_accept; returns trees, tokens, the path's width
    and the sizes of pool and table."""

    device = _gpu_of("starts", starts)
    _placed(device, "starts", starts, _I32, 1)
    trees = starts.shape[0] - 1
    if trees < 0:
        raise ValueError("starts holds one entry more than there are trees")
    _vector(device, "starts", starts, _I32, trees + 1)
    _placed(device, "ids", ids, _LONG, 1)
    tokens = ids.shape[0]
    _vector(device, "ids", ids, _LONG, tokens)
    _vector(device, "parents", parents, _I32, tokens)
    _vector(device, "targets", targets, _LONG, tokens)
    _placed(device, "path", path, _I32, 2)
    if path.shape[0] != trees or not path.is_contiguous():
        raise ValueError("path must be contiguous [{}, max_tree]".format(trees))
    max_tree = _count("path's width", path.shape[1], 1, 64)
    _vector(device, "counts", counts, _I32, trees)
    _vector(device, "next_ids", next_ids, _LONG, trees)
    if rows is not None:
        _vector(device, "rows", rows, _I32, trees)
    _check_error_word(device, error_flag)
    planes = plane_bytes = count = kv_heads = page_size = row_bytes = 0
    table_stride = sequences = width = 0
    if pages is not None:
        _placed(device, "pages", pages, _BF16, 6)
        if not pages.is_contiguous() or pages.shape[1] != 2:
            raise ValueError("pages must be contiguous [layers, 2, pages, kv_heads, "
                             "page_size, dim]")
        layers, _, count, kv_heads, page_size, dim = pages.shape
        planes, row_bytes = 2 * layers, 2 * dim
        plane_bytes = count * kv_heads * page_size * row_bytes
        table_stride = _table_stride(device, page_table)
        sequences, width = page_table.shape
        _vector(device, "lengths", lengths, _I32, sequences)
        if rows is None and trees > sequences:
            raise ValueError("more trees than page table rows (give rows)")
    elif page_table is not None or lengths is not None:
        raise ValueError("page_table and lengths without pages")
    return trees, tokens, max_tree, (planes, plane_bytes, count, kv_heads, page_size,
                                     row_bytes, table_stride, sequences, width)


def paged_tree_accept(starts, ids, parents, targets, path, counts, next_ids,
                      pages=None, page_table=None, lengths=None, rows=None,
                      error_flag=None, stream=None):
    """Follow the drawn tokens through drafted trees, and keep the K and V rows
    of the nodes on their paths.

    Tree b has the rows ``starts[b]`` .. ``starts[b + 1]`` - 1 (int32 [trees +
    1]); of each row ``ids`` (int64 [tokens]) is the node's own token,
    ``parents`` (int32 [tokens]) its parent's place in the tree, before its
    own, and ``targets`` (int64 [tokens]) the token drawn there.  From node 0 on, the
    path goes to the first child whose own token is the one drawn.  ``path``
    (int32 [trees, max_tree], max_tree <= 64) lists its nodes, -1 behind them;
    ``counts`` (int32 [trees]) their number, ``next_ids`` (int64 [trees]) the
    token drawn at the last.  No nodes, a negative ``rows[b]`` and a tree out
    of range: 0 and -1.

    ``pages``: a contiguous pool [layers, 2, pages, kv_heads, page_size, dim]
    whose rows of the path move to the front of the tree, the j-th node's to
    position lengths[r] - n + j of page table row r = ``rows[b]`` (b without
    ``rows``; no row twice) with n nodes.  Rows, lengths and pages out of range
    are left out and flagged (PAGED_ERANGE in ``error_flag``).  Returns
    ``path``."""

    try:
        index = starts.get_device()
        trees, max_tree = path.shape
        tokens, = shape = ids.shape
        each = (trees,)
        ordinary = (
            index >= 0 and tokens > 0 and trees > 0 and 0 < max_tree <= 64
            and starts.dtype is _I32 and ids.dtype is _LONG and parents.dtype is _I32
            and targets.dtype is _LONG and path.dtype is _I32 and counts.dtype is _I32
            and next_ids.dtype is _LONG
            and index == ids.get_device() == parents.get_device() == targets.get_device()
            == path.get_device() == counts.get_device() == next_ids.get_device()
            and starts.shape == (trees + 1,) and parents.shape == shape
            and targets.shape == shape and counts.shape == each and next_ids.shape == each
            and starts.is_contiguous() and ids.is_contiguous() and parents.is_contiguous()
            and targets.is_contiguous() and path.is_contiguous() and counts.is_contiguous()
            and next_ids.is_contiguous()
            and (rows is None or (
                rows.dtype is _I32 and rows.get_device() == index and rows.shape == each
                and rows.is_contiguous()))
            and (error_flag is None or (
                error_flag.dtype is _I32 and error_flag.get_device() == index
                and error_flag.numel() > 0)))
        planes = plane_bytes = count = kv_heads = page_size = row_bytes = 0
        table_stride = sequences = width = 0
        if pages is not None:
            layers, pair, count, kv_heads, page_size, dim = pages.shape
            sequences, width = page_table.shape
            table_stride, table_last = page_table.stride()
            planes, row_bytes = 2 * layers, 2 * dim
            plane_bytes = count * kv_heads * page_size * row_bytes
            ordinary = (
                ordinary and pair == 2 and pages.dtype is _BF16 and pages.is_contiguous()
                and page_table.dtype is _I32 and lengths.dtype is _I32
                and index == pages.get_device() == page_table.get_device()
                == lengths.get_device()
                and table_last == 1 and table_stride >= width
                and lengths.shape == (sequences,) and lengths.is_contiguous()
                and (rows is not None or trees <= sequences))
        elif page_table is not None or lengths is not None:
            ordinary = False
    except (AttributeError, IndexError, TypeError, ValueError, RuntimeError):
        ordinary = False
    if not ordinary:
        trees, tokens, max_tree, (planes, plane_bytes, count, kv_heads, page_size,
                                  row_bytes, table_stride, sequences, width) = (
            _check_accept(starts, ids, parents, targets, path, counts, next_ids, pages,
                          page_table, lengths, rows, error_flag))
        index = starts.get_device()
    if trees == 0:
        return path
    if tokens == 0:
        with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
            path.fill_(-1)
            counts.zero_()
            next_ids.fill_(-1)
        return path
    _call_on(
        index, stream, "cascade_paged_tree_accept", starts.data_ptr(),
        ids.data_ptr(), parents.data_ptr(), targets.data_ptr(), tokens, trees, max_tree,
        path.data_ptr(), counts.data_ptr(), next_ids.data_ptr(),
        0 if pages is None else pages.data_ptr(), planes, plane_bytes, count, kv_heads,
        page_size, row_bytes, 0 if pages is None else page_table.data_ptr(),
        table_stride, sequences, width, 0 if pages is None else lengths.data_ptr(),
        0 if rows is None else rows.data_ptr(),
        0 if error_flag is None else error_flag.data_ptr())
    return path


def sample_workspace_bytes(rows, vocab):
    """Workspace bytes of sample for up to ``rows`` rows of up to ``vocab``
    logits."""

    size = load().cascade_sample_workspace_bytes(int(rows), int(vocab))
    if size == 0:
        raise ValueError("unsupported sampling shape (rows={}, vocab={})".format(
            rows, vocab))
    return int(size)


def _setting(device, name, value, dtype, rows):
    """(pointer, number) of a per-row tensor or one number for all rows."""

    if not isinstance(value, torch.Tensor):
        return 0, value
    _vector(device, name, value, dtype, rows)
    return value.data_ptr(), 0


def sample(logits, uniform, ids, workspace, temperature=1.0, top_k=0, top_p=1.0,
           min_p=0.0, logprobs=None, stream=None):
    """Draw one token a row of fp32 ``logits`` [rows, vocab] into ``ids``
    (int64 [rows], returned).

    ``uniform``: fp32 [rows], a number in [0, 1) a row.  The settings apply in
    the order temperature, top-k, top-p, min-p; each is a number, or a tensor
    with one value a row (fp32; top_k int32).  temperature 0 takes the largest
    logit; top_k 0, top_p 1 and min_p 0 are off.  ``logprobs`` (fp32 [rows])
    receives the log-probability the token was drawn with.  A row with a NaN,
    or with every token at -inf, yields -1 (and NaN).  ``workspace``:
    sample_workspace_bytes(rows, vocab) uint8, one each for calls that may
    overlap."""

    device = _gpu_of("logits", logits)
    _placed(device, "logits", logits, _F32, 2)
    rows, vocab = logits.shape
    row_stride, last = logits.stride()
    if vocab > 1 and last != 1:
        raise ValueError("the rows of logits must be contiguous")
    if rows == 1:
        row_stride = vocab
    elif row_stride < vocab:
        raise ValueError("the rows of logits overlap")
    _vector(device, "uniform", uniform, _F32, rows)
    _vector(device, "ids", ids, _LONG, rows)
    if logprobs is not None:
        _vector(device, "logprobs", logprobs, _F32, rows)
    t_ptr, t = _setting(device, "temperature", temperature, _F32, rows)
    k_ptr, k = _setting(device, "top_k", top_k, _I32, rows)
    p_ptr, p = _setting(device, "top_p", top_p, _F32, rows)
    m_ptr, m = _setting(device, "min_p", min_p, _F32, rows)
    _check_bytes(device, workspace)
    if rows == 0:
        return ids
    _call_on(device.index, stream, "cascade_sample_f32", logits.data_ptr(),
             row_stride, rows, vocab, uniform.data_ptr(), t_ptr, t, k_ptr,
             max(0, min(int(k), 1 << 31)),  # (one past 64 bits would wrap)
             p_ptr, p, m_ptr, m, ids.data_ptr(),
             0 if logprobs is None else logprobs.data_ptr(), workspace.data_ptr(),
             workspace.numel())
    return ids


# ------------------------------------------------------------- 4-bit weights


def linear_w4_workspace_bytes(rows, n, k):
    """Workspace bytes of linear_w4 for ``rows`` rows of ``k`` values times a
    matrix of ``n`` rows (0: none is needed).  Fewer rows may need more: a buffer
    for several sizes takes the largest of theirs."""

    return int(load().cascade_linear_w4_workspace_bytes(int(rows), int(n), int(k)))


def _row_stride(device, name, tensor, dtype, shape):
    """The row stride of a [rows, columns] view with contiguous rows."""

    _placed(device, name, tensor, dtype, 2)
    if shape is not None and tensor.shape != shape:
        raise ValueError("{} has shape {}, expected {}".format(
            name, tuple(tensor.shape), tuple(shape)))
    rows, columns = tensor.shape
    stride, last = tensor.stride()
    if columns > 1 and last != 1:
        raise ValueError("the rows of {} must be contiguous".format(name))
    return columns if rows == 1 else stride


def _check_w4(x, out, dtype, residual, workspace, **matrices):
    """The checks of the products with 4-bit weights; returns (rows, the row
    strides of x, out and residual)."""

    device = _gpu_of("x", x)
    x_stride = _row_stride(device, "x", x, _BF16, None)
    m, k = x.shape
    for name, matrix in matrices.items():
        if not isinstance(matrix, W4Matrix):
            raise TypeError("{} must be a W4Matrix".format(name))
        matrix.launch  # raises where its memory is gone
        if matrix.device != device:
            raise ValueError("{} must live on {}, got {}".format(
                name, device, matrix.device))
        if matrix.k != k:
            raise ValueError("{} has {} columns, x {}".format(name, matrix.k, k))
    n = matrix.n
    y_stride = _row_stride(device, "out", out, dtype, (m, n))
    if m > 1 and y_stride < n:
        raise ValueError("the rows of out overlap")
    if m and x.data_ptr() == out.data_ptr():
        raise ValueError("out may not be x")
    residual_stride = 0
    if residual is not None:
        residual_stride = _row_stride(device, "residual", residual, _BF16, (m, n))
    if workspace is not None:
        _check_bytes(device, workspace)
    return m, x_stride, y_stride, residual_stride


def linear_w4(x, matrix, out, residual=None, workspace=None, stream=None):
    """out = x W^T (+ residual) for a W4Matrix [n, k].

    ``x`` bf16 [rows, k] (row stride a multiple of 8), ``out`` [rows, n] bf16,
    or fp32 for rows that are not rounded (logits; without residual), ``residual``
    bf16 [rows, n], which may be ``out``.  Sums are fp32, with one rounding at
    the end.  ``workspace``: linear_w4_workspace_bytes(rows, n, k) uint8, one
    each for calls that may overlap; None where that is 0."""

    try:
        index, packed, scales, zeros, n, k, group = matrix.launch
        m, x_columns = x.shape
        x_stride, x_last = x.stride()
        y_type = out.dtype
        x_ptr, y_ptr = x.data_ptr(), out.data_ptr()
        y_stride = n
        residual_stride = residual_ptr = 0
        ordinary = (
            x_columns == k and x_last == 1 and m > 0 and x.dtype is _BF16
            and out.shape == (m, n) and out.is_contiguous()
            and (y_type is _BF16 or (y_type is _F32 and residual is None))
            and index == x.get_device() == out.get_device() and x_ptr != y_ptr)
        if residual is not None:
            residual_stride, residual_ptr = n, residual.data_ptr()
            ordinary = (
                ordinary and residual.shape == (m, n) and residual.is_contiguous()
                and residual.dtype is _BF16 and residual.get_device() == index)
        space = (0, 0)
        if workspace is not None:
            space = workspace.data_ptr(), workspace.numel()
            ordinary = (
                ordinary and workspace.dtype is _U8 and workspace.is_contiguous()
                and workspace.dim() == 1 and workspace.get_device() == index)
        if m == 1:
            x_stride = k
    except (AttributeError, IndexError, TypeError, ValueError, RuntimeError):
        ordinary = False
    if not ordinary:
        y_type = _F32 if isinstance(out, torch.Tensor) and out.dtype is _F32 else _BF16
        m, x_stride, y_stride, residual_stride = _check_w4(
            x, out, y_type, residual, workspace, matrix=matrix)
        if y_type is _F32 and residual is not None:
            raise ValueError("fp32 rows take no residual")
        if m == 0:
            return out
    if y_type is _F32:
        _call_on(index, stream, "cascade_linear_w4_f32out_bf16", x_ptr, x_stride, packed,
                 scales, zeros, m, n, k, group, y_ptr, y_stride, *space)
    else:
        _call_on(index, stream, "cascade_linear_w4_bf16", x_ptr, x_stride, packed, scales,
                 zeros, m, n, k, group, residual_ptr, residual_stride, y_ptr, y_stride,
                 *space)
    return out


def gate_up_swiglu_w4(x, gate, up, out, stream=None):
    """out = silu(x Wg^T) * (x Wu^T) for two W4Matrix [n, k] of one group size,
    both with zero points or neither; ``x`` bf16 [rows, k], ``out`` bf16
    [rows, n].  Sums are fp32, with one rounding at the end."""

    try:
        index, *gate_parts, n, k, group = gate.launch
        up_index, *up_parts, up_n, up_k, up_group = up.launch
        m, x_columns = x.shape
        x_stride, x_last = x.stride()
        x_ptr, y_ptr = x.data_ptr(), out.data_ptr()
        y_stride = n
        ordinary = (
            x_columns == k == up_k and n == up_n and group == up_group and x_last == 1
            and m > 0 and (gate_parts[2] == 0) == (up_parts[2] == 0)
            and x.dtype is _BF16 and out.dtype is _BF16
            and out.shape == (m, n) and out.is_contiguous()
            and index == up_index == x.get_device() == out.get_device() and x_ptr != y_ptr)
        if m == 1:
            x_stride = k
    except (AttributeError, IndexError, TypeError, ValueError, RuntimeError):
        ordinary = False
    if not ordinary:
        m, x_stride, y_stride, _ = _check_w4(x, out, _BF16, None, None, gate=gate, up=up)
        if (up.n, up.group, up.zeros is None) != (gate.n, gate.group, gate.zeros is None):
            raise ValueError("gate and up differ in rows, group size or zero points")
        if m == 0:
            return out
    _call_on(index, stream, "cascade_gate_up_swiglu_w4_bf16", x_ptr, x_stride, *gate_parts,
             *up_parts, m, n, k, group, y_ptr, y_stride)
    return out


# ------------------------------------------------------------ copy pipeline


def memcpy_h2d_async(dst, src, nbytes, stream):
    """hipMemcpyAsync host->device of nbytes; src must be page-locked."""

    require_device(dst, "dst", contiguous=False)
    if src.device.type != "cpu":
        raise ValueError("src must be a host tensor")
    if nbytes > src.numel() * src.element_size():
        raise ValueError("copy larger than the source")
    if nbytes > dst.numel() * dst.element_size():
        raise ValueError("copy larger than the destination")
    call("cascade_memcpy_h2d_async", dst.data_ptr(), src.data_ptr(),
         int(nbytes), stream_handle(stream))


def default_copy_threads():
    """Threads for host staging copies: this process's CPUs, at most 8.

    Eight threads stage at about twice the link rate.  More slow the H2D
    copies that read host memory at the same time: on MI355X, config 5
    prefill took 286 ms with 16 threads, 277 ms with 6 to 10, and 281 ms
    with 4."""

    try:
        cpus = len(os.sched_getaffinity(0))
    except AttributeError:  # not Linux
        cpus = os.cpu_count() or 1
    return max(1, min(8, cpus))


def _host_copy_bytes(dst, src):
    for name, t in (("dst", dst), ("src", src)):
        if not isinstance(t, torch.Tensor) or t.device.type != "cpu":
            raise ValueError("{} must be a host tensor".format(name))
        if not t.is_contiguous():
            raise ValueError("{} must be contiguous".format(name))
    nbytes = src.numel() * src.element_size()
    if dst.numel() * dst.element_size() != nbytes:
        raise ValueError("host_copy needs equal byte sizes")
    return nbytes


def host_copy(dst, src, threads=None):
    """dst.copy_(src) for contiguous host tensors of equal byte size, with
    the library's multi-threaded non-temporal memcpy (threads started for
    this call only; the GIL is released for the duration of the copy)."""

    nbytes = _host_copy_bytes(dst, src)
    call("cascade_host_copy", dst.data_ptr(), src.data_ptr(), nbytes,
         int(threads or default_copy_threads()))
    return dst


def device_numa_node(device=None):
    """NUMA node of the host bridge a GPU sits behind, from the PCI
    device's sysfs entry; -1 when there is no GPU, the platform reports
    none (a one-node host writes -1 there too) or the entry is missing."""

    if not torch.cuda.is_available():
        return -1
    props = torch.cuda.get_device_properties(
        torch.cuda.current_device() if device is None else device)
    path = "/sys/bus/pci/devices/{:04x}:{:02x}:{:02x}.0/numa_node".format(
        props.pci_domain_id, props.pci_bus_id, props.pci_device_id)
    try:
        with open(path) as f:
            return int(f.read().strip())
    except (OSError, ValueError):
        return -1


class _PoolState:
    """The native pool handle and the count of copies running on it, shared
    by a CopyPool and its finalizer."""

    __slots__ = ("handle", "busy", "lock")

    def __init__(self, handle):
        self.handle = handle
        self.busy = 0
        self.lock = threading.Lock()


def _destroy_copy_pool(state):
    with state.lock:
        handle, state.handle = state.handle, 0
        if not handle or state.busy:
            # A copy is still running on the pool: only a daemon staging
            # thread at interpreter exit can be inside one when the pool is
            # finalized.  New copies are refused from here on, and the
            # native pool, whose helpers that copy is using, is left to the
            # process exit.
            return
    call("cascade_copy_pool_destroy", handle)


class CopyPool:
    """A caller-owned pool for the multi-threaded host copy: ``threads``
    threads in all (the caller and threads - 1 helpers), the helpers bound
    to the CPUs of ``numa_node`` when it is >= 0.  ``close`` joins them (as
    does garbage collection, or interpreter exit, of an unclosed pool).  A
    pool closed or finalized while a copy runs on it refuses new copies and
    leaves the native pool alive for that copy (it is not destroyed then)."""

    def __init__(self, threads=None, numa_node=-1):
        handle = _U64(0)
        call("cascade_copy_pool_create", int(threads or default_copy_threads()),
             int(numa_node), ctypes.byref(handle))
        self._state = _PoolState(handle.value)
        self._finalizer = weakref.finalize(self, _destroy_copy_pool, self._state)
        threads_out, bound = _INT(0), _INT(0)
        call("cascade_copy_pool_info", handle.value, ctypes.byref(threads_out),
             ctypes.byref(bound))
        self.threads = threads_out.value
        self.bound_cpus = bound.value
        self.numa_node = int(numa_node)

    @property
    def handle(self):
        return self._state.handle

    def copy(self, dst, src):
        nbytes = _host_copy_bytes(dst, src)
        state = self._state
        with state.lock:
            handle = state.handle
            if not handle:
                raise RuntimeError("the copy pool is closed")
            state.busy += 1
        try:
            call("cascade_copy_pool_copy", handle, dst.data_ptr(),
                 src.data_ptr(), nbytes)
        finally:
            with state.lock:
                state.busy -= 1
        return dst

    def close(self):
        self._finalizer()  # destroys the native pool, once

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()


class HipEvent:
    """A hipEvent_t created through the C ABI (duck-types torch.cuda.Event
    for ``record``, ``wait``, ``synchronize``, ``query`` and
    ``elapsed_time``)."""

    __slots__ = ("handle", "timing")

    def __init__(self, enable_timing=False):
        handle = _U64(0)
        call("cascade_event_create", ctypes.byref(handle),
             1 if enable_timing else 0)
        self.handle = handle.value
        self.timing = bool(enable_timing)

    def record(self, stream=None):
        call("cascade_event_record", self.handle, stream_handle(stream))

    def wait(self, stream=None):
        """Make ``stream`` wait for this event (hipStreamWaitEvent)."""

        call("cascade_stream_wait_event", stream_handle(stream), self.handle)

    def synchronize(self):
        call("cascade_event_synchronize", self.handle)

    def query(self):
        code = load().cascade_event_query(self.handle)
        if code in (0, 1):
            return code == 0
        _check("cascade_event_query", code)
        return False

    def elapsed_time(self, end):
        ms = _F(0.0)
        call("cascade_event_elapsed_ms", self.handle, end.handle,
             ctypes.byref(ms))
        return float(ms.value)

    def __del__(self):
        lib = _lib
        if lib is not None and self.handle:
            try:
                lib.cascade_event_destroy(self.handle)
            except Exception:  # interpreter shutdown
                pass
            self.handle = 0


def time_next_launch(start, stop):
    """Bind two timing HipEvents (or None) to this thread's next kernel
    launch through the library: their elapsed time is that kernel's own
    duration.  ``time_next_launch(None, None)`` clears pending events."""

    call("cascade_time_next_launch", start.handle if start else 0,
         stop.handle if stop else 0)


def stream_wait(stream, event):
    """stream waits for event (either a HipEvent or a torch.cuda.Event)."""

    if isinstance(event, HipEvent):
        event.wait(stream)
    else:
        stream.wait_event(event)

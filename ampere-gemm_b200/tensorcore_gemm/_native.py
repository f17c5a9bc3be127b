"""ctypes binding of the C ABI in include/b200_gemm.h (libb200gemm.so).

This is the reference-side binding of the native boundary: where the
reference bound its kernels through a pybind function generated by
load_inline (tensorcore_gemm/gemm.py:202-206, cuda_compile.py:235-245), this
package binds the prebuilt C-ABI library with ctypes.  There is no fallback:
if the library is missing or cannot be loaded every GEMM call raises.
"""
from __future__ import annotations

import ctypes
import threading
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libb200gemm.so"

# Return codes (include/b200_gemm.h).
B200_OK = 0
B200_ERR_INVALID_ARGUMENT = 1
B200_ERR_MISALIGNED = 2
B200_ERR_TOO_LARGE = 3
B200_ERR_CUDA = 4
B200_ERR_TENSOR_MAP = 5
B200_ERR_DEVICE = 6
B200_ERR_UNSUPPORTED_DEVICE = 7
B200_ERR_WORKSPACE = 8
B200_ERR_SCRATCH_LIMIT = 9

B200_VARIANT_AUTO = 0
B200_VARIANT_CTA1 = 1
B200_VARIANT_PAIR = 2
B200_VARIANT_SKINNY = 3
B200_VARIANT_PAIR_WIDE = 4
B200_VARIANT_PAIR_WIDE_224 = 5
B200_VARIANT_PAIR_WIDE_192 = 6
VARIANTS = {"auto": B200_VARIANT_AUTO, "cta1": B200_VARIANT_CTA1, "pair": B200_VARIANT_PAIR,
            "skinny": B200_VARIANT_SKINNY, "pair2m": B200_VARIANT_PAIR_WIDE,
            "pair2m_224": B200_VARIANT_PAIR_WIDE_224, "pair2m_192": B200_VARIANT_PAIR_WIDE_192}

B200_B_ROW_MAJOR = 0
B200_B_COL_MAJOR = 1
B200_A_ROW_MAJOR = 0
B200_A_COL_MAJOR = 1

B200_DTYPE_F16 = 0
B200_DTYPE_BF16 = 1
B200_DTYPE_F32 = 2
B200_LOGPROBS_MAX_TOP = 64
B200_ACT_SILU = 0
B200_ACT_GELU = 1
B200_ACT_GELU_TANH = 2

# Every symbol the header declares, with its ctypes signature.
_SIGNATURES = {
    "b200_gemm_f16": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int, ctypes.c_void_p],
    ),
    "b200_gemm_workspace_size": (
        ctypes.c_int64,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int],
    ),
    "b200_gemm_f16_ws": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "b200_gemm_f16_ex": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int, ctypes.c_int, ctypes.c_float, ctypes.c_float,
         ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "b200_gemm_workspace_size_ex": (
        ctypes.c_int64,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_int],
    ),
    "b200_kmeans_workspace_size": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int64]),
    "b200_kmeans_assign_f16": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_int64,
         ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p],
    ),
    "b200_gemm_f16_gather": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
         ctypes.c_int, ctypes.POINTER(ctypes.c_void_p), ctypes.c_int, ctypes.c_void_p],
    ),
    "b200_layer_norm_fwd": (
        ctypes.c_int,
        [ctypes.c_void_p] * 6 + [ctypes.c_int64] * 4 + [ctypes.c_int, ctypes.c_int, ctypes.c_float, ctypes.c_void_p],
    ),
    "b200_layer_norm_bwd_workspace_size": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int64]),
    "b200_layer_norm_bwd": (
        ctypes.c_int,
        [ctypes.c_void_p] * 8 + [ctypes.c_int64] * 5 +
        [ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "b200_token_logprobs_workspace_size": (ctypes.c_int64, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int]),
    "b200_token_logprobs_fwd": (
        ctypes.c_int,
        [ctypes.c_void_p] * 7 + [ctypes.c_int64] * 3 +
        [ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "b200_token_logprobs_bwd": (
        ctypes.c_int,
        [ctypes.c_void_p] * 7 + [ctypes.c_int64] * 5 + [ctypes.c_int, ctypes.c_void_p],
    ),
    "b200_gated_ffn_workspace_size": (ctypes.c_int64, [ctypes.c_int64] * 4 + [ctypes.c_int] * 2),
    "b200_gated_ffn_plan": (ctypes.c_int, [ctypes.c_int64] * 3 + [ctypes.c_int] * 2 +
                            [ctypes.POINTER(ctypes.c_int)] * 3),
    "b200_gated_ffn_fwd": (
        ctypes.c_int,
        [ctypes.c_void_p] * 5 + [ctypes.c_int64] * 8 +
        [ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "b200_gated_ffn_bwd": (
        ctypes.c_int,
        [ctypes.c_void_p] * 8 + [ctypes.c_int64] * 11 +
        [ctypes.c_int, ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "b200_ipc_handle_size": (ctypes.c_int, []),
    "b200_ipc_alloc": (ctypes.c_int, [ctypes.c_int64, ctypes.POINTER(ctypes.c_void_p), ctypes.c_void_p]),
    "b200_ipc_free": (ctypes.c_int, [ctypes.c_void_p]),
    "b200_ipc_open": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(ctypes.c_void_p)]),
    "b200_ipc_close": (ctypes.c_int, [ctypes.c_void_p]),
    "b200_gemm_strerror": (ctypes.c_char_p, [ctypes.c_int]),
    "b200_gemm_last_device_error": (ctypes.c_int, []),
    "b200_gemm_sm_count": (ctypes.c_int, []),
    "b200_gemm_version": (ctypes.c_int, []),
    "b200_gemm_set_variant": (ctypes.c_int, [ctypes.c_int]),
    "b200_gemm_plan": (ctypes.c_int, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int,
                                      ctypes.POINTER(ctypes.c_int), ctypes.POINTER(ctypes.c_int)]),
    "b200_gemm_selftest_bounded_wait": (ctypes.c_int, [ctypes.c_int64]),
    "b200_gemm_selftest_split_fixup": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
         ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p],
    ),
}

_lib = None
_lock = threading.Lock()


class NativeLibraryError(RuntimeError):
    """The native GEMM library is missing or could not be loaded."""


def load() -> ctypes.CDLL:
    """Load (once) and return the native library, raising if it is absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not LIB_PATH.exists():
                raise NativeLibraryError(
                    f"B200 GEMM library not built: {LIB_PATH} is missing "
                    "(run `python ampere-gemm_b200/build.py`)")
            try:
                lib = ctypes.CDLL(str(LIB_PATH))
            except OSError as exc:
                raise NativeLibraryError(f"cannot load {LIB_PATH}: {exc}") from exc
            for name, (res, args) in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.restype = res
                fn.argtypes = args
            _lib = lib
    return _lib


def strerror(code: int) -> str:
    return load().b200_gemm_strerror(int(code)).decode()


def check(code: int, what: str = "b200_gemm_f16") -> None:
    if code != B200_OK:
        raise RuntimeError(f"{what} failed: {strerror(code)} (code {code})")


def gemm_f16_raw(a_ptr: int, b_ptr: int, c_ptr: int, m: int, n: int, k: int,
                 lda: int, ldb: int, ldc: int, b_layout: int, stream: int) -> int:
    """Direct call of b200_gemm_f16; returns its code without raising."""
    fn = _gemm_fn
    if fn is None:
        fn = _bind_gemm()
    return fn(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, b_layout, stream)


_gemm_fn = None


def _bind_gemm():
    global _gemm_fn
    _gemm_fn = load().b200_gemm_f16
    return _gemm_fn


def workspace_size(a_ptr: int, b_ptr: int, c_ptr: int, m: int, n: int, k: int,
                   lda: int, ldb: int, ldc: int, b_layout: int) -> int:
    """Bytes of workspace b200_gemm_f16_ws needs (0 if none); raises on bad arguments."""
    v = load().b200_gemm_workspace_size(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, b_layout)
    if v < 0:
        check(-v, "b200_gemm_workspace_size")
    return v


def gemm_f16_ws_raw(a_ptr: int, b_ptr: int, c_ptr: int, m: int, n: int, k: int, lda: int, ldb: int, ldc: int,
                    b_layout: int, ws_ptr: int, ws_bytes: int, stream: int) -> int:
    return load().b200_gemm_f16_ws(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, b_layout, ws_ptr, ws_bytes, stream)


def gemm_ex_raw(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, a_layout, b_layout, alpha, beta,
                ws_ptr, ws_bytes, stream) -> int:
    return load().b200_gemm_f16_ex(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, a_layout, b_layout,
                                   float(alpha), float(beta), ws_ptr, ws_bytes, stream)


def workspace_size_ex(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, a_layout, b_layout) -> int:
    v = load().b200_gemm_workspace_size_ex(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, a_layout, b_layout)
    if v < 0:
        check(-v, "b200_gemm_workspace_size_ex")
    return v


def last_device_error() -> int:
    return load().b200_gemm_last_device_error()


def sm_count() -> int:
    return load().b200_gemm_sm_count()


def version() -> int:
    return load().b200_gemm_version()


def set_variant(variant: int | str) -> None:
    """Force one kernel variant for the whole process ("auto" restores the heuristic)."""
    v = VARIANTS[variant] if isinstance(variant, str) else int(variant)
    check(load().b200_gemm_set_variant(v), "b200_gemm_set_variant")


def selftest_bounded_wait(limit_ns: int = 10_000_000) -> int:
    """Run the bounded-wait self-test kernel; returns the error word it produced (5 = ok)."""
    return load().b200_gemm_selftest_bounded_wait(int(limit_ns))


def selftest_split_fixup(a_ptr: int, b_ptr: int, c_ptr: int, m: int, n: int, k: int,
                         limit_ns: int = 2_000_000, stream: int = 0) -> int:
    """Run the split-fixup failure self-test; returns the error word it produced (6 = ok)."""
    return load().b200_gemm_selftest_split_fixup(a_ptr, b_ptr, c_ptr, m, n, k, int(limit_ns), stream)


def gemm_gather_raw(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, b_layout, peer_ptrs, stream) -> int:
    """Direct call of b200_gemm_f16_gather; peer_ptrs is a sequence of device addresses."""
    arr = (ctypes.c_void_p * max(1, len(peer_ptrs)))(*[int(p) for p in peer_ptrs])
    return load().b200_gemm_f16_gather(a_ptr, b_ptr, c_ptr, m, n, k, lda, ldb, ldc, b_layout, arr,
                                       len(peer_ptrs), stream)


def ipc_alloc(nbytes: int) -> tuple[int, bytes]:
    """Allocate an IPC-shareable device buffer; returns (device address, handle bytes)."""
    lib = load()
    size = lib.b200_ipc_handle_size()
    handle = ctypes.create_string_buffer(size)
    ptr = ctypes.c_void_p()
    check(lib.b200_ipc_alloc(int(nbytes), ctypes.byref(ptr), handle), "b200_ipc_alloc")
    return int(ptr.value), handle.raw


def ipc_open(handle: bytes) -> int:
    """Map a peer's buffer (handle from ipc_alloc in another process); returns its address here."""
    ptr = ctypes.c_void_p()
    check(load().b200_ipc_open(ctypes.create_string_buffer(bytes(handle), len(handle)), ctypes.byref(ptr)),
          "b200_ipc_open")
    return int(ptr.value)


def ipc_close(ptr: int) -> None:
    check(load().b200_ipc_close(ctypes.c_void_p(int(ptr))), "b200_ipc_close")


def ipc_free(ptr: int) -> None:
    check(load().b200_ipc_free(ctypes.c_void_p(int(ptr))), "b200_ipc_free")


FFN_PRODUCTS = {"gate_up": 0, "out": 1, "gate_grad": 2, "in_grad": 3}


def gated_ffn_plan(rows: int, n: int, k: int, product: str, sm_count: int = 148) -> tuple[int, int, int]:
    """(CTAs of a cluster, shared memory, TMEM columns) of one of the block's products on the kernel for few
    rows, (0, 0, 0) where it runs on the GEMM's tiles (b200_gated_ffn_plan); no GPU needed."""
    out = [ctypes.c_int() for _ in range(3)]
    check(load().b200_gated_ffn_plan(int(rows), int(n), int(k), FFN_PRODUCTS[product], int(sm_count),
                                     *(ctypes.byref(v) for v in out)), "b200_gated_ffn_plan")
    return tuple(v.value for v in out)


VARIANT_NAMES = {v: k for k, v in VARIANTS.items()}


def plan(m: int, n: int, k: int, sm_count: int = 148) -> tuple[str, int]:
    """(variant name, K ranges of the last wave) the library would launch; no GPU needed."""
    v, r = ctypes.c_int(), ctypes.c_int()
    check(load().b200_gemm_plan(int(m), int(n), int(k), int(sm_count), ctypes.byref(v), ctypes.byref(r)),
          "b200_gemm_plan")
    return VARIANT_NAMES[v.value], r.value

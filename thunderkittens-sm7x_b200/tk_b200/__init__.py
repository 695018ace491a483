"""Python binding of the tk_b200 C ABI (include/tk_b200.h).

The library is the product: ``libtk_b200.so`` built in-tree for sm_100a. This module
only loads it with ctypes and passes device pointers, sizes and CUDA streams. It
never computes anything itself and has no fallback: if the shared library is
missing, or a call returns an error, it raises.

Entry points mirror ThunderKittens-SM7x's public API (include/tk_sm7x/gemm.cuh,
attention.cuh, reduce.cuh, softmax.cuh): same argument meaning and the same
error behaviour (``cudaErrorInvalidValue`` for invalid arguments, nothing
enqueued).
"""

from __future__ import annotations

import ctypes as C
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
PKG_ROOT = os.path.dirname(HERE)
LIB_PATH = os.path.join(HERE, "libtk_b200.so")

CUDA_SUCCESS = 0
CUDA_ERROR_INVALID_VALUE = 1
CUDA_ERROR_INVALID_DEVICE_FUNCTION = 98
CUDA_ERROR_NOT_SUPPORTED = 801

# Every symbol include/tk_b200.h declares, with its ctypes signature.
_VP, _I, _SZ, _F, _L = C.c_void_p, C.c_int, C.c_size_t, C.c_float, C.c_int64
_MASKED = [_VP, _VP, _VP, _VP, _VP, _I, _I, _I, _I, _I, _I, _F, _F, _VP, _VP, _VP, _I, _VP]
_APPEND = [_VP, _VP, _L, _L, _VP, _I, _I, _I, _VP, _VP, _VP, _VP, _I, _I, _VP]
_PAGED = [_VP, _L, _VP, _L, _I, _VP, _VP, _VP, _VP, _I, _I, _VP, _I, _VP, _VP, _I, _I, _I, _I, _I, _I, _F, _F, _VP, _VP]
SIGNATURES = {
    "tk_gemm_f16_f16_f32_nn": (_I, [_I, _I, _I, _VP, _I, _VP, _I, _VP, _I, _VP]),
    "tk_gemm_f16_f16_f32_nn_rowstats": (_I, [_I, _I, _I, _VP, _I, _VP, _I, _VP, _I, _VP, _VP, _VP]),
    "tk_gemm_f16_f16_f32_nn_rowstats_noalloc": (_I, [_I, _I, _I, _VP, _I, _VP, _I, _VP, _I, _VP, _VP,
                                                     _VP]),
    "tk_gemm_f16_f16_f32_nn_rowsoftmax": (_I, [_I, _I, _I, _VP, _I, _VP, _I, _VP, _I, _VP, _I, _VP]),
    "tk_gemm_f16_f16_f32_nn_gather": (_I, [_I, _I, _I, _VP, _I, _VP, _I, _VP, _I, _I, _I, _VP]),
    "tk_ipc_alloc": (_I, [_SZ, C.POINTER(C.c_void_p), _VP]),
    "tk_ipc_open": (_I, [_VP, C.POINTER(C.c_void_p)]),
    "tk_ipc_close": (_I, [_VP]),
    "tk_ipc_free": (_I, [_VP]),
    "tk_gemm_set_cta_group": (_I, [_I]),
    "tk_gemm_set_splitk_reduce": (_I, [_I]),
    "tk_tile_row_sum_f32": (_I, [_VP, _SZ, _VP, _VP]),
    "tk_tile_row_max_f32": (_I, [_VP, _SZ, _VP, _VP]),
    "tk_tile_row_softmax_f32": (_I, [_VP, _SZ, _VP, _VP]),
    "tk_tile_row_softmax_causal_f32": (_I, [_VP, _SZ, _VP, _VP]),
    "tk_tile_row_ops_f32": (_I, [_VP, _SZ, _VP, _VP, _VP, _VP, _VP]),
    "tk_attention_forward_16x16": (_I, [_VP, _VP, _VP, _VP, _VP]),
    "tk_attention_forward_16x16_causal": (_I, [_VP, _VP, _VP, _VP, _VP]),
    "tk_attention_forward_f16": (_I, [_VP, _VP, _VP, _VP, _I, _I, _I, _I, _F, _I, _VP]),
    "tk_attention_forward_gqa_f16": (_I, [_VP, _VP, _VP, _VP, _I, _I, _I, _I, _I, _F, _I, _VP]),
    "tk_attention_masked_f16": (_I, _MASKED),
    "tk_attention_masked_bf16": (_I, _MASKED),
    "tk_kv_plan": (_I, [_VP, _VP, _I, _I, _VP, _I, _VP, _I, _VP, _VP, _VP, _VP, _VP, _I, _VP, _VP]),
    "tk_kv_append_e4m3_f16": (_I, _APPEND),
    "tk_kv_append_e4m3_bf16": (_I, _APPEND),
    "tk_attention_paged_e4m3_f16": (_I, _PAGED),
    "tk_attention_paged_e4m3_bf16": (_I, _PAGED),
    "tk_attention_set_cta_group": (_I, [_I]),
    "tk_gemm_set_group_rows": (_I, [_I]),
    "tk_gemm_set_small_m": (_I, [_I]),
    "tk_device_status": (_I, [C.POINTER(C.c_uint32), _I]),
    "tk_scratch_pool_bytes": (_I, [_I, C.POINTER(C.c_uint64), C.POINTER(C.c_uint64)]),
    "tk_abi_version": (_I, []),
}

_lib = None


class TkError(RuntimeError):
    def __init__(self, fn: str, code: int):
        super().__init__(f"{fn} returned cudaError {code}")
        self.code = code


def build() -> None:
    """Compile libtk_b200.so for sm_100a (nvcc cross-compiles without a GPU)."""
    subprocess.run(["make", "-s", "-C", PKG_ROOT], check=True)


def lib():
    """The loaded C library. Raises if it was not built: there is no fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: run `make -C {PKG_ROOT}` (no CPU fallback exists)")
        handle = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def _check(name: str, code: int) -> None:
    if code != CUDA_SUCCESS:
        raise TkError(name, code)


def _ptr(t):
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def _stream(stream):
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


# ---- raw calls (pointers as ints or tensors); return the cudaError code -------------

def gemm_raw(m, n, k, a, lda, b, ldb, c, ldc, stream=None) -> int:
    return lib().tk_gemm_f16_f16_f32_nn(m, n, k, _ptr(a), lda, _ptr(b), ldb, _ptr(c), ldc, _stream(stream))


def gemm_rowstats_raw(m, n, k, a, lda, b, ldb, c, ldc, row_max, row_sum, stream=None) -> int:
    return lib().tk_gemm_f16_f16_f32_nn_rowstats(m, n, k, _ptr(a), lda, _ptr(b), ldb, _ptr(c), ldc,
                                                 _ptr(row_max), _ptr(row_sum), _stream(stream))


def gemm_rowsoftmax_raw(m, n, k, a, lda, b, ldb, c, ldc, probs, ldp, stream=None) -> int:
    return lib().tk_gemm_f16_f16_f32_nn_rowsoftmax(m, n, k, _ptr(a), lda, _ptr(b), ldb, _ptr(c), ldc,
                                                   _ptr(probs), ldp, _stream(stream))


def gemm_gather_raw(m, n, k, a, lda, b, ldb, c_ranks, rank, ldc, stream=None) -> int:
    """c_ranks: device pointers (ints) of every rank's gathered buffer, in rank order."""
    arr = (C.c_void_p * len(c_ranks))(*c_ranks)
    return lib().tk_gemm_f16_f16_f32_nn_gather(m, n, k, _ptr(a), lda, _ptr(b), ldb, C.cast(arr, C.c_void_p),
                                                len(c_ranks), rank, ldc, _stream(stream))


def ipc_alloc(nbytes: int) -> tuple[int, bytes]:
    """Shareable device allocation: (pointer, 64-byte IPC handle)."""
    ptr = C.c_void_p()
    handle = C.create_string_buffer(64)
    _check("tk_ipc_alloc", lib().tk_ipc_alloc(nbytes, C.byref(ptr), handle))
    return ptr.value, handle.raw


def ipc_open(handle: bytes) -> int:
    ptr = C.c_void_p()
    buf = C.create_string_buffer(bytes(handle), 64)
    _check("tk_ipc_open", lib().tk_ipc_open(buf, C.byref(ptr)))
    return ptr.value


def ipc_close(ptr: int) -> None:
    _check("tk_ipc_close", lib().tk_ipc_close(ptr))


def ipc_free(ptr: int) -> None:
    _check("tk_ipc_free", lib().tk_ipc_free(ptr))


def set_gemm_cta_group(g: int) -> int:
    return lib().tk_gemm_set_cta_group(g)


def set_gemm_splitk_reduce(mode: int) -> int:
    """0: split-K partials summed inside the kernel (tile clusters) where they fit;
    1: always by a second kernel. Returns the previous mode."""
    return lib().tk_gemm_set_splitk_reduce(mode)


def attention_16x16_raw(q, k, v, out, causal=False, stream=None) -> int:
    fn = lib().tk_attention_forward_16x16_causal if causal else lib().tk_attention_forward_16x16
    return fn(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _stream(stream))


def attention_raw(q, k, v, out, batch, heads, seq, head_dim, scale, causal, stream=None) -> int:
    return lib().tk_attention_forward_f16(_ptr(q), _ptr(k), _ptr(v), _ptr(out), batch, heads, seq,
                                          head_dim, float(scale), 1 if causal else 0, _stream(stream))


def attention_gqa_raw(q, k, v, out, batch, heads_q, heads_kv, seq, head_dim, scale, causal, stream=None) -> int:
    return lib().tk_attention_forward_gqa_f16(_ptr(q), _ptr(k), _ptr(v), _ptr(out), batch, heads_q, heads_kv,
                                              seq, head_dim, float(scale), 1 if causal else 0, _stream(stream))


def row_ops_raw(tiles, n_tiles, row_sum=None, row_max=None, softmax=None, softmax_causal=None,
                stream=None) -> int:
    return lib().tk_tile_row_ops_f32(_ptr(tiles), n_tiles, _ptr(row_sum), _ptr(row_max), _ptr(softmax),
                                     _ptr(softmax_causal), _stream(stream))


def device_status(clear: bool = False) -> int:
    v = C.c_uint32()
    _check("tk_device_status", lib().tk_device_status(C.byref(v), 1 if clear else 0))
    return v.value


def scratch_pool_bytes(device: int = 0) -> tuple[int, int]:
    """(reserved, used) bytes of the library's scratch pool on `device`."""
    reserved, used = C.c_uint64(), C.c_uint64()
    _check("tk_scratch_pool_bytes", lib().tk_scratch_pool_bytes(device, C.byref(reserved), C.byref(used)))
    return reserved.value, used.value


# ---- torch-level helpers (device tensors in, device tensors out) ---------------------

def gemm(a, b, c=None, *, m=None, n=None, k=None, lda=None, ldb=None, ldc=None, stream=None):
    """C = A @ B with A (m x lda) / B (k x ldb) binary16 and C (m x ldc) FP32 device tensors."""
    import torch
    m = a.shape[0] if m is None else m
    k = b.shape[0] if k is None else k
    n = b.shape[1] if n is None else n
    lda = a.stride(0) if lda is None else lda
    ldb = b.stride(0) if ldb is None else ldb
    if c is None:
        c = torch.empty((m, n), dtype=torch.float32, device=a.device)
    ldc = c.stride(0) if ldc is None else ldc
    _check("tk_gemm_f16_f16_f32_nn", gemm_raw(m, n, k, a, lda, b, ldb, c, ldc, stream))
    return c


def gemm_rowstats(a, b, c=None, *, stream=None):
    import torch
    m, n, k = a.shape[0], b.shape[1], b.shape[0]
    if c is None:
        c = torch.empty((m, n), dtype=torch.float32, device=a.device)
    row_max = torch.empty(m, dtype=torch.float32, device=a.device)
    row_sum = torch.empty(m, dtype=torch.float32, device=a.device)
    _check("tk_gemm_f16_f16_f32_nn_rowstats",
           gemm_rowstats_raw(m, n, k, a, a.stride(0), b, b.stride(0), c, c.stride(0), row_max, row_sum,
                             stream))
    return c, row_max, row_sum


def gemm_rowsoftmax(a, b, c=None, probs=None, *, in_place=False, stream=None):
    """C = A @ B and P = softmax over each row of C. With in_place=True P replaces C
    (one buffer); returns (C, P), the same tensor twice when in place."""
    import torch
    m, n, k = a.shape[0], b.shape[1], b.shape[0]
    if c is None:
        c = torch.empty((m, n), dtype=torch.float32, device=a.device)
    if in_place:
        probs = c
    elif probs is None:
        probs = torch.empty((m, n), dtype=torch.float32, device=a.device)
    _check("tk_gemm_f16_f16_f32_nn_rowsoftmax",
           gemm_rowsoftmax_raw(m, n, k, a, a.stride(0), b, b.stride(0), c, c.stride(0), probs,
                               probs.stride(0), stream))
    return c, probs


def tile_row_ops(tiles, *, ops=("sum", "max", "softmax", "causal"), stream=None):
    """Batched 16x16 tile row ops; tiles is a contiguous FP32 tensor of n*256 values."""
    import torch
    n = tiles.numel() // 256
    out = {}
    dev = tiles.device
    if "sum" in ops:
        out["sum"] = torch.empty((n, 16), dtype=torch.float32, device=dev)
    if "max" in ops:
        out["max"] = torch.empty((n, 16), dtype=torch.float32, device=dev)
    if "softmax" in ops:
        out["softmax"] = torch.empty((n, 16, 16), dtype=torch.float32, device=dev)
    if "causal" in ops:
        out["causal"] = torch.empty((n, 16, 16), dtype=torch.float32, device=dev)
    _check("tk_tile_row_ops_f32", row_ops_raw(tiles, n, out.get("sum"), out.get("max"), out.get("softmax"),
                                              out.get("causal"), stream))
    return out


def attention(q, k, v, *, scale, causal=False, out=None, stream=None):
    """q, k, v: [B, H, S, D] contiguous binary16 device tensors -> FP32 [B, H, S, D]."""
    import torch
    b, h, s, d = q.shape
    if out is None:
        out = torch.empty((b, h, s, d), dtype=torch.float32, device=q.device)
    _check("tk_attention_forward_f16", attention_raw(q, k, v, out, b, h, s, d, scale, causal, stream))
    return out


# ---- attention of language models, and the paged 8-bit cache ---------------------------
#
# The smallest calls take a few microseconds on the GPU, less than Python takes to look
# at a dozen tensors with care. So each helper tests all that it requires in one chain of
# cheap comparisons, and works out which of them failed only when one did.

_torch = None
_raw_stream = None
_Strides = C.c_int64 * 12


def _import_torch():
    global _torch, _raw_stream
    import torch
    # The handle of a device's current stream without a Stream object around it (0.1 us against 4).
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    _torch = torch
    return torch


def _require(ok, message):
    if not ok:
        raise ValueError(message)


def _half_type(t, name):
    _require(t.dtype in (_torch.float16, _torch.bfloat16), f"{name} must be float16 or bfloat16, got {t.dtype}")


def _vector(t, name, dtype, shape):
    """None, or a contiguous tensor of this type and shape."""
    _require(t is None or (t.dtype == dtype and tuple(t.shape) == tuple(shape) and t.is_contiguous()),
             f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)}" +
             ("" if t is None else f", got {t.dtype} {tuple(t.shape)}"))


def _same_device(device, **tensors):
    _require(device.type == "cuda", f"tensors must be on a CUDA device, got {device}")
    for name, t in tensors.items():
        _require(t is None or t.device == device, f"{name} is on {getattr(t, 'device', None)}, expected {device}")


class _Launch:
    """Makes `device`, and on it the stream of a call, current while the call allocates its
    outputs and launches, so that the outputs belong to that stream."""

    def __init__(self, device, stream):
        self.device = _torch.cuda.device(device)
        if isinstance(stream, int):
            stream = _torch.cuda.ExternalStream(stream, device=device)
        _require(stream is None or stream.device == device, f"stream is on {getattr(stream, 'device', None)}, tensors on {device}")
        self.scope = None if stream is None else _torch.cuda.stream(stream)

    def __enter__(self):
        self.device.__enter__()
        if self.scope is not None:
            self.scope.__enter__()

    def __exit__(self, *exc):
        if self.scope is not None:
            self.scope.__exit__(*exc)
        self.device.__exit__(*exc)


def _on(call, device, stream, *args):
    """call(stream handle, *args) on the device's current stream, or on `stream`."""
    i = device.index
    if stream is None and i == _torch.cuda.current_device():
        return call(_raw_stream(i), *args)
    with _Launch(device, stream):
        return call(_raw_stream(i), *args)


def attention_masked(q, k, v, *, scale, causal=False, softcap=0.0, alibi_slopes=None, doc_ids=None, prefix_lens=None,
                     out=None, stream=None):
    """Attention under masks and score changes (tk_attention_masked_*).

    q: [B, Hq, Sq, D], k, v: [B, Hkv, Skv, D], float16 or bfloat16, any strides with the last
    one 1 (a [B, S, H, D] tensor goes in as its transpose(1, 2)). Returns [B, Hq, Sq, D] of the
    same type, its strides ordered as q's if `out` is not given. alibi_slopes: float32 [Hq];
    doc_ids: int32 [B, Sq] (each run of equal ids a document, negative: padding);
    prefix_lens: int32 [B] (with causal). A row that may see no key is 0."""
    torch = _torch or _import_torch()
    kind, device, kshape = q.dtype, q.device, k.shape
    if not (q.dim() == 4 and k.dim() == 4 and (kind is torch.float16 or kind is torch.bfloat16)
            and device.type == "cuda" and k.dtype is kind and v.dtype is kind and k.device == device and v.device == device
            and v.shape == kshape and q.size(0) == kshape[0] and q.size(3) == kshape[3]
            and (out is None or (out.dtype is kind and out.shape == q.shape and out.device == device))):
        _masked_complaint(q, k, v, out)
    b, h, sq, d = q.shape
    for t, name, dtype, shape in ((alibi_slopes, "alibi_slopes", torch.float32, (h,)), (doc_ids, "doc_ids", torch.int32, (b, sq)),
                                  (prefix_lens, "prefix_lens", torch.int32, (b,))):
        if t is not None:
            _vector(t, name, dtype, shape)
            _require(t.device == device, f"{name} is on {t.device}, expected {device}")

    def call(handle, out):
        if out is None:
            out = torch.empty_like(q)
        if q.is_contiguous() and k.is_contiguous() and v.is_contiguous() and out.is_contiguous():
            strides = None
        else:
            (qb, qh, qs, q1), (kb, kh, ks, k1) = q.stride(), k.stride()
            (vb, vh, vs, v1), (ob, oh, os_, o1) = v.stride(), out.stride()
            _require(d == 1 or (q1 == 1 and k1 == 1 and v1 == 1 and o1 == 1), "the last strides of q, k, v and out must be 1")
            strides = _Strides(qb, qh, qs, kb, kh, ks, vb, vh, vs, ob, oh, os_)
        name = "tk_attention_masked_f16" if kind is torch.float16 else "tk_attention_masked_bf16"
        code = getattr(_lib or lib(), name)(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), strides, b, h, kshape[1], sq, kshape[2], d, scale, softcap,
            alibi_slopes if alibi_slopes is None else alibi_slopes.data_ptr(), doc_ids if doc_ids is None else doc_ids.data_ptr(),
            prefix_lens if prefix_lens is None else prefix_lens.data_ptr(), 1 if causal else 0, handle)
        if code:
            raise TkError(name, code)
        return out

    return _on(call, device, stream, out)


def _masked_complaint(q, k, v, out):
    _half_type(q, "q")
    _require(q.dim() == 4 and k.dim() == 4 and v.shape == k.shape, "q, k, v must be [B, H, S, D], k and v alike")
    _require(k.shape[0] == q.shape[0] and k.shape[3] == q.shape[3], f"k has shape {tuple(k.shape)}, q {tuple(q.shape)}")
    _require(k.dtype == q.dtype and v.dtype == q.dtype, "q, k, v must have one type")
    _same_device(q.device, k=k, v=v, out=out)
    raise ValueError("out must have q's type and shape")


def kv_plan(cached_lens, new_lens, block_table, free_pages, n_free, *, page_size, max_tokens, lens_out=None, seq_lens=None,
            starts=None, slots=None, n_free_out=None, stream=None):
    """Places for the new tokens of a step (tk_kv_plan): fills block_table in place and returns
    (lens, seq_lens, starts, slots, n_free). cached_lens, new_lens: int32 [R]; block_table: int32
    [R, max_pages]; free_pages: int32; n_free: int32 [1]. lens_out may be cached_lens and
    n_free_out n_free, for a state that moves on in place. Outputs that are not given come as
    parts of one new buffer."""
    torch = _torch or _import_torch()
    i32, device = torch.int32, cached_lens.device
    if not (device.type == "cuda" and cached_lens.dim() == 1 and block_table.dim() == 2 and n_free.numel() == 1
            and cached_lens.shape == new_lens.shape and block_table.size(0) == cached_lens.size(0)
            and cached_lens.dtype is i32 and new_lens.dtype is i32 and block_table.dtype is i32 and free_pages.dtype is i32
            and n_free.dtype is i32 and cached_lens.is_contiguous() and new_lens.is_contiguous() and block_table.is_contiguous()
            and free_pages.is_contiguous() and new_lens.device == device and block_table.device == device
            and free_pages.device == device and n_free.device == device):
        _plan_complaint(cached_lens, new_lens, block_table, free_pages, n_free)
    r, width = block_table.shape
    _require(max_tokens >= 0, "max_tokens must not be negative")
    for t, name, dtype, n in ((lens_out, "lens_out", i32, r), (seq_lens, "seq_lens", i32, r), (starts, "starts", i32, r + 1),
                              (slots, "slots", torch.int64, max_tokens), (n_free_out, "n_free_out", i32, 1)):
        if t is not None:
            _vector(t, name, dtype, (n,))
            _require(t.device == device, f"{name} is on {t.device}, expected {device}")

    def call(handle, lens_out, seq_lens, starts, slots, n_free_out):
        if lens_out is None or seq_lens is None or starts is None or slots is None or n_free_out is None:
            # Slots first: they need 8-byte alignment.
            parts = torch.empty(2 * max_tokens + 3 * r + 2, dtype=i32, device=device).split((2 * max_tokens, r, r, r + 1, 1))
            slots = parts[0].view(torch.int64) if slots is None else slots
            lens_out = parts[1] if lens_out is None else lens_out
            seq_lens = parts[2] if seq_lens is None else seq_lens
            starts = parts[3] if starts is None else starts
            n_free_out = parts[4] if n_free_out is None else n_free_out
        code = (_lib or lib()).tk_kv_plan(
            cached_lens.data_ptr(), new_lens.data_ptr(), r, page_size, block_table.data_ptr(), width, free_pages.data_ptr(),
            free_pages.numel(), n_free.data_ptr(), lens_out.data_ptr(), seq_lens.data_ptr(), starts.data_ptr(), slots.data_ptr(),
            max_tokens, n_free_out.data_ptr(), handle)
        if code:
            raise TkError("tk_kv_plan", code)
        return lens_out, seq_lens, starts, slots, n_free_out

    return _on(call, device, stream, lens_out, seq_lens, starts, slots, n_free_out)


def _plan_complaint(cached_lens, new_lens, block_table, free_pages, n_free):
    i32 = _torch.int32
    _require(cached_lens.dim() == 1, "cached_lens must be [R]")
    r = cached_lens.shape[0]
    _vector(cached_lens, "cached_lens", i32, (r,))
    _vector(new_lens, "new_lens", i32, (r,))
    _require(block_table.dim() == 2, "block_table must be [R, max_pages]")
    _vector(block_table, "block_table", i32, (r, block_table.shape[1]))
    _vector(free_pages, "free_pages", i32, free_pages.shape)
    _vector(n_free, "n_free", i32, (1,))
    _same_device(cached_lens.device, new_lens=new_lens, block_table=block_table, free_pages=free_pages, n_free=n_free)


def _cache_complaint(device, k_cache, v_cache, k_scale, v_scale):
    _require(k_cache.dim() == 4, "k_cache must be [pages, Hkv, page_size, D]")
    shape = k_cache.shape
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        _require(t.element_size() == 1, f"{name} must hold bytes (uint8 or float8_e4m3fn)")
        _vector(t, name, t.dtype, shape)
    _vector(k_scale, "k_scale", _torch.float32, shape[:2])
    _vector(v_scale, "v_scale", _torch.float32, shape[:2])
    _same_device(device, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale)


def _cache_ok(torch, device, k_cache, v_cache, k_scale, v_scale):
    f32, shape = torch.float32, k_cache.shape
    return (len(shape) == 4 and v_cache.shape == shape and k_cache.element_size() == 1 and v_cache.element_size() == 1
            and k_scale.dtype is f32 and v_scale.dtype is f32 and k_scale.shape == shape[:2] and v_scale.shape == shape[:2]
            and k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()
            and k_cache.device == device and v_cache.device == device and k_scale.device == device and v_scale.device == device)


def _tokens(t, name, heads, dim):
    """Elements between the tokens of a packed [T, heads, dim] tensor."""
    if t.is_contiguous():
        return heads * dim
    token, head, one = t.stride()
    _require(one == 1 and (heads == 1 or head == dim), f"the heads of a token of {name} must be adjacent")
    return token if t.size(0) > 1 else heads * dim


def kv_append(k, v, slots, k_cache, v_cache, k_scale, v_scale, *, stream=None):
    """Quantises packed tokens k, v [T, Hkv, D] (float16 or bfloat16) into the cache at slots
    (int64 [T], -1: skipped), in place (tk_kv_append_e4m3_*)."""
    torch = _torch or _import_torch()
    kind, device = k.dtype, k.device
    if not ((kind is torch.float16 or kind is torch.bfloat16) and v.dtype is kind and k.dim() == 3 and v.shape == k.shape
            and device.type == "cuda" and v.device == device and slots.device == device and slots.dtype is torch.int64
            and slots.dim() == 1 and slots.size(0) == k.size(0) and slots.is_contiguous()
            and _cache_ok(torch, device, k_cache, v_cache, k_scale, v_scale)
            and k.size(1) == k_cache.size(1) and k.size(2) == k_cache.size(3)):
        _append_complaint(k, v, slots, k_cache, v_cache, k_scale, v_scale)
    n, heads, dim = k.shape
    if n == 0:
        return
    k_stride, v_stride = _tokens(k, "k", heads, dim), _tokens(v, "v", heads, dim)

    def call(handle):
        name = "tk_kv_append_e4m3_f16" if kind is torch.float16 else "tk_kv_append_e4m3_bf16"
        code = getattr(_lib or lib(), name)(
            k.data_ptr(), v.data_ptr(), k_stride, v_stride, slots.data_ptr(), n, heads, dim, k_cache.data_ptr(),
            v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k_cache.size(0), k_cache.size(2), handle)
        if code:
            raise TkError(name, code)

    _on(call, device, stream)


def _append_complaint(k, v, slots, k_cache, v_cache, k_scale, v_scale):
    _half_type(k, "k")
    _cache_complaint(k.device, k_cache, v_cache, k_scale, v_scale)
    _require(k.dim() == 3 and tuple(k.shape[1:]) == (k_cache.shape[1], k_cache.shape[3]),
             f"k must be [T, {k_cache.shape[1]}, {k_cache.shape[3]}], got {tuple(k.shape)}")
    _require(v.dtype == k.dtype and v.shape == k.shape, "k and v must have one type and shape")
    _vector(slots, "slots", _torch.int64, (k.shape[0],))
    _same_device(k.device, v=v, slots=slots)


def attention_paged(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, *, scale, softcap=0.0,
                    alibi_slopes=None, max_query_len=1, max_seq_len=None, out=None, stream=None):
    """Attention of packed newest tokens q [T, Hq, D] over the paged cache
    (tk_attention_paged_e4m3_*); returns [T, Hq, D] of q's type. max_query_len: at least the most
    query tokens of a request; max_seq_len: about the longest context (default: what the block
    table can hold). Rows behind the last request are left as they were in `out`."""
    torch = _torch or _import_torch()
    kind, device, i32 = q.dtype, q.device, torch.int32
    if not ((kind is torch.float16 or kind is torch.bfloat16) and q.dim() == 3 and device.type == "cuda"
            and _cache_ok(torch, device, k_cache, v_cache, k_scale, v_scale) and q.size(2) == k_cache.size(3)
            and block_table.dim() == 2 and block_table.dtype is i32 and seq_lens.dtype is i32 and starts.dtype is i32
            and seq_lens.dim() == 1 and starts.dim() == 1 and seq_lens.size(0) == block_table.size(0)
            and starts.size(0) == block_table.size(0) + 1 and block_table.is_contiguous() and seq_lens.is_contiguous()
            and starts.is_contiguous() and block_table.device == device and seq_lens.device == device and starts.device == device
            and (out is None or (out.dtype is kind and out.shape == q.shape and out.device == device))):
        _paged_complaint(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, out)
    n, h, dim = q.shape
    r, width = block_table.shape
    pages, hkv, page, _ = k_cache.shape
    if alibi_slopes is not None:
        _vector(alibi_slopes, "alibi_slopes", torch.float32, (h,))
        _require(alibi_slopes.device == device, f"alibi_slopes is on {alibi_slopes.device}, expected {device}")
    q_stride = _tokens(q, "q", h, dim)

    def call(handle, out):
        if out is None:
            out, out_stride = torch.empty((n, h, dim), dtype=kind, device=device), h * dim
        else:
            out_stride = _tokens(out, "out", h, dim)
        if n == 0 or r == 0:
            return out
        name = "tk_attention_paged_e4m3_f16" if kind is torch.float16 else "tk_attention_paged_e4m3_bf16"
        code = getattr(_lib or lib(), name)(
            q.data_ptr(), q_stride, out.data_ptr(), out_stride, n, k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
            v_scale.data_ptr(), pages, page, block_table.data_ptr(), width, seq_lens.data_ptr(), starts.data_ptr(), r, h, hkv, dim,
            max_query_len, width * page if max_seq_len is None else max_seq_len, scale, softcap,
            alibi_slopes if alibi_slopes is None else alibi_slopes.data_ptr(), handle)
        if code:
            raise TkError(name, code)
        return out

    return _on(call, device, stream, out)


def _paged_complaint(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, starts, out):
    _half_type(q, "q")
    _cache_complaint(q.device, k_cache, v_cache, k_scale, v_scale)
    _require(q.dim() == 3 and q.shape[2] == k_cache.shape[3], f"q must be [T, Hq, {k_cache.shape[3]}], got {tuple(q.shape)}")
    _require(block_table.dim() == 2, "block_table must be [R, max_pages]")
    r = block_table.shape[0]
    _vector(block_table, "block_table", _torch.int32, block_table.shape)
    _vector(seq_lens, "seq_lens", _torch.int32, (r,))
    _vector(starts, "starts", _torch.int32, (r + 1,))
    _same_device(q.device, block_table=block_table, seq_lens=seq_lens, starts=starts, out=out)
    raise ValueError("out must have q's type and shape")

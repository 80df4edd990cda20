"""Host-side Python mirror of the gfx950 paged KV-cache library (libie_hip.so).

The library's C ABI is declared in include/ie_hip.h; this module binds it with
ctypes -- and, for the calls made per layer and step, with the CPython extension
native_calls.so -- and offers the reference's kernel-launcher interface
(src/cuda/kernels.cuh:69-102) over torch tensors, plus the page allocator
(src/cuda/cuda_runner.cu:191-313) as a class. torch supplies device memory
and streams only; all compute happens in the HIP kernels. Nothing here falls
back to a CPU implementation: every entry point raises if libie_hip.so is
missing or a call fails.

The package directory name is not an identifier; load it with ``load()`` from
``__graft_entry__`` or import it through importlib (tests do).
"""
from __future__ import annotations

import ctypes
import functools
import os
from dataclasses import dataclass

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG_DIR, "libie_hip.so")
CALLS_PATH = os.path.join(PKG_DIR, "native_calls.so")
PAGE_SIZE = 16
KV_F32, KV_F16, KV_BF16 = 0, 1, 2
KV_NAMES = {"f32": KV_F32, "f16": KV_F16, "bf16": KV_BF16}

# Status codes (include/ie_hip.h).
OK, EINVAL, ELAUNCH, EFULL, ERANGE, ESEQ = 0, 1, 2, 3, 4, 5


class IeHipError(RuntimeError):
    """A libie_hip call returned a nonzero status."""

    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


class KvLayout(ctypes.Structure):
    """ie_kv_layout: the reference's KvLayout (src/cuda/kernels.cuh:33-38) + pool size."""

    _fields_ = [("tables", ctypes.c_void_p), ("max_pages", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("kv_dtype", ctypes.c_int32),
                ("num_pages", ctypes.c_int32)]


class Matrix(ctypes.Structure):
    """ie_matrix: the reference's DeviceMatrix (src/cuda/kernels.cuh:40-46), BF16 bits or
    INT8 values with one f32 scale per row."""

    _fields_ = [("data", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("int8", ctypes.c_int32),
                ("rows", ctypes.c_int32), ("cols", ctypes.c_int32)]


class MatrixQ4(ctypes.Structure):
    """ie_matrix_q4: 4-bit weights with a scale (and a zero point) per row and group of columns."""

    _fields_ = [("data", ctypes.c_void_p), ("scale", ctypes.c_void_p), ("zero", ctypes.c_void_p),
                ("scale_dtype", ctypes.c_int32), ("group", ctypes.c_int32),
                ("rows", ctypes.c_int32), ("cols", ctypes.c_int32)]
    tensors, device = (), -1  # set by matrix_q4()


class LogitRules(ctypes.Structure):
    """ie_logit_rules: what the rows of a step ask of their logits before a token is drawn."""

    _fields_ = ([(n, ctypes.c_void_p) for n in (
        "history", "history_start", "history_len", "prompt_len", "repetition", "presence",
        "frequency", "bias_token", "bias_value", "bias_start", "bias_len", "mask", "mask_row")]
        + [("history_size", ctypes.c_int64), ("bias_size", ctypes.c_int64),
           ("mask_rows", ctypes.c_int32)])
    tensors, rows, words = (), None, None  # set by logit_rules()


_vp, _i, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
_SIGS = {
    "ie_hip_last_error": (ctypes.c_char_p, []),
    "ie_hip_version": (ctypes.c_char_p, []),
    "ie_hip_set_attention_impl": (_i, [_i]),
    "ie_hip_rope_table": (_i, [_vp, _i, _i, _f]),
    "ie_hip_set_prefill_rounding": (_i, [_i]),
    "ie_hip_range_push": (None, [ctypes.c_char_p]),
    "ie_hip_range_pop": (None, []),
    "ie_hip_rope_and_cache": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, KvLayout, _i, _i,
                                   _i, _vp]),
    "ie_hip_attention_chunk_tokens": (_i, [_i, _i, _i]),
    "ie_hip_attention_chunks": (_i, [_i, _i]),
    "ie_hip_attention_workspace_bytes": (ctypes.c_size_t, [_i, _i, _i, _i]),
    "ie_hip_attention": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _vp, KvLayout, _i, _i, _vp, _i, _i, _i,
                              _vp]),
    "ie_hip_attention_noalloc": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _vp, KvLayout, _i, _i, _i, _i,
                                      _i, _vp]),
    "ie_hip_attention_plan_ints": (ctypes.c_size_t, [_i, _i, _i]),
    "ie_hip_attention_plan": (_i, [_vp, ctypes.c_size_t, _i, _vp, _vp, _vp, _i, _i, _i, _i]),
    "ie_hip_attention_planned": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _vp, KvLayout, _i, _i, _vp, _vp,
                                      ctypes.c_size_t, _i, _i, _i, _vp]),
    "ie_hip_rope_cache_attention_planned": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp,
                                                 _vp, KvLayout, _i, _i, _vp, _vp, ctypes.c_size_t,
                                                 _i, _i, _i, _vp]),
    "ie_hip_rope_cache_attention_supported": (_i, [_i, _i, _i, _i, _i]),
    "ie_hip_rope_cache_attention": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp,
                                         KvLayout, _i, _i, _vp, _i, _i, _i, _vp]),
    "ie_hip_attention_prefill_supported": (_i, [_i, _i, _i]),
    "ie_hip_attention_prefill": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _vp, KvLayout, _i, _i, _i, _vp]),
    "ie_hip_rope_cache_attention_prefill_supported": (_i, [_i, _i, _i, _i]),
    "ie_hip_rope_cache_attention_prefill": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp,
                                                 _vp, KvLayout, _i, _i, _i, _vp]),
    "ie_hip_gather_rows": (_i, [_vp, _vp, _vp, _i, _i, _vp]),
    "ie_hip_gather_kv": (_i, [_vp, _vp, KvLayout, _i, _i, _i, _vp]),
    "ie_hip_argmax_rows": (_i, [_vp, _vp, _i, _i, _vp]),
    "ie_hip_embedding": (_i, [_vp, _vp, Matrix, _i, _vp]),
    "ie_hip_rmsnorm": (_i, [_vp, _vp, _vp, _i, _i, _f, _vp]),
    "ie_hip_matmul": (_i, [_vp, _vp, Matrix, _vp, _i, _i, _vp]),
    "ie_hip_gate_up_silu": (_i, [_vp, _vp, Matrix, Matrix, _i, _vp]),
    "ie_hip_qkv_proj": (_i, [_vp, _vp, _vp, _vp, Matrix, _vp, _i, _i, _i, _vp]),
    "ie_hip_rmsnorm_qkv_proj": (_i, [_vp, _vp, _vp, _vp, _vp, _f, Matrix, _vp, _i, _i, _i, _vp]),
    "ie_hip_rmsnorm_gate_up_silu": (_i, [_vp, _vp, _vp, _f, Matrix, Matrix, _i, _vp]),
    "ie_hip_matmul_q4_workspace_bytes": (ctypes.c_size_t, [_i, _i]),
    "ie_hip_matmul_q4": (_i, [_vp, _vp, MatrixQ4, _vp, _i, _i, _vp, _vp]),
    "ie_hip_qkv_proj_q4": (_i, [_vp, _vp, _vp, _vp, MatrixQ4, _vp, _i, _i, _i, _vp, _vp]),
    "ie_hip_gate_up_silu_q4": (_i, [_vp, _vp, MatrixQ4, MatrixQ4, _i, _vp, _vp]),
    "ie_hip_adjust_logits": (_i, [_vp, _vp, LogitRules, _i, _i, _vp]),
    "ie_hip_sample_rows_workspace_bytes": (ctypes.c_size_t, [_i, _i]),
    "ie_hip_sample_rows": (_i, [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp]),
    "ie_pages_create": (_vp, [_i, _i, _i]),
    "ie_pages_destroy": (None, [_vp]),
    "ie_pages_open_sequence": (_i, [_vp]),
    "ie_pages_close_sequence": (_i, [_vp, _i]),
    "ie_pages_ensure": (_i, [_vp, _i, _i]),
    "ie_pages_sequence_length": (_i, [_vp, _i]),
    "ie_pages_set_sequence_length": (_i, [_vp, _i, _i]),
    "ie_pages_sequence_pages": (_i, [_vp, _i, _vp, _i]),
    "ie_pages_total_pages": (_i, [_vp]),
    "ie_pages_free_pages": (_i, [_vp]),
    "ie_pages_max_batch": (_i, [_vp]),
    "ie_pages_max_seq_len": (_i, [_vp]),
    "ie_pages_max_pages_per_seq": (_i, [_vp]),
    "ie_pages_host_tables": (_vp, [_vp]),
    "ie_pages_upload_tables": (_i, [_vp, _vp, _vp, _vp]),
    "ie_pages_for": (_i, [_i]),
}
EXPORTED = tuple(_SIGS)

_lib = None


def lib() -> ctypes.CDLL:
    """The loaded libie_hip.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} is missing: build it with __graft_entry__.build() "
                "(there is no fallback implementation)")
        l = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(l, name)
            fn.restype = res
            fn.argtypes = args
        _lib = l
    return _lib


_calls = None


def _native():
    """The CPython extension's entry points (raises if it has not been built)."""
    global _calls
    if _calls is None:
        import importlib.util

        import torch
        if not os.path.exists(CALLS_PATH):
            raise FileNotFoundError(
                f"{CALLS_PATH} is missing: build it with __graft_entry__.build()")
        lib()
        spec = importlib.util.spec_from_file_location("native_calls", CALLS_PATH)
        calls = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(calls)
        calls.set_types(torch.float32, torch.float16, torch.bfloat16, Matrix, MatrixQ4, LogitRules)
        _calls = calls
    return _calls


def last_error() -> str:
    return lib().ie_hip_last_error().decode()


def _check(rc: int) -> None:
    if rc != OK:
        raise IeHipError(rc, last_error())


_raw_stream = None


def _stream(stream=None) -> int:
    global _raw_stream
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None:
        import torch
        torch.cuda.current_stream()  # initialises the device
        get, device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
        _raw_stream = lambda: get(device())
    return _raw_stream()


def layout(tables, max_pages: int, num_pages: int, kv_dtype: int) -> KvLayout:
    return KvLayout(tables.data_ptr(), max_pages, PAGE_SIZE, kv_dtype, num_pages)


def torch_kv_dtype(kv_dtype: int):
    import torch
    return {KV_F32: torch.float32, KV_F16: torch.float16, KV_BF16: torch.bfloat16}[kv_dtype]


IMPL_AUTO, IMPL_VALU, IMPL_MFMA = 0, 1, 2


def set_attention_impl(impl: int) -> int:
    """Process-wide attention kernel choice (AUTO / VALU / MFMA); returns the previous one."""
    return int(lib().ie_hip_set_attention_impl(impl))


PREFILL_SINGLE, PREFILL_SPLIT = 0, 1


def set_prefill_rounding(mode: int) -> int:
    """Process-wide operand precision of the f16 matrix-core prefill (SINGLE: q and P
    rounded once to f16; SPLIT: hi + lo halves); returns the previous one."""
    return int(lib().ie_hip_set_prefill_rounding(mode))


# ------------------------------------------------------------ kernels ----
def rope_table(n_pos: int, head_dim: int, theta: float):
    """Host RoPE table [n_pos, head_dim] (cos | sin) as a CPU float32 tensor."""
    import torch
    t = torch.empty((n_pos, head_dim), dtype=torch.float32)
    _check(lib().ie_hip_rope_table(t.data_ptr(), n_pos, head_dim, theta))
    return t


def rope_and_cache(q, k, v, k_pool, v_pool, table, row_pos, row_seq, tables, max_pages: int,
                   n_heads: int, n_kv_heads: int, head_dim: int, stream=None) -> None:
    """rope_and_cache (src/cuda/kernels.cuh:72-74); q may be None (append only)."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_rope_and_cache(
        q, k, v, k_pool, v_pool, table, table.shape[0], T, row_pos, row_seq, kv, n_heads,
        n_kv_heads, head_dim, _stream(stream)))


def attention_chunk_tokens(T: int, max_context: int, kv_dtype: int = KV_F16) -> int:
    """Chunk size for T rows of up to max_context tokens (kv_dtype picks the kernel)."""
    return int(lib().ie_hip_attention_chunk_tokens(T, max_context, kv_dtype))


def attention_chunks(context: int, chunk_tokens: int) -> int:
    return int(lib().ie_hip_attention_chunks(context, chunk_tokens))


def attention_workspace(T: int, n_heads: int, head_dim: int, num_chunks: int, device="cuda"):
    import torch
    n = int(lib().ie_hip_attention_workspace_bytes(T, n_heads, head_dim, num_chunks))
    return torch.zeros(max(n, 256), dtype=torch.uint8, device=device)


def attention(out, q, k_pool, v_pool, row_pos, row_seq, tables, max_pages: int, num_chunks: int,
              chunk_tokens: int, workspace, n_heads: int, n_kv_heads: int, head_dim: int,
              stream=None) -> None:
    """Flash-decoding attention (src/cuda/kernels.cuh:84-87)."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_attention(
        out, q, k_pool, v_pool, T, row_pos, row_seq, kv, num_chunks, chunk_tokens, workspace,
        n_heads, n_kv_heads, head_dim, _stream(stream)))


NOALLOC_SCRATCH_BYTES = 16 << 20  # IE_HIP_NOALLOC_SCRATCH_BYTES


def attention_noalloc(out, q, k_pool, v_pool, row_pos, row_seq, tables, max_pages: int,
                      num_chunks: int, chunk_tokens: int, n_heads: int, n_kv_heads: int,
                      head_dim: int, stream=None) -> None:
    """attention() with the library's fixed device scratch in place of a workspace."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_attention_noalloc(
        out, q, k_pool, v_pool, T, row_pos, row_seq, kv, num_chunks, chunk_tokens, n_heads,
        n_kv_heads, head_dim, _stream(stream)))


def attention_plan_ints(T: int, num_chunks: int, chunk_tokens: int) -> int:
    return int(lib().ie_hip_attention_plan_ints(T, num_chunks, chunk_tokens))


def attention_plan(row_pos, row_seq, tables, num_chunks: int, chunk_tokens: int):
    """The decode work list for one launch, built on the host from host copies (numpy
    int32) of the rows' positions and sequences and of the block table [seqs, max_pages];
    returns it as a numpy int32 array (copy it to the device for attention_planned)."""
    import numpy as np
    row_pos = np.ascontiguousarray(row_pos, dtype=np.int32)
    row_seq = np.ascontiguousarray(row_seq, dtype=np.int32)
    tables = np.ascontiguousarray(tables, dtype=np.int32)
    T = row_pos.size
    n = int(lib().ie_hip_attention_plan_ints(max(T, 1), num_chunks, chunk_tokens))
    if n == 0:
        raise IeHipError(EINVAL, "attention_plan: bad chunk arguments")
    plan = np.zeros(n, np.int32)
    _check(lib().ie_hip_attention_plan(plan.ctypes.data, n, T, row_pos.ctypes.data,
                                       row_seq.ctypes.data, tables.ctypes.data, tables.shape[0],
                                       tables.shape[1], num_chunks, chunk_tokens))
    return plan


def attention_planned(out, q, k_pool, v_pool, row_pos, row_seq, tables, max_pages: int,
                      num_chunks: int, chunk_tokens: int, workspace, plan, n_heads: int,
                      n_kv_heads: int, head_dim: int, stream=None) -> None:
    """attention() with a device copy of attention_plan()'s work list."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_attention_planned(
        out, q, k_pool, v_pool, T, row_pos, row_seq, kv, num_chunks, chunk_tokens, workspace,
        plan, plan.numel(), n_heads, n_kv_heads, head_dim, _stream(stream)))


def rope_cache_attention_planned(out, q, k, v, k_pool, v_pool, table, row_pos, row_seq, tables,
                                 max_pages: int, num_chunks: int, chunk_tokens: int, workspace,
                                 plan, n_heads: int, n_kv_heads: int, head_dim: int,
                                 stream=None) -> None:
    """rope_cache_attention() with a device copy of attention_plan()'s work list."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_rope_cache_attention_planned(
        out, q, k, v, k_pool, v_pool, table, table.shape[0], T, row_pos, row_seq, kv, num_chunks,
        chunk_tokens, workspace, plan, plan.numel(), n_heads, n_kv_heads, head_dim,
        _stream(stream)))


def rope_cache_attention_supported(kv_dtype: int, n_heads: int, n_kv_heads: int, head_dim: int,
                                   chunk_tokens: int) -> bool:
    return bool(lib().ie_hip_rope_cache_attention_supported(kv_dtype, n_heads, n_kv_heads,
                                                            head_dim, chunk_tokens))


def rope_cache_attention(out, q, k, v, k_pool, v_pool, table, row_pos, row_seq, tables,
                         max_pages: int, num_chunks: int, chunk_tokens: int, workspace,
                         n_heads: int, n_kv_heads: int, head_dim: int, stream=None) -> None:
    """rope_and_cache + attention of one decode step in one launch (q is not modified)."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_rope_cache_attention(
        out, q, k, v, k_pool, v_pool, table, table.shape[0], T, row_pos, row_seq, kv, num_chunks,
        chunk_tokens, workspace, n_heads, n_kv_heads, head_dim, _stream(stream)))


def rope_cache_attention_prefill_supported(kv_dtype: int, n_heads: int, n_kv_heads: int,
                                           head_dim: int) -> bool:
    return bool(lib().ie_hip_rope_cache_attention_prefill_supported(kv_dtype, n_heads, n_kv_heads,
                                                                    head_dim))


def rope_cache_attention_prefill(out, q, k, v, k_pool, v_pool, table, row_pos, row_seq, tables,
                                 max_pages: int, n_heads: int, n_kv_heads: int, head_dim: int,
                                 stream=None) -> None:
    """rope_and_cache + attention_prefill of one prompt chunk, q rotated inside the prefill
    kernel (q is not modified)."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_rope_cache_attention_prefill(
        out, q, k, v, k_pool, v_pool, table, table.shape[0], T, row_pos, row_seq, kv, n_heads,
        n_kv_heads, head_dim, _stream(stream)))


def attention_prefill_supported(n_heads: int, n_kv_heads: int, head_dim: int) -> bool:
    return bool(lib().ie_hip_attention_prefill_supported(n_heads, n_kv_heads, head_dim))


def attention_prefill(out, q, k_pool, v_pool, row_pos, row_seq, tables, max_pages: int,
                      n_heads: int, n_kv_heads: int, head_dim: int, stream=None) -> None:
    """Prompt attention (src/cuda/kernels.cuh:93-96)."""
    T = row_pos.numel()
    kv = (tables, max_pages, k_pool, n_kv_heads * head_dim)
    _check(_native().ie_hip_attention_prefill(
        out, q, k_pool, v_pool, T, row_pos, row_seq, kv, n_heads, n_kv_heads, head_dim,
        _stream(stream)))


def gather_rows(dst, src, rows, stream=None) -> None:
    """dst[r] = src[rows[r]] (src/cuda/kernels.cuh:101-102)."""
    _check(_native().ie_hip_gather_rows(
        dst, src, rows, rows.numel(), src.shape[-1], _stream(stream)))


def argmax_rows(out, logits, stream=None) -> None:
    """out[r] = first index of the maximum of logits[r] (src/cuda/kernels.cuh:106)."""
    _check(_native().ie_hip_argmax_rows(
        out, logits, logits.shape[0], logits.shape[1], _stream(stream)))


def matrix(data, scale=None) -> Matrix:
    """An ie_matrix over a device tensor of BF16 bits (int16/uint16/bfloat16) or INT8
    values [rows, cols] and, for INT8, its f32 row scales."""
    import torch
    int8 = data.dtype == torch.int8
    if int8 and scale is None:
        raise ValueError("INT8 weights need their row scales")
    return Matrix(data.data_ptr(), scale.data_ptr() if int8 else None, int(int8), data.shape[0],
                  data.shape[1])


def embedding(x, ids, e: Matrix, stream=None) -> None:
    """x[t] = E[ids[t]] widened to f32 (src/cuda/kernels.cuh:48-49)."""
    _check(_native().ie_hip_embedding(x, ids, e, ids.numel(), _stream(stream)))


def rmsnorm(y, x, weight, eps: float, stream=None) -> None:
    """y = x / rms(x) * weight per row (src/cuda/kernels.cuh:51-53)."""
    dim = weight.numel()
    _check(_native().ie_hip_rmsnorm(y, x, weight, x.numel() // dim, dim, eps, _stream(stream)))


def matmul(y, x, w: Matrix, bias=None, accumulate: bool = False, stream=None) -> None:
    """y (+)= x . W^T * scale + bias (src/cuda/kernels.cuh:55-62)."""
    _check(_native().ie_hip_matmul(
        y, x, w, bias, x.numel() // w.cols, int(accumulate), _stream(stream)))


def qkv_proj(q, k, v, x, w_qkv: Matrix, b_qkv=None, stream=None) -> None:
    """q, k, v = x . [Wq; Wk; Wv]^T + [bq; bk; bv] in one launch."""
    q_dim, kv_dim = q.shape[-1], k.shape[-1]
    _check(_native().ie_hip_qkv_proj(
        q, k, v, x, w_qkv, b_qkv, x.numel() // w_qkv.cols, q_dim, kv_dim, _stream(stream)))


def gate_up_silu(out, x, w_gate: Matrix, w_up: Matrix, stream=None) -> None:
    """out = silu(x . Wg^T) * (x . Wu^T) (src/cuda/kernels.cuh:64-66)."""
    _check(_native().ie_hip_gate_up_silu(
        out, x, w_gate, w_up, x.numel() // w_gate.cols, _stream(stream)))


def rmsnorm_qkv_proj(q, k, v, x, norm, eps: float, w_qkv: Matrix, b_qkv=None,
                     stream=None) -> None:
    """qkv_proj(rmsnorm(x, norm, eps)) in one launch (no reference counterpart)."""
    q_dim, kv_dim = q.shape[-1], k.shape[-1]
    _check(_native().ie_hip_rmsnorm_qkv_proj(
        q, k, v, x, norm, eps, w_qkv, b_qkv, x.numel() // w_qkv.cols, q_dim, kv_dim,
        _stream(stream)))


def rmsnorm_gate_up_silu(out, x, norm, eps: float, w_gate: Matrix, w_up: Matrix,
                         stream=None) -> None:
    """gate_up_silu(rmsnorm(x, norm, eps)) in one launch (no reference counterpart)."""
    _check(_native().ie_hip_rmsnorm_gate_up_silu(
        out, x, norm, eps, w_gate, w_up, x.numel() // w_gate.cols, _stream(stream)))


# ---------------------------------------- 4-bit weights, logits to tokens ----
def _tensor(t, name: str, dtype, shape, like=None):
    """Refuses a tensor the kernels would read wrongly: another type or shape, elements that do
    not follow each other, another device than `like` (the call's first tensor) or, for that
    one, than the current device, whose stream the launch goes to."""
    if t.dtype != dtype:
        raise IeHipError(EINVAL, f"{name}: expected {dtype}, not {t.dtype}")
    if shape is not None and t.shape != shape:
        raise IeHipError(EINVAL, f"{name}: expected shape {tuple(shape)}, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise IeHipError(EINVAL, f"{name}: must be contiguous")
    device = t.get_device()
    if like is not None:
        if device != like.get_device():
            raise IeHipError(EINVAL, f"{name}: on {t.device}, not on {like.device}")
    elif device < 0 or device != _current_device():
        raise IeHipError(EINVAL, f"{name}: on {t.device}, not on the current GPU")


_get_device = None


def _current_device() -> int:
    global _get_device
    if _get_device is None:
        import torch
        torch.cuda.current_device()  # initialises the device
        _get_device = torch._C._cuda_getDevice
    return _get_device()


def _f32():
    import torch
    return torch.float32


def _tokens(x, w: "MatrixQ4", name: str) -> int:
    """Rows of the activations x [..., w.cols]; checks x as _tensor does."""
    cols, device = w.cols, w.device
    T = x.numel() // cols
    if not (device >= 0 and _native().fits(x, T * cols, cols, device) and device == _current_device()):
        _tensor(x, f"{name}: x", _f32(), None)
        if x.dim() == 0 or x.shape[-1] != cols:
            raise IeHipError(EINVAL, f"{name}: x must have {cols} columns")
        raise IeHipError(EINVAL, f"{name}: the weights are not on {x.device}")
    return T


def _rows_of(t, rows: int, cols: int, name: str, like, device: int) -> None:
    """t holds `rows` rows of `cols` f32 values on `device`, which is like's."""
    if not _native().fits(t, rows * cols, cols, device):
        _tensor(t, name, _f32(), None, like)
        raise IeHipError(EINVAL, f"{name}: expected {rows} rows of {cols}, not {tuple(t.shape)}")


def _workspace(workspace, need: int, name: str, like):
    """The workspace checked, or None where the call needs none."""
    if need == 0:
        return None
    if workspace is None:
        raise IeHipError(EINVAL, f"{name}: needs a workspace of {need} bytes")
    if workspace.get_device() != like.get_device():
        raise IeHipError(EINVAL, f"{name}: workspace on {workspace.device}, not on {like.device}")
    if not workspace.is_contiguous() or workspace.numel() * workspace.element_size() < need:
        raise IeHipError(EINVAL, f"{name}: needs a contiguous workspace of {need} bytes")
    return workspace


def matrix_q4(data, scale, group: int, zero=None) -> MatrixQ4:
    """An ie_matrix_q4 over device tensors: packed weights, uint8 [rows, cols / 2] (even columns
    in the low halves); scales [rows, ceil(cols / group)] in float32, float16 or bfloat16; zero
    points, uint8 of the scales' shape, or None for 8. The tensors are kept with it."""
    import torch
    kinds = {torch.float32: KV_F32, torch.float16: KV_F16, torch.bfloat16: KV_BF16}
    if data.dim() != 2 or data.dtype != torch.uint8 or not data.is_contiguous():
        raise IeHipError(EINVAL, "matrix_q4: data must be contiguous uint8 [rows, cols / 2]")
    if group not in (32, 64, 128):
        raise IeHipError(EINVAL, "matrix_q4: groups must be of 32, 64 or 128 columns")
    rows, cols = data.shape[0], 2 * data.shape[1]
    shape = (rows, -(-cols // group))
    if scale.dtype not in kinds:
        raise IeHipError(EINVAL, f"matrix_q4: scales of {scale.dtype}")
    _tensor(scale, "matrix_q4: scale", scale.dtype, shape, data)
    if zero is not None:
        _tensor(zero, "matrix_q4: zero", torch.uint8, shape, data)
    m = MatrixQ4(data.data_ptr(), scale.data_ptr(), None if zero is None else zero.data_ptr(),
                 kinds[scale.dtype], group, rows, cols)
    m.tensors, m.device = (data, scale, zero), data.get_device()
    return m


def matmul_q4_workspace(T: int, cols: int, device="cuda"):
    """A workspace for the products of T tokens of `cols` columns (of fewer tokens, too)."""
    import torch
    n = int(lib().ie_hip_matmul_q4_workspace_bytes(T, cols))
    return torch.empty(max(n, 256), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=4096)
def _q4_need(T: int, cols: int) -> int:
    return int(lib().ie_hip_matmul_q4_workspace_bytes(T, cols))


def _q4_workspace(workspace, T: int, w: MatrixQ4, name: str, like):
    return _workspace(workspace, _q4_need(T, w.cols), name, like)


def matmul_q4(y, x, w: MatrixQ4, bias=None, accumulate: bool = False, workspace=None,
              stream=None) -> None:
    """matmul() over a 4-bit matrix: y (+)= x . W^T + bias (no reference counterpart)."""
    T = _tokens(x, w, "matmul_q4")
    _rows_of(y, T, w.rows, "matmul_q4: y", x, w.device)
    if bias is not None:
        _rows_of(bias, 1, w.rows, "matmul_q4: bias", x, w.device)
    ws = _q4_workspace(workspace, T, w, "matmul_q4", x)
    _check(_native().ie_hip_matmul_q4(y, x, w, bias, T, int(accumulate), ws, _stream(stream)))


def qkv_proj_q4(q, k, v, x, w_qkv: MatrixQ4, b_qkv=None, workspace=None, stream=None) -> None:
    """qkv_proj() over a 4-bit matrix (no reference counterpart)."""
    T = _tokens(x, w_qkv, "qkv_proj_q4")
    q_dim, kv_dim = q.shape[-1], k.shape[-1]
    _rows_of(q, T, q_dim, "qkv_proj_q4: q", x, w_qkv.device)
    _rows_of(k, T, kv_dim, "qkv_proj_q4: k", x, w_qkv.device)
    _rows_of(v, T, kv_dim, "qkv_proj_q4: v", x, w_qkv.device)
    if b_qkv is not None:
        _rows_of(b_qkv, 1, w_qkv.rows, "qkv_proj_q4: bias", x, w_qkv.device)
    ws = _q4_workspace(workspace, T, w_qkv, "qkv_proj_q4", x)
    _check(_native().ie_hip_qkv_proj_q4(q, k, v, x, w_qkv, b_qkv, T, q_dim, kv_dim, ws,
                                        _stream(stream)))


def gate_up_silu_q4(out, x, w_gate: MatrixQ4, w_up: MatrixQ4, workspace=None, stream=None) -> None:
    """gate_up_silu() over two 4-bit matrices (no reference counterpart)."""
    T = _tokens(x, w_gate, "gate_up_silu_q4")
    if w_up.device != w_gate.device:
        raise IeHipError(EINVAL, "gate_up_silu_q4: gate and up on two devices")
    _rows_of(out, T, w_gate.rows, "gate_up_silu_q4: out", x, w_gate.device)
    ws = _q4_workspace(workspace, T, w_gate, "gate_up_silu_q4", x)
    _check(_native().ie_hip_gate_up_silu_q4(out, x, w_gate, w_up, T, ws, _stream(stream)))


def logit_rules(history=None, prompt_len=None, repetition=None, presence=None, frequency=None,
                bias=None, mask=None, mask_row=None) -> LogitRules:
    """The rules of R rows for adjust_logits, over device tensors that are kept with it: history
    = (token ids, start [R], length [R]) and prompt_len [R], int32; repetition, presence and
    frequency [R], float32; bias = (tokens int32, values float32, start [R], length [R]); mask
    [mask rows, ceil(n / 32)] int32 words and mask_row [R] int32 (negative: none)."""
    import torch
    i32, f32 = torch.int32, torch.float32
    r, keep, rows = LogitRules(), [], None

    def put(field, t, dtype, per_row=True):
        nonlocal rows
        if per_row:
            if rows is None:
                rows = t.numel()
            _tensor(t, f"logit_rules: {field}", dtype, (rows,), keep[0] if keep else t)
        else:
            _tensor(t, f"logit_rules: {field}", dtype, None, keep[0] if keep else t)
        keep.append(t)
        setattr(r, field, t.data_ptr())

    if history is not None:
        put("history", history[0], i32, False)
        put("history_start", history[1], i32)
        put("history_len", history[2], i32)
        r.history_size = history[0].numel()
    elif any(t is not None for t in (prompt_len, repetition, presence, frequency)):
        raise IeHipError(EINVAL, "logit_rules: penalties need a history")
    for field, t, dtype in (("prompt_len", prompt_len, i32), ("repetition", repetition, f32),
                            ("presence", presence, f32), ("frequency", frequency, f32)):
        if t is not None:
            put(field, t, dtype)
    if bias is not None:
        put("bias_token", bias[0], i32, False)
        put("bias_value", bias[1], f32, False)
        if bias[0].numel() != bias[1].numel():
            raise IeHipError(EINVAL, "logit_rules: as many bias values as tokens")
        put("bias_start", bias[2], i32)
        put("bias_len", bias[3], i32)
        r.bias_size = bias[0].numel()
    if mask is not None:
        put("mask", mask, i32, False)
        if mask.dim() != 2:
            raise IeHipError(EINVAL, "logit_rules: mask must be [mask rows, words]")
        r.mask_rows = mask.shape[0]
        if mask_row is not None:
            put("mask_row", mask_row, i32)
    elif mask_row is not None:
        raise IeHipError(EINVAL, "logit_rules: mask rows without a mask")
    r.tensors, r.rows, r.words = tuple(keep), rows, None if mask is None else mask.shape[1]
    return r


def adjust_logits(out, logits, rules: LogitRules, stream=None) -> None:
    """out = logits [R, n] under the rules (the penalty of src/sampler.cpp, biases and masks);
    out may be logits."""
    import torch
    _tensor(logits, "adjust_logits: logits", torch.float32, None)
    if logits.dim() != 2:
        raise IeHipError(EINVAL, "adjust_logits: logits must be [R, n]")
    R, n = logits.shape
    _tensor(out, "adjust_logits: out", torch.float32, (R, n), logits)
    if rules.rows is not None and rules.rows != R:
        raise IeHipError(EINVAL, f"adjust_logits: rules of {rules.rows} rows for {R}")
    if rules.words is not None and rules.words != -(-n // 32):
        raise IeHipError(EINVAL, f"adjust_logits: a mask of {rules.words} words for {n} tokens")
    if rules.tensors and rules.tensors[0].get_device() != logits.get_device():
        raise IeHipError(EINVAL, f"adjust_logits: rules on {rules.tensors[0].device}")
    _check(_native().ie_hip_adjust_logits(out, logits, rules, R, n, _stream(stream)))


def sample_rows_workspace(R: int, n: int, device="cuda"):
    """A workspace for sample_rows of up to R rows of up to n logits."""
    import torch
    b = int(lib().ie_hip_sample_rows_workspace_bytes(R, n))
    return torch.empty(max(b, 256), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=4096)
def _sample_need(R: int, n: int) -> int:
    return int(lib().ie_hip_sample_rows_workspace_bytes(R, n))


def sample_rows(out, logits, temperature, u, top_k=None, top_p=None, min_p=None, workspace=None,
                stream=None) -> None:
    """out[r] = a token of logits[r] drawn at u[r] under its temperature, top-k, min-p and top-p
    (src/sampler.cpp after its penalty); temperature <= 0 takes the largest."""
    import torch
    _tensor(logits, "sample_rows: logits", torch.float32, None)
    if logits.dim() != 2:
        raise IeHipError(EINVAL, "sample_rows: logits must be [R, n]")
    R, n = logits.shape
    for name, t, dtype in (("out", out, torch.int32), ("temperature", temperature, torch.float32),
                           ("u", u, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if t is not None:
            _tensor(t, f"sample_rows: {name}", dtype, (R,), logits)
    ws = _workspace(workspace, _sample_need(R, n), "sample_rows", logits)
    _check(_native().ie_hip_sample_rows(out, logits, temperature, top_k, top_p, min_p, u, R, n, ws,
                                        _stream(stream)))


def gather_kv(dst, pool, tables, max_pages: int, seq: int, length: int, kv_dim: int,
              stream=None) -> None:
    """Contiguous fp32 copy of one sequence's paged rows."""
    kv = (tables, max_pages, pool, kv_dim)
    _check(_native().ie_hip_gather_kv(dst, pool, kv, seq, length, kv_dim, _stream(stream)))


# -------------------------------------------------------- page allocator ----
class PagePool:
    """The BatchRunner page allocator (src/cuda/cuda_runner.cu:191-313), host side."""

    def __init__(self, num_pages: int, max_batch: int, max_seq_len: int):
        self._h = lib().ie_pages_create(num_pages, max_batch, max_seq_len)
        if not self._h:
            raise IeHipError(EINVAL, last_error())

    def close(self) -> None:
        if self._h:
            lib().ie_pages_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def open_sequence(self) -> int:
        return int(lib().ie_pages_open_sequence(self._h))

    def close_sequence(self, seq: int) -> None:
        _check(lib().ie_pages_close_sequence(self._h, seq))

    def ensure(self, seq: int, length: int) -> None:
        _check(lib().ie_pages_ensure(self._h, seq, length))

    def sequence_length(self, seq: int) -> int:
        return int(lib().ie_pages_sequence_length(self._h, seq))

    def set_sequence_length(self, seq: int, length: int) -> None:
        _check(lib().ie_pages_set_sequence_length(self._h, seq, length))

    def pages(self, seq: int) -> list[int]:
        n = lib().ie_pages_sequence_pages(self._h, seq, None, 0)
        buf = (ctypes.c_int32 * max(n, 1))()
        lib().ie_pages_sequence_pages(self._h, seq, buf, n)
        return list(buf[:n])

    @property
    def total_pages(self) -> int:
        return int(lib().ie_pages_total_pages(self._h))

    @property
    def free_pages(self) -> int:
        return int(lib().ie_pages_free_pages(self._h))

    @property
    def max_batch(self) -> int:
        return int(lib().ie_pages_max_batch(self._h))

    @property
    def max_seq_len(self) -> int:
        return int(lib().ie_pages_max_seq_len(self._h))

    @property
    def max_pages_per_seq(self) -> int:
        return int(lib().ie_pages_max_pages_per_seq(self._h))

    def host_tables(self) -> list[int]:
        n = self.max_batch * self.max_pages_per_seq
        p = lib().ie_pages_host_tables(self._h)
        return list((ctypes.c_int32 * n).from_address(p))

    def upload_tables(self, device_tables, stream=None) -> bool:
        up = ctypes.c_int(0)
        _check(lib().ie_pages_upload_tables(self._h, device_tables.data_ptr(), _stream(stream),
                                            ctypes.byref(up)))
        return bool(up.value)


def pages_for(tokens: int) -> int:
    return int(lib().ie_pages_for(tokens))

"""ctypes bindings of the C ABI (``include/tokenserve_b200.h``) with torch-tensor wrappers.

The wrappers only translate tensors into pointers, sizes and the current CUDA stream; all
compute happens in the CUDA kernels of ``libtokenserve_b200.so``. There is no fallback: if the
library is missing or a call fails, a :class:`KernelError` is raised.
"""

from __future__ import annotations

import ctypes
import threading
from pathlib import Path

import torch

LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libtokenserve_b200.so"
ABI_VERSION = 1

TS_FLOAT32, TS_FLOAT16, TS_BFLOAT16 = 0, 1, 2
TS_ERR_INVALID_ARGUMENT, TS_ERR_UNSUPPORTED, TS_ERR_WORKSPACE, TS_ERR_MISALIGNED = -1, -2, -3, -4
DTYPE_CODES = {torch.float32: TS_FLOAT32, torch.float16: TS_FLOAT16, torch.bfloat16: TS_BFLOAT16}

_p = ctypes.c_void_p
_i32 = ctypes.c_int32
_i64 = ctypes.c_int64
_f32 = ctypes.c_float
_sz = ctypes.c_size_t

_SIGNATURES: dict[str, tuple[object, list[object]]] = {
    "ts_version": (ctypes.c_int, []),
    "ts_last_error": (ctypes.c_char_p, []),
    "ts_reshape_and_cache": (
        ctypes.c_int,
        [_p, _p, _i64, _i64, _p, _p, _p, _i64, _i32, _i32, _i32, _i64, _i32, _p, _p, _p, _p],
    ),
    "ts_paged_decode_workspace_size": (_sz, [_i32, _i32, _i32, _i32, _i32, _i32, _i32]),
    "ts_paged_decode": (
        ctypes.c_int,
        [_p, _p, _i64, _p, _p, _p, _i32, _p, _i32, _i32, _i32, _i32, _i32, _i64, _f32, _i32,
         _p, _sz, _p],
    ),
    "ts_paged_decode_planned": (
        ctypes.c_int,
        [_p, _p, _i64, _p, _p, _p, _i32, _p, _i32, _i32, _i32, _i32, _i32, _i64, _f32, _i32,
         _p, _sz, _p],
    ),
    "ts_paged_prefill": (
        ctypes.c_int,
        [_p, _p, _i64, _p, _p, _p, _i32, _p, _p, _i32, _i32, _i32, _i32, _i32, _i32, _i32,
         _i64, _f32, _i32, _p],
    ),
    "ts_copy_blocks": (ctypes.c_int, [_p, _i64, _i64, _i64, _i64, _p, _i64, _p, _p]),
    "ts_verify_tags": (ctypes.c_int, [_p, _p, _i32, _p, _p, _p, _i32, _i32, _i64, _p, _p]),
    "ts_swap_blocks": (
        ctypes.c_int, [_p, _i64, _i64, _p, _i64, _i64, _i64, _i64, _p, _i64, _p, _p]
    ),
    "ts_paged_decode_peer": (
        ctypes.c_int,
        [_p, _i32, _i32, _p, ctypes.c_uint32, _p, _i64, _p, _p, _p, _i32, _p, _i32, _i32, _i32,
         _i32, _i32, _i64, _f32, _i32, _p, ctypes.c_size_t, _i32, _p],
    ),
    "ts_paged_decode_publish": (
        ctypes.c_int,
        [_p, _i32, _i32, _p, ctypes.c_uint32, _p, _i64, _p, _p, _p, _i32, _p, _i32, _i32, _i32,
         _i32, _i32, _i64, _f32, _i32, _p, ctypes.c_size_t, _i32, _p],
    ),
    "ts_gather_peers": (
        ctypes.c_int, [_p, _i32, _i32, _p, ctypes.c_uint32, _i32, _i32, _i32, _i32, _p, _p]
    ),
    "ts_wait_peers": (ctypes.c_int, [_p, _i32, ctypes.c_uint32, _p, _p]),
    "ts_peer_alloc": (ctypes.c_int, [ctypes.c_size_t, ctypes.POINTER(ctypes.c_void_p)]),
    "ts_peer_free": (ctypes.c_int, [_p]),
    "ts_ipc_get_handle": (ctypes.c_int, [_p, _p]),
    "ts_ipc_open": (ctypes.c_int, [_p, ctypes.POINTER(ctypes.c_void_p)]),
    "ts_ipc_close": (ctypes.c_int, [_p]),
    "ts_add_rmsnorm": (ctypes.c_int, [_p, _p, _p, _p, _i64, _i32, _f32, _i32, _p]),
    "ts_rope_and_cache": (
        ctypes.c_int,
        [_p, _i64, _p, _p, _p, _p, _p, _p, _i64, _i32, _i32, _i32, _i32, _i64, _i32, _p, _p],
    ),
    "ts_silu_mul": (ctypes.c_int, [_p, _p, _i64, _i32, _i32, _p]),
    "ts_reshape_and_cache_fp8": (
        ctypes.c_int,
        [_p, _p, _i64, _i64, _p, _p, _p, _p, _p, _i64, _i32, _i32, _i32, _i64, _i32, _p, _p, _p,
         _p],
    ),
    "ts_rotary_and_cache": (
        ctypes.c_int,
        [_p, _i64, _p, _p, _p, _p, _p, _p, _p, _p, _i64, _i32, _i32, _i32, _i32, _i32, _f32, _i32,
         _i64, _i32, _p, _p],
    ),
    "ts_read_cache_fp8": (
        ctypes.c_int,
        [_p, _p, _p, _p, _p, _p, _p, _i32, _p, _i32, _i64, _i32, _i32, _i32, _i64, _i32, _p, _p],
    ),
    "ts_paged_decode_fp8": (
        ctypes.c_int,
        [_p, _p, _i64, _p, _p, _p, _p, _p, _i32, _p, _i32, _i32, _i32, _i32, _i32, _i64, _f32,
         _i32, _p, _sz, _i32, _p],
    ),
    "ts_paged_prefill_fp8": (
        ctypes.c_int,
        [_p, _p, _i64, _p, _p, _p, _p, _p, _i32, _p, _p, _i32, _i32, _i32, _i32, _i32, _i32,
         _i32, _i64, _f32, _i32, _p],
    ),
}

_lib: ctypes.CDLL | None = None
_lock = threading.Lock()


class KernelError(RuntimeError):
    """A tokenserve_b200 kernel call was rejected or failed to launch."""


def load_library() -> ctypes.CDLL:
    """Loads (once) and returns the kernel library; raises if it was not built."""
    global _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not LIB_PATH.exists():
            raise KernelError(
                f"{LIB_PATH} is missing; build it with `python -m tokenserve_b200._build` "
                "(there is no CPU fallback)"
            )
        lib = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        if lib.ts_version() != ABI_VERSION:
            raise KernelError(f"ABI version {lib.ts_version()} != {ABI_VERSION}")
        _lib = lib
        return lib


def exported_symbols() -> list[str]:
    return list(_SIGNATURES)


def _check(code: int, what: str) -> None:
    if code != 0:
        msg = load_library().ts_last_error().decode(errors="replace")
        raise KernelError(f"{what} failed (status {code}): {msg}")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _dtype(t: torch.Tensor) -> int:
    try:
        return DTYPE_CODES[t.dtype]
    except KeyError:
        raise KernelError(f"unsupported dtype {t.dtype}") from None


def _rows(t: torch.Tensor, heads: int, head_dim: int, what: str) -> int:
    """Token stride (elements) of a [tokens, heads, head_dim] view with contiguous rows."""
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != head_dim:
        raise KernelError(f"{what}: expected [tokens, {heads}, {head_dim}], got {tuple(shape)}")
    stride = t.stride()
    if stride[2] != 1 or stride[1] != head_dim:
        raise KernelError(f"{what}: heads and head_dim must be contiguous")
    return stride[0]


def _pool_dims(pool: torch.Tensor) -> tuple[int, int, int, int]:
    if pool.dim() != 4 or not pool.is_contiguous():
        raise KernelError("KV pool must be a contiguous [num_blocks, kv_heads, block_size, head_dim]")
    nb, h, bs, d = pool.shape
    return nb, h, bs, d


def reshape_and_cache(
    key: torch.Tensor,
    value: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    token_tags: torch.Tensor | None = None,
    tag_pool: torch.Tensor | None = None,
    error_flag: torch.Tensor | None = None,
) -> None:
    """K1: ``key/value [T, Hkv, D]`` -> pools at ``slot_mapping [T]`` (int64)."""
    nb, h, bs, d = _pool_dims(key_pool)
    if value_pool.shape != key_pool.shape or value_pool.dtype != key_pool.dtype:
        raise KernelError("key and value pools differ")
    if key.dtype != key_pool.dtype or value.dtype != key_pool.dtype:
        raise KernelError("K/V rows must have the pool's dtype")
    ks = _rows(key, h, d, "key")
    vs = _rows(value, h, d, "value")
    if slot_mapping.dtype != torch.int64 or slot_mapping.numel() != key.shape[0]:
        raise KernelError("slot_mapping must be int64 with one entry per token")
    code = load_library().ts_reshape_and_cache(
        _ptr(key), _ptr(value), ks, vs, _ptr(key_pool), _ptr(value_pool),
        _ptr(slot_mapping), key.shape[0], h, d, bs, nb, _dtype(key_pool),
        _ptr(token_tags), _ptr(tag_pool), _ptr(error_flag), _stream(),
    )  # fmt: skip
    _check(code, "reshape_and_cache")


def decode_workspace_size(
    batch: int, num_q_heads: int, num_kv_heads: int, head_dim: int, max_blocks: int,
    block_size: int, dtype: torch.dtype,
) -> int:  # fmt: skip
    return int(
        load_library().ts_paged_decode_workspace_size(
            batch, num_q_heads, num_kv_heads, head_dim, max_blocks, block_size, DTYPE_CODES[dtype]
        )
    )


def paged_decode(
    out: torch.Tensor,
    query: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float,
    workspace: torch.Tensor | None,
    reuse_plan: bool = False,
) -> None:
    """K2: ``query [B, Hq, D]`` over each sequence's context -> ``out [B, Hq, D]``.

    ``reuse_plan=True`` runs the work plan an earlier call left in ``workspace`` (same block
    tables, context lengths, batch, KV heads and table width: the later layers of one decode
    step) and skips the prep kernel (``ts_paged_decode_planned``).
    """
    nb, hkv, bs, d = _pool_dims(key_pool)
    hq = query.shape[1]
    qs = _rows(query, hq, d, "query")
    if not out.is_contiguous() or out.shape != (query.shape[0], hq, d):
        raise KernelError("out must be a contiguous [B, Hq, D]")
    if block_tables.dtype != torch.int32 or not block_tables.is_contiguous():
        raise KernelError("block_tables must be contiguous int32 [B, max_blocks]")
    if context_lens.dtype != torch.int32:
        raise KernelError("context_lens must be int32")
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    lib = load_library()
    fn = lib.ts_paged_decode_planned if reuse_plan else lib.ts_paged_decode
    code = fn(
        _ptr(out), _ptr(query), qs, _ptr(key_pool), _ptr(value_pool), _ptr(block_tables),
        block_tables.shape[1], _ptr(context_lens), query.shape[0], hq, hkv, d, bs, nb,
        float(scale), _dtype(key_pool), _ptr(workspace), ws_bytes, _stream(),
    )  # fmt: skip
    _check(code, "paged_decode")


def paged_prefill(
    out: torch.Tensor,
    query: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    block_tables: torch.Tensor,
    query_start_loc: torch.Tensor,
    context_lens: torch.Tensor,
    max_query_len: int,
    scale: float,
) -> None:
    """K3: causal chunk attention, ``query [T, Hq, D]`` -> ``out [T, Hq, D]``."""
    nb, hkv, bs, d = _pool_dims(key_pool)
    hq = query.shape[1]
    qs = _rows(query, hq, d, "query")
    if not out.is_contiguous() or out.shape != (query.shape[0], hq, d):
        raise KernelError("out must be a contiguous [T, Hq, D]")
    if block_tables.dtype != torch.int32 or not block_tables.is_contiguous():
        raise KernelError("block_tables must be contiguous int32")
    if query_start_loc.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise KernelError("query_start_loc and context_lens must be int32")
    code = load_library().ts_paged_prefill(
        _ptr(out), _ptr(query), qs, _ptr(key_pool), _ptr(value_pool), _ptr(block_tables),
        block_tables.shape[1], _ptr(query_start_loc), _ptr(context_lens),
        context_lens.shape[0], query.shape[0], int(max_query_len), hq, hkv, d, bs, nb,
        float(scale), _dtype(key_pool), _stream(),
    )  # fmt: skip
    _check(code, "paged_prefill")


def copy_blocks(
    planes: torch.Tensor, src_dst: torch.Tensor, error_flag: torch.Tensor | None = None
) -> None:
    """K4: ``planes [P, num_blocks, ...]`` (contiguous); copy each (src, dst) block in every plane."""
    if not planes.is_contiguous() or planes.dim() < 2:
        raise KernelError("planes must be a contiguous [P, num_blocks, ...] tensor")
    if src_dst.dtype != torch.int64 or not src_dst.is_contiguous():
        raise KernelError("src_dst must be contiguous int64 [n, 2]")
    if not planes.is_cuda or src_dst.device != planes.device:
        raise KernelError("planes and src_dst must be on the same CUDA device")
    es = planes.element_size()
    block_bytes = planes[0, 0].numel() * es
    code = load_library().ts_copy_blocks(
        _ptr(planes), planes.shape[0], planes.stride(0) * es, block_bytes, planes.shape[1],
        _ptr(src_dst), src_dst.numel() // 2, _ptr(error_flag), _stream(),
    )  # fmt: skip
    _check(code, "copy_blocks")


def swap_blocks(dst: torch.Tensor, src: torch.Tensor, src_dst: torch.Tensor,
                error_flag: torch.Tensor | None = None) -> None:  # fmt: skip
    """K4 between two arenas ``[P, blocks, ...]`` of one plane layout: ``dst[p, d] = src[p, s]``
    for each pair ``(s, d)``. One side may be pinned host memory (swap-out / swap-in)."""
    for t in (dst, src):
        if not t.is_contiguous() or t.dim() < 2:
            raise KernelError("swap_blocks: arenas must be contiguous [P, blocks, ...] tensors")
        if not t.is_cuda and not t.is_pinned():
            raise KernelError("swap_blocks: a host arena must be pinned memory")
    if dst.shape[0] != src.shape[0] or dst[0, 0].numel() * dst.element_size() != (
            src[0, 0].numel() * src.element_size()):  # fmt: skip
        raise KernelError("swap_blocks: arenas differ in planes or block size")
    if src_dst.dtype != torch.int64 or not src_dst.is_contiguous() or not src_dst.is_cuda:
        raise KernelError("swap_blocks: src_dst must be contiguous int64 [n, 2] on the device")
    bb = dst[0, 0].numel() * dst.element_size()
    code = load_library().ts_swap_blocks(
        _ptr(dst), dst.stride(0) * dst.element_size(), dst.shape[1],
        _ptr(src), src.stride(0) * src.element_size(), src.shape[1],
        dst.shape[0], bb, _ptr(src_dst), src_dst.numel() // 2, _ptr(error_flag), _stream(),
    )  # fmt: skip
    _check(code, "swap_blocks")


def verify_tags(
    tag_pool: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    expected_offsets: torch.Tensor,
    expected_tokens: torch.Tensor,
    block_size: int,
    mismatch_pos: torch.Tensor,
) -> None:
    """Device shadow-KV read-back check; ``mismatch_pos[b]`` = first bad position or -1."""
    num_blocks = tag_pool.numel() // block_size
    code = load_library().ts_verify_tags(
        _ptr(tag_pool), _ptr(block_tables), block_tables.shape[1], _ptr(context_lens),
        _ptr(expected_offsets), _ptr(expected_tokens), context_lens.shape[0], block_size,
        num_blocks, _ptr(mismatch_pos), _stream(),
    )  # fmt: skip
    _check(code, "verify_tags")


def add_rmsnorm(out: torch.Tensor, residual: torch.Tensor, x: torch.Tensor | None,
                weight: torch.Tensor, eps: float) -> None:  # fmt: skip
    """``residual += x`` (skipped when ``x`` is None), then ``out = RMSNorm(residual) * weight``."""
    rows, hidden = residual.shape
    for t in (out, residual, weight) + (() if x is None else (x,)):
        if not t.is_contiguous() or t.dtype != residual.dtype:
            raise KernelError("add_rmsnorm: tensors must be contiguous and of one dtype")
    code = load_library().ts_add_rmsnorm(_ptr(out), _ptr(residual), _ptr(x), _ptr(weight), rows,
                                         hidden, float(eps), _dtype(residual), _stream())  # fmt: skip
    _check(code, "add_rmsnorm")


def rope_and_cache(qkv: torch.Tensor, q_out: torch.Tensor, key_pool: torch.Tensor,
                   value_pool: torch.Tensor, slot_mapping: torch.Tensor, positions: torch.Tensor,
                   inv_freq: torch.Tensor, num_q_heads: int, num_kv_heads: int,
                   error_flag: torch.Tensor | None = None) -> None:  # fmt: skip
    """RoPE on q and k of fused ``qkv [T, (Hq + 2 Hkv) * D]``; q -> ``q_out``, k/v -> the pool."""
    nb, hkv, bs, d = _pool_dims(key_pool)
    if hkv != num_kv_heads or qkv.stride(1) != 1 or not q_out.is_contiguous():
        raise KernelError("rope_and_cache: bad layout")
    if slot_mapping.dtype != torch.int64 or positions.dtype != torch.int64:
        raise KernelError("rope_and_cache: slot_mapping and positions must be int64")
    code = load_library().ts_rope_and_cache(
        _ptr(qkv), qkv.stride(0), _ptr(q_out), _ptr(key_pool), _ptr(value_pool),
        _ptr(slot_mapping), _ptr(positions), _ptr(inv_freq), qkv.shape[0], num_q_heads,
        num_kv_heads, d, bs, nb, _dtype(key_pool), _ptr(error_flag), _stream(),
    )  # fmt: skip
    _check(code, "rope_and_cache")


def silu_mul(out: torch.Tensor, gate_up: torch.Tensor) -> None:
    """``out = silu(gate) * up`` for ``gate_up = [gate | up]`` of shape ``[T, 2 I]``."""
    rows, two_i = gate_up.shape
    if not gate_up.is_contiguous() or not out.is_contiguous() or out.shape != (rows, two_i // 2):
        raise KernelError("silu_mul: bad layout")
    code = load_library().ts_silu_mul(_ptr(out), _ptr(gate_up), rows, two_i // 2,
                                      _dtype(gate_up), _stream())  # fmt: skip
    _check(code, "silu_mul")


# ------------------------------------------------------------------------------ 8-bit KV cache
#
# Pools [num_blocks, kv_heads, block_size, head_dim] of torch.float8_e4m3fn with float32 scales
# [num_blocks, kv_heads, block_size]; a row stands for code * scale (include/tokenserve_b200.h).
# The operators below run on their tensors' device, on its current stream.


def _cuda(what: str, *tensors: torch.Tensor | None) -> int:
    """Index of the one CUDA device all the (present) tensors live on."""
    dev = tensors[0].get_device()  # type: ignore[union-attr]
    for t in tensors:
        if t is not None and t.get_device() != dev:
            dev = -1
    if dev < 0:
        raise KernelError(f"{what}: tensors must be on one CUDA device")
    return dev


# The raw handle of a device's current stream. torch.cuda.current_stream() builds a Stream object
# for it, 3 us of a small call's 10.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)  # fmt: skip


def _launch(what: str, device: int, name: str, *args) -> None:  # type: ignore[no-untyped-def]
    """Calls the entry point ``name`` with ``device`` current, on its current stream."""
    fn = getattr(_lib or load_library(), name)
    if torch.cuda.current_device() == device:
        code = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            code = fn(*args, _raw_stream(device))
    if code:
        _check(code, what)


_E4M3, _F32, _I32, _I64 = torch.float8_e4m3fn, torch.float32, torch.int32, torch.int64


def _fp8_pool_dims(what: str, key_pool: torch.Tensor, value_pool: torch.Tensor,
                   key_scales: torch.Tensor, value_scales: torch.Tensor) -> torch.Size:  # fmt: skip
    shape = key_pool.shape
    if (len(shape) != 4 or value_pool.shape != shape or key_pool.dtype != _E4M3
            or value_pool.dtype != _E4M3 or not key_pool.is_contiguous()
            or not value_pool.is_contiguous()):  # fmt: skip
        raise KernelError(f"{what}: 8-bit pools must be contiguous float8_e4m3fn "
                          "[num_blocks, kv_heads, block_size, head_dim]")  # fmt: skip
    rows = key_scales.shape
    if (rows != shape[:3] or value_scales.shape != rows
            or key_scales.dtype != _F32 or value_scales.dtype != _F32
            or not key_scales.is_contiguous() or not value_scales.is_contiguous()):  # fmt: skip
        raise KernelError(f"{what}: scales must be contiguous float32 "
                          "[num_blocks, kv_heads, block_size]")  # fmt: skip
    return shape


def _int_array(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, n: int) -> None:
    if t.dtype != dtype or t.numel() != n or not t.is_contiguous():
        raise KernelError(f"{what}: {name} must be a contiguous {dtype} of {n} entries, got "
                          f"{t.dtype} {tuple(t.shape)}")  # fmt: skip


def _error_flag(what: str, t: torch.Tensor | None) -> None:
    if t is not None and (t.dtype != _I32 or t.numel() < 1):
        raise KernelError(f"{what}: error_flag must be an int32 tensor")


def _tables(what: str, t: torch.Tensor, rows: int) -> int:
    shape = t.shape
    if t.dtype != _I32 or len(shape) != 2 or shape[0] != rows or not t.is_contiguous():
        raise KernelError(f"{what}: block_tables must be contiguous int32 [{rows}, max_blocks]")
    return shape[1]


def _attention_rows(what: str, out: torch.Tensor, query: torch.Tensor, kv_heads: int,
                    head_dim: int) -> tuple[int, int]:  # fmt: skip
    """Query heads and token stride of ``query [T, Hq, D]``, checked against ``out``."""
    shape = query.shape
    if len(shape) != 3 or shape[1] == 0 or shape[1] % max(kv_heads, 1):
        raise KernelError(f"{what}: query must be [tokens, heads, {head_dim}] with a multiple of "
                          f"{kv_heads} heads, got {tuple(shape)}")  # fmt: skip
    stride = _rows(query, shape[1], head_dim, f"{what}: query")
    if out.shape != shape or out.dtype != query.dtype or not out.is_contiguous():
        raise KernelError(f"{what}: out must be contiguous, of the query's shape and dtype")
    # A single row's stride says nothing.
    return shape[1], stride if shape[0] > 1 else shape[1] * head_dim


def reshape_and_cache_fp8(
    key: torch.Tensor,
    value: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    slot_mapping: torch.Tensor,
    *,
    token_tags: torch.Tensor | None = None,
    tag_pool: torch.Tensor | None = None,
    error_flag: torch.Tensor | None = None,
) -> None:
    """K1 into an 8-bit cache: ``key/value [T, Hkv, D]`` are quantised row by row as they are
    written at ``slot_mapping [T]`` (int64, distinct; negative: skipped)."""
    what = "reshape_and_cache_fp8"
    nb, h, bs, d = _fp8_pool_dims(what, key_pool, value_pool, key_scales, value_scales)
    dev = _cuda(what, key, value, key_pool, value_pool, key_scales, value_scales, slot_mapping,
                token_tags, tag_pool, error_flag)  # fmt: skip
    if key.dtype != value.dtype or key.shape != value.shape:
        raise KernelError(f"{what}: key and value must have one shape and dtype")
    ks, vs = _rows(key, h, d, f"{what}: key"), _rows(value, h, d, f"{what}: value")
    n = key.shape[0]
    if n == 1:  # a single row's stride says nothing
        ks = vs = h * d
    _int_array(what, "slot_mapping", slot_mapping, _I64, n)
    if token_tags is not None:
        _int_array(what, "token_tags", token_tags, _I32, n)
    if tag_pool is not None:
        _int_array(what, "tag_pool", tag_pool, _I32, nb * bs)
    _error_flag(what, error_flag)
    _launch(what, dev, "ts_reshape_and_cache_fp8",
            key.data_ptr(), value.data_ptr(), ks, vs, key_pool.data_ptr(), value_pool.data_ptr(),
            key_scales.data_ptr(), value_scales.data_ptr(), slot_mapping.data_ptr(), n, h, d, bs,
            nb, _dtype(key), _ptr(token_tags), _ptr(tag_pool), _ptr(error_flag))  # fmt: skip


def rotary_and_cache(
    qkv: torch.Tensor,
    q_out: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    slot_mapping: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    num_q_heads: int,
    num_kv_heads: int,
    *,
    key_scales: torch.Tensor | None = None,
    value_scales: torch.Tensor | None = None,
    interleaved: bool = False,
    attention_scaling: float = 1.0,
    error_flag: torch.Tensor | None = None,
) -> None:
    """Rotary positions on q and k of fused ``qkv [T, (Hq + 2 Hkv) * D]``; q -> ``q_out [T, Hq,
    D]``, k and v -> the pools, quantised where ``key_scales`` and ``value_scales`` are given.

    The first ``2 * len(inv_freq)`` dims of each head turn by ``positions * inv_freq`` (any
    frequencies), in pairs ``(i, i + len)`` or, ``interleaved``, ``(2i, 2i + 1)``;
    ``attention_scaling`` multiplies cos and sin. Computed in fp32, rounded once.
    """
    what = "rotary_and_cache"
    if (key_scales is None) != (value_scales is None):
        raise KernelError(f"{what}: key_scales and value_scales go together")
    if key_scales is not None:
        nb, hkv, bs, d = _fp8_pool_dims(what, key_pool, value_pool, key_scales, value_scales)
    else:
        nb, hkv, bs, d = _pool_dims(key_pool)
        if (value_pool.shape != key_pool.shape or not value_pool.is_contiguous()
                or key_pool.dtype != qkv.dtype or value_pool.dtype != qkv.dtype):  # fmt: skip
            raise KernelError(f"{what}: pools must be contiguous, of one shape and of qkv's dtype")
    dev = _cuda(what, qkv, q_out, key_pool, value_pool, key_scales, value_scales, slot_mapping,
                positions, inv_freq, error_flag)  # fmt: skip
    n, width = qkv.shape if qkv.dim() == 2 else (-1, -1)
    stride = qkv.stride()
    if hkv != num_kv_heads or num_q_heads <= 0 or width != (num_q_heads + 2 * hkv) * d or (
            stride[1] != 1):  # fmt: skip
        raise KernelError(f"{what}: qkv must be [tokens, (q heads + 2 kv heads) * head_dim] with "
                          "contiguous rows and the pool's kv heads")  # fmt: skip
    if q_out.shape != (n, num_q_heads, d) or q_out.dtype != qkv.dtype or not q_out.is_contiguous():
        raise KernelError(f"{what}: q_out must be a contiguous [tokens, q heads, head_dim] of "
                          "qkv's dtype")  # fmt: skip
    _int_array(what, "slot_mapping", slot_mapping, _I64, n)
    _int_array(what, "positions", positions, _I64, n)
    half = inv_freq.numel()
    _int_array(what, "inv_freq", inv_freq, _F32, half)
    _error_flag(what, error_flag)
    _launch(what, dev, "ts_rotary_and_cache",
            qkv.data_ptr(), stride[0] if n > 1 else width, q_out.data_ptr(),
            key_pool.data_ptr(), value_pool.data_ptr(), _ptr(key_scales), _ptr(value_scales),
            slot_mapping.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), n, num_q_heads, hkv,
            d, 2 * half, int(interleaved), float(attention_scaling), bs, nb, _dtype(qkv),
            _ptr(error_flag))  # fmt: skip


def read_cache_fp8(
    key_out: torch.Tensor,
    value_out: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    block_tables: torch.Tensor,
    token_start_loc: torch.Tensor,
    error_flag: torch.Tensor | None = None,
) -> None:
    """Reads an 8-bit cache back: position p of sequence s -> row ``token_start_loc[s] + p`` of
    ``key_out`` and ``value_out [T, Hkv, D]`` (float32, float16 or bfloat16)."""
    what = "read_cache_fp8"
    nb, h, bs, d = _fp8_pool_dims(what, key_pool, value_pool, key_scales, value_scales)
    dev = _cuda(what, key_out, value_out, key_pool, value_pool, key_scales, value_scales,
                block_tables, token_start_loc, error_flag)  # fmt: skip
    n = key_out.shape[0] if key_out.dim() == 3 else -1
    for t in (key_out, value_out):
        if t.shape != (n, h, d) or t.dtype != key_out.dtype or not t.is_contiguous():
            raise KernelError(f"{what}: outputs must be contiguous [tokens, {h}, {d}] of one dtype")
    seqs = block_tables.shape[0] if block_tables.dim() else -1
    width = _tables(what, block_tables, seqs)
    _int_array(what, "token_start_loc", token_start_loc, _I32, seqs + 1)
    _error_flag(what, error_flag)
    _launch(what, dev, "ts_read_cache_fp8",
            key_out.data_ptr(), value_out.data_ptr(), key_pool.data_ptr(), value_pool.data_ptr(),
            key_scales.data_ptr(), value_scales.data_ptr(), block_tables.data_ptr(), width,
            token_start_loc.data_ptr(), seqs, n, h, d, bs, nb, _dtype(key_out),
            _ptr(error_flag))  # fmt: skip


def paged_decode_fp8(
    out: torch.Tensor,
    query: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    block_tables: torch.Tensor,
    context_lens: torch.Tensor,
    scale: float,
    workspace: torch.Tensor | None,
    reuse_plan: bool = False,
) -> None:
    """K2 over an 8-bit cache: ``query [B, Hq, D]`` -> ``out``; see :func:`paged_decode`. The
    workspace is sized by :func:`decode_workspace_size` with the query's dtype."""
    what = "paged_decode_fp8"
    nb, hkv, bs, d = _fp8_pool_dims(what, key_pool, value_pool, key_scales, value_scales)
    dev = _cuda(what, out, query, key_pool, value_pool, key_scales, value_scales, block_tables,
                context_lens, workspace)  # fmt: skip
    hq, qs = _attention_rows(what, out, query, hkv, d)
    b = query.shape[0]
    width = _tables(what, block_tables, b)
    _int_array(what, "context_lens", context_lens, _I32, b)
    if workspace is not None and not workspace.is_contiguous():
        raise KernelError(f"{what}: workspace must be contiguous")
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _launch(what, dev, "ts_paged_decode_fp8",
            out.data_ptr(), query.data_ptr(), qs, key_pool.data_ptr(), value_pool.data_ptr(),
            key_scales.data_ptr(), value_scales.data_ptr(), block_tables.data_ptr(), width,
            context_lens.data_ptr(), b, hq, hkv, d, bs, nb, float(scale), _dtype(query),
            _ptr(workspace), ws_bytes, int(reuse_plan))  # fmt: skip


def paged_prefill_fp8(
    out: torch.Tensor,
    query: torch.Tensor,
    key_pool: torch.Tensor,
    value_pool: torch.Tensor,
    key_scales: torch.Tensor,
    value_scales: torch.Tensor,
    block_tables: torch.Tensor,
    query_start_loc: torch.Tensor,
    context_lens: torch.Tensor,
    max_query_len: int,
    scale: float,
) -> None:
    """K3 over an 8-bit cache: causal chunk attention, ``query [T, Hq, D]`` -> ``out``."""
    what = "paged_prefill_fp8"
    nb, hkv, bs, d = _fp8_pool_dims(what, key_pool, value_pool, key_scales, value_scales)
    dev = _cuda(what, out, query, key_pool, value_pool, key_scales, value_scales, block_tables,
                query_start_loc, context_lens)  # fmt: skip
    hq, qs = _attention_rows(what, out, query, hkv, d)
    seqs = context_lens.numel()
    width = _tables(what, block_tables, seqs)
    _int_array(what, "context_lens", context_lens, _I32, seqs)
    _int_array(what, "query_start_loc", query_start_loc, _I32, seqs + 1)
    _launch(what, dev, "ts_paged_prefill_fp8",
            out.data_ptr(), query.data_ptr(), qs, key_pool.data_ptr(), value_pool.data_ptr(),
            key_scales.data_ptr(), value_scales.data_ptr(), block_tables.data_ptr(), width,
            query_start_loc.data_ptr(), context_lens.data_ptr(), seqs, query.shape[0],
            int(max_query_len), hq, hkv, d, bs, nb, float(scale), _dtype(query))  # fmt: skip

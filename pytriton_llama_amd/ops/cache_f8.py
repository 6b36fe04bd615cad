"""Python faces of the kernels around a cache that is held in 8 bits (csrc/cache_f8.hip, csrc/attention_f8.hip), in the manner of
ops.kernels: operands are checked on the host, launches go to torch's current stream, what a kernel does not take raises.

The cache: codes float8_e4m3fn [pages, Hkv, page_size, D] and scales float32 [pages, Hkv], of the keys and of the values. What the
block of a (page, kv head) holds stands for code * scale; a scale is a power of two (2^-126 and more).
"""
from __future__ import annotations

import ctypes
import itertools
from typing import Optional, Sequence

import torch

from . import library
from .kernels import TICKET, KernelError, _check, _dtype_code, _i32, _need_gpu, _ptr, _stream, _tickets

CACHE_F8 = torch.float8_e4m3fn          # the codes' type


def _cache(what: str, Hkv: int, D: int, k_cache, v_cache, k_scale, v_scale):
    """(pages, page size) of an 8-bit cache; raises where its tensors do not belong together."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[1] != Hkv or k_cache.shape[3] != D:
        raise KernelError(f"{what}: caches must be [pages, {Hkv}, page_size, {D}]")
    if k_cache.dtype != CACHE_F8 or v_cache.dtype != CACHE_F8:
        raise KernelError(f"{what}: caches must be float8_e4m3fn, got {k_cache.dtype} and {v_cache.dtype}")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous() or (k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise KernelError(f"{what}: caches must be contiguous and 16-byte aligned")
    scales = (k_cache.shape[0], Hkv)
    for t in (k_scale, v_scale):
        if t.dtype != torch.float32 or t.shape != scales or not t.is_contiguous():
            raise KernelError(f"{what}: scales must be contiguous float32 [{scales[0]}, {scales[1]}]")
    return k_cache.shape[0], k_cache.shape[2]


def _one_device(what: str, *tensors) -> None:
    """All on the current device, where the launch goes."""
    at = -1
    for t in tensors:
        if t is None:
            continue
        d = t.get_device()
        if d != at or d < 0:
            _need_gpu(t)
            at = torch._C._cuda_getDevice()
            if d != at:
                raise KernelError(f"{what}: tensors must be on the current device cuda:{at}, got one on {t.device}")


def rope_store_f8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: Optional[torch.Tensor],
                  slots: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor) -> torch.Tensor:
    """``rope_store`` for an 8-bit cache: the queries, rotated by positions * inv_freq, as a new tensor [T, Hq, D]; the rotated keys
    and the values into the blocks at ``slots`` (int32, page * page_size + offset; a token with a negative slot, or one behind
    the cache, is not stored). q, k, v: [T, heads, D] views that share one row stride, float32 or bfloat16, D even, up to 640.
    inv_freq None: no rotation. slots None: no store.

    The tokens that a call brings for one page have to be rows one after the other with slots one after the other. Where the first
    of them has the page's first slot the page begins anew: what it held is dropped, and rows behind the call's are zeros.
    Otherwise its scale grows where the new tokens need it, and the page's other numbers are rounded anew. Storing the same once
    more changes nothing. Numbers that are not finite are held as NaN."""
    _one_device("rope_store_f8", q, k, v, positions, inv_freq, slots, k_cache, v_cache, k_scale, v_scale)
    if q.dim() != 3 or k.dim() != 3:
        raise KernelError("rope_store_f8: q, k and v must be [T, heads, D]")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (T, Hkv, D) or v.shape != (T, Hkv, D):
        raise KernelError("rope_store_f8: k and v must be [T, Hkv, D]")
    rs = q.stride(0)
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype != q.dtype or t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != D) or (T > 1 and t.stride(0) != rs):
            raise KernelError(f"rope_store_f8: {name} must be a [T, heads, D] view with dense heads and the common row stride")
    if D % 2 or not 0 < D <= 640:
        raise KernelError(f"rope_store_f8: head size {D} must be even, up to 640")
    _i32(positions, "positions")
    if positions.numel() != T:
        raise KernelError("rope_store_f8: one position per token")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() != D // 2 or not inv_freq.is_contiguous()):
        raise KernelError(f"rope_store_f8: inv_freq must be float32 [{D // 2}]")
    if slots is not None:
        _i32(slots, "slots")
        if slots.numel() != T:
            raise KernelError("rope_store_f8: one slot per token")
    pages, page_size = _cache("rope_store_f8", Hkv, D, k_cache, v_cache, k_scale, v_scale)
    out = torch.empty((T, Hq, D), dtype=q.dtype, device=q.device)
    _check(library.load("cache_f8").ptl_rope_store_f8(
        _ptr(out), _ptr(q), _ptr(k), _ptr(v), ctypes.c_long(rs), _ptr(positions), _ptr(inv_freq), _ptr(slots), _ptr(k_cache),
        _ptr(v_cache), _ptr(k_scale), _ptr(v_scale), T, Hq, Hkv, D, page_size, pages, _dtype_code(q), _stream()), "rope_store_f8")
    return out


def _attention(what: str, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, block_table, window, sink, *more):
    _one_device(what, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, block_table, sink, *more)
    if q.dim() != 3 or out.shape != q.shape or out.dtype != q.dtype:
        raise KernelError(f"{what}: q and out must be [T, Hq, D] of one dtype")
    T, Hq, D = q.shape
    if k_cache.dim() != 4:
        raise KernelError(f"{what}: caches must be [pages, Hkv, page_size, {D}]")
    Hkv = k_cache.shape[1]
    _, page_size = _cache(what, Hkv, D, k_cache, v_cache, k_scale, v_scale)
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise KernelError(f"{what}: {Hq} query heads are not a multiple of {Hkv} kv heads")
    if q.stride(2) != 1 or out.stride(2) != 1 or (Hq > 1 and (q.stride(1) != D or out.stride(1) != D)):
        raise KernelError(f"{what}: q and out need dense heads")
    _i32(q_start, "q_start")
    _i32(ctx_len, "ctx_len")
    if q_start.numel() != ctx_len.numel() + 1:
        raise KernelError(f"{what}: inconsistent sequence tables")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] < ctx_len.numel() \
            or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise KernelError(f"{what}: block_table must be int32 [n, max_pages]")
    if window < 0:
        raise KernelError(f"{what}: a window is not negative")
    if sink is not None and (sink.dtype != torch.float32 or sink.shape != (Hq,) or not sink.is_contiguous()):
        raise KernelError(f"{what}: sink must be a contiguous float32 tensor [{Hq}]")
    return T, Hq, Hkv, D, page_size


def _work(what: str, work_seq: torch.Tensor, work_qoff: torch.Tensor) -> int:
    _i32(work_seq, "work_seq")
    _i32(work_qoff, "work_qoff")
    if work_seq.numel() != work_qoff.numel():
        raise KernelError(f"{what}: inconsistent work list")
    return work_seq.numel()


def attention_generic_f8(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor, block_table: torch.Tensor,
                         work_seq: torch.Tensor, work_qoff: torch.Tensor, scale: float, window: int = 0,
                         sink: Optional[torch.Tensor] = None) -> None:
    """``attention_generic`` over an 8-bit cache: float32 or bfloat16 queries, head sizes up to 640, any page size; the work list names
    16-row query blocks. window, sink: as there."""
    T, Hq, Hkv, D, page_size = _attention("attention_generic_f8", out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len,
                                          block_table, window, sink, work_seq, work_qoff)
    if not 0 < D <= 640 or Hq > 65535:
        raise KernelError(f"attention_generic_f8: head size {D} exceeds the kernel's limit of 640 (or {Hq} heads that of 65,535)")
    n = _work("attention_generic_f8", work_seq, work_qoff)
    _check(library.load("attention_f8").ptl_attention_generic_f8(
        _ptr(out), ctypes.c_long(out.stride(0)), _ptr(q), ctypes.c_long(q.stride(0)), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale),
        _ptr(v_scale), _ptr(q_start), _ptr(ctx_len), _ptr(block_table), int(block_table.stride(0)), _ptr(work_seq), _ptr(work_qoff),
        n, Hq, Hkv, D, page_size, int(window), _ptr(sink), ctypes.c_float(scale), _dtype_code(q), _stream()), "attention_generic_f8")


def attention_f8_fits(dtype: torch.dtype, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int) -> bool:
    """Whether ``attention_decode_f8`` and ``attention_prefill_f8`` take this case: bfloat16, head size 32, 64, 96 or 128, a
    page size from 16 on that is a power of two, pages (of all kv heads) below 2 GiB."""
    return (dtype == torch.bfloat16 and head_dim % 32 == 0 and 0 < head_dim <= 128 and page_size >= 16
            and page_size & (page_size - 1) == 0 and num_kv_heads > 0 and num_heads % num_kv_heads == 0
            and 0 < num_heads // num_kv_heads <= 1024 and num_kv_heads * page_size * head_dim < 2 ** 31)


def attention_decode_f8(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor, block_table: torch.Tensor, n_seq: int,
                        scale: float, window: int = 0, sink: Optional[torch.Tensor] = None,
                        tickets: Optional[torch.Tensor] = None) -> None:
    """Attention of the first ``n_seq`` sequences of the tables, each of which brings exactly one query token, over an 8-bit cache
    (``attention_f8_fits`` says for which sizes). How the keys are cut is decided on the device from ctx_len. ``tickets``: as for
    ``attention_decode``, TICKET * n_seq * kv heads for every 16 heads of a kv head."""
    T, Hq, Hkv, D, page_size = _attention("attention_decode_f8", out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len,
                                          block_table, window, sink, tickets)
    if not attention_f8_fits(q.dtype, Hq, Hkv, D, page_size) or q.stride(0) % 8 or q.data_ptr() % 16:
        raise KernelError("attention_decode_f8: needs bfloat16, a head size of 32/64/96/128, a page size from 16 on that is a power "
                          "of two, aligned q rows")
    if not 0 <= n_seq <= ctx_len.numel():
        raise KernelError("attention_decode_f8: tables are shorter than n_seq")
    if n_seq == 0:
        return
    lib = library.load("attention_f8")
    cuts = lib.ptl_attention_decode_f8_cuts(n_seq, Hkv, Hq)
    heads = (n_seq + cuts) * Hq
    parts = torch.empty(heads * (D + 2), dtype=torch.float32, device=q.device)
    tickets = _tickets(tickets, TICKET * n_seq * Hkv * -(-(Hq // Hkv) // 16), q, "attention_decode_f8")
    at = parts.data_ptr()
    _check(lib.ptl_attention_decode_f8(
        _ptr(out), ctypes.c_long(out.stride(0)), _ptr(q), ctypes.c_long(q.stride(0)), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale),
        _ptr(v_scale), _ptr(q_start), _ptr(ctx_len), _ptr(block_table), int(block_table.stride(0)), ctypes.c_void_p(at),
        ctypes.c_void_p(at + 4 * heads * D), _ptr(tickets), cuts, int(n_seq), Hq, Hkv, D, page_size, int(window), _ptr(sink),
        ctypes.c_float(scale), _stream()), "attention_decode_f8")


def attention_prefill_f8(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor, block_table: torch.Tensor,
                         work_seq: torch.Tensor, work_qoff: torch.Tensor, scale: float, window: int = 0, block_rows: int = 64,
                         groups: int = 0, sink: Optional[torch.Tensor] = None) -> None:
    """``attention_prefill_mfma`` over an 8-bit cache (``attention_f8_fits`` says for which sizes): the work list names query blocks
    of ``block_rows`` (64 or 128) rows, those with the most keys first; ``groups`` workgroups a head share it (0: one for
    every block)."""
    T, Hq, Hkv, D, page_size = _attention("attention_prefill_f8", out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len,
                                          block_table, window, sink, work_seq, work_qoff)
    if not attention_f8_fits(q.dtype, Hq, Hkv, D, page_size):
        raise KernelError("attention_prefill_f8: needs bfloat16, a head size of 32/64/96/128, a page size from 16 on that is a power "
                          "of two")
    if q.stride(0) % 8 or out.stride(0) % 4 or q.data_ptr() % 16 or out.data_ptr() % 8:
        raise KernelError("attention_prefill_f8: q rows must be 16-byte aligned, out rows 8-byte")
    if block_rows not in (64, 128):
        raise KernelError("attention_prefill_f8: query blocks are 64 or 128 rows")
    if not scale > 0:
        raise KernelError("attention_prefill_f8: scale must be positive")
    n = _work("attention_prefill_f8", work_seq, work_qoff)
    _check(library.load("attention_f8").ptl_attention_prefill_f8(
        _ptr(out), ctypes.c_long(out.stride(0)), _ptr(q), ctypes.c_long(q.stride(0)), _ptr(k_cache), _ptr(v_cache), _ptr(k_scale),
        _ptr(v_scale), _ptr(q_start), _ptr(ctx_len), _ptr(block_table), int(block_table.stride(0)), _ptr(work_seq), _ptr(work_qoff),
        n, min(n, int(groups), 65535) if groups > 0 else min(n, 65535), int(block_rows), Hq, Hkv, D, page_size, int(window),
        _ptr(sink), ctypes.c_float(scale), _stream()), "attention_prefill_f8")


def copy_pages(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Page src[i] -> page dst[i] in all layers of every pool [layers, pages, ...] (contiguous, up to 16 of them, any dtype), one
    launch. src, dst: page numbers on the host; no page may be written twice, or both read and written (one may be read many
    times). The numbers go with the launch: nothing is uploaded, and a recorded launch keeps its own."""
    src, dst = list(src), list(dst)
    n = len(src)
    if n != len(dst):
        raise KernelError(f"copy_pages: {n} pages to read, {len(dst)} to write")
    _one_device("copy_pages", *pools)
    desc = []
    for t in pools:
        if t.dim() < 2 or not t.is_contiguous():
            raise KernelError("copy_pages: a pool is a contiguous tensor [layers, pages, ...]")
        layers, pages = t.shape[:2]
        if n and not (0 <= min(src) and max(src) < pages and 0 <= min(dst) and max(dst) < pages):
            raise KernelError(f"copy_pages: a page number lies outside the pool's {pages} pages")
        if t.numel():
            desc += [t.data_ptr(), layers, pages, t.numel() // (layers * pages) * t.element_size()]
    written = set(dst)
    if len(written) != n or not written.isdisjoint(src):
        raise KernelError("copy_pages: a page is written twice, or read and written")
    if n == 0 or not desc:
        return
    if len(desc) > 4 * 16:
        raise KernelError("copy_pages: up to 16 pools a call")
    numbers = (ctypes.c_int32 * (2 * n))(*itertools.chain(src, dst))
    at = ctypes.addressof(numbers)
    _check(library.load("cache_f8").ptl_copy_pages((ctypes.c_long * len(desc))(*desc), len(desc) // 4, ctypes.c_void_p(at),
                                                   ctypes.c_void_p(at + 4 * n), n, _stream()), "copy_pages")

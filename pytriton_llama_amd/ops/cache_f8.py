"""Python faces of the kernels around a cache that is held in 8 bits (csrc/cache_f8.hip, csrc/attention_f8.hip), in the manner of
ops.kernels: operands are checked on the host, launches go to torch's current stream, what a kernel does not take raises.

The cache: codes float8_e4m3fn [pages, Hkv, page_size, D] and scales float32 [pages, Hkv], of the keys and of the values. What the
block of a (page, kv head) holds stands for code * scale; a scale is a power of two (2^-126 and more).

A decode step is a row of short kernels, and what the host needs for a call shows in it: tensors are asked for each of their
properties once, and entries know their arguments' types, so that addresses go as plain numbers (a call of ``attention_decode_f8``
costs the host 12.3 us; 16.8 with addresses wrapped for each call and every tensor's properties asked for by each check).
"""
from __future__ import annotations

import array
import ctypes
from typing import Optional, Sequence

import torch

from . import library
from .kernels import TICKET, KernelError, RowScale, _check, _dtype_code, _i32, _need_gpu, _tickets, compute_units

CACHE_F8 = torch.float8_e4m3fn          # the codes' type

_TYPES = {"p": ctypes.c_void_p, "l": ctypes.c_long, "i": ctypes.c_int, "f": ctypes.c_float}
# entry -> library, types of its arguments (p: address, l: long, i: int, f: float)
_ENTRIES = {"ptl_rope_store_f8": ("cache_f8", "pppplppppppp" "iiiiii" "piif" "ip"), "ptl_copy_pages": ("cache_f8", "pippip"),
            "ptl_attention_generic_f8": ("attention_f8", "plplppppppp" "ipp" "iiiiiii" "pfip"),
            "ptl_attention_decode_f8": ("attention_f8", "plplppppppp" "ippp" "iiiiiii" "pfp"),
            "ptl_attention_prefill_f8": ("attention_f8", "plplppppppp" "ipp" "iiippiiiiii" "pfp")}
_loaded = {}


def _entry(name: str):
    f = _loaded.get(name)
    if f is None:
        lib, types = _ENTRIES[name]
        f = getattr(library.load(lib), name)
        f.argtypes = [_TYPES[t] for t in types]
        _loaded[name] = f
    return f


def _launch_stream(what: str, *tensors) -> int:
    """torch's current stream; raises unless all tensors are on the current device, where the launch goes."""
    at = -1
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if d != at or d < 0:
                _need_gpu(t)
                at = torch._C._cuda_getDevice()
                if d != at:
                    raise KernelError(f"{what}: tensors must be on the current device cuda:{at}, got one on {t.device}")
    return torch._C._cuda_getCurrentRawStream(at) if at >= 0 else 0


def _cache(what: str, Hkv: int, D: int, k_cache, v_cache, k_scale, v_scale):
    """(pages, page size, addresses) of an 8-bit cache; raises where its tensors do not belong together."""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape or shape[1] != Hkv or shape[3] != D:
        raise KernelError(f"{what}: caches must be [pages, {Hkv}, page_size, {D}]")
    if k_cache.dtype != CACHE_F8 or v_cache.dtype != CACHE_F8:
        raise KernelError(f"{what}: caches must be float8_e4m3fn, got {k_cache.dtype} and {v_cache.dtype}")
    k, v = k_cache.data_ptr(), v_cache.data_ptr()
    # (what the kernels read at once lies in one row: a layer of a pool may begin at any of its multiples of D bytes)
    need = 16 if D % 16 == 0 else 4 if D % 4 == 0 else 2 - D % 2
    if not k_cache.is_contiguous() or not v_cache.is_contiguous() or (k | v) % need:
        raise KernelError(f"{what}: caches must be contiguous and {need}-byte aligned")
    for t in (k_scale, v_scale):
        if t.dtype != torch.float32 or t.shape != shape[:2] or not t.is_contiguous():
            raise KernelError(f"{what}: scales must be contiguous float32 [{shape[0]}, {Hkv}]")
    return shape[0], shape[2], (k, v, k_scale.data_ptr(), v_scale.data_ptr())


SCALED_ROWS = 16           # rows that rope_store_f8 takes without their norm's factor (csrc/cache_f8.hip)


def rope_store_f8(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, inv_freq: Optional[torch.Tensor],
                  slots: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, row_scale: Optional[RowScale] = None) -> torch.Tensor:
    """``rope_store`` for an 8-bit cache: the queries, rotated by positions * inv_freq, as a new tensor [T, Hq, D]; the rotated keys
    and the values into the blocks at ``slots`` (int32, page * page_size + offset; a token with a negative slot, or one behind
    the cache, is not stored). q, k, v: [T, heads, D] views that share one row stride, float32 or bfloat16, D even, up to 640.
    inv_freq None: no rotation. slots None: no store.

    The tokens that a call brings for one page have to be rows one after the other with slots one after the other. Where the first
    of them has the page's first slot the page begins anew: what it held is dropped, and rows behind the call's are zeros.
    Otherwise its scale grows where the new tokens need it, and the page's other numbers are rounded anew. Storing the same once
    more changes nothing. Numbers that are not finite are held as NaN.

    ``row_scale``: a factor that the rows of q, k and v still lack (at most 16 rows): theirs is the product of rows that a norm has not
    finished."""
    stream = _launch_stream("rope_store_f8", q, k, v, positions, inv_freq, slots, k_cache, v_cache, k_scale, v_scale,
                            row_scale.partials if row_scale is not None else None)
    if q.dim() != 3 or k.dim() != 3:
        raise KernelError("rope_store_f8: q, k and v must be [T, heads, D]")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape != (T, Hkv, D) or v.shape != k.shape:
        raise KernelError("rope_store_f8: k and v must be [T, Hkv, D]")
    dtype, rs = q.dtype, q.stride(0)
    for name, t, heads in (("q", q, Hq), ("k", k, Hkv), ("v", v, Hkv)):
        rows, head, one = t.stride()
        if t.dtype != dtype or one != 1 or (heads > 1 and head != D) or (T > 1 and rows != rs):
            raise KernelError(f"rope_store_f8: {name} must be a [T, heads, D] view with dense heads and the common row stride")
    if D % 2 or not 0 < D <= 640 or Hq < 1 or Hkv < 1:
        raise KernelError(f"rope_store_f8: head size {D} must be even, up to 640, and there is a head at least")
    _i32(positions, "positions")
    if positions.numel() != T:
        raise KernelError("rope_store_f8: one position per token")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() != D // 2 or not inv_freq.is_contiguous()):
        raise KernelError(f"rope_store_f8: inv_freq must be float32 [{D // 2}]")
    if slots is not None:
        _i32(slots, "slots")
        if slots.numel() != T:
            raise KernelError("rope_store_f8: one slot per token")
    pages, page_size, cache = _cache("rope_store_f8", Hkv, D, k_cache, v_cache, k_scale, v_scale)
    partials, count, size, eps = None, 0, 0, 0.0
    if row_scale is not None:
        if T > SCALED_ROWS:
            raise KernelError(f"rope_store_f8: rows that lack a factor are at most {SCALED_ROWS}, got {T}")
        row_scale.args(T, row_scale.size, "rope_store_f8")          # (checks)
        partials, count, size, eps = row_scale.partials.data_ptr(), row_scale.partials.shape[1], row_scale.size, row_scale.eps
    out = torch.empty((T, Hq, D), dtype=dtype, device=q.device)
    _check(_entry("ptl_rope_store_f8")(
        out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), rs, positions.data_ptr(),
        inv_freq.data_ptr() if inv_freq is not None else None, slots.data_ptr() if slots is not None else None, *cache, T, Hq, Hkv, D,
        page_size, pages, partials, count, size, eps, _dtype_code(q), stream), "rope_store_f8")
    return out


def _attention(what: str, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, block_table, window, sink):
    """What the attentions have in common: (Hq, Hkv, D, page size, the entry's first arguments, address of the sink, alignment)."""
    shape = q.shape
    if len(shape) != 3 or out.shape != shape or out.dtype != q.dtype:
        raise KernelError(f"{what}: q and out must be [T, Hq, D] of one dtype")
    _, Hq, D = shape
    Hkv = k_cache.shape[1] if k_cache.dim() == 4 else 0
    _, page_size, cache = _cache(what, Hkv, D, k_cache, v_cache, k_scale, v_scale)
    if Hkv == 0 or Hq == 0 or Hq % Hkv:
        raise KernelError(f"{what}: {Hq} query heads are not a multiple of {Hkv} kv heads")
    (q_row, q_head, q_one), (out_row, out_head, out_one) = q.stride(), out.stride()
    if q_one != 1 or out_one != 1 or (Hq > 1 and (q_head != D or out_head != D)):
        raise KernelError(f"{what}: q and out need dense heads")
    _i32(q_start, "q_start")
    _i32(ctx_len, "ctx_len")
    n = ctx_len.numel()
    if q_start.numel() != n + 1:
        raise KernelError(f"{what}: inconsistent sequence tables")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] < n \
            or (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise KernelError(f"{what}: block_table must be int32 [n, max_pages]")
    if window < 0:
        raise KernelError(f"{what}: a window is not negative")
    if sink is not None and (sink.dtype != torch.float32 or sink.shape != (Hq,) or not sink.is_contiguous()):
        raise KernelError(f"{what}: sink must be a contiguous float32 tensor [{Hq}]")
    q_at, out_at = q.data_ptr(), out.data_ptr()
    args = (out_at, out_row, q_at, q_row, *cache, q_start.data_ptr(), ctx_len.data_ptr(), block_table.data_ptr(), block_table.stride(0))
    return Hq, Hkv, D, page_size, args, sink.data_ptr() if sink is not None else None, (q_at % 16 or q_row % 8, out_at % 8 or out_row % 4)


def _work(what: str, work_seq: torch.Tensor, work_qoff: torch.Tensor) -> int:
    _i32(work_seq, "work_seq")
    _i32(work_qoff, "work_qoff")
    n = work_seq.numel()
    if n != work_qoff.numel():
        raise KernelError(f"{what}: inconsistent work list")
    return n


def attention_generic_f8(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor, block_table: torch.Tensor,
                         work_seq: torch.Tensor, work_qoff: torch.Tensor, scale: float, window: int = 0,
                         sink: Optional[torch.Tensor] = None) -> None:
    """``attention_generic`` over an 8-bit cache: float32 or bfloat16 queries, head sizes up to 640, any page size; the work list names
    16-row query blocks. window, sink: as there."""
    what = "attention_generic_f8"
    stream = _launch_stream(what, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, block_table, sink, work_seq, work_qoff)
    Hq, Hkv, D, page_size, args, sink_at, _ = _attention(what, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len,
                                                         block_table, window, sink)
    if not 0 < D <= 640 or Hq > 65535:
        raise KernelError(f"{what}: head size {D} exceeds the kernel's limit of 640 (or {Hq} heads that of 65,535)")
    n = _work(what, work_seq, work_qoff)
    _check(_entry("ptl_attention_generic_f8")(*args, work_seq.data_ptr(), work_qoff.data_ptr(), n, q.shape[0], Hq, Hkv, D, page_size,
                                              int(window), sink_at, scale, _dtype_code(q), stream), what)


def attention_f8_fits(dtype: torch.dtype, num_heads: int, num_kv_heads: int, head_dim: int, page_size: int) -> bool:
    """Whether ``attention_decode_f8`` and ``attention_prefill_f8`` take this case: bfloat16, head size 32, 64, 96 or 128, a
    page size from 16 on that is a power of two, pages (of all kv heads) below 2 GiB."""
    return (dtype == torch.bfloat16 and head_dim % 32 == 0 and 0 < head_dim <= 128 and page_size >= 16
            and page_size & (page_size - 1) == 0 and num_kv_heads > 0 and num_heads % num_kv_heads == 0
            and 0 < num_heads // num_kv_heads <= 1024 and num_kv_heads * page_size * head_dim < 2 ** 31)


MOST_PARTS_F8 = 128        # parts of a (sequence, kv head) pair (csrc/attention_f8.hip)
WHOLE_KEYS_F8 = 512        # keys of a pair that is never cut


def _decode_parts(device: torch.device, num_heads: int, num_kv_heads: int) -> int:
    """Parts of all sequences' keys, some: a workgroup a compute unit."""
    return max(1, min(MOST_PARTS_F8, compute_units(device) // (num_kv_heads * -(-(num_heads // num_kv_heads) // 16))))


def attention_decode_f8(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                        v_scale: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor, block_table: torch.Tensor, n_seq: int,
                        scale: float, window: int = 0, sink: Optional[torch.Tensor] = None,
                        tickets: Optional[torch.Tensor] = None) -> None:
    """Attention of the first ``n_seq`` sequences of the tables, each of which brings exactly one query token, over an 8-bit cache
    (``attention_f8_fits`` says for which sizes). How the keys are cut is decided on the device from ctx_len. ``tickets``: as for
    ``attention_decode``, TICKET * n_seq * kv heads for every 16 heads of a kv head."""
    what = "attention_decode_f8"
    stream = _launch_stream(what, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, block_table, sink, tickets)
    Hq, Hkv, D, page_size, args, sink_at, unaligned = _attention(what, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len,
                                                                 block_table, window, sink)
    if unaligned[0] or not attention_f8_fits(q.dtype, Hq, Hkv, D, page_size):
        raise KernelError(f"{what}: needs bfloat16, a head size of 32/64/96/128, a page size from 16 on that is a power of two, "
                          "aligned q rows")
    if not 0 <= n_seq <= ctx_len.numel() or n_seq > q.shape[0]:
        raise KernelError(f"{what}: tables, or q, are shorter than n_seq")
    if n_seq == 0:
        return
    cap, parts_at, ends_at, tickets_at = 0, None, None, None
    if tickets is not None:
        _tickets(tickets, 0, q, what)                        # (checks)
    if block_table.shape[1] * page_size > WHOLE_KEYS_F8:
        tiles = -(-(Hq // Hkv) // 16)
        cap = _decode_parts(q.device, Hq, Hkv)
        heads = (n_seq + cap) * Hq                                                   # (room for parts: csrc/attention_f8.hip)
        parts = torch.empty(heads * (D + 2), dtype=torch.float32, device=q.device)
        tickets = _tickets(tickets, TICKET * n_seq * Hkv * tiles, q, what)
        parts_at, tickets_at = parts.data_ptr(), tickets.data_ptr()
        ends_at = parts_at + 4 * heads * D
    _check(_entry("ptl_attention_decode_f8")(*args, parts_at, ends_at, tickets_at, cap, int(n_seq), Hq, Hkv, D, page_size, int(window), sink_at,
                                             scale, stream), what)


WORTH_TILES = 12           # tiles of 64 keys that blocks of query rows have to become shorter by to be cut (csrc/attention_f8.hip)


def _prefill_resident(device: torch.device, num_heads: int, head_dim: int) -> int:
    """Workgroups of a head that ``attention_prefill_f8`` runs at once."""
    return compute_units(device) * (3 if head_dim <= 64 else 2) // num_heads


def attention_prefill_f8_plan(device: torch.device, num_heads: int, head_dim: int, blocks_of_64: int, blocks_of_128: int,
                              max_keys: int = 0, bound: bool = False):
    """(block_rows, groups) for ``attention_prefill_f8``; arguments as of ``attention_prefill_mfma_plan``, which it follows but where
    blocks have many keys each. With t = the workgroups of a head that run at once, four blocks of 128 rows or more, and max_keys the
    longest sequence's, blocks have 128 rows
      where blocks of 64 are cut (2 of them fill no more than t): above head size 64 from 3,000 keys a workgroup on (blocks * max_keys / t);
      where each has a workgroup: from 4,800 keys on;
      where they are more than t: from 400 keys for each block of 128 rows on, above head size 64 from 192.
    us in blocks of 64 and of 128 rows, heads x head size, rows behind keys. Cut: 8 x 64 512 behind 6,000 30 41, 2,048 behind 6,000 65 72; 16 x 64
    1,024 behind 4,000 46 54; 32 x 64 512 behind 6,000 58 66; 16 x 128 512 behind 6,000 63 66, 1,024 behind 4,000 78 87; 8 x 128 2,048 behind 6,000
    110 110; 32 x 128 500 behind 3,000 62 64, 512 behind 6,000 100 89, behind 8,000 122 109. A workgroup each: 16 x 64 2,048 behind 2,000 57 62, behind
    6,000 120 102; 32 x 64 1,024 behind 1,000 32 42, behind 4,000 79 75; 64 x 64 512 behind 6,000 106 91; 16 x 128 2,048 behind 2,000 90 97, behind
    6,000 185 175; 32 x 128 1,024 behind 1,000 49 58, 900 behind 4,000 128 123; 64 x 128 512 behind 6,000 163 150. More: 32 x 64 2,048 behind 3,000
    107 113, behind 6,000 188 179; 64 x 64 1,024 behind 4,000 124 124; 32 x 128 1,536 behind 500 67 72, 1,531 behind 1,000 97 86, 2,048 behind 2,000
    160 140; 64 x 128 1,024 behind 1,000 87 77.

    ``bound``: max_keys is only a bound of what the sequences will have (a step that is recorded). Then blocks of 128 rows are for
    head sizes above 64, a bound from 4,096 on and blocks of 64 rows that have no workgroup each at once: 2,048 rows of 128 lose 7 us
    by them where the prompt begins and win 24 behind 2,048 keys; 1,024 rows lose 17 and win 8 behind 6,000."""
    t = max(1, _prefill_resident(device, num_heads, head_dim))
    if bound:
        long = blocks_of_64 > t and head_dim > 64 and max_keys >= 4096
    elif 2 * blocks_of_64 <= t:
        long = head_dim > 64 and blocks_of_64 * max_keys >= 3000 * t
    elif blocks_of_64 <= t:
        long = max_keys >= 4800
    else:
        long = max_keys >= (192 if head_dim > 64 else 400) * blocks_of_128
    long = long and (bound or blocks_of_128 >= 4)
    rows, blocks = (128, blocks_of_128) if long or 4 * blocks_of_128 >= 5 * t else (64, blocks_of_64)
    return rows, max(1, blocks if blocks <= 2 * t else t)


def _cut_into(device: torch.device, num_heads: int, head_dim: int, blocks: int, groups: int, block_rows: int, table_keys: int) -> int:
    """Parts a head that ``attention_prefill_f8`` cuts its blocks into, some; 0: it leaves them whole. table_keys: keys that a row of
    the block table has room for."""
    if groups != blocks or blocks > 64 or table_keys <= 64 * WORTH_TILES:
        return 0
    resident = _prefill_resident(device, num_heads, head_dim)
    # (blocks of 64 rows that fill more than half of it are as fast whole, of 128 rows five sixths: csrc/attention_f8.hip has the figures)
    return resident if (2 * blocks <= resident if block_rows == 64 else 6 * blocks <= 5 * resident) else 0


def attention_prefill_f8_tickets(device: torch.device, num_heads: int, head_dim: int, blocks: int, groups: int, block_rows: int,
                                 table_keys: int) -> int:
    """How many tickets ``attention_prefill_f8`` counts in for so many blocks and groups, over a block table whose rows have room
    for ``table_keys`` keys (0: none)."""
    return TICKET * blocks * num_heads if _cut_into(device, num_heads, head_dim, blocks, groups, block_rows, table_keys) else 0


def attention_f8_workspace_bytes(device: torch.device, num_heads: int, num_kv_heads: int, head_dim: int, num_seqs: int) -> int:
    """The most that one call of ``attention_decode_f8`` with up to ``num_seqs`` sequences, or of ``attention_prefill_f8``, makes for the
    parts that it cuts keys into."""
    cap = _decode_parts(device, num_heads, num_kv_heads)
    most = (num_seqs + cap) * num_heads * (head_dim + 2)
    for rows in (64, 128):
        blocks = max((n for n in range(1, 65) if _cut_into(device, num_heads, head_dim, n, n, rows, 1 << 30)), default=0)
        if blocks:
            parts = _cut_into(device, num_heads, head_dim, blocks, blocks, rows, 1 << 30)
            most = max(most, (blocks + parts) * num_heads * rows * (head_dim + 8))
    return 4 * most


def attention_prefill_f8(out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, q_start: torch.Tensor, ctx_len: torch.Tensor, block_table: torch.Tensor,
                         work_seq: torch.Tensor, work_qoff: torch.Tensor, scale: float, window: int = 0, block_rows: int = 64,
                         groups: int = 0, sink: Optional[torch.Tensor] = None, tickets: Optional[torch.Tensor] = None) -> None:
    """``attention_prefill_mfma`` over an 8-bit cache (``attention_f8_fits`` says for which sizes): the work list names query blocks
    of ``block_rows`` (64 or 128) rows, those with the most keys first; ``groups`` workgroups a head share it (0: one for
    every block). Where blocks have a workgroup each and these fill less than the GPU, blocks are cut along their keys, on the device and
    by the contexts that it finds there.
    ``tickets``: zeros that such launches on one stream may share, as many as ``attention_prefill_f8_tickets`` says (else they are
    made)."""
    what = "attention_prefill_f8"
    stream = _launch_stream(what, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len, block_table, sink, work_seq, work_qoff,
                            tickets)
    Hq, Hkv, D, page_size, args, sink_at, unaligned = _attention(what, out, q, k_cache, v_cache, k_scale, v_scale, q_start, ctx_len,
                                                                 block_table, window, sink)
    if not attention_f8_fits(q.dtype, Hq, Hkv, D, page_size):
        raise KernelError(f"{what}: needs bfloat16, a head size of 32/64/96/128, a page size from 16 on that is a power of two")
    if unaligned[0] or unaligned[1]:
        raise KernelError(f"{what}: q rows must be 16-byte aligned, out rows 8-byte")
    if block_rows not in (64, 128):
        raise KernelError(f"{what}: query blocks are 64 or 128 rows")
    if not scale > 0:
        raise KernelError(f"{what}: scale must be positive")
    n = _work(what, work_seq, work_qoff)
    if n == 0:
        return
    groups = min(n, groups, 65535) if groups > 0 else min(n, 65535)
    cap, work_at, tickets_at = _cut_into(q.device, Hq, D, n, groups, block_rows, block_table.shape[1] * page_size), None, None
    if cap:
        work = torch.empty((n + cap) * Hq * block_rows * (D + 8), dtype=torch.float32, device=q.device)
        tickets = _tickets(tickets, TICKET * n * Hq, q, what)
        work_at, tickets_at = work.data_ptr(), tickets.data_ptr()
    _check(_entry("ptl_attention_prefill_f8")(*args, work_seq.data_ptr(), work_qoff.data_ptr(), n, groups, cap, work_at, tickets_at,
                                              block_rows, Hq, Hkv, D, page_size, int(window), sink_at, scale, stream), what)


def copy_pages(pools: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    """Page src[i] -> page dst[i] in all layers of every pool [layers, pages, ...] (contiguous, up to 16 of them, any dtype), a
    launch for 256 pages. src, dst: page numbers on the host; no page may be written twice, or both read and written (one may be read many
    times). The numbers go with the launch: nothing is uploaded, and a recorded launch keeps its own."""
    src, dst = list(src), list(dst)
    n = len(src)
    if n != len(dst):
        raise KernelError(f"copy_pages: {n} pages to read, {len(dst)} to write")
    stream = _launch_stream("copy_pages", *pools)
    if len(pools) > 16:
        raise KernelError("copy_pages: up to 16 pools a call")
    low, high = (min(min(src), min(dst)), max(max(src), max(dst))) if n else (0, -1)
    desc = []
    for t in pools:
        shape = t.shape
        if len(shape) < 2 or not t.is_contiguous():
            raise KernelError("copy_pages: a pool is a contiguous tensor [layers, pages, ...]")
        if low < 0 or high >= shape[1]:
            raise KernelError(f"copy_pages: a page number lies outside the pool's {shape[1]} pages")
        if t.numel():
            desc += (t.data_ptr(), shape[0], shape[1], t.stride(1) * t.element_size())
    written = set(dst)
    if len(written) != n or not written.isdisjoint(src):
        raise KernelError("copy_pages: a page is written twice, or read and written")
    if n == 0 or not desc:
        return
    numbers, described = array.array("i", src + dst), array.array("l", desc)
    at = numbers.buffer_info()[0]
    _check(_entry("ptl_copy_pages")(described.buffer_info()[0], len(desc) // 4, at, at + 4 * n, n, stream), "copy_pages")

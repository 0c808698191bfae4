"""4-bit paged KV cache: quantised as it is written, read back, attended, and attended sparsely.

The reference has no 4-bit cache; this module defines one and keeps the conventions of the
16-bit and FP8 entry points.

    kv4_pool : uint8 [pages, Hkv, page_size / 16, 20 * D], D = 64 or 128, page_size a multiple of 16

One pool holds K and V.  Every 32 channels of a token's row are a group with a step and a floor
of the element type (fp16 or bf16, that of Q): floor = min, step = (max - min) / 15, and a channel
is a code 0..15 that stands for code * step + floor -- 5 bits a channel, 0.31 of a 16-bit cache.
The steps travel with the codes, so a row is quantised when it is written and never again; a pool
is written and read with one element type.  The bytes of a tile are laid out in
include/qf_hotpath.h.

    pool = empty_kv_pool_int4(pages, kv_heads, head_dim, device=...)
    q = packed_qkv_rope_cache_int4(packed, positions, slots, pool)           # RoPE, quantise, store
    out = paged_decode_attention_int4(q, pool, block_table, seq_lens)        # every page
    k, v = read_kv_int4(pool, slots, dtype=q.dtype)                          # rows as 16-bit K and V

Long contexts: a query attends its newest page and the pages whose keys can score highest.

    bounds = empty_key_bounds_int4(pool, dtype)
    update_key_bounds_int4(pool, bounds, block_table, seq_lens, new_tokens=n)   # after n tokens
    out, pages, lens = sparse_decode_attention_int4(q, pool, bounds, block_table, seq_lens, num_pages=64)

Every call enqueues on the current stream of its tensors' device, reads nothing back and may be
captured into a CUDA graph; scratch is a torch allocation of the call.  There is no CPU path.
"""

from __future__ import annotations

import ctypes
import importlib.util
import sys
from pathlib import Path

TILE_TOKENS = 16
MAX_GROUP = 16

_cabi_module = None


def _cabi():
    """The ctypes binding, loaded by path so this file works under any module name."""
    global _cabi_module
    if _cabi_module is None:
        module = sys.modules.get("qf_hotpath_cabi")
        if module is None:
            path = Path(__file__).resolve().parents[1] / "_cabi.py"
            spec = importlib.util.spec_from_file_location("qf_hotpath_cabi", path)
            module = importlib.util.module_from_spec(spec)
            sys.modules["qf_hotpath_cabi"] = module
            spec.loader.exec_module(module)
        _cabi_module = module
    return _cabi_module


def _require(condition, message):
    if not condition:
        raise ValueError(message)


def _check_pool(torch, pool):
    """(kv_heads, head_dim, page_size) of a 4-bit pool."""
    _require(pool.ndim == 4 and pool.dtype == torch.uint8 and pool.shape[3] in (1280, 2560),
             "a 4-bit pool is uint8 [pages, kv_heads, page_size / 16, 20 * head_dim] with head_dim 64 or 128")
    _require(pool.shape[1] >= 1 and pool.shape[2] >= 1, "a 4-bit pool has at least one KV head and one tile a page")
    _require(pool.is_cuda, "the 4-bit cache needs a CUDA device")
    _require(pool.is_contiguous() and pool.data_ptr() % 16 == 0, "a 4-bit pool must be contiguous and 16-byte aligned")
    return pool.shape[1], pool.shape[3] // 20, pool.shape[2] * TILE_TOKENS


def _element_code(torch, dtype):
    if dtype is torch.float16:
        return 0
    if dtype is torch.bfloat16:
        return 1
    raise ValueError("a 4-bit cache is written and read as float16 or bfloat16")


def _index_code(torch, tensor, what):
    if tensor.dtype is torch.int32:
        return 0
    if tensor.dtype is torch.int64:
        return 1
    raise ValueError(f"{what} must use an integer dtype")


def empty_kv_pool_int4(num_pages, kv_heads, head_dim, *, page_size=16, device=None):
    """An uninitialised 4-bit pool for K and V; its rows are defined once they are written."""
    import torch

    _require(head_dim in (64, 128), "head_dim must be 64 or 128")
    _require(page_size >= TILE_TOKENS and page_size % TILE_TOKENS == 0, "page_size must be a multiple of 16")
    return torch.empty((num_pages, kv_heads, page_size // TILE_TOKENS, 20 * head_dim), dtype=torch.uint8,
                       device="cuda" if device is None else device)


def empty_key_bounds_int4(kv4_pool, dtype):
    """Storage for the smallest and the largest key of every page: [pages, kv_heads, 2, D]."""
    import torch

    kv_heads, dim, _ = _check_pool(torch, kv4_pool)
    _element_code(torch, dtype)
    return torch.empty((kv4_pool.shape[0], kv_heads, 2, dim), dtype=dtype, device=kv4_pool.device)


def _write(q, k, v, q_out, q_strides, k_strides, v_strides, o_strides, positions, slot_mapping, pool, *,
           rows, q_heads, kv_heads, head_dim, page_size, base, rope_table, valid_tokens=None):
    """Check what every write shares, fill qf_int4_write_args and enqueue on the current stream."""
    import torch

    cabi = _cabi()
    device = pool.device
    dtype = _element_code(torch, k.dtype)
    _require(v.dtype == k.dtype and (q is None or q.dtype == k.dtype), "Q/K/V must share FP16 or BF16 dtype")
    operands = [t for t in (q, k, v, positions, slot_mapping, rope_table, valid_tokens) if t is not None]
    _require(all(t.device == device for t in operands), "the 4-bit cache write needs CUDA tensors of one device")
    positions_code = 0
    if positions is not None:
        if positions.dtype is torch.float32 and rope_table is None:
            positions_code = cabi.INDEX_F32
        else:
            positions_code = _index_code(torch, positions, "positions")
    if rope_table is not None:
        _require(rope_table.ndim == 3 and rope_table.shape[0] >= 1 and tuple(rope_table.shape[1:]) == (head_dim // 2, 2)
                 and rope_table.dtype == torch.float32 and rope_table.is_contiguous(),
                 "rope_table must be contiguous float32 [positions, head_dim / 2, 2]")
    if valid_tokens is not None:
        _require(valid_tokens.dtype == torch.int32 and valid_tokens.numel() == 1,
                 "valid_tokens must be a CUDA int32 scalar")
    args = cabi.Int4WriteArgs(
        None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), None if q is None else q_out.data_ptr(),
        *q_strides, *k_strides, *v_strides, *o_strides,
        None if positions is None else positions.data_ptr(), 0 if positions is None else positions.stride(0),
        None if slot_mapping is None else slot_mapping.data_ptr(), 0 if slot_mapping is None else slot_mapping.stride(0),
        None if rope_table is None else rope_table.data_ptr(), pool.data_ptr(), pool.shape[0],
        None if valid_tokens is None else valid_tokens.data_ptr(),
        rows, q_heads, kv_heads, head_dim, page_size, dtype, positions_code,
        0 if slot_mapping is None else _index_code(torch, slot_mapping, "slot mapping"),
        0 if rope_table is None else rope_table.shape[0], float(base))
    with cabi.device_of(pool):
        cabi.check(cabi.library().qf_int4_rope_kv_write(ctypes.byref(args), cabi.stream_pointer(device)))


def packed_qkv_rope_cache_int4(
    packed, positions, slot_mapping, kv4_pool, *, q_heads=12, base=1_000_000.0, rope_table=None, valid_tokens=None,
):
    """packed_qkv_rope_cache for the 4-bit cache: packed (rows, (q_heads + 2 kv_heads) * D) -> q (rows, q_heads, D).

    Rotated K and V go to slot_mapping[row] (page * page_size + row in page; outside the pool: the
    row is skipped).  rope_table (positions, D / 2, 2) float32 (cos, sin) pairs; without it the
    angles are position * base^(-2i / D).  Rows at or beyond valid_tokens get zero queries and no
    cache write.  No two rows of a call may have the same slot."""
    import torch

    if packed.ndim == 3:
        _require(packed.shape[1] == 1, "packed QKV must have one decode token per row")
        packed = packed[:, 0, :]
    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    _require(q_heads >= 1, "q_heads must be positive")
    _require(packed.ndim == 2 and packed.shape[1] == (q_heads + 2 * kv_heads) * dim,
             "expected packed QKV shape (rows, (q_heads + 2 * kv_heads) * head_dim)")
    rows = packed.shape[0]
    _require(positions.shape == (rows,) and slot_mapping.shape == (rows,),
             "positions and slots must contain one value per row")
    q = torch.empty((rows, q_heads, dim), device=packed.device, dtype=packed.dtype)
    row_stride, col_stride = packed.stride()
    segment = (row_stride, dim * col_stride, col_stride)
    _write(packed, packed[:, q_heads * dim:], packed[:, (q_heads + kv_heads) * dim:], q, segment, segment, segment,
           q.stride(), positions, slot_mapping, kv4_pool, rows=rows, q_heads=q_heads, kv_heads=kv_heads, head_dim=dim,
           page_size=page_size, base=base, rope_table=rope_table, valid_tokens=valid_tokens)
    return q


def native_decode_rope_kv_write_int4(
    q, k, v, positions, slot_mapping, kv4_pool, *, base=1_000_000.0, rope_table=None, rotate_q=True,
):
    """native_decode_rope_kv_write for the 4-bit cache: q (B, Hq, 1, D), k and v (B, Hkv, 1, D).
    Returns rotated Q (or q when rotate_q=False)."""
    import torch

    _require(all(t.ndim == 4 and t.shape[2] == 1 for t in (q, k, v)),
             "decode Q/K/V must have shape (batch, heads, 1, dim)")
    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    batch = q.shape[0]
    _require(k.shape == v.shape and tuple(k.shape) == (batch, kv_heads, 1, dim) and q.shape[-1] == dim,
             "decode K/V shapes do not match Q and the pool")
    _require(positions.shape == (batch,) and slot_mapping.shape == (batch,),
             "positions and slots must contain one entry per batch row")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if rotate_q else q
    rows_of = lambda t: (t.stride(0), t.stride(1), t.stride(3))  # noqa: E731
    _write(q if rotate_q else None, k, v, out, rows_of(q), rows_of(k), rows_of(v), rows_of(out), positions, slot_mapping,
           kv4_pool, rows=batch, q_heads=q.shape[1] if rotate_q else 0, kv_heads=kv_heads, head_dim=dim,
           page_size=page_size, base=base, rope_table=rope_table)
    return out


def rope_kv_write_int4(q, k, v, positions, slot_mapping, kv4_pool, *, base=1_000_000.0, rope_table=None):
    """rope_kv_write for the 4-bit cache: q (1, Hq, T, D), k and v (1, Hkv, T, D), one prompt or a
    packed chunk of several.  Returns rotated Q shaped like q."""
    import torch

    _require(q.ndim == 4 and k.ndim == 4 and v.ndim == 4, "q, k, and v must be rank-four tensors")
    _require(q.shape[0] == 1 and k.shape[0] == 1 and v.shape[0] == 1,
             "packed q, k, and v must have batch dimension one")
    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    tokens = q.shape[2]
    _require(k.shape == v.shape and tuple(k.shape) == (1, kv_heads, tokens, dim) and q.shape[-1] == dim,
             "K/V shapes do not match Q and the pool")
    if positions.ndim == 2:
        _require(tuple(positions.shape) == (1, tokens), "positions must have shape (1, tokens)")
        positions = positions[0]
    _require(positions.shape == (tokens,) and slot_mapping.shape == (tokens,),
             "positions and slots must contain one entry per token")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    rows_of = lambda t: (t.stride(2), t.stride(1), t.stride(3))  # noqa: E731
    _write(q, k, v, out, rows_of(q), rows_of(k), rows_of(v), rows_of(out), positions, slot_mapping, kv4_pool,
           rows=tokens, q_heads=q.shape[1], kv_heads=kv_heads, head_dim=dim, page_size=page_size, base=base,
           rope_table=rope_table)
    return out


def quantize_kv_pool_int4(k_pool, v_pool):
    """A 4-bit pool with the contents of fp16 / bf16 pools [pages, page_size, Hkv, D] (keys as they are:
    already rotated).  Every row of the pools is quantised; rows with a NaN or an infinity read back as NaN."""
    import torch

    _require(k_pool.ndim == 4 and k_pool.shape == v_pool.shape and k_pool.is_contiguous() and v_pool.is_contiguous(),
             "K/V pools must be contiguous with matching rank-four shapes")
    pages, page_size, kv_heads, dim = k_pool.shape
    _require(k_pool.is_cuda and v_pool.device == k_pool.device, "K/V pools must share one CUDA device")
    pool = empty_kv_pool_int4(pages, kv_heads, dim, page_size=page_size, device=k_pool.device)
    strides = (kv_heads * dim, dim, 1)
    _write(None, k_pool, v_pool, None, strides, strides, strides, strides, None, None, pool, rows=pages * page_size,
           q_heads=0, kv_heads=kv_heads, head_dim=dim, page_size=page_size, base=1.0, rope_table=None)
    return pool


def _read(torch, kv4_pool, slot_mapping, rows, dtype):
    cabi = _cabi()
    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    code = _element_code(torch, dtype)
    k = torch.empty((rows, kv_heads, dim), dtype=dtype, device=kv4_pool.device)
    v = torch.empty((rows, kv_heads, dim), dtype=dtype, device=kv4_pool.device)
    slots = (None, 0, 0)
    if slot_mapping is not None:
        slots = (slot_mapping.data_ptr(), _index_code(torch, slot_mapping, "slot mapping"), slot_mapping.stride(0))
    with cabi.device_of(kv4_pool):
        cabi.check(cabi.library().qf_int4_read_rows(
            kv4_pool.data_ptr(), kv4_pool.shape[0], page_size, kv_heads, dim, code, *slots, rows, k.data_ptr(),
            v.data_ptr(), cabi.stream_pointer(kv4_pool.device)))
    return k, v


def read_kv_int4(kv4_pool, slot_mapping, *, dtype=None):
    """Rows of the cache at a list of slots as (k, v), both [n, Hkv, D] in `dtype` (that of the
    writes; default float16).  A slot outside the pool, -1 for one, gives a row of zeros."""
    import torch

    _require(slot_mapping.ndim == 1, "slot mapping must be a list of slots")
    _require(slot_mapping.device == kv4_pool.device, "pool and slots must share one CUDA device")
    return _read(torch, kv4_pool, slot_mapping, slot_mapping.shape[0], torch.float16 if dtype is None else dtype)


def dequantize_kv_pool_int4(kv4_pool, dtype=None):
    """The whole cache as 16-bit pools (k_pool, v_pool), both [pages, page_size, Hkv, D]."""
    import torch

    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    k, v = _read(torch, kv4_pool, None, kv4_pool.shape[0] * page_size, torch.float16 if dtype is None else dtype)
    shape = (kv4_pool.shape[0], page_size, kv_heads, dim)
    return k.view(shape), v.view(shape)


def _paged(torch, cabi, batch, kv_heads, dim, page_size, num_pages, dtype, block_table, seq_lens, *, per_head,
           q=None, out=None, pool=None, bounds=None, page_table=None, page_lens=None, new_tokens=0, take=0, scale=0.0):
    """Check table and lengths and fill qf_paged_int4_args (no workspace yet)."""
    heads_too = per_head and block_table.ndim == 3
    if heads_too:
        _require(tuple(block_table.shape[:2]) == (batch, kv_heads) and tuple(seq_lens.shape) == (batch, kv_heads),
                 "a table and lengths per KV head have shapes [batch, kv_heads, pages] and [batch, kv_heads]")
        t_sb, t_sh, t_sp = block_table.stride()
        l_sb, l_sh = seq_lens.stride()
    else:
        _require(block_table.ndim == 2 and seq_lens.ndim == 1 and block_table.shape[0] == batch
                 and seq_lens.shape[0] == batch, "batch dimensions must match")
        (t_sb, t_sp), t_sh = block_table.stride(), 0
        l_sb, l_sh = seq_lens.stride(0), 0
    q_strides = (0, 0) if q is None else (q.stride(0), q.stride(1))
    o_strides = (0, 0) if out is None else (out.stride(0), out.stride(1))
    pointer = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    return cabi.PagedInt4Args(
        pointer(q), pointer(out), pointer(pool), pointer(bounds), block_table.data_ptr(), seq_lens.data_ptr(), None,
        pointer(page_table), pointer(page_lens), *q_strides, *o_strides, t_sb, t_sh, t_sp, l_sb, l_sh,
        num_pages, block_table.shape[-1], 0, batch, 0 if q is None else q.shape[1], kv_heads, dim, page_size, dtype,
        _index_code(torch, block_table, "page table"), _index_code(torch, seq_lens, "lengths"), new_tokens, take, scale)


def _add_workspace(torch, cabi, args, call, device):
    """Scratch of one call: a torch allocation, so it is the stream's (and a captured graph's own)."""
    need = ctypes.c_int64(0)
    cabi.check(cabi.library().qf_paged_int4_workspace(ctypes.byref(args), call, ctypes.byref(need)))
    scratch = torch.empty(need.value, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = scratch.data_ptr(), need.value
    return scratch


def _check_query(torch, q, kv_heads, dim):
    """q as the kernels take it: unit inner stride, rows on 16-byte boundaries."""
    _require(q.ndim == 3 and q.shape[1] >= 1 and q.shape[2] == dim, "q must have shape [batch, query_heads, head_dim]")
    _require(q.shape[1] % kv_heads == 0, "query heads must be divisible by KV heads")
    _require(q.shape[1] // kv_heads <= MAX_GROUP, "at most 16 query heads share a KV head")
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        q = q.clone() if q.data_ptr() % 16 else q
    return q


def paged_decode_attention_int4(q, kv4_pool, block_table, seq_lens, *, scale=None):
    """GQA decode attention over the 4-bit cache: q [B, Hq, D] -> out [B, Hq, D] in q's dtype, which is
    that of the cache's writes.

    block_table [B, n] and seq_lens [B], or one table and length per KV head: [B, Hkv, n] and [B, Hkv]
    (what select_kv_pages returns).  seq_lens counts the tokens attended, the newest included; a row of
    length 0 gives zeros.  Default scale D ** -0.5.  The split over the GPU is planned on the device from
    the lengths, so there is no split_k."""
    import torch

    cabi = _cabi()
    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    dtype = _element_code(torch, q.dtype)
    q = _check_query(torch, q, kv_heads, dim)
    device = kv4_pool.device
    _require(q.device == device and block_table.device == device and seq_lens.device == device,
             "q, pool, page table and lengths must share one CUDA device")
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    args = _paged(torch, cabi, q.shape[0], kv_heads, dim, page_size, kv4_pool.shape[0], dtype, block_table, seq_lens,
                  per_head=True, q=q, out=out, pool=kv4_pool, scale=dim ** -0.5 if scale is None else scale)
    with cabi.device_of(kv4_pool):
        scratch = _add_workspace(torch, cabi, args, cabi.INT4_ATTENTION, device)
        cabi.check(cabi.library().qf_int4_decode_attention(ctypes.byref(args), cabi.stream_pointer(device)))
    del scratch
    return out


def _check_bounds(torch, bounds, dtype):
    _require(bounds.ndim == 4 and bounds.shape[2] == 2 and bounds.shape[3] in (64, 128) and bounds.dtype == dtype
             and bounds.is_contiguous() and bounds.data_ptr() % 16 == 0,
             "key bounds must be contiguous [pages, kv_heads, 2, head_dim] in the queries' dtype")
    _require(bounds.is_cuda, "key bounds must be on a CUDA device")


def update_key_bounds_int4(kv4_pool, key_bounds, block_table, seq_lens, *, new_tokens=1):
    """Recompute key_bounds for the pages that hold one of the last new_tokens tokens of each sequence
    (1 after a decode step, the prompt's length after a prefill); returns key_bounds.

    Bounds are the smallest and the largest key of a page's tokens below seq_lens, per channel, as the
    cache reads back."""
    import torch

    cabi = _cabi()
    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    dtype = _element_code(torch, key_bounds.dtype)
    _check_bounds(torch, key_bounds, key_bounds.dtype)
    _require(key_bounds.shape[0] == kv4_pool.shape[0] and key_bounds.shape[1] == kv_heads and key_bounds.shape[3] == dim,
             "key bounds do not match the pool")
    _require(isinstance(new_tokens, int) and not isinstance(new_tokens, bool) and 0 <= new_tokens < 2 ** 31,
             "new_tokens must be a non-negative integer")
    device = kv4_pool.device
    _require(key_bounds.device == device and block_table.device == device and seq_lens.device == device,
             "pool, key bounds, page table and lengths must share one CUDA device")
    args = _paged(torch, cabi, block_table.shape[0], kv_heads, dim, page_size, kv4_pool.shape[0], dtype, block_table,
                  seq_lens, per_head=False, pool=kv4_pool, bounds=key_bounds, new_tokens=new_tokens)
    with cabi.device_of(kv4_pool):
        cabi.check(cabi.library().qf_int4_key_bounds(ctypes.byref(args), cabi.stream_pointer(device)))
    return key_bounds


def _check_take(num_pages):
    _require(isinstance(num_pages, int) and not isinstance(num_pages, bool) and 1 <= num_pages < 2 ** 31,
             "num_pages must be a positive integer")


def select_kv_pages(q, key_bounds, block_table, seq_lens, *, num_pages, page_size=16):
    """The pages each sequence's queries attend, per KV head: (page_table int32 [B, Hkv, num_pages],
    page_lens int32 [B, Hkv]), a table and lengths for paged_decode_attention_int4.

    A row is the sequence's newest page and the num_pages - 1 others with the highest bound on a score,
    the largest over the KV head's query heads of sum_d max(q_d * low_d, q_d * high_d); ties go to the
    earlier page.  Pages keep the sequence's order; -1 pads a sequence that has fewer."""
    import torch

    cabi = _cabi()
    dtype = _element_code(torch, q.dtype)
    _check_bounds(torch, key_bounds, q.dtype)
    kv_heads, dim = key_bounds.shape[1], key_bounds.shape[3]
    q = _check_query(torch, q, kv_heads, dim)
    _check_take(num_pages)
    _require(page_size >= TILE_TOKENS and page_size % TILE_TOKENS == 0, "page_size must be a multiple of 16")
    device = key_bounds.device
    _require(q.device == device and block_table.device == device and seq_lens.device == device,
             "q, key bounds, page table and lengths must share one CUDA device")
    batch = q.shape[0]
    page_table = torch.empty((batch, kv_heads, num_pages), dtype=torch.int32, device=device)
    page_lens = torch.empty((batch, kv_heads), dtype=torch.int32, device=device)
    args = _paged(torch, cabi, batch, kv_heads, dim, page_size, key_bounds.shape[0], dtype, block_table, seq_lens,
                  per_head=False, q=q, bounds=key_bounds, page_table=page_table, page_lens=page_lens, take=num_pages)
    with cabi.device_of(key_bounds):
        scratch = _add_workspace(torch, cabi, args, cabi.INT4_SELECT, device)
        cabi.check(cabi.library().qf_select_kv_pages(ctypes.byref(args), cabi.stream_pointer(device)))
    del scratch
    return page_table, page_lens


def sparse_decode_attention_int4(q, kv4_pool, key_bounds, block_table, seq_lens, *, num_pages, scale=None):
    """select_kv_pages and paged_decode_attention_int4 over its choice in one call: (out, page_table,
    page_lens).  key_bounds must be up to date for every page but a sequence's newest."""
    import torch

    cabi = _cabi()
    kv_heads, dim, page_size = _check_pool(torch, kv4_pool)
    dtype = _element_code(torch, q.dtype)
    _check_bounds(torch, key_bounds, q.dtype)
    _require(key_bounds.shape[0] == kv4_pool.shape[0] and key_bounds.shape[1] == kv_heads and key_bounds.shape[3] == dim,
             "key bounds do not match the pool")
    q = _check_query(torch, q, kv_heads, dim)
    _check_take(num_pages)
    device = kv4_pool.device
    _require(q.device == device and key_bounds.device == device and block_table.device == device
             and seq_lens.device == device, "q, pool, key bounds, page table and lengths must share one CUDA device")
    batch = q.shape[0]
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    page_table = torch.empty((batch, kv_heads, num_pages), dtype=torch.int32, device=device)
    page_lens = torch.empty((batch, kv_heads), dtype=torch.int32, device=device)
    args = _paged(torch, cabi, batch, kv_heads, dim, page_size, kv4_pool.shape[0], dtype, block_table, seq_lens,
                  per_head=False, q=q, out=out, pool=kv4_pool, bounds=key_bounds, page_table=page_table,
                  page_lens=page_lens, take=num_pages, scale=dim ** -0.5 if scale is None else scale)
    with cabi.device_of(kv4_pool):
        scratch = _add_workspace(torch, cabi, args, cabi.INT4_SPARSE, device)
        cabi.check(cabi.library().qf_int4_sparse_decode_attention(ctypes.byref(args), cabi.stream_pointer(device)))
    del scratch
    return out, page_table, page_lens

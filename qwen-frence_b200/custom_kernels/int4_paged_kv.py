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

Block tables and lengths are step metadata: attention, scores and choice may read them while the
kernel in front on the stream still runs.  Copies and torch ops that rewrite them need nothing more
when a write, read or bounds call follows; in front of any other call of this library, ops that
rewrite them in place are followed by qf_order_next_launch(), as for the 16-bit cache.  What
select_kv_pages returns may go straight to paged_decode_attention_int4, whatever else is launched
between them, on this stream or another.
"""

from __future__ import annotations

import ctypes
import importlib.util
import sys
from pathlib import Path

import torch

TILE_TOKENS = 16
MAX_GROUP = 16
MAX_ITEMS = 2 ** 31 - 128  # threads of one write

def _load_cabi():
    """The ctypes binding, loaded by path so this file works under any module name."""
    module = sys.modules.get("qf_hotpath_cabi")
    if module is None:
        path = Path(__file__).resolve().parents[1] / "_cabi.py"
        spec = importlib.util.spec_from_file_location("qf_hotpath_cabi", path)
        module = importlib.util.module_from_spec(spec)
        sys.modules["qf_hotpath_cabi"] = module
        spec.loader.exec_module(module)
    return module


_cabi = _load_cabi()


def _require(condition, message):
    if not condition:
        raise ValueError(message)


_ELEMENT_CODES = {torch.float16: 0, torch.bfloat16: 1}
_INDEX_CODES = {torch.int32: 0, torch.int64: 1}


def _check_pool(pool):
    """(pages, kv_heads, head_dim, page_size) of a 4-bit pool."""
    shape = pool.shape
    if len(shape) != 4 or pool.dtype is not torch.uint8 or shape[3] not in (1280, 2560):
        raise ValueError("a 4-bit pool is uint8 [pages, kv_heads, page_size / 16, 20 * head_dim] with head_dim 64 or 128")
    pages, kv_heads, tiles, width = shape
    if kv_heads < 1 or tiles < 1:
        raise ValueError("a 4-bit pool has at least one KV head and one tile a page")
    if not pool.is_cuda:
        raise ValueError("the 4-bit cache needs a CUDA device")
    if not pool.is_contiguous() or pool.data_ptr() % 16:
        raise ValueError("a 4-bit pool must be contiguous and 16-byte aligned")
    return pages, kv_heads, width // 20, tiles * TILE_TOKENS


def _element_code(dtype):
    code = _ELEMENT_CODES.get(dtype)
    if code is None:
        raise ValueError("a 4-bit cache is written and read as float16 or bfloat16")
    return code


def _index_code(tensor, what):
    code = _INDEX_CODES.get(tensor.dtype)
    if code is None:
        raise ValueError(f"{what} must use an integer dtype")
    return code


def _enqueue(function, arguments, device):
    """One library call on the current stream of CUDA device number `device`, which is current meanwhile."""
    if torch.cuda.current_device() == device:
        status = function(*arguments, _cabi.raw_stream(device))
    else:
        with torch.cuda.device(device):
            status = function(*arguments, _cabi.raw_stream(device))
    if status:
        _cabi.check(status)


def empty_kv_pool_int4(num_pages, kv_heads, head_dim, *, page_size=16, device=None):
    """An uninitialised 4-bit pool for K and V; its rows are defined once they are written."""
    _require(head_dim in (64, 128), "head_dim must be 64 or 128")
    _require(page_size >= TILE_TOKENS and page_size % TILE_TOKENS == 0, "page_size must be a multiple of 16")
    return torch.empty((num_pages, kv_heads, page_size // TILE_TOKENS, 20 * head_dim), dtype=torch.uint8,
                       device="cuda" if device is None else device)


def empty_key_bounds_int4(kv4_pool, dtype):
    """Storage for the smallest and the largest key of every page: [pages, kv_heads, 2, D]."""
    _, kv_heads, dim, _ = _check_pool(kv4_pool)
    _element_code(dtype)
    return torch.empty((kv4_pool.shape[0], kv_heads, 2, dim), dtype=dtype, device=kv4_pool.device)


def _write(pool, geometry, pointers, strides, like, positions, slot_mapping, *, rows, q_heads, base, rope_table,
           valid_tokens=None):
    """Check what every write shares, fill qf_int4_write_args and enqueue on the current stream.
    `pointers` of q, k, v and q_out; `strides` of their rows, heads and channels, twelve numbers."""
    pages, kv_heads, dim, page_size = geometry
    device = pool.get_device()
    dtype = _element_code(like.dtype)
    position_at = position_stride = position_code = slot_at = slot_stride = slot_code = table_at = table_positions = valid_at = 0
    one_device = like.get_device() == device
    if positions is not None:
        one_device = one_device and positions.get_device() == device
        if positions.dtype is torch.float32 and rope_table is None:
            position_code = _cabi.INDEX_F32
        else:
            position_code = _index_code(positions, "positions")
        position_at = positions.data_ptr()
        position_stride, = positions.stride()
    if slot_mapping is not None:
        one_device = one_device and slot_mapping.get_device() == device
        slot_code = _index_code(slot_mapping, "slot mapping")
        slot_at = slot_mapping.data_ptr()
        slot_stride, = slot_mapping.stride()
    if rope_table is not None:
        shape = rope_table.shape
        table_positions, table_at = shape[0], rope_table.data_ptr()
        if (len(shape) != 3 or table_positions < 1 or shape[1] * 2 != dim or shape[2] != 2 or rope_table.dtype is not torch.float32
                or not rope_table.is_contiguous() or table_at % 16):
            raise ValueError("rope_table must be contiguous, 16-byte aligned float32 [positions, head_dim / 2, 2]")
        one_device = one_device and rope_table.get_device() == device
    if valid_tokens is not None:
        if valid_tokens.dtype is not torch.int32 or valid_tokens.numel() != 1 or valid_tokens.get_device() != device:
            raise ValueError("valid_tokens must be a CUDA int32 scalar")
        valid_at = valid_tokens.data_ptr()
    if not one_device:
        raise ValueError("the 4-bit cache write needs CUDA tensors of one device")
    args = _cabi.pack_int4_write(
        *pointers, *strides, position_at, position_stride, slot_at, slot_stride, table_at, pool.data_ptr(), pages, valid_at,
        rows, q_heads, kv_heads, dim, page_size, dtype, position_code, slot_code, table_positions, base)
    _enqueue(_cabi.library().qf_int4_rope_kv_write, (args,), device)


def packed_qkv_rope_cache_int4(
    packed, positions, slot_mapping, kv4_pool, *, q_heads=12, base=1_000_000.0, rope_table=None, valid_tokens=None,
):
    """packed_qkv_rope_cache for the 4-bit cache: packed (rows, (q_heads + 2 kv_heads) * D) -> q (rows, q_heads, D).

    Rotated K and V go to slot_mapping[row] (page * page_size + row in page; outside the pool: the
    row is skipped).  rope_table (positions, D / 2, 2) float32 (cos, sin) pairs; without it the
    angles are position * base^(-2i / D).  Rows at or beyond valid_tokens get zero queries and no
    cache write.  No two rows of a call may have the same slot."""
    if packed.ndim == 3:
        _require(packed.shape[1] == 1, "packed QKV must have one decode token per row")
        packed = packed[:, 0, :]
    geometry = _, kv_heads, dim, _ = _check_pool(kv4_pool)
    if q_heads < 1:
        raise ValueError("q_heads must be positive")
    shape = packed.shape
    if len(shape) != 2 or shape[1] != (q_heads + 2 * kv_heads) * dim:
        raise ValueError("expected packed QKV shape (rows, (q_heads + 2 * kv_heads) * head_dim)")
    rows = shape[0]
    if positions.shape != (rows,) or slot_mapping.shape != (rows,):
        raise ValueError("positions and slots must contain one value per row")
    q = torch.empty(rows, q_heads, dim, device=packed.device, dtype=packed.dtype)
    if rows == 0:
        return q
    row_stride, col_stride = packed.stride()
    segment = (row_stride, dim * col_stride, col_stride)
    at, head = packed.data_ptr(), 2 * dim * col_stride  # bytes from one head to the next
    _write(kv4_pool, geometry, (at, at + q_heads * head, at + (q_heads + kv_heads) * head, q.data_ptr()),
           (*segment, *segment, *segment, q_heads * dim, dim, 1), packed, positions, slot_mapping, rows=rows,
           q_heads=q_heads, base=base, rope_table=rope_table, valid_tokens=valid_tokens)
    return q


def _write_heads(q, k, v, positions, slot_mapping, kv4_pool, geometry, token_dim, rotate_q, base, rope_table):
    """The write of tensors whose tokens lie along `token_dim` and heads along dimension 1."""
    _require(k.dtype == v.dtype == q.dtype, "Q/K/V must share FP16 or BF16 dtype")
    _require(q.get_device() == k.get_device() == v.get_device(), "the 4-bit cache write needs CUDA tensors of one device")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if rotate_q else q
    strides = tuple(t.stride(n) for t in (q, k, v, out) for n in (token_dim, 1, 3))
    _write(kv4_pool, geometry, (q.data_ptr() if rotate_q else 0, k.data_ptr(), v.data_ptr(), out.data_ptr() if rotate_q else 0),
           strides, k, positions, slot_mapping, rows=k.shape[token_dim], q_heads=q.shape[1] if rotate_q else 0, base=base,
           rope_table=rope_table)
    return out


def native_decode_rope_kv_write_int4(
    q, k, v, positions, slot_mapping, kv4_pool, *, base=1_000_000.0, rope_table=None, rotate_q=True,
):
    """native_decode_rope_kv_write for the 4-bit cache: q (B, Hq, 1, D), k and v (B, Hkv, 1, D).
    Returns rotated Q (or q when rotate_q=False)."""
    _require(all(t.ndim == 4 and t.shape[2] == 1 for t in (q, k, v)),
             "decode Q/K/V must have shape (batch, heads, 1, dim)")
    geometry = _, kv_heads, dim, _ = _check_pool(kv4_pool)
    batch = q.shape[0]
    _require(k.shape == v.shape and k.shape == (batch, kv_heads, 1, dim) and q.shape[-1] == dim,
             "decode K/V shapes do not match Q and the pool")
    _require(positions.shape == (batch,) and slot_mapping.shape == (batch,),
             "positions and slots must contain one entry per batch row")
    return _write_heads(q, k, v, positions, slot_mapping, kv4_pool, geometry, 0, rotate_q, base, rope_table)


def rope_kv_write_int4(q, k, v, positions, slot_mapping, kv4_pool, *, base=1_000_000.0, rope_table=None):
    """rope_kv_write for the 4-bit cache: q (1, Hq, T, D), k and v (1, Hkv, T, D), one prompt or a
    packed chunk of several.  Returns rotated Q shaped like q."""
    _require(q.ndim == 4 and k.ndim == 4 and v.ndim == 4, "q, k, and v must be rank-four tensors")
    _require(q.shape[0] == 1 and k.shape[0] == 1 and v.shape[0] == 1,
             "packed q, k, and v must have batch dimension one")
    geometry = _, kv_heads, dim, _ = _check_pool(kv4_pool)
    tokens = q.shape[2]
    _require(k.shape == v.shape and k.shape == (1, kv_heads, tokens, dim) and q.shape[-1] == dim,
             "K/V shapes do not match Q and the pool")
    if positions.ndim == 2:
        _require(tuple(positions.shape) == (1, tokens), "positions must have shape (1, tokens)")
        positions = positions[0]
    _require(positions.shape == (tokens,) and slot_mapping.shape == (tokens,),
             "positions and slots must contain one entry per token")
    return _write_heads(q, k, v, positions, slot_mapping, kv4_pool, geometry, 2, True, base, rope_table)


def quantize_kv_pool_int4(k_pool, v_pool):
    """A 4-bit pool with the contents of fp16 / bf16 pools [pages, page_size, Hkv, D] (keys as they are:
    already rotated).  Every row of the pools is quantised; rows with a NaN or an infinity read back as NaN."""
    _require(k_pool.ndim == 4 and k_pool.shape == v_pool.shape and k_pool.is_contiguous() and v_pool.is_contiguous(),
             "K/V pools must be contiguous with matching rank-four shapes")
    pages, page_size, kv_heads, dim = k_pool.shape
    _require(k_pool.is_cuda and v_pool.device == k_pool.device, "K/V pools must share one CUDA device")
    pool = empty_kv_pool_int4(pages, kv_heads, dim, page_size=page_size, device=k_pool.device)
    _require(v_pool.dtype == k_pool.dtype, "K/V pools must share FP16 or BF16 dtype")
    step = max(1, MAX_ITEMS // (2 * kv_heads * (dim // 16) * page_size))  # pages a call has room for
    for first in range(0, pages, step):
        k, v, part = k_pool[first:first + step], v_pool[first:first + step], pool[first:first + step]
        _write(part, (part.shape[0], kv_heads, dim, page_size), (0, k.data_ptr(), v.data_ptr(), 0), (kv_heads * dim, dim, 1) * 4,
               k, None, None, rows=part.shape[0] * page_size, q_heads=0, base=1.0, rope_table=None)
    return pool


def _read(kv4_pool, slots, rows, dtype):
    """Rows at `slots` = (address, index code, stride) as K and V [rows, kv_heads, D]."""
    pages, kv_heads, dim, page_size = _check_pool(kv4_pool)
    code = _element_code(dtype)
    k = torch.empty(rows, kv_heads, dim, dtype=dtype, device=kv4_pool.device)
    v = torch.empty_like(k)
    _enqueue(_cabi.library().qf_int4_read_rows,
             (kv4_pool.data_ptr(), pages, page_size, kv_heads, dim, code, *slots, rows, k.data_ptr(), v.data_ptr()),
             kv4_pool.get_device())
    return k, v


def read_kv_int4(kv4_pool, slot_mapping, *, dtype=None):
    """Rows of the cache at a list of slots as (k, v), both [n, Hkv, D] in `dtype`, that of the writes,
    which the pool does not hold: steps and floors read as another type are other numbers (default
    float16).  A slot outside the pool, -1 for one, gives a row of zeros."""
    shape = slot_mapping.shape
    if len(shape) != 1:
        raise ValueError("slot mapping must be a list of slots")
    if slot_mapping.get_device() != kv4_pool.get_device():
        raise ValueError("pool and slots must share one CUDA device")
    slots = (slot_mapping.data_ptr(), _index_code(slot_mapping, "slot mapping"), *slot_mapping.stride())
    return _read(kv4_pool, slots, shape[0], torch.float16 if dtype is None else dtype)


def dequantize_kv_pool_int4(kv4_pool, dtype=None):
    """The whole cache as 16-bit pools (k_pool, v_pool), both [pages, page_size, Hkv, D], in `dtype`: that
    of the writes, as for read_kv_int4."""
    pages, kv_heads, dim, page_size = _check_pool(kv4_pool)
    k, v = _read(kv4_pool, (None, 0, 0), pages * page_size, torch.float16 if dtype is None else dtype)
    shape = (pages, page_size, kv_heads, dim)
    return k.view(shape), v.view(shape)


# scratch bytes by call, device and sizes: what qf_paged_int4_workspace answers is a function of these
_workspace_sizes = {}

_PAGED_DEVICE = "queries, pool, key bounds, page table and lengths must share one CUDA device"


def _run(function, call, device, batch, geometry, dtype, block_table, seq_lens, per_head, q, out, pool, bounds, choice, new_tokens,
         take, scale):
    """Check table and lengths, fill qf_paged_int4_args, add the scratch of `call` (None: it has none) and
    enqueue.  The scratch is a torch allocation, so it is the stream's, and a captured graph's own."""
    pages, kv_heads, dim, page_size = geometry
    t_shape = block_table.shape
    if per_head and len(t_shape) == 3:
        if t_shape[0] != batch or t_shape[1] != kv_heads or seq_lens.shape != (batch, kv_heads):
            raise ValueError("a table and lengths per KV head have shapes [batch, kv_heads, pages] and [batch, kv_heads]")
        t_sb, t_sh, t_sp = block_table.stride()
        l_sb, l_sh = seq_lens.stride()
        width = t_shape[2]
    else:
        if len(t_shape) != 2 or t_shape[0] != batch or seq_lens.shape != (batch,):
            raise ValueError("batch dimensions must match")
        t_sb, t_sp = block_table.stride()
        l_sb, = seq_lens.stride()
        t_sh = l_sh = 0
        width = t_shape[1]
    if block_table.get_device() != device or seq_lens.get_device() != device:
        raise ValueError(_PAGED_DEVICE)
    q_at = o_at = pages_at = held_at = q_heads = q_sb = q_sh = o_sb = scratch_at = scratch_bytes = 0
    if q is not None:
        q_at, q_heads = q.data_ptr(), q.shape[1]
        q_sb, q_sh, _ = q.stride()
    if out is not None:
        o_at, o_sb = out.data_ptr(), q_heads * dim
    if choice is not None:
        pages_at, held_at = choice[0].data_ptr(), choice[1].data_ptr()

    def fill():
        return _cabi.pack_paged_int4(
            q_at, o_at, 0 if pool is None else pool.data_ptr(), 0 if bounds is None else bounds.data_ptr(),
            block_table.data_ptr(), seq_lens.data_ptr(), scratch_at, pages_at, held_at, q_sb, q_sh, o_sb, dim, t_sb, t_sh, t_sp,
            l_sb, l_sh, pages, width, scratch_bytes, batch, q_heads, kv_heads, dim, page_size, dtype,
            _index_code(block_table, "page table"), _index_code(seq_lens, "lengths"), new_tokens, take, scale)

    if call is not None:
        key = (call, device, batch, q_heads, kv_heads, dim, page_size, width, take)
        scratch_bytes = _workspace_sizes.get(key)
        if scratch_bytes is None:
            scratch_bytes, size = 0, ctypes.c_int64()
            with torch.cuda.device(device):
                _cabi.check(_cabi.library().qf_paged_int4_workspace(fill(), call, ctypes.byref(size)))
            if len(_workspace_sizes) >= 4096:
                _workspace_sizes.clear()
            scratch_bytes = _workspace_sizes[key] = size.value
        if scratch_bytes:
            scratch = torch.empty(scratch_bytes, dtype=torch.uint8, device=block_table.device)
            scratch_at = scratch.data_ptr()
    _enqueue(function, (fill(),), device)


def _check_query(q, geometry):
    """q as the kernels take it: unit inner stride, rows on 16-byte boundaries."""
    _, kv_heads, dim, _ = geometry
    shape = q.shape
    if len(shape) != 3 or shape[1] < 1 or shape[2] != dim:
        raise ValueError("q must have shape [batch, query_heads, head_dim]")
    if shape[1] % kv_heads:
        raise ValueError("query heads must be divisible by KV heads")
    if shape[1] > MAX_GROUP * kv_heads:
        raise ValueError("at most 16 query heads share a KV head")
    row, head, inner = q.stride()
    if inner != 1 or row % 8 or head % 8 or q.data_ptr() % 16:
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
    geometry = _check_pool(kv4_pool)
    dtype = _element_code(q.dtype)
    q = _check_query(q, geometry)
    device = kv4_pool.get_device()
    if q.get_device() != device:
        raise ValueError(_PAGED_DEVICE)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _run(_cabi.library().qf_int4_decode_attention, _cabi.INT4_ATTENTION, device, q.shape[0], geometry, dtype, block_table, seq_lens,
         True, q, out, kv4_pool, None, None, 0, 0, geometry[2] ** -0.5 if scale is None else scale)
    return out


def _check_bounds(bounds, dtype, geometry=None):
    """Key bounds of a pool's geometry (default: any)."""
    shape = bounds.shape
    if (len(shape) != 4 or shape[2] != 2 or shape[3] not in (64, 128) or bounds.dtype != dtype or not bounds.is_contiguous()
            or bounds.data_ptr() % 16):
        raise ValueError("key bounds must be contiguous [pages, kv_heads, 2, head_dim] in the queries' dtype")
    if not bounds.is_cuda:
        raise ValueError("key bounds must be on a CUDA device")
    if geometry is not None and (shape[0] != geometry[0] or shape[1] != geometry[1] or shape[3] != geometry[2]):
        raise ValueError("key bounds do not match the pool")


def update_key_bounds_int4(kv4_pool, key_bounds, block_table, seq_lens, *, new_tokens=1):
    """Recompute key_bounds for the pages that hold one of the last new_tokens tokens of each sequence
    (1 after a decode step, the prompt's length after a prefill); returns key_bounds.

    Bounds are the smallest and the largest key of a page's tokens below seq_lens, per channel, as the
    cache reads back.  Sequences that share a page hold the same number of its tokens: one that holds
    more might find the bounds of fewer."""
    geometry = _check_pool(kv4_pool)
    dtype = _element_code(key_bounds.dtype)
    _check_bounds(key_bounds, key_bounds.dtype, geometry)
    _require(isinstance(new_tokens, int) and not isinstance(new_tokens, bool) and 0 <= new_tokens < 2 ** 31,
             "new_tokens must be a non-negative integer")
    device = kv4_pool.get_device()
    _require(key_bounds.get_device() == device, _PAGED_DEVICE)
    _run(_cabi.library().qf_int4_key_bounds, None, device, block_table.shape[0], geometry, dtype, block_table, seq_lens, False,
         None, None, kv4_pool, key_bounds, None, new_tokens, 0, 0.0)
    return key_bounds


def _check_take(num_pages, rows, page_size):
    """Before the choice is allocated: a row of it holds fewer than 2^30 tokens, all rows fewer than 2^30 tiles."""
    _require(isinstance(num_pages, int) and not isinstance(num_pages, bool) and 1 <= num_pages, "num_pages must be a positive integer")
    _require(num_pages < 2 ** 30 // page_size and rows * num_pages < 2 ** 30 // (page_size // TILE_TOKENS),
             "num_pages is too large: a choice holds fewer than 2^30 tokens a row and 2^30 tiles of 16 in all")


def _empty_choice(batch, kv_heads, num_pages, device):
    return (torch.empty(batch, kv_heads, num_pages, dtype=torch.int32, device=device),
            torch.empty(batch, kv_heads, dtype=torch.int32, device=device))


def select_kv_pages(q, key_bounds, block_table, seq_lens, *, num_pages, page_size=16):
    """The pages each sequence's queries attend, per KV head: (page_table int32 [B, Hkv, num_pages],
    page_lens int32 [B, Hkv]), a table and lengths for paged_decode_attention_int4.

    A row is the sequence's newest page and the num_pages - 1 others with the highest bound on a score,
    the largest over the KV head's query heads of sum_d max(q_d * low_d, q_d * high_d); ties go to the
    earlier page.  Pages keep the sequence's order; -1 pads a sequence that has fewer.  page_size is the
    pool's, kv4_pool.shape[2] * 16: the bounds do not hold it, and with another one every length is cut
    into other pages."""
    dtype = _element_code(q.dtype)
    _check_bounds(key_bounds, q.dtype)
    _require(page_size >= TILE_TOKENS and page_size % TILE_TOKENS == 0, "page_size must be a multiple of 16")
    pages, kv_heads, _, dim = key_bounds.shape
    geometry = (pages, kv_heads, dim, page_size)
    q = _check_query(q, geometry)
    _check_take(num_pages, q.shape[0] * kv_heads, page_size)
    device = key_bounds.get_device()
    _require(q.get_device() == device, _PAGED_DEVICE)
    choice = _empty_choice(q.shape[0], kv_heads, num_pages, q.device)
    _run(_cabi.library().qf_select_kv_pages, _cabi.INT4_SELECT, device, q.shape[0], geometry, dtype, block_table, seq_lens, False,
         q, None, None, key_bounds, choice, 0, num_pages, 0.0)
    return choice


def sparse_decode_attention_int4(q, kv4_pool, key_bounds, block_table, seq_lens, *, num_pages, scale=None):
    """select_kv_pages and paged_decode_attention_int4 over its choice in one call: (out, page_table,
    page_lens).  key_bounds must be up to date for every page but a sequence's newest.  The pages are
    those of the largest q . k, so scale is not negative."""
    geometry = _check_pool(kv4_pool)
    _require(scale is None or scale >= 0, "scale must not be negative: pages are chosen by their largest scores")
    dtype = _element_code(q.dtype)
    _check_bounds(key_bounds, q.dtype, geometry)
    q = _check_query(q, geometry)
    _check_take(num_pages, q.shape[0] * geometry[1], geometry[3])
    device = kv4_pool.get_device()
    _require(q.get_device() == device and key_bounds.get_device() == device, _PAGED_DEVICE)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    choice = _empty_choice(q.shape[0], geometry[1], num_pages, q.device)
    _run(_cabi.library().qf_int4_sparse_decode_attention, _cabi.INT4_SPARSE, device, q.shape[0], geometry, dtype, block_table,
         seq_lens, False, q, out, kv4_pool, key_bounds, choice, 0, num_pages, geometry[2] ** -0.5 if scale is None else scale)
    return out, *choice

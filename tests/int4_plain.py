"""The 4-bit paged cache from its definitions, on the CPU: codec and layout channel by channel,
attention and page choice in 64 bits.  What the GPU tests compare with."""

from __future__ import annotations

import math

import torch

GROUP, TILE = 32, 16


def places(dim):
    """(byte, shift) of K code [token, channel] and of V code, and byte of K step [token, group], in a tile."""
    token, ch = torch.arange(TILE)[:, None], torch.arange(dim)[None, :]
    w = dim // GROUP
    group, inner, shift = ch // GROUP, ch % GROUP, ch % 2 * 4
    k = token * (dim // 2) + inner // 8 * 4 * w + group * 4 + inner % 8 // 2
    v = 8 * dim + token // 2 * dim + inner // 4 * 4 * w + group * 4 + token % 2 * 2 + inner % 4 // 2
    step = 16 * dim + token * 2 * w + 2 * torch.arange(w)[None, :]
    return k, v, shift.expand(TILE, dim), step


def encode(x):
    """[..., D] in fp16 / bf16 -> codes [..., D] int64, step and floor [..., D / 32] in the same type."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    step = ((high - low) / torch.full_like(low, 15.0)).to(x.dtype).float()
    step = torch.where(step < 2.0 ** -60, torch.zeros_like(step), step)
    bad = ~torch.isfinite(g).all(-1)
    nan = torch.full_like(low, math.nan)
    step, low = torch.where(bad, nan, step), torch.where(bad, nan, low)
    n = torch.round((g - low[..., None]) / torch.where(step > 0, step, torch.ones_like(step))[..., None])
    n = torch.where((step > 0)[..., None], n.clamp(0, 15), torch.zeros_like(n))
    return n.flatten(-2).long(), step.to(x.dtype), low.to(x.dtype)


def decode(codes, step, low):
    """float32 values: one rounding of code * step + floor."""
    n = codes.unflatten(-1, (-1, GROUP)).double()
    return (n * step.double()[..., None] + low.double()[..., None]).float().flatten(-2)


def store(pool, slots, k, v):
    """Quantise rows [n, heads, D] into a CPU pool at their slots (out-of-range slots skipped)."""
    dim, per_page = pool.shape[3] // 20, pool.shape[2]
    page_size = per_page * TILE
    kb, vb, shift, pb = places(dim)
    sides = [(kb, 0, encode(k)), (vb, 2, encode(v))]
    for row, slot in enumerate(slots.tolist()):
        if not 0 <= slot < pool.shape[0] * page_size:
            continue
        page, inside = divmod(slot, page_size)
        tile, t = pool[page, :, inside // TILE], inside % TILE  # [heads, bytes]
        for where, which, (codes, step, low) in sides:
            low_half, high_half = codes[row][:, 0::2], codes[row][:, 1::2]
            tile[:, where[t][0::2]] = (low_half | high_half << 4).to(torch.uint8)
            for offset, values in ((which, step), (which + 1, low)):
                raw = values[row].contiguous().view(torch.uint8).view(values.shape[1], -1, 2)
                for byte in range(2):
                    tile[:, pb[t] + dim * offset + byte] = raw[:, :, byte]


def rows(pool, dtype):
    """The whole cache as float32 K, V [pages, page_size, heads, D]."""
    dim = pool.shape[3] // 20
    kb, vb, shift, pb = places(dim)
    flat = pool.reshape(-1, 20 * dim)
    out = []
    for where, which in ((kb, 0), (vb, 2)):
        codes = (flat[:, where].long() >> shift) & 15
        params = flat[:, 16 * dim:].contiguous().view(dtype).view(-1, 4, TILE, dim // GROUP)
        x = decode(codes, params[:, which], params[:, which + 1])
        x = x.view(pool.shape[0], pool.shape[1], pool.shape[2] * TILE, dim)
        out.append(x.transpose(1, 2).contiguous())
    return out


def rope(x, table, positions):
    """x [n, heads, D]: separate fp32 products, one rounding."""
    cs = table[positions.long()][:, None]
    a, b = x.float().chunk(2, -1)
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def rope_table(positions, dim, base=1e6):
    inv = base ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def attention(q, k, v, table, lens, scale=None):
    """64-bit attention of q [B, Hq, D] over CPU float pools [pages, page, heads, D]; table [B, n] or
    [B, heads, n].  Pages outside the pool read as zeros.  Returns (out float64, largest |v| a row)."""
    batch, hq, dim = q.shape
    pages, page, heads = k.shape[:3]
    scale = dim ** -0.5 if scale is None else scale
    out, top = torch.zeros(batch, hq, dim, dtype=torch.float64), torch.zeros(batch, hq, 1, dtype=torch.float64)
    for b in range(batch):
        for h in range(heads):
            row, n = (table[b], lens[b]) if table.ndim == 2 else (table[b, h], lens[b, h])
            n = min(max(int(n), 0), row.shape[0] * page)
            if n == 0:
                continue
            ids = row[: -(-n // page)].long()
            ok = ((ids >= 0) & (ids < pages))[:, None, None]
            kk, vv = (torch.where(ok, x[ids.clamp(0, pages - 1), :, h], torch.zeros(())).flatten(0, 1)[:n].double()
                      for x in (k, v))
            mine = slice(h * (hq // heads), (h + 1) * (hq // heads))
            p = torch.softmax(q[b, mine].double() @ kk.T * scale, -1)
            out[b, mine] = p @ vv
            top[b, mine] = vv.abs().max()
    return out, top


def assert_attention(actual, expected, top):
    """|out - exact| <= half a step of the output's type, of the exact value, plus 2^-9 of the row's
    largest |v|: a weight p * step is rounded to fp16 at worst (2^-11 of it, times a code up to 15, so
    2^-11 of a group's range, at most 2 max|v|), which is 2^-10; the fp32 sums, exponentials and the
    score's own rounding get as much again."""
    half = torch.finfo(actual.dtype).eps / 2
    error = (actual.double().cpu() - expected).abs()
    allowed = half * expected.abs() + 2.0 ** -9 * top + 1e-30
    assert torch.isfinite(actual).all()
    worst = (error / allowed).max().item() if error.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} of the tolerance"


def bounds(k, table, lens, dtype, new, into):
    """Key bounds of the pages that hold the last `new` tokens, in place into [pages, heads, 2, D]."""
    page = k.shape[1]
    for b in range(table.shape[0]):
        n = min(max(int(lens[b]), 0), table.shape[1] * page)
        for i in range(max(0, n - new) // page, -(-n // page)):
            ident = int(table[b, i])
            if 0 <= ident < k.shape[0] and new > 0:
                mine = k[ident, : min(page, n - i * page)].to(dtype)
                into[ident, :, 0], into[ident, :, 1] = mine.amin(0), mine.amax(0)
    return into


def select(q, limits, table, lens, take, page):
    """(page_table [B, heads, take], page_lens [B, heads]): fp32 scores, pairwise sums."""
    batch, hq, dim = q.shape
    heads = limits.shape[1]
    out = torch.full((batch, heads, take), -1, dtype=torch.int32)
    held = torch.zeros(batch, heads, dtype=torch.int32)
    for b in range(batch):
        n = min(max(int(lens[b]), 0), table.shape[1] * page)
        count = -(-n // page)
        ids = table[b, :count].long()
        for h in range(heads):
            if count <= take:
                chosen = torch.arange(count)
            else:
                x = q[b, h * (hq // heads):(h + 1) * (hq // heads)].float()[:, None]
                ok = (ids >= 0) & (ids < limits.shape[0])
                low, high = limits[ids.clamp(0, limits.shape[0] - 1), h].float().unbind(1)
                terms = torch.maximum(x * low, x * high)
                while terms.shape[-1] > 1:
                    terms = terms[..., 0::2] + terms[..., 1::2]
                score = terms[..., 0].amax(0)
                score = torch.where(torch.isnan(score), math.inf, score).masked_fill(~ok, -math.inf)[:-1]
                best = torch.sort(score, descending=True, stable=True).indices[: take - 1].sort().values
                chosen = torch.cat([best, torch.tensor([count - 1])])
            out[b, h, : len(chosen)] = ids[chosen].int()
            held[b, h] = n - (count - len(chosen)) * page
    return out, held


def make_cache(lengths, *, dtype=torch.float16, dim=128, heads=2, group=6, page=16, seed=0, extra=2, poison=True,
               gain=1.0, pad=-1):
    """q, CPU pool, table, lens: pages in random order, rows with channel offsets; what no sequence holds is
    codes of 15 with NaN steps and floors (poison)."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + extra
    pool = torch.zeros(pages, heads, page // TILE, 20 * dim, dtype=torch.uint8)
    if poison:
        pool[..., : 16 * dim] = 255
        pool[..., 16 * dim:].view(dtype).fill_(math.nan)
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lengths), max([1, *counts])), pad, dtype=torch.int32)
    slots, at = [], 0
    for b, (n, c) in enumerate(zip(lengths, counts)):
        table[b, :c] = order[at:at + c].int()
        slots.append((table[b, :c].long()[:, None] * page + torch.arange(page)).flatten()[:n])
        at += c
    slots = torch.cat(slots) if slots else torch.zeros(0, dtype=torch.long)
    offset = torch.randn(heads, dim, generator=g) * 0.5
    offset[:, 7] += 6
    k = (torch.randn(len(slots), heads, dim, generator=g) * 0.5 + offset).to(dtype)
    v = (torch.randn(len(slots), heads, dim, generator=g) * gain).to(dtype)
    store_fast(pool, slots, k, v)
    q = (torch.randn(len(lengths), heads * group, dim, generator=g)).to(dtype)
    return q, pool, table, torch.tensor(lengths, dtype=torch.int32)


def store_fast(pool, slots, k, v):
    """store() for many rows: the same places, all rows at once."""
    dim, heads, per_page = pool.shape[3] // 20, pool.shape[1], pool.shape[2]
    kb, vb, _, pb = places(dim)
    tile = (slots // (per_page * TILE))[:, None] * heads * per_page + torch.arange(heads) * per_page \
        + (slots // TILE % per_page)[:, None]
    base, t = (tile * 20 * dim)[..., None], slots % TILE
    flat = pool.view(-1)
    for where, which, (codes, step, low) in ((kb, 0, encode(k)), (vb, 2, encode(v))):
        flat[base + where[t][:, None, 0::2]] = (codes[..., 0::2] | codes[..., 1::2] << 4).to(torch.uint8)
        for offset, values in ((which, step), (which + 1, low)):
            raw = values.contiguous().view(torch.uint8).view(*values.shape, 2)
            for byte in range(2):
                flat[base + pb[t][:, None] + dim * offset + byte] = raw[..., byte]

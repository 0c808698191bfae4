"""Operators of the 4-bit paged KV cache: what they compute, in plain torch, and the sizes they run at.

The cache.  kv4_pool is uint8 [pages, kv_heads, page_size / 16, 20 * D]: tiles of 16 tokens of one KV head, K and V
side by side.  Every 32 consecutive channels of a token's row are a group with a step and a floor, both in the type of
the queries (fp16 or bf16); a channel is a code 0..15 and stands for code * step + floor.  Bytes of a tile, W = D / 32:
    [0, 8D)     K codes [16 tokens][4][W][4 bytes]: byte y of (t, w) holds channels 32w + 8t + 2y (low), + 2y + 1 (high)
    [8D, 16D)   V codes [8 token pairs][8][W][2 tokens][2 bytes]: byte y of (g, w) holds channels 32w + 4g + 2y, + 2y + 1
    [16D, 20D)  K steps [16][W], K floors [16][W], V steps [16][W], V floors [16][W], 16 bits each
Token p of a sequence lives in page table[p // page_size], tile (p % page_size) // 16, row p % 16.

The operators.
    write      RoPE on Q and K, K and V into the cache at their slots (and read back: the values the codes stand for)
    read       rows of the cache at a list of slots, as 16-bit K and V
    attention  one query token a sequence over its pages, grouped heads
    bounds     smallest and largest K of every page and channel, for the pages the newest tokens touched
    sparse     bounds of the newest page, the pages a query is to attend by an upper bound of their scores, and the
               attention over those: per sequence and KV head, the newest page always among them
"""
import math
import random

import torch

own = False

GROUP = 32


# ------------------------------------------------------------------ cases
def listed():
    qwen = dict(q_heads=12, kv_heads=2, dim=128, page=16)
    return [
        # a decode step of 64 sequences: the new token's row of each
        dict(name="write_b64", op="write", rows=64, dtype="fp16", **qwen),
        # a chunk of a long prompt
        dict(name="write_chunk8192", op="write", rows=8192, dtype="bf16", **qwen),
        # a short prefix read back for a chunk's dense attention, with padded rows, another head layout
        dict(name="read_1501", op="read", rows=1501, dtype="bf16", q_heads=16, kv_heads=4, dim=64, page=32),
        # four prompts of 32768 tokens read back
        dict(name="read_131072", op="read", rows=131072, dtype="fp16", **qwen),
        # one short chat: latency
        dict(name="attn_b1_513", op="attention", batch=1, low=513, high=513, dtype="fp16", **qwen),
        # the decode batch of 64, contexts uniform in [128, 4096]
        dict(name="attn_b64", op="attention", batch=64, low=129, high=4097, dtype="fp16", **qwen),
        # a few sequences, one of them very long
        dict(name="attn_skew_b4", op="attention", batch=4, low=513, high=32769, dtype="bf16", **qwen),
        # many sequences of a model with 64 channels a head, four query heads a KV head
        dict(name="attn_b256_d64", op="attention", batch=256, low=64, high=4096, dtype="bf16", q_heads=16, kv_heads=4, dim=64, page=32),
        # after a step: the page of each sequence's newest token
        dict(name="bounds_b64_new1", op="bounds", batch=64, low=129, high=4097, new=1, dtype="fp16", **qwen),
        # after a prompt: every page of it
        dict(name="bounds_prompt", op="bounds", batch=16, low=4096, high=8192, new=8192, dtype="bf16", q_heads=12, kv_heads=2, dim=128, page=64),
        # one long document: 64 of its 2048 pages
        dict(name="sparse_b1_32769", op="sparse", batch=1, low=32769, high=32769, take=64, dtype="fp16", **qwen),
        # a batch of long documents, pages of 64 tokens, a sixteenth or more of them attended
        dict(name="sparse_b32_p64", op="sparse", batch=32, low=8192, high=32768, take=32, dtype="bf16", q_heads=12, kv_heads=2, dim=128, page=64),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kv_heads, group, dim = rng.choice([(2, 6, 128), (4, 4, 64), (1, 8, 128), (8, 1, 64), (2, 7, 128), (4, 3, 128), (1, 16, 64)])
    case = dict(op=rng.choice(["write", "read", "attention", "attention", "bounds", "sparse"]), dtype=rng.choice(["fp16", "bf16"]),
                q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64]))
    if case["op"] == "write":
        case["rows"] = _log(rng, 1, 8192 * 256 // (kv_heads * dim))
    elif case["op"] == "read":
        case["rows"] = _log(rng, 1, 131072 * 256 // (kv_heads * dim))
    else:
        most = 200_000 * 256 // (kv_heads * dim)  # tokens of the whole batch
        case["batch"] = _log(rng, 1, 256)
        case["high"] = _log(rng, 2, min(32768, most // case["batch"]))
        case["low"] = rng.randint(1, case["high"])
        if case["op"] == "bounds":
            case["new"] = rng.choice([1, 1, 17, case["high"]])
        if case["op"] == "sparse":
            case["take"] = _log(rng, 1, 128)
    return case


def _lengths(case):
    """The sequences' lengths: the longest, the shortest, and others spread between them."""
    rng = random.Random("%d %d %d" % (case["batch"], case["low"], case["high"]))
    if case["batch"] <= 4:  # 32769, 16385, 4097, 513: a geometric fall
        ratio = case["low"] / case["high"]
        return [max(1, round(case["high"] * ratio ** (i / max(1, case["batch"] - 1)))) for i in range(case["batch"])]
    return [case["high"], case["low"]] + [rng.randint(case["low"], case["high"]) for _ in range(case["batch"] - 2)]


def _pages(case):
    return [-(-n // case["page"]) for n in _lengths(case)]


def work(case):
    hq, hkv, d, p = case["q_heads"], case["kv_heads"], case["dim"], case["page"]
    row4, row16 = 2 * hkv * (d // 2 + d // 8), 2 * hkv * d * 2  # bytes of a token's K and V in 4 and in 16 bits
    if case["op"] == "write":
        r = case["rows"]
        return {"bytes": r * ((2 * hq + 2 * hkv) * d * 2 + 2 * row4 + row16 + 4 * d + 20), "flops": r * (hq + 6 * hkv) * d * 3}
    if case["op"] == "read":
        return {"bytes": case["rows"] * (row4 + row16 + 8), "flops": case["rows"] * 4 * hkv * d}
    lens = _lengths(case)
    ends = case["batch"] * hq * d * 2 * 2  # q and out
    if case["op"] == "attention":
        return {"bytes": sum(lens) * row4 + ends + 4 * sum(_pages(case)), "flops": 4 * sum(lens) * hq * d}
    bound = 2 * hkv * d * 2  # bytes of a page's bounds
    if case["op"] == "bounds":
        pages = [(n - 1) // p - max(0, n - case["new"]) // p + 1 for n in lens]
        tokens = [n - max(0, n - case["new"]) // p * p for n in lens]
        return {"bytes": sum(tokens) * row4 // 2 + sum(pages) * (bound + 4), "flops": 4 * sum(tokens) * hkv * d}
    last = [n - (n - 1) // p * p for n in lens]  # tokens of the newest page
    seen = [min(case["take"] - 1, (n - 1) // p) * p + t for n, t in zip(lens, last)]
    scored = sum(n if n > case["take"] else 0 for n in _pages(case))
    return {"bytes": sum(last) * row4 // 2 + len(lens) * bound + scored * (bound + 4) + sum(seen) * row4 + ends,
            "flops": scored * hq * d * 4 + 4 * sum(seen) * hq * d}


# ------------------------------------------------------------------ inputs
def _dtype(case):
    return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rows(case, g, n, heads):
    """Rows as a projection with a bias gives them: N(0, 1/2) and channels with an offset, a few of them large."""
    offset = _randn(g, heads, case["dim"]) * 0.25
    offset[:, 5] += 4.0
    offset[:, case["dim"] - 3] -= 6.0
    return (_randn(g, n, heads, case["dim"]) * 0.5 + offset).to(_dtype(case))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    d, hq, hkv, page, dt = case["dim"], case["q_heads"], case["kv_heads"], case["page"], _dtype(case)
    state = dict(case=case, op=case["op"], page=page, dtype=dt, dim=d, q_heads=hq, kv_heads=hkv)
    if case["op"] in ("write", "read"):
        rows = case["rows"]
        pages = rows // page + 3
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:rows]
        pool = torch.zeros(pages, hkv, page // 16, 20 * d, dtype=torch.uint8, device="cuda")
        state.update(pool=pool, slots=slots)
        if case["op"] == "read":
            every = torch.arange(pages * page, device="cuda")
            _store(pool, every, _rows(case, g, pages * page, hkv), _rows(case, g, pages * page, hkv), page)
            slots[rows // 2::97] = -1  # rows that pad the list
            return state
        packed = torch.cat([_rows(case, g, rows, hq), _rows(case, g, rows, hkv), _rows(case, g, rows, hkv)], 1)
        start = int(torch.randint(0, 20000, (1,), generator=g, device="cuda"))
        positions = (torch.arange(rows, device="cuda") + start).int()
        inv = 1e6 ** (-torch.arange(d // 2, dtype=torch.float64, device="cuda") / (d // 2))
        angle = torch.arange(start + rows, dtype=torch.float64, device="cuda")[:, None] * inv
        table = torch.stack([angle.cos(), angle.sin()], -1).float()
        state.update(packed=packed.view(rows, -1), positions=positions, rope=table)
        return state
    lens = _lengths(case)
    counts = _pages(case)
    pages = sum(counts) + 5
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.zeros(len(lens), max(counts), dtype=torch.int32)
    place = torch.zeros(len(lens), max(counts), dtype=torch.bool)
    for b, n in enumerate(counts):
        place[b, :n] = True
    table = table.cuda()
    table[place.cuda()] = order[: sum(counts)]
    pool = torch.empty(pages, hkv, page // 16, 20 * d, dtype=torch.uint8, device="cuda")
    every = torch.arange(pages * page, device="cuda")
    _store(pool, every, _rows(case, g, pages * page, hkv), _rows(case, g, pages * page, hkv), page)
    state.update(pool=pool, table=table, lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if case["op"] != "bounds":
        state["q"] = _rows(case, g, len(lens), hq)
    if case["op"] != "attention":
        state["bounds"] = torch.zeros(pages, hkv, 2, d, dtype=dt, device="cuda")
        state["new"], state["take"] = case.get("new", 1), case.get("take")
    if case["op"] == "sparse":
        _bounds(state, max(lens))
    return state


# ------------------------------------------------------------------ the framework's calls
def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _own(s):
    ops = _package()
    if s["op"] == "write":
        q = ops.packed_qkv_rope_cache_int4(s["packed"], s["positions"], s["slots"], s["pool"], q_heads=s["q_heads"], rope_table=s["rope"])
        k, v = ops.read_kv_int4(s["pool"], s["slots"], dtype=s["dtype"])
        return {"q": q, "k": k, "v": v}
    if s["op"] == "read":
        k, v = ops.read_kv_int4(s["pool"], s["slots"], dtype=s["dtype"])
        return {"k": k, "v": v}
    if s["op"] == "attention":
        return ops.paged_decode_attention_int4(s["q"], s["pool"], s["table"], s["lens"])
    ops.update_key_bounds_int4(s["pool"], s["bounds"], s["table"], s["lens"], new_tokens=s["new"])
    if s["op"] == "bounds":
        return s["bounds"]
    out, table, lens = ops.sparse_decode_attention_int4(s["q"], s["pool"], s["bounds"], s["table"], s["lens"], num_pages=s["take"])
    return {"out": out, "pages": table, "lens": lens}


# ------------------------------------------------------------------ the plain form
def _quantize(x):
    """[n, heads, D] -> codes uint8 [n, heads, D], step and floor [n, heads, D / 32] in x's type.  The quotients are true
    divisions: in bf16 many of them lie just between two codes, and a rounded reciprocal would tip those either way."""
    g = x.float().unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1), g.amax(-1)
    step = ((high - low) / torch.full_like(low, 15.0)).to(x.dtype).float()
    step = torch.where(step < 2.0 ** -60, torch.zeros_like(step), step)
    codes = torch.round((g - low[..., None]) / torch.where(step > 0, step, torch.ones_like(step))[..., None])
    codes = torch.where(step[..., None] > 0, codes.clamp(0, 15), torch.zeros_like(codes))
    return codes.flatten(-2).to(torch.uint8), step.to(x.dtype), low.to(x.dtype)


def _store(pool, slots, k, v, page):
    """K and V rows [n, heads, D] into the cache at their slots."""
    n, heads, d = k.shape
    w = d // GROUP
    where, tile, token = slots // page, slots % page // 16, slots % 16
    flat = pool.view(-1)
    base = ((where[:, None] * heads + torch.arange(heads, device=pool.device)) * (page // 16) + tile[:, None]) * (20 * d)
    ar = lambda m: torch.arange(m, device=pool.device)  # noqa: E731
    codes, step, low = _quantize(k)
    c = codes.view(n, heads, w, 4, 4, 2).transpose(2, 3)  # [t][w][byte][nibble]
    at = base[..., None] + token[:, None, None] * (d // 2) + ar(d // 2)
    flat[at.reshape(-1)] = (c[..., 0] | c[..., 1] << 4).reshape(-1)
    v_codes, v_step, v_low = _quantize(v)
    params = torch.stack([step, low, v_step, v_low], 2).view(torch.uint8)  # [n, heads, 4, 2 W]
    at = (base[..., None] + 16 * d + token[:, None, None] * (2 * w))[..., None] + d * ar(4)[:, None] + ar(2 * w)
    flat[at.reshape(-1)] = params.reshape(-1)
    c = v_codes.view(n, heads, w, 8, 2, 2).transpose(2, 3)  # [g][w][byte][nibble]
    at = base[..., None] + 8 * d + (token // 2)[:, None, None] * d + (token % 2)[:, None, None] * 2
    at = at[..., None] + (4 * ar(8 * w))[:, None] + ar(2)
    flat[at.reshape(-1)] = (c[..., 0] | c[..., 1] << 4).reshape(-1)


def _values(tiles, dtype):
    """uint8 [..., 20 D] -> K, V float32 [..., 16, D]"""
    d = tiles.shape[-1] // 20
    w = d // GROUP
    lead = tiles.shape[:-1]
    kc, vc, par = tiles.split([8 * d, 8 * d, 4 * d], -1)
    par = par.contiguous().view(dtype).float().view(*lead, 4, 16, w, 1)
    nibbles = lambda c: torch.stack([c & 15, c >> 4], -1)  # noqa: E731
    kc = nibbles(kc).view(*lead, 16, 4, w, 8).transpose(-3, -2).reshape(*lead, 16, w, GROUP).float()
    vc = nibbles(vc).view(*lead, 8, 8, w, 2, 4)
    vc = vc.movedim(-2, -4).transpose(-3, -2).reshape(*lead, 16, w, GROUP).float()
    k = kc * par[..., 0, :, :, :] + par[..., 1, :, :, :]
    v = vc * par[..., 2, :, :, :] + par[..., 3, :, :, :]
    return k.flatten(-2), v.flatten(-2)


def _rope(x, table, positions):
    """Rotate-half in 32 bits, rounded once: x [n, heads, D]."""
    cs = table[positions.long()][:, None]  # [n, 1, D / 2, 2]
    a, b = x.float().chunk(2, -1)
    c, s = cs[..., 0], cs[..., 1]
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def _write(s):
    n = s["packed"].shape[0]
    q, k, v = s["packed"].view(n, -1, s["dim"]).split([s["q_heads"], s["kv_heads"], s["kv_heads"]], 1)
    q, k = _rope(q, s["rope"], s["positions"]), _rope(k, s["rope"], s["positions"])
    _store(s["pool"], s["slots"], k, v, s["page"])
    return {"q": q, **_read(s)}


def _read(s):
    slots, page, pool = s["slots"], s["page"], s["pool"]
    live = slots >= 0
    at = slots.clamp(min=0)
    k, v = _values(pool.transpose(1, 2)[at // page, at % page // 16], s["dtype"])  # [n, heads, 16, D]
    token = (at % 16)[:, None, None, None].expand(-1, k.shape[1], 1, k.shape[3])
    k, v = (x.gather(2, token).squeeze(2).to(s["dtype"]) * live[:, None, None] for x in (k, v))
    return {"k": k, "v": v}


def _attend(q, k, v, lens):
    """q [B, heads, group, D], k and v [B, heads, tokens, D], lens [B, heads or 1]: softmax over the first lens tokens."""
    scores = (q.float() @ k.transpose(-1, -2)) * (q.shape[-1] ** -0.5)
    out = torch.arange(k.shape[2], device=k.device) >= lens[..., None, None]
    scores = scores.masked_fill(out, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return (p @ v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _pages_of(s, table):
    """K, V float32 [B, heads, tokens, D] of a table [B, n] or [B, heads, n]."""
    heads = s["kv_heads"]
    if table.ndim == 2:
        table = table[:, None].expand(-1, heads, -1)
    tiles = s["pool"][table.long(), torch.arange(heads, device=table.device)[None, :, None]]  # [B, heads, n, tiles, 20 D]
    k, v = _values(tiles, s["dtype"])
    return k.flatten(2, 4), v.flatten(2, 4)


def _attention(s, table, lens):
    k, v = _pages_of(s, table)
    q = s["q"].unflatten(1, (s["kv_heads"], -1))
    return _attend(q, k, v, lens).flatten(1, 2).to(s["dtype"])


def _bounds(s, new):
    """Smallest and largest K of the pages that hold a sequence's last `new` tokens."""
    page, table = s["page"], s["table"]
    lens = s["lens"].long()
    n = torch.arange(table.shape[1], device=table.device)
    touched = (n >= (lens - new).clamp(min=0)[:, None] // page) & (n * page < lens[:, None])
    b, n = touched.nonzero(as_tuple=True)
    ids = table[b, n].long()
    k, _ = _values(s["pool"][ids], s["dtype"])  # [pages, heads, tiles, 16, D]
    k = k.flatten(2, 3).to(s["dtype"]).float()
    live = torch.arange(page, device=ids.device) < (lens[b] - n * page)[:, None]
    live = live[:, None, :, None]
    s["bounds"][ids, :, 0] = k.masked_fill(~live, math.inf).amin(2).to(s["dtype"])
    s["bounds"][ids, :, 1] = k.masked_fill(~live, -math.inf).amax(2).to(s["dtype"])
    return s["bounds"]


def _select(s):
    """Pages [B, heads, take] a KV head's queries attend, ascending, -1 behind the last, and the tokens they hold."""
    q, table, page, take = s["q"].float().unflatten(1, (s["kv_heads"], 1, -1)), s["table"], s["page"], s["take"]
    lens = s["lens"].long()
    count = (lens + page - 1) // page
    low, high = s["bounds"][table.long()].float().transpose(1, 2).unsqueeze(4).unbind(3)  # [B, heads, n, 1, D]
    terms = torch.maximum(q * low, q * high)  # [B, heads, n, group, D]
    while terms.shape[-1] > 1:  # pairwise, neighbours first
        terms = terms[..., 0::2] + terms[..., 1::2]
    scores = terms[..., 0].amax(-1)
    n = torch.arange(table.shape[1], device=q.device)
    scores = scores.masked_fill(n >= count[:, None, None], -math.inf)
    scores = scores.masked_fill(n == (count - 1)[:, None, None], math.inf)
    order = torch.sort(scores, dim=-1, descending=True, stable=True).indices[..., :take]
    if order.shape[-1] < take:
        order = torch.nn.functional.pad(order, (0, take - order.shape[-1]), value=table.shape[1])
    order = order.masked_fill(order >= count[:, None, None], table.shape[1]).sort(dim=-1).values
    taken = (order < table.shape[1]).sum(-1)
    at = order.clamp(max=table.shape[1] - 1)
    pages = table[:, None].expand(-1, s["kv_heads"], -1).gather(2, at).masked_fill(order == table.shape[1], -1)
    held = (taken - 1) * page + (lens - (count - 1) * page)[:, None]
    return pages.int(), held.int()


def _sparse(s):
    _bounds(s, 1)
    pages, held = _select(s)
    return {"out": _attention(s, pages.clamp(min=0), held), "pages": pages, "lens": held}


def run(state):
    if own:
        return _own(state)
    if state["op"] == "write":
        return _write(state)
    if state["op"] == "read":
        return _read(state)
    if state["op"] == "attention":
        return _attention(state, state["table"], state["lens"][:, None])
    if state["op"] == "bounds":
        return _bounds(state, state["new"])
    return _sparse(state)


# ------------------------------------------------------------------ in 64 bits, from the definitions
def _decode64(tiles, dtype):
    """uint8 [n, 20 D] -> K, V float64 [n, 16, D], by the place of every channel in the tile."""
    d = tiles.shape[1] // 20
    w = d // GROUP
    token = torch.arange(16, device=tiles.device)[:, None]
    ch = torch.arange(d, device=tiles.device)[None, :]
    group, inner = ch // GROUP, ch % GROUP
    k_byte = token * (d // 2) + (inner // 8) * 4 * w + group * 4 + inner % 8 // 2
    v_byte = 8 * d + token // 2 * d + (inner // 4) * 4 * w + group * 4 + token % 2 * 2 + inner % 4 // 2
    shift = ch % 2 * 4
    params = tiles[:, 16 * d:].contiguous().view(dtype).double().view(-1, 4, 16, w).repeat_interleave(GROUP, -1)
    code = lambda at: ((tiles[:, at].int() >> shift) & 15).double()  # noqa: E731
    return code(k_byte) * params[:, 0] + params[:, 1], code(v_byte) * params[:, 2] + params[:, 3]


def _codec64(x, dtype):
    """What rows [n, heads, D] (float64 values of type dtype) stand for once they are held in 4 bits."""
    parts = x.unflatten(-1, (-1, GROUP))
    low, high = parts.min(-1, keepdim=True).values, parts.max(-1, keepdim=True).values
    step = ((high - low) / 15).to(dtype).double()
    codes = torch.where(step > 0, ((parts - low) / step).round().clamp(0, 15), torch.zeros_like(parts))
    return (codes * step + low).flatten(-2)


def _sequence64(s, pages, head, tokens):
    k, v = _decode64(s["pool"][pages.long(), head].flatten(0, 1), s["dtype"])
    return k.reshape(-1, s["dim"])[:tokens], v.reshape(-1, s["dim"])[:tokens]


def _attention64(s, pages_of, tokens_of):
    group = s["q_heads"] // s["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(out.shape[0]):
        for h in range(s["kv_heads"]):
            tokens = tokens_of(b, h)
            if tokens:
                k, v = _sequence64(s, pages_of(b, h), h, tokens)
                heads = slice(h * group, (h + 1) * group)
                p = torch.softmax(s["q"][b, heads].double() @ k.T / math.sqrt(s["dim"]), -1)
                out[b, heads] = p @ v
    return out


def _bounds64(s, new):
    bounds = s["bounds"].double()
    for b, n in enumerate(s["lens"].tolist()):
        first = max(0, n - new) // s["page"]
        pages = s["table"][b, first:-(-n // s["page"])].long()
        for h in range(s["kv_heads"]):
            k, _ = _sequence64(s, pages, h, n - first * s["page"])
            k = k.to(s["dtype"]).double()
            short = len(pages) * s["page"] - len(k)
            rows = torch.cat([k, k[-1:].expand(short, -1)]).view(len(pages), s["page"], -1)  # the last row again: no new bound
            bounds[pages, h, 0], bounds[pages, h, 1] = rows.amin(1), rows.amax(1)
    return bounds


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "write":
        rows = s["packed"].double().view(len(s["slots"]), -1, s["dim"])
        half = s["dim"] // 2
        cs = s["rope"].double()[s["positions"].long()][:, None]
        one, two = rows[..., :half], rows[..., half:]
        turned = torch.cat([one * cs[..., 0] - two * cs[..., 1], two * cs[..., 0] + one * cs[..., 1]], -1)
        hq, hkv = s["q_heads"], s["kv_heads"]
        k = turned[:, hq:hq + hkv].to(s["dtype"]).double()  # the cache holds the key as its type rounds it
        return {"q": turned[:, :hq], "k": _codec64(k, s["dtype"]), "v": _codec64(rows[:, hq + hkv:], s["dtype"])}
    if s["op"] == "read":
        slots = s["slots"]
        at = slots.clamp(min=0)
        tiles = s["pool"].permute(0, 2, 1, 3).flatten(0, 1)[at // 16]  # [n, heads, 20 D]
        got = []
        for x in _decode64(tiles.flatten(0, 1), s["dtype"]):
            x = x.view(len(at), s["kv_heads"], 16, s["dim"])[torch.arange(len(at), device=at.device), :, at % 16]
            got.append(torch.where((slots >= 0)[:, None, None], x, torch.zeros_like(x)))
        return {"k": got[0], "v": got[1]}
    lens = s["lens"].tolist()
    if s["op"] == "attention":
        return _attention64(s, lambda b, h: s["table"][b, :-(-lens[b] // s["page"])], lambda b, h: lens[b])
    bounds = _bounds64(s, s["new"])
    if s["op"] == "bounds":
        return bounds
    chosen, held = {}, {}
    for b, n in enumerate(lens):
        count = -(-n // s["page"])
        pages = s["table"][b, :count].long()
        for h in range(s["kv_heads"]):
            group = s["q_heads"] // s["kv_heads"]
            q = s["q"][b, h * group:(h + 1) * group].double()
            low, high = bounds[pages, h, 0], bounds[pages, h, 1]
            score = (q.clamp(min=0) @ high.T + q.clamp(max=0) @ low.T).max(0).values[:-1]
            best = torch.sort(score, descending=True, stable=True).indices[: s["take"] - 1].sort().values
            chosen[b, h] = torch.cat([pages[best], pages[-1:]])
            held[b, h] = len(best) * s["page"] + n - (count - 1) * s["page"]
    return {"out": _attention64(s, lambda b, h: chosen[b, h], lambda b, h: held[b, h]), "pages": None, "lens": None}

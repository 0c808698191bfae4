"""GPU tests that every 32 tokens of every row are in the result once: across warps, CTAs, clusters and both
kernels, in caches where a lost or doubled piece is far outside the bound."""

from __future__ import annotations

import pytest
import torch

import int4_pieces as pieces
import int4_plain as plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
LAYOUTS = [(2, 6, 128, 16), (1, 16, 128, 64), (4, 4, 64, 32), (1, 9, 64, 16)]
LENGTHS = [[1], [31, 32, 33, 64], [513], [768, 769], [1024] * 3, [1500, 7, 1600], [2500] * 6, [2500] * 8, [5000], [40000], [20000, 7, 1],
           [33] * 300, [1] * 400, [100] * 149, [4096, 64, 2000, 129] * 8, [700, 9, 31, 1500, 64, 65, 3, 48, 1024, 1025, 250, 16] * 8, [12000, 9000, 32, 11000]]


def _attend(package, device, q, pool, table, lens, **more):
    return package.paged_decode_attention_int4(*(t.to(device) for t in (q, pool, table, lens)), **more)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", LAYOUTS)
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: f"{len(x)}x{max(x)}")
def test_every_unit_is_counted_once(package, cuda_device, dtype, heads, group, dim, page, lengths):
    q, pool, table, lens = pieces.counted(lengths, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=len(lengths))
    out = _attend(package, cuda_device, q, pool, table, lens)
    want, allowed = pieces.expected(q, pool, table, lens, device=cuda_device)
    assert pieces.worst(out, want, allowed) <= 1.0
    # a table far wider than the sequences: the other split of the work
    wide = torch.full((len(lengths), 4000), -1, dtype=torch.int32)
    wide[:, : table.shape[1]] = table[:, :4000]
    out = _attend(package, cuda_device, q, pool, wide, lens)
    assert pieces.worst(out, want, allowed) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", LAYOUTS)
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: f"{len(x)}x{max(x)}")
def test_ordinary_caches_within_a_channels_bound(package, cuda_device, dtype, heads, group, dim, page, lengths):
    q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=len(lengths))
    out = _attend(package, cuda_device, q, pool, table, lens)
    assert pieces.worst(out, *pieces.expected(q, pool, table, lens, device=cuda_device)) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", LAYOUTS)
@pytest.mark.parametrize("n", [33, 513, 1100, 3000, 13000])
def test_every_unit_in_turn_holds_the_weight(package, cuda_device, dtype, heads, group, dim, page, n):
    """Queries aimed at one unit after another: its maximum decides, wherever in the row, the warp or the CTA it lies."""
    patterns, pool, table, lens = pieces.signed(n, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=n)
    units = len(patterns)
    calls = -(-units // group)
    at = torch.arange(calls * group).view(calls, group) % units
    q = patterns[at].transpose(1, 2).reshape(calls, heads * group, dim).to(dtype)  # [calls, heads, group, D]
    dev = [t.to(cuda_device) for t in (pool, table, lens)]
    one_by_one = torch.cat([package.paged_decode_attention_int4(x[None].to(cuda_device), *dev, scale=0.25) for x in q])
    want, allowed = pieces.expected(q, pool, table.expand(calls, -1), lens.expand(calls), 0.25, device=cuda_device)
    assert pieces.worst(one_by_one, want, allowed) <= 1.0
    together = package.paged_decode_attention_int4(q.to(cuda_device), dev[0], dev[1].expand(calls, -1), dev[2].expand(calls), scale=0.25)
    assert pieces.worst(together, want, allowed) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("take", [1, 5, 33, 300])
def test_every_chosen_page_is_counted_once(package, cuda_device, dtype, take):
    """A choice's table through both calls, against the sum over the pages that it names."""
    lengths = [16 * 700 - 3, 16 * take, 40, 16 * 350 + 1]
    q, pool, table, lens = pieces.counted(lengths, dtype=dtype, dim=128, heads=2, group=6, page=16, seed=take)
    g = torch.Generator().manual_seed(take)
    limits = torch.randn(pool.shape[0], 2, 2, 128, generator=g).to(dtype).to(cuda_device)  # any choice will do
    out, pages, held = package.sparse_decode_attention_int4(*(t.to(cuda_device) for t in (q, pool)), limits, *(t.to(cuda_device) for t in (table, lens)), num_pages=take)
    again = package.paged_decode_attention_int4(q.to(cuda_device), pool.to(cuda_device), pages, held)
    k, v = (x.to(cuda_device) for x in plain.rows(pool, dtype))
    for b in range(len(lengths)):
        for h in range(2):
            n = int(held[b, h])
            ids = pages[b, h, : -(-n // 16)].long()
            mine = slice(6 * h, 6 * h + 6)
            parts = pieces.weighted(q[b, mine].to(cuda_device), k[ids, :, h].flatten(0, 1), v[ids, :, h].flatten(0, 1), n, 128 ** -0.5)
            for got in (out, again):
                assert ((got[b, mine].double() - parts[0]).abs() / pieces.bound(dtype, *parts)).max() <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", LAYOUTS)
@pytest.mark.parametrize("factor", [2.0 ** -6, 2.0 ** -10, 2.0 ** -14])
def test_groups_of_unlike_steps(package, cuda_device, dtype, heads, group, dim, page, factor):
    """Groups of V whose steps are far below another group's, an early token far above the rest, values of one
    sign and a large offset, and scores with a peak and a long tail: every channel within its own group's bound and
    2^-30 a token of the largest step's range."""
    lengths = [3000, 700, 40]
    q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=3)
    g = torch.Generator().manual_seed(3)
    for b, n in enumerate(lengths):
        token = torch.arange(n)
        slots = table[b, token // page].long() * page + token % page
        v = torch.randn(n, heads, dim, generator=g)
        v[..., : dim // 2] *= 8.0
        v[..., dim // 2:] *= 8.0 * factor
        v[n // 2, :, :32] *= 4.0
        v[..., dim - 32:] = v[..., dim - 32:].abs() + 50.0 * factor
        k = torch.randn(n, heads, dim, generator=g) * 0.3
        plain.store_fast(pool, slots, k.to(dtype), v.to(dtype))
    for scale in (0.02, 0.3, 2.0):
        out = _attend(package, cuda_device, q, pool, table, lens, scale=scale)
        assert pieces.worst(out, *pieces.expected(q, pool, table, lens, scale, device=cuda_device)) <= 1.0

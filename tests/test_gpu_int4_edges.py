"""GPU tests of the 4-bit cache at the edges of its definition."""

from __future__ import annotations

import pytest
import torch

import int4_plain as plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _spoil(pool, table, dtype, places):
    """Make groups of V infinite: (sequence, token, KV head, group); the row's K and other groups stay as they read."""
    page = pool.shape[2] * plain.TILE
    k, v = plain.rows(pool, dtype)
    for b, token, head, group in places:
        ident, row = int(table[b, token // page]), token % page
        kept_k, kept_v = (x[ident, row][None].to(dtype) for x in (k, v))
        kept_v[0, head, 32 * group + 7] = float("inf")
        plain.store(pool, torch.tensor([ident * page + row]), kept_k, kept_v)
        k, v = plain.rows(pool, dtype)
    return k, v


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", [(2, 6, 128, 16), (2, 4, 64, 32), (1, 16, 128, 16), (1, 12, 64, 16)])
@pytest.mark.parametrize("longest", [1, 40, 700, 3000, 20000])
def test_a_nan_group_of_v_stays_in_its_channels(package, cuda_device, dtype, heads, group, dim, page, longest):
    """A group of V with an infinity reads back as NaN: 32 channels of the sequence's result are NaN, all others
    are what they are without it, whether the row is one warp's, one CTA's, a cluster's or spread over CTAs."""
    lengths = [longest, 33, longest, 5]
    q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=longest)
    last = dim // 32 - 1
    places = [(0, longest // 2, 0, 0), (2, longest - 1, heads - 1, last), (1, 4, heads - 1, 1)]
    k, v = _spoil(pool, table, dtype, places)
    want, top = plain.attention(q, k, torch.nan_to_num(v, nan=0.0), table, lens)
    out = package.paged_decode_attention_int4(*(t.to(cuda_device) for t in (q, pool, table, lens))).cpu()
    spoiled = torch.zeros(out.shape, dtype=torch.bool)
    for b, _, head, w in places:
        spoiled[b, head * group:(head + 1) * group, 32 * w:32 * w + 32] = True
    assert torch.equal(torch.isnan(out), spoiled)
    plain.assert_attention(torch.where(spoiled, 0.0, out).to(dtype), torch.where(spoiled, 0.0, want), top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_units_of_nan_groups(package, cuda_device, dtype):
    """Whole units of 32 tokens whose V is NaN in one group, or in all of them in one sequence."""
    q, pool, table, lens = plain.make_cache([200, 200, 64], dtype=dtype, seed=5)
    places = [(0, t, 0, 2) for t in range(64, 96)] + [(1, t, 1, w) for t in range(32) for w in range(4)]
    k, v = _spoil(pool, table, dtype, places)
    want, top = plain.attention(q, k, torch.nan_to_num(v, nan=0.0), table, lens)
    out = package.paged_decode_attention_int4(*(t.to(cuda_device) for t in (q, pool, table, lens))).cpu()
    spoiled = torch.zeros(out.shape, dtype=torch.bool)
    spoiled[0, :6, 64:96] = spoiled[1, 6:] = True
    assert torch.equal(torch.isnan(out), spoiled)
    plain.assert_attention(torch.where(spoiled, 0.0, out).to(dtype), torch.where(spoiled, 0.0, want), top)


@pytest.mark.parametrize("query", [1e36, 3e37, 1e-30, 1e-36])
def test_queries_at_the_ends_of_bf16(package, cuda_device, query):
    """bf16 queries of any magnitude whose scores are ordinary."""
    q, pool, table, lens = plain.make_cache([40, 200, 1], dtype=torch.bfloat16, seed=2)
    q = (q.float() * query).bfloat16()
    scale = 0.1 / query
    want, top = plain.attention(q, *plain.rows(pool, q.dtype), table, lens, scale)
    out = package.paged_decode_attention_int4(*(t.to(cuda_device) for t in (q, pool, table, lens)), scale=scale)
    plain.assert_attention(out, want, top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pools_without_pages_are_read_and_written(package, cuda_device, dtype):
    """Every slot is outside a pool without pages: zeros are read, nothing is written, queries are rotated."""
    pool = package.empty_kv_pool_int4(0, 2, 128, device=cuda_device)
    slots = torch.tensor([0, 5, -1], device=cuda_device)
    for x in package.read_kv_int4(pool, slots, dtype=dtype):
        assert x.shape == (3, 2, 128) and (x == 0).all()
    for x in package.dequantize_kv_pool_int4(pool, dtype):
        assert x.shape == (0, 16, 2, 128)
    packed = torch.randn(3, 2048, device=cuda_device).to(dtype)
    rope = plain.rope_table(10, 128)
    q = package.packed_qkv_rope_cache_int4(packed, slots.clamp(min=0), slots, pool, rope_table=rope.to(cuda_device))
    assert torch.equal(q.cpu(), plain.rope(packed.cpu().view(3, 16, 128)[:, :12], rope, slots.cpu().clamp(min=0)))


@pytest.mark.parametrize("num_pages", [2 ** 31 - 1, 2 ** 26, 2 ** 62, 0, True])
def test_choices_too_large_are_refused_before_they_are_allocated(package, cuda_device, num_pages):
    """16 rows: 2^30 tiles over 16 rows and one tile a page leave fewer than 2^26 pages a row."""
    q, pool, table, lens = (t.to(cuda_device) for t in plain.make_cache([64] * 8))
    limits = package.empty_key_bounds_int4(pool, q.dtype).zero_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for call in (lambda: package.select_kv_pages(q, limits, table, lens, num_pages=num_pages),
                 lambda: package.sparse_decode_attention_int4(q, pool, limits, table, lens, num_pages=num_pages)):
        with pytest.raises(ValueError, match="num_pages"):
            call()
    assert torch.cuda.max_memory_allocated() - before < 2 ** 20


def test_sparse_attention_takes_scales_from_zero_on(package, cuda_device):
    q, pool, table, lens = plain.make_cache([300, 64])
    k, v = plain.rows(pool, q.dtype)
    limits = plain.bounds(k, table, lens, q.dtype, 10 ** 6, torch.zeros(pool.shape[0], 2, 2, 128, dtype=q.dtype))
    call = [t.to(cuda_device) for t in (q, pool, limits, table, lens)]
    for scale in (0.0, 0.3):
        out, pages, held = package.sparse_decode_attention_int4(*call, num_pages=5, scale=scale)
        plain.assert_attention(out, *plain.attention(q, k, v, pages.cpu(), held.cpu(), scale))
    with pytest.raises(ValueError, match="scale"):
        package.sparse_decode_attention_int4(*call, num_pages=5, scale=-0.3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", [(2, 6, 128, 16), (1, 16, 64, 32)])
@pytest.mark.parametrize("n", [20, 700, 5000])
def test_queries_that_are_not_finite_stay_in_their_heads(package, cuda_device, dtype, heads, group, dim, page, n):
    q, pool, table, lens = plain.make_cache([n, n, 3], dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=n)
    want, top = plain.attention(q, *plain.rows(pool, dtype), table, lens)
    q[0, 1, 5], q[1, group - 1, dim - 1], q[1, 0] = float("nan"), float("inf"), -float("inf")
    out = package.paged_decode_attention_int4(*(t.to(cuda_device) for t in (q, pool, table, lens))).cpu()
    spoiled = torch.zeros(out.shape, dtype=torch.bool)
    spoiled[0, 1] = spoiled[1, group - 1] = spoiled[1, 0] = True
    assert torch.equal(torch.isnan(out), spoiled)
    plain.assert_attention(torch.where(spoiled, 0.0, out).to(dtype), torch.where(spoiled, 0.0, want), top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_groups_at_the_ends_of_their_type(package, cuda_device, dtype):
    """Rows whose groups reach the largest finite numbers, of one sign and of both."""
    info = torch.finfo(dtype)
    x = torch.zeros(16, 2, 128, dtype=dtype)
    x[0, 0, 3], x[1, :, 40], x[2, 1, ::2], x[3] = info.max, -info.max, info.max, info.tiny
    x[4, 0, 0], x[4, 0, 1] = info.max, -info.max
    want = torch.zeros(1, 2, 1, 2560, dtype=torch.uint8)
    plain.store(want, torch.arange(16), x, x)
    got = package.quantize_kv_pool_int4(x[None].to(cuda_device), x[None].to(cuda_device))
    k, v = (t.cpu()[0] for t in package.dequantize_kv_pool_int4(got, dtype))
    value = plain.rows(want, dtype)[0][0].to(dtype)
    wide = torch.zeros(16, 2, 128, dtype=torch.bool)
    wide[4, 0, :32] = dtype is torch.bfloat16  # its range is beyond fp32
    for back in (k, v):
        assert torch.isnan(back)[wide].all() and torch.equal(back[~wide], value[~wide])

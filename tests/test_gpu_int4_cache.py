"""GPU tests of the 4-bit cache's write, read-back and key bounds: bytes and values equal the plain
codec's, whatever the layout of the inputs."""

from __future__ import annotations

from unittest import mock

import pytest
import torch

import int4_plain as plain
from conftest import with_gaps

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


def _rows(generator, n, heads, dim, dtype):
    offset = torch.randn(heads, dim, generator=generator)
    offset[:, 9] += 20
    return (torch.randn(n, heads, dim, generator=generator) * 0.5 + offset).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, q_heads, kv_heads, dim, page", [
    (1, 12, 2, 128, 16), (67, 12, 2, 128, 16), (33, 8, 8, 64, 32), (130, 7, 1, 128, 64), (5, 40, 8, 128, 16), (3, 1, 1, 64, 16)])
def test_packed_write(package, cuda_device, dtype, rows, q_heads, kv_heads, dim, page):
    """Bytes of the whole pool, rows that no slot names among them, and the rotated queries, bit for bit."""
    g = torch.Generator().manual_seed(rows)
    pages = rows // page + 3
    packed = torch.cat([_rows(g, rows, n, dim, dtype) for n in (q_heads, kv_heads, kv_heads)], 1)
    packed[0, q_heads, 1] = float("nan")
    packed[rows - 1, -1, dim - 2] = float("inf")
    packed[rows // 2, q_heads:] = 0.5
    slots = torch.randperm(pages * page, generator=g)[:rows]
    slots[rows // 3] = -1 if rows > 2 else slots[rows // 3]
    positions = torch.randint(0, 900, (rows,), generator=g).int()
    table = plain.rope_table(900, dim)
    pool = torch.randint(0, 256, (pages, kv_heads, page // 16, 20 * dim), generator=g, dtype=torch.uint8)
    dev = pool.to(cuda_device)
    q = package.packed_qkv_rope_cache_int4(packed.view(rows, -1).to(cuda_device), positions.to(cuda_device), slots.to(cuda_device),
                                           dev, q_heads=q_heads, rope_table=table.to(cuda_device))
    want_q, k = (plain.rope(x, table, positions) for x in packed.split([q_heads, kv_heads, kv_heads], 1)[:2])
    plain.store(pool, slots, k, packed[:, q_heads + kv_heads:])
    assert torch.equal(q.cpu().view(torch.int16), want_q.view(torch.int16)) or torch.equal(
        torch.nan_to_num(q.cpu().float()), torch.nan_to_num(want_q.float()))
    _same_cache(dev.cpu(), pool, dtype)


def _same_cache(actual, expected, dtype):
    """Equal bytes; NaN steps and floors may differ in their payload."""
    dim = expected.shape[3] // 20
    assert torch.equal(actual[..., : 16 * dim], expected[..., : 16 * dim])
    a, e = (x[..., 16 * dim:].contiguous().view(dtype) for x in (actual, expected))
    same = (a.view(torch.int16) == e.view(torch.int16)) | (torch.isnan(a) & torch.isnan(e))
    assert same.all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_forms_and_strides(package, cuda_device, dtype):
    """The three input layouts, strided and unaligned ones, int32 and int64 and float positions, and the
    angles computed in the kernel: the keys are then those of the 16-bit write, quantised."""
    g = torch.Generator().manual_seed(4)
    rows, hq, hkv, dim = 21, 6, 2, 128
    packed = torch.cat([_rows(g, rows, n, dim, dtype) for n in (hq, hkv, hkv)], 1).to(cuda_device)
    positions = torch.randint(0, 30000, (rows,), generator=g).to(cuda_device)
    slots = torch.randperm(64, generator=g)[:rows].to(cuda_device)
    k16, v16 = (torch.zeros(4, 16, hkv, dim, dtype=dtype, device=cuda_device) for _ in range(2))
    q, k, v = (x.unsqueeze(2) for x in packed.split([hq, hkv, hkv], 1))
    want_q = package.native_decode_rope_kv_write(q, k, v, positions, slots, k16, v16)
    want = torch.zeros(4, hkv, 1, 20 * dim, dtype=torch.uint8)
    keys, values = (x.cpu().view(64, hkv, dim)[slots.cpu()] for x in (k16, v16))
    plain.store(want, slots.cpu(), keys, values)

    def check(call, position=positions, slot=slots):
        pool = torch.zeros(want.shape, dtype=torch.uint8, device=cuda_device)
        got = call(position, slot, pool)
        assert torch.equal(pool.cpu(), want)
        return got

    flat = packed.view(rows, -1)
    decode = package.native_decode_rope_kv_write_int4
    assert torch.equal(check(lambda p, s, c: package.packed_qkv_rope_cache_int4(flat, p, s, c, q_heads=hq)), want_q[:, :, 0])
    check(lambda p, s, c: package.packed_qkv_rope_cache_int4(flat[:, None], p, s, c, q_heads=hq), positions.int(), slots.int())
    check(lambda p, s, c: package.packed_qkv_rope_cache_int4(with_gaps(flat), p, s, c, q_heads=hq), positions.float(), with_gaps(slots))
    shifted = torch.empty(rows * flat.shape[1] + 1, dtype=dtype, device=cuda_device)[1:].view(rows, -1).copy_(flat)
    check(lambda p, s, c: package.packed_qkv_rope_cache_int4(shifted, p, s, c, q_heads=hq), with_gaps(positions))
    assert torch.equal(check(lambda p, s, c: decode(q, k, v, p, s, c)), want_q)
    assert torch.equal(check(lambda p, s, c: decode(with_gaps(q), with_gaps(k), v, p, s, c)), want_q)
    kept = check(lambda p, s, c: decode(q, k, v, p, s, c, rotate_q=False))
    assert kept is q
    chunk = tuple(x.squeeze(2).transpose(0, 1)[None] for x in (q, k, v))
    got = check(lambda p, s, c: package.rope_kv_write_int4(*chunk, p[None], s, c))
    assert torch.equal(got[0].transpose(0, 1), want_q[:, :, 0])
    # a pool converted from 16-bit pools holds the same rows
    whole = package.quantize_kv_pool_int4(k16, v16)
    per_slot = lambda pool: [x.view(64, hkv, dim)[slots] for x in package.dequantize_kv_pool_int4(pool, dtype)]  # noqa: E731
    for a, b in zip(per_slot(whole), per_slot(want.to(cuda_device))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_quotients_between_two(package, cuda_device, dtype):
    """Values on and beside the borders between two codes, and tiny, huge and equal ones: the kernel's quotients are
    the correctly rounded ones, tie for tie."""
    g = torch.Generator().manual_seed(2)
    rows, heads, dim = 4096, 2, 128
    info = torch.finfo(dtype)
    step = torch.rand(rows, heads, dim // 32, 1, generator=g).mul(8).sub(4).exp()
    low = torch.randn(rows, heads, dim // 32, 1, generator=g) * step * 20
    x = low + step * (torch.randint(0, 31, (rows, heads, dim // 32, 32), generator=g) * 0.5)
    x = x.flatten(-2).to(dtype)
    x[:64] = (x[:64].float() * info.tiny * 4).to(dtype)           # down to subnormal steps
    x[64:128] = (x[64:128].float().sign() * info.max * 0.25 * torch.rand(64, heads, dim, generator=g)).to(dtype)
    x[128:140] = 0.0
    k, v = x, x.flip(-1)
    pool = torch.zeros(rows // 16, heads, 1, 20 * dim, dtype=torch.uint8)
    plain.store_fast(pool, torch.arange(rows), k, v)
    got = package.quantize_kv_pool_int4(*(t.to(cuda_device).view(rows // 16, 16, heads, dim) for t in (k, v)))
    _same_cache(got.cpu(), pool, dtype)


def test_converting_pools_in_parts(package, cuda_device):
    """Pools of more threads than one write takes are converted page range by page range: the same bytes."""
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(7, 32, 2, 128, generator=g).half().to(cuda_device) for _ in range(2))
    whole = package.quantize_kv_pool_int4(k, v)
    with mock.patch.object(package.kernel_module("int4_paged_kv"), "MAX_ITEMS", 3 * 32 * 32 + 5):
        parts = package.quantize_kv_pool_int4(k, v)
    assert torch.equal(whole, parts)


def test_valid_tokens_empty_calls_and_positions_past_the_table(package, cuda_device):
    g = torch.Generator().manual_seed(8)
    packed = torch.randn(6, 2048, generator=g).half().to(cuda_device)
    pool = torch.zeros(2, 2, 1, 2560, dtype=torch.uint8, device=cuda_device)
    table = plain.rope_table(10, 128).to(cuda_device)
    index = torch.arange(6, device=cuda_device)
    q = package.packed_qkv_rope_cache_int4(packed, index, index, pool, rope_table=table,
                                           valid_tokens=torch.tensor([4], dtype=torch.int32, device=cuda_device))
    assert (q[4:] == 0).all() and (q[:4] != 0).any(-1).all()
    k, v = package.read_kv_int4(pool, index)
    assert (k[4:] == 0).all() and (v[4:] == 0).all() and (v[:4] != 0).any(-1).all()
    before = pool.clone()
    none = package.packed_qkv_rope_cache_int4(packed[:0], index[:0], index[:0], pool, rope_table=table)
    assert none.shape == (0, 12, 128) and torch.equal(pool, before)
    assert [x.shape for x in package.read_kv_int4(pool, index[:0])] == [(0, 2, 128)] * 2
    late = package.packed_qkv_rope_cache_int4(packed, index + 7, index, pool, rope_table=table)
    assert package.cabi.device_status() == 4
    last = package.packed_qkv_rope_cache_int4(packed, index.clamp(min=9, max=9), index, pool, rope_table=table)
    assert torch.equal(late[3:], last[3:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, dim, page, rows", [(2, 128, 16, 1), (2, 128, 16, 1000), (4, 64, 32, 333), (1, 128, 64, 77), (8, 64, 16, 48)])
def test_read_rows(package, cuda_device, dtype, heads, dim, page, rows):
    """Rows in any order, repeated, and slots outside the pool."""
    q, pool, table, lens = plain.make_cache([page * 20 - 3], dtype=dtype, dim=dim, heads=heads, group=1, page=page, seed=rows, extra=0)
    g = torch.Generator().manual_seed(rows)
    slots = torch.randint(0, pool.shape[0] * page, (rows,), generator=g)
    slots[rows // 2:: 7] = torch.tensor([-1, pool.shape[0] * page, 2 ** 40, -2 ** 40])[torch.arange(len(slots[rows // 2:: 7])) % 4]
    k, v = (x.reshape(-1, heads, dim) for x in plain.rows(pool, dtype))
    live = (slots >= 0) & (slots < pool.shape[0] * page)
    for where in (slots, with_gaps(slots)):
        got = package.read_kv_int4(pool.to(cuda_device), where.to(cuda_device) if where is slots else with_gaps(slots.to(cuda_device)), dtype=dtype)
        for x, want in zip(got, (k, v)):
            want = torch.where(live[:, None, None], want[slots.clamp(0, len(want) - 1)], torch.zeros(())).to(dtype)
            assert torch.equal(torch.nan_to_num(x.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))
    whole = package.dequantize_kv_pool_int4(pool.to(cuda_device), dtype)
    for x, want in zip(whole, (k, v)):
        assert torch.equal(torch.nan_to_num(x.cpu().view(want.shape), nan=77.0), torch.nan_to_num(want.to(dtype), nan=77.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, dim, page", [(2, 128, 16), (4, 64, 64), (1, 128, 32), (3, 64, 16)])
@pytest.mark.parametrize("new", [0, 1, 40, 5000])
def test_key_bounds(package, cuda_device, dtype, heads, dim, page, new):
    """Pages of the newest tokens get exact extremes; all others, and rows behind a sequence's end, are left alone."""
    lengths = [0, 1, page - 1, page, page + 1, 300, 0, 1000]
    q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, dim=dim, heads=heads, group=1, page=page, seed=new)
    limits = torch.full((pool.shape[0], heads, 2, dim), 3.0, dtype=dtype)
    dev = limits.to(cuda_device)
    back = package.update_key_bounds_int4(pool.to(cuda_device), dev, table.long().to(cuda_device), lens.to(cuda_device), new_tokens=new)
    assert back is dev
    k, _ = plain.rows(pool, dtype)
    assert torch.equal(dev.cpu(), plain.bounds(k, table, lens, dtype, new, limits))


def test_key_bounds_keep_a_nan_and_report_bad_pages(package, cuda_device):
    q, pool, table, lens = plain.make_cache([40, 20], group=1, poison=False)
    k = torch.randn(1, 2, 128).half()
    k[0, 1, 70] = float("nan")
    plain.store(pool, table[0, 1:2].long() * 16 + 3, k, k)
    table[1, 0] = pool.shape[0]
    limits = torch.zeros(pool.shape[0], 2, 2, 128, dtype=torch.float16, device=cuda_device)
    package.update_key_bounds_int4(pool.to(cuda_device), limits, table.to(cuda_device), lens.to(cuda_device), new_tokens=40)
    assert package.cabi.device_status() == 2
    bad = torch.isnan(limits[table[0, 1].item()])
    assert bad[1, :, 64:96].all() and not bad[1, :, :64].any() and not bad[0].any()
    assert not torch.isnan(limits[table[0, 0].item()]).any()

"""GPU tests of attention over the 4-bit cache, of the page choice, and of both with the write, as a
decode loop uses them."""

from __future__ import annotations

import pytest
import torch

import int4_plain as plain
from conftest import with_gaps

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
MIXED = [0, 1, 15, 16, 17, 100, 513, 0, 2048, 31, 1000, 3]


def _check(package, device, q, pool, table, lens, /, *, scale=None, **forms):
    want, top = plain.attention(q, *plain.rows(pool, q.dtype), table, lens, scale)
    out = package.paged_decode_attention_int4(*(forms.get(n, t.to(device)) for n, t in
                                                (("q", q), ("pool", pool), ("table", table), ("lens", lens))), scale=scale)
    assert out.dtype == q.dtype and out.shape == q.shape
    plain.assert_attention(out, want, top)
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", [
    (2, 6, 128, 16), (1, 1, 128, 16), (2, 8, 64, 32), (8, 1, 64, 16), (1, 16, 128, 64), (3, 5, 64, 64), (4, 9, 128, 32), (2, 2, 128, 48)])
def test_lengths_layouts_and_types(package, cuda_device, dtype, heads, group, dim, page):
    """Empty rows, one token, page borders; what no sequence holds is NaN, table entries behind the last -1."""
    q, pool, table, lens = plain.make_cache(MIXED, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=group)
    out = _check(package, cuda_device, q, pool, table, lens)
    assert (out[lens == 0] == 0).all()
    assert package.cabi.device_status() == 0


@pytest.mark.parametrize("lengths", [[1], [16], [5000], [40000], [20000, 7, 1], [33] * 300, [1] * 700, [0, 0], list(range(0, 400, 3)),
                                     [700, 9, 31, 1500, 64, 65, 3, 48, 1024, 1025, 250, 16] * 8])
def test_splits(package, cuda_device, lengths):
    """One long row, many short ones, and shares whose borders fall inside rows."""
    q, pool, table, lens = plain.make_cache(lengths, seed=len(lengths))
    _check(package, cuda_device, q, pool, table, lens)


@pytest.mark.parametrize("heads, group, dim, page", [(2, 6, 128, 16), (1, 16, 64, 32), (4, 4, 64, 16), (2, 9, 128, 16)])
@pytest.mark.parametrize("batch, longest", [(1, 1), (1, 33), (2, 384), (1, 513), (3, 1024), (13, 1024), (14, 1024), (20, 1100), (1, 2000), (6, 2500), (7, 2500),
                                            (37, 400), (38, 400), (74, 300), (75, 300), (148, 100), (149, 100)])
def test_short_tables(package, cuda_device, batch, longest, heads, group, dim, page):
    """Rows that one CTA or the CTAs of one cluster hold alone, and the sizes around them: no token, fewer
    units than warps or CTAs, full rows; twice the same bits, then other lengths in the same tables."""
    lengths = [longest, *([0, 1, longest // 2, 40, 33, 32, 31, longest - 1, longest] * batch)][:batch]
    lengths = [min(n, longest) for n in lengths]
    q, pool, table, lens = plain.make_cache(lengths, dim=dim, heads=heads, group=group, page=page, seed=batch)
    out = _check(package, cuda_device, q, pool, table, lens)
    assert torch.equal(out, _check(package, cuda_device, q, pool, table, lens))
    _check(package, cuda_device, q, pool, table, lens // 3)


@pytest.mark.parametrize("take, page", [(32, 64), (16, 32), (5, 16)])
def test_choices_of_equal_length(package, cuda_device, take, page):
    """The tables of a choice: most rows full, some short or empty."""
    lengths = [page * take * 2 - 5] * 32
    lengths[3], lengths[9], lengths[31] = 0, 1, page * take // 2
    q, pool, table, lens = plain.make_cache(lengths, dtype=torch.bfloat16, page=page, seed=take)
    k, v = plain.rows(pool, q.dtype)
    limits = plain.bounds(k, table, lens, q.dtype, 10 ** 6, torch.zeros(pool.shape[0], 2, 2, 128, dtype=q.dtype))
    for n in (32, 13, 1):
        call = [t.to(cuda_device) for t in (q[:n], pool, limits, table[:n], lens[:n])]
        out, pages, held = package.sparse_decode_attention_int4(*call, num_pages=take)
        want, top = plain.attention(q[:n], k, v, pages.cpu(), held.cpu())
        plain.assert_attention(out, want, top)


@pytest.mark.parametrize("dtype", DTYPES)
def test_magnitudes(package, cuda_device, dtype):
    """Values and queries far from one, scores far apart, one row far larger than the rest, and a scale of its own."""
    lengths = [5, 300, 64, 1]
    for gain, query in ((1e-3, 1.0), (100.0, 0.01), (1.0, 30.0)):
        q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, gain=gain, seed=3)
        q = (q.float() * query).to(dtype)
        _check(package, cuda_device, q, pool, table, lens, scale=0.05)
    # the value of one late token dwarfs the others, and so does, elsewhere, the score of one
    k = torch.randn(2, 2, 128).to(dtype)
    v = (torch.randn(2, 2, 128) * 1000).to(dtype)
    plain.store(pool, torch.tensor([table[1, 17] * 16 + 3, table[1, 2] * 16 + 1]), k * 4, v)
    _check(package, cuda_device, q, pool, table, lens)


def test_large_and_tiny_bf16(package, cuda_device):
    for gain in (1e15, 1e-15, 1e33, 1e37):
        q, pool, table, lens = plain.make_cache([40, 200], dtype=torch.bfloat16, gain=gain, seed=2)
        _check(package, cuda_device, q, pool, table, lens)
    for query in (1e15, 1e-15):
        q, pool, table, lens = plain.make_cache([40, 200], dtype=torch.bfloat16, seed=2)
        _check(package, cuda_device, (q.float() * query).bfloat16(), pool, table, lens, scale=0.1 / query)


def test_equal_rows_of_zeros_and_constants(package, cuda_device):
    """A cache of zeros and groups without range: the mean of the values, exactly their value."""
    pool = torch.zeros(3, 2, 1, 2560, dtype=torch.uint8)
    plain.store(pool, torch.arange(32), torch.zeros(32, 2, 128).half(), torch.full((32, 2, 128), 0.75).half())
    q = torch.randn(1, 12, 128).half()
    out = package.paged_decode_attention_int4(q.to(cuda_device), pool.to(cuda_device), torch.tensor([[0, 1]], dtype=torch.int32, device=cuda_device),
                                              torch.tensor([30], dtype=torch.int32, device=cuda_device))
    assert (out == 0.75).all()


def test_strides_index_types_and_tables_a_head(package, cuda_device):
    q, pool, table, lens = plain.make_cache(MIXED, seed=9)
    dev = cuda_device
    _check(package, dev, q, pool, table, lens, table=table.long().to(dev), lens=lens.long().to(dev))
    _check(package, dev, q, pool, table, lens, table=with_gaps(table.to(dev)), lens=with_gaps(lens.to(dev)), q=with_gaps(q.to(dev)))
    wide = torch.zeros(len(MIXED), 40, 128, dtype=q.dtype, device=dev)
    wide[:, 8:20] = q.to(dev)
    _check(package, dev, q, pool, table, lens, q=wide[:, 8:20])
    shifted = torch.empty(q.numel() + 1, dtype=q.dtype, device=dev)[1:].view(q.shape).copy_(q)
    _check(package, dev, q, pool, table, lens, q=shifted)
    # a table and a length for every KV head: the second head's rows in reverse order of the batch
    both = torch.stack([table, table.flip(0)], 1)
    lens_both = torch.stack([lens, lens.flip(0)], 1)
    _check(package, dev, q, pool, both, lens_both)
    _check(package, dev, q, pool, both, lens_both, table=both.transpose(0, 1).contiguous().to(dev).transpose(0, 1), lens=lens_both.long().to(dev))


def test_lengths_outside_the_table_and_bad_pages(package, cuda_device):
    q, pool, table, lens = plain.make_cache([64, 64, 64, 64], seed=1)
    lens = torch.tensor([64, -5, 10 ** 6, 2 ** 31 - 1], dtype=torch.int32)
    _check(package, cuda_device, q, pool, table, lens)
    table[0, 1], table[2, 0], table[2, 3] = -1, pool.shape[0], 2 ** 31 - 1
    _check(package, cuda_device, q, pool, table, lens)
    assert package.cabi.device_status() == 2


def test_empty_batch_and_infinite_values(package, cuda_device):
    q, pool, table, lens = plain.make_cache([64, 30], seed=1)
    empty = package.paged_decode_attention_int4(*(t.to(cuda_device) for t in (q[:0], pool, table[:0], lens[:0])))
    assert empty.shape == (0, 12, 128)
    v = torch.zeros(1, 2, 128).half()
    v[0, 1, 3] = float("inf")
    plain.store(pool, table[0, :1].long() * 16, v, v)
    out = package.paged_decode_attention_int4(*(t.to(cuda_device) for t in (q, pool, table, lens))).cpu()
    assert torch.isnan(out[0, 6:]).all() and torch.isfinite(out[0, :6]).all() and torch.isfinite(out[1]).all()


def test_tables_without_pages_and_pools_without_pages(package, cuda_device):
    """A table of width 0 holds no token; a pool without pages has none to read."""
    q, pool, table, lens = (t.to(cuda_device) for t in plain.make_cache([40, 20], seed=1))
    limits = torch.zeros(pool.shape[0], 2, 2, 128, dtype=q.dtype, device=cuda_device)
    out = package.paged_decode_attention_int4(q, pool, table[:, :0], lens)
    assert (out == 0).all()
    pages, held = package.select_kv_pages(q, limits, table[:, :0], lens, num_pages=3)
    assert (pages == -1).all() and (held == 0).all()
    out, pages, held = package.sparse_decode_attention_int4(q, pool, limits, table[:, :0], lens, num_pages=3)
    assert (out == 0).all() and (pages == -1).all() and (held == 0).all()
    package.update_key_bounds_int4(pool, limits, table[:, :0], lens, new_tokens=5)
    assert package.cabi.device_status() == 0
    out = package.paged_decode_attention_int4(q, pool[:0], table, lens)
    assert (out == 0).all() and package.cabi.device_status() == 2


@pytest.mark.parametrize("scale", [0.0, -0.07, 3.0])
def test_scales(package, cuda_device, scale):
    q, pool, table, lens = plain.make_cache([0, 1, 33, 200, 700], seed=8)
    _check(package, cuda_device, (q * 0.3).half(), pool, table, lens, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_rows_than_shared_memory_keeps(package, cuda_device, dtype):
    """Thousands of rows, many of them empty: lengths come from global memory and threads take several rows."""
    g = torch.Generator().manual_seed(1)
    lengths = torch.randint(0, 40, (700,), generator=g).tolist() + [900, 0, 0, 0, 5]
    q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, dim=64, heads=4, group=2, seed=4)
    out = _check(package, cuda_device, q, pool, table, lens)
    assert (out[lens == 0] == 0).all()


def test_pool_beyond_four_gigabytes(package, cuda_device):
    q, pool, table, lens = plain.make_cache([100, 333], seed=6)
    far = 2 ** 32 // (2 * 2560) + 1000
    big = torch.empty(far + pool.shape[0], *pool.shape[1:], dtype=torch.uint8, device=cuda_device)
    big[far:] = pool.to(cuda_device)
    moved = torch.where(table >= 0, table + far, table).to(cuda_device)
    want, top = plain.attention(q, *plain.rows(pool, q.dtype), table, lens)
    plain.assert_attention(package.paged_decode_attention_int4(q.to(cuda_device), big, moved, lens.to(cuda_device)), want, top)
    slots = (moved[1, :3].long()[:, None] * 16 + torch.arange(16, device=cuda_device)).flatten()
    near = slots - far * 16
    for a, b in zip(package.read_kv_int4(big, slots), package.read_kv_int4(pool.to(cuda_device), near)):
        assert torch.equal(a, b)


def _selection(package, device, q, limits, table, lens, take, page):
    want = plain.select(q, limits, table, lens, take, page)
    got = package.select_kv_pages(q.to(device), limits.to(device), table.to(device), lens.to(device), num_pages=take, page_size=page)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads, group, dim, page", [(2, 6, 128, 16), (4, 4, 64, 32), (1, 16, 128, 64), (8, 1, 64, 16), (2, 3, 128, 32)])
@pytest.mark.parametrize("take", [1, 2, 17, 64])
def test_selection_and_sparse_attention(package, cuda_device, dtype, heads, group, dim, page, take):
    lengths = [0, 1, page * take, page * take + 1, 3000, 700, page * (take - 1) + 2, 1600]
    q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=take)
    k, v = plain.rows(pool, dtype)
    limits = plain.bounds(k, table, lens, dtype, 10 ** 6, torch.zeros(pool.shape[0], heads, 2, dim, dtype=dtype))
    pages, held = _selection(package, cuda_device, q, limits, table, lens, take, page)
    out, pages2, held2 = package.sparse_decode_attention_int4(q.to(cuda_device), pool.to(cuda_device), limits.to(cuda_device), table.to(cuda_device),
                                                              lens.to(cuda_device), num_pages=take)
    assert torch.equal(pages, pages2) and torch.equal(held, held2)
    want, top = plain.attention(q, k, v, pages.cpu(), held.cpu())
    plain.assert_attention(out, want, top)
    plain.assert_attention(package.paged_decode_attention_int4(q.to(cuda_device), pool.to(cuda_device), pages, held), want, top)


def test_selection_of_ties_specials_and_many_pages(package, cuda_device):
    """Equal scores go to the earlier pages; NaN first; pages outside the pool last; zeros of both signs tie."""
    g = torch.Generator().manual_seed(0)
    pages, heads, dim = 300, 2, 64
    q = torch.randn(3, 4, dim, generator=g).half()
    limits = torch.zeros(pages, heads, 2, dim).half()
    limits[::3] = -0.0
    table = torch.stack([torch.randperm(pages, generator=g) for _ in range(3)]).int()
    lens = torch.tensor([pages * 16, 4001, 50 * 16], dtype=torch.int32)
    _selection(package, cuda_device, q, limits, table, lens, 20, 16)
    limits[:] = torch.randint(-2, 3, limits.shape, generator=g).half()  # many ties of whole numbers
    q = torch.randint(-1, 2, q.shape, generator=g).half()
    _selection(package, cuda_device, q, limits, table, lens, 20, 16)
    limits[7, 0, 0, 5], limits[9], limits[11] = float("nan"), float("inf"), -float("inf")
    q = torch.randn(3, 4, dim, generator=g).half()
    _selection(package, cuda_device, q, limits, table, lens, 41, 16)
    table[0, 30], table[1, 200], table[2, 3] = -1, pages, 10 ** 6
    _selection(package, cuda_device, q, limits, table, lens, 41, 16)
    assert package.cabi.device_status() == 2
    many = 70000
    limits = torch.randn(many, 1, 2, dim, generator=g).half()
    table = torch.randperm(many, generator=g)[None]
    _selection(package, cuda_device, q[:1], limits, table, torch.tensor([many * 16 - 9]), 1500, 16)
    _selection(package, cuda_device, q[:1], limits, table, torch.tensor([many * 16 - 9]), many - 1, 16)


@pytest.mark.parametrize("kind", ["wide", "near", "signs", "two values", "few bits", "huge", "one large"])
@pytest.mark.parametrize("count", [2, 511, 1024, 2560, 2561, 9000])
def test_selection_of_scores_of_all_kinds(package, cuda_device, kind, count):
    """Scores that differ in their high bits, in their low ones, in sign, in one place, or not at all, at
    the sizes where a thread holds more keys or none."""
    g = torch.Generator().manual_seed(count)
    x = torch.randn(count, 3, generator=g, dtype=torch.float64)
    x = {"wide": lambda: x * torch.exp2(torch.randint(-12, 12, (count, 3), generator=g)), "signs": lambda: x.sign(),
         "near": lambda: 1 + x.abs() * 0.01, "two values": lambda: (x > 0).double(), "huge": lambda: x * 6000,
         "few bits": lambda: torch.cat([torch.full((count, 2), 512.0, dtype=torch.float64), x[:, :1].round() / 256], 1),
         "one large": lambda: torch.where(torch.arange(count)[:, None] == count // 2, 100.0, 0.0) + torch.zeros(3)}[kind]()
    limits = torch.zeros(count, 1, 2, 64)
    limits[:, 0, :, 8] = x[:, :1]
    limits[:, 0, :, 9], limits[:, 0, :, 40] = x[:, 1:2], x[:, 2:]
    q = torch.zeros(1, 1, 64)
    q[0, 0, [8, 9, 40]] = torch.tensor([1.0, 1.0, 2.0 ** -6])
    table, lens = torch.randperm(count, generator=g)[None].int(), torch.tensor([count * 16 - 3], dtype=torch.int32)
    for take in {1, 2, min(33, count), count // 2 + 1, count - 1} - {0}:
        _selection(package, cuda_device, q.half(), limits.half(), table, lens, take, 16)


def _decode_state(device, dtype=torch.float16, page=32, prompt=(200, 37, 90), steps=70):
    """Sequences with room to grow, their packed rows for a prompt and for every step."""
    g = torch.Generator().manual_seed(12)
    width = max(-(-(n + steps) // page) for n in prompt)
    table = torch.randperm(len(prompt) * width + 3, generator=g)[: len(prompt) * width].view(len(prompt), -1).int()
    rows = lambda n: (torch.randn(n, 2048, generator=g) * 0.7).to(dtype)  # noqa: E731
    return table, torch.tensor(prompt), rows(sum(prompt)), [rows(len(prompt)) for _ in range(steps)], plain.rope_table(width * page, 128)


def _slots(table, b, positions, page):
    return table[b, positions // page].long() * page + positions % page


def test_page_ids_beyond_32_bits_stay_outside_the_pool(package, cuda_device):
    """An id of 2^32 + 5 must not come out of the choice as page 5."""
    q, pool, table, lens = plain.make_cache([64, 300], seed=4)
    k, _ = plain.rows(pool, q.dtype)
    limits = plain.bounds(k, table, lens, q.dtype, 10 ** 6, torch.zeros(pool.shape[0], 2, 2, 128, dtype=q.dtype))
    wide = table.long()
    wide[0, 1], wide[1, 18] = 2 ** 32 + 5, 2 ** 33  # a page of a row whose pages are all taken, and a newest page
    out, pages, held = package.sparse_decode_attention_int4(*(t.to(cuda_device) for t in (q, pool, limits, wide, lens)), num_pages=6)
    assert package.cabi.device_status() == 2
    assert pages[0, :, 1].tolist() == [-1, -1] and pages[1, :, 5].tolist() == [-1, -1]
    plain.assert_attention(out, *plain.attention(q, *plain.rows(pool, q.dtype), pages.cpu(), held.cpu()))


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prompt_and_a_decode_loop(package, cuda_device, dtype, captured):
    """Prompt written in one call, bounds of all its pages, then steps of write, bounds and sparse attention
    (captured once and replayed, or called), against the plain forms on the cache as it then is."""
    page, take = 32, 4
    table, lens, prompt, steps, rope = _decode_state(cuda_device, dtype, page)
    batch = len(lens)
    owner = torch.repeat_interleave(torch.arange(batch), lens)
    positions = torch.cat([torch.arange(n) for n in lens.tolist()])
    dev = lambda t: t.to(cuda_device)  # noqa: E731
    pool = package.empty_kv_pool_int4(int(table.max()) + 4, 2, 128, page_size=page, device=cuda_device)
    pool.fill_(255)
    limits = package.empty_key_bounds_int4(pool, dtype)
    limits.fill_(float("nan"))
    rope_dev, table_dev = dev(rope), dev(table)
    package.packed_qkv_rope_cache_int4(dev(prompt), dev(positions), dev(_slots(table, owner, positions, page)), pool, rope_table=rope_dev)
    length = dev(lens.int())
    package.update_key_bounds_int4(pool, limits, table_dev, length, new_tokens=int(lens.max()))
    packed, position, slot = torch.zeros(batch, 2048, dtype=dtype, device=cuda_device), length.clone(), length.long()

    def step():
        q = package.packed_qkv_rope_cache_int4(packed, position, slot, pool, rope_table=rope_dev)
        package.update_key_bounds_int4(pool, limits, table_dev, length)
        return q, *package.sparse_decode_attention_int4(q, pool, limits, table_dev, length, num_pages=take)

    graph = None
    for i, rows in enumerate(steps):
        position.copy_(lens)
        slot.copy_(_slots(table, torch.arange(batch), lens, page))
        lens = lens + 1
        length.copy_(lens)
        packed.copy_(rows)
        if not captured:
            outputs = step()
        elif graph is None:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outputs = step()
            graph.replay()
        else:
            graph.replay()
        if i % 23 == 0 or i == len(steps) - 1:
            q, out, pages, held = (t.cpu() for t in outputs)
            k, v = plain.rows(pool.cpu(), dtype)
            fresh = plain.bounds(k, table, lens, dtype, 10 ** 6, torch.zeros(limits.shape, dtype=dtype))
            used = torch.zeros(pool.shape[0], dtype=torch.bool)
            for b in range(batch):
                used[table[b, : -(-int(lens[b]) // page)].long()] = True
            assert torch.equal(limits.cpu()[used], fresh[used])
            want_pages, want_held = plain.select(q, fresh, table, lens, take, page)
            assert torch.equal(pages, want_pages) and torch.equal(held, want_held)
            plain.assert_attention(out, *plain.attention(q, k, v, pages, held))
            assert torch.equal(q, plain.rope(rows.view(batch, -1, 128)[:, :12], rope, lens - 1))


def test_same_bits_again_other_streams_and_two_graphs(package, cuda_device):
    """The same call twice gives the same bits, on any stream; two captured calls replayed in any order, on two
    streams at once, do not disturb each other."""
    inputs = [tuple(t.to(cuda_device) for t in plain.make_cache(lengths, seed=s)) for s, lengths in ((1, [3000, 20, 900]), (2, [64] * 50))]
    want = [package.paged_decode_attention_int4(*x) for x in inputs]
    again = [package.paged_decode_attention_int4(*x) for x in inputs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [package.paged_decode_attention_int4(*x) for x in inputs]
    torch.cuda.synchronize()
    for a, b, c in zip(want, again, other):
        assert torch.equal(a, b) and torch.equal(a, c)
    graphs = []
    for x in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = package.paged_decode_attention_int4(*x)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out), b in zip(graphs, want):
        assert torch.equal(out, b)


def test_two_captured_sparse_calls_side_by_side(package, cuda_device):
    """Scratch and choices are each graph's own: replayed together they give what they give alone."""
    cases = []
    for seed, lengths in ((3, [4000, 900, 2500]), (4, [1500] * 6)):
        q, pool, table, lens = plain.make_cache(lengths, seed=seed)
        k, _ = plain.rows(pool, q.dtype)
        limits = plain.bounds(k, table, lens, q.dtype, 10 ** 6, torch.zeros(pool.shape[0], 2, 2, 128, dtype=q.dtype))
        cases.append(tuple(t.to(cuda_device) for t in (q, pool, limits, table, lens)))
    alone = [package.sparse_decode_attention_int4(*c, num_pages=20) for c in cases]
    graphs = []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = package.sparse_decode_attention_int4(*c, num_pages=20)
        graphs.append((graph, outputs, torch.cuda.Stream()))
    for _ in range(30):
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, outputs, _), want in zip(graphs, alone):
        assert all(torch.equal(a, b) for a, b in zip(outputs, want))


def test_neighbouring_calls_do_not_race(package, cuda_device):
    """Launches chained back to back: a step's write must be seen by the attention behind it, and an attention
    must be done with the cache before the next step's write changes it."""
    q, pool, table, lens = plain.make_cache([257] * 40, seed=5)
    dev = [t.to(cuda_device) for t in (q, pool, table, lens)]
    rope = plain.rope_table(300, 128).to(cuda_device)
    slots = (table[:, 16].long() * 16).to(cuda_device)
    positions = torch.full((40,), 256, device=cuda_device)
    rows = [torch.randn(40, 2048, device=cuda_device).half() for _ in range(6)]
    chained, apart = [], []
    for results, wait in ((apart, True), (chained, False)):
        for packed in rows * 5:
            turned = package.packed_qkv_rope_cache_int4(packed, positions, slots, dev[1], rope_table=rope)
            torch.cuda.synchronize() if wait else None
            results.append(package.paged_decode_attention_int4(turned, dev[1], dev[2], dev[3]))
            torch.cuda.synchronize() if wait else None
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(chained, apart))


def test_refusals_on_the_device(package, cuda_device):
    q, pool, table, lens = (t.to(cuda_device) for t in plain.make_cache([40, 20]))
    attend = package.paged_decode_attention_int4
    limits = package.empty_key_bounds_int4(pool, torch.float16)
    for match, call in (("head_dim", lambda: attend(q[..., :64], pool, table, lens)), ("divisible", lambda: attend(q[:, :11], pool, table, lens)),
                        ("batch dimensions", lambda: attend(q, pool, table[:1], lens)), ("integer", lambda: attend(q, pool, table.float(), lens)),
                        ("integer", lambda: attend(q, pool, table, lens.half())), ("float16 or bfloat16", lambda: attend(q.float(), pool, table, lens)),
                        ("contiguous", lambda: attend(q, pool.transpose(0, 1), table, lens)), ("device", lambda: attend(q.cpu(), pool, table, lens)),
                        ("per KV head", lambda: attend(q, pool, table[:, None], lens)), ("at most 16", lambda: attend(q.repeat(1, 3, 1), pool, table, lens)),
                        ("batch dimensions", lambda: package.update_key_bounds_int4(pool, limits, table[:, None], lens)),
                        ("new_tokens", lambda: package.update_key_bounds_int4(pool, limits, table, lens, new_tokens=-1)),
                        ("match the pool", lambda: package.update_key_bounds_int4(pool, limits[1:], table, lens)),
                        ("queries' dtype", lambda: package.select_kv_pages(q.bfloat16(), limits, table, lens, num_pages=2)),
                        ("num_pages", lambda: package.select_kv_pages(q, limits, table, lens, num_pages=0)),
                        ("page_size", lambda: package.select_kv_pages(q, limits, table, lens, num_pages=2, page_size=8)),
                        ("num_pages", lambda: package.sparse_decode_attention_int4(q, pool, limits, table, lens, num_pages=1.5)),
                        ("per row", lambda: package.packed_qkv_rope_cache_int4(q.new_zeros(2, 2048), lens[:1], lens, pool)),
                        ("packed QKV", lambda: package.packed_qkv_rope_cache_int4(q.view(2, -1), lens, lens, pool)),
                        ("integer", lambda: package.read_kv_int4(pool, lens.float()))):
        with pytest.raises(ValueError, match=match):
            call()

"""GPU tests of the 4-bit cache's calls beside others: what a call reads is what the calls before it on its
own stream wrote, whatever is launched between them on this stream or another."""

from __future__ import annotations

import threading

import pytest
import torch

import int4_plain as plain

pytestmark = pytest.mark.gpu


def _choices(device, seed, *, heads=2, group=6, batch=24, steps=24):
    """A cache whose rows have thousands of pages (some shared, so that it stays small) and a query a step:
    the choice takes a while and differs from step to step."""
    g = torch.Generator().manual_seed(seed)
    _, pool, _, _ = plain.make_cache([16 * 600], heads=heads, group=group, seed=seed, extra=0)
    limits = plain.bounds(plain.rows(pool, torch.float16)[0], torch.arange(600)[None], torch.tensor([16 * 600]), torch.float16, 16 * 600,
                          torch.zeros(600, heads, 2, 128, dtype=torch.float16))
    table = torch.randint(0, 600, (batch, 3000), generator=g).int()
    lens = torch.randint(16 * 2000, 16 * 3000, (batch,), generator=g).int()
    queries = torch.randn(steps, batch, heads * group, 128, generator=g).half()
    return [t.to(device) for t in (pool, limits, table, lens, queries)]


def _select(package, case, step):
    pool, limits, table, lens, queries = case
    return package.select_kv_pages(queries[step], limits, table, lens, num_pages=20)


def _attend(package, case, step, choice, flat=False):
    pages, held = choice
    pages, held = (pages[:, 0], held[:, 0]) if flat else (pages, held)
    return package.paged_decode_attention_int4(case[4][step], case[0], pages, held)


@pytest.mark.parametrize("heads, flat", [(2, False), (1, False), (1, True)])
def test_choices_and_attentions_of_two_streams_interleave(package, cuda_device, heads, flat):
    """One thread, two micro-batches on two streams: choose, choose, attend, attend.  flat: the only KV head's
    table as one of the sequences."""
    cases = [_choices(cuda_device, seed, heads=heads) for seed in (1, 2)]
    steps = len(cases[0][4])
    alone = []
    for case in cases:
        alone.append([])
        for step in range(steps):
            choice = _select(package, case, step)
            torch.cuda.synchronize()
            alone[-1].append((*choice, _attend(package, case, step, choice, flat)))
            torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        results = [[], []]
        for step in range(steps):
            choices = []
            for case, stream in zip(cases, streams):
                with torch.cuda.stream(stream):
                    choices.append(_select(package, case, step))
            for got, case, choice, stream in zip(results, cases, choices, streams):
                with torch.cuda.stream(stream):
                    got.append((*choice, _attend(package, case, step, choice, flat)))
        torch.cuda.synchronize()
        for got, want in zip(results, alone):
            assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


def test_a_call_on_another_stream_between_a_choice_and_its_attention(package, cuda_device):
    case = _choices(cuda_device, 3)
    steps = len(case[4])
    alone = []
    for step in range(steps):
        choice = _select(package, case, step)
        torch.cuda.synchronize()
        alone.append(_attend(package, case, step, choice))
    side, slots = torch.cuda.Stream(), torch.arange(64, device=cuda_device)
    got = []
    for step in range(steps):
        choice = _select(package, case, step)
        with torch.cuda.stream(side):
            package.read_kv_int4(case[0], slots, dtype=torch.float16)
        got.append((choice, _attend(package, case, step, choice)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for (_, a), b in zip(got, alone))


def test_a_call_on_the_same_stream_between_a_choice_and_its_attention(package, cuda_device):
    """A kernel that lets the next one stand by from its start lies between the two."""
    case = _choices(cuda_device, 4)
    steps, slots = len(case[4]), torch.arange(64, device=cuda_device)
    want, got = [], []
    for results, wait in ((want, True), (got, False)):
        for step in range(steps):
            choice = _select(package, case, step)
            torch.cuda.synchronize() if wait else None
            package.read_kv_int4(case[0], slots, dtype=torch.float16)
            torch.cuda.synchronize() if wait else None
            results.append((choice, _attend(package, case, step, choice)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for (_, a), (_, b) in zip(got, want))


def test_choices_and_attentions_of_two_threads(package, cuda_device):
    cases = [_choices(cuda_device, seed) for seed in (5, 6)]
    steps = len(cases[0][4])
    alone = []
    for case in cases:
        alone.append([])
        for step in range(steps):
            choice = _select(package, case, step)
            torch.cuda.synchronize()
            alone[-1].append(_attend(package, case, step, choice))
    torch.cuda.synchronize()
    results, start = [[], []], threading.Barrier(2, timeout=60)

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for step in range(steps):
                choice = _select(package, cases[i], step)
                results[i].append((choice, _attend(package, cases[i], step, choice)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for got, want in zip(results, alone):
        assert len(got) == steps and all(torch.equal(a, b) for (_, a), b in zip(got, want))


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("between", ["write", "read", "bounds", "nothing", "advance"])
def test_lengths_moved_on_by_a_kernel_in_front(package, cuda_device, between, captured):
    """seq_lens.add_(1), as a decode loop does it, then a call, then attention: no copy and no request in between."""
    batch, steps, first = 40, 60, 257
    _, pool, table, lens = (t.to(cuda_device) for t in plain.make_cache([first + steps + 1] * batch, seed=7))
    g = torch.Generator().manual_seed(7)
    packed = (torch.randn(steps, batch, 2048, generator=g) * 0.7).half().to(cuda_device)
    rope = plain.rope_table(400, 128).to(cuda_device)
    limits = package.empty_key_bounds_int4(pool, torch.float16).zero_()
    queries = torch.randn(steps, batch, 12, 128, generator=g).half().to(cuda_device)
    positions = torch.full((batch,), first, device=cuda_device)
    slots = table[:, first // 16].long() * 16 + first % 16

    def run(wait):
        """A copy of the cache, its steps one after another; the attention's results."""
        cache, length, position, slot = pool.clone(), torch.full_like(lens, first), positions - int(between == "advance"), slots.clone()
        bounds, results = limits.clone(), []
        pause = torch.cuda.synchronize if wait else (lambda: None)
        for step in range(steps):
            if between == "advance":
                package.advance_decode_state(position, length, slot, table, num_pages=cache.shape[0])
            else:
                length.add_(1)
            pause()
            if between in ("write", "advance"):
                package.packed_qkv_rope_cache_int4(packed[step], position, slot, cache, rope_table=rope)
            elif between == "read":
                package.read_kv_int4(cache, slot, dtype=torch.float16)
            elif between == "bounds":
                package.update_key_bounds_int4(cache, bounds, table, length)
            pause()
            results.append(package.paged_decode_attention_int4(queries[step], cache, table, length))
            if between == "bounds":
                results.append(package.sparse_decode_attention_int4(queries[step], cache, bounds, table, length, num_pages=4)[1])
            pause()
        return results

    want = run(True)
    for _ in range(3):
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = run(False)
            graph.replay()
        else:
            got = run(False)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))

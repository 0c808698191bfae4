"""Attention over the 4-bit cache held to a bound per channel, and caches in which every 32 tokens show in the result:
a piece of a row that is lost, or counted twice, is then far outside that bound."""

from __future__ import annotations

import torch

import int4_plain as plain

UNIT = 32  # tokens that a warp takes at a time


def weighted(q, k, v, tokens, scale):
    """One (sequence, KV head) in 64 bits: q [group, D], k and v [tokens, D] as read back -> (out, spread, size, reach,
    tail), [group, D] or [group, 1]: the result; sum of weight * (value - its group's smallest); sum of weight * the
    group's largest |value|; what scores can reach; what fp16 weights below 2^-14 are off by at most."""
    q, k, v = q.double(), k[:tokens].double(), v[:tokens].double()
    scores = q @ k.T * scale
    w = torch.softmax(scores, -1)
    groups = v.unflatten(-1, (-1, 32))
    low, high = groups.amin(-1, keepdim=True), groups.amax(-1, keepdim=True)
    every = lambda x: x.expand_as(groups).flatten(-2)  # noqa: E731
    size = w @ every(groups.abs().amax(-1, keepdim=True))
    # scores: |q| times the largest |k| of every group
    reach = (q.unflatten(-1, (-1, 32)).abs().sum(-1) @ k.unflatten(-1, (-1, 32)).abs().amax(-1).T).amax(-1, keepdim=True) * abs(scale)
    tail = tokens * 2.0 ** -30 * float((high - low).max()) * w.amax(-1, keepdim=True)
    return w @ v, w @ (v - every(low)), size, reach, tail


def bound(dtype, out, spread, size, reach, tail):
    """Per channel: half a step of the result's type; 2^-11 of every weight * step * code, as fp16 holds weight * step
    (steps times codes are values less their group's smallest); the scores' error, two terms of 2^-22 in their
    floors and fp32 sums, 2^-20 of what they reach, in the weights and in their sum; 2^-16 for exponentials, quotient
    and the fp32 sums of fewer than 100 products; the tail."""
    return torch.finfo(dtype).eps / 2 * out.abs() + 2.0 ** -11 * spread + (2.0 ** -19 * reach + 2.0 ** -16) * size + tail + 1e-30


def expected(q, pool, table, lens, scale=None, device="cpu"):
    """(out, allowed), both float64 [B, Hq, D], for a table [B, n] without bad pages."""
    k, v = (x.to(device) for x in plain.rows(pool, q.dtype))
    page, heads = k.shape[1], k.shape[2]
    group = q.shape[1] // heads
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, allowed = (torch.zeros(q.shape, dtype=torch.float64, device=device) for _ in range(2))
    for b, n in enumerate(lens.tolist()):
        if n == 0:
            continue
        ids = table[b, : -(-n // page)].long().to(device)
        for h in range(heads):
            mine = slice(h * group, (h + 1) * group)
            parts = weighted(q[b, mine].to(device), k[ids, :, h].flatten(0, 1), v[ids, :, h].flatten(0, 1), n, scale)
            out[b, mine], allowed[b, mine] = parts[0], bound(q.dtype, *parts)
    return out.cpu(), allowed.cpu()


def worst(actual, out, allowed):
    """The largest error as a share of what is allowed."""
    return ((actual.double().cpu() - out).abs() / allowed).max().item()


def counted(lengths, *, dtype, dim, heads, group, page, seed=0, skip=None):
    """A cache whose keys are all zero and whose tokens of unit u have V = 1 in channel u % D of an order that
    depends on the sequence and head, 0 elsewhere: a channel of the result is the share of the tokens in its units.
    Queries are ordinary, scores all zero.  `skip`: (sequence, unit) whose tokens have V = 0."""
    q, pool, table, lens = plain.make_cache(lengths, dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=seed)
    g = torch.Generator().manual_seed(seed)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        token = torch.arange(n)
        v = torch.zeros(n, heads, dim)
        for h in range(heads):
            order = torch.randperm(dim, generator=g)
            v[token, h, order[token // UNIT % dim]] = 1.0
        if skip is not None and skip[0] == b:
            v[UNIT * skip[1]: UNIT * skip[1] + UNIT] = 0
        plain.store_fast(pool, table[b, token // page].long() * page + token % page, torch.zeros(n, heads, dim).to(dtype), v.to(dtype))
    return q, pool, table, lens


def signed(n, *, dtype, dim, heads, group, page, seed=0):
    """One sequence whose units have keys of random signs, one pattern a unit, and V of their own; a query that is a
    unit's pattern gives that unit nearly all of the weight.  Returns (patterns [units, heads, D], pool, table, lens)."""
    _, pool, table, lens = plain.make_cache([n], dtype=dtype, dim=dim, heads=heads, group=group, page=page, seed=seed)
    g = torch.Generator().manual_seed(seed)
    units = -(-n // UNIT)
    patterns = torch.randint(0, 2, (units, heads, dim), generator=g).float() * 2 - 1
    token = torch.arange(n)
    v = torch.randn(units, heads, dim, generator=g)[token // UNIT] + 0.2 * torch.randn(n, heads, dim, generator=g)
    plain.store_fast(pool, table[0, token // page].long() * page + token % page, patterns[token // UNIT].to(dtype), v.to(dtype))
    return patterns, pool, table, lens

"""CPU tests that the bound of int4_pieces sees what it is for: a result without one unit, or with one unit
twice, is far outside it at every length the GPU tests use."""

from __future__ import annotations

import pytest
import torch

import int4_pieces as pieces
import int4_plain as plain


def _units_of(n):
    units = -(-n // pieces.UNIT)
    return sorted({0, 1, units // 3, units // 2, units - 2, units - 1} & set(range(units)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 513, 3000, 40000])
def test_a_lost_or_doubled_unit_is_outside_the_bound(dtype, n):
    q, pool, table, lens = pieces.counted([n], dtype=dtype, dim=128, heads=1, group=2, page=16)
    out, allowed = pieces.expected(q, pool, table, lens)
    assert pieces.worst(out.to(dtype), out, allowed) <= 1.0
    k, v = (x[table[0].long(), :, 0].flatten(0, 1)[:n] for x in plain.rows(pool, dtype))
    for unit in _units_of(n):
        rows = torch.arange(n)
        inside = rows // pieces.UNIT == unit
        for mine in (rows[~inside], torch.cat([rows, rows[inside]])):
            wrong = pieces.weighted(q[0], k[mine], v[mine], len(mine), 128 ** -0.5)[0][None]
            assert pieces.worst(wrong.to(dtype), out, allowed) > 4.0, unit


@pytest.mark.parametrize("n", [513, 3000])
def test_a_lost_unit_that_holds_the_weight_is_outside_the_bound(n):
    patterns, pool, table, lens = pieces.signed(n, dtype=torch.float16, dim=128, heads=1, group=1, page=16)
    k, v = (x[table[0].long(), :, 0].flatten(0, 1)[:n] for x in plain.rows(pool, torch.float16))
    rows = torch.arange(n)
    for unit in _units_of(n):
        q = patterns[unit][None].half()
        out, allowed = pieces.expected(q, pool, table, lens, 0.25)
        mine = rows[rows // pieces.UNIT != unit]
        wrong = pieces.weighted(q[0], k[mine], v[mine], len(mine), 0.25)[0][None]
        assert pieces.worst(out.half(), out, allowed) <= 1.0 and pieces.worst(wrong.half(), out, allowed) > 20.0

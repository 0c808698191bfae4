"""CPU tests of the 4-bit cache: refusals before any device work, struct layout, and the plain
codec the GPU tests compare with."""

from __future__ import annotations

import ctypes
import shutil
import subprocess

import pytest
import torch

import int4_plain as plain
from conftest import REPO_ROOT


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_structs_match_c_layout(package, tmp_path):
    structs = {"qf_int4_write_args": package.cabi.Int4WriteArgs, "qf_paged_int4_args": package.cabi.PagedInt4Args}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "qf_hotpath.h"', "int main(void) {"]
    for struct, cls in structs.items():
        lines.append(f'printf("{struct} %zu\\n", sizeof({struct}));')
        lines += [f'printf("{struct}.{name} %zu\\n", offsetof({struct}, {name}));' for name, _ in cls._fields_]
    source, binary = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run(["gcc", "-I", str(REPO_ROOT / "include"), str(source), "-o", str(binary)], check=True)
    reported = dict(line.split() for line in subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.splitlines())
    for struct, cls in structs.items():
        assert int(reported[struct]) == ctypes.sizeof(cls)
        for name, _ in cls._fields_:
            assert int(reported[f"{struct}.{name}"]) == getattr(cls, name).offset, (struct, name)


def test_packed_arguments_are_the_structures_bytes(package):
    cabi = package.cabi
    for cls, pack in ((cabi.Int4WriteArgs, cabi.pack_int4_write), (cabi.PagedInt4Args, cabi.pack_paged_int4)):
        values = [(i * 37 + 5) / 4 if kind in (ctypes.c_float, ctypes.c_double) else i * 1000003 + 1 for i, (_, kind) in enumerate(cls._fields_)]
        assert pack(*values) == bytes(cls(*values)) and len(pack(*values)) == ctypes.sizeof(cls)


def _write_args(cabi, **changes):
    args = cabi.Int4WriteArgs()
    values = dict(rows=1, q_heads=0, kv_heads=2, head_dim=128, page_size=16, dtype=0, k=16, v=16, pool=16, num_pages=4, base=1e6)
    for name, value in {**values, **changes}.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("changes, message", [
    (dict(head_dim=96), b"64 or 128"), (dict(page_size=24), b"multiple of 16"), (dict(page_size=0), b"multiple of 16"),
    (dict(dtype=2), b"float16 or bfloat16"), (dict(kv_heads=0), b"head counts"), (dict(rows=-1), b"rows"),
    (dict(k=None), b"must not be null"), (dict(pool=8), b"aligned"), (dict(q_heads=4), b"q and q_out"),
    (dict(positions=16, positions_dtype=3), b"positions"), (dict(positions=16, positions_dtype=2, rope_table=16, table_positions=4), b"positions"),
    (dict(positions=16, base=0.0), b"base"), (dict(positions=16, rope_table=16), b"table is empty"),
    (dict(slot_mapping=16, slot_dtype=2), b"slot mapping"), (dict(num_pages=-1), b"2^31 slots"), (dict(num_pages=1 << 27), b"2^31 slots"), (dict(rows=(1 << 31) - 1), b"too many rows"),
])
def test_write_refusals(package, changes, message):
    lib = package.cabi.library()
    assert lib.qf_int4_rope_kv_write(ctypes.byref(_write_args(package.cabi, **changes)), None) == -1
    assert message in lib.qf_last_error()


def test_nothing_to_do_launches_nothing(package):
    cabi, lib = package.cabi, package.cabi.library()
    assert lib.qf_int4_rope_kv_write(ctypes.byref(_write_args(cabi, rows=0, k=None)), None) == 0
    assert lib.qf_int4_read_rows(None, 4, 16, 2, 128, 0, None, 0, 0, 0, None, None, None) == 0
    args = _paged_args(cabi, batch=0)
    for name in ("qf_int4_decode_attention", "qf_int4_key_bounds", "qf_select_kv_pages", "qf_int4_sparse_decode_attention"):
        assert getattr(lib, name)(ctypes.byref(args), None) == 0, name
    for name in ("qf_int4_rope_kv_write", "qf_int4_decode_attention", "qf_select_kv_pages"):
        assert getattr(lib, name)(None, None) == -1


def test_read_refusals(package):
    lib = package.cabi.library()
    read = lambda pool=16, pages=4, page=16, heads=2, dim=128, dtype=0, slots=16, code=0, rows=1, k=16, v=16: (  # noqa: E731
        lib.qf_int4_read_rows(pool, pages, page, heads, dim, dtype, slots, code, 1, rows, k, v, None))
    for changes, message in ((dict(dim=80), b"64 or 128"), (dict(dtype=5), b"float16 or bfloat16"), (dict(code=2), b"slot mapping"),
                             (dict(pool=None), b"must not be null"), (dict(k=8), b"aligned"), (dict(rows=-1), b"geometry")):
        assert read(**changes) == -1 and message in lib.qf_last_error(), changes


def _paged_args(cabi, **changes):
    args = cabi.PagedInt4Args()
    values = dict(batch=2, q_heads=12, kv_heads=2, head_dim=128, page_size=16, dtype=0, q=16, out=16, pool=16, key_bounds=16,
                  block_table=16, seq_lens=16, workspace=16, page_table=16, page_lens=16, num_pages=4, table_width=8, take=2, new_tokens=1)
    for name, value in {**values, **changes}.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("changes, message", [
    (dict(head_dim=256), b"64 or 128"), (dict(page_size=20), b"multiple of 16"), (dict(dtype=-1), b"float16 or bfloat16"),
    (dict(q_heads=13), b"divisible"), (dict(q_heads=34), b"at most 16"), (dict(q_heads=0), b"divisible"),
    (dict(batch=-1), b"batch"), (dict(q=None), b"aligned"), (dict(q=8), b"aligned"), (dict(q_stride_b=4), b"multiple of 8"),
    (dict(out=None), b"out must"), (dict(pool=8), b"pool must"), (dict(seq_lens=None), b"must not be null"),
    (dict(block_table=None), b"must not be null"), (dict(table_dtype=2), b"page table"), (dict(lens_dtype=2), b"lengths"),
    (dict(table_width=1 << 28), b"2^30 tokens"), (dict(table_width=(1 << 26) - 1, batch=16), b"2^30 tiles"), (dict(take=1 << 26), b"2^30 tokens"), (dict(num_pages=1 << 31), b"pool or table size"),
    (dict(take=0), b"at least one page"), (dict(page_table=None), b"page_table"), (dict(key_bounds=None), b"key bounds"),
    (dict(workspace=None), b"workspace"), (dict(workspace_bytes=8), b"workspace"),
])
def test_paged_refusals(package, changes, message):
    lib = package.cabi.library()
    args = _paged_args(package.cabi, **changes)
    assert lib.qf_int4_sparse_decode_attention(ctypes.byref(args), None) != 0
    # without a GPU the status word has no address, which is the last of the checks before the workspace's
    assert message in lib.qf_last_error() or b"status word" in lib.qf_last_error() and "workspace" in str(changes), lib.qf_last_error()


def test_workspace_sizes(package):
    cabi, lib = package.cabi, package.cabi.library()
    size = ctypes.c_int64(-1)
    assert lib.qf_paged_int4_workspace(ctypes.byref(_paged_args(cabi)), 7, ctypes.byref(size)) == -1
    assert lib.qf_paged_int4_workspace(None, 0, ctypes.byref(size)) == -1
    assert lib.qf_paged_int4_workspace(ctypes.byref(_paged_args(cabi)), cabi.INT4_SELECT, ctypes.byref(size)) == 0
    assert size.value == 2 * 2 * 8 * 4  # a 32-bit key for every page of every row

    def attention(**changes):
        assert lib.qf_paged_int4_workspace(ctypes.byref(_paged_args(cabi, **changes)), cabi.INT4_ATTENTION, ctypes.byref(size)) == 0
        return size.value

    # none for short tables, whatever the batch up to a row an SM; never more for a smaller call than for a larger one
    assert attention(table_width=48) == attention(batch=74, table_width=48) == attention(table_width=0) == attention(batch=0) == 0
    for sizes in (dict(head_dim=128), dict(head_dim=64), dict(head_dim=128, q_heads=20), dict(head_dim=64, q_heads=32)):
        bytes_of = [[attention(batch=b, table_width=w, **sizes) for w in (1, 16, 32, 33, 48, 49, 64, 65, 200, 2048)] for b in (1, 8, 40, 74, 75, 300)]
        for rows in (*bytes_of, *zip(*bytes_of)):
            assert list(rows) == sorted(rows)


def test_wrappers_refuse_before_any_device_work(package):
    pool = torch.zeros(4, 2, 1, 2560, dtype=torch.uint8)
    q, table, lens = torch.zeros(2, 12, 128, dtype=torch.float16), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    bounds = torch.zeros(4, 2, 2, 128, dtype=torch.float16)
    packed, index = torch.zeros(2, 2048, dtype=torch.float16), torch.zeros(2, dtype=torch.int64)
    heads = q[:, :, None]
    calls = [lambda: package.paged_decode_attention_int4(q, pool, table, lens), lambda: package.read_kv_int4(pool, index),
             lambda: package.packed_qkv_rope_cache_int4(packed, index, index, pool),
             lambda: package.native_decode_rope_kv_write_int4(heads, heads[:, :2], heads[:, :2], index, index, pool),
             lambda: package.rope_kv_write_int4(q[None].transpose(1, 2), q[None, :, :2].transpose(1, 2), q[None, :, :2].transpose(1, 2), index, index, pool),
             lambda: package.update_key_bounds_int4(pool, bounds, table, lens),
             lambda: package.select_kv_pages(q, bounds, table, lens, num_pages=1),
             lambda: package.sparse_decode_attention_int4(q, pool, bounds, table, lens, num_pages=1),
             lambda: package.dequantize_kv_pool_int4(pool), lambda: package.empty_key_bounds_int4(pool, torch.float16),
             lambda: package.quantize_kv_pool_int4(torch.zeros(4, 16, 2, 128, dtype=torch.float16), torch.zeros(4, 16, 2, 128, dtype=torch.float16))]
    for call in calls:
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for bad in (pool.float(), pool[..., :2000], pool[0]):
        with pytest.raises(ValueError, match="4-bit pool"):
            package.paged_decode_attention_int4(q, bad, table, lens)
    for arguments in (dict(head_dim=96), dict(head_dim=128, page_size=8)):
        with pytest.raises(ValueError):
            package.empty_kv_pool_int4(4, 2, **arguments)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_plain_codec(dtype, dim):
    """The codec the GPU tests hold the kernels to: the two layouts agree, and a value is off by half a step
    and what rounding the step to the type can add: 15 half units in its last place."""
    g = torch.Generator().manual_seed(3)
    k, v = ((torch.randn(40, 2, dim, generator=g) * 3).to(dtype) for _ in range(2))
    k[5, 0, 3], v[6, 1, dim - 1], k[7] = float("inf"), float("nan"), 1.25
    slots = torch.randperm(96, generator=g)[:40]
    one, two = (torch.zeros(3, 2, 2, 20 * dim, dtype=torch.uint8) for _ in range(2))
    plain.store(one, slots, k, v)
    plain.store_fast(two, slots, k, v)
    assert torch.equal(one, two)
    for x, back in zip((k, v), plain.rows(one, dtype)):
        back = back.reshape(-1, 2, dim)[slots]
        group = x.float().unflatten(-1, (-1, 32))
        finite = torch.isfinite(group).all(-1, keepdim=True).expand_as(group).flatten(-2)
        step = ((group.amax(-1) - group.amin(-1)) / 15).repeat_interleave(32, -1)
        limit = step * (0.5 + 15 * torch.finfo(dtype).eps / 2) + 1e-6
        assert ((back - x.float()).abs() <= limit)[finite].all() and torch.isnan(back)[~finite].all()
    assert (plain.rows(one, dtype)[0].reshape(-1, 2, dim)[slots[7]] == 1.25).all()

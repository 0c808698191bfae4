"""CPU tests of what the 4-bit calls promise beside their results: what their kernels may assume of memory,
what a C caller may pass, and how the package hands its functions out."""

from __future__ import annotations

import ctypes
import re

import pytest

from conftest import REPO_ROOT

SOURCES = ("qf_int4_kv.cu", "qf_int4_attention.cu", "qf_kv_select.cu")


@pytest.mark.parametrize("name", SOURCES)
def test_chained_kernels_promise_nothing_about_memory(name):
    """A kernel that is resident while the one in front still writes must not declare its memory unchanging."""
    text = (REPO_ROOT / "qwen-frence_b200" / "csrc" / name).read_text()
    kernels = re.findall(r"__global__[^{;]*\{", text)
    assert kernels
    assert not [k for k in kernels if "__restrict__" in k]
    assert "ld.global.nc" not in text and "__ldg(" not in text


def _sparse_args(cabi, **changes):
    args = cabi.PagedInt4Args()
    values = dict(batch=2, q_heads=12, kv_heads=2, head_dim=128, page_size=16, q=16, out=16, pool=16, key_bounds=16, block_table=16, seq_lens=16,
                  workspace=16, workspace_bytes=1 << 30, page_table=16, page_lens=16, num_pages=4, table_width=8, take=2, new_tokens=1)
    for name, value in {**values, **changes}.items():
        setattr(args, name, value)
    return args


@pytest.mark.parametrize("name", ["qf_int4_decode_attention", "qf_select_kv_pages", "qf_int4_sparse_decode_attention"])
@pytest.mark.parametrize("workspace", [8, 24, 17])
def test_workspaces_are_aligned(package, name, workspace):
    """Kernels store 16 bytes at a time into it."""
    lib = package.cabi.library()
    assert getattr(lib, name)(ctypes.byref(_sparse_args(package.cabi, workspace=workspace)), None) == -1
    assert b"workspace" in lib.qf_last_error() and b"aligned" in lib.qf_last_error()


@pytest.mark.parametrize("changes", [dict(block_table=18), dict(table_dtype=1, block_table=20), dict(seq_lens=18), dict(lens_dtype=1, seq_lens=20),
                                     dict(page_table=18), dict(page_lens=18)])
def test_tables_and_lengths_are_aligned_to_their_elements(package, changes):
    lib = package.cabi.library()
    assert lib.qf_int4_sparse_decode_attention(ctypes.byref(_sparse_args(package.cabi, **changes)), None) == -1
    assert b"aligned" in lib.qf_last_error()


def test_inputs_of_reads_and_writes_are_aligned_to_their_elements(package):
    cabi, lib = package.cabi, package.cabi.library()
    for slots, code in ((18, 0), (20, 1)):
        assert lib.qf_int4_read_rows(16, 4, 16, 2, 128, 0, slots, code, 1, 1, 16, 16, None) == -1
        assert b"slots must be aligned" in lib.qf_last_error()
    for changes in (dict(k=17), dict(v=17), dict(positions=18), dict(positions=20, positions_dtype=1), dict(slot_mapping=18),
                    dict(slot_mapping=20, slot_dtype=1), dict(valid_tokens=18), dict(q_heads=2, q=17, q_out=16), dict(q_heads=2, q=16, q_out=17)):
        args = cabi.Int4WriteArgs()
        for name, value in {**dict(rows=1, kv_heads=2, head_dim=128, page_size=16, k=16, v=16, pool=16, num_pages=4, base=1e6), **changes}.items():
            setattr(args, name, value)
        assert lib.qf_int4_rope_kv_write(ctypes.byref(args), None) == -1
        assert b"aligned to their elements" in lib.qf_last_error(), changes


@pytest.mark.parametrize("name, module", [("rms_norm", "fused_rms"), ("packed_qkv_rope_cache", "packed_qkv_rope_cache"),
                                          ("paged_decode_attention_int4", "int4_paged_kv")])
def test_the_package_hands_out_what_its_modules_hold(package, monkeypatch, name, module):
    """A function replaced on a drop-in module is the package's, before and after."""
    before = getattr(package, name)
    stand_in = object()
    monkeypatch.setattr(package.kernel_module(module), name, stand_in)
    assert getattr(package, name) is stand_in
    monkeypatch.undo()
    assert getattr(package, name) is before is getattr(package.kernel_module(module), name)


def test_sparse_attention_refuses_a_negative_scale(package):
    """Its pages are those of the largest q . k, which a negative scale would make the smallest scores."""
    lib = package.cabi.library()
    assert lib.qf_int4_sparse_decode_attention(ctypes.byref(_sparse_args(package.cabi, scale=-0.1)), None) == -1
    assert b"scale" in lib.qf_last_error()
    assert lib.qf_int4_sparse_decode_attention(ctypes.byref(_sparse_args(package.cabi, batch=0, scale=0.0)), None) == 0

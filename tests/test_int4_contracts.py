"""CPU tests of what the 4-bit calls promise beside their results: what their kernels may assume of memory,
what a C caller may pass, and how the package hands its functions out."""

from __future__ import annotations

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

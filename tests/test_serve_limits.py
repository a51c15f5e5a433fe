"""Sizes that the packed and cache calls plan and check by."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys

import pytest
import torch

from quantumdlblocks_amd import (
    _native,
    born_cache_evict,
    flash_born_attention_packed,
    flash_born_attention_paged,
    fused_qk_rope_l2_normalize_append,
)
from quantumdlblocks_amd.kernels import flash_born_packed as packed
from test_cache import _append_block, _evict_block, _paged_block


def test_a_windows_workspace_does_not_grow_with_the_table():
    size = _native.load().qdl_flash_born_paged_workspace_size
    # 32 sequences of 32 heads over 8, D128, pages of 16, the weights kept.
    near, far = (size(32, 32, 8, 128, pages, 16, 512, 1) for pages in (64, 8192))
    assert near == far < 16 << 20
    assert size(32, 32, 8, 128, 8192, 16, 0, 1) > size(32, 32, 8, 128, 64, 16, 0, 1)  # without one it has to


def test_windows_past_every_key_are_cut(monkeypatch):
    # As the paged call cuts them: a caller's "no window" may be any large number.
    seen = []
    monkeypatch.setattr(packed, "_eager_packed", lambda *a: seen.append(a[8]))
    x = torch.rand(3, 1, 8)
    for window in (sys.maxsize, 1 << 31, (1 << 30) + 1, 1 << 30, 5, -1):
        flash_born_attention_packed(x, x, x, 1.0, torch.tensor([0, 3]), window_size=window)
    assert seen == [1 << 30] * 4 + [5, 0]


MASK = """
#include <initializer_list>
#include "%s"
using namespace qdl;
// In a constant expression an overflow of a signed sum is a compile error.
constexpr bool agree(bool causal, int64_t window) {
    const int lower = packed_lower(causal), upper = packed_upper(window);
    const uint32_t span = packed_span(lower, upper);
    // The farthest positions of 2^28 queries and keys, and those next to the bounds.
    for (int lag : {-(1 << 29), -1, 0, 1, 99, 100, 101, (1 << 29)})
        if (((uint32_t)(lag - lower) < span) != ((!causal || lag >= 0) && (window <= 0 || lag < window))) return false;
    return true;
}
static_assert(agree(false, 0) && agree(true, 0) && agree(false, 100) && agree(true, 100) && agree(false, 1 << 30) && agree(true, 1 << 30), "mask");
static_assert(packed_span(packed_lower(false), packed_upper(0)) == 0x80000000u, "both bounds far away");
int main() {}
""" % os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quantumdlblocks_amd", "csrc", "packed_mask.h")


def test_the_masks_span_does_not_overflow(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    (tmp_path / "mask.cpp").write_text(MASK)
    subprocess.run([gxx, "-std=c++17", "-fsyntax-only", str(tmp_path / "mask.cpp")], check=True)


@pytest.mark.parametrize("pages,page", [(1 << 40, 1 << 24), (1 << 62, 4), ((1 << 63) - 1, 2), ((1 << 30) + 1, 1)])
def test_tables_whose_keys_leave_64_bits(pages, page):
    # The product that is checked wraps to a small number.
    lib = _native.load()
    over = dict(pages=pages, page=page, ld=(1 << 63) - 1)
    assert lib.qdl_flash_born_paged_forward_call(_paged_block(**over, ws_bytes=1 << 60), None) == -15
    assert lib.qdl_flash_born_cache_append_call(_append_block(**over), None) == -15
    assert lib.qdl_flash_born_cache_evict_call(_evict_block(**over), None) == -15
    assert lib.qdl_flash_born_paged_workspace_size(2, 4, 2, 64, pages, page, 0, 1) == 0


def test_one_tensor_as_both_caches():
    # Read and moved to other pages it may be both; two writers of one row it may not.
    c = torch.rand(6, 4, 1, 8)
    table, lens, to = torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([6], dtype=torch.int32), torch.tensor([[3]], dtype=torch.int32)
    x, w = torch.rand(1, 1, 8), torch.rand(1, 1, 8)
    flash_born_attention_paged(x, c, c, table, lens, 1.0)
    before = c.clone()
    with pytest.raises(ValueError, match="share"):
        fused_qk_rope_l2_normalize_append(x, x, 2 * x, None, None, c, c, table, lens)
    with pytest.raises(ValueError, match="share"):
        born_cache_evict(c, c, table, lens, w, 3)
    assert torch.equal(c, before)
    _, _, kept = born_cache_evict(c, c, table, lens, w, 3, 0, to)
    assert torch.equal(c[3, :3], before[:2].flatten(0, 1)[kept[0, 0].long()])
    none = torch.rand(0, 4, 1, 8)  # nothing to share
    fused_qk_rope_l2_normalize_append(x, x, x, None, None, none, none, table, lens)

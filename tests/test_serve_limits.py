"""Sizes that the packed and cache calls plan and check by."""

from __future__ import annotations

from quantumdlblocks_amd import _native


def test_a_windows_workspace_does_not_grow_with_the_table():
    size = _native.load().qdl_flash_born_paged_workspace_size
    # 32 sequences of 32 heads over 8, D128, pages of 16, the weights kept.
    near, far = (size(32, 32, 8, 128, pages, 16, 512, 1) for pages in (64, 8192))
    assert near == far < 16 << 20
    assert size(32, 32, 8, 128, 8192, 16, 0, 1) > size(32, 32, 8, 128, 64, 16, 0, 1)  # without one it has to

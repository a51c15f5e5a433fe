"""Sizes that the packed and cache calls plan and check by."""

from __future__ import annotations

import sys

import torch

from quantumdlblocks_amd import _native, flash_born_attention_packed
from quantumdlblocks_amd.kernels import flash_born_packed as packed


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

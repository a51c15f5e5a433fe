"""Windows over caches much longer than they are, with the keys' weights kept:
the raw weights' workspace spans the window only."""

from __future__ import annotations

import sys

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import flash_born_attention_packed, flash_born_attention_paged
from test_cache import make_cache

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("window", [1, 31, 300, 1025, 2999])
@pytest.mark.parametrize("page,H,Hkv", [(16, 4, 2), (24, 3, 1), (7, 20, 1)])
def test_weights_of_a_window(cuda_device, dtype, window, page, H, Hkv):
    lens, D, dt = [3000, 700, 0, 301], 64, DT[dtype]
    kc, vc, table, n, _ = make_cache(lens, page, Hkv, D, torch.float32, 25)
    kc = torch.nn.functional.normalize(kc + 0.1, dim=-1)
    q = torch.nn.functional.normalize(torch.randn(4, H, D, generator=torch.Generator().manual_seed(26)) + 0.1, dim=-1)
    q, kc, vc = (x.to(device=cuda_device, dtype=dt) for x in (q, kc, vc))
    weight = torch.full((4, Hkv, 2900), 0.5, device=cuda_device)  # narrower than the longest cache
    out = flash_born_attention_paged(q, kc, vc, table.to(cuda_device), n.to(cuda_device), 2.0, 1e-12, window, weight)
    o, w = ref.paged(q, kc, vc, table, n, 2.0, 1e-12, window)
    assert ref.worst(out, o) <= 1.0
    x, e = w[0][..., :2900] + 0.5, w[1][..., :2900] + 2.0 ** -24 * 2.0 * (w[0][..., :2900] + 0.5)
    assert ref.worst(weight, (x, e)) <= 1.0
    for b, m in enumerate(lens):  # nothing is added outside the windows
        assert (weight[b, :, : max(0, m - window)] == 0.5).all() and (weight[b, :, m:] == 0.5).all()


def test_packed_windows_past_every_key(cuda_device):
    g = torch.Generator().manual_seed(27)
    q, k, v = (torch.randn(90, h, 64, generator=g).to(device=cuda_device, dtype=torch.bfloat16) for h in (4, 2, 2))
    cu = torch.tensor([0, 20, 90], dtype=torch.int32, device=cuda_device)
    want = flash_born_attention_packed(q, k, v, 1.0, cu)
    for window in (90, 1 << 30, 1 << 31, sys.maxsize):
        assert torch.equal(flash_born_attention_packed(q, k, v, 1.0, cu, window_size=window), want)

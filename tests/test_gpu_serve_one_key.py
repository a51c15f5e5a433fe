"""Rows that one key takes whole are that key's values: what rounds a weight is in
the numerator and in the denominator."""

from __future__ import annotations

import pytest
import torch

from quantumdlblocks_amd import flash_born_attention_packed, flash_born_attention_paged

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("n", [200, 3000])  # blocks whose waves share rows, and whole ones
def test_packed_rows_of_one_key(cuda_device, dtype, D, n):
    g = torch.Generator().manual_seed(50)
    q, k, v = (torch.randn(n, h, D, generator=g).abs().to(device=cuda_device, dtype=DT[dtype]) for h in (16, 8, 8))
    cu = torch.arange(n + 1, dtype=torch.int32, device=cuda_device)
    one = v.repeat_interleave(2, 1)
    for kw in (dict(cu_seqlens_q=cu), dict(cu_seqlens_q=cu[[0, n]], window_size=1)):
        out = flash_born_attention_packed(q, k, v, 0.3, eps=0.0, **kw)
        if dtype == "fp32":  # the product, the reciprocal and its product
            assert ((out - one).abs() <= 2.0 ** -22 * one.abs()).all()
        else:
            assert torch.equal(out, one)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1])
def test_paged_rows_of_one_key(cuda_device, dtype, D, window):
    g = torch.Generator().manual_seed(51)
    B, page = 64, 16
    kc, vc, q = (torch.randn(*s, generator=g).abs().to(device=cuda_device, dtype=DT[dtype]) for s in
                 ((B, page, 2, D), (B, page, 2, D), (B, 4, D)))
    table = torch.arange(B, dtype=torch.int32, device=cuda_device).view(B, 1)
    n = 10 if window else 1
    out = flash_born_attention_paged(q, kc, vc, table, torch.full((B,), n, dtype=torch.int32, device=cuda_device), 0.3, 0.0, window)
    one = vc[:, n - 1].repeat_interleave(2, 1)
    if dtype == "fp32":
        assert ((out - one).abs() <= 2.0 ** -22 * one.abs()).all()
    else:
        # The two parts leave 2^-16 (bf16) or 2^-22 of a weight out, well under half a step.
        assert torch.equal(out, one)

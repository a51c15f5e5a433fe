"""Attention of one token in 16 bits: the weights keep 16 bits and more, so that an
output is off by its own rounding and what fp32 costs."""

from __future__ import annotations

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import flash_born_attention_paged
from test_cache import make_cache

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,Hkv,page", [(4, 2, 16), (32, 1, 24)])
@pytest.mark.parametrize("lens", [[200, 3, 90], [4000, 1100]])
def test_only_the_output_is_rounded(cuda_device, dtype, D, H, Hkv, page, lens):
    dt, u = DT[dtype], ref.HALF_STEP[DT[dtype]]
    kc, vc, table, n, _ = make_cache(lens, page, Hkv, D, torch.float32, 48)
    kc = torch.nn.functional.normalize(kc + 0.1, dim=-1)
    q = torch.nn.functional.normalize(torch.randn(len(lens), H, D, generator=torch.Generator().manual_seed(49)) + 0.1, dim=-1)
    q, kc, vc = (x.to(dt) for x in (q, kc, vc))
    out = flash_born_attention_paged(*(x.to(cuda_device) for x in (q, kc, vc, table, n)), 2.0)
    # An fp32 kernel's bound on the same values; the two parts of a weight, the
    # second rounded to half a step of a half step; the output's rounding.
    (x, e), _ = ref.paged(*(t.float() for t in (q, kc, vc)), table, n, 2.0)
    e = e + 1.1 * u * u * vc.abs().max() + 1.02 * u * x.abs()
    if dtype == "fp16":  # its smallest step in a weight's second part, under a largest weight of at least 64^2; in the output
        e = e + 2.0 ** -25 / 4096 * max(lens) * vc.abs().max() + 2.0 ** -25
    assert ref.worst(out, (x, e)) <= 1.0

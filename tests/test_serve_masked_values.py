"""What the CPU formulas make of infinities and NaN where nothing is seen, of
autocast, and of batches without sequences."""

from __future__ import annotations

import pytest
import torch

from quantumdlblocks_amd import fused_qk_rope_l2_normalize_append

BAD = [float("nan"), float("inf"), -float("inf")]


def _cache(lens=(2,), page=4, Hkv=1, D=8):
    g = torch.Generator().manual_seed(0)
    kc, vc = (torch.rand(4, page, Hkv, D, generator=g) for _ in range(2))
    table = torch.arange(2 * len(lens), dtype=torch.int32).view(len(lens), 2)
    return kc, vc, table, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.parametrize("bad", BAD)
def test_tokens_of_no_sequence_are_zero_queries(bad):
    kc, vc, table, lens = _cache()
    q = torch.rand(4, 2, 8)
    q[2:] = bad
    cu = torch.tensor([0, 2], dtype=torch.int32)
    out = fused_qk_rope_l2_normalize_append(q, q[:, :1], q[:, :1], None, None, kc, vc, table, lens, cu)
    assert not out[2:].any() and out[:2].isfinite().all() and kc.isfinite().all() and vc.isfinite().all()
    zero = torch.zeros(3, 2, 8)  # 0 / 0 in rows that no sequence owns
    out = fused_qk_rope_l2_normalize_append(zero, zero[:, :1], zero[:, :1], None, None, kc, vc, table, lens * 0,
                                            torch.tensor([0, 0]), eps=0.0)
    assert not out.any() and not out.isnan().any()

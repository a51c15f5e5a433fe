"""A compiler that traces a caller leaves the cache operators alone: their calls
take the device, the stream and the addresses of the moment."""

from __future__ import annotations

import pytest
import torch

from quantumdlblocks_amd import born_cache_evict, flash_born_attention_paged, fused_qk_rope_l2_normalize_append
from quantumdlblocks_amd.kernels import born_cache


@pytest.fixture
def traced(monkeypatch):
    """Whether each call's checks were traced."""
    seen = []
    check = born_cache._check_cache

    def look(*a, **kw):
        seen.append(torch.compiler.is_compiling())
        return check(*a, **kw)

    monkeypatch.setattr(born_cache, "_check_cache", look)
    torch._dynamo.reset()
    return seen


def test_cache_operators_run_untraced(traced):
    kc, vc = torch.rand(3, 4, 1, 8), torch.rand(3, 4, 1, 8)
    table, lens = torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([6], dtype=torch.int32)

    def step(x, kc, vc):
        q = fused_qk_rope_l2_normalize_append(2 * x, x, x, None, None, kc, vc, table, lens)
        weight = torch.zeros(1, 1, 8)
        out = flash_born_attention_paged(q, kc, vc, table, lens, 1.0, key_weight=weight)
        new, weight, kept = born_cache_evict(kc, vc, table, lens, weight, 4, 1)
        return out + 1, new, weight, kept, kc, vc

    x = torch.rand(1, 1, 8)
    with torch.no_grad():
        want = step(x, kc.clone(), vc.clone())
        got = torch.compile(step, backend="eager")(x, kc.clone(), vc.clone())
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert traced == [False] * 6

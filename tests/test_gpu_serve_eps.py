"""The smallest eps, where its reciprocal leaves fp32's range: rows that see
nothing, or whose overlaps are all negative, are zeros and have zero gradients."""

from __future__ import annotations

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import flash_born_attention_packed, flash_born_attention_paged
from test_cache import make_cache

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = torch.finfo(torch.float32).tiny
EPS = [TINY, 8 * TINY, 2.0 ** -149, 0.0]


def _cu(c, dev):
    return torch.tensor(c, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,H", [(64, 2), (128, 2), (256, 2), (64, 12)])
@pytest.mark.parametrize("eps", EPS)
def test_packed_rows_without_weight(cuda_device, dtype, D, H, eps):
    # Fewer keys than queries (rows that see nothing), a sequence without keys,
    # and queries that every key is turned away from.
    g = torch.Generator().manual_seed(22)
    cq, ck = ref.starts([150, 40, 70]), ref.starts([33, 0, 70])
    q, k, v, do = (torch.randn(n, h, D, generator=g) for n, h in ((cq[-1], H), (ck[-1], 1), (ck[-1], 1), (cq[-1], H)))
    q, k = (torch.nn.functional.normalize(x.abs(), dim=-1) for x in (q, k))
    q[200:230] *= -1.0
    q, k, v, do = (x.to(device=cuda_device, dtype=DT[dtype]) for x in (q, k, v, do))
    for causal in (True, False):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        scale = torch.tensor([8.0], device=cuda_device, requires_grad=True)
        out = flash_born_attention_packed(*leaves, scale, _cu(cq, cuda_device), _cu(ck, cuda_device), causal, eps)
        grads = torch.autograd.grad(out, [*leaves, scale], do)
        want = ref.packed(q, k, v, 8.0, cq, ck, causal, eps, 0, do, DT[dtype])
        for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
            assert ref.worst(x, want[name]) <= 1.0, name
        empty = [*range(150, 190), *range(200, 230), *(range(117) if causal else ())]
        assert not out[empty].any() and not grads[0][empty].any() and grads[3].isfinite().all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("eps", EPS)
@pytest.mark.parametrize("weigh", [False, True])
def test_paged_rows_without_weight(cuda_device, dtype, D, eps, weigh):
    for lens in ([100, 0, 60, 2000], [40, 0, 3, 64]):  # joined from splits, and of one
        kc, vc, table, n, _ = make_cache(lens, 16, 1, D, torch.float32, 23)
        kc = torch.nn.functional.normalize(kc.abs(), dim=-1)
        q = torch.nn.functional.normalize(torch.randn(4, 2, D, generator=torch.Generator().manual_seed(24)).abs(), dim=-1)
        q[2, 1] *= -1.0
        table[0] = -1
        q, kc, vc = (x.to(device=cuda_device, dtype=DT[dtype]) for x in (q, kc, vc))
        weight = torch.zeros(4, 1, max(lens), device=cuda_device) if weigh else None
        out = flash_born_attention_paged(q, kc, vc, table.to(cuda_device), n.to(cuda_device), 8.0, eps, 0, weight)
        o, w = ref.paged(q, kc, vc, table, n, 8.0, eps)
        assert ref.worst(out, o) <= 1.0
        assert not out[0].any() and not out[1].any() and not out[2, 1].any()
        if weigh:
            x, e = (t[..., : max(lens)] for t in w)
            assert ref.worst(weight, (x, e + 2.0 ** -23 * x)) <= 1.0

"""Pages that are no multiple of 16 tokens at every head dim, with the keys'
weights and without, and evictions from caches of every width that the selection
has a kernel for."""

from __future__ import annotations

import pytest
import torch

from quantumdlblocks_amd import born_cache_evict
from test_cache import make_cache
from test_gpu_cache import DT, _attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [40, 64, 104, 128, 232, 256])
@pytest.mark.parametrize("page,window", [(5, 0), (24, 0), (24, 70), (100, 333)])
@pytest.mark.parametrize("weigh", [False, True])
def test_pages_of_odd_sizes(cuda_device, dtype, D, page, window, weigh):
    scale = torch.tensor([2.0, -1.0, 3.0, 0.5, -4.0, 1.0])
    _attend([500, 0, 1, 129], page, 6, 2, D, DT[dtype], cuda_device, window=window, scale=scale, weigh=weigh, seed=45)


@pytest.mark.parametrize("longest", [1, 64, 1024, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385])
@pytest.mark.parametrize("inplace", [False, True])
def test_evictions_from_caches_of_every_width(cuda_device, longest, inplace):
    lens, page, Hkv, D = [longest, longest // 3], 1, 2, 8
    budget, recent = max(1, longest // 2), longest // 7
    kc, vc, table, n, free = make_cache(lens, page, Hkv, D, torch.float32, 46, spare=2 * budget)
    to = None if inplace else free[: 2 * budget].view(2, budget).to(torch.int32)
    g = torch.Generator().manual_seed(47)
    w = torch.randint(0, 50, (2, Hkv, longest), generator=g).float()  # many ties
    w[1, 1] = w[1, 1].exp()
    dev = [x if x is None else x.to(cuda_device) for x in (kc, vc, table, n, w, to)]
    got = born_cache_evict(*dev[:5], budget, recent, dev[5])
    want = born_cache_evict(kc, vc, table, n, w, budget, recent, to)
    assert all(torch.equal(a.cpu(), b) for a, b in zip((*got, *dev[:2]), (*want, kc, vc)))

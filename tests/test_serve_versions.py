"""The cache operators write through addresses: they count their writes for
autograd, so that a backward that saved what they changed says so."""

from __future__ import annotations

import pytest
import torch

from quantumdlblocks_amd import born_cache_evict, flash_born_attention_paged, fused_qk_rope_l2_normalize_append
from quantumdlblocks_amd.kernels import born_cache

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _state(dev):
    g = torch.Generator().manual_seed(0)
    kc, vc, x = (torch.rand(*s, generator=g).to(dev) for s in ((5, 4, 1, 8), (5, 4, 1, 8), (1, 1, 8)))
    table, lens = torch.tensor([[0, 1]], dtype=torch.int32, device=dev), torch.tensor([6], dtype=torch.int32, device=dev)
    return kc, vc, x, table, lens


def _paged(kc, vc, x, table, lens, w):
    flash_born_attention_paged(x, kc, vc, table, lens, 1.0, key_weight=w)


def _append(kc, vc, x, table, lens, w):
    fused_qk_rope_l2_normalize_append(x, x, x, None, None, kc, vc, table, lens)


def _evict(kc, vc, x, table, lens, w):
    born_cache_evict(kc, vc, table, lens, w, 3)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("call,written", [(_paged, "w"), (_append, "kv"), (_evict, "kv")])
def test_a_backward_that_saved_a_written_tensor_raises(dev, call, written):
    if dev == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")
    for name in "kvw":
        kc, vc, x, table, lens = _state(dev)
        w = torch.rand(1, 1, 8, device=dev)
        saved = {"k": kc, "v": vc, "w": w}[name]
        leaf = torch.ones((), device=dev, requires_grad=True)
        loss = (leaf * saved).sum()
        with torch.no_grad():
            call(kc, vc, x, table, lens, w)
        if name in written:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
        else:
            loss.backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_inference_tensors_are_written(dev):
    if dev == "cuda" and not torch.cuda.is_available():
        pytest.skip("no GPU")
    with torch.inference_mode():
        kc, vc, x, table, lens = _state(dev)
        w = torch.zeros(1, 1, 8, device=dev)
        for call in (_append, _paged, _evict):
            call(kc, vc, x, table, lens, w)
        assert w.any()


def test_what_the_kernels_write_is_counted():
    a, b = torch.zeros(3), torch.zeros(3)
    before = a._version, b._version
    born_cache._written((a, b))
    assert (a._version, b._version) == (before[0] + 1, before[1] + 1)

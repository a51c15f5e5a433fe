"""Derivatives that the packed and cache operators do not have are refused, never
dropped.  On the CPU; the GPU's path of the packed call is run with the library
call recorded in place of the launch."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from quantumdlblocks_amd import born_cache_evict, flash_born_attention_packed, flash_born_attention_paged, fused_qk_rope_l2_normalize_append
from quantumdlblocks_amd.kernels import flash_born_packed as packed

NAMES = ("q", "k", "v", "scale")


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(packed, "_run_call", lambda fn, what, device, block: made.append(what))
    return made


def _packed_inputs():
    g = torch.Generator().manual_seed(0)
    x = dict(zip(NAMES, (torch.randn(5, h, 8, generator=g) for h in (4, 2, 2))), scale=torch.tensor([2.0]))
    return x, torch.tensor([0, 2, 5], dtype=torch.int32)


def _on_gpu(x, cu):
    return packed._on_gpu(*(x[n] for n in NAMES), cu, cu, True, 1e-12, 0)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("grad", [True, False])
def test_packed_forward_mode(calls, name, grad):
    x, cu = _packed_inputs()
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        _on_gpu(x, cu)  # a level without tangents
        dual = dict(x, **{name: forward_ad.make_dual(x[name], torch.ones_like(x[name]))})
        with pytest.raises(RuntimeError):
            _on_gpu(dual, cu)
        # The formulas on the CPU have it.
        out = flash_born_attention_packed(*(dual[n] for n in NAMES), cu, eps=0.5)
        assert forward_ad.unpack_dual(out).tangent is not None
    _on_gpu(x, cu)


def _cache():
    kc, vc = torch.randn(3, 4, 1, 8), torch.randn(3, 4, 1, 8)
    table, lens = torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)
    return dict(k_cache=kc, v_cache=vc, block_table=table, cache_lens=lens)


def _operators():
    one, w = torch.randn(1, 1, 8), torch.rand(1, 1, 8)
    ang = torch.rand(8, 4)
    return {
        "paged": (flash_born_attention_paged, dict(q=one, **_cache(), scale=torch.tensor([2.0]), key_weight=w),
                  ("q", "k_cache", "v_cache", "scale", "key_weight")),
        "append": (fused_qk_rope_l2_normalize_append, dict(q=one, k=one.clone(), v=one.clone(), cos=ang.cos(), sin=ang.sin(), **_cache()),
                   ("q", "k", "v", "cos", "sin", "k_cache", "v_cache")),
        "evict": (born_cache_evict, dict(**_cache(), key_weight=w, budget=3), ("k_cache", "v_cache", "key_weight")),
    }


@pytest.mark.parametrize("op", ["paged", "append", "evict"])
def test_cache_operators_refuse_recorded_derivatives(op):
    fn, kw, names = _operators()[op]
    for name in names:
        before = {n: t.clone() for n, t in kw.items() if isinstance(t, torch.Tensor)}
        leaf = kw[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no backward"):
            fn(**dict(kw, **{name: leaf}))
        for inner in (torch.enable_grad, torch.no_grad):
            with forward_ad.dual_level(), inner():
                dual = forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))
                with pytest.raises(RuntimeError, match="no forward-mode"):
                    fn(**dict(kw, **{name: dual}))
        assert all(torch.equal(kw[n], t) for n, t in before.items())
        with torch.no_grad():
            fn(**dict(kw, **{name: leaf}))
    with forward_ad.dual_level():
        fn(**kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])  # float64: rows that the call casts
@pytest.mark.parametrize("wrt", range(4))
def test_packed_second_derivative(calls, dtype, wrt):
    x, cu = _packed_inputs()
    leaves = [x["q"].to(dtype), x["k"].to(dtype), x["v"], x["scale"].to(dtype)]
    leaves = [t.requires_grad_() for t in leaves]
    out = packed._on_gpu(*leaves, cu, cu, True, 1e-12, 0)
    (g,) = torch.autograd.grad(out.sum(), leaves[wrt], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        (g.square().sum() + leaves[0].sum()).backward()
    # A recorded backward by itself is none.
    out = packed._on_gpu(*leaves, cu, cu, True, 1e-12, 0)
    out.sum().backward(create_graph=True)
    assert all(t.grad.shape == t.shape for t in leaves)
    for t in leaves:
        t.grad = None  # with its graph

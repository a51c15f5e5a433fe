"""The packed backward's gradients where autograd gives it other tensors than the
forward's: checkpoints, offloading to the host, hooks that copy."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import serve_ref as ref
from quantumdlblocks_amd import flash_born_attention_packed

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(dtype, D, dev):
    g = torch.Generator().manual_seed(21)
    lens = [130, 1, 65]
    cu = torch.tensor(ref.starts(lens), dtype=torch.int32, device=dev)
    x, do = (torch.randn(sum(lens), h, D, generator=g).to(device=dev, dtype=dtype) for h in (8, 4))
    scale = torch.tensor([1.0, -2.0, 3.0, 0.5], device=dev)
    return x, do, scale, cu


def _grads(x, do, scale, cu, around=None):
    """Gradients of one projection's output, whose rows the call reads in place, and of the scale."""
    leaf, s = x.clone().requires_grad_(), scale.clone().requires_grad_()

    def layer(leaf, s):
        y = leaf * 0.5
        return flash_born_attention_packed(y[:, :4], y[:, 4:6], y[:, 6:], s, cu, eps=0.5)

    out = layer(leaf, s) if around is None else around(layer, leaf, s)
    torch.full_like(x, float("nan"))  # takes memory that was given back
    return (out.detach(), *torch.autograd.grad(out, (leaf, s), do))


def _hooked(pack, unpack):
    def around(layer, leaf, s):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            return layer(leaf, s)

    return around


def _offloaded(layer, leaf, s):
    with torch.autograd.graph.save_on_cpu():
        return layer(leaf, s)


WAYS = {
    "checkpoint": lambda layer, leaf, s: checkpoint(layer, leaf, s, use_reentrant=False),
    "offload": _offloaded,
    "copies": _hooked(lambda t: t.detach().clone(), lambda t: t.clone()),
    "on the host": _hooked(lambda t: t.cpu(), lambda t: t),
    "strides": _hooked(lambda t: t, lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)),
}


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 20])
@pytest.mark.parametrize("way", list(WAYS))
def test_gradients_are_those_without_hooks(cuda_device, dtype, D, way):
    case = _case(DT[dtype], D, cuda_device)
    for a, b in zip(_grads(*case), _grads(*case, WAYS[way])):
        assert torch.equal(a, b)

"""What the packed backward passes on: the tensors that autograd gives it back,
which a saved tensor's hook (a checkpoint, offloading) may have replaced.  On the
CPU, with the library call recorded in place of the launch."""

from __future__ import annotations

import pytest
import torch

from quantumdlblocks_amd import _native
from quantumdlblocks_amd.kernels import flash_born_packed as packed

FIELDS = ("size dtype sequences n_q n_k H h_kv D q k v qs0 qs1 ks0 ks1 vs0 vs1 out z cu_q cu_k scale n_scale value causal "
          "window eps dout ds0 ds1 dq dk dv dscale ws ws_bytes").split()
SAVED = ("q", "k", "v", "out", "z", "scale", "cu_q", "cu_k")


@pytest.fixture
def blocks(monkeypatch):
    """The argument blocks of the calls that were made, as dicts."""
    made = []

    def record(fn, what, device, block):
        made.append(dict(zip(FIELDS, _native.packed_call.unpack(block)), what=what))

    monkeypatch.setattr(packed, "_run_call", record)
    return made


def _inputs(strided=False):
    g = torch.Generator().manual_seed(0)
    if strided:  # one projection's output
        x = torch.randn(7, 8, 16, generator=g)
        q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    else:
        q, k, v = (torch.randn(7, h, 16, generator=g) for h in (4, 2, 2))
    return [t.requires_grad_() if not strided else t.detach().requires_grad_() for t in (q, k, v)]


def _call(q, k, v, scale, cu, cu_k=None):
    return packed._FlashBornPackedFn.apply(q, k, v, scale, cu, cu if cu_k is None else cu_k, True, 1e-12, 0)


@pytest.mark.parametrize("strided", [False, True])
def test_backward_takes_what_the_hooks_return(blocks, strided):
    cu, scale = torch.tensor([0, 3, 7], dtype=torch.int32), torch.tensor([1.0, 2.0, 3.0, 4.0], requires_grad=True)
    leaves = _inputs(strided)
    given = []

    def unpack(t):
        given.append(t.clone(memory_format=torch.contiguous_format))
        return given[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack):
        out = _call(*leaves, scale, cu, cu.clone())
    torch.autograd.grad(out, leaves, torch.ones_like(out))
    forward, backward = blocks
    assert forward["what"].endswith("forward_call") and backward["what"].endswith("backward_call")
    assert len(given) == len(SAVED)
    for name, t in zip(SAVED, given):
        assert backward[name] == t.data_ptr() != forward[name], name
    # The clones are contiguous, whatever the forward's rows were.
    assert [backward[n] for n in ("qs0", "qs1", "ks0", "ks1", "vs0", "vs1")] == [64, 16, 32, 16, 32, 16]
    assert [backward[n] for n in FIELDS[1:8]] == [forward[n] for n in FIELDS[1:8]]
    assert (backward["n_scale"], backward["causal"], backward["eps"]) == (4, 1, 1e-12)


def test_backward_takes_rows_of_other_strides_and_types(blocks):
    # Hooks may also keep a tensor in other strides or in more bits.
    cu = torch.tensor([0, 7], dtype=torch.int32)
    leaves = _inputs()

    def unpack(t):
        return t.double() if t.dtype == torch.float32 and t.dim() == 2 else t.transpose(0, -1).contiguous().transpose(0, -1)

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        out = _call(*leaves, 2.0, cu)
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
    backward = blocks[1]
    assert [backward[n] for n in ("qs0", "qs1", "ks0", "ks1", "vs0", "vs1")] == [64, 16, 32, 16, 32, 16]
    assert backward["scale"] == 0 and backward["value"] == 2.0
    assert all(g.is_contiguous() and g.shape == x.shape for g, x in zip(grads, leaves))


def test_a_checkpoint_takes_the_second_forward(blocks):
    from torch.utils.checkpoint import checkpoint

    cu = torch.tensor([0, 7], dtype=torch.int32)
    w = torch.randn(16, 16, requires_grad=True)
    x = torch.randn(7, 2, 16)

    def layer(x):
        return _call(x @ w, x @ (2 * w), x @ (3 * w), 2.0, cu)

    out = checkpoint(layer, x, use_reentrant=False)
    hold = [torch.zeros(7, 2, 16) for _ in range(8)]  # takes the first forward's freed memory
    out.backward(torch.ones_like(out))
    first, second, backward = blocks
    names = ("q", "k", "v", "out", "z")
    assert all(backward[n] == second[n] for n in names) and hold
    assert any(first[n] != second[n] for n in names)


def test_without_hooks_nothing_is_copied(blocks):
    cu = torch.tensor([0, 7], dtype=torch.int32)
    out = _call(*_inputs(True), torch.ones(4), cu)
    out.backward(torch.ones_like(out))
    forward, backward = blocks
    assert all(forward[n] == backward[n] for n in FIELDS[:27])


def test_hooks_that_leave_a_tensor_elsewhere(blocks):
    # The library takes addresses on its own device only: others are brought
    # there, or, where there is nothing to bring, refused.
    cu = torch.tensor([0, 7], dtype=torch.int32)
    leaves = _inputs()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.to("meta"), lambda t: t):
        out = _call(*leaves, 2.0, cu)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.autograd.grad(out, leaves, torch.ones_like(out))
    assert len(blocks) == 1

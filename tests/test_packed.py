"""Packed attention on the CPU: the formulas, their gradients, refusals, and the
C ABI's checks of its argument block (which return before any HIP call)."""

from __future__ import annotations

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import _native, flash_born_attention, flash_born_attention_packed


def _inputs(lens, past, H, Hkv, D, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    N, M = sum(lens), sum(lens) + past * len(lens)
    q = torch.randn(N, H, D, generator=g, dtype=torch.float64)
    k, v = (torch.randn(M, Hkv, D, generator=g, dtype=torch.float64) for _ in range(2))
    cq, ck = ref.starts(lens), ref.starts([n + past for n in lens])
    return q.to(dtype), k.to(dtype), v.to(dtype), cq, ck, torch.tensor(cq), torch.tensor(ck)


@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 3), (False, 2)])
@pytest.mark.parametrize("lens,past", [([5, 0, 1, 7], 0), ([3, 4], 2), ([1], 0)])
def test_formula_and_gradients(lens, past, causal, window):
    q, k, v, cq, ck, tq, tk = _inputs(lens, past, 4, 2, 6)
    scale = torch.tensor([2.0, -1.5, 0.7, 1.1], dtype=torch.float64)
    grad = torch.randn(q.shape, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, scale)]
    out = flash_born_attention_packed(*leaves[:3], leaves[3], tq, tk, causal, 0.3, window)
    got = torch.autograd.grad(out, leaves, grad)
    want = ref.packed(q, k, v, scale, cq, ck, causal, 0.3, window, grad, torch.float32)
    for name, x in zip(("out", "dq", "dk", "dv", "ds"), (out, *got)):
        assert torch.allclose(x, want[name][0], rtol=1e-10, atol=1e-12), name


def test_gradients_against_differences():
    q, k, v, cq, ck, tq, tk = _inputs([4, 3], 1, 2, 1, 4, seed=5)
    scale = torch.tensor(1.3, dtype=torch.float64)
    leaves = [x.requires_grad_() for x in (q, k, v, scale)]
    fn = lambda q, k, v, s: flash_born_attention_packed(q, k, v, s, tq, tk, True, 0.2, 0)  # noqa: E731
    assert torch.autograd.gradcheck(fn, leaves, eps=1e-6, atol=1e-7)


def test_matches_the_dense_call_and_leaves_rows_behind_zero():
    q, k, v, cq, ck, tq, tk = _inputs([6], 0, 3, 3, 8, torch.float32)
    more = torch.cat([q, torch.ones(2, 3, 8)])
    out = flash_born_attention_packed(more, k, v, 2.0, tq, tk)
    dense = flash_born_attention(*(x.transpose(0, 1).unsqueeze(0) for x in (q, k, v)), 2.0)
    assert torch.allclose(out[:6], dense[0].transpose(0, 1), atol=1e-5)
    assert not out[6:].any()


def test_rows_without_keys_are_zero():
    q, k, v, cq, ck, tq, tk = _inputs([4], 0, 2, 1, 8, torch.float32)
    out = flash_born_attention_packed(q, k[:2], v[:2], 1.0, tq, torch.tensor([0, 2]), eps=0.0)
    assert not out[:2].any() and out[2:].isfinite().all()


def test_refusals():
    q, k, v, cq, ck, tq, tk = _inputs([4, 3], 0, 4, 2, 8, torch.float32)
    call = flash_born_attention_packed
    for bad in (
        lambda: call(q.view(7, 2, 2, 8), k, v, 1.0, tq),
        lambda: call(q, k, v[:5], 1.0, tq),
        lambda: call(q, k[..., :4], v[..., :4], 1.0, tq),
        lambda: call(q[:, :3], k, v, 1.0, tq),
        lambda: call(q, k, v, torch.ones(3), tq),
        lambda: call(q, k, v, 1.0, tq.float()),
        lambda: call(q, k, v, 1.0, tq, tk[:2]),
        lambda: call(q, k, v, 1.0, torch.tensor([0, 5, 4])),
        lambda: call(q, k, v, 1.0, torch.tensor([0, 4, 9])),
        lambda: call(q, k, v, 1.0, torch.tensor([1, 4, 7])),
        lambda: call(q, k, v, 1.0, tq, eps=-1.0),
        lambda: call(q, k, v, 1.0, tq, eps=float("nan")),
    ):
        with pytest.raises(ValueError):
            bad()


def _packed_block(**over):
    a = dict(dtype=2, sequences=1, n_q=4, n_k=4, H=4, h_kv=2, D=64, q=16, k=16, v=16, qs0=256, qs1=64, ks0=128, ks1=64, vs0=128,
             vs1=64, out=16, z=16, cu_q=16, cu_k=16, scale=0, n_scale=1, value=1.0, causal=1, window=0, eps=0.0, dout=16, ds0=256,
             ds1=64, dq=16, dk=16, dv=16, dscale=0, ws=16, ws_bytes=1 << 20)
    a.update(over)
    return _native.packed_call(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(dtype=5), -1), (dict(n_q=-1), -2), (dict(sequences=1 << 27), -2), (dict(eps=-1.0), -2), (dict(eps=float("nan")), -2),
    (dict(D=12), -3), (dict(D=264), -3), (dict(q=8), -4), (dict(out=8), -4), (dict(k=0), -5), (dict(cu_q=0), -5),
    (dict(scale=16, n_scale=3), -6), (dict(window=-1), -7), (dict(window=1 << 31), -7), (dict(H=3), -13), (dict(h_kv=0), -13),
    (dict(qs0=32), -14), (dict(qs0=257), -14), (dict(ks1=-64), -14), (dict(vs0=1 << 23), -14), (dict(H=1 << 20, h_kv=2), -2),
])
def test_argument_block_checks(over, code):
    lib = _native.load()
    assert lib.qdl_flash_born_packed_forward_call(_packed_block(**over), None) == code


def test_backward_block_checks():
    lib = _native.load()
    call = lib.qdl_flash_born_packed_backward_call
    assert call(_packed_block(ws_bytes=0), None) == -8
    assert call(_packed_block(ws=0), None) == -8
    assert call(_packed_block(dout=0), None) == -5
    assert call(_packed_block(dk=0), None) == -5
    assert call(_packed_block(z=0), None) == -5
    assert call(_packed_block(dq=8), None) == -4
    assert call(_packed_block(ds0=16), None) == -14
    assert call(None, None) == -5
    assert lib.qdl_flash_born_packed_forward_call(_packed_block(n_q=0), None) == 0
    short = _packed_block()
    assert lib.qdl_flash_born_packed_forward_call(b"\x08" + short[1:], None) == -2
    assert lib.qdl_flash_born_packed_workspace_size(_packed_block()) >= 2 * 4 * 4 * 4
    assert lib.qdl_flash_born_packed_workspace_size(_packed_block(D=12)) == 0


def test_many_sequences_fit_the_launches_of_both_directions():
    # dK/dV's workgroups of 512 threads: 2^23 of them leave the 32 bits that count a launch's threads.
    lib = _native.load()
    assert lib.qdl_flash_born_packed_workspace_size(_packed_block(H=1, h_kv=1, sequences=(1 << 23) - 4)) > 0
    assert lib.qdl_flash_born_packed_workspace_size(_packed_block(H=1, h_kv=1, sequences=1 << 23)) == 0
    assert lib.qdl_flash_born_packed_forward_call(_packed_block(H=1, h_kv=1, sequences=1 << 23), None) == -2

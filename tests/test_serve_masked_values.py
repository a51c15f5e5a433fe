"""What the CPU formulas make of infinities and NaN where nothing is seen, of
autocast, and of batches without sequences."""

from __future__ import annotations

import threading

import pytest
import torch

from quantumdlblocks_amd import flash_born_attention_packed, flash_born_attention_paged, fused_qk_rope_l2_normalize_append
from quantumdlblocks_amd.kernels import born_cache
from quantumdlblocks_amd.kernels import flash_born_packed as packed

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


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 2), (True, 2)])
def test_packed_keys_that_a_row_does_not_see(bad, causal, window):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.rand(9, h, 8, generator=g) for h in (4, 2, 2))
    cu = torch.tensor([0, 4, 9])
    want = flash_born_attention_packed(q, k, v, 2.0, cu, None, causal, 1e-12, window)
    at = 3 if causal else 0  # seen by the first sequence's last row, or by its first two
    k[at] = bad
    out = flash_born_attention_packed(q, k, v, 2.0, cu, None, causal, 1e-12, window)
    blind = [0, 1, 2, 4, 5, 6, 7, 8] if causal else [2, 3, 4, 5, 6, 7, 8]
    assert torch.equal(out[blind], want[blind])
    # Rows that see no key, whatever they hold.
    q[:2] = bad
    out = flash_born_attention_packed(q[:4], k[:2], v[:2], 2.0, torch.tensor([0, 4]), torch.tensor([0, 2]), eps=0.0)
    assert not out[:2].any()


@pytest.mark.parametrize("bad", BAD)
@pytest.mark.parametrize("window", [0, 3])
def test_paged_rows_without_keys(bad, window):
    table = _cache((0, 5, 5))[2]
    kc, vc = torch.rand(6, 4, 1, 8), torch.rand(6, 4, 1, 8)
    table[2] = -1
    q = torch.rand(3, 2, 8)
    weight = torch.zeros(3, 1, 8)
    want = flash_born_attention_paged(q, kc, vc, table, torch.tensor([0, 5, 5]), 2.0, 0.0, window, weight.clone())
    q[0] = q[2] = bad
    out = flash_born_attention_paged(q, kc, vc, table, torch.tensor([0, 5, 5]), 2.0, 0.0, window, weight)
    assert torch.equal(out, want) and not out[0].any() and not out[2].any()
    assert not weight[0].any() and not weight[2].any() and weight[1].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_autocast_leaves_the_formulas_in_fp32(dtype):
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(9, h, 8, generator=g).to(dtype) for h in (4, 2, 2))
    cu = torch.tensor([0, 4, 9])
    kc, vc, table, lens = _cache((7,))
    kc, vc = kc.to(dtype), vc.to(dtype)

    def run(autocast):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        with torch.autocast("cpu", dtype=torch.bfloat16, enabled=autocast):
            out = flash_born_attention_packed(*leaves, 2.0, cu)
            one = flash_born_attention_paged(q[:1], kc, vc, table, lens, 2.0)
        return (out, one, *torch.autograd.grad(out, leaves, torch.ones_like(out)))

    assert all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(run(True), run(False)))


def test_packed_batches_without_sequences_have_zero_gradients():
    leaves = [torch.rand(5, h, 8, requires_grad=True) for h in (4, 2, 2)] + [torch.tensor([2.0], requires_grad=True)]
    out = flash_born_attention_packed(*leaves, torch.zeros(1, dtype=torch.int32))
    assert not out.any()
    for x, g in zip(leaves, torch.autograd.grad(out.sum(), leaves)):
        assert g.shape == x.shape and not g.any()


@pytest.mark.parametrize("op", ["packed", "paged"])
def test_calls_from_two_threads_leave_each_its_autocast(op, monkeypatch):
    # One call ends while the other, of a thread without autocast, is on its way.
    inside, ended = threading.Event(), threading.Event()
    state = {}
    x = torch.rand(4, 2, 8)
    kc, vc, table, lens = _cache((5,))

    class Late(torch.Tensor):
        """Starts, or lengths, that the call reads once it is on its way."""

        @classmethod
        def __torch_function__(cls, func, types, args=(), kwargs=None):
            if func in (torch.Tensor.tolist, torch.Tensor.long):
                if threading.current_thread().name == "outer":
                    assert inside.wait(30)
                else:
                    inside.set()
                    assert ended.wait(30)
            return super().__torch_function__(func, types, args, kwargs or {})

    def call():
        if op == "packed":
            cu = torch.tensor([0, 4]).as_subclass(Late)
            packed._eager_packed(x, x[:, :1], x[:, :1], torch.tensor(1.0), cu, cu, True, 0.1, 0, x.dtype)
        else:
            born_cache._eager_paged(x[:1], kc, vc, table, lens.as_subclass(Late), torch.tensor(1.0), 0.1, 0, None)

    def outer():
        with torch.autocast("cpu", dtype=torch.bfloat16):
            call()
            state["outer"] = torch.is_autocast_enabled("cpu")
        ended.set()

    def inner():
        call()
        state["inner"] = torch.is_autocast_enabled("cpu")

    threads = [threading.Thread(target=f, name=f.__name__) for f in (outer, inner)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert state == {"outer": True, "inner": False}

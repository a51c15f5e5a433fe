"""Packed attention on the GPU against its formulas in 64 bits, element by
element within the bounds of serve_ref."""

from __future__ import annotations

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import flash_born_attention_packed

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _inputs(lens, past, H, Hkv, D, dtype, dev, seed=0, unit=True, behind=0):
    g = torch.Generator().manual_seed(seed)
    N, M = sum(lens) + behind, sum(lens) + past * len(lens) + behind
    q, k, v, do = (torch.randn(n, h, D, generator=g) for n, h in ((N, H), (M, Hkv), (M, Hkv), (N, H)))
    if unit:
        way = 0.5 * torch.randn(1, 1, D, generator=g)
        q, k = (torch.nn.functional.normalize(x + way, dim=-1) for x in (q, k))
    q, k, v, do = (x.to(device=dev, dtype=dtype) for x in (q, k, v, do))
    return q, k, v, do, ref.starts(lens), ref.starts([n + past for n in lens])


def _cu(c, dev):
    return torch.tensor(c, dtype=torch.int32, device=dev)


def _check(q, k, v, do, scale, cq, ck, causal, eps, window, names=("out", "dq", "dk", "dv")):
    dev = q.device
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    out = flash_born_attention_packed(*leaves, scale, _cu(cq, dev), _cu(ck, dev), causal, eps, window)
    grads = torch.autograd.grad(out, leaves, do)
    want = ref.packed(q, k, v, scale, cq, ck, causal, eps, window, do, q.dtype)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        if name in names:
            assert ref.worst(x, want[name]) <= 1.0, name


MASKS = [(True, 0), (False, 0), (True, 100), (False, 40)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("causal,window", MASKS)
def test_masks_and_head_dims(cuda_device, dtype, D, causal, window):
    lens = [131, 1, 0, 64, 257]
    _check(*_case(lens, 0, 4, 2, D, DT[dtype], cuda_device), causal, 1e-12, window)


def _case(lens, past, H, Hkv, D, dtype, dev, scale=3.0, **kw):
    q, k, v, do, cq, ck = _inputs(lens, past, H, Hkv, D, dtype, dev, **kw)
    return q, k, v, do, scale, cq, ck


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [8, 20, 32, 72, 200])
def test_odd_head_dims(cuda_device, dtype, D):
    _check(*_case([65, 30, 200], 0, 3, 1, D, DT[dtype], cuda_device, seed=2), True, 1e-12, 0)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (8, 1), (6, 3), (24, 8)])
def test_groups(cuda_device, dtype, H, Hkv):
    _check(*_case([70, 129], 0, H, Hkv, 64, DT[dtype], cuda_device, seed=3), True, 1e-12, 0)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 60)])
def test_heads_of_a_group_shared_out(cuda_device, dtype, D, causal, window):
    # Few blocks, many heads on one key head: dK and dV are summed from parts.
    q, k, v, do, cq, ck = _inputs([700, 1, 333], 0, 12, 1, D, DT[dtype], cuda_device, seed=16)
    scale = torch.tensor([2.0, -1.0, 3.0] * 4, device=cuda_device)
    _check(q, k, v, do, scale, cq, ck, causal, 1e-12, window)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("causal,window", MASKS)
def test_long_blocks(cuda_device, dtype, D, causal, window):
    # Enough key blocks for the eight-wave dK/dV kernel.
    lens = [300, 129, 1, 40] * 9
    q, k, v, do, cq, ck = _inputs(lens, 3, 8, 4, D, DT[dtype], cuda_device, seed=17)
    scale = torch.tensor([2.0, -1.0, 3.0, 1.0, -2.0, -3.0, 1.0, 1.0], device=cuda_device)
    _check(q, k, v, do, scale, cq, ck, causal, 1e-12, window)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("past", [1, 63, 300])
@pytest.mark.parametrize("causal,window", MASKS)
def test_more_keys_than_queries(cuda_device, dtype, past, causal, window):
    _check(*_case([40, 1, 150], past, 4, 2, 64, DT[dtype], cuda_device, seed=4), causal, 1e-12, window)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("causal", [True, False])
def test_fewer_keys_than_queries(cuda_device, dtype, causal):
    # Under causality the first rows see nothing; the second sequence has no keys.
    q, k, v, do, cq, _ = _inputs([150, 40, 9], 0, 4, 2, 64, DT[dtype], cuda_device, seed=5)
    ck = [0, 33, 33, 60]
    _check(q, k[:60], v[:60], do, 2.0, cq, ck, causal, 1e-12, 0)
    out = flash_born_attention_packed(q, k[:60], v[:60], 2.0, _cu(cq, cuda_device), _cu(ck, cuda_device), causal, eps=0.0)
    assert out.isfinite().all() and not out[150:190].any()
    assert not causal or not out[:117].any()


@pytest.mark.parametrize("dtype", list(DT))
def test_scales_and_their_gradient(cuda_device, dtype):
    # eps of the size of the sums, so that the scale matters.
    q, k, v, do, cq, ck = _inputs([100, 33], 0, 4, 2, 64, DT[dtype], cuda_device, seed=6)
    for values in ([2.5], [1.5, -2.0, 0.3, 40.0]):
        scale = torch.tensor(values, device=cuda_device, requires_grad=True)
        out = flash_born_attention_packed(q, k, v, scale, _cu(cq, cuda_device), _cu(ck, cuda_device), True, 0.5, 0)
        (ds,) = torch.autograd.grad(out, scale, do)
        want = ref.packed(q, k, v, values if len(values) > 1 else values[0], cq, ck, True, 0.5, 0, do, q.dtype)
        assert ref.worst(out, want["out"]) <= 1.0
        x, e = want["ds"]
        x, e = (x, e) if len(values) > 1 else (x.sum().view(1), e.sum().view(1))
        assert ds.shape == scale.shape and ref.worst(ds, (x, e + 2.0 ** -23 * x.abs())) <= 1.0
    zero = flash_born_attention_packed(q, k, v, 0.0, _cu(cq, cuda_device), _cu(ck, cuda_device))
    assert not zero.any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [1e-3, 30.0, 300.0])
def test_overlaps_of_any_size_keep_their_weight(cuda_device, dtype, size):
    # fp16's square leaves its range above 255 and its normal range below 2^-7.
    q, k, v, do, cq, ck = _inputs([200, 65], 0, 2, 1, 64, DT[dtype], cuda_device, seed=7, unit=False)
    ramp = torch.linspace(0.05, 1.0, k.shape[0], device=cuda_device).view(-1, 1, 1)
    k = (k.float() * ramp * size).to(k.dtype)
    _check(q, k, v, do, 1.0, cq, ck, True, 1e-12, 0, names=("out",))
    _check(q, k, v, do, 1.0, cq, ck, False, 1e-12, 0, names=("out",))


@pytest.mark.parametrize("dtype", list(DT))
def test_rows_behind_the_last_sequence(cuda_device, dtype):
    q, k, v, do, cq, ck = _inputs([40, 9], 0, 4, 2, 64, DT[dtype], cuda_device, seed=8, behind=200)
    q[49:] = float("nan")
    k[49:] = float("inf")
    v[49:] = float("nan")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = flash_born_attention_packed(*leaves, 2.0, _cu(cq, cuda_device))
    grads = torch.autograd.grad(out, leaves, do)
    for x in (out, *grads):
        assert not x[49:].any() and x[:49].isfinite().all()
    want = ref.packed(*(x.detach()[:49] for x in leaves), 2.0, cq, ck, grad=do[:49], dt=q.dtype)
    for name, x in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert ref.worst(x[:49], want[name]) <= 1.0, name


def test_no_sequences_and_no_tokens(cuda_device):
    q = torch.randn(5, 2, 64, device=cuda_device, dtype=torch.bfloat16, requires_grad=True)
    none = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    out = flash_born_attention_packed(q, q, q, 1.0, none)
    assert not out.any()
    (g,) = torch.autograd.grad(out.sum(), q)
    assert not g.any()
    e = q[:0]
    out = flash_born_attention_packed(e, e, e, 1.0, torch.zeros(4, dtype=torch.int32, device=cuda_device))
    assert out.shape == (0, 2, 64)
    some = flash_born_attention_packed(q, e, e, 1.0, torch.tensor([0, 5], device=cuda_device), torch.tensor([0, 0], device=cuda_device))
    assert not some.any()


def test_many_sequences(cuda_device):
    # More than one round of the 64-way search.
    lens = [(7 * i) % 5 for i in range(5000)]
    q, k, v, do, cq, ck = _inputs(lens, 0, 2, 1, 32, torch.float32, cuda_device, seed=9)
    cu = _cu(cq, cuda_device)
    out = flash_born_attention_packed(q, k, v, 2.0, cu)
    pick = [0, 1, 63, 64, 65, 2500, 4095, 4096, 4998, 4999]
    for s in pick:
        a, b = cq[s], cq[s + 1]
        want = ref.packed(q[a:b], k[a:b], v[a:b], 2.0, [0, b - a], [0, b - a])
        assert ref.worst(out[a:b], want["out"]) <= 1.0, s
    assert out[: cq[-1]].abs().sum(-1).ne(0).float().mean() > 0.9


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strided_rows(cuda_device, dtype):
    # One projection's output holds q, k and v; heads-first tensors; a broadcast key head.
    g = torch.Generator().manual_seed(10)
    lens, H, Hkv, D = [77, 60], 4, 2, 64
    N = sum(lens)
    qkv = torch.randn(N, H + 2 * Hkv, D, generator=g).to(device=cuda_device, dtype=DT[dtype])
    q, k, v = qkv[:, :H], qkv[:, H : H + Hkv], qkv[:, H + Hkv :]
    cq = ref.starts(lens)
    do = torch.randn(N, H, D, generator=g).to(device=cuda_device, dtype=DT[dtype])
    _check(q, k, v, do, 0.5, cq, cq, True, 1e-12, 0)
    out = flash_born_attention_packed(q, k, v, 0.5, _cu(cq, cuda_device))
    first = flash_born_attention_packed(q.transpose(0, 1).contiguous().transpose(0, 1), k.clone(), v.clone(), 0.5, _cu(cq, cuda_device))
    assert torch.equal(out, first)
    one = k[:, :1].expand(N, Hkv, D)
    assert torch.equal(flash_born_attention_packed(q, one, v, 0.5, _cu(cq, cuda_device)),
                       flash_born_attention_packed(q, one.contiguous(), v, 0.5, _cu(cq, cuda_device)))
    wide = torch.zeros(N, H, D + 1, device=cuda_device, dtype=DT[dtype])  # rows that are not aligned
    wide[..., 1:] = q
    assert torch.equal(flash_born_attention_packed(wide[..., 1:], k, v, 0.5, _cu(cq, cuda_device)), out)
    lead = out.sum()  # a gradient of expanded strides
    leaf = q.detach().clone().requires_grad_()
    flash_born_attention_packed(leaf, k, v, 0.5, _cu(cq, cuda_device)).sum().backward()
    ones = torch.ones_like(q)
    ref_leaf = q.detach().clone().requires_grad_()
    flash_born_attention_packed(ref_leaf, k, v, 0.5, _cu(cq, cuda_device)).backward(ones)
    assert torch.equal(leaf.grad, ref_leaf.grad) and lead.isfinite()


def test_long_sequence_against_blocks_of_its_rows(cuda_device):
    q, k, v, do, cq, ck = _inputs([5000], 0, 2, 1, 128, torch.bfloat16, cuda_device, seed=11)
    _check(q, k, v, do, 3.0, cq, ck, True, 1e-12, 0)


def test_same_results_every_time(cuda_device):
    q, k, v, do, scale, cq, ck = _case([300, 77, 512], 0, 8, 2, 64, torch.bfloat16, cuda_device, seed=12)
    runs = []
    for _ in range(3):
        leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
        out = flash_born_attention_packed(*leaves, scale, _cu(cq, cuda_device))
        runs.append((out, *torch.autograd.grad(out, leaves, do)))
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_autocast_and_mixed_dtypes(cuda_device):
    q, k, v, do, cq, ck = _inputs([64, 30], 0, 2, 2, 64, torch.float32, cuda_device, seed=13)
    cu = _cu(cq, cuda_device)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        leaf = q.clone().requires_grad_()
        out = flash_born_attention_packed(leaf, k, v, 2.0, cu)
    assert out.dtype == torch.bfloat16
    assert torch.equal(out, flash_born_attention_packed(q.bfloat16(), k.bfloat16(), v.bfloat16(), 2.0, cu))
    out.sum().backward()
    assert leaf.grad.dtype == torch.float32


def test_on_another_stream_and_in_a_graph(cuda_device):
    q, k, v, do, cq, ck = _inputs([200, 120], 0, 4, 2, 64, torch.bfloat16, cuda_device, seed=14)
    cu = _cu(cq, cuda_device)
    with torch.no_grad():
        want = flash_born_attention_packed(q, k, v, 2.0, cu)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = flash_born_attention_packed(q, k, v, 2.0, cu)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = flash_born_attention_packed(q, k, v, 2.0, cu)
        for lens in ([200, 120], [1, 319], [160, 160]):  # the starts may change between replays
            cu.copy_(_cu(ref.starts(lens), cuda_device))
            q.copy_(torch.randn_like(q))
            graph.replay()
            eager = flash_born_attention_packed(q, k, v, 2.0, cu)
            torch.cuda.synchronize()
            assert torch.equal(held, eager)


def test_training_step_in_a_graph(cuda_device):
    q, k, v, do, cq, ck = _inputs([200, 120], 0, 4, 2, 64, torch.bfloat16, cuda_device, seed=15)
    cu = _cu(cq, cuda_device)

    def step(leaves):
        out = flash_born_attention_packed(*leaves, 2.0, cu)
        return (out.detach(), *torch.autograd.grad(out, leaves, do))

    static = [x.clone().requires_grad_() for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(static)
    for i in range(3):
        with torch.no_grad():
            static[0].copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)).to(q))
        graph.replay()
        torch.cuda.synchronize()
        eager = step([x.detach().clone().requires_grad_() for x in static])
        assert all(torch.equal(a, b) for a, b in zip(held, eager))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 96, 256])
def test_gradients_of_some_inputs_only(cuda_device, dtype, D):
    # Whichever are asked for, each is the one of the whole backward; heads are shared out here too.
    q, k, v, do, cq, _ = _inputs([200, 1, 65], 0, 8, 1, D, DT[dtype], cuda_device, seed=18)
    cu, scale = _cu(cq, cuda_device), torch.tensor([2.0], device=cuda_device)
    leaves = [x.requires_grad_() for x in (q, k, v, scale)]
    every = torch.autograd.grad(flash_born_attention_packed(*leaves, cu, eps=0.5), leaves, do)
    for pick in ((0,), (1,), (2,), (3,), (0, 3), (0, 1), (1, 2), (2, 3)):
        some = [x if i in pick else x.detach() for i, x in enumerate(leaves)]
        out = flash_born_attention_packed(*some, cu, eps=0.5)
        for i, g in zip(pick, torch.autograd.grad(out, [leaves[i] for i in pick], do)):
            assert torch.equal(g, every[i]), (pick, i)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_offsets_past_32_bits(cuda_device, dtype):
    # Token strides of half a step under the limit: rows lie over more than 4 GiB.
    lens, H, Hkv, D = [500, 200], 2, 1, 64
    q, k, v, do, cq, _ = _inputs(lens, 0, H, Hkv, D, DT[dtype], cuda_device, seed=19)
    cu = _cu(cq, cuda_device)
    stride = (1 << 23) // q.element_size()  # 8 MiB a token

    def far(x):
        n, h, d = x.shape
        big = torch.empty((n - 1) * stride + h * d, dtype=x.dtype, device=x.device).as_strided((n, h, d), (stride, d, 1))
        return big.copy_(x)

    def run(*xs):
        xs = [x.detach().requires_grad_() for x in xs]
        out = flash_born_attention_packed(*xs, 2.0, cu)
        return (out, *torch.autograd.grad(out, xs, do))

    assert 700 * stride * q.element_size() > 1 << 32
    for a, b in zip(run(q, k, v), run(far(q), far(k), far(v))):
        assert torch.equal(a, b)


def test_keys_without_queries(cuda_device):
    q, k, v, _, _, _ = _inputs([70], 0, 4, 2, 64, torch.bfloat16, cuda_device, seed=20)
    none, some = torch.tensor([0, 0], device=cuda_device), torch.tensor([0, 70], device=cuda_device)
    leaves = [x.requires_grad_() for x in (q[:0].detach(), k, v)]
    out = flash_born_attention_packed(*leaves, 1.0, none, some)
    for x, g in zip(leaves, torch.autograd.grad(out.sum(), leaves)):
        assert g.shape == x.shape and not g.any()

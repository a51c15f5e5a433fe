"""Launches that fill the chip, which take other kernels than small ones do: the
append of many tokens, four rows of a token to a group of lanes, and packed
attention in blocks whose waves share no rows; and gradients of overlaps of any
size.  Bounds as in serve_ref."""

from __future__ import annotations

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import flash_born_attention_packed, fused_qk_rope_l2_normalize_append
from test_cache import make_cache

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _lanes(D, dtype):
    """Lanes of a row in the append kernel."""
    vec = 8 if dtype != torch.float32 and D % 16 == 0 else 4
    n = 1
    while n * vec < D // 2:
        n *= 2
    return n


# Rows of a token that are no multiple of four, groups that lie across queries,
# keys and values in every way.
@pytest.mark.parametrize("H,Hkv", [(6, 2), (5, 1), (3, 3), (2, 1)])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,freqs", [(24, 5), (64, 32), (128, 64), (256, 100)])
def test_append_of_many_tokens(cuda_device, dtype, D, freqs, H, Hkv):
    dt, page = DT[dtype], 16
    N = (1 << 20) // ((H + 2 * Hkv) * _lanes(D, dt)) + 3  # just enough for groups of four rows
    assert N * (H + 2 * Hkv) * _lanes(D, dt) >= 1 << 20
    new = [N // 2, 0, 1, N - N // 2 - 1 - 50]  # 50 tokens of no sequence
    full = [new[0] + 70, 5, 1, new[3] + 3]
    kc, vc, table, n, _ = make_cache(full, page, Hkv, D, dt, seed=41)
    table[0, 9] = -1
    g = torch.Generator().manual_seed(42)
    q, k, v = (torch.randn(N, h, D, generator=g).to(dt) for h in (H, Hkv, Hkv))
    q[-50:] = float("nan")
    cu = torch.tensor(ref.starts(new), dtype=torch.int32)
    pos = torch.randint(0, 60, (N,), generator=g, dtype=torch.int32)  # some past the tables
    ang = torch.rand(50, freqs, generator=g) * 6
    wide = [x.double() for x in (q, k, v, kc, vc)]
    kd, vd = wide[3].clone(), wide[4].clone()
    qd = fused_qk_rope_l2_normalize_append(*wide[:3], ang.cos(), ang.sin(), kd, vd, table, n, cu, pos, 1e-6)
    dev = [x.to(cuda_device) for x in (q, k, v, ang.cos(), ang.sin(), kc, vc, table, n, cu, pos)]
    got = fused_qk_rope_l2_normalize_append(*dev, eps=1e-6)
    u = ref.HALF_STEP[dt] * 1.02
    for x, y in ((got, qd), (dev[5], kd)):
        y = y.to(cuda_device)
        assert ((x.double() - y).abs() <= u * y.abs() + (D + 32) * 2.0 ** -24).all()
    assert torch.equal(dev[6].cpu().double(), vd) and not got[-50:].any()
    still = ~(vd != wide[4]).any(-1)
    assert torch.equal(dev[5].cpu()[still], kc[still])


def _inputs(lens, past, H, Hkv, D, dtype, dev, seed, unit=True):
    g = torch.Generator().manual_seed(seed)
    N, M = sum(lens), sum(lens) + past * len(lens)
    q, k, v, do = (torch.randn(n, h, D, generator=g) for n, h in ((N, H), (M, Hkv), (M, Hkv), (N, H)))
    if unit:
        way = 0.5 * torch.randn(1, 1, D, generator=g)
        q, k = (torch.nn.functional.normalize(x + way, dim=-1) for x in (q, k))
    return [x.to(device=dev, dtype=dtype) for x in (q, k, v, do)], ref.starts(lens), ref.starts([n + past for n in lens])


def _check(x, cq, ck, scale, causal, window):
    q, k, v, do = x
    cu_q, cu_k = (torch.tensor(c, dtype=torch.int32, device=q.device) for c in (cq, ck))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = flash_born_attention_packed(*leaves, scale, cu_q, cu_k, causal, 1e-12, window)
    grads = torch.autograd.grad(out, leaves, do)
    want = ref.packed(q, k, v, scale, cq, ck, causal, 1e-12, window, do, q.dtype)
    for name, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        assert ref.worst(t, want[name]) <= 1.0, name


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("causal,window,past", [(True, 0, 0), (False, 0, 0), (True, 200, 0), (False, 333, 20), (True, 0, 70)])
def test_packed_blocks_of_whole_waves(cuda_device, dtype, D, causal, window, past):
    x, cq, ck = _inputs([1500, 1, 1333, 1290], past, 16, 8, D, DT[dtype], cuda_device, 43)
    scale = torch.tensor([2.0, -1.0, 3.0, 0.5] * 4, device=cuda_device)
    _check(x, cq, ck, scale, causal, window)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", [1e-3, 30.0, 300.0])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,H,Hkv,D", [([200, 65], 2, 1, 64), ([1100, 1300, 900, 1000], 16, 8, 64), ([300, 41], 4, 2, 128), ([190], 2, 2, 256)])
def test_gradients_of_overlaps_of_any_size(cuda_device, dtype, size, causal, lens, H, Hkv, D):
    # Growing along the keys, so that fp16's factors change on the way.
    (q, k, v, do), cq, ck = _inputs(lens, 0, H, Hkv, D, DT[dtype], cuda_device, 44, unit=False)
    ramp = torch.linspace(0.05, 1.0, k.shape[0], device=cuda_device).view(-1, 1, 1)
    k = (k.float() * ramp * size).to(k.dtype)
    _check((q, k, v, do), cq, ck, 1.0, causal, 0)

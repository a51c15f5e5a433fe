"""The paged cache's operators on the GPU: attention of one token against its
formula in 64 bits within the bounds of serve_ref, appending and evicting against
the same calls on the CPU."""

from __future__ import annotations

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import (
    born_cache_evict,
    flash_born_attention_packed,
    flash_born_attention_paged,
    fused_qk_rope_l2_normalize,
    fused_qk_rope_l2_normalize_append,
)
from test_cache import make_cache

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _attend(lens, page, H, Hkv, D, dtype, dev, window=0, scale=2.0, eps=1e-12, weigh=False, unit=True, size=1.0, seed=0):
    kc, vc, table, n, _ = make_cache(lens, page, Hkv, D, torch.float32, seed)
    q = torch.randn(len(lens), H, D, generator=torch.Generator().manual_seed(seed + 1))
    if unit:
        q, kc = (torch.nn.functional.normalize(x + 0.1, dim=-1) for x in (q, kc))
    kc = kc * size
    q, kc, vc = (x.to(device=dev, dtype=dtype) for x in (q, kc, vc))
    table, n = table.to(dev), n.to(dev)
    s = scale.to(dev) if isinstance(scale, torch.Tensor) else scale
    weight = torch.full((len(lens), Hkv, max(lens + [1])), 0.5, device=dev) if weigh else None
    out = flash_born_attention_paged(q, kc, vc, table, n, s, eps, window, weight)
    o, w = ref.paged(q, kc, vc, table, n.cpu(), scale, eps, window)
    assert ref.worst(out, o) <= 1.0
    if weigh:
        m = min(weight.shape[2], w[0].shape[2])
        x, e = w[0][..., :m] + 0.5, w[1][..., :m] + 2.0 ** -24 * 2.0 * (w[0][..., :m] + 0.5)
        assert ref.worst(weight[..., :m], (x, e)) <= 1.0
        assert (weight[..., m:] == 0.5).all()
    return out


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("H,Hkv", [(4, 2), (1, 1), (20, 1)])
def test_head_dims_and_groups(cuda_device, dtype, D, H, Hkv):
    _attend([130, 0, 1, 33], 16, H, Hkv, D, DT[dtype], cuda_device)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_pages_and_windows(cuda_device, dtype, page, window):
    _attend([300, 31, 32, 129], page, 4, 2, 64, DT[dtype], cuda_device, window=window, weigh=True, seed=2)


@pytest.mark.parametrize("dtype", list(DT))
def test_long_caches_are_split(cuda_device, dtype):
    scale = torch.tensor([1.0, -2.0, 30.0, 0.1])
    _attend([2500, 5, 1024, 1025], 16, 4, 2, 128, DT[dtype], cuda_device, scale=scale, weigh=True, seed=3)
    _attend([2500], 32, 4, 4, 64, DT[dtype], cuda_device, scale=scale, eps=0.3, seed=4)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("size", [1e-3, 30.0, 300.0])
def test_overlaps_of_any_size_keep_their_weight(cuda_device, dtype, size):
    _attend([700, 40], 16, 4, 2, 64, DT[dtype], cuda_device, unit=False, size=size, scale=1.0, weigh=True, seed=5)


def test_missing_pages_and_empty_rows(cuda_device):
    for dt in DT.values():
        kc, vc, table, n, _ = make_cache([100, 100, 100], 16, 2, 64, dt, seed=6, device=cuda_device)
        kc[-1] = float("nan")  # pages of nobody
        table[0, 2] = -1
        table[1, 3] = kc.shape[0] + 5
        n[1], n[2] = 5000, -3
        q = torch.randn(3, 4, 64, device=cuda_device).to(dt)
        used = torch.unique(table[(table >= 0) & (table < kc.shape[0])])
        free = [i for i in range(kc.shape[0]) if i not in used.tolist()]
        kc[free] = float("nan")
        vc[free] = float("inf")
        out = flash_born_attention_paged(q, kc, vc, table, n, 1.0, 0.0)
        o, _ = ref.paged(q, kc, vc, table, n.cpu(), 1.0, 0.0)
        assert ref.worst(out, o) <= 1.0 and not out[2].any()
        # What lies in a sequence's last page behind its length is not read.
        n[0] = 90
        kc[table[0, 5].long(), 10:] = float("nan")
        vc[table[0, 5].long(), 10:] = float("nan")
        out = flash_born_attention_paged(q, kc, vc, table, n, 1.0, 0.0)
        assert out[0].isfinite().all()


def test_strides_and_index_types(cuda_device):
    g = torch.Generator().manual_seed(7)
    B, Hkv, D, page = 3, 2, 64, 16
    kc, vc, table, n, _ = make_cache([70, 20, 48], page, Hkv, D, torch.bfloat16, seed=7, device=cuda_device)
    q = torch.randn(B, 4, D, generator=g).to(device=cuda_device, dtype=torch.bfloat16)
    want = flash_born_attention_paged(q, kc, vc, table, n, 2.0)
    heads_first = kc.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.stack([kc, vc], 1)  # one allocation: (pages, 2, page, Hkv, D)
    assert torch.equal(flash_born_attention_paged(q, heads_first, both[:, 1], table, n, 2.0), want)
    wide = torch.full((B, table.shape[1] + 3), -1, dtype=torch.int32, device=cuda_device)
    wide[:, : table.shape[1]] = table
    got = flash_born_attention_paged(q.transpose(0, 1).contiguous().transpose(0, 1), kc, vc, wide[:, : table.shape[1]], n, 2.0)
    assert torch.equal(got, want)
    assert torch.equal(flash_born_attention_paged(q, kc, vc, table.long(), n.long(), torch.tensor(2.0, device=cuda_device)), want)
    with pytest.raises(ValueError):
        flash_born_attention_paged(q[..., :32], kc[..., ::2], vc[..., ::2], table, n, 2.0)
    with pytest.raises(NotImplementedError):
        flash_born_attention_paged(q[..., :60], kc[..., :60], vc[..., :60], table, n, 2.0)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,freqs", [(64, 32), (128, 64), (24, 5), (256, 200), (8, 4)])
@pytest.mark.parametrize("rope", [True, False])
def test_append(cuda_device, dtype, D, freqs, rope):
    dt = DT[dtype]
    page, H, Hkv = 16, 6, 2
    full, new = [50, 3, 0, 200], [20, 3, 0, 37]
    kc, vc, table, n, _ = make_cache(full, page, Hkv, D, dt, seed=8)
    table[3, 12] = -1  # the last slots have no page
    g = torch.Generator().manual_seed(9)
    N = sum(new) + 2
    q, k, v = (torch.randn(N, h, D, generator=g).to(dt) for h in (H, Hkv, Hkv))
    cu = torch.tensor(ref.starts(new), dtype=torch.int32)
    pos = torch.randint(0, 40, (N,), generator=g, dtype=torch.int32)
    pos[3] = 1000
    ang = torch.rand(40, freqs, generator=g) * 6
    tables = (ang.cos(), ang.sin()) if rope else (None, None)
    for positions in (pos, None):
        wide = [x.double() for x in (q, k, v, kc, vc)]
        kd, vd = wide[3].clone(), wide[4].clone()
        qd = fused_qk_rope_l2_normalize_append(*wide[:3], *tables, kd, vd, table, n, cu, positions, 1e-6)
        dev = [x.to(cuda_device) if x is not None else None for x in (q, k, v, *tables, kc, vc, table, n, cu, positions)]
        got = fused_qk_rope_l2_normalize_append(*dev, eps=1e-6)
        # Rounded once; before that, sums of D squares and a handful of fp32 operations.
        u = ref.HALF_STEP[dt] * 1.02
        for x, y in ((got, qd), (dev[5], kd)):
            d = (x.double().cpu() - y).abs()
            assert (d <= u * y.abs() + (D + 32) * 2.0 ** -24).all()
        assert torch.equal(dev[6].double().cpu(), vd) and not got[-2:].any()
        touched = (vd != wide[4]).any(-1)
        assert torch.equal(dev[5].cpu()[~touched], kc[~touched])


def test_append_one_token_each_equals_the_prologue_in_fp32(cuda_device):
    B, H, D, page = 40, 4, 64, 16
    kc, vc, table, n, _ = make_cache([page] * B, page, H, D, seed=10, device=cuda_device)
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(B, H, D, generator=g).to(cuda_device) for _ in range(3))
    ang = torch.rand(page, D // 2, generator=g).to(cuda_device)
    got = fused_qk_rope_l2_normalize_append(q, k, v, ang.cos(), ang.sin(), kc, vc, table, n)
    at = torch.full((B,), page - 1)
    cos, sin = ang.cos()[at].view(1, 1, B, -1), ang.sin()[at].view(1, 1, B, -1)
    qp, kp = fused_qk_rope_l2_normalize(q.transpose(0, 1).unsqueeze(0), k.transpose(0, 1).unsqueeze(0), cos, sin)
    assert torch.allclose(got, qp[0].transpose(0, 1), atol=1e-6)
    assert torch.allclose(kc[table[:, 0].long(), page - 1], kp[0].transpose(0, 1), atol=1e-6)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lens,budget,recent", [
    ([100, 20, 0, 65], 64, 16), ([100, 7], 64, 64), ([300], 0, 0), ([5000, 1300], 1024, 100), ([17000, 20000], 9000, 3), ([70], 69, 0),
])
def test_evict(cuda_device, dtype, lens, budget, recent, inplace):
    page, Hkv, D = 16, 2, 24
    dt = DT[dtype]
    room = max(1, -(-min(budget, max(lens)) // page))
    kc, vc, table, n, free = make_cache(lens, page, Hkv, D, dt, seed=12, spare=len(lens) * room)
    to = None if inplace else free[: len(lens) * room].view(len(lens), room).to(torch.int32)
    g = torch.Generator().manual_seed(13)
    w = torch.randn(len(lens), Hkv, max(lens) - 3, generator=g).exp()
    w = torch.where(torch.rand(w.shape, generator=g) < 0.4, torch.zeros_like(w), w)  # ties
    w[0, 0, 5], w[0, 1, 7], w[0, 1, 9] = float("nan"), float("inf"), -1.0
    dev = [x.to(cuda_device) if x is not None else None for x in (kc, vc, table, n, w, to)]
    got = born_cache_evict(*dev[:5], budget, recent, dev[5])
    want = born_cache_evict(kc, vc, table, n, w, budget, recent, to)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[2].cpu(), want[2])
    assert torch.equal(got[1].cpu().nan_to_num(9e9, 8e8), want[1].nan_to_num(9e9, 8e8))
    assert torch.equal(dev[0].cpu(), kc) and torch.equal(dev[1].cpu(), vc)
    assert torch.equal(dev[4].cpu().nan_to_num(9e9, 8e8), w.nan_to_num(9e9, 8e8))


def test_evict_with_missing_pages(cuda_device):
    kc, vc, table, n, _ = make_cache([100, 90], 16, 2, 64, torch.bfloat16, seed=14)
    table[0, 1] = -1
    w = torch.rand(2, 2, 100, generator=torch.Generator().manual_seed(15))
    dev = [x.to(cuda_device) for x in (kc, vc, table, n, w)]
    got = born_cache_evict(*dev, 60, 10)
    want = born_cache_evict(kc, vc, table, n, w, 60, 10)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    assert torch.equal(dev[0].cpu(), kc) and torch.equal(dev[1].cpu(), vc)


def test_a_server_run_on_the_gpu(cuda_device):
    """Prompt, tokens one by one in a replayed graph, an eviction, more tokens,
    against the same run on the CPU in fp32."""
    lens, page, H, Hkv, D, steps = [150, 37], 16, 8, 2, 64, 4
    cap = 208
    kc, vc, table, n, _ = make_cache([cap, cap], page, Hkv, D, seed=16)
    g = torch.Generator().manual_seed(17)
    n.copy_(torch.tensor(lens, dtype=torch.int32))
    cu = torch.tensor(ref.starts(lens), dtype=torch.int32)
    pre = torch.randn(sum(lens), H + 2 * Hkv, D, generator=g) + 0.3
    ang = torch.rand(cap, D // 2, generator=g) * 3
    more = torch.randn(2 * steps, 2, H + 2 * Hkv, D, generator=g) + 0.3

    def split(x):
        return x[:, :H], x[:, H : H + Hkv], x[:, H + Hkv :]

    def serve(dev, graphs):
        c = [x.to(dev, copy=True) for x in (kc, vc, table, n, cu, ang.cos(), ang.sin())]
        k_, v_, tb, ln, cs, co, si = c
        outs = []
        q = fused_qk_rope_l2_normalize_append(*split(pre.to(dev)), co, si, k_, v_, tb, ln, cs)
        rows = [(tb[b, torch.arange(x, device=dev) // page].long(), torch.arange(x, device=dev) % page) for b, x in enumerate(lens)]
        keys, vals = (torch.cat([t[r] for r in rows]) for t in (k_, v_))
        outs.append(flash_born_attention_packed(q, keys, vals, 2.0, cs))
        weight = torch.zeros(2, Hkv, cap, device=dev)
        pos = torch.tensor(lens, dtype=torch.int32, device=dev)
        x_in = torch.zeros(2, H + 2 * Hkv, D, device=dev)

        def step():
            q = fused_qk_rope_l2_normalize_append(*split(x_in), co, si, k_, v_, tb, ln, None, pos)
            return flash_born_attention_paged(q, k_, v_, tb, ln, 2.0, 1e-12, 0, weight)

        run = step
        if graphs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held = step()

            def run():
                graph.replay()
                return held

        for i in range(2 * steps):
            if i == steps:
                new, w2, _ = born_cache_evict(k_, v_, tb, ln, weight, 32, 8)
                ln.copy_(new)
                weight.copy_(w2)
            x_in.copy_(more[i].to(dev))
            ln += 1
            outs.append(run().clone())
            pos += 1
        return outs, weight, ln

    with torch.no_grad():
        a, wa, la = serve(torch.device("cpu"), False)
        b, wb, lb = serve(cuda_device, True)
    assert la.tolist() == lb.tolist() == [36, 36]
    for x, y in zip(a, b):
        assert torch.allclose(x, y.cpu(), atol=2e-5)
    assert torch.allclose(wa, wb.cpu(), atol=2e-4)


def test_streams_and_two_graphs(cuda_device):
    # Two captured graphs own their workspaces, and replay beside each other.
    kc, vc, table, n, _ = make_cache([2500, 900], 16, 2, 64, torch.bfloat16, seed=18, device=cuda_device)
    g = torch.Generator().manual_seed(19)
    q1, q2 = (torch.randn(2, 8, 64, generator=g).to(device=cuda_device, dtype=torch.bfloat16) for _ in range(2))
    want = [flash_born_attention_paged(q, kc, vc, table, n, 2.0) for q in (q1, q2)]
    graphs, held = [], []
    for q in (q1, q2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(flash_born_attention_paged(q, kc, vc, table, n, 2.0))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for _ in range(3):
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            other = flash_born_attention_paged(q1, kc, vc, table, n, 2.0)
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]) and torch.equal(other, want[0])


def test_batches_without_sequences_or_tokens(cuda_device):
    for dev in ("cpu", cuda_device):
        kc, vc = (torch.randn(3, 16, 2, 64, device=dev) for _ in range(2))
        before = kc.clone(), vc.clone()
        table, lens = torch.zeros(0, 2, dtype=torch.int32, device=dev), torch.zeros(0, dtype=torch.int32, device=dev)
        weight = torch.zeros(0, 2, 32, device=dev)
        x = torch.randn(5, 4, 64, device=dev)
        assert flash_born_attention_paged(x[:0], kc, vc, table, lens, 1.0, key_weight=weight).shape == (0, 4, 64)
        cu = torch.zeros(1, dtype=torch.int32, device=dev)
        q = fused_qk_rope_l2_normalize_append(x, x[:, :2], x[:, :2], None, None, kc, vc, table, lens, cu)
        assert q.shape == x.shape and not q.any()
        one, n = torch.ones(1, 2, dtype=torch.int32, device=dev), torch.full((1,), 3, dtype=torch.int32, device=dev)
        cu = torch.zeros(2, dtype=torch.int32, device=dev)
        q = fused_qk_rope_l2_normalize_append(x[:0], x[:0, :2], x[:0, :2], None, None, kc, vc, one, n, cu)
        assert q.shape == (0, 4, 64)
        lens_out, w, kept = born_cache_evict(kc, vc, table, lens, weight, 8)
        assert lens_out.shape == (0,) and w.shape == weight.shape and kept.shape == (0, 2, 8)
        assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


def test_int64_tables_name_no_other_page(cuda_device):
    # 2^32 is no page of the cache: nothing is read there, and nothing written.
    g = torch.Generator().manual_seed(31)
    kc, vc, x = (torch.randn(*s, generator=g).to(cuda_device) for s in ((4, 16, 2, 64), (4, 16, 2, 64), (1, 4, 64)))
    before = kc.clone(), vc.clone()
    lens = torch.tensor([20], device=cuda_device)
    far = torch.tensor([[1, 1 << 32]], device=cuda_device)
    near = torch.tensor([[1, -1]], device=cuda_device, dtype=torch.int32)
    assert torch.equal(flash_born_attention_paged(x, kc, vc, far, lens, 1.0), flash_born_attention_paged(x, kc, vc, near, lens, 1.0))
    fused_qk_rope_l2_normalize_append(x, x[:, :2], x[:, :2], None, None, kc, vc, far, lens)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])


@pytest.mark.parametrize("page", [16, 24])
def test_offsets_past_32_bits(cuda_device, page):
    # The same rows in a cache's first pages and behind its first 4 GiB give the same.
    B, Hkv, D, n = 2, 8, 128, 100
    per = -(-n // page)
    pages = (9 << 29) // (page * Hkv * D * 2) + 4 * per * B  # 4.5 GiB and more of bf16
    g = torch.Generator().manual_seed(32)
    kc, vc = (torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    lens = torch.full((B,), n, dtype=torch.int32, device=cuda_device)
    low = torch.arange(B * per, dtype=torch.int32, device=cuda_device).view(B, per)
    high = pages - 1 - low
    to_low, to_high = low + B * per, high - B * per
    assert int(to_high.min()) * page * Hkv * D * 2 > 1 << 32
    q, k, v = (torch.randn(B * n, h, D, generator=g).to(device=cuda_device, dtype=torch.bfloat16) for h in (16, Hkv, Hkv))
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=cuda_device)
    weight = torch.rand(B, Hkv, n, generator=g).to(cuda_device)
    got = []
    for table, to in ((low, to_low), (high, to_high)):
        qn = fused_qk_rope_l2_normalize_append(q, k, v, None, None, kc, vc, table, lens, cu)
        out = flash_born_attention_paged(qn[n - 1 :: n], kc, vc, table, lens, 1.0)
        cut, _, kept = born_cache_evict(kc, vc, table, lens, weight, 50, 10, to)
        moved = flash_born_attention_paged(qn[n - 1 :: n], kc, vc, to, cut, 1.0)
        born_cache_evict(kc, vc, table, lens, weight, 50, 10)
        own = flash_born_attention_paged(qn[n - 1 :: n], kc, vc, table, cut, 1.0)
        assert torch.equal(own, moved) and out.any() and moved.any()
        got.append((out, moved, kept))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_evict_over_one_span_of_the_selection(cuda_device):
    # More keys than the workgroup's threads hold at once, with ties across the spans.
    n, budget, recent = 40000, 17000, 100
    g = torch.Generator().manual_seed(33)
    w = torch.randint(0, 500, (1, 2, n), generator=g).float()
    w[0, 1, 5000:30000] = 0.0
    kc, vc, table, lens, _ = make_cache([n], 64, 2, 8, torch.float32, 34)
    want = born_cache_evict(kc.clone(), vc.clone(), table, lens, w, budget, recent)
    k2, v2 = kc.to(cuda_device), vc.to(cuda_device)
    got = born_cache_evict(k2, v2, table.to(cuda_device), lens.to(cuda_device), w.to(cuda_device), budget, recent)
    k1, v1 = kc.clone(), vc.clone()
    born_cache_evict(k1, v1, table, lens, w, budget, recent)
    for a, b in zip((*got, k2, v2), (*want, k1, v1)):
        assert torch.equal(a.cpu().to(b.dtype), b)


def test_two_streams_at_once(cuda_device):
    # Calls that overlap share nothing: each has its own workspace.
    cases = [make_cache([3000, 700], 16, 2, 64, torch.float32, s) for s in (35, 36)]
    sets = []
    for i, (kc, vc, table, lens, _) in enumerate(cases):
        q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(37 + i))
        sets.append([x.to(cuda_device) for x in (q, kc, vc, table, lens)])
    alone = [flash_born_attention_paged(*s, 1.0) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                outs[i].append(flash_born_attention_paged(*s, 1.0))
    torch.cuda.synchronize()
    for a, many in zip(alone, outs):
        assert all(torch.equal(a, x) for x in many)

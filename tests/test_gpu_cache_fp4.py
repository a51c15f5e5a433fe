"""The 4-bit paged cache on the GPU: what is stored against the same call on the
CPU, bit for bit; attention against its formula in 64 bits within fp4_ref's bounds."""

from __future__ import annotations

import math

import pytest
import torch

import fp4_ref as ref
import serve_ref
from quantumdlblocks_amd import (
    born_cache_evict_fp4,
    born_cache_fp4,
    born_cache_read_fp4,
    flash_born_attention_packed,
    flash_born_attention_paged_fp4,
    fused_qk_rope_l2_normalize_append,
    fused_qk_rope_l2_normalize_append_fp4,
)

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INT = dict(dtype=torch.int32)


def _to(dev, *xs):
    return [tuple(t.to(dev) for t in x) if isinstance(x, tuple) else x.to(dev) if isinstance(x, torch.Tensor) else x for x in xs]


# ---------------------------------------------------------------------------
# Storing and reading
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,freqs", [(64, 32), (128, 64), (24, 5), (256, 200), (8, 4), (80, 40), (96, 48), (40, 20)])
@pytest.mark.parametrize("rope", [True, False])
def test_append(cuda_device, dtype, D, freqs, rope):
    dt, page, H, Hkv = DT[dtype], 16, 6, 2
    full, new = [50, 3, 0, 200], [20, 3, 0, 37]
    cache, table, n, _ = ref.make_cache(full, page, Hkv, D, seed=8)
    table[3, 12] = -1  # the last slots have no page
    g = torch.Generator().manual_seed(9)
    N = sum(new) + 2
    q, k, v = (torch.randn(N, h, D, generator=g).to(dt) for h in (H, Hkv, Hkv))
    cu = torch.tensor(serve_ref.starts(new), **INT)
    pos = torch.randint(0, 40, (N,), generator=g, **INT)
    pos[3] = 1000
    ang = torch.rand(40, freqs, generator=g) * 6
    tables = (ang.cos(), ang.sin()) if rope else (None, None)
    for positions in (pos, None):
        want = tuple(t.clone() for t in cache)
        qd = fused_qk_rope_l2_normalize_append_fp4(q.double(), k.double(), v.double(), *tables, want, table, n, cu, positions, 1e-6)
        dev = _to(cuda_device, q, k, v, *tables, cache, table, n, cu, positions)
        got = fused_qk_rope_l2_normalize_append_fp4(*dev, eps=1e-6)
        # Rounded once; before that, sums of D squares and a handful of fp32 operations.
        d = (got.double().cpu() - qd).abs()
        assert (d <= serve_ref.HALF_STEP[dt] * 1.02 * qd.abs() + (D + 32) * 2.0 ** -24).all() and not got[-2:].any()
        # The key's bits differ in 64 bits by the order of a sum at most, 2^-45 of
        # it: no code of 10^4 random ones lies that near its border.
        for a, b in zip(dev[5], want):
            assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [128, 72])
def test_append_of_many_tokens(cuda_device, dtype, D):
    """Enough of them that a token's lanes take several heads."""
    dt, page, H, Hkv = DT[dtype], 16, 42 if D == 72 else 35, 7
    half, vec = D // 2, 8 if dtype != "fp32" and D % 16 == 0 else 4
    lanes = 1 << (-(-half // vec) - 1).bit_length()
    N = -(-(1 << 20) // (H * lanes)) + 3
    new, B = [N - 50, 7, 0, 40], 4
    full = [N - 50 + 20, 7, 5, 60]
    cache, table, n, _ = ref.make_cache(full, page, Hkv, D, seed=19)
    g = torch.Generator().manual_seed(19)
    q, k, v = (torch.randn(N, h, D, generator=g).to(dt) for h in (H, Hkv, Hkv))
    cu = torch.tensor(serve_ref.starts(new), **INT)
    ang = torch.rand(N, half - 1, generator=g) * 6
    want = tuple(t.clone() for t in cache)
    qd = fused_qk_rope_l2_normalize_append_fp4(q.double(), k.double(), v.double(), ang.cos(), ang.sin(), want, table, n, cu)
    dev = _to(cuda_device, q, k, v, ang.cos(), ang.sin(), cache, table, n, cu)
    got = fused_qk_rope_l2_normalize_append_fp4(*dev)
    d = (got.double().cpu() - qd).abs()
    assert (d <= serve_ref.HALF_STEP[dt] * 1.02 * qd.abs() + (D + 32) * 2.0 ** -24).all() and not got[-3:].any()
    for a, b in zip(dev[5], want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", list(DT))
def test_values_at_the_codes_borders(cuda_device, dtype):
    ties = [0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.0, -0.0]
    near = [x * (1 + s * torch.finfo(DT[dtype]).eps) for x in ties for s in (-1, 1)]
    rows = []
    for size in (1.0, 2.0 ** -10, 8.0, 2.0 ** -3 * 1.5):
        for some in (ties, near, near[::-1], near[7:]):
            rows.append(([7.0 * size] + [x * size for x in some] + [0.0] * 32)[:32])
    rows.append([0.0] * 32)
    if dtype != "fp16":
        rows += [[x * 2.0 ** 120 for x in rows[0]], [x * 2.0 ** -130 for x in rows[0]], [2.0 ** -133] * 32]
        rows += [[x * 2.0 ** 125 for x in rows[0]], [x * 1.01 * 2.0 ** 125 for x in rows[0]]]  # as far as it goes, and past it
    v = torch.tensor(rows).to(DT[dtype]).view(-1, 1, 32)
    N = v.shape[0]
    table, n = torch.arange(N, **INT).view(-1, 1), torch.ones(N, **INT)
    want, got = born_cache_fp4(N, 1, 1, 32, device="cpu"), born_cache_fp4(N, 1, 1, 32, device=cuda_device)
    fused_qk_rope_l2_normalize_append_fp4(v, v, v, None, None, want, table, n)
    fused_qk_rope_l2_normalize_append_fp4(*_to(cuda_device, v, v, v), None, None, got, *_to(cuda_device, table, n))
    assert torch.equal(got.v.cpu(), want.v) and torch.equal(got.v_scale.cpu(), want.v_scale)
    assert dtype == "fp16" or want.v_scale[-2:].view(-1).tolist() == [252, 255]
    # Read back exactly, in every type that can hold them.
    cu = torch.arange(N + 1, **INT)
    for dt in DT.values():
        a = born_cache_read_fp4(got, *_to(cuda_device, table, n, cu), N, dtype=dt)
        b = born_cache_read_fp4(want, table, n, cu, N, dtype=dt)
        assert all(torch.equal(x.cpu().nan_to_num(8.0), y.nan_to_num(8.0)) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [8, 40, 64, 96, 256])
def test_read(cuda_device, dtype, D):
    lens, cu = [70, 0, 33, 129], [0, 70, 75, 80, 99]
    for page in (1, 16, 24):
        cache, table, n, _ = ref.make_cache(lens, page, 3, D, seed=2)
        table[3, 2] = -1
        total = 101
        want = born_cache_read_fp4(cache, table, n, torch.tensor(cu, **INT), total, D, DT[dtype])
        dev = _to(cuda_device, cache, table, n, torch.tensor(cu, **INT))
        got = born_cache_read_fp4(*dev, total, D, DT[dtype])
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def _attend(dev, lens, page, H, Hkv, D, dtype, new=None, window=0, scale=2.0, eps=1e-12, weigh=False, seed=0, size=1.0, columns=0):
    cache, table, n, _ = ref.make_cache(lens, page, Hkv, D, seed)
    table = torch.nn.functional.pad(table, (0, max(0, columns - table.shape[1])), value=-1)
    cu = None if new is None else serve_ref.starts(new)
    N = len(lens) if new is None else cu[-1] + 2  # two rows behind the last sequence
    q = torch.nn.functional.normalize(torch.randn(N, H, D, generator=torch.Generator().manual_seed(seed + 1)) + 0.1, dim=-1) * size
    q = q.to(dtype)
    weight = torch.full((len(lens), Hkv, max(lens + [1])), 0.5, device=dev) if weigh else None
    c, t, l, x, s, starts = _to(dev, cache, table, n, q, scale, None if cu is None else torch.tensor(cu, **INT))
    out = flash_born_attention_paged_fp4(x, c, t, l, s, starts, eps, window, weight)
    o, w = ref.attend(q, cache, table[:, : max(1, -(-max(lens + [1]) // page))], n, scale, cu, eps, window)
    assert out.dtype is dtype and ref.worst(out, o) <= 1.0
    if new is not None:
        assert not out[-2:].any()
    if weigh:
        m = min(weight.shape[2], w[0].shape[2])
        y, e = w[0][..., :m] + 0.5, w[1][..., :m] + 2.0 ** -24 * 2.0 * (w[0][..., :m] + 0.5)
        assert ref.worst(weight[..., :m], (y, e)) <= 1.0 and (weight[..., m:] == 0.5).all()
    return out


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [8, 40, 64, 80, 96, 128, 160, 256])
@pytest.mark.parametrize("H,Hkv", [(4, 2), (1, 1), (20, 1)])
def test_one_token_head_dims_and_groups(cuda_device, dtype, D, H, Hkv):
    _attend(cuda_device, [130, 0, 1, 33], 16, H, Hkv, D, DT[dtype])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_one_token_pages_and_windows(cuda_device, dtype, page, window):
    _attend(cuda_device, [300, 31, 32, 129], page, 4, 2, 64, DT[dtype], window=window, weigh=True, seed=2)


@pytest.mark.parametrize("dtype", list(DT))
def test_one_token_long_caches_are_split(cuda_device, dtype):
    scale = torch.tensor([1.0, -2.0, 30.0, 0.1])
    _attend(cuda_device, [2500, 5, 1024, 1025], 16, 4, 2, 128, DT[dtype], scale=scale, weigh=True, seed=3)
    _attend(cuda_device, [2500], 32, 4, 4, 64, DT[dtype], scale=scale, eps=0.3, seed=4)
    _attend(cuda_device, [1500, 700], 16, 40, 2, 96, DT[dtype], weigh=True, seed=4)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 200.0])
def test_overlaps_of_any_size_keep_their_weight(cuda_device, dtype, size):
    _attend(cuda_device, [700, 40], 16, 4, 2, 64, DT[dtype], size=size, scale=1.0, weigh=True, seed=5)
    _attend(cuda_device, [700, 40], 16, 4, 2, 64, DT[dtype], new=[40, 3], size=size, scale=1.0, seed=5)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [8, 40, 64, 96, 128, 256])
@pytest.mark.parametrize("H,Hkv", [(4, 2), (3, 3), (20, 1)])
def test_several_tokens_head_dims_and_groups(cuda_device, dtype, D, H, Hkv):
    _attend(cuda_device, [130, 0, 1, 33, 64], 16, H, Hkv, D, DT[dtype], new=[5, 0, 1, 33, 2], seed=6)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("page", [1, 7, 16, 24, 64])
@pytest.mark.parametrize("window", [0, 1, 50])
@pytest.mark.parametrize("H", [4, 16])  # all rows narrow, some wide
def test_several_tokens_pages_and_windows(cuda_device, dtype, page, window, H):
    _attend(cuda_device, [300, 31, 2, 129, 8], page, H, 2, 64, DT[dtype], new=[70, 31, 1, 4, 12], window=window, seed=7)  # 12 of 8


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
def test_several_tokens_long_and_mixed(cuda_device, dtype, D):
    scale = torch.tensor([1.0, -2.0, 30.0, 0.1])
    _attend(cuda_device, [1500, 700, 1, 333], 16, 4, 2, D, DT[dtype], new=[1, 300, 1, 9], scale=scale, seed=8)
    _attend(cuda_device, [900, 2000, 333], 16, 4, 1, D, DT[dtype], new=[40, 1, 50], scale=scale, seed=13)
    _attend(cuda_device, [1200], 16, 8, 2, D, DT[dtype], new=[260], window=300, seed=9)
    _attend(cuda_device, [900], 32, 4, 4, D, DT[dtype], new=[1], scale=scale, eps=0.3, seed=10)


@pytest.mark.parametrize("dtype", list(DT))
def test_several_tokens_over_tables_of_one_step(cuda_device, dtype):
    """No more than 128 keys a sequence: nothing to share out."""
    for H in (2, 8):
        _attend(cuda_device, [112, 90, 0, 7, 100], 16, H, 2, 64, DT[dtype], new=[112, 50, 0, 7, 33], seed=11)
    _attend(cuda_device, [100, 90, 3], 5, 6, 1, 128, DT[dtype], new=[1, 80, 3], window=40, seed=12)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 10])
def test_few_tokens_each_over_wide_tables(cuda_device, dtype, D, page):
    """Tables of 2^17 keys: narrow and wide sequences in launches of their own."""
    new = [60, 1, 4, 0, 9, 8, 3] + [5] * 14
    _attend(cuda_device, [60, 300, 4, 7, 1000, 20, 33] + [40 + i for i in range(14)], page, 4, 1, D, DT[dtype], new=new, seed=16,
            columns=(1 << 17) // page)
    for weigh in (False, True):
        _attend(cuda_device, [60, 300, 0, 7], page, 4, 1, D, DT[dtype], seed=16, columns=(1 << 17) // page, weigh=weigh)


@pytest.mark.parametrize("several", [False, True])
def test_missing_pages_lengths_and_bytes_of_nobody(cuda_device, several):
    new = [40, 60, 3] if several else None
    for dt in DT.values():
        cache, table, n, free = ref.make_cache([100, 100, 100], 16, 2, 64, seed=6)
        for t in cache:
            t[free] = 255  # scales that are not numbers, in pages of nobody
        table[0, 2] = -1
        table[1, 3] = cache[0].shape[0] + 5
        n[0], n[1], n[2] = 90, 5000, -3
        cache[2][table[0, 5].long(), 10:] = 255  # behind the last key
        cache[3][table[0, 5].long(), 10:] = 255
        cu = None if new is None else serve_ref.starts(new)
        q = torch.randn(3 if new is None else cu[-1], 4, 64, generator=torch.Generator().manual_seed(2)).to(dt)
        dev = _to(cuda_device, q, cache, table, n)
        out = flash_born_attention_paged_fp4(*dev, 1.0, None if cu is None else torch.tensor(cu, **INT).to(cuda_device), 0.0)
        o, _ = ref.attend(q, cache, table, n, 1.0, cu, 0.0)
        assert ref.worst(out, o) <= 1.0 and not out[-1].any()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tokens_that_are_no_numbers_reach_those_that_see_them_alone(cuda_device, dtype, D):
    dt = DT[dtype]
    for n_new, page, G in ((9, 4, 2), (150, 16, 2), (150, 16, 8), (150, 1, 4)):
        g = torch.Generator().manual_seed(7)
        k, v, x = (torch.rand(n_new, h, D, generator=g).to(dt) for h in (2, 2, 2 * G))
        a, b = n_new // 3, 2 * n_new // 3
        k[a, 0, 5], v[b, 1, 40] = math.nan, math.inf
        cache = born_cache_fp4(-(-n_new // page), page, 2, D, device=cuda_device)
        table, n = torch.arange(-(-n_new // page), **INT).view(1, -1), torch.tensor([n_new], **INT)
        cu = torch.tensor([0, n_new], **INT)
        table, n, cu, x, k, v = _to(cuda_device, table, n, cu, x, k, v)
        q = fused_qk_rope_l2_normalize_append_fp4(x, k, v, None, None, cache, table, n, cu)
        out = flash_born_attention_paged_fp4(q, cache, table, n, -1.0, cu, window_size=2)
        nan = out.isnan()
        assert torch.equal(nan.all(-1), nan.any(-1))
        for h, at in ((0, a), (1, b)):
            for i in range(G * h, G * h + G):
                assert torch.nonzero(nan[:, i].any(-1)).view(-1).tolist() == [at, at + 1]
        # One token, which sees them all.
        weight = torch.zeros(1, 2, n_new, device=cuda_device)
        one = flash_born_attention_paged_fp4(q[-1:], cache, table, n, 1.0, key_weight=weight)
        assert one.isnan().all() and weight.isnan().all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
def test_queries_that_are_no_numbers_are_rows_of_their_own(cuda_device, dtype, D):
    for new, G in (([9, 3], 2), ([300, 7], 4), ([1, 1], 8)):
        cache, table, n, _ = ref.make_cache([330, 200], 16, 2, D, seed=17, device=cuda_device)
        N = sum(new)
        q = torch.randn(N, 2 * G, D, generator=torch.Generator().manual_seed(17)).to(device=cuda_device, dtype=DT[dtype])
        cu = torch.tensor(serve_ref.starts(new), device=cuda_device, **INT)
        want = flash_born_attention_paged_fp4(q, cache, table, n, 1.0, cu)
        for bad in (math.nan, -math.nan, math.inf):
            for scale in (1.0, -1.0):
                x = q.clone()
                x[N // 2, 1, 3] = x[N - 1, 0, D - 1] = bad
                out = flash_born_attention_paged_fp4(x, cache, table, n, scale, cu)
                if scale > 0:
                    same = torch.ones(N, 2 * G, dtype=torch.bool, device=cuda_device)
                    same[N // 2, 1] = same[N - 1, 0] = False
                    assert torch.equal(out[same], want[same])
                # An infinite overlap has a weight of infinity, or none where all of them are negative.
                assert bad == math.inf or (out[N // 2, 1].isnan().all() and out[N - 1, 0].isnan().all())


def test_starts_that_do_not_ascend_stay_in_bounds(cuda_device):
    """They have no meaning, but nothing behind the tensors is touched, and rows
    that the call is right about elsewhere are not changed by one before."""
    for B, room, N, H in ((100, 2000, 64, 16), (100, 100, 64, 16), (1100, 400, 96, 8), (6, 4000, 600, 8), (6, 100, 600, 8), (80, 3000, 700, 4)):
        cache, table, n, _ = ref.make_cache([room] * 2, 16, 2, 64, seed=18, device=cuda_device)
        table, n = table.repeat(B // 2, 1), n.repeat(B // 2)
        q = torch.randn(N, H, 64, generator=torch.Generator().manual_seed(18)).to(device=cuda_device, dtype=torch.bfloat16)
        for starts in ([0, N] * (B // 2) + [N], [0] + [N - i % 7 * 5 for i in range(B)], [N] * B + [0], [-5, N + 9] * (B // 2) + [N]):
            cu = torch.tensor(starts, device=cuda_device, **INT)
            out = flash_born_attention_paged_fp4(q, cache, table, n, 1.0, cu)
            assert out.shape == q.shape
            torch.cuda.synchronize()
        even = torch.tensor([i * N // B for i in range(B + 1)], device=cuda_device, **INT)
        got = flash_born_attention_paged_fp4(q, cache, table, n, 1.0, even)
        assert got.isfinite().all()


def test_strides_and_index_types(cuda_device):
    cache, table, n, _ = ref.make_cache([70, 20, 48], 16, 2, 64, seed=7, device=cuda_device)
    g = torch.Generator().manual_seed(7)
    q = torch.randn(9, 4, 64, generator=g).to(device=cuda_device, dtype=torch.bfloat16)
    cu = torch.tensor([0, 3, 4, 9], device=cuda_device, **INT)
    want = flash_born_attention_paged_fp4(q, cache, table, n, 2.0, cu)
    tokens_first = tuple(t.contiguous() for t in cache)
    both = torch.stack(cache[:2], 1)  # one allocation: (pages, 2, page, Hkv, W / 2)
    odd = torch.zeros(*cache[2].shape[:3], 5, dtype=torch.uint8, device=cuda_device)[..., 2:4]  # scales need no alignment
    odd.copy_(cache[2])
    for c in (tokens_first, (both[:, 0], both[:, 1], odd, cache[3])):
        assert torch.equal(flash_born_attention_paged_fp4(q, c, table, n, 2.0, cu), want)
        k = born_cache_read_fp4(c, table, n, cu, 9)
        assert all(torch.equal(a, b) for a, b in zip(k, born_cache_read_fp4(cache, table, n, cu, 9)))
    wide = torch.full((3, table.shape[1] + 3), -1, device=cuda_device, **INT)
    wide[:, : table.shape[1]] = table
    got = flash_born_attention_paged_fp4(q.transpose(0, 1).contiguous().transpose(0, 1), cache, wide[:, : table.shape[1]], n, 2.0, cu)
    assert torch.equal(got, want)
    assert torch.equal(flash_born_attention_paged_fp4(q, cache, table.long(), n.long(), torch.tensor(2.0, device=cuda_device), cu.long()), want)
    with pytest.raises(ValueError):
        flash_born_attention_paged_fp4(q, (cache[0].contiguous().view(-1, 2, 16, 32).transpose(1, 2)[..., ::2], *cache[1:]), table, n, 2.0, cu)
    with pytest.raises(NotImplementedError):
        flash_born_attention_paged_fp4(q[..., :60], cache, table, n, 2.0, cu)
    with pytest.raises(NotImplementedError):
        flash_born_attention_paged_fp4(q.double(), cache, table, n, 2.0, cu)
    with pytest.raises(NotImplementedError):
        born_cache_read_fp4(cache, table, n, cu, 9, dtype=torch.float64)
    with pytest.raises(NotImplementedError):
        flash_born_attention_paged_fp4(torch.zeros(1, 1, 288, device=cuda_device), born_cache_fp4(1, 16, 1, 288, cuda_device), table[:1], n[:1], 1.0)


def test_offsets_past_32_bits(cuda_device):
    """Pages that start past 2^32 bytes, and a page past 2^31."""
    for pages, page in ((40000, 64), (2, 1 << 20)):
        if pages > 2:
            codes = [torch.zeros(pages, 33, page, 64, dtype=torch.uint8, device=cuda_device).transpose(1, 2) for _ in range(2)]
            assert codes[0].stride(0) * (pages - 1) > 1 << 32
        else:
            codes = [torch.zeros(pages, page, 33, 64, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
            assert codes[0].stride(1) * (page - 1) > 1 << 31
        scales = [torch.full((*c.shape[:3], 4), 127, dtype=torch.uint8, device=cuda_device) for c in codes]
        n_keys = 200 if pages > 2 else page
        last = pages - 1
        table = torch.arange(last, last - 4, -1, device=cuda_device, **INT).view(1, -1) if pages > 2 else torch.tensor([[1]], device=cuda_device, **INT)
        n = torch.tensor([n_keys], device=cuda_device, **INT)
        g = torch.Generator().manual_seed(0)
        k, v, x = (torch.randn(50, 33, 128, generator=g).to(cuda_device, torch.bfloat16) for _ in range(3))
        cu = torch.tensor([0, 50], device=cuda_device, **INT)
        cache = (*codes, *scales)
        q = fused_qk_rope_l2_normalize_append_fp4(x, k, v, None, None, cache, table, n, cu)
        small = born_cache_fp4(4, 64, 33, 128, device=cuda_device)
        near = torch.arange(4, device=cuda_device, **INT).view(1, -1)
        few = torch.tensor([200], device=cuda_device, **INT)
        fused_qk_rope_l2_normalize_append_fp4(x, k, v, None, None, small, near, few, cu)
        assert all(torch.equal(a, b) for a, b in zip(born_cache_read_fp4(cache, table, n, cu, 50), born_cache_read_fp4(small, near, few, cu, 50)))
        for starts, rows in ((cu, q), (torch.tensor([0, 1], device=cuda_device, **INT), q[-1:])):
            a = flash_born_attention_paged_fp4(rows, cache, table, n, 1.0, starts, window_size=60)
            b = flash_born_attention_paged_fp4(rows, small, near, few, 1.0, starts, window_size=60)
            # Splits may differ: fp32 sums in another order, then one rounding.
            assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=1e-5)
        del codes, scales, cache


# ---------------------------------------------------------------------------
# Eviction
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("D", [24, 128, 160, 256])
@pytest.mark.parametrize("lens,budget,recent", [
    ([100, 20, 0, 65], 64, 16), ([100, 7], 64, 64), ([300], 0, 0), ([5000, 1300], 1024, 100), ([70], 69, 0),
])
def test_evict(cuda_device, lens, budget, recent, D, inplace):
    page, Hkv = 16, 2
    room = max(1, -(-min(budget, max(lens)) // page))
    cache, table, n, free = ref.make_cache(lens, page, Hkv, D, seed=12, spare=len(lens) * room)
    table[0, 1] = -1
    to = None if inplace else free[: len(lens) * room].view(len(lens), room).to(torch.int32)
    g = torch.Generator().manual_seed(13)
    w = torch.randn(len(lens), Hkv, max(lens) - 3, generator=g).exp()
    w = torch.where(torch.rand(w.shape, generator=g) < 0.4, torch.zeros_like(w), w)  # ties
    w[0, 0, 5], w[0, 1, 7], w[0, 1, 9] = float("nan"), float("inf"), -1.0
    dev = _to(cuda_device, cache, table, n, w)
    got = born_cache_evict_fp4(*dev, budget, recent, None if to is None else to.to(cuda_device))
    want = born_cache_evict_fp4(cache, table, n, w, budget, recent, to)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[2].cpu(), want[2])
    assert torch.equal(got[1].cpu().nan_to_num(9e9, 8e8), want[1].nan_to_num(9e9, 8e8))
    for a, b in zip(dev[0], cache):
        assert torch.equal(a.cpu(), b)


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
def _run_server(dev, dtype, H, Hkv, D, page):
    """Prompts, decoding with the keys' weights kept, an eviction, a second turn,
    drafted tokens; every output, and the cache as it ends."""
    g = torch.Generator().manual_seed(21)
    prompts, B = [40, 3, 77], 3
    cache = born_cache_fp4(40, page, Hkv, D, device=dev)
    table = torch.randperm(36, generator=g)[:30].view(B, 10).to(**INT).to(dev)
    way = 0.6 * D ** 0.5 * torch.nn.functional.normalize(torch.randn(Hkv, D, generator=g), dim=-1)
    ang = torch.outer(torch.arange(200.0), 1.0 / 100.0 ** (torch.arange(D // 2) / (D // 2)))
    cos, sin = ang.cos().to(dev), ang.sin().to(dev)
    outs, lens, at = [], [0] * B, [0] * B
    weight = torch.zeros(B, Hkv, 10 * page, device=dev)

    def step(new, decode=False):
        n = sum(new)
        q = torch.randn(n, H, D, generator=g) + way.repeat_interleave(H // Hkv, 0)
        k, v = torch.randn(n, Hkv, D, generator=g) + way, torch.randn(n, Hkv, D, generator=g)
        pos = torch.cat([torch.arange(a, a + x) for a, x in zip(at, new)]).to(**INT).to(dev)
        for b in range(B):
            lens[b] += new[b]
            at[b] += new[b]
        l = torch.tensor(lens, **INT).to(dev)
        cu = None if decode else torch.tensor(serve_ref.starts(new), **INT).to(dev)
        q = fused_qk_rope_l2_normalize_append_fp4(*(x.to(dev, dtype) for x in (q, k, v)), cos, sin, cache, table, l, cu, pos)
        outs.append(flash_born_attention_paged_fp4(q, cache, table, l, 3.0, cu, key_weight=weight if decode else None))
        return l

    step(prompts)
    for _ in range(4):
        l = step([1, 1, 1], decode=True)
    l, new_weight, kept = born_cache_evict_fp4(cache, table, l, weight, 32, 8)
    weight.copy_(new_weight)
    lens[:] = l.tolist()
    outs += [new_weight]
    step([20, 0, 5])
    step([4, 4, 4])
    step([1, 1, 1], decode=True)
    return outs, weight, kept, cache, lens


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (80, 5)])
def test_a_server_run_on_the_gpu(cuda_device, dtype, D, page):
    page = 16 if page == 16 else 13
    got = _run_server(cuda_device, DT[dtype], 4, 2, D, page)
    want = _run_server(torch.device("cpu"), DT[dtype], 4, 2, D, page)
    assert got[4] == want[4] and torch.equal(got[2].cpu(), want[2])
    for a, b in zip(got[3], want[3]):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(got[0], want[0]):
        # Queries rounded to the type by either side may differ by a step, an
        # overlap by as much, its square by twice it, on top and below; the output by one more.
        assert torch.allclose(a.float().cpu(), b.float(), rtol=8 * torch.finfo(DT[dtype]).eps, atol=8 * torch.finfo(DT[dtype]).eps)


def test_captured_steps_follow_their_lengths(cuda_device):
    H, Hkv, D, page, B = 8, 2, 128, 16, 3
    cache, table, n, _ = ref.make_cache([700, 20, 300], page, Hkv, D, seed=3, device=cuda_device)
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(6, h, D, generator=g).to(cuda_device, torch.bfloat16) for h in (H, Hkv, Hkv))
    cu = torch.tensor([0, 3, 4, 6], device=cuda_device, **INT)
    weight = torch.zeros(B, Hkv, 700, device=cuda_device)

    def step():
        x = fused_qk_rope_l2_normalize_append_fp4(q, k, v, None, None, cache, table, n, cu)
        several = flash_born_attention_paged_fp4(x, cache, table, n, 2.0, cu)
        one = flash_born_attention_paged_fp4(x[:3], cache, table, n, 2.0, key_weight=weight)
        return several, one, *born_cache_read_fp4(cache, table, n, cu, 6)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    start = tuple(t.clone() for t in cache)
    for lens, starts in (([700, 20, 300], [0, 3, 4, 6]), ([3, 20, 5], [0, 1, 2, 6]), ([640, 7, 123], [0, 6, 6, 6]), ([700, 20, 300], [0, 3, 4, 6])):
        for t, s in zip(cache, start):
            t.copy_(s)
        weight.zero_()
        n.copy_(torch.tensor(lens, **INT))
        cu.copy_(torch.tensor(starts, **INT))
        graph.replay()
        replayed, kept, stored = [x.clone() for x in got], weight.clone(), [t.clone() for t in cache]
        torch.cuda.synchronize()
        for t, s in zip(cache, start):
            t.copy_(s)
        weight.zero_()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(replayed, eager)) and torch.equal(kept, weight)
        assert all(torch.equal(a, b) for a, b in zip(stored, cache))


def test_two_streams_share_nothing(cuda_device):
    cache, table, n, _ = ref.make_cache([3000, 20, 2500], 16, 2, 128, seed=3, device=cuda_device)
    g = torch.Generator().manual_seed(6)
    a, b = (torch.randn(3, 8, 128, generator=g).to(cuda_device, torch.bfloat16) for _ in range(2))
    want = [flash_born_attention_paged_fp4(x, cache, table, n, 2.0) for x in (a, b)]
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for stream, x in ((s, a), (t, b)):
            with torch.cuda.stream(stream):
                got.append(flash_born_attention_paged_fp4(x, cache, table, n, 2.0))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


def test_many_sequences(cuda_device):
    """More sequences than a workgroup looks through to share out the keys."""
    lens = [i % 7 for i in range(1100)]
    _attend(cuda_device, lens, 4, 2, 1, 32, torch.bfloat16, seed=30)
    _attend(cuda_device, lens, 4, 2, 1, 32, torch.bfloat16, new=[(i // 3) % 3 for i in range(1100)], seed=31)
    _attend(cuda_device, [40 * (i % 9) for i in range(130)], 16, 2, 1, 32, torch.bfloat16, seed=32)
    _attend(cuda_device, [40 * (i % 9) for i in range(130)], 16, 2, 1, 32, torch.bfloat16, new=[(i % 5) * (i % 9) for i in range(130)], seed=33)
    new = [70 if i in (3, 500, 1099) else i % 2 for i in range(1100)]
    _attend(cuda_device, [2 * x + i % 5 for i, x in enumerate(new)], 16, 2, 1, 32, torch.bfloat16, new=new, seed=34)


def test_empty_calls(cuda_device):
    cache, table, n, _ = ref.make_cache([5, 5], 16, 2, 64, device=cuda_device)
    none = dict(device=cuda_device)
    z = lambda n_, h: torch.zeros(n_, h, 64, **none)  # noqa: E731
    e_table, e_lens, cu = torch.zeros(0, 3, **INT, **none), torch.zeros(0, **INT, **none), torch.zeros(1, **INT, **none)
    assert flash_born_attention_paged_fp4(z(0, 4), cache, e_table, e_lens, 1.0).shape == (0, 4, 64)
    assert not flash_born_attention_paged_fp4(z(2, 4) + 1, cache, e_table, e_lens, 1.0, cu).any()
    assert fused_qk_rope_l2_normalize_append_fp4(z(0, 4), z(0, 2), z(0, 2), None, None, cache, e_table, e_lens).shape == (0, 4, 64)
    assert not fused_qk_rope_l2_normalize_append_fp4(z(2, 4), z(2, 2), z(2, 2), None, None, cache, e_table, e_lens, cu).any()
    assert not born_cache_read_fp4(cache, e_table, e_lens, cu, 2)[0].any()
    narrow = table[:, :0]
    assert not flash_born_attention_paged_fp4(z(2, 4) + 1, cache, narrow, n, 1.0).any()
    empty = born_cache_fp4(0, 16, 2, 64, device=cuda_device)
    assert not flash_born_attention_paged_fp4(z(2, 4) + 1, empty, table, n, 1.0).any()
    q = fused_qk_rope_l2_normalize_append_fp4(z(2, 4) + 1, z(2, 2), z(2, 2), None, None, empty, table, n)
    assert torch.allclose(q.norm(dim=-1), torch.ones(2, 4, **none), atol=1e-5)
    assert born_cache_evict_fp4(cache, e_table, e_lens, torch.zeros(0, 2, 4, **none), 3)[2].shape == (0, 2, 3)


def test_second_turns_agree_with_the_wide_attention(cuda_device):
    """Over the values read back, the packed attention gives the same rows."""
    lens, new = [900, 250, 411], [300, 250, 7]
    cache, table, n, _ = ref.make_cache(lens, 16, 2, 128, seed=14, device=cuda_device)
    cu, ck = (torch.tensor(serve_ref.starts(x), device=cuda_device, **INT) for x in (new, lens))
    q = torch.nn.functional.normalize(torch.randn(sum(new), 8, 128, generator=torch.Generator().manual_seed(15)), dim=-1)  # 2228 rows
    q = q.to(cuda_device, torch.float32)
    k, v = born_cache_read_fp4(cache, table, n, ck, sum(lens), dtype=torch.float32)
    for window in (0, 100):
        a = flash_born_attention_paged_fp4(q, cache, table, n, 2.0, cu, window_size=window)
        b = flash_born_attention_packed(q, k, v, 2.0, cu, ck, window_size=window)
        # Each within its sums' 1000-odd fp32 roundings of the formula, of values up to 12.
        assert torch.allclose(a, b, rtol=0, atol=2 * 12 * 1000 * 2.0 ** -24)

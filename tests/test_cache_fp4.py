"""The 4-bit paged cache on the CPU: its format, appending, reading, attention of
one and of several tokens, evicting, refusals, and the C ABI's checks."""

from __future__ import annotations

import math
import os
import shutil
import subprocess

import pytest
import torch

import fp4_ref as ref
import serve_ref
from quantumdlblocks_amd import (
    BornCacheFp4,
    _native,
    born_cache_evict,
    born_cache_evict_fp4,
    born_cache_fp4,
    born_cache_read_fp4,
    flash_born_attention_packed,
    flash_born_attention_paged_fp4,
    fused_qk_rope_l2_normalize_append,
    fused_qk_rope_l2_normalize_append_fp4,
)
from quantumdlblocks_amd.kernels import born_fp4

INT = dict(dtype=torch.int32)


def test_the_stored_codes_are_the_nearest():
    g = torch.Generator().manual_seed(0)
    blocks = [torch.randn(32, generator=g).tolist() for _ in range(30)]
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0, -0.25, -5.0, -0.0, 6.0, 7.0]
    for size in (1.0, 2.0 ** -20, 3.0 * 2.0 ** 60):
        blocks.append([x * size for x in ties] + [0.0] * 19)
        blocks.append([x * size * (1 + 2.0 ** -40) for x in ties] + [0.0] * 19)
        blocks.append([x * size * (1 - 2.0 ** -40) for x in ties] + [7.0 * size] + [0.0] * 18)
    blocks += [[0.0] * 32, [2.0 ** -140] * 32, [math.inf] + [1.0] * 31, [1.0] * 31 + [math.nan]]
    blocks += [[7 * 2.0 ** 125] * 32, [7 * 2.0 ** 125 * (1 + 2.0 ** -24)] + [1.0] * 31, [-1.99 * 2.0 ** 127] * 32]
    codes, scales = born_fp4._encode(torch.tensor(blocks, dtype=torch.float64))
    for x, c, s in zip(blocks, codes.tolist(), scales.tolist()):
        e, want = ref.store_block(x)
        assert s == [e]
        assert [c[i // 2] >> 4 * (i % 2) & 15 for i in range(32)] == want
    got = born_fp4._decode(codes, scales)
    assert torch.equal(got.nan_to_num(9e99), ref.value(codes, scales).nan_to_num(9e99))


def test_the_stored_rows_are_near():
    x = torch.randn(4000, 128, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    y = born_fp4._decode(*born_fp4._encode(x))
    # Uniform rounding errors of normal values: 0.112 in norm; a block is off by
    # half its largest step, 1/7 of the largest value, at most.
    assert float((y - x).norm() / x.norm()) < 0.115
    top = x.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    assert bool(((y - x).unflatten(-1, (-1, 32)).abs() <= top / 3.5).all())
    for dt in (torch.bfloat16, torch.float32):
        assert torch.equal(y.to(dt).double(), y)


def test_an_empty_cache():
    c = born_cache_fp4(5, 16, 2, 80, device="cpu")
    assert isinstance(c, BornCacheFp4) and [tuple(t.shape) for t in c] == [(5, 16, 2, 48)] * 2 + [(5, 16, 2, 3)] * 2
    assert all(t.dtype == torch.uint8 and t.transpose(1, 2).is_contiguous() and not t.any() for t in c)
    for bad in ((-1, 16, 2, 64), (1, 0, 2, 64), (1, 16, 0, 64), (1, 16, 2, 0)):
        with pytest.raises(ValueError):
            born_cache_fp4(*bad, device="cpu")


@pytest.mark.parametrize("D", [8, 40, 64])
def test_append_stores_what_the_wide_cache_gets(D):
    page, Hkv, H = 4, 2, 4
    full, new = [7, 3, 9], [2, 0, 5]
    cache, table, n, _ = ref.make_cache(full, page, Hkv, D)
    before = [t.clone() for t in cache]
    N = sum(new) + 1  # one token behind the last sequence
    g = torch.Generator().manual_seed(4)
    q = torch.randn(N, H, D, generator=g)
    k, v = (torch.randn(N, Hkv, D, generator=g) for _ in range(2))
    ang = torch.rand(20, D // 2 - 1, generator=g)
    cu = torch.tensor(serve_ref.starts(new), **INT)
    pos = torch.tensor([5, 6, 30, 4, 5, 6, 7, 0], **INT)
    got = fused_qk_rope_l2_normalize_append_fp4(q, k, v, ang.cos(), ang.sin(), cache, table, n, cu, pos, 1e-6)
    kc, vc = (torch.zeros(cache[0].shape[0], page, Hkv, D, dtype=torch.float64) for _ in range(2))
    want = fused_qk_rope_l2_normalize_append(q.double(), k.double(), v.double(), ang.cos(), ang.sin(), kc, vc, table, n, cu, pos, 1e-6)
    assert torch.allclose(got.double(), want, atol=1e-6) and not got[-1:].any()
    written = torch.zeros(cache[0].shape[:2], dtype=torch.bool)
    for b, x in enumerate(new):
        for i in range(full[b] - x, full[b]):
            t, r = int(table[b, i // page]), i % page
            written[t, r] = True
            for h in range(Hkv):
                for codes, scales, row in ((cache[0], cache[2], kc[t, r, h]), (cache[1], cache[3], vc[t, r, h])):
                    row = row.tolist() + [0.0] * (-D % 32)
                    for blk in range(len(row) // 32):
                        e, want_c = ref.store_block(row[32 * blk : 32 * blk + 32])
                        c = codes[t, r, h, 16 * blk : 16 * blk + 16].tolist()
                        assert int(scales[t, r, h, blk]) == e and [c[i // 2] >> 4 * (i % 2) & 15 for i in range(32)] == want_c
    for a, b in zip(cache, before):
        assert torch.equal(a[~written], b[~written])


@pytest.mark.parametrize("cu", [[0, 3, 3, 10, 11], [0, 7, 7, 7, 7]])
def test_read_gives_a_sequences_last_keys(cu):
    lens, page, Hkv, D = [7, 0, 9, 5], 4, 2, 40
    cache, table, n, _ = ref.make_cache(lens, page, Hkv, D)
    table[2, 1] = -1
    total = cu[-1] + 2
    k, v = born_cache_read_fp4(cache, table, n, torch.tensor(cu, **INT), total, head_dim=D, dtype=torch.float32)
    want = torch.zeros(2, total, Hkv, D)
    for b, x in enumerate(lens):
        m = cu[b + 1] - cu[b]
        kk, vv, ok, _ = ref.rows(cache, table[b], x, D)
        for i in range(m):
            j = x - m + i
            if j >= 0 and ok[j]:
                want[0, cu[b] + i], want[1, cu[b] + i] = kk[j], vv[j]
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert born_cache_read_fp4(cache, table, n, torch.tensor(cu, **INT), total)[0].shape == (total, Hkv, 64)


@pytest.mark.parametrize("window", [0, 1, 3])
@pytest.mark.parametrize("page", [1, 4, 5])
def test_attention_of_one_token(page, window):
    lens = [7, 0, 1, 12]
    cache, table, n, _ = ref.make_cache(lens, page, 2, 40)
    q = torch.randn(4, 4, 40, generator=torch.Generator().manual_seed(3))
    scale = torch.tensor([1.0, 2.0, -0.5, 3.0])
    weight = torch.ones(4, 2, 11)
    out = flash_born_attention_paged_fp4(q, cache, table, n, scale, None, 0.01, window, weight)
    o, w = ref.attend(q, cache, table, n, scale, None, 0.01, window)
    assert torch.allclose(out.double(), o[0], atol=1e-5) and not out[1].any()
    m = min(11, w[0].shape[2])
    assert torch.allclose(weight[..., :m].double() - 1.0, w[0][..., :m], atol=1e-5)


@pytest.mark.parametrize("window", [0, 1, 4])
def test_attention_of_several_tokens(window):
    lens, new = [7, 4, 1, 12, 3], [3, 0, 1, 12, 5]  # the last has more tokens than keys
    cache, table, n, _ = ref.make_cache(lens, 4, 2, 32)
    cu = serve_ref.starts(new)
    q = torch.randn(cu[-1] + 2, 4, 32, generator=torch.Generator().manual_seed(5))
    out = flash_born_attention_paged_fp4(q, cache, table, n, 2.0, torch.tensor(cu, **INT), 0.0, window)
    o, _ = ref.attend(q, cache, table, n, 2.0, cu, 0.0, window)
    assert torch.allclose(out.double(), o[0], atol=1e-5) and not out[-2:].any() and not out[cu[4] : cu[4] + 2].any()
    # The same, from the keys read back, by the packed attention.
    k, v = born_cache_read_fp4(cache, table, n, torch.tensor(serve_ref.starts(lens), **INT), sum(lens), dtype=torch.float32)
    got = flash_born_attention_packed(q[: cu[-1]], k, v, 2.0, torch.tensor(cu), torch.tensor(serve_ref.starts(lens)), eps=0.0,
                                      window_size=window)
    assert torch.allclose(out[: cu[-1]], got, atol=1e-5)


def test_missing_pages_and_lengths_past_the_table():
    cache, table, n, _ = ref.make_cache([10, 10], 4, 1, 32)
    table[0, 1] = -1
    table[1, 2] = 1000
    n[0] = 99
    q = torch.randn(4, 2, 32)
    cu = torch.tensor([0, 2, 4], **INT)
    out = flash_born_attention_paged_fp4(q, cache, table, n, 1.0, cu, 0.0)
    o, _ = ref.attend(q, cache, table, n, 1.0, cu, 0.0)
    assert torch.allclose(out.double(), o[0], atol=1e-5)
    table.fill_(-1)
    assert not flash_born_attention_paged_fp4(q, cache, table, n, 1.0, cu, 0.0).any()
    none = tuple(t[:0] for t in cache)
    assert not flash_born_attention_paged_fp4(q[:2], none, table, n, 1.0).any()


def test_tokens_that_are_no_numbers_reach_those_that_see_them_alone():
    D, page = 64, 4
    cache = born_cache_fp4(4, page, 1, D, device="cpu")
    table, n, cu = torch.tensor([[0, 1, 2]], **INT), torch.tensor([9], **INT), torch.tensor([0, 9], **INT)
    g = torch.Generator().manual_seed(7)
    k, v = (torch.rand(9, 1, D, generator=g) for _ in range(2))
    k[3, 0, 5], v[6, 0, 40] = math.nan, math.inf
    q = fused_qk_rope_l2_normalize_append_fp4(torch.rand(9, 1, D, generator=g), k, v, None, None, cache, table, n, cu)
    assert int((cache.k_scale == 255).sum()) == 2 and int((cache.v_scale == 255).sum()) == 1
    out = flash_born_attention_paged_fp4(q, cache, table, n, 1.0, cu, window_size=2)
    assert out.isnan().all(-1).view(-1).tolist() == [i in (3, 4, 6, 7) for i in range(9)]
    assert out[[0, 1, 2, 5, 8]].isfinite().all()


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("budget,recent", [(4, 0), (4, 2), (0, 0), (20, 3)])
def test_evict_keeps_what_the_wide_cache_keeps(budget, recent, inplace):
    lens, page, Hkv, D = [9, 3, 0, 12], 3, 2, 40
    room = 4 * max(1, -(-budget // page))
    cache, table, n, free = ref.make_cache(lens, page, Hkv, D, spare=room)
    w = torch.randint(0, 3, (4, Hkv, 10), generator=torch.Generator().manual_seed(6)).float()
    to = None if inplace else free[:room].view(4, -1).to(torch.int32)
    kc, vc = ref.value(cache[0], cache[2]), ref.value(cache[1], cache[3])
    got = born_cache_evict_fp4(cache, table, n, w, budget, recent, to)
    want = born_cache_evict(kc, vc, table, n, w, budget, recent, to)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(ref.value(cache[0], cache[2]), kc) and torch.equal(ref.value(cache[1], cache[3]), vc)


def test_refusals():
    cache, table, n, _ = ref.make_cache([5, 5], 4, 2, 64)
    q, k = torch.rand(2, 4, 64), torch.rand(2, 2, 64)
    w = torch.rand(2, 2, 8)
    cu = torch.tensor([0, 1, 2], **INT)

    def append(**over):
        a = dict(q=q, k=k, v=k, cos=None, sin=None, cache=cache, block_table=table, cache_lens=n)
        fused_qk_rope_l2_normalize_append_fp4(**(a | over))

    def attend(**over):
        a = dict(q=q, cache=cache, block_table=table, cache_lens=n, scale=1.0)
        flash_born_attention_paged_fp4(**(a | over))

    def evict(**over):
        a = dict(cache=cache, block_table=table, cache_lens=n, key_weight=w, budget=3)
        born_cache_evict_fp4(**(a | over))

    def read(**over):
        a = dict(cache=cache, block_table=table, cache_lens=n, cu_seqlens=cu, total=2)
        born_cache_read_fp4(**(a | over))

    other = [cache[:3], (*cache[:3], cache[3][:, :2]), (*cache[:2], cache[2][..., :1], cache[3][..., :1]),
             tuple(t.int() for t in cache), tuple(t[0] for t in cache)]
    for call in (append, attend, evict, read):
        for c in other:
            with pytest.raises(ValueError):
                call(cache=c)
        for bad in (dict(block_table=table[:1]), dict(block_table=table.float()), dict(block_table=table[0]), dict(cache_lens=n[:1]),
                    dict(cache_lens=n.float()), dict(block_table=torch.zeros(2, 1, **INT).expand(2, (1 << 28) + 1))):
            with pytest.raises(ValueError):
                call(**bad)
    for bad in (dict(q=q[..., :32], k=k[..., :32], v=k[..., :32]), dict(q=q[:, :3]), dict(k=k[:1]), dict(v=k[..., :32]), dict(k=k[:, :1], v=k[:, :1]),
                dict(q=torch.rand(3, 4, 64), k=torch.rand(3, 2, 64), v=torch.rand(3, 2, 64)), dict(cu_seqlens=cu[:2]), dict(cu_seqlens=cu.float()),
                dict(positions=cu), dict(cos=torch.rand(4, 32)), dict(eps=-1.0), dict(eps=math.nan),
                dict(cos=torch.rand(4, 32), sin=torch.rand(5, 32)), dict(cache=(cache[0], cache[0], cache[2], cache[3])),
                dict(cache=(cache[0][:, :1].expand(-1, 4, -1, -1), *cache[1:]))):
        with pytest.raises(ValueError):
            append(**bad)
    for bad in (dict(q=q[0]), dict(q=q[..., :32]), dict(q=q[:, :3]), dict(q=q[:1]), dict(scale=torch.rand(3)), dict(eps=-1.0),
                dict(key_weight=w[:1]), dict(key_weight=w.double()), dict(key_weight=torch.zeros(2, 2, 1).expand(2, 2, 8)), dict(cu_seqlens=cu[:2])):
        with pytest.raises(ValueError):
            attend(**bad)
    with pytest.raises(NotImplementedError):
        attend(key_weight=w, cu_seqlens=cu)
    for bad in (dict(budget=-1), dict(recent=-1), dict(key_weight=w[:, :1]), dict(out_block_table=table[:1]), dict(out_block_table=table),
                dict(budget=8, out_block_table=table[:, :1].clone())):
        with pytest.raises(ValueError):
            evict(**bad)
    for bad in (dict(total=-1), dict(head_dim=32), dict(head_dim=65), dict(cu_seqlens=cu[:2]), dict(dtype=torch.int32)):
        with pytest.raises(ValueError):
            read(**bad)


def test_derivatives_are_refused():
    cache, table, n, _ = ref.make_cache([5, 5], 4, 2, 64)
    q, k = torch.rand(2, 4, 64, requires_grad=True), torch.rand(2, 2, 64, requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward"):
        flash_born_attention_paged_fp4(q, cache, table, n, 1.0)
    with pytest.raises(RuntimeError, match="no backward"):
        fused_qk_rope_l2_normalize_append_fp4(q.detach(), k, k.detach(), None, None, cache, table, n)
    with pytest.raises(RuntimeError, match="no backward"):
        born_cache_evict_fp4(cache, table, n, torch.rand(2, 2, 8, requires_grad=True), 3)
    with torch.no_grad():
        flash_born_attention_paged_fp4(q, cache, table, n, 1.0)
        versions = [t._version for t in cache]
        fused_qk_rope_l2_normalize_append_fp4(q, k, k, None, None, cache, table, n)
    assert all(t._version > x for t, x in zip(cache, versions))


def test_compiled_callers_break_the_graph():
    cache, table, n, _ = ref.make_cache([5, 5], 4, 2, 64)
    q = torch.rand(2, 4, 64)
    f = torch.compile(lambda x: flash_born_attention_paged_fp4(2 * x, cache, table, n, 1.0) + 1, backend="eager")
    assert torch.equal(f(q), flash_born_attention_paged_fp4(2 * q, cache, table, n, 1.0) + 1)


# ---------------------------------------------------------------------------
# The C ABI: every call below is rejected before any HIP call, or has nothing to do.
# ---------------------------------------------------------------------------
P = 64  # a dummy address

FIELDS = dict(k=P, v=P, ks=P, vs=P, kst=(512, 32, 512), vst=(512, 32, 512), kss=(32, 2, 32), vss=(32, 2, 32), cache_pages=9, page=16,
              table=P, pages=4, ld=4, lens=P)


def _cache_fields(a):
    return (a["k"], a["v"], a["ks"], a["vs"], *a["kst"], *a["vst"], *a["kss"], *a["vss"], a["cache_pages"], a["page"], a["table"],
            a["pages"], a["ld"], a["lens"])


def _block(name, **over):
    a = dict(FIELDS, dtype=2, n=2, B=2, H=4, Hkv=2, D=64, q=P, qs=(256, 64), kv=P, kvs=(128, 64), out=P, cu=0, scale=0, n_scale=1, window=0,
             eps=1e-12, weight=0, w_len=0, ws=P, ws_bytes=1 << 40, cos=0, rows=0, freqs=0, freq_ld=0, budget=3, recent=0, to=0, to_pages=0,
             to_ld=0, lens_out=2 * P, kept=P, weight_out=0)
    a.update(over)
    c = _cache_fields(a)
    if name == "append":
        return _native.fp4_append_call(a["dtype"], a["n"], a["B"], a["H"], a["Hkv"], a["D"], a["q"], a["kv"], a["kv"], *a["qs"], *a["kvs"],
                                       *a["kvs"], a["out"], *c, a["cu"], a["cos"], a["cos"], a["rows"], a["freqs"], a["freq_ld"], 0, a["eps"])
    if name == "read":
        return _native.fp4_read_call(a["dtype"], a["n"], a["B"], a["Hkv"], a["D"], a["out"], a["out"], *c, a["cu"])
    if name == "paged":
        return _native.fp4_paged_call(a["dtype"], a["n"], a["B"], a["H"], a["Hkv"], a["D"], a["q"], *a["qs"], a["out"], *c, a["cu"], a["scale"],
                                      a["n_scale"], 1.0, a["window"], a["eps"], a["weight"], 0, 0, a["w_len"], a["ws"], a["ws_bytes"])
    return _native.fp4_evict_call(a["B"], a["Hkv"], a["D"], *c, a["weight"], 0, 0, a["w_len"], a["budget"], a["recent"], a["to"], a["to_pages"],
                                  a["to_ld"], a["weight_out"], a["lens_out"], a["kept"])


def test_argument_blocks_are_checked():
    lib = _native.load()
    calls = {n: getattr(lib, f"qdl_flash_born_fp4_{n}{'_forward' if n == 'paged' else ''}_call") for n in ("append", "read", "paged", "evict")}

    def rc(name, **over):
        return calls[name](_block(name, **over), None)

    far = (1 << 63) - 1
    for name, call in calls.items():
        assert call(None, None) == -5
        assert call(b"\0" * 8 + _block(name)[8:], None) == -2
        assert rc(name, D=12) == -3 and rc(name, D=264) == -3 and rc(name, Hkv=0) == -13
        assert rc(name, B=-1) == -2
        assert rc(name, kst=(512, 24, 512)) == -14 and rc(name, vst=(-16, 32, 512)) == -14 and rc(name, kss=(-1, 2, 32)) == -14
        assert rc(name, page=0) == -15 and rc(name, pages=5) == -15 and rc(name, cache_pages=-1) == -15
        for pages, page in ((1 << 40, 1 << 24), (1 << 62, 4), (far, 2), ((1 << 30) + 1, 1)):
            assert rc(name, pages=pages, page=page, ld=far) == -15
        assert rc(name, k=0) == -5 and rc(name, vs=0) == -5 and rc(name, table=0) == -5 and rc(name, lens=0) == -5
        assert rc(name, k=P + 8) == -4
    for name in ("append", "read", "paged"):
        assert rc(name, dtype=7) == -1
        assert rc(name, n=-1) == -2 and rc(name, n=0, B=0, cu=P) == 0
        assert rc(name, out=0, cu=P) == -5 and rc(name, out=P + 4, cu=P) == -4
    for name in ("append", "paged"):
        assert rc(name, H=3) == -13 and rc(name, n=3) == -2 and rc(name, eps=-1.0) == -2 and rc(name, eps=math.nan) == -2
        assert rc(name, qs=(256, 60)) == -14 and rc(name, q=0) == -5
    assert rc("append", cos=P, rows=0) == -10 and rc("append", cos=P, rows=4, freqs=33, freq_ld=33) == -10
    assert rc("read", cu=0) == -5
    assert rc("paged", scale=P, n_scale=3) == -6 and rc("paged", window=-1) == -7 and rc("paged", ws=0) == -8 and rc("paged", ws_bytes=8) == -8
    assert rc("paged", weight=P, cu=P) == -2 and rc("paged", n=1 << 28, H=256, B=1, cu=P, qs=(1 << 14, 64)) == -2
    assert rc("paged", n=500, B=0, cu=P) == -2  # tokens of no sequence
    assert rc("evict", budget=-1) == -16 and rc("evict", lens_out=P) == -2 and rc("evict", to=P) == -15 and rc("evict", kept=0) == -5
    assert rc("evict", weight=P, w_len=4, weight_out=P) == -2 and rc("evict", to=2 * P, to_pages=3, to_ld=2) == -15
    assert lib.qdl_flash_born_fp4_paged_workspace_size(2, 2, 4, 2, 64, 1 << 40, 1 << 24, 0, 0, 1) == 0


SHARES = r"""
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>
#include "%s"
using namespace qdl;
int main() {
    std::mt19937_64 g(1);
    auto upto = [&](int64_t most) { return (int64_t)(g() %% (uint64_t)(most + 1)); };
    auto log_upto = [&](int bits) { return upto((int64_t)1 << upto(bits)); };
    for (int round = 0; round < 200000; ++round) {
        const int64_t B = 1 + upto(round %% 50 == 0 ? 3000 : 20), h_kv = 1 + upto(8), G = 1 + log_upto(6), H = h_kv * G, D = 64;
        const int64_t page = 1 + log_upto(8), pages = log_upto(round %% 7 ? 10 : 22), room = pages * page;
        const int64_t window = upto(2) ? 0 : 1 + log_upto(12);
        const bool packed = upto(3) != 0, weighed = !packed && upto(1);
        std::vector<int64_t> nq(B, 1), n(B);
        int64_t N = 0;
        for (int64_t b = 0; b < B; ++b) {
            if (packed) nq[b] = upto(3) ? upto(8) : log_upto(10);
            N += nq[b];
            n[b] = upto(3) ? std::min(room, log_upto(30)) : room;
        }
        if (packed) N += upto(2);
        if (!N || room > (int64_t)1 << 30) continue;
        const Fp4Plan r = fp4_plan(N, B, H, h_kv, D, pages, page, window, packed, weighed, (1 << 24) - 1);
        uint64_t total = 0;
        int64_t wide = 0, units = 0, cols = 16 * r.nc;
        auto is_wide = [&](int64_t b) { return packed && nq[b] * G > r.limit; };
        auto steps = [&](int64_t b) { return fp4_steps((int)n[b], fp4_first((int)n[b], (int)nq[b], (int)window)); };
        auto columns = [&](int64_t b) { return is_wide(b) ? 0 : fp4_blocks(nq[b] * G, (int)cols); };
        for (int64_t b = 0; b < B; ++b) {
            total += (uint64_t)steps(b) * columns(b);
            if (is_wide(b)) wide += (nq[b] * G + kFp4Rows - 1) / kFp4Rows;
            if (columns(b) > r.cblocks || (!is_wide(b) && nq[b] * G > r.most)) return printf("rows %%d\n", round), 1;
            const int64_t base = fp4_first((int)n[b], (int)nq[b], (int)window) & ~31;
            if (weighed && (n[b] - base + 31) / 32 * 32 > r.raw_ld) return printf("raw %%d\n", round), 1;
        }
        if (wide && !r.slots) return printf("no slots %%d\n", round), 1;
        if (r.items > 0) {
            const int64_t step = fp4_step(total, r.items);
            if (step < 1 || step > 1 << 23) return printf("step %%d\n", round), 1;
            for (int64_t b = 0; b < B; ++b) units += (steps(b) + step - 1) / step * columns(b);
            if (wide > r.slots) return printf("slots %%d\n", round), 1;
        } else {
            units = B * r.cblocks;
            if (r.slots && r.slots < N * G / kFp4Rows + B + 1) return printf("slots by starts %%d\n", round), 1;
        }
        if (units > r.units) return printf("units %%d: %%ld of %%ld\n", round, (long)units, (long)r.units), 1;
        const int64_t parts = r.items > 0 || weighed ? r.units * h_kv * cols * (D + 4) * 4 : 0;
        if (r.part_bytes != parts || r.grid != (r.units + r.slots * r.splits) * h_kv) return 1;
        if (r.fits && r.items > 0 && r.join.narrow != (r.slots ? B * h_kv * r.most : 0)) return 1;
        if (r.fits && r.join.rows != ((r.slots ? r.splits > 1 : r.items > 0) ? N * H : 0)) return 1;
    }
    return 0;
}
"""


def test_what_the_device_shares_out_fits_what_the_host_made_room_for(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no host compiler")
    header = os.path.join(os.path.dirname(born_fp4.__file__), "..", "csrc", "fp4_plan.h")
    (tmp_path / "shares.cpp").write_text(SHARES % os.path.abspath(header))
    subprocess.run([gxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", str(tmp_path / "shares.cpp"), "-o",
                    str(tmp_path / "shares")], check=True)
    got = subprocess.run([str(tmp_path / "shares")], capture_output=True, text=True)
    assert got.returncode == 0, got.stdout + got.stderr

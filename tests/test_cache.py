"""The paged cache on the CPU: attention of one token, appending, evicting, their
refusals, missing pages, and the C ABI's checks of the argument blocks."""

from __future__ import annotations

import pytest
import torch

import serve_ref as ref
from quantumdlblocks_amd import (
    _native,
    born_cache_evict,
    flash_born_attention_packed,
    flash_born_attention_paged,
    fused_qk_rope_l2_normalize_append,
)


def make_cache(lens, page, Hkv, D, dtype=torch.float32, seed=0, extra=4, spare=0, device="cpu"):
    """Caches whose pages lie in any order; tables padded with -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra + spare
    order = torch.randperm(total, generator=g)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n].to(torch.int32)
        at += n
    kc, vc = (torch.randn(total, page, Hkv, D, generator=g).to(dtype) for _ in range(2))
    return (kc.to(device), vc.to(device), table.to(device), torch.tensor(lens, dtype=torch.int32, device=device),
            order[at:].to(device))


@pytest.mark.parametrize("page", [1, 4, 5])
@pytest.mark.parametrize("window", [0, 3])
def test_attention_of_one_token(page, window):
    lens = [7, 0, 1, 12]
    kc, vc, table, n, _ = make_cache(lens, page, 2, 8)
    q = torch.randn(4, 4, 8, generator=torch.Generator().manual_seed(3))
    weight = torch.ones(4, 2, 12)
    out = flash_born_attention_paged(q, kc, vc, table, n, torch.tensor([1.0, 2.0, -0.5, 3.0]), 0.01, window, weight)
    o, w = ref.paged(q, kc, vc, table, n, torch.tensor([1.0, 2.0, -0.5, 3.0]), 0.01, window)
    assert torch.allclose(out.double(), o[0], atol=1e-5)
    m = min(12, w[0].shape[2])
    assert torch.allclose(weight[..., :m].double() - 1.0, w[0][..., :m], atol=1e-5)
    assert not out[1].any()


def test_missing_pages_and_lengths_past_the_table():
    kc, vc, table, n, _ = make_cache([10, 10], 4, 1, 8)
    table[0, 1] = -1
    table[1, 2] = 1000
    n[0] = 99
    q = torch.randn(2, 2, 8)
    out = flash_born_attention_paged(q, kc, vc, table, n, 1.0, 0.0)
    o, _ = ref.paged(q, kc, vc, table, n, 1.0, 0.0)
    assert torch.allclose(out.double(), o[0], atol=1e-5)
    table.fill_(-1)
    assert not flash_born_attention_paged(q, kc, vc, table, n, 1.0, 0.0).any()


def test_append_writes_slots_and_leaves_the_rest():
    page, Hkv, D = 4, 2, 8
    kc, vc, table, n, _ = make_cache([7, 3, 9], page, Hkv, D)
    new = [2, 0, 5]
    cu = torch.tensor(ref.starts(new))
    N = sum(new) + 1  # one token behind the last sequence
    g = torch.Generator().manual_seed(4)
    q = torch.randn(N, 4, D, generator=g)
    k, v = (torch.randn(N, Hkv, D, generator=g) for _ in range(2))
    ang = torch.rand(20, 3, generator=g)
    pos = torch.tensor([5, 6, 30, 4, 5, 6, 7, 0])  # 30: past the tables
    k0, v0 = kc.clone(), vc.clone()
    out = fused_qk_rope_l2_normalize_append(q, k, v, ang.cos(), ang.sin(), kc, vc, table, n, cu, pos, eps=1e-6)

    def turned(x, p):
        c, s = torch.ones(4), torch.zeros(4)
        c[:3], s[:3] = ang[min(p, 19)].cos(), ang[min(p, 19)].sin()
        y = torch.cat([x[..., :4] * c - x[..., 4:] * s, x[..., :4] * s + x[..., 4:] * c], -1)
        return y / (y.square().sum(-1, keepdim=True) + 1e-6).sqrt()

    t = 0
    for b, x in enumerate(new):
        for i in range(x):
            slot = int(n[b]) - x + i
            pg, r = int(table[b, slot // page]), slot % page
            k0[pg, r], v0[pg, r] = turned(k[t], int(pos[t])), v[t]
            assert torch.allclose(out[t], turned(q[t], int(pos[t])), atol=1e-6)
            t += 1
    assert torch.allclose(kc, k0, atol=1e-6) and torch.equal(vc, v0)
    assert not out[t:].any()


def test_append_of_missing_slots_writes_nothing():
    kc, vc, table, n, _ = make_cache([5, 5], 4, 1, 8)
    table[0, 1] = -1
    n[1] = 50
    k0, v0 = kc.clone(), vc.clone()
    out = fused_qk_rope_l2_normalize_append(torch.randn(2, 1, 8), torch.randn(2, 1, 8), torch.randn(2, 1, 8), None, None, kc, vc,
                                            table, n)
    assert torch.equal(kc, k0) and torch.equal(vc, v0) and torch.allclose(out.norm(dim=-1), torch.ones(2, 1))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("budget,recent", [(4, 0), (4, 2), (4, 9), (0, 0), (20, 3)])
def test_evict(budget, recent, inplace):
    lens, page, Hkv = [9, 3, 0, 12], 3, 2
    kc, vc, table, n, free = make_cache(lens, page, Hkv, 8, spare=4 * max(1, -(-budget // page)))
    g = torch.Generator().manual_seed(6)
    w = torch.randint(0, 3, (4, Hkv, 10), generator=g).float()
    w[0, 0, 2] = float("nan")
    to = free[: 4 * max(1, -(-budget // page))].view(4, -1).to(torch.int32)
    k0, v0 = kc.clone(), vc.clone()
    new, weight, kept = born_cache_evict(kc, vc, table, n, w, budget, recent, None if inplace else to)
    dst = table if inplace else to
    for b, x in enumerate(lens):
        m = min(x, budget)
        assert int(new[b]) == m
        for h in range(Hkv):
            full = [float(w[b, h, j]) if j < 10 else 0.0 for j in range(x)]
            want = ref.evict(full, x, budget, recent)
            assert kept[b, h].tolist() == want + [-1] * (budget - m)
            for i, j in enumerate(want):
                a, d = (int(table[b, j // page]), j % page), (int(dst[b, i // page]), i % page)
                assert torch.equal(kc[d[0], d[1], h], k0[a[0], a[1], h]) and torch.equal(vc[d[0], d[1], h], v0[a[0], a[1], h])
                if i < 10:
                    assert full[j] == float(weight[b, h, i]) or full[j] != full[j]
            assert not weight[b, h, m:].any()


def test_prompt_then_tokens_then_eviction():
    """The operators as a server runs them: the packed prompt, its keys into the
    cache, tokens one by one with their weight kept, an eviction, more tokens."""
    lens, page, H, Hkv, D = [5, 9], 4, 4, 2, 8
    g = torch.Generator().manual_seed(8)
    cap = 16
    kc, vc, table, n, _ = make_cache([cap, cap], page, Hkv, D)
    tokens = [torch.randn(x + 3, H + 2 * Hkv, D, generator=g) for x in lens]
    pre = torch.cat([t[:x] for t, x in zip(tokens, lens)])
    cu = torch.tensor(ref.starts(lens))
    n.copy_(torch.tensor(lens))
    q = fused_qk_rope_l2_normalize_append(pre[:, :H], pre[:, H : H + Hkv], pre[:, H + Hkv :], None, None, kc, vc, table, n, cu)
    k = torch.cat([ref.gather(kc, table[b], x, page)[0] for b, x in enumerate(lens)])
    v = torch.cat([ref.gather(vc, table[b], x, page)[0] for b, x in enumerate(lens)])
    out = flash_born_attention_packed(q, k, v, 2.0, cu)
    last = flash_born_attention_paged(q[cu[1:] - 1], kc, vc, table, n, 2.0)
    assert torch.allclose(out[cu[1:] - 1], last, atol=1e-5)  # a prompt's last row is its token's
    weight, want = torch.zeros(2, Hkv, cap), torch.zeros(2, Hkv, cap, dtype=torch.float64)
    for i in range(3):
        n += 1
        x = torch.stack([t[l + i] for t, l in zip(tokens, lens)])
        q = fused_qk_rope_l2_normalize_append(x[:, :H], x[:, H : H + Hkv], x[:, H + Hkv :], None, None, kc, vc, table, n)
        flash_born_attention_paged(q, kc, vc, table, n, 2.0, key_weight=weight)
        want += ref.paged(q, kc, vc, table, n, 2.0)[1][0]
    assert torch.allclose(weight.double(), want, atol=1e-5)
    n2, weight, kept = born_cache_evict(kc, vc, table, n, weight, 6, 2)
    assert n2.tolist() == [6, 6] and (kept[:, :, -2:] == torch.stack([n - 2, n - 1], -1).view(2, 1, 2)).all()
    assert flash_born_attention_paged(q, kc, vc, table, n2, 2.0).isfinite().all()


def test_refusals():
    kc, vc, table, n, free = make_cache([5, 6], 4, 2, 8, spare=4)
    q, k, v = torch.randn(2, 4, 8), torch.randn(2, 2, 8), torch.randn(2, 2, 8)
    w = torch.zeros(2, 2, 8)
    to = free[:4].view(2, 2).to(torch.int32)
    att = flash_born_attention_paged
    app = fused_qk_rope_l2_normalize_append
    for bad in (
        lambda: att(q.view(2, 2, 2, 8), kc, vc, table, n, 1.0),
        lambda: att(q[:, :3], kc, vc, table, n, 1.0),
        lambda: att(q[..., :4], kc, vc, table, n, 1.0),
        lambda: att(q, kc, vc[:2], table, n, 1.0),
        lambda: att(q, kc, vc.double(), table, n, 1.0),
        lambda: att(q, kc, vc, table[:1], n, 1.0),
        lambda: att(q, kc, vc, table.float(), n, 1.0),
        lambda: att(q, kc, vc, table, n[:1], 1.0),
        lambda: att(q, kc, vc, table, n, torch.ones(3)),
        lambda: att(q, kc, vc, table, n, 1.0, eps=-1.0),
        lambda: att(q, kc, vc, table, n, 1.0, key_weight=w[:, :1]),
        lambda: att(q, kc, vc, table, n, 1.0, key_weight=w.double()),
        lambda: att(q, kc, vc, table, n, 1.0, key_weight=w[:1].expand(2, 2, 8)),
        lambda: app(q, k[:1], v, None, None, kc, vc, table, n),
        lambda: app(q[:1], k[:1], v[:1], None, None, kc, vc, table, n),
        lambda: app(q, k, v, torch.ones(4, 4), None, kc, vc, table, n),
        lambda: app(q, k, v, torch.ones(2, 4, 4), torch.ones(2, 4, 4), kc, vc, table, n),
        lambda: app(q, k, v, torch.ones(4, 4), torch.ones(4, 3), kc, vc, table, n),
        lambda: app(q, k, v, None, None, kc, vc, table, n, cu_seqlens=torch.tensor([0, 2])),
        lambda: app(q, k, v, None, None, kc, vc, table, n, positions=torch.tensor([0])),
        lambda: app(q, k, v, None, None, kc[:1].expand(4, 4, 2, 8), vc[:1].expand(4, 4, 2, 8), table, n),
        lambda: born_cache_evict(kc, vc, table, n, w, -1),
        lambda: born_cache_evict(kc, vc, table, n, w, 4, -1),
        lambda: born_cache_evict(kc, vc, table, n, w[:, :1], 4),
        lambda: born_cache_evict(kc, vc, table, n, w, 8, 0, to[:, :1]),
        lambda: born_cache_evict(kc, vc, table, n, w, 4, 0, to[:1]),
        lambda: born_cache_evict(kc, vc, table, n, w, 4, 0, table),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        att(q.requires_grad_(), kc, vc, table, n, 1.0)
    with torch.no_grad():
        att(q, kc, vc, table, n, 1.0)


def _paged_block(**over):
    a = dict(dtype=2, B=2, H=4, h_kv=2, D=64, q=16, qs0=256, qs1=64, out=16, k=16, v=16, ks0=2048, ks1=128, ks2=64, vs0=2048, vs1=128,
             vs2=64, cache_pages=8, page=16, table=16, pages=4, ld=4, lens=16, scale=0, n_scale=1, value=1.0, window=0, eps=0.0,
             weight=0, w0=0, w1=0, w_len=0, ws=16, ws_bytes=1 << 24)
    a.update(over)
    return _native.paged_call(*a.values())


def _append_block(**over):
    a = dict(dtype=2, n=2, B=2, H=4, h_kv=2, D=64, q=16, k=16, v=16, qs0=256, qs1=64, ks0=128, ks1=64, vs0=128, vs1=64, q_out=16,
             kc=16, vc=16, c0=2048, c1=128, c2=64, d0=2048, d1=128, d2=64, cache_pages=8, page=16, table=16, pages=4, ld=4, lens=16,
             cu=0, cos=16, sin=16, rows=10, n_freq=32, freq_ld=32, positions=0, eps=0.0)
    a.update(over)
    return _native.append_call(*a.values())


def _evict_block(**over):
    a = dict(dtype=2, B=2, h_kv=2, D=64, kc=16, vc=16, c0=2048, c1=128, c2=64, d0=2048, d1=128, d2=64, cache_pages=8, page=16,
             table=16, pages=4, ld=4, lens=16, weight=16, w0=128, w1=64, w_len=64, budget=32, recent=4, to=0, to_pages=0, to_ld=0,
             weight_out=16, lens_out=16, kept=16)
    a.update(over)
    return _native.evict_call(*a.values())


_CACHE = [(dict(page=0), -15), (dict(ld=3), -15), (dict(pages=1 << 27, ld=1 << 27), -15), (dict(cache_pages=-1), -15),
          (dict(table=0), -5), (dict(lens=0), -5), (dict(D=20), -3), (dict(dtype=3), -1), (dict(h_kv=0), -13)]


@pytest.mark.parametrize("over,code", _CACHE + [
    (dict(q=0), -5), (dict(q=8), -4), (dict(k=8), -4), (dict(ks1=4), -14), (dict(qs0=-64), -14), (dict(H=5), -13), (dict(ws=0), -8),
    (dict(ws_bytes=64), -8), (dict(window=-1), -7), (dict(eps=-1.0), -2), (dict(scale=16, n_scale=2), -6), (dict(B=-1), -2),
])
def test_paged_block_checks(over, code):
    more = dict(weight=16, w_len=64)  # a workspace is needed
    assert _native.load().qdl_flash_born_paged_forward_call(_paged_block(**more, **over), None) == code


@pytest.mark.parametrize("over,code", _CACHE + [
    (dict(kc=8), -4), (dict(c1=4), -14), (dict(qs1=3), -14), (dict(n=3), -2), (dict(sin=0), -10), (dict(n_freq=33), -10),
    (dict(freq_ld=8), -10), (dict(rows=0), -10), (dict(q_out=0), -5), (dict(eps=-1.0), -2),
])
def test_append_block_checks(over, code):
    assert _native.load().qdl_flash_born_cache_append_call(_append_block(**over), None) == code


@pytest.mark.parametrize("over,code", _CACHE + [
    (dict(kc=8), -4), (dict(c1=4), -14), (dict(budget=-1), -16), (dict(recent=-1), -16), (dict(budget=1 << 31), -16),
    (dict(w_len=-1), -2), (dict(weight=0), -5), (dict(kept=0), -5), (dict(lens_out=0), -5), (dict(to=16, to_pages=4, to_ld=2), -15),
])
def test_evict_block_checks(over, code):
    assert _native.load().qdl_flash_born_cache_evict_call(_evict_block(**over), None) == code


def test_empty_calls_launch_nothing():
    lib = _native.load()
    assert lib.qdl_flash_born_paged_forward_call(_paged_block(B=0), None) == 0
    assert lib.qdl_flash_born_cache_append_call(_append_block(n=0, B=0), None) == 0
    assert lib.qdl_flash_born_cache_evict_call(_evict_block(B=0), None) == 0
    assert lib.qdl_flash_born_paged_workspace_size(0, 4, 2, 64, 4, 16, 0, 0) == 0
    assert lib.qdl_flash_born_paged_workspace_size(2, 4, 3, 64, 4, 16, 0, 0) == 0
    for call in (lib.qdl_flash_born_paged_forward_call, lib.qdl_flash_born_cache_append_call, lib.qdl_flash_born_cache_evict_call):
        assert call(None, None) == -5
        assert call(b"\x08" + bytes(511), None) == -2


def test_int64_indices_outside_32_bits_are_not_wrapped():
    # 2^32 is page 0 with its upper half cut off, 2^32 + 5 a length of 5.
    from quantumdlblocks_amd.kernels import born_cache, flash_born_packed

    table = torch.tensor([[1 << 32, 2, -(1 << 40), (1 << 62) + 1]])
    got, _ = born_cache._table(table)
    assert got.dtype is torch.int32 and got[0, 1] == 2
    assert all(not 0 <= got[0, i] < 1000 for i in (0, 2, 3))
    lens = born_cache._index(torch.tensor([(1 << 32) + 5, 7, -(1 << 33)]))
    assert lens[0] == 2 ** 31 - 1 and lens[1] == 7 and lens[2] < 0
    cu = flash_born_packed._starts(torch.tensor([0, 9, (1 << 32) + 1]), torch.device("cpu"))
    assert cu.tolist() == [0, 9, 2 ** 31 - 1]


def test_append_counts_the_groups_that_it_launches():
    # Five rows a token are two groups of four: 2^24 workgroups, where 5 / 4 of a group would pass.
    over = dict(n=1 << 28, B=1, cu=16, H=3, h_kv=1, D=128, qs0=384, qs1=128, ks0=128, ks1=128, vs0=128, vs1=128)
    assert _native.load().qdl_flash_born_cache_append_call(_append_block(**over), None) == -2


@pytest.mark.parametrize("over,code", [(dict(lens_out=32, lens=32), -2), (dict(weight_out=32, weight=32), -2),
                                       (dict(to=32, table=32, to_pages=4, to_ld=4), -15)])
def test_evict_refuses_outputs_that_are_its_inputs(over, code):
    # Other workgroups still read them.
    base = dict(lens_out=48, lens=64, weight_out=80, weight=96)
    assert _native.load().qdl_flash_born_cache_evict_call(_evict_block(**{**base, **over}), None) == code

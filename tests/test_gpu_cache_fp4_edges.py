"""The 4-bit paged cache on the GPU where it is easiest to get wrong: precision
whatever else is in the batch, values that are not numbers, exact ties, large
batches, wide tables, and memory behind the tensors."""

from __future__ import annotations

import math

import pytest
import torch

import fp4_ref as ref
import serve_ref
from quantumdlblocks_amd import (
    _native,
    born_cache_fp4,
    flash_born_attention_paged_fp4,
    fused_qk_rope_l2_normalize_append_fp4,
)
from quantumdlblocks_amd.kernels import born_fp4

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
INT = dict(dtype=torch.int32)


def _rows(cache, table, n, D):
    """fp4_ref.rows for long caches: every key at once."""
    kc, vc, ks, vs = (t.cpu() for t in cache)
    page, j = kc.shape[1], torch.arange(n)
    t = table[j // page].long()
    ok = (t >= 0) & (t < kc.shape[0])
    t, r = torch.where(ok, t, torch.zeros_like(t)), torch.where(ok, j % page, torch.zeros_like(j))
    bad = (ks[t, r] == 255).any(-1) | (vs[t, r] == 255).any(-1)
    return ref.value(kc[t, r], ks[t, r])[..., :D], ref.value(vc[t, r], vs[t, r])[..., :D], ok, bad


@pytest.fixture(autouse=True)
def _every_key_at_once(monkeypatch):
    monkeypatch.setattr(ref, "rows", _rows)


def _queries(N, H, D, dtype, seed):
    x = torch.randn(N, H, D, generator=torch.Generator().manual_seed(seed)) + 0.1
    return torch.nn.functional.normalize(x, dim=-1).to(dtype)


def _tight(q, cache, table, lens, scale, cu, eps=1e-12, window=0):
    """fp4_ref.attend a few tokens at a time: the bound of 32 rows or fewer."""
    G, outs = q.shape[1] // cache[0].shape[2], []
    for b in range(len(cu) - 1):
        new, few = cu[b + 1] - cu[b], max(1, 32 // G)
        for i in range(0, new, few):
            m = min(few, new - i)
            n = torch.tensor([int(lens[b]) - new + i + m])
            outs.append(ref.attend(q[cu[b] + i : cu[b] + i + m], cache, table[b : b + 1], n, scale, [0, m], eps, window)[0])
    return tuple(torch.cat(x) for x in zip(*outs))


# ---------------------------------------------------------------------------
# Precision
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_rows_precision_is_its_own(cuda_device, dtype, D):
    """The same bound whether a sequence has few new tokens or many, alone, beside
    others, or beside sequences without new tokens."""
    scale = torch.tensor([1.0, -2.0, 30.0, 0.1, 1.0, 2.0, 3.0, 4.0])
    for new in ([60], [60, 0, 0, 0], [60, 300], [1, 60, 9], [4, 5]):
        lens = [x + 200 + 10 * i for i, x in enumerate(new)]
        cache, table, n, _ = ref.make_cache(lens, 16, 2, D, seed=41)
        cu = serve_ref.starts(new)
        q = _queries(cu[-1], 8, D, DT[dtype], 42)
        out = flash_born_attention_paged_fp4(q.to(cuda_device), tuple(t.to(cuda_device) for t in cache), table.to(cuda_device), n.to(cuda_device),
                                             scale.to(cuda_device), torch.tensor(cu, device=cuda_device, **INT))
        assert ref.worst(out, _tight(q, cache, table, n, scale, cu)) <= 1.0


# ---------------------------------------------------------------------------
# Large batches
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("weigh", [False, True])
def test_sequences_of_several_column_blocks_each(cuda_device, weigh):
    """Forty heads over one key head: two or three blocks of columns a sequence,
    more of them than a grid's second dimension holds."""
    B, H, D = 33000, 40, 8
    cache, _, _, _ = ref.make_cache([16] * 64, 16, 1, D, seed=45, extra=0)
    table, n = (torch.arange(B, **INT) % 64).view(-1, 1), torch.arange(B, **INT) % 17
    q = _queries(B, H, D, torch.bfloat16, 46)
    dev = tuple(t.to(cuda_device) for t in cache)
    weight = torch.zeros(B, 1, 16, device=cuda_device) if weigh else None
    out = flash_born_attention_paged_fp4(q.to(cuda_device), dev, table.to(cuda_device), n.to(cuda_device), 2.0, key_weight=weight)
    # The first, the last, and those about the 65536th block.
    some = torch.tensor([*range(70), *range(32700, 32840), *range(B - 70, B)])
    o, w = ref.attend(q[some], cache, table[some], n[some], 2.0)
    assert ref.worst(out[some.to(cuda_device)], o) <= 1.0
    if weigh:
        assert ref.worst(weight[some.to(cuda_device)], (w[0], w[1] + 2.0 ** -24 * w[0])) <= 1.0


def test_many_long_sequences_share_the_keys(cuda_device):
    """More than two rounds of 64 sequences, with keys enough to be split."""
    g = torch.Generator().manual_seed(43)
    lens = [int(x) for x in torch.randint(150, 900, (200,), generator=g)]
    lens[7], lens[70], lens[199] = 6000, 0, 5000
    some = [int(x) for x in torch.randint(0, 6, (200,), generator=g)]
    wide = [90 if i in (3, 68, 199) else x for i, x in enumerate(some)]
    cache, table, n, _ = ref.make_cache(lens, 16, 1, 64, seed=43)
    dev = tuple(t.to(cuda_device) for t in cache)
    for new, window in ((None, 0), (None, 300), (some, 0), (wide, 0), (wide, 100)):
        cu = list(range(201)) if new is None else serve_ref.starts(new)
        q = _queries(cu[-1], 2, 64, torch.bfloat16, 44)
        weight = torch.zeros(200, 1, 6000, device=cuda_device) if new is None else None
        out = flash_born_attention_paged_fp4(q.to(cuda_device), dev, table.to(cuda_device), n.to(cuda_device), 2.0,
                                             None if new is None else torch.tensor(cu, device=cuda_device, **INT), 1e-12, window, weight)
        o, w = ref.attend(q, cache, table, n, 2.0, None if new is None else cu, 1e-12, window)
        assert ref.worst(out, o) <= 1.0
        if new is None:
            y, e = (t[..., :6000] for t in w)
            assert ref.worst(weight, (y, e + 2.0 ** -24 * y)) <= 1.0


# ---------------------------------------------------------------------------
# The keys' weights
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
def test_weights_of_few_keys_over_wide_tables(cuda_device, dtype):
    """Tables of 2^20 keys a sequence for 520 sequences of 8 key heads: neither the
    launch nor its workspace goes by them where the weights kept are few."""
    B, Hkv = 520, 8
    lens = [300 if i % 40 == 0 else i % 50 for i in range(B)]
    cache, table, n, _ = ref.make_cache(lens, 256, Hkv, 32, seed=47)
    wide = torch.full((B, 4096), -1, **INT)
    wide[:, : table.shape[1]] = table
    q = _queries(B, Hkv, 32, DT[dtype], 48)
    weight = torch.full((B, Hkv, 280), 0.25, device=cuda_device)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = flash_born_attention_paged_fp4(q.to(cuda_device), tuple(t.to(cuda_device) for t in cache), wide.to(cuda_device), n.to(cuda_device), 2.0,
                                         key_weight=weight)
    assert torch.cuda.max_memory_allocated() - before < 256 << 20
    o, w = ref.attend(q, cache, table, n, 2.0)
    y, e = (t[..., :280] for t in w)
    assert ref.worst(out, o) <= 1.0 and ref.worst(weight, (y + 0.25, e + 2.0 ** -24 * (y + 0.25))) <= 1.0


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("kept", [1, 50, 100, 700])
def test_weights_of_some_of_the_keys(cuda_device, window, kept):
    lens = [690, 33, 0, 100]
    for page in (16, 7):
        cache, table, n, _ = ref.make_cache(lens, page, 2, 64, seed=49)
        q = _queries(4, 8, 64, torch.float16, 50)
        room = torch.full((4, 2, kept + 40), 0.25, device=cuda_device)  # rows with others' values behind them
        flash_born_attention_paged_fp4(q.to(cuda_device), tuple(t.to(cuda_device) for t in cache), table.to(cuda_device), n.to(cuda_device), 2.0,
                                       window_size=window, key_weight=room[..., :kept])
        y, e = ref.attend(q, cache, table, n, 2.0, None, 1e-12, window)[1]
        m = min(kept, y.shape[2])
        assert ref.worst(room[..., :m], (y[..., :m] + 0.25, e[..., :m] + 2.0 ** -24 * (y[..., :m] + 0.25))) <= 1.0
        assert (room[..., m:] == 0.25).all()


def test_keys_that_are_not_seen_keep_their_weights(cuda_device):
    """A row that is not a number makes NaN of the weights that it sees, of no other."""
    for dt in DT.values():
        for page, window in ((16, 0), (16, 30), (5, 0), (5, 30)):
            cache, table, n, _ = ref.make_cache([90, 60], page, 2, 64, seed=51)
            table[0, 40 // page] = -1
            table[0, 70 // page] = cache[0].shape[0] + 2
            t, r = int(table[0, 85 // page]), 85 % page
            cache[2][t, r, 1, 0] = 255
            q = _queries(2, 4, 64, dt, 52)
            q[1, 0, 7] = math.nan
            weight = torch.full((2, 2, 120), 0.5, device=cuda_device)
            flash_born_attention_paged_fp4(q.to(cuda_device), tuple(x.to(cuda_device) for x in cache), table.to(cuda_device), n.to(cuda_device),
                                           1.0, window_size=window, key_weight=weight)
            j = torch.arange(120)
            for b, h in ((0, 1), (1, 0)):  # the bad key's head, the bad query's
                m = int(n[b])
                at = torch.div(j, page, rounding_mode="floor").clamp(max=table.shape[1] - 1)
                seen = (j < m) & (j >= (m - window if window else 0)) & (table[b][at] >= 0) & (table[b][at] < cache[0].shape[0])
                assert torch.equal(weight[b, h].cpu().isnan(), seen)
                assert (weight[b, h].cpu()[~seen] == 0.5).all()
            assert weight[0, 0].isfinite().all() and weight[1, 1].isfinite().all()


def test_weights_of_heads_without_a_scale(cuda_device):
    """0 times a key that is not a number is none either, for all that the row sees."""
    cache, table, n, _ = ref.make_cache([90, 60], 16, 2, 64, seed=61)
    cache[3][int(table[0, 2]), 7, 1, 1] = 255
    q = _queries(2, 4, 64, torch.bfloat16, 62)
    weight = torch.full((2, 2, 90), 0.5, device=cuda_device)
    out = flash_born_attention_paged_fp4(q.to(cuda_device), tuple(x.to(cuda_device) for x in cache), table.to(cuda_device), n.to(cuda_device),
                                         0.0, key_weight=weight)
    assert out[0, 2:].isnan().all() and not out[0, :2].any() and not out[1].any()
    assert weight[0, 1].isnan().all() and (weight[0, 0] == 0.5).all() and (weight[1] == 0.5).all()


# ---------------------------------------------------------------------------
# Ties
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_keys_that_lie_halfway_between_two_codes(cuda_device, dtype):
    """Keys of a whole norm whose normalised values are exact: a code that is one
    of two as near, or the block's exponent, goes by the quotient's last bit."""
    rows = []
    for norm in (49, 75, 77, 91, 93, 99, 103, 105, 107, 117):
        for t in (7, 6, 5, 3):  # eighths of the norm: 7 / 8 is the largest value of its exponent
            rest = (8 * norm) ** 2 - (t * norm) ** 2
            parts = []
            for _ in range(5):  # sums of squares, the largest first
                parts.append(math.isqrt(rest))
                rest -= parts[-1] ** 2
            if rest == 0 and max(parts) < t * norm:
                rows.append([t * norm / 8] + [x / 8 for x in parts] + [0.0, -0.0] + [0.0] * 8)
    k = torch.tensor(rows, dtype=torch.float64).to(DT[dtype]).view(-1, 1, 16)
    assert len(rows) > 10 and torch.equal(k.double().flatten().cpu(), torch.tensor(rows, dtype=torch.float64).flatten())
    N = k.shape[0]
    table, n = torch.arange(N, **INT).view(-1, 1), torch.ones(N, **INT)
    got = born_cache_fp4(N, 1, 1, 16, device=cuda_device)
    fused_qk_rope_l2_normalize_append_fp4(*(k.to(cuda_device) for _ in range(3)), None, None, got, table.to(cuda_device), n.to(cuda_device), eps=0.0)
    for i, row in enumerate(rows):
        norm = math.sqrt(sum(x * x for x in row))
        assert norm == int(norm)
        e, codes = ref.store_block([x / norm for x in row] + [0.0] * 16)
        c = got.k[i, 0, 0].tolist()
        assert int(got.k_scale[i, 0, 0, 0]) == e and [c[j // 2] >> 4 * (j % 2) & 15 for j in range(32)] == codes


# ---------------------------------------------------------------------------
# Queries that are infinite, or nearly so
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [[9, 3, 5], [200, 3, 100]])
def test_infinite_queries_follow_the_formula(cuda_device, dtype, D, new):
    """An overlap with an infinity is infinite, its weight too or, where it is
    negative, none; with a value of 0 it is not a number."""
    cache, table, n, _ = ref.make_cache([210, 40, 150], 16, 2, D, seed=53)
    kc = cache[0]
    # Column 4 of every key: of one sign, but for head 1's, where some are zeros.
    byte = kc[..., 2]
    byte[...] = (byte & 0xF0) | 0x0A
    byte[1::3, :, 1] &= 0xF0
    cu = serve_ref.starts(new)
    G, dt = 4, DT[dtype]
    for bad, scale in ((math.inf, 1.0), (-math.inf, 1.0), (math.inf, -1.0), (-math.inf, -2.0)):
        q = _queries(cu[-1], 2 * G, D, dt, 54)
        at = [(cu[b] + i, h) for b in range(3) for i, h in ((0, 1), (new[b] - 1, 6), (new[b] // 2, 0))]
        for i, h in at:
            q[i, h, 4] = bad
        out = flash_born_attention_paged_fp4(q.to(cuda_device), tuple(t.to(cuda_device) for t in cache), table.to(cuda_device),
                                             n.to(cuda_device), scale, torch.tensor(cu, device=cuda_device, **INT)).cpu()
        for i, h in at:
            b = max(x for x in range(3) if cu[x] <= i)
            m = int(n[b]) - cu[b + 1] + i + 1  # the keys that this token sees
            k, v, _, _ = _rows(cache, table[b], m, D)
            r = scale * (q[i, h].double() * k[:, h // G]).sum(-1)
            p = torch.where(r < 0, torch.zeros_like(r), r * r)
            want = ((p / (p.sum() + 1e-12)).unsqueeze(-1) * v[:, h // G]).sum(0)
            assert want.isnan().all() or not want.any()
            assert torch.equal(out[i, h].isnan(), want.isnan()) and not out[i, h].nan_to_num().any()
        fine = torch.ones(cu[-1], 2 * G, dtype=torch.bool)
        for i, h in at:
            fine[i, h] = False
        assert out[fine].isfinite().all()


def test_queries_as_large_as_they_get(cuda_device):
    """Past bf16's largest, over keys so small that the overlaps are ordinary."""
    for new in ([1, 1], [40, 70]):
        cache, table, n, _ = ref.make_cache([100, 80], 16, 2, 64, seed=55)
        cache[2].fill_(127 - 120)
        cu = serve_ref.starts(new)
        q = _queries(cu[-1], 8, 64, torch.float32, 56)
        big = torch.finfo(torch.float32).max
        q = q / q.abs().amax(-1, keepdim=True) * big
        q[:, :, 3], q[:, :, 5] = big, -big * (1 - 2.0 ** -20)
        out = flash_born_attention_paged_fp4(q.to(cuda_device), tuple(t.to(cuda_device) for t in cache), table.to(cuda_device), n.to(cuda_device),
                                             1.0, torch.tensor(cu, device=cuda_device, **INT))
        assert ref.worst(out, ref.attend(q, cache, table, n, 1.0, cu)[0]) <= 1.0


# ---------------------------------------------------------------------------
# Memory behind the tensors
# ---------------------------------------------------------------------------
def _guarded(dev, size):
    """size bytes with a pattern on both sides, and what is left of the pattern."""
    pad = 1 << 16
    room = torch.full((pad + size + pad,), 0xA5, dtype=torch.uint8, device=dev)
    return room[pad : pad + size], lambda: bool((room[:pad] == 0xA5).all() and (room[pad + size :] == 0xA5).all())


def _attend_guarded(q, cache, table, n, cu, window=0, weight=None):
    """The library's call with guards about its output and its workspace."""
    N, H, D = q.shape
    B, pages = table.shape
    page, Hkv = cache[0].shape[1:3]
    fields = born_fp4._check_fp4(cache, table, n, B, D, written=False)
    size = born_fp4._paged_workspace(N, B, H, Hkv, D, pages, page, window, cu is not None, 0 if weight is None else weight.shape[2])
    size = -(-size // 4) * 4
    out, out_ok = _guarded(q.device, q.numel() * q.element_size())
    ws, ws_ok = _guarded(q.device, size)
    w = (0, 0, 0, 0) if weight is None else (weight.data_ptr(), weight.stride(0), weight.stride(1), weight.shape[2])
    block = _native.fp4_paged_call(born_fp4._DTYPE_CODE[q.dtype], N, B, H, Hkv, D, q.data_ptr(), q.stride(0), q.stride(1), out.data_ptr(),
                                   *fields, table.data_ptr(), pages, table.stride(0), n.data_ptr(), 0 if cu is None else cu.data_ptr(), 0, 1, 1.0,
                                   window, 1e-12, *w, ws.data_ptr(), size)
    assert _native.load().qdl_flash_born_fp4_paged_forward_call(block, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert out_ok() and ws_ok()
    return out.view(q.dtype).view(N, H, D)


@pytest.mark.parametrize("B,room,N,H", [(100, 2000, 64, 16), (100, 100, 64, 16), (1100, 400, 96, 8), (6, 4000, 600, 8), (6, 100, 600, 8),
                                        (80, 3000, 700, 4), (3, 5000, 40, 4)])
def test_starts_of_any_order_write_nothing_else(cuda_device, B, room, N, H):
    cache, table, n, _ = ref.make_cache([room, room - 90], 16, 2, 64, seed=57, device=cuda_device)
    table, n = table.repeat(-(-B // 2), 1)[:B].contiguous(), n.repeat(-(-B // 2))[:B].contiguous()
    q = _queries(N, H, 64, torch.bfloat16, 58).to(cuda_device)
    even = torch.tensor([i * N // B for i in range(B + 1)], device=cuda_device, **INT)
    for window in (0, 70):
        want = _attend_guarded(q, cache, table, n, even, window)
        assert torch.equal(want, flash_born_attention_paged_fp4(q, cache, table, n, 1.0, even, window_size=window))
        for starts in (([0, N] * B)[:B] + [N], [0] + [N - i % 7 * 5 for i in range(B)], [N] * B + [0], ([-5, N + 9] * B)[:B] + [N],
                       [0] + [N // 2] * (B - 1) + [N // 3], [0, N] + [N // 3] * (B - 1)):
            _attend_guarded(q, cache, table, n, torch.tensor(starts, device=cuda_device, **INT), window)
        assert torch.equal(_attend_guarded(q, cache, table, n, even, window), want)


@pytest.mark.parametrize("lens,H,page", [([3000, 1, 700], 4, 16), ([3000, 1, 700], 40, 16), ([100] * 80, 2, 7), ([60000], 4, 64)])
def test_one_token_writes_nothing_else(cuda_device, lens, H, page):
    cache, table, n, _ = ref.make_cache(lens, page, 2, 64, seed=59, device=cuda_device)
    q = _queries(len(lens), H, 64, torch.float16, 60).to(cuda_device)
    for window in (0, 1, 333):
        for keys in (0, 1, 50, max(lens)):
            room, ok = _guarded(cuda_device, len(lens) * 2 * keys * 4)
            weight = room.view(torch.float32).view(len(lens), 2, keys) if keys else None
            _attend_guarded(q, cache, table, n, None, window, weight)
            assert ok()

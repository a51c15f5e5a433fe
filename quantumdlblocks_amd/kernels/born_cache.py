"""A paged key-value cache for Born attention: filling it, attending over it and
shrinking it.

``k_cache`` and ``v_cache`` are (pages, page_size, Hkv, D) tensors of one dtype,
in any strides with unit stride along D; ``block_table`` (B, P) int32 names the
pages of each of B sequences, in order, and ``cache_lens`` (B,) int32 how many
keys each of them holds.  Key j of sequence b is row ``j % page_size`` of page
``block_table[b, j // page_size]``.  Table entries outside the cache (-1, say)
are missing pages: their keys are not seen and nothing is written to them.

    fused_qk_rope_l2_normalize_append   a step's new tokens: rotate and normalise
                                        q and k, write k and v to their slots
    flash_born_attention_paged          one new token per sequence attends
    born_cache_evict                    keep the recent keys and the heaviest

No call copies anything to the host, so a decoding step can be captured into a
HIP graph; tables and lengths may change between replays.  CPU tensors run the
same formulas in torch operations.  None of these has a backward: they refuse
tensors that a gradient is recorded for.
"""

from __future__ import annotations

import torch

from .. import _native
from .flash_born import _DTYPE_CODE, MAX_HEAD_DIM, _parameter, _run_call

__all__ = ["born_cache_evict", "flash_born_attention_paged", "fused_qk_rope_l2_normalize_append"]

_LIMIT = 1 << 30


def _no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no backward: call it under torch.no_grad(), or with detached tensors")


def _check_cache(k_cache, v_cache, block_table, cache_lens, B, written: bool):
    """The caches' (page, token, head) strides."""
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError(f"k_cache and v_cache must share one (pages, page_size, key_heads, head_dim) shape and dtype, got "
                         f"{k_cache.dtype} {tuple(k_cache.shape)}, {v_cache.dtype} {tuple(v_cache.shape)}")
    P, page, Hkv, D = k_cache.shape
    if page < 1 or Hkv < 1 or D < 1:
        raise ValueError(f"page_size, key_heads and head_dim must be positive, got {tuple(k_cache.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"block_table must be (B={B}, pages) int32, got {block_table.dtype} {tuple(block_table.shape)}")
    if tuple(cache_lens.shape) != (B,) or cache_lens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cache_lens must be (B={B},) int32, got {cache_lens.dtype} {tuple(cache_lens.shape)}")
    if block_table.shape[1] * page > _LIMIT:
        raise ValueError(f"block_table holds {block_table.shape[1]} pages of {page}: more than 2^30 keys a sequence")
    for name, t in (("v_cache", v_cache), ("block_table", block_table), ("cache_lens", cache_lens)):
        if t.device != k_cache.device:
            raise ValueError(f"{name} must be on the caches' device {k_cache.device}, got {t.device}")
    strides = []
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if written and any(n > 1 and s == 0 for n, s in zip(c.shape, c.stride())):
            raise ValueError(f"{name} is written and must not overlap itself, got strides {c.stride()}")
        if k_cache.is_cuda:
            if D % 8 or D > MAX_HEAD_DIM or c.dtype not in _DTYPE_CODE:
                raise NotImplementedError(f"paged caches take fp32, fp16 or bf16 and head dims that are multiples of 8 up to "
                                          f"{MAX_HEAD_DIM}, got {c.dtype} and {D}")
            st = [s if n > 1 else 0 for n, s in zip(c.shape, c.stride())]
            if c.stride(3) != 1 or c.data_ptr() % 16 or any(s * c.element_size() % 16 for s in st[:3]):
                raise ValueError(f"{name} needs unit stride along head_dim, other strides that are multiples of 16 bytes "
                                 f"and a 16-byte aligned base, got strides {c.stride()}")
            strides += st[:3]
    return strides


def _index(t: torch.Tensor) -> torch.Tensor:
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t if t.numel() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _table_ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _table(t: torch.Tensor) -> torch.Tensor:
    t = _index(t)
    return t if t.shape[0] <= 1 or t.stride(0) >= t.shape[1] else t.contiguous()


def _heads(t: torch.Tensor, dtype: torch.dtype):
    """(n, heads, D) rows in ``dtype`` and their (row, head) strides."""
    if t.dtype != dtype:
        t = t.to(dtype)
    item = t.element_size()
    st = [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())]
    if t.stride(2) != 1 or t.data_ptr() % 16 or any(s * item % 16 or s < 0 for s in st[:2]):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        st = list(t.stride())
    return t, st[0], st[1]


def _slots(block_table, page, slots):
    """Pages and rows of slots (B, n) on the CPU path; page -1 where there is none."""
    width = block_table.shape[1]
    col = slots // page
    if width == 0:
        return torch.full_like(slots, -1), slots % page
    pages = block_table.long().gather(1, col.clamp(0, width - 1))
    return torch.where((slots >= 0) & (col < width), pages, torch.full_like(pages, -1)), slots % page


# ---------------------------------------------------------------------------
# One new token per sequence
# ---------------------------------------------------------------------------
def _eager_paged(q, k_cache, v_cache, block_table, cache_lens, scale_t, eps, window, key_weight):
    B, H, D = q.shape
    P, page, Hkv, _ = k_cache.shape
    G, L = H // Hkv, block_table.shape[1] * page
    wide = torch.float64 if k_cache.dtype == torch.float64 else torch.float32
    j = torch.arange(L, device=q.device).view(1, L).expand(B, L)
    pages, rows = _slots(block_table, page, j)
    n = cache_lens.long().clamp(0, L).view(B, 1)
    keep = (pages >= 0) & (pages < P) & (j < n)
    if window > 0:
        keep = keep & (j >= n - window)
    at = torch.where(keep, pages, torch.zeros_like(pages))
    mask = keep.view(B, L, 1, 1)
    if P == 0:
        k = v = torch.zeros((B, L, Hkv, D), dtype=wide, device=q.device)
    else:
        k, v = (torch.where(mask, c[at, rows].to(wide), torch.zeros((), dtype=wide, device=q.device)) for c in (k_cache, v_cache))
    s = scale_t.to(device=q.device, dtype=wide).reshape(-1).expand(H).view(1, Hkv, G, 1)
    r = torch.matmul(q.to(wide).view(B, Hkv, G, D), k.permute(0, 2, 3, 1))
    p = torch.relu(r * s).square() * keep.view(B, 1, 1, L)
    den = p.sum(-1, keepdim=True) + eps
    w = p / torch.where(den > 0, den, torch.ones_like(den))
    if key_weight is not None:
        m = min(L, key_weight.shape[2])
        key_weight[:, :, :m] += w.sum(2)[:, :, :m].to(key_weight.dtype)
    return torch.matmul(w, v.permute(0, 2, 1, 3)).reshape(B, H, D).to(k_cache.dtype)


def flash_born_attention_paged(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    scale: float | torch.Tensor,
    eps: float = 1e-12,
    window_size: int = 0,
    key_weight: torch.Tensor | None = None,
) -> torch.Tensor:
    """Born attention of one new token per sequence over the cache; returns
    (B, H, D) in the caches' dtype.

    ``q`` (B, H, D), H a multiple of the caches' Hkv.  The token is the last of
    its sequence's ``cache_lens`` keys (its own key is in the cache already) and
    sees all of them, or the last ``window_size``:

        p_j = max(0, scale_h q . k_j) ** 2,  out = sum_j p_j v_j / (sum_j p_j + eps)

    ``scale``: a float or a tensor of 1 or H values.  ``key_weight`` (B, Hkv, L)
    fp32: each visible key's weight p_j / (sum p + eps), summed over the heads
    that read it, is added in place at j < L: what ``born_cache_evict`` goes by.
    Lengths past the table's pages are cut to them; a sequence without visible
    keys gets zeros.
    """
    _no_grad("flash_born_attention_paged", q, k_cache, v_cache, scale, key_weight)
    if q.dim() != 3:
        raise ValueError(f"q must be (B, heads, head_dim), got shape {tuple(q.shape)}")
    B, H, D = q.shape
    strides = _check_cache(k_cache, v_cache, block_table, cache_lens, B, written=False)
    P, page, Hkv, Dk = k_cache.shape
    if Dk != D or H < 1 or H % Hkv:
        raise ValueError(f"q {tuple(q.shape)} does not fit caches of {Hkv} key heads of {Dk}")
    if q.device != k_cache.device:
        raise ValueError(f"q must be on the caches' device {k_cache.device}, got {q.device}")
    n_scale = scale.numel() if isinstance(scale, torch.Tensor) else 1
    if n_scale not in (1, H):
        raise ValueError(f"scale must hold 1 value or H={H} per-head values, got {n_scale}")
    if not float(eps) >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    window = min(max(int(window_size), 0), _LIMIT)
    w_ptr = w_sb = w_sh = w_len = 0
    if key_weight is not None:
        if (key_weight.dim() != 3 or tuple(key_weight.shape[:2]) != (B, Hkv) or key_weight.dtype != torch.float32
                or key_weight.device != k_cache.device or (key_weight.numel() and key_weight.shape[2] > 1 and key_weight.stride(2) != 1)
                or any(n > 1 and s == 0 for n, s in zip(key_weight.shape, key_weight.stride()))):
            raise ValueError(f"key_weight must be (B={B}, key_heads={Hkv}, keys) fp32 on {k_cache.device} with unit stride along "
                             f"the keys, got {key_weight.dtype} {tuple(key_weight.shape)} on {key_weight.device}, strides "
                             f"{key_weight.stride()}")
        w_ptr, w_sb, w_sh, w_len = key_weight.data_ptr(), key_weight.stride(0), key_weight.stride(1), key_weight.shape[2]
    if not q.is_cuda:
        scale_t = scale if isinstance(scale, torch.Tensor) else torch.tensor(float(scale), dtype=torch.float64)
        return _eager_paged(q.detach(), k_cache, v_cache, block_table, cache_lens, scale_t.detach(), float(eps), window, key_weight)
    lib = _native.load()
    dev = q.device
    # Kept alive here until the call: the block holds addresses.
    scale_flat, scale_p, n_scale, scale_value = _parameter(scale, dev)
    q_c, sb, sh = _heads(q.detach(), k_cache.dtype)
    table, lens = _table(block_table), _index(cache_lens)
    out = torch.empty((B, H, D), dtype=k_cache.dtype, device=dev)
    head = (_DTYPE_CODE[k_cache.dtype], B, H, Hkv, D, q_c.data_ptr(), sb, sh, out.data_ptr(), k_cache.data_ptr(),
            v_cache.data_ptr(), *strides, P, page, table.data_ptr(), table.shape[1], _table_ld(table), lens.data_ptr(),
            scale_p, n_scale, scale_value, window, float(eps), w_ptr, w_sb, w_sh, w_len)
    size = int(lib.qdl_flash_born_paged_workspace_size(_native.paged_call(*head, 0, 0)))
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _run_call(lib.qdl_flash_born_paged_forward_call, "qdl_flash_born_paged_forward_call", dev,
              _native.paged_call(*head, 0 if ws is None else ws.data_ptr(), size))
    return out


# ---------------------------------------------------------------------------
# New tokens
# ---------------------------------------------------------------------------
def _tables(cos, sin, half, device):
    """(rows, n) fp32 tables with n = min(width, half)."""
    out = []
    for t in (cos, sin):
        t = t.detach()
        while t.dim() > 2:
            if t.shape[0] != 1:
                raise ValueError(f"rotary tables must be (rows, n) or (1, 1, rows, n), got shape {tuple(t.shape)}")
            t = t[0]
        if t.dim() != 2 or t.shape[0] < 1:
            raise ValueError(f"rotary tables must be (rows, n) or (1, 1, rows, n), got shape {tuple(t.shape)}")
        out.append(t[:, :half])
    if out[0].shape != out[1].shape:
        raise ValueError(f"cos and sin differ in shape: {tuple(cos.shape)}, {tuple(sin.shape)}")
    out = [t.to(device=device, dtype=torch.float32) for t in out]
    n = out[0].shape[1]
    same = out[0].stride() == out[1].stride() and (n <= 1 or out[0].stride(1) == 1) and (
        out[0].shape[0] == 1 or out[0].stride(0) >= n)
    return out if same else [t.contiguous() for t in out]


def _eager_append(q, k, v, tables, k_cache, v_cache, block_table, cache_lens, cu, positions, eps):
    N, B = q.shape[0], cache_lens.shape[0]
    P, page = k_cache.shape[:2]
    dev = q.device
    t = torch.arange(N, device=dev)
    if cu is None:
        s, end = t, t + 1
        here = torch.ones_like(t, dtype=torch.bool)
    else:
        c = cu.long()
        s = (torch.searchsorted(c, t, right=True) - 1).clamp(0, max(B - 1, 0))
        end = c[(s + 1).clamp(max=B)]
        here = (t >= c[s]) & (t < end) if B else torch.zeros_like(t, dtype=torch.bool)
    slot = torch.full_like(t, -1)
    if B:
        slot = torch.where(here, cache_lens.long()[s] - (end - t), slot)
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    half = q.shape[2] // 2
    if tables is None:
        cos, sin = torch.ones((N, 1, half), dtype=wide, device=dev), torch.zeros((N, 1, half), dtype=wide, device=dev)
    else:
        at = (slot if positions is None else positions.long()).clamp(0, tables[0].shape[0] - 1)
        pad = (0, half - tables[0].shape[1])
        cos, sin = (torch.nn.functional.pad(x.to(wide)[at], pad, value=one).unsqueeze(1) for x, one in zip(tables, (1.0, 0.0)))

    def turned(x):
        x1, x2 = x.to(wide)[..., :half], x.to(wide)[..., half:]
        y = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1)
        return y * (y.square().sum(-1, keepdim=True) + eps).rsqrt()

    if B:
        pages, rows = _slots(block_table[s], page, slot.view(-1, 1))
        pages, rows = pages.view(-1), rows.view(-1)
        ok = here & (pages >= 0) & (pages < P)
        k_cache[pages[ok], rows[ok]] = turned(k)[ok].to(k_cache.dtype)
        v_cache[pages[ok], rows[ok]] = v[ok].to(v_cache.dtype)
    return (turned(q) * here.view(-1, 1, 1)).to(k_cache.dtype)


def fused_qk_rope_l2_normalize_append(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor | None,
    sin: torch.Tensor | None,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    eps: float = 1e-12,
) -> torch.Tensor:
    """The Q/K prologue of a serving step, with the keys and values written to
    their slots of the cache; returns the normalised queries (N, H, D).

    ``q`` (N, H, D), ``k`` and ``v`` (N, Hkv, D): the step's new tokens,
    ``cu_seqlens`` (B + 1,) the starts of the sequences among them, or None for
    one token each (N == B).  ``cache_lens`` counts the new tokens already, as
    ``flash_born_attention_paged`` takes it: a sequence's new tokens go to its
    last slots.  Queries and keys are rotated by row ``positions[t]`` of
    ``cos``, ``sin`` ((rows, n) or (1, 1, rows, n), cut or padded to D / 2
    columns; None: not rotated) and divided by sqrt(sum of squares + eps).
    ``positions`` (N,) int32 defaults to the slots; after an eviction they
    differ.  Positions past the tables take the last row.

    As ``fused_qk_rope_l2_normalize`` but for its roundings: this one works in
    fp32 and rounds once, where the training prologue rounds every step to
    16 bits as the reference does.  Values that no sequence owns come out as
    zero queries; slots without a page are not written.
    """
    what = "fused_qk_rope_l2_normalize_append"
    _no_grad(what, q, k, v, k_cache, v_cache)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"q must be (N, heads, head_dim) and k, v (N, key_heads, head_dim), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    N, H, D = q.shape
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    strides = _check_cache(k_cache, v_cache, block_table, cache_lens, B, written=True)
    P, page, Hkv, Dk = k_cache.shape
    if Dk != D or k.shape[1] != Hkv or H < 1 or H % Hkv or D % 2:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} do not fit caches of {Hkv} key heads of {Dk}, or "
                         f"head_dim is odd")
    if cu_seqlens is None:
        if N != B:
            raise ValueError(f"without cu_seqlens there is one token per sequence, got {N} tokens and {B} sequences")
    elif tuple(cu_seqlens.shape) != (B + 1,) or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cu_seqlens must be (B + 1 = {B + 1},) int32, got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)}")
    if positions is not None and (tuple(positions.shape) != (N,) or positions.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"positions must be (N={N},) int32, got {positions.dtype} {tuple(positions.shape)}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    if not float(eps) >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    dev = k_cache.device
    for name, t in (("q", q), ("k", k), ("v", v), ("cu_seqlens", cu_seqlens), ("positions", positions)):
        if t is not None and t.device != dev:
            raise ValueError(f"{name} must be on the caches' device {dev}, got {t.device}")
    tables = None if cos is None else _tables(cos, sin, D // 2, dev)
    if not q.is_cuda:
        return _eager_append(q.detach(), k.detach(), v.detach(), tables, k_cache, v_cache, block_table, cache_lens, cu_seqlens,
                             positions, float(eps))
    lib = _native.load()
    dt = k_cache.dtype
    (q_c, *qs), (k_c, *ks), (v_c, *vs) = (_heads(x.detach(), dt) for x in (q, k, v))
    table, lens = _table(block_table), _index(cache_lens)
    cu, pos = (None if x is None else _index(x) for x in (cu_seqlens, positions))
    out = torch.empty((N, H, D), dtype=dt, device=dev)
    if tables is None:
        rot = (0, 0, 0, 0, 0)
    else:
        c, s = tables
        rot = (c.data_ptr(), s.data_ptr(), c.shape[0], c.shape[1], c.stride(0) if c.shape[0] > 1 else c.shape[1])
    _run_call(lib.qdl_flash_born_cache_append_call, "qdl_flash_born_cache_append_call", dev, _native.append_call(
        _DTYPE_CODE[dt], N, B, H, Hkv, D, q_c.data_ptr(), k_c.data_ptr(), v_c.data_ptr(), *qs, *ks, *vs, out.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), *strides, P, page, table.data_ptr(), table.shape[1], _table_ld(table),
        lens.data_ptr(), 0 if cu is None else cu.data_ptr(), *rot, 0 if pos is None else pos.data_ptr(), float(eps)))
    return out


# ---------------------------------------------------------------------------
# Eviction
# ---------------------------------------------------------------------------
def _eager_evict(k_cache, v_cache, block_table, cache_lens, key_weight, budget, recent, out_table):
    P, page, Hkv, D = k_cache.shape
    B, _, L = key_weight.shape
    room = block_table.shape[1] * page
    dev = k_cache.device
    n = cache_lens.long().clamp(0, room)
    lens = n.clamp(max=budget)
    weight = torch.zeros((B, Hkv, L), dtype=torch.float32, device=dev)
    kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device=dev)
    to = block_table if out_table is None else out_table
    moves = []
    for b in range(B):
        x, m = int(n[b]), int(lens[b])
        tail = m if x <= budget else min(recent, m)
        w = torch.zeros((Hkv, x), dtype=torch.float32, device=dev)
        w[:, : min(x, L)] = key_weight[b, :, : min(x, L)]
        best = w[:, : x - tail].sort(dim=-1, descending=True, stable=True).indices[:, : m - tail].sort(dim=-1).values
        idx = torch.cat([best, torch.arange(x - tail, x, device=dev).expand(Hkv, tail)], dim=1)  # (Hkv, m)
        kept[b, :, :m] = idx.to(torch.int32)
        weight[b, :, : min(m, L)] = w.gather(1, idx)[:, : min(m, L)]
        heads = torch.arange(Hkv, device=dev).view(-1, 1).expand_as(idx)
        src, row = _slots(block_table[b : b + 1].expand(Hkv, -1), page, idx)
        dst, drow = _slots(to[b : b + 1].expand(Hkv, -1), page, torch.arange(m, device=dev).expand(Hkv, m))
        ok, there = (src >= 0) & (src < P), (dst >= 0) & (dst < P)
        if P:
            rows = [torch.where(ok.unsqueeze(-1), c[src.clamp(0, P - 1), row, heads], torch.zeros((), dtype=c.dtype, device=dev))
                    for c in (k_cache, v_cache)]
            moves.append((dst[there], drow[there], heads[there], *(r[there] for r in rows)))
    for dst, drow, heads, kr, vr in moves:
        k_cache[dst, drow, heads] = kr
        v_cache[dst, drow, heads] = vr
    return lens.to(torch.int32), weight, kept


def born_cache_evict(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    key_weight: torch.Tensor,
    budget: int,
    recent: int = 0,
    out_block_table: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Shrink every sequence's cache to at most ``budget`` keys by accumulated
    attention weight; returns ``(cache_lens, key_weight, kept)``.

    Where a sequence holds more, each key head keeps its last ``min(recent,
    budget)`` keys and, of the others, those with the greatest ``key_weight``
    (B, Hkv, L), ties to the lowest index (NaN counts as above all numbers; keys
    at L and after have weight 0).  They keep their order and move to the
    sequence's first slots, in the pages of ``out_block_table`` (B, P'), which
    must not be any of ``block_table``'s (its own pages can be freed afterwards),
    or without one in ``block_table``'s own; sequences must then not share pages.
    Rows behind the last kept one stay as they were.

    Returned are new tensors: the lengths (B,) int32, the kept keys' weights
    (B, Hkv, L), 0 behind the last, so that the next steps can go on adding to
    them, and ``kept`` (B, Hkv, budget) int32, the kept keys' old slots, -1
    behind the last.  Keys stay rotated by the positions that they were appended
    at: pass ``positions`` to the next append.
    """
    _no_grad("born_cache_evict", k_cache, v_cache, key_weight)
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    strides = _check_cache(k_cache, v_cache, block_table, cache_lens, B, written=True)
    P, page, Hkv, D = k_cache.shape
    budget, recent = int(budget), int(recent)
    if not 0 <= budget <= _LIMIT or not 0 <= recent <= _LIMIT:
        raise ValueError(f"budget and recent must be at least 0 and within 2^30, got {budget} and {recent}")
    if (key_weight.dim() != 3 or tuple(key_weight.shape[:2]) != (B, Hkv) or key_weight.dtype != torch.float32
            or key_weight.device != k_cache.device):
        raise ValueError(f"key_weight must be (B={B}, key_heads={Hkv}, keys) fp32 on {k_cache.device}, got {key_weight.dtype} "
                         f"{tuple(key_weight.shape)} on {key_weight.device}")
    most = min(budget, block_table.shape[1] * page)
    if out_block_table is not None:
        if (out_block_table.dim() != 2 or out_block_table.shape[0] != B or out_block_table.dtype not in (torch.int32, torch.int64)
                or out_block_table.device != k_cache.device):
            raise ValueError(f"out_block_table must be (B={B}, pages) int32 on {k_cache.device}, got {out_block_table.dtype} "
                             f"{tuple(out_block_table.shape)} on {out_block_table.device}")
        if out_block_table.shape[1] * page < most:
            raise ValueError(f"out_block_table holds {out_block_table.shape[1]} pages of {page}: fewer than the {most} keys kept")
        if out_block_table.shape[1] * page > _LIMIT:
            raise ValueError(f"out_block_table holds {out_block_table.shape[1]} pages of {page}: more than 2^30 keys a sequence")
        if out_block_table.numel() and out_block_table.data_ptr() == block_table.data_ptr():
            raise ValueError("out_block_table is block_table itself: leave it out to compact in place")
    if not k_cache.is_cuda:
        return _eager_evict(k_cache, v_cache, block_table, cache_lens, key_weight, budget, recent, out_block_table)
    lib = _native.load()
    dev = k_cache.device
    w = key_weight if key_weight.numel() == 0 or key_weight.shape[2] <= 1 or key_weight.stride(2) == 1 else key_weight.contiguous()
    table, lens = _table(block_table), _index(cache_lens)
    to = None if out_block_table is None else _table(out_block_table)
    weight = torch.empty((B, Hkv, w.shape[2]), dtype=torch.float32, device=dev)
    new_lens = torch.empty(B, dtype=torch.int32, device=dev)
    kept = torch.empty((B, Hkv, budget), dtype=torch.int32, device=dev)
    _run_call(lib.qdl_flash_born_cache_evict_call, "qdl_flash_born_cache_evict_call", dev, _native.evict_call(
        _DTYPE_CODE[k_cache.dtype], B, Hkv, D, k_cache.data_ptr(), v_cache.data_ptr(), *strides, P, page, table.data_ptr(),
        table.shape[1], _table_ld(table), lens.data_ptr(), w.data_ptr(), w.stride(0), w.stride(1), w.shape[2], budget, recent,
        0 if to is None else to.data_ptr(), 0 if to is None else to.shape[1], 0 if to is None else _table_ld(to),
        weight.data_ptr(), new_lens.data_ptr(), kept.data_ptr()))
    return new_lens, weight, kept

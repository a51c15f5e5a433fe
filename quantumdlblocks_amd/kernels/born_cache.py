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
same formulas in torch operations.  None of these has a derivative: they refuse
tensors that one is recorded for, backward or forward.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version as _written  # counts a kernel's writes, as torch's in-place operations do

from .. import _native
from .flash_born import _DTYPE_CODE, MAX_HEAD_DIM, _parameter, _run_call
from .flash_born_packed import _LIMIT, _call_uncompiled, _int32, _is_dual

__all__ = ["born_cache_evict", "flash_born_attention_paged", "fused_qk_rope_l2_normalize_append"]

_INDEX = (torch.int32, torch.int64)


def _no_grad(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise RuntimeError(f"{what} has no backward: call it under torch.no_grad(), or with detached tensors")
    if forward_ad._current_level >= 0 and _is_dual(*tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative: call it with the tensors' primals")


def _bad_cache(name: str, c: torch.Tensor):
    return ValueError(f"{name} needs unit stride along head_dim, other strides that are multiples of 16 bytes and a 16-byte "
                      f"aligned base, got strides {c.stride()}")


def _check_cache(k_cache, v_cache, block_table, cache_lens, B, written: bool, apart: bool = False):
    """The caches' (page, token, head) strides on the GPU.  ``apart``: the two
    are written each for itself, so that one row may not be of both.  Decoding
    calls this for every layer and token: plain tests in a row, no loops over
    tensors."""
    shape, dt = k_cache.shape, k_cache.dtype
    if len(shape) != 4 or shape != v_cache.shape or v_cache.dtype != dt:
        raise ValueError(f"k_cache and v_cache must share one (pages, page_size, key_heads, head_dim) shape and dtype, got "
                         f"{dt} {tuple(shape)}, {v_cache.dtype} {tuple(v_cache.shape)}")
    P, page, Hkv, D = shape
    if page < 1 or Hkv < 1 or D < 1:
        raise ValueError(f"page_size, key_heads and head_dim must be positive, got {tuple(shape)}")
    tshape, lshape = block_table.shape, cache_lens.shape
    if len(tshape) != 2 or tshape[0] != B or block_table.dtype not in _INDEX:
        raise ValueError(f"block_table must be (B={B}, pages) int32, got {block_table.dtype} {tuple(tshape)}")
    if len(lshape) != 1 or lshape[0] != B or cache_lens.dtype not in _INDEX:
        raise ValueError(f"cache_lens must be (B={B},) int32, got {cache_lens.dtype} {tuple(lshape)}")
    if tshape[1] * page > _LIMIT:
        raise ValueError(f"block_table holds {tshape[1]} pages of {page}: more than 2^30 keys a sequence")
    dev = k_cache.get_device()
    if v_cache.get_device() != dev or block_table.get_device() != dev or cache_lens.get_device() != dev:
        raise ValueError(f"k_cache, v_cache, block_table and cache_lens must be on one device, got {k_cache.device}, "
                         f"{v_cache.device}, {block_table.device}, {cache_lens.device}")
    ks, vs = k_cache.stride(), v_cache.stride()
    if written:
        for name, st in (("k_cache", ks), ("v_cache", vs)):
            if (st[0] == 0 and P > 1) or (st[1] == 0 and page > 1) or (st[2] == 0 and Hkv > 1) or (st[3] == 0 and D > 1):
                raise ValueError(f"{name} is written and must not overlap itself, got strides {st}")
    if apart and P and k_cache.data_ptr() == v_cache.data_ptr():
        raise ValueError("k_cache and v_cache are both written and must not share memory")
    if dev < 0:
        return ()
    if D % 8 or D > MAX_HEAD_DIM or dt not in _DTYPE_CODE:
        raise NotImplementedError(f"paged caches take fp32, fp16 or bf16 and head dims that are multiples of 8 up to "
                                  f"{MAX_HEAD_DIM}, got {dt} and {D}")
    pieces = 4 if dt is torch.float32 else 8  # elements of 16 bytes
    k0, k1, k2 = ks[0] if P > 1 else 0, ks[1] if page > 1 else 0, ks[2] if Hkv > 1 else 0
    v0, v1, v2 = vs[0] if P > 1 else 0, vs[1] if page > 1 else 0, vs[2] if Hkv > 1 else 0
    if ks[3] != 1 or k0 % pieces or k1 % pieces or k2 % pieces or k_cache.data_ptr() % 16:
        raise _bad_cache("k_cache", k_cache)
    if vs[3] != 1 or v0 % pieces or v1 % pieces or v2 % pieces or v_cache.data_ptr() % 16:
        raise _bad_cache("v_cache", v_cache)
    return k0, k1, k2, v0, v1, v2


def _index(t: torch.Tensor) -> torch.Tensor:
    """1-D int32, contiguous."""
    t = _int32(t)
    return t if t.is_contiguous() else t.contiguous()


def _table(t: torch.Tensor):
    """int32 rows of unit stride, and their distance."""
    t = _int32(t)
    if t.is_contiguous():
        return t, t.shape[1]
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _heads(t: torch.Tensor, dtype: torch.dtype):
    """(n, heads, D) rows in ``dtype`` and their (row, head) strides."""
    if t.dtype is not dtype:
        t = t.to(dtype)
    n, h, _ = t.shape
    s0, s1, s2 = t.stride()
    pieces = 4 if dtype is torch.float32 else 8
    if n <= 1:
        s0 = 0
    if h <= 1:
        s1 = 0
    if s2 != 1 or s0 % pieces or s1 % pieces or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        s0, s1, _ = t.stride()
    return t, s0, s1


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
@functools.lru_cache(maxsize=256)
def _paged_workspace(*sizes) -> int:
    return int(_native.load().qdl_flash_born_paged_workspace_size(*sizes))


def _eager_paged(*args):
    with torch.autocast("cpu", enabled=False):  # not as a decorator, which is one object for all threads
        return _paged_formula(*args)


def _paged_formula(q, k_cache, v_cache, block_table, cache_lens, scale_t, eps, window, key_weight):
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
    p = torch.relu(torch.where(keep.view(B, 1, 1, L), r * s, torch.zeros_like(r))).square()
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
    sees all of them, or the last ``window_size``, counted in slots: after an
    eviction these reach back farther than as many positions.  The formula:

        p_j = max(0, scale_h q . k_j) ** 2,  out = sum_j p_j v_j / (sum_j p_j + eps)

    ``scale``: a float or a tensor of 1 or H values.  ``key_weight`` (B, Hkv, L)
    fp32: each visible key's weight p_j / (sum p + eps), summed over the heads
    that read it, is added in place at j < L: what ``born_cache_evict`` goes by.
    Lengths past the table's pages are cut to them; a sequence without visible
    keys gets zeros, and so does a head whose (sum p + eps) / scale_h ** 2 lies
    below fp32's normal range, 2^-126.
    """
    if torch.compiler.is_compiling():  # one graph break, as the other operators
        return _call_uncompiled(flash_born_attention_paged, (q, k_cache, v_cache, block_table, cache_lens, scale, eps, window_size,
                                                             key_weight))
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_grad("flash_born_attention_paged", q, k_cache, v_cache, scale, key_weight)
    if q.dim() != 3:
        raise ValueError(f"q must be (B, heads, head_dim), got shape {tuple(q.shape)}")
    B, H, D = q.shape
    strides = _check_cache(k_cache, v_cache, block_table, cache_lens, B, written=False)
    P, page, Hkv, Dk = k_cache.shape
    if Dk != D or H < 1 or H % Hkv:
        raise ValueError(f"q {tuple(q.shape)} does not fit caches of {Hkv} key heads of {Dk}")
    if q.get_device() != k_cache.get_device():
        raise ValueError(f"q must be on the caches' device {k_cache.device}, got {q.device}")
    dev, eps = q.device, float(eps)
    # A scale tensor is kept alive here until the call: the block holds addresses.
    if isinstance(scale, torch.Tensor):
        if scale.numel() not in (1, H):
            raise ValueError(f"scale must hold 1 value or H={H} per-head values, got {scale.numel()}")
        scale_flat, scale_p, n_scale, scale_value = _parameter(scale, dev)
    else:
        scale_flat, scale_p, n_scale, scale_value = None, 0, 1, float(scale)
    if not eps >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    window = min(max(int(window_size), 0), _LIMIT)
    w_ptr = w_sb = w_sh = w_len = 0
    if key_weight is not None:
        if (key_weight.dim() != 3 or tuple(key_weight.shape[:2]) != (B, Hkv) or key_weight.dtype != torch.float32
                or key_weight.device != dev or (key_weight.numel() and key_weight.shape[2] > 1 and key_weight.stride(2) != 1)
                or any(n > 1 and s == 0 for n, s in zip(key_weight.shape, key_weight.stride()))):
            raise ValueError(f"key_weight must be (B={B}, key_heads={Hkv}, keys) fp32 on {dev} with unit stride along "
                             f"the keys, got {key_weight.dtype} {tuple(key_weight.shape)} on {key_weight.device}, strides "
                             f"{key_weight.stride()}")
        w_ptr, w_sb, w_sh, w_len = key_weight.data_ptr(), key_weight.stride(0), key_weight.stride(1), key_weight.shape[2]
    if not q.is_cuda:
        scale_t = scale.detach() if isinstance(scale, torch.Tensor) else torch.tensor(scale_value, dtype=torch.float64)
        return _eager_paged(q.detach(), k_cache, v_cache, block_table, cache_lens, scale_t, eps, window, key_weight)
    lib = _native.load()
    dt = k_cache.dtype
    out = k_cache.new_empty((B, H, D))
    if B == 0:
        return out
    q_c, sb, sh = _heads(q, dt)
    (table, ld), lens = _table(block_table), _index(cache_lens)
    pages = table.shape[1]
    size = _paged_workspace(B, H, Hkv, D, pages, page, window, w_ptr != 0)
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    _run_call(lib.qdl_flash_born_paged_forward_call, "qdl_flash_born_paged_forward_call", dev, _native.paged_call(
        _DTYPE_CODE[dt], B, H, Hkv, D, q_c.data_ptr(), sb, sh, out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), *strides,
        P, page, table.data_ptr(), pages, ld, lens.data_ptr(), scale_p, n_scale, scale_value, window, eps, w_ptr, w_sb, w_sh, w_len,
        0 if ws is None else ws.data_ptr(), size))
    if key_weight is not None:
        _written((key_weight,))
    return out


# ---------------------------------------------------------------------------
# New tokens
# ---------------------------------------------------------------------------
def _tables(cos, sin, half, device):
    """(rows, n) fp32 tables with n = min(width, half), and their row stride."""
    if (cos.dim() == 2 and cos.shape == sin.shape and cos.shape[1] <= half and cos.shape[0] > 0 and cos.dtype is torch.float32
            and sin.dtype is torch.float32 and cos.device == device and sin.device == device and cos.is_contiguous()
            and sin.is_contiguous()):
        return cos, sin, cos.shape[1]  # the usual tables: as they are
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
    if not same:
        out = [t.contiguous() for t in out]
    return *out, out[0].stride(0) if out[0].shape[0] > 1 else n


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
        cos, sin = (torch.nn.functional.pad(x.to(wide)[at], pad, value=one).unsqueeze(1) for x, one in zip(tables[:2], (1.0, 0.0)))

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
    queries = turned(q)
    return torch.where(here.view(-1, 1, 1), queries, torch.zeros_like(queries)).to(k_cache.dtype)


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
    if torch.compiler.is_compiling():  # one graph break, as the other operators
        return _call_uncompiled(fused_qk_rope_l2_normalize_append, (q, k, v, cos, sin, k_cache, v_cache, block_table, cache_lens,
                                                                    cu_seqlens, positions, eps))
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_grad("fused_qk_rope_l2_normalize_append", q, k, v, cos, sin, k_cache, v_cache)
    kshape = k.shape
    if q.dim() != 3 or len(kshape) != 3 or kshape != v.shape or kshape[0] != q.shape[0] or kshape[2] != q.shape[2]:
        raise ValueError(f"q must be (N, heads, head_dim) and k, v (N, key_heads, head_dim), got {tuple(q.shape)}, "
                         f"{tuple(kshape)}, {tuple(v.shape)}")
    N, H, D = q.shape
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    strides = _check_cache(k_cache, v_cache, block_table, cache_lens, B, written=True, apart=True)
    P, page, Hkv, Dk = k_cache.shape
    if Dk != D or kshape[1] != Hkv or H < 1 or H % Hkv or D % 2:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(kshape)} do not fit caches of {Hkv} key heads of {Dk}, or "
                         f"head_dim is odd")
    dev, at = k_cache.device, k_cache.get_device()
    if q.get_device() != at or k.get_device() != at or v.get_device() != at:
        raise ValueError(f"q, k and v must be on the caches' device {dev}, got {q.device}, {k.device}, {v.device}")
    if cu_seqlens is None:
        if N != B:
            raise ValueError(f"without cu_seqlens there is one token per sequence, got {N} tokens and {B} sequences")
    elif cu_seqlens.dim() != 1 or cu_seqlens.shape[0] != B + 1 or cu_seqlens.dtype not in _INDEX or cu_seqlens.get_device() != at:
        raise ValueError(f"cu_seqlens must be (B + 1 = {B + 1},) int32 on {dev}, got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)} "
                         f"on {cu_seqlens.device}")
    if positions is not None and (positions.dim() != 1 or positions.shape[0] != N or positions.dtype not in _INDEX
                                  or positions.get_device() != at):
        raise ValueError(f"positions must be (N={N},) int32 on {dev}, got {positions.dtype} {tuple(positions.shape)} on "
                         f"{positions.device}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    tables = None if cos is None else _tables(cos, sin, D // 2, dev)
    if at < 0:
        return _eager_append(q.detach(), k.detach(), v.detach(), tables, k_cache, v_cache, block_table, cache_lens, cu_seqlens,
                             positions, eps)
    lib = _native.load()
    dt = k_cache.dtype
    out = k_cache.new_empty((N, H, D))
    if N == 0:
        return out
    if B == 0:
        return out.zero_()  # tokens of no sequence
    q_c, q0, q1 = _heads(q, dt)
    k_c, k0, k1 = _heads(k, dt)
    v_c, v0, v1 = _heads(v, dt)
    (table, ld), lens = _table(block_table), _index(cache_lens)
    cu = None if cu_seqlens is None else _index(cu_seqlens)
    pos = None if positions is None else _index(positions)
    if tables is None:
        rot = (0, 0, 0, 0, 0)
    else:
        rot = (tables[0].data_ptr(), tables[1].data_ptr(), *tables[0].shape, tables[2])
    _run_call(lib.qdl_flash_born_cache_append_call, "qdl_flash_born_cache_append_call", dev, _native.append_call(
        _DTYPE_CODE[dt], N, B, H, Hkv, D, q_c.data_ptr(), k_c.data_ptr(), v_c.data_ptr(), q0, q1, k0, k1, v0, v1, out.data_ptr(),
        k_cache.data_ptr(), v_cache.data_ptr(), *strides, P, page, table.data_ptr(), table.shape[1], ld, lens.data_ptr(),
        0 if cu is None else cu.data_ptr(), *rot, 0 if pos is None else pos.data_ptr(), eps))
    _written((k_cache, v_cache))
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
    if torch.compiler.is_compiling():  # one graph break, as the other operators
        return _call_uncompiled(born_cache_evict, (k_cache, v_cache, block_table, cache_lens, key_weight, budget, recent,
                                                   out_block_table))
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_grad("born_cache_evict", k_cache, v_cache, key_weight)
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    strides = _check_cache(k_cache, v_cache, block_table, cache_lens, B, written=True, apart=out_block_table is None)
    P, page, Hkv, D = k_cache.shape
    dev, at = k_cache.device, k_cache.get_device()
    budget, recent = int(budget), int(recent)
    if not 0 <= budget <= _LIMIT or not 0 <= recent <= _LIMIT:
        raise ValueError(f"budget and recent must be at least 0 and within 2^30, got {budget} and {recent}")
    wshape = key_weight.shape
    if len(wshape) != 3 or wshape[0] != B or wshape[1] != Hkv or key_weight.dtype is not torch.float32 or key_weight.get_device() != at:
        raise ValueError(f"key_weight must be (B={B}, key_heads={Hkv}, keys) fp32 on {dev}, got {key_weight.dtype} "
                         f"{tuple(wshape)} on {key_weight.device}")
    if out_block_table is not None:
        tshape = out_block_table.shape
        if len(tshape) != 2 or tshape[0] != B or out_block_table.dtype not in _INDEX or out_block_table.get_device() != at:
            raise ValueError(f"out_block_table must be (B={B}, pages) int32 on {dev}, got {out_block_table.dtype} {tuple(tshape)} "
                             f"on {out_block_table.device}")
        most = min(budget, block_table.shape[1] * page)
        if tshape[1] * page < most:
            raise ValueError(f"out_block_table holds {tshape[1]} pages of {page}: fewer than the {most} keys kept")
        if tshape[1] * page > _LIMIT:
            raise ValueError(f"out_block_table holds {tshape[1]} pages of {page}: more than 2^30 keys a sequence")
        if tshape[1] and B and out_block_table.data_ptr() == block_table.data_ptr():
            raise ValueError("out_block_table is block_table itself: leave it out to compact in place")
    if at < 0:
        return _eager_evict(k_cache, v_cache, block_table, cache_lens, key_weight, budget, recent, out_block_table)
    lib = _native.load()
    w = key_weight
    if not w.is_contiguous() and wshape[2] > 1 and w.stride(2) != 1:
        w = w.contiguous()
    (table, ld), lens = _table(block_table), _index(cache_lens)
    to, to_ld = (None, 0) if out_block_table is None else _table(out_block_table)
    weight = w.new_empty(wshape)
    new_lens, kept = lens.new_empty(B), lens.new_empty((B, Hkv, budget))
    if B == 0:
        return new_lens, weight, kept
    _run_call(lib.qdl_flash_born_cache_evict_call, "qdl_flash_born_cache_evict_call", dev, _native.evict_call(
        _DTYPE_CODE[k_cache.dtype], B, Hkv, D, k_cache.data_ptr(), v_cache.data_ptr(), *strides, P, page, table.data_ptr(),
        table.shape[1], ld, lens.data_ptr(), w.data_ptr(), w.stride(0), w.stride(1), wshape[2], budget, recent,
        0 if to is None else to.data_ptr(), 0 if to is None else to.shape[1], to_ld,
        weight.data_ptr(), new_lens.data_ptr(), kept.data_ptr()))
    _written((k_cache, v_cache))
    return new_lens, weight, kept

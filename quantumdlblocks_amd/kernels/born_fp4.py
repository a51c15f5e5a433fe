"""A paged key-value cache for Born attention in 4 bits: a quarter of the memory
and of the traffic of the 16-bit one (``born_cache``), whose pages, tables and
lengths it shares.

A row (one head of one token) is stored in blocks of 32 columns, the head dim
rounded up to whole blocks: a 4-bit code for each column, two in a byte, the
lower nibble the even one (sign, two exponent bits, one mantissa bit: 0, 0.5, 1,
1.5, 2, 3, 4, 6), and a byte e for each block; a value is its code times
2 ** (e - 127).  e is the least with max |x| <= 7 * 2 ** (e - 127) over the block
(at least 1), codes are the nearest, halfway to the even one, and at most 6.
The values stored for a row of normal ones are off by 0.112 of it in norm.
They are exact in bf16; a block with an infinity, a NaN or a magnitude past
7 * 2 ** 125 has e = 255: not a number.

    born_cache_fp4                            an empty cache
    fused_qk_rope_l2_normalize_append_fp4     a step's new tokens, written to their slots
    flash_born_attention_paged_fp4            one new token per sequence attends, or several
    born_cache_read_fp4                       rows as values again
    born_cache_evict_fp4                      keep the recent keys and the heaviest

No call copies anything to the host, so a step can be captured into a HIP graph;
tables and lengths may change between replays.  CPU tensors run the same formulas
in torch operations.  None of these has a derivative: they refuse tensors that
one is recorded for, backward or forward.
"""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from .. import _native
from .born_cache import _eager_evict, _heads, _index, _INDEX, _no_grad, _slots, _table, _tables, _written
from .flash_born import _DTYPE_CODE, MAX_HEAD_DIM, _parameter, _run_call
from .flash_born_packed import _LIMIT, _call_uncompiled

__all__ = [
    "BornCacheFp4",
    "born_cache_evict_fp4",
    "born_cache_fp4",
    "born_cache_read_fp4",
    "flash_born_attention_paged_fp4",
    "fused_qk_rope_l2_normalize_append_fp4",
]

_BLOCK = 32
_BAD = 255
_U8 = torch.uint8


class BornCacheFp4(NamedTuple):
    """The tensors of a cache, uint8: codes (pages, page_size, Hkv, W / 2) and
    scales (pages, page_size, Hkv, W / 32), W the head dim rounded up to 32s, in
    any strides with unit stride along the last dimension (codes: others that are
    multiples of 16 bytes).  The calls take any tuple of the four."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def born_cache_fp4(pages: int, page_size: int, key_heads: int, head_dim: int, device="cuda") -> BornCacheFp4:
    """An empty cache whose pages hold one head after the other, so that a head's
    tokens lie side by side: what the attention reads fastest."""
    if pages < 0 or page_size < 1 or key_heads < 1 or head_dim < 1:
        raise ValueError(f"page_size, key_heads and head_dim must be positive and pages not negative, got {pages}, {page_size}, "
                         f"{key_heads}, {head_dim}")
    nb = -(-head_dim // _BLOCK)
    made = [torch.zeros((pages, key_heads, page_size, nb * n), dtype=torch.uint8, device=device).transpose(1, 2) for n in (16, 16, 1, 1)]
    return BornCacheFp4(*made)


def _check_fp4(cache, block_table, cache_lens, B, head_dim, written: bool):
    """The cache's fields of the argument blocks up to page_size, on the GPU.
    ``head_dim`` None: any.  ``written``: the tensors are, so none may overlap
    itself or be another.  Plain tests in a row, as for the 16-bit cache: decoding
    calls this for every layer and token."""
    if len(cache) != 4:
        raise ValueError(f"a 4-bit cache is its codes and scales (k, v, k_scale, v_scale), got {len(cache)} tensors")
    k, v, ks, vs = cache
    shape, sshape, tshape = k.shape, ks.shape, block_table.shape
    if len(shape) != 4 or v.shape != shape or len(sshape) != 4 or vs.shape != sshape or sshape[:3] != shape[:3] or shape[3] != 16 * sshape[3]:
        raise ValueError(f"a 4-bit cache is codes (pages, page_size, key_heads, 16 n) and scales (pages, page_size, key_heads, n), "
                         f"got {[tuple(t.shape) for t in cache]}")
    if k.dtype is not _U8 or v.dtype is not _U8 or ks.dtype is not _U8 or vs.dtype is not _U8:
        raise ValueError(f"a 4-bit cache is held in uint8, got {[t.dtype for t in cache]}")
    P, page, Hkv, nb = sshape
    if page < 1 or Hkv < 1 or nb < 1:
        raise ValueError(f"page_size, key_heads and head_dim must be positive, got {tuple(shape)}")
    if head_dim is not None and not _BLOCK * (nb - 1) < head_dim <= _BLOCK * nb:
        raise ValueError(f"head_dim {head_dim} does not fit a cache of {nb} blocks of {_BLOCK} columns")
    if len(tshape) != 2 or tshape[0] != B or block_table.dtype not in _INDEX:
        raise ValueError(f"block_table must be (B={B}, pages) int32, got {block_table.dtype} {tuple(tshape)}")
    if cache_lens.shape != (B,) or cache_lens.dtype not in _INDEX:
        raise ValueError(f"cache_lens must be (B={B},) int32, got {cache_lens.dtype} {tuple(cache_lens.shape)}")
    if tshape[1] * page > _LIMIT:
        raise ValueError(f"block_table holds {tshape[1]} pages of {page}: more than 2^30 keys a sequence")
    dev = k.get_device()
    if not (v.get_device() == ks.get_device() == vs.get_device() == block_table.get_device() == cache_lens.get_device() == dev):
        raise ValueError(f"the cache, block_table and cache_lens must be on one device, got {[t.device for t in cache]}, "
                         f"{block_table.device}, {cache_lens.device}")
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    s0, s1, s2, s3 = ks.stride()
    u0, u1, u2, u3 = vs.stride()
    pk, pv, ps, pu = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()
    if written:
        if not (k0 and k1 and k2 and k3 and v0 and v1 and v2 and v3 and s0 and s1 and s2 and s3 and u0 and u1 and u2 and u3):
            for name, t in zip(("k", "v", "k_scale", "v_scale"), cache):
                if any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
                    raise ValueError(f"{name} is written and must not overlap itself, got strides {t.stride()}")
        if P and (pk == pv or ps == pu or pk == ps or pk == pu or pv == ps or pv == pu):
            raise ValueError("the cache's four tensors are all written and must not share memory")
    if dev < 0:
        return ()
    if nb * _BLOCK > MAX_HEAD_DIM:
        raise NotImplementedError(f"paged caches take head dims up to {MAX_HEAD_DIM}, got {nb} blocks of {_BLOCK}")
    if P <= 1:
        k0 = v0 = s0 = u0 = 0
    if page == 1:
        k1 = v1 = s1 = u1 = 0
    if Hkv == 1:
        k2 = v2 = s2 = u2 = 0
    any_stride = k0 | k1 | k2 | v0 | v1 | v2
    if k3 != 1 or v3 != 1 or (any_stride | pk | pv) & 15:
        raise ValueError(f"codes need unit stride along a row, other strides that are multiples of 16 and a 16-byte aligned base, "
                         f"got strides {k.stride()} and {v.stride()}")
    if (any_stride | s0 | s1 | s2 | u0 | u1 | u2) >> 32:
        raise ValueError(f"a cache's strides lie under 2^32, got {[t.stride() for t in cache]}")
    if nb > 1 and (s3 != 1 or u3 != 1):
        raise ValueError(f"scales need unit stride along a row, got strides {ks.stride()} and {vs.stride()}")
    return pk, pv, ps, pu, k0, k1, k2, v0, v1, v2, s0, s1, s2, u0, u1, u2, P, page


def _check_type(D: int, dtype: torch.dtype) -> None:
    if D % 8 or dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"4-bit caches take fp32, fp16 or bf16 rows and head dims that are multiples of 8, got {dtype} and {D}")


def _check_starts(cu_seqlens, B, dev, at) -> None:
    if cu_seqlens.shape != (B + 1,) or cu_seqlens.dtype not in _INDEX or cu_seqlens.get_device() != at:
        raise ValueError(f"cu_seqlens must be (B + 1 = {B + 1},) int32 on {dev}, got {cu_seqlens.dtype} {tuple(cu_seqlens.shape)} "
                         f"on {cu_seqlens.device}")


# ---------------------------------------------------------------------------
# The format, in torch operations
# ---------------------------------------------------------------------------
def _power(e: torch.Tensor) -> torch.Tensor:
    """2 ** e in fp64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _encode(x: torch.Tensor):
    """Rows (..., D) -> codes (..., W / 2) and scales (..., W / 32)."""
    D = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -D % _BLOCK)).unflatten(-1, (-1, _BLOCK))
    top = x.abs().amax(-1)
    bad = ~(top <= 7 * 2.0**125)
    m, e = torch.frexp(torch.where(bad, torch.ones_like(top), top))
    e = torch.where(top == 0, torch.full_like(e, -126), e - 3 + (m > 0.875)).clamp(min=-126)
    y = torch.where(bad.unsqueeze(-1), torch.zeros_like(x), x * _power(-e).unsqueeze(-1))
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    a = torch.round(a / step) * step  # halfway to even
    code = torch.where(a < 2.0, 2 * a, torch.where(a < 4.0, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).flatten(-2)
    scale = torch.where(bad, torch.full_like(e, _BAD), e + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


_CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Codes and scales -> values (..., W) in fp64."""
    table = torch.tensor(_CODES, dtype=torch.float64, device=codes.device)
    y = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()].unflatten(-1, (-1, _BLOCK))
    y = y * _power(scales.int() - 127).unsqueeze(-1)
    return torch.where((scales == _BAD).unsqueeze(-1), torch.full_like(y, float("nan")), y).flatten(-2)


def _packed_slots(n, cu, cache_lens, B, device):
    """Of packed rows: their sequence, whether they have one, their slot (-1 where not)."""
    t = torch.arange(n, device=device)
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
    return s, here, slot


def _packed_pages(cache, block_table, s, here, slot):
    """Pages and rows of packed rows, and whether they are there."""
    P, page = cache[0].shape[:2]
    if not block_table.shape[0]:
        return slot, slot, torch.zeros_like(here)
    pages, rows = _slots(block_table[s], page, slot.view(-1, 1))
    pages, rows = pages.view(-1), rows.view(-1)
    return pages, rows, here & (pages >= 0) & (pages < P)


# ---------------------------------------------------------------------------
# New tokens
# ---------------------------------------------------------------------------
def _eager_append(q, k, v, tables, cache, block_table, cache_lens, cu, positions, eps):
    N, B = q.shape[0], cache_lens.shape[0]
    s, here, slot = _packed_slots(N, cu, cache_lens, B, q.device)
    half = q.shape[2] // 2

    def turned(x, wide):
        if tables is None:
            cos, sin = torch.ones((N, 1, half), dtype=wide, device=q.device), torch.zeros((N, 1, half), dtype=wide, device=q.device)
        else:
            at = (slot if positions is None else positions.long()).clamp(0, tables[0].shape[0] - 1)
            pad = (0, half - tables[0].shape[1])
            cos, sin = (torch.nn.functional.pad(y.to(wide)[at], pad, value=one).unsqueeze(1) for y, one in zip(tables[:2], (1.0, 0.0)))
        x1, x2 = x.to(wide)[..., :half], x.to(wide)[..., half:]
        y = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1)
        return y / (y.square().sum(-1, keepdim=True) + eps).sqrt()

    pages, rows, ok = _packed_pages(cache, block_table, s, here, slot)
    for codes, scales, x in ((cache[0], cache[2], turned(k, torch.float64)), (cache[1], cache[3], v)):
        codes[pages[ok], rows[ok]], scales[pages[ok], rows[ok]] = _encode(x[ok])
    queries = turned(q, torch.float64 if q.dtype == torch.float64 else torch.float32)
    return torch.where(here.view(-1, 1, 1), queries, torch.zeros_like(queries)).to(q.dtype)


def fused_qk_rope_l2_normalize_append_fp4(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cos: torch.Tensor | None,
    sin: torch.Tensor | None,
    cache: BornCacheFp4,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    eps: float = 1e-12,
) -> torch.Tensor:
    """``fused_qk_rope_l2_normalize_append`` into a 4-bit cache: the Q/K prologue
    of a serving step, with the keys and values stored in their slots; returns
    the normalised queries (N, H, D) in ``q``'s dtype.

    The arguments are the same but for ``cache``; ``k`` and ``v`` have ``q``'s
    dtype or are cast to it.  Keys are rotated and normalised in 64 bits before
    their codes are chosen, so these do not depend on the order of a sum; queries
    in fp32, rounded once.  A token with an infinity or NaN in its key or value,
    or a value past 7 * 2 ** 125, makes NaN of the rows that see it.
    """
    if torch.compiler.is_compiling():  # one graph break, as the other operators
        return _call_uncompiled(fused_qk_rope_l2_normalize_append_fp4, (q, k, v, cos, sin, cache, block_table, cache_lens, cu_seqlens,
                                                                        positions, eps))
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_grad("fused_qk_rope_l2_normalize_append_fp4", q, k, v, cos, sin)
    kshape = k.shape
    if q.dim() != 3 or len(kshape) != 3 or kshape != v.shape or kshape[0] != q.shape[0] or kshape[2] != q.shape[2]:
        raise ValueError(f"q must be (N, heads, head_dim) and k, v (N, key_heads, head_dim), got {tuple(q.shape)}, "
                         f"{tuple(kshape)}, {tuple(v.shape)}")
    N, H, D = q.shape
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    fields = _check_fp4(cache, block_table, cache_lens, B, D, written=True)
    Hkv = cache[0].shape[2]
    if kshape[1] != Hkv or H < 1 or H % Hkv or D % 2:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(kshape)} do not fit a cache of {Hkv} key heads, or head_dim is odd")
    dev, at = q.device, q.get_device()
    if cache[0].get_device() != at or k.get_device() != at or v.get_device() != at:
        raise ValueError(f"q, k and v must be on the cache's device {cache[0].device}, got {q.device}, {k.device}, {v.device}")
    if cu_seqlens is None:
        if N != B:
            raise ValueError(f"without cu_seqlens there is one token per sequence, got {N} tokens and {B} sequences")
    else:
        _check_starts(cu_seqlens, B, dev, at)
    if positions is not None and (positions.shape != (N,) or positions.dtype not in _INDEX
                                  or positions.get_device() != at):
        raise ValueError(f"positions must be (N={N},) int32 on {dev}, got {positions.dtype} {tuple(positions.shape)} on "
                         f"{positions.device}")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    tables = None if cos is None else _tables(cos, sin, D // 2, dev)
    dt = q.dtype
    if at < 0:
        return _eager_append(q.detach(), k.detach().to(dt), v.detach().to(dt), tables, cache, block_table, cache_lens, cu_seqlens,
                             positions, eps)
    _check_type(D, dt)
    lib = _native.load()
    out = q.new_empty((N, H, D))
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
    rot = (0, 0, 0, 0, 0) if tables is None else (tables[0].data_ptr(), tables[1].data_ptr(), *tables[0].shape, tables[2])
    _run_call(lib.qdl_flash_born_fp4_append_call, "qdl_flash_born_fp4_append_call", dev, _native.fp4_append_call(
        _DTYPE_CODE[dt], N, B, H, Hkv, D, q_c.data_ptr(), k_c.data_ptr(), v_c.data_ptr(), q0, q1, k0, k1, v0, v1, out.data_ptr(),
        *fields, table.data_ptr(), table.shape[1], ld, lens.data_ptr(), 0 if cu is None else cu.data_ptr(), *rot,
        0 if pos is None else pos.data_ptr(), eps))
    _written(cache)
    return out


# ---------------------------------------------------------------------------
# Reading back
# ---------------------------------------------------------------------------
def born_cache_read_fp4(
    cache: BornCacheFp4,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    cu_seqlens: torch.Tensor,
    total: int,
    head_dim: int | None = None,
    dtype: torch.dtype = torch.bfloat16,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values as packed rows (total, Hkv, D) of ``dtype``, as
    ``flash_born_attention_packed`` takes them: rows ``cu_seqlens[b] :
    cu_seqlens[b + 1]`` are the last keys of sequence b, all of them where these
    are as many as ``cache_lens`` counts.

    Values are exact in bf16 and fp32, and in fp16 but for those past its range
    or below its normal numbers.  ``head_dim`` defaults to the cache's columns.
    Rows of no sequence, and keys without a page, are zeros.
    """
    if torch.compiler.is_compiling():  # one graph break, as the other operators
        return _call_uncompiled(born_cache_read_fp4, (cache, block_table, cache_lens, cu_seqlens, total, head_dim, dtype))
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    fields = _check_fp4(cache, block_table, cache_lens, B, head_dim, written=False)
    Hkv, nb = cache[2].shape[2:]
    D, N = _BLOCK * nb if head_dim is None else int(head_dim), int(total)
    dev, at = cache[0].device, cache[0].get_device()
    _check_starts(cu_seqlens, B, dev, at)
    if N < 0:
        raise ValueError(f"total must be at least 0, got {N}")
    if not dtype.is_floating_point:
        raise ValueError(f"dtype must be a floating one, got {dtype}")
    if at < 0:
        pages, rows, ok = _packed_pages(cache, block_table, *_packed_slots(N, cu_seqlens, cache_lens, B, dev))
        out = []
        for codes, scales in ((cache[0], cache[2]), (cache[1], cache[3])):
            x = torch.zeros((N, Hkv, D), dtype=dtype, device=dev)
            x[ok] = _decode(codes[pages[ok], rows[ok]], scales[pages[ok], rows[ok]])[..., :D].to(dtype)
            out.append(x)
        return tuple(out)
    _check_type(D, dtype)
    lib = _native.load()
    k = torch.empty((N, Hkv, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    if N == 0:
        return k, v
    if B == 0:
        return k.zero_(), v.zero_()  # rows of no sequence
    (table, ld), lens, cu = _table(block_table), _index(cache_lens), _index(cu_seqlens)
    _run_call(lib.qdl_flash_born_fp4_read_call, "qdl_flash_born_fp4_read_call", dev, _native.fp4_read_call(
        _DTYPE_CODE[dtype], N, B, Hkv, D, k.data_ptr(), v.data_ptr(), *fields, table.data_ptr(), table.shape[1], ld, lens.data_ptr(),
        cu.data_ptr()))
    return k, v


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
@functools.lru_cache(maxsize=256)
def _paged_workspace(*sizes) -> int:
    return int(_native.load().qdl_flash_born_fp4_paged_workspace_size(*sizes))


def _eager_paged(*args):
    with torch.autocast("cpu", enabled=False):  # not as a decorator, which is one object for all threads
        return _paged_formula(*args)


def _paged_formula(q, cache, block_table, cache_lens, scale_t, cu, eps, window, key_weight):
    N, H, D = q.shape
    B, width = block_table.shape
    P, page, Hkv = cache[0].shape[:3]
    G, L = H // Hkv, width * page
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros((N, H, D), dtype=q.dtype, device=q.device)
    starts = list(range(B + 1)) if cu is None else [0] + [min(max(int(x), 0), N) for x in cu.tolist()[1:]]
    s = scale_t.to(device=q.device, dtype=wide).reshape(-1).expand(H).view(Hkv, G, 1, 1)
    j = torch.arange(L, device=q.device)
    for b in range(B):
        a0, new = starts[b], max(starts[b + 1] - starts[b], 0)
        n = min(max(int(cache_lens[b]), 0), L)
        pages, rows = _slots(block_table[b : b + 1], page, j.view(1, L))
        pages, rows = pages[0], rows[0]
        there = (pages >= 0) & (pages < P) & (j < n)
        at, rows = torch.where(there, pages, torch.zeros_like(pages)), torch.where(there, rows, torch.zeros_like(rows))
        if P == 0 or L == 0:
            k = v = torch.zeros((L, Hkv, D), dtype=wide, device=q.device)
        else:
            k, v = (_decode(c[at, rows], e[at, rows])[..., :D].to(wide) for c, e in ((cache[0], cache[2]), (cache[1], cache[3])))
            bad = (cache[2][at, rows] == _BAD).any(-1) | (cache[3][at, rows] == _BAD).any(-1)  # (L, Hkv)
            k = torch.where(bad.unsqueeze(-1), torch.full_like(k, float("nan")), k)
            v = torch.where(bad.unsqueeze(-1) | ~there.view(-1, 1, 1), torch.zeros_like(v), v)
        i = n - new + torch.arange(new, device=q.device).view(-1, 1)
        keep = there.view(1, L) & (j.view(1, L) <= i)
        if window > 0:
            keep = keep & (i - j.view(1, L) < window)
        x = q[a0 : a0 + new].to(wide).view(new, Hkv, G, D).permute(1, 2, 0, 3)
        r = torch.matmul(x, k.permute(1, 2, 0).unsqueeze(1))  # (Hkv, G, new, L)
        p = torch.relu(torch.where(keep, r * s, torch.zeros_like(r))).square()
        den = p.sum(-1, keepdim=True) + eps
        w = p / torch.where(den == 0, torch.ones_like(den), den)
        if key_weight is not None:
            m = min(L, key_weight.shape[2])
            seen = torch.where(keep, w, torch.zeros_like(w))  # a row that is not a number is NaN throughout
            key_weight[b, :, :m] += seen.sum((1, 2))[:, :m].to(key_weight.dtype)
        o = torch.matmul(w, v.permute(1, 0, 2).unsqueeze(1))
        out[a0 : a0 + new] = o.permute(2, 0, 1, 3).reshape(new, H, D).to(q.dtype)
    return out


def flash_born_attention_paged_fp4(
    q: torch.Tensor,
    cache: BornCacheFp4,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    scale: float | torch.Tensor,
    cu_seqlens: torch.Tensor | None = None,
    eps: float = 1e-12,
    window_size: int = 0,
    key_weight: torch.Tensor | None = None,
) -> torch.Tensor:
    """Born attention of new tokens over a 4-bit cache; returns (N, H, D) in
    ``q``'s dtype.

    ``q`` (N, H, D), H a multiple of the cache's Hkv: one new token per sequence
    (N == B), or several, packed, with ``cu_seqlens`` (B + 1,) the starts of the
    sequences among them (the first is 0), 65536 sequences at most.  Their keys
    are in the cache already and ``cache_lens`` counts them: a sequence's i-th
    token of m stands at ``cache_lens - m + i`` and sees the keys up to there, or
    the last ``window_size`` of them, counted in slots.  The formula, over the
    stored values:

        p_ij = max(0, scale_h q_i . k_j) ** 2,  out_i = sum_j p_ij v_j / (sum_j p_ij + eps)

    ``scale``: a float or a tensor of 1 or H values.  ``key_weight`` (B, Hkv, L)
    fp32, only without ``cu_seqlens``: each visible key's weight p_j / (sum p +
    eps), summed over the heads that read it, is added in place at j < L: what
    ``born_cache_evict_fp4`` goes by; the call's workspace holds B H fp32 values
    for each of these L keys, or of the table's where it has fewer.  Lengths past
    the table's pages are cut to them first.  Tokens that see no key get zeros, so
    do tokens of no sequence, and heads whose (sum p + eps) / scale_h ** 2 lies
    below fp32's normal range, 2^-126; overlaps q_i . k_j from 2^64 on, whose
    squares lie past it, are infinite whatever the scale.  A row's precision does
    not go by the others in the batch.  A key that is not a number makes NaN of
    the rows that see it.
    """
    if torch.compiler.is_compiling():  # one graph break, as the other operators
        return _call_uncompiled(flash_born_attention_paged_fp4, (q, cache, block_table, cache_lens, scale, cu_seqlens, eps,
                                                                 window_size, key_weight))
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_grad("flash_born_attention_paged_fp4", q, scale, key_weight)
    if q.dim() != 3:
        raise ValueError(f"q must be (tokens, heads, head_dim), got shape {tuple(q.shape)}")
    N, H, D = q.shape
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    fields = _check_fp4(cache, block_table, cache_lens, B, D, written=False)
    page, Hkv = cache[0].shape[1:3]
    if H < 1 or H % Hkv:
        raise ValueError(f"the {H} query heads must be a multiple of the cache's {Hkv} key heads")
    dev, at = q.device, q.get_device()
    if cache[0].get_device() != at:
        raise ValueError(f"q must be on the cache's device {cache[0].device}, got {dev}")
    if cu_seqlens is None:
        if N != B:
            raise ValueError(f"without cu_seqlens there is one token per sequence, got {N} tokens and {B} sequences")
    else:
        _check_starts(cu_seqlens, B, dev, at)
    eps = float(eps)
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
        if cu_seqlens is not None:
            raise NotImplementedError("key_weight is kept for one new token per sequence, without cu_seqlens")
        if (key_weight.dim() != 3 or tuple(key_weight.shape[:2]) != (B, Hkv) or key_weight.dtype != torch.float32
                or key_weight.device != dev or (key_weight.numel() and key_weight.shape[2] > 1 and key_weight.stride(2) != 1)
                or any(n > 1 and s == 0 for n, s in zip(key_weight.shape, key_weight.stride()))):
            raise ValueError(f"key_weight must be (B={B}, key_heads={Hkv}, keys) fp32 on {dev} with unit stride along "
                             f"the keys, got {key_weight.dtype} {tuple(key_weight.shape)} on {key_weight.device}, strides "
                             f"{key_weight.stride()}")
        w_ptr, w_sb, w_sh, w_len = key_weight.data_ptr(), key_weight.stride(0), key_weight.stride(1), key_weight.shape[2]
    if at < 0:
        scale_t = scale.detach() if isinstance(scale, torch.Tensor) else torch.tensor(scale_value, dtype=torch.float64)
        return _eager_paged(q.detach(), cache, block_table, cache_lens, scale_t, cu_seqlens, eps, window, key_weight)
    dt = q.dtype
    _check_type(D, dt)
    lib = _native.load()
    out = q.new_empty((N, H, D))
    if N == 0:
        return out
    if B == 0:
        return out.zero_()  # tokens of no sequence
    q_c, st, sh = _heads(q, dt)
    (table, ld), lens = _table(block_table), _index(cache_lens)
    cu = None if cu_seqlens is None else _index(cu_seqlens)
    pages = table.shape[1]
    size = _paged_workspace(N, B, H, Hkv, D, pages, page, window, cu is not None, max(w_len, 2) if w_ptr else 0)
    ws = lens.new_empty((size + 3) // 4)
    _run_call(lib.qdl_flash_born_fp4_paged_forward_call, "qdl_flash_born_fp4_paged_forward_call", dev, _native.fp4_paged_call(
        _DTYPE_CODE[dt], N, B, H, Hkv, D, q_c.data_ptr(), st, sh, out.data_ptr(), *fields, table.data_ptr(), pages, ld,
        lens.data_ptr(), 0 if cu is None else cu.data_ptr(), scale_p, n_scale, scale_value, window, eps, w_ptr, w_sb, w_sh, w_len,
        ws.data_ptr(), size))
    if key_weight is not None:
        _written((key_weight,))
    return out


# ---------------------------------------------------------------------------
# Eviction
# ---------------------------------------------------------------------------
def born_cache_evict_fp4(
    cache: BornCacheFp4,
    block_table: torch.Tensor,
    cache_lens: torch.Tensor,
    key_weight: torch.Tensor,
    budget: int,
    recent: int = 0,
    out_block_table: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``born_cache_evict`` for a 4-bit cache: every sequence keeps at most
    ``budget`` keys, chosen and moved as there, codes and scales as they are;
    returns ``(cache_lens, key_weight, kept)``."""
    if torch.compiler.is_compiling():  # one graph break, as the other operators
        return _call_uncompiled(born_cache_evict_fp4, (cache, block_table, cache_lens, key_weight, budget, recent, out_block_table))
    if torch.is_grad_enabled() or forward_ad._current_level >= 0:
        _no_grad("born_cache_evict_fp4", key_weight)
    B = block_table.shape[0] if block_table.dim() == 2 else -1
    fields = _check_fp4(cache, block_table, cache_lens, B, None, written=True)
    page, Hkv, nb = cache[2].shape[1:]
    dev, at = cache[0].device, cache[0].get_device()
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
        k, v, ks, vs = cache
        rows = [torch.cat([c, e], -1) for c, e in ((k, ks), (v, vs))]
        got = _eager_evict(*rows, block_table, cache_lens, key_weight, budget, recent, out_block_table)
        for both, c, e in zip(rows, (k, v), (ks, vs)):
            c.copy_(both[..., : 16 * nb])
            e.copy_(both[..., 16 * nb :])
        return got
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
    _run_call(lib.qdl_flash_born_fp4_evict_call, "qdl_flash_born_fp4_evict_call", dev, _native.fp4_evict_call(
        B, Hkv, _BLOCK * nb, *fields, table.data_ptr(), table.shape[1], ld, lens.data_ptr(), w.data_ptr(), w.stride(0), w.stride(1),
        wshape[2], budget, recent, 0 if to is None else to.data_ptr(), 0 if to is None else to.shape[1], to_ld, weight.data_ptr(),
        new_lens.data_ptr(), kept.data_ptr()))
    _written(tuple(cache))
    return new_lens, weight, kept

"""The 4-bit cache's format and its attention in 64 bits, written apart from the
package, and how far a kernel's outputs may be from them.

Stored values are exact in bf16, so an overlap is an fp32 sum of exact products
(the query's bf16 parts times the key): |dr| <= parts D 2^-24 sum |q k|.  The
weights go into their product in two bf16 parts, what is left of them below
2^-17 relative (each part takes half a step of 2^-8), fp32's in three, below two
roundings of the square; bf16's in one, half a step of 2^-8, where a sequence
has more than 32 rows (new tokens x heads of a group), but for calls of 512 rows
or fewer and at most 64 a sequence in the mean.  Sums of n terms are fp32 sums, the output is rounded
once."""

from __future__ import annotations

import math

import torch

from serve_ref import HALF_STEP, LEAST, U32

CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
PARTS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}
WEIGHT = {torch.bfloat16: 2.0 ** -17 + 3 * U32, torch.float16: 2.0 ** -17 + 3 * U32, torch.float32: 3 * U32}


def store_block(x):
    """32 Python floats -> (scale byte, 32 codes), by trying every code."""
    if not all(abs(v) <= 7.0 * 2.0 ** 125 for v in x):
        return 255, [0] * 32
    top = max(abs(v) for v in x)
    e = -126
    while top > 7.0 * 2.0 ** e:
        e += 1
    codes = []
    for v in x:
        a = abs(v) / 2.0 ** e
        # Nearest; of two as near the even code.
        c = min(range(8), key=lambda i: (abs(a - CODES[i]), i % 2))
        codes.append(c + (8 if math.copysign(1.0, v) < 0 else 0))
    return e + 127, codes


def value(codes, scales):
    """uint8 rows (..., 16 n), (..., n) -> fp64 values (..., 32 n)."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    y = torch.tensor(CODES + [-x for x in CODES], dtype=torch.float64, device=codes.device)[c]
    p = torch.tensor([2.0 ** (e - 127) if e < 255 else math.nan for e in range(256)], dtype=torch.float64, device=codes.device)
    return y * p[scales.long()].repeat_interleave(32, -1)


def rows(cache, table, n, D):
    """(n, Hkv, D) keys and values of one sequence, which of them are there, and
    which are not numbers (n, Hkv)."""
    kc, vc, ks, vs = (t.cpu() for t in cache)
    page = kc.shape[1]
    ok, k, v, bad = [], [], [], []
    for j in range(n):
        t = int(table[j // page])
        ok.append(0 <= t < kc.shape[0])
        t, r = (t, j % page) if ok[-1] else (0, 0)
        k.append(value(kc[t, r], ks[t, r])[..., :D])
        v.append(value(vc[t, r], vs[t, r])[..., :D])
        bad.append((ks[t, r] == 255).any(-1) | (vs[t, r] == 255).any(-1))
    if not n:
        return torch.zeros(0, kc.shape[2], D, dtype=torch.float64), None, torch.zeros(0, dtype=torch.bool), None
    return torch.stack(k), torch.stack(v), torch.tensor(ok), torch.stack(bad)


def attend(q, cache, table, lens, scale, cu=None, eps=1e-12, window=0):
    """out (N, H, D) and its bounds; the keys' weights (B, Hkv, room) and theirs,
    where there is one token a sequence.  On the CPU, in fp64."""
    dt = q.dtype
    q, table, lens = q.detach().cpu().double(), table.cpu(), lens.cpu()
    N, H, D = q.shape
    B, Hkv, page = table.shape[0], cache[0].shape[2], cache[0].shape[1]
    room, G = table.shape[1] * page, H // Hkv

    def wide(new):  # rows of the kernel for many new tokens
        return new * G > 32 and not (N * G <= 512 and N * G <= 64 * B)

    cu = list(range(B + 1)) if cu is None else [int(x) for x in cu]
    s = torch.as_tensor(scale, dtype=torch.float64).detach().reshape(-1).cpu()
    s = s if s.numel() == H else s.repeat(H)
    o, eo = torch.zeros(N, H, D, dtype=torch.float64), torch.full((N, H, D), 1e-30, dtype=torch.float64)
    w_all, ew_all = torch.zeros(B, Hkv, room, dtype=torch.float64), torch.full((B, Hkv, room), 1e-30, dtype=torch.float64)
    parts, u = PARTS[dt], HALF_STEP[dt]
    for b in range(B):
        n, new = min(max(int(lens[b]), 0), room), cu[b + 1] - cu[b]
        k, v, ok, bad = rows(cache, table[b], n, D)
        if n == 0 or new == 0:
            continue
        i, j = n - new + torch.arange(new).view(-1, 1), torch.arange(n).view(1, -1)
        up = HALF_STEP[dt] + 3 * U32 if dt is torch.bfloat16 and wide(new) else WEIGHT[dt]
        keep = ok.view(1, -1) & (j <= i)
        if window > 0:
            keep = keep & (i - j < window)
        for h in range(H):
            g = h * Hkv // H
            kk, vv = (torch.where(bad[:, g].view(-1, 1), torch.zeros_like(x[:, g]), x[:, g]) for x in (k, v))
            x = q[cu[b] : cu[b + 1], h] * (-1.0 if s[h] < 0 else 1.0)
            r, dr = x @ kk.t(), 1.01 * parts * D * U32 * (x.abs() @ kk.abs().t())
            a, da = r.clamp(min=0.0) * keep, dr * keep
            s2 = float(s[h]) ** 2
            p, dp = s2 * a * a, s2 * (2 * a * da + da * da) + up * s2 * a * a
            z = p.sum(1, keepdim=True) + eps
            zz = torch.where(z > 0, z, torch.ones_like(z))
            w, dw = p / zz, dp / zz
            dz = dw.sum(1, keepdim=True) + (n + 16) * U32
            y, A = w @ vv, w @ vv.abs()
            e = (dw @ vv.abs() + (dz + (parts * n + 16) * U32) * A) * 1.02 + u * y.abs() * 1.02 + LEAST[dt]
            nan = (keep & bad[:, g].view(1, -1)).any(1)
            y[nan], w[nan] = math.nan, math.nan
            o[cu[b] : cu[b + 1], h], eo[cu[b] : cu[b + 1], h] = y, e
            if new == 1:
                w_all[b, g, :n] += torch.where(keep[0], w[0], torch.zeros_like(w[0]))
                ew_all[b, g, :n] += (dw + w * dz)[0] + w[0] * 8 * U32
    return (o, eo), (w_all, ew_all)


def worst(got, ref):
    """The largest |got - ref| over its bound; NaN only where the reference has it."""
    x, e = ref
    y = got.detach().double().cpu().reshape(x.shape)
    assert torch.equal(torch.isnan(x), torch.isnan(y)), "NaN elsewhere"
    fine = ~torch.isnan(x)
    return float(((y - x).abs() / e)[fine].max()) if fine.any() else 0.0


def make_cache(lens, page, Hkv, D, seed=0, extra=4, spare=0, device="cpu"):
    """A filled cache, pages in any order, tables padded with -1: (cache, table,
    lens, pages of nobody)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    total, nb = sum(need) + extra + spare, -(-D // 32)
    order = torch.randperm(total, generator=g)
    table = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at : at + n].to(torch.int32)
        at += n
    codes = [torch.randint(0, 256, (total, Hkv, page, 16 * nb), generator=g, dtype=torch.uint8).transpose(1, 2) for _ in range(2)]
    scales = [torch.randint(122, 128, (total, Hkv, page, nb), generator=g, dtype=torch.uint8).transpose(1, 2) for _ in range(2)]
    cache = tuple(t.to(device) for t in (codes[0], codes[1], scales[0], scales[1]))
    return cache, table.to(device), torch.tensor(lens, dtype=torch.int32, device=device), order[at:].to(device)

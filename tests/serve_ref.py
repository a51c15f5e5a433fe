"""Packed, paged and cache operators in 64 bits, and how far a kernel's outputs
may be from them.

The bounds follow the kernels' steps, element by element: the overlaps are fp32
sums of D exact products (|dr| <= D 2^-24 sum |q k|), a weight or a gradient's
factor is rounded once to the element type (relative ``half_step``: bf16 2^-8,
fp16 2^-11, fp32 2^-24, doubled for fp32's square), sums of n terms are fp32
sums (relative n 2^-24), and the output is rounded once."""

from __future__ import annotations

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
U32 = 2.0 ** -24
# fp16 values below 2^-14 lie 2^-24 apart, so rounding moves them by up to half
# of that whatever their size; bf16 and fp32 have no such values here.
LEAST = {torch.bfloat16: 1e-30, torch.float16: 2.0 ** -25, torch.float32: 1e-30}


def visible(nq, nk, causal, window, device="cpu"):
    lag = torch.arange(nk - nq, nk, device=device).view(-1, 1) - torch.arange(nk, device=device).view(1, -1)
    keep = torch.ones_like(lag, dtype=torch.bool)
    if causal:
        keep &= lag >= 0
    if window > 0:
        keep &= lag < window
    return keep


def head(q, k, v, s, keep, eps, dt, grad=None):
    """One head of one sequence: q (n, D), k and v (m, D), float64.  Returns the
    outputs and their bounds, by name ("out", "dq", "dk", "dv", "ds")."""
    D, m, n = q.shape[1], k.shape[0], q.shape[0]
    u = HALF_STEP[dt]
    up = u if dt != torch.float32 else 4 * u
    sg = -1.0 if s < 0 else 1.0
    r = torch.mm(q, k.t()) * sg
    dr = D * U32 * torch.mm(q.abs(), k.abs().t())
    a = r.clamp(min=0.0) * keep
    da = dr * keep
    s2 = s * s
    p, dp = s2 * a * a, s2 * (2 * a * da + da * da) + up * s2 * a * a
    if dt == torch.float16:  # fp16's smallest step, under a largest weight of at least 64^2
        dp = dp + 2.0 ** -25 / 4096 * p.amax(1, keepdim=True) if m else dp
    z = p.sum(1, keepdim=True) + eps
    zz = torch.where(z > 0, z, torch.ones_like(z))
    w, dw = p / zz, dp / zz
    dz = dw.sum(1, keepdim=True) + (m + 16) * U32  # relative error of z
    o = torch.mm(w, v)
    A = torch.mm(w, v.abs())
    eo = torch.mm(dw, v.abs()) + (dz + (m + 16) * U32) * A
    eo = eo * 1.02 + u * o.abs() * 1.02 + LEAST[dt]
    out = {"out": (o, eo)}
    if grad is None:
        return out, w, dw + w * dz
    ob = A * 0 + o.abs() + eo
    delta = (grad * o).sum(1, keepdim=True)
    edelta = (grad.abs() * eo).sum(1, keepdim=True) + 2 * D * U32 * (grad.abs() * ob).sum(1, keepdim=True)
    t = torch.mm(grad, v.t()) - delta
    et = 2 * D * U32 * (torch.mm(grad.abs(), v.abs().t()) + delta.abs()) + edelta
    f = 2 * s2 * sg * a * t / zz
    ef = 2 * s2 / zz * (da * (t.abs() + et) + a * et) + f.abs() * (up + dz + 8 * U32)
    ew = dw + w * (dz + up)
    if dt == torch.float16:
        # Half of fp16's smallest step: in p / Z, which is scaled up by 16, and
        # in the factor of dS, whose largest of a row (for dQ) or of a column
        # (for dK) is scaled to 2^14 at least.
        ew = ew + 2.0 ** -25 / 16 * keep
        top = torch.maximum(f.abs().amax(1, keepdim=True), f.abs().amax(0, keepdim=True)) if f.numel() else f
        ef = ef + 2.0 ** -25 * 2.0 ** -14 * top
    dq, dk, dv = torch.mm(f, k), torch.mm(f.t(), q), torch.mm(w.t(), grad)
    edq = torch.mm(ef, k.abs()) + (m + 16) * U32 * torch.mm(f.abs(), k.abs())
    edk = torch.mm(ef.t(), q.abs()) + (n + 16) * U32 * torch.mm(f.abs().t(), q.abs())
    edv = torch.mm(ew.t(), grad.abs()) + (n + 16) * U32 * torch.mm(w.t(), grad.abs())
    out |= {"dq": (dq, edq), "dk": (dk, edk), "dv": (dv, edv)}
    ds = 2.0 / s * (delta * eps / zz).sum() if s != 0 else torch.zeros((), dtype=torch.float64, device=q.device)
    eds = abs(2.0 / s) * ((edelta + delta.abs() * (2 * dz + 8 * U32)) * eps / zz).sum() if s != 0 else ds * 0
    out["ds"] = (ds, eds)
    return out, w, dw


def packed(q, k, v, scale, cu_q, cu_k, causal=True, eps=1e-12, window=0, grad=None, dt=None):
    """Outputs and bounds of flash_born_attention_packed, float64 on q's device."""
    dt = dt or v.dtype
    q, k, v = (x.detach().double() for x in (q, k, v))
    g = None if grad is None else grad.detach().double()
    H, Hkv = q.shape[1], k.shape[1]
    s = torch.as_tensor(scale, dtype=torch.float64).detach().reshape(-1).cpu()
    s = s if s.numel() == H else s.repeat(H)
    like = {"out": q, "dq": q, "dk": k, "dv": v}
    res = {n: (torch.zeros_like(x), torch.full_like(x, 1e-30)) for n, x in like.items() if g is not None or n == "out"}
    if g is not None:
        res["ds"] = (torch.zeros(H, dtype=torch.float64, device=q.device), torch.full((H,), 1e-30, dtype=torch.float64, device=q.device))
    u = HALF_STEP[dt]
    for a0, a1, b0, b1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        keep = visible(a1 - a0, b1 - b0, causal, window, q.device)
        for h in range(H):
            kh = h * Hkv // H
            one, _, _ = head(q[a0:a1, h], k[b0:b1, kh], v[b0:b1, kh], float(s[h]), keep, eps, dt, None if g is None else g[a0:a1, h])
            for name, (x, e) in one.items():
                rows, hh = (slice(a0, a1), h) if name in ("out", "dq") else (slice(b0, b1), kh)
                for i, y in ((0, x), (1, e)):
                    if name == "ds":
                        res[name][i][h] += y
                    elif name == "out":
                        res[name][i][rows, hh] = y
                    else:
                        res[name][i][rows, hh] += y
    for name in ("dq", "dk", "dv"):
        if name in res:  # the heads' sum and the final rounding
            x, e = res[name]
            e.mul_(1.02).add_(u * 1.02 * x.abs() + LEAST[dt])
    return res


def worst(got, ref):
    """The largest |got - ref| over its bound (at most 1 where all hold).  Where
    the exact value may lie beyond the type's largest (fp16's 65504: a row whose
    overlaps are all small has gradients that large), infinity is its rounding."""
    x, e = ref
    if x.numel() == 0:
        return 0.0
    y = got.detach().double().to(x.device).reshape(x.shape)
    assert not torch.isnan(y).any(), "not a number"
    d = torch.where((x.abs() + e > torch.finfo(got.dtype).max) & torch.isinf(y) & (y * x > 0), torch.zeros_like(x), (y - x).abs())
    return float((d / e).max())


def starts(lens):
    s = [0]
    for n in lens:
        s.append(s[-1] + n)
    return s


def gather(cache, table, n, page):
    """(n, Hkv, D) keys or values of one sequence; zeros for missing pages, and
    whether each key's page is there."""
    rows, ok = [], []
    for j in range(n):
        t = int(table[j // page])
        ok.append(0 <= t < cache.shape[0])
        rows.append(cache[t, j % page] if ok[-1] else torch.zeros_like(cache[0, 0]))
    if not rows:
        return cache.new_zeros((0, *cache.shape[2:])), torch.zeros(0, dtype=torch.bool)
    return torch.stack(rows), torch.tensor(ok)


def paged(q, k_cache, v_cache, table, lens, scale, eps=1e-12, window=0):
    """out and key weights of flash_born_attention_paged with their bounds, on the CPU."""
    dt = k_cache.dtype
    q, kc, vc, table = (x.detach().cpu() for x in (q, k_cache, v_cache, table))
    B, H, D = q.shape
    page, Hkv = kc.shape[1], kc.shape[2]
    room = table.shape[1] * page
    s = torch.as_tensor(scale, dtype=torch.float64).detach().reshape(-1).cpu()
    s = s if s.numel() == H else s.repeat(H)
    o, eo = torch.zeros((B, H, D), dtype=torch.float64), torch.full((B, H, D), 1e-30, dtype=torch.float64)
    w, ew = torch.zeros((B, Hkv, room), dtype=torch.float64), torch.full((B, Hkv, room), 1e-30, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(lens[b]), 0), room)
        k, ok = gather(kc, table[b], n, page)
        v, _ = gather(vc, table[b], n, page)
        k, v = torch.where(ok.view(-1, 1, 1), k, torch.zeros_like(k)).double(), torch.where(ok.view(-1, 1, 1), v, torch.zeros_like(v)).double()
        keep = ok.clone()
        if window > 0:
            keep[: max(0, n - window)] = False
        for h in range(H):
            kh = h * Hkv // H
            one, wh, dwh = head(q[b, h].double().view(1, -1), k[:, kh], v[:, kh], float(s[h]), keep.view(1, -1), eps, dt)
            o[b, h], eo[b, h] = one["out"][0][0], one["out"][1][0]
            w[b, kh, :n] += wh[0]
            # The key weights come from the unrounded fp32 weights.
            x32 = head(q[b, h].double().view(1, -1), k[:, kh], v[:, kh], float(s[h]), keep.view(1, -1), eps, torch.float32)
            ew[b, kh, :n] += x32[2][0] + x32[1][0] * 8 * U32
    return (o, eo), (w, ew)


def evict(weight, n, budget, recent):
    """Kept slots of one (sequence, key head), by sorting; weight: a list of n."""
    m = min(n, budget)
    tail = m if n <= budget else min(recent, m)
    old = n - tail
    rank = sorted(range(old), key=lambda j: (0 if weight[j] != weight[j] else 1, -weight[j] if weight[j] == weight[j] else 0.0, j))
    return sorted(rank[: m - tail]) + list(range(old, n))

"""The packed, paged and cache operators of Born attention: their cases, their
plain forms and their definition in 64 bits.

A model that trains on ragged batches and then serves runs them in this order:
``flash_born_attention_packed`` over prompts or documents of different lengths
with grouped heads, ``fused_qk_rope_l2_normalize_append`` to fill the pages of
its cache, ``flash_born_attention_paged`` for each new token, and
``born_cache_evict`` when a cache has to shrink.

Keys of a case: ``op``; ``H`` / ``Hkv`` query and key heads; ``D``; ``dtype``;
and by operator ``lens`` (tokens of each sequence, a text), ``past`` (keys
before a sequence's first query), ``causal``, ``window``, ``scale`` ("float" or
"heads"), ``train``, ``page`` (tokens a page), ``weigh`` (keep the keys'
accumulated weight), ``cached`` (tokens that a sequence had), ``budget`` and
``recent``.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SCALE = 8.0
EPS = 1e-12
SHARED = 0.6  # length of the rows' shared part over that of their own


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _packed(lens, H, Hkv, D, dtype="bf16", train=False, causal=True, window=0, past=0, scale="float", name=None):
    c = dict(op="packed", lens=lens, H=H, Hkv=Hkv, D=D, dtype=dtype, train=train, causal=causal, window=window,
             past=past, scale=scale)
    return dict(c, name=name) if name else c


def _paged(lens, H, Hkv, D, dtype="bf16", page=16, window=0, weigh=False, scale="float", name=None):
    c = dict(op="paged", lens=lens, H=H, Hkv=Hkv, D=D, dtype=dtype, page=page, window=window, weigh=weigh, scale=scale)
    return dict(c, name=name) if name else c


def _append(lens, H, Hkv, D, dtype="bf16", page=16, cached=0, name=None):
    c = dict(op="append", lens=lens, H=H, Hkv=Hkv, D=D, dtype=dtype, page=page, cached=cached)
    return dict(c, name=name) if name else c


def _evict(lens, Hkv, D, budget, recent, dtype="bf16", page=16, name=None):
    c = dict(op="evict", lens=lens, Hkv=Hkv, D=D, budget=budget, recent=recent, dtype=dtype, page=page)
    return dict(c, name=name) if name else c


def _ragged(rng, n, least, most):
    """n lengths, spread over their logarithm."""
    return " ".join(str(int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))) for _ in range(n))


def listed():
    rng = random.Random(1)
    return [
        # Three short prompts of a small model: latency and launches.
        _packed("100 29 131", 4, 2, 64, name="packed_prompts_3_d64"),
        # A prefill batch of ragged prompts, 16 heads over 4 key heads.
        _packed("1531 900 2048 313 1024 77 1800 1203", 16, 4, 64, name="packed_prompts_8_d64"),
        # A training step on packed documents of 16384 tokens, head dim 128.
        _packed("4096 1111 2900 3500 512 1777 1024 1464", 16, 4, 128, train=True, name="packed_train_8_d128"),
        # Fine-tuning in fp16 with a window, a padded head dim and odd lengths.
        _packed("701 1100 33 1 1290", 6, 2, 96, dtype="fp16", train=True, window=384, name="packed_train_fp16_5_d96"),
        # Training without autocast: fp32, every head its own keys.
        _packed("500 129 371", 8, 8, 64, dtype="fp32", train=True, name="packed_train_fp32_3_d64"),
        # One conversation, one new token: latency.
        _paged("1531", 16, 4, 128, name="paged_1x1531_d128"),
        # A serving batch of long ragged conversations.
        _paged(_ragged(rng, 32, 2048, 16384), 32, 8, 128, name="paged_32_long_d128"),
        # The same with the keys' weight kept for eviction, and fp16.
        _paged(_ragged(rng, 16, 512, 8192), 16, 4, 64, dtype="fp16", page=64, weigh=True, scale="heads",
               name="paged_weigh_16_d64"),
        # A decoding step's new tokens: one for each of 64 sequences.
        _append(" ".join(["1"] * 64), 16, 4, 128, cached=1000, name="append_64_tokens"),
        # A prefill's new tokens.
        _append("4096 1111 2900 3500 512 1777 1024 1464", 32, 8, 128, name="append_prompts_8"),
        # One conversation's cache halved.
        _evict("2048", 4, 64, 1024, 256, name="evict_1x2048_d64"),
        # A batch of long caches cut to 4096 tokens.
        _evict(_ragged(rng, 16, 4000, 10000), 8, 128, 4096, 1024, page=32, name="evict_16_long_d128"),
    ]


def _cost(case):
    """Rough microseconds, to keep drawn cases below the largest listed ones."""
    w = work(case)
    us = w["bytes"] / 4e6 + w["flops"] / (4e7 if case["dtype"] == "fp32" else 3e8)
    if case["op"] == "packed":  # the plain form pads every sequence to the longest
        n = _lens(case)
        pairs = len(n) * max(n) * (max(n) + case["past"])
        us = max(us, (10.0 if case["train"] else 4.0) * case["D"] * case["H"] * pairs / 3e8)
    return us


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["packed", "packed", "packed", "paged", "paged", "append", "evict"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        D = rng.choice([64, 64, 128, 128, 32, 80, 96, 256])
        Hkv = rng.choice([1, 2, 3, 4, 8])
        H = Hkv * rng.choice([1, 2, 3, 4, 8])
        page = rng.choice([8, 16, 16, 32, 64, 24])
        if op == "packed":
            top = int(math.exp(rng.uniform(math.log(32), math.log(4096))))
            lens = _ragged(rng, rng.choice([1, 2, 3, 5, 8, 13]), max(1, top // 16), top)
            kind = rng.choice(["causal", "causal", "causal", "window", "full"])
            c = _packed(lens, H, Hkv, D, dtype, train=rng.random() < 0.6, causal=kind != "full",
                        window=rng.choice([100, 256, 384, 512]) if kind == "window" else 0,
                        past=rng.choice([0, 0, 0, 17, 256]))
            c["scale"] = "float" if c["train"] else rng.choice(["float", "heads"])
        elif op == "paged":
            top = int(math.exp(rng.uniform(math.log(64), math.log(16384))))
            c = _paged(_ragged(rng, rng.choice([1, 2, 3, 7, 16, 32]), max(1, top // 16), top), H, Hkv, D, dtype, page,
                       window=rng.choice([0, 0, 0, 512]), weigh=rng.random() < 0.3, scale=rng.choice(["float", "heads"]))
        elif op == "append":
            if rng.random() < 0.5:
                lens = " ".join(["1"] * rng.choice([1, 5, 16, 33, 64, 128]))
            else:
                top = int(math.exp(rng.uniform(math.log(32), math.log(4096))))
                lens = _ragged(rng, rng.choice([1, 2, 3, 5, 8]), max(1, top // 16), top)
            c = _append(lens, H, Hkv, D, dtype, page, cached=rng.choice([0, 0, 100, 1000, 1531]))
        else:
            budget = int(math.exp(rng.uniform(math.log(64), math.log(6000))))
            c = _evict(_ragged(rng, rng.choice([1, 2, 5, 16]), max(1, budget // 2), 3 * budget), Hkv, D, budget,
                       rng.choice([0, budget // 8, budget // 4, budget]), dtype, page)
        if _cost(c) <= most:
            return c


def _lens(case):
    return [int(n) for n in case["lens"].split()]


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------
def _pairs(n, past, causal, window):
    """Visible pairs of n queries behind `past` keys."""
    if not causal and not window:
        return float(n) * (n + past)
    total = 0
    for i in range(past, past + n):
        seen = min(i + 1, window) if window else i + 1
        total += seen if causal else seen + (n + past - 1 - i)
    return float(total)


def work(case):
    item = 4 if case["dtype"] == "fp32" else 2
    n, Hkv, D = _lens(case), case["Hkv"], case["D"]
    H = case.get("H", Hkv)
    if case["op"] == "packed":
        q = sum(n) * H * D * item
        k = (sum(n) + len(n) * case["past"]) * Hkv * D * item
        flops = 4.0 * D * H * sum(_pairs(x, case["past"], case["causal"], case["window"]) for x in n)
        if case["train"]:  # q, k, v, dout in; out, dq, dk, dv out
            return {"bytes": 4.0 * q + 4.0 * k, "flops": 3.5 * flops}
        return {"bytes": 2.0 * q + 2.0 * k, "flops": flops}
    if case["op"] == "paged":
        seen = sum(min(x, case["window"]) if case["window"] else x for x in n)
        nbytes = 2.0 * seen * Hkv * D * item + 2.0 * len(n) * H * D * item
        if case["weigh"]:
            nbytes += 8.0 * seen * Hkv
        return {"bytes": nbytes, "flops": 4.0 * seen * H * D}
    if case["op"] == "append":
        rows = float(sum(n))
        return {"bytes": 2.0 * rows * (H + 2 * Hkv) * D * item + rows * D * 4.0, "flops": 6.0 * rows * (H + Hkv) * D}
    kept = sum(min(x, case["budget"]) for x in n)
    # Weights once; the kept rows of K and V, their weights and indices read and written.
    return {"bytes": Hkv * (4.0 * sum(n) + kept * (4.0 * D * item + 8.0)), "flops": 2.0 * Hkv * sum(n)}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _normal(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def _direction(Hkv, D, gen):
    """One direction for each key head, shared by its queries and keys, so that
    most overlaps are positive, as in a trained head."""
    return SHARED * math.sqrt(D) * _unit(_normal((Hkv, D), gen))


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(n):
    s = [0]
    for x in n:
        s.append(s[-1] + x)
    return s


def _scale(case, gen):
    if case["scale"] == "heads":
        return SCALE * (0.8 + 0.4 * torch.rand(case["H"], generator=gen, device="cuda"))
    return SCALE


def _pages(n, page, gen, spare=0):
    """Tables of pages that lie anywhere in the cache, -1 past a sequence's
    last one, and the number of pages in the cache."""
    need = [-(-x // page) for x in n]
    total = sum(need) + spare + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    wide = max(1, max(need))
    start = torch.tensor(_starts(need)[:-1], device="cuda").view(-1, 1)
    col = torch.arange(wide, device="cuda").view(1, -1)
    here = col < torch.tensor(need, device="cuda").view(-1, 1)
    table = torch.where(here, order[torch.clamp(start + col, max=total - 1)], -1).to(torch.int32)
    return table, order[sum(need):], total


def prepare(case, seed):
    """Unit rows for queries and keys (the layers normalise them), standard
    normal values and upstream gradients."""
    gen = torch.Generator("cuda").manual_seed(seed)
    n, Hkv, D, dt = _lens(case), case["Hkv"], case["D"], DTYPES[case["dtype"]]
    H = case.get("H", Hkv)
    st = {"case": case}
    if case["op"] == "packed":
        N, M = sum(n), sum(n) + len(n) * case["past"]
        way = _direction(Hkv, D, gen)
        q = _unit(_normal((N, H, D), gen) + way.repeat_interleave(H // Hkv, 0))
        k = _unit(_normal((M, Hkv, D), gen) + way)
        v, g = _normal((M, Hkv, D), gen), _normal((N, H, D), gen)
        st["q"], st["k"], st["v"] = (x.to(dt).requires_grad_(case["train"]) for x in (q, k, v))
        st["grad"] = g.to(dt)
        st["cu_q"] = _int32(_starts(n))
        st["cu_k"] = _int32(_starts([x + case["past"] for x in n])) if case["past"] else st["cu_q"]
        st["max_q"], st["max_k"] = max(n), max(n) + case["past"]
        st["scale"] = _scale(case, gen)
        return st
    page = case["page"]
    if case["op"] == "append":
        full = [x + case["cached"] for x in n]
        st["table"], _, total = _pages(full, page, gen)
        N, way = sum(n), _direction(Hkv, D, gen)
        st["q"] = (_normal((N, H, D), gen) + way.repeat_interleave(H // Hkv, 0)).to(dt)
        st["k"], st["v"] = (_normal((N, Hkv, D), gen) + way).to(dt), _normal((N, Hkv, D), gen).to(dt)
        st["k_cache"], st["v_cache"] = (_normal((total, page, Hkv, D), gen).to(dt) for _ in range(2))
        st["lens"], st["cu"] = _int32(full), _int32(_starts(n))
        half = D // 2
        freqs = 1.0 / (10000.0 ** (torch.arange(half, dtype=torch.float64) / half))
        ang = torch.outer(torch.arange(max(full) + 8, dtype=torch.float64), freqs)
        st["cos"], st["sin"] = ang.cos().float().cuda(), ang.sin().float().cuda()
        st["positions"] = torch.cat([torch.arange(f - x, f) for x, f in zip(n, full)]).to(torch.int32).cuda()
        return st
    spare = -(-case["budget"] // page) * len(n) if case["op"] == "evict" else 0
    st["table"], free, total = _pages(n, page, gen, spare)
    st["lens"] = _int32(n)
    way = _direction(Hkv, D, gen)
    st["k_cache"] = _unit(_normal((total, page, Hkv, D), gen) + way).to(dt)
    st["v_cache"] = _normal((total, page, Hkv, D), gen).to(dt)
    if case["op"] == "paged":
        st["q"] = _unit(_normal((len(n), H, D), gen) + way.repeat_interleave(H // Hkv, 0)).to(dt)
        st["scale"] = _scale(case, gen)
        if case["weigh"]:
            st["weight"] = torch.rand((len(n), Hkv, max(n)), generator=gen, device="cuda").square()
        return st
    # Accumulated weights: a long tail, and keys that no query ever weighed.
    w = _normal((len(n), Hkv, max(n)), gen)
    st["weight"] = torch.where(w > 0.5, torch.zeros_like(w), (2.0 * w).exp())
    st["to"] = free[:spare].view(len(n), -1).contiguous()
    return st


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    return {"packed": _run_packed, "paged": _run_paged, "append": _run_append, "evict": _run_evict}[state["case"]["op"]](state)


def _run_packed(st):
    case = st["case"]
    if own:
        from quantumdlblocks_amd import flash_born_attention_packed

        kw = dict(cu_seqlens_k=st["cu_k"], is_causal=case["causal"], eps=EPS, window_size=case["window"])
        if not case["train"]:
            with torch.no_grad():
                return {"out": flash_born_attention_packed(st["q"], st["k"], st["v"], st["scale"], st["cu_q"], **kw)}
        out = flash_born_attention_packed(st["q"], st["k"], st["v"], st["scale"], st["cu_q"], **kw)
        dq, dk, dv = torch.autograd.grad(out, [st["q"], st["k"], st["v"]], st["grad"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        return _plain_packed(st, case)


def _pad(x, cu, longest, groups):
    """(N, h, D) -> (S, h / groups, groups * longest, D), fp32, zeros behind each sequence."""
    at = torch.arange(longest, device=x.device)
    n = (cu[1:] - cu[:-1]).long()
    idx = cu[:-1].long().view(-1, 1) + at
    y = x.detach().float()[torch.clamp(idx, max=x.shape[0] - 1)] * (at < n.view(-1, 1)).view(len(n), -1, 1, 1)
    S, T, h, D = y.shape
    return y.view(S, T, h // groups, groups, D).permute(0, 2, 3, 1, 4).reshape(S, h // groups, groups * T, D)


def _unpad(y, cu, N, groups):
    """The way back."""
    S, h, GT, D = y.shape
    y = y.view(S, h * groups, GT // groups, D)
    t = torch.arange(N, device=y.device)
    s = torch.searchsorted(cu.long(), t, right=True) - 1
    return y[s, :, t - cu.long()[s]]


def _plain_packed(st, case):
    G, Tq, Tk = case["H"] // case["Hkv"], st["max_q"], st["max_k"]
    cq, ck = st["cu_q"], st["cu_k"]
    q, g = (_pad(x, cq, Tq, G) for x in (st["q"], st["grad"]))
    k, v = (_pad(x, ck, Tk, 1) for x in (st["k"], st["v"]))
    S, h = q.shape[:2]
    s = torch.as_tensor(st["scale"], device="cuda").float().reshape(-1)
    s = s.expand(case["H"]).view(1, h, G, 1, 1).expand(1, h, G, Tq, 1).reshape(1, h, G * Tq, 1)
    nq, nk = (cq[1:] - cq[:-1]).view(-1, 1, 1), (ck[1:] - ck[:-1]).view(-1, 1, 1)
    i = torch.arange(Tq, device="cuda").view(1, -1, 1) + (nk - nq)
    j = torch.arange(Tk, device="cuda").view(1, 1, -1)
    keep = j < nk
    if case["causal"]:
        keep = keep & (j <= i)
    if case["window"]:
        keep = keep & (i - j < case["window"])
    a = (q @ k.transpose(-1, -2)).mul_(s).relu_()
    a.view(S, h, G, Tq, Tk).mul_(keep[:, None, None])
    w = a.square()
    z = w.sum(-1, keepdim=True) + EPS
    w.div_(z)
    o = w @ v
    dt = st["q"].dtype
    out = _unpad(o, cq, st["q"].shape[0], G).to(dt)
    if not case["train"]:
        return {"out": out}
    dv = w.transpose(-1, -2) @ g
    ds = g @ v.transpose(-1, -2)
    ds.sub_((g * o).sum(-1, keepdim=True)).mul_(a).mul_(2.0 * s / z)
    dq, dk = ds @ k, ds.transpose(-1, -2) @ q
    N, M = st["q"].shape[0], st["k"].shape[0]
    return {"out": out, "dq": _unpad(dq, cq, N, G).to(dt), "dk": _unpad(dk, ck, M, 1).to(dt),
            "dv": _unpad(dv, ck, M, 1).to(dt)}


def _run_paged(st):
    case = st["case"]
    weight = st["weight"].clone() if case["weigh"] else None  # a step goes on from the state's weights
    if own:
        from quantumdlblocks_amd import flash_born_attention_paged

        out = flash_born_attention_paged(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lens"], st["scale"],
                                         eps=EPS, window_size=case["window"], key_weight=weight)
        return {"out": out, "weight": weight} if case["weigh"] else {"out": out}
    B, H, D = st["q"].shape
    Hkv = case["Hkv"]
    G = H // Hkv
    page = st["table"].clamp(min=0).long()
    k = st["k_cache"][page].flatten(1, 2).float().permute(0, 2, 1, 3)  # (B, Hkv, L, D)
    v = st["v_cache"][page].flatten(1, 2).float().permute(0, 2, 1, 3)
    s = torch.as_tensor(st["scale"], device="cuda").float().reshape(-1).expand(H).view(1, Hkv, G, 1)
    j = torch.arange(k.shape[2], device="cuda").view(1, 1, 1, -1)
    n = st["lens"].view(-1, 1, 1, 1)
    keep = j < n
    if case["window"]:
        keep = keep & (j >= n - case["window"])
    r = st["q"].float().view(B, Hkv, G, D) @ k.transpose(-1, -2)
    p = (r * s).relu_().square_() * keep
    w = p / (p.sum(-1, keepdim=True) + EPS)
    out = (w @ v).view(B, H, D).to(st["q"].dtype)
    if not case["weigh"]:
        return {"out": out}
    weight += w.sum(2)[..., : weight.shape[-1]]
    return {"out": out, "weight": weight}


def _run_append(st):
    if own:
        from quantumdlblocks_amd import fused_qk_rope_l2_normalize_append

        q = fused_qk_rope_l2_normalize_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["k_cache"], st["v_cache"],
                                              st["table"], st["lens"], cu_seqlens=st["cu"], positions=st["positions"], eps=EPS)
        return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    cos, sin = (t[st["positions"].long()].unsqueeze(1) for t in (st["cos"], st["sin"]))

    def turned(x):
        x1, x2 = x.float().chunk(2, dim=-1)
        y = torch.cat([x1 * cos - x2 * sin, x1 * sin + x2 * cos], dim=-1)
        return (y * (y.square().sum(-1, keepdim=True) + EPS).rsqrt()).to(x.dtype)

    page = st["k_cache"].shape[1]
    t = torch.arange(st["q"].shape[0], device="cuda")
    cu = st["cu"].long()
    s = torch.searchsorted(cu, t, right=True) - 1
    at = st["lens"].long()[s] - cu[s + 1] + t
    where = (st["table"].long()[s, at // page], at % page)
    st["k_cache"][where] = turned(st["k"])
    st["v_cache"][where] = st["v"]
    return {"q": turned(st["q"]), "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _run_evict(st):
    case = st["case"]
    budget, recent, page = case["budget"], case["recent"], case["page"]
    if own:
        from quantumdlblocks_amd import born_cache_evict

        lens, weight, kept = born_cache_evict(st["k_cache"], st["v_cache"], st["table"], st["lens"], st["weight"], budget,
                                              recent, out_block_table=st["to"])
        return {"lens": lens, "weight": weight, "kept": kept, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    B, Hkv, L = st["weight"].shape
    n = st["lens"].long().view(-1, 1, 1)
    j = torch.arange(L, device="cuda").view(1, 1, -1)
    top = torch.finfo(torch.float32).max
    # The recent ones first, then by weight.
    w = torch.where(j >= n - min(recent, budget), top, st["weight"].clamp(max=top / 2))
    w = torch.where(j < n, w, -1.0)
    width = min(budget, L)
    best = w.sort(dim=-1, descending=True, stable=True).indices[..., :width]
    lens = n.clamp(max=budget)
    here = torch.arange(width, device="cuda").view(1, 1, -1) < lens
    kept = torch.where(here, best, L).sort(dim=-1).values
    weight = torch.zeros_like(st["weight"])
    at = kept.clamp(max=L - 1)
    weight[..., :width] = st["weight"].gather(-1, at) * here
    b, h, i = torch.nonzero(here.expand(B, Hkv, width), as_tuple=True)
    src = at[b, h, i]
    frm = (st["table"].long()[b, src // page], src % page, h)
    to = (st["to"].long()[b, i // page], i % page, h)
    st["k_cache"][to] = st["k_cache"][frm]
    st["v_cache"][to] = st["v_cache"][frm]
    whole = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device="cuda")
    whole[..., :width] = torch.where(here, kept, -1)
    return {"lens": lens.view(-1).to(torch.int32), "weight": weight, "kept": whole, "k_cache": st["k_cache"],
            "v_cache": st["v_cache"]}


# ---------------------------------------------------------------------------
# The definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"packed": _exact_packed, "paged": _exact_paged, "append": _exact_append, "evict": _exact_evict}[case["op"]](st, case)


def _head_scales(st, H):
    s = torch.as_tensor(st["scale"], device="cuda", dtype=torch.float64).reshape(-1)
    return s if s.numel() == H else s.repeat(H)


def _exact_packed(st, case):
    n, past, H, G = _lens(case), case["past"], case["H"], case["H"] // case["Hkv"]
    q, k, v, g = (x.detach().double() for x in (st["q"], st["k"], st["v"], st["grad"]))
    scales = _head_scales(st, H)
    o = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    a0 = b0 = 0
    for x in n:
        a1, b1 = a0 + x, b0 + x + past
        lag = torch.arange(past, past + x, device="cuda").unsqueeze(1) - torch.arange(past + x, device="cuda").unsqueeze(0)
        seen = torch.ones_like(lag, dtype=torch.bool)
        if case["causal"]:
            seen &= lag >= 0
        if case["window"]:
            seen &= lag < case["window"]
        for h in range(H):
            qs, ks, vs = q[a0:a1, h], k[b0:b1, h // G], v[b0:b1, h // G]
            amp = torch.clamp(scales[h] * torch.mm(qs, ks.t()), min=0.0) * seen
            p = amp * amp
            z = p.sum(1, keepdim=True) + EPS
            os_ = torch.mm(p, vs) / z
            o[a0:a1, h] = os_
            if case["train"]:
                gs = g[a0:a1, h]
                dv[b0:b1, h // G] += torch.mm((p / z).t(), gs)
                dr = 2.0 * scales[h] * amp * (torch.mm(gs, vs.t()) - (gs * os_).sum(1, keepdim=True)) / z
                dq[a0:a1, h] = torch.mm(dr, ks)
                dk[b0:b1, h // G] += torch.mm(dr.t(), qs)
        a0, b0 = a1, b1
    return {"out": o, "dq": dq, "dk": dk, "dv": dv} if case["train"] else {"out": o}


def _exact_paged(st, case):
    H, G = case["H"], case["H"] // case["Hkv"]
    scales = _head_scales(st, H).view(-1, 1, G)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    weight = st["weight"].double() if case["weigh"] else None
    for b, n in enumerate(_lens(case)):
        pages = st["table"][b, : -(-n // case["page"])].long()
        first = max(0, n - case["window"]) if case["window"] else 0
        k, v = (c[pages].flatten(0, 1)[first:n].double() for c in (st["k_cache"], st["v_cache"]))
        q = st["q"][b].double().view(-1, G, case["D"])
        amp = torch.clamp(torch.bmm(k.transpose(0, 1), q.transpose(1, 2).contiguous()) * scales, min=0.0)  # (Hkv, n, G)
        p = amp * amp
        w = p / (p.sum(1, keepdim=True) + EPS)
        out[b] = torch.bmm(w.transpose(1, 2), v.transpose(0, 1).contiguous()).reshape(H, -1)
        if case["weigh"]:
            weight[b, :, first:n] += w.sum(2)
    return {"out": out, "weight": weight} if case["weigh"] else {"out": out}


def _exact_append(st, case):
    n, page = _lens(case), case["page"]
    half = case["D"] // 2
    c, s = (t.double()[st["positions"].long()].view(-1, 1, half) for t in (st["cos"], st["sin"]))

    def rows(x):
        x = x.double()
        z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(c, s)
        y = torch.cat([z.real, z.imag], -1)
        return y / torch.sqrt((y * y).sum(-1, keepdim=True) + EPS)

    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    k, t = rows(st["k"]), 0
    for b, x in enumerate(n):
        at = torch.arange(case["cached"], case["cached"] + x, device="cuda")
        pages = st["table"][b].long()[at // page]
        kc[pages, at % page] = k[t : t + x]
        vc[pages, at % page] = st["v"][t : t + x].double()
        t += x
    return {"q": rows(st["q"]), "k_cache": kc, "v_cache": vc}


def _exact_evict(st, case):
    page, budget, recent = case["page"], case["budget"], case["recent"]
    n = _lens(case)
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    weight = torch.zeros_like(st["weight"], dtype=torch.float64)
    all_w = st["weight"].double().cpu().numpy()
    table, to = st["table"].long(), st["to"].long()
    for b, x in enumerate(n):
        m = min(x, budget)
        tail = min(recent, m)
        i = torch.arange(m, device="cuda")
        for h in range(case["Hkv"]):
            if x <= budget:
                kept = list(range(x))
            else:
                old = all_w[b, h, : x - tail]
                kept = sorted((-old).argsort(kind="stable")[: m - tail].tolist()) + list(range(x - tail, x))
            src = torch.tensor(kept, dtype=torch.long, device="cuda")
            weight[b, h, :m] = st["weight"][b, h, src].double()
            frm, dst = table[b][src // page], to[b][i // page]
            kc[dst, i % page, h] = st["k_cache"][frm, src % page, h].double()
            vc[dst, i % page, h] = st["v_cache"][frm, src % page, h].double()
    return {"lens": None, "weight": weight, "kept": None, "k_cache": kc, "v_cache": vc}

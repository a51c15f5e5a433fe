"""Flash-Born attention over packed sequences with grouped heads, forward and
backward: the ragged form of ``flash_born_attention``.

Several sequences of different lengths share rows of tokens, ``q`` (N, H, D) and
``k``, ``v`` (M, Hkv, D) with ``H`` a multiple of ``Hkv``: sequence s owns query
rows ``cu_seqlens_q[s] : cu_seqlens_q[s + 1]`` and key rows likewise, and query
head h reads key head ``h // (H // Hkv)``.  Per sequence, with len_q queries
standing at the last len_q of len_k positions,

    a_ij = max(0, scale_h * q_i . k_j) * M_ij,   p_ij = a_ij ** 2
    O_i  = sum_j p_ij v_j / (sum_j p_ij + eps)
    M_ij = [causal => j <= i + len_k - len_q]
           & [window_size > 0 => i + len_k - len_q - j < window_size]

Rows that see no key are zero, and so are their gradients; so are rows whose
(sum_j p_ij + eps) / scale_h^2 lies below fp32's normal range, 2^-126.

GPU tensors with head dim <= 256 run the HIP kernels; CPU tensors and larger
head dims the formulation in torch operations.
"""

from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from .. import _native
from .flash_born import _DTYPE_CODE, MAX_HEAD_DIM, _aligned, _apply, _autocast_dtype, _pad_head, _parameter, _run_call

__all__ = ["flash_born_attention_packed"]

_LIMIT = 1 << 30  # positions, windows


def _token_rows(t: torch.Tensor, dtype: torch.dtype, dp: int):
    """``t`` (N, heads, D) in ``dtype``, zero-padded to ``dp`` columns, and its
    (token, head) strides, read in place where the kernels can: unit stride
    along D, 16-byte pieces, tokens that do not overlap."""
    if t.dtype is not dtype:
        t = t.to(dtype)
    n, h, d = t.shape
    if d != dp:
        t = _pad_head(t, dp)
    st, sh, sd = t.stride()
    if n <= 1:
        st = h * dp
    if h <= 1:
        sh = 0
    pieces = 4 if dtype is torch.float32 else 8  # elements of 16 bytes
    if sd != 1 or st % pieces or sh % pieces or st < dp or st >= pieces << 20 or t.data_ptr() % 16:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        st, sh = h * dp, dp
    return t, st, sh


def _whole(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """``t`` in ``dtype``, contiguous and 16-byte aligned: itself where it is."""
    if t.dtype is dtype and t.is_contiguous() and not t.data_ptr() % 16:
        return t
    return _aligned(t.to(dtype))


def _int32(t: torch.Tensor) -> torch.Tensor:
    """int32, values outside its range cut to it: what lies outside the tensors stays outside."""
    return t if t.dtype is torch.int32 else t.clamp(-(1 << 31), (1 << 31) - 1).to(torch.int32)


def _starts(cu: torch.Tensor, device: torch.device) -> torch.Tensor:
    cu = _int32(cu)
    if cu.device != device:
        cu = cu.to(device)
    return cu if cu.is_contiguous() else cu.contiguous()


def _bad_starts(name, cu):
    return ValueError(f"{name} must be a 1-D int32 or int64 tensor of sequences + 1 starts, got {cu.dtype} {tuple(cu.shape)}")


def _check(q, k, v, n_scale, cu_q, cu_k):
    qs, ks = q.shape, k.shape
    if len(qs) != 3:
        raise ValueError(f"q must be (tokens, heads, head_dim), got shape {tuple(qs)}")
    if len(ks) != 3 or ks != v.shape or ks[2] != qs[2]:
        raise ValueError(f"k and v must share one (tokens, key_heads, head_dim) shape with q's head_dim, got "
                         f"{tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    H, Hkv = qs[1], ks[1]
    if Hkv < 1 or H < 1 or H % Hkv or qs[2] < 1:
        raise ValueError(f"the {H} query heads must be a multiple of the {Hkv} key heads, and head_dim positive")
    if n_scale != 1 and n_scale != H:
        raise ValueError(f"scale must hold 1 value or H={H} per-head values, got {n_scale}")
    if cu_q.dim() != 1 or cu_q.shape[0] < 1 or cu_q.dtype not in (torch.int32, torch.int64):
        raise _bad_starts("cu_seqlens_q", cu_q)
    if cu_k is not cu_q:
        if cu_k.dim() != 1 or cu_k.shape[0] < 1 or cu_k.dtype not in (torch.int32, torch.int64):
            raise _bad_starts("cu_seqlens_k", cu_k)
        if cu_q.shape[0] != cu_k.shape[0]:
            raise ValueError(f"cu_seqlens_q and cu_seqlens_k name {cu_q.shape[0] - 1} and {cu_k.shape[0] - 1} sequences")
    at = q.get_device()
    if k.get_device() != at or v.get_device() != at:
        raise ValueError(f"q, k, v must be on one device, got {q.device}, {k.device}, {v.device}")


def _forward(q, k, v, scale, cu_q, cu_k, is_causal, eps, window, train):
    """The call: (output, its sizes, what the backward needs).  The argument
    block holds addresses: the tensors stay here until the call."""
    lib = _native.load()
    target = _autocast_dtype(q) or v.dtype
    if target not in _DTYPE_CODE:
        raise TypeError(f"flash_born_attention_packed: unsupported dtype {target}")
    dev = q.device
    scale_flat, scale_p, n_scale, scale_value = _parameter(scale, dev)
    N, H, D = q.shape
    M, Hkv, _ = k.shape
    dp = (D + 7) // 8 * 8
    q_c, q0, q1 = _token_rows(q, target, dp)
    k_c, k0, k1 = _token_rows(k, target, dp)
    v_c, v0, v1 = _token_rows(v, target, dp)
    cs_q = _starts(cu_q, dev)
    cs_k = cs_q if cu_k is cu_q else _starts(cu_k, dev)
    out = q_c.new_empty((N, H, dp))
    z = torch.empty((H, N), dtype=torch.float32, device=dev) if train else None
    sizes = (_DTYPE_CODE[target], cs_q.shape[0] - 1, N, M, H, Hkv, dp)
    _run_call(lib.qdl_flash_born_packed_forward_call, "qdl_flash_born_packed_forward_call", dev, _native.packed_call(
        *sizes, q_c.data_ptr(), k_c.data_ptr(), v_c.data_ptr(), q0, q1, k0, k1, v0, v1, out.data_ptr(), z.data_ptr() if train else 0,
        cs_q.data_ptr(), cs_k.data_ptr(), scale_p, n_scale, scale_value, 1 if is_causal else 0, window, eps, 0, 0, 0, 0, 0, 0, 0, 0, 0))
    return (out if dp == D else out[..., :D].contiguous(), sizes,
            (q_c, k_c, v_c, out, z, scale_flat, cs_q, None if cs_k is cs_q else cs_k))


@torch.compiler.disable
def _call_uncompiled(fn, args):
    return fn(*args)


def _uncompiled(fn, *args):
    return _call_uncompiled(fn, args) if torch.compiler.is_compiling() else fn(*args)


@functools.lru_cache(maxsize=256)
def _workspace(dtype, sequences, N, M, H, Hkv, dp, window) -> int:
    """Bytes of the backward's workspace, by sizes alone (the block's addresses and strides are not looked at)."""
    piece = 16
    block = _native.packed_call(dtype, sequences, N, M, H, Hkv, dp, piece, piece, piece, H * dp, dp, Hkv * dp, dp, Hkv * dp, dp, piece,
                                piece, piece, piece, 0, 1, 1.0, 1, window, 0.0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    return int(_native.load().qdl_flash_born_packed_workspace_size(block))


def _is_dual(*values) -> bool:
    """Whether a forward-mode derivative runs through any of them.  Outside of a
    dual level (forward_ad._current_level < 0) there are none."""
    return any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in values)


class _OnlyOnce(torch.autograd.Function):
    """A gradient of a recorded backward (``create_graph``): the kernels have no
    second derivative, so to differentiate it again is an error, not a zero."""

    @staticmethod
    def forward(ctx, grad, anchor):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError("flash_born_attention_packed has no second derivative on the GPU")


class _FlashBornPackedFn(torch.autograd.Function):
    """forward: computes in the autocast dtype (CUDA autocast active) else
    ``v.dtype``; saves the rows, ``out``, Z (fp32) and the starts.  backward:
    dq, dk, dv in the inputs' dtypes, dscale in the scale's shape and dtype.

    The context holds no address and no stride: a saved tensor's hook
    (checkpoints, offloading) gives the backward other tensors than these."""

    @staticmethod
    def forward(ctx, q, k, v, scale, cu_q, cu_k, is_causal, eps, window):
        out, sizes, saved = _forward(q, k, v, scale, cu_q, cu_k, is_causal, eps, window, True)
        ctx.sizes, ctx.dtype = sizes, saved[3].dtype
        ctx.modes = 1 if is_causal else 0, window, eps
        ctx.scale_value = 0.0 if isinstance(scale, torch.Tensor) else float(scale)
        ctx.save_for_backward(*saved)
        ctx.head_dim = q.shape[2]
        if isinstance(scale, torch.Tensor):
            ctx.scale_shape, ctx.scale_dtype = scale.shape, scale.dtype
        ctx.dtypes = (q.dtype, k.dtype, v.dtype)
        return out

    @staticmethod
    def backward(ctx, do):
        lib = _native.load()
        q, k, v, out, z, scale_flat, cu_q, cu_k = ctx.saved_tensors
        sizes, dt, dev = ctx.sizes, ctx.dtype, do.device
        if q.device != dev or k.device != dev or v.device != dev or out.device != dev or z.device != dev:
            q, k, v, out, z = (t.to(dev) for t in (q, k, v, out, z))  # a hook left them elsewhere
        _, _, N, M, H, Hkv, dp = sizes
        D = ctx.head_dim
        q, q0, q1 = _token_rows(q, dt, dp)
        k, k0, k1 = _token_rows(k, dt, dp)
        v, v0, v1 = _token_rows(v, dt, dp)
        do, d0, d1 = _token_rows(do, dt, dp)
        out, z, cu_q = _whole(out, dt), _whole(z, torch.float32), _starts(cu_q, dev)
        cu_k = cu_q if cu_k is None else _starts(cu_k, dev)
        scale_p, n_scale = 0, 1
        if scale_flat is not None:
            scale_flat, scale_p, n_scale, _ = _parameter(scale_flat, dev)
        _, want_k, want_v, want_scale = ctx.needs_input_grad[:4]
        dq = out.new_empty((N, H, dp))
        # dK and dV come together, and not at all where neither is wanted.
        dk = dv = None
        if want_k or want_v:
            dk, dv = out.new_empty((M, Hkv, dp)), out.new_empty((M, Hkv, dp))
        # The scale's gradient costs launches of its own: only where wanted.
        dscale = z.new_empty(n_scale) if want_scale else None
        size = _workspace(*sizes, ctx.modes[1])
        ws = z.new_empty((size + 15) // 16 * 4)
        _run_call(lib.qdl_flash_born_packed_backward_call, "qdl_flash_born_packed_backward_call", dev, _native.packed_call(
            *sizes, q.data_ptr(), k.data_ptr(), v.data_ptr(), q0, q1, k0, k1, v0, v1, out.data_ptr(), z.data_ptr(),
            cu_q.data_ptr(), cu_k.data_ptr(), scale_p, n_scale, ctx.scale_value, *ctx.modes, do.data_ptr(), d0, d1, dq.data_ptr(),
            0 if dk is None else dk.data_ptr(), 0 if dv is None else dv.data_ptr(), 0 if dscale is None else dscale.data_ptr(),
            ws.data_ptr(), size))
        grads, again = [], torch.is_grad_enabled()
        for g, want in zip((dq, dk, dv), ctx.dtypes):
            if g is not None:
                if dp != D:
                    g = g[..., :D]
                if g.dtype is not want:
                    g = g.to(want)
            grads.append(g)
        grads.append(None if dscale is None else dscale.view(ctx.scale_shape).to(ctx.scale_dtype))
        if again:
            anchor = torch.empty(0, requires_grad=True)
            grads = [None if g is None else _OnlyOnce.apply(g, anchor) for g in grads]
        return (*grads, None, None, None, None, None)


def _on_gpu(q, k, v, scale, *rest):
    """Through the autograd function where a derivative is recorded; it refuses a forward-mode one."""
    recorded = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                            or (isinstance(scale, torch.Tensor) and scale.requires_grad))
    if recorded or (forward_ad._current_level >= 0 and _is_dual(q, k, v, scale)):
        return _apply(_FlashBornPackedFn, q, k, v, scale, *rest)
    return _uncompiled(_forward, q, k, v, scale, *rest, False)[0]


def _eager_packed(q, k, v, scale_t, cu_q, cu_k, is_causal, eps, window, target):
    """The formulas in torch operations, in fp32 (fp64 for fp64 values) under
    autocast too, one sequence at a time; the output in ``target``."""
    with torch.autocast(q.device.type, enabled=False):  # not as a decorator, which is one object for all threads
        return _packed_formula(q, k, v, scale_t, cu_q, cu_k, is_causal, eps, window).to(target)


def _packed_formula(q, k, v, scale_t, cu_q, cu_k, is_causal, eps, window):
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for name, c, n in (("cu_seqlens_q", cq, q.shape[0]), ("cu_seqlens_k", ck, k.shape[0])):
        if c[0] != 0 or c[-1] > n or any(a > b for a, b in zip(c, c[1:])):
            raise ValueError(f"{name} must start at 0, never decrease and end within the {n} rows, got {c}")
    H, Hkv = q.shape[1], k.shape[1]
    G = H // Hkv
    wide = torch.float64 if v.dtype == torch.float64 else torch.float32
    s = scale_t.to(device=q.device, dtype=wide).reshape(-1).expand(H).view(Hkv, G, 1, 1)
    outs = []
    if len(cq) == 1:  # no sequences: an empty one, for the gradients
        cq, ck = cq * 2, ck * 2
    for a0, a1, b0, b1 in zip(cq, cq[1:], ck, ck[1:]):
        nq, nk = a1 - a0, b1 - b0
        qs = q[a0:a1].to(wide).view(nq, Hkv, G, q.shape[2]).permute(1, 2, 0, 3)
        ks, vs = (x[b0:b1].to(wide).permute(1, 0, 2).unsqueeze(1) for x in (k, v))
        lag = (torch.arange(nq, device=q.device) + nk - nq).view(-1, 1) - torch.arange(nk, device=q.device).view(1, -1)
        keep = torch.ones_like(lag, dtype=torch.bool)
        if is_causal:
            keep = keep & (lag >= 0)
        if window > 0:
            keep = keep & (lag < window)
        r = torch.matmul(qs, ks.transpose(-1, -2)) * s
        p = torch.relu(torch.where(keep, r, torch.zeros_like(r))).square()
        den = p.sum(-1, keepdim=True) + eps
        # Rows without weight are zero, with eps == 0 too.
        w = p / torch.where(den > 0, den, torch.ones_like(den))
        outs.append(torch.matmul(w, vs).permute(2, 0, 1, 3).reshape(nq, H, q.shape[2]))
    outs.append(torch.zeros((q.shape[0] - cq[-1], H, v.shape[2]), dtype=wide, device=q.device))
    return torch.cat(outs)


def flash_born_attention_packed(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    scale: float | torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor | None = None,
    is_causal: bool = True,
    eps: float = 1e-12,
    window_size: int = 0,
) -> torch.Tensor:
    """Born attention over packed sequences; returns (N, H, D) in the compute dtype.

    ``q`` (N, H, D), ``k`` and ``v`` (M, Hkv, D): rows of tokens, any strides
    with unit stride along D are read in place.  ``scale``: a float or a tensor
    of 1 or H values.  ``cu_seqlens_q``, ``cu_seqlens_k`` (default: the
    queries'): the sequences' S + 1 starts, int32 (int64 is converted), the
    first 0, never decreasing, the last at most the rows; they stay on the
    device, so on the GPU values that break this are not reported: such calls
    read and write nothing outside the tensors, and their outputs are undefined.
    Rows behind the last sequence come out as zeros.  ``is_causal`` and
    ``window_size`` count positions from the sequences' ends: fewer queries than
    keys are the last ones (a prompt's next part behind its cache).
    Differentiable in q, k, v and scale (on the GPU once, and not forward-mode);
    the sums over a group's heads are taken in a fixed order.  An infinity or NaN
    in v may reach rows of its sequence that do not see it, as 0 times that does
    in the formula; one in k does not reach their outputs.  In 16 bits the
    weights and the gradients' factors are rounded for the products that take
    them: dq and dk are about 1.9 and 1.5 times as far from exact gradients as
    those rounded to 16 bits are (in norm bf16 3e-3, fp16 4e-4), seldom more (5.8
    and 4.4 times, 8.7e-3, the worst of 1228 drawn batches: short sequences, some
    of whose rows one key takes nearly whole with a small overlap); fp32 rounds
    nothing on the way.
    """
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    n_scale = scale.numel() if isinstance(scale, torch.Tensor) else 1
    _check(q, k, v, n_scale, cu_seqlens_q, cu_seqlens_k)
    window = min(max(int(window_size), 0), _LIMIT)
    if not float(eps) >= 0.0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    if q.is_cuda and q.shape[2] <= MAX_HEAD_DIM:
        return _on_gpu(q, k, v, scale, cu_seqlens_q, cu_seqlens_k, bool(is_causal), float(eps), window)
    scale_t = scale if isinstance(scale, torch.Tensor) else torch.tensor(float(scale), dtype=torch.float64)
    target = _autocast_dtype(q) or v.dtype
    return _eager_packed(q, k, v, scale_t, cu_seqlens_q, cu_seqlens_k, bool(is_causal), float(eps), window, target)

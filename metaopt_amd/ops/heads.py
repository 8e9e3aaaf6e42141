"""Attention-head operators of the population LM beyond :mod:`.lm`'s plain causal attention: query /
key head norms with the position rotation in the same pass, and attention with a sliding window and
sink tokens, grouped heads, padded batches and queries at an offset in a cache -- HIP kernels
(csrc/lm_qknorm.hip, csrc/lm_window.hip) behind autograd Functions, with PyTorch references of the
same math (the CPU backend).

Layouts are :mod:`.lm`'s: rows ``[R, .]`` ordered (trial, sequence, position), heads
``[B', heads, T, D]``, per-trial parameters ``[P, .]``.  The kernels take bf16 and fp16 and head
dimensions 64 and 128; other calls on a GPU are refused.
"""
from __future__ import annotations

import ctypes
import math
from functools import reduce
from operator import or_
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .lm import _hip

c_void_p, c_int, c_float, c_int64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64

_lib.register_signatures({
    "mopt_qk_norm_rope_fwd": ([c_void_p, c_int64] + [c_void_p] * 9 + [c_int] * 8 +
                              [c_float, c_int, c_int, c_void_p], c_int),
    "mopt_qk_norm_rope_bwd": ([c_void_p, c_int64] + [c_void_p] * 11 + [c_int] * 7 +
                              [c_float, c_int, c_int, c_void_p], c_int),
    "mopt_window_fwd": ([c_void_p] * 6 + [c_int] + [c_void_p] * 3 + [c_int] * 8 +
                        [c_float, c_int, c_void_p], c_int),
    "mopt_window_step": ([c_void_p] * 6 + [c_int] + [c_void_p] * 2 + [c_int] * 9 +
                         [c_float, c_int, c_void_p], c_int),
    "mopt_window_bwd": ([c_void_p] * 6 + [c_int] + [c_void_p] * 9 + [c_int] * 11 +
                        [c_float, c_int, c_void_p], c_int),
})

_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_Strides6, _Strides9 = c_int64 * 6, c_int64 * 9
#: longest sequence and cache of :func:`window_attention`
MAX_LENGTH = 1 << 29


def _call(t: torch.Tensor, name: str, *args) -> None:
    """Launch on the current stream of ``t``'s device, whichever device is current."""
    fn = getattr(_lib.get_lib(), name)
    index = t.get_device()
    if index != torch.cuda.current_device():
        with torch.cuda.device(index):
            rc = fn(*args, _lib.stream_ptr(t.device))
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc or _lib.SYNC_CHECK:
        _lib.check(rc, name)


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """``t`` with contiguous 16-byte aligned rows (a copy only where it has none)."""
    s = t.stride()
    if s[-1] != 1 or t.data_ptr() % 16 or reduce(or_, s[:-1]) % 8 or \
            s[-2] >= 1 << 24:                  # (a tile's 64 rows are reached by 32-bit offsets)
        return t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def _needs_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def _no_tangents(what: str, *tensors) -> None:
    """The kernels carry no forward-mode derivatives.  (A dual tensor need not require a gradient:
    its tangent would be lost without a word.)"""
    if getattr(forward_ad, "_current_level", 0) < 0:       # out of dual_level(): the cheap way out
        return
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what} on a GPU has no forward-mode derivatives")


def _same(t: torch.Tensor, names: str, *others) -> None:
    index = t.get_device()                       # (-1: the CPU)
    for i, o in enumerate(others):
        if o.get_device() != index:
            raise ValueError(f"{names.split()[i]} is on {o.device}, the input on {t.device}")


def _once(backward):
    """``once_differentiable`` at the price of one test where no graph of the backward is asked for."""
    strict = torch.autograd.function.once_differentiable(backward)

    def call(ctx, *grads):
        return strict(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return staticmethod(call)


def _int32(name: str, t: torch.Tensor, n: int) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of {n} values, one a sequence")


# ============================================================================ qk norm + rotation
def rope_tables(T: int, dim: int = 64, base: float = 10000.0, device=None):
    """(cos, sin) float32 [T, dim / 2] of the angles ``t base^(-2 j / dim)``."""
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    ang = torch.arange(T, dtype=torch.float64)[:, None] * inv[None, :]
    return (torch.cos(ang).float().contiguous().to(device),
            torch.sin(ang).float().contiguous().to(device))


def _rotate_ref(x, cos, sin, il):
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if il else (x[..., :half], x[..., half:])
    u, w = a * cos - b * sin, b * cos + a * sin
    return torch.stack([u, w], -1).flatten(-2) if il else torch.cat([u, w], -1)


def qk_norm_rope_ref(qkv, wq, wk, cos, sin, T, H, kv_heads=None, eps=1e-5, il=False, start=None):
    """q, k, v heads of the QKV activation in (at least) fp32; tokens of sequence b stand at
    positions ``start[b] + t`` (default: t)."""
    KV, D, P = kv_heads or H, wq.shape[1], wq.shape[0]
    n = qkv.shape[0] // T
    f = torch.promote_types(qkv.dtype, torch.float32)
    x = qkv.to(f).view(n, T, H + 2 * KV, D).transpose(1, 2)
    at = torch.arange(T, device=qkv.device)[None]
    if start is not None:
        at = at + start.long()[:, None]
    c, s = cos.to(f)[at][:, None], sin.to(f)[at][:, None]

    def norm(t, w):
        w = w.to(f).repeat_interleave(n // P, 0)[:, None, None]
        return _rotate_ref(t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + eps) * w, c, s, il)
    return tuple(t.to(qkv.dtype).contiguous() for t in
                 (norm(x[:, :H], wq), norm(x[:, H:H + KV], wk), x[:, H + KV:]))


def _check_qk(qkv, wq, wk, cos, sin, T, H, KV):
    if qkv.dim() != 2 or wq.dim() != 2 or wq.shape != wk.shape:
        raise ValueError("qkv is [rows, (H + 2 KV) D], wq and wk are [trials, D]")
    P, D = wq.shape
    R = qkv.shape[0]
    if T < 1 or H < 1 or KV < 1 or H % KV:
        raise ValueError(f"tokens {T}, heads {H} and kv_heads {KV} must be positive, heads a "
                         "multiple of kv_heads")
    if qkv.shape[1] != (H + 2 * KV) * D:
        raise ValueError(f"qkv has {qkv.shape[1]} columns, {H} + 2 x {KV} heads of {D} need "
                         f"{(H + 2 * KV) * D}")
    if P < 1 or R % (P * T):
        raise ValueError(f"{R} rows are not {P} trials of whole sequences of {T} tokens")
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape != cos.shape or \
                t.shape[1] != D // 2 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float32 table [positions, {D // 2}]")
        if t.requires_grad:
            raise ValueError(f"{name} has no gradient here: detach it")
    if not (wq.dtype == wk.dtype == qkv.dtype):
        raise ValueError("qkv, wq and wk must be of one type")
    _same(qkv, "wq wk cos sin", wq, wk, cos, sin)
    if D % 2:
        raise ValueError(f"head dimension {D}: pairs are rotated")
    return P, D, R


def _check_kernel(what, t, D):
    if t.dtype not in _TYPES:
        raise ValueError(f"{what} on a GPU takes bfloat16 or float16, not {t.dtype}")
    if D not in (64, 128):
        raise ValueError(f"{what} on a GPU takes head dimensions 64 and 128, not {D}")


def _qk_fwd(qkv, wq, wk, cos, sin, T, H, KV, eps, il, k, v, start, cap):
    R, (P, D) = qkv.shape[0], wq.shape
    q = torch.empty(R // T, H, T, D, dtype=qkv.dtype, device=qkv.device)
    if R:
        strides = _Strides6(*k.stride()[:3], *v.stride()[:3])
        _call(qkv, "mopt_qk_norm_rope_fwd", _p(qkv), qkv.stride(0), _p(wq), _p(wk), _p(cos), _p(sin),
              _p(start), _p(q), _p(k), _p(v), strides, R, T, H, KV, R // P, D, cos.shape[0], cap, eps,
              int(il), _TYPES[qkv.dtype])
    return q


def _qk_blocks(rows: int, P: int, columns: int) -> int:
    """Workgroups of the backward for each trial's ``rows``: 8 a CU over all trials, each with 4 steps
    (of 2048 values) at least."""
    return max(1, min(-(-2048 // P), -(-rows * columns // 8192), rows))


def _qk_heads(qkv, wq, wk, cos, sin, T, H, KV, eps, il):
    shape = qkv.shape[0] // T, KV, T, wq.shape[1]
    k = torch.empty(shape, dtype=qkv.dtype, device=qkv.device)
    v = torch.empty_like(k)
    return _qk_fwd(qkv, wq, wk, cos, sin, T, H, KV, eps, il, k, v, None, T), k, v


class _QKNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, wq, wk, cos, sin, T, H, KV, eps, il):
        ctx.save_for_backward(qkv, wq, wk, cos, sin)
        ctx.meta = (T, H, KV, eps, il)
        return _qk_heads(qkv, wq, wk, cos, sin, T, H, KV, eps, il)

    @_once
    def backward(ctx, dq, dk, dv):
        qkv, wq, wk, cos, sin = ctx.saved_tensors
        T, H, KV, eps, il = ctx.meta
        (P, D), R = wq.shape, qkv.shape[0]
        dx = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        if R == 0:
            return (dx, torch.zeros_like(wq), torch.zeros_like(wk)) + (None,) * 7
        dq, dk, dv = _dense16(dq), _dense16(dk), _dense16(dv)
        dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
        blocks = _qk_blocks(R // P, P, (H + 2 * KV) * D)
        part = torch.empty(P * blocks * 2 * D, dtype=torch.float32, device=qkv.device)
        _call(qkv, "mopt_qk_norm_rope_bwd", _p(qkv), qkv.stride(0), _p(wq), _p(wk), _p(cos), _p(sin),
              _p(dq), _p(dk), _p(dv), _p(dx), _p(part), _p(dwq), _p(dwk), R, T, H, KV, R // P, D,
              blocks, eps, int(il), _TYPES[qkv.dtype])
        return (dx, dwq, dwk) + (None,) * 7


def _dense16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def qk_norm_rope(qkv, wq, wk, cos, sin, T, H, kv_heads=None, eps=1e-5, il=False):
    """(q ``[B', H, T, D]``, k, v ``[B', KV, T, D]``) of the QKV activation ``qkv``
    ``[B' T, (H + 2 KV) D]``: every query and key head is RMS-normalised, scaled by its trial's
    weight (``wq``, ``wk`` ``[P, D]``) and rotated by its position, in one pass.

    ``cos``, ``sin``: float32 ``[>= T, D / 2]`` (:func:`rope_tables`); pairs are (j, j + D / 2), or
    (2 j, 2 j + 1) with ``il``.  Differentiable in ``qkv``, ``wq`` and ``wk``; the sums over rows of
    the weights' gradients are taken in a fixed order."""
    KV = H if kv_heads is None else int(kv_heads)
    P, D, R = _check_qk(qkv, wq, wk, cos, sin, T, H, KV)
    if cos.shape[0] < T:
        raise ValueError(f"the tables hold {cos.shape[0]} positions, the sequences {T} tokens")
    if not _hip(qkv, "qk_norm_rope"):
        return qk_norm_rope_ref(qkv, wq, wk, cos, sin, T, H, KV, eps, il)
    _check_kernel("qk_norm_rope", qkv, D)
    _no_tangents("qk_norm_rope", qkv, wq, wk, cos, sin)
    args = _rows16(qkv), _dense16(wq), _dense16(wk), cos, sin, T, H, KV, float(eps), bool(il)
    return _QKNormRope.apply(*args) if _needs_grad(qkv, wq, wk) else _qk_heads(*args)


def _extent(t: torch.Tensor) -> int:
    """Bytes from the first element of ``t`` to behind its last."""
    if t.is_contiguous():
        return t.nbytes
    return (1 + sum([(m - 1) * s for m, s in zip(t.shape, t.stride())])) * t.element_size()


def _meet(off: int, dims) -> bool:
    """Whether ``off`` is a difference of two places of a layout: (stride, size) from the largest stride
    on, each larger than what the strides behind it reach."""
    if not dims:
        return off == 0
    (s, m), rest = dims[0], dims[1:]
    return any(abs(i) < m and _meet(off - i * s, rest) for i in (off // s, off // s + 1))


def _check_written(kcache, vcache, qkv) -> None:
    """Both caches are written while qkv is read: no place of theirs may be another's."""
    k0, v0, x0 = kcache.data_ptr(), vcache.data_ptr(), qkv.data_ptr()
    if kcache.is_contiguous() and vcache.is_contiguous() and qkv.is_contiguous():
        n = kcache.nbytes                        # the cheap way: three dense tensors, one behind another
        x1 = x0 + qkv.nbytes
        if (k0 + n <= v0 or v0 + n <= k0) and (k0 + n <= x0 or x1 <= k0) and (v0 + n <= x0 or x1 <= v0):
            return
    k1, v1, x1 = k0 + _extent(kcache), v0 + _extent(vcache), x0 + _extent(qkv)
    if not kcache.numel():
        return
    for c in (kcache, vcache):
        if not c.is_contiguous():
            reach = 0
            for s, m in sorted([(s, m) for s, m in zip(c.stride(), c.shape) if m > 1]):
                if s <= reach:
                    raise ValueError("the caches are written: no expanded tensors, none that overlap themselves")
                reach += (m - 1) * s
    if k0 < v1 and v0 < k1:                      # apart, or one between the other's rows in one layout
        off, rest = divmod(v0 - k0, kcache.element_size())
        layout = [[(s, m) for s, m in zip(c.stride(), c.shape) if m > 1] for c in (kcache, vcache)]
        if rest or layout[0] != layout[1] or _meet(off, sorted(layout[0], reverse=True)):
            raise ValueError("the caches are written: not one for both, and no overlapping ones")
    if (k0 < x1 and x0 < k1) or (v0 < x1 and x0 < v1):
        raise ValueError("the caches are written while qkv is read: not in one another's memory")


def qk_norm_rope_cached(qkv, wq, wk, cos, sin, T, H, kcache, vcache, start, eps=1e-5, il=False):
    """:func:`qk_norm_rope` of the next ``T`` tokens of every sequence: sequence b's stand at
    positions ``start[b] ... start[b] + T - 1`` (int32 ``[B']``, on the device), their keys and
    values are written into ``kcache``, ``vcache`` ``[B', KV, capacity, D]`` at these positions
    (nothing else of the caches is touched), and their queries ``[B', H, T, D]`` are returned.
    The caches may lie side by side in one tensor, but overlap neither each other nor ``qkv``.
    A token whose position lies outside the cache or the tables is not written, its query is 0.
    No gradients."""
    if kcache.dim() != 4 or kcache.shape != vcache.shape:
        raise ValueError("kcache and vcache are [sequences, kv_heads, capacity, D], both alike")
    KV, cap = kcache.shape[1], kcache.shape[2]
    P, D, R = _check_qk(qkv, wq, wk, cos, sin, T, H, KV)
    n = R // T
    if kcache.shape[0] != n or kcache.shape[3] != D:
        raise ValueError(f"the caches are {tuple(kcache.shape)}: {n} sequences of heads of {D}")
    if kcache.dtype != qkv.dtype or vcache.dtype != qkv.dtype:
        raise ValueError("the caches must be of qkv's type")
    _check_written(kcache, vcache, qkv)
    _same(qkv, "kcache vcache start", kcache, vcache, start)
    _int32("start", start, n)
    if not _hip(qkv, "qk_norm_rope"):
        return _cached_ref(qkv, wq, wk, cos, sin, T, H, kcache, vcache, start, eps, il)
    _check_kernel("qk_norm_rope_cached", qkv, D)
    _no_tangents("qk_norm_rope_cached", qkv, wq, wk, cos, sin, kcache, vcache)
    for name, c in (("kcache", kcache), ("vcache", vcache)):
        s = c.stride()
        if s[3] != 1 or c.data_ptr() % 16 or (s[0] | s[1] | s[2]) % 8:
            raise ValueError(f"{name} needs contiguous rows at multiples of 16 bytes: it is written "
                             "in place")
    if cap == 0 or not len(cos):
        return torch.zeros(n, H, T, D, dtype=qkv.dtype, device=qkv.device)
    q = _qk_fwd(_rows16(qkv), _dense16(wq), _dense16(wk), cos, sin, T, H, KV, float(eps), il, kcache,
                vcache, start, cap)
    torch.autograd.graph.increment_version((kcache, vcache))     # written behind torch's back
    return q


@torch.no_grad()
def _cached_ref(qkv, wq, wk, cos, sin, T, H, kcache, vcache, start, eps, il):
    n, KV, cap = kcache.shape[:3]
    if cap == 0 or not len(cos):                 # no token has a place
        return qkv.new_zeros(n, H, T, wq.shape[1])
    at = start.long()[:, None] + torch.arange(T, device=qkv.device)
    ok = (at >= 0) & (at < min(cap, cos.shape[0]))
    rows = torch.where(ok, at, torch.zeros_like(at)).reshape(-1)     # the tables' rows, one a token
    q, k, v = qk_norm_rope_ref(qkv, wq, wk, cos[rows], sin[rows], T, H, KV, eps, il,
                               start=torch.arange(n, device=qkv.device) * T)
    b, t = ok.nonzero(as_tuple=True)
    kcache[b, :, at[b, t]] = k[b, :, t]
    vcache[b, :, at[b, t]] = v[b, :, t]
    return torch.where(ok[:, None, :, None], q, torch.zeros_like(q))


# ============================================================================ window attention
def window_mask(Tq, Tk, window, sinks, start, lengths, device=None):
    """Visible pairs ``[B', Tq, Tk]`` of :func:`window_attention`."""
    i = start.long()[:, None, None] + torch.arange(Tq, device=device)[None, :, None]
    j = torch.arange(Tk, device=device)[None, None]
    n = lengths.long().clamp(0, Tk)[:, None, None]
    return (j <= i) & (i < n) & ((i - j < window) | (j < sinks))


def window_attention_ref(q, k, v, window=None, sinks=0, scale=None, start=None, lengths=None):
    """The same in (at least) fp32 with a full score matrix."""
    B, H, Tq, D = q.shape
    KV, Tk = k.shape[1], k.shape[2]
    f = torch.promote_types(q.dtype, torch.float32)
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    start = Tk - Tq if start is None else start
    first = start if torch.is_tensor(start) else torch.full((B,), start, device=q.device)
    lengths = first + Tq if lengths is None else lengths
    see = window_mask(Tq, Tk, Tk + Tq if window is None else window, sinks, first, lengths,
                      q.device)[:, None, None]
    # keys behind a sequence's length do not exist, whatever the tensors hold there
    live = (torch.arange(Tk, device=q.device) < lengths.long()[:, None])[:, None, :, None]
    kf, vf = (torch.where(live, t.to(f), torch.zeros((), dtype=f, device=q.device)) for t in (k, v))
    real = see.any(-1, keepdim=True)                     # [B, 1, 1, Tq, 1]
    qf = torch.where(real, q.to(f).view(B, KV, H // KV, Tq, D), torch.zeros((), dtype=f, device=q.device))
    s = torch.matmul(qf, kf[:, :, None].transpose(3, 4)) * scale
    s = s.masked_fill(~see, -math.inf).masked_fill(~real, 0.0)
    p = s.softmax(-1) * real
    o = torch.matmul(p, vf[:, :, None])
    return o.reshape(B, H, Tq, D).permute(0, 2, 1, 3).reshape(B * Tq, H * D).to(q.dtype)


def _span(sinks: int, heads: int, Tq: int) -> int:
    """Queries of one item of the dK / dV kernel that adds up sinks' pairs out of the window
    (csrc/lm_window.hip): 512 where there are so many of these that they fill the CUs (125M step: 95
    us, with 128 107), else 128, as the others wait for the last of them (8192 tokens, 4 key heads of
    128: 206 us, with 512 264); and so many that the 4 partial sums of the sinks' rows that each
    leaves are no more than there are queries."""
    near = 512 if heads * -(-Tq // 512) >= 256 else 128
    return max(near, -(-4 * sinks // 64) * 64)


def _geometry(q, k, v):
    return _Strides9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])


def _splits(heads: int, tokens: int) -> int:
    """Workgroups that share the ``tokens`` keys of each of ``heads`` key heads: at most one a CU
    over all heads (32768 keys of 8 heads: 25 us, with two a CU 29), and each with 1024 keys at
    least: joining them costs a launch, 3.4 us, as much as about 1000 keys do."""
    return max(1, min(256 // heads, tokens // 1024))


def _window_fwd(q, k, v, window, sinks, scale, start, start0, lengths, train):
    B, H, Tq, D = q.shape
    KV, Tk = k.shape[1], k.shape[2]
    o = torch.empty(B * Tq, H * D, dtype=q.dtype, device=q.device)
    # for the backward: the log-sums and what the rounding of o left off
    lse = torch.empty(B, H, -(-Tq // 128) * 128, dtype=torch.float32, device=q.device) if train else None
    rest = torch.empty_like(o) if train else None
    if o.numel() and Tk and not train and H // KV * Tq <= 16:
        splits = _splits(B * KV, min(Tk, window + sinks))
        part = torch.empty(B * KV * splits * 16 * (D + 4), dtype=torch.float32,
                           device=q.device) if splits > 1 else None
        _call(q, "mopt_window_step", _p(q), _p(k), _p(v), _geometry(q, k, v), _p(start), _p(lengths),
              start0, _p(o), _p(part), splits, B, H, KV, Tq, Tk, D, window, sinks, scale,
              _TYPES[q.dtype])
    elif o.numel() and Tk:
        _call(q, "mopt_window_fwd", _p(q), _p(k), _p(v), _geometry(q, k, v), _p(start), _p(lengths),
              start0, _p(o), _p(rest), _p(lse), B, H, KV, Tq, Tk, D, window, sinks, scale,
              _TYPES[q.dtype])
    else:
        o.zero_()
    return o, rest, lse


def _parts(blocks: int, steps: int) -> int:
    """Workgroups that share the queries of each of ``blocks`` key blocks in the dK / dV kernel,
    where there are fewer blocks than two a CU (8192 tokens of 4 key heads, window 1024: heads of 64
    124 + 8 us against 171 + 5, of 128 206 + 14 against 240 + 6), each with 8 of the block's ``steps``
    groups of 32 queries at least.  Their sums are added up by another launch."""
    return max(1, min(512 // max(1, blocks), steps // 8))


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, start, start0, lengths):
        o, rest, lse = _window_fwd(q, k, v, window, sinks, scale, start, start0, lengths, True)
        ctx.save_for_backward(q, k, v, o, rest, lse, start, lengths)
        ctx.meta = (window, sinks, scale, start0)
        return o

    @_once
    def backward(ctx, do):
        q, k, v, o, rest, lse, start, lengths = ctx.saved_tensors
        window, sinks, scale, start0 = ctx.meta
        B, H, Tq, D = q.shape
        KV, Tk = k.shape[1], k.shape[2]
        new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        dq, dk, dv = new(q), new(k), new(v)
        if not o.numel() or not Tk:
            return (dq.zero_(), dk.zero_(), dv.zero_()) + (None,) * 6
        dsum = torch.empty_like(lse)
        span = _span(sinks, B * KV, Tq)
        spans = -(-Tq // span) if sinks and Tk > window else 0
        parts = _parts(B * KV * -(-Tk // 128), H // KV * (min(Tq, window + 128) // 32))
        part = None
        if parts > 1 or spans:
            rows = parts * (Tk if parts > 1 else sinks) + 4 * spans * sinks
            part = torch.empty(rows * B * KV * 2 * D, dtype=torch.float32, device=q.device)
        _call(q, "mopt_window_bwd", _p(q), _p(k), _p(v), _geometry(q, k, v), _p(start), _p(lengths),
              start0, _p(o), _p(rest), _p(_dense16(do)), _p(lse), _p(dsum), _p(dq), _p(dk), _p(dv), _p(part),
              parts, spans, span, B, H, KV, Tq, Tk, D, window, sinks, scale, _TYPES[q.dtype])
        return (dq, dk, dv) + (None,) * 6


def window_attention(q, k, v, window: Optional[int] = None, sinks: int = 0, scale=None, start=None,
                     lengths=None):
    """Causal attention rows ``[B' Tq, H D]`` of q ``[B', H, Tq, D]`` over k, v ``[B', KV, Tk, D]``
    (H a multiple of KV: query head h reads key head ``h // (H / KV)``).

    Query t of sequence b stands at position ``i = start[b] + t`` and sees the keys
    ``j <= i < lengths[b]`` with ``i - j < window`` (None: all) or ``j < sinks``.

    ``start``: an int or int32 ``[B']``; default ``Tk - Tq`` (the last queries of the keys; 0 for
    self-attention).  ``lengths``: int32 ``[B']``, default ``start + Tq``; values over ``Tk`` count
    as ``Tk``.  Queries outside ``[0, lengths[b])`` are padding: their rows are 0, what q, k, v and
    the output's gradient hold there is not read, and their gradients are 0.  So a batch padded at
    its end passes ``lengths``; one new token over a cache passes Tq = 1 and ``start`` = the tokens
    before it.  Within a sequence all values must be finite: a score outside the mask counts as
    absent, but a value's infinity or NaN reaches the queries whose tiles it shares.

    ``scale``: positive (within [1e-30, 1e30]), default ``1 / sqrt(D)``.  Scores and log-sums are
    kept in 32 bits: beyond 2^16 in size their last bits are felt in the gradients.  Probabilities and
    score gradients enter their products as two 16-bit pieces (2^-16 of themselves in bf16, 2^-22 in
    fp16), so that results are as near as rounded once.  Any strides
    (copied where rows are not contiguous at multiples of 16 bytes).  Differentiable in q, k and v,
    with sums in a fixed order."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError("q is [B, H, Tq, D], k and v are [B, KV, Tk, D]")
    B, H, Tq, D = q.shape
    KV, Tk = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)} does not fit k {tuple(k.shape)}")
    if H < 1 or KV < 1 or H % KV:
        raise ValueError(f"{H} query heads are not a multiple of {KV} key heads")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q, k and v must be of one type")
    if window is not None and window < 1:
        raise ValueError(f"window {window}: a query sees itself at least (None: no window)")
    if sinks < 0:
        raise ValueError(f"sinks {sinks} must not be negative")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:               # (its reciprocal is taken in 32 bits, too)
        raise ValueError(f"scale {scale} must be positive, within [1e-30, 1e30]")
    if max(Tq, Tk) > MAX_LENGTH:
        raise ValueError(f"sequences and caches hold at most {MAX_LENGTH} tokens")
    _same(q, "k v", k, v)
    start0 = Tk - Tq
    if torch.is_tensor(start):
        _int32("start", start, B)
        _same(q, "start", start)
    elif start is not None:
        start0, start = int(start), None
        if abs(start0) > MAX_LENGTH:
            raise ValueError(f"start {start0} is no position")
    if lengths is not None:
        _int32("lengths", lengths, B)
        _same(q, "lengths", lengths)
    if not _hip(q, "window_attn"):
        return window_attention_ref(q, k, v, window, sinks, scale, start0 if start is None else start,
                                    lengths)
    _check_kernel("window_attention", q, D)
    _no_tangents("window_attention", q, k, v)
    # a window over all positions is no window; sinks within every window are none
    reach = 1 << 30 if window is None else min(int(window), 1 << 30)
    sinks = min(int(sinks), Tk) if reach < Tk else 0
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    if _needs_grad(q, k, v):
        return _WindowAttention.apply(q, k, v, reach, sinks, scale, start, start0, lengths)
    return _window_fwd(q, k, v, reach, sinks, scale, start, start0, lengths, False)[0]

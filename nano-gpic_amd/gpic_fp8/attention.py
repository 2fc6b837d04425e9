"""Attention of queries to an encoder's states of another length, on the HIP kernels of nano-gpic_amd/csrc/attention.hip: the
operator between the projections and the output projection of a text-conditioned block. (The reference's attentions call torch's
scaled_dot_product_attention, attention_op.py:4.)

    cross_attention(q, k, v, kv_lens, mask, scale)    o = softmax(scale q k^T over the valid keys) v, differentiable
    cross_attention_fwd, cross_attention_bwd          its two passes

One query a head (a decode step) takes a kernel of its own that splits the keys over the chip. o lies in memory as [B, N, H, D], so
merging its heads for the output projection (o.transpose(1, 2).reshape(B, N, H D)) copies nothing, and fp8_heads_linear_f8 takes it
as it is. Differentiable once: a backward under create_graph=True raises.
"""
import ctypes
import math
from typing import Optional

import torch

from . import _lib as L
from .layernorm import no_tangents, once
from .rows import _PLAIN, _call, _run, _same_device

DTYPES = {torch.bfloat16: 0, torch.float16: 2}
MAX_D = 128
F32 = torch.float32


def _strides(t):
    """The strides of a batch entry, a head and a row; of an extent of one, 0."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:3], t.shape[:3])]


def _heads(t):
    """t [B, H, N, D] as the kernels read it: a row's elements beside each other, rows 16-byte aligned; copied only where they are
    not (to [B, N, H, D] in memory)."""
    if t.numel() and (t.stride(3) != 1 or t.data_ptr() % 16 or any(s % 8 for s in _strides(t))):
        t = L.aligned(t.transpose(1, 2).contiguous()).transpose(1, 2)
    return t, (ctypes.c_int64 * 3)(*_strides(t))


def _new(like, B, H, N, D):
    return torch.empty(B, N, H, D, dtype=like.dtype, device=like.device).transpose(1, 2)


def _check(q, k, v, lens, mask, scale):
    L.require_gpu(q, k, v, lens, mask)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError(f"cross_attention takes q [B, H, N, D] and k, v [B, Hk, L, D], got {tuple(q.shape)}, {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"cross_attention takes bf16 or fp16 q, k and v of one type, got {q.dtype}, {k.dtype} and {v.dtype}")
    B, H, N, D = q.shape
    Hk, n = k.shape[1], k.shape[2]
    if not 0 < D <= MAX_D or D % 8 or Hk == 0 or H == 0 or H % Hk:
        raise ValueError(f"cross_attention needs D % 8 == 0, 0 < D <= {MAX_D} and H a multiple of Hk, got D = {D}, H = {H}, Hk = {Hk}")
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite, got {scale}")
    if lens is not None and (lens.shape != (B,) or lens.dtype not in (torch.int32, torch.int64)):
        raise ValueError(f"kv_lens must be int32 or int64 [{B}], got {lens.dtype} {tuple(lens.shape)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape not in ((B, n), (B, 1, 1, n))):
        raise ValueError(f"mask must be bool [{B}, {n}] or [{B}, 1, 1, {n}], true where a key takes part, got {mask.dtype} "
                         f"{tuple(mask.shape)}")
    _same_device(q.device, k=k, v=v, kv_lens=lens, mask=mask)
    no_tangents("cross_attention", q, k, v)


def _keys(lens, mask, n):
    """lens as int32 and mask as rows of bytes, and the rows' stride."""
    if lens is not None:
        lens = (lens if lens.dtype == torch.int32 else lens.clamp(0, n).to(torch.int32)).contiguous()
    ld = 0
    if mask is not None:
        mask = mask.view(mask.shape[0], n)
        if n > 1 and mask.stride(1) != 1:
            mask = mask.contiguous()
        ld = mask.stride(0) if mask.shape[0] > 1 else 0
    return lens, mask, ld


@L.step_op("gpic::cross_attention_fwd")
def cross_attention_fwd_op(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_lens: Optional[torch.Tensor],
                           mask: Optional[torch.Tensor], scale: float, want_lse: bool = True
                           ) -> tuple[torch.Tensor, torch.Tensor]:
    """cross_attention_fwd, as an op."""
    o = L.native("attention", q, q, k, v, kv_lens, mask, scale, want_lse)
    if o is not None:
        return o
    _check(q, k, v, kv_lens, mask, scale)
    B, H, N, D = q.shape
    Hk, n = k.shape[1:3]
    (q, qs), (k, ks), (v, vs) = _heads(q), _heads(k), _heads(v)
    lens, m, ldm = _keys(kv_lens, mask, n)
    o = _new(q, B, H, N, D)
    lse = torch.empty((B, H, N) if want_lse else (0,), dtype=F32, device=q.device)
    with L.on_device(q.device):
        nws = L.lib().gpic_fp8_attention_workspace_bytes(B, H, Hk, N, n, D)
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws else None
        L.check(L.lib().gpic_fp8_attention(
            q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, DTYPES[q.dtype], L.ptr(lens), L.ptr(m), ldm, B, H, Hk, N, n, D,
            float(scale), o.data_ptr(), (ctypes.c_int64 * 3)(*_strides(o)), lse.data_ptr() if want_lse else None, L.ptr(ws), nws,
            L.stream_ptr(q.device)), "gpic_fp8_attention")
    return o, lse


@cross_attention_fwd_op.register_fake
def _(q, k, v, kv_lens, mask, scale, want_lse=True):
    B, H, N, D = q.shape
    return q.new_empty(B, N, H, D).transpose(1, 2), q.new_empty((B, H, N) if want_lse else (0,), dtype=F32)


@L.step_op("gpic::cross_attention_bwd")
def cross_attention_bwd_op(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                           lse: torch.Tensor, kv_lens: Optional[torch.Tensor], mask: Optional[torch.Tensor], scale: float,
                           want_kv: bool = True) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """cross_attention_bwd, as an op (dk and dv empty unless want_kv)."""
    r = L.native("attention_bwd", q, dout, q, k, v, o, lse, kv_lens, mask, scale, want_kv)
    if r is not None:
        return r
    _check(q, k, v, kv_lens, mask, scale)
    L.require_gpu(dout, o, lse)
    _same_device(q.device, dout=dout, o=o, lse=lse)
    B, H, N, D = q.shape
    Hk, n = k.shape[1:3]
    if dout.shape != q.shape or o.shape != q.shape or o.dtype != q.dtype:
        raise ValueError(f"dout and o must be like q {tuple(q.shape)}, got {tuple(dout.shape)} and {o.dtype} {tuple(o.shape)}")
    if lse.shape != (B, H, N) or lse.dtype != F32:
        raise ValueError(f"lse must be fp32 {(B, H, N)}, got {lse.dtype} {tuple(lse.shape)}")
    (dout, ds), (q, qs), (k, ks), (v, vs), (o, os) = (_heads(t) for t in (dout.to(q.dtype), q, k, v, o))
    lse = lse.contiguous()
    lens, m, ldm = _keys(kv_lens, mask, n)
    dq = _new(q, B, H, N, D)
    dk, dv = (_new(q, B, Hk, n, D) if want_kv else q.new_empty(0) for _ in range(2))
    s3 = lambda t: (ctypes.c_int64 * 3)(*_strides(t)) if want_kv else None  # noqa: E731
    with L.on_device(q.device):
        nws = L.lib().gpic_fp8_attention_bwd_workspace_bytes(B, H, Hk, N, n, D)
        ws = torch.empty(max(nws, 16), dtype=torch.uint8, device=q.device)
        L.check(L.lib().gpic_fp8_attention_bwd(
            dout.data_ptr(), ds, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, o.data_ptr(), os, lse.data_ptr(),
            DTYPES[q.dtype], L.ptr(lens), L.ptr(m), ldm, B, H, Hk, N, n, D, float(scale), dq.data_ptr(),
            (ctypes.c_int64 * 3)(*_strides(dq)), dk.data_ptr() if want_kv else None, s3(dk), dv.data_ptr() if want_kv else None,
            s3(dv), ws.data_ptr(), nws, L.stream_ptr(q.device)), "gpic_fp8_attention_bwd")
    return dq, dk, dv


@cross_attention_bwd_op.register_fake
def _(dout, q, k, v, o, lse, kv_lens, mask, scale, want_kv=True):
    new = lambda t: t.new_empty(t.shape[0], t.shape[2], t.shape[1], t.shape[3]).transpose(1, 2)  # noqa: E731
    return (new(q), new(k), new(v)) if want_kv else (new(q), q.new_empty(0), q.new_empty(0))


def _scale(scale, q):
    return float(scale) if scale is not None else q.shape[-1] ** -0.5 if q.dim() and q.shape[-1] else 1.0


def cross_attention_fwd(q, k, v, kv_lens=None, mask=None, scale=None):
    """cross_attention's o and its rows' log2-sums [B, H, N] fp32 (of 2^(scores log2 e); +inf where no key is valid), which
    cross_attention_bwd takes."""
    return _run(cross_attention_fwd_op, "attention", q, q, k, v, kv_lens, mask, _scale(scale, q), True)


def cross_attention_bwd(dout, q, k, v, o, lse, kv_lens=None, mask=None, scale=None):
    """The gradients (dq, dk, dv) of cross_attention from o's, and the forward's o and lse."""
    return _run(cross_attention_bwd_op, "attention_bwd", q, dout, q, k, v, o, lse, kv_lens, mask, _scale(scale, q), True)


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_lens, mask, scale):
        train = any(ctx.needs_input_grad)
        o, lse = _call(cross_attention_fwd_op, q, k, v, kv_lens, mask, scale, train)
        ctx.save_for_backward(q, k, v, o, lse, kv_lens, mask)
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        return o

    @staticmethod
    @once("cross_attention")
    def backward(ctx, do):
        if do is None:
            return (None,) * 6
        q, k, v, o, lse, kv_lens, mask = ctx.saved_tensors
        nq, nk, nv = ctx.needs_input_grad[:3]
        dq, dk, dv = _call(cross_attention_bwd_op, do, q, k, v, o, lse, kv_lens, mask, ctx.scale, nk or nv)
        return dq if nq else None, dk if nk else None, dv if nv else None, None, None, None


def cross_attention(q, k, v, kv_lens=None, mask=None, scale=None):
    """o [B, H, N, D] = softmax(scale q k^T) v of q [B, H, N, D] and an encoder's k, v [B, Hk, L, D], bf16 or fp16, over the keys that
    are valid: below kv_lens[b] (int32 or int64 [B]; taken into 0..L) and where mask (bool [B, L] or [B, 1, 1, L]) is true, both
    together if both are given. A batch entry without a valid key gives zeros, and zeros as gradients; what k and v hold at keys that
    are not valid is not used, whatever it is. H is a multiple of Hk: head h reads key head h Hk // H. D % 8 == 0, D <= 128. scale > 0
    (None: 1 / sqrt(D)). Any strides (rows that are not contiguous or 16-byte aligned are copied). o lies as [B, N, H, D].
    Differentiable (once) in q, k and v."""
    scale = _scale(scale, q)
    if type(q) in _PLAIN:
        o = L.native("attention_call", q, q, k, v, kv_lens, mask, scale)
        if o is not None:
            return o
    return _CrossAttention.apply(q, k, v, kv_lens, mask, scale)

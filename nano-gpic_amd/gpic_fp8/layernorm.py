"""Layer norm on the HIP kernels of nano-gpic_amd/csrc/layernorm.hip, beside the root-mean-square norms (rows.py, norm.py). No
counterpart in the reference, whose norms take no mean (fused_norm.py:64-91).

    layer_norm(x, weight, bias, eps, a)        x_new = x + a;  h = (x_new - mean) / deviation weight + bias, differentiable
    layer_norm_rows(x, weight, bias, eps, a)   the same with h as e4m3 and one scale a row, for fp8_gemm_rows in a server
    layer_norm_bwd                             the backward pass, with the weight's and the bias's gradient

They run in the type of x (bf16, fp16 or fp32) with fp32 inside and one rounding. layer_norm is differentiable once: a backward
under create_graph=True raises.
"""
import functools
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L
from .fp8_native import E4, _rows
from .rows import BF, NORM_MAX_C, _PLAIN, _call, _run, _same_device

F32 = torch.float32


def once(what):
    """once_differentiable for the backward of `what`, which raises under create_graph=True: its gradients would be constants
    there, and a term of a loss made of them would be lost without a word."""
    def deco(backward):
        inner = once_differentiable(backward)

        @functools.wraps(backward)
        def call(ctx, *grads):
            if torch.is_grad_enabled() and not torch.compiler.is_compiling():
                raise RuntimeError(f"{what} is differentiable once: its backward does not run under create_graph=True")
            return inner(ctx, *grads)
        return call
    return deco


def no_tangents(what, *tensors):
    """Raises for a tensor that carries a forward-mode gradient, which the kernels would drop."""
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode gradient")


def _vec3(t, C, name):
    """A weight or bias [C] of a type the kernels take, 16-byte aligned; None as it is."""
    if t is None:
        return None
    if t.shape != (C,):
        raise ValueError(f"{name} must be [{C}], got {tuple(t.shape)}")
    if t.dtype not in L.DTYPE_CODE_3:
        t = t.float()
    return L.aligned(t.contiguous())


def _code(t):
    return L.DTYPE_CODE_3[t.dtype] if t is not None else 0


def _check(x, a, weight, bias, name, dtypes):
    L.require_gpu(x, a, weight, bias)
    if x.dim() < 1 or x.dtype not in dtypes or x.shape[-1] % 8 or not 0 < x.shape[-1] <= NORM_MAX_C:
        raise ValueError(f"{name} takes {', '.join(str(d)[6:] for d in dtypes)} x [..., C] with C % 8 == 0 and 0 < C <= "
                         f"{NORM_MAX_C}, got {x.dtype} {tuple(x.shape)}")
    if a is not None and a.shape != x.shape:
        raise ValueError(f"a must have x's shape {tuple(x.shape)}, got {tuple(a.shape)}")
    _same_device(x.device, a=a, weight=weight, bias=bias)
    no_tangents(name, x, a, weight, bias)


def _forward(x, weight, bias, eps, a, want_h, stats, rows):
    """(x_new, h, mean, rstd, q, s), the ones not asked for empty."""
    C, dev = x.shape[-1], x.device
    w, b = _vec3(weight, C, "weight"), _vec3(bias, C, "bias")
    x2, ldx = _rows(x.reshape(-1, C))
    a2, lda = _rows(a.to(x.dtype).reshape(-1, C)) if a is not None else (None, 0)
    M = x2.shape[0]
    none = x.new_empty(0)
    xn = torch.empty(x.shape, dtype=x.dtype, device=dev) if a is not None else none
    h = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_h else x.new_empty(0)
    mean, rstd = (torch.empty(M if stats else 0, dtype=F32, device=dev) for _ in range(2))
    q = torch.empty(x.shape if rows else (0,), dtype=E4, device=dev)
    s = torch.empty(M if rows else 0, dtype=F32, device=dev)
    with L.on_device(dev):
        L.check(L.lib().gpic_fp8_layer_norm(
            x2.data_ptr(), L.DTYPE_CODE_3[x.dtype], ldx, L.ptr(a2), lda, L.ptr(w), _code(w), L.ptr(b), _code(b), M, C,
            float(eps), xn.data_ptr() if a is not None else None, h.data_ptr() if want_h else None,
            mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None, q.data_ptr() if rows else None,
            s.data_ptr() if rows else None, L.stream_ptr(dev)), "gpic_fp8_layer_norm")
    return xn, h, mean, rstd, q, s


# ------------------------------------------------------------------------------------------------ ops

@L.step_op("gpic::layer_norm_fwd")
def layer_norm_fwd_op(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
                      a: Optional[torch.Tensor] = None, stats: bool = True
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(x_new, empty without a; h; mean [rows]; rstd [rows], the last two empty unless stats)."""
    o = L.native("layer_norm", x, x, weight, bias, eps, a, stats)
    if o is not None:
        return o
    _check(x, a, weight, bias, "layer_norm", tuple(L.DTYPE_CODE_3))
    return _forward(x, weight, bias, eps, a, True, stats, False)[:4]


@layer_norm_fwd_op.register_fake
def _(x, weight, bias, eps, a=None, stats=True):
    M = x.shape[:-1].numel() if stats else 0
    return (x.new_empty(x.shape) if a is not None else x.new_empty(0), x.new_empty(x.shape), x.new_empty(M, dtype=F32),
            x.new_empty(M, dtype=F32))


@L.step_op("gpic::layer_norm_rows")
def layer_norm_rows_op(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5, a: Optional[torch.Tensor] = None, want_h: bool = False
                       ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """layer_norm_rows, as an op."""
    o = L.native("layer_norm_rows", x, x, weight, bias, eps, a, want_h)
    if o is not None:
        return o
    _check(x, a, weight, bias, "layer_norm_rows", (BF,))
    xn, h, _, _, q, s = _forward(x, weight, bias, eps, a, want_h, False, True)
    return xn, h, q, s


@layer_norm_rows_op.register_fake
def _(x, weight=None, bias=None, eps=1e-5, a=None, want_h=False):
    return (x.new_empty(x.shape) if a is not None else x.new_empty(0), x.new_empty(x.shape) if want_h else x.new_empty(0),
            x.new_empty(x.shape, dtype=E4), x.new_empty(x.shape[:-1].numel(), dtype=F32))


@L.step_op("gpic::layer_norm_bwd")
def layer_norm_bwd_op(dh: torch.Tensor, dxn: Optional[torch.Tensor], xs: torch.Tensor, weight: Optional[torch.Tensor],
                      mean: torch.Tensor, rstd: torch.Tensor, bias_dtype: Optional[torch.dtype] = None
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """layer_norm_bwd, as an op: (dx; dw, empty without a weight; db, empty without a bias_dtype)."""
    o = L.native("layer_norm_bwd", xs, dh, dxn, xs, weight, mean, rstd, bias_dtype)
    if o is not None:
        return o
    _check(xs, None, weight, None, "layer_norm_bwd", tuple(L.DTYPE_CODE_3))
    L.require_gpu(dh, dxn, mean, rstd)
    dev, C, dt = xs.device, xs.shape[-1], xs.dtype
    _same_device(dev, dh=dh, dxn=dxn, mean=mean, rstd=rstd)
    M = xs.numel() // C
    if dh.shape != xs.shape or (dxn is not None and dxn.shape != xs.shape):
        raise ValueError(f"dh and dxn must have xs's shape {tuple(xs.shape)}")
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.numel() != M or t.dtype != F32:
            raise ValueError(f"{name} must be fp32 with {M} elements, got {t.dtype} {tuple(t.shape)}")
    dhc, xc = L.aligned(dh.to(dt).contiguous()), L.aligned(xs.contiguous())
    nc = L.aligned(dxn.to(dt).contiguous()) if dxn is not None else None
    w, mc, rc = _vec3(weight, C, "weight"), mean.contiguous(), rstd.contiguous()
    dx = torch.empty(xs.shape, dtype=dt, device=dev)
    dw = torch.empty(C if w is not None else 0, dtype=w.dtype if w is not None else F32, device=dev)
    bdt = bias_dtype if bias_dtype in L.DTYPE_CODE_3 else F32
    db = torch.empty(C if bias_dtype is not None else 0, dtype=bdt, device=dev)
    with L.on_device(dev):
        nws = L.lib().gpic_fp8_layer_norm_bwd_workspace_bytes(M, C)
        ws = torch.empty(max(nws, 16), dtype=torch.uint8, device=dev)
        L.check(L.lib().gpic_fp8_layer_norm_bwd(
            dhc.data_ptr(), L.ptr(nc), xc.data_ptr(), L.DTYPE_CODE_3[dt], L.ptr(w), _code(w), mc.data_ptr(), rc.data_ptr(),
            M, C, dx.data_ptr(), dw.data_ptr() if w is not None else None, L.DTYPE_CODE_3[dw.dtype],
            db.data_ptr() if bias_dtype is not None else None, L.DTYPE_CODE_3[bdt], ws.data_ptr(), nws, L.stream_ptr(dev)),
            "gpic_fp8_layer_norm_bwd")
    return dx, dw, db


@layer_norm_bwd_op.register_fake
def _(dh, dxn, xs, weight, mean, rstd, bias_dtype=None):
    C = xs.shape[-1]
    kept = lambda d: d if d in L.DTYPE_CODE_3 else F32  # noqa: E731
    return (xs.new_empty(xs.shape), xs.new_empty(C if weight is not None else 0, dtype=kept(getattr(weight, "dtype", None))),
            xs.new_empty(C if bias_dtype is not None else 0, dtype=kept(bias_dtype)))


# ------------------------------------------------------------------------------------------------ public calls

def layer_norm_rows(x, weight=None, bias=None, eps=1e-5, a=None, want_h=False):
    """x_new = x + a (without a: x), h = (x_new - mean) / sqrt(variance + eps) weight + bias ->
    (x_new bf16, empty without a; h bf16, empty unless want_h; h's e4m3 bytes; their scales [rows]).
    x, a [..., C] bf16, C % 8 == 0, C <= 16384; weight, bias [C], or None. h is rounded once, to e4m3 (and once, to bf16, for
    want_h). The bytes and scales are fp8_gemm_rows' operand. Forward only."""
    return _run(layer_norm_rows_op, "layer_norm_rows", x, x, weight, bias, eps, a, want_h)


def layer_norm_bwd(dh, dxn, xs, weight, mean, rstd, bias_dtype=None):
    """The backward of layer_norm: dh (of h) and dxn (of x_new, or None) like xs (x_new, or x without a) [..., C] bf16, fp16 or
    fp32; mean, rstd [rows] fp32 -> (dx, which is a's gradient too, of xs's type; dw [C] of weight's type, empty without one; db
    [C] of bias_dtype, empty for None). The sums are fp32 in a fixed order, rounded once."""
    return _run(layer_norm_bwd_op, "layer_norm_bwd", xs, dh, dxn, xs, weight, mean, rstd, bias_dtype)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, a):
        xn, h, mean, rstd = _call(layer_norm_fwd_op, x, weight, bias, eps, a, any(ctx.needs_input_grad))
        ctx.save_for_backward(x if a is None else xn, weight, mean, rstd)
        ctx.set_materialize_grads(False)
        ctx.bdt, ctx.adt = None if bias is None else bias.dtype, None if a is None else a.dtype
        return h if a is None else (xn, h)

    @staticmethod
    @once("layer_norm")
    def backward(ctx, *grads):
        xs, weight, mean, rstd = ctx.saved_tensors
        dxn, dh = grads if len(grads) == 2 else (None, grads[0])
        nx, nw, nb, _, na = ctx.needs_input_grad
        if dh is None:
            if dxn is None:
                return (None,) * 5
            # x_new alone was used: its gradient as it is, and zeros that no value of x can spoil
            dx = dxn.to(xs.dtype)
            dw = torch.zeros_like(weight) if nw else None
            db = xs.new_zeros(xs.shape[-1], dtype=ctx.bdt) if nb else None
        else:
            dx, dw, db = _call(layer_norm_bwd_op, dh, dxn, xs, weight, mean, rstd, ctx.bdt if nb else None)
            dw = dw.to(weight.dtype) if nw else None
            db = db.to(ctx.bdt) if nb else None
        return dx if nx else None, dw, db, None, dx.to(ctx.adt) if na else None


def layer_norm(x, weight=None, bias=None, eps=1e-5, a=None):
    """h = (x_new - mean) / sqrt(variance + eps) weight + bias of x_new = x + a: (x_new, h); without a h alone.
    x [..., C] bf16, fp16 or fp32, C % 8 == 0, C <= 16384; a of x's shape; weight, bias [C] or None. The statistics are over the
    last dimension, in fp32; x_new and h are rounded once to x's type. Differentiable (once): the gradients of x, a, weight and
    bias."""
    if a is not None and a.shape != x.shape:
        raise ValueError(f"a must have x's shape {tuple(x.shape)}, got {tuple(a.shape)}")
    if type(x) in _PLAIN:
        o = L.native("layer_norm_call", x, x, weight, bias, eps, a)
        if o is not None:
            return o
    return _LayerNorm.apply(x, weight, bias, eps, a)

"""The row-scaled operators: e4m3 with one scale a row (a token, or an output channel of a weight) instead of one a tensor,
on the HIP kernels of nano-gpic_amd/csrc/rows.hip and gemm.hip. No counterpart in the reference, whose casts are tensorwise
(fp8_native.py:33-49).

    rmsnorm_rows      x_new = x + gate a;  h = RMSNorm(x_new) (1 + scale) + shift  -> e4m3 and scales by row
    tcast_rows        the row cast of a matrix
    fp8_gemm_rows     y = residual + gate act(sa sb a b^T + bias), one rounding; act: none, silu, gelu_tanh, swiglu
    act_bwd_rows      the epilogue's backward: dz, and dz times the weight's scales cast by row
    rmsnorm_rows_bwd  the norm's backward
and over them
    fp8_linear_rows(x, weight, ...)               a linear with activation and residual
    fp8_rmsnorm_linear_rows(x, w_norm, ..., weight, ...)   the norm feeding one

A row's scale needs no maximum over the chip, so one token's norm or linear is a short launch, and a token's bytes do not
depend on the others of its batch (nor its linear on their values; their number chooses the GEMM's tiles, whose sums differ in
the last bits). With weights that rows_weight has cast once (a sampler, a server) a linear is the cast of
x and one GEMM; with ordinary weights the two are differentiable: the forward and the dgrad in FP8, the weight's gradient
in bf16 (a token's scale lies on its reduction), from the bf16 input and the bf16 gradient of z. They are differentiable
once: under create_graph=True their gradients are constants, with a warning.
"""
import functools
import warnings
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from .fp8_native import E4, _gemm_operand, _no_autocast, _r16, _rows, bf16_wgrad
from .norm import BWD_MAX_C, res_mod_rmsnorm_bwd_k

ACTS = {"none": 0, "silu": 1, "gelu_tanh": 2, "swiglu": 3}
NORM_MAX_C = 16384    # the norm's widest row
CAST_MAX_C = 32768    # the row casts'
BF = torch.bfloat16


def _act(act, train=False):
    if act not in ACTS or (train and act == "swiglu"):
        raise ValueError(f"act must be one of {sorted(a for a in ACTS if not (train and a == 'swiglu'))}, got {act!r}")
    return ACTS[act]


_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _run(op, name, x, *args):
    """A public call of op: the native host module's function `name` on args, else the op's function (L.call); the op itself
    where a gradient is recorded (it says that it has none) and for tensors without memory of their own (fake ones)."""
    if type(x) in _PLAIN:
        o = L.native(name, x, *(ACTS[a] if type(a) is str else a for a in args))
        if o is not None:
            return o
    tensors = [t for t in args if isinstance(t, torch.Tensor)]
    if any(type(t) not in _PLAIN for t in tensors) or (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)):
        return op(*args)
    return L.call(op, *args)


def _has_memory(t):
    """Whether t has memory of its own: a fake tensor, or a subclass that wraps others, has none to read."""
    return type(t).__torch_dispatch__ is torch.Tensor.__torch_dispatch__


def _call(op, t, *args):
    """L.call for a linear's own calls; the op itself, with its fake kernel, for tensors without memory (t says it for all)."""
    return L.call(op, t, *args) if torch.compiler.is_compiling() or _has_memory(t) else op(t, *args)


def _same_device(dev, **named):
    for name, t in named.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {dev}")


def _vec(t, C, batch, rows, name):
    """Rows of a modulation ([B, 1, C], [B, C] or [C]) as a bf16 [B, C] view with 16-byte rows (copied only where it is none),
    B the batch of x [B, N, C], or any divisor of a 2-D x's rows."""
    if t.shape[-1] != C:
        raise ValueError(f"{name} must have {C} columns, got {tuple(t.shape)}")
    t = t.reshape(-1, C)
    B = t.shape[0]
    if B != 1 and (B != batch if batch is not None else rows % B if B else rows):
        raise ValueError(f"{name} has {B} rows for a batch of {batch if batch is not None else rows}")
    if t.dtype != BF:
        t = t.to(BF)
    if t.stride(1) != 1 or (B > 1 and (t.stride(0) % 8 or t.stride(0) < C)) or t.data_ptr() % 16:
        t = L.aligned(t.contiguous())
    return t, B, (t.stride(0) if B > 1 else C)


def _weight_vec(w, C, name):
    if w.shape != (C,):
        raise ValueError(f"{name} must be [{C}], got {tuple(w.shape)}")
    if w.dtype not in L.DTYPE_CODE:
        w = w.float()
    return L.aligned(w.contiguous())


# ------------------------------------------------------------------------------------------------ row cast

@L.step_op("gpic::fp8_tcast_rows")
def tcast_rows_op(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., C] (any float dtype, C % 8 == 0, C <= 32768) -> (q e4m3, x's shape; s [rows] fp32): each row's own amax."""
    o = L.native("cast_rows", x, x)
    if o is not None:
        return o
    L.require_gpu(x)
    if x.dim() < 1 or x.shape[-1] % 8 or not 0 < x.shape[-1] <= CAST_MAX_C or not x.is_floating_point():
        raise ValueError(f"tcast_rows needs float x [..., C] with C % 8 == 0 and 0 < C <= {CAST_MAX_C}, got {x.dtype} "
                         f"{tuple(x.shape)}")
    C = x.shape[-1]
    x2 = x.reshape(-1, C)
    if x2.dtype not in L.DTYPE_CODE:
        x2 = x2.float()
    x2, ld = _rows(x2)
    q = torch.empty(x.shape, dtype=E4, device=x.device)
    s = torch.empty(x2.shape[0], dtype=torch.float32, device=x.device)
    with L.on_device(x.device):
        L.check(L.lib().gpic_fp8_tcast_rows(x2.data_ptr(), L.DTYPE_CODE[x2.dtype], ld, x2.shape[0], C, q.data_ptr(),
                                            s.data_ptr(), None, 0, 0, 0, None, None, L.stream_ptr(x.device)),
                "gpic_fp8_tcast_rows")
    return q, s


@tcast_rows_op.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=E4), x.new_empty(x.shape[:-1].numel(), dtype=torch.float32)


def tcast_rows(x):
    """x [..., C] (any float dtype, C % 8 == 0, C <= 32768) -> (q e4m3, x's shape; s [rows] fp32): tcast with one amax, and
    one scale, a row. A NaN in a row makes its scale NaN."""
    return _run(tcast_rows_op, "cast_rows", x, x)


class RowsWeight(NamedTuple):
    """A weight cast once by rows_weight: e4m3 [N, K] and its rows' scales [N]; swiglu: its rows in a SwiGLU's order."""
    q: torch.Tensor
    s: torch.Tensor
    swiglu: bool


def swiglu_layout(t):
    """w12's rows (or its bias) [2 H, ...], the gate's half first, in the order of act="swiglu": runs of 4 of the gate's and
    4 of its partners', so that one lane's 8 columns hold both (H % 16 == 0)."""
    if t.shape[0] % 32:
        raise ValueError(f"swiglu_layout needs 2 H rows with H % 16 == 0, got {tuple(t.shape)}")
    return t.reshape(2, t.shape[0] // 8, 4, *t.shape[1:]).transpose(0, 1).reshape(t.shape)


def rows_weight(w, act="none"):
    """A linear's weight [N, K] (w12 [2 H, K] for act="swiglu") cast once, for forward calls. A SwiGLU's rows are reordered
    (swiglu_layout), so its calls take the bias in that order too: swiglu_layout(b12), made once beside the weight."""
    if w.dim() != 2 or w.shape[0] % 16 or w.shape[1] % 16:
        raise ValueError(f"rows_weight needs w [N, K] with N % 16 == 0 and K % 16 == 0, got {tuple(w.shape)}")
    swiglu = _act(act) == ACTS["swiglu"]
    w = w.detach()
    return RowsWeight(*tcast_rows(swiglu_layout(w) if swiglu else w), swiglu)


# ------------------------------------------------------------------------------------------------ norm

@L.step_op("gpic::fp8_rmsnorm_rows")
def rmsnorm_rows_op(x: torch.Tensor, w: torch.Tensor, eps: float, a: Optional[torch.Tensor] = None,
                    gate: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                    scale: Optional[torch.Tensor] = None, want_h: bool = False
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """rmsnorm_rows, as an op."""
    o = L.native("norm_rows", x, x, w, eps, a, gate, shift, scale, want_h)
    if o is not None:
        return o
    L.require_gpu(x, w, a, gate, shift, scale)
    if x.dim() < 2 or x.dtype != BF or x.shape[-1] % 8 or not 0 < x.shape[-1] <= NORM_MAX_C:
        raise ValueError(f"rmsnorm_rows takes bf16 x [..., C] with C % 8 == 0 and 0 < C <= {NORM_MAX_C}, got {x.dtype} "
                         f"{tuple(x.shape)}")
    if a is not None and a.shape != x.shape:
        raise ValueError(f"a must have x's shape {tuple(x.shape)}, got {tuple(a.shape)}")
    if gate is not None and a is None:
        raise ValueError("gate needs a")
    if (shift is None) != (scale is None):
        raise ValueError("shift and scale come together")
    dev, C = x.device, x.shape[-1]
    _same_device(dev, w=w, a=a, gate=gate, shift=shift, scale=scale)
    x2, ldx = _rows(x.reshape(-1, C))
    M = x2.shape[0]
    batch = x.shape[0] if x.dim() > 2 else None
    a2, lda = _rows(a.to(BF).reshape(-1, C)) if a is not None else (None, 0)
    wc = _weight_vec(w, C, "w")
    vecs, Bs = {}, set()
    for name, t in (("gate", gate), ("shift", shift), ("scale", scale)):
        v, B, ld = _vec(t, C, batch, M, name) if t is not None else (None, None, 0)
        vecs[name] = (v, ld)
        if B is not None:
            Bs.add(B)
    if len(Bs) > 1:
        raise ValueError("gate, shift and scale must have the same number of rows")
    ntok = max(M // max(Bs.pop() if Bs else 1, 1), 1)
    xn = torch.empty(x.shape, dtype=BF, device=dev) if a is not None else x.new_empty(0)
    h = torch.empty(x.shape, dtype=BF, device=dev) if want_h else x.new_empty(0)
    q = torch.empty(x.shape, dtype=E4, device=dev)
    s = torch.empty(M, dtype=torch.float32, device=dev)
    rstd = torch.empty(M, dtype=torch.float32, device=dev)
    (g, sg), (sh, ssh), (sc, ssc) = vecs["gate"], vecs["shift"], vecs["scale"]
    with L.on_device(dev):
        L.check(L.lib().gpic_fp8_rmsnorm_rows(
            x2.data_ptr(), ldx, L.ptr(a2), lda, L.ptr(g), sg, wc.data_ptr(), L.DTYPE_CODE[wc.dtype], L.ptr(sh), ssh,
            L.ptr(sc), ssc, M, ntok, C, float(eps), xn.data_ptr() if a is not None else None,
            h.data_ptr() if want_h else None, rstd.data_ptr(), q.data_ptr(), s.data_ptr(), None, 0, 0, None, None,
            L.stream_ptr(dev)), "gpic_fp8_rmsnorm_rows")
    return xn, h, q, s, rstd


@rmsnorm_rows_op.register_fake
def _(x, w, eps, a=None, gate=None, shift=None, scale=None, want_h=False):
    M = x.shape[:-1].numel()
    return (x.new_empty(x.shape) if a is not None else x.new_empty(0), x.new_empty(x.shape) if want_h else x.new_empty(0),
            x.new_empty(x.shape, dtype=E4), x.new_empty(M, dtype=torch.float32), x.new_empty(M, dtype=torch.float32))


def rmsnorm_rows(x, w, eps, a=None, gate=None, shift=None, scale=None, want_h=False):
    """x_new = x + gate a (without a: x; without gate: x + a), h = RMSNorm(x_new) w (1 + scale) + shift (both or neither) ->
    (x_new bf16, empty without a; h bf16, empty unless want_h; h's e4m3 bytes; their scales [rows]; rstd [rows]).
    x, a [..., C] bf16, C % 8 == 0, C <= 16384; w [C]; gate, shift, scale [B, 1, C] for x [B, N, C] (or one row for all;
    for x [M, C] any number of rows that divides M). h is rounded once, to e4m3 (and once, to bf16, for want_h)."""
    return _run(rmsnorm_rows_op, "norm_rows", x, x, w, eps, a, gate, shift, scale, want_h)


@L.step_op("gpic::fp8_rmsnorm_rows_bwd")
def rmsnorm_rows_bwd_op(dh: torch.Tensor, dxn: Optional[torch.Tensor], xs: torch.Tensor, w: torch.Tensor,
                        rstd: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """rmsnorm_rows_bwd, as an op."""
    o = L.native("norm_rows_bwd", xs, dh, dxn, xs, w, rstd)
    if o is not None:
        return o
    L.require_gpu(dh, dxn, xs, w, rstd)
    if xs.dim() < 1 or xs.dtype != BF or xs.shape[-1] % 8 or not 0 < xs.shape[-1] <= NORM_MAX_C:
        raise ValueError(f"rmsnorm_rows_bwd takes bf16 xs [..., C] with C % 8 == 0 and 0 < C <= {NORM_MAX_C}, got {xs.dtype} "
                         f"{tuple(xs.shape)}")
    dev, C = xs.device, xs.shape[-1]
    _same_device(dev, dh=dh, dxn=dxn, w=w, rstd=rstd)
    M = xs.numel() // C
    if dh.shape != xs.shape or (dxn is not None and dxn.shape != xs.shape):
        raise ValueError(f"dh and dxn must have xs's shape {tuple(xs.shape)}")
    if rstd.numel() != M or rstd.dtype != torch.float32:
        raise ValueError(f"rstd must be fp32 with {M} elements, got {rstd.dtype} {tuple(rstd.shape)}")
    dhc, xc = L.aligned(dh.to(BF).contiguous()), L.aligned(xs.contiguous())
    nc = L.aligned(dxn.to(BF).contiguous()) if dxn is not None else None
    wc, rc = _weight_vec(w, C, "w"), rstd.contiguous()
    dx = torch.empty_like(xc)
    dw = torch.empty(C, dtype=w.dtype if w.dtype in L.DTYPE_CODE else torch.float32, device=dev)
    with L.on_device(dev):
        nws = L.lib().gpic_fp8_rmsnorm_rows_bwd_workspace_bytes(M, C)
        ws = torch.empty(max(nws, 16), dtype=torch.uint8, device=dev)
        L.check(L.lib().gpic_fp8_rmsnorm_rows_bwd(
            dhc.data_ptr(), L.ptr(nc), xc.data_ptr(), wc.data_ptr(), L.DTYPE_CODE[wc.dtype], rc.data_ptr(), M, C,
            dx.data_ptr(), dw.data_ptr(), L.DTYPE_CODE[dw.dtype], ws.data_ptr(), nws, L.stream_ptr(dev)),
            "gpic_fp8_rmsnorm_rows_bwd")
    return dx, dw


@rmsnorm_rows_bwd_op.register_fake
def _(dh, dxn, xs, w, rstd):
    return xs.new_empty(xs.shape), xs.new_empty(xs.shape[-1], dtype=w.dtype if w.dtype in L.DTYPE_CODE else torch.float32)


def rmsnorm_rows_bwd(dh, dxn, xs, w, rstd):
    """The backward of rmsnorm_rows without gate, shift and scale: dh (of h) and dxn (of x_new, or None) like xs (x_new, or
    x without a) [..., C] bf16, rstd [rows] -> (dx, which is a's gradient too, bf16; dw [C] of w's dtype, summed in fp32 in a
    fixed order)."""
    return _run(rmsnorm_rows_bwd_op, "norm_rows_bwd", xs, dh, dxn, xs, w, rstd)


# ------------------------------------------------------------------------------------------------ GEMM

def _scales(s, n, name):
    if s is None:
        return None
    if s.numel() != n or s.dtype != torch.float32:
        raise ValueError(f"{name} must be fp32 with {n} elements, got {s.dtype} {tuple(s.shape)}")
    return L.aligned(s.contiguous())


@L.step_op("gpic::fp8_gemm_rows")
def gemm_rows_op(a: torch.Tensor, sa: Optional[torch.Tensor], b: torch.Tensor, sb: Optional[torch.Tensor],
                 bias: Optional[torch.Tensor] = None, act: str = "none", residual: Optional[torch.Tensor] = None,
                 gate: Optional[torch.Tensor] = None, want_z: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """fp8_gemm_rows, as an op: (y, z as bf16 when want_z, else an empty tensor)."""
    code = _act(act)
    o = L.native("gemm_rows", a, a, sa, b, sb, bias, code, residual, gate, want_z)
    if o is not None:
        return o
    L.require_gpu(a, sa, b, sb, bias, residual, gate)
    _same_device(a.device, sa=sa, b=b, sb=sb, bias=bias, residual=residual, gate=gate)
    a, b = _gemm_operand(a, "a"), _gemm_operand(b, "b")
    (M, K), N = a.shape, b.shape[0]
    half = code == ACTS["swiglu"]
    if b.shape[1] != K or K == 0 or K % 16 or N % (32 if half else 16):
        raise ValueError(f"fp8_gemm_rows needs a [M, K], b [N, K] with K % 16 == 0, K > 0 and N % 16 == 0 (swiglu: 32), got "
                         f"{tuple(a.shape)} and {tuple(b.shape)}")
    No = N // 2 if half else N
    dev = a.device
    sa, sb = _scales(sa, M, "sa"), _scales(sb, N, "sb")
    if bias is not None:
        bias = _weight_vec(bias, N, "bias")
    ldr = No
    batch = None
    if residual is not None:
        if residual.shape[-1] != No or residual.numel() != M * No:
            raise ValueError(f"residual must be [{M}, {No}], got {tuple(residual.shape)}")
        residual, ldr = _rows(residual.to(BF).reshape(-1, No))
    g, sg, ntok = None, 0, 1
    if gate is not None:
        g, B, sg = _vec(gate, No, batch, M, "gate")
        ntok = max(M // max(B, 1), 1)
    y = torch.empty(M, No, dtype=BF, device=dev)
    z = torch.empty((M, N) if want_z else (0,), dtype=BF, device=dev)
    lda = a.stride(0) if M > 1 else max(a.stride(0), K) // 16 * 16
    ldb = b.stride(0) if N > 1 else K
    with L.on_device(dev):
        nws = L.gemm_workspace_bytes(dev, M, N, K)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws else None
        L.check(L.lib().gpic_fp8_gemm_rows(
            a.data_ptr(), lda, L.ptr(sa), b.data_ptr(), ldb, L.ptr(sb), L.ptr(bias),
            L.DTYPE_CODE[bias.dtype] if bias is not None else 0, code, L.ptr(residual), ldr, L.ptr(g), sg, ntok,
            y.data_ptr(), No, z.data_ptr() if want_z else None, N, M, N, K, L.ptr(ws), nws, L.stream_ptr(dev)),
            "gpic_fp8_gemm_rows")
    return y, z


@gemm_rows_op.register_fake
def _(a, sa, b, sb, bias=None, act="none", residual=None, gate=None, want_z=False):
    M, N = a.shape[0], b.shape[0]
    return (a.new_empty(M, N // 2 if act == "swiglu" else N, dtype=BF),
            a.new_empty((M, N) if want_z else (0,), dtype=BF))


def fp8_gemm_rows(a, sa, b, sb, bias=None, act="none", residual=None, gate=None):
    """a [M, K], b [N, K] e4m3 with their rows' scales sa [M], sb [N] fp32 (None: ones) ->
    y [M, N] bf16 = residual + gate act(sa sb a b^T + bias), in fp32 and rounded once. act: "none", "silu", "gelu_tanh", or
    "swiglu" (b's rows as rows_weight(w12, "swiglu") lays them out, and sb and bias in the same order: swiglu_layout(b12);
    y [M, N / 2]). bias [N] bf16 or fp32; residual [M, N]
    bf16; gate [B, 1, N] bf16, B dividing M: a block's gate, one row for M / B rows of y."""
    _act(act)
    return _run(gemm_rows_op, "gemm_rows", a, a, sa, b, sb, bias, act, residual, gate, False)[0]


@L.step_op("gpic::fp8_act_bwd_rows")
def act_bwd_rows_op(dy: torch.Tensor, z: Optional[torch.Tensor], act: str, sw: torch.Tensor,
                    wq: Optional[torch.Tensor] = None, want_db: bool = False, db32: bool = False
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """act_bwd_rows, as an op: (dz, empty for act="none"; q; s; wq [N, K]'s bytes transposed [K, N16]; the sum of dz over the
    rows, bf16 or db32), the last two empty unless asked for."""
    L.require_gpu(dy, z, sw, wq)
    code = _act(act, train=True)
    if dy.dim() != 2 or dy.dtype != BF or dy.shape[1] % 8 or not 0 < dy.shape[1] <= CAST_MAX_C:
        raise ValueError(f"act_bwd_rows takes bf16 dy [M, N] with N % 8 == 0 and 0 < N <= {CAST_MAX_C}, got {dy.dtype} "
                         f"{tuple(dy.shape)}")
    M, N = dy.shape
    dev = dy.device
    _same_device(dev, z=z, sw=sw, wq=wq)
    if code and (z is None or z.shape != dy.shape or z.dtype != BF):
        raise ValueError("act_bwd_rows needs the forward's bf16 z, of dy's shape")
    if wq is not None and (wq.dtype != E4 or wq.dim() != 2 or wq.shape[0] != N or wq.shape[1] % 16):
        raise ValueError(f"wq must be e4m3 [{N}, K] with K % 16 == 0, got {wq.dtype} {tuple(wq.shape)}")
    sw = _scales(sw, N, "sw")
    dy, ldy = _rows(dy)
    z, ldz = _rows(z) if code else (None, 0)
    dz = torch.empty((M, N) if code else (0,), dtype=BF, device=dev)
    q = torch.empty(M, N, dtype=E4, device=dev)
    s = torch.empty(M, dtype=torch.float32, device=dev)
    K = 0 if wq is None else wq.shape[1]
    wq = None if wq is None else L.aligned(wq.contiguous())
    wqt = torch.empty((0,) if wq is None else (K, _r16(N)), dtype=E4, device=dev)
    db = torch.empty(N if want_db else 0, dtype=torch.float32 if db32 else BF, device=dev)
    with L.on_device(dev):
        nws = L.lib().gpic_fp8_act_bwd_rows_workspace_bytes(M, N) if want_db else 0
        ws = torch.empty(max(nws, 16), dtype=torch.uint8, device=dev) if want_db else None
        L.check(L.lib().gpic_fp8_act_bwd_rows(
            dy.data_ptr(), ldy, L.ptr(z), ldz, code, sw.data_ptr(), M, N, dz.data_ptr() if code else None, q.data_ptr(),
            s.data_ptr(), L.ptr(wq), K, wqt.data_ptr() if wq is not None else None, _r16(N),
            db.data_ptr() if want_db else None, L.DTYPE_CODE[db.dtype], L.ptr(ws), nws, L.stream_ptr(dev)),
            "gpic_fp8_act_bwd_rows")
    return dz, q, s, wqt, db


@act_bwd_rows_op.register_fake
def _(dy, z, act, sw, wq=None, want_db=False, db32=False):
    N = dy.shape[1]
    return (dy.new_empty(dy.shape if act != "none" else (0,)), dy.new_empty(dy.shape, dtype=E4),
            dy.new_empty(dy.shape[0], dtype=torch.float32),
            dy.new_empty((0,) if wq is None else (wq.shape[1], _r16(N)), dtype=E4),
            dy.new_empty(N if want_db else 0, dtype=torch.float32 if db32 else BF))


def act_bwd_rows(dy, z, act, sw):
    """dy [M, N] bf16 and the forward's z [M, N] bf16 (unused for act="none") -> (dz = dy act'(z) as bf16, dy itself for
    "none"; dz sw as e4m3; its scales [M]): the operands of the weight's gradient and, against the weight's bytes
    transposed, of the dgrad (sw [N]: the weight's scales, which lie on its reduction)."""
    dz, q, s, _, _ = _run(act_bwd_rows_op, None, None, dy, z, act, sw)
    return (dy if act == "none" else dz), q, s


# ------------------------------------------------------------------------------------------------ linears

def _linear_bwd(ctx, dy2, z, wq, sw, x2, need_dx, need_dw, need_db):
    """(dx [M, K] bf16, dw, db) of y = act(x w^T + b), each None unless needed."""
    r = None
    if _has_memory(dy2):
        r = L.native("linear_rows_bwd", dy2, dy2, z, ACTS[ctx.act], wq, sw, x2, need_dx, need_dw, need_db,
                     ctx.wdt == torch.float32, ctx.bdt == torch.float32)
    if r is not None:
        dx, dw, db = r
        return dx, dw if dw is None else dw.to(ctx.wdt), db if db is None else db.to(ctx.bdt)
    dz, dq, sd, wqt, db = _call(act_bwd_rows_op, dy2, z, ctx.act, sw, wq if need_dx else None, need_db,
                                ctx.bdt == torch.float32)
    if ctx.act == "none":
        dz = dy2
    dx = _call(gemm_rows_op, dq, sd, wqt, None)[0] if need_dx else None
    dw = _call(bf16_wgrad, dz, x2, ctx.wdt == torch.float32).to(ctx.wdt) if need_dw else None
    return dx, dw, db.to(ctx.bdt) if need_db else None


def _once(backward):
    """once_differentiable, with a warning where a backward under create_graph=True returns constants that are none (the last
    input's gradient, a residual's, is y's own): a term made of them would be lost without a word from a sum whose other terms
    have a gradient."""
    inner = once_differentiable(backward)

    @functools.wraps(backward)
    def call(ctx, *grads):
        if (torch.is_grad_enabled() and not torch.compiler.is_compiling() and grads[-1] is not None
                and any(ctx.needs_input_grad[:-1]) and not any(g is not None and g.requires_grad for g in grads)):
            warnings.warn("the row-scaled linears are differentiable once: the gradients of a backward under create_graph=True "
                          "do not require a gradient, and a loss made of them has none through these linears")
        return inner(ctx, *grads)
    return call


class _LinearRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, act, residual):
        x2 = x.reshape(-1, x.shape[-1])
        xq, sx = _call(tcast_rows_op, x2)
        wq, sw = _call(tcast_rows_op, w)
        y, z = _call(gemm_rows_op, xq, sx, wq, sw, b, act, None if residual is None else residual.reshape(-1, w.shape[0]), None,
                     act != "none" and any(ctx.needs_input_grad))
        ctx.save_for_backward(x2, z, wq, sw)
        ctx.set_materialize_grads(False)
        ctx.act, ctx.wdt, ctx.bdt, ctx.shape = act, w.dtype, None if b is None else b.dtype, x.shape
        return y.view(*x.shape[:-1], w.shape[0])

    @staticmethod
    @_once
    def backward(ctx, dy):
        x2, z, wq, sw = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if dy is None:
            return None, None, None, None, None
        if any(need[:3]):
            dx, dw, db = _linear_bwd(ctx, dy.reshape(-1, dy.shape[-1]).to(BF), z, wq, sw, x2, *need[:3])
        return dx.view(ctx.shape) if need[0] else None, dw, db, None, dy if need[4] else None


class _NormLinearRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, gate, wn, shift, scale, eps, w, b, act):
        C = x.shape[-1]
        train = any(ctx.needs_input_grad)
        want_z = train and act != "none"
        r = None
        if _has_memory(x):
            r = L.native("norm_linear_rows_fwd", x, x, wn, eps, a, gate, shift, scale, w, b, ACTS[act], train, want_z)
        if r is not None:
            xn, h, rstd, y, z, wq, sw = r
        else:
            xn, h, hq, sh, rstd = _call(rmsnorm_rows_op, x, wn, eps, a, gate, shift, scale, train)
            wq, sw = _call(tcast_rows_op, w)
            y, z = _call(gemm_rows_op, hq.view(-1, C), sh, wq, sw, b, act, None, None, want_z)
        xs = x if a is None else xn
        ctx.save_for_backward(xs, a if gate is not None else None, gate, wn, shift, scale, rstd,
                              h.view(-1, C) if train else None, z, wq, sw)
        ctx.set_materialize_grads(False)
        ctx.act, ctx.wdt, ctx.bdt = act, w.dtype, None if b is None else b.dtype
        y = y.view(*x.shape[:-1], w.shape[0])
        return y if a is None else (xn, y)

    @staticmethod
    @_once
    def backward(ctx, *grads):
        xs, a, gate, wn, shift, scale, rstd, h, z, wq, sw = ctx.saved_tensors
        dxn, dy = grads if len(grads) == 2 else (None, grads[0])
        need = ctx.needs_input_grad
        if dy is None:
            if dxn is None:
                return (None,) * 10
            # x_new alone was used: its gradient as it is, and zeros that no value of h or z can spoil (gate's and a's by the
            # norm's backward of zero rows, whose dx is dxn)
            zeros = lambda t, dtype=None: torch.zeros_like(t, dtype=dtype)  # noqa: E731
            dx = da = dxn.to(BF)
            dgate = None
            if gate is not None and (need[1] or need[2]):
                none = zeros(xs)
                _, da, dg, *_ = _call(res_mod_rmsnorm_bwd_k, none, dx, none, a, gate, zeros(wn), zeros(scale), zeros(rstd))
                dgate = dg.view(gate.shape).to(gate.dtype)
            return (dx if need[0] else None, da if need[1] else None, dgate if need[2] else None,
                    *[zeros(t) if n else None for t, n in zip((wn, shift, scale), need[3:6])], None,
                    zeros(wq, ctx.wdt) if need[7] else None,
                    sw.new_zeros(wq.shape[0], dtype=ctx.bdt) if need[8] else None, None)
        below = any(need[:6])   # a gradient through the norm
        dy2 = dy.reshape(-1, dy.shape[-1]).to(BF)
        dx = da = dgate = dwn = dshift = dscale = None
        dh, dw, db = _linear_bwd(ctx, dy2, z, wq, sw, h, below, need[7], need[8])
        if below and shift is None:
            dx, dwn = _call(rmsnorm_rows_bwd_op, dh.view(xs.shape), dxn, xs, wn, rstd)
            dwn, da = dwn.to(wn.dtype), dx
        elif below:
            dx, da, dg, dwn, dsh, dsc = _call(res_mod_rmsnorm_bwd_k, dh.view(xs.shape), dxn, xs, a, gate, wn, scale, rstd)
            dwn = dwn.to(wn.dtype)
            dshift, dscale = dsh.view(shift.shape).to(shift.dtype), dsc.view(scale.shape).to(scale.dtype)
            dgate = dg.view(gate.shape).to(gate.dtype) if gate is not None else None
        out = [dx, da, dgate, dwn, dshift, dscale, None, dw, db, None]
        return tuple(g if n else None for g, n in zip(out, need))


def _check_linear(x, weight, act, train):
    _act(act, train)
    w = weight.q if isinstance(weight, RowsWeight) else weight
    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1] or w.shape[0] % 16 or w.shape[1] % 16:
        raise ValueError(f"the linear needs x [..., K] and a weight [N, K] with K % 16 == 0 and N % 16 == 0, got "
                         f"{tuple(x.shape)} and {tuple(w.shape)}")
    if isinstance(weight, RowsWeight):
        if weight.swiglu != (act == "swiglu"):
            raise ValueError('a weight for act="swiglu" is cast by rows_weight(w12, "swiglu"), and no other is')
    elif w.shape[0] > CAST_MAX_C or w.shape[1] > CAST_MAX_C:
        raise ValueError(f"the linear takes at most {CAST_MAX_C} features in and out, got {tuple(w.shape)}")


def _no_gradient(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("a RowsWeight is for forward calls: give the weight itself, or call under torch.no_grad()")


def fp8_linear_rows(x, weight, bias=None, act="none", residual=None, gate=None):
    """residual + gate act(x weight^T + bias), x [..., K] -> [..., N] bf16, with row-scaled e4m3 operands. weight [N, K]:
    differentiable (the forward and the dgrad in FP8, the weight's gradient in bf16; act none, silu or gelu_tanh; no gate).
    weight a RowsWeight (rows_weight): forward only, with act="swiglu" (N / 2 columns) and gate as well: [B, 1, N] for x
    [B, ..., K], or one row for all; for x [M, K] any number of rows that divides M. act="swiglu": bias is
    swiglu_layout(b12), w12's bias in the order of the RowsWeight's rows."""
    serving = isinstance(weight, RowsWeight)
    _check_linear(x, weight, act, not serving)
    if serving and type(x) in _PLAIN:
        y = L.native("linear_served", x, x, weight.q, weight.s, bias, ACTS[act], residual, gate)
        if y is not None:
            return y
    with _no_autocast():
        x = x.to(BF)
        if residual is not None:
            residual = residual.to(BF)
        if not serving:
            if gate is not None:
                raise ValueError("gate needs a RowsWeight")
            if residual is not None and residual.shape != (*x.shape[:-1], weight.shape[0]):
                raise ValueError(f"residual must be {(*x.shape[:-1], weight.shape[0])}, got {tuple(residual.shape)}")
            if type(x) in _PLAIN and type(weight) in _PLAIN:   # (the usual form, recorded or not)
                y = L.native("linear_rows", x, x, weight, bias, ACTS[act], residual)
                if y is not None:
                    return y
            return _LinearRows.apply(x, weight, bias, act, residual)
        _no_gradient(x, weight.q, weight.s, bias, residual, gate)
        K, N = x.shape[-1], weight.q.shape[0] // (2 if weight.swiglu else 1)
        if residual is not None:
            if residual.shape != (*x.shape[:-1], N):
                raise ValueError(f"residual must be {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
            residual = residual.reshape(-1, N)
        if gate is not None and x.dim() > 2 and gate.numel() not in (N, x.shape[0] * N):
            raise ValueError(f"gate has {gate.numel() // N} rows of {N} for a batch of {x.shape[0]}")
        q, s = _call(tcast_rows_op, x.reshape(-1, K))
        y = _call(gemm_rows_op, q, s, weight.q, weight.s, bias, act, residual, gate)[0]
        return y.view(*x.shape[:-1], N)


def fp8_rmsnorm_linear_rows(x, w_norm, eps, weight, bias=None, act="none", a=None, gate=None, shift=None, scale=None):
    """(x_new, act(h weight^T + bias)) for x_new, h of rmsnorm_rows(x, w_norm, eps, a, gate, shift, scale); x_new is x without
    a. h goes to the GEMM as the norm's bytes. weight as in fp8_linear_rows; with a gradient: a with gate, shift and scale,
    or a alone, or neither, or shift and scale alone (then C <= 2048). act="swiglu": bias is swiglu_layout(b12)."""
    serving = isinstance(weight, RowsWeight)
    _check_linear(x, weight, act, not serving)
    if serving and type(x) in _PLAIN:
        r = L.native("norm_linear_served", x, x, w_norm, eps, a, gate, shift, scale, weight.q, weight.s, bias, ACTS[act])
        if r is not None:
            return (x if a is None else r[0]), r[1]
    with _no_autocast():
        x = x.to(BF)
        if a is not None:
            a = a.to(BF)
        if serving:
            _no_gradient(x, w_norm, weight.q, weight.s, bias, a, gate, shift, scale)
            xn, _, q, s, _ = _call(rmsnorm_rows_op, x, w_norm, eps, a, gate, shift, scale)
            y = _call(gemm_rows_op, q.view(-1, x.shape[-1]), s, weight.q, weight.s, bias, act)[0]
            return (x if a is None else xn), y.view(*x.shape[:-1], y.shape[-1])
        if shift is not None or gate is not None:
            if shift is None or (a is not None and gate is None):
                raise ValueError("with a weight that is not a RowsWeight: gate, shift and scale (and a), or shift and scale "
                                 "without a, or none of them")
            if x.dim() != 3 or any(t is not None and t.numel() != x.shape[0] * x.shape[-1] for t in (gate, shift, scale)):
                raise ValueError("gate, shift and scale [B, 1, C] need x [B, N, C]")
            if x.shape[-1] > BWD_MAX_C:
                raise ValueError(f"the modulated norm's backward takes rows of at most {BWD_MAX_C}, got C = {x.shape[-1]}")
        elif type(x) in _PLAIN and type(weight) in _PLAIN:
            r = L.native("norm_linear_rows", x, x, w_norm, eps, a, weight, bias, ACTS[act])
            if r is not None:
                return (x if a is None else r[0]), r[1]
        out = _NormLinearRows.apply(x, a, gate, w_norm, shift, scale, eps, weight, bias, act)
        return (x, out) if a is None else out

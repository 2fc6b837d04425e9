"""Plain 64-bit statements of the row-scaled operators, and the bounds their tests hold the kernels to."""
import math

import torch

E4, BF, F32, F64 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float64
U32 = 2.0 ** -24           # half a step of fp32, relative
UBF = 2.0 ** -8            # of bf16
UE4, SUB4 = 2.0 ** -4, 2.0 ** -10   # of e4m3: relative, and of its subnormals (steps of 2^-9)


def rowq(h):
    """The row cast of fp32 h on the CPU, IEEE fp32 throughout: (q, s)."""
    h = h.float().cpu()
    a = h.abs().amax(-1, keepdim=True).clamp_min(1e-12)
    k = torch.full_like(a, 448.0)
    return (h * (k / a)).clamp(-448.0, 448.0).to(E4), (a / k).squeeze(-1)


def deq(q, s):
    return q.double() * s.double().view(*q.shape[:-1], 1)


def sigmoid(z):
    return 1.0 / (1.0 + torch.exp(-z))


def act(z, name):
    if name == "silu":
        return z * sigmoid(z)
    if name == "gelu_tanh":
        return z * sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    if name == "swiglu":
        v = z.reshape(z.shape[0], -1, 2, 4)
        return (v[:, :, 0] * sigmoid(v[:, :, 0]) * v[:, :, 1]).reshape(z.shape[0], -1)
    return z


def dact(z, name):
    if name == "silu":
        p = sigmoid(z)
        return p * (1 + z * (1 - p))
    if name == "gelu_tanh":
        c = 2.0 * math.sqrt(2.0 / math.pi)
        p = sigmoid(c * (z + 0.044715 * z ** 3))
        return p + z * p * (1 - p) * c * (1 + 0.134145 * z ** 2)
    return torch.ones_like(z)


def gemm(a, sa, b, sb, bias=None, name="none", res=None, gate=None, slack=2.0 ** -16):
    """(y, how far a kernel's may be off) of fp8_gemm_rows in 64 bits. z carries `slack` of the sum of |terms| (the MFMA's
    summation of a block of 128 products, parity.assert_elementwise's allowance) and 4 fp32 roundings; an activation's slope is
    at most 1.13 (SwiGLU: 1.1 |z2| and |silu(z1)|) and its own value 16 fp32 roundings off (|z| 2^-24 in e^z for |z| <= 8, the
    hardware's two functions, the products); gate and residual two more; then one bf16 rounding."""
    one = torch.ones((), dtype=F64, device=a.device)
    sa = one if sa is None else sa.double()[:, None]
    sb = one if sb is None else sb.double()
    A, B = a.double() * sa, b.double() * (sb[:, None] if sb.dim() else sb)
    z = A @ B.t()
    ez = (A.abs() @ B.abs().t()) * slack
    if bias is not None:
        z = z + bias.double()
        ez = ez + bias.double().abs() * U32
    ez = ez + 4 * U32 * z.abs()
    y = act(z, name)
    if name == "swiglu":
        v, e = z.reshape(z.shape[0], -1, 2, 4), ez.reshape(z.shape[0], -1, 2, 4)
        sl = v[:, :, 0] * sigmoid(v[:, :, 0])
        ey = (1.1 * v[:, :, 1].abs() * e[:, :, 0] + sl.abs() * e[:, :, 1] + 1.1 * e[:, :, 0] * e[:, :, 1]).reshape(y.shape)
    else:
        ey = (1.0 if name == "none" else 1.13) * ez
    if name != "none":
        ey = ey + y.abs() * U32 * (16 + z.abs().max().item())
    if gate is not None:
        g = gate.double().reshape(-1, y.shape[1])
        g = g.repeat_interleave(y.shape[0] // g.shape[0], 0)
        y, ey = y * g, ey * g.abs() + (y * g).abs() * U32
    if res is not None:
        y = y + res.double()
        ey = ey + y.abs() * U32
    return y, ey + (y.abs() + ey) * UBF + 1e-38


def within(x, ref, bound, what=""):
    err = (x.double() - ref).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst excess {(err - bound).max().item():.3g}"


def norm(x, w, eps, a=None, gate=None, shift=None, scale=None):
    """(x_new bf16, rstd, h, the magnitude h's error is relative to) in 64 bits; gate, shift, scale [B, C] with B dividing the
    rows of x [M, C]."""
    M = x.shape[0]
    rep = lambda t: t.double().reshape(-1, x.shape[1]).repeat_interleave(M // t.reshape(-1, x.shape[1]).shape[0], 0)  # noqa: E731
    xn = x
    if a is not None:
        xn = (x.double() + (rep(gate) * a.double() if gate is not None else a.double())).to(F32).to(BF)
    v = xn.double()
    rstd = (v.square().mean(-1, keepdim=True) + eps) ** -0.5
    n = w.double() * v * rstd
    h, mag = n, n.abs()
    if shift is not None:
        h = n * (1 + rep(scale)) + rep(shift)
        mag = n.abs() * (1 + rep(scale)).abs() + rep(shift).abs()
    return xn, rstd.squeeze(-1), h, mag


def check_rowq(q, s, h, eps_h):
    """q, s as the row cast of h (64 bits, known to eps_h): the scale of the row's largest within that row's largest error and
    two roundings; each value within half a step of e4m3 (4 roundings of fp32 ahead of it)."""
    a = h.abs().amax(-1).clamp_min(1e-12)
    within(s, a / 448, (eps_h.amax(-1) + 2 * U32 * a) / 448, "scales")
    s = s.double()[:, None]
    within(q.double() * s, h, (torch.maximum(h.abs() * UE4, s * SUB4) + eps_h) * (1 + 8 * U32) + 4 * U32 * h.abs(), "bytes")


def norm_f64(x, w, eps):
    """RMSNorm of 64-bit x and w, nothing rounded."""
    return w * x * (x.square().mean(-1, keepdim=True) + eps) ** -0.5

"""The row-scaled operators (gpic_fp8.rows) against their 64-bit statements (rows_ref.py), on the GPU."""
import math
import warnings

import pytest
import torch

import gpic_fp8 as G
import rows_ref as R
from gpic_fp8 import _lib as L
from gpic_fp8 import rows as GR

pytestmark = pytest.mark.gpu
E4, BF, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32
U = R.U32


def gen(dev, seed=0):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape, std=1.0, dtype=BF):
    return (torch.randn(*shape, generator=g, device=g.device) * std).to(dtype)


def u8(t):
    return t.contiguous().view(torch.uint8).cpu()


# ------------------------------------------------------------------------------------------------ row cast

@pytest.mark.parametrize("dtype", [BF, F32, torch.float16])
@pytest.mark.parametrize("rows,C", [(1, 8), (1, 1024), (3, 16), (5, 504), (7, 512), (9, 520), (130, 1000), (33, 2048),
                                    (6, 2056), (5, 4104), (4, 8192), (3, 8200), (2, 16392), (3, 32768)])
def test_tcast_rows_bytes(dev, rows, C, dtype):
    x = randn(gen(dev), rows, C, dtype=dtype) * (10.0 ** torch.arange(rows, device=dev).clamp(max=3))[:, None].to(dtype)
    q, s = G.tcast_rows(x)
    rq, rs = R.rowq(x)
    assert q.shape == x.shape and torch.equal(s.cpu(), rs) and torch.equal(u8(q), u8(rq))


def test_tcast_rows_special_rows(dev):
    """Zeros; tiny; the largest; a NaN, and an infinity, anywhere in the row, also in another lane's and wave's part."""
    for C in (64, 1024, 5000 // 8 * 8, 20000):
        x = randn(gen(dev), 9, C, dtype=F32)
        x[0] = 0
        x[1] = 1e-30
        x[2] = 3e38
        x[3, 5] = math.nan
        x[4, C - 1] = math.nan
        x[5, C // 2] = math.inf
        x[6, :] = math.nan
        x[7, 0] = -math.inf
        q, s = G.tcast_rows(x)
        s = s.cpu()
        assert torch.isnan(s[[3, 4, 6]]).all() and torch.isinf(s[[5, 7]]).all() and torch.isfinite(s[[0, 1, 2, 8]]).all()
        ok = [0, 1, 2, 8]
        rq, rs = R.rowq(x[ok])
        assert torch.equal(s[ok], rs) and torch.equal(u8(q)[ok], u8(rq))
        assert (q[0].float() == 0).all() and s[0] == torch.tensor(1e-12) / 448


def test_tcast_rows_strides(dev):
    g = gen(dev)
    big = randn(g, 12, 2080)
    for x in (big[:, 16:1040], big[::2, :1024], big[1:2, 8:1032], big.t()[:1024, :8], big[:, 1:1025], big[:0, :64],
              randn(g, 2, 3, 64).transpose(0, 1), randn(g, 64)[None].expand(5, 64)):
        q, s = G.tcast_rows(x)
        rq, rs = R.rowq(x)
        assert q.shape == x.shape and q.is_contiguous()
        assert torch.equal(s.cpu(), rs.reshape(-1)) and torch.equal(u8(q), u8(rq))
    one = torch.randn(40, device=dev, dtype=BF)[None, 8:24]      # a single row whose stride is no multiple of anything
    q, s = G.tcast_rows(one)
    assert torch.equal(u8(q), u8(R.rowq(one)[0]))


def test_tcast_rows_past_32_bits(dev):
    """Rows whose offset passes 2^31 elements."""
    C, rows = 8192, 2 ** 18 + 3
    x = torch.zeros(rows, C, dtype=BF, device=dev)
    x[-4:] = randn(gen(dev), 4, C)
    q, s = G.tcast_rows(x)
    rq, rs = R.rowq(x[-5:])
    assert torch.equal(s[-5:].cpu(), rs) and torch.equal(u8(q[-5:]), u8(rq))
    assert not q[:1000].view(torch.uint8).any()


# ------------------------------------------------------------------------------------------------ norm

def eps_of(C, mag):
    """h's fp32 error, relative to `mag`: the sum's chain (C / 64 terms a lane at most, the butterfly, 16 waves), halved by the
    root, and 12 roundings."""
    return mag * (C / 64 + 48) * U


MODES = ["plain", "res", "res_gate", "mod", "res_mod", "res_gate_mod"]


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("B,N,C", [(1, 1, 8), (1, 1, 1024), (2, 3, 16), (3, 5, 520), (2, 33, 896), (4, 17, 1024),
                                   (2, 5, 1792), (1, 7, 2048), (2, 3, 2056), (1, 3, 4096), (1, 5, 6152), (1, 2, 16384)])
def test_rmsnorm_rows(dev, mode, B, N, C):
    g = gen(dev, C + N)
    x, a = randn(g, B, N, C, std=2.0), randn(g, B, N, C)
    w = (1 + 0.1 * torch.randn(C, generator=g, device=dev)).to(F32 if N % 2 else BF)
    m = randn(g, B, 1, 3 * C, std=0.3).chunk(3, dim=-1)
    kw = dict(a=a if "res" in mode else None, gate=m[0] if "gate" in mode else None,
              shift=m[1] if "mod" in mode else None, scale=m[2] if "mod" in mode else None)
    xn, h16, q, s, rstd = G.rmsnorm_rows(x, w, 1e-6, want_h=True, **kw)
    flat = {k: v.reshape(-1, C) if v is not None else None for k, v in kw.items()}
    rxn, rr, rh, mag = R.norm(x.reshape(-1, C), w, 1e-6, **flat)
    if kw["a"] is not None:
        assert torch.equal(xn.reshape(-1, C), rxn)
    else:
        assert xn.numel() == 0
    R.within(rstd, rr, rr * (C / 64 + 32) * U, "rstd")
    eps = eps_of(C, mag)
    R.check_rowq(q.reshape(-1, C), s, rh, eps)
    R.within(h16.reshape(-1, C), rh, rh.abs() * R.UBF + eps * (1 + R.UBF), "h")
    q2 = G.rmsnorm_rows(x, w, 1e-6, **kw)
    assert q2[1].numel() == 0 and torch.equal(u8(q2[2]), u8(q)) and torch.equal(q2[3], s)


def test_rmsnorm_rows_forms(dev):
    """Strided rows, one modulation row for all, several for a 2-D x, no rows, NaN and zero rows."""
    g = gen(dev)
    big, w = randn(g, 24, 2048), torch.ones(512, device=dev)
    x, a = big[:, 512:1024], big[:, 1024:1536]
    sh, sc = randn(g, 4, 512, std=0.2), randn(g, 4, 512, std=0.2)
    for B in (1, 4):
        kw = dict(a=a, shift=sh[:B], scale=sc[:B])
        _, _, q, s, _ = G.rmsnorm_rows(x, w, 1e-6, **kw)
        _, _, rh, mag = R.norm(x, w, 1e-6, **kw)
        R.check_rowq(q, s, rh, eps_of(512, mag))
    out = G.rmsnorm_rows(x[:0], w, 1e-6, a=a[:0])
    assert [t.shape[0] for t in out] == [0, 0, 0, 0, 0]
    x = x.contiguous()
    x[3, 7], x[5] = math.nan, 0
    _, _, q, s, rstd = G.rmsnorm_rows(x, w, 1e-6)
    assert torch.isnan(s[3]) and torch.isfinite(s[[2, 4, 5]]).all() and not q[5].float().any()
    assert abs(rstd[5].item() - 1e3) < 1e-2


@pytest.mark.parametrize("dxn", [False, True])
@pytest.mark.parametrize("M,C", [(1, 8), (1, 1024), (3, 520), (5, 1024), (67, 896), (4099, 64), (2051, 1024), (9, 2048),
                                 (1500, 1792), (5, 2056), (600, 4096), (7, 8192), (3, 8200), (530, 16384)])
def test_rmsnorm_rows_bwd(dev, M, C, dxn):
    g = gen(dev, M + C)
    xs, dh, dn = randn(g, M, C), randn(g, M, C), randn(g, M, C) if dxn else None
    for w in (1 + 0.1 * torch.randn(C, generator=g, device=dev), randn(g, C)):
        rstd = torch.rsqrt(xs.float().square().mean(-1) + 1e-6)
        dx, dw = G.rmsnorm_rows_bwd(dh, dn, xs, w, rstd)
        t, dt = xs.double() * rstd.double()[:, None], dh.double() * w.double()
        rs = rstd.double()[:, None]
        ref = rs * (dt - t * (dt * t).mean(-1, keepdim=True))
        mag = rs * (dt.abs() + t.abs() * (dt * t).abs().mean(-1, keepdim=True))
        if dxn:
            ref, mag = ref + dn.double(), mag + dn.double().abs()
        eps = mag * (C / 64 + 48) * U
        R.within(dx, ref, ref.abs() * R.UBF + 2 * eps, "dx")
        # dw: a chain of rows per team, 3 teams, the workgroups' partials by 16ths, 16; and two roundings a term
        rw, mw = (dh.double() * t).sum(0), (dh.double() * t).abs().sum(0)
        assert dw.dtype == w.dtype
        R.within(dw, rw, mw * (M / 512 + 80) * U + (rw.abs() * R.UBF if dw.dtype == BF else 0), "dw")
        again = G.rmsnorm_rows_bwd(dh, dn, xs, w, rstd)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


def test_rmsnorm_rows_bwd_differences(dev):
    """dx and dw against central differences of the 64-bit norm, along random directions."""
    g = gen(dev, 3)
    M, C, eps = 5, 256, 1e-3
    x, w, dh, dn = randn(g, M, C), 1 + 0.1 * torch.randn(C, generator=g, device=dev), randn(g, M, C), randn(g, M, C)
    f = lambda x, w: (R.norm_f64(x, w, eps) * dh.double()).sum() + (x * dn.double()).sum()  # noqa: E731
    rstd = torch.rsqrt(x.float().square().mean(-1) + eps)
    dx, dw = G.rmsnorm_rows_bwd(dh, dn, x, w, rstd)
    vx, vw = torch.randn(M, C, generator=g, device=dev).double(), torch.randn(C, generator=g, device=dev).double()
    t = 1e-4
    x, w = x.double(), w.double()
    nx = ((f(x + t * vx, w) - f(x - t * vx, w)) / (2 * t)).item()
    nw = ((f(x, w + t * vw) - f(x, w - t * vw)) / (2 * t)).item()
    # the difference's own error ~ t^2; dx: a bf16 rounding of each element
    assert abs((dx.double() * vx).sum().item() - nx) <= R.UBF * (dx.double() * vx).abs().sum().item() * 0.25 + 1e-4
    assert abs((dw.double() * vw).sum().item() - nw) <= 1e-5 * (dw.double() * vw).abs().sum().item() + 1e-4


def test_rmsnorm_rows_bwd_no_rows(dev):
    w = torch.ones(64, device=dev)
    e = torch.empty(0, 64, dtype=BF, device=dev)
    dx, dw = G.rmsnorm_rows_bwd(e, None, e, w, torch.empty(0, device=dev))
    assert dx.shape == (0, 64) and not dw.any()


# ------------------------------------------------------------------------------------------------ GEMM

def ints(g, *shape, hi=4):
    return torch.randint(-hi, hi + 1, shape, generator=g, device=g.device).float()


# every class: few rows (1-32), the small tiles, 256 x 128, 256 x 256, split K; ragged M, N, K
SHAPES = [(1, 16, 16), (1, 64, 128), (1, 4096, 1024), (2, 48, 400), (15, 80, 528), (16, 128, 2048), (17, 1024, 1040),
          (32, 256, 4112), (33, 64, 64), (33, 1040, 1008), (100, 96, 144), (257, 528, 1024), (512, 1024, 1024),
          (512, 272, 8192), (1000, 2064, 272), (2049, 1024, 1024), (4097, 2064, 528), (700, 4112, 2064),
          (2500, 512, 8208), (6592, 4096, 256), (9000, 1040, 400)]
# more rows than 32 in few tiles of 16 columns: one a workgroup, two; and the small tiles past them
SHAPES += [(33, 16, 16), (45, 208, 8176), (250, 512, 2064), (1000, 112, 400), (2048, 16, 2048), (8190, 16, 48), (64, 4080, 5632),
           (1021, 240, 8112), (130, 1520, 6160), (333, 1040, 272), (700, 2064, 400), (1500, 2064, 400)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_rows_exact(dev, M, N, K):
    """Small whole operands and power-of-two scales: every sum is exact, and so is every result whose magnitude fits
    bf16's 8 bits -- forced here by one nonzero product in most sums."""
    g = gen(dev, M)
    a, b = torch.zeros(M, K, device=dev), torch.zeros(N, K, device=dev)
    ka, kb = torch.arange(M, device=dev) * 7 % K, torch.arange(N, device=dev) * 5 % K
    a[torch.arange(M, device=dev), ka] = ints(g, M)
    b[torch.arange(N, device=dev), kb] = ints(g, N)
    b[:, K - 1] = 1.0
    a[:, K - 1] += 1.0
    sa = 2.0 ** (torch.arange(M, device=dev) % 3).float()
    sb = 2.0 ** (torch.arange(N, device=dev) % 2).float()
    bias, res = ints(g, N), ints(g, M, N).to(BF)
    gate = ints(g, 1, N, hi=1).to(BF)
    z = (a @ b.t()) * sa[:, None] * sb + bias
    want = (z * gate.float() + res.float()).to(BF)
    for bias_ in (bias, bias.to(BF)):
        y = G.fp8_gemm_rows(a.to(E4), sa, b.to(E4), sb, bias_, "none", res, gate)
        assert torch.equal(y, want)
    y, z16 = GR.gemm_rows_op(a.to(E4), sa, b.to(E4), sb, bias, "none", None, None, True)
    assert torch.equal(y, z.to(BF)) and torch.equal(z16, y)
    assert torch.equal(G.fp8_gemm_rows(a.to(E4), None, b.to(E4), None), (a @ b.t()).to(BF))


@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("M,N,K", [(1, 4096, 1024), (1, 32, 16), (5, 96, 272), (31, 512, 4096), (64, 160, 48), (300, 1024, 1024),
                                   (2049, 1056, 1024), (4100, 2080, 528), (520, 1024, 8192), (205, 96, 272), (130, 1536, 6160),
                                   (335, 1056, 272)])
def test_gemm_rows_epilogue(dev, M, N, K, act):
    g = gen(dev, N + K)
    a, sa = R.rowq(randn(g, M, K))
    b, sb = R.rowq(randn(g, N, K, std=K ** -0.5, dtype=F32) * 2.0)
    a, sa, b, sb = (t.to(dev) for t in (a, sa, b, sb))
    No = N // 2 if act == "swiglu" else N
    bias, res = randn(g, N), randn(g, M, No)
    B = 5 if M % 5 == 0 else 1
    gate = randn(g, B, 1, 2 * No).chunk(2, dim=-1)[1]
    for kw in (dict(), dict(bias=bias), dict(bias=bias.float(), res=res), dict(res=res, gate=gate), dict(gate=gate)):
        y = G.fp8_gemm_rows(a, sa, b, sb, kw.get("bias"), act, kw.get("res"), kw.get("gate"))
        ref, bound = R.gemm(a, sa, b, sb, kw.get("bias"), act, kw.get("res"), kw.get("gate"))
        assert y.shape == ref.shape and y.dtype == BF
        R.within(y, ref, bound, str(sorted(kw)))
        assert torch.equal(y, G.fp8_gemm_rows(a, sa, b, sb, kw.get("bias"), act, kw.get("res"), kw.get("gate")))


@pytest.mark.parametrize("M,N,K", [(3, 64, 64), (300, 512, 512), (5000, 2048, 528), (700, 1024, 8192), (100, 256, 4112)])
def test_gemm_rows_keeps_z(dev, M, N, K):
    g = gen(dev, M)
    a, sa, b, sb = (t.to(dev) for t in (*R.rowq(randn(g, M, K)), *R.rowq(randn(g, N, K, std=K ** -0.5))))
    bias = randn(g, N)
    y, z = GR.gemm_rows_op(a, sa, b, sb, bias, "silu", None, None, True)
    ref, bound = R.gemm(a, sa, b, sb, bias)
    R.within(z, ref, bound, "z")
    ref, bound = R.gemm(a, sa, b, sb, bias, "silu")
    R.within(y, ref, bound, "y")


def test_gemm_rows_strides_and_empty(dev):
    g = gen(dev)
    A, B = randn(g, 70, 256).to(E4), randn(g, 96, 512).to(E4)
    a, b = A[::2, 64:192], B[:, 128:256]
    res = randn(g, 35, 400)[:, 8:104]
    y = G.fp8_gemm_rows(a, None, b, None, residual=res)
    ref, bound = R.gemm(a, None, b, None, res=res)
    R.within(y, ref, bound)
    one = A[5:6, 16:144]
    R.within(G.fp8_gemm_rows(one, None, b, None), *R.gemm(one, None, b, None))
    assert G.fp8_gemm_rows(A[:0, :128], None, b, None).shape == (0, 96)
    assert G.fp8_gemm_rows(a, None, B[:0, :128], None).shape == (35, 0)


@pytest.mark.parametrize("M,N,K,act", [(20, 96, 64, "none"), (300, 96, 512, "silu"), (4099, 1040, 256, "none"),
                                       (4099, 1056, 256, "swiglu"), (9000, 2064, 400, "gelu_tanh"), (9001, 2080, 384, "swiglu"),
                                       (700, 1040, 8192, "silu"), (90, 96, 2064, "swiglu"), (100, 2080, 5136, "silu")])
def test_gemm_rows_strided_residual_and_gate(dev, M, N, K, act):
    """A residual that is a column range ending with its storage, a gate whose rows change within and between the waves' 64
    rows, with and without z, in every tile class."""
    g = gen(dev, M + N)
    a, sa, b, sb = (t.to(dev) for t in (*R.rowq(randn(g, M, K)), *R.rowq(randn(g, N, K, std=K ** -0.5))))
    No = N // 2 if act == "swiglu" else N
    res = randn(g, M, No + 72)[:, 72:]
    bias = randn(g, N)
    for B in {1, 3 if M % 3 == 0 else 1, M // 50 if M % 50 == 0 else 1, M}:
        gate = randn(g, B, 1, 3 * No).chunk(3, dim=-1)[1]
        y = G.fp8_gemm_rows(a, sa, b, sb, bias, act, res, gate)
        R.within(y, *R.gemm(a, sa, b, sb, bias, act, res, gate), f"gate of {B}")
    y, z = GR.gemm_rows_op(a, sa, b, sb, bias, act, res, gate, True)
    R.within(y, *R.gemm(a, sa, b, sb, bias, act, res, gate), "y beside z")
    R.within(z, *R.gemm(a, sa, b, sb, bias), "z")
    R.within(G.fp8_gemm_rows(a, sa, b, sb, bias, act, res), *R.gemm(a, sa, b, sb, bias, act, res), "residual alone")


def test_gemm_rows_not_finite(dev):
    """A NaN scale reaches its own row alone, and so does an infinite one; an infinite residual stays."""
    g = gen(dev)
    for M in (8, 300):
        x = randn(g, M, 128)
        x[3, 5], x[4, 6] = math.nan, math.inf
        a, sa = G.tcast_rows(x)
        b, sb = G.tcast_rows(randn(g, 64, 128))
        res = randn(g, M, 64)
        res[6, 1], res[7, 2] = math.inf, math.nan
        y = G.fp8_gemm_rows(a, sa, b, sb, act="silu", residual=res)
        assert torch.isnan(y[3]).all() and not torch.isfinite(y[4]).any()
        bad = ~torch.isfinite(y)
        bad[3:5] = False
        assert bad.sum() == 2 and torch.isinf(y[6, 1]) and torch.isnan(y[7, 2])


def test_gemm_rows_past_32_bits(dev):
    """Outputs and residuals past 2^31 elements."""
    M, N, K = 2 ** 18 + 20, 8192, 16
    a = torch.zeros(M, K, device=dev).to(E4)
    a[-3:] = 1.0
    b = torch.ones(N, K, device=dev).to(E4)
    res = torch.zeros(M, N, dtype=BF, device=dev)
    res[-3:] = 2.0
    y = G.fp8_gemm_rows(a, None, b, None, residual=res)
    assert (y[-3:] == 18).all() and not y[:-3].any()


# ------------------------------------------------------------------------------------------------ activation's backward

@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh"])
@pytest.mark.parametrize("M,N", [(1, 8), (3, 520), (65, 1024), (9, 2048), (5, 4096), (3, 7168), (2, 16384), (2, 32768)])
def test_act_bwd_rows(dev, M, N, act):
    g = gen(dev, N)
    dy, z = randn(g, M, N), randn(g, M, N, std=2.0)
    sw = torch.rand(N, generator=g, device=dev) + 0.5
    dz, q, s = G.act_bwd_rows(dy, z, act, sw)
    ref = dy.double() * R.dact(z.double(), act)
    # the derivative's fp32 error: 24 roundings relative to |terms| <= 1 + |z|(1 + z^2) on |z| <= 10, and |z| 2^-24 in e^z
    eps = 0 * ref if act == "none" else dy.double().abs() * U * (24 + z.double().abs()) * 3
    if act == "none":
        assert dz is dy
    else:
        R.within(dz, ref, ref.abs() * R.UBF + 2 * eps, "dz")
    R.check_rowq(q, s, ref * sw.double(), (eps + ref.abs() * U) * sw.double())


@pytest.mark.parametrize("act", ["none", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (0, 64, 32), (5, 72, 48), (3, 1040, 200 // 16 * 16), (1000, 2048, 64),
                                   (7, 4104, 80), (900, 2056, 16), (2, 16392, 176), (4000, 64, 1024)])
def test_act_bwd_rows_transpose_and_sum(dev, M, N, K, act):
    """The weight's bytes transposed in the same launch, and the column sums of the dz that it wrote."""
    g = gen(dev, N)
    dy, z, sw = randn(g, M, N), randn(g, M, N), torch.rand(N, generator=g, device=dev) + 0.5
    wq = torch.randint(0, 256, (N, K), generator=g, device=dev, dtype=torch.uint8).view(E4)
    for b32 in (False, True):
        dz, q, s, wqt, db = GR.act_bwd_rows_op(dy, z, act, sw, wq, True, b32)
        assert wqt.shape == (K, (N + 15) // 16 * 16)
        assert torch.equal(u8(wqt)[:, :N], u8(wq).t()) and not u8(wqt)[:, N:].any()
        d = (dy if act == "none" else dz).double()
        # a chain of rows per team (M over 768 x 4, 768, or all in one), 3 teams, 16 partial rows, 6 pairs
        chain = -(-M // 3072) if N <= 2048 else -(-M // 768)
        bound = d.abs().sum(0) * (chain + 28) * U + (0 if b32 else d.sum(0).abs() * R.UBF)
        assert db.dtype == (F32 if b32 else BF)
        R.within(db, d.sum(0), bound + 1e-38, "db")
        plain = GR.act_bwd_rows_op(dy, z, act, sw)
        assert torch.equal(u8(plain[1]), u8(q)) and torch.equal(plain[0], dz) and torch.equal(plain[2], s)
        assert torch.equal(db, GR.act_bwd_rows_op(dy, z, act, sw, None, True, b32)[4])


def test_act_bwd_differences(dev):
    """act' against central differences of the activation, over the range where it changes."""
    z = torch.linspace(-12, 12, 2048, device=dev).to(BF)[None]
    for act in ("silu", "gelu_tanh"):
        dz, _, _ = G.act_bwd_rows(torch.ones_like(z), z, act, torch.ones(2048, device=dev))
        t = 1e-5
        num = (R.act(z.double() + t, act) - R.act(z.double() - t, act)) / (2 * t)
        R.within(dz, num, num.abs() * R.UBF + 1e-5, act)


# ------------------------------------------------------------------------------------------------ linears

@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_act_bwd_rows_far_values(dev, act):
    """The activation's derivative where it is 0 or 1 to the last bit, up to the type's largest values, whose square
    overflows; NaN stays NaN."""
    z = torch.tensor([30., -300., 1e4, -1e9, 1e18, -1e20, 1e25, -3e38], dtype=BF, device=dev).repeat(2, 2)
    dy = torch.full_like(z, 3.0)
    sw = torch.ones(16, device=dev)
    dz, q, s = G.act_bwd_rows(dy, z, act, sw)
    assert torch.equal(dz, torch.where(z > 0, dy, torch.zeros_like(dy)))
    ref = torch.where(z > 0, 3.0, 0.0).double()
    assert ((R.deq(q, s) - ref).abs() <= 2 ** -24 * ref).all()   # (448 times the rounded 3 / 448)
    z[1, 5] = float("nan")
    dz, q, s = G.act_bwd_rows(dy, z, act, sw)
    assert torch.isnan(dz[1, 5]) and torch.isnan(s[1]) and torch.isfinite(s[0]) and torch.isfinite(dz).sum() == 31


def rel(x, ref):
    return (torch.linalg.norm(x.double() - ref) / torch.linalg.norm(ref)).item()


@pytest.mark.parametrize("act", ["none", "silu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,K,wdt", [(1, 64, 32, BF), (37, 96, 160, F32), (700, 1024, 512, BF), (3000, 512, 1040, F32)])
def test_linear_rows_train(dev, M, N, K, wdt, act):
    """y and every gradient against 64 bits from the same bytes; relative Frobenius errors within 1e-2 (bf16 roundings
    2^-8 at most, and the gradient's e4m3 bytes that a last bit of z moves by a step)."""
    g = gen(dev, M)
    x, res = randn(g, M, K).requires_grad_(), randn(g, M, N).requires_grad_()
    w, b = randn(g, N, K, std=K ** -0.5, dtype=wdt).requires_grad_(), randn(g, N, dtype=wdt).requires_grad_()
    dy = randn(g, M, N)
    y = G.fp8_linear_rows(x, w, b, act, res)
    gx, gw, gb, gr = torch.autograd.grad(y, (x, w, b, res), dy)
    assert gw.dtype == wdt and gb.dtype == wdt and gx.dtype == BF and torch.equal(gr, dy)
    with torch.no_grad():
        (xq, sx), (wq, sw) = G.tcast_rows(x), G.tcast_rows(w)
        z = R.deq(xq, sx) @ R.deq(wq, sw).t() + b.double()
        assert rel(y, R.act(z, act) + res.double()) < 1e-2
        dz = dy.double() * R.dact(z.to(BF).double(), act)
        dq, sd = R.rowq(dz.float() * sw)
        assert rel(gx, R.deq(dq.to(dev), sd.to(dev)) @ wq.double()) < 1e-2
        assert rel(gw, dz.t() @ x.double()) < 1e-2 and rel(gb, dz.sum(0)) < 1e-2
        # and the dgrad against the unquantized one: e4m3's rounding (rms of 2^-4 / sqrt 3 at most) in both operands
        assert rel(gx, dz @ w.double()) < 2 * 2 ** -4


def test_linear_rows_some_gradients(dev):
    """Only what is asked for: no input gradient, no weight gradient, no bias, an fp32 x, a batch [B, N, K]."""
    g = gen(dev)
    x, w, b = randn(g, 2, 9, 64), randn(g, 32, 64).requires_grad_(), randn(g, 32, dtype=F32).requires_grad_()
    y = G.fp8_linear_rows(x, w, b, "silu")
    assert y.shape == (2, 9, 32)
    gw, gb = torch.autograd.grad(y.float().sum(), (w, b))
    x32 = x.float().requires_grad_()
    y = G.fp8_linear_rows(x32, w.detach(), None, "silu")
    (gx,) = torch.autograd.grad(y.float().sum(), x32)
    assert gx.dtype == F32 and gx.shape == x.shape and gw.shape == w.shape and gb.dtype == F32
    res = randn(g, 2, 9, 32).requires_grad_()
    y = G.fp8_linear_rows(x, w.detach(), None, "none", res)
    (gr,) = torch.autograd.grad(y, res, torch.ones_like(y))
    assert (gr == 1).all()
    y = G.fp8_linear_rows(x32[:, :0], w, b, "gelu_tanh")
    gx, gw, gb = torch.autograd.grad(y.sum(), (x32, w, b))
    assert y.shape == (2, 0, 32) and not gw.any() and not gb.any() and not gx.any()
    a = randn(g, 2, 9, 64).requires_grad_()
    wn = torch.ones(64, device=dev, requires_grad=True)
    xn, y = G.fp8_rmsnorm_linear_rows(x32, wn, 1e-6, w, b, "silu", a)   # one output alone
    ga, gw0 = torch.autograd.grad(xn.float().sum(), (a, wn), retain_graph=True)
    assert (ga == 1).all() and not gw0.any()
    ga, gx = torch.autograd.grad(y.float().sum(), (a, x32))
    assert torch.equal(ga.float(), gx) and ga.any()
    y = G.fp8_linear_rows(x32, w, b, "silu").expand(3, 2, 9, 32)        # an expanded gradient
    (gx,) = torch.autograd.grad(y.sum(), x32)
    assert torch.isfinite(gx).all()
    with pytest.raises(RuntimeError):
        y = G.fp8_linear_rows(x32, w, b, "silu")
        (gx,) = torch.autograd.grad(y.float().sum(), x32, create_graph=True)
        gx.sum().backward()


@pytest.mark.parametrize("mode", ["plain", "res", "mod", "res_gate_mod"])
@pytest.mark.parametrize("B,N,C,O,act", [(2, 5, 64, 96, "silu"), (3, 100, 896, 512, "gelu_tanh"), (1, 1, 1024, 64, "none")])
def test_rmsnorm_linear_rows_train(dev, mode, B, N, C, O, act):
    """The norm feeding a linear: outputs and all gradients against 64 bits from the same bytes, and (e4m3's noise) against
    torch's autograd of the unquantized formulas in 64 bits."""
    g = gen(dev, C)
    x, a = randn(g, B, N, C).requires_grad_(), randn(g, B, N, C).requires_grad_()
    wn, w = randn(g, C, std=0.1).add_(1).requires_grad_(), randn(g, O, C, std=C ** -0.5).requires_grad_()
    b = randn(g, O).requires_grad_()
    gate, shift, scale = (randn(g, B, 1, C, std=0.3).requires_grad_() for _ in range(3))
    kw = dict(a=a if "res" in mode else None, gate=gate if "gate" in mode else None,
              shift=shift if "mod" in mode else None, scale=scale if "mod" in mode else None)
    xn, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, act, **kw)
    leaves = [x, wn, w, b] + [t for t in kw.values() if t is not None]
    dxn, dy = randn(g, B, N, C, std=0.1), randn(g, B, N, O)
    outs = (xn, y) if kw["a"] is not None else (y,)
    grads = torch.autograd.grad(outs, leaves, (dxn, dy) if kw["a"] is not None else (dy,))
    d = {id(t): t.detach().double().requires_grad_() for t in leaves}
    D = lambda t: d[id(t)]  # noqa: E731
    xr = D(x)
    if kw["a"] is not None:
        xr = xr + (D(gate) * D(a) if kw["gate"] is not None else D(a))
        assert torch.equal(xn, xr.detach().to(F32).to(BF))
    else:
        assert xn is x
    h = D(wn) * xr * (xr.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
    if kw["shift"] is not None:
        h = h * (1 + D(scale)) + D(shift)
    yr = R.act((h @ D(w).t() + D(b)).reshape(-1, O), act).reshape(y.shape)
    # e4m3 in h and w: 2^-4 / sqrt 3 of each rms at most, both independent of the other
    assert rel(y, yr.detach()) < 2 * 2 ** -4
    refs = torch.autograd.grad((xr, yr) if kw["a"] is not None else (yr,), list(d.values()),
                               (dxn.double(), dy.double()) if kw["a"] is not None else (dy.double(),))
    for t, gr, ref in zip(leaves, grads, refs):
        assert gr.shape == t.shape and gr.dtype == t.dtype
        assert rel(gr, ref) < 3 * 2 ** -4, (mode, rel(gr, ref))


def block(dev, g, B, N, C, H):
    mod = randn(g, B, 1, 6 * C, std=0.3).chunk(6, dim=-1)
    return dict(x=randn(g, B, N, C), a=randn(g, B, N, C), wn=1 + 0.1 * torch.randn(C, generator=g, device=dev), mod=mod,
                w12=randn(g, 2 * H, C, std=C ** -0.5), w3=randn(g, C, H, std=H ** -0.5))


def serve(s, w12, w3):
    """A block's second half as a sampler runs it: norm site 2, the SwiGLU MLP, the gated residual."""
    m = s["mod"]
    xn, hid = G.fp8_rmsnorm_linear_rows(s["x"], s["wn"], 1e-6, w12, None, "swiglu", s["a"], m[2], m[3], m[4])
    return xn, hid, G.fp8_linear_rows(hid, w3, None, "none", xn, m[5])


@pytest.mark.parametrize("B,N,C,H", [(1, 1, 64, 128), (2, 256, 1024, 1024), (3, 51, 896, 1792), (16, 256, 256, 512)])
def test_block_serving(dev, B, N, C, H):
    """The operators together, as a sampler runs them, each step against 64 bits from the bytes before it."""
    s = block(dev, gen(dev, C), B, N, C, H)
    m = s["mod"]
    w12, w3 = G.rows_weight(s["w12"], "swiglu"), G.rows_weight(s["w3"])
    with torch.no_grad():
        xn, hid, y = serve(s, w12, w3)
        _, _, q, sc, _ = G.rmsnorm_rows(s["x"], s["wn"], 1e-6, s["a"], m[2], m[3], m[4])
        rxn, _, rh, mag = R.norm(s["x"].reshape(-1, C), s["wn"], 1e-6, s["a"].reshape(-1, C), m[2], m[3], m[4])
        assert torch.equal(xn.reshape(-1, C), rxn)
        R.check_rowq(q.reshape(-1, C), sc, rh, eps_of(C, mag))
        ref, bound = R.gemm(q.reshape(-1, C), sc, w12.q, w12.s, name="swiglu")
        R.within(hid.reshape(-1, H), ref, bound, "hidden")
        # the layout of w12: the plain SwiGLU of its dequantized halves
        wd = torch.empty(2 * H, C, dtype=torch.float64, device=dev)
        wd[G.swiglu_layout(torch.arange(2 * H, device=dev))] = R.deq(w12.q, w12.s)
        z = R.deq(q.reshape(-1, C), sc) @ wd.t()
        assert rel(hid.reshape(-1, H), R.act(z[:, :H], "silu") * z[:, H:]) < 2 * R.UBF
        hq, hs = G.tcast_rows(hid.reshape(-1, H))
        ref, bound = R.gemm(hq, hs, w3.q, w3.s, res=rxn, gate=m[5])
        R.within(y.reshape(-1, C), ref, bound, "y")


def test_block_serving_graph_and_streams(dev):
    """Captured and replayed with new inputs, with eager work between the replays; and on a stream of its own."""
    g = gen(dev)
    for B, N in ((1, 1), (2, 200)):
        s = block(dev, g, B, N, 512, 1024)
        w12, w3 = G.rows_weight(s["w12"], "swiglu"), G.rows_weight(s["w3"])
        with torch.no_grad():
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                first = serve(s, w12, w3)
            torch.cuda.current_stream().wait_stream(side)
            assert all(torch.equal(p, q) for p, q in zip(first, serve(s, w12, w3)))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = serve(s, w12, w3)
            for k in range(4):
                s["x"].copy_(randn(g, B, N, 512))
                s["a"].copy_(randn(g, B, N, 512, std=1.0 + k))
                want = [t.clone() for t in serve(s, w12, w3)]
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_train_graph(dev):
    """A training step of norm, linear, activation and residual captured whole and replayed against the eager one."""
    g = gen(dev)
    x, a, dy = randn(g, 300, 256), randn(g, 300, 256), randn(g, 300, 256)
    wn, w1, b1 = randn(g, 256), randn(g, 512, 256, std=1 / 16), randn(g, 512)
    w2, b2 = randn(g, 256, 512, std=1 / 22), randn(g, 256)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, a, wn, w1, b1, w2, b2)]
        X, A, WN, W1, B1, W2, B2 = leaves
        xn, h = G.fp8_rmsnorm_linear_rows(X, WN, 1e-6, W1, B1, "gelu_tanh", A)
        y = G.fp8_linear_rows(h, W2, B2, "none", xn)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.copy_(randn(g, 300, 256))
        dy.copy_(randn(g, 300, 256))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want))


def test_compiled_and_autocast(dev):
    g = gen(dev)
    x, w, b = randn(g, 20, 64), randn(g, 48, 64).requires_grad_(), randn(g, 48).requires_grad_()
    wn = torch.ones(64, device=dev)

    def f(x):
        xn, h = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, "silu", x)
        return h.float().sum() + xn.float().sum()
    want = torch.autograd.grad(f(x), (w, b))
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager", fullgraph=True)(x), (w, b))
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    with torch.autocast("cuda", dtype=BF):
        assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(f(x), (w, b))))


def test_the_raw_calls_have_no_gradient(dev):
    """A gradient asked of an operator that has none is an error, not a silent loss."""
    g = gen(dev)
    x = randn(g, 4, 64).requires_grad_()
    xn = G.rmsnorm_rows(x, torch.ones(64, device=dev), 1e-6, x)[0]
    with pytest.raises(RuntimeError):
        xn.float().sum().backward()


@pytest.mark.parametrize("act", ["none", "silu"])
def test_host_module_and_general_form(dev, monkeypatch, act):
    """The native host module's calls and the general Python form give the same bits."""
    g = gen(dev)
    x, a, w, b = randn(g, 3, 50, 256), randn(g, 3, 50, 256), randn(g, 128, 256, dtype=F32), randn(g, 128, dtype=F32)
    w2, mod = randn(g, 256, 128), randn(g, 3, 1, 6 * 256, std=0.3).chunk(6, dim=-1)
    wn = 1 + 0.1 * torch.randn(256, generator=g, device=dev)
    dy, dxn = randn(g, 3, 50, 256), randn(g, 3, 50, 256)

    def passes():
        out = []
        for m in (False, True):
            leaves = [t.detach().requires_grad_() for t in (x, a, wn, w, b, w2)]
            X, A, WN, W, B, W2 = leaves
            kw = dict(gate=mod[2], shift=mod[3], scale=mod[4]) if m else {}
            xn, h = G.fp8_rmsnorm_linear_rows(X, WN, 1e-6, W, B, act, A, **kw)
            y = G.fp8_linear_rows(h, W2, None, "none", xn)
            out += [y.detach(), *torch.autograd.grad((xn, y), leaves, (dxn, dy))]
        with torch.no_grad():
            s = dict(x=x, a=a, wn=wn, mod=mod)
            out += serve(s, G.rows_weight(randn(gen(dev, 5), 256, 256), "swiglu"), G.rows_weight(w2))
            dh = dy.reshape(-1, 256)
            out += G.rmsnorm_rows_bwd(dh, None, dxn.reshape(-1, 256), wn, torch.rand(150, generator=gen(dev), device=dev))
        return out
    want = passes()
    monkeypatch.setattr(L, "native", lambda *a: None)
    got = passes()
    assert len(want) == len(got) and all(torch.equal(p, q) for p, q in zip(want, got))


def subsets(n):
    return [[i >> k & 1 == 1 for k in range(n)] for i in range(1, 1 << n)]


def grads_of(outs, dys, leaves, needs):
    need = [t for t, r in zip(leaves, needs) if r and t is not None]
    pairs = [(o, d) for o, d in zip(outs, dys) if o.requires_grad]
    got = iter(torch.autograd.grad([o for o, _ in pairs], need, [d for _, d in pairs], allow_unused=True))
    return [next(got) if r and t is not None else None for t, r in zip(leaves, needs)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("res", [False, True])
@pytest.mark.parametrize("act", ["none", "gelu_tanh"])
def test_linear_rows_gradient_of_each_set(dev, bias, res, act):
    """Every set of leaves that take a gradient, with and without bias and residual: the graph's native node gives the bits
    of the general Function, which is fed an output's gradient of another layout too."""
    g = gen(dev)
    leaves = [randn(g, 2, 9, 64), randn(g, 48, 64, dtype=F32), randn(g, 48) if bias else None,
              randn(g, 2, 9, 48) if res else None]
    dy = randn(g, 9, 2, 48).transpose(0, 1)
    for needs in subsets(4):
        if not any(r and t is not None for t, r in zip(leaves, needs)):
            continue
        x, w, b, r = [t if t is None else t.detach().requires_grad_(n) for t, n in zip(leaves, needs)]
        y = G.fp8_linear_rows(x, w, b, act, r)
        y2 = GR._LinearRows.apply(x, w, b, act, r)
        assert y.grad_fn.name() != y2.grad_fn.name() and torch.equal(y, y2)
        for p, q in zip(grads_of([y], [dy], [x, w, b, r], needs), grads_of([y2], [dy], [x, w, b, r], needs)):
            assert (p is None) == (q is None) and (p is None or (torch.equal(p, q) and p.dtype == q.dtype)), needs


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("add", [False, True])
def test_rmsnorm_linear_rows_gradient_of_each_set(dev, bias, add):
    g = gen(dev)
    leaves = [randn(g, 2, 9, 64), randn(g, 64, dtype=F32), randn(g, 48, 64), randn(g, 2, 9, 64) if add else None,
              randn(g, 48, dtype=F32) if bias else None]
    dxn, dy = randn(g, 2, 9, 64), randn(g, 2, 9, 48)
    for needs in subsets(5):
        if not any(r and t is not None for t, r in zip(leaves, needs)):
            continue
        x, wn, w, a, b = [t if t is None else t.detach().requires_grad_(n) for t, n in zip(leaves, needs)]
        xn, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, "silu", a)
        o = GR._NormLinearRows.apply(x, a, None, wn, None, None, 1e-6, w, b, "silu")
        outs, outs2 = ([xn, y], list(o)) if add else ([y], [o])
        assert y.grad_fn.name() != outs2[-1].grad_fn.name() and all(torch.equal(p, q) for p, q in zip(outs, outs2))
        for keep in ([0, 1], [0], [1]) if add else ([0],):   # (both outputs used, or one)
            dys = [dxn, dy] if add else [dy]
            args = ([x, wn, w, a, b], needs)
            o = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, "silu", a)
            p = grads_of([o[i if add else 1] for i in keep], [dys[i] for i in keep], *args)
            o = GR._NormLinearRows.apply(x, a, None, wn, None, None, 1e-6, w, b, "silu")
            q = grads_of([o[i] if add else o for i in keep], [dys[i] for i in keep], *args)
            for i, (s, t) in enumerate(zip(p, q)):
                assert (s is None) == (t is None) and (s is None or (torch.equal(s, t) and s.dtype == t.dtype)), (needs, keep, i)


def test_linear_rows_nodes_in_a_graph(dev):
    """What a node of the graph owes: a gradient of a gradient is refused (and a recorded first one alone is not), an input
    changed in place after the forward is refused, checkpointing and hooks work, two backward passes are the same."""
    from torch.utils.checkpoint import checkpoint
    g = gen(dev)
    x, wn, w = randn(g, 5, 64).requires_grad_(), torch.ones(64, device=dev, requires_grad=True), randn(g, 64, 64).requires_grad_()
    a = randn(g, 5, 64).requires_grad_()
    calls = [lambda x: G.fp8_linear_rows(x, w, None, "silu"),
             lambda x: G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, None, "silu")[1],
             lambda x: sum(G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, None, "silu", a))]
    for f in calls:
        y = f(x)
        dy = randn(g, *y.shape).requires_grad_()
        gx, gw = torch.autograd.grad(y, (x, w), dy.detach(), retain_graph=True, create_graph=True)
        assert not gx.requires_grad
        rx, rw = torch.autograd.grad(y, (x, w), dy, retain_graph=True, create_graph=True)
        assert torch.equal(rx, gx) and torch.equal(rw, gw) and rx.requires_grad
        with pytest.raises(RuntimeError, match="differentiable once"):
            rx.float().sum().backward()
        p, q = torch.autograd.grad(checkpoint(f, x, use_reentrant=False), (x, w), dy.detach())
        assert torch.equal(p, gx) and torch.equal(q, gw)
        seen = []
        h = x.register_hook(lambda t: seen.append(t.clone()))
        y.backward(dy.detach())
        h.remove()
        assert torch.equal(seen[0], gx) and torch.equal(x.grad, gx) and torch.equal(w.grad, gw)
        x.grad = w.grad = wn.grad = a.grad = None
        with torch.autograd.graph.save_on_cpu():
            y = f(x)
        p, q = torch.autograd.grad(y, (x, w), dy.detach())
        assert torch.equal(p, gx) and torch.equal(q, gw)
        for back in (lambda t: t.cpu(), lambda t: t.t().contiguous().t() if t.dim() == 2 else t):   # (hooks that change them)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), back):
                y = f(x)
            with pytest.raises(RuntimeError, match="as they were saved"):
                torch.autograd.grad(y, (x, w), dy.detach())
        with torch.autograd.detect_anomaly(check_nan=False):
            p, q = torch.autograd.grad(f(x), (x, w), dy.detach())
        assert torch.equal(p, gx) and torch.equal(q, gw)
        with torch.autograd.forward_ad.dual_level():
            for leaf in (x.detach(), x):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    f(torch.autograd.forward_ad.make_dual(leaf, torch.ones_like(leaf)))
        x2 = x.detach().clone()
        y = f(x2)
        x2.add_(1)
        if f is calls[2]:        # (it keeps x + a, not x)
            torch.autograd.grad(y, w, dy.detach())
        else:
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad(y, w, dy.detach())
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).float().sum())(x.detach())
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x.detach()[None])
    xn, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, None, "silu", a)   # (an output that is kept, changed in place)
    xn.mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        y.float().sum().backward()


def test_linear_rows_inference_mode_and_threads(dev):
    """Under inference mode, and from four threads at once, each on a stream of its own: the bits of a call alone."""
    import threading
    g = gen(dev)
    x, a, wn = randn(g, 70, 256), randn(g, 70, 256), torch.ones(256, device=dev)
    w, w2 = randn(g, 512, 256, std=1 / 16), randn(g, 256, 512, std=1 / 22)

    def step(train):
        leaves = [t.detach().requires_grad_(train) for t in (x, a, wn, w, w2)]
        X, A, WN, W, W2 = leaves
        xn, h = G.fp8_rmsnorm_linear_rows(X, WN, 1e-6, W, None, "gelu_tanh", A)
        y = G.fp8_linear_rows(h, W2, None, "none", xn)
        return [y.detach(), *torch.autograd.grad(y, leaves, x)] if train else [y]

    want = step(True)
    with torch.inference_mode():
        (y,) = step(False)
        assert y.is_inference() and torch.equal(y, want[0])
        q, s = G.tcast_rows(x)
        assert q.is_inference() and torch.equal(u8(q), u8(G.tcast_rows(x)[0]))
    torch.cuda.synchronize()
    bad = []

    def work():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = step(True)
                    torch.cuda.current_stream().synchronize()
                    bad.extend(i for i, (p, q) in enumerate(zip(got, want)) if not torch.equal(p, q))
        except Exception as e:   # noqa: BLE001 (reported by the thread that waits)
            bad.append(e)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_linear_rows_past_32_bits(dev):
    """A linear whose output has more than 2^31 bytes, and its gradients: the last rows, and the sums over all."""
    M, K, N = 140000, 64, 8192
    g = gen(dev)
    x, w, b = (randn(g, *s).requires_grad_() for s in ((M, K), (N, K), (N,)))
    y = G.fp8_linear_rows(x, w, b, "silu")
    dy = randn(g, N, std=0.1).expand(M, N)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
    with torch.no_grad():
        (xq, sx), (wq, sw) = G.tcast_rows(x), G.tcast_rows(w)
        X, W = R.deq(xq, sx), R.deq(wq, sw)
        dw, db = torch.zeros(N, K, dtype=torch.float64, device=dev), torch.zeros(N, dtype=torch.float64, device=dev)
        for i in range(0, M, 10000):
            z = X[i:i + 10000] @ W.t() + b.double()
            dz = dy[i:i + 10000].double() * R.dact(z.to(BF).double(), "silu")
            dw += dz.t() @ x[i:i + 10000].double()
            db += dz.sum(0)
        assert rel(y[-1000:], R.act(z, "silu")[-1000:]) < 1e-2 and rel(gw, dw) < 1e-2 and rel(gb, db) < 1e-2
        dq, sd = R.rowq((dz[-1000:]).float() * sw)
        assert rel(gx[-1000:], R.deq(dq.to(dev), sd.to(dev)) @ wq.double()) < 1e-2


@pytest.mark.parametrize("shape", [(256,), (1, 256), (2, 3, 5, 256), (40, 256)])
def test_served_linears_native_and_general(dev, monkeypatch, shape):
    """Linears on a RowsWeight: the native call gives the general form's bits, and what neither takes is refused."""
    g = gen(dev)
    x, a, wn = randn(g, *shape), randn(g, *shape), 1 + 0.1 * torch.randn(256, generator=g, device=dev)
    M = x.numel() // 256
    w, w12 = G.rows_weight(randn(g, 96, 256)), G.rows_weight(randn(g, 192, 256), "swiglu")
    b, b12, res = randn(g, 96), randn(g, 192, dtype=F32), randn(g, *shape[:-1], 96)
    gate = randn(g, 2 if M % 2 == 0 else 1, 1, 192).chunk(2, dim=-1)[1]

    def calls():
        out = [G.fp8_linear_rows(x, w, b, "gelu_tanh", res, gate), G.fp8_linear_rows(x, w), G.fp8_linear_rows(x, w, None, "silu", res),
               G.fp8_linear_rows(x, w12, b12, "swiglu", res, gate), G.fp8_linear_rows(x.float(), w12, None, "swiglu")]
        if len(shape) > 1:
            out += [*G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, "silu"), *G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w12, b12, "swiglu", a)]
        return out
    for r in (res[..., :80], res.reshape(1, *res.shape)):
        with pytest.raises(ValueError, match="residual"):
            G.fp8_linear_rows(x, w, None, "none", r)
    with pytest.raises(ValueError):
        G.fp8_linear_rows(x, w, None, "none", res, gate.repeat(M + 1, 1, 1))
    with pytest.raises(ValueError, match="RowsWeight"):
        G.fp8_linear_rows(x.requires_grad_(), w)
    x.requires_grad_(False)
    want = calls()
    assert all(y.shape == (*shape[:-1], 96) for y in want[:5])
    monkeypatch.setattr(L, "native", lambda *a: None)
    got = calls()
    assert len(want) == len(got) and all(torch.equal(p, q) for p, q in zip(want, got))


def test_operands_that_take_a_gradient(dev):
    """A gradient asked of the GEMM through any of its operands is an error, not a silent loss, also through the e4m3 ones."""
    g = gen(dev)
    a, b = randn(g, 4, 64).to(E4), randn(g, 32, 64).to(E4)
    ins = [a, torch.ones(4, device=dev), b, torch.ones(32, device=dev), randn(g, 32), randn(g, 4, 32), randn(g, 1, 32)]
    for i in range(len(ins)):
        t = [v.detach().requires_grad_(k == i) for k, v in enumerate(ins)]
        y = G.fp8_gemm_rows(*t[:5], "none", t[5], t[6])
        with pytest.raises(RuntimeError):
            y.float().sum().backward()
        with torch.no_grad():
            assert not G.fp8_gemm_rows(*t[:5], "none", t[5], t[6]).requires_grad
    for w in (G.RowsWeight(b.detach().requires_grad_(), ins[3], False), G.RowsWeight(b, ins[3].detach().requires_grad_(), False)):
        with pytest.raises(ValueError, match="RowsWeight"):
            G.fp8_linear_rows(randn(g, 4, 64), w)
        with pytest.raises(ValueError, match="RowsWeight"):
            G.fp8_rmsnorm_linear_rows(randn(g, 4, 64), torch.ones(64, device=dev), 1e-6, w)


def test_gate_rows_follow_the_batch(dev, monkeypatch):
    """A gate of a linear on a RowsWeight: one row, or x's batch's; for a 2-D x any number that divides its rows."""
    g = gen(dev)
    x, w, gates = randn(g, 2, 6, 64), G.rows_weight(randn(g, 32, 64)), randn(g, 12, 1, 32)
    z = G.fp8_linear_rows(x, w).double()
    for native in (True, False):
        if not native:
            monkeypatch.setattr(L, "native", lambda *a: None)
        for n in (3, 4, 6, 12):
            with pytest.raises(ValueError, match="gate has"):
                G.fp8_linear_rows(x, w, gate=gates[:n])
        with pytest.raises(ValueError, match="gate has"):
            G.fp8_linear_rows(x.view(1, 12, 64), w, gate=gates[:2])
        for n in (1, 2, 3, 4, 6, 12):
            y = G.fp8_linear_rows(x.view(12, 64), w, gate=gates[:n])
            ref = z.view(12, 32) * gates[:n].double().view(n, 32).repeat_interleave(12 // n, 0)
            assert rel(y, ref) < 2 * R.UBF
            if n <= 2:
                assert torch.equal(G.fp8_linear_rows(x, w, gate=gates[:n]).view(12, 32), y)


@pytest.mark.parametrize("B,N", [(0, 3), (2, 0), (0, 0)])
def test_no_rows(dev, B, N):
    """An empty batch, and entries without tokens, with a block's gate, shift and scale: outputs without rows, zero gradients."""
    g = gen(dev)
    leaves = [randn(g, *s) for s in ((B, N, 64), (64,), (32, 64), (32,), (B, N, 64), (B, 1, 64), (B, 1, 64), (B, 1, 64))]
    w, w12, res = G.rows_weight(leaves[2]), G.rows_weight(randn(g, 64, 64), "swiglu"), randn(g, B, N, 32)
    x, wn, _, b, a, gate, shift, scale = leaves
    for kw in (dict(), dict(a=a), dict(a=a, gate=gate), dict(shift=shift, scale=scale), dict(a=a, gate=gate, shift=shift, scale=scale)):
        xn, h, q, s, rstd = G.rmsnorm_rows(x, wn, 1e-6, want_h=True, **kw)
        assert h.shape == q.shape == (B, N, 64) and s.numel() == rstd.numel() == 0 and xn.numel() == 0
        for weight, act in ((w, "silu"), (w12, "swiglu")):
            xn, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, weight, None, act, **kw)
            assert xn.shape == x.shape and y.shape == (B, N, 32)
            assert G.fp8_linear_rows(x, weight, None, act, res, randn(g, B, 1, 32)).shape == (B, N, 32)
        if "gate" not in kw or "shift" in kw:
            t = {k: v.detach().requires_grad_() for k, v in dict(x=x, wn=wn, w=leaves[2], b=b, **kw).items()}
            xn, y = G.fp8_rmsnorm_linear_rows(t["x"], t["wn"], 1e-6, t["w"], t["b"], "silu", *[t.get(k) for k in ("a", "gate", "shift", "scale")])
            grads = torch.autograd.grad(xn.float().sum() + y.float().sum(), list(t.values()))
            assert all(d.shape == v.shape and d.dtype == v.dtype and not d.any() for d, v in zip(grads, t.values()))
    for rows in (0, 1, 3):   # (x without a batch: any number of modulation rows that divides none)
        mod = randn(g, rows, 64)
        assert G.rmsnorm_rows(x.reshape(-1, 64), wn, 1e-6, a.reshape(-1, 64), mod, mod, mod)[2].shape == (0, 64)
        assert G.fp8_linear_rows(x.reshape(-1, 64), w, gate=randn(g, rows, 32)).shape == (0, 32)


@pytest.mark.parametrize("form", ["native", "general", "gated"])
def test_x_new_alone(dev, form):
    """Only x_new in the loss: its gradient as it is, and zeros for what the norm and the linear have, also where h is not finite."""
    g = gen(dev)
    x, a, wn, w, b = randn(g, 2, 9, 64), randn(g, 2, 9, 64), randn(g, 64), randn(g, 48, 64), randn(g, 48, dtype=F32)
    x[0, 3, 7], x[1, 2, 0] = math.inf, math.nan
    mod = randn(g, 2, 1, 3 * 64, std=0.3).chunk(3, -1) if form == "gated" else (None, None, None)
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, a, wn, w, b, *mod)]
    x, a, wn, w, b, gate, shift, scale = leaves
    if form == "general":
        xn, y = GR._NormLinearRows.apply(x, a, None, wn, None, None, 1e-6, w, b, "silu")
    else:
        xn, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, "silu", a, gate, shift, scale)
    dxn = randn(g, 9, 2, 64).transpose(0, 1)
    need = [t for t in leaves if t is not None]
    grads = dict(zip(map(id, need), torch.autograd.grad(xn, need, dxn, retain_graph=True)))
    assert torch.equal(grads[id(x)], dxn)
    for t in (wn, w, b, shift, scale):
        if t is not None:
            assert grads[id(t)].shape == t.shape and grads[id(t)].dtype == t.dtype and not grads[id(t)].any()
    if gate is None:
        assert torch.equal(grads[id(a)], dxn)
    else:
        assert torch.equal(grads[id(a)], (gate.double() * dxn.double()).to(BF))
        assert rel(grads[id(gate)], (dxn.double() * a.double()).sum(1, keepdim=True)) < R.UBF
    for t in need:   # (and each alone)
        (got,) = torch.autograd.grad(xn, t, dxn, retain_graph=True)
        assert torch.equal(got, grads[id(t)])


def test_linears_on_fake_tensors(dev):
    """Forward and backward as a shape pass over a program makes them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device=dev)  # noqa: E731
        x, a, w, b = e(2, 9, 64).requires_grad_(), e(2, 9, 64).requires_grad_(), e(48, 64).requires_grad_(), e(48, dt=F32).requires_grad_()
        wn, m = e(64, dt=F32).requires_grad_(), [t.requires_grad_() for t in (e(2, 1, 64), e(2, 1, 64), e(2, 1, 64))]
        y = G.fp8_linear_rows(x, w, b, "silu", e(2, 9, 48))
        assert [t.shape for t in torch.autograd.grad(y, (x, w, b), e(2, 9, 48))] == [x.shape, w.shape, b.shape]
        for mod in ((None, None, None), m):
            leaves = [t for t in (x, wn, w, b, a, *mod) if t is not None]
            xn, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, "gelu_tanh", a, *mod)
            for outs, dys in (((xn, y), (e(2, 9, 64), e(2, 9, 48))), ((y,), (e(2, 9, 48),)), ((xn,), (e(2, 9, 64),))):
                got = torch.autograd.grad(outs, leaves, dys, retain_graph=True)
                assert [(t.shape, t.dtype) for t in got] == [(t.shape, t.dtype) for t in leaves]


@pytest.mark.parametrize("form", ["native", "general"])
def test_recorded_backward_warns(dev, form, monkeypatch):
    """A backward that is itself recorded, from an output's gradient that is a constant: what comes back is a constant too (as
    torch's once_differentiable has it), and a warning says so. The usual backward gives none."""
    g = gen(dev)
    x, w, a = (randn(g, *s).requires_grad_() for s in ((5, 64), (64, 64), (5, 64)))
    wn = torch.ones(64, device=dev, requires_grad=True)
    if form == "general":
        monkeypatch.setattr(L, "native", lambda *a: None)
    res = randn(g, 5, 64).requires_grad_()
    calls = [lambda: G.fp8_linear_rows(x, w, None, "silu", res), lambda: G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, None, "silu")[1],
             lambda: sum(G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, None, "silu", a))]
    for f in calls:
        y = f()
        dy = randn(g, 5, 64)
        with pytest.warns(UserWarning, match="differentiable once"):
            gx, gw = torch.autograd.grad(y, (x, w), dy, create_graph=True)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            px, pw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
            rx, rw = torch.autograd.grad(y, (x, w), dy.detach().requires_grad_(), create_graph=True)   # (refused by rx's node)
        assert all(torch.equal(p, q) for p, q in ((gx, px), (gw, pw), (rx, px), (rw, pw)))
        with pytest.raises(RuntimeError):
            rx.float().sum().backward()
    with warnings.catch_warnings():   # (gradients that are constants: a residual's, and x_new's own)
        warnings.simplefilter("error")
        y = G.fp8_linear_rows(x.detach(), w.detach(), None, "silu", res)
        assert torch.equal(torch.autograd.grad(y, res, dy, create_graph=True)[0], dy)
        xn, _ = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, None, "silu", a)
        assert torch.equal(torch.autograd.grad(xn, x, dy, create_graph=True)[0], dy)


@pytest.mark.parametrize("M", [5, 700])
def test_swiglu_bias_order(dev, M):
    """w12 and its bias through swiglu_layout and rows_weight: the plain silu(x w1^T + b1) (x w2^T + b2)."""
    g = gen(dev, M)
    K, H = 256, 512
    x, w12, b12 = randn(g, M, K), randn(g, 2 * H, K, std=K ** -0.5), randn(g, 2 * H)
    w = G.rows_weight(w12, "swiglu")
    (xq, sx), (wq, sw) = G.tcast_rows(x), G.tcast_rows(w12)
    z = R.deq(xq, sx) @ R.deq(wq, sw).t() + b12.double()
    ref = R.act(z[:, :H], "silu") * z[:, H:]
    assert rel(G.fp8_linear_rows(x, w, G.swiglu_layout(b12), "swiglu"), ref) < 2 * R.UBF
    assert rel(G.fp8_linear_rows(x, w, b12, "swiglu"), ref) > 0.1   # (in w12's own order it is another bias)
    assert rel(G.fp8_gemm_rows(xq, sx, w.q, w.s, G.swiglu_layout(b12), "swiglu"), ref) < 2 * R.UBF
    wn = torch.ones(K, device=dev)
    _, _, hq, sh, _ = G.rmsnorm_rows(x, wn, 1e-6)
    z = R.deq(hq, sh) @ R.deq(wq, sw).t() + b12.double()
    _, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, G.swiglu_layout(b12), "swiglu")
    assert rel(y, R.act(z[:, :H], "silu") * z[:, H:]) < 2 * R.UBF


@pytest.mark.parametrize("M,N,K,act", [(4099, 1040, 256, "none"), (4099, 2080, 128, "swiglu"), (16500, 1008, 1024, "silu"),
                                       (6529, 1024, 1024, "gelu_tanh"), (6529, 1024, 1024, "swiglu")])
def test_gemm_rows_one_gate_row(dev, M, N, K, act):
    """One gate row for all rows, whose number no tile divides."""
    g = gen(dev, M)
    a, b = randn(g, M, K).to(E4), randn(g, N, K).to(E4)
    sa, sb = torch.rand(M, generator=g, device=dev) / K ** 0.5, torch.rand(N, generator=g, device=dev) + 0.5
    No = N // 2 if act == "swiglu" else N
    gate, res = randn(g, 1, No), randn(g, M, No)
    for r in (None, res):
        y = G.fp8_gemm_rows(a, sa, b, sb, None, act, r, gate)
        ref, bound = R.gemm(a, sa, b, sb, None, act, r, gate)
        R.within(y, ref, bound)


@pytest.mark.parametrize("mode", ["plain", "res", "mod", "res_gate_mod"])
@pytest.mark.parametrize("B,N,C,O,act", [(2, 5, 64, 96, "silu"), (3, 100, 896, 512, "gelu_tanh"), (1, 1, 1024, 64, "none")])
def test_rmsnorm_linear_rows_train_same_bytes(dev, mode, B, N, C, O, act):
    """The norm feeding a linear: outputs, z and all gradients against 64 bits from the forward's bytes (norm's, weight's and z's
    roundings as they are, the gradient's row cast and dh's rounding to bf16 made again). An output is off by half a step of bf16,
    and by another where dh rounds the other way: 2 UBF. The norm's backward without the mean of dt t, its smallest term, is
    further off than that wherever there are rows to average over."""
    g = gen(dev, C + N)
    x, a = randn(g, B, N, C).requires_grad_(), randn(g, B, N, C).requires_grad_()
    wn, w = randn(g, C, std=0.1).add_(1).requires_grad_(), randn(g, O, C, std=C ** -0.5).requires_grad_()
    b = randn(g, O).requires_grad_()
    gate, shift, scale = (randn(g, B, 1, C, std=0.3).requires_grad_() for _ in range(3))
    kw = dict(a=a if "res" in mode else None, gate=gate if "gate" in mode else None,
              shift=shift if "mod" in mode else None, scale=scale if "mod" in mode else None)
    res = kw["a"] is not None
    xn, y = G.fp8_rmsnorm_linear_rows(x, wn, 1e-6, w, b, act, **kw)
    names = ["x", "wn", "w", "b"] + [k for k, t in kw.items() if t is not None]
    leaves = [x, wn, w, b] + [t for t in kw.values() if t is not None]
    dxn, dy = randn(g, B, N, C, std=0.1), randn(g, B, N, O)
    got = dict(zip(names, torch.autograd.grad((xn, y) if res else (y,), leaves, (dxn, dy) if res else (dy,))))
    with torch.no_grad():
        xn2, h16, hq, sh, _ = G.rmsnorm_rows(x, wn, 1e-6, want_h=True, **kw)
        wq, sw = G.tcast_rows(w)
        y2, z = GR.gemm_rows_op(hq.view(-1, C), sh, wq, sw, b, act, None, None, True)
        rz, bound = R.gemm(hq.view(-1, C), sh, wq, sw, b)
        R.within(z, rz, bound, "z")
        R.within(y2, *R.gemm(hq.view(-1, C), sh, wq, sw, b, act), "y")
        assert torch.equal(y.view(-1, O), y2) and (not res or torch.equal(xn, xn2))
        xs, M, z, d = xn if res else x, B * N, z.double(), dy.double().view(-1, O)
        dz = d * R.dact(z, act)
        dq, sd = R.rowq(dz.float() * sw)
        dh = (R.deq(dq.to(dev), sd.to(dev)) @ wq.double()).to(BF).double().view(B, N, C)
        dz16 = dz.to(BF).double()
        ref = {"w": dz16.t() @ h16.double().view(M, C), "b": dz16.sum(0)}
        v = xs.double()
        rstd = (v.square().mean(-1, keepdim=True) + 1e-6) ** -0.5
        t = v * rstd
        dn = dh
        if kw["shift"] is not None:
            n = wn.double() * t
            dn = dh * (1 + scale.double())
            ref["shift"], ref["scale"] = dh.sum(1, keepdim=True), (dh * n).sum(1, keepdim=True)
        dt = dn * wn.double()
        ref["wn"] = (dn * t).sum((0, 1))
        base = dxn.double() if res else 0.0
        ref["x"] = rstd * (dt - t * (dt * t).mean(-1, keepdim=True)) + base
        if res:
            ref["a"] = ref["x"] * (gate.double() if kw["gate"] is not None else 1.0)
        if kw["gate"] is not None:
            ref["gate"] = (ref["x"] * a.double()).sum(1, keepdim=True)
        for k in got:
            assert rel(got[k], ref[k]) < 2 * R.UBF, (k, rel(got[k], ref[k]))
        assert set(ref) == set(got) and (M == 1 or rel(rstd * dt + base, ref["x"]) > 3 * R.UBF)

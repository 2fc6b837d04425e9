"""The row-scaled operators without a GPU: the C ABI's status codes, the Python refusals, layouts and fake kernels."""
import ctypes

import pytest
import torch

import gpic_fp8 as G
from gpic_fp8 import _lib as L
from gpic_fp8 import rows as GR

BF, F32, E4 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
EINVAL, EDTYPE, ESHAPE, EALIGN, EWORKSPACE = -1, -2, -3, -4, -5


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096 + 16)
    p.keep = buf
    return (ctypes.addressof(buf) + 15) // 16 * 16


def test_tcast_rows_codes(p):
    def f(x=p, dt=0, ld=64, rows=4, cols=64, q=p, s=p, x2=p, dt2=1, ld2=64, rows2=4, q2=p, s2=p):
        return L.lib().gpic_fp8_tcast_rows(x, dt, ld, rows, cols, q, s, x2, dt2, ld2, rows2, q2, s2, None)
    assert f(rows=0, rows2=0) == 0 and f(rows=0, x=None, q=None, s=None, x2=None, q2=None, s2=None) == 0
    assert f(rows2=-1) == EINVAL and f(q2=None) == EINVAL and f(s2=None) == EINVAL and f(dt2=9) == EDTYPE
    assert f(ld2=68) == ESHAPE and f(ld2=56) == ESHAPE and f(x2=p + 8) == EALIGN and f(q2=p + 8) == EALIGN
    assert f(rows=-1) == EINVAL and f(cols=0) == EINVAL and f(x=None) == EINVAL and f(q=None) == EINVAL and f(s=None) == EINVAL
    assert f(dt=7) == EDTYPE
    assert f(cols=60) == ESHAPE and f(ld=68) == ESHAPE and f(ld=56) == ESHAPE and f(cols=32776, ld=32776) == ESHAPE
    assert f(x=p + 8) == EALIGN and f(q=p + 8) == EALIGN


def test_rmsnorm_rows_codes(p):
    def f(x=p, ldx=64, a=p, lda=64, gate=p, sg=64, w=p, wd=1, sh=p, ssh=64, sc=p, ssc=64, rows=4, ntok=2, C=64, xn=p, h=None,
          rstd=p, q=p, s=p, wt=None, td=0, N=16, wq=p, sw=p):
        return L.lib().gpic_fp8_rmsnorm_rows(x, ldx, a, lda, gate, sg, w, wd, sh, ssh, sc, ssc, rows, ntok, C, 1e-6, xn, h,
                                             rstd, q, s, wt, td, N, wq, sw, None)
    assert f(rows=0) == 0
    assert f(wt=p, N=-1) == EINVAL and f(wt=p, wq=None) == EINVAL and f(wt=p, sw=None) == EINVAL and f(wt=p, td=3) == EDTYPE
    assert f(wt=p + 8) == EALIGN and f(wt=p, wq=p + 8) == EALIGN
    for bad in (dict(rows=-1), dict(C=0), dict(ntok=0), dict(a=None), dict(sh=None), dict(sc=None), dict(x=None), dict(w=None),
                dict(rstd=None), dict(q=None), dict(s=None), dict(xn=None)):
        assert f(**bad) == EINVAL, bad
    assert f(wd=2) == EDTYPE
    for bad in (dict(C=60), dict(C=16392, ldx=16392), dict(rows=5), dict(ldx=60), dict(ldx=56), dict(lda=60), dict(lda=56),
                dict(sg=60), dict(sg=56), dict(ssh=60), dict(ssh=56), dict(ssc=60), dict(ssc=56), dict(rows=1 << 31)):
        assert f(**bad) == ESHAPE, bad
    for name in ("x", "a", "gate", "w", "sh", "sc", "xn", "h", "q"):
        assert f(**{name: p + 8}) == EALIGN, name


def test_rmsnorm_rows_bwd_codes(p):
    def f(dh=p, dxn=p, xs=p, w=p, wd=0, rstd=p, rows=4, C=64, dx=p, dw=p, dd=1, ws=p, nws=1 << 20):
        return L.lib().gpic_fp8_rmsnorm_rows_bwd(dh, dxn, xs, w, wd, rstd, rows, C, dx, dw, dd, ws, nws, None)
    need = L.lib().gpic_fp8_rmsnorm_rows_bwd_workspace_bytes
    assert need(0, 64) == 0 and need(4, 64) >= 64 * 4 and need(1 << 20, 1024) % (1024 * 4) == 0
    for bad in (dict(rows=-1), dict(C=0), dict(dh=None), dict(xs=None), dict(w=None), dict(rstd=None), dict(dx=None),
                dict(dw=None)):
        assert f(**bad) == EINVAL, bad
    assert f(wd=5) == EDTYPE and f(dd=5) == EDTYPE
    assert f(C=60) == ESHAPE and f(C=16392) == ESHAPE
    assert f(nws=need(4, 64) - 1) == EWORKSPACE and f(ws=None) == EWORKSPACE
    for name in ("dh", "dxn", "xs", "w", "dx", "dw", "ws"):
        assert f(**{name: p + 8}) == EALIGN, name


def test_gemm_rows_codes(p):
    def f(A=p, lda=64, sa=p, B=p, ldb=64, sb=p, bias=p, bd=0, act=0, res=p, ldr=32, gate=p, sg=32, ntok=2, C=p, ldc=32, z=p,
          ldz=32, M=4, N=32, K=64, ws=None, nws=0):
        return L.lib().gpic_fp8_gemm_rows(A, lda, sa, B, ldb, sb, bias, bd, act, res, ldr, gate, sg, ntok, C, ldc, z, ldz, M, N,
                                          K, ws, nws, None)
    assert f(M=0) == 0 and f(N=0) == 0
    for bad in (dict(M=-1), dict(N=-16), dict(K=0), dict(A=None), dict(B=None), dict(C=None), dict(act=4), dict(act=-1),
                dict(ntok=0)):
        assert f(**bad) == EINVAL, bad
    assert f(bd=3) == EDTYPE
    for bad in (dict(K=72), dict(N=24), dict(lda=48), dict(ldb=48), dict(lda=72), dict(ldc=24), dict(ldc=36), dict(ldr=24),
                dict(ldr=36), dict(ldz=24), dict(sg=24), dict(M=5), dict(ldr=1 << 22), dict(ldz=1 << 22), dict(ldc=1 << 22), dict(sg=1 << 22),
                dict(act=3, N=48, ldz=48), dict(act=3, ldc=8), dict(act=3, ldr=8)):
        assert f(**bad) == ESHAPE, bad
    for name in ("A", "B", "C", "sb", "bias", "res", "gate", "z"):
        assert f(**{name: p + 8}) == EALIGN, name
    # (a plan that splits K: the workspace)
    assert L.lib().gpic_fp8_gemm_workspace_bytes(64, 1024, 8192) > 0
    assert f(M=64, N=1024, K=8192, lda=8192, ldb=8192, ldc=1024, ldr=1024, ldz=1024, sg=1024) == EWORKSPACE


def test_act_bwd_rows_codes(p):
    def f(dy=p, ldy=64, z=p, ldz=64, act=1, sw=p, rows=4, N=64, dz=p, q=p, s=p, wq=p, K=32, wqt=p, ldt=64, db=p, dd=0, ws=p,
          nws=1 << 20):
        return L.lib().gpic_fp8_act_bwd_rows(dy, ldy, z, ldz, act, sw, rows, N, dz, q, s, wq, K, wqt, ldt, db, dd, ws, nws, None)
    need = L.lib().gpic_fp8_act_bwd_rows_workspace_bytes
    assert need(0, 64) == 0 and need(4, 64) >= 64 * 4 and need(1 << 20, 1024) % (1024 * 4) == 0
    assert f(rows=0, wq=None, wqt=None, db=None) == 0
    for bad in (dict(rows=-1), dict(N=0), dict(act=3), dict(act=-1), dict(dy=None), dict(z=None), dict(sw=None), dict(dz=None),
                dict(q=None), dict(s=None), dict(wq=None), dict(wqt=None), dict(K=-16)):
        assert f(**bad) == EINVAL, bad
    assert f(dd=4) == EDTYPE
    for bad in (dict(N=60), dict(N=32776, ldy=32776, ldz=32776), dict(ldy=60), dict(ldy=56), dict(ldz=60), dict(ldz=56),
                dict(K=24), dict(ldt=48), dict(ldt=72), dict(K=1 << 40)):
        assert f(**bad) == ESHAPE, bad
    for name in ("dy", "z", "sw", "dz", "q", "wq", "wqt", "db", "ws"):
        assert f(**{name: p + 8}) == EALIGN, name
    assert f(nws=need(4, 64) - 1) == EWORKSPACE and f(ws=None) == EWORKSPACE


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 64, dtype=BF), torch.zeros(32, 64, dtype=BF)
    q, s = torch.zeros(4, 64).to(E4), torch.ones(4)
    for call in (lambda: G.tcast_rows(x), lambda: G.rmsnorm_rows(x, w[0], 1e-6), lambda: G.rows_weight(w),
                 lambda: G.rmsnorm_rows_bwd(x, None, x, w[0], s), lambda: G.fp8_gemm_rows(q, s, q, s),
                 lambda: G.act_bwd_rows(x, x, "silu", torch.ones(64)), lambda: G.fp8_linear_rows(x, w),
                 lambda: G.fp8_rmsnorm_linear_rows(x, w[0], 1e-6, w)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


@pytest.fixture
def no_gpu_check(monkeypatch):
    """The checks that follow the device's, on CPU tensors: none of these calls reaches the library."""
    monkeypatch.setattr(L, "require_gpu", lambda *t: None)

    def reached(*a):
        raise AssertionError("launched")
    monkeypatch.setattr(L, "lib", reached)


def test_refusals(no_gpu_check):
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)  # noqa: E731
    q, one = z(4, 64, dt=F32).to(E4), torch.ones(4)
    w = torch.ones(64)
    bad = [
        lambda: G.tcast_rows(z(4, 60)), lambda: G.tcast_rows(z(4, 0)), lambda: G.tcast_rows(z(2, 32776)),
        lambda: G.tcast_rows(torch.zeros(4, 64, dtype=torch.int32)),
        lambda: G.rmsnorm_rows(z(4, 60), w[:60], 1e-6), lambda: G.rmsnorm_rows(z(4, 64, dt=F32), w, 1e-6),
        lambda: G.rmsnorm_rows(z(2, 16392), torch.ones(16392), 1e-6), lambda: G.rmsnorm_rows(z(4, 64), w[:32], 1e-6),
        lambda: G.rmsnorm_rows(z(4, 64), w, 1e-6, z(4, 32)), lambda: G.rmsnorm_rows(z(4, 64), w, 1e-6, None, z(1, 64)),
        lambda: G.rmsnorm_rows(z(4, 64), w, 1e-6, None, None, z(1, 64)),
        lambda: G.rmsnorm_rows(z(4, 64), w, 1e-6, z(4, 64), z(3, 64)),
        lambda: G.rmsnorm_rows(z(4, 2, 64), w, 1e-6, z(4, 2, 64), z(2, 1, 64)),
        lambda: G.rmsnorm_rows(z(4, 64), w, 1e-6, None, None, z(2, 64), z(4, 64)),
        lambda: G.rmsnorm_rows(z(4, 64), w, 1e-6, None, None, z(1, 32), z(1, 32)),
        lambda: G.rmsnorm_rows_bwd(z(4, 64), z(3, 64), z(4, 64), w, one),
        lambda: G.rmsnorm_rows_bwd(z(4, 64), None, z(4, 64), w, one[:3]),
        lambda: G.rmsnorm_rows_bwd(z(4, 64), None, z(4, 64), w, one.double()),
        lambda: G.fp8_gemm_rows(q, one, q[:, :32], one), lambda: G.fp8_gemm_rows(q, one[:3], z(16, 64, dt=F32).to(E4), None),
        lambda: G.fp8_gemm_rows(q, None, z(24, 64, dt=F32).to(E4), None),
        lambda: G.fp8_gemm_rows(q, None, z(16, 64, dt=F32).to(E4), None, None, "swiglu"),
        lambda: G.fp8_gemm_rows(q, None, z(16, 64, dt=F32).to(E4), None, None, "relu6"),
        lambda: G.fp8_gemm_rows(q, None, z(16, 64, dt=F32).to(E4), None, torch.ones(8)),
        lambda: G.fp8_gemm_rows(q, None, z(16, 64, dt=F32).to(E4), None, None, "none", z(4, 32)),
        lambda: G.fp8_gemm_rows(q, None, z(16, 64, dt=F32).to(E4), None, None, "none", None, z(3, 16)),
        lambda: G.fp8_gemm_rows(z(4, 64), None, z(16, 64, dt=F32).to(E4), None),
        lambda: G.fp8_gemm_rows(q[:, :0], None, q[:, :0], None),
        lambda: G.act_bwd_rows(z(4, 64), None, "silu", w), lambda: G.act_bwd_rows(z(4, 64), z(4, 64), "swiglu", w),
        lambda: GR.act_bwd_rows_op(z(4, 64), None, "none", w, q), lambda: GR.act_bwd_rows_op(z(4, 64), None, "none", w, z(64, 32)),
        lambda: G.act_bwd_rows(z(4, 64, dt=F32), None, "none", w), lambda: G.act_bwd_rows(z(4, 64), None, "none", w[:32]),
        lambda: G.rows_weight(z(24, 64)), lambda: G.rows_weight(z(32, 24)), lambda: G.rows_weight(z(32, 64), "relu6"),
        lambda: G.rows_weight(z(16, 64), "swiglu"), lambda: G.swiglu_layout(z(16)),
        lambda: G.fp8_linear_rows(z(4, 32), z(16, 64)), lambda: G.fp8_linear_rows(z(4, 64), z(24, 64)),
        lambda: G.fp8_linear_rows(z(4, 64), z(32, 64), None, "swiglu"),
        lambda: G.fp8_linear_rows(z(4, 64), z(16, 64), None, "none", None, z(1, 16)),
        lambda: G.fp8_linear_rows(z(4, 64), z(16, 64), None, "none", z(2, 16)),
        lambda: G.fp8_linear_rows(z(4, 64), G.RowsWeight(z(32, 64, dt=F32).to(E4), torch.ones(32), True)),
        lambda: G.fp8_linear_rows(z(4, 64), G.RowsWeight(z(32, 64, dt=F32).to(E4), torch.ones(32), False), None, "swiglu"),
        lambda: G.fp8_linear_rows(z(4, 64).requires_grad_(), G.RowsWeight(z(32, 64, dt=F32).to(E4), torch.ones(32), False)),
        lambda: G.fp8_linear_rows(z(4, 64), G.RowsWeight(z(32, 64, dt=F32).to(E4), torch.ones(32), False), None, "none", z(2, 32)),
        lambda: G.fp8_linear_rows(z(4, 64), G.RowsWeight(z(32, 64, dt=F32).to(E4), torch.ones(32), True), None, "swiglu", z(4, 32)),
        lambda: G.fp8_rmsnorm_linear_rows(z(4, 64), w, 1e-6, z(16, 64), None, "none", None, None, z(1, 64), z(1, 64)),
        lambda: G.fp8_rmsnorm_linear_rows(z(1, 4, 64), w, 1e-6, z(16, 64), None, "none", z(1, 4, 64), z(1, 1, 64)),
        lambda: G.fp8_rmsnorm_linear_rows(z(1, 4, 64), w, 1e-6, z(16, 64), None, "none", z(1, 4, 64), None, z(1, 1, 64),
                                          z(1, 1, 64)),
        lambda: G.fp8_rmsnorm_linear_rows(z(1, 4, 4096), torch.ones(4096), 1e-6, z(16, 4096), None, "none", None, None,
                                          z(1, 1, 4096), z(1, 1, 4096)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_two_devices_are_refused(no_gpu_check):
    m = lambda *s: torch.zeros(*s, dtype=BF, device="meta")  # noqa: E731
    with pytest.raises(ValueError, match="is on"):
        G.rmsnorm_rows(torch.zeros(4, 64, dtype=BF), m(64), 1e-6)
    with pytest.raises(ValueError, match="is on"):
        G.fp8_gemm_rows(torch.zeros(4, 64).to(E4), None, torch.zeros(16, 64).to(E4), None, residual=m(4, 16))


def test_swiglu_layout():
    t = torch.arange(2 * 48 * 3).view(96, 3)
    o = G.swiglu_layout(t)
    for h in range(48):
        r = h // 4 * 8 + h % 4
        assert torch.equal(o[r], t[h]) and torch.equal(o[r + 4], t[48 + h])
    assert torch.equal(G.swiglu_layout(t[:, 0]), o[:, 0])


def test_fake_kernels():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        q, s = GR.tcast_rows_op(e(2, 3, 64))
        assert q.shape == (2, 3, 64) and q.dtype == E4 and s.shape == (6,) and s.dtype == F32
        xn, h, q, s, r = GR.rmsnorm_rows_op(e(2, 3, 64), e(64, dt=F32), 1e-6, e(2, 3, 64), None, None, None, True)
        assert xn.shape == h.shape == q.shape == (2, 3, 64) and s.shape == r.shape == (6,) and xn.dtype == h.dtype == BF
        assert GR.rmsnorm_rows_op(e(3, 64), e(64), 1e-6)[0].numel() == 0
        dx, dw = GR.rmsnorm_rows_bwd_op(e(3, 64), None, e(3, 64), e(64), e(3, dt=F32))
        assert dx.shape == (3, 64) and dw.shape == (64,) and dw.dtype == BF
        y, z = GR.gemm_rows_op(e(3, 64, dt=E4), None, e(32, 64, dt=E4), None, None, "swiglu", None, None, True)
        assert y.shape == (3, 16) and z.shape == (3, 32) and y.dtype == z.dtype == BF
        dz, q, s, t, b = GR.act_bwd_rows_op(e(3, 64), e(3, 64), "silu", e(64, dt=F32), e(64, 32, dt=E4), True, True)
        assert dz.shape == q.shape == (3, 64) and s.shape == (3,) and q.dtype == E4
        assert t.shape == (32, 64) and b.shape == (64,) and b.dtype == F32


def test_host_module_takes_no_cpu_tensors():
    h = L.host()
    x, w, v = torch.zeros(16, 16, dtype=BF), torch.zeros(16, 16), torch.ones(16)
    q = torch.zeros(16, 16).to(E4)
    n = None
    assert h.cast_rows(x, 0, 0, 0) is None
    assert h.norm_rows(x, v, 1e-6, n, n, n, n, False, 0, 0, 0) is None
    assert h.norm_rows_bwd(x, n, x, v, v, 0, 0, 0) is None
    assert h.gemm_rows(q, n, q, n, n, 0, n, n, False, 0, 0, 0) is None
    assert h.linear_rows(x, w, n, 0, n, 0, 0, 0) is None
    assert h.norm_linear_rows(x, v, 1e-6, n, w, n, 0, 0, 0, 0) is None
    assert h.linear_served(x, q, v, n, 0, n, n, 0, 0, 0) is None
    assert h.norm_linear_served(x, v, 1e-6, n, n, n, n, q, v, n, 0, 0, 0, 0) is None
    assert h.linear_rows_bwd(x, x, 0, q, v, x, True, True, True, True, True, 0, 0, 0) is None
    assert h.norm_linear_rows_fwd(x, v, 1e-6, n, n, n, n, w, n, 0, True, True, 0, 0, 0) is None


def test_public_calls_on_fake_tensors():
    """Tensors without memory (a shape pass over a program) go to the ops' fake kernels."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        q, s = G.tcast_rows(e(6, 64))
        assert G.rmsnorm_rows(e(2, 3, 64), e(64), 1e-6, e(2, 3, 64))[0].shape == (2, 3, 64)
        assert G.rmsnorm_rows_bwd(e(3, 64), None, e(3, 64), e(64), e(3, dt=F32))[1].shape == (64,)
        assert G.fp8_gemm_rows(q, s, e(32, 64, dt=E4), e(32, dt=F32), act="swiglu").shape == (6, 16)
        assert G.act_bwd_rows(e(3, 64), e(3, 64), "silu", e(64, dt=F32))[1].dtype == E4


def test_served_weights_that_take_a_gradient(no_gpu_check):
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)  # noqa: E731
    q, s = z(32, 64, dt=F32).to(E4), torch.ones(32)
    for w in (G.RowsWeight(q.clone().requires_grad_(), s, False), G.RowsWeight(q, s.clone().requires_grad_(), False)):
        with pytest.raises(ValueError, match="RowsWeight"):
            G.fp8_linear_rows(z(4, 64), w)
        with pytest.raises(ValueError, match="RowsWeight"):
            G.fp8_rmsnorm_linear_rows(z(4, 64), torch.ones(64), 1e-6, w)


def test_gate_rows_follow_the_batch(no_gpu_check):
    z = lambda *s, dt=BF: torch.zeros(*s, dtype=dt)  # noqa: E731
    w = G.RowsWeight(z(32, 64, dt=F32).to(E4), torch.ones(32), False)
    for x, gate in ((z(2, 3, 64), z(3, 1, 32)), (z(2, 3, 64), z(6, 32)), (z(1, 6, 64), z(2, 1, 32)), (z(2, 3, 4, 64), z(6, 32))):
        with pytest.raises(ValueError, match="gate has"):
            G.fp8_linear_rows(x, w, None, "none", None, gate)


def test_no_rows_need_no_memory(p):
    """No rows: their tensors have no memory, and the modulation's may have some."""
    def f(x=None, a=None, gate=p, sh=p, sc=p, rows=0, xn=None):
        return L.lib().gpic_fp8_rmsnorm_rows(x, 64, a, 64, gate, 64, p, 1, sh, 64, sc, 64, rows, 1, 64, 1e-6, xn, None, None, None,
                                             None, None, 0, 0, None, None, None)
    assert f() == 0 and f(gate=None) == 0 and f(gate=None, sh=None, sc=None) == 0 and f(sh=None) == EINVAL
    assert f(x=p, rows=4) == EINVAL


def test_linears_on_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        w, b, wn = e(32, 64).requires_grad_(), e(32), e(64, dt=F32)
        served = G.RowsWeight(e(32, 64, dt=E4), e(32, dt=F32), True)
        assert G.fp8_linear_rows(e(2, 3, 64), w, b, "silu", e(2, 3, 32)).shape == (2, 3, 32)
        assert G.fp8_linear_rows(e(2, 3, 64), served, None, "swiglu", e(2, 3, 16), e(2, 1, 16)).shape == (2, 3, 16)
        assert [t.shape for t in G.fp8_rmsnorm_linear_rows(e(2, 3, 64), wn, 1e-6, w, b, "silu", e(2, 3, 64))] == [(2, 3, 64), (2, 3, 32)]
        m = e(2, 1, 6 * 64).chunk(6, -1)
        for weight, act, n in ((w, "gelu_tanh", 32), (served, "swiglu", 16)):
            xn, y = G.fp8_rmsnorm_linear_rows(e(2, 3, 64), wn, 1e-6, weight, None, act, e(2, 3, 64), m[2], m[3], m[4])
            assert xn.shape == (2, 3, 64) and y.shape == (2, 3, n) and y.dtype == BF


def test_host_module_takes_no_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        e = lambda *s, dt=BF: torch.empty(*s, dtype=dt, device="cuda")  # noqa: E731
        x, w, v, q = e(16, 16), e(16, 16), e(16, dt=F32), e(16, 16, dt=E4)
    h, n = L.host(), None
    assert h.cast_rows(x, 0, 0, 0) is None
    assert h.gemm_rows(q, n, q, n, n, 0, n, n, False, 0, 0, 0) is None
    assert h.linear_served(x, q, v, n, 0, n, n, 0, 0, 0) is None
    for mod in ((n, n, n), (x, v, v)):   # (the modulation's rows are looked at apart)
        assert h.norm_rows(x, v, 1e-6, x, *mod, False, 0, 0, 0) is None
    assert h.norm_rows_bwd(x, n, x, v, v, 0, 0, 0) is None
    assert h.linear_rows(x, w, n, 0, n, 0, 0, 0) is None
    assert h.norm_linear_rows(x, v, 1e-6, n, w, n, 0, 0, 0, 0) is None
    assert h.norm_linear_served(x, v, 1e-6, n, n, n, n, q, v, n, 0, 0, 0, 0) is None
    assert h.linear_rows_bwd(x, x, 0, q, v, x, True, True, True, True, True, 0, 0, 0) is None
    assert h.norm_linear_rows_fwd(x, v, 1e-6, n, n, n, n, w, n, 0, True, True, 0, 0, 0) is None

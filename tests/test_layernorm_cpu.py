"""Layer norm without a GPU: the formula of its gradients against differences, refusals, fake kernels, the C entry's checks."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gpic_fp8 as G
from gpic_fp8 import _lib as L
from norm_ref import layer_norm64, layer_norm_grads64

BF, F32 = torch.bfloat16, torch.float32


def test_the_formulas_gradients_are_the_differences():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x, w, b, dh = r(5, 24) * 3 + 1, r(24), r(24), r(5, 24)
    dx, dw, db = layer_norm_grads64(dh, None, x, w, 1e-5)
    loss = lambda x, w, b: (layer_norm64(x, w, b, 1e-5)[0] * dh).sum()  # noqa: E731
    for v, grad, f in ((r(5, 24), dx, lambda e, v: loss(x + e * v, w, b)), (r(24), dw, lambda e, v: loss(x, w + e * v, b)),
                       (r(24), db, lambda e, v: loss(x, w, b + e * v))):
        e = 1e-5   # differences off by e^2 and by 1e-16 / e of the loss
        diff = (f(e, v) - f(-e, v)) / (2 * e)
        assert abs(diff - (grad * v).sum()) < 1e-7 * (1 + abs(diff))


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=BF)
    for call in (lambda: G.layer_norm(x), lambda: G.layer_norm_rows(x),
                 lambda: G.layer_norm_bwd(x, None, x, None, torch.zeros(2), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_fake_tensors_take_the_fake_kernels():
    with FakeTensorMode():
        x = torch.empty(3, 5, 64, dtype=BF, device="cuda")
        w = torch.empty(64, dtype=F32, device="cuda")
        xn, h = G.layer_norm(x, w, w, 1e-5, x)
        assert xn.shape == h.shape == x.shape and h.dtype == BF
        xn, h, q, s = G.layer_norm_rows(x, w, w)
        assert xn.numel() == h.numel() == 0 and q.shape == x.shape and q.dtype == G.E4 and s.shape == (15,)
        dx, dw, db = G.layer_norm_bwd(x, None, x, w, s, s, BF)
        assert dx.shape == x.shape and dw.shape == (64,) and dw.dtype == F32 and db.shape == (64,) and db.dtype == BF


def test_the_c_entry_checks():
    lib = L.lib()
    buf = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    fwd, bwd, nws = lib.gpic_fp8_layer_norm, lib.gpic_fp8_layer_norm_bwd, lib.gpic_fp8_layer_norm_bwd_workspace_bytes
    ok = dict(x=p, dt=0, ldx=64, a=None, lda=0, w=p, wt=0, b=p, bt=0, rows=2, C=64, eps=1e-5, xn=None, h=p, mean=None,
              rstd=None, q=None, s=None)
    call = lambda **k: fwd(*{**ok, **k}.values(), None)  # noqa: E731
    assert call(rows=0) == 0
    assert call(rows=-1) == call(C=0) == call(x=None) == call(h=None) == call(a=p) == call(mean=p) == call(q=p) == -1
    assert call(dt=3) == call(wt=-1) == call(bt=7) == call(dt=2, q=p, s=p) == -2
    assert call(C=60) == call(C=16392, ldx=16392) == call(ldx=56) == call(ldx=68) == call(rows=1 << 31) == -3
    assert call(a=p, xn=p, lda=8) == -3
    assert call(x=p + 8) == call(w=p + 2) == call(b=p + 4) == call(h=p + 8) == -4
    okb = dict(dh=p, dxn=None, xs=p, dt=0, w=p, wt=0, mean=p, rstd=p, rows=2, C=64, dx=p, dw=p, dwt=0, db=p, dbt=0, ws=p, n=4096)
    call = lambda **k: bwd(*{**okb, **k}.values(), None)  # noqa: E731
    assert nws(0, 64) == nws(2, 0) == 0 and nws(2, 64) == 1 * 64 * 8
    assert call(rows=-1) == call(dh=None) == call(xs=None) == call(mean=None) == call(dx=None) == -1
    assert call(dt=5) == call(wt=3) == call(dwt=3) == call(dbt=4) == -2
    assert call(C=60) == call(C=16392) == -3
    assert call(dh=p + 2) == call(dw=p + 8) == call(ws=p + 4) == -4
    assert call(n=511) == call(ws=None) == -5

"""Cross attention without a GPU: the reference's gradients against differences, refusals, fake kernels, the C entries' checks."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gpic_fp8 as G
from attn_ref import attend, valid_keys
from gpic_fp8 import _lib as L

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def test_the_formulas_gradients_are_the_differences():
    """The formulas that the GPU tests hold the backward to, against differences of the 64-bit forward."""
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    q, k, v, do = r(2, 4, 3, 8), r(2, 2, 5, 8), r(2, 2, 5, 8), r(2, 4, 3, 8)
    ok = valid_keys(2, 5, torch.tensor([4, 2]), torch.tensor([[1, 0, 1, 1, 1], [1, 1, 1, 1, 1]], dtype=torch.bool))
    s = 0.4
    o, P, _, q6, k6, v6 = attend(q, k, v, ok, s)
    d6 = do.reshape(2, 2, 6, 8)
    dS = P * (d6 @ v6.transpose(2, 3) - (d6 * o).sum(-1, keepdim=True))
    grads = {"q": s * (dS @ k6).reshape(q.shape), "k": s * (dS.transpose(2, 3) @ q6), "v": P.transpose(2, 3) @ d6}
    base = dict(q=q, k=k, v=v)
    for name, t in base.items():
        x = r(*t.shape)
        f = lambda e: (attend(**{**base, name: t + e * x}, ok=ok, scale=s)[0] * d6).sum()  # noqa: E731
        diff = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(diff - (grads[name] * x).sum()) < 1e-8 * (1 + abs(diff)), name


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(1, 2, 3, 16, dtype=BF), torch.zeros(1, 2, 5, 16, dtype=BF)
    for call in (lambda: G.cross_attention(q, k, k), lambda: G.cross_attention_fwd(q, k, k),
                 lambda: G.cross_attention_bwd(q, q, k, k, q, torch.zeros(1, 2, 3))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_fake_tensors_take_the_fake_kernels():
    with FakeTensorMode():
        q = torch.empty(2, 7, 8, 64, dtype=BF, device="cuda").transpose(1, 2).requires_grad_()
        k = torch.empty(2, 2, 9, 64, dtype=BF, device="cuda")
        lens = torch.empty(2, dtype=torch.int32, device="cuda")
        o = G.cross_attention(q, k, k, lens)
        assert o.shape == q.shape and o.stride() == q.stride() and o.dtype == BF
        o, lse = G.cross_attention_fwd(q.detach(), k, k)
        assert lse.shape == (2, 8, 7) and lse.dtype == F32
        dq, dk, dv = G.cross_attention_bwd(o, q.detach(), k, k, o, lse)
        assert dq.shape == q.shape and dk.shape == dv.shape == k.shape


@pytest.fixture(scope="module")
def p():
    buf = ctypes.create_string_buffer(4096 + 16)
    p.keep = buf
    return (ctypes.addressof(buf) + 15) // 16 * 16


S = lambda *v: (ctypes.c_int64 * 3)(*v)  # noqa: E731


def test_forward_codes(p):
    ok = dict(q=p, qs=S(0, 16, 16), k=p, ks=S(0, 16, 16), v=p, vs=S(0, 16, 16), dt=0, lens=None, mask=None, ldm=0, B=1, H=2, Hk=1,
              N=3, L=5, D=16, scale=0.25, o=p, os=S(0, 16, 32), lse=None, ws=None, n=0)
    call = lambda **k: L.lib().gpic_fp8_attention(*{**ok, **k}.values(), None)  # noqa: E731
    need = L.lib().gpic_fp8_attention_workspace_bytes
    assert call(N=0) == 0 and call(B=0, q=None, o=None) == 0
    for bad in (dict(B=-1), dict(H=0), dict(Hk=0), dict(N=-1), dict(L=-1), dict(D=0), dict(q=None), dict(k=None), dict(v=None),
                dict(o=None), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(qs=None),
                dict(mask=p, ldm=-1), dict(ks=S(0, -8, 8))):
        assert call(**bad) == -1, bad
    assert call(dt=1) == call(dt=3) == -2
    for bad in (dict(D=12), dict(D=136), dict(H=3, Hk=2), dict(N=1 << 31), dict(L=1 << 31), dict(B=1 << 24),
                dict(H=1 << 20, N=1 << 12)):
        assert call(**bad) == -3, bad
    for bad in (dict(q=p + 8), dict(k=p + 2), dict(v=p + 8), dict(o=p + 4), dict(qs=S(0, 12, 16)), dict(os=S(4, 16, 32))):
        assert call(**bad) == -4, bad
    assert need(0, 2, 1, 3, 5, 16) == need(1, 2, 1, 0, 5, 16) == need(1, 3, 2, 4, 5, 16) == 0
    n = need(1, 2, 1, 1, 8192, 64)   # few rows over long states: split
    assert n > 0 and n % (2 * 66 * 4) == 0
    assert call(N=1, L=8192, n=n - 1, ws=p) == call(N=1, L=8192, n=n, ws=None) == -5


def test_backward_codes(p):
    s = S(0, 16, 16)
    ok = dict(do=p, ds=s, q=p, qs=s, k=p, ks=s, v=p, vs=s, o=p, os=s, lse=p, dt=0, lens=None, mask=None, ldm=0, B=1, H=2, Hk=1, N=3,
              L=5, D=16, scale=0.25, dq=p, dqs=s, dk=p, dks=s, dv=p, dvs=s, ws=p, n=1 << 20)
    call = lambda **k: L.lib().gpic_fp8_attention_bwd(*{**ok, **k}.values(), None)  # noqa: E731
    assert call(B=0) == 0 and call(N=0, L=0) == 0
    for bad in (dict(do=None), dict(q=None), dict(o=None), dict(lse=None), dict(dq=None), dict(k=None), dict(v=None), dict(dk=None),
                dict(dv=None), dict(scale=0.0), dict(Hk=0), dict(dqs=None), dict(dks=None)):
        assert call(**bad) == -1, bad
    assert call(dt=1) == -2 and call(D=20) == call(H=3, Hk=2) == -3
    for bad in (dict(do=p + 8), dict(dq=p + 2), dict(dk=p + 8), dict(dv=p + 8), dict(dvs=S(0, 16, 4)), dict(ws=p + 8)):
        assert call(**bad) == -4, bad
    n = L.lib().gpic_fp8_attention_bwd_workspace_bytes(1, 2, 1, 3, 5, 16)
    assert n >= 4 * 6 and call(n=n - 1) == call(ws=None, n=n) == -5


def test_workspaces_of_nothing():
    fwd, bwd = L.lib().gpic_fp8_attention_workspace_bytes, L.lib().gpic_fp8_attention_bwd_workspace_bytes
    for B, N, n in ((0, 4, 5), (0, 100, 5), (2, 0, 5), (2, 4, 0), (0, 0, 0)):
        assert fwd(B, 4, 4, N, n, 64) == 0 and bwd(B, 4, 2, N, n, 64) >= 0

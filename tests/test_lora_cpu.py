"""Per-request adapters without a GPU: refusals, the fake kernel, the C entry's checks."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import gpic_fp8 as G
from gpic_fp8 import _lib as L

BF = torch.bfloat16


def test_cpu_tensors_are_refused():
    y, x, A, B = (torch.zeros(*s, dtype=BF) for s in ((2, 16), (2, 32), (1, 8, 32), (1, 16, 8)))
    with pytest.raises(RuntimeError, match="GPU only"):
        G.lora_rows(y, x, A, B, torch.zeros(2, dtype=torch.int32))


def test_fake_tensors_take_the_fake_kernel():
    with FakeTensorMode():
        y, x, A, B = (torch.empty(*s, dtype=BF, device="cuda") for s in ((2, 3, 16), (2, 3, 32), (1, 8, 32), (1, 16, 8)))
        out = G.lora_rows(y, x, A, B, torch.empty(2, dtype=torch.int32, device="cuda"))
        assert out.shape == y.shape and out.dtype == BF


def test_the_c_entry_checks():
    buf = ctypes.create_string_buffer(4096 + 16)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    ok = dict(y=p, ldy=16, x=p, ldx=32, A=p, B=p, s=None, ids=p, wide=0, per=1, dt=0, M=4, N=16, K=32, R=8, n=2, out=p, ws=p, nws=4096)
    call = lambda **k: L.lib().gpic_fp8_lora_rows(*{**ok, **k}.values(), None)  # noqa: E731
    need = L.lib().gpic_fp8_lora_rows_workspace_bytes
    assert call(M=0) == 0 and call(M=0, y=None, x=None, ids=None, out=None, ws=None, nws=0) == 0
    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(R=0), dict(n=0), dict(per=0), dict(y=None), dict(x=None), dict(A=None),
                dict(B=None), dict(ids=None), dict(out=None)):
        assert call(**bad) == -1, bad
    assert call(dt=1) == call(dt=3) == -2
    for bad in (dict(N=20), dict(K=20), dict(R=12), dict(R=136), dict(ldx=24), dict(ldx=36), dict(ldy=8), dict(ldy=20),
                dict(M=1 << 30), dict(n=1 << 30), dict(N=1 << 24, ldy=1 << 24), dict(ldx=1 << 24), dict(ldy=1 << 24),
                dict(K=1 << 24, ldx=1 << 24)):
        assert call(**bad) == -3, bad
    for bad in (dict(y=p + 8), dict(x=p + 2), dict(A=p + 8), dict(B=p + 8), dict(out=p + 8), dict(ws=p + 8)):
        assert call(**bad) == -4, bad
    assert need(0, 16, 32, 8, 2) == need(4, 16, 32, 136, 2) == 0
    n = need(4, 16, 32, 8, 2)
    assert n >= 4 * 8 * 4 and call(nws=n - 1) == call(ws=None) == -5

"""Layer norm on the GPU against 64 bits: types, widths, strides, residual, absent weights, far means, odd values, gradients, graphs,
streams, the e4m3 form into the row-scaled GEMM."""
import pytest
import torch

import gpic_fp8 as G
from norm_ref import (U32, dx_bound, grads_of, h_bound, layer_norm64, layer_norm_grads64, stats64, sum_bound)
from rows_ref import deq, rowq

pytestmark = pytest.mark.gpu
BF, FP, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
EPS = 1e-5


def make(shape, dt, seed=0, mean=0.3, std=1.0, wdt=None, bdt=None, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = (r(*shape) * std + mean).to(dt)
    a, dh, dxn = r(*shape).to(dt), (0.1 * r(*shape)).to(dt), (0.1 * r(*shape)).to(dt)
    w, b = (1 + 0.2 * r(C)).to(wdt or dt), (0.2 * r(C)).to(bdt or dt)
    return [t.to(dev) for t in (x, a, w, b, dh, dxn)]


def inside(got, ref, bound, what=""):
    err = (got.to(F64) - ref).abs()
    over = err > bound
    assert not over.any(), (what, int(over.sum()), float((err / bound.clamp_min(1e-300)).max()))


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("shape", [(1, 8), (1, 1024), (3, 64), (7, 520), (5, 3, 1032), (257, 896), (9, 2056), (6, 4104), (3, 8200),
                                   (2, 16384), (8195, 64), (2, 2049, 136)])
@pytest.mark.parametrize("res", [False, True])
def test_forward(dev, dt, shape, res):
    x, a, w, b, _, _ = make(shape, dt)
    out = G.layer_norm(x, w, b, EPS, a if res else None)
    xs = x
    if res:
        xn, h = out
        xs = (x.float() + a.float()).to(dt)
        assert torch.equal(xn, xs) and xn.shape == x.shape
    else:
        h = out
    assert h.dtype == dt and h.shape == x.shape
    w64, b64 = w.to(F64), b.to(F64)
    ref, t = layer_norm64(xs.to(F64), w64, b64, EPS)
    inside(h, ref, h_bound(ref, t, w64, b64, dt))


@pytest.mark.parametrize("dt,wdt,bdt", [(BF, F32, FP), (F32, BF, None), (FP, F32, BF), (BF, F64, F32)])
def test_weights_of_other_types(dev, dt, wdt, bdt):
    x, a, w, b, dh, dxn = make((33, 264), dt, 1, wdt=wdt, bdt=bdt)
    w, b, x = w.requires_grad_(), b.requires_grad_(), x.requires_grad_()
    h = G.layer_norm(x, w, b, EPS)
    w64, b64 = w.detach().to(F64), b.detach().to(F64)
    if wdt == F64:
        w64 = w.detach().to(F32).to(F64)
    ref, t = layer_norm64(x.detach().to(F64), w64, b64, EPS)
    inside(h, ref, h_bound(ref, t, w64, b64, dt))
    dx, dw, db = torch.autograd.grad(h, (x, w, b), dh)
    assert dx.dtype == dt and dw.dtype == w.dtype and db.dtype == b.dtype
    inside(db, dh.to(F64).sum(0), sum_bound(dh.to(F64).sum(0), dh.to(F64).abs().sum(0), 33, F32 if b.dtype == F64 else b.dtype))


@pytest.mark.parametrize("w_on,b_on", [(False, False), (True, False), (False, True)])
def test_absent_weight_or_bias(dev, w_on, b_on):
    x, a, w, b, dh, dxn = make((19, 512), BF, 2)
    w, b = w if w_on else None, b if b_on else None
    leaves = [t.requires_grad_() for t in (x, w, b) if t is not None]
    h = G.layer_norm(x, w, b, EPS)
    f = lambda t: None if t is None else t.detach().to(F64)  # noqa: E731
    ref, t = layer_norm64(f(x), f(w), f(b), EPS)
    inside(h, ref, h_bound(ref, t, f(w), f(b), BF))
    grads = torch.autograd.grad(h, leaves, dh)
    _, r, d = stats64(f(x), EPS)
    dx, dw, db, size = grads_of(f(dh), None, d * r, r, f(w))
    # (the kernel's mean and rstd are rounded to fp32: 2^-24 of |mean| rstd in t, 2^-24 of t, against values of order one)
    inside(grads[0], dx, dx_bound(dx, 2 * size, BF))
    if w_on:
        inside(grads[1], dw, sum_bound(dw, 2 * ((f(dh) * t).abs()).sum(0), 19, BF))
    if b_on:
        inside(grads[-1], db, sum_bound(db, f(dh).abs().sum(0), 19, BF))


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("shape", [(1, 8), (1, 1024), (7, 520), (5, 3, 1032), (2051, 256), (9, 2056), (6, 4104), (3, 8200),
                                   (2, 16384), (4099, 64)])
@pytest.mark.parametrize("res", [False, True])
def test_backward_op(dev, dt, shape, res):
    """Given mean and rstd: the formula on them, in 64 bits."""
    x, a, w, b, dh, dxn = make(shape, dt, 3)
    if not res:
        dxn = None
    mu, r, _ = stats64(x.to(F64), EPS)
    mean, rstd = mu.reshape(-1).float(), r.reshape(-1).float()
    dx, dw, db = G.layer_norm_bwd(dh, dxn, x, w, mean, rstd, dt)
    r64 = rstd.to(F64).view(r.shape)
    t = (x.to(F64) - mean.to(F64).view(mu.shape)) * r64
    f = lambda t: None if t is None else t.to(F64)  # noqa: E731
    rx, rw, rb, size = grads_of(f(dh), f(dxn), t, r64, f(w))
    rows, C = mean.numel(), shape[-1]
    inside(dx, rx, dx_bound(rx, size, dt), "dx")
    inside(dw, rw, sum_bound(rw, (f(dh) * t).abs().reshape(rows, C).sum(0), rows, dt), "dw")
    inside(db, rb, sum_bound(rb, f(dh).abs().reshape(rows, C).sum(0), rows, dt), "db")
    again = G.layer_norm_bwd(dh, dxn, x, w, mean, rstd, dt)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def test_gradients_through_autograd(dev):
    x, a, w, b, dh, dxn = make((3, 41, 768), F32, 4)
    for t in (x, a, w, b):
        t.requires_grad_()
    xn, h = G.layer_norm(x, w, b, EPS, a)
    gx, ga, gw, gb = torch.autograd.grad((xn, h), (x, a, w, b), (dxn, dh))
    assert torch.equal(gx, ga)
    xs = xn.detach().to(F64)
    w64 = w.detach().to(F64)
    _, r, d = stats64(xs, EPS)
    rx, rw, rb, size = grads_of(dh.to(F64), dxn.to(F64), d * r, r, w64)
    # rstd is off by (K + 8) 2^-24 and mean by K 2^-24 deviations (h_bound): t and r by as much, which enters dx twice
    inside(gx, rx, dx_bound(rx, 64 * size, F32))
    inside(gw, rw, sum_bound(rw, 8 * (dh.to(F64) * d * r).abs().reshape(123, -1).sum(0) + 8 * dh.to(F64).abs().reshape(123, -1).sum(0),
                             123, F32))
    inside(gb, rb, sum_bound(rb, dh.to(F64).abs().reshape(123, -1).sum(0), 123, F32))
    # differences of the 64-bit forward along a direction
    v = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).to(x.device, F64)
    e = 1e-6
    loss = lambda s: (layer_norm64(s, w64, b.detach().to(F64), EPS)[0] * dh.to(F64)).sum() + (s * dxn.to(F64)).sum()  # noqa: E731
    diff = (loss(xs + e * v) - loss(xs - e * v)) / (2 * e)
    proj = (gx.to(F64) * v).sum()
    assert abs(diff - proj) <= (dx_bound(rx, 64 * size, F32) * v.abs()).sum() + 1e-6 * abs(diff) + 1e-6


def test_outputs_used_alone_and_partly(dev):
    x, a, w, b, dh, dxn = make((5, 64), BF, 6)
    for t in (x, a, w, b):
        t.requires_grad_()
    xn, h = G.layer_norm(x, w, b, EPS, a)
    gx, ga, gw, gb = torch.autograd.grad(xn, (x, a, w, b), dxn)
    assert torch.equal(gx, dxn) and torch.equal(ga, dxn) and not gw.any() and not gb.any()
    xn, h = G.layer_norm(x, w, b, EPS, a)
    (ga,) = torch.autograd.grad(h, (a,), dh)
    assert torch.isfinite(ga).all()
    h = G.layer_norm(x.detach(), w, b.detach(), EPS)
    (gw,) = torch.autograd.grad(h, (w,), dh)
    _, r, d = stats64(x.detach().to(F64), EPS)
    ref = (dh.to(F64) * d * r).sum(0)
    inside(gw, ref, sum_bound(ref, 8 * (dh.to(F64).abs() * (1 + (d * r).abs())).sum(0), 5, BF))


def test_far_means_keep_their_digits(dev):
    """Rows of mean 4096 and deviation 1 in fp32: the deviations are exact to 2^-12 steps of the inputs, not of a rounded mean."""
    x, a, w, b, _, _ = make((64, 1000), F32, 7, mean=4096.0)
    h = G.layer_norm(x, w, b, EPS)
    ref, t = layer_norm64(x.to(F64), w.to(F64), b.to(F64), EPS)
    inside(h, ref, h_bound(ref, t, w.to(F64), b.to(F64), F32))


def test_constant_rows_and_special_values(dev):
    x = torch.full((4, 128), 3.25, dtype=BF, device=dev)
    w, b = torch.ones(128, device=dev), torch.full((128,), 0.5, device=dev)
    assert torch.equal(G.layer_norm(x, w, b), torch.full_like(x, 0.5))
    x[1, 5], x[2, 7] = float("nan"), float("inf")
    h = G.layer_norm(x, w, b)
    assert h[1].isnan().all() and h[2].isnan().all() and torch.equal(h[[0, 3]], torch.full_like(x[:2], 0.5))
    q, s = G.layer_norm_rows(x, w, b)[2:]
    assert s[1].isnan() and s[2].isnan() and s[[0, 3]].isfinite().all()


def test_strides_orders_and_offsets(dev):
    x, a, w, b, _, _ = make((6, 5, 128), BF, 8)
    ref = G.layer_norm(x, w, b, EPS, a)
    wide = torch.zeros(6, 5, 384, dtype=BF, device=dev)
    wide[..., 128:256] = x
    odd = torch.zeros(30 * 128 + 1, dtype=BF, device=dev)
    odd[1:] = a.reshape(-1)
    back = torch.empty(128, dtype=BF, device=dev).copy_(w.flip(0)).flip(0)
    for xv, av in ((wide[..., 128:256], a), (x, odd[1:].view(6, 5, 128)), (x.transpose(0, 1).contiguous().transpose(0, 1), a),
                   (x, a.to(F32))):
        got = G.layer_norm(xv, back, b, EPS, av)
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
    same = x[:1].expand(6, 5, 128)
    assert torch.equal(G.layer_norm(same, w, b)[3], G.layer_norm(x[:1].contiguous(), w, b)[0])


def test_no_rows(dev):
    x = torch.empty(0, 64, dtype=BF, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    h = G.layer_norm(x, w, w.detach())
    gx, gw = torch.autograd.grad(h, (x, w), torch.empty_like(h))
    assert h.shape == gx.shape == (0, 64) and not gw.any()
    assert G.layer_norm_rows(x.detach(), w.detach())[2].shape == (0, 64)


@pytest.mark.parametrize("shape", [(1, 1024), (7, 520), (3, 11, 1032), (2, 16384), (4097, 64), (5, 2056)])
@pytest.mark.parametrize("res,want_h", [(False, False), (True, False), (True, True)])
def test_rows_form(dev, shape, res, want_h):
    x, a, w, b, _, _ = make(shape, BF, 9, wdt=F32)
    xn, h, q, s = G.layer_norm_rows(x, w, b, EPS, a if res else None, want_h)
    xs = (x.float() + a.float()).to(BF) if res else x
    assert torch.equal(xn, xs) if res else xn.numel() == 0
    w64, b64 = w.to(F64), b.to(F64)
    ref, t = layer_norm64(xs.to(F64), w64, b64, EPS)
    e = h_bound(ref, t, w64, b64, F32)
    if want_h:
        inside(h, ref, h_bound(ref, t, w64, b64, BF))
    C = shape[-1]
    amax = ref.abs().reshape(-1, C).amax(1)
    inside(s, amax / 448, (e.reshape(-1, C).amax(1) + 3 * U32 * amax) / 448)
    # a value over its scale rounds to e4m3: half a step is 2^-4 of it, or 2^-10 among the subnormals
    inside(deq(q.cpu(), s.cpu()).to(dev), ref,
           (2.0 ** -4 * ref.abs()).clamp_min(1e-30) + 2.0 ** -10 * s.to(F64).view(*shape[:-1], 1) + 2 * e + 4 * U32 * ref.abs())


def test_rows_form_feeds_the_gemm(dev):
    """The norm's bytes into a served projection, against the projection of the norm's bf16 output."""
    x, a, w, b, _, _ = make((37, 512), BF, 10)
    W = (torch.randn(256, 512, generator=torch.Generator().manual_seed(1)) * 512 ** -0.5).to(dev, BF)
    W8 = G.rows_weight(W)
    _, _, q, s = G.layer_norm_rows(x, w, b, EPS, a)
    y = G.fp8_gemm_rows(q, s, W8.q, W8.s)
    ref = deq(q.cpu(), s.cpu()) @ deq(W8.q.cpu(), W8.s.cpu()).t()
    size = deq(q.cpu(), s.cpu()).abs() @ deq(W8.q.cpu(), W8.s.cpu()).abs().t()
    assert ((y.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -12 * size).all()


def test_refusals(dev):
    x, a, w, b, dh, _ = make((4, 64), BF, 11)
    bad = [lambda: G.layer_norm(x[:, :60], w[:60]), lambda: G.layer_norm(x.to(F64)), lambda: G.layer_norm(x, w[:32]),
           lambda: G.layer_norm(x, w, b[None]), lambda: G.layer_norm(x, w, b, EPS, a[:2]),
           lambda: G.layer_norm(torch.zeros(1, 16392, dtype=BF, device=dev)), lambda: G.layer_norm_rows(x.half()),
           lambda: G.layer_norm(x, w.cpu().to(dev), b.cpu().to(dev), EPS, a.view(2, 2, 64)),
           lambda: G.layer_norm_bwd(dh[:2], None, x, w, torch.zeros(4, device=dev), torch.zeros(4, device=dev)),
           lambda: G.layer_norm_bwd(dh, None, x, w, torch.zeros(3, device=dev), torch.zeros(4, device=dev))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="GPU only"):
        G.layer_norm(x, w.cpu())
    x.requires_grad_()
    h = G.layer_norm(x, w, b)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(h, x, dh, create_graph=True)
    with pytest.raises(Exception):
        h = G.layer_norm_rows(x, w, b)
        h[2].float().sum().backward()
    x = x.detach()
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(x, a)
        for call in (lambda: G.layer_norm(d, w, b), lambda: G.layer_norm_rows(d, w, b)):
            with pytest.raises((NotImplementedError, RuntimeError)):
                call()


def test_other_stream_and_threads_of_work(dev):
    x, a, w, b, dh, dxn = make((513, 1024), BF, 12)
    ref = G.layer_norm(x, w, b, EPS, a)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = G.layer_norm(x, w, b, EPS, a)
        rows = G.layer_norm_rows(x, w, b, EPS, a)
    torch.cuda.current_stream().wait_stream(st)
    assert all(torch.equal(p, q) for p, q in zip(got, ref)) and torch.equal(rows[0], ref[0])


def test_captured_and_replayed(dev):
    """Forward and backward in a graph, replayed with other inputs and eager work between, against the eager calls. (The leaves are
    made inside the capture: torch's engine waits for the stream of a leaf's older graph.)"""
    x, a, w, b, dh, dxn = make((300, 520), BF, 13)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, a, w, b)]
        xn, h = G.layer_norm(leaves[0], leaves[2], leaves[3], EPS, leaves[1])
        return [xn.detach(), h.detach(), *torch.autograd.grad((xn, h), leaves, (dxn, dh))]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        for t, n in zip((x, a, w, b, dh, dxn), make((300, 520), BF, 20 + i)):
            t.copy_(n)
        ref = [t.clone() for t in step()]
        torch.cuda.synchronize()
        g.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, ref)), i


def test_compiled(dev):
    x, a, w, b, dh, dxn = make((64, 256), BF, 14)
    for t in (x, w, b):
        t.requires_grad_()
    f = lambda x, w, b: G.layer_norm(x, w, b, EPS)  # noqa: E731
    h = torch.compile(f, backend="aot_eager")(x, w, b)
    ref = f(x, w, b)
    assert torch.equal(h, ref)
    for p, q in zip(torch.autograd.grad(h, (x, w, b), dh), torch.autograd.grad(ref, (x, w, b), dh)):
        assert torch.equal(p, q)


def test_saved_tensor_hooks_and_versions(dev):
    x, a, w, b, dh, dxn = make((40, 256), BF, 15)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    ref = torch.autograd.grad(G.layer_norm(*leaves), leaves, dh)
    with torch.autograd.graph.save_on_cpu():
        h = G.layer_norm(*leaves)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(h, leaves, dh), ref))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu()):
        h = G.layer_norm(*leaves)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(h, leaves, dh)
    h = G.layer_norm(*leaves)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, leaves, dh)


@pytest.mark.parametrize("native", [True, False])
def test_every_set_of_leaves(dev, native):
    """The node of the usual form and the general form (a weight whose elements are not beside each other) give the same bits,
    whichever leaves take a gradient, with either output's gradient missing."""
    x, a, w, b, dh, dxn = make((33, 264), BF, 16)
    if not native:
        w = torch.stack([w, w], 1)[:, 0]
    full = [t.detach().requires_grad_() for t in (x, a, w, b)]
    xn, h = G.layer_norm(full[0], full[2], full[3], EPS, full[1])
    ref = dict(zip("xawb", torch.autograd.grad((xn, h), full, (dxn, dh))))
    only_h = dict(zip("xawb", torch.autograd.grad(G.layer_norm(full[0], full[2], full[3], EPS, full[1])[1], full, dh)))
    for i in range(1, 16):
        on = [n for j, n in enumerate("xawb") if i >> j & 1]
        t = {n: v.detach().requires_grad_(n in on) for n, v in zip("xawb", (x, a, w, b))}
        xn, h = G.layer_norm(t["x"], t["w"], t["b"], EPS, t["a"])
        outs = [o for o in (xn, h) if o.requires_grad]
        assert len(outs) == 2
        got = torch.autograd.grad(outs, [t[n] for n in on], (dxn, dh), retain_graph=True)
        assert all(torch.equal(g, ref[n]) for n, g in zip(on, got)), on
        got = torch.autograd.grad(h, [t[n] for n in on], dh)
        assert all(torch.equal(g, only_h[n]) for n, g in zip(on, got)), on


def test_gradients_of_other_layouts_and_types(dev):
    x, a, w, b, dh, dxn = make((30, 64), BF, 17)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    run = lambda d: torch.autograd.grad(G.layer_norm(*leaves), leaves, d)  # noqa: E731
    ref = run(dh)
    for d in (dh.t().contiguous().t(), torch.empty(dh.numel() + 1, dtype=BF, device=dev)[1:].view(dh.shape).copy_(dh)):
        assert all(torch.equal(p, q) for p, q in zip(run(d), ref))
    total = torch.autograd.grad(G.layer_norm(*leaves).sum(), leaves)
    assert all(torch.equal(p, q) for p, q in zip(total, run(torch.ones_like(x))))

"""Per-request adapters on the GPU against 64 bits: ranks, sizes, orders of ids, rows without an adapter, strides, what other
adapters hold, graphs and streams; and the operators of a text-conditioned block together, served and trained."""
import math

import pytest
import torch

import gpic_fp8 as G

pytestmark = pytest.mark.gpu
BF, FP, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
U32 = 2.0 ** -24
HALF = {BF: 2.0 ** -8, FP: 2.0 ** -11}


def make(M, K, N, n, R, dt=BF, seed=0, dev="cuda", wide=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, y = r(M, K), r(M, N)
    A, B = r(n, R, K) * K ** -0.5, r(n, N, R) * R ** -0.5
    ids = torch.randint(-1, n, (M,), generator=g, dtype=torch.int64 if wide else torch.int32)
    s = torch.rand(n, generator=g) + 0.5
    return [*(t.to(dev, dt) for t in (y, x, A, B)), ids.to(dev), s.to(dev)]


def check(out, y, x, A, B, ids, s):
    """t's sums of K terms (K 2^-23 of their magnitudes), t as two 16-bit numbers (2^-16 of it, and in fp16 2^-22 of the row's
    largest), the sums of 2 R terms, a few fp32 steps, and one rounding."""
    K, R, N = x.shape[-1], A.shape[1], y.shape[-1]
    y6, x6, A6, B6 = (t.to(F64) for t in (y.reshape(-1, N), x.reshape(-1, K), A, B))
    ref, bound = y6.clone(), torch.zeros_like(y6)
    ids = ids.reshape(-1).long()
    for i in range(A.shape[0]):
        m = (ids == i).nonzero().squeeze(-1)
        if not m.numel():
            continue
        t, ta = x6[m] @ A6[i].t(), x6[m].abs() @ A6[i].abs().t()
        k = 1.0 if s is None else float(s[i])
        d = k * (t @ B6[i].t())
        ref[m] += d
        et = 2 * K * U32 * ta + 2.0 ** -16 * t.abs() + 2.0 ** -22 * t.abs().amax(1, keepdim=True)
        bound[m] = abs(k) * ((et + 4 * R * U32 * t.abs()) @ B6[i].abs().t()) + 4 * U32 * (y6[m].abs() + d.abs())
    bound = bound + HALF[y.dtype] * (ref.abs() + bound) + (2.0 ** -25 if y.dtype == FP else 0)
    err = (out.reshape(-1, N).to(F64) - ref).abs()
    assert (err <= bound).all(), (float(err.max()), float((err / bound.clamp_min(1e-300)).max()))
    none = (ids < 0) | (ids >= A.shape[0])
    assert torch.equal(out.reshape(-1, N)[none], y.reshape(-1, N)[none])


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("R", [8, 16, 24, 32, 64, 72, 128])
@pytest.mark.parametrize("M,K,N,n", [(1, 8, 8, 1), (1, 1024, 1024, 4), (5, 72, 200, 3), (16, 512, 136, 20), (64, 2048, 264, 32),
                                     (77, 1000, 1032, 2), (300, 264, 520, 5), (2051, 136, 1160, 7)])
def test_against_64_bits(dev, dt, R, M, K, N, n):
    y, x, A, B, ids, s = make(M, K, N, n, R, dt, wide=R == 16)
    check(G.lora_rows(y, x, A, B, ids, s), y, x, A, B, ids, s)
    if R == 8:
        check(G.lora_rows(y, x, A, B, ids), y, x, A, B, ids, None)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("M,K,N,n,R", [(300, 4104, 264, 3, 24), (700, 8192, 136, 40, 64), (1500, 4160, 72, 2, 128), (260, 20000, 8, 1, 8),
                                         (8200, 4104, 72, 3, 40), (5000, 2056, 40, 5, 72), (16390, 520, 24, 2, 16)])
def test_long_reductions_in_parts(dev, dt, M, K, N, n, R):
    y, x, A, B, ids, s = make(M, K, N, n, R, dt, 9)
    check(G.lora_rows(y, x, A, B, ids, s), y, x, A, B, ids, s)
    out = G.lora_rows(y, x, A, B, ids, s)
    assert torch.equal(G.lora_rows(y, x, A, B, ids, s), out)


@pytest.mark.parametrize("order", ["runs", "same", "none", "mixed", "outside"])
@pytest.mark.parametrize("M", [40, 2500])
def test_orders_of_ids(dev, order, M):
    y, x, A, B, ids, s = make(M, 256, 384, 6, 16, BF, 1)
    if order == "runs":
        ids = ids.sort()[0]
    elif order == "same":
        ids.fill_(3)
    elif order == "none":
        ids.fill_(-1)
    elif order == "outside":   # indices that no adapter has keep y
        ids[::3], ids[1::3] = 6, -(1 << 31)
    out = G.lora_rows(y, x, A, B, ids, s)
    check(out, y, x, A, B, ids, s)
    # a row's bits do not depend on the order of the rows, nor on the others'
    perm = torch.randperm(M, generator=torch.Generator().manual_seed(2)).to(dev)
    assert torch.equal(G.lora_rows(y[perm], x[perm], A, B, ids[perm], s), out[perm])
    if order == "outside":
        assert torch.equal(G.lora_rows(y, x, A, B, ids.long() + (1 << 40), s), y)


def test_ids_of_the_batch(dev):
    y, x, A, B, ids, s = make(6 * 35, 128, 256, 4, 16, BF, 3)
    y, x, b = y.view(6, 35, 256), x.view(6, 35, 128), ids[:6].contiguous()
    out = G.lora_rows(y, x, A, B, b, s)
    assert torch.equal(out, G.lora_rows(y, x, A, B, b[:, None].expand(6, 35), s)) and out.shape == y.shape
    check(out, y, x, A, B, b.repeat_interleave(35), s)


def test_other_adapters_may_hold_anything(dev):
    for M in (48, 2100):
        y, x, A, B, ids, s = make(M, 256, 264, 5, 24, BF, 4)
        out = G.lora_rows(y, x, A, B, ids, s)
        A2, B2 = A.clone(), B.clone()
        A2[2], B2[2] = math.nan, math.inf
        got, row = G.lora_rows(y, x, A2, B2, ids, s), ids == 2
        assert torch.equal(got[~row], out[~row]) and got[row].isnan().all()
        x2 = x.clone()
        x2[7, 3] = math.inf
        keep = torch.arange(M, device=dev) != 7
        assert torch.equal(G.lora_rows(y, x2, A, B, ids, s)[keep], out[keep])


@pytest.mark.parametrize("scale", [1e-6, 3e4])
def test_small_and_large_intermediates_in_fp16(dev, scale):
    """x A^T far below fp16's normal numbers, or above its largest, where the product with B is neither."""
    y, x, A, B, ids, s = make(33, 512, 136, 3, 32, FP, 5)
    A = (A.float() * scale).to(FP)
    s = s / scale
    x = (x.float() * 4).to(FP)
    check(G.lora_rows(y, x, A, B, ids, s), y, x, A, B, ids, s)


def test_strides(dev):
    y, x, A, B, ids, s = make(50, 128, 256, 4, 16, BF, 6)
    ref = G.lora_rows(y, x, A, B, ids, s)
    wide = torch.zeros(50, 400, dtype=BF, device=dev)
    wide[:, 8:136] = x
    yw = torch.zeros(50, 264, dtype=BF, device=dev)
    yw[:, 8:] = y
    odd = torch.zeros(50 * 128 + 1, dtype=BF, device=dev)
    odd[1:] = x.view(-1)
    AB = torch.zeros(4, 16, 200, dtype=BF, device=dev)
    AB[:, :, 4:132] = A
    Bt = B.transpose(1, 2).contiguous().transpose(1, 2)
    for yy, xx, aa, bb in ((yw[:, 8:], wide[:, 8:136], A, B), (y, odd[1:].view(50, 128), AB[:, :, 4:132], Bt),
                           (y.t().contiguous().t(), x, A, B)):
        assert torch.equal(G.lora_rows(yy, xx, aa, bb, ids, s), ref)
    two = torch.stack([ids, ids], 1)[:, 0]
    assert torch.equal(G.lora_rows(y, x, A, B, two, torch.stack([s, s], 1)[:, 0]), ref)
    one = x[:1].expand(50, 128)
    check(G.lora_rows(y, one, A, B, ids, s), y, one.contiguous(), A, B, ids, s)


def test_no_rows(dev):
    y, x, A, B, ids, s = make(4, 64, 64, 2, 8)
    assert G.lora_rows(y[:0], x[:0], A, B, ids[:0], s).shape == (0, 64)
    assert G.lora_rows(y[:0].view(0, 3, 64), x[:0].view(0, 3, 64), A, B, ids[:0], s).shape == (0, 3, 64)


def test_far_offsets(dev):
    """An adapter and rows beyond 2^31 elements of their tensors' starts."""
    K, R = 8192, 128
    n = (1 << 31) // (K * R) + 2
    A = torch.empty(n, R, K, dtype=BF, device=dev)
    y, x, A1, B1, _, s1 = make(40, K, 64, 1, R, BF, 7)
    A[n - 1] = A1[0]
    B = torch.zeros(n, 64, R, dtype=BF, device=dev)
    B[n - 1] = B1[0]
    ids = torch.full((40,), n - 1, dtype=torch.int32, device=dev)
    got = G.lora_rows(y, x, A, B, ids)
    check(got, y, x, A1, B1, torch.zeros_like(ids), None)


def test_refusals(dev):
    y, x, A, B, ids, s = make(6, 64, 128, 2, 16)
    bad = [lambda: G.lora_rows(y[:5], x, A, B, ids, s), lambda: G.lora_rows(y, x, A, B[:1], ids, s),
           lambda: G.lora_rows(y, x[:, :32], A, B, ids, s), lambda: G.lora_rows(y, x, A[:, :8], B, ids, s),
           lambda: G.lora_rows(y, x.half(), A, B, ids, s), lambda: G.lora_rows(*(t.float() for t in (y, x, A, B)), ids, s),
           lambda: G.lora_rows(y[:, :124], x, A, B[:, :124], ids, s), lambda: G.lora_rows(y, x, A[:, :12], B[:, :, :12], ids, s),
           lambda: G.lora_rows(y, x, A, B, ids[:5], s), lambda: G.lora_rows(y, x, A, B, ids.short(), s),
           lambda: G.lora_rows(y, x, A, B, ids, s.double()), lambda: G.lora_rows(y, x, A, B, ids, s[:1]),
           lambda: G.lora_rows(y, x, A[:0], B[:0], ids, s[:0]),
           lambda: G.lora_rows(y, x, torch.zeros(2, 136, 64, dtype=BF, device=dev), torch.zeros(2, 128, 136, dtype=BF, device=dev), ids)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="GPU only"):
        G.lora_rows(y, x, A, B, ids.cpu(), s)
    with pytest.raises(Exception):
        G.lora_rows(y, x.requires_grad_(), A, B, ids, s).sum().backward()


def test_captured_replayed_and_on_another_stream(dev):
    for M in (3, 40, 2200):
        y, x, A, B, ids, s = make(M, 520, 264, 6, 16, BF, 8)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            side = G.lora_rows(y, x, A, B, ids, s)
        torch.cuda.current_stream().wait_stream(st)
        assert torch.equal(side, G.lora_rows(y, x, A, B, ids, s))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = G.lora_rows(y, x, A, B, ids, s)
        for i in range(4):
            for t, n in zip((y, x, A, B, ids, s), make(M, 520, 264, 6, 16, BF, 20 + i)):
                t.copy_(n)
            ref = G.lora_rows(y, x, A, B, ids, s)
            torch.cuda.synchronize()
            g.replay()
            assert torch.equal(out, ref)


# ------------------------------------------------------------------------------------------------ the operators together

class Block:
    """A text-conditioned block's cross-attention sublayer: norm, query projection, attention to a caption's states, output
    projection with the residual."""

    def __init__(self, dev, C=256, H=4, T=320, n=3, R=16):
        g = torch.Generator().manual_seed(9)
        r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dev, BF)  # noqa: E731
        self.C, self.H = C, H
        self.wn, self.bn = 1 + r(C, std=0.1), r(C, std=0.1)
        self.wq, self.wkv, self.wo = r(C, C, std=C ** -0.5), r(2 * C, T, std=T ** -0.5), r(C, C, std=C ** -0.5)
        self.bo = r(C, std=0.1)
        self.qa, self.qb, self.oa, self.ob = r(n, R, C, std=C ** -0.5), r(n, C, R, std=0.25), r(n, R, C, std=C ** -0.5), r(n, C, R, std=0.25)
        self.x, self.a, self.text = r(4, 60, C), r(4, 60, C), r(4, 77, T)
        self.lens = torch.tensor([77, 20, 0, 1], dtype=torch.int32, device=dev)
        self.ids = torch.tensor([2, -1, 0, 2], dtype=torch.int32, device=dev)

    def heads(self, t):
        return t.view(*t.shape[:2], self.H, -1).transpose(1, 2)

    def serve(self, W, x, a, text, lens, ids, lora=True):
        xn, h, q8, s8 = G.layer_norm_rows(x, self.wn, self.bn, 1e-5, a, True)
        q = G.fp8_gemm_rows(q8.view(-1, self.C), s8, W[0].q, W[0].s).view(x.shape)
        if lora:
            q = G.lora_rows(q, h, self.qa, self.qb, ids)
        k, v = G.fp8_linear_rows(text, W[1]).chunk(2, -1)
        o = G.cross_attention(self.heads(q), self.heads(k), self.heads(v), lens).transpose(1, 2).reshape(x.shape)
        y = G.fp8_linear_rows(o, W[2], self.bo, residual=xn)
        return G.lora_rows(y, o, self.oa, self.ob, ids) if lora else y

    def train(self, x, a, text, lens):
        xn, h = G.layer_norm(x, self.wn, self.bn, 1e-5, a)
        q = G.fp8_linear_rows(h, self.wq)
        k, v = G.fp8_linear_rows(text, self.wkv).chunk(2, -1)
        o = G.cross_attention(self.heads(q), self.heads(k), self.heads(v), lens).transpose(1, 2).reshape(x.shape)
        return G.fp8_linear_rows(o, self.wo, self.bo, residual=xn)


def test_block_served(dev):
    b = Block(dev)
    W = [G.rows_weight(w) for w in (b.wq, b.wkv, b.wo)]
    with torch.no_grad():
        plain = b.serve(W, b.x, b.a, b.text, b.lens, b.ids, lora=False)
        y = b.serve(W, b.x, b.a, b.text, b.lens, b.ids)
        assert torch.equal(y[1], plain[1]) and not torch.equal(y[0], plain[0])   # (the request without adapters)
        # an empty caption: the attention gives zeros, and y is the residual, the bias and the output adapter of zeros
        xn = (b.x.float() + b.a.float()).to(BF)
        assert torch.equal(y[2], (xn[2].float() + b.bo.float()).to(BF))
        # the training form without gradients is the same block, its e4m3 operand cast from the norm's bf16 output
        t = b.train(b.x, b.a, b.text, b.lens)
        assert ((t - plain).float().norm() / plain.float().norm()) < 2.0 ** -4
        g = torch.cuda.CUDAGraph()
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            b.serve(W, b.x, b.a, b.text, b.lens, b.ids)
        torch.cuda.current_stream().wait_stream(st)
        with torch.cuda.graph(g):
            out = b.serve(W, b.x, b.a, b.text, b.lens, b.ids)
        for i in range(3):
            gen = torch.Generator().manual_seed(30 + i)
            for t in (b.x, b.a, b.text):
                t.copy_(torch.randn(t.shape, generator=gen))
            b.lens.copy_(torch.randint(0, 78, (4,), generator=gen))
            b.ids.copy_(torch.randint(-1, 3, (4,), generator=gen))
            ref = b.serve(W, b.x, b.a, b.text, b.lens, b.ids)
            torch.cuda.synchronize()
            g.replay()
            assert torch.equal(out, ref)


def test_block_trained(dev):
    """The block's gradients are those of its operators one after another, and those of an fp32 block to what e4m3 leaves."""
    b = Block(dev)
    leaves = [t.requires_grad_() for t in (b.x, b.a, b.text, b.wn, b.bn, b.wq, b.wkv, b.wo, b.bo)]
    y = b.train(b.x, b.a, b.text, b.lens)
    dy = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(dev, BF)
    got = torch.autograd.grad(y, leaves, dy)
    again = torch.autograd.grad(b.train(b.x, b.a, b.text, b.lens), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(got, again))

    f = [t.detach().to(F32).requires_grad_() for t in leaves]
    x, a, text, wn, bn, wq, wkv, wo, bo = f
    xn = x + a
    h = torch.nn.functional.layer_norm(xn, (b.C,), wn, bn, 1e-5)
    q, (k, v) = h @ wq.t(), (text @ wkv.t()).chunk(2, -1)
    s = b.heads(q) @ b.heads(k).transpose(2, 3) * (b.C // b.H) ** -0.5
    ok = (torch.arange(77, device=dev) < b.lens[:, None])[:, None, None]
    p = torch.where(ok, torch.softmax(s.masked_fill(~ok, -1e30), -1), torch.zeros_like(s))
    o = (p @ b.heads(v)).transpose(1, 2).reshape(x.shape)
    ref = torch.autograd.grad(xn + o @ wo.t() + bo, f, dy.to(F32))
    for name, p, r in zip(("x", "a", "text", "wn", "bn", "wq", "wkv", "wo", "bo"), got, ref):
        # a product of e4m3 operands is off by up to 2^-4 of each; a gradient here passes at most four of them: eight operands
        assert (p.float() - r).norm() <= 8 * 2.0 ** -4 * r.norm(), name
        assert not p[2].any() if name == "text" else p.isfinite().all()

"""Cross attention on the GPU against 64 bits: types, shared heads, lengths from none, masks with holes, head dimensions, strides,
what padding holds, gradients, graphs, streams, far offsets, and the operators of a block together."""
import math

import pytest
import torch

import gpic_fp8 as G
from attn_ref import check, valid_keys

pytestmark = pytest.mark.gpu
BF, FP, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def make(B, H, Hk, N, L, D, dt=BF, seed=0, dev="cuda", do_std=0.1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, do = r(B, N, H, D), do_std * r(B, N, H, D)
    k, v = r(B, L, Hk, D), r(B, L, Hk, D)
    return [t.to(dev, dt).transpose(1, 2) for t in (q, k, v, do)]


def keys(B, L, kind, seed=0, dev="cuda"):
    g = torch.Generator().manual_seed(seed + 100)
    lens = mask = None
    if "lens" in kind:
        lens = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        lens[0] = L
        if B > 1:
            lens[1] = 0
        lens = lens.to(dev)
    if "mask" in kind:
        mask = torch.rand(B, L, generator=g) < 0.7
        if B > 2:
            mask[2] = False
        mask = mask.to(dev)
    return lens, mask


def both(q, k, v, do, lens, mask, scale=None):
    """Forward and backward through autograd, and the check."""
    s = scale or q.shape[-1] ** -0.5
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = G.cross_attention(q, k, v, lens, mask, scale)
    assert o.shape == q.shape and o.dtype == q.dtype
    grads = torch.autograd.grad(o, (q, k, v), do)
    ok = valid_keys(k.shape[0], k.shape[2], lens, mask, k.device)
    check(q.detach(), k.detach(), v.detach(), ok, s, o.detach(), do, grads)
    served = G.cross_attention(q.detach(), k.detach(), v.detach(), lens, mask, scale)
    assert torch.equal(served, o)
    return o.detach(), grads


SHAPES = [  # B, H, Hk, N, L, D
    (1, 1, 1, 1, 1, 8), (2, 3, 3, 5, 7, 16), (1, 2, 2, 16, 32, 64), (3, 4, 2, 17, 33, 64), (2, 2, 2, 64, 64, 64),
    (3, 2, 1, 65, 129, 72), (2, 2, 2, 200, 77, 64), (4, 8, 2, 1, 300, 128), (3, 16, 1, 1, 1000, 64), (2, 2, 1, 333, 511, 128),
    (3, 1, 1, 40, 64, 80), (4, 16, 16, 1, 65, 32), (2, 5, 5, 3, 2049, 96), (1, 1, 1, 1000, 3, 64), (33, 16, 16, 256, 77, 64)]


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["all", "lens", "mask", "lens+mask"])
def test_forward_and_backward(dev, dt, shape, kind):
    B, H, Hk, N, L, D = shape
    q, k, v, do = make(*shape, dt)
    both(q, k, v, do, *keys(B, L, kind))


@pytest.mark.parametrize("shape", [(8, 32, 8, 1, 8191, 128), (1, 4, 4, 2, 5000, 64), (2, 2, 2, 100, 4000, 64), (64, 16, 16, 256, 320, 64),
                                   (1, 4, 1, 1024, 2111, 128), (40, 16, 16, 129, 257, 128)])
@pytest.mark.parametrize("kind", ["lens", "mask"])
def test_larger_and_split(dev, shape, kind):
    B, H, Hk, N, L, D = shape
    q, k, v, do = make(*shape, BF, 1)
    both(q, k, v, do, *keys(B, L, kind, 1))


@pytest.mark.parametrize("B,H,Hk,N,L,D", [(9, 16, 8, 1, 6200, 128), (64, 16, 4, 4, 3100, 64), (2, 8, 1, 2, 262144, 96), (3, 64, 64, 1, 4100, 72)])
@pytest.mark.parametrize("kind", ["none", "ones", "one long", "tiles", "full", "drawn", "mask"])
def test_one_token_of_unlike_lengths(dev, B, H, Hk, N, L, D, kind):
    """Lengths that put an entry's ends inside, at and outside the runs that workgroups take; o and lse, with 64-bit lengths too."""
    g = torch.Generator(device="cuda").manual_seed(B)
    r = lambda h, n: torch.randn(B, n, h, D, generator=g, device="cuda").to(BF).transpose(1, 2)  # noqa: E731
    q, k, v = r(H, N), r(Hk, L), r(Hk, L)
    few = torch.arange(B, dtype=torch.int32, device="cuda")
    drawn = torch.randint(0, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens = {"none": 0 * few, "ones": 0 * few + 1, "one long": torch.where(few == B // 2, L, few % 3), "tiles": 32 * (few % 5) + 256,
            "full": 0 * few + L, "drawn": drawn, "mask": drawn}[kind].to(torch.int32)
    mask = torch.rand(B, L, generator=g, device="cuda") < 0.02 if kind == "mask" else None
    o, lse = G.cross_attention_fwd(q, k, v, lens, mask)
    assert torch.equal(G.cross_attention(q, k, v, lens.long(), mask), o)
    ok = valid_keys(B, L, lens, mask, "cuda")
    for b in range(B):   # (an entry at a time: 64 bits of all would not fit beside each other)
        check(q[b:b + 1], k[b:b + 1], v[b:b + 1], ok[b:b + 1], D ** -0.5, o[b:b + 1])
        _, alone = G.cross_attention_fwd(q[b:b + 1], k[b:b + 1], v[b:b + 1], lens[b:b + 1], None if mask is None else mask[b:b + 1])
        assert torch.equal(torch.isinf(alone), torch.isinf(lse[b:b + 1]))
        # (p's sums in another order: fp32 steps of the sum, as many as its longest chain of additions, and of the maximum's exponent)
        assert ((alone - lse[b:b + 1]).nan_to_num(0).abs() <= 2.0 ** -24 * (L / 8 + 64)).all()


def test_captured_lengths_change(dev):
    B, H, Hk, L, D = 9, 16, 8, 6200, 128
    g = torch.Generator(device="cuda").manual_seed(4)
    r = lambda h, n: torch.randn(B, n, h, D, generator=g, device="cuda").to(FP).transpose(1, 2)  # noqa: E731
    q, k, v = r(H, 1), r(Hk, L), r(Hk, L)
    lens = torch.full((B,), L, dtype=torch.int32, device="cuda")
    G.cross_attention(q, k, v, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = G.cross_attention(q, k, v, lens)
    for i in range(5):
        lens.copy_(torch.randint(0, L + 1, (B,), generator=g, device="cuda") * (i != 2))
        ref = G.cross_attention(q, k, v, lens)
        graph.replay()
        assert torch.equal(o, ref), i
    assert not torch.equal(o, torch.zeros_like(o))


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("N", [1, 100])
def test_padding_may_hold_anything(dev, dt, N):
    q, k, v, do = make(3, 4, 2, N, 150, 64, dt, 2)
    lens = torch.tensor([150, 70, 0], dtype=torch.int32, device=dev)
    mask = torch.ones(3, 150, dtype=torch.bool, device=dev)
    mask[0, 10:90] = False
    ok = valid_keys(3, 150, lens, mask, dev)
    o, grads = both(q, k, v, do, lens, mask)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dt).max):
        kb, vb = (torch.where(ok[:, None, :, None], t, torch.full_like(t, bad)) for t in (k, v))
        o2, grads2 = both(q, kb, vb, do, lens, mask)
        assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_infinities_and_nan_where_keys_are_valid(dev):
    """A row's own business: NaN in one query's row, an infinite value of one key."""
    for N in (1, 40):
        q, k, v, do = make(2, 2, 2, N, 70, 64, BF, 3)
        q[0, 0, 0, 3] = math.nan
        v[1, 1, 5, 7] = math.inf
        o = G.cross_attention(q, k, v)
        assert o[0, 0, 0].isnan().all() and o[0, 1].isfinite().all() and o[1, 0].isfinite().all()
        assert (o[1, 1, :, 7] == math.inf).all() and o[1, 1, :, 8].isfinite().all()
        if N > 1:
            assert o[0, 0, 1:].isfinite().all()


@pytest.mark.parametrize("dt,std", [(BF, 1e-6), (FP, 1e-6), (FP, 300.0), (BF, 1e4)])
def test_small_and_large_gradients(dev, dt, std):
    q, k, v, do = make(2, 2, 2, 130, 900, 64, dt, 4, do_std=std)
    both(q, k, v, do, None, None)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 7.5])
def test_scales_and_sharp_rows(dev, scale):
    q, k, v, do = make(2, 2, 1, 70, 200, 64, BF, 5)
    both(q, k, v, do, None, None, scale)


def test_rising_scores(dev):
    """Keys in rising order of their scores: the running maximum moves in every tile."""
    q, k, v, do = make(1, 2, 2, 80, 700, 64, BF, 6)
    q = q.abs()
    k = (k.abs() * torch.linspace(0.01, 4, 700, device=dev).view(1, 1, -1, 1)).to(BF)
    both(q, k, v, do, None, None)
    both(q[:, :, :1], k, v, do[:, :, :1], None, None)


def test_strides_and_layouts(dev):
    q, k, v, do = make(2, 4, 2, 50, 90, 64, BF, 7)
    ref = G.cross_attention(q, k, v)
    cont = lambda t: t.contiguous()  # noqa: E731
    pad = torch.zeros(2, 2, 90, 136, dtype=BF, device=dev)
    pad[..., 8:72], odd = k, torch.zeros(k.numel() + 1, dtype=BF, device=dev)
    odd[1:] = k.contiguous().view(-1)
    last = k.transpose(2, 3).contiguous().transpose(2, 3)
    for kk in (cont(k), pad[..., 8:72], odd[1:].view(k.shape), last, pad[..., 8:72].transpose(0, 1).contiguous().transpose(0, 1)):
        assert torch.equal(G.cross_attention(cont(q), kk, cont(v)), ref)
        o, lse = G.cross_attention_fwd(q, kk, v)
        g1, g2 = G.cross_attention_bwd(do, q, kk, v, o, lse), G.cross_attention_bwd(cont(do), q, k, v, cont(o), lse)
        assert all(torch.equal(a, b) for a, b in zip(g1, g2))
    one = G.cross_attention(q, k[:1].expand(2, 2, 90, 64), v[:1].expand(2, 2, 90, 64))
    assert torch.equal(one[0], ref[0])
    lens, mask = keys(2, 90, "lens+mask")
    wide = torch.zeros(2, 200, dtype=torch.bool, device=dev)
    wide[:, 5:95] = mask
    a = G.cross_attention(q, k, v, lens, mask)
    for l2, m2 in ((lens.long(), wide[:, 5:95]), (lens, mask.view(2, 1, 1, 90)), (lens, mask.t().contiguous().t())):
        assert torch.equal(G.cross_attention(q, k, v, l2, m2), a)
    assert torch.equal(G.cross_attention(q, k, v, torch.tensor([1 << 40, 95], device=dev)), ref)
    assert not G.cross_attention(q, k, v, torch.tensor([-5, -(1 << 40)], device=dev)).any()
    assert not G.cross_attention(q, k, v, torch.tensor([-5, -9], dtype=torch.int32, device=dev)).any()


def test_broadcast_inputs_sum_their_gradients(dev):
    q, k, v, do = make(3, 2, 2, 20, 40, 64, BF, 8)
    k1, v1 = k[:1].detach().requires_grad_(), v[:1].detach().requires_grad_()
    o = G.cross_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1))
    gk, gv = torch.autograd.grad(o, (k1, v1), do)
    o, lse = G.cross_attention_fwd(q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1))
    _, dk, dv = G.cross_attention_bwd(do, q, k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), o, lse)
    assert torch.equal(gk, dk.sum(0, keepdim=True)) and torch.equal(gv, dv.sum(0, keepdim=True))


def test_which_gradients(dev):
    q, k, v, do = make(2, 4, 2, 30, 50, 64, BF, 9)
    o, lse = G.cross_attention_fwd(q, k, v)
    ref = dict(zip("qkv", G.cross_attention_bwd(do, q, k, v, o, lse)))
    for on in ("q", "k", "v", "qk", "kv", "qv"):
        t = {n: x.detach().requires_grad_(n in on) for n, x in zip("qkv", (q, k, v))}
        got = torch.autograd.grad(G.cross_attention(t["q"], t["k"], t["v"]), [t[n] for n in on], do)
        assert all(torch.equal(g, ref[n]) for n, g in zip(on, got)), on


@pytest.mark.parametrize("B,N,L", [(0, 4, 5), (2, 0, 5), (2, 4, 0), (0, 0, 0)])
def test_nothing(dev, B, N, L):
    q, k, v, do = (torch.zeros(B, n, 4, 64, dtype=BF, device=dev).transpose(1, 2) for n in (N, L, L, N))
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = G.cross_attention(q, k, v, torch.full((B,), 3, dtype=torch.int32, device=dev), torch.ones(B, L, dtype=torch.bool, device=dev))
    grads = torch.autograd.grad(o, (q, k, v), do)
    assert not o.any() and all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v)))


def test_lse(dev):
    q, k, v, _ = make(2, 4, 2, 9, 70, 64, BF, 10)
    lens = torch.tensor([70, 0], dtype=torch.int32, device=dev)
    for n in (9, 1):
        _, lse = G.cross_attention_fwd(q[:, :, :n], k, v, lens)
        ref = torch.logsumexp(q[0, :, :n].double() @ k[0].double().repeat_interleave(2, 0).transpose(1, 2) / 8, -1) / math.log(2)
        assert (lse[0] - ref).abs().max() < 64 * 2.0 ** -20 and (lse[1] == math.inf).all()


def test_same_bits_again(dev):
    for shape in ((2, 4, 4, 1, 3000, 64), (1, 2, 1, 300, 900, 128), (2, 1, 1, 40, 5000, 64)):
        q, k, v, do = make(*shape, BF, 11)
        first = G.cross_attention_fwd(q, k, v)
        g1 = G.cross_attention_bwd(do, q, k, v, *first)
        for _ in range(3):
            again = G.cross_attention_fwd(q, k, v)
            assert all(torch.equal(a, b) for a, b in zip(first, again))
            assert all(torch.equal(a, b) for a, b in zip(g1, G.cross_attention_bwd(do, q, k, v, *again)))


def test_far_offsets(dev):
    """Rows of k and v beyond 2^31 elements of their tensors' starts."""
    D, L, far = 64, 130, (1 << 31) + 64
    buf = torch.empty(far + L * D, dtype=BF, device=dev)
    q, k, v, do = make(2, 1, 1, 20, L, D, BF, 12)
    kk = torch.as_strided(buf, (2, 1, L, D), (far, D, D, 1))
    kk.copy_(k)
    o, lse = G.cross_attention_fwd(q, kk, kk)
    ref, lse2 = G.cross_attention_fwd(q, k, k)
    assert torch.equal(o, ref) and torch.equal(lse, lse2)
    assert torch.equal(G.cross_attention(q[:, :, :1], kk, kk), G.cross_attention(q[:, :, :1], k, k))
    for a, b in zip(G.cross_attention_bwd(do, q, kk, kk, o, lse), G.cross_attention_bwd(do, q, k, k, ref, lse2)):
        assert torch.equal(a, b)


def test_refusals(dev):
    q, k, v, do = make(2, 4, 2, 6, 9, 64, BF, 13)
    lens = torch.tensor([9, 9], dtype=torch.int32, device=dev)
    mask = torch.ones(2, 9, dtype=torch.bool, device=dev)
    bad = [lambda: G.cross_attention(q[0], k, v), lambda: G.cross_attention(q, k, v[:, :, :5]), lambda: G.cross_attention(q, k[:1], v[:1]),
           lambda: G.cross_attention(q, k[..., :32], v[..., :32]), lambda: G.cross_attention(q[:, :3], k, v),
           lambda: G.cross_attention(q.float(), k.float(), v.float()), lambda: G.cross_attention(q, k.half(), v.half()),
           lambda: G.cross_attention(q[..., :60], k[..., :60], v[..., :60]), lambda: G.cross_attention(q, k, v, scale=0.0),
           lambda: G.cross_attention(q, k, v, scale=-0.1), lambda: G.cross_attention(q, k, v, scale=math.nan),
           lambda: G.cross_attention(q, k, v, scale=math.inf), lambda: G.cross_attention(q, k, v, lens[:1]),
           lambda: G.cross_attention(q, k, v, lens.float()), lambda: G.cross_attention(q, k, v, None, mask[:, :8]),
           lambda: G.cross_attention(q, k, v, None, mask.float()), lambda: G.cross_attention(q, k, v, None, mask[:1]),
           lambda: G.cross_attention(*(torch.zeros(1, 1, 2, 136, dtype=BF, device=dev) for _ in range(3))),
           lambda: G.cross_attention_bwd(do[:, :, :5], q, k, v, q, torch.zeros(2, 4, 6, device=dev)),
           lambda: G.cross_attention_bwd(do, q, k, v, q, torch.zeros(2, 4, 5, device=dev))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(str(i))
    with pytest.raises(RuntimeError, match="GPU only"):
        G.cross_attention(q, k.cpu(), v.cpu())
    with pytest.raises(RuntimeError, match="GPU only"):
        G.cross_attention(q, k, v, lens.cpu())
    qg = q.detach().requires_grad_()
    o = G.cross_attention(qg, k, v)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(o, qg, do, create_graph=True)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(q, q)
        for call in (lambda: G.cross_attention(d, k, v), lambda: G.cross_attention_fwd(d, k, v)):
            with pytest.raises((NotImplementedError, RuntimeError)):
                call()


def test_other_stream(dev):
    q, k, v, do = make(4, 8, 8, 128, 300, 64, BF, 14)
    lens, mask = keys(4, 300, "lens+mask")
    ref, lse = G.cross_attention_fwd(q, k, v, lens, mask)
    refs = G.cross_attention_bwd(do, q, k, v, ref, lse, lens, mask)
    one = G.cross_attention(q[:, :, :1], k, v, lens, mask)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o, lse = G.cross_attention_fwd(q, k, v, lens, mask)
        got = G.cross_attention_bwd(do, q, k, v, o, lse, lens, mask)
        few = G.cross_attention(q[:, :, :1], k, v, lens, mask)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(o, ref) and torch.equal(few, one) and all(torch.equal(a, b) for a, b in zip(got, refs))


@pytest.mark.parametrize("shape", [(2, 4, 2, 1, 2000, 64), (2, 4, 2, 70, 2000, 64), (3, 4, 4, 128, 90, 128)])
def test_captured_and_replayed(dev, shape):
    """Forward and backward in a graph, replayed with other inputs, lengths and masks and eager work between. (The leaves are made
    inside the capture: torch's engine waits for the stream of a leaf's older graph.)"""
    B, H, Hk, N, L, D = shape
    q, k, v, do = make(*shape, BF, 15)
    lens, mask = keys(B, L, "lens+mask")

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = G.cross_attention(*leaves, lens, mask)
        return [o.detach(), *torch.autograd.grad(o, leaves, do), G.cross_attention(q, k, v, lens)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step()
    torch.cuda.current_stream().wait_stream(st)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        for t, n in zip((q, k, v, do), make(*shape, BF, 20 + i)):
            t.copy_(n)
        for t, n in zip((lens, mask), keys(B, L, "lens+mask", 20 + i)):
            t.copy_(n)
        ref = [t.clone() for t in step()]
        torch.cuda.synchronize()
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, ref)), i


def test_compiled(dev):
    q, k, v, do = make(2, 4, 2, 40, 60, 64, BF, 16)
    lens, mask = keys(2, 60, "lens+mask")
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    f = lambda q, k, v: G.cross_attention(q, k, v, lens, mask)  # noqa: E731
    o, ref = torch.compile(f, backend="aot_eager")(q, k, v), f(q, k, v)
    assert torch.equal(o, ref)
    for a, b in zip(torch.autograd.grad(o, (q, k, v), do), torch.autograd.grad(ref, (q, k, v), do)):
        assert torch.equal(a, b)


def test_output_feeds_the_heads_linear(dev):
    """o as the tensorwise heads linear and the row-scaled linear take it: no copy to merge its heads."""
    q, k, v, _ = make(2, 4, 4, 32, 50, 64, BF, 17)
    o = G.cross_attention(q, k, v)
    merged = o.transpose(1, 2).reshape(2, 32, 256)
    assert merged.data_ptr() == o.data_ptr()
    W = (torch.randn(256, 256, generator=torch.Generator().manual_seed(1)) / 16).to(dev, BF)
    assert torch.equal(G.fp8_heads_linear_f8(o, W, None), G.fp8_linear_f8(merged, W, None))
    y = G.fp8_linear_rows(merged, G.rows_weight(W))
    assert y.shape == (2, 32, 256) and y.isfinite().all()


def test_saved_tensor_hooks_and_versions(dev):
    """What the nodes owe autograd: hooks that bring the tensors back as they were change nothing, others raise; an input changed
    in place after the forward raises."""
    q, k, v, do = make(2, 4, 2, 30, 50, 64, BF, 18)
    lens = torch.tensor([50, 20], dtype=torch.int32, device=dev)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    ref = torch.autograd.grad(G.cross_attention(*leaves, lens), leaves, do)
    with torch.autograd.graph.save_on_cpu():
        o = G.cross_attention(*leaves, lens)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o, leaves, do), ref))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu()):
        o = G.cross_attention(*leaves, lens)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(o, leaves, do)
    o = G.cross_attention(*leaves, lens)
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, leaves, do)


def test_gradients_of_other_layouts(dev):
    """o's gradient as autograd makes it: expanded (a sum's), transposed, fp32."""
    q, k, v, do = make(2, 4, 2, 30, 50, 64, BF, 19)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    run = lambda d: torch.autograd.grad(G.cross_attention(*leaves), leaves, d)  # noqa: E731
    ref = run(do)
    last = do.transpose(2, 3).contiguous().transpose(2, 3)
    odd = torch.empty(do.numel() + 1, dtype=BF, device=dev)[1:].view(do.shape).copy_(do)
    for d in (do.contiguous(), last, odd):
        assert all(torch.equal(a, b) for a, b in zip(run(d), ref))
    one = torch.ones(2, 4, 30, 64, dtype=BF, device=dev)
    total = torch.autograd.grad(G.cross_attention(*leaves).sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(total, run(one)))


def test_retained_and_shared_graphs(dev):
    q, k, v, do = make(2, 2, 2, 40, 60, 64, BF, 20)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = G.cross_attention(*leaves)
    first = torch.autograd.grad(o, leaves, do, retain_graph=True)
    again = torch.autograd.grad(o, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    same = q.detach().requires_grad_()   # the same tensor three times over: its gradient is the sum
    (g,) = torch.autograd.grad(G.cross_attention(same, same, same), same, do)
    o, lse = G.cross_attention_fwd(q, q, q)
    dq, dk, dv = G.cross_attention_bwd(do, q, q, q, o, lse)
    ref = dq.float() + dk.float() + dv.float()
    assert ((g.float() - ref).abs() <= 3 * 2.0 ** -8 * (dq.float().abs() + dk.float().abs() + dv.float().abs())).all()
    for t in leaves:
        t.grad = None
    for _ in range(2):
        G.cross_attention(*leaves).backward(do)
    assert all(((t.grad.float() - 2 * g.float()).abs() <= 2.0 ** -7 * g.float().abs()).all() for t, g in zip(leaves, first))

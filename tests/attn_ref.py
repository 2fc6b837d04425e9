"""Attention over valid keys and its gradients in 64 bits, and the bounds its tests hold the kernels to."""
import torch

U32 = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative
F64 = torch.float64


def valid_keys(B, L, lens=None, mask=None, device="cpu"):
    ok = torch.ones(B, L, dtype=torch.bool, device=device)
    if lens is not None:
        ok &= torch.arange(L, device=device) < lens.to(device)[:, None]
    if mask is not None:
        ok &= mask.reshape(B, L)
    return ok


def attend(q, k, v, ok, scale):
    """fp64 (o, P, S) of q [B, H, N, D], k, v [B, Hk, L, D] as [B, Hk, G N, .] rows; invalid rows of k and v count as zeros."""
    B, H, N, D = q.shape
    Hk, L = k.shape[1], k.shape[2]
    z = ok[:, None, :, None]
    k, v = (torch.where(z, t.to(F64), torch.zeros((), dtype=F64, device=t.device)) for t in (k, v))
    q = q.to(F64).reshape(B, Hk, H // Hk * N, D)
    S = scale * (q @ k.transpose(2, 3).contiguous())
    M = S.masked_fill(~ok[:, None, None], -torch.inf)
    m = M.amax(-1, keepdim=True) if L else torch.zeros(*S.shape[:3], 1, dtype=F64, device=S.device)
    e = torch.exp(M - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    l = e.sum(-1, keepdim=True)
    P = e / torch.where(l == 0, torch.ones_like(l), l)
    return P @ v, P, S, q, k, v


def check(q, k, v, ok, scale, o=None, do=None, grads=None):
    """Asserts o and the gradients (dq, dk, dv) against 64 bits.

    Scores: D products, exact in fp32, summed in fp32 (D 2^-23 of the terms' magnitudes, twice the sum's bound for the matrix
    instruction's own order); their scaling, maximum and 2^x add a few fp32 steps of the score and the maximum. P's relative error E
    is that of its score and of its row's sum. P (dS) is rounded to the type: u of it, and in fp16 an absolute 2^-25 of its largest
    unit (P: of a row's maximum in the forward, 2^-10 of that in the backward; dS: 2^-4 of the row norm of do at most, doubled by the
    exponent's floor). The sums over keys or rows add one fp32 step a term at most of 32, and the result is rounded once."""
    B, H, N, D = q.shape
    Hk, L = k.shape[1], k.shape[2]
    dt, u = q.dtype, HALF[q.dtype]
    fp16 = dt == torch.float16
    ro, P, S, q6, k6, v6 = attend(q, k, v, ok, scale)
    okf = ok[:, None, None].to(F64)
    E = scale * D * 2 * U32 * (q6.abs() @ k6.abs().transpose(2, 3).contiguous()) + 4 * U32 * (1 + S.abs())
    if L:
        E = E + 4 * U32 * (S * okf).abs().amax(-1, keepdim=True)
    E = (E + (P * E).sum(-1, keepdim=True)) * okf
    n = (L / 8 + 32) * U32
    va = v6.abs()
    bo = u * ro.abs() + (P * (E + u + n)) @ va * 1.01 + (2.0 ** -25 * va.sum(-2, keepdim=True) if fp16 else 0) + (2.0 ** -25 if fp16 else 0)
    rows = lambda t: t.to(F64).reshape(B, Hk, -1, D)  # noqa: E731
    if o is not None:
        inside(rows(o), ro, bo, "o")
    if do is None:
        return
    d6 = rows(do)
    da = d6.abs()
    T = lambda t: t.transpose(2, 3).contiguous()  # noqa: E731
    r = (q6.shape[2] / 8 + 32) * U32
    dP = d6 @ T(v6)
    delta = (d6 * ro).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    rv = T(P) @ d6
    bv = u * rv.abs() + T(P * (E + u + r)) @ da * 1.01 + (2.0 ** -35 * da.sum(-2, keepdim=True) if fp16 else 0)
    dd = (da * (u * ro.abs() + bo)).sum(-1, keepdim=True)   # (delta is the rounded o's)
    e = P * (E * (dP - delta).abs() + 2 * D * U32 * (da @ T(va)) + dd + 8 * U32 * (dP.abs() + delta.abs() + (da * ro.abs()).sum(-1, keepdim=True)))
    norm = d6.square().sum(-1, keepdim=True).sqrt()
    e = (e + u * (dS.abs() + e)) * okf
    eq = e + (2.0 ** -28 * norm * okf if fp16 else 0)
    ek = e + (2.0 ** -28 * norm.amax(2, keepdim=True) * okf if fp16 else 0) if q6.shape[2] else e
    rq, rk = scale * (dS @ k6), scale * (T(dS) @ q6)
    bq = u * rq.abs() + scale * ((eq + n * dS.abs()) @ k6.abs()) * 1.01
    bk = u * rk.abs() + scale * (T(ek + r * dS.abs()) @ q6.abs()) * 1.01
    tiny = 2.0 ** -25 if fp16 else 0   # (an fp16 result's own subnormal rounding)
    dq, dk, dv = grads
    inside(rows(dq), rq, bq + tiny, "dq")
    if dk is not None:
        inside(dk.to(F64), rk, bk + tiny, "dk")
        inside(dv.to(F64), rv, bv + tiny, "dv")
        bad = ~ok[:, None, :, None]
        assert not (dk * bad).any() and not (dv * bad).any()


def inside(got, ref, bound, what):
    err = (got - ref).abs()
    over = ~(err <= bound)
    assert not over.any(), (what, int(over.sum()), float(err.max()), float((err / bound.clamp_min(1e-300)).max()))

"""Layer norm in 64 bits, and the bounds its tests hold the kernels to."""
import torch

U32 = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative
SUB = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}                 # half a step of the subnormals
# Steps of a sum over a row: 8 elements of up to 4 steps a thread, 6 halvings of the wave, 16 waves
K = 8 * 4 + 6 + 16


def stats64(x, eps):
    mu = x.mean(-1, keepdim=True)
    d = x - mu
    return mu, (d.square().mean(-1, keepdim=True) + eps) ** -0.5, d


def layer_norm64(x, w, b, eps):
    """(h, t) of fp64 x; w, b or None."""
    _, r, d = stats64(x, eps)
    t = d * r
    h = t if w is None else t * w
    return (h if b is None else h + b), t


def layer_norm_grads64(dh, dxn, x, w, eps):
    _, r, d = stats64(x, eps)
    return grads_of(dh, dxn, d * r, r, w)[:3]


def grads_of(dh, dxn, t, r, w):
    """(dx, dw, db, the terms' magnitudes that dx's error goes by)."""
    dt = dh if w is None else dh * w
    m1, m2 = dt.mean(-1, keepdim=True), (dt * t).mean(-1, keepdim=True)
    dx = r * (dt - m1 - t * m2)
    a1, a2 = dt.abs().mean(-1, keepdim=True), (dt * t).abs().mean(-1, keepdim=True)
    size = r * (6 * (dt.abs() + m1.abs() + (t * m2).abs()) + (K + 2) * a1 + (K + 6) * a2 * t.abs())
    if dxn is not None:
        dx = dx + dxn
        size = size + dxn.abs()
    rows = t.shape[:-1].numel()
    return dx, (dh * t).reshape(rows, -1).sum(0), dh.reshape(rows, -1).sum(0), size


def h_bound(h, t, w, b, dt):
    """t is off by (K + 8) 2^-24 of itself (the deviation's sums over a row, the division, the root) and by K 2^-24 (the mean's,
    in deviations); the product and the addition round once each; then the type's rounding."""
    aw = 1.0 if w is None else w.abs()
    ab = 0.0 if b is None else b.abs()
    e = U32 * ((2 * K + 8) * (t.abs() + 1.0) * aw + 4 * (t.abs() * aw + ab))
    return HALF[dt] * (h.abs() + e) + SUB[dt] + e


def dx_bound(dx, size, dt):
    e = U32 * size
    return HALF[dt] * (dx.abs() + e) + SUB[dt] + e


def sum_bound(ref, terms_abs_sum, rows, dt):
    """Rows of a thread one after another (512 workgroups, at least one team each), up to 4 teams, then 512 partial rows by 64
    groups and 6 halvings; a term's own 3 roundings."""
    e = U32 * (rows / 512 + 1 + 4 + 8 + 6 + 3) * terms_abs_sum
    return HALF[dt] * (ref.abs() + e) + SUB[dt] + e

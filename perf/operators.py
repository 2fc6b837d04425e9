"""The row-scaled FP8 operators as timed cases: the root-mean-square norm with the residual's addition and an e4m3 output
with one scale a row, its backward, the row cast, and the matrix product on row-scaled operands with bias, activation and
residual in its epilogue, forward for a sampler or a server and as a training linear.

own says which of the two run() computes: the operators' plain form in torch's elementary operations (fp32), or the
framework's calls. listed() names the cases, draw(rng) gives further ones of the same ranges, prepare(case, seed) makes
what a program holds before the call, run(state) is one pass, work(case) the bytes and operations that a pass cannot do
without, and exact(case, seed) the results in 64 bits, rounded only where the operators' definition rounds.
"""
import math
import os
import sys

import torch

own = False

E4, BF, F32, F64 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float64
EPS = 1e-6
FMAX, TINY = 448.0, 1e-12
GELU_C = math.sqrt(2.0 / math.pi)


def _api():
    """The framework's package, which only `own` needs."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-gpic_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gpic_fp8
    return gpic_fp8


# ------------------------------------------------------------------------------------------------ cases

def _norm(name, batch, tokens, width, residual=True, mod=False):
    """batch x tokens rows of `width`; residual: x + a first; mod: the block's gate, shift and scale, one row per batch
    entry."""
    return {"name": name, "kind": "norm", "batch": batch, "tokens": tokens, "width": width, "residual": residual,
            "mod": mod}


def _norm_bwd(name, rows, width, residual=True):
    return {"name": name, "kind": "norm_bwd", "rows": rows, "width": width, "residual": residual}


def _cast(name, rows, width, fp32=False):
    return {"name": name, "kind": "cast", "rows": rows, "width": width, "fp32": fp32}


def _gemm(name, batch, tokens, width, out, act="none", bias=False, residual=False, gate=False):
    """[batch x tokens, width] . [out, width]^T; out counts both halves of a swiglu."""
    return {"name": name, "kind": "gemm", "batch": batch, "tokens": tokens, "width": width, "out": out, "act": act,
            "bias": bias, "residual": residual, "gate": gate}


def _linear(name, rows, width, out, act="none", bias=True, residual=False):
    return {"name": name, "kind": "linear", "rows": rows, "width": width, "out": out, "act": act, "bias": bias,
            "residual": residual}


def _norm_linear(name, rows, width, out, act="none", bias=True, residual=True):
    return {"name": name, "kind": "norm_linear", "rows": rows, "width": width, "out": out, "act": act, "bias": bias,
            "residual": residual}


def listed():
    return [
        # One token's norm with its residual in a server's decode step: the smallest call, latency.
        _norm("norm_1_token", 1, 1, 1024),
        # A d12 image block's second norm site over the batch, with the block's gate, shift and scale.
        _norm("norm_d12_site2", 128, 256, 1024, mod=True),
        # The norm's backward over a batch of captions (128 of 51 tokens), plain residual, training.
        _norm_bwd("norm_bwd_text", 6528, 1024),
        # The same of a wide model over an odd number of packed tokens.
        _norm_bwd("norm_bwd_wide", 16381, 4096),
        # A d12 block's w12 in fp32 (DDP's master weights), cast per output channel.
        _cast("cast_w12_fp32", 8192, 1024, fp32=True),
        # The hidden activations of a d12 MLP over the batch, cast per token.
        _cast("cast_hidden", 32768, 4096),
        # One token through an MLP's first product: bias and activation in the epilogue, the weight's bytes bound it.
        _gemm("gemm_1_token_gelu", 1, 1, 1024, 4096, act="gelu_tanh", bias=True),
        # A sampler's MLP for one image with guidance (two rows of 256 tokens): w12 with SwiGLU in its epilogue.
        _gemm("gemm_sampler_swiglu", 2, 256, 1024, 8192, act="swiglu"),
        # A d12 MLP's second product over the batch with the gated residual in its epilogue.
        _gemm("gemm_d12_down_residual", 128, 256, 4096, 1024, residual=True, gate=True),
        # A text-refine sized MLP's first linear over 6592 caption tokens with SiLU, training.
        _linear("linear_text_train", 6592, 1024, 4096, act="silu"),
        # A short odd batch through norm, linear and GELU, training: launches and host time.
        _norm_linear("norm_linear_331_train", 331, 896, 3584, act="gelu_tanh"),
        # A d18 micro-batch of 64 images through norm, the MLP's first linear and GELU, training: the largest call.
        _norm_linear("norm_linear_d18_train", 16384, 1792, 7168, act="gelu_tanh"),
    ]


def _cost(c):
    """A pass's time for keeping draws below the largest listed case: seconds of the plain form, roughly."""
    w = work(c)
    return w["flops"] / 1e14 + w["bytes"] / 5e11


def _log(rng, lo, hi, step=1):
    return max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step)


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("norm", "norm_bwd", "cast", "gemm", "linear", "norm_linear"))
        yes = lambda: rng.random() < 0.5  # noqa: E731
        if kind == "norm":
            batch = _log(rng, 1, 128)
            c = _norm("", batch, _log(rng, 1, 512), _log(rng, 64, 8192, 8), yes(), yes())
        elif kind == "norm_bwd":
            c = _norm_bwd("", _log(rng, 1, 32768), _log(rng, 64, 8192, 8), yes())
        elif kind == "cast":
            c = _cast("", _log(rng, 1, 32768), _log(rng, 64, 16384, 8), yes())
        elif kind == "gemm":
            act = rng.choice(("none", "silu", "gelu_tanh", "swiglu"))
            res = yes()
            c = _gemm("", _log(rng, 1, 64), _log(rng, 1, 512), _log(rng, 64, 8192, 16),
                      _log(rng, 64, 8192, 32 if act == "swiglu" else 16), act, yes(), res, res and yes())
        else:
            c = (_linear if kind == "linear" else _norm_linear)(
                "", _log(rng, 16, 32768), _log(rng, 128, 4096, 16), _log(rng, 128, 8192, 16),
                rng.choice(("none", "silu", "gelu_tanh")), yes(), yes())
        del c["name"]
        if _cost(c) <= limit:
            return c


# ------------------------------------------------------------------------------------------------ inputs

def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=g.device) * std


def _acts(g, *shape):
    """N(0, 1) activations with 1% of the channels x20, rounded to bf16."""
    x = _randn(g, *shape)
    cols = torch.randperm(shape[-1], generator=g, device=g.device)[:max(1, round(0.01 * shape[-1]))]
    x[..., cols] *= 20.0
    return x.to(BF)


def _rowq(h):
    """The row cast in fp32: (e4m3, scale [rows])."""
    a = h.abs().amax(-1, keepdim=True).clamp_min(TINY)
    k = torch.full_like(a, FMAX)
    return (h * (k / a)).clamp(-FMAX, FMAX).to(E4), (a / k).squeeze(-1)


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c, "kind": kind}
    C = c["width"]
    if kind == "norm":
        B, N = c["batch"], c["tokens"]
        s["x"] = _acts(g, B, N, C)
        s["w"] = 1.0 + _randn(g, C, std=0.1)
        if c["residual"]:
            s["a"] = _randn(g, B, N, C).to(BF)
        if c["mod"]:
            mod = _randn(g, B, 1, 6 * C, std=0.2).to(BF).chunk(6, dim=-1)   # adaLN's output and its views
            s["shift"], s["scale"] = mod[3], mod[4]
            if c["residual"]:
                s["gate"] = mod[2]
    elif kind == "norm_bwd":
        x = _acts(g, c["rows"], C)
        s["xs"] = x
        s["w"] = 1.0 + _randn(g, C, std=0.1)
        s["rstd"] = torch.rsqrt(x.float().square().mean(-1) + EPS)
        s["dh"] = _randn(g, c["rows"], C, std=0.1).to(BF)
        if c["residual"]:
            s["dxn"] = _randn(g, c["rows"], C, std=0.1).to(BF)
    elif kind == "cast":
        s["x"] = _randn(g, c["rows"], C, std=C ** -0.5) if c["fp32"] else _acts(g, c["rows"], C)
    elif kind == "gemm":
        M, O = c["batch"] * c["tokens"], c["out"]
        s["aq"], s["sa"] = _rowq(_acts(g, M, C).float())
        s["bq"], s["sb"] = _rowq(_randn(g, O, C, std=C ** -0.5))   # a swiglu's rows in the order rows_weight lays out
        y = O // 2 if c["act"] == "swiglu" else O
        if c["bias"]:
            s["bias"] = _randn(g, O, std=0.1).to(BF)
        if c["residual"]:
            s["res"] = _randn(g, M, y).to(BF)
        if c["gate"]:
            s["gate"] = _randn(g, c["batch"], 1, 6 * y, std=0.5).to(BF).chunk(6, dim=-1)[5]
    else:
        M, O = c["rows"], c["out"]
        s["x"] = _acts(g, M, C)
        s["w"] = _randn(g, O, C, std=C ** -0.5).to(BF)
        if c["bias"]:
            s["b"] = _randn(g, O, std=0.1).to(BF)
        if kind == "norm_linear":
            s["wn"] = (1.0 + _randn(g, C, std=0.1)).to(BF)
            if c["residual"]:
                s["a"] = _randn(g, M, C).to(BF)
                s["dxn"] = _randn(g, M, C, std=0.1).to(BF)
        elif c["residual"]:
            s["res"] = _randn(g, M, O).to(BF)
        s["dy"] = _randn(g, M, O, std=0.1).to(BF)
        for k in ("x", "a", "wn", "w", "b", "res"):
            if k in s:
                s[k] = s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    s = state
    kind = s["kind"]
    if own:
        return _run_own(s, kind)
    with torch.no_grad():
        return {"norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "cast": _plain_cast, "gemm": _plain_gemm,
                "linear": _plain_linear, "norm_linear": _plain_norm_linear}[kind](s)


def _run_own(s, kind):
    G = _api()
    if kind == "norm":
        xn, _, q, sc, rstd = G.rmsnorm_rows(s["x"], s["w"], EPS, s.get("a"), s.get("gate"), s.get("shift"), s.get("scale"))
        return ([xn] if "a" in s else []) + [q, sc, rstd]
    if kind == "norm_bwd":
        return list(G.rmsnorm_rows_bwd(s["dh"], s.get("dxn"), s["xs"], s["w"], s["rstd"]))
    if kind == "cast":
        return list(G.tcast_rows(s["x"]))
    if kind == "gemm":
        return G.fp8_gemm_rows(s["aq"], s["sa"], s["bq"], s["sb"], s.get("bias"), s["case"]["act"], s.get("res"),
                               s.get("gate"))
    ins = [s[k] for k in ("x", "a", "wn", "w", "b", "res") if k in s]
    if kind == "linear":
        y = G.fp8_linear_rows(s["x"], s["w"], s.get("b"), s["case"]["act"], s.get("res"))
        return [y, *torch.autograd.grad(y, ins, s["dy"])]
    xn, y = G.fp8_rmsnorm_linear_rows(s["x"], s["wn"], EPS, s["w"], s.get("b"), s["case"]["act"], s.get("a"))
    if "a" in s:
        return [xn, y, *torch.autograd.grad((xn, y), ins, (s["dxn"], s["dy"]))]
    return [y, *torch.autograd.grad(y, ins, s["dy"])]


def _act(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(GELU_C * (z + 0.044715 * z * z * z)))
    return z


def _act_bwd(z, act):
    """act'(z)."""
    if act == "silu":
        sg = torch.sigmoid(z)
        return sg * (1.0 + z * (1.0 - sg))
    if act == "gelu_tanh":
        t = torch.tanh(GELU_C * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_C * (1.0 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _swiglu(z):
    """Rows laid out in runs of 4 of the gate's half and 4 of the other's."""
    v = z.reshape(z.shape[0], -1, 2, 4)
    g = v[:, :, 0]
    return (g * torch.sigmoid(g) * v[:, :, 1]).reshape(z.shape[0], -1)


def _plain_norm(s):
    x, shape = s["x"], s["x"].shape
    out = []
    v = x.float()
    if "a" in s:
        a = s["a"].float()
        x = (v + (s["gate"].float() * a if "gate" in s else a)).to(BF)
        v = x.float()
        out.append(x)
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    h = s["w"].float() * (v * rstd)
    if "shift" in s:
        h = h * (1.0 + s["scale"].float()) + s["shift"].float()
    q, sc = _rowq(h.reshape(-1, shape[-1]))
    return out + [q.view(shape), sc, rstd.reshape(-1)]


def _norm_grads(dh, dxn, xs, w, rstd):
    t = xs.float() * rstd[:, None]
    dt = dh.float() * w.float()
    dx = rstd[:, None] * (dt - t * (dt * t).mean(-1, keepdim=True))
    if dxn is not None:
        dx = dx + dxn.float()
    return dx.to(BF), (dh.float() * t).sum(0)


def _plain_norm_bwd(s):
    return list(_norm_grads(s["dh"], s.get("dxn"), s["xs"], s["w"], s["rstd"]))


def _plain_cast(s):
    return list(_rowq(s["x"].float()))


def _plain_gemm(s):
    c = s["case"]
    z = (s["aq"].float() @ s["bq"].float().t()) * s["sa"][:, None] * s["sb"]
    if "bias" in s:
        z = z + s["bias"].float()
    y = _swiglu(z) if c["act"] == "swiglu" else _act(z, c["act"])
    if "gate" in s:
        y = (y.view(c["batch"], c["tokens"], -1) * s["gate"].float()).view(y.shape)
    if "res" in s:
        y = y + s["res"].float()
    return y.to(BF)


def _linear_train(s, xq, sx, x, act):
    """y, and the gradients of the linear's bf16 input, weight and bias."""
    wq, sw = _rowq(s["w"].float())
    z = (xq.float() @ wq.float().t()) * sx[:, None] * sw
    if "b" in s:
        z = z + s["b"].float()
    y = _act(z, act)
    if "res" in s:
        y = y + s["res"].float()
    dz = s["dy"].float()
    if act != "none":
        dz = dz * _act_bwd(z.to(BF).float(), act)   # (the linear keeps z as bf16)
    dq, sd = _rowq(dz * sw)
    dx = ((dq.float() @ wq.float()) * sd[:, None]).to(BF)
    dz16 = dz.to(BF).float()
    grads = [(dz16.t() @ x.float()).to(BF)]
    if "b" in s:
        grads.append(dz16.sum(0).to(BF))
    return y.to(BF), dx, grads


def _plain_linear(s):
    xq, sx = _rowq(s["x"].float())
    y, dx, grads = _linear_train(s, xq, sx, s["x"], s["case"]["act"])
    return [y, dx, *grads] + ([s["dy"]] if "res" in s else [])


def _plain_norm_linear(s):
    xs = (s["x"].float() + s["a"].float()).to(BF) if "a" in s else s["x"]
    v = xs.float()
    rstd = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    h = s["wn"].float() * (v * rstd)
    hq, sh = _rowq(h)
    y, dh, grads = _linear_train(s, hq, sh, h.to(BF), s["case"]["act"])
    dx, dwn = _norm_grads(dh, s.get("dxn"), xs, s["wn"], rstd.squeeze(-1))
    if "a" in s:
        return [xs, y, dx, dx, dwn.to(BF), *grads]
    return [y, dx, dwn.to(BF), *grads]


# ------------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    c, kind, C = case, case["kind"], case["width"]
    if kind == "norm":
        M = c["batch"] * c["tokens"]
        per = 3 + (4 if c["residual"] else 0)   # x, q; a, x_new
        mod = (3 if c["residual"] else 2) * 2 * c["batch"] * C if c["mod"] else 0
        return {"bytes": per * M * C + 8 * M + 4 * C + mod, "flops": 0}
    if kind == "norm_bwd":
        M = c["rows"]
        return {"bytes": (6 + (2 if c["residual"] else 0)) * M * C + 4 * M + 8 * C, "flops": 0}
    if kind == "cast":
        return {"bytes": (5 if c["fp32"] else 3) * c["rows"] * C + 4 * c["rows"], "flops": 0}
    O = c["out"]
    if kind == "gemm":
        M, y = c["batch"] * c["tokens"], O // 2 if c["act"] == "swiglu" else O
        n = M * C + O * C + 4 * (M + O) + 2 * M * y
        n += 2 * O * c["bias"] + 2 * M * y * c["residual"] + 2 * c["batch"] * y * c["gate"]
        return {"bytes": n, "flops": 2 * M * O * C}
    M = c["rows"]
    n = 4 * M * C + 4 * M * O + 4 * O * C + 4 * O * c["bias"]   # x, dx; y, dy; w, dw; b, db
    if kind == "norm_linear":
        n += 4 * C + (8 * M * C if c["residual"] else 0)        # wn, dwn; a, da, x_new, dxn
    elif c["residual"]:
        n += 2 * M * O
    return {"bytes": n, "flops": 6 * M * O * C}


# ------------------------------------------------------------------------------------------------ 64 bits

def _b64(t):
    """Rounded to bf16 where the definition holds a bf16 tensor."""
    return t.to(BF).to(F64)


def _scaled64(h):
    """(h over its row's scale, before the rounding to e4m3; the scale)."""
    a = h.abs().amax(-1, keepdim=True).clamp_min(TINY)
    return h * (FMAX / a), (a / FMAX).squeeze(-1)


def _q64(h):
    """(the values of the row cast's e4m3, the scale) of h for the products that read them: the cast's rule, which divides
    and multiplies in IEEE fp32."""
    f = h.to(F32)
    a = f.abs().amax(-1, keepdim=True).clamp_min(TINY)
    k = torch.full_like(a, FMAX)
    return (f * (k / a)).clamp(-FMAX, FMAX).to(E4).to(F64), (a / k).squeeze(-1).to(F64)


def _sig64(z):
    return 1.0 / (1.0 + torch.exp(-z))


def _act64(z, act):
    """(act(z), act'(z))."""
    if act == "silu":
        p = _sig64(z)
        return z * p, p + z * p * (1.0 - p)
    if act == "gelu_tanh":   # z sigmoid(2 u): 1 + tanh(u) = 2 sigmoid(2 u)
        p = _sig64(2.0 * GELU_C * (z + 0.044715 * z ** 3))
        return z * p, p + z * p * (1.0 - p) * 2.0 * GELU_C * (1.0 + 0.134145 * z ** 2)
    return z, torch.ones_like(z)


def exact(case, seed):
    c, kind, C = case, case["kind"], case["width"]
    with torch.no_grad():
        s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
        d = {k: v.to(F64) for k, v in s.items() if isinstance(v, torch.Tensor)}
        if kind == "cast":
            return list(_scaled64(d["x"]))
        if kind == "norm":
            out, x = [], d["x"]
            if "a" in d:
                x = x + (d["gate"] * d["a"] if "gate" in d else d["a"])
                out.append(x)
                x = _b64(x)
            rstd = (x.square().mean(-1, keepdim=True) + EPS) ** -0.5
            h = d["w"] * x * rstd
            if "shift" in d:
                h = h * (1.0 + d["scale"]) + d["shift"]
            v, sc = _scaled64(h.reshape(-1, C))
            return out + [v.view(x.shape), sc, rstd.reshape(-1)]
        if kind == "norm_bwd":
            return _exact_norm_bwd(d["dh"], d.get("dxn"), d["xs"], d["w"], d["rstd"][:, None])
        if kind == "gemm":
            z = (d["aq"] @ d["bq"].t()) * d["sa"][:, None] * d["sb"]
            if "bias" in d:
                z = z + d["bias"]
            if c["act"] == "swiglu":
                v = z.view(z.shape[0], -1, 2, 4)
                y = (v[:, :, 0] * _sig64(v[:, :, 0]) * v[:, :, 1]).reshape(z.shape[0], -1)
            else:
                y = _act64(z, c["act"])[0]
            if "gate" in d:
                y = y * d["gate"].reshape(c["batch"], -1).repeat_interleave(c["tokens"], 0)
            return y + d["res"] if "res" in d else y
        x = d["x"]
        if kind == "norm_linear":
            if "a" in d:
                x = _b64(x + d["a"])
            rstd = (x.square().mean(-1, keepdim=True) + EPS) ** -0.5
            h = d["wn"] * x * rstd
        else:
            h = x
        hq, sh = _q64(h)
        wq, sw = _q64(d["w"])
        z = (hq @ wq.t()) * sh[:, None] * sw
        if "b" in d:
            z = z + d["b"]
        y = _act64(z, c["act"])[0]
        if "res" in d:
            y = y + d["res"]
        dz = d["dy"] * _act64(_b64(z), c["act"])[1]
        dq, sd = _q64(dz * sw)
        dh = (dq @ wq) * sd[:, None]
        dz16 = _b64(dz)
        grads = [dz16.t() @ _b64(h)] + ([dz16.sum(0)] if "b" in d else [])
        if kind == "linear":
            return [y, dh, *grads] + ([d["dy"]] if "res" in d else [])
        dx, dwn = _exact_norm_bwd(_b64(dh), d.get("dxn"), x, d["wn"], rstd)
        return ([x, y, dx, dx] if "a" in d else [y, dx]) + [dwn, *grads]


def _exact_norm_bwd(dh, dxn, x, w, rstd):
    t = x * rstd
    dt = dh * w
    dx = (dt - t * (dt * t).mean(-1, keepdim=True)) * rstd
    return [dx if dxn is None else dx + dxn, (dh * t).sum(0)]

"""The operators of a text-conditioned block's cross-attention sublayer as timed cases: the layer norm with the residual's
addition (for a server writing e4m3 with one scale a row, for training with its backward pass), attention to an encoder's
states of another length (forward, backward, and one query a head), and the low-rank adapters of many requests beside a shared
projection.

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

E4, BF, FP, F32, F64 = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32, torch.float64
DTYPES = {"bf16": BF, "fp16": FP, "fp32": F32}
EPS = 1e-5
FMAX, TINY = 448.0, 1e-12


def _api():
    """The framework's package, which only `own` needs."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-gpic_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gpic_fp8
    return gpic_fp8


# ------------------------------------------------------------------------------------------------ cases

def _norm_rows(name, rows, width, residual=True):
    """The served form: h as e4m3 with one scale a row."""
    return {"name": name, "kind": "norm_rows", "rows": rows, "width": width, "residual": residual}


def _norm(name, rows, width, residual=True, dtype="bf16"):
    """Forward and backward."""
    return {"name": name, "kind": "norm", "rows": rows, "width": width, "residual": residual, "dtype": dtype}


def _attn(name, batch, heads, kv_heads, q_len, kv_len, dim, keys="all", train=False, dtype="bf16"):
    """batch x heads x q_len queries over kv_len states of kv_heads heads; keys: "all", "lens" (each batch entry's own
    length, some of them none), "mask" (truth values, with holes)."""
    return {"name": name, "kind": "attn", "batch": batch, "heads": heads, "kv_heads": kv_heads, "q_len": q_len,
            "kv_len": kv_len, "dim": dim, "keys": keys, "train": train, "dtype": dtype}


def _lora(name, requests, tokens, adapters, rank, width, out, dtype="bf16"):
    """requests x tokens rows, each request on one of the adapters, a few on none."""
    return {"name": name, "kind": "lora", "requests": requests, "tokens": tokens, "adapters": adapters, "rank": rank,
            "width": width, "out": out, "dtype": dtype}


def listed():
    return [
        # One token's norm with its residual in a server's decode step: the smallest call, latency.
        _norm_rows("norm_rows_1_token", 1, 1024),
        # The norm before a served block's projection, over a batch of 128 images of 256 tokens.
        _norm_rows("norm_rows_d12", 32768, 1024),
        # A batch of captions (128 of 51 tokens) through the norm, training.
        _norm("norm_text_train", 6528, 1024),
        # A wide model's packed tokens, an odd number, in fp32 without a residual (a final norm), training.
        _norm("norm_wide_fp32_train", 8191, 4096, residual=False, dtype="fp32"),
        # A decode step of eight requests: one query a head over long encoder states, four heads to a key's: its bytes bound it.
        _attn("attn_1_query_long", 8, 32, 8, 1, 8191, 128, keys="lens"),
        # A sampler's image with guidance: two of 256 tokens over captions of up to 77 states.
        _attn("attn_sampler", 2, 16, 16, 256, 77, 64, keys="lens"),
        # A d12 block's batch over captions of up to 320 states, training.
        _attn("attn_d12_train", 128, 16, 16, 256, 320, 64, keys="lens", train=True),
        # Long odd sequences over longer states with holes in their mask and shared heads, training: the largest.
        _attn("attn_long_train", 2, 16, 4, 2047, 4097, 128, keys="mask", train=True),
        # One token of one request, one adapter: latency.
        _lora("lora_1_token", 1, 1, 4, 16, 1024, 1024),
        # A decode step of 64 requests on 32 adapters, one token each.
        _lora("lora_decode_64", 64, 1, 32, 16, 4096, 4096),
        # Eight sampler requests of 331 tokens, rank 64, into an MLP's first product.
        _lora("lora_sampler", 8, 331, 8, 64, 1024, 4096, dtype="fp16"),
        # Prompts of sixteen requests together.
        _lora("lora_prompts", 16, 1024, 8, 32, 4096, 4096),
    ]


def _cost(c):
    """A pass's time for keeping draws below the largest listed case: seconds of the plain form, roughly."""
    w = work(c)
    if c["kind"] == "lora":
        return w["flops"] * c["adapters"] / 1e14 + w["bytes"] / 5e11
    if c["kind"] == "attn":   # the plain form's scores in memory
        s = c["batch"] * c["heads"] * c["q_len"] * c["kv_len"]
        return w["flops"] / 1e14 + (w["bytes"] + (80 if c["train"] else 30) * s) / 4e12
    return w["bytes"] / 5e11


def _log(rng, lo, hi, step=1):
    return max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step) * step)


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(("norm_rows", "norm", "attn", "attn", "lora", "lora"))
        yes = lambda: rng.random() < 0.5  # noqa: E731
        if kind == "norm_rows":
            c = _norm_rows("", _log(rng, 1, 32768), _log(rng, 64, 8192, 8), yes())
        elif kind == "norm":
            c = _norm("", _log(rng, 1, 32768), _log(rng, 64, 8192, 8), yes(), rng.choice(("bf16", "fp16", "fp32")))
        elif kind == "attn":
            kv = _log(rng, 1, 32)
            group = rng.choice((1, 1, 2, 4, 8))
            train = yes()
            q_len = _log(rng, 1, 4096) if train or yes() else 1
            c = _attn("", _log(rng, 1, 128), kv * group, kv, q_len, _log(rng, 1, 8192), rng.choice((32, 64, 64, 72, 80, 128, 128)),
                      rng.choice(("all", "lens", "mask")), train, rng.choice(("bf16", "bf16", "fp16")))
        else:
            c = _lora("", _log(rng, 1, 64), _log(rng, 1, 1024), _log(rng, 1, 64), _log(rng, 8, 128, 8), _log(rng, 64, 8192, 16),
                      _log(rng, 64, 8192, 16), rng.choice(("bf16", "bf16", "fp16")))
        del c["name"]
        if _cost(c) <= limit:
            return c


# ------------------------------------------------------------------------------------------------ inputs

def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device=g.device) * std


def _acts(g, *shape):
    """N(0.1, 1) activations with 1% of the channels x20."""
    x = _randn(g, *shape) + 0.1
    cols = torch.randperm(shape[-1], generator=g, device=g.device)[:max(1, round(0.01 * shape[-1]))]
    x[..., cols] *= 20.0
    return x


def prepare(case, seed):
    c, kind = case, case["kind"]
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c, "kind": kind}
    if kind in ("norm", "norm_rows"):
        M, C = c["rows"], c["width"]
        dt = DTYPES[c.get("dtype", "bf16")]
        s["x"] = _acts(g, M, C).to(dt)
        if c["residual"]:
            s["a"] = _randn(g, M, C).to(dt)
        s["w"] = (1.0 + _randn(g, C, std=0.1)).to(dt)
        s["b"] = _randn(g, C, std=0.1).to(dt)
        if kind == "norm":
            s["dh"] = _randn(g, M, C, std=0.1).to(dt)
            if c["residual"]:
                s["dxn"] = _randn(g, M, C, std=0.1).to(dt)
            for k in ("x", "a", "w", "b"):
                if k in s:
                    s[k] = s[k].requires_grad_(True)
    elif kind == "attn":
        B, H, Hk, N, L, D = (c[k] for k in ("batch", "heads", "kv_heads", "q_len", "kv_len", "dim"))
        dt = DTYPES[c["dtype"]]
        s["q"] = _randn(g, B, N, H, D).to(dt).transpose(1, 2)          # the query projection's output and its view
        kv = _randn(g, B, L, 2, Hk, D).to(dt)                           # the states' one projection to keys and values
        s["k"], s["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        if c["keys"] == "lens":   # captions: from none to all of the states
            lens = torch.randint(0, L + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
            lens[0] = L
            s["lens"] = lens
        elif c["keys"] == "mask":
            m = torch.rand(B, L, generator=g, device="cuda") < 0.8
            m &= torch.arange(L, device="cuda") < torch.randint(L // 2, L + 1, (B, 1), generator=g, device="cuda")
            s["mask"] = m
        if c["train"]:
            s["do"] = _randn(g, B, N, H, D, std=0.1).to(dt).transpose(1, 2)
            for k in ("q", "k", "v"):
                s[k] = s[k].detach().requires_grad_(True)
    else:
        n, R, K, N = c["adapters"], c["rank"], c["width"], c["out"]
        M, dt = c["requests"] * c["tokens"], DTYPES[c["dtype"]]
        s["x"] = _acts(g, M, K).to(dt)
        s["y"] = _randn(g, M, N).to(dt)   # the shared projection's output
        s["A"] = _randn(g, n, R, K, std=K ** -0.5).to(dt)
        s["B"] = _randn(g, n, N, R, std=R ** -0.5).to(dt)
        s["scale"] = torch.rand(n, generator=g, device="cuda") + 0.5
        ids = torch.randint(0, n, (c["requests"],), generator=g, device="cuda", dtype=torch.int32)
        if c["requests"] > 4:
            ids[3] = -1   # a request without an adapter
        s["ids"] = ids.repeat_interleave(c["tokens"])
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    s = state
    kind = s["kind"]
    if own:
        return _run_own(s, kind)
    with torch.no_grad():
        return {"norm": _plain_norm, "norm_rows": _plain_norm_rows, "attn": _plain_attn, "lora": _plain_lora}[kind](s)


def _run_own(s, kind):
    G = _api()
    if kind == "norm_rows":
        xn, _, q, sc = G.layer_norm_rows(s["x"], s["w"], s["b"], EPS, s.get("a"))
        return ([xn] if "a" in s else []) + [q, sc]
    if kind == "norm":
        if "a" in s:
            xn, h = G.layer_norm(s["x"], s["w"], s["b"], EPS, s["a"])
            return [xn, h, *torch.autograd.grad((xn, h), (s["x"], s["a"], s["w"], s["b"]), (s["dxn"], s["dh"]))]
        h = G.layer_norm(s["x"], s["w"], s["b"], EPS)
        return [h, *torch.autograd.grad(h, (s["x"], s["w"], s["b"]), s["dh"])]
    if kind == "attn":
        o = G.cross_attention(s["q"], s["k"], s["v"], kv_lens=s.get("lens"), mask=s.get("mask"))
        return [o, *torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])] if "do" in s else o
    return G.lora_rows(s["y"], s["x"], s["A"], s["B"], s["ids"], s["scale"])


def _stats(s):
    """(x_new in the inputs' type, its normalised rows, 1 / its deviation)."""
    x = s["x"]
    if "a" in s:
        x = (x.float() + s["a"].float()).to(x.dtype)
    v = x.float()
    d = v - v.mean(-1, keepdim=True)
    rstd = torch.rsqrt(d.square().mean(-1, keepdim=True) + EPS)
    return x, d * rstd, rstd


def _plain_norm_rows(s):
    x, t, _ = _stats(s)
    h = t * s["w"].float() + s["b"].float()
    a = h.abs().amax(-1, keepdim=True).clamp_min(TINY)
    k = torch.full_like(a, FMAX)
    q = (h * (k / a)).clamp(-FMAX, FMAX).to(E4)
    return ([x] if "a" in s else []) + [q, (a / k).squeeze(-1)]


def _plain_norm(s):
    x, t, rstd = _stats(s)
    dt = x.dtype
    h = t * s["w"].float() + s["b"].float()
    dh = s["dh"].float()
    d = dh * s["w"].float()
    dx = rstd * (d - d.mean(-1, keepdim=True) - t * (d * t).mean(-1, keepdim=True))
    if "dxn" in s:
        dx = dx + s["dxn"].float()
    dx = dx.to(dt)
    dw, db = (dh * t).sum(0).to(dt), dh.sum(0).to(dt)
    return [x, h.to(dt), dx, dx, dw, db] if "a" in s else [h.to(dt), dx, dw, db]


def _plain_attn(s):
    c = s["case"]
    B, H, Hk, N, L, D = (c[k] for k in ("batch", "heads", "kv_heads", "q_len", "kv_len", "dim"))
    dt, scale, rows = s["q"].dtype, D ** -0.5, H // Hk * N
    q = s["q"].float().reshape(B * Hk, rows, D)   # a key's heads as rows beside each other
    k, v = (s[n].float().reshape(B * Hk, L, D) for n in ("k", "v"))
    valid = None
    if "lens" in s:
        valid = torch.arange(L, device=q.device) < s["lens"][:, None]
    elif "mask" in s:
        valid = s["mask"]
    z = torch.bmm(q, k.transpose(1, 2)) * scale
    if valid is not None:
        z = z.view(B, Hk, rows, L).masked_fill(~valid[:, None, None], -math.inf).view(B * Hk, rows, L)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, torch.ones_like(l), l)
    o = torch.bmm(p, v)
    out = o.view(B, H, N, D).to(dt)
    if "do" not in s:
        return out
    do = s["do"].float().reshape(B * Hk, rows, D)
    dv = torch.bmm(p.transpose(1, 2), do)
    ds = p * (torch.bmm(do, v.transpose(1, 2)) - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.bmm(ds, k)
    dk = torch.bmm(ds.transpose(1, 2), q)
    return [out, dq.view(B, H, N, D).to(dt), dk.view(B, Hk, L, D).to(dt), dv.view(B, Hk, L, D).to(dt)]


def _plain_lora(s):
    c = s["case"]
    n, R, K, N = c["adapters"], c["rank"], c["width"], c["out"]
    x, ids = s["x"].float(), s["ids"].long()
    t = (x @ s["A"].float().view(n * R, K).t()).view(-1, n, R)   # every adapter's, and of them the row's own
    own_one = ids[:, None] == torch.arange(n, device=x.device)
    t = torch.where(own_one[:, :, None], t * s["scale"][:, None], torch.zeros_like(t))
    d = t.view(-1, n * R) @ s["B"].float().transpose(1, 2).reshape(n * R, N)
    return (s["y"].float() + d).to(s["y"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass needs

def work(case):
    c, kind = case, case["kind"]
    if kind == "norm_rows":
        M, C = c["rows"], c["width"]
        return {"bytes": (3 + 4 * c["residual"]) * M * C + 4 * M + 4 * C, "flops": 0}
    if kind == "norm":
        M, C, e = c["rows"], c["width"], 4 if c["dtype"] == "fp32" else 2
        # x, h, dh, dx; a, x_new, dx_new; w, b, dw, db (dx is a's gradient too)
        return {"bytes": e * ((4 + 3 * c["residual"]) * M * C + 4 * C), "flops": 0}
    if kind == "attn":
        B, H, Hk, N, L, D = (c[k] for k in ("batch", "heads", "kv_heads", "q_len", "kv_len", "dim"))
        keys = {"all": 1.0, "lens": 0.5 + 0.5 / B, "mask": 0.6}[c["keys"]]   # of the states, those that take part
        rows = 2 * B * H * N * D * 2
        n, f = rows + 2 * B * Hk * L * D * 2 * keys, 4 * B * H * N * L * D * keys
        if c["train"]:   # do, dq; dk, dv; five products
            n, f = n + rows + 2 * B * Hk * L * D * 2, f * 3.5
        return {"bytes": int(n), "flops": int(f)}
    n, R, K, N = c["adapters"], c["rank"], c["width"], c["out"]
    M = c["requests"] * c["tokens"]
    used = n * (1.0 - (1.0 - 1.0 / n) ** c["requests"])   # adapters that some request takes, of uniform choices
    return {"bytes": int(2 * (M * K + 2 * M * N + used * R * (K + N)) + 4 * M), "flops": 2 * M * R * (K + N)}


# ------------------------------------------------------------------------------------------------ 64 bits

def exact(case, seed):
    c, kind = case, case["kind"]
    with torch.no_grad():
        s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
        d = {k: v.to(F64) for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
        if kind == "attn":
            return _exact_attn(c, s, d)
        if kind == "lora":
            out = d["y"].clone()
            for i in range(c["adapters"]):
                r = (s["ids"] == i).nonzero().squeeze(-1)
                if r.numel():
                    out[r] += d["scale"][i] * ((d["x"][r] @ d["A"][i].t()) @ d["B"][i].t())
            return out
        x = d["x"]
        out = []
        if "a" in d:
            x = x + d["a"]
            out.append(x)
            x = x.to(s["x"].dtype).to(F64)   # (x_new is handed on in the inputs' type)
        var, mu = torch.var_mean(x, -1, correction=0, keepdim=True)
        r = (var + EPS) ** -0.5
        t = (x - mu) * r
        h = d["w"] * t + d["b"]
        if kind == "norm_rows":
            a = h.abs().amax(-1, keepdim=True).clamp_min(TINY)
            return out + [h * (FMAX / a), (a / FMAX).squeeze(-1)]
        n = x.shape[-1]
        y = d["dh"] * d["w"]
        dx = r / n * (n * y - y.sum(-1, keepdim=True) - t * (y * t).sum(-1, keepdim=True))
        if "dxn" in d:
            dx = dx + d["dxn"]
        return out + [h, dx] + ([dx] if "a" in d else []) + [(d["dh"] * t).sum(0), d["dh"].sum(0)]


def _exact_attn(c, s, d):
    B, H, Hk, N, L, D = (c[k] for k in ("batch", "heads", "kv_heads", "q_len", "kv_len", "dim"))
    G, scale = H // Hk, 1.0 / math.sqrt(D)
    o, dq = torch.zeros(B, H, N, D, dtype=F64, device="cuda"), torch.zeros(B, H, N, D, dtype=F64, device="cuda")
    dk, dv = torch.zeros(B, Hk, L, D, dtype=F64, device="cuda"), torch.zeros(B, Hk, L, D, dtype=F64, device="cuda")
    for b in range(B):   # a batch entry's valid keys alone
        if "lens" in s:
            i = torch.arange(int(s["lens"][b]), device="cuda")
        elif "mask" in s:
            i = s["mask"][b].nonzero().squeeze(-1)
        else:
            i = torch.arange(L, device="cuda")
        if not i.numel():
            continue
        k, v = (d[n][b, :, i].repeat_interleave(G, 0) for n in ("k", "v"))
        q = d["q"][b].contiguous()
        p = torch.softmax(scale * (q @ k.transpose(1, 2).contiguous()), -1)
        o[b] = p @ v
        if c["train"]:
            do = d["do"][b].contiguous()
            dv[b, :, i] = (p.transpose(1, 2).contiguous() @ do).view(Hk, G, -1, D).sum(1)
            dp = do @ v.transpose(1, 2).contiguous()
            ds = p * (dp - (dp * p).sum(-1, keepdim=True)) * scale
            dq[b] = ds @ k
            dk[b, :, i] = (ds.transpose(1, 2).contiguous() @ q).view(Hk, G, -1, D).sum(1)
    return [o, dq, dk, dv] if c["train"] else o

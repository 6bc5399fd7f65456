"""The operators of a transformer block beside the framework's linear, layer_norm and attention: what is measured of them.

Five operators of ``miphei_vit_amd.torch_ops``:

* ``add_rms_norm`` (training, gradients) and ``add_rms_norm_fp8`` (serving): h = x + residual, kept in the residual stream's type;
  y = h / sqrt(mean(h^2) + eps) * weight.  The 8-bit form gives y as e4m3 with one scale a row: scale = max(max |y|, 1e-30) / 448, q = e4m3(y / scale).
* ``quantize_fp8``: the same quantisation of rows that no norm precedes (attention's output, the MLP's hidden activation).
* ``rotary``: rotary positions with several axes.  Pair i of a head turns by position[axis of i] * inv_freq[i].
* ``linear_act``: y = residual + act(x W^T + bias), 16-bit operands, with gradients.
* ``linear_fp8``: the same product of e4m3 operands with a scale for each row of x and of W (serving).

Where ``own`` is false, ``run`` computes them with elementary torch operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

EPS = 1e-6
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # H-Optimus-0's residual stream (f32, D = 1536) in a training step on 64 tiles of 256 x 256 (329 tokens each), forward and backward
        {"name": "norm train 64 tiles", "op": "norm", "rows": 64 * 329, "dim": 1536, "type": "bf16", "stream": "f32"},
        # a small odd-sized width with a 16-bit stream, as a user's own block has it: ragged rows and a width that no vector load fits
        {"name": "norm train odd width", "op": "norm", "rows": 1301, "dim": 459, "type": "fp16", "stream": "fp16"},
        # serving, one token: latency
        {"name": "norm fp8 one token", "op": "norm8", "rows": 1, "dim": 1536, "type": "bf16", "stream": "f32"},
        # serving, 16 tiles of 512 x 512 (1301 tokens each), 16-bit stream
        {"name": "norm fp8 16 large tiles", "op": "norm8", "rows": 16 * 1301, "dim": 1536, "type": "bf16", "stream": "bf16"},
        # the attention output of one tile
        {"name": "quantise one tile", "op": "quant", "rows": 329, "dim": 1536, "type": "bf16"},
        # the MLP's hidden activation of 64 tiles
        {"name": "quantise hidden 64 tiles", "op": "quant", "rows": 64 * 329, "dim": 4096, "type": "bf16"},
        # one token's packed q | k | v, turned for serving
        {"name": "rotary one token", "op": "rotary", "layout": "packed", "batch": 1, "tokens": 1, "prefix": 0, "heads": 24, "head_dim": 64,
         "axes": 1, "rotated": 64, "type": "bf16", "interleaved": False, "train": False},
        # packed q | k | v of 64 tiles: two axes (row, column) on the 18 x 18 patch grid behind class and register tokens, forward and backward
        {"name": "rotary 2-d train 64 tiles", "op": "rotary", "layout": "packed", "batch": 64, "tokens": 329, "prefix": 5, "heads": 24,
         "head_dim": 64, "axes": 2, "rotated": 64, "type": "bf16", "interleaved": False, "train": True},
        # a focal stack or a video, three axes, head-major f32 queries, neighbouring pairs, a part of each head turned
        {"name": "rotary 3-d head-major f32", "op": "rotary", "layout": "heads", "batch": 1, "tokens": 8 * 1297, "prefix": 0, "heads": 16,
         "head_dim": 128, "axes": 3, "rotated": 96, "type": "f32", "interleaved": True, "train": False},
        # MLP up-projection of 16 tiles in training, forward and the gradients of x, weight and bias
        {"name": "linear gelu train 16 tiles", "op": "linear", "rows": 16 * 329, "k": 1536, "n": 4096, "act": "gelu", "type": "bf16",
         "residual": "none", "train": True},
        # output projection of one token in serving: the weight is read once
        {"name": "linear fp8 one token", "op": "linear8", "rows": 1, "k": 1536, "n": 1536, "act": "none", "type": "bf16", "residual": "f32"},
        # MLP up-projection of 64 tiles in serving
        {"name": "linear fp8 64 tiles", "op": "linear8", "rows": 64 * 329, "k": 1536, "n": 8192, "act": "silu", "type": "bf16", "residual": "none"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm8", "quant", "rotary", "linear", "linear8"])
    t = rng.choice(["bf16", "fp16"])
    if op in ("norm", "norm8"):
        dim = _log(rng, 64, 8192)
        dim = dim if rng.random() < 0.4 else max(64, dim // 64 * 64)
        rows = _log(rng, 1, min(64 * 329, 64 * 329 * 1536 // dim))
        return {"op": op, "rows": rows, "dim": dim, "type": t, "stream": rng.choice(["f32", t])}
    if op == "quant":
        dim = _log(rng, 64, 8192)
        dim = dim if rng.random() < 0.4 else max(64, dim // 64 * 64)
        rows = _log(rng, 1, min(64 * 329, 64 * 329 * 4096 // dim))
        return {"op": op, "rows": rows, "dim": dim, "type": rng.choice([t, t, "f32"])}
    if op == "rotary":
        layout, train = rng.choice(["packed", "heads"]), rng.random() < 0.5
        axes, head_dim, heads = rng.choice([1, 2, 3, 4]), rng.choice([32, 40, 48, 64, 80, 96, 128, 256]), rng.choice([1, 2, 3, 4, 8, 16, 24])
        rotated = rng.choice([head_dim, head_dim, max(8, head_dim // 2 // 2 * 2)])
        prefix = rng.choice([0, 0, 1, 5])
        per_token = (3 if layout == "packed" else 1) * heads * head_dim
        tokens = prefix + _log(rng, 1, min(20000, 64 * 329 * 4608 // per_token // 2))
        batch = _log(rng, 1, max(1, min(64, 64 * 329 * 4608 // (per_token * tokens * 2))))
        return {"op": op, "layout": layout, "batch": batch, "tokens": tokens, "prefix": prefix, "heads": heads, "head_dim": head_dim, "axes": axes,
                "rotated": rotated, "type": rng.choice([t, "f32"]), "interleaved": rng.random() < 0.5, "train": train}
    if op == "linear":
        k, n = 8 * _log(rng, 8, 512), _log(rng, 32, 8192)
        rows = _log(rng, 1, max(1, min(16 * 1301, 5264 * 1536 * 4096 // (k * n))))
        return {"op": op, "rows": rows, "k": k, "n": n, "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), "type": t,
                "residual": rng.choice(["none", "f32", t]), "train": rng.random() < 0.5}
    k, n = 16 * _log(rng, 4, 512), _log(rng, 32, 8192)
    rows = _log(rng, 1, max(1, min(64 * 329, 64 * 329 * 1536 * 4096 // (k * n))))
    return {"op": op, "rows": rows, "k": k, "n": n, "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), "type": t,
            "residual": rng.choice(["none", "f32", t])}


def work(case):
    c, size = case, {"bf16": 2, "fp16": 2, "f32": 4}
    op, t = c["op"], size[c["type"]]
    if op in ("norm", "norm8"):
        m, s = c["rows"] * c["dim"], size[c["stream"]]
        wb = c["dim"] * 4
        if op == "norm8":   # x, residual in; q, scale, h out
            return {"bytes": m * (t + s + 1 + s) + wb + 4 * c["rows"], "flops": 6 * m}
        # forward: x, residual in, y, h out; backward: dy, dh, h in, dx, d(residual) out (one tensor where the types agree); weight and its gradient
        return {"bytes": m * (t + s + t + s) + m * (t + s + s + (s if s == t else t + s)) + 3 * wb, "flops": 16 * m}
    if op == "quant":
        m = c["rows"] * c["dim"]
        return {"bytes": m * (t + 1) + 4 * c["rows"], "flops": 3 * m}
    if op == "rotary":
        groups, turned = (3, 2) if c["layout"] == "packed" else (1, 1)
        per = c["batch"] * c["tokens"] * c["heads"] * c["head_dim"]
        moved = per * groups
        pos = (c["tokens"] - c["prefix"]) * c["axes"] * 4
        passes = 2 if c["train"] else 1
        return {"bytes": passes * (2 * moved * t + pos), "flops": passes * 3 * per * turned * c["rotated"] // c["head_dim"]}
    m, k, n = c["rows"], c["k"], c["n"]
    res = 0 if c["residual"] == "none" else size[c["residual"]]
    out = res or t
    if op == "linear8":
        return {"bytes": m * k + n * k + 4 * (m + n) + n * t + m * n * (res + out), "flops": 2 * m * n * k}
    fwd = (m * k + n * k + n) * t + m * n * (res + out)
    if not c["train"]:
        return {"bytes": fwd, "flops": 2 * m * n * k}
    return {"bytes": 2 * fwd + (m * k + n * k) * t, "flops": 6 * m * n * k}


# ------------------------------------------------------------------ what a user's program has in hand
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activation(g, rows, dim, t):
    """Activations with channels of different size and a few large ones, as transformer blocks give them."""
    channel = torch.exp(0.5 * _randn(g, dim))
    return (_randn(g, rows, dim) * channel).to(t)


def _rows_e4m3(v):
    scale = v.float().abs().amax(1).clamp_min(1e-30) / 448
    return (v.float() / scale[:, None]).clamp(-448, 448).to(E4M3), scale


def prepare(case, seed):
    g, c = _gen(seed), case
    op, t = c["op"], TYPES[c["type"]]
    s = {"case": c}
    if op in ("norm", "norm8"):
        m, d, stream = c["rows"], c["dim"], TYPES[c["stream"]]
        s["x"], s["residual"] = _activation(g, m, d, t), (3 * _activation(g, m, d, torch.float32)).to(stream)
        s["weight"] = 1 + 0.2 * _randn(g, d)
        if op == "norm":
            s["dy"], s["dh"] = (0.1 * _randn(g, m, d)).to(t), (0.1 * _randn(g, m, d)).to(stream)
            for k in ("x", "residual", "weight"):
                s[k].requires_grad_()
    elif op == "quant":
        s["x"] = _activation(g, c["rows"], c["dim"], t)
    elif op == "rotary":
        b, n, h, dh, pre, axes = (c[k] for k in ("batch", "tokens", "heads", "head_dim", "prefix", "axes"))
        pairs = c["rotated"] // 2
        sections = [pairs // axes + (a < pairs % axes) for a in range(axes)]
        where = torch.arange(n - pre, device="cuda")
        side = [max(1, math.isqrt(n - pre)) if axes == 2 else max(1, round((n - pre) ** (1 / axes)))] * axes
        start = int(torch.randint(0, 1000, (1,), device="cuda", generator=g)) if axes == 1 else 0   # one token stands behind others
        pos = [(where // math.prod(side[a + 1:])) % (side[a] if a else n) + start for a in range(axes)]
        s["positions"] = torch.stack(pos, -1).int()
        s["sections"] = sections
        s["inv_freq"] = torch.cat([100.0 ** (-torch.arange(k, device="cuda", dtype=torch.float64) / k) for k in sections])
        s["axis"] = torch.tensor([a for a, k in enumerate(sections) for _ in range(k)], device="cuda")
        if c["layout"] == "packed":
            s["x"] = _activation(g, b * n, 3 * h * dh, t).view(b, n, 3 * h, dh)
        else:
            s["x"] = _activation(g, b * h * n, dh, t).view(b, h, n, dh).transpose(1, 2)
        if c["train"]:
            s["dy"] = (0.1 * torch.randn(s["x"].shape, device="cuda", generator=g)).to(t)
            s["x"] = s["x"].detach().requires_grad_()
    else:
        m, k, n = c["rows"], c["k"], c["n"]
        x, w = _activation(g, m, k, torch.float32), _randn(g, n, k) * k ** -0.5
        s["bias"] = (0.1 * _randn(g, n)).to(t)
        s["residual"] = None if c["residual"] == "none" else _randn(g, m, n).to(TYPES[c["residual"]])
        if op == "linear8":
            (s["x"], s["x_scale"]), (s["weight"], s["w_scale"]) = _rows_e4m3(x), _rows_e4m3(w)
        else:
            s["x"], s["weight"] = x.to(t), w.to(t)
            if c["train"]:
                s["dy"] = (0.1 * _randn(g, m, n)).to(s["residual"].dtype if s["residual"] is not None else t)
                for key in ("x", "weight", "bias"):
                    s[key].requires_grad_()
                if s["residual"] is not None:
                    s["residual"].requires_grad_()
    return s


# ------------------------------------------------------------------ the plain forms
def _plain_norm(s):
    x, res, w = s["x"], s["residual"], s["weight"]
    h = (x.float() + res.float()).to(res.dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    return h, hf, rstd, hf * rstd * w


def _plain_act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def _plain_act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        u = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + u) + 0.5 * z * (1 - u * u) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_e4m3(y):
    scale = y.abs().amax(1).clamp_min(1e-30) / 448
    return (y / scale[:, None]).to(E4M3), scale


def _turn(v, cos, sin, pairs, interleaved):
    if interleaved:
        a, b = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = v[..., :pairs], v[..., pairs:2 * pairs]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, v[..., 2 * pairs:]), -1)


def _plain_rotary(s, v, turned, sign):
    """`turned` leading heads of v [B, N, heads, head_dim], tokens behind the prefix."""
    c = s["case"]
    angle = s["positions"].double()[:, s["axis"]] * s["inv_freq"]
    cos, sin = angle.cos().float()[:, None], sign * angle.sin().float()[:, None]
    part = _turn(v[:, c["prefix"]:, :turned].float(), cos, sin, c["rotated"] // 2, c["interleaved"]).to(v.dtype)
    behind = torch.cat((part, v[:, c["prefix"]:, turned:]), 2)
    return torch.cat((v[:, :c["prefix"]], behind), 1)


def _run_plain(s):
    c = s["case"]
    op = c["op"]
    if op == "norm8":
        h, _, _, y = _plain_norm(s)
        q, scale = _plain_e4m3(y)
        return {"q": q, "scale": scale, "h": h}
    if op == "norm":
        h, hf, rstd, y = _plain_norm(s)
        dy, w = s["dy"].float(), s["weight"]
        xhat, gw = hf * rstd, dy * w
        total = s["dh"].float() + rstd * (gw - xhat * (gw * xhat).mean(1, keepdim=True))
        return {"y": y.to(s["x"].dtype), "h": h, "dx": total.to(s["x"].dtype), "dresidual": total.to(h.dtype), "dweight": (dy * xhat).sum(0)}
    if op == "quant":
        q, scale = _plain_e4m3(s["x"].float())
        return {"q": q, "scale": scale}
    if op == "rotary":
        turned = (2 if c["layout"] == "packed" else 1) * c["heads"]
        y = _plain_rotary(s, s["x"], turned, 1)
        return {"y": y, "dx": _plain_rotary(s, s["dy"], turned, -1)} if c["train"] else {"y": y}
    res, out = s["residual"], TYPES[c["type"]] if s["residual"] is None else s["residual"].dtype
    z = s["x"].float() @ s["weight"].float().t()
    if op == "linear8":
        z = z * s["x_scale"][:, None] * s["w_scale"]
    z = z + s["bias"].float()
    y = _plain_act(z, c["act"])
    y = (y if res is None else res.float() + y).to(out)
    if op == "linear8" or not c["train"]:
        return {"y": y}
    dz = s["dy"].float() * _plain_act_grad(z, c["act"])
    t = s["x"].dtype
    got = {"y": y, "dx": (dz @ s["weight"].float()).to(t), "dweight": (dz.t() @ s["x"].float()).to(t), "dbias": dz.sum(0).to(t)}
    return got if res is None else {**got, "dresidual": s["dy"]}


# ------------------------------------------------------------------ the framework's calls
def _run_own(s):
    import miphei_vit_amd.torch_ops as T
    c = s["case"]
    op = c["op"]
    if op == "norm8":
        q, scale, h = T.add_rms_norm_fp8(s["x"], s["residual"], s["weight"], EPS)
        return {"q": q, "scale": scale, "h": h}
    if op == "norm":
        y, h = T.add_rms_norm(s["x"], s["residual"], s["weight"], EPS)
        dx, dres, dw = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dresidual": dres, "dweight": dw}
    if op == "quant":
        q, scale = T.quantize_fp8(s["x"])
        return {"q": q, "scale": scale}
    if op == "rotary":
        heads = (2 if c["layout"] == "packed" else 1) * c["heads"]
        args = (s["positions"], s["inv_freq"], s["sections"], heads, c["prefix"], c["interleaved"])
        y = T.rotary(s["x"], *args)
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]} if c["train"] else {"y": y}
    if op == "linear8":
        return {"y": T.linear_fp8(s["x"], s["x_scale"], s["weight"], s["w_scale"], s["bias"], s["residual"], c["act"], TYPES[c["type"]])}
    y = T.linear_act(s["x"], s["weight"], s["bias"], s["residual"], c["act"])
    if not c["train"]:
        return {"y": y}
    leaves = [s[k] for k in ("x", "weight", "bias", "residual") if s[k] is not None]
    grads = torch.autograd.grad(y, leaves, s["dy"])
    return {"y": y.detach(), **{"d" + k: v for k, v in zip(("x", "weight", "bias", "residual"), grads)}}


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _run_plain(state)


# ------------------------------------------------------------------ the definitions in 64 bits
def _e4m3_of(v):
    """v rounded to the nearest e4m3 value (ties to even): 3 bits behind the leading one, exponents from -6, up to 448."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _act_pair(z, act):
    """act(z) and its derivative."""
    zero = torch.zeros_like(z)
    if act == "none":
        return z, zero + 1
    if act == "relu":
        return torch.maximum(z, zero), torch.where(z > 0, zero + 1, zero)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p + z * p * (1 - p)
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * math.pi) ** 0.5
    k = (2 / math.pi) ** 0.5
    p = 1 / (1 + torch.exp(-2 * k * (z + 0.044715 * z ** 3)))
    return z * p, p + z * p * (1 - p) * 2 * k * (1 + 0.134145 * z ** 2)


@torch.no_grad()
def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c["op"]
    x = s["x"].detach().double()
    if op in ("norm", "norm8"):
        h = (x + s["residual"].double()).to(s["residual"].dtype).double()
        w = s["weight"].double()
        r = (h.pow(2).sum(1, keepdim=True) / c["dim"] + EPS).pow(-0.5)
        y = h * r * w
        if op == "norm8":
            scale = torch.clamp(y.abs().max(1).values, min=1e-30) / 448
            return {"q": _e4m3_of(y / scale.unsqueeze(1)), "scale": scale, "h": h}
        dy = s["dy"].double()
        # d/dh of sum_j dy_j w_j h_j r(h) with r = (|h|^2 / D + eps)^(-1/2), dr/dh_i = -r^3 h_i / D
        dot = (dy * w * h).sum(1, keepdim=True)
        total = s["dh"].double() + r * w * dy - r.pow(3) * h * dot / c["dim"]
        return {"y": y, "h": h, "dx": total, "dresidual": total, "dweight": (dy * h * r).sum(0)}
    if op == "quant":
        scale = torch.clamp(x.abs().max(1).values, min=1e-30) / 448
        return {"q": _e4m3_of(x / scale.unsqueeze(1)), "scale": scale}
    if op == "rotary":
        pairs, heads = c["rotated"] // 2, (2 if c["layout"] == "packed" else 1) * c["heads"]
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double().index_select(1, s["axis"]) * s["inv_freq"])
        if c["interleaved"]:
            first, second = torch.arange(0, 2 * pairs, 2, device="cuda"), torch.arange(1, 2 * pairs, 2, device="cuda")
        else:
            first, second = torch.arange(pairs, device="cuda"), torch.arange(pairs, 2 * pairs, device="cuda")

        def turned(v, by):
            out = v.clone()
            z = torch.complex(v[..., first], v[..., second])[:, c["prefix"]:, :heads] * by.unsqueeze(1)
            out[:, c["prefix"]:, :heads, first.tolist()] = z.real
            out[:, c["prefix"]:, :heads, second.tolist()] = z.imag
            return out

        return {"y": turned(x, turn), "dx": turned(s["dy"].double(), turn.conj())} if c["train"] else {"y": turned(x, turn)}
    w = s["weight"].detach().double()
    z = torch.matmul(x, w.t())
    if op == "linear8":
        z = z * torch.outer(s["x_scale"].double(), s["w_scale"].double())
    y, slope = _act_pair(z + s["bias"].double(), c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().double()
    if op == "linear8" or not c["train"]:
        return {"y": y}
    dz = s["dy"].double() * slope
    got = {"y": y, "dx": torch.matmul(dz, w), "dweight": torch.matmul(dz.t(), x), "dbias": dz.sum(0)}
    return got if s["residual"] is None else {**got, "dresidual": s["dy"].double()}

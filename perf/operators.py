"""Operators of an attention or feed-forward block, through the entry points of `torchllmtuner_b200.ops`.

Five kinds of case, on one GPU:

  linear      `ops.linear_act`: a linear layer with bias, activation and residual; forward and every gradient
  layer_norm  `ops.layer_norm`: LayerNorm over the width of a vision tower; forward and every gradient
  rope        `ops.rope`: rotary positions on part of a head, pairs in halves or side by side; forward and gradient
  tables      `ops.rope_tables` with frequencies scaled for long contexts
  qk          `ops.qk_norm_rope`: per-head norms of queries and keys with the rotation in the same pass; forward and every gradient
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # the first MLP layer of the default tower (128 -> 256) on one 14 x 14 image: the smallest call, where launches count
        {"name": "linear_small", "kind": "linear", "rows": 196, "in": 128, "out": 256, "act": "gelu_tanh", "bias": True, "residual": False},
        # the first MLP layer of a tower with 16 heads of 72 on sixteen images of 32 x 32 patches
        {"name": "linear_up", "kind": "linear", "rows": 16384, "in": 1152, "out": 4608, "act": "gelu_tanh", "bias": True, "residual": False},
        # that tower's attention output projection, added to the residual stream
        {"name": "linear_proj", "kind": "linear", "rows": 16384, "in": 1152, "out": 1152, "act": "none", "bias": True, "residual": True},
        # the merger's first layer on the 2 x 2 neighbourhoods of a few images of unequal size
        {"name": "linear_merger", "kind": "linear", "rows": 1021, "in": 4608, "out": 4608, "act": "gelu", "bias": True, "residual": False},
        # the default tower's norm on one image
        {"name": "layer_norm_small", "kind": "layer_norm", "rows": 196, "dim": 128, "dtype": "bf16"},
        # the norm of a 1152-wide tower, twice per block
        {"name": "layer_norm_tower", "kind": "layer_norm", "rows": 16384, "dim": 1152, "dtype": "bf16"},
        # queries and keys of that tower as one view of the packed projection, pairs side by side (2-D positions)
        {"name": "rope_tower", "kind": "rope", "rows": 16384, "heads": 32, "of": 48, "dim": 72, "offset": 0, "rot": 72, "layout": "interleaved",
         "dtype": "bf16"},
        # the trailing half of DeepSeek-V4's heads (the recipe among the examples), an odd number of tokens
        {"name": "rope_trailing", "kind": "rope", "rows": 1001, "heads": 16, "of": 16, "dim": 128, "offset": 64, "rot": 64, "layout": "interleaved",
         "dtype": "bf16"},
        # the longest context of the Qwen3 configuration, extended four times from 32768
        {"name": "tables_long", "kind": "tables", "rows": 131072, "dim": 128, "theta": 1e6, "rope_type": "yarn", "factor": 4.0, "original": 32768},
        # a short packed batch with positions divided by 8
        {"name": "tables_short", "kind": "tables", "rows": 700, "dim": 64, "theta": 1e4, "rope_type": "linear", "factor": 8.0, "original": 2048},
        # Qwen3.5's gated attention at its training length: zero-centred norms, a quarter of the head rotates, queries lie beside their gates
        {"name": "qk_gated", "kind": "qk", "rows": 8192, "heads": 16, "kv_heads": 4, "dim": 256, "offset": 0, "rot": 64, "layout": "half",
         "norm": "zero_centered", "gated": True, "dtype": "bf16"},
        # DeepSeek-V4's queries (no weight) and its one shared key on a short document
        {"name": "qk_shared_key", "kind": "qk", "rows": 77, "heads": 16, "kv_heads": 1, "dim": 128, "offset": 64, "rot": 64, "layout": "interleaved",
         "norm": "unit_q", "gated": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "layer_norm", "rope", "tables", "qk"])
    if kind == "linear":
        if rng.random() < 0.25:                    # widths that are no multiple of anything
            n_in, n_out = _log(rng, 33, 2000), _log(rng, 33, 2000)
        else:
            n_in, n_out = 8 * _log(rng, 8, 576), 8 * _log(rng, 8, 576)
        rows = min(_log(rng, 16, 16384), 16384 * 1152 * 4608 // (n_in * n_out))
        return {"kind": kind, "rows": rows, "in": n_in, "out": n_out, "act": rng.choice(["none", "gelu", "gelu_tanh", "silu", "relu"]),
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.5}
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "layer_norm":
        dim = rng.choice([8 * _log(rng, 2, 1024), _log(rng, 17, 4000)])
        return {"kind": kind, "rows": min(_log(rng, 1, 16384), 9437184 // dim), "dim": dim, "dtype": dtype}
    if kind == "tables":
        return {"kind": kind, "rows": _log(rng, 1, 131072), "dim": 2 * rng.randint(4, 64), "theta": rng.choice([1e4, 1e6, 1e7]),
                "rope_type": rng.choice(["linear", "llama3", "yarn"]), "factor": rng.choice([2.0, 4.0, 8.0]), "original": rng.choice([4096, 32768])}
    layout = rng.choice(["half", "interleaved"])
    dim = rng.choice([64, 72, 80, 96, 128, 192, 256, 2 * rng.randint(8, 128)])
    rot = dim if rng.random() < 0.4 else 2 * rng.randint(1, dim // 2)
    if rot < dim and rng.random() < 0.5 and dim % 16 == 0:
        rot = dim // 2
    offset = rng.choice([0, dim - rot])
    if kind == "rope":
        heads = _log(rng, 1, 48)
        return {"kind": kind, "rows": min(_log(rng, 1, 16384), 37748736 // (heads * dim)), "heads": heads,
                "of": heads * rng.choice([1, 2, 3]), "dim": dim, "offset": offset, "rot": rot, "layout": layout, "dtype": dtype}
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4])
    return {"kind": kind, "rows": min(_log(rng, 1, 8192), 16777216 // (heads * dim)), "heads": heads, "kv_heads": kv, "dim": dim, "offset": offset, "rot": rot,
            "layout": layout, "norm": rng.choice(["weight", "zero_centered", "unit_q", "none"]), "gated": rng.random() < 0.4, "dtype": dtype}


# ------------------------------------------------------------------------------------------------------------ inputs
class _Make:
    """Tensors of one seed, in the order they are asked for."""

    def __init__(self, seed, dtype):
        self.g, self.dtype = torch.Generator(device=DEV).manual_seed(int(seed)), dtype

    def normal(self, *shape, std=1.0, mean=0.0, spread=None):
        t = torch.empty(*shape, dtype=torch.float32, device=DEV).normal_(mean, std, generator=self.g)
        if spread is not None:                     # a few channels much larger than the rest, as in a trained residual stream
            t[..., ::spread] *= 8.0
        return t.to(self.dtype)

    def positions(self, n):
        """Document-relative positions of a packed row: two documents, the second starting at a place that depends on the seed."""
        cut = int(torch.randint(0, n, (1,), generator=self.g, device=DEV))
        return torch.cat((torch.arange(cut, device=DEV), torch.arange(n - cut, device=DEV)))


def _angles(positions, rot, theta=1e4):
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    return positions.double()[:, None] * inv


def _inputs(c, seed):
    m, kind, n = _Make(seed, TYPES[c.get("dtype", "bf16")]), c["kind"], c["rows"]
    if kind == "linear":
        s = {"x": m.normal(n, c["in"]), "w": m.normal(c["out"], c["in"], std=c["in"] ** -0.5), "dy": m.normal(n, c["out"])}
        if c["bias"]:
            s["b"] = m.normal(c["out"], std=0.5)
        if c["residual"]:
            s["r"] = m.normal(n, c["out"], std=2.0)
        return s
    if kind == "layer_norm":
        return {"x": m.normal(n, c["dim"], mean=0.3, spread=37), "w": m.normal(c["dim"], std=0.1, mean=1.0), "b": m.normal(c["dim"], std=0.1),
                "dy": m.normal(n, c["dim"])}
    if kind == "tables":
        return {"positions": m.positions(n)}
    ang = _angles(m.positions(n), c["rot"])
    s = {"cos": ang.cos().float(), "sin": ang.sin().float()}
    if kind == "rope":
        return s | {"x": m.normal(n, c["of"], c["dim"])[:, :c["heads"]], "dy": m.normal(n, c["heads"], c["dim"])}
    H, K, d = c["heads"], c["kv_heads"], c["dim"]
    s["q"] = m.normal(n, H, 2 * d)[..., :d] if c["gated"] else m.normal(n, H, d)
    s["k"] = m.normal(n, K, d)
    mean = 0.0 if c["norm"] == "zero_centered" else 1.0
    if c["norm"] in ("weight", "zero_centered"):
        s["qw"] = m.normal(d, std=0.1, mean=mean)
    if c["norm"] != "none":
        s["kw"] = m.normal(d, std=0.1, mean=mean)
    return s | {"dq": m.normal(n, H, d), "dk": m.normal(n, K, d)}


LEAVES = {"linear": ("x", "w", "b", "r"), "layer_norm": ("x", "w", "b"), "rope": ("x",), "tables": (), "qk": ("q", "k", "qw", "kw")}


def prepare(case, seed):
    s = _inputs(case, seed)
    for name in LEAVES[case["kind"]]:
        if name in s:
            s[name] = s[name].detach().requires_grad_()
    s["case"] = case
    return s


def _scaling(c):
    s = {"rope_type": c["rope_type"], "factor": c["factor"], "original_max_position_embeddings": c["original"]}
    return s | {"low_freq_factor": 1.0, "high_freq_factor": 4.0} if c["rope_type"] == "llama3" else s


# --------------------------------------------------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z.clamp(min=0.0) if act == "relu" else z


def _rotate(x, cos, sin, c):
    a, r = c["offset"], c["rot"]
    t = x[..., a:a + r]
    cos, sin = cos[:, None, :], sin[:, None, :]
    if c["layout"] == "half":
        u, v = t[..., :r // 2], t[..., r // 2:]
        t = torch.cat((u * cos - v * sin, v * cos + u * sin), -1)
    else:
        u, v = t[..., 0::2], t[..., 1::2]
        t = torch.stack((u * cos - v * sin, v * cos + u * sin), -1).flatten(-2)
    return torch.cat((x[..., :a], t, x[..., a + r:]), -1)


def _unit(x):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain(t, c):
    """The outputs that have gradients, from 32-bit leaves."""
    kind = c["kind"]
    if kind == "linear":
        z = t["x"] @ t["w"].t()
        z = z + t["b"] if "b" in t else z
        y = _act(z, c["act"])
        return {"y": y + t["r"] if "r" in t else y}
    if kind == "layer_norm":
        d = t["x"] - t["x"].mean(-1, keepdim=True)
        return {"y": d * torch.rsqrt((d * d).mean(-1, keepdim=True) + EPS) * t["w"] + t["b"]}
    if kind == "rope":
        return {"y": _rotate(t["x"], t["cos"], t["sin"], c)}
    q, k = t["q"], t["k"]
    if c["norm"] != "none":
        shift = 1.0 if c["norm"] == "zero_centered" else 0.0
        q, k = _unit(q), _unit(k) * (t["kw"] + shift)
        q = q * (t["qw"] + shift) if "qw" in t else q
    return {"q": _rotate(q, t["cos"], t["sin"], c), "k": _rotate(k, t["cos"], t["sin"], c)}


def _frequencies(c, device):
    """Scaled inverse frequencies in 64 bits and the factor on both tables."""
    d, s, L = c["dim"], c["factor"], c["original"]
    j = torch.arange(0, d // 2, dtype=torch.float64, device=device)
    inv = torch.exp(-2.0 * j / d * math.log(c["theta"]))
    if c["rope_type"] == "linear":
        return inv / s, 1.0
    if c["rope_type"] == "llama3":
        turns = L * inv / (2.0 * math.pi)                          # rotations within the original context
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return inv * keep + inv / s * (1.0 - keep), 1.0
    at = lambda turns: d * math.log(L / (turns * 2.0 * math.pi)) / (2.0 * math.log(c["theta"]))  # noqa: E731
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
    ramp = ((j - low) / (high - low if high != low else 0.001)).clamp(0.0, 1.0)
    return inv * (1.0 - ramp) + inv / s * ramp, 0.1 * math.log(s) + 1.0


GRADS = {"linear": ("dy",), "layer_norm": ("dy",), "rope": ("dy",), "qk": ("dq", "dk")}


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "tables":
        if own:
            from torchllmtuner_b200 import ops
            cos, sin = ops.rope_tables(s["positions"], c["dim"], c["theta"], scaling=_scaling(c))
            return {"cos": cos, "sin": sin}
        inv, factor = _frequencies(c, s["positions"].device)
        ang = s["positions"].double()[:, None] * inv
        return {"cos": (ang.cos() * factor).float(), "sin": (ang.sin() * factor).float()}
    names = [n for n in LEAVES[kind] if n in s]
    upstream = [s[n] for n in GRADS[kind]]
    if own:
        from torchllmtuner_b200 import ops
        if kind == "linear":
            outs = {"y": ops.linear_act(s["x"], s["w"], s.get("b"), activation=None if c["act"] == "none" else c["act"], residual=s.get("r"))}
        elif kind == "layer_norm":
            outs = {"y": ops.layer_norm(s["x"], s["w"], s["b"], EPS)}
        elif kind == "rope":
            outs = {"y": ops.rope(s["x"], s["cos"], s["sin"], layout=c["layout"], offset=c["offset"])}
        else:
            q, k = ops.qk_norm_rope(s["q"], s["k"], s.get("qw"), s.get("kw"), s["cos"], s["sin"], EPS, layout=c["layout"], offset=c["offset"],
                                    norm=c["norm"] != "none", zero_centered=c["norm"] == "zero_centered")
            outs = {"q": q, "k": k}
        grads = torch.autograd.grad(list(outs.values()), [s[n] for n in names], upstream)
        return {n: t.detach() for n, t in outs.items()} | {"d_" + n: g for n, g in zip(names, grads)}
    leaves = {n: s[n].detach().float().requires_grad_() for n in names}
    outs = _plain(leaves | {n: s[n] for n in ("cos", "sin") if n in s}, c)
    grads = torch.autograd.grad(list(outs.values()), list(leaves.values()), [g.float() for g in upstream])
    dtype = upstream[0].dtype
    return {n: t.detach().to(dtype) for n, t in outs.items()} | {"d_" + n: g.to(dtype) for n, g in zip(names, grads)}


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, kind, n = case, case["kind"], case["rows"]
    size = 4 if c.get("dtype") == "fp32" else 2
    if kind == "linear":
        i, o = c["in"], c["out"]
        values = 2 * n * i + 2 * i * o + 2 * n * o + (2 * o if c["bias"] else 0) + (2 * n * o if c["residual"] else 0)
        return {"bytes": 2 * values, "flops": 6 * n * i * o}
    if kind == "layer_norm":
        return {"bytes": size * (4 * n * c["dim"] + 4 * c["dim"]), "flops": 20 * n * c["dim"]}
    if kind == "tables":
        return {"bytes": 8 * n + 4 * n * c["dim"], "flops": 20 * n * c["dim"]}
    if kind == "rope":
        return {"bytes": size * 4 * n * c["heads"] * c["dim"] + 4 * n * c["rot"], "flops": 6 * n * c["heads"] * c["rot"]}
    heads, norm = c["heads"] + c["kv_heads"], c["norm"] != "none"
    # without a norm the gradient needs the tables alone: queries and keys are read once either way
    return {"bytes": size * 4 * n * heads * c["dim"] + 4 * n * c["rot"], "flops": n * heads * (6 * c["rot"] + (20 * c["dim"] if norm else 0))}


# -------------------------------------------------------------------------------------------------------- in 64 bits
def _act64(z, act):
    """The activation and its derivative, from their definitions."""
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * k * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    return z, torch.ones_like(z)


def _turn64(x, cos, sin, c, sign):
    """Rotation as complex numbers: by the tables' angles (sign 1) or back (sign -1)."""
    a, r = c["offset"], c["rot"]
    t, turn = x[..., a:a + r], torch.complex(cos, sign * sin)[:, None, :]
    if c["layout"] == "half":
        z = torch.complex(t[..., :r // 2].contiguous(), t[..., r // 2:].contiguous()) * turn
        t = torch.cat((z.real, z.imag), -1)
    else:
        t = torch.view_as_real(torch.view_as_complex(t.reshape(*t.shape[:-1], r // 2, 2).contiguous()) * turn).flatten(-2)
    out = x.clone()
    out[..., a:a + r] = t
    return out


def _norm64(x, w, dn):
    """x / rms(x) * w for one operand, with its gradients from those of the result."""
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    h, g = x * r, dn * w
    return h * w, r * (g - h * (g * h).mean(-1, keepdim=True)), (dn * h).sum((0, 1))


def exact(case, seed):
    c, kind = case, case["kind"]
    s = {n: t.double() if t.is_floating_point() else t for n, t in _inputs(c, seed).items()}
    if kind == "linear":
        z = torch.nn.functional.linear(s["x"], s["w"], s.get("b"))
        y, slope = _act64(z, c["act"])
        dz = s["dy"] * slope
        out = {"y": y + s["r"] if "r" in s else y, "d_x": dz @ s["w"], "d_w": dz.t() @ s["x"]}
        if "b" in s:
            out["d_b"] = dz.sum(0)
        if "r" in s:
            out["d_r"] = s["dy"]
        return out
    if kind == "layer_norm":
        var, mean = torch.var_mean(s["x"], -1, correction=0, keepdim=True)
        r = (var + EPS).rsqrt()
        h, g = (s["x"] - mean) * r, s["dy"] * s["w"]
        return {"y": torch.addcmul(s["b"], h, s["w"]), "d_x": r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True)),
                "d_w": (s["dy"] * h).sum(0), "d_b": s["dy"].sum(0)}
    if kind == "tables":
        d, f, L = c["dim"], c["factor"], c["original"]
        inv, scale = [c["theta"] ** (-2.0 * j / d) for j in range(d // 2)], 1.0
        if c["rope_type"] == "linear":
            inv = [v / f for v in inv]
        elif c["rope_type"] == "llama3":
            mixed = []
            for v in inv:
                length = 2.0 * math.pi / v
                smooth = (L / length - 1.0) / 3.0
                mixed.append(v / f if length > L else v if length < L / 4.0 else (1 - smooth) * v / f + smooth * v)
            inv = mixed
        else:
            edge = [d * math.log(L / (2.0 * math.pi * b)) / (2.0 * math.log(c["theta"])) for b in (32.0, 1.0)]
            lo, hi = max(0, math.floor(edge[0])), min(d - 1, math.ceil(edge[1]))
            hi = hi + 0.001 if hi == lo else hi
            inv = [v / f * w + v * (1 - w) for v, w in ((v, min(1.0, max(0.0, (j - lo) / (hi - lo)))) for j, v in enumerate(inv))]
            scale = 1.0 + 0.1 * math.log(f)
        ang = torch.outer(s["positions"].double(), torch.tensor(inv, dtype=torch.float64, device=DEV))
        return {"cos": scale * ang.cos(), "sin": scale * ang.sin()}
    if kind == "rope":
        return {"y": _turn64(s["x"], s["cos"], s["sin"], c, 1), "d_x": _turn64(s["dy"], s["cos"], s["sin"], c, -1)}
    back = {n: _turn64(s["d" + n], s["cos"], s["sin"], c, -1) for n in "qk"}
    out = {"q": s["q"], "k": s["k"], "d_q": back["q"], "d_k": back["k"]}
    if c["norm"] != "none":
        one = 1.0 if c["norm"] == "zero_centered" else 0.0
        for n in "qk":
            w = s[n + "w"] + one if n + "w" in s else torch.ones(c["dim"], dtype=torch.float64, device=DEV)
            out[n], out["d_" + n], dw = _norm64(s[n], w, back[n])
            if n + "w" in s:
                out[f"d_{n}w"] = dw
    turned = {n: _turn64(out[n], s["cos"], s["sin"], c, 1) for n in "qk"}
    return turned | {n: out[n] for n in ("d_q", "d_k", "d_qw", "d_kw") if n in out}

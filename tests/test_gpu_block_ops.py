"""Linear layers with an epilogue, LayerNorm, rotary positions and per-head norms with rotation against their formulas in 64 bits.

Bounds are element-wise: each rounding to the storage type is off by at most half a step, U = eps / 2 relative to the value (bf16 2^-8, fp32
2^-24); fp32 arithmetic in front of it by N 2^-24 of the sum of the absolute values of the terms, with N the number of dependent additions plus
a few for the functions in between (64 covers the trees over a row, a thread's terms and rsqrt / exp / erfc)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
E32 = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(*shape, seed=0, dtype=torch.bfloat16, std=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std + mean).to(dtype)


def _near(out, ref, bound, name):
    assert out.shape == ref.shape, f"{name}: {tuple(out.shape)} against {tuple(ref.shape)}"
    assert torch.isfinite(out).all(), f"{name}: not finite"
    off = (out.double() - ref).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    if worst > 0:
        at = tuple(int(i) for i in torch.unravel_index((off - bound).argmax(), off.shape))
        raise AssertionError(f"{name}{list(at)}: {out[at].item()} against {ref[at].item()}, bound {bound[at].item()}, {(off > bound).sum().item()} outside")


# ------------------------------------------------------------------------------------------------------------ linear
def _act64(z, act):
    """Value, first derivative and a bound on the second."""
    if act == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        pdf = torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
        return z * cdf, cdf + z * pdf, 0.8                  # |(2 - z^2) pdf| <= 2 / sqrt(2 pi)
    if act == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (z + 0.044715 * z ** 3))
        du = k * (1 + 3 * 0.044715 * z * z)
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * du, 0.85
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s)), 0.5
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    return z, torch.ones_like(z), 0.0


def _linear_check(x, w, b, r, act, dy, outs):
    u = _u(torch.bfloat16)
    X, W, G = (t.double() for t in (x, w, dy))
    x2, g2 = X.reshape(-1, X.shape[-1]), G.reshape(-1, G.shape[-1])
    M, K, N = x2.shape[0], x2.shape[1], W.shape[0]
    z = x2 @ W.t() + (b.double() if b is not None else 0)
    size = x2.abs() @ W.abs().t() + (b.double().abs() if b is not None else 0)
    y, slope, curve = _act64(z, act)
    ez = (K + 8) * E32 * size
    R = r.double().expand(*x.shape[:-1], N).reshape(M, N) if r is not None else torch.zeros_like(y)
    ref = y + R
    # |act'| <= 1.13; the functions are off by 8 steps of fp32 relative to z
    _near(outs["y"].reshape(M, N), ref, u * ref.abs() + 1.13 * ez + 16 * E32 * (z.abs() + R.abs()) + 1e-30, "y")
    dz = g2 * slope
    edz = u * dz.abs() + g2.abs() * (curve * (u * z.abs() + ez) + 16 * E32 * (1 + z.abs())) if act else torch.zeros_like(dz)
    if act == "relu":
        keep = z.abs() > ez                                 # next to the kink either slope is right
        edz = torch.where(keep, edz, g2.abs())
    _near(outs["dx"].reshape(M, K), dz @ W, u * (dz @ W).abs() + edz @ W.abs() + (N + 8) * E32 * ((dz.abs() + edz) @ W.abs()) + 1e-30, "dx")
    dw = dz.t() @ x2
    _near(outs["dw"], dw, u * dw.abs() + edz.t() @ x2.abs() + (M + 8) * E32 * ((dz.abs() + edz).t() @ x2.abs()) + 1e-30, "dw")
    if b is not None:
        db = dz.sum(0)
        edb = edz - u * dz.abs() if act else edz            # summed before dz is rounded
        ub = _u(b.dtype)
        _near(outs["db"], db, ub * db.abs() + edb.sum(0).clamp(min=0) + (M + 64) * E32 * dz.abs().sum(0) + 1e-30, "db")


def _linear_run(x, w, b, r, act, dy):
    from torchllmtuner_b200 import ops
    leaves = [t for t in (x, w, b, r) if t is not None]
    y = ops.linear_act(x, w, b, activation=act, residual=r)
    grads = dict(zip([n for n, t in zip(("dx", "dw", "db", "dr"), (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, dy)))
    return {"y": y.detach(), **grads}


@pytest.mark.parametrize("act", [None, "gelu", "gelu_tanh", "silu", "relu"])
@pytest.mark.parametrize("M,K,N", [(1, 64, 128), (196, 128, 256), (130, 72, 264), (333, 1152, 200), (257, 40, 1000), (1021, 256, 520)])
def test_linear_act(M, K, N, act):
    x, w = _rand(M, K, seed=1).requires_grad_(), _rand(N, K, seed=2, std=K ** -0.5).requires_grad_()
    b, r, dy = _rand(N, seed=3, std=0.5).requires_grad_(), _rand(M, N, seed=4).requires_grad_(), _rand(M, N, seed=5)
    outs = _linear_run(x, w, b, r, act, dy)
    _linear_check(x.detach(), w.detach(), b.detach(), r.detach(), act, dy, outs)
    assert torch.equal(outs["dr"], dy)
    outs = _linear_run(x, w, None, None, act, dy)
    _linear_check(x.detach(), w.detach(), None, None, act, dy, outs)


@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (5, 33, 7), (129, 65, 131), (300, 577, 259), (64, 100, 36), (40, 64, 1153), (700, 1001, 33)])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
def test_linear_act_widths_off_the_vector_grid(M, K, N, act):
    x, w = _rand(M, K, seed=1).requires_grad_(), _rand(N, K, seed=2, std=K ** -0.5).requires_grad_()
    b, r, dy = _rand(N, seed=3, dtype=torch.float32).requires_grad_(), _rand(M, N, seed=4).requires_grad_(), _rand(M, N, seed=5)
    _linear_check(x.detach(), w.detach(), b.detach(), r.detach(), act, dy, _linear_run(x, w, b, r, act, dy))


def test_linear_act_strides_and_broadcast_residual():
    """Rows of a wider buffer, a transposed weight, a strided upstream gradient, a residual broadcast over rows, an input with more dimensions."""
    big = _rand(3, 50, 200, seed=1)
    x = big[..., 3:131].detach().requires_grad_()
    w = _rand(128, 96, seed=2, std=0.1).t().detach().requires_grad_()
    b, r = _rand(96, seed=3).requires_grad_(), _rand(50, 96, seed=4).requires_grad_()
    dy = _rand(3, 96, 50, seed=5).transpose(1, 2)
    outs = _linear_run(x, w, b, r, "gelu", dy)
    assert torch.equal(outs["dr"], dy.sum(0))
    _linear_check(x.detach(), w.detach(), b.detach(), r.detach(), "gelu", dy, outs)


def test_linear_act_partial_gradients_and_no_grad():
    from torchllmtuner_b200 import ops
    x, w, b = _rand(200, 64, seed=1), _rand(72, 64, seed=2, std=0.1), _rand(72, seed=3)
    dy = _rand(200, 72, seed=4)
    full = _linear_run(*(t.clone().requires_grad_() for t in (x, w, b)), None, "silu", dy)
    for i, name in enumerate(("dx", "dw", "db")):
        args = [t.clone() for t in (x, w, b)]
        args[i].requires_grad_()
        g, = torch.autograd.grad(ops.linear_act(*args, activation="silu"), args[i], dy)
        assert torch.equal(g, full[name])
    with torch.no_grad():
        assert torch.equal(ops.linear_act(x, w, b, activation="silu"), full["y"])
    for shape in ((0, 64), (0, 3, 64)):
        e = torch.empty(*shape, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        y = ops.linear_act(e, w.requires_grad_(), b, activation="gelu")
        assert y.shape == (*shape[:-1], 72)
        assert torch.autograd.grad(y.sum(), w)[0].abs().max() == 0


def test_linear_act_special_values():
    """Infinities, NaN and values far out in the tails: what the activation's formula gives, and rows keep to themselves."""
    from torchllmtuner_b200 import ops
    K = 64
    w = torch.eye(K, device=DEV).bfloat16()
    x = torch.zeros(130, K, device=DEV).bfloat16()
    x[0, :6] = torch.tensor([float("nan"), 1e30, -1e30, 40.0, -40.0, 3e38], device=DEV)
    for act, far in (("relu", 0.0), ("gelu", 0.0), ("gelu_tanh", 0.0), ("silu", 0.0)):
        y = ops.linear_act(x, w, activation=act)
        assert y[0].isnan().all() or (y[0, 0].isnan() and y[0, 4].abs() <= 1e-12)       # NaN spreads through the product of its row
        assert torch.equal(y[1:], torch.zeros_like(y[1:]))
    z = torch.tensor([-1e30, -40.0, -8.0, -5.0, -3.0, -0.0, 0.0, 3.0, 40.0, 1e30], device=DEV)
    x = torch.zeros(10, K, device=DEV).bfloat16()
    x[:, 0] = z.bfloat16()
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        y = ops.linear_act(x, w, activation=act)[:, 0].double()
        ref = _act64(x[:, 0].double(), act)[0]
        assert ((y - ref).abs() <= _u(torch.bfloat16) * ref.abs() * 1.01 + 1e-20).all(), (act, y, ref)


# --------------------------------------------------------------------------------------------------------- LayerNorm
def _norm_check(x, w, b, dy, y, dx, dw, db, eps):
    u = _u(x.dtype)
    D = x.shape[-1]
    X, G = x.double().reshape(-1, D), dy.double().reshape(-1, D)
    W, B = w.double(), b.double()
    mean = X.mean(1, keepdim=True)
    r = ((X - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    h = (X - mean) * r
    A = (X.abs() + mean.abs() + X.abs().mean(1, keepdim=True)) * r
    n = 64 + D / 256
    ref = h * W + B
    _near(y.reshape(-1, D), ref, u * ref.abs() + n * E32 * (A * W.abs() * (1 + (A * A).mean(1, keepdim=True)) + B.abs()), "y")
    g = G * W
    ref = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    cond = 1 + (A * A).mean(1, keepdim=True)                # of the variance: how much cancels in x - mean
    _near(dx.reshape(-1, D), ref, u * ref.abs() + n * E32 * cond * r * (g.abs() + g.abs().mean(1, keepdim=True) + A * (g.abs() * A).mean(1, keepdim=True)) + 1e-30, "dx")
    R = X.shape[0]
    _near(dw, (G * h).sum(0), u * (G * h).sum(0).abs() + (n + R) * E32 * (G.abs() * A * cond).sum(0) + 1e-30, "dw")
    _near(db, G.sum(0), u * G.sum(0).abs() + (n + R) * E32 * G.abs().sum(0) + 1e-30, "db")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("R,D", [(1, 1), (1, 8), (3, 2), (196, 128), (7, 129), (1000, 1152), (33, 1001), (517, 255), (2, 2047), (65, 2056), (9, 4099), (5, 8192), (3, 10007)])
def test_layer_norm(R, D, dtype):
    from torchllmtuner_b200 import ops
    if D > 8190 and dtype == "fp32":
        D = 8185
    dt = TYPES[dtype]
    x = _rand(R, D, seed=1, dtype=dt, mean=0.5)
    x[..., ::37] *= 8
    x.requires_grad_()
    w, b, dy = _rand(D, seed=2, dtype=dt, mean=1, std=0.1).requires_grad_(), _rand(D, seed=3, dtype=dt).requires_grad_(), _rand(R, D, seed=4, dtype=dt)
    y = ops.layer_norm(x, w, b, 1e-6)
    assert type(y.grad_fn).__name__.startswith("CppFunction") or "LayerNorm" in type(y.grad_fn).__name__
    _norm_check(x.detach(), w.detach(), b.detach(), dy, y.detach(), *torch.autograd.grad(y, (x, w, b), dy), 1e-6)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_layer_norm_strides_and_alignment(dtype):
    """Rows inside a wider buffer at every start, weights off the 16-byte boundary, a transposed upstream gradient; neighbours are NaN."""
    from torchllmtuner_b200 import ops
    dt = TYPES[dtype]
    for D in (128, 131):
        for start in range(0, 9):
            base = torch.full((50, D + 24), float("nan"), device=DEV, dtype=dt)
            base[:, start:start + D] = _rand(50, D, seed=start, dtype=dt)
            x = base[:, start:start + D].detach().requires_grad_()
            wb = _rand(2 * D + 8, seed=2, dtype=dt, mean=1, std=0.1)
            w, b = wb[start:start + D].detach().requires_grad_(), wb[D + 3:2 * D + 3].detach().requires_grad_()
            dy = _rand(D, 50, seed=4, dtype=dt).t()
            y = ops.layer_norm(x, w, b, 1e-5)
            _norm_check(x.detach(), w.detach(), b.detach(), dy, y.detach(), *torch.autograd.grad(y, (x, w, b), dy), 1e-5)


def test_layer_norm_constant_and_special_rows():
    from torchllmtuner_b200 import ops
    x = _rand(6, 256, seed=1)
    x[0] = 3.0                                             # no variance: the bias alone
    x[1, 5] = float("inf")
    x[2, 7] = float("nan")
    w, b = _rand(256, seed=2), _rand(256, seed=3)
    y = ops.layer_norm(x, w, b, 1e-6)
    assert torch.equal(y[0], b) and y[1].isnan().any() and y[2].isnan().all() and torch.isfinite(y[3:]).all()
    e = torch.empty(0, 256, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    w.requires_grad_()
    g = torch.autograd.grad(ops.layer_norm(e, w, b, 1e-6).sum(), (e, w))
    assert g[0].shape == (0, 256) and g[1].abs().max() == 0


# ---------------------------------------------------------------------------------------------------------- rotation
def _tables(T, P, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ang = torch.rand(T, P, generator=g, device=DEV, dtype=torch.float64) * 2 * math.pi
    return ang.cos().float(), ang.sin().float()


def _turn64(x, cos, sin, layout, off, sign=1.0):
    """Rotated heads and the sum of the terms' absolute values."""
    P = cos.shape[1]
    c, s = cos.double()[:, None], sign * sin.double()[:, None]
    first = torch.arange(P, device=x.device) + off if layout == "half" else torch.arange(P, device=x.device) * 2 + off
    second = first + (P if layout == "half" else 1)
    y, size = x.clone(), x.abs().clone()
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first], size[..., second] = a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs()
    return y, size


ROTARY = [(1, 1, 2, 1, 0), (5, 3, 64, 32, 0), (77, 16, 128, 32, 64), (300, 20, 72, 36, 0), (9, 5, 80, 16, 8), (33, 2, 256, 32, 0), (17, 7, 66, 33, 0), (4, 40, 50, 9, 31),
          (13, 64, 192, 64, 64), (6, 1, 96, 48, 0), (3, 300, 128, 64, 0)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,d,P,off", ROTARY)
def test_rope(T, H, d, P, off, layout, dtype):
    from torchllmtuner_b200 import ops
    dt = TYPES[dtype]
    cos, sin = _tables(T, P)
    x, dy = _rand(T, H, d, seed=1, dtype=dt).requires_grad_(), _rand(T, H, d, seed=2, dtype=dt)
    for inverse in (False, True):
        y = ops.rope(x, cos, sin, layout=layout, offset=off, inverse=inverse)
        sign = -1.0 if inverse else 1.0
        ref, size = _turn64(x.detach().double(), cos, sin, layout, off, sign)
        _near(y.detach(), ref, _u(dt) * ref.abs() + 4 * E32 * size, "y")
        keep = torch.ones(d, dtype=torch.bool, device=DEV)
        keep[off:off + 2 * P] = False
        assert torch.equal(y.detach()[..., keep], x.detach()[..., keep])
        dx, = torch.autograd.grad(y, x, dy)
        ref, size = _turn64(dy.double(), cos, sin, layout, off, -sign)
        _near(dx, ref, _u(dt) * ref.abs() + 4 * E32 * size, "dx")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_strides(layout):
    """Heads of a packed projection, heads-first memory, an odd start, tables of wider rows, a 2-D operand, a transposed upstream gradient."""
    from torchllmtuner_b200 import ops
    T, H, d, P, off = 41, 6, 64, 16, 32
    wide_c, wide_s = _tables(T, 2 * P + 3)
    cos, sin = wide_c[:, 1:1 + P], wide_s[:, 1:1 + P]
    views = {"packed": _rand(T, 3 * H, d, seed=1)[:, H:2 * H], "heads first": _rand(H, T, d, seed=2).transpose(0, 1),
             "odd start": _rand(T, H, d + 9, seed=3)[..., 5:5 + d], "channels strided": _rand(T, H, 2 * d, seed=4)[..., ::2],
             "one head for all": _rand(T, 1, d, seed=5).expand(T, H, d)}
    dy = _rand(d, H, T, seed=6).permute(2, 1, 0)
    for name, x in views.items():
        x = x.detach().requires_grad_()
        y = ops.rope(x, cos, sin, layout=layout, offset=off)
        ref, size = _turn64(x.detach().double(), cos, sin, layout, off)
        _near(y.detach(), ref, _u(x.dtype) * ref.abs() + 4 * E32 * size, name)
        dx, = torch.autograd.grad(y, x, dy)
        ref, size = _turn64(dy.double(), cos, sin, layout, off, -1.0)
        _near(dx, ref, _u(x.dtype) * ref.abs() + 4 * E32 * size, name)
    x = _rand(T, d, seed=7)
    assert torch.equal(ops.rope(x, cos, sin, layout=layout, offset=off), ops.rope(x[:, None], cos, sin, layout=layout, offset=off)[:, 0])
    x = _rand(T, 2, H, d, seed=8)
    assert torch.equal(ops.rope(x, cos, sin, layout=layout, offset=off).flatten(1, 2), ops.rope(x.flatten(1, 2), cos, sin, layout=layout, offset=off))
    assert ops.rope(x[:0], cos[:0], sin[:0], layout=layout, offset=off).shape == (0, 2, H, d)


def _head_norm64(x, w, eps):
    """x / rms(x) * w in 64 bits and the reciprocal of the rms."""
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return x * r * w, r


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("mode", ["weight", "zero_centered", "unit", "unit_q", "weight_k", "none"])
@pytest.mark.parametrize("T,H,K,d,P,off", [(1, 1, 1, 64, 32, 0), (77, 16, 1, 128, 32, 64), (300, 8, 2, 256, 32, 0), (50, 5, 5, 72, 36, 0), (9, 3, 2, 96, 8, 16),
                                           (21, 4, 1, 66, 33, 0), (200, 12, 4, 40, 20, 0), (3, 2, 1, 520, 100, 7), (1000, 4, 4, 64, 16, 0)])
def test_qk_norm_rope_forms(T, H, K, d, P, off, mode, layout, dtype):
    from torchllmtuner_b200 import ops
    dt, eps = TYPES[dtype], 1e-6
    cos, sin = _tables(T, P)
    q, k = _rand(T, H, d, seed=1, dtype=dt).requires_grad_(), _rand(T, K, d, seed=2, dtype=dt).requires_grad_()
    dq, dk = _rand(T, H, d, seed=3, dtype=dt), _rand(T, K, d, seed=4, dtype=dt)
    zero = mode == "zero_centered"
    qw = _rand(d, seed=5, dtype=dt, std=0.1, mean=0.0 if zero else 1.0).requires_grad_() if mode in ("weight", "zero_centered") else None
    kw = _rand(d, seed=6, dtype=dt, std=0.1, mean=0.0 if zero else 1.0).requires_grad_() if mode in ("weight", "zero_centered", "unit_q", "weight_k") else None
    norm = {"none": False, "weight_k": None}.get(mode, True)
    yq, yk = ops.qk_norm_rope(q, k, qw, kw, cos, sin, eps, layout=layout, offset=off, norm=norm, zero_centered=zero)
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    grads = dict(zip([n for n, t in zip(("q", "k", "qw", "kw"), (q, k, qw, kw)) if t is not None], torch.autograd.grad((yq, yk), leaves, (dq, dk))))
    u = _u(dt)
    for name, x, y, dy, w in (("q", q, yq, dq, qw), ("k", k, yk, dk, kw)):
        X, G = x.detach().double(), dy.double()
        normed = norm is True or (norm is None and w is not None)
        W = (w.detach().double() + (1.0 if zero else 0.0)) if w is not None else torch.ones(d, device=DEV, dtype=torch.float64)
        n, r = _head_norm64(X, W, eps) if normed else (X, None)
        ref, _ = _turn64(n, cos, sin, layout, off)
        size = _turn64(n.abs(), cos.abs(), -sin.abs(), layout, off)[1]
        _near(y.detach(), ref, u * ref.abs() + 64 * E32 * size, f"{name} forward")
        back, bsize = _turn64(G, cos, sin, layout, off, -1.0)
        if not normed:
            _near(grads[name], back, u * back.abs() + 4 * E32 * bsize, f"d{name}")
            continue
        g, gs = back * W, bsize * W.abs()
        ref = r * (g - X * r * r * (g * X).mean(-1, keepdim=True))
        _near(grads[name], ref, u * ref.abs() + 64 * E32 * r * (gs + X.abs() * r * r * (gs * X.abs()).mean(-1, keepdim=True)), f"d{name}")
        if w is not None:
            dw = (back * X * r).sum((0, 1))
            _near(grads[name + "w"], dw, u * dw.abs() + (64 + T * x.shape[1] / 8) * E32 * (bsize * X.abs() * r).sum((0, 1)), f"d{name}w")


def test_qk_norm_rope_views_beside_gates():
    """Queries interleaved with their gates, keys of a packed projection, tables with doubled columns: what the gated attention hands over."""
    from torchllmtuner_b200 import ops
    T, H, K, d, P = 130, 8, 2, 128, 16
    qg, kv = _rand(T, H, 2 * d, seed=1), _rand(T, 2 * K, d, seed=2)
    cos, sin = _tables(T, P)
    cos2, sin2 = torch.cat((cos, cos), -1), torch.cat((sin, sin), -1)
    qw, kw = _rand(d, seed=3, std=0.1), _rand(d, seed=4, std=0.1)
    kind = dict(norm=True, zero_centered=True)
    a = ops.qk_norm_rope(qg[..., :d], kv[:, :K], qw, kw, cos2[:, :P], sin2[:, :P], 1e-6, **kind)
    b = ops.qk_norm_rope(qg[..., :d].contiguous(), kv[:, :K].contiguous(), qw, kw, cos, sin, 1e-6, **kind)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_qk_norm_rope_operands_have_a_node_each():
    from torchllmtuner_b200 import ops
    T, d = 20, 64
    cos, sin = _tables(T, 16)
    for norm in (True, False):
        q, k, w = _rand(T, 4, d, seed=1).requires_grad_(), _rand(T, 2, d, seed=2).requires_grad_(), _rand(d, seed=3).requires_grad_()
        yq, yk = ops.qk_norm_rope(q, k, w if norm else None, w if norm else None, cos, sin, 1e-6, norm=norm)
        yq.sum().backward()
        assert q.grad is not None and k.grad is None
        yk.sum().backward()
        assert k.grad is not None


# ------------------------------------------------------------------------------------------------------------ tables
SCALINGS = [{"rope_type": "linear", "factor": 8.0}, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
            {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0}]


@pytest.mark.parametrize("scaling", SCALINGS, ids=lambda s: s["rope_type"])
@pytest.mark.parametrize("T,d", [(1, 2), (7, 6), (700, 64), (1000, 128), (33, 72), (5, 512)])
def test_scaled_rope_tables(T, d, scaling):
    from torchllmtuner_b200 import ops
    from torchllmtuner_b200.ops import reference as ref
    g = torch.Generator(device=DEV).manual_seed(T)
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=DEV)
    pos[0] = 0
    inv, factor = ref.scaled_frequencies(d, 1e6, scaling)
    ang = pos.double()[:, None] * torch.tensor(inv, dtype=torch.float64, device=DEV)
    for p in (pos, pos.int(), torch.stack((pos, pos), 1)[:, 0]):
        cos, sin = ops.rope_tables(p, d, 1e6, scaling=scaling)
        # the reduced angle (at most pi) and the function's value are each rounded to fp32, and the factor's product
        bound = factor * (math.pi + 4) * E32 + 2.0 ** -50 * ang
        _near(cos, ang.cos() * factor, bound, "cos")
        _near(sin, ang.sin() * factor, bound, "sin")
    assert ops.rope_tables(pos[:0], d, 1e6, scaling=scaling)[0].shape == (0, d // 2)


# --------------------------------------------------------------------------- derivatives, transforms, streams, graphs
def _cases():
    from torchllmtuner_b200 import ops
    T, d = 6, 64
    cos, sin = _tables(T, 16)
    return {
        "linear_act": (lambda x, w, b: ops.linear_act(x, w, b, activation="gelu_tanh"), (_rand(T, d, seed=1), _rand(24, d, seed=2, std=0.1), _rand(24, seed=3))),
        "layer_norm": (lambda x, w, b: ops.layer_norm(x, w, b, 1e-6), (_rand(T, d, seed=1), _rand(d, seed=2), _rand(d, seed=3))),
        "rope": (lambda x: ops.rope(x, cos, sin, offset=8), (_rand(T, 3, d, seed=1),)),
        "qk": (lambda q, k, w: torch.cat(ops.qk_norm_rope(q, k, w, w, cos, sin, 1e-6, norm=True, zero_centered=True), 1),
               (_rand(T, 3, d, seed=1), _rand(T, 2, d, seed=2), _rand(d, seed=3, std=0.1))),
    }


@pytest.mark.parametrize("name", ["linear_act", "layer_norm", "rope", "qk"])
def test_second_derivatives_and_batched_gradients(name):
    fn, args = _cases()[name]
    args = [a.clone().requires_grad_() for a in args]
    y = fn(*args)
    dy = _rand(*y.shape, seed=9).requires_grad_()
    first = torch.autograd.grad(y, args, dy, create_graph=True)
    plain = torch.autograd.grad(fn(*args), args, dy)
    for a, b in zip(first, plain):
        assert ((a - b).float().norm() <= 2e-2 * b.float().norm()), name
    total = sum((g.float() ** 2).sum() for g in first)
    for g in torch.autograd.grad(total, [dy, *args], allow_unused=True):      # a bias behind the norm has no second derivative
        assert g is None or torch.isfinite(g).all()
    y = fn(*args)
    batch = torch.stack([_rand(*y.shape, seed=s) for s in (1, 2)])
    got = torch.autograd.grad(y, args, batch, is_grads_batched=True, retain_graph=True)
    for i in range(2):
        for a, b in zip(got, torch.autograd.grad(y, args, batch[i], retain_graph=True)):
            assert (a[i] - b).float().norm() <= 2e-2 * b.float().norm()


@pytest.mark.parametrize("name", ["linear_act", "layer_norm", "rope", "qk"])
def test_gradients_against_differences(name):
    """The directional derivative along the gradients' own direction, from outputs in 64 bits of slightly moved fp32 inputs."""
    fn, args = _cases()[name]
    if name != "linear_act":                               # bf16 alone on the device: its kernel is compared with the formula above
        args = tuple(a.float() for a in args)
    args = [a.clone().requires_grad_() for a in args]
    y = fn(*args)
    dy = _rand(*y.shape, seed=9, dtype=y.dtype)
    grads = torch.autograd.grad(y, args, dy)
    norm = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    step = 2.0 ** -6 if name != "linear_act" else 2.0 ** -2
    with torch.no_grad():
        up = fn(*(a + step * g / norm for a, g in zip(args, grads))).double()
        down = fn(*(a - step * g / norm for a, g in zip(args, grads))).double()
    slope = ((up - down) * dy.double()).sum().item() / (2 * step)
    # second-order terms cancel in the symmetric difference; third-order ones are of the order of step^2; bf16 outputs add their rounding
    assert abs(slope - norm) <= (0.01 if name != "linear_act" else 0.08) * norm, (slope, norm)


@pytest.mark.parametrize("name", ["linear_act", "layer_norm", "rope", "qk"])
def test_transforms_and_tracing(name):
    fn, args = _cases()[name]
    y = fn(*args)
    stacked = [torch.stack((a, a * 0.5)) for a in args]
    out = torch.func.vmap(fn)(*stacked)
    assert (out[0] - y).float().norm() <= 1e-2 * y.float().norm()
    traced = torch.jit.trace(fn, tuple(args), check_trace=False)
    other = [a * 0.5 for a in args]
    ref = fn(*other)
    assert (traced(*other) - ref).float().norm() <= 1e-2 * ref.float().norm()


@pytest.mark.parametrize("name", ["linear_act", "layer_norm", "rope", "qk"])
def test_other_streams_and_captured_graphs(name):
    """The same bits on a side stream, from a captured and replayed forward + backward with new inputs, and from two graphs that run at once."""
    fn, args = _cases()[name]

    def step(*a):
        leaves = [t.detach().requires_grad_() for t in a]
        y = fn(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, torch.ones_like(y)))
    want = step(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = step(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        static = [a.clone() for a in args]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*static)
        graphs.append((static, graph, outs))
    other = [a * 0.5 for a in args]
    want2 = step(*other)
    for static, src in ((graphs[0][0], args), (graphs[1][0], other)):
        for s, a in zip(static, src):
            s.copy_(a)
    torch.cuda.synchronize()
    for _ in range(3):
        graphs[0][1].replay()
        with torch.cuda.stream(side):
            graphs[1][1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][2], want))
    assert all(torch.equal(a, b) for a, b in zip(graphs[1][2], want2))


def test_repeated_calls_give_the_same_bits():
    from torchllmtuner_b200 import ops
    x, w, b = _rand(3000, 264, seed=1).requires_grad_(), _rand(136, 264, seed=2, std=0.1).requires_grad_(), _rand(136, seed=3).requires_grad_()
    lw, lb = _rand(264, seed=4).requires_grad_(), _rand(264, seed=5).requires_grad_()
    dy = _rand(3000, 136, seed=6)

    def step():
        y = ops.linear_act(ops.layer_norm(x, lw, lb, 1e-6), w, b, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b, lw, lb), dy))
    want = step()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_refusals_name_the_argument():
    """What the kernels cannot take is refused on the host, before a launch, with the argument's name."""
    from torchllmtuner_b200 import ops
    from torchllmtuner_b200.errors import ConfigError
    x, w, b = _rand(6, 64), _rand(8, 64), _rand(8)
    for bad in (lambda: ops.linear_act(x, _rand(8, 63)), lambda: ops.linear_act(x, w, _rand(7)), lambda: ops.linear_act(x, w, activation="tanh"),
                lambda: ops.linear_act(x, w.cpu()), lambda: ops.linear_act(x, w, b.cpu()), lambda: ops.linear_act(x, _rand(8, 64, 1)), lambda: ops.linear_act(x, None),
                lambda: ops.linear_act(x, w, residual=_rand(6, 8).cpu())):
        with pytest.raises(ConfigError):
            bad()
    n = _rand(64)
    for bad in (lambda: ops.layer_norm(x, n[:63], n, 1e-6), lambda: ops.layer_norm(x, n, n[:, None], 1e-6), lambda: ops.layer_norm(x, n.cpu(), n, 1e-6),
                lambda: ops.layer_norm(x, n, None, 1e-6)):
        with pytest.raises(ConfigError):
            bad()
    cos, sin = _tables(6, 8)
    h = _rand(6, 2, 32)
    for bad in (lambda: ops.rope(h, cos, sin, offset=17), lambda: ops.rope(h, cos, sin, offset=-1), lambda: ops.rope(h, cos[:5], sin[:5]),
                lambda: ops.rope(h, cos, sin[:, :4]), lambda: ops.rope(h, cos, sin, layout="pairs"), lambda: ops.rope(h, cos.cpu(), sin.cpu()),
                lambda: ops.qk_norm_rope(h, h[..., :16], None, None, cos, sin, 1e-6, norm=True),
                lambda: ops.qk_norm_rope(h, h, n, None, cos, sin, 1e-6, norm=True), lambda: ops.qk_norm_rope(h, h.float(), None, None, cos, sin, 1e-6, norm=True),
                lambda: ops.qk_norm_rope(h, h, None, None, cos, sin, 1e-6, norm=True, offset=17)):
        with pytest.raises(ConfigError):
            bad()
    pos = torch.arange(4, device=DEV)
    for bad in ({"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "yarn", "factor": 2.0}, {"rope_type": "linear", "factor": [2.0]}):
        with pytest.raises(ConfigError):
            ops.rope_tables(pos, 8, 1e4, scaling=bad)


def test_residual_broadcast_over_columns():
    from torchllmtuner_b200 import ops
    x, w, r = _rand(40, 64, seed=1), _rand(24, 64, seed=2, std=0.1), _rand(40, 1, seed=3).requires_grad_()
    y = ops.linear_act(x, w, residual=r)
    ref = x.double() @ w.double().t() + r.detach().double()
    _near(y.detach(), ref, _u(torch.bfloat16) * ref.abs() + 80 * E32 * (x.double().abs() @ w.double().abs().t() + r.detach().double().abs()), "y")
    dy = _rand(40, 24, seed=4)
    g, = torch.autograd.grad(y, r, dy)
    ref = dy.double().sum(1, keepdim=True)
    _near(g, ref, _u(torch.bfloat16) * ref.abs() + 32 * E32 * dy.double().abs().sum(1, keepdim=True), "dr")


# ------------------------------------------------------------------------------------------------------ a run of them
def _tower_block(kind):
    from torchllmtuner_b200.models import moonvit, qwen_vit
    cfg = dict(hidden_size=288, intermediate_size=520, num_heads=4)                      # heads of 72
    return (qwen_vit.QwenViTBlock(qwen_vit.QwenViTConfig(**cfg)) if kind == "qwen" else moonvit.MoonViTBlock(moonvit.MoonViTConfig(**cfg)))


@pytest.mark.parametrize("kind", ["qwen", "moon"])
def test_tower_block_against_its_fp32_statement(kind):
    """LayerNorm -> packed projection with bias -> rotation -> attention -> projection + residual -> LayerNorm -> two-layer GELU MLP + residual, as the
    towers call it, forward and every gradient. About 12 roundings to bf16 lie on a path forwards and as many again backwards, each off by at most
    half a step: 12 and 24 times 2^-8 in the 2-norm."""
    import copy

    from torchllmtuner_b200.ops import AttnMeta
    from torchllmtuner_b200.ops.cuda_ext import load
    torch.manual_seed(3)
    block = _tower_block(kind)
    with torch.no_grad():
        for name, p in block.named_parameters():
            p.copy_(1 + 0.1 * torch.randn(p.shape) if "norm" in name and name.endswith("weight") else torch.randn(p.shape) * (0.1 if p.dim() == 1 else p.shape[-1] ** -0.5))
    block = block.bfloat16()
    plain = copy.deepcopy(block).float()
    block = block.to(DEV)
    x = torch.randn(300, 288).bfloat16()
    dy = torch.randn(300, 288).bfloat16()
    ang = torch.rand(300, 36) * 6
    ang = torch.cat((ang, ang), -1) if kind == "qwen" else ang
    cuts = torch.tensor([0, 77, 300])

    def run(m, dev, dtype):
        leaf = x.to(dev, dtype).requires_grad_()
        y = m(leaf, ang.cos().to(dev), ang.sin().to(dev), AttnMeta.build(cuts, causal=False, device=dev if dev == DEV else None))
        names = [n for n, _ in m.named_parameters()]
        return {"y": y, **dict(zip(["x", *names], torch.autograd.grad(y, [leaf, *m.parameters()], dy.to(dev, dtype))))}
    before = load().launch_count()
    got = run(block, DEV, torch.bfloat16)
    assert load().launch_count() - before >= 20
    want = run(plain, "cpu", torch.float32)
    for name, ref in want.items():
        off = (got[name].detach().float().cpu() - ref.detach()).norm() / ref.detach().norm()
        # the key's bias shifts every score of a query alike: its gradient is zero but for rounding, and shares a tensor with the queries' and values'
        assert off <= (12 if name == "y" else 24) * 2.0 ** -8, (name, off.item())


def test_gated_attention_against_its_fp32_statement():
    """The gated attention of Qwen3.5: queries beside their gates, zero-centred norms and partial rotation in one pass; about 10 roundings each way."""
    import copy

    from torchllmtuner_b200.models.qwen3_5 import GatedFullAttention, Qwen35Config, Qwen35Context, mrope_tables
    from torchllmtuner_b200.ops import AttnMeta
    torch.manual_seed(4)
    cfg = Qwen35Config(hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64, num_experts=0)
    block = GatedFullAttention(cfg)
    with torch.no_grad():
        for p in block.parameters():
            p.copy_(torch.randn(p.shape) * (0.1 if p.dim() == 1 else p.shape[-1] ** -0.5))
    block = block.bfloat16()
    plain = copy.deepcopy(block).float()
    block = block.to(DEV)
    x, dy = torch.randn(150, 128).bfloat16(), torch.randn(150, 128).bfloat16()
    cuts = torch.tensor([0, 61, 150])
    pos = torch.cat((torch.arange(61), torch.arange(89)))

    def run(m, dev, dtype):
        cos, sin = mrope_tables(pos.to(dev), cfg.rotary_dim, cfg.rope_theta, cfg.mrope_section)
        ctx = Qwen35Context(cos, sin, AttnMeta.build(cuts, causal=True, device=dev if dev == DEV else None), positions=pos.to(dev))
        leaf = x.to(dev, dtype).requires_grad_()
        y = m(leaf, ctx)
        return {"y": y, **dict(zip(["x", *(n for n, _ in m.named_parameters())], torch.autograd.grad(y, [leaf, *m.parameters()], dy.to(dev, dtype))))}
    got, want = run(block, DEV, torch.bfloat16), run(plain, "cpu", torch.float32)
    for name, ref in want.items():
        off = (got[name].detach().float().cpu() - ref.detach()).norm() / ref.detach().norm()
        assert off <= (10 if name == "y" else 20) * 2.0 ** -8, (name, off.item())


def test_linear_act_with_more_rows_than_a_grid_of_16_bit_tiles():
    """2^24 + 300 rows: 131 075 tile rows of one narrow column. A row is 8 products of values that bf16 holds exactly, so z is off by fp32's rounding
    alone, 8 steps of 2^-24 of the sum of magnitudes, and y by one rounding to bf16 more; dW sums 2^24 rows of magnitude 1 and random sign."""
    from torchllmtuner_b200 import ops
    m = (1 << 24) + 300
    g = torch.Generator(DEV).manual_seed(5)
    x = torch.randint(-8, 9, (m, 8), device=DEV, generator=g).bfloat16() / 8
    w = (torch.randint(-8, 9, (8, 8), device=DEV, generator=g).bfloat16() / 8).requires_grad_()
    y = ops.linear_act(x, w, activation="relu")
    dw, = torch.autograd.grad(y, w, torch.ones_like(y))
    for rows in (slice(0, 600), slice(m // 2, m // 2 + 600), slice(m - 600, m)):
        want = (x[rows].double() @ w.detach().double().t()).relu()
        assert ((y[rows].double() - want).abs() <= want * 2.0 ** -8 + 8 * 8 * 2.0 ** -24).all()
    z = x.double() @ w.detach().double().t()
    want = (z > 0).double().t() @ x.double()
    # exact multiples of 1/8 up to 2^24: fp32 sums (in parts) are off by at most a few hundred half steps of their magnitude; one rounding to bf16
    assert ((dw.double() - want).abs() <= want.abs() * 2.0 ** -8 + x.double().abs().sum(0) * 2.0 ** -12).all()


def test_gelu_tanh_gradient_of_enormous_values():
    """act' is 1 and 0 far out, also where z^3 overflows fp32."""
    from torchllmtuner_b200 import ops
    z = torch.tensor([1e3, 1e10, 1e20, 3e38, -1e3, -1e10, -1e20, -3e38], device=DEV).bfloat16().unsqueeze(1)
    one = torch.zeros(8, 8, device=DEV, dtype=torch.bfloat16)
    one[:, 0] = 1
    x = torch.cat((z, torch.zeros(8, 7, device=DEV, dtype=torch.bfloat16)), 1).requires_grad_()
    for act in ("gelu_tanh", "gelu", "silu", "relu"):
        y = ops.linear_act(x, one, activation=act)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert (dx[:4, 0] == 8).all() and (dx[4:, 0] == 0).all(), (act, dx[:, 0])


@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear_act_gradient_into_an_owners_buffer(act):
    """A weight with `main_grad` gets its gradient there: written the first time, added the second, and None is returned for it; x and bias as ever."""
    from torchllmtuner_b200 import ops
    x, w, b = _rand(300, 200, seed=1), _rand(136, 200, seed=2, std=0.07), _rand(136, seed=3)
    dy = _rand(300, 136, seed=4)

    def grads(owned):
        leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]
        if owned:
            leaves[1].main_grad, leaves[1].main_grad_initialized = torch.full((136, 200), 7.0, device=DEV, dtype=torch.bfloat16), False
        out = []
        for _ in range(2):
            y = ops.linear_act(*leaves, activation=act)
            out.append(torch.autograd.grad(y, leaves, dy, allow_unused=True))
        return leaves, out
    _, plain = grads(False)
    leaves, owned = grads(True)
    assert owned[0][1] is None and owned[1][1] is None
    for i in (0, 2):
        for got in owned:
            assert torch.equal(got[i], plain[0][i])
    # the sum of two equal gradients, each product rounded once: the second launch adds to the rounded first
    want = 2 * plain[0][1].double()
    assert ((leaves[1].main_grad.double() - want).abs() <= want.abs() * 3 * 2.0 ** -8 + want.abs().max() * 2.0 ** -16).all()


def test_scaled_tables_under_another_default_device():
    """The frequencies are kept on the host whatever device new tensors go to; a residual that fits nothing is named on the device too."""
    from torchllmtuner_b200 import ops
    from torchllmtuner_b200.errors import ConfigError
    scaling = {"rope_type": "linear", "factor": 3.5}
    with torch.device(DEV):
        cos, sin = ops.rope_tables(torch.arange(50), 48, 5e4, scaling=scaling)
    ang = torch.arange(50, dtype=torch.float64)[:, None] * torch.tensor([5e4 ** (-2 * j / 48) / 3.5 for j in range(24)], dtype=torch.float64)
    assert (cos.cpu().double() - ang.cos()).abs().max() < 2.0 ** -22 and (sin.cpu().double() - ang.sin()).abs().max() < 2.0 ** -22
    with pytest.raises(ConfigError, match="residual"):
        ops.linear_act(_rand(4, 8), _rand(6, 8), residual=_rand(5, 6))


@pytest.mark.parametrize("start", [1, 2, 3, 8])
@pytest.mark.parametrize("M,K,N", [(37, 1, 9), (130, 63, 40), (600, 200, 71), (9, 520, 264)])
def test_linear_act_rows_between_foreign_values(M, K, N, start):
    """Operands as rows of buffers whose other values are NaN, on odd and even starts and pitches: none of those may reach a result."""
    def between(rows, cols, seed, std=1.0):
        buf = torch.full((rows, cols + 2 * start + seed), float("nan"), device=DEV, dtype=torch.bfloat16)
        buf[:, start:start + cols] = _rand(rows, cols, seed=seed, std=std)
        return buf[:, start:start + cols].detach()
    x, w, r, dy = between(M, K, 1), between(N, K, 2, K ** -0.5), between(M, N, 3), between(M, N, 4)
    b = _rand(N, seed=5)
    for act in (None, "gelu_tanh"):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        _linear_check(x, w, b, r, act, dy, _linear_run(*leaves, act, dy))


def test_saved_tensors_through_the_host():
    """Offloaded saved tensors come back dense, whatever strides went out: the gradients are the same bits."""
    from torchllmtuner_b200 import ops
    ang = torch.rand(90, 12, device=DEV) * 6
    cos, sin = ang.cos()[:, :10], ang.sin()[:, :10]

    def run():
        x = _rand(90, 71, seed=1)[:, :67].detach().requires_grad_()
        w, b = _rand(132, 67, seed=2, std=0.1).requires_grad_(), _rand(132, seed=3).requires_grad_()
        lw, lb, qw = (_rand(n, seed=i).requires_grad_() for i, n in ((4, 132), (5, 132), (6, 33)))
        h = ops.layer_norm(ops.linear_act(x, w, b, activation="gelu"), lw, lb, 1e-5)
        q, k = ops.qk_norm_rope(h.view(90, 4, 33)[:, :3], h.view(90, 4, 33)[:, 3:], qw, None, cos, sin, 1e-6, offset=5, norm=True)
        y = ops.linear_act(torch.cat((q, ops.rope(k, cos, sin, layout="interleaved", offset=1)), 1).flatten(1), w.t()[:, :132])
        return [y, *torch.autograd.grad(y, [x, w, b, lw, lb, qw], torch.ones_like(y))]
    plain = run()
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        moved = run()
    for i, (a, b) in enumerate(zip(plain, moved)):
        assert torch.isfinite(a).all() and torch.equal(a, b), i


@pytest.mark.parametrize("op", ["linear", "layer_norm", "rope", "qk"])
def test_offsets_past_32_bits(op):
    """Tensors of more than 2^31 elements: the last rows are those of the same call on the last rows alone, forward and backward."""
    from torchllmtuner_b200 import ops
    rows, tail = (1 << 31) // 4096 + 300, 200
    if op == "linear":
        x, w = _rand(rows, 64, seed=1), _rand(4096, 64, seed=2, std=0.125)
        run = lambda t: ops.linear_act(t, w, activation="silu")  # noqa: E731
    else:
        x = torch.empty(rows, 4096, device=DEV, dtype=torch.bfloat16).normal_()
        ang = torch.rand(rows, 32, device=DEV)
        lw, lb, qw = _rand(4096, seed=3), _rand(4096, seed=4), _rand(256, seed=5)
        part = lambda t, n: ang[-n:].cos() if t else ang[-n:].sin()  # noqa: E731
        run = {"layer_norm": lambda t: ops.layer_norm(t, lw, lb, 1e-5),
               "rope": lambda t: ops.rope(t.view(-1, 16, 256), part(1, len(t)), part(0, len(t)), layout="interleaved", offset=8).view(t.shape),
               "qk": lambda t: ops.qk_norm_rope(t.view(-1, 16, 256), t.view(-1, 16, 256)[:, :0], qw, None, part(1, len(t)), part(0, len(t)), 1e-6,
                                                norm=True)[0].reshape(t.shape)}[op]
    x.requires_grad_()
    y = run(x)
    assert y.numel() > 1 << 31
    dy = torch.empty_like(y).normal_()
    dx, = torch.autograd.grad(y, x, dy)
    x2 = x.detach()[-tail:].clone().requires_grad_()
    y2 = run(x2)
    dx2, = torch.autograd.grad(y2, x2, dy[-tail:].clone())
    for name, a, b in (("y", y[-tail:], y2), ("dx", dx[-tail:], dx2)):
        # other tiles add in another order: each side is off by half a step of bf16, and what is rounded before (z) once more
        assert torch.equal(a, b) if op != "linear" else (a.double() - b.double()).norm() <= 4 * 2.0 ** -8 * b.double().norm(), name
    del y, dy, dx
    torch.cuda.empty_cache()


def test_two_threads_on_their_own_streams():
    """Workspaces and cut tables belong to a call and a thread: two threads at once get the bits of one alone."""
    import threading

    from torchllmtuner_b200 import ops

    def work(seed):
        m, k, n = (300, 1200, 520) if seed else (700, 264, 136)
        x, w, b = _rand(m, k, seed=seed).requires_grad_(), _rand(n, k, seed=seed + 1, std=k ** -0.5).requires_grad_(), _rand(n, seed=seed + 2).requires_grad_()
        lw, lb = _rand(n, seed=seed + 3).requires_grad_(), _rand(n, seed=seed + 4).requires_grad_()
        y = ops.layer_norm(ops.linear_act(x, w, b, activation="gelu"), lw, lb, 1e-5)
        return [t.detach() for t in (y, *torch.autograd.grad(y, [x, w, b, lw, lb], _rand(m, n, seed=seed + 5)))]
    alone = [work(0), work(1)]
    got, faults = {}, []

    def repeat(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[seed] = [work(seed) for _ in range(20)]
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            faults.append(e)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=repeat, args=(s,)) for s in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not faults
    for seed in (0, 1):
        for run in got[seed]:
            assert all(torch.equal(a, b) for a, b in zip(run, alone[seed]))

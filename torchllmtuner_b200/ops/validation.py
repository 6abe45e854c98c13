"""Argument contracts of the kernel facade (reference: llmtuner/kernel/validation.py:1-133): shape, dtype, device and
alignment checks that turn a bad call into a `ConfigError` with the operand's name instead of a failed launch."""
from __future__ import annotations

import torch

from ..errors import ConfigError


def require_tensor(x, name: str, *, dims: int | None = None, dtype=None, device_type: str | None = None) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise ConfigError(f"{name} must be a tensor, got {type(x).__name__}")
    if dims is not None and x.dim() != dims:
        raise ConfigError(f"{name} must have {dims} dimensions, got shape {tuple(x.shape)}")
    if dtype is not None and x.dtype not in (dtype if isinstance(dtype, (tuple, list)) else (dtype,)):
        raise ConfigError(f"{name} must have dtype {dtype}, got {x.dtype}")
    if device_type is not None and x.device.type != device_type:
        raise ConfigError(f"{name} must live on {device_type}, got {x.device}")
    return x


def require_same_device(*named) -> None:
    devs = {t.device for _, t in named}
    if len(devs) > 1:
        raise ConfigError("operands on different devices: " + ", ".join(f"{n}={t.device}" for n, t in named))


def require_last_dim_contiguous(x: torch.Tensor, name: str, multiple: int = 8) -> None:
    """The tcgen05 / TMA paths need a unit inner stride, 16-byte aligned rows and a 16-byte aligned base."""
    if x.stride(-1) != 1:
        raise ConfigError(f"{name} must be contiguous in its last dimension")
    if x.dim() >= 2 and x.stride(-2) % multiple:
        raise ConfigError(f"{name}: row stride {x.stride(-2)} is not a multiple of {multiple} elements")
    if x.data_ptr() % 16:
        raise ConfigError(f"{name}: base address is not 16-byte aligned")


def validate_attention_inputs(q, k, v) -> None:
    """q [T, Hq, d], k [S, Hkv, d], v [S, Hkv, dv]; Hq a multiple of Hkv; on the device d and dv at most 256."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        require_tensor(t, n, dims=3)
    require_same_device(("q", q), ("k", k), ("v", v))
    if k.shape[:2] != v.shape[:2]:
        raise ConfigError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must agree in rows and heads")
    if q.shape[2] != k.shape[2] or q.shape[1] % k.shape[1]:
        raise ConfigError(f"q {tuple(q.shape)} is not compatible with k {tuple(k.shape)} (head_dim equal, Hq % Hkv == 0)")


def validate_rms_norm_inputs(x, weight) -> None:
    require_tensor(x, "x")
    require_tensor(weight, "weight", dims=1)
    if x.shape[-1] != weight.shape[0]:
        raise ConfigError(f"weight has {weight.shape[0]} elements, the normalised dimension has {x.shape[-1]}")


def validate_router_inputs(logits, k: int) -> None:
    require_tensor(logits, "logits", dims=2)
    if not (1 <= k <= logits.shape[1]):
        raise ConfigError(f"top-k {k} must be in [1, {logits.shape[1]}]")


def validate_layer_norm_inputs(x, weight, bias) -> None:
    require_tensor(x, "x")
    for n, t in (("weight", weight), ("bias", bias)):
        require_tensor(t, n, dims=1)
        if x.dim() == 0 or x.shape[-1] != t.shape[0]:
            raise ConfigError(f"{n} has {t.shape[0]} elements, x has shape {tuple(x.shape)}")
    require_same_device(("x", x), ("weight", weight), ("bias", bias))


def validate_rotary_inputs(x, cos, sin, layout: str, offset: int, name: str = "x") -> None:
    """x [T, ..., d]; cos, sin [T, P] with offset + 2 P <= d."""
    require_tensor(x, name)
    require_tensor(cos, "cos", dims=2)
    require_tensor(sin, "sin", dims=2)
    require_same_device((name, x), ("cos", cos), ("sin", sin))
    if layout not in ("half", "interleaved"):
        raise ConfigError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    if x.dim() < 2 or cos.shape != sin.shape or cos.shape[0] != x.shape[0]:
        raise ConfigError(f"{name} {tuple(x.shape)} needs cos and sin [{x.shape[0] if x.dim() else 0}, P], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    if offset < 0 or cos.shape[1] < 1 or offset + 2 * cos.shape[1] > x.shape[-1]:
        raise ConfigError(f"{2 * cos.shape[1]} rotated channels from {offset} on do not lie in a head of {x.shape[-1]}")


def validate_qk_inputs(q, k, q_weight, k_weight, cos, sin, layout: str, offset: int) -> None:
    validate_rotary_inputs(q, cos, sin, layout, offset, "q")
    validate_rotary_inputs(k, cos, sin, layout, offset, "k")
    if q.dim() != 3 or k.dim() != 3 or q.shape[2] != k.shape[2] or q.dtype != k.dtype:
        raise ConfigError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} must be [T, heads, d] of one head width and type")
    for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            require_tensor(w, n, dims=1)
            require_same_device(("q", q), (n, w))
            if w.shape[0] != q.shape[2]:
                raise ConfigError(f"{n} has {w.shape[0]} elements, a head has {q.shape[2]}")


def validate_linear_act_inputs(x, w, bias, activation, residual, activations) -> None:
    require_tensor(x, "x")
    require_tensor(w, "w", dims=2)
    if x.dim() == 0 or x.shape[-1] != w.shape[1]:
        raise ConfigError(f"x {tuple(x.shape)} and w {tuple(w.shape)} do not agree in their last dimension")
    if activation not in activations:
        raise ConfigError(f"activation must be one of {[a for a in activations if a]} or None, got {activation!r}")
    require_same_device(("x", x), ("w", w))
    if bias is not None:
        require_tensor(bias, "bias", dims=1)
        require_same_device(("x", x), ("bias", bias))
        if bias.shape[0] != w.shape[0]:
            raise ConfigError(f"bias has {bias.shape[0]} elements, w has {w.shape[0]} rows")
    if residual is not None:
        require_tensor(residual, "residual")
        require_same_device(("x", x), ("residual", residual))
        shape = (*x.shape[:-1], w.shape[0])
        try:
            torch.broadcast_shapes(residual.shape, shape)
        except RuntimeError:
            raise ConfigError(f"residual {tuple(residual.shape)} does not broadcast with the result {shape}") from None


ROPE_SCALINGS = ("linear", "llama3", "yarn")


def validate_rope_scaling(scaling, kinds=ROPE_SCALINGS) -> dict:
    """`scaling` itself where `rope_tables` has a form for it."""
    if not isinstance(scaling, dict) or scaling.get("rope_type") not in kinds:
        raise ConfigError(f"rotary scaling must be a dict with rope_type in {list(kinds)}, got {scaling!r}")
    need = {"linear": ("factor",), "llama3": ("factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"),
            "yarn": ("factor", "original_max_position_embeddings")}[scaling["rope_type"]]
    for key in need:
        v = scaling.get(key)
        if isinstance(v, bool) or not isinstance(v, (int, float)) or not v > 0:
            raise ConfigError(f"{scaling['rope_type']!r} rotary scaling needs a positive {key}, got {v!r}")
    if scaling["factor"] < 1:
        raise ConfigError(f"the rotary scaling factor must be at least 1, got {scaling['factor']!r}")
    if scaling["rope_type"] == "llama3" and not scaling["high_freq_factor"] > scaling["low_freq_factor"]:
        raise ConfigError("llama3 rotary scaling needs high_freq_factor > low_freq_factor")
    return scaling

"""Linear layers with an epilogue, LayerNorm and rotary positions without a GPU: statements against plain formulas and the transformers library,
refusals, and the models that call them."""
import json
import math

import pytest
import torch

from torchllmtuner_b200 import ops
from torchllmtuner_b200.errors import ConfigError, UnsupportedCombinationError
from torchllmtuner_b200.ops import reference as ref

YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192, "low_freq_factor": 1.0, "high_freq_factor": 4.0}
LINEAR = {"rope_type": "linear", "factor": 8.0}


# ---------------------------------------------------------------------------------------------------------- statements
def test_linear_act_statement():
    g = torch.Generator().manual_seed(0)
    x, w, b, r = (torch.randn(*s, generator=g) for s in ((3, 5, 7), (4, 7), (4,), (3, 5, 4)))
    F = torch.nn.functional
    z = F.linear(x, w, b)
    for name, f in ((None, lambda t: t), ("gelu", F.gelu), ("gelu_tanh", lambda t: F.gelu(t, approximate="tanh")), ("silu", F.silu), ("relu", F.relu)):
        assert torch.allclose(ops.linear_act(x, w, b, activation=name, residual=r), f(z) + r, atol=1e-6)
        assert torch.allclose(ops.linear_act(x, w, activation=name), f(F.linear(x, w)), atol=1e-6)
    assert torch.allclose(ops.linear_act(x, w, b, residual=r[0, 0]), z + r[0, 0], atol=1e-6)


def test_layer_norm_statement():
    x, w, b = torch.randn(3, 4, 10), torch.randn(10), torch.randn(10)
    assert torch.allclose(ops.layer_norm(x, w, b, 1e-5), torch.nn.functional.layer_norm(x, (10,), w, b, 1e-5), atol=1e-6)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,P,off", [(8, 4, 0), (10, 3, 2), (10, 3, 4), (6, 1, 5 - 1)])
def test_rope_statement_turns_pairs_as_complex_numbers(d, P, off, layout):
    ang = torch.rand(5, P, dtype=torch.float64) * 6
    cos, sin = ang.cos(), ang.sin()
    x = torch.randn(5, 3, d, dtype=torch.float64)
    y = ref.rope(x, cos, sin, layout=layout, offset=off).double()
    first = torch.arange(P) + off if layout == "half" else 2 * torch.arange(P) + off
    second = first + (P if layout == "half" else 1)
    z = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(ang), ang)[:, None]
    assert torch.allclose(y[..., first], z.real, atol=1e-6) and torch.allclose(y[..., second], z.imag, atol=1e-6)
    rest = [c for c in range(d) if c not in first.tolist() + second.tolist()]
    assert torch.equal(y[..., rest], x[..., rest])
    assert torch.allclose(ref.rope(y, cos, sin, layout=layout, offset=off, inverse=True), x, atol=1e-6)


def test_qk_norm_rope_statement():
    T, d = 6, 12
    cos, sin = (t(torch.rand(T, 4) * 6) for t in (torch.cos, torch.sin))
    q, k, qw, kw = torch.randn(T, 3, d), torch.randn(T, 2, d), torch.randn(d), torch.randn(d)
    unit = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    turn = lambda t: ops.rope(t, cos, sin, offset=2)  # noqa: E731
    for norm, zero, fq, fk in ((True, False, qw, kw), (True, True, 1 + qw, 1 + kw)):
        a, b = ops.qk_norm_rope(q, k, qw, kw, cos, sin, 1e-6, offset=2, norm=norm, zero_centered=zero)
        assert torch.allclose(a, turn(unit(q) * fq), atol=1e-6) and torch.allclose(b, turn(unit(k) * fk), atol=1e-6)
    a, b = ops.qk_norm_rope(q, k, None, kw, cos, sin, 1e-6, offset=2, norm=True)
    assert torch.allclose(a, turn(unit(q)), atol=1e-6) and torch.allclose(b, turn(unit(k) * kw), atol=1e-6)
    a, b = ops.qk_norm_rope(q, k, None, kw, cos, sin, 1e-6, offset=2)
    assert torch.equal(a, turn(q)) and torch.allclose(b, turn(unit(k) * kw), atol=1e-6)
    a, b = ops.qk_norm_rope(q, k, qw, kw, cos, sin, 1e-6, offset=2, norm=False)
    assert torch.equal(a, turn(q)) and torch.equal(b, turn(k))


@pytest.mark.parametrize("scaling", [YARN, {**YARN, "beta_fast": 16.0, "beta_slow": 2.0, "attention_factor": 1.5}, {**YARN, "truncate": False},
                                     {**YARN, "mscale": 1.0, "mscale_all_dim": 0.5}, LLAMA3, LINEAR])
@pytest.mark.parametrize("d,theta", [(128, 1e6), (64, 1e4)])
def test_scaled_frequencies_are_those_of_the_library(scaling, d, theta):
    T = pytest.importorskip("transformers")
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    cfg = T.Qwen3Config(hidden_size=4 * d, num_attention_heads=4, num_key_value_heads=2, head_dim=d, max_position_embeddings=131072,
                        rope_parameters={"rope_theta": theta, **scaling})
    want, gain = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    inv, factor = ref.scaled_frequencies(d, theta, scaling)
    got = torch.tensor(inv, dtype=torch.float64)
    # the library works in fp32: about ten roundings in a frequency and its mixing weight
    assert ((got - want.double()).abs() <= 2e-6 * got).all() and math.isclose(factor, gain, rel_tol=1e-6)


def test_scaled_tables_on_far_positions():
    pos = torch.tensor([0, 1, 131071, 10 ** 9])
    cos, sin = ops.rope_tables(pos, 8, 1e4, scaling=LINEAR)
    for i, p in enumerate(pos.tolist()):
        for j in range(4):
            a = p * 1e4 ** (-2 * j / 8) / 8.0
            assert abs(cos[i, j].item() - math.cos(a)) < 1e-6 and abs(sin[i, j].item() - math.sin(a)) < 1e-6
    assert all(torch.equal(a, b) for a, b in zip(ops.rope_tables(pos, 8, 1e4), ref.rope_tables(pos, 8, 1e4)))


# ------------------------------------------------------------------------------------------------------------ refusals
def test_linear_act_refusals():
    x, w = torch.randn(3, 8), torch.randn(4, 8)
    for bad in (lambda: ops.linear_act(x, torch.randn(4, 7)), lambda: ops.linear_act(x, w, torch.randn(5)), lambda: ops.linear_act(x, w, torch.randn(4, 1)),
                lambda: ops.linear_act(x, w, activation="tanh"), lambda: ops.linear_act(x, torch.randn(8)), lambda: ops.linear_act([1.0], w),
                lambda: ops.linear_act(torch.tensor(1.0), w), lambda: ops.linear_act(x, w, residual=1.0), lambda: ops.linear_act(x, w.to("meta"))):
        with pytest.raises(ConfigError):
            bad()


def test_layer_norm_refusals():
    x = torch.randn(3, 8)
    for w, b in ((torch.ones(7), torch.ones(8)), (torch.ones(8), torch.ones(7)), (torch.ones(8, 1), torch.ones(8)), (None, torch.ones(8)),
                 (torch.ones(8), torch.ones(8, device="meta"))):
        with pytest.raises(ConfigError):
            ops.layer_norm(x, w, b, 1e-6)


def test_rotary_refusals():
    x, cos, sin = torch.randn(5, 2, 8), torch.ones(5, 3), torch.ones(5, 3)
    for bad in (lambda: ops.rope(x, cos, sin, offset=3), lambda: ops.rope(x, cos, sin, offset=-1), lambda: ops.rope(x, cos[:4], sin[:4]),
                lambda: ops.rope(x, cos, sin[:, :2]), lambda: ops.rope(x, cos, sin, layout="pairs"), lambda: ops.rope(x[0, 0], cos, sin),
                lambda: ops.rope(x, cos[:, :0], sin[:, :0]), lambda: ops.rope(x, torch.ones(5, 5), torch.ones(5, 5)),
                lambda: ops.qk_norm_rope(x, x[:, :1, :7], None, None, cos, sin, 1e-6), lambda: ops.qk_norm_rope(x, x.double(), None, None, cos, sin, 1e-6),
                lambda: ops.qk_norm_rope(x, x, torch.ones(7), None, cos, sin, 1e-6, norm=True),
                lambda: ops.qk_norm_rope(x[0], x[0], None, None, cos[:2], sin[:2], 1e-6)):
        with pytest.raises(ConfigError):
            bad()


def test_scaling_refusals():
    pos = torch.arange(4)
    for bad in ({"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "yarn", "factor": 2.0}, {"rope_type": "linear"}, {"rope_type": "linear", "factor": 0.5},
                {"rope_type": "linear", "factor": "2"}, {**LLAMA3, "high_freq_factor": 1.0}, "yarn"):
        with pytest.raises(ConfigError):
            ops.rope_tables(pos, 8, 1e4, scaling=bad)
    for args in ((pos[None], 8, 1e4), (pos, 7, 1e4), (pos, 8, 1.0)):
        with pytest.raises(ConfigError):
            ops.rope_tables(*args, scaling=LINEAR)


# -------------------------------------------------------------------------------------------------------------- models
def test_qwen3_reads_scaled_rotary_settings(tmp_path):
    from torchllmtuner_b200.config.model_config import ModelConfig
    from torchllmtuner_b200.models.qwen3 import Qwen3Config
    from torchllmtuner_b200.models.registry import build_registered_model
    from torchllmtuner_b200.models.state import Qwen3StateFormat
    from torchllmtuner_b200.ops import AttnMeta
    hf = dict(model_type="qwen3", vocab_size=32, hidden_size=32, intermediate_size=64, num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=1,
              head_dim=16, rms_norm_eps=1e-6, hidden_act="silu", rope_theta=1e6, max_position_embeddings=131072)
    for key, value in (("rope_scaling", {**YARN, "type": "yarn"}), ("rope_parameters", {"rope_theta": 1e6, **YARN})):
        (tmp_path / "config.json").write_text(json.dumps({**hf, key: value}))
        model = build_registered_model(ModelConfig(model_name_or_path=str(tmp_path)))
        assert model.config.rope_scaling == YARN and model.config.rope_theta == 1e6
        pos = torch.arange(40000, 40008)
        ctx = model.build_context(pos, AttnMeta.build(torch.tensor([0, 8]), causal=True))
        want = ref.rope_tables(pos, 16, 1e6, scaling=YARN)
        assert torch.equal(ctx.cos, want[0]) and torch.equal(ctx.sin, want[1])
        back = Qwen3StateFormat().hf_config(model.config)
        assert Qwen3StateFormat().arch_from_hf({**back, "hidden_act": "silu"})["rope_scaling"] == YARN
    assert Qwen3Config(rope_scaling={"rope_type": "default"}).rope_scaling is None
    with pytest.raises(ConfigError):
        Qwen3Config(rope_scaling={"rope_type": "yarn", "factor": 2.0})
    (tmp_path / "config.json").write_text(json.dumps({**hf, "rope_scaling": {"rope_type": "longrope", "factor": 2.0}}))
    with pytest.raises(UnsupportedCombinationError, match="longrope"):
        build_registered_model(ModelConfig(model_name_or_path=str(tmp_path)))


def test_families_with_tables_of_their_own_refuse_scaling():
    from torchllmtuner_b200.models.deepseek_v4 import DeepseekV4Config
    from torchllmtuner_b200.models.kimi_k3 import KimiConfig
    from torchllmtuner_b200.models.qwen3_5 import Qwen35Config
    for cls in (Qwen35Config, DeepseekV4Config, KimiConfig):
        with pytest.raises(UnsupportedCombinationError):
            cls(rope_scaling=LINEAR, num_experts=4, num_experts_per_tok=2)


def test_scaled_qwen3_logits_are_those_of_the_library():
    T = pytest.importorskip("transformers")
    from torchllmtuner_b200.models.qwen3 import Qwen3Config, Qwen3ForCausalLM
    from torchllmtuner_b200.ops import AttnMeta
    sizes = dict(vocab_size=48, hidden_size=32, intermediate_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=16)
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}
    torch.manual_seed(0)
    theirs = T.Qwen3ForCausalLM(T.Qwen3Config(**sizes, tie_word_embeddings=False, max_position_embeddings=256,
                                              rope_parameters={"rope_theta": 1e4, **scaling})).eval()
    ours = Qwen3ForCausalLM(Qwen3Config(**sizes, rope_theta=1e4, rope_scaling=scaling))
    ours.load_state_dict(theirs.state_dict(), strict=False)
    tok = torch.randint(0, 48, (200,))
    with torch.no_grad():
        got = ours(tok, ours.build_context(torch.arange(200), AttnMeta.build(torch.tensor([0, 200]), causal=True)))
        want = theirs(input_ids=tok[None], use_cache=False).logits[0]
    assert torch.allclose(got.float(), want, atol=2e-5), (got - want).abs().max()


def test_refusals_name_what_does_not_fit():
    from torchllmtuner_b200.errors import ConfigError
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ConfigError, match="residual"):
        ops.linear_act(x, w, residual=torch.zeros(5, 6))
    with pytest.raises(ConfigError, match="positions"):
        ops.rope_tables([0, 1, 2], 8, 1e4, scaling={"rope_type": "linear", "factor": 2.0})
    with pytest.raises(ConfigError, match="positions"):
        ops.rope_tables(torch.zeros(2, 3, dtype=torch.int64), 8, 1e4, scaling={"rope_type": "linear", "factor": 2.0})

"""Rotary settings of Hugging Face configs, against transformers' own models; no device is needed."""

import pytest
import torch

from saelens_b200.models.lm.hf import hooked_lm_from_hf

transformers = pytest.importorskip("transformers")


def converted(family, rope, **kw):
    torch.manual_seed(0)
    cfg = getattr(transformers, family + "Config")(
        vocab_size=300, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
        num_key_value_heads=2, head_dim=16, max_position_embeddings=64, rope_parameters={"rope_theta": 10000.0, **rope}, **kw)
    return getattr(transformers, family + "ForCausalLM")(cfg).eval()


def check_same_logits(hf, length=60):
    toks = torch.randint(0, 300, (2, length))
    with torch.no_grad():
        # fp32 on both sides, sums in another order: far below what a wrong angle moves (1e-3 and more)
        assert torch.allclose(hooked_lm_from_hf(hf).eval()(toks), hf(input_ids=toks).logits, atol=1e-5, rtol=1e-5)


@pytest.mark.parametrize("family", ["Llama", "Mistral", "Qwen2", "Gemma2"])
@pytest.mark.parametrize("where", ["rope_parameters", "config"])
def test_a_partial_factor_that_the_type_does_not_read(family, where):
    part = {"partial_rotary_factor": 0.5}
    hf = converted(family, {"rope_type": "default", **(part if where == "rope_parameters" else {})},
                   **(part if where == "config" else {}))
    check_same_logits(hf)


YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}


@pytest.mark.parametrize("more", [{"truncate": False}, {"truncate": True}, {"truncate": False, "beta_fast": 8.0, "beta_slow": 2.0}])
def test_yarn_between_pairs(more):
    check_same_logits(converted("Llama", {**YARN, **more}))


def tiny_config(**kw):
    from saelens_b200.models.lm import preset_config

    return preset_config("llama-3-8b", **{**dict(n_layers=1, d_model=64, n_heads=4, n_key_value_heads=2, d_mlp=128, d_vocab=300,
                                                 n_ctx=64, d_head=16, dtype="float32"), **kw})


@pytest.mark.parametrize("scaling,match", [
    ({"rope_type": "linear", "factor": 0.5}, "factor"), ({"rope_type": "linear"}, "factor"),
    ({"type": "yarn", "factor": 4.0}, "original_max"), ({"rope_type": "other", "factor": 2.0}, "unknown"),
    ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0, "original_max_position_embeddings": 32}, "high_freq"),
])
def test_a_scaling_is_checked_when_the_config_is_made(scaling, match):
    with pytest.raises(ValueError, match=match):
        tiny_config(rope_scaling=scaling)


def test_scalings_that_are_not_used_or_need_no_length():
    for kw in ({"rope_scaling": {"rope_type": "default"}}, {"rope_scaling": {}}, {"rope_scaling": {"rope_type": "dynamic", "factor": 2.0}},
               {"positional": "standard", "rope_scaling": {"rope_type": "other"}}):
        cfg = tiny_config(**kw)
        assert cfg.rope_scaling == kw["rope_scaling"]
    from saelens_b200.models.lm import HookedLM

    torch.manual_seed(0)
    lm = HookedLM(tiny_config(rope_scaling={"rope_type": "dynamic", "factor": 2.0}))
    near, far = lm._rotary(64), lm._rotary(100)
    assert torch.equal(near.freq, lm._rotary(10).freq) and (far.freq <= near.freq).all() and far.freq[-1] < near.freq[-1]


def test_a_scaling_that_is_not_computed_is_refused():
    """It was taken as no scaling at all."""
    hf = converted("Llama", {"rope_type": "longrope", "factor": 2.0, "short_factor": [1.0] * 8, "long_factor": [2.0] * 8,
                             "original_max_position_embeddings": 32})
    with pytest.raises(ValueError, match="longrope"):
        hooked_lm_from_hf(hf)


@pytest.mark.parametrize("rope", [
    {"rope_type": "default"}, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "yarn", "factor": 4.0}, YARN,
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0},
    {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 32},
])
@pytest.mark.parametrize("family", ["Llama", "Qwen2", "Gemma2"])
def test_scalings_that_are_computed(family, rope):
    check_same_logits(converted(family, rope), 100 if rope["rope_type"] == "dynamic" else 60)

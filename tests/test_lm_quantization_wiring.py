"""8-bit weights of the producer LM as a program reaches them; no device is needed."""

import pytest
import torch

from saelens_b200.models.lm import HookedLM, preset_config

TINY = dict(n_layers=2, d_model=128, n_heads=4, n_key_value_heads=2, d_mlp=192, d_vocab=300, n_ctx=64, d_head=32, dtype="float32")


def test_a_shared_config_stays_as_it_is():
    cfg = preset_config("llama-3-8b", **TINY)
    lm = HookedLM(cfg).quantize_weights()
    assert lm.cfg.weight_quantization == "fp8" and cfg.weight_quantization is None
    assert HookedLM(cfg).blocks[0].attn.qkv_fp8 is None

"""Refusals of the block operators and the frequencies of rotary positions; no device is needed."""

import math

import pytest
import torch

from saelens_b200 import ops

E4 = torch.float8_e4m3fn


def fp8_args():
    return {"x": torch.zeros(4, 256), "weight": torch.zeros(384, 256).to(E4), "scale": torch.zeros(3, 2)}


@pytest.mark.parametrize("change,match", [
    ({"x": torch.zeros(4, 256, dtype=torch.float64)}, "x must be"),
    ({"x": torch.zeros(4, 0)}, "x must be"),
    ({"x": torch.zeros(4, 255)}, "weight must be"),
    ({"weight": torch.zeros(384, 256)}, "weight must be"),
    ({"weight": torch.zeros(384 * 256).to(E4)}, "weight must be"),
    ({"weight": torch.zeros(384, 272).to(E4)[:, 1:257]}, "16 bytes"),
    ({"weight": torch.zeros(384, 264).to(E4)[:, :256]}, "16 bytes"),
    ({"weight": torch.zeros(256, 384).to(E4).t()}, "contiguous"),
    ({"scale": torch.zeros(2, 2)}, "scales"),
    ({"scale": torch.zeros(3, 2, dtype=torch.float64)}, "scales"),
    ({"bias": torch.zeros(383)}, "bias"),
    ({"bias": torch.zeros(384, dtype=torch.bfloat16)}, "bias"),
    ({}, "CUDA"),
])
def test_linear_fp8_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        ops.linear_fp8(**{**fp8_args(), **change})


def test_gemm_and_quantize_refuse():
    a, s = torch.zeros(4, 256).to(E4), torch.zeros(2, 4).t()
    w = fp8_args()
    for args, match in (((a.float(), s), "a must be"), ((a, s[:, :1]), "scales"), ((a, s.contiguous()), "laid out"),
                        ((torch.zeros(4, 264).to(E4)[:, :256], s), "laid out"), ((a, s), "CUDA")):
        with pytest.raises(ValueError, match=match):
            ops.gemm_fp8(*args, w["weight"], w["scale"])
    for x, rows, match in ((torch.zeros(4), 1, "rows, columns"), (torch.zeros(4, 4), 64, "block_rows"),
                           (torch.zeros(4, 4, dtype=torch.int32), 1, "bf16"), (torch.zeros(4, 4), 128, "CUDA")):
        with pytest.raises(ValueError, match=match):
            ops.quantize_fp8(x, rows)


def norm_args():
    return {"x": torch.zeros(2, 3, 16), "branch": torch.zeros(2, 3, 16), "weight": torch.zeros(16)}


@pytest.mark.parametrize("change,match", [
    ({"x": torch.zeros(2, 3, 16, dtype=torch.float64)}, "x must be"),
    ({"branch": torch.zeros(2, 16)}, "shape"),
    ({"branch": torch.zeros(2, 3, 16, dtype=torch.bfloat16)}, "branch must be"),
    ({"weight": torch.zeros(15)}, "weight must be"),
    ({"weight": torch.zeros(16, dtype=torch.bfloat16)}, "weight must be"),
    ({"bias": torch.zeros(16)}, "no bias"),
    ({"kind": "layer", "post_bias": torch.zeros(16)}, "without post_weight"),
    ({"kind": "batch"}, "kind"),
    ({"gate": torch.zeros(1, 3, 16)}, "gate"),
    ({"gate": torch.zeros(3, 16)}, "gate"),
    ({"gate": torch.zeros(2, 3, 1)}, "gate"),
    ({"gate": torch.zeros(2, 2, 3, 16)}, "gate"),
    ({}, "CUDA"),
])
def test_residual_norm_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        ops.residual_norm(**{**norm_args(), **change})


@pytest.mark.parametrize("change,match", [
    ({"q": torch.zeros(2, 3, 16)}, "q must be"),
    ({"q": torch.zeros(2, 3, 4, 16, dtype=torch.float64)}, "q must be"),
    ({"k": torch.zeros(2, 3, 4, 8)}, "does not match"),
    ({"k": torch.zeros(2, 3, 4, 16, dtype=torch.bfloat16)}, "does not match"),
    ({"freq": torch.ones(8)}, "freq"),
    ({"freq": torch.ones(9, dtype=torch.float64)}, "freq"),
    ({"freq": torch.ones(0, dtype=torch.float64)}, "freq"),
    ({"positions": torch.zeros(2, 3)}, "positions"),
    ({"positions": torch.zeros(2, 4, dtype=torch.int64)}, "broadcast"),
    ({"positions": torch.zeros(1, 2, 3, dtype=torch.int64)}, "positions"),
    ({"positions": torch.zeros(2, 3, dtype=torch.int64), "offset": 1}, "either"),
    ({}, "CUDA"),
])
def test_rotary_refuses(change, match):
    args = {"q": torch.zeros(2, 3, 4, 16), "k": None, "freq": torch.ones(8, dtype=torch.float64), **change}
    with pytest.raises(ValueError, match=match):
        ops.rotary(args.pop("q"), args.pop("k"), args.pop("freq"), **args)


def test_frequencies():
    f, a = ops.rotary_frequencies(64, 10000.0)
    assert f.dtype == torch.float64 and a == 1.0 and torch.allclose(f, 10000.0 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-15)
    lin, a = ops.rotary_frequencies(64, 10000.0, {"type": "linear", "factor": 4})
    assert torch.equal(lin, f / 4) and a == 1.0
    assert torch.equal(ops.rotary_frequencies(64, 10000.0, {"rope_type": "default"})[0], f)

    # by frequency bands: short wavelengths kept, long ones divided, a monotone blend between
    s = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
    g, _ = ops.rotary_frequencies(128, 500000.0, s)
    f = ops.rotary_frequencies(128, 500000.0)[0]
    turns = 8192 * f / (2 * math.pi)
    assert torch.equal(g[turns > 4], f[turns > 4]) and torch.allclose(g[turns < 1], f[turns < 1] / 8, rtol=1e-14)
    assert (g.diff() < 0).all() and (g <= f).all() and (g >= f / 8 * (1 - 1e-12)).all()

    # by pairs: the ends kept and divided, the factor on cos and sin logarithmic unless given
    y = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    g, a = ops.rotary_frequencies(128, 10000.0, y)
    f = ops.rotary_frequencies(128, 10000.0)[0]
    turns = 4096 * f / (2 * math.pi)
    assert a == pytest.approx(0.1 * math.log(16) + 1, rel=1e-15)
    assert torch.allclose(g[turns > 40], f[turns > 40], rtol=1e-14) and torch.allclose(g[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-14)
    assert ops.rotary_frequencies(128, 10000.0, {**y, "attention_factor": 1.0})[1] == 1.0
    ratio = (0.0707 * math.log(16) + 1) / (0.1 * math.log(16) + 1)
    assert ops.rotary_frequencies(128, 10000.0, {**y, "mscale": 0.707, "mscale_all_dim": 1.0})[1] == pytest.approx(ratio, rel=1e-14)
    assert ops.rotary_frequencies(128, 10000.0, {**y, "factor": 1.0})[1] == 1.0

    # with the length: unchanged up to the original context, a larger base beyond
    d = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}
    assert torch.equal(ops.rotary_frequencies(64, 10000.0, d, n_positions=2048)[0], ops.rotary_frequencies(64, 10000.0)[0])
    longer = ops.rotary_frequencies(64, 10000.0, d, n_positions=4096)[0]
    assert torch.allclose(longer, ops.rotary_frequencies(64, 10000.0 * 3.0 ** (64 / 62))[0], rtol=1e-13)


@pytest.mark.parametrize("args,match", [
    ((63,), "even"), ((64, 0.0), "base"), ((64, 1e4, {"rope_type": "other", "factor": 2}), "unknown"),
    ((64, 1e4, {"rope_type": "linear"}), "factor"), ((64, 1e4, {"rope_type": "yarn", "factor": 2}), "original_max"),
    ((64, 1e4, {"rope_type": "linear", "factor": 0.5}), "factor"),
    ((64, 1e4, {"rope_type": "llama3", "factor": 2, "original_max_position_embeddings": 8, "low_freq_factor": 4.0}), "high_freq"),
])
def test_frequencies_refuse(args, match):
    with pytest.raises(ValueError, match=match):
        ops.rotary_frequencies(*args)

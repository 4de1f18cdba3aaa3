"""The block operators inside the producer LM: stretched contexts against transformers' own models,
8-bit projections, branch gates and scales, and the CUDA path against the PyTorch one."""

import math

import pytest
import torch

from saelens_b200.models.lm import HookedLM, preset_config
from saelens_b200.models.lm import transformer as lm_mod
from saelens_b200.models.lm.fp8 import quantize_torch

TINY = dict(n_layers=3, d_model=256, n_heads=4, n_key_value_heads=2, d_mlp=384, d_vocab=300, n_ctx=64)
gpu = pytest.mark.gpu


def tiny(preset="llama-3-8b", device=None, seed=0, **kw):
    torch.manual_seed(seed)
    return HookedLM(preset_config(preset, **{**TINY, "d_head": 64, "dtype": "float32", **kw}), device=device).eval()


@pytest.mark.parametrize("scaling", [
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 32},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32},
    {"rope_type": "dynamic", "factor": 2.0},
])
def test_stretched_contexts_match_transformers(scaling):
    transformers = pytest.importorskip("transformers")
    from saelens_b200.models.lm.hf import hooked_lm_from_hf

    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(vocab_size=300, hidden_size=64, intermediate_size=128, num_hidden_layers=2,
                                   num_attention_heads=4, num_key_value_heads=2, max_position_embeddings=64,
                                   rope_parameters={"rope_theta": 10000.0, **scaling})
    hf = transformers.LlamaForCausalLM(cfg).eval()
    lm = hooked_lm_from_hf(hf).eval()
    assert lm.cfg.rope_scaling["rope_type"] == scaling["rope_type"]
    for n in (12, 100 if scaling["rope_type"] == "dynamic" else 60):
        toks = torch.randint(0, 300, (2, n))
        with torch.no_grad():
            assert torch.allclose(lm(toks), hf(input_ids=toks).logits, atol=1e-4, rtol=1e-4)


def test_partial_interleaved_rotary_turns_pairs():
    lm = tiny(rotary_dim=16, rotary_interleaved=True)
    rot = lm._rotary(7)
    assert isinstance(rot, lm_mod.RotaryFrequencies) and rot.freq.shape == (8,)
    q, k = torch.randn(2, 7, 4, 64), torch.randn(2, 7, 2, 64)
    for t, got in zip((q, k), rot.turn(q, k)):
        z = torch.view_as_complex(t[..., :16].double().unflatten(-1, (8, 2)).contiguous())
        z = z * torch.polar(torch.ones(7, 8, dtype=torch.float64), torch.outer(torch.arange(7.0).double(), rot.freq))[None, :, None]
        # a fp32 rotation: two products and a sum of rounded terms
        assert (got[..., :16].double() - torch.view_as_real(z).flatten(-2)).abs().max() <= 8 * 2.0**-24 * t.abs().max()
        assert torch.equal(got[..., 16:], t[..., 16:])
    assert isinstance(tiny(rotary_dim=64)._rotary(7), tuple)  # the whole head in halves: the tables, as before


def test_gates_and_scales_of_branches():
    lm = tiny(branch_gate=True, residual_scale=0.5)
    toks = torch.randint(0, 300, (2, 9))
    with torch.no_grad():
        for blk in lm.blocks:
            blk.attn_gate.normal_()
            blk.mlp_gate.zero_()
        out, cache = lm.run_with_cache(toks)
    for i in range(3):
        p = f"blocks.{i}."
        mid = cache[p + "hook_resid_pre"] + cache[p + "hook_attn_out"]
        assert torch.equal(cache[p + "hook_resid_mid"], mid) and torch.equal(cache[p + "hook_resid_post"], mid)
    (g,) = torch.autograd.grad(lm(toks, return_type="loss"), [lm.blocks[1].mlp_gate])
    assert g.abs().max() > 0
    ones = tiny(branch_gate=True)
    assert torch.equal(ones(toks), tiny()(toks))  # gates start at one


def test_config_refusals():
    with pytest.raises(ValueError, match="rotary_dim"):
        tiny(rotary_dim=65)
    with pytest.raises(ValueError, match="rotary_dim"):
        tiny(rotary_dim=128)
    with pytest.raises(ValueError, match="weight_quantization"):
        tiny(weight_quantization="int4")
    with pytest.raises(ValueError, match="kind"):
        tiny().quantize_weights("int8")
    with pytest.raises(ValueError, match="already"):
        tiny(weight_quantization="fp8").quantize_weights()
    from saelens_b200.models.lm.tp import shard_lm_tensor_parallel

    with pytest.raises(ValueError, match="shard the model before"):
        shard_lm_tensor_parallel(tiny(weight_quantization="fp8"), None)


@pytest.mark.parametrize("preset", ["llama-3-8b", "gpt2", "gemma-2-9b", "qwen-14b"])
def test_quantized_model(preset):
    """A quantised projection is the product with the values that its 8 bits stand for, of rows that
    e4m3 holds: off by 2^-4 of each value (half a step of 3 bits), or half the least step, 2^-10 scales."""
    kw = dict(d_mlp=200, attn_softcap=None) if preset != "gpt2" else dict(n_key_value_heads=None, d_mlp=200)
    lm, ref = tiny(preset, **kw), tiny(preset, **kw)
    lm.quantize_weights("fp8")
    assert lm.cfg.weight_quantization == "fp8"
    x = torch.randn(2, 5, 256)
    for a, b in zip(lm.blocks, ref.blocks):
        pairs = [(a.attn.q, b.attn.q), (a.attn.k, b.attn.k), (a.attn.v, b.attn.v), (a.attn.o, b.attn.o), (a.mlp.up, b.mlp.up)]
        pairs += [(a.mlp.gate, b.mlp.gate)] if a.mlp.gated else []
        for p, r in pairs:
            y, want = p(x).flatten(0, 1).detach(), r(x).flatten(0, 1).detach()
            q, s = quantize_torch(x.flatten(0, 1), 1)
            w = r.weight.detach()
            held = 2.0**-4 * x.abs().flatten(0, 1) + 2.0**-10 * s.repeat_interleave(128, 1)
            err_w = 2.0**-4 * w.abs() + 2.0**-10 * w.abs().max() / 448
            tol = held @ w.abs().T + (x.abs().flatten(0, 1) + held) @ err_w.T
            assert ((y - want).abs() <= tol + 1e-5).all()
    toks = torch.randint(0, 300, (2, 11))
    with torch.no_grad():
        a, b = lm(toks).double(), ref(toks).double()
    assert torch.isfinite(a).all() and (a - b).norm() <= 0.25 * b.norm()
    # reload and change of type
    again = tiny(preset, seed=3, **kw).quantize_weights("fp8")
    again.load_state_dict(lm.state_dict())
    with torch.no_grad():
        assert torch.equal(again(toks), lm(toks))
    again.to(torch.bfloat16)
    assert again.blocks[0].attn.o.data.dtype == torch.float8_e4m3fn and again.blocks[0].attn.o.scale.dtype == torch.float32


def test_gradient_through_a_quantized_model():
    lm = tiny(weight_quantization="fp8", n_layers=2)
    x = torch.randn(2, 6, 256, requires_grad=True)
    y = lm.blocks[0].mlp(x)
    (g,) = torch.autograd.grad(y.square().sum(), x)
    assert torch.isfinite(g).all() and g.abs().max() > 0
    assert not any(p.dtype == torch.float8_e4m3fn for p in lm.parameters())


# ------------------------------------------------------------------------------------ on the device
PRESETS = [("llama-3-8b", {}), ("gemma-2-9b", {}), ("gpt2", {"n_key_value_heads": None}), ("qwen-14b", {}),
           ("llama-3-8b", {"branch_gate": True, "residual_scale": 0.5}),
           ("gemma-2-9b", {"branch_gate": True, "weight_quantization": "fp8"}),
           ("llama-3-8b", {"rotary_dim": 32, "rotary_interleaved": True, "weight_quantization": "fp8"}),
           ("llama-3-8b", {"rope_scaling": {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 32}})]


@gpu
@pytest.mark.parametrize("preset,kw", PRESETS)
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_same_bits_with_and_without_hooks(preset, kw, dtype):
    """Hooks that read every value turn the fused updates into single steps; nothing may change."""
    lm = tiny(preset, device="cuda", dtype=dtype, **kw)
    if kw.get("branch_gate"):
        with torch.no_grad():
            for blk in lm.blocks:
                blk.attn_gate.normal_()
                blk.mlp_gate.normal_()
    toks = torch.randint(0, 300, (3, 37), device="cuda")
    # fp32 gates and scales: the fused kernel's product and sum round once
    exact = not (dtype == "float32" and kw.get("branch_gate"))
    with torch.no_grad():
        plain = lm(toks)
        hooked, cache = lm.run_with_cache(toks)
        same = torch.equal if exact else lambda a, b: torch.allclose(a, b, rtol=1e-5, atol=1e-5)
        assert same(plain, hooked)
        for name in ("blocks.1.hook_resid_pre", "blocks.1.hook_resid_mid", "blocks.2.ln2.hook_normalized", "ln_final.hook_normalized",
                     "blocks.0.hook_resid_post", "blocks.2.ln1.hook_normalized", "blocks.0.attn.hook_rot_q"):
            if name in cache:
                _, one = lm.run_with_cache(toks, names_filter=name)
                assert same(one[name], cache[name]), name
        stop = lm(toks, stop_at_layer=2)
        assert same(stop, cache["blocks.2.hook_resid_pre"])
        # an edit of the stream reaches everything behind it, a module hook is called
        seen = []
        handle = lm.blocks[1].ln2.register_forward_hook(lambda m, i, o: seen.append(o))
        with lm.hooks(fwd_hooks=[("blocks.1.hook_resid_pre", lambda t, hook: t * 0)]):
            edited = lm(toks)
        handle.remove()
        assert len(seen) == 1 and not torch.equal(edited, plain)
        start = lm(toks, start_at_layer=1, residual=cache["blocks.1.hook_resid_pre"])
        assert same(start, plain)


@gpu
@pytest.mark.parametrize("preset,kw", PRESETS)
def test_cuda_matches_torch(preset, kw):
    """bf16 on the kernels against the same weights in fp32 PyTorch on the device: bf16 rounds each of
    about 12 steps a layer by 2^-9; a quantised model rounds its rows alike on both sides, up to
    values on a border."""
    lm = tiny(preset, device="cuda", dtype="bfloat16", init_std=0.06, **kw)
    toks = torch.randint(0, 300, (3, 37), device="cuda")
    with torch.no_grad():
        got = lm(toks).double()
        want = tiny(preset, device="cuda", init_std=0.06, **{**kw, "weight_quantization": None})
        src = {n: p for n, p in lm.state_dict().items()}
        if kw.get("weight_quantization"):
            lm_mod.FORCE_TORCH = True
            try:
                ref = lm(toks).double()
            finally:
                lm_mod.FORCE_TORCH = False
        else:
            want.load_state_dict({n: p.float() for n, p in src.items()})
            lm_mod.FORCE_TORCH = True
            try:
                ref = want(toks).double()
            finally:
                lm_mod.FORCE_TORCH = False
    bound = math.sqrt(36) * 2.0**-8 * (4 if kw.get("weight_quantization") else 1)
    assert (got - ref).norm() <= bound * ref.norm(), ((got - ref).norm() / ref.norm()).item()


@gpu
def test_gradients_through_a_quantized_model_on_cuda():
    """The gradient at an early hook, on the kernels and in PyTorch."""
    lm = tiny("llama-3-8b", device="cuda", dtype="bfloat16", weight_quantization="fp8", rotary_dim=32)
    toks = torch.randint(0, 300, (2, 20), device="cuda")
    with torch.no_grad():
        _, cache = lm.run_with_cache(toks, names_filter="blocks.1.hook_resid_pre")

    def gradient():
        x = cache["blocks.1.hook_resid_pre"].clone().requires_grad_()
        loss = lm(toks, start_at_layer=1, residual=x, return_type="loss")
        return torch.autograd.grad(loss, x)[0].double()

    got = gradient()
    lm_mod.FORCE_TORCH = True
    try:
        want = gradient()
    finally:
        lm_mod.FORCE_TORCH = False
    assert torch.isfinite(got).all()
    # bf16 and e4m3 borders: each of the two layers' steps rounds by 2^-9, quantised rows flip rarely
    assert (got - want).norm() <= 0.06 * want.norm(), ((got - want).norm() / want.norm()).item()


@gpu
def test_operators_in_a_row():
    """norm -> q/k/v -> rotary -> attention -> output -> norm, as a block chains them, captured in a graph."""
    from saelens_b200 import ops

    B, S, H, KV, d, D = 2, 50, 4, 2, 64, 256
    bf = torch.bfloat16
    w1, w2 = (ops.quantize_fp8(torch.randn(n, k, device="cuda").to(bf) * k**-0.5, 128) for n, k in (((H + 2 * KV) * d, D), (D, H * d)))
    x, branch = (torch.randn(B, S, D, device="cuda").to(bf) for _ in range(2))
    g1, g2 = (torch.rand(D, device="cuda").to(bf) + 0.5 for _ in range(2))
    freq, factor = ops.rotary_frequencies(d, 10000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}, device="cuda")
    st = ops.StatusWord("cuda")

    def block():
        stream, h = ops.residual_norm(x, branch, g1)
        qkv = ops.linear_fp8(h, *w1, status=st)
        q, k = qkv[..., : H * d].view(B, S, H, d), qkv[..., H * d : (H + KV) * d].view(B, S, KV, d)
        v = qkv[..., (H + KV) * d :].view(B, S, KV, d)
        q, k = ops.rotary(q, k, freq, factor=factor, inplace=True)
        z = ops.attention(q, k, v, d**-0.5, status=st)
        return ops.residual_norm(stream, ops.linear_fp8(z.reshape(B, S, H * d), *w2, status=st), g2, post_weight=g1)

    def plain():
        def norm(t, w):
            return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-5) * w.double()

        def linear(t, q, s):
            xq, xs = quantize_torch(t.reshape(-1, t.shape[-1]).to(bf), 1)
            held = xq.double() * xs.double().repeat_interleave(128, 1)[:, : t.shape[-1]]
            w = q.double() * s.double().repeat_interleave(128, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]
            return (held @ w.T).view(*t.shape[:-1], -1)

        stream = x.double() + branch.double()
        h = norm(stream, g1)
        qkv = linear(h, *w1)
        q, k = qkv[..., : H * d].view(B, S, H, d), qkv[..., H * d : (H + KV) * d].view(B, S, KV, d)
        v = qkv[..., (H + KV) * d :].view(B, S, KV, d)
        c = torch.polar(torch.full((S, d // 2), factor, dtype=torch.float64, device="cuda"),
                        torch.outer(torch.arange(S, device="cuda").double(), freq))[None, :, None]
        q, k = (torch.view_as_real(torch.complex(t[..., : d // 2], t[..., d // 2 :]) * c).movedim(-1, -2).flatten(-2) for t in (q, k))
        k, v = (t.repeat_interleave(H // KV, 2) for t in (k, v))
        att = torch.einsum("bshd,bthd->bhst", q, k) * d**-0.5
        att = att.masked_fill(~torch.ones(S, S, dtype=torch.bool, device="cuda").tril(), -math.inf).softmax(-1)
        z = torch.einsum("bhst,bthd->bshd", att, v).reshape(B, S, H * d)
        stream = stream + norm(linear(z, *w2), g1)
        return stream, norm(stream, g2)

    with torch.no_grad():
        got, want = block(), plain()
        for a, b in zip(got, want):
            # seven bf16 roundings of 2^-9 and e4m3 borders that they move
            assert (a.double() - b).norm() <= 0.03 * b.norm(), ((a.double() - b).norm() / b.norm()).item()
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block()
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            held = block()
        for _ in range(2):
            x.copy_(torch.randn_like(x))
            graph.replay()
            for a, b in zip(held, block()):
                assert torch.equal(a, b)
        st.check()

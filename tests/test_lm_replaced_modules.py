"""Modules of the producer LM that a program replaced or watches: the fused residual update may not go
past them."""

import pytest
import torch
from torch import nn

from saelens_b200.models.lm import HookedLM, preset_config
from saelens_b200.models.lm import transformer as lm_mod
from saelens_b200.utils.hooks import HookPoint

gpu = pytest.mark.gpu


def tiny(preset="llama-3-8b", device=None, **kw):
    torch.manual_seed(0)
    args = dict(n_layers=3, d_model=256, n_heads=4, n_key_value_heads=2, d_mlp=384, d_vocab=300, n_ctx=64, d_head=64, dtype="float32")
    return HookedLM(preset_config(preset, **{**args, **kw}), device=device).eval()


class Doubled(lm_mod.Norm):
    """A subclass with a forward of its own."""

    def __init__(self, norm):
        nn.Module.__init__(self)
        self.__dict__.update(norm.__dict__)

    def forward(self, x):
        return 2 * super().forward(x)


class Watched(HookPoint):
    def forward(self, x):
        return x + 1


def patched(norm):
    norm.forward = lambda x: 2 * lm_mod.Norm.forward(norm, x)
    return norm


REPLACED = [Doubled, patched, lambda norm: nn.Identity()]
HOOKS = ["register_forward_hook", "register_forward_pre_hook"]


@pytest.mark.parametrize("replace", REPLACED)
def test_a_replaced_norm_is_not_fused(replace, monkeypatch):
    monkeypatch.setattr(lm_mod, "_native_ok", lambda t: True)
    lm = tiny("gemma-2-9b")
    blk, x, hook = lm.blocks[0], torch.randn(1, 3, 256), HookPoint()
    assert lm_mod._fuses_residual(x, x, blk.ln1_post, hook, hook, blk.ln2, lm.cfg)
    blk.ln2 = replace(blk.ln2)
    assert not lm_mod._fuses_residual(x, x, blk.ln1_post, hook, hook, blk.ln2, lm.cfg)
    blk.ln1_post = replace(blk.ln1_post)
    assert not lm_mod._fuses_residual(x, x, blk.ln1_post, hook, hook, blk.ln1, lm.cfg)
    assert not lm_mod._fuses_residual(x, x, None, Watched(), hook, blk.ln1, lm.cfg)


@pytest.mark.parametrize("where", HOOKS)
def test_hooks_of_all_modules_are_not_passed(where, monkeypatch):
    monkeypatch.setattr(lm_mod, "_native_ok", lambda t: True)
    lm = tiny()
    x, hook = torch.randn(1, 3, 256), HookPoint()
    handle = getattr(nn.modules.module, "register_module_" + where[len("register_"):])(lambda *a: None)
    try:
        assert not lm_mod._fuses_residual(x, x, None, hook, hook, lm.ln_final, lm.cfg)
    finally:
        handle.remove()
    assert lm_mod._fuses_residual(x, x, None, hook, hook, lm.ln_final, lm.cfg)


def residual_norm_torch(x, branch, weight, bias, *, kind, eps, one_plus, post_weight, post_bias, gate, scale, round_branch,
                        post_eps=None):
    """`ops.residual_norm` by its definition, in fp32."""
    def norm(t, w, b, e):
        if kind == "layer":
            t = t - t.mean(-1, keepdim=True)
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + e) * (w + 1 if one_plus else w)
        return t if b is None else t + b

    if post_weight is not None:
        branch = norm(branch, post_weight, post_bias, eps if post_eps is None else post_eps)
    stream = x + branch * scale
    return stream, norm(stream, weight, bias, eps)


@pytest.mark.parametrize("normalization", ["RMS", "LN"])
@pytest.mark.parametrize("one_plus", [False, True])
@pytest.mark.parametrize("change", [{}, {"eps": 0.5}, {"one_plus": True}, {"one_plus": False}])
def test_the_fused_update_has_the_norms_settings(normalization, one_plus, change, monkeypatch):
    """A post-norm's own eps, a layer norm that ignores `one_plus`, norms that weigh differently."""
    from saelens_b200 import ops

    lm = tiny("gemma-2-9b", normalization=normalization, rms_one_plus=one_plus)
    blk, hook = lm.blocks[0], HookPoint()
    for n, norm in enumerate((blk.ln1_post, blk.ln2)):
        with torch.no_grad():
            norm.w.normal_()
            if norm.b is not None:
                norm.b.normal_()
    for name, value in change.items():
        setattr(blk.ln1_post, name, value)
    x, out = torch.randn(2, 5, 256), torch.randn(2, 5, 256)
    with torch.no_grad():
        stream = x + blk.ln1_post(out)
        want = blk.ln2(stream)
        # the update alone believes that its kernel runs, which is its definition here
        fuses = lm_mod._fuses_residual
        monkeypatch.setattr(lm_mod, "_native_ok", lambda t: True)
        ok = fuses(x, out, blk.ln1_post, hook, hook, blk.ln2, lm.cfg)
        monkeypatch.undo()
        monkeypatch.setattr(lm_mod, "_fuses_residual", lambda *a: ok)
        monkeypatch.setattr(ops, "residual_norm", residual_norm_torch)
        got, normed = blk._join(x, out, blk.ln1_post, None, hook, hook, blk.ln2)
        normed = blk.ln2(got) if normed is None else normed
    # fp32 in two orders: 256 addends and a few products, 2^-24 each
    assert torch.allclose(got, stream, atol=1e-4, rtol=1e-5) and torch.allclose(normed, want, atol=1e-4, rtol=1e-4)
    assert ok or "one_plus" in change  # what may be fused still is


class Twice(nn.Module):
    """A block of a program's own."""

    def __init__(self, block):
        super().__init__()
        self.block = block

    def forward(self, x, rot):
        return self.block(self.block(x, rot), rot)


def replaced_blocks(lm):
    toks = torch.randint(0, 300, (2, 9), device=lm.device)
    args = []
    handle = lm.blocks[1].register_forward_pre_hook(lambda m, a: args.append(len(a)))
    with torch.no_grad():
        lm(toks)
        handle.remove()
        assert args == [2]  # a hook of a block sees what a block was always called with
        x = lm(toks, stop_at_layer=1)
        want = lm.blocks[1](lm.blocks[1](x, lm._rotary(9)), lm._rotary(9))
        lm.blocks[1] = Twice(lm.blocks[1])
        assert torch.equal(lm(toks, stop_at_layer=2), want)
        logits = lm.unembed(lm.ln_final(lm.blocks[2](want, lm._rotary(9))))
        assert torch.equal(lm(toks), logits)


def test_a_replaced_block():
    replaced_blocks(tiny())


@gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_replaced_block_on_cuda(dtype):
    replaced_blocks(tiny(device="cuda", dtype=dtype))


@gpu
@pytest.mark.parametrize("preset,names", [("llama-3-8b", ["ln1", "ln2"]), ("gemma-2-9b", ["ln1_post", "ln2", "ln2_post"])])
@pytest.mark.parametrize("replace", REPLACED)
def test_a_replaced_norm_is_called_on_cuda(preset, names, replace):
    """The same bits as with hooks on every value, where each module is called."""
    lm = tiny(preset, device="cuda", dtype="bfloat16")
    toks = torch.randint(0, 300, (2, 9), device="cuda")
    with torch.no_grad():
        before = lm(toks)
        for name in names:
            setattr(lm.blocks[1], name, replace(getattr(lm.blocks[1], name)))
        lm.ln_final = replace(lm.ln_final)
        got = lm(toks)
        hooked, _ = lm.run_with_cache(toks)
    assert torch.equal(got, hooked) and not torch.equal(got, before)

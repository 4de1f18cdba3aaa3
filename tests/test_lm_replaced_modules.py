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

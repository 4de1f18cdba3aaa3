"""8-bit weights of the producer LM as a program reaches them."""

import pytest
import torch

from saelens_b200.models.lm import HookedLM, preset_config

TINY = dict(n_layers=2, d_model=128, n_heads=4, n_key_value_heads=2, d_mlp=192, d_vocab=300, n_ctx=64, d_head=32, dtype="float32")


def test_a_shared_config_stays_as_it_is():
    cfg = preset_config("llama-3-8b", **TINY)
    lm = HookedLM(cfg).quantize_weights()
    assert lm.cfg.weight_quantization == "fp8" and cfg.weight_quantization is None
    assert HookedLM(cfg).blocks[0].attn.qkv_fp8 is None


class _Fake:
    """`ops.linear_fp8` whose backward pass reports a wait that ran out."""

    class Linear(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, status):
            ctx.status, ctx.d_in = status, x.shape[-1]
            return x.new_zeros(*x.shape[:-1], weight.shape[0])

        @staticmethod
        def backward(ctx, dy):
            ctx.status.tensor.fill_(_Fake.code)
            _Fake.ran += 1
            return dy.new_zeros(*dy.shape[:-1], ctx.d_in), None, None

    code = ran = 0

    @staticmethod
    def linear_fp8(x, weight, scale, bias=None, status=None):
        return _Fake.Linear.apply(x, weight, status)


def test_a_wait_that_ran_out_in_a_backward_pass_raises_there(monkeypatch):
    from saelens_b200 import ops
    from saelens_b200.models.lm import fp8
    from saelens_b200.models.lm import transformer as lm_mod
    from saelens_b200.ops.status import KernelTimeoutError, StatusWord

    lm = HookedLM(preset_config("llama-3-8b", **TINY)).quantize_weights()
    status = StatusWord("cpu")
    read = []
    monkeypatch.setattr(status, "code", lambda: read.append(1) or int(status.tensor))
    monkeypatch.setattr(fp8, "_native", lambda x: True)
    monkeypatch.setattr(lm_mod, "_status_for", lambda x: status)
    monkeypatch.setattr(ops, "linear_fp8", _Fake.linear_fp8)
    x = torch.randn(1, 4, 128, requires_grad=True)
    for code in (0, 2, 0, 3, 2):
        _Fake.code, _Fake.ran = code, 0
        read.clear()
        y = lm.blocks[0].mlp(x) + lm.blocks[1].mlp(x)
        if code:
            with pytest.raises(KernelTimeoutError, match="backward"):
                y.sum().backward()
        else:
            y.sum().backward()
        assert _Fake.ran == 4 and len(read) == 1 and int(status.tensor) == 0  # one read for the whole pass
    with torch.no_grad():
        lm.blocks[0].mlp(x)


@pytest.mark.gpu
def test_a_backward_pass_on_cuda_reads_its_status():
    """The word is read at the end of the pass, whichever thread ends it, and not under capture."""
    from saelens_b200.models.lm import transformer as lm_mod
    from saelens_b200.ops.status import KernelTimeoutError

    lm = HookedLM(preset_config("llama-3-8b", **{**TINY, "dtype": "bfloat16"}), device="cuda").quantize_weights()
    mlp = lm.blocks[0].mlp
    x = torch.randn(2, 40, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    status = lm_mod._status_for(x)

    def gradient():
        return torch.autograd.grad(mlp(x).float().square().sum(), x)[0]

    want = gradient()
    y = mlp(x).float().square().sum()
    status.tensor.fill_(2)  # as a wait that ran out writes it
    with pytest.raises(KernelTimeoutError, match="backward"):
        torch.autograd.grad(y, x)
    assert status.code() == 0 and torch.equal(gradient(), want)
    del y  # autograd ties a leaf to the stream of a graph that lives, which a capture may not join

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        gradient()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = gradient()
    for _ in range(2):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        assert torch.equal(held, gradient())
    status.check()

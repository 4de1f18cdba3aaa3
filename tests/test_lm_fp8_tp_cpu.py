"""8-bit weights under producer tensor parallelism (gloo on CPU): the model is split first, then each
rank quantises its slices, by hand and through the training runner."""

import json
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp


def _port() -> int:
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _join(rank, world, port):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank))
    import torch.distributed as dist

    dist.init_process_group("gloo", rank=rank, world_size=world)
    return dist


def _model(preset):
    from saelens_b200.models.lm import HookedLM, preset_config

    # widths and slices that are no multiples of the blocks of 128
    over = dict(n_layers=1, d_model=192, n_heads=6, n_key_value_heads=6 if preset == "gpt2" else 2, d_head=32, d_mlp=328,
                d_vocab=300, n_ctx=32, dtype="float32", init_std=0.1)
    torch.manual_seed(0)
    lm = HookedLM(preset_config(preset, **over))
    with torch.no_grad():
        for name, p in lm.named_parameters():
            if name.endswith("bias"):
                p.normal_()
    return lm


def _slices_worker(rank, world, port, preset, tmp):
    dist = _join(rank, world, port)
    from saelens_b200.models.lm.fp8 import Fp8Linear
    from saelens_b200.models.lm.tp import shard_lm_tensor_parallel
    from saelens_b200.models.lm.transformer import NativeLinear, _act

    def part(lin, rows=None, cols=None):
        """An 8-bit projection of rows or columns of a whole one; what is split by columns has no bias."""
        w = lin.weight if rows is None else lin.weight[rows[0] : rows[1]]
        w = w if cols is None else w[:, cols[0] : cols[1]]
        bias = None if lin.bias is None or cols is not None else lin.bias[rows[0] : rows[1]]
        m = NativeLinear(w.shape[1], w.shape[0], bias is not None, torch.float32)
        m.weight.data, m.bias = w.detach().clone(), None if bias is None else torch.nn.Parameter(bias.detach().clone())
        return Fp8Linear([m])

    full, names = _model(preset), ["ln1.hook_normalized", "attn.hook_q", "attn.hook_k", "attn.hook_v", "attn.hook_z", "hook_attn_out",
                                   "ln2.hook_normalized", "hook_mlp_out"]
    tp = shard_lm_tensor_parallel(_model(preset), dist.group.WORLD).quantize_weights()
    assert tp.blocks[0].attn.qkv_fp8 is not None and tp.cfg.weight_quantization == "fp8"
    toks = torch.randint(0, 300, (2, 12), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        _, got = tp.run_with_cache(toks, names_filter=["blocks.0." + n for n in names])
        got = {n: got["blocks.0." + n] for n in names}
        at, mlp, cfg = full.blocks[0].attn, full.blocks[0].mlp, full.cfg
        ranges = lambda n: [(r * n // world, (r + 1) * n // world) for r in range(world)]  # noqa: E731
        x, want = got["ln1.hook_normalized"], {}
        for n, lin, heads in (("q", at.q, cfg.n_heads), ("k", at.k, cfg.n_key_value_heads), ("v", at.v, cfg.n_key_value_heads)):
            want["attn.hook_" + n] = torch.cat([part(lin, rows=r)(x) for r in ranges(heads * cfg.d_head)], -1)
        z = got["attn.hook_z"].flatten(2)
        out = sum(part(at.o, cols=r)(z[..., r[0] : r[1]]) for r in ranges(z.shape[-1]))
        want["hook_attn_out"] = out if at.o.bias is None else out + at.o.bias
        x, out = got["ln2.hook_normalized"], 0
        for r in ranges(cfg.d_mlp):
            pre = part(mlp.gate if mlp.gated else mlp.up, rows=r)(x)
            post = _act(cfg.act_fn, pre) * part(mlp.up, rows=r)(x) if mlp.gated else _act(cfg.act_fn, pre)
            out = out + part(mlp.down, cols=r)(post)
        want["hook_mlp_out"] = out if mlp.down.bias is None else out + mlp.down.bias
    errs = {}
    for n, w in want.items():
        # q, k and v of a rank share blocks of 128 rows where their slices meet: their weights' values differ by
        # an e4m3 rounding, 2^-4 of a value; what is split by columns is quantised alike
        own = n in ("hook_attn_out", "hook_mlp_out")
        errs[n] = ((got[n].flatten(2) - w).norm() / w.norm() / (1e-5 if own and not (n == "hook_mlp_out" and mlp.gated) else 2.0**-4)).item()
    with open(os.path.join(tmp, f"r{rank}.json"), "w") as f:
        json.dump(errs, f)
    dist.destroy_process_group()


@pytest.mark.parametrize("preset", ["llama-3-8b", "gpt2"])
def test_a_split_model_is_quantised_slice_by_slice(tmp_path, preset):
    mp.spawn(_slices_worker, args=(2, _port(), preset, str(tmp_path)), nprocs=2, join=True)
    for rank in range(2):
        errs = json.loads((tmp_path / f"r{rank}.json").read_text())
        assert len(errs) == 5 and max(errs.values()) <= 1, errs


def _runner_worker(rank, world, port, tmp, vtp):
    dist = _join(rank, world, port)
    from saelens_b200.config import LanguageModelSAERunnerConfig, LoggingConfig
    from saelens_b200.models.standard import StandardTrainingSAEConfig
    from saelens_b200.runners.llm_sae_training_runner import LanguageModelSAETrainingRunner

    kwargs = dict(n_layers=2, d_model=64, n_heads=4, d_mlp=128, d_vocab=500, n_ctx=64, dtype="float32", seed=0,
                  weight_quantization="fp8")
    cfg = LanguageModelSAERunnerConfig(
        sae=StandardTrainingSAEConfig(d_in=64, d_sae=128, l1_coefficient=1e-3), model_name="gpt2",
        model_from_pretrained_kwargs=dict(kwargs), hook_name="blocks.1.hook_resid_pre",
        dataset_path="synthetic:uniform:500:32", context_size=16, training_tokens=64 * 2, train_batch_size_tokens=64,
        store_batch_size_prompts=4, n_batches_in_buffer=2, output_path=os.path.join(tmp, "out"),
        logger=LoggingConfig(log_to_wandb=False), device="cpu", n_checkpoints=0, verbose=False, routing_transport="collective")
    runner = LanguageModelSAETrainingRunner(cfg, vllm_dp_size=1, sae_dp_size=1, vllm_tp_size=vtp, use_shard_routing=True)
    info = {"role": runner.role}
    if runner.model is not None:
        blk = runner.model.blocks[0]
        info.update(width=blk.attn.qkv_fp8.d_out, quantised=runner.model.cfg.weight_quantization,
                    sharded=getattr(runner.model, "tp", None) is not None)
    assert cfg.model_from_pretrained_kwargs == kwargs
    out = runner.run()
    if out is not None:
        info["steps"] = runner.trainer.n_training_steps
    with open(os.path.join(tmp, f"r{rank}.json"), "w") as f:
        json.dump(info, f)
    dist.destroy_process_group()


@pytest.mark.parametrize("vtp", [1, 2])
def test_the_runner_splits_before_it_quantises(tmp_path, vtp):
    mp.spawn(_runner_worker, args=(vtp + 1, _port(), str(tmp_path), vtp), nprocs=vtp + 1, join=True)
    r = [json.loads((tmp_path / f"r{i}.json").read_text()) for i in range(vtp + 1)]
    for producer in r[:vtp]:
        assert producer == {"role": "producer", "width": 3 * 64 // vtp, "quantised": "fp8", "sharded": vtp > 1}
    assert r[vtp]["role"] == "consumer" and r[vtp]["steps"] == 2

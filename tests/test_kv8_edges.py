"""The 8-bit key/value cache on the CPU: what the kernels' reports name, and which models take the cache."""
import argparse
import glob
import json
import os
import re

import pytest
import torch

from mp_util import run_ranks
from slopllm_b200.models.dense import DenseConfig, DenseModel, load_dense_model, random_dense_model
from slopllm_b200.ops import kv8 as K8
from slopllm_b200.parallel.dist import ParallelContext

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "slopllm_b200", "csrc")


def test_reports_name_one_kernel():
    """Numbers of failed self-checks and of expired waits in the 8-bit cache's kernels are no other kernel's, and are written by name."""
    text = {os.path.basename(f): open(f).read() for f in glob.glob(os.path.join(CSRC, "*.cu*"))}
    own = dict(re.findall(r"(KV8_(?:SITE|WAIT)_\w+) = (\d+)", text["kv8.cuh"]))
    sites, waits = ([int(v) for k, v in own.items() if k.startswith(f"KV8_{what}")] for what in ("SITE", "WAIT"))
    assert len(set(sites)) == 4 and len(set(waits)) == 2
    used = {"site": {}, "wait": {}}
    for name, source in text.items():
        for what, pattern in (("site", r"(?:guard_ok|kv8_slot)\(\s*[\w.>-]+(?:\([^()]*\))?,\s*(\d+)\s*,"), ("wait", r"atomicExch\([^;]*?,\s*(\d+)\)")):
            for number in re.findall(pattern, source):
                used[what].setdefault(int(number), set()).add(name)
    assert used["site"] and used["wait"]
    assert not set(sites) & set(used["site"]) and not set(waits) & set(used["wait"])
    assert not any(name.startswith("kv8") for names in (*used["site"].values(), *used["wait"].values()) for name in names)


def wide(**kw):
    """Qwen3.5's widths: 16 heads of 256 over 2, a quarter of them rotated, a gate behind each query."""
    return DenseConfig(hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=16, num_key_value_heads=2, head_dim=256, vocab_size=100,
                       partial_rotary_factor=0.25, attn_output_gate=True, **kw)


def raw_config(head_dim):
    return {"model_type": "qwen3", "hidden_size": 64, "intermediate_size": 128, "num_hidden_layers": 1, "num_attention_heads": 16, "num_key_value_heads": 2,
            "head_dim": head_dim, "vocab_size": 100, "eos_token_id": 1}


def test_widths_without_prompts_are_refused_before_loading(tmp_path, capsys):
    """A GPU has no attention of prompts for heads of 256 over this cache: the model, its loading and the plan say so, in front of weights and pages.  The CPU has it."""
    from slopllm_b200.cli import plan as plan_cli
    from slopllm_b200.utils.sizing import plan_dense
    gpu = ParallelContext(device=torch.device("cuda", 0))
    for head_dim in (256, 96):
        (tmp_path / "config.json").write_text(json.dumps(raw_config(head_dim)))
        for call in (lambda: DenseModel(wide() if head_dim == 256 else DenseConfig(head_dim=96), None, gpu, kv_dtype="e4m3"),
                     lambda: load_dense_model(str(tmp_path), gpu, kv_dtype="e4m3"), lambda: plan_dense(DenseConfig(head_dim=head_dim), kv_dtype="e4m3")):
            with pytest.raises(ValueError, match=f"64 or 128 values, not {head_dim}"):
                call()
        with pytest.raises(SystemExit, match="64 or 128"):
            plan_cli.main(["--model", str(tmp_path), "--kv-dtype", "e4m3"])
        assert plan_cli.main(["--model", str(tmp_path)]) == 0
    capsys.readouterr()
    cfg = wide()
    w, _ = random_dense_model(cfg, seed=1, device="cpu", dtype=torch.float32)
    assert DenseModel(cfg, w, ParallelContext(device=torch.device("cpu")), kv_dtype="e4m3").allocate_cache(2).kv8


def test_checkpoints_that_do_not_take_the_cache_end_the_command(tmp_path):
    """One line of text, as with random weights, not a traceback."""
    from slopllm_b200.cli.model_cli import add_model_args, build_runtime
    ap = argparse.ArgumentParser()
    add_model_args(ap)
    for raw, what in (({"model_type": "zemezen"}, "zemezen does not cache keys and values in e4m3"), (raw_config(72), "multiple of 16")):
        (tmp_path / "config.json").write_text(json.dumps(raw))
        with pytest.raises(SystemExit, match=what):
            build_runtime(ap.parse_args(["--cpu", "--model", str(tmp_path), "--kv-dtype", "e4m3"]))


def test_both_types_reach_the_loader(tmp_path):
    """`dtype` and `kv_dtype` together: a family that has both gets both."""
    from slopllm_b200.models.registry import ModelRegistration, load_registered
    got = []
    reg = ModelRegistration(False, False, False, False, lambda *a, **k: got.append(k), float32=True, kv8=True)
    gpu, cpu = ParallelContext(device=torch.device("cuda", 0)), ParallelContext(device=torch.device("cpu"))
    load_registered(reg, str(tmp_path), gpu, 0, "float32", "e4m3")
    load_registered(reg, str(tmp_path), cpu, 0, "float32", "e4m3")
    load_registered(reg, str(tmp_path), cpu, 0, None, None)
    assert got == [{"dtype": torch.float32, "kv_dtype": "e4m3"}, {"kv_dtype": "e4m3"}, {}]


def _two_ranks(rank, world, hybrid):
    from slopllm_b200.parallel.dist import init_from_env
    from slopllm_b200.runtime.engine import Engine
    cfg = DenseConfig.tiny(hybrid=hybrid)
    prompt = torch.randint(2, cfg.vocab_size, (90,), generator=torch.Generator().manual_seed(5)).tolist()

    def serve(ctx, r, n):
        w, _ = random_dense_model(cfg, 3, "cpu", torch.float32, r, n)
        eng = Engine(cfg, DenseModel(cfg, w, ctx, kv_dtype="e4m3"), num_pages=8, max_batch=2, max_seq_len=256)
        s, _ = eng.kv.start_request(prompt)
        _, hid = eng.prefill([s], [prompt], chunk_size=64, want_hidden=True)
        return [eng.model.compute_logits(hid[0])[-1:].float(), *(eng.step([s], [[7 + i]], [[0]])[0][None].float() for i in range(3))], eng.cache

    got, cache = serve(init_from_env("gloo"), rank, world)
    want, whole = serve(ParallelContext(device=torch.device("cpu")), 0, 1)
    i = min(cache.kv8)
    n_kv = cache.kv8[i].k.shape[1]
    heads = slice(rank * n_kv, (rank + 1) * n_kv)
    # (the first full-attention layer's rows see no sum over ranks in front of them where it is the model's first layer)
    same = hybrid or all(torch.equal(getattr(cache.kv8[i], x), getattr(whole.kv8[i], x)[:, heads]) for x in ("k", "v", "exps"))
    return same, n_kv * world == whole.kv8[i].k.shape[1], max(((a - b).abs().max() / b.abs().max()).item() for a, b in zip(got, want))


@pytest.mark.parametrize("hybrid", [False, True])
def test_two_ranks(hybrid):
    """Key heads over two ranks: each rank's part of the cache is the whole one's, and so are the logits, up to the order of sums over ranks, which can move a
    value of a later layer to the next code (2^-3 of it, of some 64 in a head)."""
    for same, shared, err in run_ranks(_two_ranks, 2, hybrid):
        assert same and shared and err < 2e-2, err


def test_negative_positions_have_no_keys():
    """Any negative position, as on a GPU."""
    cache = K8.Kv8Cache.allocate(1, 16, 1, 16, "cpu")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)
    got = K8.kv8_attention(torch.ones(3, 2, 16), cache, i32(-1, -2, -70), i32(0, 0, 0), i32(0)[None], 1.0)
    assert (got == 0).all()

"""What is made of rows' and weights' arguments before a kernel sees them, and what loaders and plans say about FP8 projections."""
import pytest
import torch

from fp8_util import near, some_rows, weight
from slopllm_b200.models.weights import LinearWeight
from slopllm_b200.ops import fp8 as F8


def test_scales_that_the_kernels_take():
    s = torch.rand(3, 4)
    assert F8._scales(s) is s and F8._scales(part := torch.rand(3, 8)[:, :4]) is part
    for scale in (s[:1].expand(3, 4), s.flatten()[:8].as_strided((3, 4), (2, 1)), torch.rand(4, 3).t(), s.double(), s[:1].as_strided((1, 4), (1, 1)),
                  torch.rand(4, 1).t()):
        got = F8._scales(scale)
        assert got.dtype == torch.float32 and got.stride() == (4, 1) and torch.equal(got, scale.float())
    far = torch.empty(2, 2 ** 31, device="meta")[:, :4]
    assert F8._scales(far).stride() == (4, 1)
    w, values = weight(300, 400, device="cpu")
    rows, scale = some_rows(5, 400, device="cpu"), w.fp8_scale[:1].expand(3, 4)
    values = values / w.fp8_scale.double().repeat_interleave(128, 0)[:300].repeat_interleave(128, 1)[:, :400]
    assert near(F8.fp8_linear(rows, LinearWeight(w.weight, fp8_scale=scale), out_f32=True), rows, values * scale[:1].double().repeat_interleave(128, 1)[:, :400])


def test_weights_that_the_kernels_take():
    w = torch.zeros(64, 256, dtype=torch.uint8)
    assert F8._codes(w) is w and F8._codes(part := w[3:40:2, 16:160]) is part
    w.copy_(torch.arange(64 * 256).view(64, 256) % 251)
    for codes in (w[:1].expand(64, 256), w.flatten().as_strided((64, 256), (16, 1)), w[:1].as_strided((1, 256), (16, 1)), w[:, :144].t().contiguous().t(),
                  torch.zeros(64, 264, dtype=torch.uint8)[:, :256]):
        got = F8._codes(codes)
        assert got.stride() == (codes.shape[1], 1) and torch.equal(got, codes)
    assert F8._codes(torch.empty(2, 2 ** 31, dtype=torch.uint8, device="meta")[:, :256]).stride() == (256, 1)


def test_plans_count_what_loaders_expand():
    """Weights of a rank against the plan: projections that end on the edges of blocks, shards and parts of fused matrices that do not."""
    from slopllm_b200.models.dense import DenseConfig, random_dense_model
    from slopllm_b200.runtime.workspace import walk_tensors
    from slopllm_b200.utils.sizing import dense_weight_bytes
    configs = [dict(hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=4, head_dim=64),
               dict(hidden_size=272, intermediate_size=1216, num_attention_heads=8, num_key_value_heads=2, head_dim=64),
               dict(hidden_size=128, intermediate_size=192, num_attention_heads=2, num_key_value_heads=2, head_dim=32),
               dict(hidden_size=400, intermediate_size=1024, num_attention_heads=6, num_key_value_heads=2, head_dim=128)]
    some = set()
    for cfg in [DenseConfig(num_hidden_layers=2, vocab_size=512, **c) for c in configs] + [DenseConfig.tiny(), DenseConfig.tiny(hybrid=True)]:
        for tp in (1, 2):
            w, _ = random_dense_model(cfg, 0, "cpu", torch.bfloat16, 0, tp, fp8=True)
            seen, total = set(), [0]

            def add(t):
                if t.data_ptr() not in seen:
                    seen.add(t.data_ptr())
                    total[0] += t.numel() * t.element_size()
            walk_tensors(w, add)
            assert dense_weight_bytes(cfg, tp, fp8=True) == total[0], (cfg, tp)
            layer = w.layers[-1]
            some.add((layer.w_qkv.is_fp8, layer.o_proj.is_fp8, layer.mlp_w13.is_fp8, layer.mlp_w2.is_fp8))
    assert len(some) > 3


def fp8_checkpoint(path, cfg, keep):
    """A checkpoint of `cfg` whose projections named by `keep` are FP8, others bf16."""
    import json
    import struct
    from slopllm_b200.models.dense import random_dense_model
    from slopllm_b200.ops import dense as D
    _, tensors = random_dense_model(cfg, seed=3, device="cpu", dtype=torch.bfloat16)
    for name in [n for n in tensors if any(n.endswith(k + ".weight") for k in keep)]:
        tensors[name], tensors[name + "_scale_inv"] = D.fp8_block_quantize(tensors[name])
    names = {torch.bfloat16: "BF16", torch.float32: "F32", torch.float8_e4m3fn: "F8_E4M3"}
    head, blobs, at = {}, [], 0
    for n, t in tensors.items():
        blobs.append(bytes(t.contiguous().view(torch.uint8).numpy()))
        head[n] = {"dtype": names[t.dtype], "shape": list(t.shape), "data_offsets": [at, at + len(blobs[-1])]}
        at += len(blobs[-1])
    text = json.dumps(head).encode()
    text += b" " * (-len(text) % 8)
    path.mkdir()
    (path / "model.safetensors").write_bytes(struct.pack("<Q", len(text)) + text + b"".join(blobs))
    raw = dict(model_type=cfg.model_type, hidden_size=cfg.hidden_size, intermediate_size=cfg.intermediate_size, num_hidden_layers=cfg.num_hidden_layers,
               num_attention_heads=cfg.num_attention_heads, num_key_value_heads=cfg.num_key_value_heads, head_dim=cfg.head_dim, vocab_size=cfg.vocab_size)
    if cfg.model_type == "qwen3_5":
        raw.update(layer_types=cfg.layer_types, linear_num_key_heads=cfg.linear_num_key_heads, linear_key_head_dim=cfg.linear_key_head_dim,
                   linear_num_value_heads=cfg.linear_num_value_heads, linear_value_head_dim=cfg.linear_value_head_dim, attn_output_gate=True,
                   rope_parameters=dict(partial_rotary_factor=cfg.partial_rotary_factor))
    (path / "config.json").write_text(json.dumps(raw))
    return str(path)


def model_args(*more):
    import argparse
    from slopllm_b200.cli import model_cli
    ap = argparse.ArgumentParser()
    model_cli.add_model_args(ap)
    return ap.parse_args(["--cpu", "--act-dtype", "e4m3", "--max-pages", "8", *more])


def test_checkpoints_whose_fp8_projections_take_no_rows(tmp_path, monkeypatch):
    """FP8 in recurrent layers or in the down projection alone: refused by name, before anything is loaded."""
    from slopllm_b200.cli import model_cli
    from slopllm_b200.models import dense
    from slopllm_b200.parallel.dist import ParallelContext
    cfg, plain, cpu = dense.DenseConfig.tiny(hybrid=True), dense.DenseConfig.tiny(), ParallelContext(device=torch.device("cpu"))
    linear = ("linear_attn.in_proj_qkv", "linear_attn.in_proj_z", "linear_attn.out_proj")
    some = {"linear": (cfg, linear), "down": (plain, ("down_proj",)), "both": (cfg, (*linear, "self_attn.o_proj"))}
    paths = {n: fp8_checkpoint(tmp_path / n, *x) for n, x in some.items()}
    assert not dense.has_fp8_projections(plain, ["model.visual.layers.0.mlp.up_proj.weight_scale_inv", "mtp.layers.0.self_attn.q_proj.weight_scale_inv"])
    _, model = dense.load_dense_model(paths["both"], cpu, act_dtype="e4m3")
    assert [lw.o_proj.is_fp8 for lw in model.w.layers if lw.kind == "full_attention"] == [True]
    monkeypatch.setattr(dense, "assemble_dense_weights", None)
    for name in ("linear", "down"):
        with pytest.raises(ValueError, match="has none"):
            dense.load_dense_model(paths[name], cpu, act_dtype="e4m3")
        with pytest.raises(SystemExit, match="has none"):
            model_cli.build_runtime(model_args("--model", paths[name]), with_scheduler=False)


def test_matrices_that_take_no_rows_in_8_bits_are_told(capsys, monkeypatch):
    from slopllm_b200.cli import model_cli
    from slopllm_b200.models.dense import DenseConfig, DenseModel, random_dense_model
    from slopllm_b200.parallel.dist import ParallelContext
    cpu = ParallelContext(device=torch.device("cpu"))
    of = lambda cfg, tp=1: DenseModel(cfg, random_dense_model(cfg, 0, "cpu", torch.float32, 0, tp, fp8=True)[0], cpu, act_dtype="e4m3").fp8_layers()
    assert of(DenseConfig.tiny()) == (8, 8) and of(DenseConfig.tiny(hybrid=True)) == (10, 16)
    cut = DenseConfig(num_hidden_layers=1, vocab_size=512, hidden_size=256, intermediate_size=1216, num_attention_heads=4, num_key_value_heads=4, head_dim=64)
    assert of(cut) == (2, 4) and of(cut, 2) == (2, 4)
    for spec, told in (("qwen3-tiny", ""), ("qwen35-tiny", "10 of 16 matrices")):
        model_cli.build_runtime(model_args("--random-init", spec), with_scheduler=False)
        err = capsys.readouterr().err
        assert told in err and bool(told) == ("--act-dtype" in err)


def test_communicators_join_rows_in_8_bits():
    """Sums over the ranks and their norm in 8 bits are one call of the communicator, as those in 16 bits: what it overrides is used."""
    from slopllm_b200.models.dense import DenseConfig, DenseModel, random_dense_model
    from slopllm_b200.parallel.dist import Comm, ParallelContext
    from slopllm_b200.runtime.engine import Engine
    told = []

    class Told(Comm):
        def allreduce_add_rmsnorm_fp8(self, *args):
            told.append(8)
            return super().allreduce_add_rmsnorm_fp8(*args)

        def allreduce_add_rmsnorm(self, *args, **kw):
            told.append(16)
            return super().allreduce_add_rmsnorm(*args, **kw)

        def _reduce_partial(self, partial):
            return super()._reduce_partial(partial) * 2

    cfg, ctx = DenseConfig.tiny(), ParallelContext(device=torch.device("cpu"))
    w, _ = random_dense_model(cfg, 0, "cpu", torch.float32, fp8=True)
    logits = []
    for comm in (Told(ctx), Comm(ctx)):
        model = DenseModel(cfg, w, ctx, comm=comm, act_dtype="e4m3")
        eng = Engine(cfg, model, num_pages=8, max_batch=2, max_seq_len=256)
        s, _ = eng.kv.start_request([5, 6, 7])
        _, hid = eng.prefill([s], [[5, 6, 7]], chunk_size=32, want_hidden=True)
        logits.append(model.compute_logits(hid[0]))
    assert told == [8, 8, 8, 16] and not torch.equal(*logits)


@pytest.mark.parametrize("keep", [("o_proj",), ("gate_proj", "up_proj"), ("q_proj", "k_proj", "down_proj"), ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")])
def test_plans_count_what_a_checkpoint_holds(tmp_path, keep):
    """A checkpoint that is partly FP8: its loaded weights against the plan from its tensors' names."""
    from slopllm_b200.cli.model_cli import _tensor_names
    from slopllm_b200.models.dense import DenseConfig, load_dense_model
    from slopllm_b200.parallel.dist import ParallelContext
    from slopllm_b200.runtime.workspace import walk_tensors
    from slopllm_b200.utils.sizing import dense_weight_bytes
    cfg = DenseConfig(num_hidden_layers=2, vocab_size=512, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=4, head_dim=64)
    path = fp8_checkpoint(tmp_path / "model", cfg, keep)
    if keep != ("q_proj", "k_proj", "down_proj"):
        cfg, model = load_dense_model(path, ParallelContext(device=torch.device("cpu")), act_dtype="e4m3")
        w = model.w
    else:                                                 # (q, k and v are one matrix: nothing takes rows in 8 bits, the plan counts it all the same)
        from slopllm_b200.checkpoint.safetensors_io import load_dir
        from slopllm_b200.models.dense import assemble_dense_weights
        w = assemble_dense_weights(cfg, load_dir(path), "cpu", torch.bfloat16, keep_fp8=True)
    seen = {}
    walk_tensors(w, lambda t: seen.setdefault(t.data_ptr(), t.numel() * t.element_size()))
    assert dense_weight_bytes(cfg, 1, fp8=set(_tensor_names(path))) == sum(seen.values())


def test_what_a_layer_calls(monkeypatch):
    """Which operators a forward pass goes through, with which weights, epsilon and types of results: what a comparison of logits is too wide to see."""
    from slopllm_b200.models.dense import DenseConfig, DenseModel, random_dense_model
    from slopllm_b200.parallel.dist import ParallelContext
    from slopllm_b200.runtime.engine import Engine
    cfg = DenseConfig(num_hidden_layers=2, vocab_size=512, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=4, head_dim=64,
                      rms_norm_eps=3e-3)
    w, _ = random_dense_model(cfg, 0, "cpu", torch.float32, fp8=True)
    told = []

    def spy(name, which):
        plain = getattr(F8, name)

        def call(*args, **kw):
            told.append((name, *which(*args, **kw)))
            return plain(*args, **kw)
        monkeypatch.setattr(F8, name, call)

    at = {id(x): (i, n) for i, lw in enumerate(w.layers) for n in ("w_qkv", "o_proj", "mlp_w13", "mlp_w2", "input_norm", "post_attn_norm") for x in [getattr(lw, n)]}
    spy("fp8_add_rmsnorm", lambda x, r, n, eps: (at[id(n)], eps, r is None))
    spy("fp8_rows", lambda x: (tuple(x.shape),))
    spy("fp8_linear", lambda rows, m, out_f32=False: (at[id(m)], out_f32))
    spy("fp8_gate_up", lambda rows, m: (at[id(m)],))
    eng = Engine(cfg, DenseModel(cfg, w, ParallelContext(device=torch.device("cpu")), act_dtype="e4m3"), num_pages=8, max_batch=2, max_seq_len=256)
    s = eng.kv.new_sequence()
    eng.prefill([s], [[5, 6, 7]], chunk_size=32)
    want = []
    for i in (0, 1):
        want += [("fp8_add_rmsnorm", (i, "input_norm"), 3e-3, i == 0), ("fp8_linear", (i, "w_qkv"), True), ("fp8_rows", (3, 256)), ("fp8_linear", (i, "o_proj"), True),
                 ("fp8_add_rmsnorm", (i, "post_attn_norm"), 3e-3, False), ("fp8_gate_up", (i, "mlp_w13")), ("fp8_linear", (i, "mlp_w13"), True),
                 ("fp8_linear", (i, "mlp_w2"), True)]
    assert told == want

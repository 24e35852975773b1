"""Qwen3 / Qwen3.5 from FP8 checkpoints with activations in 8 bits (`--act-dtype e4m3`): the engine against the whole-sequence implementation of
`test_dense_models.py` whose FP8 products take rows of the format, two ranks, graphs, and the command line."""
import argparse
import json
import struct

import pytest
import torch

from fp8_util import nearest
from slopllm_b200.models.dense import DenseConfig, DenseModel, assemble_dense_weights, load_dense_model, random_dense_model
from slopllm_b200.ops import dense as D
from slopllm_b200.ops import quant
from slopllm_b200.ops import reference as R
from slopllm_b200.parallel.dist import ParallelContext
from slopllm_b200.runtime.engine import Engine
from test_dense_models import oracle_logits
from mp_util import run_ranks


class Fp8Matrix:
    """An FP8 weight in the whole-sequence implementation: `h @ w.to(...).t()` multiplies the values that rows of `h` have in 8 bits, in 64 bits."""

    def __init__(self, codes, scale):
        self.w = (codes.double() * scale.double().repeat_interleave(128, 0)[:codes.shape[0]].repeat_interleave(128, 1)[:, :codes.shape[1]]).t()

    def to(self, *_):
        return self

    def t(self):
        return self

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        h, m = args
        return (nearest(h.double())[0] @ m.w).float()


def oracle(cfg, tensors, ids):
    """Logits of the last token.  (No norms of queries and keys where there are none.)"""
    t = {n: Fp8Matrix(x, tensors[n + "_scale_inv"]) if n + "_scale_inv" in tensors else x for n, x in tensors.items()}
    plain, none = R.rmsnorm, torch.ones(cfg.head_dim)
    bare = not any(n.endswith("q_norm.weight") for n in tensors)
    if bare:
        for i in range(cfg.num_hidden_layers):
            for x in "qk":
                t[f"{cfg.weight_prefix}layers.{i}.self_attn.{x}_norm.weight"] = none
    with pytest.MonkeyPatch.context() as m:
        m.setattr(R, "rmsnorm", lambda x, w, eps: x if bare and x.dim() == 3 else plain(x, w, eps))
        return oracle_logits(cfg, t, torch.tensor(ids))[-1]


def bare_model(cfg, rank=0, world=1):
    """Weights for the CPU without norms of queries and keys, which would leave them in bf16: rows of the engine and of the whole sequence then are the same
    up to fp32 before they are rounded to 8 bits.  Larger differences would grow from product to product (a code is 2^-3 of a value)."""
    _, tensors = random_dense_model(cfg, seed=3, device="cpu", dtype=torch.float32, fp8=True)
    tensors = {n: t for n, t in tensors.items() if not n.endswith(("q_norm.weight", "k_norm.weight"))}
    return assemble_dense_weights(cfg, tensors, "cpu", torch.float32, rank, world, keep_fp8=True), tensors


def engine(cfg, w, device, **kw):
    model = DenseModel(cfg, w, ParallelContext(device=torch.device(device)), act_dtype="e4m3")
    return Engine(cfg, model, num_pages=24, max_batch=4, max_seq_len=512, **kw)


def errors(cfg, w, tensors, device, prompt, steps, chunk, **kw):
    """Chunked prefill, then decode steps fed with the oracle's tokens: largest error of the logits relative to their peak at each."""
    eng = engine(cfg, w, device, **kw)
    s, _ = eng.kv.start_request(prompt)
    _, hid = eng.prefill([s], [prompt], chunk_size=chunk, want_hidden=True)
    got, ids, errs = eng.model.compute_logits(hid[0])[-1].float().cpu(), list(prompt), []
    for _ in range(steps):
        want = oracle(cfg, tensors, ids)
        errs.append(((want - got).abs().max() / want.abs().max()).item())
        ids.append(int(want.argmax()))
        got = eng.step([s], [[ids[-1]]], [[0]])[0].cpu()
    return errs


@pytest.mark.parametrize("hybrid", [False, True])
def test_engine_on_the_cpu(hybrid):
    """Attention layers alone have every rounding of the oracle: the bound of the plain checkpoint's test.  The recurrent layers leave theirs in bf16: the bound of
    the test on a GPU, where all rows are."""
    cfg = DenseConfig.tiny(hybrid=hybrid)
    w, tensors = bare_model(cfg)
    prompt = torch.randint(2, cfg.vocab_size, (70,), generator=torch.Generator().manual_seed(5)).tolist()
    errs = errors(cfg, w, tensors, "cpu", prompt, 4, 32)
    assert max(errs) < (0.12 if hybrid else 2e-2), errs


@pytest.mark.gpu
@pytest.mark.parametrize("hybrid,graph", [(False, False), (False, True), (True, True)])
def test_engine_on_a_gpu(hybrid, graph):
    """bf16 rows differ from the oracle's before they are rounded to 8 bits, and differences grow until the roundings of the two have nothing to do with each
    other.  A rounding to four bits is off by 2^-4 of a value at most, evenly spread, and by 2^-5 where the significand is near 2: 0.026 of the
    value's size in the root mean square, 0.037 between two independent ones, and as much of a product's result.  A sublayer has two such products
    in a row (0.052), and what it reads is off by that from the sublayers in front (0.075 together).  The largest of 512 errors stands to the largest
    of 512 logits as their sizes do, give or take half: 0.11, and 0.01 for bf16 itself."""
    cfg = DenseConfig.tiny(hybrid=hybrid)
    _, tensors = random_dense_model(cfg, seed=3, device="cpu", dtype=torch.float32, fp8=True)
    w, _ = random_dense_model(cfg, seed=3, device="cuda", dtype=torch.bfloat16, fp8=True)
    assert all(m.is_fp8 for layer in w.layers for m in (layer.mlp_w13, layer.mlp_w2))
    prompt = torch.randint(2, cfg.vocab_size, (150,), generator=torch.Generator().manual_seed(7)).tolist()
    errs = errors(cfg, w, tensors, "cuda", prompt, 4, 64, cuda_graph=graph)
    assert max(errs) < 0.12, errs


@pytest.mark.gpu
def test_captured_steps_and_batches():
    """A captured decode step gives the eager one's tokens, for one sequence and several, over the 8-bit cache as well."""
    cfg = DenseConfig.tiny()
    w, _ = random_dense_model(cfg, seed=4, device="cuda", dtype=torch.bfloat16, fp8=True)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(2, cfg.vocab_size, (n,), generator=g).tolist() for n in (5, 150, 64)]
    for kv_dtype in (None, "e4m3"):
        told = []
        for graph in (False, True):
            model = DenseModel(cfg, w, ParallelContext(device=torch.device("cuda", 0)), kv_dtype=kv_dtype, act_dtype="e4m3")
            eng = Engine(cfg, model, num_pages=24, max_batch=4, max_seq_len=512, cuda_graph=graph)
            seqs = [eng.kv.new_sequence() for _ in prompts]
            last, _ = eng.prefill(seqs, prompts, chunk_size=128)
            out = [last]
            for _ in range(6):
                out.append(eng.decode_step(seqs, out[-1]))
            told.append(out)
        assert told[0] == told[1]


def _two_ranks(rank, world):
    from slopllm_b200.parallel.dist import init_from_env
    cfg = DenseConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=4, head_dim=64, vocab_size=512,
                      eos_token_ids=[1])
    prompt = torch.randint(2, cfg.vocab_size, (40,), generator=torch.Generator().manual_seed(5)).tolist()

    def serve(ctx, r, n):
        w, _ = bare_model(cfg, r, n)
        model = DenseModel(cfg, w, ctx, act_dtype="e4m3")
        eng = Engine(cfg, model, num_pages=8, max_batch=2, max_seq_len=256)
        s, _ = eng.kv.start_request(prompt)
        _, hid = eng.prefill([s], [prompt], chunk_size=32, want_hidden=True)
        return model.compute_logits(hid[0])[-1].float(), all(x.fp8_input for x in model.sublayers) and all(x.o_proj.is_fp8 and x.mlp_w2.is_fp8 for x in w.layers)

    got, eight = serve(init_from_env("gloo"), rank, world)
    want, _ = serve(ParallelContext(device=torch.device("cpu")), 0, 1)
    return eight, ((got - want).abs().max() / want.abs().max()).item()


def test_two_ranks():
    """Shards whose groups of 128 values are whole: the same rows but for sums that are split over the ranks, which can move a value to the next code."""
    for eight, err in run_ranks(_two_ranks, 2):
        assert eight and err < 2e-2, err


def write_checkpoint(path, cfg, fp8=True):
    _, tensors = random_dense_model(cfg, seed=3, device="cpu", dtype=torch.bfloat16, fp8=fp8)
    names = {torch.bfloat16: "BF16", torch.float32: "F32", torch.float8_e4m3fn: "F8_E4M3"}
    head, blobs, at = {}, [], 0
    for n, t in tensors.items():
        raw = t.contiguous().view(torch.uint8).numpy().tobytes()
        head[n] = {"dtype": names[t.dtype], "shape": list(t.shape), "data_offsets": [at, at + len(raw)]}
        at += len(raw)
        blobs.append(raw)
    text = json.dumps(head).encode()
    text += b" " * (-len(text) % 8)
    (path / "model.safetensors").write_bytes(struct.pack("<Q", len(text)) + text + b"".join(blobs))
    (path / "config.json").write_text(json.dumps(dict(
        model_type="qwen3", hidden_size=cfg.hidden_size, intermediate_size=cfg.intermediate_size, num_hidden_layers=cfg.num_hidden_layers,
        num_attention_heads=cfg.num_attention_heads, num_key_value_heads=cfg.num_key_value_heads, head_dim=cfg.head_dim, vocab_size=cfg.vocab_size)))


def test_checkpoints_and_commands(tmp_path, capsys):
    from slopllm_b200.cli import model_cli
    from slopllm_b200.cli import plan as plan_cli
    from slopllm_b200.models.registry import MODEL_REGISTRY, load_any, load_registered
    cfg, cpu = DenseConfig.tiny(), ParallelContext(device=torch.device("cpu"))
    write_checkpoint(tmp_path, cfg)
    _, model = load_any(str(tmp_path), cpu, act_dtype="e4m3")
    assert model.act_dtype == "e4m3" and model.w.layers[0].w_qkv.is_fp8 and all(s.fp8_input for s in model.sublayers)
    _, model = load_dense_model(str(tmp_path), cpu)
    assert not model.w.layers[0].w_qkv.is_fp8 and not any(s.fp8_input for s in model.sublayers)
    _, model, _ = model_cli._random_model("qwen35-tiny", cpu, 0, None, None, "e4m3")
    assert [s.fp8_input for s in model.sublayers[::2]] == [k == "full_attention" for k in model.cfg.layer_types] and all(s.fp8_input for s in model.sublayers[1::2])
    ap = argparse.ArgumentParser()
    model_cli.add_model_args(ap)
    args = lambda *a: ap.parse_args(["--cpu", "--act-dtype", "e4m3", "--max-pages", "8", *a])
    rt = model_cli.build_runtime(args("--random-init", "qwen3-tiny"), with_scheduler=False)
    assert rt.engine.model.act_dtype == "e4m3"
    # refusals: other families, checkpoints without FP8 projections, rows that are no multiple of 16
    with pytest.raises(ValueError, match="does not take activations"):
        load_registered(MODEL_REGISTRY["zemezen"], str(tmp_path), cpu, act_dtype="e4m3")
    for spec in ("zemezen-tiny", "tiny"):
        with pytest.raises(SystemExit, match="does not take activations"):
            model_cli._random_model(spec, cpu, 0, None, None, "e4m3")
    for spec in ("glm5", "gidisun"):
        with pytest.raises(SystemExit):
            plan_cli.main(["--random-init", spec, "--act-dtype", "e4m3"])
    plain = tmp_path / "plain"
    plain.mkdir()
    write_checkpoint(plain, cfg, fp8=False)
    with pytest.raises(ValueError, match="has none"):
        load_dense_model(str(plain), cpu, act_dtype="e4m3")
    with pytest.raises(SystemExit, match="has none"):
        model_cli.build_runtime(args("--model", str(plain)))
    w, _ = random_dense_model(cfg, seed=1, device="cpu", dtype=torch.float32)
    with pytest.raises(ValueError, match="have none"):
        DenseModel(cfg, w, cpu, act_dtype="e4m3")
    for bad in (DenseConfig(hidden_size=1000), DenseConfig(intermediate_size=200), DenseConfig(num_attention_heads=1, num_key_value_heads=1, head_dim=72)):
        with pytest.raises(ValueError, match="multiples of 16"):
            DenseModel(bad, None, cpu, act_dtype="e4m3")
    with pytest.raises(ValueError, match="no activations of type"):
        DenseModel(cfg, w, cpu, act_dtype="int8")
    capsys.readouterr()
    weights = []
    for extra in ([], ["--act-dtype", "e4m3"]):
        assert plan_cli.main(["--random-init", "qwen3", "--max-pages", "64", *extra]) == 0
        weights.append(json.loads(capsys.readouterr().out.splitlines()[-1])["weights_bytes"])
    assert weights[1] < 0.8 * weights[0]


def test_weights_that_are_partly_fp8():
    """A product whose weight was expanded (a shard's edge inside a block) takes its rows as before, beside products in 8 bits."""
    cfg = DenseConfig.tiny()
    _, tensors = bare_model(cfg)
    prompt = torch.randint(2, cfg.vocab_size, (20,), generator=torch.Generator().manual_seed(5)).tolist()
    for some in (("down_proj",), ("gate_proj", "up_proj"), ("q_proj", "k_proj", "v_proj"), ("o_proj", "down_proj")):
        t = dict(tensors)
        for n in [n for n in tensors if any(x in n for x in some) and n.endswith("_scale_inv")]:
            t[n[:-10]] = D.fp8_block_dequant(t[n[:-10]], t.pop(n))
        w = assemble_dense_weights(cfg, t, "cpu", torch.float32, keep_fp8=True)
        if "up_proj" in some:                            # the activation then is not in 8 bits, nor what it is multiplied with
            for n in [n for n in t if n.endswith("down_proj.weight")]:
                t[n] = quant.fp8_block_dequantize(t[n], t.pop(n + "_scale_inv"))
        errs = errors(cfg, w, t, "cpu", prompt, 2, 32)
        assert max(errs) < 2e-2, (some, errs)


@pytest.mark.gpu
def test_weights_that_are_partly_fp8_on_a_gpu():
    """A feed-forward of rows in 8 bits whose down projection is bf16: as its parts."""
    from slopllm_b200.models.weights import LinearWeight
    from slopllm_b200.ops import fp8 as F8
    from slopllm_b200.ops.cuda_ops import CudaOps
    cfg = DenseConfig.tiny()
    w, _ = random_dense_model(cfg, seed=3, device="cuda", dtype=torch.bfloat16, fp8=True)
    layer, ops = w.layers[0], CudaOps(cfg)
    rows = F8.fp8_rows(torch.randn(5, cfg.hidden_size, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    layer.mlp_w2 = LinearWeight(layer.mlp_w2.dequant(torch.bfloat16))
    y = ops.dense_mlp(rows, layer)
    gu = F8.fp8_linear(rows, layer.mlp_w13).double()
    g, u = gu.chunk(2, -1)
    want = (g * torch.sigmoid(g) * u) @ layer.mlp_w2.weight.double().t()
    # the activation is rounded to bf16 (2^-8 of each value), sums are fp32
    most = (g * torch.sigmoid(g) * u).abs() @ layer.mlp_w2.weight.double().abs().t()
    assert y.dtype == torch.float32 and ((y.double() - want).abs() <= 2.0 ** -7 * most).all()

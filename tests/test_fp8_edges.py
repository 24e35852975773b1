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

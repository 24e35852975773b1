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

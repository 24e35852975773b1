"""Rows in 8 bits and their products with FP8 weights: the definition on the CPU, and what is refused."""
import pytest
import torch

from fp8_util import held, near, nearest, same, some_rows, weight
from slopllm_b200.models.weights import LinearWeight
from slopllm_b200.ops import fp8 as F8


@pytest.mark.parametrize("t,k", [(1, 16), (3, 128), (2, 144), (5, 1040), (0, 128)])
def test_rows(t, k):
    x = torch.randn(t, k, generator=torch.Generator().manual_seed(t + k)) * torch.tensor([1e-3, 1.0, 300.0, 1e6, 1.0])[:t, None]
    assert same(F8.fp8_rows(x), x.double())
    assert same(F8.fp8_silu_mul(torch.cat([x, x + 1], 1)), x.double() * torch.sigmoid(x.double()) * (x + 1).double())
    values = F8.fp8_values(F8.fp8_rows(x))
    assert values.dtype == torch.bfloat16 and (values.double() == nearest(x.double())[0]).all()


def test_exponents_at_their_limits():
    edge = 448.0 * 2.0 ** torch.arange(-3, 4)
    for x, step in ((edge, 0), (torch.nextafter(edge, edge * 2), 1), (torch.nextafter(edge, edge * 0), 0)):
        row = torch.zeros(7, 128)
        row[:, 5] = x
        rows = F8.fp8_rows(row)
        assert rows.exps[:, 0].tolist() == [127 + e + step for e in range(-3, 4)]
    row = torch.zeros(4, 128)
    row[1, 0], row[2, 0], row[3, 0] = 1e-30, 3e38, float("inf")
    row[3, 1] = 2.0
    rows = F8.fp8_rows(row)
    assert rows.exps[:, 0].tolist() == [67, 67, 187, 127 + 1 - 8]
    assert rows.codes[2, 0] == 0x7e and rows.codes[3, 0] & 127 == 127 and held(rows)[3, 1] == 2.0


def test_norm():
    g = torch.Generator().manual_seed(0)
    x, res, w = torch.randn(3, 272, generator=g), torch.randn(3, 272, generator=g) * 4, torch.randn(272, generator=g)
    rows, r = F8.fp8_add_rmsnorm(x, res, w, 1e-6)
    assert (r == res + x).all()
    v = r.double()
    assert same(rows, v / (v.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double())
    first, r = F8.fp8_add_rmsnorm(x.bfloat16(), None, w.bfloat16(), 1e-6)
    assert (r == x.bfloat16().float()).all()


def test_products():
    w, values = weight(200, 272, device="cpu")
    rows = some_rows(5, 272, device="cpu")
    assert near(F8.fp8_linear(rows, w, out_f32=True), rows, values)
    assert near(F8.fp8_linear(rows, w), rows, values)
    w, values = weight(2 * 48, 272, device="cpu")
    gu = F8.fp8_linear(rows, w, out_f32=True).double()
    assert same(F8.fp8_gate_up(rows, w), gu[:, :48] * torch.sigmoid(gu[:, :48]) * gu[:, 48:])


def test_refusals():
    rows = some_rows(4, 256, device="cpu")
    w, _ = weight(64, 256, device="cpu")
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    for codes, exps in ((u8(4, 256), u8(4, 3)), (u8(4, 256), u8(3, 16)[:, :2]), (torch.zeros(4, 256), u8(4, 16)[:, :2]), (u8(4, 24), u8(4, 16)[:, :1]),
                        (u8(4, 256), u8(4, 2)), (u8(4, 264)[:, :256], u8(4, 16)[:, :2]), (u8(4, 512)[:, ::2], u8(4, 16)[:, :2]), (u8(4, 0), u8(4, 0)),
                        (u8(256), u8(2))):
        with pytest.raises(ValueError):
            F8.Fp8Rows(codes, exps)
    F8.Fp8Rows(u8(1, 256), u8(1, 2))
    for bad in (LinearWeight(torch.zeros(64, 256)), LinearWeight(w.weight[:, :128], fp8_scale=w.fp8_scale), LinearWeight(w.weight, fp8_scale=w.fp8_scale[:, :1]),
                LinearWeight(w.weight, fp8_scale=w.fp8_scale[:0])):
        with pytest.raises(ValueError):
            F8.fp8_linear(rows, bad)
    with pytest.raises(ValueError):
        F8.fp8_gate_up(rows, weight(72, 256, device="cpu")[0])
    x = torch.randn(4, 256)
    for call in (lambda: F8.fp8_rows(torch.randn(4, 40)), lambda: F8.fp8_rows(torch.randn(256)), lambda: F8.fp8_silu_mul(torch.randn(4, 33)),
                 lambda: F8.fp8_silu_mul(torch.randn(4, 40)), lambda: F8.fp8_add_rmsnorm(x, x[:3], torch.ones(256), 1e-6),
                 lambda: F8.fp8_add_rmsnorm(x, x, torch.ones(128), 1e-6)):
        with pytest.raises(ValueError):
            call()


def test_more_rows_and_wider_strides_than_the_kernels_count():
    """Rows, values and strides of 2^31 and more: refused, or (rows that are only read) a copy."""
    far = lambda n, k, dtype: torch.empty(n, 2 ** 31, dtype=dtype, device="meta")[:, :k]
    u8, one = torch.uint8, torch.zeros(1, 16)
    near_by, spread = torch.empty(2, 16, dtype=u8, device="meta"), torch.empty(1, 16, dtype=u8, device="meta").expand(2 ** 31, 16)
    tall = LinearWeight(torch.zeros(1, 16, dtype=u8).expand(2 ** 31, 16), fp8_scale=torch.ones(1, 1).expand(2 ** 24, 1))
    for codes, exps in ((far(2, 16, u8), near_by[:, :1]), (near_by, far(2, 1, u8)), (spread, spread[:, :1])):
        with pytest.raises(ValueError, match="up to"):
            F8.Fp8Rows(codes, exps)
    for call in (lambda: F8.fp8_rows(one.expand(2 ** 31, 16)), lambda: F8.fp8_silu_mul(one.expand(2 ** 32 + 1, 16)),
                 lambda: F8.fp8_rows(one[:, :1].expand(1, 2 ** 31)),
                 lambda: F8.fp8_add_rmsnorm(one.expand(2 ** 31, 16), None, torch.ones(16), 1e-6),
                 lambda: F8.fp8_linear(some_rows(1, 16, device="cpu"), tall)):
        with pytest.raises(ValueError, match="up to"):
            call()
    for dtype in (torch.bfloat16, torch.float32):
        x = far(2, 32, dtype)
        assert x.stride(0) == 2 ** 31 and F8._aligned(x).stride() == (32, 1)
        assert F8._aligned(x[:1]).stride(0) == 2 ** 31                           # (one row: its stride is not used)

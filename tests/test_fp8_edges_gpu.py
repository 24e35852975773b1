"""Rows in 8 bits and their products on a GPU where they are easily wrong: numbers by the limits of fp32, status words that a captured call makes, strides, what lies
around results, and the activation that is made in a product's epilogue."""
import numpy as np
import pytest
import torch

from fp8_util import held, near, nearest, same, some_rows, weight
from slopllm_b200.models.weights import LinearWeight
from slopllm_b200.ops import fp8 as F8
from slopllm_b200.ops import native as N
from slopllm_b200.ops import tcgen05

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def silu_mul(gu):
    g, u = gu.double().chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def rms(r, w, eps):
    v = r.double()
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.double()


# ---- numbers by the limits of fp32 -------------------------------------------------------------------------------------------------

def test_norms_whose_factor_is_subnormal():
    """Rows of 3e38: 1 / rms lies below 2^-126, where fp32 has fewer bits.  Gains put every value next to the middle between two codes."""
    g, largest, h = np.random.default_rng(2), np.finfo(np.float32).max, 4096
    shape, rows = g.uniform(0.99, 1.0, h), 0
    for size in np.linspace(0.9, 1.0, 4000):
        v = (shape * size * largest).astype(np.float32)
        inv = 1 / np.sqrt(np.mean(v.astype(np.float64) ** 2))
        if abs(np.float64(np.float32(inv)) / inv - 1) < 3.75 * 2.0 ** -24:
            continue
        middles = (1 + (g.integers(0, 2, h) + 0.5) / 8) * 2.0 ** g.integers(3, 8, h)
        w = torch.from_numpy((middles / (v.astype(np.float64) * inv)).astype(np.float32)).cuda()
        x = torch.from_numpy(v).cuda()[None]
        got, _ = F8.fp8_add_rmsnorm(x, None, w, 0.0)
        assert same(got, rms(x, w, 0.0)), size
        rows += 1
    assert rows > 50
    x = torch.randn(300, 1040, generator=gen(0), device="cuda").clamp(-3, 3) * 1e38
    w = torch.randn(1040, generator=gen(1), device="cuda")
    for weight_type in (torch.float32, torch.bfloat16):
        assert same(F8.fp8_add_rmsnorm(x, None, w.to(weight_type), 1e-6)[0], rms(x, w.to(weight_type), 1e-6))

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gates_that_are_subnormal(dtype):
    """silu(gate) below 2^-126 times a large value, and the other way round."""
    size = torch.exp2(torch.rand(64, 512, generator=gen(2), device="cuda") * 14 - 138)
    gate = size * torch.where(torch.rand(64, 512, generator=gen(3), device="cuda") < 0.5, -1.0, 1.0)
    up = torch.randn(64, 512, generator=gen(4), device="cuda").clamp(-3, 3) * 1e38
    for gu in (torch.cat([gate, up], 1), torch.cat([up.abs(), gate], 1)):
        assert same(F8.fp8_silu_mul(gu.to(dtype)), silu_mul(gu.to(dtype)))

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gains_that_bring_tiny_values_back(dtype):
    """Values 2^-140 of the row's size, times gains of 2^126."""
    x = torch.randn(20, 1024, generator=gen(5), device="cuda")
    x[:, 128:] *= 2.0 ** -140
    w = torch.randn(1024, generator=gen(6), device="cuda").clamp(-3, 3)
    w[128:] *= 2.0 ** 126
    x, w = x.to(dtype), w.to(dtype)
    for size in (1.0, 2.0 ** 40):
        assert same(F8.fp8_add_rmsnorm(x.float() * size, None, w, 0.0)[0], rms(x.float() * size, w, 0.0))

def test_products_by_the_largest_number():
    """Gate times up where fp32 rounds to infinity and 64 bits to the largest finite number: a code, not NaN; beyond it, NaN."""
    limit = (2 - 2.0 ** -24) * 2.0 ** 127                 # from here on fp32 has infinity
    g = np.random.default_rng(0)
    gate = g.uniform(16.7, 24, 4096).astype(np.float32)
    up = (limit / gate.astype(np.float64)).astype(np.float32)
    up = np.stack([np.nextafter(up, np.float32(0)), up, np.nextafter(up, np.float32(np.inf))])
    d = gate.astype(np.float64) / (1 + np.exp(-gate.astype(np.float64))) * up
    with np.errstate(over="ignore"):
        assert (np.isinf(gate * up) & (d < limit)).any()
    rows = torch.from_numpy(np.concatenate([np.stack([gate] * 3), up], 1)).cuda()
    assert same(F8.fp8_silu_mul(rows), silu_mul(rows))
    # the norm: rows of one large value, gains that take it there
    x = torch.zeros(1, 256, device="cuda")
    x[0, 5] = 3.0
    for step in range(-3, 4):
        w = torch.ones(256, device="cuda")
        w[5] = float(np.float32(limit / 16)) * (1 + step * 2.0 ** -23)
        for value in (3.0, 1.7, 1.1):
            x[0, 5] = value
            assert same(F8.fp8_add_rmsnorm(x, None, w, 0.0)[0], rms(x, w, 0.0))


# ---- status words, strides, what lies around results -----------------------------------------------------------------------------------

def test_status_words_that_a_captured_call_makes(monkeypatch):
    """A device's first call may be a captured one.  A replay leaves what a kernel has written into the status words."""
    rows, (w, _) = some_rows(4, 256), weight(64, 256)
    F8.fp8_linear(rows, w)
    monkeypatch.setattr(tcgen05, "_err", {})
    monkeypatch.setattr(F8, "_status", lambda device: tcgen05.error_flag(torch.device("cuda", device)).data_ptr())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        F8.fp8_linear(rows, w)
    words = tcgen05.error_flag(rows.device)
    assert words.tolist() == [0] * tcgen05.ERROR_WORDS
    words[0] = 7
    graph.replay()
    assert words[0] == 7
    with pytest.raises(N.NativeError, match="site 7"):
        tcgen05.check_errors(rows.device)
    assert words.tolist() == [0] * tcgen05.ERROR_WORDS

@pytest.mark.parametrize("t", [3, 200])
def test_scales_whose_rows_lie_in_one_another(t):
    """Scales that are one row for all blocks, a single row with a stride of its own, windows that overlap: as their contiguous copies."""
    (w, _), rows = weight(300, 400, 20), some_rows(t, 400, 21)
    s = w.fp8_scale
    for scale in (s[:1].expand(3, 4), s.flatten()[:8].as_strided((3, 4), (2, 1)), s.flatten()[:8].as_strided((3, 4), (1, 2))):
        got = F8.fp8_linear(rows, LinearWeight(w.weight, fp8_scale=scale), out_f32=True)
        assert torch.equal(got, F8.fp8_linear(rows, LinearWeight(w.weight, fp8_scale=scale.contiguous()), out_f32=True))
    few = LinearWeight(w.weight[:100], fp8_scale=s[:1].as_strided((1, 4), (1, 1)))
    assert torch.equal(F8.fp8_linear(rows, few), F8.fp8_linear(rows, LinearWeight(w.weight[:100], fp8_scale=s[:1].clone())))
    gated, _ = weight(512, 400, 22)
    scale = gated.fp8_scale[:1].expand(4, 4)
    got, want = (F8.fp8_gate_up(rows, LinearWeight(gated.weight, fp8_scale=x)) for x in (scale, scale.contiguous()))
    assert torch.equal(got.codes, want.codes) and torch.equal(got.exps, want.exps)

@pytest.mark.parametrize("t", [3, 200])
def test_weights_whose_rows_lie_in_one_another(t):
    """One row for all columns, windows of a longer row, a single row with a stride of its own."""
    (w, _), rows = weight(256, 400, 23), some_rows(t, 400, 24)
    codes = w.weight.view(torch.uint8)
    for part in (codes[:1].expand(256, 400), codes.flatten().as_strided((256, 400), (16, 1)), codes[:1].as_strided((1, 400), (16, 1))):
        scale = w.fp8_scale[:-(-part.shape[0] // 128)]
        got = F8.fp8_linear(rows, LinearWeight(part, fp8_scale=scale), out_f32=True)
        assert torch.equal(got, F8.fp8_linear(rows, LinearWeight(part.clone(memory_format=torch.contiguous_format), fp8_scale=scale), out_f32=True))
    tcgen05.check_errors(rows.device)

def test_more_columns_than_a_grid_has():
    """Refused in words, and not copied before."""
    n = 65535 * 128 + 1
    codes = torch.zeros(1, 16, dtype=torch.uint8, device="cuda").expand(n, 16)
    w = LinearWeight(codes, fp8_scale=torch.ones(1, 1, device="cuda").expand(65536, 1))
    for t in (1, 100):
        with pytest.raises(ValueError, match="up to 8388480"):
            F8.fp8_linear(some_rows(t, 16), w)
    y = F8.fp8_linear(some_rows(1, 16), LinearWeight(codes[1:].contiguous(), fp8_scale=w.fp8_scale[1:]))
    assert y.shape == (1, n - 1) and (y == 0).all()

class Around:
    """Rows of `width` bytes, `ld` apart, in a piece of memory whose every other byte is 0xa5 and has to stay so, but for those up to the next multiple of `piece`
    behind a row."""

    def __init__(self, rows, width, ld, piece=1, margin=8192):
        self.rows, self.width, self.ld, self.margin, self.written = rows, width, ld, margin, -(-width // piece) * piece
        self.space = torch.full((2 * margin + rows * ld,), 0xa5, dtype=torch.uint8, device="cuda")
        self.at = self.space.data_ptr() + margin

    def get(self, dtype=torch.uint8):
        """The rows, once nothing else is found to be written."""
        inside = self.space[self.margin:self.margin + self.rows * self.ld].view(self.rows, self.ld)
        for other in (self.space[:self.margin], self.space[self.margin + self.rows * self.ld:], inside[:, self.written:]):
            assert (other == 0xa5).all()
        return inside[:, :self.width].contiguous().view(dtype)


# forms of the product: one SM with 16, 32 and 64 rows, pairs with 128 and 256 columns, shares of K
@pytest.mark.parametrize("t,n,k", [(1, 1, 16), (3, 130, 4112), (17, 130, 400), (40, 1001, 400), (65, 1001, 400), (129, 1001, 2064), (257, 130, 400), (1500, 1001, 400),
                                   (4500, 130, 272), (333, 2321, 2064), (300, 1001, 144), (2500, 2321, 144), (1000, 1001, 16)])
@pytest.mark.parametrize("f32", [True, False])
def test_what_lies_around_a_product(t, n, k, f32):
    """Columns behind the last piece of 16 bytes, rows behind the last and what is in front of the first are left as they were."""
    (w, _), rows = weight(n, k, 25), some_rows(t, k, 26)
    size = 4 if f32 else 2
    for more in (0, 32):
        ld = -(-n * size // 16) * 16 + more
        y = Around(t, n * size, ld, 16)
        F8._multiply("sl_fp8_linear", 0, rows, w.weight, n, w.fp8_scale, y.at, ld // size, f32)
        assert torch.equal(y.get(torch.float32 if f32 else torch.bfloat16), F8.fp8_linear(rows, w, out_f32=f32))
    tcgen05.check_errors(rows.device)


@pytest.mark.parametrize("t,inner,k", [(65, 128, 144), (129, 384, 400), (257, 256, 144), (300, 512, 400), (2100, 1152, 272)])
def test_what_lies_around_gated_rows_of_a_product(t, inner, k):
    (w, _), rows = weight(2 * inner, k, 27), some_rows(t, k, 28)
    codes, exps = Around(t, inner, inner + 32), Around(t, inner // 128, -(-inner // 2048) * 16 + 16)
    F8._multiply("sl_fp8_gate_up", 0, rows, w.weight, 2 * inner, w.fp8_scale, codes.at, codes.ld, False, exps.at, exps.ld)
    want = F8.fp8_silu_mul(F8.fp8_linear(rows, w, out_f32=True))
    assert (exps.get() == want.exps).all() and (codes.get() != want.codes).float().mean() < 1e-4
    if F8._on_pairs(t, 2 * inner, k):
        got = F8.fp8_gate_up(rows, w)
        assert torch.equal(codes.get(), got.codes) and torch.equal(exps.get(), got.exps)
    tcgen05.check_errors(rows.device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t,k", [(1, 16), (3, 144), (17, 272), (300, 4112), (2500, 1040)])
def test_what_lies_around_rows(t, k, dtype):
    """Codes, exponents, residuals and values that are read back."""
    import ctypes as C
    x = torch.randn(t, 2 * k, generator=gen(29), device="cuda").to(dtype)
    w, groups = torch.rand(k, generator=gen(30), device="cuda"), -(-k // 128)
    f32 = dtype is torch.float32
    res = torch.randn(t, k, generator=gen(31), device="cuda")

    def rows():
        return Around(t, k, k + 16), Around(t, groups, F8._padded(k) + 16)

    def put(codes, exps):
        return codes.at, codes.ld, exps.at, exps.ld

    for gated, want in ((False, F8.fp8_rows(x[:, :k])), (True, F8.fp8_silu_mul(x))):
        codes, exps = rows()
        p = F8.Fp8RowsParams(x.data_ptr(), x.stride(0), t, k, *put(codes, exps))
        F8._call(0, "sl_fp8_rows", C.byref(p), gated, f32)
        assert torch.equal(codes.get(), want.codes) and torch.equal(exps.get(), want.exps)
    values = Around(t, 2 * k, 2 * k)
    p = F8.Fp8ValuesParams(*want._where(), t, k, values.at)
    F8._call(0, "sl_fp8_values", C.byref(p))
    assert torch.equal(values.get(torch.bfloat16), F8.fp8_values(want))
    part = x[:, :k]
    (codes, exps), r = rows(), Around(t, 4 * k, 4 * k)
    p = F8.Fp8NormParams(part.data_ptr(), part.stride(0), res.data_ptr(), res.stride(0), w.data_ptr(), k, 1e-6, r.at, *put(codes, exps))
    F8._call(0, "sl_fp8_add_rmsnorm", C.byref(p), t, f32, True)
    want, r_want = F8.fp8_add_rmsnorm(part, res, w, 1e-6)
    assert torch.equal(codes.get(), want.codes) and torch.equal(exps.get(), want.exps) and torch.equal(r.get(torch.float32), r_want)

def test_residuals_and_scales_far_apart():
    """Rows of the residual and of scales more than 2^31 values apart."""
    step = 2 ** 31 + 64
    space = torch.empty(step + 512, dtype=torch.float32, device="cuda")
    far = torch.as_strided(space, (2, 512), (step, 1))
    far.copy_(torch.randn(2, 512, generator=gen(32), device="cuda"))
    x, w = torch.randn(2, 512, generator=gen(33), device="cuda"), torch.rand(512, generator=gen(34), device="cuda")
    (got, r), (want, r_want) = (F8.fp8_add_rmsnorm(x, a, w, 1e-6) for a in (far, far.contiguous()))
    assert torch.equal(r, r_want) and torch.equal(got.codes, want.codes) and torch.equal(got.exps, want.exps)
    for n in (200, 512):
        (w, _), rows = weight(n, 500 // 16 * 16, 35), some_rows(100, 496, 36)
        scale = torch.as_strided(space, (w.fp8_scale.shape[0], 4), (step // (w.fp8_scale.shape[0] - 1) // 4 * 4, 1))
        assert n > 256 or scale.stride(0) > 2 ** 31
        scale.copy_(w.fp8_scale)
        assert torch.equal(F8.fp8_linear(rows, LinearWeight(w.weight, fp8_scale=scale)), F8.fp8_linear(rows, w))
    tcgen05.check_errors(rows.device)


# ---- the activation in a product's epilogue --------------------------------------------------------------------------------------------
#
# Against `fp8_silu_mul` of the fp32 product, which is the definition's nearest.  Codes may be the neighbour's where the two fp32 values lie on different sides of a
# middle: both are within some 20 units of 2^-24 (gates of -16) of the value, middles are 2^-4 of a value apart or more, so that fewer than
# 2 * 20 * 2^-24 * 2^4 = 4e-5 of evenly spread codes are; an exponent likewise where a group's largest value lies next to a limit, of which these cases have none.
# Products of two codes are not evenly spread, many are a middle themselves: where sums are exact, the value of each code that differs is looked at.

def fused_and_apart(rows, w, t, n, k):
    assert F8._on_pairs(t, n, k)
    return F8.fp8_gate_up(rows, w), F8.fp8_silu_mul(F8.fp8_linear(rows, w, out_f32=True))


def agree(got, want, value=None):
    tcgen05.check_errors(got.device)
    a, b = held(got), held(want)
    assert torch.equal(got.exps, want.exps) and torch.equal(a.isnan(), b.isnan())
    step = torch.exp2(want.exps.double() - 127).repeat_interleave(128, 1)
    off = (a - b).nan_to_num(0.0).abs()
    assert (off <= torch.maximum(2.0 ** -3 * b.nan_to_num(0.0).abs(), 2.0 ** -9 * step)).all()
    if value is None:
        assert (off > 0).sum() <= 2 + 4e-5 * off.numel(), (off > 0).sum()
    else:
        middle = (a + b) / 2
        assert ((off == 0) | ((value - middle).abs() <= 20 * 2.0 ** -24 * middle.abs())).all()


def chosen(gate, up):
    """Rows and weights whose product has column j of weight row i at [j, i]: gates and ups [t, inner] as they are given, up to a power of two."""
    t, inner = gate.shape
    k = -(-t // 128) * 128
    codes = torch.zeros(2 * inner, k, dtype=torch.uint8, device="cuda")
    codes[:inner, :t] = gate.t().to(torch.float8_e4m3fn).view(torch.uint8)
    codes[inner:, :t] = up.t().to(torch.float8_e4m3fn).view(torch.uint8)
    rows = F8.Fp8Rows.allocate(t, k, "cuda")
    rows.codes.copy_(torch.nn.functional.pad(torch.eye(t, device="cuda") * 2.0, (0, k - t)).to(torch.float8_e4m3fn).view(torch.uint8))
    rows.exps.fill_(126)                                  # 2 * 2^-1
    return rows, LinearWeight(codes.view(torch.float8_e4m3fn), fp8_scale=torch.ones(2 * inner // 128, k // 128, device="cuda"))


def test_gates_of_all_sizes_in_the_epilogue():
    """Gates of every code (up to 448 either way: those below -87 are zeros), and around -16, -88 and 88, times ups of every code."""
    t, inner = 254, 512
    codes = torch.tensor([c for c in range(256) if c & 127 != 127], dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).float()
    gate = codes[:, None].expand(t, inner)
    up = codes[torch.randint(0, 254, (t, inner), generator=gen(40), device="cuda")]
    for g in (gate, gate[torch.randperm(254, generator=gen(41), device="cuda")], torch.tensor([-15., -16, -18, -80, -88, -96, 80, 88, 96, 448.], device="cuda")[
            torch.randint(0, 10, (t, inner), generator=gen(42), device="cuda")]):
        rows, w = chosen(g, up)
        got, want = fused_and_apart(rows, w, t, 2 * inner, rows.shape[1])
        value = silu_mul(torch.cat([g.to(torch.float8_e4m3fn).float(), up], 1))
        assert same(want, value)
        agree(got, want, value)


@pytest.mark.parametrize("t,inner,k", [(129, 384, 400), (300, 512, 400), (700, 1024, 528)])
def test_numbers_that_are_not_finite_in_the_epilogue(t, inner, k):
    """A NaN code of a row spoils its row, one of a gate's or an up's weight its column, and no other value or exponent."""
    (w, _), rows = weight(2 * inner, k, 43), some_rows(t, k, 44)
    clean, _ = fused_and_apart(rows, w, t, 2 * inner, k)
    rows.codes[t // 2, 3] = 0x7f
    codes = w.weight.view(torch.uint8)
    codes[5, 390], codes[inner + 130, 17] = 0xff, 0x7f
    got, want = fused_and_apart(rows, w, t, 2 * inner, k)
    agree(got, want)
    bad = torch.zeros(t, inner, dtype=torch.bool, device="cuda")
    bad[t // 2], bad[:, 5], bad[:, 130] = True, True, True
    assert torch.equal(held(got).isnan(), bad) and (got.exps[t // 2] == 67).all()
    assert (got.codes == clean.codes)[:, 256:][~bad[:, 256:]].all()


@pytest.mark.parametrize("t,inner,k", [(129, 384, 400), (300, 512, 400), (700, 1024, 528)])
def test_limits_of_the_format_in_the_epilogue(t, inner, k):
    """Rows of zeros, products that saturate and that leave fp32, that lie below the smallest code, and scales far apart from block to block."""
    for up, more, spread in ((0, 0, 6), (60, 30, 1), (60, 57, 1), (-50, -25, 1), (-50, -50, 1)):       # (powers of two of up's scales and of the rows)
        (w, _), rows = weight(2 * inner, k, 45, spread=spread), some_rows(t, k, 46, spread=40 if spread > 1 else 1)
        rows.codes[1::3] = 0
        scale = w.fp8_scale.clone()
        scale[inner // 128:] *= 2.0 ** up
        rows.exps.add_(more)
        got, want = fused_and_apart(rows, LinearWeight(w.weight, fp8_scale=scale), t, 2 * inner, k)
        agree(got, want)
        assert (got.codes[1::3] == 0).all() and (got.exps[1::3] == 67).all()
        if (up, more) == (60, 30):
            assert (got.exps == 187).any() and (got.codes & 127 == 126).any()
        if more == 57:
            assert held(got).isnan().any() and held(got).isfinite().any()
        if more == -50:
            assert (got.exps == 67).all()


def test_a_checkpoint_that_a_command_serves(tmp_path, capsys):
    """Partly FP8: planned by its tensors' names, loaded, told about, and a token made."""
    from slopllm_b200.cli import model_cli
    from slopllm_b200.models.dense import DenseConfig
    from test_fp8_edges import fp8_checkpoint
    import argparse
    cfg = DenseConfig(num_hidden_layers=2, vocab_size=512, hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=4, head_dim=64)
    path = fp8_checkpoint(tmp_path / "model", cfg, ("o_proj", "gate_proj", "up_proj", "down_proj"))
    ap = argparse.ArgumentParser()
    model_cli.add_model_args(ap)
    args = ["--act-dtype", "e4m3", "--max-pages", "8", "--batch-size", "2", "--model", path]
    rt = model_cli.build_runtime(ap.parse_args(args), with_scheduler=False)
    assert "6 of 8 matrices" in capsys.readouterr().err and rt.engine.model.fp8_layers() == (6, 8)
    s = rt.engine.kv.new_sequence()
    last, _ = rt.engine.prefill([s], [list(range(2, 100))], chunk_size=64)
    assert 0 <= last[0] < cfg.vocab_size and 0 <= rt.engine.decode_step([s], last)[0] < cfg.vocab_size
    plan = model_cli.check_memory_plan(ap.parse_args([*args, "--max-pages", str(10 ** 8)]), rt.ctx, path, "qwen3")
    assert "memory plan" in plan

"""Rows in 8 bits and their products with FP8 weights on a GPU (`csrc/fp8_rows.cu`, `csrc/fp8_gemm_tcgen05.cu`) against 64 bits."""
import pytest
import torch

from fp8_util import held, near, nearest, same, some_rows, weight
from slopllm_b200.models.weights import LinearWeight
from slopllm_b200.ops import fp8 as F8
from slopllm_b200.ops import tcgen05

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def silu_mul(gu):
    g, u = gu.double().chunk(2, -1)
    return g / (1 + torch.exp(-g)) * u


def rms(r, w, eps):
    v = r.double()
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k", [(0, 128), (1, 16), (1, 128), (2, 144), (3, 272), (5, 1024), (7, 4112), (300, 2048), (1, 16384), (64, 31264), (2500, 4096),
                                 (700, 14352)])
def test_rows(t, k, dtype):
    """Whole and cut groups, sizes that differ from token to token, one token and many."""
    x = (torch.randn(t, 2 * k, generator=gen(t + k), device="cuda") * torch.exp(torch.randn(t, 1, generator=gen(1), device="cuda") * 2)).to(dtype)
    plain = F8.fp8_rows(x[:, :k])
    assert same(plain, x[:, :k].double())
    assert same(F8.fp8_silu_mul(x), silu_mul(x))
    values = F8.fp8_values(plain)
    assert values.dtype == torch.bfloat16 and (values.double() == nearest(x[:, :k].double())[0]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("wdtype", TYPES)
@pytest.mark.parametrize("t,h", [(0, 128), (1, 16), (1, 1024), (2, 144), (3, 4112), (61, 5120), (300, 1040), (297, 4096), (5, 16384), (300, 16384)])
def test_norm(t, h, dtype, wdtype):
    x = (torch.randn(t, h, generator=gen(t + h), device="cuda") * 0.3).to(dtype)
    w = (1 + 0.1 * torch.randn(h, generator=gen(2), device="cuda")).to(wdtype)
    res = torch.randn(t, h, generator=gen(3), device="cuda") * torch.exp(torch.randn(t, 1, generator=gen(4), device="cuda"))
    for residual in (res, None):
        rows, r = F8.fp8_add_rmsnorm(x, residual, w, 1e-6)
        want = x.float() if residual is None else residual + x.float()
        assert r.dtype == torch.float32 and (r == want).all()
        assert same(rows, rms(want, w, 1e-6))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_stride(dtype):
    """Rows behind one another, every second row, values every second place, starts that no wide load takes."""
    big = torch.randn(40, 700, generator=gen(5), device="cuda").to(dtype)
    w = torch.ones(272, dtype=dtype, device="cuda")
    for x in (big[:, :272], big[::2, 8:280], big[:, 1:273], big[3:4, 3:275], big[:, 2:546:2], big[:, 200:472].t().contiguous().t()):
        assert same(F8.fp8_rows(x), x.double())
        rows, r = F8.fp8_add_rmsnorm(x, x.float(), w, 1e-5)
        assert same(rows, rms(x.float() + x.float(), w, 1e-5))
        rows, r = F8.fp8_add_rmsnorm(big[:x.shape[0], :272], torch.cat([x.float(), x.float()], 1)[:, :272], w, 1e-5)
        assert (r == big[:x.shape[0], :272].float() + x.float()).all()
        if x.shape[1] % 32 == 0:
            assert same(F8.fp8_silu_mul(x), silu_mul(x))
    gu = big[:, 5:517]
    assert same(F8.fp8_silu_mul(gu), silu_mul(gu))


def test_exponents_and_middles():
    """Magnitudes at and next to the limits of an exponent, values in and next to the middle between two codes, denormal steps among them."""
    from fp8_util import held_codes
    edge = 448.0 * 2.0 ** torch.arange(-62, 63, device="cuda").float()
    rows = torch.zeros(3 * edge.numel(), 256, device="cuda")
    rows[:, 7] = torch.cat([edge, torch.nextafter(edge, edge * 2), torch.nextafter(edge, edge * 0)])
    rows[:, 200] = -rows[:, 7] * 0.3
    assert same(F8.fp8_rows(rows), rows.double())
    table = held_codes(torch.arange(127, device="cuda")).float()
    middle = (table[1:] + table[:-1]) / 2
    x = torch.cat([middle, torch.nextafter(middle, middle * 2), torch.nextafter(middle, middle * 0), -middle])
    x = torch.nn.functional.pad(x, (0, -x.numel() % 127)).view(-1, 127)
    x = torch.cat([x, torch.full_like(x[:, :1], 448.0)], 1)
    for scale in (1.0, 2.0 ** -20, 2.0 ** 30):
        assert same(F8.fp8_rows(x * scale), x.double() * scale)


def test_values_that_are_not_finite():
    x = torch.randn(6, 256, generator=gen(6), device="cuda")
    x[0, 3], x[1, 130], x[2, 5], x[3] = float("nan"), float("inf"), -float("inf"), 0.0
    x[4, :128], x[5, 1] = float("nan"), 3e38
    rows = F8.fp8_rows(x)
    assert same(rows, x.double()) and (rows.exps[4, 0] == 67).all()
    ones = torch.ones(256, device="cuda")
    got, r = F8.fp8_add_rmsnorm(x, None, ones, 1e-6)
    assert same(got, rms(x, ones, 1e-6))
    gu = torch.randn(5, 512, generator=gen(7), device="cuda") * 3
    gu[0, 3], gu[1, 400], gu[2, 5], gu[3, 6], gu[4, 7] = float("nan"), float("inf"), -float("inf"), -200.0, 200.0
    assert same(F8.fp8_silu_mul(gu), silu_mul(gu))


def test_norms_of_extreme_rows():
    """Squares beyond fp32 on either side, no epsilon, a row of zeros, gains far apart."""
    x = torch.randn(6, 512, generator=gen(8), device="cuda")
    x[0] *= 1e30
    x[1] *= 1e-25
    x[2] *= 1e-38
    x[3] = 0
    w = torch.exp(torch.randn(512, generator=gen(9), device="cuda") * 4)
    for eps in (1e-6, 0.0):
        rows, _ = F8.fp8_add_rmsnorm(x, None, w, eps)
        assert same(rows, rms(x, w, eps))


def test_gates_far_out():
    """Gates for which the exponential's argument is large, and groups that have no others."""
    gu = torch.randn(64, 1024, generator=gen(10), device="cuda") * 12
    gu[:8, :512] = -18 - gu[:8, :512].abs()
    gu[8:16, :512] = 18 + gu[8:16, :512].abs()
    for x in (gu, gu.bfloat16()):
        assert same(F8.fp8_silu_mul(x), silu_mul(x))


@pytest.mark.parametrize("t", [0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 200, 257, 384, 1000])
@pytest.mark.parametrize("n,k", [(1, 16), (130, 144), (256, 128), (384, 1024), (1001, 4112)])
def test_products(t, n, k):
    """Every form of the kernel, cut tiles of rows, columns and blocks of K; results behind the columns are left alone."""
    w, values = weight(n, k, t + n)
    rows = some_rows(t, k, t + k)
    for f32 in (True, False):
        y = F8.fp8_linear(rows, w, out_f32=f32)
        assert y.shape == (t, n) and y.dtype == (torch.float32 if f32 else torch.bfloat16)
        assert near(y, rows, values)
    tcgen05.check_errors(y.device)


@pytest.mark.parametrize("t,n,k", [(1, 6144, 4096), (8, 2048, 14336), (40, 4096, 8192), (300, 5120, 2048), (777, 2321, 5136), (2048, 4096, 1024), (4500, 512, 256),
                                   (3, 128, 32768), (130, 128, 32768)])
def test_products_of_all_sizes(t, n, k):
    w, values = weight(n, k, 3)
    rows = some_rows(t, k, 4)
    assert near(F8.fp8_linear(rows, w, out_f32=True), rows, values)
    assert near(F8.fp8_linear(rows, w), rows, values)
    tcgen05.check_errors(rows.device)


@pytest.mark.parametrize("t,n,k", [(65, 16, 272), (192, 6144, 4096), (512, 4096, 2064), (777, 2064, 5136), (1000, 2048, 1168), (20000, 100, 400)])
def test_products_of_narrow_tiles(t, n, k):
    """Tiles of 128 columns on pairs of SMs: more and fewer than there are pairs, even and odd numbers of blocks of K, cut rows, columns and blocks."""
    w, values = weight(n, k, 31, spread=3)
    rows = some_rows(t, k, 32, spread=8)
    y = F8.fp8_linear(rows, w, out_f32=True)
    assert near(y, rows, values)
    assert torch.equal(F8.fp8_linear(rows, w), y.bfloat16())
    tcgen05.check_errors(rows.device)


@pytest.mark.parametrize("t,n,k", [(150000, 112, 16), (90000, 64, 144)])
def test_tiles_that_follow_each_other(t, n, k):
    """Tiles of one or two blocks of K, several of a pair: a result is on its way out when the next one is written."""
    w, values = weight(n, k, 33)
    rows = some_rows(t, k, 34)
    want = F8.fp8_linear(rows, w, out_f32=True)
    assert near(want, rows, values)
    want = want.bfloat16()
    assert all(torch.equal(F8.fp8_linear(rows, w), want) for _ in range(20))
    tcgen05.check_errors(rows.device)


@pytest.mark.parametrize("t", [3, 50, 300])
def test_scales_far_apart(t):
    """Exponents and scales that differ by many powers of two from block to block: a scale that meets another block would show."""
    w, values = weight(384, 2064, 5, spread=6)
    rows = some_rows(t, 2064, 6, spread=40)
    assert near(F8.fp8_linear(rows, w, out_f32=True), rows, values)


@pytest.mark.parametrize("t", [1, 20, 140, 600])
def test_codes_that_are_not_finite(t):
    """A NaN code of a row spoils the row's results, one of a weight its column's."""
    w, values = weight(300, 400, 7)
    rows = some_rows(t, 400, 8)
    w.weight.view(torch.uint8)[77, 390] = 0x7f
    rows.codes[t // 2, 3] = 0xff
    y = F8.fp8_linear(rows, w, out_f32=True)
    bad = torch.zeros(t, 300, dtype=torch.bool, device="cuda")
    bad[t // 2], bad[:, 77] = True, True
    assert (y.isnan() == bad).all()


@pytest.mark.parametrize("t", [1, 9, 100, 500])
def test_products_of_any_stride(t):
    """Some rows of a larger set, weights that are columns or rows of larger ones, scales of another type, rows of exponents without room behind them."""
    w, values = weight(512, 1024, 9)
    rows = some_rows(2 * t, 1024, 10)
    part = F8.Fp8Rows(rows.codes[::2], rows.exps[::2])
    assert near(F8.fp8_linear(part, w, out_f32=True), part, values)
    part = F8.Fp8Rows(rows.codes[:t, 256:768], F8.fp8_rows(torch.zeros(t, 512, device="cuda")).exps.copy_(rows.exps[:t, 2:6]))
    from slopllm_b200.models.weights import LinearWeight
    cut = LinearWeight(w.weight[128:401, 256:768], fp8_scale=w.fp8_scale[1:4, 2:6])
    assert near(F8.fp8_linear(part, cut, out_f32=True), part, values[128:401, 256:768])
    odd = LinearWeight(torch.nn.functional.pad(w.weight.view(torch.uint8), (3, 5))[:, 3:1027].view(torch.float8_e4m3fn), fp8_scale=w.fp8_scale.double())
    assert near(F8.fp8_linear(rows, odd, out_f32=True), rows, values)


@pytest.mark.parametrize("t", [1, 7, 40, 129, 700])
@pytest.mark.parametrize("inner", [16, 128, 144, 1024])
def test_gate_up(t, inner):
    """The activation of the product's fp32 sums.  A code may be the neighbour's where a sum lies by the middle between two: values are compared, within a
    step of the format (2^-3 of the value, 2^-9 of the group's scale) wherever they are not the nearest ones."""
    w, values = weight(2 * inner, 528, 11)
    rows = some_rows(t, 528, 12)
    got = F8.fp8_gate_up(rows, w)
    assert got.shape == (t, inner)
    x = held(rows)
    gu, most = x @ values.t(), x.abs() @ values.abs().t()
    want = silu_mul(gu)
    off = 2.0 ** -16 * most                              # (`near`'s bound on a sum; SiLU's slope is below 1.1)
    g, u = gu.chunk(2, -1)
    off = 1.1 * off[:, :inner] * (u.abs() + off[:, inner:]) + g.abs() * off[:, inner:]
    step = torch.exp2(got.exps.double() - 127).repeat_interleave(128, 1)[:, :inner]
    assert ((held(got) - want).abs() <= off + torch.maximum(2.0 ** -4 * (want.abs() + off), 2.0 ** -10 * step)).all()
    tcgen05.check_errors(rows.device)


def test_gate_up_of_many_tiles():
    """More tiles than pairs of SMs, some of them cut by the last row: the codes of the product and the activation by themselves, all but those next to a middle."""
    w, _ = weight(4096, 1040, 21)
    rows = some_rows(2100, 1040, 22)
    got, want = F8.fp8_gate_up(rows, w), F8.fp8_silu_mul(F8.fp8_linear(rows, w, out_f32=True))
    assert (got.exps == want.exps).all() and (got.codes != want.codes).float().mean() < 1e-4
    assert ((held(got) - held(want)).abs() <= 2.0 ** -3 * held(want).abs() + 2.0 ** -9 * torch.exp2(want.exps.double() - 127).repeat_interleave(128, 1)).all()
    tcgen05.check_errors(rows.device)


def test_calls_side_by_side():
    """The forms of the product on several streams at once, over the same rows and weights: each gives what it gives by itself."""
    (w, _), (big, _) = weight(1024, 2048, 23), weight(6144, 2048, 24)
    some, many = some_rows(20, 2048, 25), some_rows(900, 2048, 26)
    calls = [lambda: F8.fp8_linear(some, w), lambda: F8.fp8_linear(some, big, out_f32=True), lambda: F8.fp8_linear(many, big),
             lambda: F8.fp8_gate_up(many, big).codes, lambda: F8.fp8_gate_up(some, big).codes]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        got = []
        for c, s in zip(calls, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    tcgen05.check_errors(w.weight.device)


def layer(x, res, norm, gate_up, down):
    rows, r = F8.fp8_add_rmsnorm(x, res, norm, 1e-6)
    return F8.fp8_linear(F8.fp8_gate_up(rows, gate_up), down), r


@pytest.mark.parametrize("t", [1, 13, 200, 700])
def test_a_feed_forward(t):
    """The operators one after the other, eagerly, on another stream and as a captured graph with other inputs: the same bits each time, and near what 64 bits give
    with codes of their own (each rounding to codes is 2^-4 of a value at most, of random sign: 2^-5 of a result's size)."""
    h, inner = 528, 784
    (gate_up, vg), (down, vd) = weight(2 * inner, h, 13), weight(h, inner, 14)
    norm = (1 + 0.1 * torch.randn(h, generator=gen(15), device="cuda")).bfloat16()
    x, res = torch.randn(t, h, generator=gen(16), device="cuda").bfloat16(), torch.randn(t, h, generator=gen(17), device="cuda")
    y, r = layer(x, res, norm, gate_up, down)
    want = silu_mul(nearest(rms(res + x.float(), norm, 1e-6))[0] @ vg.t())
    want = nearest(want)[0] @ vd.t()
    assert (y.double() - want).norm() <= 2.0 ** -7 * want.norm() and (y.double() - want).abs().max() <= 2.0 ** -5 * want.square().mean().sqrt() * 8
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again, _ = layer(x, res, norm, gate_up, down)
    torch.cuda.current_stream().wait_stream(side)
    assert (again == y).all()
    xs, rs = torch.zeros_like(x), torch.zeros_like(res)
    with torch.cuda.stream(side):
        layer(xs, rs, norm, gate_up, down)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, cr = layer(xs, rs, norm, gate_up, down)
    xs.copy_(x), rs.copy_(res)
    graph.replay()
    assert (captured == y).all() and (cr == r).all()
    tcgen05.check_errors(x.device)


def test_a_row_is_the_same_in_any_batch():
    """Rows are quantised by themselves."""
    x = torch.randn(400, 1040, generator=gen(18), device="cuda")
    w = torch.ones(1040, device="cuda")
    all_rows, _ = F8.fp8_add_rmsnorm(x, None, w, 1e-6)
    for i in (0, 7, 399):
        one, _ = F8.fp8_add_rmsnorm(x[i:i + 1], None, w, 1e-6)
        assert (one.codes == all_rows.codes[i:i + 1]).all() and (one.exps == all_rows.exps[i:i + 1]).all()


def test_rows_far_apart():
    """Strides that pass 32 bits: rows, residual, weights and their scales."""
    step = 2 ** 31 + 64
    space = torch.empty(2 * step, dtype=torch.uint8, device="cuda")
    rows = torch.as_strided(torch.empty(step + 512, dtype=torch.bfloat16, device="cuda"), (2, 512), (step, 1))
    rows.copy_(torch.randn(2, 512, generator=gen(0), device="cuda"))
    near_by = rows.clone(memory_format=torch.contiguous_format)
    for call in (F8.fp8_rows, F8.fp8_silu_mul, lambda x: F8.fp8_add_rmsnorm(x, None, torch.ones(512, device="cuda"), 1e-6)[0]):
        far, close = call(rows), call(near_by)
        assert torch.equal(far.codes, close.codes) and torch.equal(far.exps, close.exps)
    w, _ = weight(2, 256)
    x = some_rows(3, 256)
    codes = torch.as_strided(space, (2, 256), (step, 1))
    codes.copy_(w.weight.view(torch.uint8))
    assert torch.equal(F8.fp8_linear(x, LinearWeight(codes, fp8_scale=w.fp8_scale)), F8.fp8_linear(x, w))


def test_refusals():
    rows, (w, _) = some_rows(4, 256), weight(64, 256)
    with pytest.raises(ValueError):
        F8.fp8_linear(rows, w.to("cpu"))
    with pytest.raises(ValueError):
        F8.Fp8Rows(rows.codes, rows.exps.cpu())
    with pytest.raises(ValueError):
        F8.Fp8Rows(rows.codes, torch.zeros(4, 2, dtype=torch.uint8, device="cuda"))
    with pytest.raises(ValueError):
        F8.Fp8Rows(rows.codes[:1], torch.zeros(2, dtype=torch.uint8, device="cuda")[None])
    with pytest.raises(ValueError):
        F8.Fp8Rows(torch.zeros(4 * 256 + 8, dtype=torch.uint8, device="cuda")[8:].view(4, 256), rows.exps)
    x = torch.randn(4, 256, device="cuda")
    for call in (lambda: F8.fp8_rows(x.half()), lambda: F8.fp8_silu_mul(x.double()), lambda: F8.fp8_add_rmsnorm(x, x.bfloat16(), x[0], 1e-6),
                 lambda: F8.fp8_add_rmsnorm(x, x, x[0].half(), 1e-6), lambda: F8.fp8_add_rmsnorm(x, x.cpu(), x[0], 1e-6),
                 lambda: F8.fp8_add_rmsnorm(x, x, x[0].cpu(), 1e-6),
                 lambda: F8.fp8_add_rmsnorm(torch.zeros(1, 16400, device="cuda"), None, torch.ones(16400, device="cuda"), 1e-6)):
        with pytest.raises(ValueError):
            call()

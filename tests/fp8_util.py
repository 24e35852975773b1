"""Rows in 8 bits and FP8 weights for tests, and what they hold in 64 bits, from the format's definition."""
import torch

from slopllm_b200.models.weights import LinearWeight
from slopllm_b200.ops import fp8 as F8

GROUP = 128


def held_codes(codes):
    """fp64 numbers of e4m3 bytes, from their bits."""
    c = codes.to(torch.int64)
    exp, man = c >> 3 & 15, (c & 7).double() / 8
    mag = torch.where(exp == 0, man * 2.0 ** -6, (1 + man) * torch.exp2((exp - 7).double()))
    mag = torch.where((c & 127) == 127, torch.full_like(mag, float("nan")), mag)
    return torch.where(c >= 128, -mag, mag)


def held(rows):
    """fp64 values of rows in 8 bits."""
    up = torch.exp2(rows.exps.double() - 127).repeat_interleave(GROUP, 1)[:, :rows.codes.shape[1]]
    return held_codes(rows.codes) * up


def nearest(v):
    """fp64 rows -> (fp64 values of the nearest rows in 8 bits, exponents), by looking magnitudes up between the middles of neighbouring codes."""
    table = held_codes(torch.arange(127, device=v.device))
    middle = (table[1:] + table[:-1]) / 2
    v = torch.where(v.float().isfinite(), v, torch.full_like(v, float("nan")))
    out, exps = torch.empty_like(v), torch.empty(v.shape[0], -(-v.shape[1] // GROUP), dtype=torch.float64, device=v.device)
    for g in range(exps.shape[1]):
        x = v[:, g * GROUP:(g + 1) * GROUP]
        top = x.abs().nan_to_num(0.0).amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -200) / 448)).clamp(-60, 60)
        e = torch.where(top > 448 * torch.exp2(e), (e + 1).clamp(max=60), torch.where(top <= 448 * torch.exp2(e - 1), (e - 1).clamp(min=-60), e))
        y = (x.abs() * torch.exp2(-e)).nan_to_num(0.0).contiguous()
        below, above = torch.bucketize(y, middle), torch.bucketize(y, middle, right=True)
        at = torch.where(below % 2 == 0, below, above)
        q = torch.sign(x) * table[at] * torch.exp2(e)
        out[:, g * GROUP:(g + 1) * GROUP] = torch.where(x.isnan(), x, q)
        exps[:, g] = e[:, 0]
    return out, exps


def same(rows, v):
    """Whether rows hold the nearest values of fp64 rows `v`, with their exponents."""
    want, exps = nearest(v)
    got = held(rows)
    return bool(((got == want) | (got.isnan() & want.isnan())).all()) and bool((rows.exps.double() - 127 == exps).all())


def weight(n, k, seed=0, device="cuda", spread=0.3):
    """FP8 weights whose blocks differ in size, and their fp64 values."""
    g = torch.Generator(device=device).manual_seed(seed)
    codes = (torch.randn(n, k, generator=g, device=device) * 110).clamp(-448, 448).to(torch.float8_e4m3fn)
    scale = torch.exp(torch.randn(-(-n // GROUP), -(-k // GROUP), generator=g, device=device) * spread) / (110 * k ** 0.5)
    values = held_codes(codes.view(torch.uint8)) * scale.double().repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    return LinearWeight(codes, fp8_scale=scale), values


def some_rows(t, k, seed=1, device="cuda", spread=2):
    """Rows in 8 bits whose groups' exponents differ by up to 2 `spread`; the bytes between rows of exponents are 255."""
    g = torch.Generator(device=device).manual_seed(seed)
    rows = F8.Fp8Rows.allocate(t, k, device)
    rows.codes.copy_((torch.randn(t, k, generator=g, device=device) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
    if t:
        rows.exps.as_strided((t, rows.exps.stride(0)), rows.exps.stride()).fill_(255)
    rows.exps.copy_(torch.randint(120 - spread, 121 + spread, rows.exps.shape, generator=g, device=device))
    return rows


def near(y, rows, values, x=None):
    """A product against 64 bits.  What may be off, relative to the sum of the products' magnitudes: the tensor core adds 32 products and a running sum at a
    time, each cut at 2^-24 of the largest at worst, four times a block of K: 2^-17 of the magnitudes; times the scale and added up in fp32
    over K / 128 blocks: (K / 128 + 2) 2^-24.  A bf16 result is rounded by 2^-8 of itself."""
    x = held(rows) if x is None else x
    want, most = x @ values.t(), x.abs() @ values.abs().t()
    off = (2.0 ** -17 + (x.shape[1] / 128 + 2) * 2.0 ** -24) * most
    if y.dtype == torch.bfloat16:
        off = off + 2.0 ** -8 * (want.abs() + off)
    bad = ~((y.double() - want).abs() <= off)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), int(bad.sum()), (y.double() - want).abs().max().item())
    return True

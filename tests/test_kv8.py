"""The 8-bit key/value cache on the CPU: the format, what the operators refuse, and the fp32 definitions against 64 bits."""
import pytest
import torch

from kv8_util import attend, exponent, filled, held, near, round_e4m3, table_of
from slopllm_b200.ops import kv8 as K8
from slopllm_b200.ops.rotary import rotary_table


def test_the_format():
    """Rows of all sizes, at the border of a scale, of zeros, with values that are not finite and values beyond the largest scale."""
    x = torch.randn(400, 32, generator=torch.Generator().manual_seed(0)) * torch.logspace(-9, 9, 400)[:, None]
    x[0] = 0.0
    x[1, 5], x[2, 6], x[3, 7] = float("inf"), float("-inf"), float("nan")
    x[4, 0], x[4, 1:] = 448.0, 1.0
    x[5, 0], x[5, 1:] = 448.0 * (1 + 2 ** -20), 1.0
    x[6, 0] = 1e30
    codes, exps = K8.kv8_quantize(x)
    assert exps[0] == 127 - 60 and exps[4] == 127 and exps[5] == 128 and exps[6] == 127 + 60
    fine = x.isfinite()
    top = torch.where(fine, x, torch.zeros(())).abs().amax(-1)
    assert torch.equal(exps.double() - 127, exponent(top))
    scale = torch.exp2(exps.double() - 127)[:, None]
    want = (round_e4m3((x.double() / scale).clamp(-448, 448)) * scale).masked_fill(~fine, float("nan"))
    assert torch.equal(held(codes, exps).nan_to_num(-7.0), want.nan_to_num(-7.0))
    assert torch.equal(K8.kv8_values(codes, exps).double().nan_to_num(-7.0), want.nan_to_num(-7.0))
    # what the cache holds is exact in bf16
    kept = K8.kv8_values(codes, exps)
    assert torch.equal(kept.to(torch.bfloat16).float().nan_to_num(-7.0), kept.nan_to_num(-7.0))


@pytest.mark.parametrize("page", [16, 64])
def test_store_read_and_attention(page):
    """Definitions on the CPU: rows appended in two steps, read back, attended over as portions and as single tokens."""
    T, h, kv, hd, dims = 70, 4, 2, 32, 16
    g = torch.Generator().manual_seed(1)
    proj = torch.randn(T, (h * 2 + 2 * kv) * hd, generator=g)
    q, k, v = proj[:, :h * 2 * hd], proj[:, h * 2 * hd:(h * 2 + kv) * hd], proj[:, (h * 2 + kv) * hd:]
    qn, kn = (1 + 0.1 * torch.randn(hd, generator=g) for _ in range(2))
    rot = rotary_table(dims, 1e4)
    table, rows, total = table_of([T, 3], page, 1, "cpu")
    cache = K8.Kv8Cache.allocate(total, page, kv, hd, "cpu")
    pos, idx = torch.arange(T, dtype=torch.int32), torch.zeros(T, dtype=torch.int32)
    parts = [K8.kv8_store(q[a:b], k[a:b], v[a:b], qn, kn, rot, pos[a:b], idx[a:b], table, cache, h, 1e-6, q_stride=2 * hd) for a, b in ((0, 50), (50, T))]
    qo = torch.cat(parts)
    x = k.reshape(T, kv, hd).double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * kn.double()
    ang = torch.outer(pos.double(), rot.freq.double())[:, None]
    a, b = x[..., :dims // 2], x[..., dims // 2:dims]
    want = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), x[..., dims:]], -1)
    kk, vv = K8.kv8_read(cache, torch.tensor([[0, 0, T, 0]], dtype=torch.int32), T, T, table)
    size = want.abs().amax(-1, keepdim=True)
    # half a step of e4m3: 2^-4 of the value, or 2^-10 of the scale (the scale is at most size / 224)
    assert ((kk.double() - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * size / 224 + 2.0 ** -18 * size).all()
    wv = v.reshape(T, kv, hd).double()
    assert ((vv.double() - wv).abs() <= 2.0 ** -4 * wv.abs() + 2.0 ** -10 * wv.abs().amax(-1, keepdim=True) / 224).all()
    some = K8.kv8_read(cache, torch.tensor([[0, 17, 5, 2], [0, 60, 2, 0]], dtype=torch.int32), 7, 5, table)
    assert torch.equal(some[0], torch.cat([kk[60:62], kk[17:22]])) and torch.equal(some[1], torch.cat([vv[60:62], vv[17:22]]))
    got = K8.kv8_attention(qo, cache, pos, idx, table, hd ** -0.5, qo_indptr=torch.tensor([0, T], dtype=torch.int32), max_q=T)
    ref = attend(qo, kk.double(), vv.double(), pos, hd ** -0.5)
    assert (got.double() - ref).abs().max() < 2.0 ** -14 * vv.abs().max()
    one = K8.kv8_attention(qo[[69, 3]], cache, pos[[69, 3]], idx[:2], table, hd ** -0.5)
    assert torch.equal(one, got[[69, 3]])
    assert cache.k.float().sum() > 0 and len(rows[1]) == 3


def test_rows_without_keys_and_padding():
    """A position of -1: attention gives zeros, the writer leaves the cache alone."""
    cache, table, _, values, g = filled([5], 2, 16, 2, 16, "cpu")
    before = [x.clone() for x in (cache.k, cache.v, cache.exps)]
    q = torch.randn(2, 4, 16, generator=g)
    pos, idx = torch.tensor([-1, 4], dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    got = K8.kv8_attention(q, cache, pos, idx, table, 0.25)
    assert (got[0] == 0).all() and got[1].abs().max() > 0
    K8.kv8_store(torch.randn(1, 64), torch.randn(1, 32), torch.randn(1, 32), None, None, rotary_table(16, 1e4), pos[:1], idx[:1], table, cache, 4, 1e-6)
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.exps)))


def test_refusals():
    """What the operators do not take is said before anything is written."""
    cache, table, _, _, _ = filled([5], 2, 16, 2, 16, "cpu")
    pos, idx = torch.tensor([4], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    for k, v, e in ((u8(64, 2, 24), u8(64, 2, 24), u8(1, 2, 2, 64)), (u8(64, 2, 272), u8(64, 2, 272), u8(1, 2, 2, 64)), (u8(64, 2, 16), u8(64, 2, 32), u8(1, 2, 2, 64)),
                    (u8(64, 2, 16), u8(64, 2, 16), u8(1, 1, 2, 64)), (u8(20, 2, 16), u8(20, 2, 16), u8(1, 2, 2, 20)),
                    (u8(64, 2, 16).float(), u8(64, 2, 16), u8(1, 2, 2, 64)), (u8(64, 2, 32)[..., :16], u8(64, 2, 16), u8(1, 2, 2, 64))):
        with pytest.raises(ValueError):
            K8.Kv8Cache(k, v, e)
    att = lambda q=torch.zeros(1, 4, 16), pos=pos, idx=idx, table=table: K8.kv8_attention(q, cache, pos, idx, table, 0.25)
    for bad in (dict(q=torch.zeros(1, 3, 16)), dict(q=torch.zeros(1, 4, 32)), dict(q=torch.zeros(2, 4, 16)), dict(pos=pos.long()), dict(table=table.long()),
                dict(idx=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            att(**bad)
    rot = rotary_table(16, 1e4)
    store = lambda q=torch.zeros(1, 64), k=torch.zeros(1, 32), rot=rot, heads=4, stride=None: K8.kv8_store(
        q, k, torch.zeros(1, 32), None, None, rot, pos, idx, table, cache, heads, 1e-6, q_stride=stride)
    for bad in (dict(q=torch.zeros(1, 48)), dict(k=torch.zeros(1, 16)), dict(rot=rotary_table(32, 1e4)), dict(heads=3), dict(stride=8)):
        with pytest.raises(ValueError):
            store(**bad)
    for r in (torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.int64)):
        with pytest.raises(ValueError):
            K8.kv8_read(cache, r, 1, 1, table)
    assert near(att().float(), att().double(), torch.ones(1))

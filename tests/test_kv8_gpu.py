"""The 8-bit key/value cache on a GPU (`csrc/kv8.cu`, `csrc/kv8_attn.cu`) against 64 bits: writer, reader, attention of single tokens and of prompts."""
import pytest
import torch

from kv8_util import attend, exponent, filled, held, near, round_e4m3, table_of
from slopllm_b200.ops import kv8 as K8
from slopllm_b200.ops import tcgen05
from slopllm_b200.ops.native import NativeError
from slopllm_b200.ops.rotary import RotaryTable, rotary_table

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def decode(histories, h, kv, hd, seed=3, page=64, scale=1.0, sizes=0.7):
    cache, table, keys, values, g = filled(histories, kv, hd, seed, page, sizes=sizes)
    q = (torch.randn(len(histories), h, hd, generator=g, device="cuda") * scale).to(torch.bfloat16)
    pos, idx = ints([n - 1 for n in histories]), torch.arange(len(histories), dtype=torch.int32, device="cuda")
    got = K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5, max_kv_len=max(histories))
    tcgen05.check_errors(q.device)
    for b in range(len(histories)):
        want = attend(q[b:b + 1], keys[b], values[b], pos[b:b + 1], hd ** -0.5)
        assert near(got[b:b + 1], want, values[b]), (b, histories[b], (got[b:b + 1].double() - want).abs().max().item())
    return cache, table, q, pos, idx, got


@pytest.mark.parametrize("histories,h,kv,hd,scale", [
    ([1], 16, 8, 128, 1.0), ([2, 15, 16, 17, 47, 48, 63, 64, 65], 8, 8, 128, 1.0), ([127, 128, 129, 700, 3], 32, 2, 128, 3.0), ([130] * 33, 8, 4, 64, 1.0),
    ([9000], 4, 1, 64, 1.0), ([77, 500, 1], 4, 2, 256, 2.0), ([40, 4100], 16, 1, 128, 1.0), ([1, 3000, 2], 64, 8, 128, 1.0), ([5000, 70], 16, 1, 256, 1.0),
    ([640] * 300, 2, 2, 64, 1.0), ([700, 30, 2000], 40, 40, 64, 1.0), ([3000, 5, 1200], 100, 50, 128, 1.0), ([900] * 30, 66, 33, 256, 1.0),
])
def test_decoding(histories, h, kv, hd, scale):
    """Tile edges, one and several pieces of a history, ragged batches, 1 to 16 query heads a key head, caches of NaN outside the histories."""
    decode(histories, h, kv, hd, scale=scale)


@pytest.mark.parametrize("hd", [16, 32, 48, 80, 96, 112, 144, 160, 192, 240])
@pytest.mark.parametrize("h,kv", [(8, 8), (6, 3), (32, 2), (12, 1)])
def test_decoding_of_all_widths(hd, h, kv):
    """Widths between the instances, and counts of query heads that are no power of two."""
    decode([1, 31, 64, 65, 700], h, kv, hd)


@pytest.mark.parametrize("page", [16, 32, 48, 128, 192])
def test_decoding_of_other_pages(page):
    decode([1, 15, 16, 17, 48, 49, 500, 1030], 8, 2, 128, page=page)


@pytest.mark.parametrize("histories,h,kv,hd", [([700], 16, 8, 128), ([64, 65, 1, 0, 2048], 8, 2, 128), ([513, 1500], 16, 1, 64), ([300, 2000], 8, 1, 256),
                                               ([128 * i + 1 for i in range(1, 9)], 6, 3, 96), ([1025], 32, 1, 80), ([449], 1, 1, 16),
                                               ([90 * i + 57 for i in range(8)], 16, 8, 128), ([0, 700, *range(1, 17)], 16, 8, 128),
                                               ([15 * i + 1 for i in range(64)], 16, 1, 64), ([33 * i + 2 for i in range(30)], 8, 2, 256)])
@pytest.mark.parametrize("page", [64, 48])
def test_decoding_in_clusters(histories, h, kv, hd, page):
    """Little work: eight, four or two blocks that join their parts in shared memory; fewer tiles than blocks, rows without keys, 16 query heads a key head and more."""
    cache, table, keys, values, g = filled([max(n, 1) for n in histories], kv, hd, 11, page)
    q = torch.randn(len(histories), h, hd, generator=g, device="cuda").to(torch.bfloat16)
    pos, idx = ints([n - 1 for n in histories]), torch.arange(len(histories), dtype=torch.int32, device="cuda")
    for longest in (max(histories), 0):
        got = K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5, max_kv_len=longest)
        tcgen05.check_errors(q.device)
        for b, n in enumerate(histories):
            if n == 0:
                assert (got[b] == 0).all()
            else:
                assert near(got[b:b + 1], attend(q[b:b + 1], keys[b], values[b], pos[b:b + 1], hd ** -0.5), values[b]), (longest, n)


@pytest.mark.parametrize("longest", [0, 1, 512, 2048, 100000])
def test_decoding_with_any_hint(longest):
    """The longest history is told for speed only: one that is wrong changes nothing but roundings."""
    cache, table, q, pos, idx, got = decode([700, 65, 1, 5000], 8, 2, 128)
    again = K8.kv8_attention(q, cache, pos, idx, table, 128 ** -0.5, max_kv_len=longest)
    assert torch.allclose(again.float(), got.float(), rtol=2 ** -7, atol=2 ** -12)


def test_decoding_of_many_rows():
    """More rows than one launch takes."""
    decode([1 + i % 70 for i in range(1500)], 4, 2, 64)


def test_decoding_of_sizes_far_apart():
    """Values whose scales differ by more than the range of fp16 within a history, zero rows among them, and a key that dominates although its
    value is zero."""
    cache, table, keys, values, g = filled([300], 2, 64, 5, sizes=6.0)
    page, hd = 64, 64
    slots = (table[0, :5].long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:300]
    q = torch.randn(1, 4, hd, generator=g, device="cuda").to(torch.bfloat16)
    for i, kv_row in ((7, torch.zeros(2, hd, device="cuda")), (200, torch.zeros(2, hd, device="cuda"))):
        c, e = K8.kv8_quantize(kv_row)
        cache.v[slots[i]], cache.exps[slots[i] // page, :, 1, slots[i] % page] = c, e
        values[0][i] = held(c, e)
    c, e = K8.kv8_quantize(q[0, [0, 2]].float() * 4)
    cache.k[slots[200]], cache.exps[slots[200] // page, :, 0, slots[200] % page] = c, e
    keys[0][200] = held(c, e)
    pos, idx = ints([299]), ints([0])
    got = K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5)
    want = attend(q, keys[0], values[0], pos, hd ** -0.5)
    # (2^-13: the largest score is 36, good to 2^-21 of it; a term of the sum is good to 2^-21 of the largest term)
    terms = torch.softmax(torch.einsum("hd,khd->hk", q[0].double(), keys[0].repeat_interleave(2, 1)) * hd ** -0.5, -1)
    most = (terms[:, :, None] * values[0].repeat_interleave(2, 1).transpose(0, 1).abs()).sum(1)
    assert ((got[0].double() - want[0]).abs() <= 2.0 ** -8 * want[0].abs() + 2.0 ** -13 * most.amax(-1, keepdim=True)).all()
    tcgen05.check_errors(q.device)


@pytest.mark.parametrize("h,kv,hd", [(4, 2, 64), (8, 1, 128), (2, 2, 256)])
def test_decoding_of_values_that_are_not_finite(h, kv, hd):
    """A NaN code of a key spoils the heads that read it, one of a value its column; neighbours and rows that end in front of it stay clean."""
    cache, table, keys, values, g = filled([100, 100], kv, hd, 6)
    q = torch.randn(3, h, hd, generator=g, device="cuda").to(torch.bfloat16)
    slot = int(table[0, 1]) * 64 + 20                                   # position 84
    cache.v[slot, 0, 5] = 0x7f
    pos, idx = ints([99, 83, 99]), ints([0, 0, 1])
    got = K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5)
    assert got[0, :h // kv, 5].isnan().all() and got.isnan().sum() == h // kv
    cache.k[slot, 0, 5] = 0xff
    got = K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5)
    assert got[0, :h // kv].isnan().all() and got.isnan().sum() == h // kv * hd
    assert near(got[1:2], attend(q[1:2], keys[0], values[0], pos[1:2], hd ** -0.5), values[0])
    assert near(got[2:3], attend(q[2:3], keys[1], values[1], pos[2:3], hd ** -0.5), values[1])
    tcgen05.check_errors(q.device)


@pytest.mark.parametrize("histories", [[0], [0, 70, 0], [0, 0, 5, 900]])
def test_rows_without_keys(histories):
    """Zeros, wherever such rows lie in a batch; no rows at all."""
    cache, table, keys, values, g = filled([max(n, 1) for n in histories], 2, 128, 7)
    q = torch.randn(len(histories), 8, 128, generator=g, device="cuda").to(torch.bfloat16)
    pos, idx = ints([n - 1 for n in histories]), torch.arange(len(histories), dtype=torch.int32, device="cuda")
    got = K8.kv8_attention(q, cache, pos, idx, table, 128 ** -0.5)
    for b, n in enumerate(histories):
        if n == 0:
            assert (got[b] == 0).all()
        else:
            assert near(got[b:b + 1], attend(q[b:b + 1], keys[b], values[b], pos[b:b + 1], 128 ** -0.5), values[b])
    assert K8.kv8_attention(q[:0], cache, pos[:0], idx[:0], table, 1.0).shape == (0, 8, 128)
    tcgen05.check_errors(q.device)


def test_rows_of_any_order_views_and_streams():
    """Several tokens of one page-table row, rows in another order, queries that start between two 16-byte pieces or lie apart, another stream:
    the same bits."""
    cache, table, q, pos, idx, got = decode([700, 65, 129, 2000], 8, 2, 128)
    perm = torch.tensor([2, 0, 3, 1], device="cuda")
    again = K8.kv8_attention(q[perm], cache, pos[perm], idx[perm], table, 128 ** -0.5, max_kv_len=2000)
    close = lambda a, b: torch.allclose(a.float(), b.float(), rtol=2 ** -7, atol=2 ** -12)
    assert close(again, got[perm])
    odd = torch.cat([q.new_zeros(1), q.flatten()])[1:].view_as(q)
    apart = torch.stack([q, q], 2)[:, :, 0]
    for x in (odd, apart):
        assert torch.equal(K8.kv8_attention(x, cache, pos, idx, table, 128 ** -0.5, max_kv_len=2000), got)
    both = K8.kv8_attention(q[[0, 0]], cache, ints([699, 350]), ints([0, 0]), table, 128 ** -0.5)
    assert close(both[:1], got[:1])
    wide = torch.cat([table, table], 1)[:, :table.shape[1]]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        on_s = K8.kv8_attention(q, cache, pos, idx, wide, 128 ** -0.5, max_kv_len=2000)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(on_s, got)
    tcgen05.check_errors(q.device)


def test_decoding_in_captured_graphs():
    """Two graphs of one size, replayed in turn after positions and queries have changed."""
    cache, table, keys, values, g = filled([900, 400], 2, 128, 8)
    idx, scale = ints([0, 1]), 128 ** -0.5
    runs = []
    for _ in range(2):
        q, pos = torch.randn(2, 16, 128, generator=g, device="cuda").to(torch.bfloat16), ints([5, 399])
        K8.kv8_attention(q, cache, pos, idx, table, scale)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = K8.kv8_attention(q, cache, pos, idx, table, scale)
        runs.append((graph, q, pos, out))
    for step in ([899, 3], [64, 127], [0, 399]):
        for graph, q, pos, out in runs:
            q.copy_(torch.randn(2, 16, 128, generator=g, device="cuda"))
            pos.copy_(ints(step))
        for graph, *_ in runs:
            graph.replay()
        for _, q, pos, out in runs:
            for b in range(2):
                assert near(out[b:b + 1], attend(q[b:b + 1], keys[b], values[b], pos[b:b + 1], scale), values[b])
    tcgen05.check_errors(q.device)


def test_tables_that_point_nowhere():
    """Page ids, rows and positions outside the tables are reported after the step; nothing is read or written there."""
    cache, table, _, _, g = filled([100], 2, 64, 9)
    q = torch.randn(1, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    k = torch.randn(1, 128, generator=g, device="cuda").to(torch.bfloat16)
    before = [x.clone() for x in (cache.k, cache.v, cache.exps)]
    rot = rotary_table(64, 1e4).to("cuda")
    far = table.clone()
    far[0, 1] = 1 << 20
    for t, pos, row in ((far, 99, 0), (table, 64 * table.shape[1], 0), (table, 99, 5), (table, 99, -1)):
        calls = (lambda: K8.kv8_attention(q, cache, ints([pos]), ints([row]), t, 0.125),
                 lambda: K8.kv8_store(q.view(1, 256), k, k, None, None, rot, ints([pos]), ints([row]), t, cache, 4, 1e-6),
                 lambda: K8.kv8_read(cache, ints([[row, pos, 1, 0]]), 1, 1, t))
        for call in calls:
            call()
            with pytest.raises(NativeError):
                tcgen05.check_errors(q.device)
    K8.kv8_read(cache, ints([[0, 0, 10, 5]]), 12, 10, table)
    with pytest.raises(NativeError):
        tcgen05.check_errors(q.device)
    K8.kv8_read(cache, ints([[0, -1, 1, 0]]), 1, 1, table)
    with pytest.raises(NativeError):
        tcgen05.check_errors(q.device)
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.exps)))


@pytest.mark.parametrize("T,h,kv,hd,dims,norm,gated,first", [
    (1, 16, 8, 128, 128, True, False, 699), (33, 9, 1, 128, 64, True, True, 0), (511, 3, 2, 64, 64, True, False, 70), (513, 5, 2, 64, 16, False, False, 5),
    (520, 16, 4, 256, 64, True, True, 100), (9, 4, 2, 128, 96, True, False, 1000000), (7, 2, 1, 96, 96, True, False, 262000), (5, 2, 2, 80, 20, True, True, 3),
    (65, 4, 4, 16, 0, True, False, 63), (12, 4, 2, 48, 34, False, True, 1)])
def test_store(T, h, kv, hd, dims, norm, gated, first):
    """Widths, rotated parts, head counts around a block's eight warps, both grids, far positions, strided rows; then reading back.  Queries
    are off by half a step of bf16 (2^-8 of the value), keys by half a step of e4m3 (2^-4 of the value, or 2^-10 of the scale, which is at
    most the row's largest magnitude / 224), both by 2^-18 of the row's largest magnitude for fp32 sums, sines and products; values are the definition's bits."""
    g = torch.Generator(device="cuda").manual_seed(T + hd)
    qs = 2 * hd if gated else hd
    wide = torch.randn(T, h * qs + 2 * kv * hd + 16, generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = wide[:, :h * qs], wide[:, h * qs:(h * qs + kv * hd)], wide[:, h * qs + kv * hd:h * qs + 2 * kv * hd]
    qn, kn = ((1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(torch.bfloat16) if norm else None for _ in range(2))
    lo, hi = first // 64, -(-(first + T) // 64)
    table = torch.zeros(1, hi, dtype=torch.int32, device="cuda")
    table[0, lo:] = torch.randperm(hi - lo + 2, generator=torch.Generator().manual_seed(T))[:hi - lo].to(torch.int32)
    cache = K8.Kv8Cache.allocate(hi - lo + 2, 64, kv, hd, "cuda")
    cache.k.fill_(7), cache.v.fill_(7), cache.exps.fill_(7)
    pos, idx = torch.arange(first, first + T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    rot = RotaryTable(dims, rotary_table(dims, 1e6).freq.cuda(), 1.25)
    got = K8.kv8_store(q, k, v, qn, kn, rot, pos, idx, table, cache, h, 1e-6, q_stride=qs)
    tcgen05.check_errors(q.device)

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        ang = torch.outer(pos.double(), rot.freq.double())[:, None]
        a, b = x[..., :dims // 2], x[..., dims // 2:dims]
        return torch.cat([(a * ang.cos() - b * ang.sin()) * 1.25, (b * ang.cos() + a * ang.sin()) * 1.25, x[..., dims:]], -1)

    want = turned(q.reshape(T, h, qs)[..., :hd], qn)
    size = want.abs().amax(-1, keepdim=True)
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * size).all()
    slots = table[0, (pos // 64).long()].long() * 64 + pos.long() % 64
    exps = cache.exps[slots // 64, :, :, slots % 64]
    want = turned(k.reshape(T, kv, hd), kn)
    size = want.abs().amax(-1, keepdim=True)
    keys = held(cache.k[slots], exps[..., 0])
    assert ((keys - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * size / 224 + 2.0 ** -18 * size).all()
    assert ((exps[..., 0].double() - 127 - exponent(size[..., 0])).abs() <= 1).all() and (exps[..., 0].double() - 127 != exponent(size[..., 0])).sum() <= 1
    c, e = K8.kv8_quantize(v.reshape(T, kv, hd).float())
    assert torch.equal(cache.v[slots], c) and torch.equal(exps[..., 1], e)
    others = torch.ones(cache.k.shape[0], dtype=torch.bool, device="cuda")
    others[slots] = False
    assert (cache.k[others] == 7).all() and (cache.v[others] == 7).all() and (cache.exps.permute(0, 3, 1, 2).flatten(0, 1)[others] == 7).all()
    kk, vv = K8.kv8_read(cache, ints([[0, first, T, 0]]), T, T, table)
    assert torch.equal(kk.double(), keys) and torch.equal(vv.double(), held(c, e))
    # rows between two vector loads: the same bits
    odd = torch.cat([wide.new_zeros(T, 1), wide], 1)[:, 1:]
    assert odd.data_ptr() % 4 and torch.equal(K8.kv8_store(odd[:, :h * qs], odd[:, h * qs:h * qs + kv * hd], odd[:, h * qs + kv * hd:h * qs + 2 * kv * hd], qn, kn,
                                                           rot, pos, idx, table, cache, h, 1e-6, q_stride=qs), got)
    assert torch.equal(held(cache.k[slots], exps[..., 0]), keys)


def test_store_of_rows_that_are_not_finite_and_of_padding():
    """Zeros, infinities, NaN and magnitudes beyond the largest scale as the definition has them; a position of -1 leaves the cache alone."""
    hd = 64
    v = torch.randn(6, 2 * hd, device="cuda").to(torch.bfloat16)
    v[0] = 0
    v[1, 3], v[2, 70], v[3, 5] = float("inf"), float("nan"), float("-inf")
    v[4, 9] = 3e38
    pos, idx, table = ints([0, 1, 2, 3, 64, -1]), torch.zeros(6, dtype=torch.int32, device="cuda"), ints([[1, 0]])
    cache = K8.Kv8Cache.allocate(2, 64, 2, hd, "cuda")
    cache.k.fill_(9), cache.v.fill_(9), cache.exps.fill_(9)
    K8.kv8_store(v, v, v, None, None, RotaryTable(0, torch.empty(0, device="cuda"), 1.0), pos, idx, table, cache, 2, 1e-6)
    c, e = K8.kv8_quantize(v.reshape(6, 2, hd).float())
    slots = torch.tensor([64, 65, 66, 67, 0], device="cuda")
    for which, codes in enumerate((cache.k, cache.v)):
        assert torch.equal(held(codes[slots], e[:5]).nan_to_num(-1.5), held(c[:5], e[:5]).nan_to_num(-1.5))
        assert torch.equal(cache.exps[slots // 64, :, which, slots % 64], e[:5])
    assert (cache.k == 9).flatten(1).all(1).sum() == 128 - 5
    tcgen05.check_errors(v.device)


def test_store_of_normed_rows_without_a_finite_mean():
    """Means of squares of zero, beyond fp32 and infinite, as the definition on a CPU has them: zeros beside a value that is not finite."""
    hd, w = 64, torch.ones(64, dtype=torch.bfloat16)
    x = torch.randn(5, 2 * hd, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    x[0] = 0
    x[1, 3], x[2, 70], x[3, 5] = float("inf"), 3e38, float("nan")
    results = []
    for device in ("cpu", "cuda"):
        y, weights = x.to(device), w.to(device)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
        cache, table = K8.Kv8Cache.allocate(1, 64, 2, hd, device), i32([[0]])
        q = K8.kv8_store(y, y, y, weights, weights, RotaryTable(0, torch.empty(0, device=device), 1.0), i32(list(range(5))), i32([0] * 5), table, cache, 2, 1e-6)
        results.append([t.float().cpu() for t in (q, *K8.kv8_read(cache, i32([[0, 0, 5, 0]]), 5, 5, table))])
    for a, b in zip(*results):
        assert torch.equal(a.isnan(), b.isnan()) and torch.allclose(a.nan_to_num(7.0), b.nan_to_num(7.0), rtol=2.0 ** -7, atol=0)
    assert results[0][0].isnan().any() and (results[0][0][1, 0].nan_to_num(0.0) == 0).all()
    tcgen05.check_errors(torch.device("cuda"))


@pytest.mark.parametrize("kv,hd,page", [(1, 16, 16), (3, 80, 64), (8, 128, 64), (2, 256, 48)])
def test_read(kv, hd, page):
    """Ranges of all lengths and starts, in any order, and rows between them that stay as they are."""
    cache, table, keys, values, _ = filled([500, 1, 64, 130], kv, hd, 4, page)
    ranges = [[0, 0, 500, 200], [3, 63, 67, 0], [1, 0, 1, 67], [2, 5, 0, 70], [2, 10, 54, 100], [0, 499, 1, 80]]
    got = K8.kv8_read(cache, ints(ranges), 700, 500, table)
    for out, rows in zip(got, (keys, values)):
        assert out.shape == (700, kv, hd)
        for b, first, n, row in ranges:
            assert torch.equal(out[row:row + n].double(), rows[b][first:first + n])
    tcgen05.check_errors(cache.k.device)


@pytest.mark.parametrize("spans,h,kv,hd,scale,page", [
    ([(0, 1), (0, 64), (0, 65)], 4, 2, 128, 1.0, 64), ([(0, 127), (0, 128), (0, 129)], 2, 2, 128, 1.0, 64), ([(63, 1), (64, 2), (190, 130)], 8, 1, 128, 1.0, 64),
    ([(0, 700)], 4, 1, 128, 3.0, 64), ([(1000, 300), (0, 17)], 2, 1, 64, 1.0, 64), ([(5, 59), (0, 257)], 16, 4, 64, 3.0, 64), ([(31, 40)], 4, 2, 128, 1.0, 32),
    ([(0, 16)] * 32, 16, 2, 64, 1.0, 64),
])
def test_prompts(spans, h, kv, hd, scale, page, monkeypatch):
    """(cached, new) tokens of each sequence: tile and page edges, ragged batches; all at once and in groups of sequences, with the longest history
    known or not, and with the first sequence's tokens as two ranges.  Bound as for decoding."""
    cache, table, keys, values, g = filled([c + n for c, n in spans], kv, hd, 1, page)
    T = sum(n for _, n in spans)
    q = (torch.randn(T, h, hd, generator=g, device="cuda") * scale).to(torch.bfloat16)
    pos = torch.cat([torch.arange(c, c + n) for c, n in spans]).to(torch.int32).cuda()
    idx = torch.cat([torch.full((n,), b) for b, (_, n) in enumerate(spans)]).to(torch.int32).cuda()
    cuts = torch.tensor([n for _, n in spans]).cumsum(0).tolist()
    longest = max(c + n for c, n in spans)
    for ends, known in (([0, *cuts], longest), ([0, *cuts], 0), (sorted({0, *cuts, (spans[0][1] + 1) // 2}), longest)):
        got = K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5, qo_indptr=ints(ends), max_q=max(n for _, n in spans), max_kv_len=known)
        tcgen05.check_errors(q.device)
        for b in range(len(spans)):
            a, e = [0, *cuts][b], cuts[b]
            assert near(got[a:e], attend(q[a:e], keys[b], values[b], pos[a:e], hd ** -0.5), values[b])
        monkeypatch.setattr(K8, "UNPACK_BUDGET_BYTES", 1)
        assert torch.equal(K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5, qo_indptr=ints(ends), max_q=max(n for _, n in spans), max_kv_len=known), got)
        monkeypatch.undo()
    tcgen05.check_errors(q.device)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("apart", [14, 15, 16, 40, 100])
def test_prompts_of_values_far_apart(hd, apart):
    """Pages whose values' scales are 2^apart apart, small ones first: what a query does not see yet leaves its result alone.  Tokens 100 on are the large ones,
    then every fifth from 300 on.  Bound as elsewhere, of the largest value that the query sees."""
    n, kv, h = 460, 2, 4
    cache, table, keys, _, g = filled([n], kv, hd, 5)
    x = torch.randn(n, kv, hd, generator=g, device="cuda")
    large = torch.zeros(n, dtype=torch.bool, device="cuda")
    large[100:140], large[300::5] = True, True
    x = torch.where(large[:, None, None], x * 2.0 ** (apart - apart // 2), x * 2.0 ** -(apart // 2))
    c, e = K8.kv8_quantize(x)
    slots = (table[0, torch.arange(n, device="cuda") // 64].long() * 64 + torch.arange(n, device="cuda") % 64)
    cache.v[slots] = c
    cache.exps[slots // 64, :, 1, slots % 64] = e
    values = held(c, e)
    first = 30
    q = torch.randn(n - first, h, hd, generator=g, device="cuda").to(torch.bfloat16)
    pos, idx = torch.arange(first, n, dtype=torch.int32, device="cuda"), torch.zeros(n - first, dtype=torch.int32, device="cuda")
    got = K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5, qo_indptr=ints([0, n - first]), max_q=n - first, max_kv_len=n)
    tcgen05.check_errors(q.device)
    want = attend(q, keys[0], values, pos, hd ** -0.5)
    for a, b in ((0, 100 - first), (100 - first, n - first)):
        assert near(got[a:b], want[a:b], values[:b + first])


def test_calls_in_a_captured_graph():
    """A step of prompts and one of single tokens, written, attended over and read back in one graph that is replayed with other rows, on another stream."""
    h, kv, hd, n = 8, 2, 128, 200
    rot = rotary_table(hd, 1e4).to("cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    rows = lambda t: torch.randn(t, (h + 2 * kv) * hd, generator=g, device="cuda").to(torch.bfloat16)
    table = ints([[3, 1, 0, 5]])
    cache, plain = (K8.Kv8Cache.allocate(6, 64, kv, hd, "cuda") for _ in range(2))
    prompt, token = rows(n), rows(1)
    pos, last, zeros = torch.arange(n, dtype=torch.int32, device="cuda"), ints([n]), torch.zeros(n, dtype=torch.int32, device="cuda")
    ends, ranges = ints([0, n]), ints([[0, 0, n + 1, 0]])

    def step(cache):
        out = []
        for x, p, more in ((prompt, pos, dict(qo_indptr=ends, max_q=n, max_kv_len=n)), (token, last, dict(max_kv_len=n + 1))):
            q, k, v = x.split([h * hd, kv * hd, kv * hd], 1)
            q = K8.kv8_store(q, k, v, None, None, rot, p, zeros[:x.shape[0]], table, cache, h, 1e-6)
            out.append(K8.kv8_attention(q, cache, p, zeros[:x.shape[0]], table, hd ** -0.5, **more))
        return [*out, *K8.kv8_read(cache, ranges, n + 1, n + 1, table)]

    step(cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache)
    other = torch.cuda.Stream()
    for _ in range(3):
        prompt.copy_(rows(n)), token.copy_(rows(1))
        want = step(plain)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graph.replay()
        torch.cuda.current_stream().wait_stream(other)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    tcgen05.check_errors(torch.device("cuda"))


def test_refusals_on_a_gpu():
    cache, table, _, _, g = filled([70], 2, 96, 2)
    pos, idx = ints([69]), ints([0])
    q = torch.randn(1, 4, 96, generator=g, device="cuda").to(torch.bfloat16)
    rot = rotary_table(96, 1e4).to("cuda")
    row = q.view(1, 384)
    for call in (lambda: K8.kv8_attention(q, cache, pos, idx, table, 0.1, qo_indptr=ints([0, 1])), lambda: K8.kv8_attention(q.float(), cache, pos, idx, table, 0.1),
                 lambda: K8.kv8_attention(q, cache, pos.cpu(), idx, table, 0.1), lambda: K8.kv8_attention(q.cpu(), cache, pos, idx, table, 0.1),
                 lambda: K8.kv8_store(row.float(), row[:, :192], row[:, :192], None, None, rot, pos, idx, table, cache, 4, 1e-6),
                 lambda: K8.kv8_store(row, row[:, :192], row[:, :192], torch.ones(96, device="cuda"), None, rot, pos, idx, table, cache, 4, 1e-6),
                 lambda: K8.kv8_store(row, row[:, :192], row[:, :192], None, None, rotary_table(96, 1e4), pos, idx, table, cache, 4, 1e-6)):
        with pytest.raises(ValueError):
            call()

"""The 8-bit key/value cache on a GPU where it is easily wrong: codes at the middle between two, bits that must not depend on the batch, weights of values whose
scales are the format's limits apart, values that are not finite behind a query, workspaces, ranges without keys."""
import numpy as np
import pytest
import torch

from kv8_util import attend, filled, held, near, round_e4m3
from slopllm_b200.ops import dense as D
from slopllm_b200.ops import kv8 as K8
from slopllm_b200.ops import tcgen05
from slopllm_b200.ops.native import NativeError
from slopllm_b200.ops.rotary import RotaryTable, rotary_table

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def put(cache, table, b, positions, which, rows):
    """fp32 rows [n, kv, hd] into places of sequence b, as keys (0) or values (1); what the cache then holds of them."""
    codes, exps = K8.kv8_quantize(rows)
    page = cache.page_size
    slots = table[b, (positions // page).long()].long() * page + positions.long() % page
    (cache.v if which else cache.k)[slots] = codes
    cache.exps[slots // page, :, which, slots % page] = exps
    return held(codes, exps)


# ---- writer ------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,h,kv,hd,dims,norm", [(3, 32, 8, 128, 128, True), (300, 9, 2, 64, 64, True), (5000, 32, 8, 128, 64, False), (700, 3, 1, 80, 20, True)])
def test_queries_do_not_depend_on_the_batch(T, h, kv, hd, dims, norm):
    """A token's query has the same bits alone, in a batch and in a chunk, whichever warp makes it."""
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, (h + 2 * kv) * hd, generator=g, device="cuda").to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(torch.bfloat16) if norm else None
    rot = rotary_table(dims, 1e6).to("cuda")
    pos = torch.randint(0, 100000, (T,), generator=g, device="cuda").to(torch.int32)
    idx, table = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    cache = K8.Kv8Cache.allocate(1, 64, kv, hd, "cuda")

    def queries(n):                                  # (places beyond the table are reported; only the queries count here)
        q, k, v = x[:n].split([h * hd, kv * hd, kv * hd], 1)
        out = K8.kv8_store(q, k, v, w, w, rot, pos[:n], idx[:n], table, cache, h, 1e-6)
        tcgen05.error_flag(out.device).zero_()
        return out

    whole = queries(T)
    for n in {1, 2, 17, 64, 299, 1100} & set(range(T)):
        assert torch.equal(queries(n), whole[:n]), n


@pytest.mark.parametrize("seed", [0, 1, 2, 3])
@pytest.mark.parametrize("hd,dims,norm,size", [(128, 128, True, 1.5), (128, 128, False, 1.5), (80, 20, True, 1.5), (256, 64, True, 1e-3), (64, 34, False, 1.5), (64, 64, True, 100.0)])
def test_stored_keys_are_the_nearest_codes(hd, dims, norm, size, seed):
    """Exponent and code of every key are those of the value in 64 bits.  Left out: values nearer than 2^-36 of the row's largest to the middle between two codes
    (the angle of position 6000 in quarter turns is good to 2^-41, products to 2^-52; fp32 gets some five of four million wrong, one if only the end is rounded to it)."""
    T, kv = 4096, 1024 // hd
    g = torch.Generator(device="cuda").manual_seed(hd + dims + 1000 * seed)
    k = (torch.randn(T, kv * hd, generator=g, device="cuda") * size).to(torch.bfloat16)
    w = (1 + 0.1 * torch.randn(hd, generator=g, device="cuda")).to(torch.bfloat16) if norm else None
    first = 2000
    pos, idx = torch.arange(first, first + T, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    table = ints([[max(0, i - first // 64) for i in range((first + T) // 64 + 1)]])
    cache = K8.Kv8Cache.allocate(int(table.max()) + 1, 64, kv, hd, "cuda")
    rot = RotaryTable(dims, rotary_table(dims, 1e6).freq.cuda(), 1.25)
    K8.kv8_store(k[:, :hd], k, k, None, w, rot, pos, idx, table, cache, 1, 1e-6)
    tcgen05.check_errors(k.device)
    x = k.view(T, kv, hd).double()
    if norm:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.double()
    ang = (pos.double()[:, None] * rot.freq.double())[:, None]
    a, b = x[..., :dims // 2], x[..., dims // 2:dims]
    want = torch.cat([(a * ang.cos() - b * ang.sin()) * 1.25, (b * ang.cos() + a * ang.sin()) * 1.25, x[..., dims:]], -1)
    slots = table[0, (pos // 64).long()].long() * 64 + pos.long() % 64
    exps = cache.exps[slots // 64, :, 0, slots % 64]
    top = want.abs().amax(-1)
    m, e = torch.frexp(top)                          # (logarithms on a GPU are off by a bit at powers of two)
    assert torch.equal(exps.int() - 127, e - 9 + (m > 0.875))
    scale = torch.exp2(exps.double() - 127)[..., None]
    z = want / scale
    step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    middle = (torch.floor(z.abs() / step) + 0.5) * step
    off = (z.abs() - middle).abs()
    sure = (off == 0) | (off > 2.0 ** -36 * (top[..., None] / scale))
    assert sure.double().mean() > 1 - 1e-5
    assert torch.equal(held(cache.k[slots], exps)[sure], (round_e4m3(z) * scale)[sure])


def test_keys_take_epsilon_and_gain_as_they_are():
    """`eps` and the rotation's gain are not rounded to fp32 on their way to a key: either would move these across the middle between two codes."""
    hd = 64
    ones = torch.ones(1, hd, device="cuda").to(torch.bfloat16)
    cache, table, zero = K8.Kv8Cache.allocate(1, 64, 1, hd, "cuda"), ints([[0]]), ints([0])
    free = RotaryTable(0, torch.empty(0, device="cuda"), 1.0)
    checked = [0, 0]
    for code in range(8, 15):                        # the middle between significands code / 8 and (code + 1) / 8
        m = (code + 0.5) / 16
        for up in (1, -1):
            eps = 1 / m ** 2 - 1 - up * 1e-12        # smaller: the key lies above the middle
            if (float(np.float32(eps)) - (1 / m ** 2 - 1)) * up > 0:
                K8.kv8_store(ones, ones, ones, None, torch.ones(hd, device="cuda").to(torch.bfloat16), free, zero, zero, table, cache, 1, eps)
                key = K8.kv8_read(cache, ints([[0, 0, 1, 0]]), 1, 1, table)[0].double()
                assert ((key - m) * up > 0).all(), (code, up)
                checked[0] += 1
        gain = m + 1e-12                             # (fp32 holds the middle itself, which would go to the even code)
        rot = RotaryTable(hd, torch.zeros(hd // 2, device="cuda"), gain)
        K8.kv8_store(ones, ones, ones, None, None, rot, zero, zero, table, cache, 1, 1e-6)
        assert (K8.kv8_read(cache, ints([[0, 0, 1, 0]]), 1, 1, table)[0].double() > m).all(), code
        checked[1] += 1
    assert min(checked) >= 3
    tcgen05.check_errors(ones.device)


def test_ranges_longer_than_promised_are_reported():
    """A range of more tokens than `longest` covers would leave rows unwritten."""
    cache, table, keys, values, _ = filled([500], 2, 64, 4)
    for longest in (400, 0):
        K8.kv8_read(cache, ints([[0, 0, 500, 0]]), 500, longest, table)
        with pytest.raises(NativeError):
            tcgen05.check_errors(cache.k.device)
    K8.kv8_read(cache, ints([[0, 0, 0, 0]]), 0, 0, table)
    got = K8.kv8_read(cache, ints([[0, 0, 500, 0]]), 500, 500, table)
    assert torch.equal(got[0].double(), keys[0]) and torch.equal(got[1].double(), values[0])
    tcgen05.check_errors(cache.k.device)


def test_reports_name_the_operator():
    """What a self-check finds is reported under the operator's own number."""
    cache, table, _, _, g = filled([100], 2, 64, 9)
    q = torch.randn(1, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    k, pos, row = q[:, :2].reshape(1, 128), ints([99]), ints([5])
    for site, call in ((60, lambda: K8.kv8_store(q.view(1, 256), k, k, None, None, rotary_table(64, 1e4).to("cuda"), pos, row, table, cache, 4, 1e-6)),
                       (61, lambda: K8.kv8_read(cache, ints([[5, 0, 1, 0]]), 1, 1, table)),
                       (62, lambda: K8.kv8_attention(q, cache, pos, row, table, 0.125)),
                       (63, lambda: K8.kv8_attention(q, cache, pos, row, table, 0.125, qo_indptr=ints([0, 1]), max_q=1, max_kv_len=100))):
        call()
        with pytest.raises(NativeError, match=f"site {site}:"):
            tcgen05.check_errors(q.device)


# ---- attention ---------------------------------------------------------------------------------------------------------------

def limits_apart(n, at, above, hd, page=64):
    """A history of keys and values of zero (exponent -60) with, at `at`, a row of the largest scale whose score lies 2^above above the others'."""
    cache, table, _, _, g = filled([n], 1, hd, n + at, page)
    every = torch.arange(n, device="cuda")
    keys, values = torch.zeros(n, 1, hd, device="cuda"), torch.zeros(n, 1, hd, device="cuda")
    values[at] = torch.randn(1, hd, generator=g, device="cuda").clamp(-3, 3) * 2.0 ** 66
    keys[at, 0, 0] = above * 0.6931471805599453
    k = put(cache, table, 0, every, 0, keys)
    v = put(cache, table, 0, every, 1, values)
    assert cache.exps[table[0, at // page].long(), 0, 1, at % page] > 127 + 56
    return cache, table, k, v


@pytest.mark.parametrize("above", [5, 9, 12])
@pytest.mark.parametrize("n,at", [(8000, 0), (8000, 4321), (8000, 7999), (300, 40), (300, 299)])
@pytest.mark.parametrize("h,hd", [(4, 64), (8, 128), (4, 256), (16, 64)])
def test_scales_at_the_limits_in_decoding(n, at, above, h, hd):
    """Rows of zeros count in the denominator beside a value of the largest scale, in the same warp, another one, another block.  A result is one weight
    (fp16, 2^-11) over a sum in fp32, rounded to bf16 (2^-8)."""
    cache, table, k, v = limits_apart(n, at, above, hd)
    q = torch.ones(1, h, hd, device="cuda").to(torch.bfloat16)
    pos, idx = ints([n - 1]), ints([0])
    want = attend(q, k, v, pos, 1.0)
    for longest in (n, 0):
        got = K8.kv8_attention(q, cache, pos, idx, table, 1.0, max_kv_len=longest)
        assert ((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -10) * want.abs()).all(), (got.double() / want).flatten()[:4]
    tcgen05.check_errors(q.device)


@pytest.mark.parametrize("above", [5, 9, 11])
@pytest.mark.parametrize("n,at", [(2000, 0), (2000, 1000), (2000, 1700), (150, 20)])
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_at_the_limits_in_prompts(n, at, above, hd):
    """The same for prompts, in pages of one scale and in those with a scale per token; queries in front of the large value give zeros."""
    cache, table, k, v = limits_apart(n, at, above, hd)
    first = n - 140
    q = torch.ones(140, 4, hd, device="cuda").to(torch.bfloat16)
    pos, idx = torch.arange(first, n, dtype=torch.int32, device="cuda"), torch.zeros(140, dtype=torch.int32, device="cuda")
    got = K8.kv8_attention(q, cache, pos, idx, table, 1.0, qo_indptr=ints([0, 140]), max_q=140, max_kv_len=n)
    want = attend(q, k, v, pos, 1.0)
    assert ((got.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -10) * want.abs()).all()
    tcgen05.check_errors(q.device)


@pytest.mark.parametrize("apart", [0, 40])
@pytest.mark.parametrize("n,first,h,kv,hd,scale", [(300, 0, 4, 2, 128, 0.1), (300, 100, 8, 2, 64, 0.1), (300, 0, 4, 2, 64, -0.1), (30, 0, 4, 2, 64, 0.1), (300, 230, 2, 2, 128, -0.1),
                                                   (2500, 2300, 16, 4, 128, 0.05)])
def test_values_that_are_not_finite_in_prompts(n, first, h, kv, hd, scale, apart):
    """A value's NaN code spoils its column for the queries that see it, a key's the heads of those queries, and nothing in front of them: both prompt kernels, pages of one
    scale and pages with a scale per token.  Bound as for decoding."""
    cache, table, keys, values, g = filled([n], kv, hd, n + hd)
    if apart:                                        # every seventh row is small
        x = torch.randn(n, kv, hd, generator=g, device="cuda")
        x[::7] *= 2.0 ** -apart
        values[0] = put(cache, table, 0, torch.arange(n, device="cuda"), 1, x)
    slot = lambda p: int(table[0, p // 64]) * 64 + p % 64
    bad = [(first + (n - first) * 2 // 5, 0, 5), (first + (n - first) // 2, kv - 1, 9), (first + (n - first) // 2 + 1, kv - 1, 9), (n - 1, 0, hd - 1)]
    spoiled_key = n - 3
    for p, head, d in bad:
        cache.v[slot(p), head, d] = 0xff if d == 9 else 0x7f
        values[0][p, head, d] = 0
    cache.k[slot(spoiled_key), kv - 1, 3] = 0x7f
    keys[0][spoiled_key, kv - 1, 3] = 0
    T = n - first
    q = torch.randn(T, h, hd, generator=g, device="cuda").to(torch.bfloat16)
    pos, idx = torch.arange(first, n, dtype=torch.int32, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    want = attend(q, keys[0], values[0], pos, scale)
    spoiled = torch.zeros_like(want, dtype=torch.bool)
    group = h // kv
    for p, head, d in bad:
        spoiled[:, head * group:(head + 1) * group, d] |= (pos >= p)[:, None]
    spoiled[:, (kv - 1) * group:] |= (pos >= spoiled_key)[:, None, None]
    assert spoiled.any() and not spoiled.all()
    got = K8.kv8_attention(q, cache, pos, idx, table, scale, qo_indptr=ints([0, T]), max_q=T, max_kv_len=n)
    tcgen05.check_errors(q.device)
    assert torch.equal(got.isnan(), spoiled)
    if scale > 0:
        assert near(got.masked_fill(spoiled, 0), want.masked_fill(spoiled, 0), values[0])
    else:                                            # (weights are one bf16 term in that kernel: 2^-8 of each)
        assert ((got.double() - want).masked_fill(spoiled, 0).abs() <= 2.0 ** -8 * (want.abs() + values[0].abs().max())).all()
    # single tokens have the same definition
    one = K8.kv8_attention(q, cache, pos, idx, table, scale, max_kv_len=n)
    assert torch.equal(one.isnan(), spoiled) and near(one.masked_fill(spoiled, 0), want.masked_fill(spoiled, 0), values[0])
    tcgen05.check_errors(q.device)


@pytest.mark.parametrize("scale", [-0.09, 0.0])
@pytest.mark.parametrize("hd", [64, 128])
def test_scales_of_scores_that_are_not_positive(scale, hd):
    """Negative and zero `sm_scale`, for which prompts take the other kernel."""
    n, first = 200, 60
    cache, table, keys, values, g = filled([n], 2, hd, 3)
    q = torch.randn(n - first, 4, hd, generator=g, device="cuda").to(torch.bfloat16)
    pos, idx = torch.arange(first, n, dtype=torch.int32, device="cuda"), torch.zeros(n - first, dtype=torch.int32, device="cuda")
    want = attend(q, keys[0], values[0], pos, scale)
    one = K8.kv8_attention(q, cache, pos, idx, table, scale, max_kv_len=n)
    assert near(one, want, values[0])
    got = K8.kv8_attention(q, cache, pos, idx, table, scale, qo_indptr=ints([0, n - first]), max_q=n - first, max_kv_len=n)
    # (weights are one bf16 term there: 2^-8 of each)
    assert ((got.double() - want).abs() <= 2.0 ** -8 * (want.abs() + values[0].abs().max())).all()
    tcgen05.check_errors(q.device)


@pytest.mark.parametrize("hd,kv,budget_pages_of_a_head", [(128, 4, 20), (64, 6, 45), (128, 4, 9)])
def test_the_workspace_keeps_its_budget(hd, kv, budget_pages_of_a_head, monkeypatch):
    """One history beyond the budget goes in groups of key heads: the same bits, and no more memory than the budget (of one key head, where that is more)."""
    n, T, h = 64 * 9 - 5, 6, 3 * kv
    cache, table, keys, values, g = filled([n, 100], kv, hd, 8)
    q = torch.randn(T + 3, h, hd, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.cat([torch.arange(n - T, n), torch.arange(97, 100)]).to(torch.int32).cuda()
    idx, ends = ints([0] * T + [1] * 3), ints([0, T, T + 3])
    call = lambda: K8.kv8_attention(q, cache, pos, idx, table, hd ** -0.5, qo_indptr=ends, max_q=T, max_kv_len=n)
    plain = call()
    budget = budget_pages_of_a_head * (64 * hd * 4 + 4 * 129 + 4)
    monkeypatch.setattr(K8, "UNPACK_BUDGET_BYTES", budget)
    torch.cuda.synchronize()
    base = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = call()
    torch.cuda.synchronize()
    # beside the workspace: the result, queries and results of the heads of a group, what the allocator rounds up
    more = 3 * q.numel() * 2 + 8 * 512 + 8 * T
    assert torch.cuda.max_memory_allocated() - base <= budget + more
    assert torch.equal(got, plain)
    tcgen05.check_errors(q.device)
    for b, (a, e) in enumerate(((0, T), (T, T + 3))):
        assert near(got[a:e], attend(q[a:e], keys[b], values[b], pos[a:e], hd ** -0.5), values[b])


@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_ranges_without_keys(scale):
    """Positions of -1 in a range of queries: rows without keys are zero, whole blocks of them too, also over the bf16 cache."""
    cache, table, keys, values, g = filled([100, 70], 2, 64, 5)
    q = torch.randn(400, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    pos = ints([-1] * 150 + list(range(100)) + [-1] * 10 + list(range(70)) + [-1] * 70)
    idx = ints([0] * 250 + [1] * 150)
    got = K8.kv8_attention(q, cache, pos, idx, table, scale, qo_indptr=ints([0, 250, 330, 400]), max_q=250, max_kv_len=100)
    tcgen05.check_errors(q.device)
    assert (got[pos < 0] == 0).all()
    for b, (a, e) in enumerate(((150, 250), (260, 330))):
        want = attend(q[a:e], keys[b], values[b], pos[a:e], scale)
        # (weights are one bf16 term in the kernel for a negative scale: 2^-8 of each)
        assert near(got[a:e], want, values[b]) if scale > 0 else ((got[a:e].double() - want).abs() <= 2.0 ** -8 * (want.abs() + values[b].abs().max())).all()
    rows = [torch.zeros(cache.k.shape, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, kept in zip(rows, (keys, values)):
        for b, y in enumerate(kept):
            at = torch.arange(y.shape[0], device="cuda")
            x[table[b, at // 64].long() * 64 + at % 64] = y.to(torch.bfloat16)
    plain = D.paged_attention(q, *rows, pos, idx, table, 64, scale, qo_indptr=ints([0, 250, 330, 400]), max_q=250, max_kv_len=100)
    tcgen05.check_errors(q.device)
    assert (plain[pos < 0] == 0).all() and not plain.isnan().any()


def test_any_negative_position_has_no_keys():
    """Not only -1: decoding and both prompt kernels."""
    cache, table, keys, values, g = filled([100], 2, 64, 6)
    q = torch.randn(6, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    pos, idx = ints([-1000, -64, -2, -90, -7, 99]), ints([0] * 6)
    for scale, more in ((0.1, {}), (0.1, dict(qo_indptr=ints([0, 3, 6]), max_q=3, max_kv_len=100)), (-0.1, dict(qo_indptr=ints([0, 3, 6]), max_q=3, max_kv_len=100))):
        got = K8.kv8_attention(q, cache, pos, idx, table, scale, **more)
        tcgen05.check_errors(q.device)
        assert (got[:5] == 0).all() and got[5].abs().max() > 0


@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_groups_of_key_heads_change_nothing(scale, monkeypatch):
    """A history that goes in groups of key heads, with values that are not finite, pages with a scale per token and other page sizes: the same bits."""
    n, first, h, kv, hd = 300, 90, 9, 3, 64
    for page in (64, 48):
        cache, table, _, _, g = filled([n], kv, hd, page, page)
        x = torch.randn(n, kv, hd, generator=g, device="cuda")
        x[::7, 1] *= 2.0 ** -40
        put(cache, table, 0, torch.arange(n, device="cuda"), 1, x)
        for p, head, d in ((120, 0, 3), (200, 2, 63), (201, 1, 0)):
            cache.v[int(table[0, p // page]) * page + p % page, head, d] = 0x7f
        q = torch.randn(n - first, h, hd, generator=g, device="cuda").to(torch.bfloat16)
        pos, idx = torch.arange(first, n, dtype=torch.int32, device="cuda"), torch.zeros(n - first, dtype=torch.int32, device="cuda")
        call = lambda: K8.kv8_attention(q, cache, pos, idx, table, scale, qo_indptr=ints([0, n - first]), max_q=n - first, max_kv_len=n)
        whole = call()
        assert whole.isnan().any() and not whole.isnan().all()
        for heads in (1, 2):
            monkeypatch.setattr(K8, "UNPACK_BUDGET_BYTES", heads * 5 * 17600)
            assert torch.equal(call().view(torch.int16), whole.view(torch.int16))
            monkeypatch.undo()
    tcgen05.check_errors(q.device)

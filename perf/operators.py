"""Operators of the 8-bit key/value cache of the grouped-query families, as cases that can be timed and checked:

* "store": a step's projection rows -> per-head norms of queries and keys, rotation, queries in bf16, keys and values quantised into the
  paged cache; the rows are then read back from the cache, so that what it holds comes back as the values that it stands for;
* "read": the cached rows of several sequences, out of their pages, as bf16 rows (what prompts attend over);
* "decode": attention of one new token per sequence over its cached rows;
* "prompt": causal attention of portions of prompts over the cached rows, the portion's own among them.

The cache: a token's row of one key head is `hd` e4m3 codes and one exponent byte b, for keys and for values; value = code * 2^(b - 127).
The exponent is the smallest with which the row's largest magnitude is at most 448, between -60 and 60.  Codes lie at [slot, head, :] with
slot = page * 64 + offset, exponent bytes at [page, head, 0 (keys) or 1 (values), offset].

A case: {"op", "seqs": sequences, "tokens": new tokens of all sequences (store, prompt) or the longest history (read, decode), "start": the
longest history in front of the new tokens (store, prompt), "heads", "kv": query and key heads, "hd": values of a head, "rot": rotated
ones, "norm": whether queries and keys are normed, "gate": whether a gate of `hd` values lies behind each query in the projection}.
"""
import math
import random

import torch

own = False

PAGE = 64
EPS = 1e-6
LOW, HIGH = -60, 60                     # limits of the exponent
F32, F64 = torch.float32, torch.float64


def _case(name, op, seqs, tokens, start, heads, kv, hd, rot=0, norm=False, gate=False):
    return {"name": name, "op": op, "seqs": seqs, "tokens": tokens, "start": start, "heads": heads, "kv": kv, "hd": hd, "rot": rot, "norm": norm,
            "gate": gate}


def listed():
    return [
        # one user's next token on the smallest dense model: latency
        _case("store-1", "store", 1, 1, 699, 16, 8, 128, 128, True),
        # a ragged decoding batch far into long histories
        _case("store-61-far", "store", 61, 61, 130000, 32, 8, 128, 128, True),
        # wide heads with a gate behind each query and a part of the values rotated, a few prompts' portions
        _case("store-333-gate", "store", 3, 333, 1000, 16, 2, 256, 64, True, True),
        # a whole chunk of a long prompt
        _case("store-4096", "store", 1, 4096, 8192, 32, 8, 128, 128, True),
        # what a chunk behind ragged histories attends over
        _case("read-ragged", "read", 5, 9000, 0, 8, 8, 128),
        # one short conversation: latency
        _case("decode-1-short", "decode", 1, 700, 0, 16, 8, 128),
        # one very long conversation: the keys of one sequence over the whole device
        _case("decode-1-long", "decode", 1, 131072, 0, 32, 8, 128),
        # a serving batch of ragged histories
        _case("decode-48-ragged", "decode", 48, 8192, 0, 32, 8, 128),
        # many users, narrow heads, many query heads a key head
        _case("decode-200-narrow", "decode", 200, 2500, 0, 64, 4, 64),
        # wide heads, 8 query heads a key head
        _case("decode-7-wide", "decode", 7, 5000, 0, 16, 2, 256),
        # several prompts packed into a chunk
        _case("prompt-ragged", "prompt", 3, 1700, 900, 16, 4, 64),
        # a chunk of a long prompt
        _case("prompt-4096", "prompt", 1, 4096, 8192, 32, 8, 128),
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    """Another call of the same kinds: sizes over their whole ranges, odd ones among them."""
    case = _draw(rng)
    del case["name"]
    return case


def _draw(rng):
    op = rng.choice(["store", "store", "read", "decode", "decode", "decode", "prompt"])
    hd = rng.choice([64, 128]) if op == "prompt" else rng.choice([128, 128, 64, 256, 32, 80, 96, 112, 192])
    kv, group = rng.choice([1, 2, 4, 8, 8, 16]), rng.choice([1, 2, 4, 4, 8, 16])
    while kv * group > 64:
        group //= 2
    heads = kv * group
    if op == "store":
        seqs = _log(rng, 1, 256)
        tokens = max(seqs, _log(rng, 1, 4096))
        rot = hd // rng.choice([1, 1, 2, 4]) // 2 * 2
        return _case("", op, seqs, tokens, _log(rng, 1, 200000), heads, kv, hd, rot, rng.random() < 0.7, rng.random() < 0.3)
    row = kv * hd
    if op == "prompt":
        tokens, start = _log(rng, 2, 4096), _log(rng, 1, 8192)
        return _case("", op, rng.randint(1, max(1, min(6, tokens // 16))), tokens, start, min(heads, 32), min(kv, min(heads, 32)), hd)
    seqs = _log(rng, 1, 256 if op == "decode" else 16)
    most = max(64, min(131072, (1 << 28) // (seqs * row)))
    return _case("", op, seqs, _log(rng, 1, most), 0, heads, kv, hd)


# ---- layout of a case --------------------------------------------------------------------------------------------------------

def _lengths(case):
    """(tokens in front, new tokens) of every sequence."""
    B, n, r = case["seqs"], case["tokens"], random.Random(case["seqs"] * 100003 + case["tokens"])
    if case["op"] in ("read", "decode"):
        return [(n - 1, 1)] + [(max(1, round(n * r.uniform(0.1, 1.0))) - 1, 1) for _ in range(B - 1)]
    cuts = sorted(r.sample(range(1, n), B - 1)) if B > 1 else []
    new = [b - a for a, b in zip([0, *cuts], [*cuts, n])]
    return [(case["start"] if b == 0 else round(case["start"] * r.uniform(0.0, 1.0)), m) for b, m in enumerate(new)]


def _row_bytes(case):
    return 2 * case["kv"] * (case["hd"] + 1)


def work(case):
    spans = _lengths(case)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    T = sum(m for _, m in spans)
    total = sum(a + m for a, m in spans)
    if case["op"] == "store":
        return {"bytes": 2 * T * (h + 2 * kv) * hd + 2 * T * h * hd + T * _row_bytes(case) + 4 * T * kv * hd, "flops": 12 * T * (h + 2 * kv) * hd}
    if case["op"] == "read":
        return {"bytes": total * (_row_bytes(case) + 4 * kv * hd), "flops": 2 * total * kv * hd}
    pairs = sum(m * a + m * (m + 1) // 2 for a, m in spans)
    return {"bytes": total * _row_bytes(case) + 4 * T * h * hd, "flops": 4 * pairs * h * hd}


def _quantised(x):
    """fp32 rows [..., hd] -> (codes as e4m3, exponents)."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = (e - 9 + (m > 0.875)).clamp(LOW, HIGH)
    e = torch.where(m == 0, torch.full_like(e, LOW), e)
    return torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn), e


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    spans = _lengths(case)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    # (pages of each sequence that the call touches: all of them, or those that get rows)
    per = [(a // PAGE if case["op"] == "store" else 0, -(-(a + m) // PAGE)) for a, m in spans]
    need = sum(hi - lo for lo, hi in per)
    pages = need + 3
    order = random.Random(seed).sample(range(pages), need)
    table = torch.zeros(len(spans), max(hi for _, hi in per) + 1, dtype=torch.int32)
    at = 0
    for b, (lo, hi) in enumerate(per):
        table[b, lo:hi] = torch.tensor(order[at:at + hi - lo], dtype=torch.int32)
        at += hi - lo
    new = [m for _, m in spans]
    T = sum(new)
    s = {"case": case, "page_table": table.to(dev),
         "positions": torch.cat([torch.arange(a, a + m, dtype=torch.int32) for a, m in spans]).to(dev),
         "batch_idx": torch.repeat_interleave(torch.arange(len(spans), dtype=torch.int32), torch.tensor(new)).to(dev),
         "ends": torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=dev),
         "spans": spans, "longest": max(a + m for a, m in spans), "scale": hd ** -0.5,
         "codes": [], "exps": torch.zeros(pages, kv, 2, PAGE, dtype=torch.uint8, device=dev)}
    for i in range(2):                                   # keys of about unit size, values whose size differs from token to token
        codes = torch.zeros(pages * PAGE, kv, hd, dtype=torch.uint8, device=dev)
        if case["op"] != "store":
            step = max(1, (1 << 26) // (PAGE * kv * hd))
            for p in range(0, pages, step):
                n = min(step, pages - p)
                x = torch.randn(n * PAGE, kv, hd, generator=g, device=dev)
                if i:
                    x = x * torch.exp(torch.randn(n * PAGE, kv, 1, generator=g, device=dev) * 0.7)
                c, e = _quantised(x)
                codes[p * PAGE:(p + n) * PAGE] = c.view(torch.uint8)
                s["exps"][p:p + n, :, i] = (e + 127).to(torch.uint8).view(n, PAGE, kv).transpose(1, 2)
        s["codes"].append(codes)
    if case["op"] == "store":
        qs = hd * (2 if case["gate"] else 1)
        s["q_stride"] = qs
        s["proj"] = (torch.randn(T, h * qs + 2 * kv * hd, generator=g, device=dev) * 1.5).to(torch.bfloat16)
        s["norms"] = [(1 + 0.1 * torch.randn(hd, generator=g, device=dev)).to(torch.bfloat16) if case["norm"] else None for _ in range(2)]
        s["freq"] = torch.tensor([1e6 ** (-2.0 * i / case["rot"]) for i in range(case["rot"] // 2)], dtype=F32, device=dev)
    elif case["op"] != "read":
        s["q"] = (torch.randn(T, h, hd, generator=g, device=dev) * 1.5).to(torch.bfloat16)
    # the tokens to be read back: (row of the page table, first position, count, first row of the result) of each sequence
    first = [(a, m) if case["op"] == "store" else (0, a + m) for a, m in spans]
    ends = [0, *torch.tensor([n for _, n in first]).cumsum(0).tolist()]
    s["ranges"] = torch.tensor([[b, a, n, ends[b]] for b, (a, n) in enumerate(first)], dtype=torch.int32, device=dev)
    s["rows"], s["most_rows"] = ends[-1], max(n for _, n in first)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------

def _parts(s):
    """Query, key and value rows [T, heads, hd] of the projection, fp32."""
    c, x, T = s["case"], s["proj"], s["proj"].shape[0]
    kb = c["heads"] * s["q_stride"]
    vb = kb + c["kv"] * c["hd"]
    q = x[:, :kb].view(T, c["heads"], s["q_stride"])[..., :c["hd"]]
    return q.to(F32), x[:, kb:vb].view(T, c["kv"], c["hd"]).to(F32), x[:, vb:].view(T, c["kv"], c["hd"]).to(F32)


def _plain_turn(x, w, s):
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(F32)
    angle = s["positions"].to(F64)[:, None] * s["freq"].to(F64)              # (far positions: 32 bits lose the angle)
    cos, sin = angle.cos().to(F32)[:, None], angle.sin().to(F32)[:, None]
    half, dims = s["case"]["rot"] // 2, s["case"]["rot"]
    a, b = x[..., :half], x[..., half:dims]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., dims:]], -1)


def _plain_store(s):
    q, k, v = _parts(s)
    out = [_plain_turn(q, s["norms"][0], s).to(torch.bfloat16)]
    codes, e = _quantised(torch.stack([_plain_turn(k, s["norms"][1], s), v]))
    back = torch.ldexp(codes.to(F32), e[..., None]).to(torch.bfloat16)
    return out + [back[0], back[1]]


def _plain_rows(s):
    """Keys and values of every page of the page table, fp32 [seqs, tokens, kv, hd]."""
    c, table = s["case"], s["page_table"].long()
    B, P = table.shape
    slots = (table[..., None] * PAGE + torch.arange(PAGE, device=table.device)).view(B, P * PAGE)
    exps = s["exps"][table].permute(3, 0, 1, 4, 2).reshape(2, B, P * PAGE, c["kv"], 1).to(torch.int32) - 127
    k = torch.ldexp(s["codes"][0][slots].view(torch.float8_e4m3fn).to(F32), exps[0])
    return k, torch.ldexp(s["codes"][1][slots].view(torch.float8_e4m3fn).to(F32), exps[1])


def _plain_read(s):
    """The rows of every range, one range behind the other."""
    width = s["page_table"].shape[1] * PAGE
    b, first, n, row = s["ranges"].long().unbind(1)
    at = torch.repeat_interleave(b * width + first - row, n) + torch.arange(s["rows"], device="cuda")
    return [x.view(-1, s["case"]["kv"], s["case"]["hd"])[at].to(torch.bfloat16) for x in _plain_rows(s)]


def _plain_attention(s):
    """Queries padded to [seqs, longest portion], scores of all pairs."""
    c, q = s["case"], s["q"].to(F32)
    T, B, g = q.shape[0], c["seqs"], c["heads"] // c["kv"]
    bi = s["batch_idx"].long()
    at = torch.arange(T, device="cuda") - s["ends"].long()[bi]
    most = max(m for _, m in s["spans"])
    x = torch.zeros(B, most, c["heads"], c["hd"], device="cuda")
    pos = torch.full((B, most), -1, device="cuda")
    x[bi, at] = q
    pos[bi, at] = s["positions"].long()
    k, v = _plain_rows(s)
    # (a place behind the history may hold anything)
    seen = torch.arange(k.shape[1], device="cuda") <= pos.max(1).values[:, None]
    k, v = (torch.where(seen[..., None, None], y, torch.zeros((), device="cuda")).permute(0, 2, 1, 3) for y in (k, v))
    x = x.view(B, most, c["kv"], g, c["hd"]).permute(0, 2, 3, 1, 4).reshape(B, c["kv"], g * most, c["hd"])
    sc = (x @ k.transpose(-1, -2)).view(B, c["kv"], g, most, -1) * s["scale"]
    sc = sc.masked_fill(torch.arange(sc.shape[-1], device="cuda") > pos[:, None, None, :, None], float("-inf"))
    e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-1e30))
    o = (e.view(B, c["kv"], g * most, -1) @ v).view(B, c["kv"], g, most, -1) / e.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, most, c["heads"], c["hd"])[bi, at].to(torch.bfloat16)


# ---- the framework's operators -------------------------------------------------------------------------------------------------

def _own(s):
    from slopllm_b200.ops import kv8 as K8
    from slopllm_b200.ops.rotary import RotaryTable
    c = s["case"]
    cache = K8.Kv8Cache(s["codes"][0], s["codes"][1], s["exps"])
    step = (s["positions"], s["batch_idx"], s["page_table"])
    if c["op"] == "store":
        x, kb = s["proj"], c["heads"] * s["q_stride"]
        vb = kb + c["kv"] * c["hd"]
        q = K8.kv8_store(x[:, :kb], x[:, kb:vb], x[:, vb:], *s["norms"], RotaryTable(c["rot"], s["freq"], 1.0), *step, cache, c["heads"], EPS,
                         q_stride=s["q_stride"])
        return [q, *K8.kv8_read(cache, s["ranges"], s["rows"], s["most_rows"], s["page_table"])]
    if c["op"] == "read":
        return list(K8.kv8_read(cache, s["ranges"], s["rows"], s["most_rows"], s["page_table"]))
    if c["op"] == "decode":
        return K8.kv8_attention(s["q"], cache, *step, s["scale"], max_kv_len=s["longest"])
    return K8.kv8_attention(s["q"], cache, *step, s["scale"], qo_indptr=s["ends"], max_q=max(m for _, m in s["spans"]), max_kv_len=s["longest"])


def run(s):
    if own:
        return _own(s)
    if s["case"]["op"] == "store":
        return _plain_store(s)
    return _plain_read(s) if s["case"]["op"] == "read" else _plain_attention(s)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def _e4m3_values(x):
    """fp64 -> the nearest numbers with 4 significant bits, ties to even, steps of 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _e4m3_of(codes):
    """fp64 numbers of e4m3 bytes, from their bits."""
    c = codes.to(torch.int64)
    exp, man = c >> 3 & 15, (c & 7).to(F64) / 8
    mag = torch.where(exp == 0, man * 2.0 ** -6, (1 + man) * torch.exp2((exp - 7).to(F64)))
    return torch.where(c >= 128, -mag, mag)


def _exact_store(s, case):
    h, kv, hd, dims = case["heads"], case["kv"], case["hd"], case["rot"]
    x, T = s["proj"].to(F64), s["proj"].shape[0]
    turn = torch.outer(s["positions"].to(F64), s["freq"].to(F64))[:, None]

    def rotated(y, w):
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w.to(F64)
        z = torch.complex(y[..., :dims // 2], y[..., dims // 2:dims]) * torch.polar(torch.ones_like(turn), turn)
        return torch.cat([z.real, z.imag, y[..., dims:]], -1)

    def held(y):
        top = y.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2(top / 448)).clamp(LOW, HIGH)
        return _e4m3_values(y * torch.exp2(-e)) * torch.exp2(e)

    n = h * s["q_stride"]
    q = rotated(x[:, :n].reshape(T, h, s["q_stride"])[..., :hd], s["norms"][0])
    k = held(rotated(x[:, n:n + kv * hd].reshape(T, kv, hd), s["norms"][1]))
    return [q, k, held(x[:, n + kv * hd:].reshape(T, kv, hd))]


def _exact_rows(s, case, b, n, which, head=None):
    """Rows 0 .. n-1 of sequence b, fp64 [n, kv, hd] (or of one head)."""
    pages = s["page_table"][b, :-(-n // PAGE)].long()
    heads = slice(None) if head is None else slice(head, head + 1)
    slots = (pages[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()[:n]
    e = s["exps"][pages][:, heads, which].transpose(1, 2).flatten(0, 1)[:n].to(F64) - 127
    return _e4m3_of(s["codes"][which][slots, heads]) * torch.exp2(e)[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(s, case)
    if case["op"] == "read":
        return [torch.cat([_exact_rows(s, case, b, a + m, which) for b, (a, m) in enumerate(s["spans"])]) for which in (0, 1)]
    out, at, g = [], 0, case["heads"] // case["kv"]
    for b, (a, m) in enumerate(s["spans"]):
        o = torch.zeros(m, case["heads"], case["hd"], dtype=F64, device="cuda")
        hidden = torch.arange(a + m, device="cuda")[None] > torch.arange(a, a + m, device="cuda")[:, None]
        for head in range(case["kv"]):
            k, v = (_exact_rows(s, case, b, a + m, which, head)[:, 0] for which in (0, 1))
            for j in range(head * g, head * g + g):
                sc = s["q"][at:at + m, j].to(F64) @ k.t() * s["scale"]
                o[:, j] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ v
        out.append(o)
        at += m
    return torch.cat(out)

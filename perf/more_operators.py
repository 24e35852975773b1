"""Operators of linear layers whose activations are quantised to 8 bits in front of FP8 weights, as cases that can be timed and checked:

* "norm": residual addition and RMS norm, with the normed rows in 8 bits; the rows are then read back, so that they come as the values that they stand for;
* "act": SiLU of the gate times up of a gated feed-forward (or, without a gate, rows as they are), in 8 bits; read back likewise;
* "product": rows in 8 bits times a matrix of FP8 weights;
* "mlp": a whole feed-forward as a decoder layer runs it: norm, gate and up products with their activation, down product.

Rows in 8 bits: groups of 128 values (the last may be shorter), a group is e4m3 codes and one exponent byte b; value = code * 2^(b - 127).  The
exponent is the smallest between -60 and 60 with which the group's largest magnitude is at most 448 * 2^exponent.  Weights: e4m3 codes [N, K] with one
fp32 scale for each block of 128 x 128.

A case: {"op", "tokens", "width": values of a row that goes in (norm, product, mlp) or comes out (act), "out": columns of the product or of the
feed-forward's gate, "f32": whether the input (norm, act) or the result (product) is fp32 in place of bf16, "first": no residual yet (norm),
"gated": (act)}.
"""
import math

import torch

own = False

GROUP = 128
EPS = 1e-6
LOW, HIGH = -60, 60                     # limits of the exponent
F32, F64, BF16 = torch.float32, torch.float64, torch.bfloat16
MOST = 4096 * 12288 * 4096              # products of the largest case


def _case(name, op, tokens, width, out=0, f32=False, first=False, gated=False):
    return {"name": name, "op": op, "tokens": tokens, "width": width, "out": out, "f32": f32, "first": first, "gated": gated}


def listed():
    return [
        # one user's next token on a small dense model: latency
        _case("norm-1", "norm", 1, 1024, f32=True),
        # an odd decoding batch of a wide model, behind a product in bf16
        _case("norm-61", "norm", 61, 5120),
        # a whole chunk of a prompt
        _case("norm-4096", "norm", 4096, 4096, f32=True),
        # a small decoding batch
        _case("act-7", "act", 7, 8192, gated=True),
        # attention's output in front of its projection, a few prompts' portions
        _case("rows-777", "act", 777, 2048),
        # a whole chunk of a prompt
        _case("act-4096", "act", 4096, 14336, gated=True),
        # one user's next token: the weights are streamed once
        _case("product-1", "product", 1, 4096, 6144),
        # a decoding batch, long rows into the residual stream
        _case("product-29", "product", 29, 12288, 4096, f32=True),
        # ragged sizes: neither rows, columns nor groups are whole
        _case("product-333-odd", "product", 333, 5136, 2321),
        # a whole chunk of a prompt
        _case("product-4096", "product", 4096, 4096, 12288),
        # a decoding batch through a feed-forward
        _case("mlp-8", "mlp", 8, 4096, 14336),
        # portions of prompts through a smaller one
        _case("mlp-1500", "mlp", 1500, 2048, 8192),
    ]


def _log(rng, lo, hi):
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    """Another call of the same kinds: sizes over their whole ranges, odd ones among them."""
    op = rng.choice(["norm", "act", "product", "product", "product", "mlp"])
    tokens = _log(rng, 1, 4096)
    width = 16 * _log(rng, 16, 896)
    if op == "norm":
        case = _case("", op, tokens, min(width, 8192), f32=rng.random() < 0.5, first=rng.random() < 0.2)
    elif op == "act":
        case = _case("", op, tokens, width, f32=rng.random() < 0.3, gated=rng.random() < 0.7)
    elif op == "product":
        out = _log(rng, 128, 14336)
        case = _case("", op, min(tokens, MOST // (width * out)), width, out, f32=rng.random() < 0.4)
    else:
        width, out = min(width, 5120), 16 * _log(rng, 32, 896)
        case = _case("", op, min(tokens, MOST // (3 * width * out)), width, out)
    del case["name"]
    return case


def _groups(n):
    return -(-n // GROUP)


def work(case):
    T, H, N = case["tokens"], case["width"], case["out"]
    size = 4 if case["f32"] else 2
    row = H + _groups(H)
    if case["op"] == "norm":
        return {"bytes": T * (H * size + (0 if case["first"] else 4 * H) + 4 * H + row + 2 * H) + 2 * H, "flops": 6 * T * H}
    if case["op"] == "act":
        return {"bytes": T * (H * size * (2 if case["gated"] else 1) + row + 2 * H), "flops": (6 if case["gated"] else 2) * T * H}
    if case["op"] == "product":
        return {"bytes": T * row + N * H + 4 * _groups(N) * _groups(H) + T * N * size, "flops": 2 * T * N * H}
    return {"bytes": T * (2 + 4 + 4 + 2) * H + 2 * H + 3 * N * H + 12 * _groups(N) * _groups(H), "flops": 6 * T * N * H}


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _weight(g, n, k):
    """Codes of normally distributed weights whose blocks differ in size, and the blocks' scales."""
    codes = torch.empty(n, k, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // k)
    for i in range(0, n, step):
        x = torch.randn(min(step, n - i), k, generator=g, device="cuda") * 110
        codes[i:i + step] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    scale = torch.exp(torch.randn(_groups(n), _groups(k), generator=g, device="cuda") * 0.3) / (110 * math.sqrt(k))
    return codes, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, H, N, op = case["tokens"], case["width"], case["out"], case["op"]
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    kind = F32 if case["f32"] else BF16
    s = {"case": case}
    if op in ("norm", "mlp"):                            # a residual stream whose tokens and channels differ in size
        size = torch.exp(rand(T, 1) * 0.5) * torch.exp(rand(1, H) * 0.5)
        s["x"] = (rand(T, H) * 0.3 * size).to(kind)
        s["residual"] = None if case["first"] else rand(T, H) * size
        s["norm"] = (1 + 0.1 * rand(H)).to(BF16)
    elif op == "act":
        s["x"] = (rand(T, H * (2 if case["gated"] else 1)) * torch.exp(rand(T, 1) * 0.5)).to(kind)
    else:                                                # normed rows: groups of about the same size, a few of them far larger
        s["codes"] = (rand(T, H) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        large = torch.rand(T, _groups(H), generator=g, device="cuda") < 0.02
        held = torch.zeros(T, -(-_groups(H) // 16) * 16, dtype=torch.uint8, device="cuda")       # (rows of exponents start at multiples of 16 bytes)
        s["exps"] = held[:, :_groups(H)]
        s["exps"].copy_(torch.randint(119, 122, large.shape, generator=g, device="cuda") + 3 * large)
        s["weight"] = _weight(g, N, H)
    if op == "mlp":
        s["gate_up"], s["down"] = _weight(g, 2 * N, H), _weight(g, H, N)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------

def _rows(v):
    """fp64 rows -> the values that their 8 bits stand for, fp32."""
    T, K = v.shape
    x = torch.nn.functional.pad(v, (0, -K % GROUP)).view(T, -1, GROUP)
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    e = torch.where(m == 0, torch.full_like(e, LOW), (e - 9 + (m > 0.875)).clamp(LOW, HIGH))
    x = torch.ldexp(x, -e).clamp(-448, 448)
    _, at = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    x = torch.ldexp(torch.round(torch.ldexp(x, 4 - at)), at - 4)             # 4 significant bits, ties to even
    return torch.ldexp(x, e).to(F32).view(T, -1)[:, :K]


def _plain_norm(s):
    r = s["x"].to(F32) if s["residual"] is None else s["residual"] + s["x"].to(F32)
    v = r.to(F64)
    return _rows(v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * s["norm"].to(F64)), r


def _plain_act(x):
    """(64 bits: values next to the border between two codes)"""
    g, u = x.to(F64).chunk(2, -1)
    return _rows(g / (1 + torch.exp(-g)) * u)


def _blocks(scale, n, k):
    return scale.repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]


def _plain_product(x, weight):
    """fp32 rows times a matrix of codes with the scales of its blocks."""
    codes, scale = weight
    return x @ (codes.view(torch.float8_e4m3fn).to(F32) * _blocks(scale, *codes.shape)).t()


def _plain(s):
    op = s["case"]["op"]
    if op == "norm":
        v, r = _plain_norm(s)
        return [v.to(BF16), r]
    if op == "act":
        return (_plain_act(s["x"]) if s["case"]["gated"] else _rows(s["x"].to(F64))).to(BF16)
    if op == "product":
        e = (s["exps"].to(torch.int32) - 127).repeat_interleave(GROUP, 1)[:, :s["codes"].shape[1]]
        x = torch.ldexp(s["codes"].view(torch.float8_e4m3fn).to(F32), e)
        return _plain_product(x, s["weight"]).to(F32 if s["case"]["f32"] else BF16)
    v, r = _plain_norm(s)
    act = _plain_act(_plain_product(v, s["gate_up"]))
    return [_plain_product(act, s["down"]).to(BF16), r]


# ---- the framework's operators -------------------------------------------------------------------------------------------------

def _own(s):
    from slopllm_b200.models.weights import LinearWeight
    from slopllm_b200.ops import fp8 as F8
    op, f32 = s["case"]["op"], s["case"]["f32"]
    weight = lambda name: LinearWeight(s[name][0], fp8_scale=s[name][1])
    if op == "norm":
        rows, r = F8.fp8_add_rmsnorm(s["x"], s["residual"], s["norm"], EPS)
        return [F8.fp8_values(rows), r]
    if op == "act":
        return F8.fp8_values(F8.fp8_silu_mul(s["x"]) if s["case"]["gated"] else F8.fp8_rows(s["x"]))
    if op == "product":
        return F8.fp8_linear(F8.Fp8Rows(s["codes"], s["exps"]), weight("weight"), out_f32=f32)
    rows, r = F8.fp8_add_rmsnorm(s["x"], s["residual"], s["norm"], EPS)
    return [F8.fp8_linear(F8.fp8_gate_up(rows, weight("gate_up")), weight("down")), r]


def run(s):
    return _own(s) if own else _plain(s)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------

def _table(device):
    """The 127 magnitudes of e4m3 in ascending order, from their bits."""
    c = torch.arange(127, device=device)
    exp, man = c >> 3, (c & 7).to(F64) / 8
    return torch.where(exp == 0, man * 2.0 ** -6, (1 + man) * torch.exp2((exp - 7).to(F64)))


def _codes_of(codes):
    mag = _table(codes.device)[(codes & 127).long()]
    return torch.where(codes >= 128, -mag, mag)


def _held(v):
    """fp64 rows -> the nearest values of the format, looked up."""
    T, K = v.shape
    table = _table(v.device)
    middle = (table[1:] + table[:-1]) / 2
    out = torch.empty_like(v)
    for a in range(0, K, GROUP):
        x = v[:, a:a + GROUP]
        e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -200) / 448)).clamp(LOW, HIGH)
        y = (x.abs() * torch.exp2(-e)).contiguous()
        below, above = torch.bucketize(y, middle), torch.bucketize(y, middle, right=True)
        at = torch.where(below % 2 == 0, below, above)                       # in the middle: the even one of both
        out[:, a:a + GROUP] = torch.sign(x) * table[at] * torch.exp2(e)
    return out


def _exact_product(x, weight, most=1 << 27):
    """x [T, K] fp64 times the matrix, some of its columns at a time."""
    codes, scale = weight
    n, k = codes.shape
    step = max(GROUP, most // k // GROUP * GROUP)
    out = torch.empty(x.shape[0], n, dtype=F64, device=x.device)
    for i in range(0, n, step):
        w = _codes_of(codes[i:i + step])
        w = w * _blocks(scale[i // GROUP:(i + step) // GROUP].to(F64), *w.shape)
        out[:, i:i + step] = torch.einsum("tk,nk->tn", x, w)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "act":
        x = s["x"].to(F64)
        if case["gated"]:
            half = case["width"]
            x = x[:, :half] * torch.sigmoid(x[:, :half]) * x[:, half:]
        return _held(x)
    if op == "product":
        x = _codes_of(s["codes"])
        for j in range(s["exps"].shape[1]):
            x[:, j * GROUP:(j + 1) * GROUP] *= torch.exp2(s["exps"][:, j:j + 1].to(F64) - 127)
        return _exact_product(x, s["weight"])
    r = s["x"].to(F32)
    if s["residual"] is not None:
        r = r + s["residual"]                            # (the residual stream is fp32: what is normed is what is kept)
    y = r.to(F64)
    rows = _held(y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * s["norm"].to(F64))
    if op == "norm":
        return [rows, r.to(F64)]
    gu, n = _exact_product(rows, s["gate_up"]), case["out"]
    return [_exact_product(_held(gu[:, :n] * torch.sigmoid(gu[:, :n]) * gu[:, n:]), s["down"]), r.to(F64)]

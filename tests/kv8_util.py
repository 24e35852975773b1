"""Caches of the 8-bit key/value format for tests, and what they hold in 64 bits, from the format's definition."""
import torch

from slopllm_b200.ops import kv8 as K8


def held(codes, exps):
    """fp64 values of code bytes [..., hd] and exponent bytes [...], from their bits."""
    c = codes.to(torch.int64)
    exp, man = c >> 3 & 15, (c & 7).double() / 8
    mag = torch.where(exp == 0, man * 2.0 ** -6, (1 + man) * torch.exp2((exp - 7).double()))
    mag = torch.where((c & 127) == 127, torch.full_like(mag, float("nan")), mag)
    return torch.where(c >= 128, -mag, mag) * torch.exp2(exps.double() - 127)[..., None]


def round_e4m3(x):
    """fp64 -> the nearest number of 4 significant bits, ties to even, in steps of 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exponent(top):
    """Smallest e in [-60, 60] with top * 2^-e <= 448."""
    return torch.ceil(torch.log2(top.double().clamp(min=1e-300) / 448)).clamp(-60, 60)


def table_of(histories, page, seed, device, spare=3):
    """Random pages for histories: (page table, slots of every sequence, number of pages)."""
    per = [-(-n // page) for n in histories]
    total = sum(per) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.zeros(len(histories), max(per) + 1, dtype=torch.int32)
    rows = []
    for b, n in enumerate(histories):
        pages = torch.tensor([order.pop() for _ in range(per[b])], dtype=torch.int32)
        table[b, :per[b]] = pages
        rows.append((pages.long()[:, None] * page + torch.arange(page)).flatten()[:n].to(device))
    return table.to(device), rows, total


def filled(histories, kv, hd, seed, page=64, device="cuda", sizes=0.7):
    """A cache whose rows outside the histories are NaN codes with the byte 255; (cache, page table, fp64 keys and values of every sequence)."""
    table, rows, total = table_of(histories, page, seed, device)
    cache = K8.Kv8Cache.allocate(total, page, kv, hd, device)
    cache.k.fill_(0x7f), cache.v.fill_(0xff), cache.exps.fill_(255)
    g = torch.Generator(device=device).manual_seed(seed)
    keys, values = [], []
    for s in rows:
        for which, (codes, out) in enumerate(((cache.k, keys), (cache.v, values))):
            x = torch.randn(s.numel(), kv, hd, generator=g, device=device)
            x = x * torch.exp(torch.randn(s.numel(), kv, 1, generator=g, device=device) * (sizes if which else 0.1))
            c, e = K8.kv8_quantize(x)
            codes[s] = c
            cache.exps[s // page, :, which, s % page] = e
            out.append(held(c, e))
    return cache, table, keys, values, g


def attend(q, k, v, positions, scale):
    """fp64 causal attention of q [T, h, hd] over k, v [n, kv, hd]."""
    g = q.shape[1] // k.shape[1]
    k, v = (x.repeat_interleave(g, 1) for x in (k, v))
    s = torch.einsum("thd,khd->htk", q.double(), k) * scale
    s = s.masked_fill(torch.arange(k.shape[0], device=q.device) > positions[:, None], float("-inf"))
    return torch.einsum("htk,khd->thd", torch.softmax(s, -1), v)


def near(got, want, values):
    """bf16 results of fp32 attention: half a step of bf16 (2^-8 of the value), and 2^-14 of the largest cached value for scores (below 64) that are
    good to 2^-21 and weights of one fp16 term: 2^-11 of each, of either sign, over the tens of keys that make a row's sum."""
    return bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * values.abs().max()).all())

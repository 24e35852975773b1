"""An 8-bit paged key/value cache for grouped-query attention: norm, rotation and quantised write, reading back, attention of prompts and of
single tokens.  It takes the place of the bf16 cache of `ops/dense.py` at half of its bytes (`--kv-dtype e4m3`).

A token's row of one key head is `hd` e4m3 codes and one exponent byte b, for keys and for values; value = code * 2^(b - 127).  The exponent
is the smallest between -60 and 60 with which the largest finite magnitude of the row is at most 448; larger values saturate, and a value that
is not finite is the NaN code: in attention a value's spoils its column, a key's the whole head, for the queries that see it and no other.
Codes lie at [slot, head, :] with slot = page * page_size + offset, exponent bytes at [page, head, 0 (keys) or 1 (values), offset].

CUDA tensors run `csrc/kv8.cu` and `csrc/kv8_attn.cu` (prompts: the tcgen05 kernel of `csrc/prefill_attn.cu` over rows read back, which bf16 holds
exactly); CPU tensors run the fp32 definition below.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from functools import lru_cache
from itertools import accumulate
from typing import Optional, Tuple

import torch

from . import native as N, reference as R, tcgen05
from .dense import AttnParams, _slots
from .rotary import RotaryTable

PROMPT_HEADS = (64, 128)               # widths of heads whose prompts the kernels attend over
LOW, HIGH, BIAS = -60, 60, 127         # limits of the exponent, and what is added to it in its byte
# Transient rows of a prompt step: more sequences go in groups, a longer history in groups of key heads (one head of 128 values takes it at 2.0 million tokens).
UNPACK_BUDGET_BYTES = 1 << 30


# (Kv8Pages and Kv8Rows of the kernels, spliced into the structures that hold them: a call makes one object)
_PAGES = [("page_table", C.c_void_p), ("pt_stride", C.c_int), ("pt_rows", C.c_int), ("pt_width", C.c_int), ("page_size", C.c_int),
          ("num_slots", C.c_int), ("guard", C.c_void_p)]
_ROWS = [("k_codes", C.c_void_p), ("v_codes", C.c_void_p), ("exps", C.c_void_p), *_PAGES, ("n_kv", C.c_int), ("hd", C.c_int)]


class Kv8StoreParams(C.Structure):
    _fields_ = [("q", C.c_void_p), ("ldq", C.c_int), ("k", C.c_void_p), ("ldk", C.c_int), ("v", C.c_void_p), ("ldv", C.c_int),
                ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("freq", C.c_void_p), ("gain", C.c_double), ("rot_dims", C.c_int),
                ("positions", C.c_void_p), ("batch_idx", C.c_void_p), *_PAGES, ("n_heads", C.c_int), ("n_kv", C.c_int),
                ("hd", C.c_int), ("q_stride", C.c_int), ("eps", C.c_double), ("q_out", C.c_void_p), ("k_codes", C.c_void_p),
                ("v_codes", C.c_void_p), ("exps", C.c_void_p), ("T", C.c_int)]


class Kv8ReadParams(C.Structure):
    _fields_ = [*_ROWS, ("ranges", C.c_void_p), ("rows", C.c_int), ("k", C.c_void_p), ("v", C.c_void_p)]


class Kv8UnpackParams(C.Structure):
    _fields_ = [*_ROWS, ("heads", C.c_int), ("qo_indptr", C.c_void_p), ("positions", C.c_void_p), ("batch_idx", C.c_void_p), ("per_seq", C.c_int),
                ("k", C.c_void_p), ("v", C.c_void_p), ("table", C.c_void_p), ("rows_out", C.c_void_p), ("positions_out", C.c_void_p),
                ("exps_out", C.c_void_p), ("scales", C.c_void_p), ("spoiled_pages", C.c_void_p), ("spoiled_dims", C.c_void_p)]


class Kv8DecodeParams(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k_codes", C.c_void_p), ("v_codes", C.c_void_p), ("exps", C.c_void_p), ("positions", C.c_void_p),
                ("batch_idx", C.c_void_p), *_PAGES, ("n_heads", C.c_int), ("n_kv", C.c_int), ("hd", C.c_int), ("scale", C.c_float),
                ("out", C.c_void_p), ("o_part", C.c_void_p), ("lse_part", C.c_void_p), ("jobs", C.c_void_p), ("T", C.c_int), ("err", C.c_void_p)]


@dataclass
class Kv8Cache:
    """One layer's cache.  `k`, `v`: uint8 [slots, n_kv, hd] e4m3 codes; `exps`: uint8 [pages, n_kv, 2, page_size]."""

    k: torch.Tensor
    v: torch.Tensor
    exps: torch.Tensor

    def __post_init__(self):
        slots, n_kv, hd = self.k.shape
        pages, heads, two, page_size = self.exps.shape
        if self.v.shape != self.k.shape or (pages * page_size, heads, two) != (slots, n_kv, 2):
            raise ValueError(f"codes {tuple(self.k.shape)} and {tuple(self.v.shape)} do not go with exponents {tuple(self.exps.shape)}")
        if slots >> 31:
            raise ValueError(f"{slots} slots: they are numbered in 31 bits")
        if hd % 16 or not 16 <= hd <= 256 or page_size % 16 or not page_size:
            raise ValueError(f"heads of {hd} values in pages of {page_size} tokens: the 8-bit cache takes multiples of 16, heads of up to 256")
        device = self.k.device
        for x in (self.k, self.v, self.exps):
            if x.dtype is not torch.uint8 or not x.is_contiguous() or x.device != device:
                raise ValueError("the tensors of an 8-bit cache are contiguous, of type uint8 and on one device")
        if (self.k.data_ptr() | self.v.data_ptr() | self.exps.data_ptr()) % 16:
            raise ValueError("the tensors of an 8-bit cache start at multiples of 16 bytes")

    @property
    def page_size(self) -> int:
        return self.exps.shape[3]

    @staticmethod
    def allocate(num_pages: int, page_size: int, n_kv: int, hd: int, device) -> "Kv8Cache":
        codes = lambda: torch.zeros(num_pages * page_size, n_kv, hd, dtype=torch.uint8, device=device)
        return Kv8Cache(codes(), codes(), torch.zeros(num_pages, n_kv, 2, page_size, dtype=torch.uint8, device=device))


def _check_step(device: int, cache: Kv8Cache, *tables: torch.Tensor) -> None:
    """Tables of a step are int32 on the device of the data and the cache, with values side by side."""
    if cache.k.get_device() != device:
        raise ValueError(f"data on device {device}, cache on {cache.k.device}")
    for t in tables:
        if t.dtype is not torch.int32 or t.get_device() != device or not (t.is_contiguous() or t.stride(-1) == 1 or t.shape[-1] <= 1):
            raise ValueError("positions, rows, ranges and page tables are int32, on the device of the data, with values side by side")


@lru_cache(maxsize=None)
def _status(device: int) -> int:
    """Address of a device's status words, which stay where they are."""
    return tcgen05.error_flag(torch.device("cuda", device)).data_ptr()


def _pages(cache: Kv8Cache, page_table: torch.Tensor) -> tuple:
    rows, width = page_table.shape
    return (page_table.data_ptr(), page_table.stride(0), rows, width, cache.exps.shape[3], cache.k.shape[0],
            _status(cache.k.get_device()) + 16)


def _rows(cache: Kv8Cache, page_table: torch.Tensor) -> tuple:
    return (cache.k.data_ptr(), cache.v.data_ptr(), cache.exps.data_ptr(), *_pages(cache, page_table), cache.k.shape[1], cache.k.shape[2])


def _call(device: int, name: str, *args) -> None:
    """A kernel call on the current stream of a device."""
    if device == torch._C._cuda_getDevice():
        N.call(name, *args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            N.call(name, *args, N.stream())


# ---- the format ----------------------------------------------------------------------------------------------------------------------

def kv8_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows [..., hd] -> (e4m3 codes, exponent bytes [...]), both uint8 (the definition)."""
    x = torch.where(x.isfinite(), x, torch.full_like(x, float("nan")))
    m, e = torch.frexp(x.nan_to_num(0.0).abs().amax(-1))
    e = torch.where(m == 0, torch.full_like(e, LOW), (e - 9 + (m > 0.875)).clamp(LOW, HIGH))
    codes = torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, (e + BIAS).to(torch.uint8)


def kv8_values(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """The fp32 values of codes [..., hd] with exponent bytes [...]."""
    return torch.ldexp(codes.view(torch.float8_e4m3fn).to(torch.float32), (exps.to(torch.int32) - BIAS)[..., None])


def _cached(cache: Kv8Cache, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 keys and values [n, n_kv, hd] of slots."""
    e = cache.exps[slots // cache.page_size, :, :, slots % cache.page_size]
    return kv8_values(cache.k[slots], e[..., 0]), kv8_values(cache.v[slots], e[..., 1])


# ---- operators -----------------------------------------------------------------------------------------------------------------------

def kv8_store(q, k, v, q_norm, k_norm, rot: RotaryTable, positions, batch_idx, page_table, cache: Kv8Cache, n_heads: int, eps: float,
              q_stride: Optional[int] = None) -> torch.Tensor:
    """:func:`~slopllm_b200.ops.dense.qk_norm_rope_cache` for the 8-bit cache: per-head RMS norm (weights [hd], or None) and rotation of the first
    `rot.dims` values of queries and keys; key and value rows go into their places quantised.  q [T, n_heads * q_stride] (head h starts at
    h * q_stride), k / v [T, n_kv * hd], bf16 on a GPU with rows of any stride.  Between the rows and the one rounding of a result everything
    is fp32, angles (position * frequency) are 64 bits, and on a GPU keys are, too.  A token whose position is negative leaves the cache as it is;
    no two tokens of a call have the same place.  Returns the queries [T, n_heads, hd]."""
    (T, width), (_, n_kv, hd), device = q.shape, cache.k.shape, q.get_device()
    q_stride = hd if q_stride is None else q_stride
    if width != n_heads * q_stride or q_stride < hd or k.shape != (T, n_kv * hd) or v.shape != k.shape:
        raise ValueError(f"projections {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} for {n_heads} heads over {n_kv} of {hd} values")
    if rot.dims > hd or rot.freq.numel() != rot.dims // 2 or rot.dims % 2:
        raise ValueError(f"{rot.dims} rotated values with {rot.freq.numel()} frequencies in heads of {hd}")
    if positions.shape != (T,) or batch_idx.shape != (T,):
        raise ValueError(f"{T} tokens with positions {tuple(positions.shape)} and rows {tuple(batch_idx.shape)}")
    _check_step(device, cache, positions, batch_idx, page_table)
    if device >= 0:
        (ldq, q_by), (ldk, k_by), (ldv, v_by) = q.stride(), k.stride(), v.stride()
        weights = [w for w in (q_norm, k_norm) if w is not None]
        for x in (q, k, v, *weights):
            if x.dtype is not torch.bfloat16 or x.get_device() != device:
                raise ValueError("projection rows and norm weights are bf16 and on one device")
        if q_by != 1 or k_by != 1 or v_by != 1 or any(w.stride(-1) != 1 for w in weights):
            raise ValueError("the values of projection rows and norm weights lie side by side")
        for w in weights:
            if w.shape != (hd,):
                raise ValueError(f"norm weights of {tuple(w.shape)} for heads of {hd} values")
        freq = rot.freq
        if freq.dtype is not torch.float32 or freq.get_device() != device or not freq.is_contiguous():
            raise ValueError("frequencies are fp32, contiguous and on the device of the data")
        out = q.new_empty((T, n_heads, hd))
        p = Kv8StoreParams(q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv, N.ptr(q_norm), N.ptr(k_norm), freq.data_ptr(), rot.gain,
                           rot.dims, positions.data_ptr(), batch_idx.data_ptr(), *_pages(cache, page_table), n_heads, n_kv, hd,
                           q_stride, eps, out.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.exps.data_ptr())
        _call(device, "sl_kv8_store", C.byref(p), T)
        return out

    def turned(x, w):
        x = x.to(torch.float32)
        if w is not None:
            x = R.rmsnorm(x, w, eps)
        half, ang = rot.dims // 2, (positions.double()[:, None] * rot.freq.double())[:, None]
        cos, sin = (ang.cos() * rot.gain).float(), (ang.sin() * rot.gain).float()
        a, b = x[..., :half], x[..., half:rot.dims]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot.dims:]], -1)

    on = positions >= 0
    slots = _slots(positions[on], batch_idx[on], page_table, cache.page_size)
    for which, (codes, x) in enumerate(((cache.k, turned(k.reshape(T, n_kv, hd), k_norm)), (cache.v, v.reshape(T, n_kv, hd).to(torch.float32)))):
        c, e = kv8_quantize(x[on])
        codes[slots] = c
        cache.exps[slots // cache.page_size, :, which, slots % cache.page_size] = e
    return turned(q.reshape(T, n_heads, q_stride)[..., :hd], q_norm).to(q.dtype)


def kv8_read(cache: Kv8Cache, ranges: torch.Tensor, rows: int, longest: int, page_table: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cached keys and values [rows, n_kv, hd] in bf16, which holds them exactly.  `ranges` int32 [R, 4]: page-table row, first position, number
    of tokens (at most `longest`; more are reported after the step), first row of the result; rows in no range are not written."""
    if ranges.dim() != 2 or ranges.shape[1] != 4 or not ranges.is_contiguous():
        raise ValueError(f"ranges are [R, 4] and contiguous, not {tuple(ranges.shape)}")
    device = ranges.get_device()
    _check_step(device, cache, ranges, page_table)
    _, n_kv, hd = cache.k.shape
    k = torch.empty(rows, n_kv, hd, dtype=torch.bfloat16, device=cache.k.device)
    v = torch.empty_like(k)
    if device >= 0:
        p = Kv8ReadParams(*_rows(cache, page_table), ranges.data_ptr(), rows, k.data_ptr(), v.data_ptr())
        _call(device, "sl_kv8_read", C.byref(p), ranges.shape[0], longest)
        return k, v
    for b, first, n, row in ranges.tolist():
        pos = torch.arange(first, first + n)
        kv = _cached(cache, _slots(pos, torch.full_like(pos, b), page_table, cache.page_size))
        k[row:row + n], v[row:row + n] = kv
    return k, v


def kv8_attention(q, cache: Kv8Cache, positions, batch_idx, page_table, sm_scale: float, qo_indptr: Optional[torch.Tensor] = None, max_q: int = 0,
                  max_kv_len: int = 0) -> torch.Tensor:
    """:func:`~slopllm_b200.ops.dense.paged_attention` over the 8-bit cache: causal attention of each query token (position positions[t],
    page-table row batch_idx[t]) over the keys 0..position of its sequence.  q [T, n_heads, hd], bf16 on a GPU -> [T, n_heads, hd].  With
    `qo_indptr` ([B + 1], contiguous token ranges of the sequences, at most `max_q` tokens and `max_kv_len` keys each; 0: not known; positions ascend
    within a range) heads have 64 or 128 values on a GPU, and rows in no range are not written; without it `max_kv_len` is a hint.  A row
    may have no keys (a negative position) and is zero.  At most 1024 query heads."""
    (T, n_heads, hd), device = q.shape, q.get_device()
    _, n_kv, width = cache.k.shape
    if hd != width or n_heads % n_kv:
        raise ValueError(f"{n_heads} query heads of {hd} values over {n_kv} key heads of {width}")
    if positions.shape != (T,) or batch_idx.shape != (T,):
        raise ValueError(f"{T} tokens with positions {tuple(positions.shape)} and rows {tuple(batch_idx.shape)}")
    _check_step(device, cache, positions, batch_idx, page_table)
    if device < 0:
        out = torch.zeros(T, n_heads, hd, dtype=torch.float32)
        for t in range(T):
            n = max(int(positions[t]) + 1, 0)
            kp = torch.arange(n)
            if n:
                k, v = _cached(cache, _slots(kp, torch.full_like(kp, int(batch_idx[t])), page_table, cache.page_size))
                out[t] = R.dense_attention(q[t:t + 1], k, v, sm_scale, causal_offset=n - 1)[0]
        return out.to(q.dtype)
    if q.dtype is not torch.bfloat16:
        raise ValueError(f"queries of type {q.dtype}: the kernels take bf16")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_like(q)
    if T == 0:
        return out
    if qo_indptr is None:
        blocks, parts, rows, wide = _decode_plan(device, n_heads, n_kv, hd)
        part = torch.empty(parts * (2 * rows * (wide + 1) + 4), dtype=torch.float32, device=q.device)
        sums = part.data_ptr() + parts * 16
        p = Kv8DecodeParams(q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.exps.data_ptr(), positions.data_ptr(), batch_idx.data_ptr(),
                            *_pages(cache, page_table), n_heads, n_kv, hd, sm_scale, out.data_ptr(), sums,
                            sums + parts * 2 * rows * wide * 4, part.data_ptr(), 0, _status(device))
        _call(device, "sl_kv8_decode", C.byref(p), T, blocks, max_kv_len)
        return out
    _check_step(device, cache, qo_indptr)
    if hd not in PROMPT_HEADS:
        raise ValueError(f"heads of {hd} values: attention of prompts takes 64 or 128")
    _prompts(q, cache, positions, batch_idx, page_table, sm_scale, qo_indptr, max_q or T, max_kv_len, out)
    return out


@lru_cache(maxsize=None)
def _decode_plan(device: int, n_heads: int, n_kv: int, hd: int) -> Tuple[int, ...]:
    """(blocks, partial results, their rows and width) of the decode kernel on a device."""
    out = (C.c_int * 4)()
    at = C.addressof(out)
    with torch.cuda.device(device):
        N.check(N.fn("sl_kv8_decode_plan")(n_heads, n_kv, hd, at, at + 4, at + 8, at + 12), "sl_kv8_decode_plan")
    return tuple(out)


def _prompts(q, cache, positions, batch_idx, page_table, sm_scale, qo_indptr, max_q, max_kv_len, out) -> None:
    """Histories are read back into pages of 64 tokens (keys bf16; values fp16 with a power of two per page and head, where the tcgen05 kernel
    takes them; values that are not finite as zeros, with a note of where they were), over which the prompt kernel attends.  Done once per key
    head and token, that costs less than codes that every block of the kernel (query heads x 128 queries) turns into an operand anew."""
    (T, n_heads, hd), device, dev = q.shape, q.get_device(), q.device
    n_kv, B = cache.k.shape[1], qo_indptr.numel() - 1
    most = page_table.shape[1] * cache.page_size
    per_seq = max(1, -(-min(max_kv_len or most, most) // 64))
    # one piece of memory: keys, values, then what the kernels know of pages and tokens (in words of 4 bytes a page)
    layout = lambda n: (32 * n * hd, 32 * n * hd, n * 128, n, n, n * hd // 4, 1)
    room = max(1, UNPACK_BUDGET_BYTES // (4 * per_seq))          # words a page, if one sequence has them all
    heads, group = n_kv, max(1, min(B, 65535, room // sum(layout(n_kv))))
    if sum(layout(n_kv)) > room:                                 # one history is too long: some key heads at a time
        heads = max(1, (room - 1) // (sum(layout(1)) - 1))
        heads = -(-n_kv // -(-n_kv // heads))
    pages, parts = group * per_seq, layout(heads)
    space = torch.empty(pages * sum(parts) + 2 * T, dtype=torch.int32, device=dev)
    k, v, scales, exps, spoiled, dims, table, rows_out = (space.data_ptr() + 4 * pages * x for x in accumulate((0, *parts)))
    positions_out = rows_out + 4 * T
    k_codes, v_codes, exps_in, *rows = _rows(cache, page_table)
    for h in range(0, n_kv, heads):
        n_h, per = min(heads, n_kv - h), n_heads // n_kv
        mine = slice(h * per, (h + n_h) * per)
        q_h, out_h = (q, out) if n_h == n_kv else (q[:, mine].contiguous(), out.new_empty(T, n_h * per, hd))
        for s in range(0, B, group):
            n, ends = min(group, B - s), qo_indptr.data_ptr() + 4 * s
            up = Kv8UnpackParams(k_codes + h * hd, v_codes + h * hd, exps_in + h * 2 * cache.page_size, *rows, n_h, ends, positions.data_ptr(),
                                 batch_idx.data_ptr(), per_seq, k, v, table, rows_out, positions_out, exps, scales, spoiled, dims)
            p = AttnParams(q_h.data_ptr(), k, v, positions_out, rows_out, table, per_seq, 64, ends, n_h * per, n_h, hd, sm_scale, out_h.data_ptr(), T,
                           pages * 64, max_kv_len, _status(device))
            _call(device, "sl_kv8_prompts", C.byref(up), C.byref(p), n, int(max_q))
        if out_h is not out:
            out[:, mine] = out_h

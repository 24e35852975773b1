"""Linear layers with 8-bit activations in front of FP8 weights: rows in 8 bits (made from rows, from the residual stream and its norm, from a
feed-forward's gate and up rows) and their products.  Qwen3 / Qwen3.5 from FP8 checkpoints run on them with `--act-dtype e4m3`.

A row's values lie in groups of 128 (the last may be shorter): e4m3 codes and one exponent byte b a group, value = code * 2^(b - 127).  The exponent
is the smallest between -60 and 60 with which the group's largest finite magnitude is at most 448 * 2^exponent; larger values saturate, and a
value that is not finite in fp32 is the NaN code.  Rows have a multiple of 16 values; codes lie at [t, k], exponent bytes at [t, k / 128], rows of
either start at multiples of 16 bytes.  Codes are the nearest ones (ties to even) of what 64 bits give.

Weights are those of FP8 checkpoints (:class:`~slopllm_b200.models.weights.LinearWeight`): e4m3 [N, K], one fp32 scale for each block of 128 x 128.

CUDA tensors run `csrc/fp8_rows.cu` and `csrc/fp8_gemm_tcgen05.cu`; CPU tensors run the definition below.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import native as N, quant, tcgen05

GROUP = 128
LOW, HIGH, BIAS = -60, 60, 127         # limits of the exponent, and what is added to it in its byte
MAX_NORM = 16384                       # values of a row that the norm takes on a GPU


class Fp8NormParams(C.Structure):
    _fields_ = [("x", C.c_void_p), ("ldx", C.c_int), ("residual", C.c_void_p), ("ldr", C.c_int), ("w", C.c_void_p), ("H", C.c_int),
                ("eps", C.c_double), ("res_out", C.c_void_p), ("codes", C.c_void_p), ("ldc", C.c_int), ("exps", C.c_void_p), ("lde", C.c_int)]


class Fp8RowsParams(C.Structure):
    _fields_ = [("x", C.c_void_p), ("ldx", C.c_int), ("T", C.c_int), ("K", C.c_int), ("codes", C.c_void_p), ("ldc", C.c_int), ("exps", C.c_void_p),
                ("lde", C.c_int)]


class Fp8ValuesParams(C.Structure):
    _fields_ = [("codes", C.c_void_p), ("ldc", C.c_int), ("exps", C.c_void_p), ("lde", C.c_int), ("T", C.c_int), ("K", C.c_int), ("out", C.c_void_p)]


class Fp8LinearParams(C.Structure):
    _fields_ = [("exps", C.c_void_p), ("lde", C.c_int), ("scale", C.c_void_p), ("lds", C.c_int), ("y", C.c_void_p), ("ldy", C.c_int),
                ("out_f32", C.c_int), ("T", C.c_int), ("N", C.c_int), ("K", C.c_int), ("exps_out", C.c_void_p), ("lde_out", C.c_int), ("err", C.c_void_p)]


def _padded(k: int) -> int:
    """Bytes of a row of exponents for k values: whole pieces of 16."""
    return (k + 16 * GROUP - 1) // (16 * GROUP) * 16


@dataclass
class Fp8Rows:
    """`codes`: uint8 [T, K], e4m3; `exps`: uint8 [T, ceil(K / 128)], rows a multiple of 16 bytes apart (the bytes up to it may be read)."""

    codes: torch.Tensor
    exps: torch.Tensor

    def __post_init__(self):
        codes, exps = self.codes, self.exps
        if codes.dim() != 2 or exps.shape != (codes.shape[0], -(-codes.shape[1] // GROUP)):
            raise ValueError(f"codes {tuple(codes.shape)} do not go with exponents {tuple(exps.shape)}")
        (T, K), (ldc, by), (lde, by_e) = codes.shape, codes.stride(), exps.stride()
        if codes.dtype is not torch.uint8 or exps.dtype is not torch.uint8 or codes.device != exps.device:
            raise ValueError("rows in 8 bits are two tensors of type uint8 on one device")
        if K % 16 or K == 0:
            raise ValueError(f"rows of {K} values: rows in 8 bits have a multiple of 16")
        if T > 1 and (ldc % 16 or lde % 16 or ldc < K or lde < _padded(K)) or by != 1 or (by_e != 1 and exps.shape[1] > 1):
            raise ValueError("rows of codes and of exponents start at multiples of 16 bytes, with bytes side by side")
        if T and codes.is_cuda and ((codes.data_ptr() | exps.data_ptr()) % 16
                                    or exps.storage_offset() + (T - 1) * lde + _padded(K) > exps.untyped_storage().nbytes()):
            raise ValueError("rows of codes and of exponents start at multiples of 16 bytes and are readable in pieces of 16")

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @staticmethod
    def allocate(tokens: int, values: int, device) -> "Fp8Rows":
        if values % 16 or values <= 0:
            raise ValueError(f"rows of {values} values: rows in 8 bits have a multiple of 16")
        rows = object.__new__(Fp8Rows)
        rows.codes = torch.empty(tokens, values, dtype=torch.uint8, device=device)
        rows.exps = torch.empty(tokens, _padded(values), dtype=torch.uint8, device=device)[:, :-(-values // GROUP)]
        return rows


def _call(device: int, name: str, *args) -> None:
    """A kernel call on the current stream of a device."""
    if device == torch._C._cuda_getDevice():
        N.call(name, *args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            N.call(name, *args, N.stream())


@lru_cache(maxsize=None)
def _status(device: int) -> int:
    """Address of a device's status words, which stay where they are."""
    return tcgen05.error_flag(torch.device("cuda", device)).data_ptr()


def _aligned(x: torch.Tensor) -> torch.Tensor:
    """Rows that loads of four values take: a copy where they do not start at multiples of that."""
    size = 4 * x.element_size()
    if x.stride(1) == 1 and x.data_ptr() % size == 0 and (x.stride(0) % 4 == 0 or x.shape[0] <= 1):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _check_rows(x: torch.Tensor, what: str) -> None:
    if x.dim() != 2:
        raise ValueError(f"{what} of shape {tuple(x.shape)}: rows are [tokens, values]")
    if x.is_cuda and x.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{what} of type {x.dtype}: the kernels take bf16 and fp32")


# ---- the format ----------------------------------------------------------------------------------------------------------------------

def _quantize(v: torch.Tensor) -> Fp8Rows:
    """fp64 rows [T, K] -> rows in 8 bits (the definition)."""
    T, K = v.shape
    out = Fp8Rows.allocate(T, K, v.device)
    v = torch.where(v.to(torch.float32).isfinite(), v, torch.full_like(v, float("nan")))
    x = torch.nn.functional.pad(v, (0, -K % GROUP)).view(T, -(-K // GROUP), GROUP)
    m, e = torch.frexp(x.nan_to_num(0.0).abs().amax(-1))
    e = torch.where(m == 0, torch.full_like(e, LOW), (e - 9 + (m > 0.875)).clamp(LOW, HIGH))
    x = torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0)
    _, at = torch.frexp(x.nan_to_num(0.0).abs().clamp(min=2.0 ** -6))
    x = torch.ldexp(torch.round(torch.ldexp(x, 4 - at)), at - 4)            # four significant bits, steps of 2^-9 at least
    out.codes.copy_(x.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8).flatten(1)[:, :K])
    out.exps.copy_(e + BIAS)
    return out


def _values(rows: Fp8Rows) -> torch.Tensor:
    """The fp32 values of rows (the definition)."""
    e = (rows.exps.to(torch.int32) - BIAS).clamp(LOW, HIGH).repeat_interleave(GROUP, 1)[:, :rows.codes.shape[1]]
    return torch.ldexp(rows.codes.view(torch.float8_e4m3fn).to(torch.float32), e)


def fp8_values(rows: Fp8Rows) -> torch.Tensor:
    """The values [T, K] of rows in 8 bits, in bf16, which holds them exactly."""
    (T, K), device = rows.codes.shape, rows.codes.get_device()
    if device < 0:
        return _values(rows).to(torch.bfloat16)
    out = torch.empty(T, K, dtype=torch.bfloat16, device=rows.codes.device)
    p = Fp8ValuesParams(rows.codes.data_ptr(), rows.codes.stride(0), rows.exps.data_ptr(), rows.exps.stride(0), T, K, out.data_ptr())
    _call(device, "sl_fp8_values", C.byref(p))
    return out


# ---- making rows -----------------------------------------------------------------------------------------------------------------------

def _make(x: torch.Tensor, values: int, gated: bool) -> Fp8Rows:
    x = _aligned(x)
    out = Fp8Rows.allocate(x.shape[0], values, x.device)
    p = Fp8RowsParams(x.data_ptr(), x.stride(0), x.shape[0], values, out.codes.data_ptr(), out.codes.stride(0), out.exps.data_ptr(), out.exps.stride(0))
    _call(x.get_device(), "sl_fp8_rows", C.byref(p), int(gated), int(x.dtype is torch.float32))
    return out


def fp8_rows(x: torch.Tensor) -> Fp8Rows:
    """Rows [T, K], bf16 or fp32, of any stride, in 8 bits."""
    _check_rows(x, "rows")
    return _make(x, x.shape[1], False) if x.is_cuda else _quantize(x.to(torch.float64))


def fp8_silu_mul(gate_up: torch.Tensor) -> Fp8Rows:
    """silu(gate) * up of rows gate | up [T, 2 K], bf16 or fp32, of any stride, in 8 bits: nothing is rounded in between."""
    _check_rows(gate_up, "gate and up rows")
    if gate_up.shape[1] % 2:
        raise ValueError(f"gate and up rows of {gate_up.shape[1]} values together")
    if gate_up.is_cuda:
        return _make(gate_up, gate_up.shape[1] // 2, True)
    g, u = gate_up.to(torch.float64).chunk(2, -1)
    return _quantize(g / (1.0 + torch.exp(-g)) * u)


def fp8_add_rmsnorm(x: torch.Tensor, residual: Optional[torch.Tensor], w: torch.Tensor, eps: float) -> Tuple[Fp8Rows, torch.Tensor]:
    """residual' = residual + x (fp32; x alone where there is no residual yet) and the rows residual' / rms(residual') * w in 8 bits.  x [T, H] bf16 or fp32, residual
    fp32, w [H] bf16 or fp32; H at most 16384 on a GPU.  The norm is that of the fp32 residual', in 64 bits.  Returns (rows, residual')."""
    _check_rows(x, "rows")
    (T, H), device = x.shape, x.get_device()
    if w.shape != (H,) or (residual is not None and residual.shape != x.shape):
        raise ValueError(f"rows {tuple(x.shape)} with a norm of {tuple(w.shape)} and a residual of {None if residual is None else tuple(residual.shape)}")
    if w.get_device() != device or (residual is not None and residual.get_device() != device):
        raise ValueError("rows, residual and norm weight are on one device")
    if device < 0:
        r = x.to(torch.float32) if residual is None else residual.to(torch.float32) + x.to(torch.float32)
        v = r.to(torch.float64)
        return _quantize(v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.to(torch.float64)), r
    if H > MAX_NORM:
        raise ValueError(f"rows of {H} values: the norm takes up to {MAX_NORM}")
    if (residual is not None and residual.dtype is not torch.float32) or w.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("the residual is fp32, the norm weight bf16 or fp32")
    x = _aligned(x)
    if residual is not None:
        residual = _aligned(residual)
    if w.stride(0) != 1 or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    out = Fp8Rows.allocate(T, H, x.device)
    res = torch.empty(T, H, dtype=torch.float32, device=x.device)
    p = Fp8NormParams(x.data_ptr(), x.stride(0), N.ptr(residual), 0 if residual is None else residual.stride(0), w.data_ptr(), H, eps, res.data_ptr(),
                      out.codes.data_ptr(), out.codes.stride(0), out.exps.data_ptr(), out.exps.stride(0))
    _call(device, "sl_fp8_add_rmsnorm", C.byref(p), T, int(x.dtype is torch.float32), int(w.dtype is torch.float32))
    return out, res


# ---- products ----------------------------------------------------------------------------------------------------------------------------

def _operands(rows: Fp8Rows, w) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of FP8 weights, checked and (on a GPU) as the kernels take them."""
    codes, scale = w.weight, w.fp8_scale
    if scale is None or codes.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise ValueError("rows in 8 bits are multiplied with FP8 weights (e4m3 and a scale for each block of 128 x 128)")
    (n, k), device = codes.shape, rows.codes.get_device()
    if k != rows.codes.shape[1] or scale.shape[0] < -(-n // GROUP) or scale.shape[1] < -(-k // GROUP):
        raise ValueError(f"rows {tuple(rows.codes.shape)}, weights {tuple(codes.shape)} with scales {tuple(scale.shape)}")
    if codes.get_device() != device or scale.get_device() != device:
        raise ValueError("rows, weights and scales are on one device")
    if device >= 0:
        if codes.stride(1) != 1 or codes.stride(0) % 16 or codes.data_ptr() % 16:
            codes = codes.clone(memory_format=torch.contiguous_format)
        if scale.dtype is not torch.float32 or scale.stride(1) != 1:
            scale = scale.to(torch.float32).contiguous()
    return codes, scale


def _multiply(name: str, rows: Fp8Rows, codes: torch.Tensor, scale: torch.Tensor, y, ldy: int, f32: int, exps_out=None, lde_out: int = 0) -> None:
    (T, K), x, e, device = rows.codes.shape, rows.codes, rows.exps, rows.codes.get_device()
    ldx, lde = (x.stride(0), e.stride(0)) if T > 1 else (K, _padded(K))
    p = Fp8LinearParams(e.data_ptr(), lde, scale.data_ptr(), scale.stride(0), y.data_ptr(), ldy, f32, T, codes.shape[0], K, N.ptr(exps_out), lde_out,
                        _status(device))
    _call(device, name, x.data_ptr(), ldx, codes.data_ptr(), codes.stride(0), C.byref(p))


@lru_cache(maxsize=4096)
def _on_pairs(tokens: int, n: int, k: int) -> bool:
    return bool(N.fn("sl_fp8_on_pairs")(tokens, n, k))


def fp8_linear(rows: Fp8Rows, w, out_f32: bool = False) -> torch.Tensor:
    """y = rows @ W^T [T, N], fp32 sums, in bf16 or fp32.  `w`: a :class:`~slopllm_b200.models.weights.LinearWeight` in FP8.  A NaN code spoils its row's (a
    weight's: its column's) results and no other."""
    codes, scale = _operands(rows, w)
    n, kind = codes.shape[0], torch.float32 if out_f32 else torch.bfloat16
    if rows.codes.get_device() < 0:
        return (_values(rows) @ quant.fp8_block_dequantize(codes, scale).t()).to(kind)
    pad = 4 if out_f32 else 8                        # whole pieces of 16 bytes a row
    ld = -(-n // pad) * pad
    y = torch.empty(rows.codes.shape[0], ld, dtype=kind, device=rows.codes.device)
    _multiply("sl_fp8_linear", rows, codes, scale, y, ld, int(out_f32))
    return y if ld == n else y[:, :n]


def fp8_gate_up(rows: Fp8Rows, w) -> Fp8Rows:
    """silu(rows @ Wg^T) * (rows @ Wu^T) in 8 bits, W = gate rows | up rows [2 I, K]: :func:`fp8_silu_mul` of the product's fp32 sums.  Many rows make the
    activation in the product's epilogue, in fp32 (`inner` a multiple of 128): a value next to the middle between two codes may get the other one."""
    inner = w.weight.shape[0] // 2
    if w.weight.shape[0] % 32:
        raise ValueError(f"{w.weight.shape[0]} gate and up rows: rows in 8 bits have a multiple of 16 values")
    if not rows.codes.is_cuda or inner % GROUP or not _on_pairs(rows.codes.shape[0], 2 * inner, rows.codes.shape[1]):
        return fp8_silu_mul(fp8_linear(rows, w, out_f32=True))
    codes, scale = _operands(rows, w)
    out = Fp8Rows.allocate(rows.codes.shape[0], inner, rows.codes.device)
    _multiply("sl_fp8_gate_up", rows, codes, scale, out.codes, inner, 0, out.exps, out.exps.stride(0))
    return out

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
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import native as N, quant, tcgen05

GROUP = 128
LOW, HIGH, BIAS = -60, 60, 127         # limits of the exponent, and what is added to it in its byte
MAX_NORM = 16384                       # values of a row that the norm takes on a GPU
MAX_COLUMNS = 65535 * 128              # columns of a product on a GPU (a grid's second extent)
MOST = 2 ** 31 - 2 ** 20               # rows, values of a row, values from row to row: the kernels count them, and some steps beyond, in 32 bits


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


class Fp8Rows:
    """`codes`: uint8 [T, K], e4m3; `exps`: uint8 [T, ceil(K / 128)], rows a multiple of 16 bytes apart (the bytes up to it may be read)."""

    __slots__ = ("shape", "_space", "_codes", "_exps")         # (rows that were allocated here are one piece of memory, with views where asked for)

    def __init__(self, codes: torch.Tensor, exps: torch.Tensor):
        if codes.dim() != 2 or exps.shape != (codes.shape[0], -(-codes.shape[1] // GROUP)):
            raise ValueError(f"codes {tuple(codes.shape)} do not go with exponents {tuple(exps.shape)}")
        (T, K), (ldc, by), (lde, by_e) = codes.shape, codes.stride(), exps.stride()
        device = codes.get_device()
        if codes.dtype is not torch.uint8 or exps.dtype is not torch.uint8 or device != exps.get_device():
            raise ValueError("rows in 8 bits are two tensors of type uint8 on one device")
        if K % 16 or K == 0:
            raise ValueError(f"rows of {K} values: rows in 8 bits have a multiple of 16")
        if max(T, K) > MOST or (T > 1 and max(ldc, lde) > MOST):
            raise ValueError(f"{T} rows of {K} values, {ldc} and {lde} bytes apart: up to {MOST} of each")
        if T > 1 and (ldc % 16 or lde % 16 or ldc < K or lde < _padded(K)) or by != 1 or (by_e != 1 and exps.shape[1] > 1):
            raise ValueError("rows of codes and of exponents start at multiples of 16 bytes, with bytes side by side")
        if T and device >= 0 and ((codes.data_ptr() | exps.data_ptr()) % 16
                                  or exps.storage_offset() + (T - 1) * lde + _padded(K) > exps.untyped_storage().nbytes()):
            raise ValueError("rows of codes and of exponents start at multiples of 16 bytes and are readable in pieces of 16")
        self.shape, self._space, self._codes, self._exps = (T, K), None, codes, exps

    @staticmethod
    def allocate(tokens: int, values: int, device) -> "Fp8Rows":
        if values % 16 or values <= 0:
            raise ValueError(f"rows of {values} values: rows in 8 bits have a multiple of 16")
        rows = object.__new__(Fp8Rows)
        rows.shape, rows._codes, rows._exps = (tokens, values), None, None
        rows._space = torch.empty(tokens * (values + _padded(values)), dtype=torch.uint8, device=device)
        return rows

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            T, K = self.shape
            self._codes = self._space[:T * K].view(T, K)
        return self._codes

    @property
    def exps(self) -> torch.Tensor:
        if self._exps is None:
            T, K = self.shape
            self._exps = self._space[T * K:].view(T, _padded(K))[:, :-(-K // GROUP)]
        return self._exps

    @property
    def _memory(self) -> torch.Tensor:
        return self._codes if self._space is None else self._space

    @property
    def device(self) -> torch.device:
        return self._memory.device

    def _where(self) -> tuple:
        """Addresses and row strides of codes and exponents (one row: those of an allocated one)."""
        T, K = self.shape
        if self._space is not None:
            at = self._space.data_ptr()
            return at, K, at + T * K, _padded(K)
        codes, exps = self._codes, self._exps
        return (codes.data_ptr(), codes.stride(0), exps.data_ptr(), exps.stride(0)) if T > 1 else (codes.data_ptr(), K, exps.data_ptr(), _padded(K))


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
    """Rows that loads of four values take: a copy where they do not start at multiples of that, or are too far apart."""
    ld, by = x.stride()
    if by == 1 and (ld % 4 == 0 and ld <= MOST or x.shape[0] <= 1) and x.data_ptr() % (16 if x.dtype is torch.float32 else 8) == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _check_rows(x: torch.Tensor, what: str) -> tuple:
    """(tokens, values, device number) of rows that the operators take."""
    if x.dim() != 2:
        raise ValueError(f"{what} of shape {tuple(x.shape)}: rows are [tokens, values]")
    device, kind = x.get_device(), x.dtype
    if device >= 0 and kind is not torch.bfloat16 and kind is not torch.float32:
        raise ValueError(f"{what} of type {kind}: the kernels take bf16 and fp32")
    T, K = x.shape
    if T > MOST or K > MOST:
        raise ValueError(f"{what} of shape {(T, K)}: up to {MOST} rows and values of a row")
    return T, K, device


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
    e = (rows.exps.to(torch.int32) - BIAS).clamp(LOW, HIGH).repeat_interleave(GROUP, 1)[:, :rows.shape[1]]
    return torch.ldexp(rows.codes.view(torch.float8_e4m3fn).to(torch.float32), e)


def fp8_values(rows: Fp8Rows) -> torch.Tensor:
    """The values [T, K] of rows in 8 bits, in bf16, which holds them exactly."""
    (T, K), memory = rows.shape, rows._memory
    device = memory.get_device()
    if device < 0:
        return _values(rows).to(torch.bfloat16)
    out = memory.new_empty((T, K), dtype=torch.bfloat16)
    p = Fp8ValuesParams(*rows._where(), T, K, out.data_ptr())
    _call(device, "sl_fp8_values", C.byref(p))
    return out


# ---- making rows -----------------------------------------------------------------------------------------------------------------------

def _make(x: torch.Tensor, tokens: int, values: int, device: int, gated: bool) -> Fp8Rows:
    x = _aligned(x)
    out = Fp8Rows.allocate(tokens, values, x.device)
    p = Fp8RowsParams(x.data_ptr(), x.stride(0), tokens, values, *out._where())
    _call(device, "sl_fp8_rows", C.byref(p), gated, x.dtype is torch.float32)
    return out


def fp8_rows(x: torch.Tensor) -> Fp8Rows:
    """Rows [T, K], bf16 or fp32, of any stride, in 8 bits."""
    T, K, device = _check_rows(x, "rows")
    return _make(x, T, K, device, False) if device >= 0 else _quantize(x.to(torch.float64))


def fp8_silu_mul(gate_up: torch.Tensor) -> Fp8Rows:
    """silu(gate) * up of rows gate | up [T, 2 K], bf16 or fp32, of any stride, in 8 bits: nothing is rounded in between."""
    T, K, device = _check_rows(gate_up, "gate and up rows")
    if K % 2:
        raise ValueError(f"gate and up rows of {K} values together")
    if device >= 0:
        return _make(gate_up, T, K // 2, device, True)
    g, u = gate_up.to(torch.float64).chunk(2, -1)
    return _quantize(g / (1.0 + torch.exp(-g)) * u)


def fp8_add_rmsnorm(x: torch.Tensor, residual: Optional[torch.Tensor], w: torch.Tensor, eps: float) -> Tuple[Fp8Rows, torch.Tensor]:
    """residual' = residual + x (fp32; x alone where there is no residual yet) and the rows residual' / rms(residual') * w in 8 bits.  x [T, H] bf16 or
    fp32, residual fp32, w [H] bf16 or fp32; H at most 16384 on a GPU.  The norm is that of the fp32 residual', in 64 bits.  Returns (rows, residual')."""
    T, H, device = _check_rows(x, "rows")
    if w.dim() != 1 or w.shape[0] != H or (residual is not None and residual.shape != x.shape):
        raise ValueError(f"rows {tuple(x.shape)} with a norm of {tuple(w.shape)} and a residual of {None if residual is None else tuple(residual.shape)}")
    if w.get_device() != device or (residual is not None and residual.get_device() != device):
        raise ValueError("rows, residual and norm weight are on one device")
    if device < 0:
        r = x.to(torch.float32) if residual is None else residual.to(torch.float32) + x.to(torch.float32)
        v = r.to(torch.float64)
        return _quantize(v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.to(torch.float64)), r
    if H > MAX_NORM:
        raise ValueError(f"rows of {H} values: the norm takes up to {MAX_NORM}")
    kind, f32 = w.dtype, torch.float32
    if (residual is not None and residual.dtype is not f32) or (kind is not torch.bfloat16 and kind is not f32):
        raise ValueError("the residual is fp32, the norm weight bf16 or fp32")
    x = _aligned(x)
    at, ld = 0, 0
    if residual is not None:
        residual = _aligned(residual)
        at, ld = residual.data_ptr(), residual.stride(0)
    if w.stride(0) != 1 or w.data_ptr() % 16:
        w = w.clone(memory_format=torch.contiguous_format)
    out = Fp8Rows.allocate(T, H, x.device)
    res = x.new_empty((T, H), dtype=f32)
    p = Fp8NormParams(x.data_ptr(), x.stride(0), at, ld, w.data_ptr(), H, eps, res.data_ptr(), *out._where())
    _call(device, "sl_fp8_add_rmsnorm", C.byref(p), T, x.dtype is f32, kind is f32)
    return out, res


# ---- products ----------------------------------------------------------------------------------------------------------------------------

def _codes(codes: torch.Tensor) -> torch.Tensor:
    """Weights that the kernels take: a copy where rows do not start at multiples of 16 bytes, or lie in one another or too far apart."""
    ld, by = codes.stride()
    if by == 1 and ld % 16 == 0 and codes.shape[1] <= ld <= MOST and codes.data_ptr() % 16 == 0:
        return codes
    return codes.clone(memory_format=torch.contiguous_format)


def _scales(scale: torch.Tensor) -> torch.Tensor:
    """Scales that the kernels take: a copy where they are no fp32, not side by side, or rows lie in one another or too far apart."""
    ld, by = scale.stride()
    if scale.dtype is torch.float32 and by == 1 and scale.shape[1] <= ld <= MOST:
        return scale
    return scale.to(torch.float32).clone(memory_format=torch.contiguous_format)


def _operands(rows: Fp8Rows, w) -> Tuple[torch.Tensor, torch.Tensor, int]:
    """Codes and scales of FP8 weights, checked and (on a GPU) as the kernels take them, and the device's number."""
    codes, scale = w.weight, w.fp8_scale
    if scale is None or (codes.dtype is not torch.float8_e4m3fn and codes.dtype is not torch.uint8):
        raise ValueError("rows in 8 bits are multiplied with FP8 weights (e4m3 and a scale for each block of 128 x 128)")
    (n, k), (nb, kb), device = codes.shape, scale.shape, rows._memory.get_device()
    if k != rows.shape[1] or nb * GROUP < n or kb * GROUP < k:
        raise ValueError(f"rows {rows.shape}, weights {(n, k)} with scales {(nb, kb)}")
    if codes.get_device() != device or scale.get_device() != device:
        raise ValueError("rows, weights and scales are on one device")
    most = MOST if device < 0 else MAX_COLUMNS
    if n > most:
        raise ValueError(f"weights of shape {(n, k)}: up to {most} rows")
    if device >= 0:
        codes, scale = _codes(codes), _scales(scale)
    return codes, scale, device


def _multiply(name: str, device: int, rows: Fp8Rows, codes: torch.Tensor, n: int, scale: torch.Tensor, y: int, ldy: int, f32: bool, exps_out: int = 0,
              lde_out: int = 0) -> None:
    T, K = rows.shape
    x, ldx, e, lde = rows._where()
    p = Fp8LinearParams(e, lde, scale.data_ptr(), scale.stride(0), y, ldy, f32, T, n, K, exps_out, lde_out, _status(device))
    _call(device, name, x, ldx, codes.data_ptr(), codes.stride(0), C.byref(p))


@lru_cache(maxsize=4096)
def _on_pairs(tokens: int, n: int, k: int) -> bool:
    return bool(N.fn("sl_fp8_on_pairs")(tokens, n, k))


def fp8_linear(rows: Fp8Rows, w, out_f32: bool = False) -> torch.Tensor:
    """y = rows @ W^T [T, N], fp32 sums, in bf16 or fp32.  `w`: a :class:`~slopllm_b200.models.weights.LinearWeight` in FP8.  A NaN code spoils its row's (a
    weight's: its column's) results and no other.  A block's factor, its scale times 2^exponent, is an fp32 number: results are those of the values as
    long as it is a normal one (scales of 2^68 and more, or below 2^-66, leave that range together with exponents at their limits)."""
    codes, scale, device = _operands(rows, w)
    n, kind = codes.shape[0], torch.float32 if out_f32 else torch.bfloat16
    if device < 0:
        return (_values(rows) @ quant.fp8_block_dequantize(codes, scale).t()).to(kind)
    pad = 4 if out_f32 else 8                        # whole pieces of 16 bytes a row
    ld = -(-n // pad) * pad
    y = codes.new_empty((rows.shape[0], ld), dtype=kind)
    _multiply("sl_fp8_linear", device, rows, codes, n, scale, y.data_ptr(), ld, out_f32)
    return y if ld == n else y[:, :n]


def fp8_gate_up(rows: Fp8Rows, w) -> Fp8Rows:
    """silu(rows @ Wg^T) * (rows @ Wu^T) in 8 bits, W = gate rows | up rows [2 I, K]: :func:`fp8_silu_mul` of the product's fp32 sums.  Many rows make the
    activation in the product's epilogue, in fp32 (I a multiple of 128): a value next to the middle between two codes may get the other one, and a gate
    below -87 gives zeros (its SiLU is below 1e-36)."""
    n = w.weight.shape[0]
    if n % 32:
        raise ValueError(f"{n} gate and up rows: rows in 8 bits have a multiple of 16 values")
    T, K = rows.shape
    if n % (2 * GROUP) or rows._memory.get_device() < 0 or not _on_pairs(T, n, K):
        return fp8_silu_mul(fp8_linear(rows, w, out_f32=True))
    codes, scale, device = _operands(rows, w)
    out = Fp8Rows.allocate(T, n // 2, codes.device)
    to, ld, exps, lde = out._where()
    _multiply("sl_fp8_gate_up", device, rows, codes, n, scale, to, ld, False, exps, lde)
    return out

"""Residual addition and RMSNorm between two projections, with the rows rounded for the next one (HIP kernel
k_add_rmsnorm of libkrq.so): one launch where the reference's step runs add_rmsnorm (engine/kernels/ops.py:42-79) and its
FP8 products then scale and cast their rows.

  d    = bf16(p_0 + p_1 + ..)     delta: the fp32 split-K partials of a projection, summed in order, or bf16 rows
  res  = bf16(x + d)              the new residual rows
  h    = bf16(bf16(res * rstd) * ln),  rstd = 1 / sqrt(mean(res^2) + eps), its sum of squares in fp64
and of h, besides or instead of the bf16 rows:
  add_rmsnorm_fp8   e4m3 rows with per-token scales (the bytes and scales of fp8.quant_rows(h)) or with a given scale (those of
                    linear_fp8's cast), row-major or in the tiled activation layout
  add_rmsnorm_mx    MX blocks (mxfp4.quant_rows(h))
delta=None normalizes x itself (a model's first norm). Rows are of any number, K a multiple of 16 (tiled rows 64, MX
blocks 32) up to 16,384; rows may lie apart in memory. Not to be confused with fused_gemv, which folds the norm into a
GEMV of at most 32 rows: this is for rows that several products and low-rank adapters (kernels.lora) share, for
partials, for prefill, and for MXFP4 weights. rstd there is of an fp32 sum, so a value of h can differ by a rounding.
"""

import torch

from . import _lib as L
from . import fp8 as _fp8
from . import mxfp4 as _mx

MAX_K = 16384
SPLIT_MAX = 64


def _strided(t, ld, unit):
    """Whether rows `ld` apart of consecutive values can be read as they lie: on 16 bytes, `unit` values to 16 bytes."""
    return t.stride(-1) == 1 and ld >= t.shape[-1] and ld % unit == 0 and t.data_ptr() % 16 == 0


def _own_memory(t):
    return t.clone(memory_format=torch.contiguous_format) if t.is_contiguous() else t.contiguous()


def _rows(t, what):
    """(t, row stride) of bf16 rows [M, K] as the kernel reads them (a copy where it cannot)."""
    if t.dtype is not torch.bfloat16 or t.dim() != 2:
        raise ValueError(f"{what} must be bf16 [M, K], got {t.dtype} {tuple(t.shape)}")
    ld = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if not _strided(t, ld, 8):
        t, ld = _own_memory(t), t.shape[1]
    return t, ld


def _partials(t, M, K):
    """(t, row stride, slice stride) of fp32 partials [S, M, K]."""
    if t.dtype is not torch.float32 or t.dim() != 3:
        raise ValueError(f"delta must be bf16 [M, K] or fp32 partials [S, M, K], got {t.dtype} {tuple(t.shape)}")
    S = t.shape[0]
    if not 1 <= S <= SPLIT_MAX:
        raise ValueError(f"delta: {S} partials (1 to {SPLIT_MAX})")
    ld, part = t.stride(1) if M > 1 else K, t.stride(0) if S > 1 else M * K
    if not _strided(t, ld, 4) or part % 4 or part < 0:
        t, ld, part = _own_memory(t), K, M * K
    return t, ld, part


def _extent(t):
    """First byte and the one past the last of what t spans."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _apart(out, t, same):
    """Refuses an output that overlaps an input, unless each element lies on its own."""
    if t is None or (same and out.data_ptr() == t.data_ptr()):
        return
    a0, a1 = _extent(out)
    b0, b1 = _extent(t)
    if a0 < b1 and b0 < a1:
        raise ValueError("res_out overlaps an input (it may be x itself)")


def _launch(x, delta, ln, eps, res_out, kind, inv, h, out, scale):
    """Checks the operands, makes res, launches; returns res. h, out, scale: functions of the checked x that make them."""
    L.require_device(x, delta, ln, inv, res_out)
    for t in (delta, ln, inv, res_out):
        if t is not None and t.get_device() != x.get_device():
            raise ValueError(f"tensors on {x.device} and {t.device}")
    res = x
    x, ldx = _rows(x, "x")
    M, K = x.shape
    if K % 16 or not 16 <= K <= MAX_K:
        raise ValueError(f"K={K} must be a multiple of 16 up to {MAX_K}")
    if ln.dtype is not torch.bfloat16 or tuple(ln.shape) != (K,):
        raise ValueError(f"ln must be bf16 [{K}], got {ln.dtype} {tuple(ln.shape)}")
    ln = ln if ln.is_contiguous() and ln.data_ptr() % 16 == 0 else _own_memory(ln)
    split = ldd = part = 0
    if delta is not None:
        if tuple(delta.shape[-2:]) != (M, K):
            raise ValueError(f"x {tuple(x.shape)} and delta {tuple(delta.shape)} do not match")
        if delta.dim() == 2:
            delta, ldd = _rows(delta, "delta")
        else:
            delta, ldd, part = _partials(delta, M, K)
            split = delta.shape[0]
        if res_out is None:
            res = torch.empty((M, K), device=x.device, dtype=torch.bfloat16)
        else:
            res = res_out
            if res.dtype is not torch.bfloat16 or tuple(res.shape) != (M, K) or not res.is_contiguous() or res.data_ptr() % 16:
                raise ValueError(f"res_out must be contiguous bf16 [{M}, {K}] on 16 bytes, got {res.dtype} {tuple(res.shape)}")
            _apart(res, x, ldx == K)
            _apart(res, delta, split == 0 and ldd == K)
            _apart(res, ln, False)
    elif res_out is not None:
        raise ValueError("res_out without delta: there is no new residual")
    if M:
        _mx._call(x.get_device(), "krq_add_rmsnorm", L.ptr(x), ldx, L.ptr(delta), split, ldd, part, L.ptr(ln), float(eps), M, K, kind,
                  L.ptr(inv), L.ptr(res) if delta is not None else None, h, out, scale)
    return res


def _shape(x):
    if x.dim() != 2:
        raise ValueError(f"x must be bf16 [M, K], got {x.dtype} {tuple(x.shape)}")
    return x.shape


def add_rmsnorm(x, delta, ln, eps=1e-6, res_out=None):
    """x [M, K] bf16, delta None, bf16 [M, K] or fp32 partials [S, M, K], ln [K] bf16 -> (res, h), both bf16 [M, K].
    res_out: where res goes (contiguous; may be x, whose rows are then replaced); res is x itself where delta is None."""
    M, K = _shape(x)
    h = torch.empty((M, K), device=x.device, dtype=torch.bfloat16)
    return _launch(x, delta, ln, eps, res_out, L.NORM_ROWS, None, L.ptr(h), None, None), h


def add_rmsnorm_fp8(x, delta, ln, eps=1e-6, a=None, tiled=False, with_h=False, res_out=None):
    """add_rmsnorm with h in e4m3: (res, x8, xs), or (res, x8, xs, h) with_h.
    a None: per-token scales, x8 and xs fp32 [M, 1] equal to fp8.quant_rows(h)'s; an ActScale / SharedScale: its scale, x8
    equal to linear_fp8's cast of h, xs = a.scale. x8 is float8_e4m3fn [M, K] for gemv_fp8(x8, q, split, xs=xs),
    gemm_fp8(x8, q, xs=xs) and their kin; tiled=True (K % 64 == 0): uint8 in the tiled activation layout, padded to
    16 * ceil(M / 16) rows, for gemv_fp8_tiled_launch(x8, xs, q, M, ..) at up to 32 rows."""
    M, K = _shape(x)
    if tiled and K % 64:
        raise ValueError(f"tiled rows need K={K} a multiple of 64")
    if tiled:
        x8 = torch.empty(((M + 15) // 16 * 16 * K,), device=x.device, dtype=torch.uint8)
    else:
        x8 = torch.empty((M, K), device=x.device, dtype=torch.float8_e4m3fn)
    if a is None:
        inv, xs = None, torch.empty((M, 1), device=x.device, dtype=torch.float32)
        kind = L.NORM_FP8_TOKEN_TILED if tiled else L.NORM_FP8_TOKEN
    else:
        inv, xs = _fp8._one(a.inv), _fp8._one(a.scale)
        if inv.numel() != 1 or xs.numel() != 1:
            raise ValueError("a must have one inverse and one scale")
        kind = L.NORM_FP8_GIVEN_TILED if tiled else L.NORM_FP8_GIVEN
    h = torch.empty((M, K), device=x.device, dtype=torch.bfloat16) if with_h else None
    res = _launch(x, delta, ln, eps, res_out, kind, inv, L.ptr(h), L.ptr(x8), None if a is not None else L.ptr(xs))
    return (res, x8, xs, h) if with_h else (res, x8, xs)


def add_rmsnorm_mx(x, delta, ln, eps=1e-6, elem="e4m3", with_h=False, res_out=None):
    """add_rmsnorm with h in MX blocks of elem: (res, rows), or (res, rows, h) with_h; rows is the MXRows of
    mxfp4.quant_rows(h, elem), for every product on an MXFP4Weight. K % 32 == 0."""
    M, K = _shape(x)
    if K % _mx.BLOCK:
        raise ValueError(f"MX blocks need K={K} a multiple of {_mx.BLOCK}")
    e = _mx._elem(elem)
    at, nbytes = _mx._rows_bytes(M, K, e)
    data = torch.empty((nbytes,), device=x.device, dtype=torch.uint8)
    h = torch.empty((M, K), device=x.device, dtype=torch.bfloat16) if with_h else None
    p = data.data_ptr()
    res = _launch(x, delta, ln, eps, res_out, L.NORM_MX_E4M3 if e == L.MX_E4M3 else L.NORM_MX_E2M1, None, L.ptr(h), p, p + at)
    rows = _mx.MXRows(data, at, (M, K), elem)
    return (res, rows, h) if with_h else (res, rows)

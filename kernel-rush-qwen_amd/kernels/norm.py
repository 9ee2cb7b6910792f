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


def _misplaced(x, *tensors):
    L.require_device(x, *tensors)
    raise ValueError("tensors on " + ", ".join(sorted({str(t.device) for t in (x, *tensors) if t is not None})))


def _operands(x, delta, ln, res_out):
    """(x, its row stride, delta, partials or 0, its row and slice strides, ln, res, M, K, device) as the kernel takes them. A
    call of a few rows is host work as much as a launch: operands that lie as they should are looked at once, by attribute."""
    dev = x.get_device()
    if dev < 0 or ln.get_device() != dev or (delta is not None and delta.get_device() != dev) or (
            res_out is not None and res_out.get_device() != dev):
        _misplaced(x, delta, ln, res_out)
    shape = x.shape
    if x.dtype is not torch.bfloat16 or len(shape) != 2:
        raise ValueError(f"x must be bf16 [M, K], got {x.dtype} {tuple(shape)}")
    M, K = shape
    if K & 15 or not 16 <= K <= MAX_K:
        raise ValueError(f"K={K} must be a multiple of 16 up to {MAX_K}")
    if ln.dtype is not torch.bfloat16 or ln.dim() != 1 or ln.shape[0] != K:
        raise ValueError(f"ln must be bf16 [{K}], got {ln.dtype} {tuple(ln.shape)}")
    res, ldx, split, ldd, part = x, K, 0, 0, 0
    if not x.is_contiguous() or x.data_ptr() & 15:
        x, ldx = _rows(x, "x")
    if not ln.is_contiguous() or ln.data_ptr() & 15:
        ln = _own_memory(ln)
    if delta is not None:
        dshape = delta.shape
        if dshape[-2:] != shape or not 2 <= len(dshape) <= 3:
            raise ValueError(f"x {tuple(shape)} and delta {tuple(dshape)} do not match")
        plain = delta.is_contiguous() and not delta.data_ptr() & 15
        if len(dshape) == 2:
            if plain and delta.dtype is torch.bfloat16:
                ldd = K
            else:
                delta, ldd = _rows(delta, "delta")
        else:
            split = dshape[0]
            if plain and delta.dtype is torch.float32 and 1 <= split <= SPLIT_MAX:
                ldd, part = K, M * K
            else:
                delta, ldd, part = _partials(delta, M, K)
        if res_out is None:
            res = torch.empty_like(x) if ldx == K else x.new_empty(shape)
        else:
            res = res_out
            if res.dtype is not torch.bfloat16 or res.shape != shape or not res.is_contiguous() or res.data_ptr() & 15:
                raise ValueError(f"res_out must be contiguous bf16 [{M}, {K}] on 16 bytes, got {res.dtype} {tuple(res.shape)}")
            _apart(res, x, ldx == K)
            _apart(res, delta, split == 0 and ldd == K)
            _apart(res, ln, False)
    elif res_out is not None:
        raise ValueError("res_out without delta: there is no new residual")
    return x, ldx, delta, split, ldd, part, ln, res, M, K, dev


def _launch(operands, eps, kind, inv, h, out, scale):
    x, ldx, delta, split, ldd, part, ln, res, M, K, dev = operands
    if M == 0:
        return
    if delta is None:
        _mx._call(dev, "krq_add_rmsnorm", x.data_ptr(), ldx, None, 0, 0, 0, ln.data_ptr(), eps, M, K, kind, inv, None, h, out, scale)
    else:
        _mx._call(dev, "krq_add_rmsnorm", x.data_ptr(), ldx, delta.data_ptr(), split, ldd, part, ln.data_ptr(), eps, M, K, kind, inv,
                  res.data_ptr(), h, out, scale)


def add_rmsnorm(x, delta, ln, eps=1e-6, res_out=None):
    """x [M, K] bf16, delta None, bf16 [M, K] or fp32 partials [S, M, K], ln [K] bf16 -> (res, h), both bf16 [M, K].
    res_out: where res goes (contiguous; may be x, whose rows are then replaced); res is x itself where delta is None."""
    ops = _operands(x, delta, ln, res_out)
    h = torch.empty_like(ops[0]) if ops[1] == ops[9] else ops[0].new_empty(ops[8:10])
    _launch(ops, eps, L.NORM_ROWS, None, h.data_ptr(), None, None)
    return ops[7], h


def add_rmsnorm_fp8(x, delta, ln, eps=1e-6, a=None, tiled=False, with_h=False, res_out=None):
    """add_rmsnorm with h in e4m3: (res, x8, xs), or (res, x8, xs, h) with_h.
    a None: per-token scales, x8 and xs fp32 [M, 1] equal to fp8.quant_rows(h)'s; an ActScale / SharedScale: its scale, x8
    equal to linear_fp8's cast of h, xs = a.scale. x8 is float8_e4m3fn [M, K] for gemv_fp8(x8, q, split, xs=xs),
    gemm_fp8(x8, q, xs=xs) and their kin; tiled=True (K % 64 == 0): uint8 in the tiled activation layout, padded to
    16 * ceil(M / 16) rows, for gemv_fp8_tiled_launch(x8, xs, q, M, ..) at up to 32 rows."""
    ops = _operands(x, delta, ln, res_out)
    x, M, K = ops[0], ops[8], ops[9]
    if not tiled:
        x8 = torch.empty_like(x, dtype=torch.float8_e4m3fn) if ops[1] == K else x.new_empty(M, K, dtype=torch.float8_e4m3fn)
    elif K % 64:
        raise ValueError(f"tiled rows need K={K} a multiple of 64")
    else:
        x8 = x.new_empty((M + 15) // 16 * 16 * K, dtype=torch.uint8)
    if a is None:
        inv = None
        xs = x.new_empty(M, 1, dtype=torch.float32)
        kind, ps = L.NORM_FP8_TOKEN_TILED if tiled else L.NORM_FP8_TOKEN, xs.data_ptr()
    else:
        one, xs = _fp8._one(a.inv), _fp8._one(a.scale)
        if one.get_device() != ops[10] or xs.get_device() != ops[10]:
            _misplaced(x, one, xs)
        kind, inv, ps = L.NORM_FP8_GIVEN_TILED if tiled else L.NORM_FP8_GIVEN, one.data_ptr(), None
    h = x.new_empty(M, K) if with_h else None
    _launch(ops, eps, kind, inv, h.data_ptr() if with_h else None, x8.data_ptr(), ps)
    return (ops[7], x8, xs, h) if with_h else (ops[7], x8, xs)


def add_rmsnorm_mx(x, delta, ln, eps=1e-6, elem="e4m3", with_h=False, res_out=None):
    """add_rmsnorm with h in MX blocks of elem: (res, rows), or (res, rows, h) with_h; rows is the MXRows of
    mxfp4.quant_rows(h, elem), for every product on an MXFP4Weight. K % 32 == 0."""
    ops = _operands(x, delta, ln, res_out)
    x, M, K = ops[0], ops[8], ops[9]
    if K % _mx.BLOCK:
        raise ValueError(f"MX blocks need K={K} a multiple of {_mx.BLOCK}")
    e = _mx._elem(elem)
    at, nbytes = _mx._rows_bytes(M, K, e)
    data = x.new_empty(nbytes, dtype=torch.uint8)
    h = x.new_empty(M, K) if with_h else None
    p = data.data_ptr()
    _launch(ops, eps, L.NORM_MX_E4M3 if e == L.MX_E4M3 else L.NORM_MX_E2M1, None, h.data_ptr() if with_h else None, p, p + at)
    rows = _mx.MXRows(data, at, (M, K), elem)
    return (ops[7], rows, h) if with_h else (ops[7], rows)

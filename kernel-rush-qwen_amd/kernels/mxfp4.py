"""Microscaled 4-bit weights (MXFP4, OCP MX v1.0) on MI355X: quantizers, the decode and prefill products
on the matrix cores' scaled instructions, and the embedding lookup of a packed table. The 4-bit
counterpart of kernels.fp8 (the reference has none): 4.25 bits a weight, no calibration.

A row is cut into blocks of 32 values along K with one E8M0 scale each, a power of two:
  scale   c = max(0, floor(log2(max|v|)) + 127 - emax), standing for 2^(c - 127); emax 2 (e2m1), 8 (e4m3)
  element v / 2^(c - 127) rounded to the nearest of the format, ties to even, clamped to 6 (e2m1) or 448 (e4m3)
A block with a NaN or an infinity has scale 255, NaN: every value of it, and every product that reads it, is
NaN. Weights are e2m1; activation rows are rounded per call to e4m3 blocks (the default) or to e2m1 blocks
(elem="e2m1": half the bytes and twice the matrix rate in prefill, 4-bit accuracy):
  linear_mxfp4 et al.  y = bf16(sum_k x[m, k] w[n, k]) over the rounded values, accumulated in fp32
The kernels read operands in the tiled layout of include/krq.h ("mx tiled"). K is a multiple of 32; N and M
are any.
"""

import torch

from . import _lib as L

ELEMS = {"e2m1": L.MX_E2M1, "e4m3": L.MX_E4M3}
DECODE_MAX_ROWS = 32  # rows of the skinny kernels
BLOCK = 32


class MXFP4Weight(tuple):
    """(w4 uint8 [N, K/2], scale uint8 [N, K/32]) row-major, as checkpoints hold them (element 2i in the low
    half of byte i), with the tiled copies the products read (`tiled`, `tiled_scale`). quantize() and
    pack() make them; a w4 or scale changed in place afterwards needs pack() again."""

    def __new__(cls, w4, scale, tiled, tiled_scale):
        self = super().__new__(cls, (w4, scale))
        self.tiled, self.tiled_scale = tiled, tiled_scale
        self.shape = (w4.shape[0], 2 * w4.shape[1])
        return self


class MXRows:
    """Activation rows [M, K] in MX blocks of `elem`, tiled (quant_rows)."""

    def __init__(self, tiled, tiled_scale, shape, elem):
        self.tiled, self.tiled_scale, self.shape, self.elem = tiled, tiled_scale, shape, elem


def _elem(elem):
    if elem not in ELEMS:
        raise ValueError(f"elem must be one of {sorted(ELEMS)}, got {elem!r}")
    return ELEMS[elem]


def _on(t):
    """t's device is made current for the launch where it is not (its stream belongs to it)."""
    return torch.cuda.device(t.device)


def _call(t, name, *args):
    L_args = args + (L.stream(t),)
    if t.get_device() == torch.cuda.current_device():
        L.call(name, *L_args)
    else:
        with _on(t):
            L.call(name, *L_args)


def _same_device(first, *tensors):
    L.require_device(first, *tensors)
    for t in tensors:
        if t.get_device() != first.get_device():
            raise ValueError(f"tensors on {first.device} and {t.device}")


def _bf16_rows(x, what):
    """x [M, K] bf16 as the kernels read it: contiguous rows that start on 16 bytes."""
    L.require_device(x)
    if x.dim() != 2 or x.dtype != torch.bfloat16:
        raise ValueError(f"expected bf16 {what}, got {x.dtype} {tuple(x.shape)}")
    M, K = x.shape
    if K == 0 or K % BLOCK:
        raise ValueError(f"{what}: K={K} must be a positive multiple of {BLOCK}")
    if x.stride(1) != 1 or (M > 1 and (x.stride(0) < K or x.stride(0) % 8)):
        x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _ld(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _tiles(M, K, elem, device):
    lib = L.lib()
    return (torch.empty((lib.krq_mx_tiled_bytes(M, K, elem),), device=device, dtype=torch.uint8),
            torch.empty((lib.krq_mx_scale_bytes(M, K),), device=device, dtype=torch.uint8))


@torch.no_grad()
def quantize(w):
    """w [N, K] bf16 -> MXFP4Weight, w ~= e2m1 values times their blocks' scales. K % 32 == 0."""
    w = _bf16_rows(w, "weight [N, K]")
    N, K = w.shape
    if N == 0:
        raise ValueError("weight [N, K]: N must be positive")
    w4 = torch.empty((N, K // 2), device=w.device, dtype=torch.uint8)
    scale = torch.empty((N, K // BLOCK), device=w.device, dtype=torch.uint8)
    tiled, tscale = _tiles(N, K, L.MX_E2M1, w.device)
    _call(w, "krq_quant_mxfp4", L.ptr(w), N, K, _ld(w), L.ptr(w4), L.ptr(scale), L.ptr(tiled), L.ptr(tscale))
    return MXFP4Weight(w4, scale, tiled, tscale)


@torch.no_grad()
def pack(w4, scale):
    """The MXFP4Weight of codes and scales quantized elsewhere: w4 uint8 [N, K/2] (element 2i in the low half
    of byte i), scale uint8 [N, K/32] (E8M0)."""
    _same_device(w4, scale)
    if w4.dtype != torch.uint8 or w4.dim() != 2 or scale.dtype != torch.uint8 or scale.dim() != 2:
        raise ValueError("pack expects uint8 w4 [N, K/2] and scale [N, K/32]")
    N, K = w4.shape[0], 2 * w4.shape[1]
    if N == 0 or K == 0 or K % BLOCK or tuple(scale.shape) != (N, K // BLOCK):
        raise ValueError(f"pack: w4 {tuple(w4.shape)} and scale {tuple(scale.shape)} do not match")
    w4, scale = w4.contiguous(), scale.contiguous()
    if w4.data_ptr() % 16:
        w4 = w4.clone()
    tiled, tscale = _tiles(N, K, L.MX_E2M1, w4.device)
    _call(w4, "krq_pack_mxfp4", L.ptr(w4), L.ptr(scale), N, K, L.ptr(tiled), L.ptr(tscale))
    return MXFP4Weight(w4, scale, tiled, tscale)


def _weight(q):
    if not isinstance(q, MXFP4Weight):
        raise ValueError("expected an MXFP4Weight (mxfp4.quantize or mxfp4.pack)")
    return q.shape


def dequantize(q):
    """The bf16 values an MXFP4Weight or MXRows stands for, [N, K] or [M, K] (its tiled copy's)."""
    if isinstance(q, MXRows):
        (M, K), elem = q.shape, ELEMS[q.elem]
    else:
        (M, K), elem = _weight(q), L.MX_E2M1
    out = torch.empty((M, K), device=q.tiled.device, dtype=torch.bfloat16)
    if M:
        _call(out, "krq_dequant_mx", L.ptr(q.tiled), L.ptr(q.tiled_scale), elem, M, K, L.ptr(out))
    return out


def quant_rows(x, elem="e4m3"):
    """x [M, K] bf16 -> MXRows: the rows rounded to MX blocks, in the layout the products read. Several
    products on the same rows can share them."""
    x = _bf16_rows(x, "rows [M, K]")
    M, K = x.shape
    e = _elem(elem)
    if M == 0:
        none = torch.empty((0,), device=x.device, dtype=torch.uint8)
        return MXRows(none, none, (0, K), elem)
    tiled, tscale = _tiles(M, K, e, x.device)
    _call(x, "krq_quant_mx_rows", L.ptr(x), M, K, _ld(x), e, L.ptr(tiled), L.ptr(tscale))
    return MXRows(tiled, tscale, (M, K), elem)


def _decode(x, q, split, mode, elem):
    N, K = _weight(q)
    if isinstance(x, MXRows):
        rows = x
    else:
        x = _bf16_rows(x, "rows [M, K]")
        rows = None
    M, kx = x.shape
    if kx != K:
        raise ValueError(f"x [{M}, {kx}] and w [{N}, {K}] do not match")
    if M > DECODE_MAX_ROWS:
        raise ValueError(f"M={M} > {DECODE_MAX_ROWS} rows: use gemm_mxfp4 or linear_mxfp4")
    if mode == L.OUT_SWIGLU and N % 32:
        raise ValueError(f"SwiGLU needs w = [gate; up] of 2 I rows with I a multiple of 16, got N={N}")
    e = _elem(elem)
    dev = q.tiled.device
    if mode == L.OUT_PARTIAL:
        out = torch.empty((split, M, N), device=dev, dtype=torch.float32)
    else:
        out = torch.empty((M, N // 2 if mode == L.OUT_SWIGLU else N), device=dev, dtype=torch.bfloat16)
    if M == 0:
        return out
    if rows is None and M > L.MX_BF16_ROWS:
        rows = quant_rows(x, elem)
    if rows is None:
        _same_device(x, q.tiled)
        _call(x, "krq_gemv_mxfp4", L.ptr(x), None, L.MX_X_BF16, e, _ld(x), L.ptr(q.tiled), L.ptr(q.tiled_scale), M, N, K,
              split, mode, L.ptr(out))
    else:
        _same_device(rows.tiled, q.tiled)
        _call(out, "krq_gemv_mxfp4", L.ptr(rows.tiled), L.ptr(rows.tiled_scale), L.MX_X_TILED, ELEMS[rows.elem], 0,
              L.ptr(q.tiled), L.ptr(q.tiled_scale), M, N, K, split, mode, L.ptr(out))
    return out


def gemv_mxfp4(x, q, split=1, elem="e4m3"):
    """MXFP4 counterpart of fp8.gemv_fp8: x [M, K] bf16 (M <= 32; rounded to blocks of elem) or MXRows, q an
    MXFP4Weight [N, K]. split == 1: bf16 [M, N]. split > 1: fp32 partials [split, M, N] whose in-order sum is
    the product; split s covers the groups of 512 k [s G / split, (s + 1) G / split), G = ceil(K / 512), so
    split <= G."""
    return _decode(x, q, split, L.OUT_BF16 if split == 1 else L.OUT_PARTIAL, elem)


def gemv_swiglu_mxfp4(x, q, elem="e4m3"):
    """MXFP4 counterpart of fp8.gemv_swiglu_fp8: q packs w_gu [2I, K] = [gate; up], I % 16 == 0. Returns
    bf16(silu(g) * u) [M, I] from the fp32 g and u (one rounding, where the FP8 form rounds g, silu(g) and
    u first as the reference's does)."""
    return _decode(x, q, 1, L.OUT_SWIGLU, elem)


def gemm_mxfp4(x, q, elem="e4m3"):
    """MXFP4 prefill product: x [M, K] bf16 (rounded to blocks of elem by quant_rows) or MXRows, any M;
    q an MXFP4Weight [N, K]. Returns bf16 [M, N]."""
    N, K = _weight(q)
    if x.shape[1] != K:
        raise ValueError(f"x {tuple(x.shape)} and w [{N}, {K}] do not match")
    rows = x if isinstance(x, MXRows) else quant_rows(x, elem)
    M = rows.shape[0]
    _same_device(rows.tiled, q.tiled)
    out = torch.empty((M, N), device=q.tiled.device, dtype=torch.bfloat16)
    if M:
        _call(out, "krq_gemm_mxfp4", L.ptr(rows.tiled), L.ptr(rows.tiled_scale), ELEMS[rows.elem], L.ptr(q.tiled),
              L.ptr(q.tiled_scale), M, N, K, L.ptr(out))
    return out


def linear_mxfp4(x, q, elem="e4m3"):
    """bf16 [M, N] ~= x @ W^T on q = quantize(W): gemv_mxfp4 up to 32 rows, gemm_mxfp4 from 33."""
    return gemv_mxfp4(x, q, 1, elem) if x.shape[0] <= DECODE_MAX_ROWS else gemm_mxfp4(x, q, elem)


def embedding(ids, q, scale=1.0):
    """Rows of the packed table q [N, K] by index, times scale (a model's embedding multiplier): bf16
    [*ids.shape, K] = bf16(w[id] * scale) from the row-major codes, so a model with tied embeddings keeps one
    packed table for this and the lm head. ids int64 or int32; an index outside [0, N) gives a row of NaN."""
    N, K = _weight(q)
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32, got {ids.dtype}")
    _same_device(ids, q[0])
    ids = ids.contiguous()
    out = torch.empty((*ids.shape, K), device=ids.device, dtype=torch.bfloat16)
    if ids.numel():
        _call(ids, "krq_embed_mxfp4", L.ptr(ids), int(ids.dtype == torch.int64), ids.numel(), L.ptr(q[0]), L.ptr(q[1]), N, K,
              float(scale), L.ptr(out))
    return out

"""Microscaled 4-bit weights (MXFP4, OCP MX v1.0) on MI355X: quantizers, the decode and prefill products
on the matrix cores' scaled instructions, and the embedding lookup of a quantized table. The 4-bit
counterpart of kernels.fp8 (the reference has none): a product reads 4.25 bits a weight; no calibration. A weight
keeps its codes and scales twice, row-major and tiled, 8.5 bits in memory.

A row is cut into blocks of 32 values along K with one E8M0 scale each, a power of two:
  scale   c = max(0, floor(log2(max|v|)) + 127 - emax), standing for 2^(c - 127); emax 2 (e2m1), 8 (e4m3)
  element v / 2^(c - 127) rounded to the nearest of the format, ties to even, clamped to 6 (e2m1) or 448 (e4m3)
A block with a NaN or an infinity has scale 255, NaN: every value of it, and every product that reads it, is
NaN. Weights are e2m1; activation rows are rounded per call to e4m3 blocks (the default) or to e2m1 blocks
(elem="e2m1": half the bytes and twice the matrix rate in prefill, 4-bit accuracy):
  linear_mxfp4 et al.  y = bf16(sum_k x[m, k] w[n, k]) over the rounded values, accumulated in fp32
The products read operands in the tiled layout of include/krq.h ("mx tiled"), the embedding the row-major one. K is a
multiple of 32, N any. M is any in gemm_mxfp4 and linear_mxfp4; the decode products gemv_mxfp4 and gemv_swiglu_mxfp4 take at
most 32 rows (the FP8 ones go on in chunks), whose split-K shares out groups of 512 k.
"""

import torch

from . import _lib as L

ELEMS = {"e2m1": L.MX_E2M1, "e4m3": L.MX_E4M3}
DECODE_MAX_ROWS = 32  # rows of the skinny kernels
BLOCK = 32
ROW_MAX_K = 10240  # up to here the skinny kernels round a single bf16 row themselves, without a workspace,
ROWS_MAX_K = 5120  # and up to here L.MX_BF16_ROWS of them
GROUP, SPLIT_MAX = 512, 64  # k of a group, the unit that split-K shares out; the most parts


class MXFP4Weight(tuple):
    """(w4 uint8 [N, K/2], scale uint8 [N, K/32]) row-major, as checkpoints hold them (element 2i in the low
    half of byte i), with the tiled copies the products read (`tiled`, `tiled_scale`). quantize() and
    pack() make them; a w4 or scale changed in place afterwards needs pack() again."""

    def __new__(cls, w4, scale, tiled, tiled_scale):
        self = super().__new__(cls, (w4, scale))
        self.shape = (w4.shape[0], 2 * w4.shape[1])
        N, K = self.shape
        if N < 1 or K < BLOCK or K % BLOCK or tuple(scale.shape) != (N, K // BLOCK):
            raise ValueError(f"MXFP4Weight: w4 {tuple(w4.shape)} and scale {tuple(scale.shape)} do not match")
        cls._check("w4", w4, N * K // 2)
        cls._check("scale", scale, N * K // BLOCK)
        self.tiled, self.tiled_scale = tiled, tiled_scale
        return self

    @staticmethod
    def _check(name, t, size):
        if t.dtype != torch.uint8 or t.numel() != size or not t.is_contiguous():
            raise ValueError(f"MXFP4Weight: {name} must be {size} contiguous bytes, got {t.dtype} {tuple(t.shape)}")

    def __setattr__(self, name, value):  # (the kernels read as many bytes as the shape needs)
        if name == "tiled":
            self._check(name, value, L.lib().krq_mx_tiled_bytes(*self.shape, L.MX_E2M1))
        elif name == "tiled_scale":
            self._check(name, value, L.lib().krq_mx_scale_bytes(*self.shape))
        super().__setattr__(name, value)

    def __getnewargs__(self):  # (copies and pickles make a new one of these)
        return self[0], self[1], self.tiled, self.tiled_scale


class MXRows:
    """Activation rows [M, K] in MX blocks of `elem`, tiled (quant_rows): `data` uint8, the elements, then
    from byte scale_at the scales."""

    __slots__ = ("data", "scale_at", "shape", "elem")

    def __init__(self, data, scale_at, shape, elem):
        self.data, self.scale_at, self.shape, self.elem = data, scale_at, shape, elem

    @property
    def tiled(self):
        return self.data[:L.lib().krq_mx_tiled_bytes(*self.shape, ELEMS[self.elem])]

    @property
    def tiled_scale(self):
        return self.data[self.scale_at:]


def _elem(elem):
    if elem not in ELEMS:
        raise ValueError(f"elem must be one of {sorted(ELEMS)}, got {elem!r}")
    return ELEMS[elem]


_cuda = torch._C


def _call(dev, name, *args):
    """L.call on device dev (made current for it where it is not) and torch's current stream of it. A call on a
    few rows is host work as much as a launch (a product of one row 8.1 us, 3.4 of them the kernel's; 6.1 with
    the library's function taken once and no Stream or device objects made)."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(L.lib(), name)
    if dev == _cuda._cuda_getDevice():
        rc = fn(*args, _cuda._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _cuda._cuda_getCurrentRawStream(dev))
    if rc != L.KRQ_OK:
        L.fail(name, rc)


_functions = {}


def _same_device(first, *tensors):
    """Refuses tensors of the host, whose addresses a kernel would read as its own, and of two devices."""
    L.require_device(first, *tensors)
    for t in tensors:
        if t.get_device() != first.get_device():
            raise ValueError(f"tensors on {first.device} and {t.device}")


def _bf16_rows(x, what):
    """(x, row stride): x [M, K] bf16 as the kernels read it, rows of consecutive values that start on 16 bytes."""
    if not x.is_cuda:
        L.require_device(x)
    shape = x.shape
    if x.dtype is not torch.bfloat16 or len(shape) != 2:
        raise ValueError(f"expected bf16 {what}, got {x.dtype} {tuple(shape)}")
    K = ld = shape[1]
    if K == 0 or K % BLOCK:
        raise ValueError(f"{what}: K={K} must be a positive multiple of {BLOCK}")
    if not x.is_contiguous():
        ld, unit = x.stride()
        if shape[0] == 1 and unit == 1:
            ld = K
        elif unit != 1 or ld < K or ld % 8:
            x, ld = x.contiguous(), K
    if x.data_ptr() % 16:
        x, ld = x.clone(memory_format=torch.contiguous_format), K
    return x, ld


def _tiles(M, K, elem, device):
    lib = L.lib()
    return (torch.empty((lib.krq_mx_tiled_bytes(M, K, elem),), device=device, dtype=torch.uint8),
            torch.empty((lib.krq_mx_scale_bytes(M, K),), device=device, dtype=torch.uint8))


@torch.no_grad()
def quantize(w):
    """w [N, K] bf16 -> MXFP4Weight, w ~= e2m1 values times their blocks' scales. K % 32 == 0."""
    w, ld = _bf16_rows(w, "weight [N, K]")
    N, K = w.shape
    if N == 0:
        raise ValueError("weight [N, K]: N must be positive")
    w4 = torch.empty((N, K // 2), device=w.device, dtype=torch.uint8)
    scale = torch.empty((N, K // BLOCK), device=w.device, dtype=torch.uint8)
    tiled, tscale = _tiles(N, K, L.MX_E2M1, w.device)
    _call(w.get_device(), "krq_quant_mxfp4", L.ptr(w), N, K, ld, L.ptr(w4), L.ptr(scale), L.ptr(tiled), L.ptr(tscale))
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
    _call(w4.get_device(), "krq_pack_mxfp4", L.ptr(w4), L.ptr(scale), N, K, L.ptr(tiled), L.ptr(tscale))
    return MXFP4Weight(w4, scale, tiled, tscale)


def _weight(q):
    if not isinstance(q, MXFP4Weight):
        raise ValueError("expected an MXFP4Weight (mxfp4.quantize or mxfp4.pack)")
    return q.shape


def dequantize(q):
    """The bf16 values an MXFP4Weight or MXRows stands for, [N, K] or [M, K] (its tiled copy's)."""
    if isinstance(q, MXRows):
        (M, K), elem, t = q.shape, ELEMS[q.elem], q.data
        _same_device(t)
        data = t.data_ptr()
        scale = data + q.scale_at
    else:
        (M, K), elem, t = _weight(q), L.MX_E2M1, q.tiled
        _same_device(t, q.tiled_scale)
        data, scale = t.data_ptr(), q.tiled_scale.data_ptr()
    out = t.new_empty((M, K), dtype=torch.bfloat16)
    if M:
        _call(t.get_device(), "krq_dequant_mx", data, scale, elem, M, K, out.data_ptr())
    return out


def _rows_bytes(M, K, e):
    """(where the scales start, the size) of M tiled rows: krq_mx_tiled_bytes and krq_mx_scale_bytes, tiles of 1 or 2 KiB
    and 256 bytes of scales per four of them, without two calls."""
    mb = (M + 15) >> 4
    at = (mb * ((K + 127) >> 7)) << (10 + e)
    return at, at + (mb * ((K + 511) >> 9) << 8)


def quant_rows(x, elem="e4m3"):
    """x [M, K] bf16 -> MXRows: the rows rounded to MX blocks, in the layout the products read. Several
    products on the same rows can share them."""
    x, ld = _bf16_rows(x, "rows [M, K]")
    M, K = x.shape
    e = _elem(elem)
    if M == 0:
        return MXRows(x.new_empty((0,), dtype=torch.uint8), 0, (0, K), elem)
    at, nbytes = _rows_bytes(M, K, e)
    data = x.new_empty((nbytes,), dtype=torch.uint8)
    p = data.data_ptr()
    _call(x.get_device(), "krq_quant_mx_rows", x.data_ptr(), M, K, ld, e, p, p + at)
    return MXRows(data, at, (M, K), elem)


def _operand(x, q, elem):
    """(the tensor that keeps x's memory, its address, its scales', x_kind, element type, row stride, M) of bf16 rows or
    MXRows that multiply q."""
    N, K = _weight(q)
    if x.shape[-1] != K:
        raise ValueError(f"x {tuple(x.shape)} and w [{N}, {K}] do not match")
    if isinstance(x, MXRows):
        t, M, ld, kind, elem = x.data, x.shape[0], 0, L.MX_X_TILED, x.elem
        p = t.data_ptr()
        scale = p + x.scale_at
    else:
        t, ld = _bf16_rows(x, "rows [M, K]")
        M, p, scale, kind = t.shape[0], t.data_ptr(), None, L.MX_X_BF16
    dev = t.get_device()
    if dev < 0 or q.tiled.get_device() != dev or q.tiled_scale.get_device() != dev:
        _same_device(t, q.tiled, q.tiled_scale)
    return t, p, scale, kind, ELEMS[elem] if elem in ELEMS else _elem(elem), ld, M


def _check_split(split, K):
    """Refuses a split that some part of K would have no group for."""
    if not 1 <= split <= min(-(-K // GROUP), SPLIT_MAX):
        raise ValueError(f"split={split} of {-(-K // GROUP)} groups of {GROUP} (K={K}), at most {SPLIT_MAX}")


def _decode(x, q, split, mode, elem):
    t, p, scale, kind, e, ld, M = _operand(x, q, elem)
    N, K = q.shape
    if M > DECODE_MAX_ROWS:
        raise ValueError(f"M={M} > {DECODE_MAX_ROWS} rows: use gemm_mxfp4 or linear_mxfp4")
    if mode == L.OUT_PARTIAL:
        _check_split(split, K)
        out = t.new_empty((split, M, N), dtype=torch.float32)
    else:
        if mode == L.OUT_SWIGLU:
            if N % 32:
                raise ValueError(f"SwiGLU needs w = [gate; up] of 2 I rows with I a multiple of 16, got N={N}")
            cols = N // 2
        else:
            cols = N
        out = t.new_empty((M, cols)) if kind == L.MX_X_BF16 else t.new_empty((M, cols), dtype=torch.bfloat16)
    if M == 0:
        return out
    ws, nbytes = None, 0
    if kind == L.MX_X_BF16 and K > (ROW_MAX_K if M == 1 else ROWS_MAX_K if M <= L.MX_BF16_ROWS else 0):
        # (more rows always need room for the rounded ones)
        nbytes = _rows_bytes(M, K, e)[1] if M > L.MX_BF16_ROWS else L.lib().krq_gemv_mxfp4_ws_bytes(kind, e, M, K, split)
        if nbytes > 0:
            ws = t.new_empty((nbytes,), dtype=torch.uint8)
    _call(t.get_device(), "krq_gemv_mxfp4", p, scale, kind, e, ld, q.tiled.data_ptr(), q.tiled_scale.data_ptr(), M, N, K, split, mode,
          L.ptr(ws), nbytes, out.data_ptr())
    return out


def gemv_mxfp4(x, q, split=1, elem="e4m3"):
    """MXFP4 counterpart of fp8.gemv_fp8: x [M, K] bf16 (M <= 32; rounded to blocks of elem) or MXRows, q an
    MXFP4Weight [N, K]. split == 1: bf16 [M, N]. split > 1: fp32 partials [split, M, N] whose in-order sum is
    the product; split s covers the groups of 512 k [s G / split, (s + 1) G / split), G = ceil(K / 512), so
    split <= G, and at most 64."""
    return _decode(x, q, split, L.OUT_BF16 if split == 1 else L.OUT_PARTIAL, elem)


def gemv_swiglu_mxfp4(x, q, elem="e4m3"):
    """MXFP4 counterpart of fp8.gemv_swiglu_fp8 for x of at most 32 rows: q packs w_gu [2I, K] = [gate; up], I % 16 == 0.
    Returns bf16(silu(g) * u) [M, I] from the fp32 g and u (one rounding, where the FP8 form rounds g, silu(g) and
    u first as the reference's does). More rows: silu(g) * u of the halves that linear_mxfp4 gives."""
    return _decode(x, q, 1, L.OUT_SWIGLU, elem)


def gemm_mxfp4(x, q, elem="e4m3"):
    """MXFP4 prefill product: x [M, K] bf16 (rounded to blocks of elem by a launch before the product's) or
    MXRows, any M; q an MXFP4Weight [N, K]. Returns bf16 [M, N]."""
    t, p, scale, kind, e, ld, M = _operand(x, q, elem)
    N, K = q.shape
    out = t.new_empty((M, N), dtype=torch.bfloat16)
    if M == 0:
        return out
    dev = t.get_device()
    if dev == _cuda._cuda_getDevice():
        nbytes = L.lib().krq_gemm_mxfp4_ws_bytes(kind, e, M, N, K)
    else:
        with torch.cuda.device(dev):  # (the plan is the current device's)
            nbytes = L.lib().krq_gemm_mxfp4_ws_bytes(kind, e, M, N, K)
    if nbytes < 0:
        raise RuntimeError("krq_gemm_mxfp4_ws_bytes: device query failed")
    ws = t.new_empty((nbytes,), dtype=torch.uint8) if nbytes else None
    _call(dev, "krq_gemm_mxfp4", p, scale, kind, e, ld, q.tiled.data_ptr(), q.tiled_scale.data_ptr(), M, N, K, L.ptr(ws), nbytes,
          out.data_ptr())
    return out


def linear_mxfp4(x, q, elem="e4m3"):
    """bf16 [M, N] ~= x @ W^T on q = quantize(W): gemv_mxfp4 up to 32 rows, gemm_mxfp4 from 33."""
    return _decode(x, q, 1, L.OUT_BF16, elem) if x.shape[0] <= DECODE_MAX_ROWS else gemm_mxfp4(x, q, elem)


def embedding(ids, q, scale=1.0):
    """Rows of the quantized table q [N, K] by index, times scale (a model's embedding multiplier): bf16
    [*ids.shape, K] = bf16(w[id] * scale) from the row-major codes. A model with tied embeddings passes one MXFP4Weight
    here and to the lm head, which reads its tiled copy. ids int64 or int32; an index outside [0, N) gives a row of NaN."""
    N, K = _weight(q)
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"ids must be int64 or int32, got {ids.dtype}")
    w4, scale_codes = q
    dev = w4.get_device()
    if dev < 0 or ids.get_device() != dev or scale_codes.get_device() != dev:
        _same_device(ids, w4, scale_codes)
    ids = ids.contiguous()
    out = w4.new_empty((*ids.shape, K), dtype=torch.bfloat16)
    n = ids.numel()
    if n:
        _call(dev, "krq_embed_mxfp4", ids.data_ptr(), ids.dtype is torch.int64, n, w4.data_ptr(), scale_codes.data_ptr(), N, K,
              float(scale), out.data_ptr())
    return out

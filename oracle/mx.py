"""CPU oracle of the microscaled (OCP MX v1.0) operators - TEST INFRASTRUCTURE, NOT PRODUCT CODE.

Written from the format's definition: blocks of 32 along K, E8M0 scale code c = max(0, floor(log2 amax) + 127
- emax) (255 for a block with a NaN or an infinity), elements by search for the nearest value of the format
in float64. Pinned in tests/test_mxfp4.py: the element tables by known answers of the formats and
(e4m3) torch's float8_e4m3fn, the rounding by brute force, the layout by a loop over its definition.
bf16 tensors are uint16 bit patterns, as in oracle.py.
"""

import numpy as np

from .oracle import bf16_to_f32

EMAX = {"e2m1": 2, "e4m3": 8}


def table(elem):
    """The non-negative values of the format by code."""
    if elem == "e2m1":
        return np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
    c = np.arange(127)
    e, m = c >> 3, c & 7
    return np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))


def encode(v, elem):
    """float64 magnitudes and signs -> element codes: nearest, ties to the even code, clamped."""
    t = table(elem)
    a = np.abs(v)
    i = np.searchsorted((t[1:] + t[:-1]) / 2, a, side="left")  # a tie falls to the lower code
    mid = (t[1:] + t[:-1]) / 2
    tie = (i < len(mid)) & (a == mid[np.minimum(i, len(mid) - 1)]) & (i % 2 == 1)
    sign = 8 if elem == "e2m1" else 128
    return (i + tie + np.where(np.signbit(v), sign, 0)).astype(np.uint8)


def quantize(x_u16, elem):
    """bf16 bits [M, K] -> (element codes uint8 [M, K], one per value; scale codes uint8 [M, K/32])."""
    M, K = x_u16.shape
    x = bf16_to_f32(x_u16).astype(np.float64).reshape(M, K // 32, 32)
    finite = np.isfinite(x).all(-1)
    x = np.where(finite[..., None], x, 0.0)
    amax = np.abs(x).max(-1)
    top = np.frexp(amax)[1] - 1  # floor(log2 amax)
    c = np.where(amax > 0, np.maximum(top + 127 - EMAX[elem], 0), 0)
    q = encode(x / 2.0 ** (c[..., None] - 127.0), elem)
    q = np.where(finite[..., None], q, 0).astype(np.uint8)
    return q.reshape(M, K), np.where(finite, c, 255).astype(np.uint8)


def values(codes, scale, elem):
    """float64 [M, K] of element codes and scales."""
    t = table(elem)
    sign = 8 if elem == "e2m1" else 128
    v = t[codes & (sign - 1)] * np.where(codes & sign, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
    return (v.reshape(*scale.shape, 32) * s[..., None]).reshape(codes.shape)


def pack4(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack4(w4):
    out = np.empty((w4.shape[0], 2 * w4.shape[1]), np.uint8)
    out[:, 0::2], out[:, 1::2] = w4 & 15, w4 >> 4
    return out


def tile(codes, scale, elem):
    """(elements, scales) in the "mx tiled" layout of include/krq.h, flat uint8."""
    M, K = codes.shape
    mb, kt, ks = -(-M // 16), -(-K // 128), -(-K // 512)
    full = np.zeros((16 * mb, 128 * kt), np.uint8)
    full[:M, :K] = codes
    f = full.reshape(mb, 16, kt, 128)
    if elem == "e2m1":
        b = (f[..., 0::2] | (f[..., 1::2] << 4)).reshape(mb, 16, kt, 4, 16)  # row block, r, tile, g, byte
        data = b.transpose(0, 2, 3, 1, 4)
    else:
        b = f.reshape(mb, 16, kt, 2, 4, 16)  # row block, r, tile, half, g, byte
        data = b.transpose(0, 2, 3, 4, 1, 5)
    s = np.zeros((16 * mb, 16 * ks), np.uint8)
    s[:M, :K // 32] = scale
    s = s.reshape(mb, 16, ks, 4, 4).transpose(0, 2, 4, 1, 3)  # row block, group, g, r, tile
    return np.ascontiguousarray(data).reshape(-1), np.ascontiguousarray(s).reshape(-1)


def norm_limit(xv, wv, elem, step):
    """How far the outputs of a product of rounded rows xv [M, K] and weights wv [N, K] may be from xv wv^T in the 2-norm over
    all of them, for data whose products have independent signs. A bound on one element has to allow for every rounding of its
    sum to fall one way; over many outputs they do not, and a product that is lost everywhere, or sums kept in too few
    bits, show here. In the 2-norm, R^2 = sum_k x^2 w^2 of an output, which is what the square of its sum, and of every
    partial sum at most, amounts to on average:
      output       half a step `step` of the value: step |y|
      accumulator  ceil(K / 128) + 16 results (instructions; additions of waves and parts), each of at most four fp32
                   sums that are off by a step 2^-23 of a partial sum: (ceil(K / 128) + 16) 2^-21 R, all of them one way
      e4m3         a product loses less than u = 2^-13 max|x| max|w| of its block, in the direction of its own sign: the squares
                   of the block's 32 losses add up, sqrt(sum_b 32 u_b^2)"""
    M, K = xv.shape
    y = np.linalg.norm(xv @ wv.T)
    R = np.sqrt(((xv ** 2) @ (wv ** 2).T).sum())
    cut = 0.0
    if elem == "e4m3":
        top = lambda v: (np.abs(v).reshape(len(v), -1, 32).max(-1)) ** 2
        cut = 2.0 ** -13 * np.sqrt(32 * (top(xv) @ top(wv).T).sum())
    return step * y + (-(-K // 128) + 16) * 2.0 ** -21 * R + cut

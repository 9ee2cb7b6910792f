"""The MXFP4 operators on the GPU against the float64 oracle of the format (oracle/mx.py).

Codes, scales, tiles, dequantised values and embedding rows are compared exactly. Products: the operands are
equal on both sides, so the error is the accumulation's and the output's rounding.
  Output: bf16, half a step, 2^-8 |y| (fp32 partials: 2^-24).
  Accumulator: one matrix instruction adds its 128 products and the accumulator in at most four fp32 sums, each
at most a step 2^-23 of the magnitudes' sum S = sum |x w| off; a result goes through at most ceil(K / 128)
instructions and one addition per wave (at most 8) or part: (ceil(K / 128) + 16) 2^-21 S.
  Products with an e4m3 operand: the instruction aligns the products it adds to the largest of them and cuts
what lies 2^-13 of that below it (one product of 2^8 beside one of 2^-5 is exact, beside one of 2^-6 it is the
2^8 alone; e2m1 products are exact beside each other, as are the sums of different blocks). A product's error
is therefore below 2^-13 max|x| max|w| of its block, a block's below 32 times that: 2^-8 sum_b max|x_b| max|w_b|."""

import numpy as np
import pytest
import torch

from kernels import _lib as L
from kernels import fp8, lmhead
from kernels import mxfp4 as X
from kernels.mlp import PersistentMLP
from oracle import mx as MX
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def bits(t):
    return t.detach().cpu().contiguous().view(torch.int16).numpy().view(np.uint16)


def u8(t):
    return t.cpu().numpy()


def bf(shape, seed, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16()


def spread(shape, seed):
    """Values over many powers of two, with blocks of zeros among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-12, 13, shape, generator=g).float())
    x.view(-1, 32)[::7] = 0
    return x.bfloat16()


def patterns():
    """Every bf16 bit pattern, in blocks whose largest member sets scales over the whole range: pattern p beside
    patterns of up to 4 binades more, then NaN and infinities in blocks of their own."""
    p = np.arange(65536, dtype=np.uint16).reshape(2048, 32)
    rolled = np.arange(65536, dtype=np.uint16).reshape(32, 2048).T.copy()  # one block spans 32 exponents
    return torch.from_numpy(np.concatenate([p, rolled]).view(np.int16)).view(torch.bfloat16)


def rounded(x, elem):
    codes, scale = MX.quantize(bits(x), elem)
    return MX.values(codes, scale, elem)


def weight(N, K, seed, dev, spread_out=False):
    w = spread((N, K), seed) if spread_out else bf((N, K), seed, 0.02)
    q = X.quantize(w.to(dev))
    return q, rounded(w, "e2m1")


def reference(xv, wv, elem="e4m3"):
    """The product and how far the accumulation may be off."""
    K = xv.shape[1]
    E = (-(-K // 128) + 16) * 2.0 ** -21 * (np.abs(xv) @ np.abs(wv).T)
    if elem == "e4m3":
        E += 2.0 ** -8 * (np.abs(xv).reshape(len(xv), -1, 32).max(-1) @ np.abs(wv).reshape(len(wv), -1, 32).max(-1).T)
    return xv @ wv.T, E


def check(y, ref, E, what, step=2.0 ** -8):
    y = y.double().cpu().numpy()
    assert y.shape == ref.shape
    lim = step * np.abs(ref) + E + 1e-40
    bad = ~(np.abs(y - ref) <= lim)
    assert not bad.any(), (what, np.argwhere(bad)[:4], y[bad][:4], ref[bad][:4], lim[bad][:4])


# ------------------------------------------------------------------------------------------ quantisation
SHAPES = [(1, 32), (16, 128), (17, 160), (33, 2880), (5, 544), (100, 1056), (48, 512), (2, 4096), (31, 96)]


@pytest.mark.parametrize("N,K", SHAPES)
def test_quantize_bytes(dev, N, K):
    w = spread((N, K), N + K)
    q = X.quantize(w.to(dev))
    codes, scale = MX.quantize(bits(w), "e2m1")
    assert np.array_equal(u8(q[0]), MX.pack4(codes)) and np.array_equal(u8(q[1]), scale)
    t, s = MX.tile(codes, scale, "e2m1")
    assert np.array_equal(u8(q.tiled), t) and np.array_equal(u8(q.tiled_scale), s)
    p = X.pack(q[0], q[1])
    assert torch.equal(p.tiled, q.tiled) and torch.equal(p.tiled_scale, q.tiled_scale)
    assert np.array_equal(X.dequantize(q).double().cpu().numpy(), MX.values(codes, scale, "e2m1"))


@pytest.mark.parametrize("elem", ["e2m1", "e4m3"])
@pytest.mark.parametrize("M,K", SHAPES)
def test_quant_rows_bytes(dev, M, K, elem):
    x = spread((M, K), M * K)
    rows = X.quant_rows(x.to(dev), elem)
    codes, scale = MX.quantize(bits(x), elem)
    t, s = MX.tile(codes, scale, elem)
    assert np.array_equal(u8(rows.tiled), t) and np.array_equal(u8(rows.tiled_scale), s)
    assert np.array_equal(X.dequantize(rows).double().cpu().numpy(), MX.values(codes, scale, elem))


@pytest.mark.parametrize("elem", ["e2m1", "e4m3"])
def test_every_bf16_pattern(dev, elem):
    x = patterns()
    rows = X.quant_rows(x.to(dev), elem)
    codes, scale = MX.quantize(bits(x), elem)
    t, s = MX.tile(codes, scale, elem)
    assert np.array_equal(u8(rows.tiled_scale), s)
    assert np.array_equal(u8(rows.tiled), t)
    v = MX.values(codes, scale, elem)
    want = torch.from_numpy(v.astype(np.float32)).bfloat16().double().numpy()  # (below 2^-126 bf16 holds fewer bits)
    assert np.array_equal(X.dequantize(rows).double().cpu().numpy(), want, equal_nan=True)


def test_pack_holds_any_codes(dev):
    g = np.random.default_rng(3)
    w4 = g.integers(0, 256, (37, 80)).astype(np.uint8)
    scale = g.integers(0, 256, (37, 5)).astype(np.uint8)
    q = X.pack(torch.from_numpy(w4).to(dev), torch.from_numpy(scale).to(dev))
    t, s = MX.tile(MX.unpack4(w4), scale, "e2m1")
    assert np.array_equal(u8(q.tiled), t) and np.array_equal(u8(q.tiled_scale), s)
    v = MX.values(MX.unpack4(w4), scale, "e2m1")
    with np.errstate(over="ignore"):
        want = torch.from_numpy(v).bfloat16().double().numpy()  # (scale 254: 1.5 and more pass the largest bf16)
    assert np.array_equal(X.dequantize(q).double().cpu().numpy(), want, equal_nan=True)


def test_strided_and_unaligned_rows(dev):
    big = bf((40, 1000), 5).to(dev)
    for view in (big[:, 8:168], big[::2, :160], big[3:4, 1:97], big[:, 1:161], big[:, :320:2], big[:20, :160].t().contiguous().t()):
        q = X.quantize(view)
        codes, scale = MX.quantize(bits(view), "e2m1")
        assert np.array_equal(u8(q[0]), MX.pack4(codes)) and np.array_equal(u8(q[1]), scale)
        qw, wv = weight(24, view.shape[1], 6, dev)
        M = min(view.shape[0], 7)
        ref, E = reference(rounded(view[:M], "e4m3"), wv)
        check(X.linear_mxfp4(view[:M], qw), ref, E, "view")


# ------------------------------------------------------------------------------------------ decode product
@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M", [1, 2, 4, 5, 8, 9, 16, 17, 32])
@pytest.mark.parametrize("N,K", [(16, 32), (1, 128), (33, 160), (100, 544), (64, 2880), (2560, 1024)])
def test_gemv(dev, M, N, K, elem):
    q, wv = weight(N, K, N + K, dev, spread_out=N < 2560)
    x = spread((M, K), M) if N < 2560 else bf((M, K), M)
    ref, E = reference(rounded(x, elem), wv, elem)
    xd = x.to(dev)
    y = X.gemv_mxfp4(xd, q, elem=elem)
    check(y, ref, E, (M, N, K, elem))
    rows = X.quant_rows(xd, elem)
    check(X.gemv_mxfp4(rows, q), ref, E, "rows")
    assert torch.equal(X.linear_mxfp4(xd, q, elem), y)


@pytest.mark.parametrize("M,N,K,split", [(1, 2560, 4096, 1), (3, 2560, 9728, 1), (32, 2560, 9728, 1), (16, 6144, 2560, 1),
                                         (1, 6144, 2560, 2), (5, 2560, 9728, 4), (32, 2560, 4096, 8), (20, 100, 1056, 3),
                                         (7, 48, 16384, 1), (12, 48, 16384, 5), (1, 16, 33 * 512 + 96, 34),
                                         # every place of the rows and the weights: one or several row blocks per workgroup,
                                         # one or two groups per wave, operands beside the weights
                                         (1, 18000, 1056, 1), (8, 16400, 2560, 1), (16, 17000, 5632, 1), (32, 16500, 2080, 1),
                                         (1, 9000, 10240, 1), (3, 100, 5152, 1), (20, 10000, 4096, 1), (32, 300, 4608, 1),
                                         (16, 96, 10272, 1), (1, 9000, 6016, 2), (32, 64, 12288, 3),
                                         (32, 16500, 4096, 1), (9, 48, 32, 1)])
def test_gemv_large_and_split(dev, M, N, K, split):
    q, wv = weight(N, K, 1, dev)
    x = bf((M, K), 2)
    ref, E = reference(rounded(x, "e4m3"), wv)
    y = X.gemv_mxfp4(x.to(dev), q, split)
    if split == 1:
        check(y, ref, E, "whole")
    else:
        assert y.shape == (split, M, N) and y.dtype == torch.float32
        check(y.double().sum(0), ref, E, "sum", 2.0 ** -24)
        G = -(-K // 512)
        for s in range(split):
            a, b = 512 * (G * s // split), min(K, 512 * (G * (s + 1) // split))
            r, t = reference(rounded(x, "e4m3")[:, a:b], wv[:, a:b])
            check(y[s], r, t, s, 2.0 ** -24)


def swiglu_check(y, xv, wv, elem="e4m3"):
    I = wv.shape[0] // 2
    ref, e = reference(xv, wv, elem)
    g, u = ref[:, :I], ref[:, I:]
    sig = 1 / (1 + np.exp(-g))
    act = g * sig * u
    # |d silu| <= 1.1 |dg|; expf, the division and two products are within 2^-20 of the value
    lim = (2.0 ** -8 + 2.0 ** -20) * np.abs(act) + 1.1 * e[:, :I] * (np.abs(u) + e[:, I:]) + np.abs(g * sig) * e[:, I:] + 1e-40
    y = y.double().cpu().numpy()
    bad = ~(np.abs(y - act) <= lim)
    assert not bad.any(), (y[bad][:4], act[bad][:4], lim[bad][:4])


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,I,K", [(1, 16, 32), (1, 9728, 2560), (3, 48, 160), (8, 80, 1056), (9, 64, 2880), (16, 1024, 2560), (32, 112, 544),
                                   (32, 48, 4096), (17, 32, 4640), (2, 80, 9728)])
def test_gemv_swiglu(dev, M, I, K, elem):
    q, wv = weight(2 * I, K, 4, dev)
    x = bf((M, K), 5)
    swiglu_check(X.gemv_swiglu_mxfp4(x.to(dev), q, elem), rounded(x, elem), wv, elem)


def test_swiglu_far_gates(dev):
    """Gates of -200 and 200: silu ends in -0 and the gate itself, without NaN from the exponential."""
    w = torch.zeros(32, 32)
    w[0, 0], w[1, 0], w[16:, 1] = 100, -100, 1
    x = torch.zeros(1, 32)
    x[0, 0], x[0, 1] = 2, 3
    y = X.gemv_swiglu_mxfp4(x.bfloat16().to(dev), X.quantize(w.bfloat16().to(dev))).float().cpu()
    wv, xv = rounded(w.bfloat16(), "e2m1"), rounded(x.bfloat16(), "e4m3")
    assert y[0, 0] == float(torch.tensor(xv[0, 0] * wv[0, 0] * 3).bfloat16()) and y[0, 1] == 0 and y[0, 2:].eq(0).all()


@pytest.mark.parametrize("M", [1, 6, 20, 50])
def test_nan_stays_in_its_row_and_column(dev, M):
    K, N = 1056, 48
    w, x = bf((N, K), 1, 0.02), bf((M, K), 2)
    x[M // 2, 700] = float("inf")
    w[11, 3] = float("nan")
    q = X.quantize(w.to(dev))
    xv, wv = rounded(x, "e4m3"), rounded(w, "e2m1")
    assert np.isnan(xv[M // 2, 672:704]).all() and np.isnan(wv[11, :32]).all()
    y = X.linear_mxfp4(x.to(dev), q).double().cpu().numpy()
    bad = np.zeros((M, N), bool)
    bad[M // 2], bad[:, 11] = True, True
    assert np.array_equal(np.isnan(y), bad)
    ref, E = reference(np.nan_to_num(xv), np.nan_to_num(wv))
    check(torch.from_numpy(np.where(bad, ref, y)), ref, E, "rest")


@pytest.mark.parametrize("ex,ew", [(60, -70), (-110, 100), (100, -20), (-60, -40)])
def test_scales_far_from_one(dev, ex, ew):
    K, N = 544, 48
    w, x = bf((N, K), 1) * 2.0 ** ew, bf((40, K), 2) * 2.0 ** ex
    q = X.quantize(w.to(dev))
    ref, E = reference(rounded(x, "e4m3"), rounded(w, "e2m1"))
    check(X.linear_mxfp4(x.to(dev), q), ref, E, "gemm")
    for M in (1, 6, 20):
        check(X.linear_mxfp4(x[:M].to(dev), q), ref[:M], E[:M], M)


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(1, 65536, 64), (4, 65549, 544), (1, 70003, 1056), (5, 32768, 32), (8, 32770, 3552), (16, 33001, 96),
                                   (16, 32784, 2560), (17, 32769, 1184), (32, 32800, 3584), (32, 50002, 160)])
def test_gemv_many_columns(dev, M, N, K, elem):
    """Enough row blocks for a wave to take whole ones, odd columns and ends of K, rows of NaN among them; equal to nothing but
    the reference behind the last row."""
    w, x = bf((N, K), N, 0.05), bf((M, K), M)
    x[M // 2, K // 2] = float("inf")
    w[32001, K - 1] = float("nan")
    q = X.quantize(w.to(dev))
    xv, wv = rounded(x, elem), rounded(w, "e2m1")
    bad = np.zeros((M, N), bool)
    bad[M // 2], bad[:, 32001] = True, True
    ref, E = reference(np.nan_to_num(xv), np.nan_to_num(wv))
    for src in (x.to(dev), X.quant_rows(x.to(dev), elem)):
        y = X.gemv_mxfp4(src, q, elem=elem).double().cpu().numpy()
        assert np.array_equal(np.isnan(y), bad)
        check(torch.from_numpy(np.where(bad, ref, y)), ref, E, (M, N, K, elem))
    rows = X.quant_rows(x.to(dev), elem)
    out = torch.full((M + 3, N), 7.0, device=dev, dtype=torch.bfloat16)
    L.call("krq_gemv_mxfp4", L.ptr(rows.tiled), L.ptr(rows.tiled_scale), L.MX_X_TILED, X.ELEMS[elem], 0, L.ptr(q.tiled),
           L.ptr(q.tiled_scale), M, N, K, 1, L.OUT_BF16, None, 0, L.ptr(out), L.stream(out))
    assert out[M:].eq(7).all() and torch.equal(out[:M].nan_to_num(), X.gemv_mxfp4(rows, q).nan_to_num())


def test_outputs_end_where_they_should(dev):
    """Through the C ABI into larger buffers: nothing behind the last row is touched."""
    M, N, K = 19, 37, 544
    q, wv = weight(N, K, 1, dev)
    x = bf((M, K), 2).to(dev)
    rows = X.quant_rows(x)
    ref, E = reference(rounded(x, "e4m3"), wv)
    for name, extra in (("krq_gemv_mxfp4", True), ("krq_gemm_mxfp4", False)):
        out = torch.full((M + 16, N), 7.0, device=dev, dtype=torch.bfloat16)
        tail = (1, L.OUT_BF16) if extra else ()
        L.call(name, L.ptr(rows.tiled), L.ptr(rows.tiled_scale), L.MX_X_TILED, L.MX_E4M3, 0, L.ptr(q.tiled), L.ptr(q.tiled_scale),
               M, N, K, *tail, None, 0, L.ptr(out), L.stream(x))
        check(out[:M], ref, E, name)
        assert out[M:].eq(7).all()


# ------------------------------------------------------------------------------------------ prefill product
@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (33, 17, 160), (77, 6144, 512), (128, 128, 128), (129, 257, 2880), (300, 1000, 1056),
                                   (64, 2560, 4096), (257, 256, 9728), (520, 768, 640), (1000, 2560, 2560), (2049, 304, 512),
                                   # every output tile on 256 compute units, several tiles per workgroup, groups of one stage:
                                   # 256 x 256, 192 x 256, 128 x 256 (and N not of whole 16-byte pieces), 128 x 128, 64 x 64
                                   (4096, 4096, 640), (4000, 2560, 544), (4000, 6100, 640), (4000, 6104, 640), (500, 2560, 2176),
                                   (700, 1100, 1152),
                                   # K in parts: whole and ragged columns
                                   (77, 520, 8224), (40, 99, 16384), (64, 2560, 9728), (77, 520, 8320),
                                   # odd and even numbers of tiles of K: one and two a stage
                                   (4096, 4096, 1024), (1000, 2560, 1024), (1000, 2560, 1152), (200, 640, 1280), (200, 640, 1184)])
def test_gemm(dev, M, N, K, elem):
    q, wv = weight(N, K, 3, dev, spread_out=M < 77)
    x = bf((M, K), 4)
    ref, E = reference(rounded(x, elem), wv, elem)
    y = X.gemm_mxfp4(x.to(dev), q, elem)
    check(y, ref, E, (M, N, K, elem))
    assert torch.equal(X.gemm_mxfp4(X.quant_rows(x.to(dev), elem), q), y)
    if M > 32:
        assert torch.equal(X.linear_mxfp4(x.to(dev), q, elem), y)


def test_empty_rows(dev):
    q, _ = weight(64, 96, 1, dev)
    none = torch.empty((0, 96), device=dev, dtype=torch.bfloat16)
    assert X.linear_mxfp4(none, q).shape == (0, 64) and X.gemm_mxfp4(none, q).shape == (0, 64)
    assert X.gemv_swiglu_mxfp4(none, q).shape == (0, 32) and X.dequantize(X.quant_rows(none)).shape == (0, 96)
    assert X.embedding(torch.empty((0, 3), device=dev, dtype=torch.int64), q).shape == (0, 3, 96)
    with pytest.raises(ValueError):
        X.quantize(none)
    with pytest.raises(ValueError):
        lmhead.lm_head_argmax(none, q)


# ------------------------------------------------------------------------------------------ sizes past 32 bits
def test_far_offsets(dev):
    """2.2 million rows of 4,096: 18 GB of bf16, 4.5 GB of codes and of tiles, more row blocks than the second axis of a
    grid. The last rows are what they are on their own."""
    N, K = 2_200_003, 4096
    w = torch.empty((N, K), device=dev, dtype=torch.bfloat16).normal_(0, 0.02, generator=torch.Generator(device=dev).manual_seed(1))
    tail = w[-115:].clone()
    q, small = X.quantize(w), X.quantize(tail)
    assert torch.equal(q[0][-115:], small[0]) and torch.equal(q[1][-115:], small[1])
    p = X.pack(q[0], q[1])
    assert torch.equal(p.tiled[-(1 << 20):], q.tiled[-(1 << 20):]) and torch.equal(p.tiled_scale[-(1 << 20):], q.tiled_scale[-(1 << 20):])
    del p, w
    want = X.dequantize(small)
    assert torch.equal(X.dequantize(q)[-115:], want)
    ids = torch.arange(N - 115, N, device=dev)
    assert torch.equal(X.embedding(ids, q), want)
    for M in (1, 20):
        x = bf((M, K), M).to(dev)
        assert torch.equal(X.linear_mxfp4(x, q)[:, -115:], X.linear_mxfp4(x, small))


def test_far_columns(dev):
    """3,000,017 columns of K = 1,632: 2.5 GB of tiles under waves that take whole row blocks."""
    N, K = 3_000_017, 1632
    at = N - 17 - 80_000 + 16
    w = torch.empty((N, K), device=dev, dtype=torch.bfloat16).normal_(0, 0.02, generator=torch.Generator(device=dev).manual_seed(4))
    q, small = X.quantize(w), X.quantize(w[at:])
    del w
    assert at % 16 == 0
    for M in (3, 16, 32):
        x = bf((M, K), M).to(dev)
        assert torch.equal(X.linear_mxfp4(x, q)[:, at:], X.linear_mxfp4(x, small))


def test_far_rows(dev):
    """600,001 rows through the prefill product: 9.8 GB of output; and more rows than a grid's second axis of row blocks."""
    M, N, K = 600_001, 8192, 512
    q = X.quantize(bf((N, K), 1, 0.02).to(dev))
    x = torch.empty((M, K), device=dev, dtype=torch.bfloat16).normal_(generator=torch.Generator(device=dev).manual_seed(2))
    for elem in ("e4m3", "e2m1"):
        y = X.linear_mxfp4(x, q, elem)
        assert torch.equal(y[-77:], X.linear_mxfp4(x[-77:].clone(), q, elem)) and torch.equal(y[:77], X.linear_mxfp4(x[:77].clone(), q, elem))
        del y
    x = x.view(-1, 32)[:1_100_000]
    assert torch.equal(X.dequantize(X.quant_rows(x))[-99:], X.dequantize(X.quant_rows(x[-99:].clone())))
    ids = torch.randint(8192, (300_001,), device=dev)
    assert torch.equal(X.embedding(ids, q)[-99:], X.embedding(ids[-99:].clone(), q))


# ------------------------------------------------------------------------------------------ lm head
@pytest.mark.parametrize("M,V,K", [(1, 16, 32), (1, 70000, 512), (5, 4112, 2560), (1, 16400, 2560), (32, 20000, 2560), (2, 9008, 6400), (20, 4096, 6400), (16, 1040, 10752), (7, 48, 512), (8, 1024, 160), (9, 32000, 1024), (16, 4096, 2880),
                                   (32, 2048, 544), (32, 4112, 4096), (25, 1040, 5120), (1, 33008, 5632), (16, 9008, 10240), (1, 1040, 10272),
                                   (9, 16000, 32), (16, 17008, 3552), (32, 16400, 3552), (24, 40000, 160), (17, 16016, 1024)])
def test_head(dev, M, V, K):
    q, wv = weight(V, K, 7, dev)
    h = bf((M, K), 8)
    idx, logits = lmhead.lm_head_argmax(h.to(dev), q, return_logits=True)
    ref, E = reference(rounded(h, "e4m3"), wv)
    check(logits, ref, E, (M, V, K))
    assert idx.dtype == torch.int64 and torch.equal(idx.cpu(), torch.argmax(logits.float().cpu(), -1))
    assert torch.equal(lmhead.lm_head_argmax(h.to(dev), q), idx)


@pytest.mark.parametrize("M", [1, 8, 16, 32])
def test_head_ties_and_nan(dev, M):
    """Equal rows give equal logits wherever they lie: the lowest index wins; a NaN logit is the maximum."""
    V, K = 8208, 512
    w, h = bf((V, K), 1, 0.02), bf((M, K), 2)
    best = (50 * h[0].float() / h[0].float().norm()).bfloat16()
    for i in (8200, 4095, 37, 36):
        w[i] = best
    h[1:] = h[0]
    idx = lmhead.lm_head_argmax(h.to(dev), X.quantize(w.to(dev)))
    assert idx.tolist() == [36] * M
    w[5000, 7] = float("nan")
    assert lmhead.lm_head_argmax(h.to(dev), X.quantize(w.to(dev))).tolist() == [5000] * M
    w = torch.cat([w[:, :256], w[:, :256]])  # more row blocks: the ties at 36, 37, 4095, 8200 and 8208 further on, the NaN twice
    assert lmhead.lm_head_argmax(h[:, :256].to(dev), X.quantize(w.to(dev))).tolist() == [5000] * M
    tied = bf((V, 256), 3, 0.02)
    tied = torch.cat([tied, tied])
    tied[[36, 37, 4095, 8200, 8244, 16000]] = best[:256]
    assert lmhead.lm_head_argmax(h[:, :256].to(dev), X.quantize(tied.to(dev))).tolist() == [36] * M
    with pytest.raises(ValueError, match="ActScale"):
        lmhead.lm_head_argmax(h.to(dev), X.quantize(w.to(dev)), a=fp8.ActScale(h.to(dev)))


# ------------------------------------------------------------------------------------------ embedding
@pytest.mark.parametrize("N,K", [(7, 32), (1000, 2560), (33, 2880), (50, 1056)])
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_embedding(dev, N, K, dtype):
    w = spread((N, K), 1)
    q = X.quantize(w.to(dev))
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(N, (3, 41), generator=g)
    ids[0, :4] = torch.tensor([0, N - 1, 0, N - 1])
    v = torch.from_numpy(rounded(w, "e2m1"))[ids].float()
    for scale in (1.0, 50.596442562694074, 0.0):
        y = X.embedding(ids.to(dev, dtype), q, scale)
        assert torch.equal(y.cpu(), (v * torch.tensor(scale, dtype=torch.float32)).bfloat16())
    out = ids.clone()
    out[1, 5], out[2, 7] = N, -1
    y = X.embedding(out.to(dev, dtype), q).cpu()
    bad = (out < 0) | (out >= N)
    assert torch.isnan(y[bad].float()).all() and torch.equal(y[~bad], v[~bad].bfloat16())
    assert torch.equal(X.embedding(ids.to(dev, dtype)[:, ::2], q).cpu(), v[:, ::2].bfloat16())
    one = X.embedding(torch.tensor(N - 1, device=dev, dtype=dtype), q)
    assert one.shape == (K,) and torch.equal(one.cpu(), torch.from_numpy(rounded(w, "e2m1"))[N - 1].bfloat16())


# ------------------------------------------------------------------------------------------ together
def layer(dev, H, I, V, seed):
    return {"emb": X.quantize(bf((V, H), seed, 0.02).to(dev)), "qkv": X.quantize(bf((H + 64, H), seed + 1, 0.02).to(dev)),
            "gu": X.quantize(bf((2 * I, H), seed + 2, 0.02).to(dev)), "down": X.quantize(bf((H, I), seed + 3, 0.02).to(dev))}


def step(ids, p, scale):
    """Embedding, a projection, the MLP and the head, as a 4-bit model's step calls them."""
    x = X.embedding(ids, p["emb"], scale)
    y = X.linear_mxfp4(x, p["qkv"])
    if x.shape[0] <= 32:
        act = X.gemv_swiglu_mxfp4(x, p["gu"])
    else:
        g, u = X.linear_mxfp4(x, p["gu"]).float().chunk(2, -1)
        act = (torch.nn.functional.silu(g) * u).bfloat16()
    z = X.linear_mxfp4(act, p["down"])
    last = z[-8:]
    return (x, y, act, z) + lmhead.lm_head_argmax(last, p["emb"], return_logits=True)


@pytest.mark.parametrize("M", [1, 7, 24, 90])
def test_model_step(dev, M):
    H, I, V = 544, 1056, 2064
    p = layer(dev, H, I, V, 10)
    ids = torch.randint(V, (M,), generator=torch.Generator().manual_seed(M))
    x, y, act, z, idx, logits = step(ids.to(dev), p, 20.0)
    val = {k: X.dequantize(q).double().cpu().numpy() for k, q in p.items()}
    assert torch.equal(x.cpu(), (torch.from_numpy(val["emb"])[ids].float() * 20.0).bfloat16())
    for rows, name, out in ((x, "qkv", y), (act, "down", z), (z[-8:], "emb", logits)):
        ref, E = reference(rounded(rows, "e4m3"), val[name])
        check(out, ref, E, name)
    if M <= 32:
        swiglu_check(act, rounded(x, "e4m3"), val["gu"])
    assert torch.equal(idx.cpu(), torch.argmax(logits.float().cpu(), -1))


@pytest.mark.parametrize("M", [1, 9, 40])
def test_graph_replays(dev, M):
    """A captured step against eager ones, replayed with eager work and new inputs between the replays."""
    p = layer(dev, 512, 1024, 1024, 20)
    ids = torch.zeros(M, device=dev, dtype=torch.int64)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(ids, p, 8.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(ids, p, 8.0)
    for k in range(4):
        new = torch.randint(1024, (M,), generator=torch.Generator().manual_seed(k)).to(dev)
        ids.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(new, p, 8.0)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_two_streams(dev):
    p = layer(dev, 512, 1024, 1024, 30)
    ids = [torch.randint(1024, (m,), generator=torch.Generator().manual_seed(m)).to(dev) for m in (12, 70)]
    want = [step(i, p, 3.0) for i in ids]
    streams = [torch.cuda.Stream() for _ in ids]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(step(ids[k], p, 3.0))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[k]))


@pytest.mark.parametrize("M", [1, 4, 16])
def test_persistent_mlp(dev, M):
    H, I = 512, 2048
    p = layer(dev, H, I, 64, 40)
    h = bf((M, H), 1).to(dev)
    mlp = PersistentMLP(M, H, I, dev)
    out = mlp(h, p["gu"], p["down"])
    assert out.shape == (4, M, H) and torch.equal(mlp.act, X.gemv_swiglu_mxfp4(h, p["gu"]))
    assert torch.equal(out, X.gemv_mxfp4(mlp.act, p["down"], 4))
    with pytest.raises(ValueError):
        mlp(h, p["gu"], fp8.quantize(torch.zeros(H, I, device=dev, dtype=torch.bfloat16)))
    with pytest.raises(ValueError):
        PersistentMLP(M, H, I, dev, one_launch=True)(h, p["gu"], p["down"])
    assert PersistentMLP(M, H, I, dev, split=1)(h, p["gu"], p["down"]).shape == (1, M, H)


def test_refusals_on_the_device(dev):
    q, _ = weight(64, 96, 1, dev)
    x = bf((4, 96), 1).to(dev)
    for call in (lambda: X.gemv_mxfp4(bf((33, 96), 1).to(dev), q), lambda: X.gemv_mxfp4(x, q, 2), lambda: X.gemv_mxfp4(x, q, 0),
                 lambda: X.gemv_mxfp4(x[:, :64], q), lambda: X.gemv_mxfp4(x.float(), q), lambda: X.gemm_mxfp4(x, q, "e5m2"),
                 lambda: X.gemv_swiglu_mxfp4(x, weight(48, 96, 1, dev)[0]), lambda: X.quantize(x[:, :40]),
                 lambda: X.quantize(x[0]), lambda: X.pack(q[0], q[1][:, :2]), lambda: X.pack(q[0].int(), q[1]),
                 lambda: fp8.gemv_fp8(x, q), lambda: fp8.linear_fp8(x, q), lambda: X.dequantize((q[0], q[1])),
                 lambda: lmhead.lm_head_argmax(x, weight(40, 96, 1, dev)[0]),
                 lambda: lmhead.lm_head_argmax(bf((33, 96), 1).to(dev), q)):
        with pytest.raises(ValueError):
            call()


def test_tiles_that_moved(dev):
    """A weight whose tiles were copied elsewhere is read from there."""
    q, _ = weight(80, 2880, 2, dev)
    x = bf((3, 2880), 3).to(dev)
    want = [X.gemv_mxfp4(x, q), X.gemm_mxfp4(x, q), lmhead.lm_head_argmax(x, q)]
    q.tiled, q.tiled_scale = q.tiled.clone(), q.tiled_scale.clone()
    for a, b in zip([X.gemv_mxfp4(x, q), X.gemm_mxfp4(x, q), lmhead.lm_head_argmax(x, q)], want):
        assert torch.equal(a, b)


def test_tensors_of_the_cpu_are_refused(dev):
    q, _ = weight(64, 96, 1, dev)
    with pytest.raises(RuntimeError, match="ROCm device"):
        X.linear_mxfp4(torch.zeros(1, 96, dtype=torch.bfloat16), q)
    with pytest.raises(RuntimeError, match="ROCm device"):
        X.embedding(torch.zeros(1, dtype=torch.int64), q)


def test_oracle_bits_agree(dev):
    """The oracle's bf16 view is the tensor's."""
    x = patterns()[:64]
    assert np.array_equal(O.bf16_to_f32(bits(x)).view(np.uint32), x.float().numpy().view(np.uint32))

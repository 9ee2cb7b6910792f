"""Every product's outputs together against the 64-bit oracle: the 2-norm of their error (oracle/mx.py, norm_limit, which says what it
allows for and why), in each kernel and for both types of rows. test_gpu_mxfp4.py bounds each output by itself."""

import numpy as np
import pytest
import torch

from kernels import lmhead
from kernels import mxfp4 as X
from kernels.mlp import PersistentMLP
from oracle import mx as MX
from test_gpu_mxfp4 import bf, check, reference, rounded, weight

pytestmark = pytest.mark.gpu
BF16, FP32 = 2.0 ** -8, 2.0 ** -24  # half a step


def near(y, xv, wv, elem, step, what):
    off, limit = np.linalg.norm(y.double().cpu().numpy() - xv @ wv.T), MX.norm_limit(xv, wv, elem, step)
    assert off <= limit, (what, off, limit)


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K,split", [
    # rows held, bf16 and rounded before: one and two groups a wave, one and two row tiles
    (1, 2560, 2560, 2), (1, 300, 9728, 1), (1, 6144, 10240, 2), (5, 2560, 9728, 4), (8, 2560, 2560, 1), (12, 48, 16384, 5), (16, 2560, 9728, 1),
    (20, 100, 1056, 3), (32, 2560, 4096, 8), (32, 300, 4096, 1),
    # streamed
    (1, 48, 40960, 1), (7, 48, 16384, 1), (16, 96, 12288, 1), (9, 96, 24576, 2), (32, 2560, 9728, 1), (24, 64, 12288, 2), (17, 33, 33 * 512 + 96, 3),
    # operands in LDS
    (4, 65536, 544, 1), (8, 32770, 2560, 1), (16, 32784, 3552, 1), (32, 32800, 1056, 1)])
def test_gemv(dev, M, N, K, split, elem):
    q, wv = weight(N, K, 1, dev)
    x = bf((M, K), 2)
    xv = rounded(x, elem)
    G = -(-K // 512)
    for src in (x.to(dev), X.quant_rows(x.to(dev), elem)):
        y = X.gemv_mxfp4(src, q, split, elem)
        if split == 1:
            near(y, xv, wv, elem, BF16, "whole")
            continue
        assert y.dtype == torch.float32 and y.shape == (split, M, N)
        near(y.double().sum(0), xv, wv, elem, FP32, "sum")
        for s in range(split):
            a, b = 512 * (G * s // split), min(K, 512 * (G * (s + 1) // split))
            near(y[s], xv[:, a:b], wv[:, a:b], elem, FP32, s)
            ref, E = reference(xv[:, a:b], wv[:, a:b], elem)
            check(y[s], ref, E, s, FP32)


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
# every output tile, one and two tiles a stage, K in parts, too few stages for the stream
@pytest.mark.parametrize("M,N,K", [(33, 640, 384), (77, 6144, 2560), (200, 640, 1184), (64, 2560, 9728), (77, 520, 8224), (500, 2560, 2176),
                                   (1000, 2560, 1152), (1000, 2560, 2560), (4000, 2560, 544), (4000, 2560, 1024), (4096, 4096, 640), (4096, 4096, 1024)])
def test_gemm(dev, M, N, K, elem):
    q, wv = weight(N, K, 3, dev)
    x = bf((M, K), 4)
    near(X.gemm_mxfp4(x.to(dev), q, elem), rounded(x, elem), wv, elem, BF16, (M, N, K))


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,V,K", [(1, 16400, 2560), (6, 4112, 4096), (16, 4096, 6400), (32, 4112, 4096), (16, 1040, 10752), (32, 2048, 9728),
                                   (16, 17008, 3552), (32, 16400, 2560)])
def test_head(dev, M, V, K, elem):
    q, wv = weight(V, K, 7, dev)
    h = bf((M, K), 8)
    idx, logits = lmhead.lm_head_argmax(X.quant_rows(h.to(dev), elem), q, return_logits=True)
    near(logits, rounded(h, elem), wv, elem, BF16, (M, V, K))
    assert torch.equal(idx.cpu(), torch.argmax(logits.float().cpu(), -1))
    if elem == "e4m3":
        near(lmhead.lm_head_argmax(h.to(dev), q, return_logits=True)[1], rounded(h, elem), wv, elem, BF16, "bf16 rows")


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,I,K", [(1, 48, 6016), (1, 1024, 2560), (1, 32, 10272), (5, 1024, 2560), (16, 80, 9728), (32, 112, 4096), (32, 48, 9728)])
def test_swiglu_gate_and_up(dev, M, I, K, elem):
    """silu(32) is 32: with gates of exactly 32 SwiGLU shows the up sums."""
    w, x = bf((2 * I, K), 4, 0.02), bf((M, K), 5)
    x[:, :32] = 0
    x[:, 0] = 8.0
    w[:, :32] = 0
    w[:I] = 0
    w[:I, 0] = 4.0
    q = X.quantize(w.to(dev))
    xv, wv = rounded(x, elem), rounded(w, "e2m1")
    gate, up = xv @ wv[:I].T, wv[I:]
    assert (gate == 32).all()
    for src in (x.to(dev), X.quant_rows(x.to(dev), elem)):
        near(X.gemv_swiglu_mxfp4(src, q, elem).double() / 32, xv, up, elem, BF16, (M, I, K))


@pytest.mark.parametrize("M", [1, 4, 16, 32])
def test_persistent_mlp(dev, M):
    """Both of its products: the partials' sum is the down product of the activations it kept."""
    H, I = 512, 2048
    gu, _ = weight(2 * I, H, 1, dev)
    down, dv = weight(H, I, 2, dev)
    mlp = PersistentMLP(M, H, I, dev)
    out = mlp(bf((M, H), 3).to(dev), gu, down)
    xv = rounded(mlp.act, "e4m3")
    for s in range(4):
        near(out[s], xv[:, 512 * s:512 * s + 512], dv[:, 512 * s:512 * s + 512], "e4m3", FP32, s)

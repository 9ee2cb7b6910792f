"""Calls of the MXFP4 operators on the GPU beside those of test_gpu_mxfp4.py: rounded rows in the head, the borders of the
formats' ranges, launch shapes. Bounds of one element are test_gpu_mxfp4.py's."""

import numpy as np
import pytest
import torch

from kernels import _lib as L
from kernels import lmhead
from kernels import mxfp4 as X
from oracle import mx as MX
from test_gpu_mxfp4 import bf, check, reference, rounded, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
# rows held in registers (one and two groups a wave, one and two row tiles), streamed, in LDS
@pytest.mark.parametrize("M,V,K", [(1, 1040, 2560), (7, 48, 512), (16, 4112, 1056), (8, 1040, 6400), (25, 2064, 2560), (3, 1040, 10752),
                                   (32, 1040, 4640), (9, 16000, 160), (16, 17008, 3552), (17, 16016, 1024), (32, 16400, 3552)])
def test_head_of_rounded_rows(dev, M, V, K, elem):
    """The head on MXRows of either type: logits, their argmax, and the ids alone."""
    q, wv = weight(V, K, 7, dev)
    h = bf((M, K), 8)
    rows = X.quant_rows(h.to(dev), elem)
    idx, logits = lmhead.lm_head_argmax(rows, q, return_logits=True)
    ref, E = reference(rounded(h, elem), wv, elem)
    check(logits, ref, E, (M, V, K, elem))
    assert idx.dtype == torch.int64 and torch.equal(idx.cpu(), torch.argmax(logits.float().cpu(), -1))
    assert torch.equal(lmhead.lm_head_argmax(rows, q), idx)
    if elem == "e4m3":
        check(lmhead.lm_head_argmax(h.to(dev), q, return_logits=True)[1], ref, E, "bf16 rows")


@pytest.mark.parametrize("sets", [513, 514, 771, 1025, 1027, 1281])
def test_a_long_launch_has_a_workgroup_per_compute_unit_at_most(dev, sets):
    """The head's candidates, one per workgroup and row block of a pair, counted in its workspace: no more than two for each
    of 256 compute units, where one unit with a second workgroup would take twice as long as the others. They still cover
    every column."""
    V, K = 32 * sets, 512
    q, _ = weight(V, K, 3, dev)
    h = bf((1, K), 4).to(dev)
    nbytes = L.lib().krq_lmhead_mxfp4_ws_bytes(L.MX_X_BF16, L.MX_E4M3, 1, V, K)
    ws = torch.full((nbytes // 8,), 0x5A5A5A5A5A5A5A5A, device=dev, dtype=torch.int64)
    logits, idx = torch.empty((1, V), device=dev, dtype=torch.bfloat16), torch.empty((1,), device=dev, dtype=torch.int64)
    L.call("krq_lmhead_argmax_mxfp4", L.ptr(h), None, L.MX_X_BF16, L.MX_E4M3, K, L.ptr(q.tiled), L.ptr(q.tiled_scale), 1, V, K, L.ptr(logits),
           L.ptr(ws), nbytes, L.ptr(idx), L.stream(h))
    assert 0 < int(ws.ne(0x5A5A5A5A5A5A5A5A).sum()) <= 2 * 256
    assert idx.item() == int(torch.argmax(logits.float().cpu(), -1))


@pytest.mark.parametrize("mult", [1.0, 0.5, 0.25, 2.0 ** -8, 50.596442562694074, 3.0e-38, 2.0 ** -140, 2.0 ** -149, 2.0 ** 100, -1.0, 0.0])
def test_embedding_of_every_scale(dev, mult):
    """Every element under every scale code, a row each, times multipliers from the smallest to large ones: the value times mult in
    64 bits, then the one rounding of fp32 and that of bf16. Codes 253 and 254 hold values beyond fp32 whose products are not."""
    K = 32
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, K // 16))
    scale = np.arange(256, dtype=np.uint8)[:, None].copy()
    q = X.pack(torch.from_numpy(MX.pack4(codes)).to(dev), torch.from_numpy(scale).to(dev))
    y = X.embedding(torch.arange(256, device=dev), q, mult).cpu()
    v = torch.from_numpy(MX.values(codes, scale, "e2m1")) * float(np.float32(mult))
    want = v.float().bfloat16()
    assert torch.equal(y.isnan(), want.isnan()) and want[255].isnan().all()
    assert torch.equal(y.nan_to_num(0), want.nan_to_num(0))


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M", [1, 6, 12, 20, 40])
def test_products_under_every_pair_of_scales(dev, M, elem):
    """One element of a row against weights of every scale code: a product of two values is exact, in bf16 too, from 2^-126 up to
    the largest bf16 value and is infinite above it; below 2^-126 it is off by less than that at most."""
    K = 32
    g = np.random.default_rng(5)
    codes = g.integers(0, 16, (255, K)).astype(np.uint8)
    scale = np.arange(255, dtype=np.uint8)[:, None].copy()
    q = X.pack(torch.from_numpy(MX.pack4(codes)).to(dev), torch.from_numpy(scale).to(dev))
    wv = MX.values(codes, scale, "e2m1")
    for start in range(-126, 121, M):
        x = torch.zeros(M, K)
        for m in range(M):
            x[m, (7 * m + start) % K] = 1.5 * 2.0 ** min(start + m, 121) * (-1) ** m
        x = x.bfloat16()
        with np.errstate(over="ignore"):
            want = torch.from_numpy(rounded(x, elem) @ wv.T).float().bfloat16().double().numpy()
        for src in (x.to(dev), X.quant_rows(x.to(dev), elem)):
            y = X.linear_mxfp4(src, q, elem).double().cpu().numpy()
            with np.errstate(invalid="ignore"):  # (infinity less itself)
                bad = ~((y == want) | (np.abs(y - want) < 2.0 ** -126))
            assert not bad.any(), (start, np.argwhere(bad)[:4], y[bad][:4], want[bad][:4])

"""The bound on a product's outputs together (oracle/mx.py, norm_limit) holds for the arithmetic it was derived for and shows the mistakes
that a bound on each output lets through, planted in the oracle's product here."""

import numpy as np
import pytest
import torch

from oracle import mx as MX
from oracle.oracle import bf16_to_f32


def bits(t):
    return t.contiguous().view(torch.int16).numpy().view(np.uint16)


def operands(M, N, K, elem, seed=1):
    g = torch.Generator().manual_seed(seed)
    x, w = torch.randn(M, K, generator=g).bfloat16(), (torch.randn(N, K, generator=g) * 0.02).bfloat16()
    return MX.values(*MX.quantize(bits(x), elem), elem), MX.values(*MX.quantize(bits(w), "e2m1"), "e2m1")


def to_bf16(y):
    return torch.from_numpy(np.asarray(y, np.float32)).bfloat16().double().numpy()


def product(xv, wv, elem, acc=np.float32):
    """The instruction's way: 128 products at a time (with e4m3 rows each cut 13 bits below the largest of its block of 32), added to an
    accumulator of type `acc` ("bf16" as well)."""
    y = np.zeros((len(xv), len(wv)))
    for k in range(0, xv.shape[1], 128):
        p = xv[:, None, k:k + 128] * wv[None, :, k:k + 128]
        if elem == "e4m3":
            b = p.reshape(*p.shape[:2], -1, 32)
            u = np.exp2(np.frexp(np.abs(b).max(-1, keepdims=True))[1] - 1.0 - 13)
            p = np.where(u > 0, np.trunc(b / np.where(u > 0, u, 1)) * u, 0).reshape(p.shape)
        y = y + p.sum(-1)
        y = to_bf16(y) if acc == "bf16" else y.astype(acc).astype(np.float64)
    return y


CASES = [(1, 64, 512), (5, 48, 2560), (7, 48, 9728), (3, 16, 16384)]


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", CASES)
def test_the_instructions_arithmetic_is_within(M, N, K, elem):
    xv, wv = operands(M, N, K, elem)
    y, ref = product(xv, wv, elem), xv @ wv.T
    assert np.linalg.norm(y - ref) <= MX.norm_limit(xv, wv, elem, 2.0 ** -24)
    assert np.linalg.norm(to_bf16(y) - ref) <= MX.norm_limit(xv, wv, elem, 2.0 ** -8)


@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
@pytest.mark.parametrize("M,N,K", CASES)
def test_mistakes_are_not(M, N, K, elem):
    xv, wv = operands(M, N, K, elem)
    ref = xv @ wv.T
    off = lambda y: np.linalg.norm(y - ref)
    fp32, bf16 = (MX.norm_limit(xv, wv, elem, s) for s in (2.0 ** -24, 2.0 ** -8))
    assert off(to_bf16(ref)) > fp32                                    # partials kept in bf16
    assert off(xv[:, :-4] @ wv[:, :-4].T) > bf16                       # the last four k left out
    one = xv.copy()
    one[:, K // 2 + 5] = 0
    assert off(one @ wv.T) > bf16                                      # one product of each sum lost
    if K >= 9728:
        assert off(product(xv, wv, elem, acc="bf16")) > bf16           # a running sum in bf16

"""Calls of the MXFP4 operators on the GPU beside those of test_gpu_mxfp4.py: rounded rows in the head, the borders of the
formats' ranges, launch shapes. Bounds of one element are test_gpu_mxfp4.py's."""

import numpy as np
import pytest
import torch

from kernels import lmhead
from kernels import mxfp4 as X
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

"""Beam search behind the lm head (HIP kernels k_beam_rows, k_beam_pick and k_beam_reorder of libkrq.so): the choice over
beams and vocabulary, and the states put in the chosen order. The counterpart of lmhead.lm_head_argmax for several
hypotheses per request (the reference decodes greedily): logits come from gemv(h, lm_head), linear_mxfp4,
lm_head_argmax(..., return_logits=True) or any head, with a grammar's or sampler's masks as -inf.

  scores, beams, tokens = beam.select(logits, scores)       # 2 W candidates of every request, best first
  ... finished hypotheses leave, W candidates stay ...
  beam.reorder([*k_caches, *v_caches], beams, dim=.., lengths=.., length_dim=..)

Both take device tensors alone, wait for nothing and can be captured.
"""

import functools
import math

import torch

from . import _lib as L
from . import mxfp4 as _mx

MAX_BEAMS, MAX_N, MAX_VOCAB, MAX_ROWS = 64, 64, 1 << 20, 65535
MAX_STATES = 64  # states of one launch


def _same_device(first, *tensors):
    L.require_device(first, *tensors)
    for t in tensors:
        if t is not None and t.get_device() != first.get_device():
            raise ValueError(f"tensors on {first.device} and {t.device}")


@functools.lru_cache(maxsize=4096)
def _ws_bytes(B, W, V, n, fp32):
    return L.lib().krq_beam_select_ws_bytes(B, W, V, n, fp32)


def select(logits, scores, n=None):
    """logits [B W, V] (or [B, W, V]) bf16 or fp32, scores [B, W] fp32 (sums of log probabilities so far) -> (scores [B, n]
    fp32, beams [B, n] int64, tokens [B, n] int64): the n (default 2 W) largest of
      scores[b, w] + log_softmax(logits[b, w])[t]
    over beams and tokens, best first; ties to the lower beam, then to the lower token. The log of the sum of exponentials is
    off by less than 2^-18 (fp32 terms; all behind them is fp64): a beam's candidates are in the order of its logits, those of
    two beams within 2^-17 of each other may come in either order, and beams of the same logits have the same sum. -inf logits
    are never preferred to others; a beam with nothing else, or with the score -inf (a first step's copies), has candidates of
    -inf. Mask with -inf: beside logits past 2^34, a type's lowest value among them, the log of the sum is below fp64's last place, so that
    a beam of nothing else counts its tokens as certain. A beam with a NaN or +inf among its logits, or as its score, has candidates
    of NaN, which count as the largest, as in lm_head_argmax. W and n up to 64, n <= W V, V up to 2^20, B W up to 65,535."""
    fp32 = logits.dtype is torch.float32
    shape = logits.shape
    if not (fp32 or logits.dtype is torch.bfloat16) or not 2 <= len(shape) <= 3:
        raise ValueError(f"logits must be bf16 or fp32 [B W, V] or [B, W, V], got {logits.dtype} {tuple(shape)}")
    if scores.dtype is not torch.float32 or scores.dim() != 2:
        raise ValueError(f"scores must be fp32 [B, W], got {scores.dtype} {tuple(scores.shape)}")
    dev = logits.get_device()
    if dev < 0 or scores.get_device() != dev:
        _same_device(logits, scores)
    B, W = scores.shape
    V = shape[-1]
    if shape[0] != (B * W if len(shape) == 2 else B) or (len(shape) == 3 and shape[1] != W):
        raise ValueError(f"logits {tuple(shape)} and scores {tuple(scores.shape)} do not match")
    n = 2 * W if n is None else int(n)
    if not 1 <= W <= MAX_BEAMS or not 1 <= V <= MAX_VOCAB or B * W > MAX_ROWS:
        raise ValueError(f"{B} x {W} beams, vocabulary {V}: at most {MAX_BEAMS} beams, {MAX_ROWS} rows, {MAX_VOCAB} tokens")
    if not 1 <= n <= min(MAX_N, W * V):
        raise ValueError(f"n={n} (1 to {min(MAX_N, W * V)})")
    ld = V
    if not logits.is_contiguous():
        logits = logits.reshape(B * W, V)
        ld = logits.stride(0) if B * W > 1 else V
        if (V > 1 and logits.stride(1) != 1) or ld < V:
            logits, ld = logits.contiguous(), V
    if not scores.is_contiguous():
        scores = scores.contiguous()
    out_scores = scores.new_empty(B, n)
    beams = torch.empty_like(out_scores, dtype=torch.int64)
    tokens = torch.empty_like(beams)
    if B:
        nbytes = _ws_bytes(B, W, V, n, fp32)
        ws = scores.new_empty((nbytes + 3) // 4)
        _mx._call(dev, "krq_beam_select", logits.data_ptr(), fp32, ld, scores.data_ptr(), B, W, V, n, ws.data_ptr(), nbytes,
                  out_scores.data_ptr(), beams.data_ptr(), tokens.data_ptr())
    return out_scores, beams, tokens


def reorder(states, beams, dim=0, lengths=None, length_dim=None):
    """Put states in the order of the chosen beams, in place: row b W + w along `dim` of every state becomes what row
    b W + beams[b, w] was. states: a contiguous tensor of any type, or a list of them that do not overlap, with the same B W rows along dim; beams
    int64 or int32 [B, W] (the first W columns of what select gave, or the W that stayed; repeats are the rule). lengths int32 or int64
    [B] with length_dim (after dim): of each entry only the positions before its length move, those behind stay as they are.
    A beam outside [0, W) leaves its row as it is. Rows whose beam is their own are neither read nor written. One launch for every 64 states
    of a shape, behind a copy of beams where they are columns of a wider tensor. Returns states."""
    many = [states] if isinstance(states, torch.Tensor) else list(states)
    shape, dev = beams.shape, beams.get_device()
    if not (beams.dtype is torch.int64 or beams.dtype is torch.int32) or len(shape) != 2:
        raise ValueError(f"beams must be int64 or int32 [B, W], got {beams.dtype} {tuple(shape)}")
    if (lengths is None) != (length_dim is None):
        raise ValueError("lengths and length_dim go together")
    B, W = shape
    if W > MAX_BEAMS or B > 1 << 20:
        raise ValueError(f"{B} x {W} beams (at most {MAX_BEAMS} beams, 2^20 entries)")
    if dev < 0 or (lengths is not None and lengths.get_device() != dev):
        _same_device(beams, lengths)
    if lengths is not None:
        if not (lengths.dtype is torch.int64 or lengths.dtype is torch.int32) or lengths.shape != (B,):
            raise ValueError(f"lengths must be int64 or int32 [{B}], got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    beams = beams.contiguous()
    groups, spans = {}, []
    for t in many:
        if t.get_device() != dev:
            _same_device(beams, t)
        if not t.is_contiguous():
            raise ValueError(f"state {tuple(t.shape)} strides {t.stride()}: states are reordered in place and must be contiguous")
        size = t.element_size()
        geometry = _geometry(t.shape, size, B, W, dim, length_dim)
        size *= t.numel()
        if size:
            p = t.data_ptr()
            groups.setdefault(geometry, []).append(p)
            spans.append((p, size))
    if len(spans) > 1:
        spans.sort()
        for (a, size), (b, _) in zip(spans, spans[1:]):
            if a + size > b:
                raise ValueError("states overlap: each would be reordered more than once")
    for (outer, mid, S, size), ptrs in groups.items():
        for i in range(0, len(ptrs), MAX_STATES):
            part = ptrs[i:i + MAX_STATES]
            _mx._call(dev, "krq_beam_reorder", (L.ctypes.c_void_p * len(part))(*part), len(part), outer, B, W, mid, S, size, beams.data_ptr(),
                      beams.dtype is torch.int64, L.ptr(lengths), lengths is not None and lengths.dtype is torch.int64)
    return states


@functools.lru_cache(maxsize=4096)
def _geometry(shape, size, B, W, dim, length_dim):
    """(entries before the rows, between rows and positions, positions, bytes of a position) of a state of elements of `size` bytes."""
    d = dim + len(shape) if dim < 0 else dim
    s = len(shape) if length_dim is None else length_dim + len(shape) if length_dim < 0 else length_dim
    if not 0 <= d < len(shape) or shape[d] != B * W or (length_dim is not None and not d < s < len(shape)):
        raise ValueError(f"state {tuple(shape)}: {B} x {W} rows along dim={dim}, positions along length_dim={length_dim} after it")
    outer, mid = math.prod(shape[:d]), math.prod(shape[d + 1:s])
    if length_dim is None:
        return outer, 1, 1, mid * size
    return outer, mid, shape[s], math.prod(shape[s + 1:]) * size

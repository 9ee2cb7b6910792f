"""Beam search behind the lm head (HIP kernels k_beam_rows, k_beam_pick and k_beam_reorder of libkrq.so): the choice over
beams and vocabulary, and the states put in the chosen order. The counterpart of lmhead.lm_head_argmax for several
hypotheses per request (the reference decodes greedily): logits come from gemv(h, lm_head), linear_mxfp4,
lm_head_argmax(..., return_logits=True) or any head, with a grammar's or sampler's masks as -inf.

  scores, beams, tokens = beam.select(logits, scores)       # 2 W candidates of every request, best first
  ... finished hypotheses leave, W candidates stay ...
  beam.reorder([*k_caches, *v_caches], beams, dim=.., lengths=.., length_dim=..)

Both take device tensors alone, wait for nothing and can be captured.
"""

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


def select(logits, scores, n=None):
    """logits [B W, V] (or [B, W, V]) bf16 or fp32, scores [B, W] fp32 (sums of log probabilities so far) -> (scores [B, n]
    fp32, beams [B, n] int64, tokens [B, n] int64): the n (default 2 W) largest of
      scores[b, w] + log_softmax(logits[b, w])[t]
    over beams and tokens, best first, compared in fp64; ties to the lower beam, then to the lower token. -inf logits are
    never preferred to others; a beam with nothing else, or with the score -inf (a first step's copies), has candidates of -inf. A beam with
    a NaN or +inf among its logits, or as its score, has candidates of NaN, which count as the largest, as in lm_head_argmax. W and n up to
    64, n <= W V, V up to 2^20, B W up to 65,535."""
    if logits.dtype not in (torch.bfloat16, torch.float32) or logits.dim() not in (2, 3):
        raise ValueError(f"logits must be bf16 or fp32 [B W, V] or [B, W, V], got {logits.dtype} {tuple(logits.shape)}")
    if scores.dtype is not torch.float32 or scores.dim() != 2:
        raise ValueError(f"scores must be fp32 [B, W], got {scores.dtype} {tuple(scores.shape)}")
    _same_device(logits, scores)
    B, W = scores.shape
    V = logits.shape[-1]
    if tuple(logits.shape[:-1]) not in ((B * W,), (B, W)):
        raise ValueError(f"logits {tuple(logits.shape)} and scores {tuple(scores.shape)} do not match")
    n = 2 * W if n is None else int(n)
    if not 1 <= W <= MAX_BEAMS or not 1 <= V <= MAX_VOCAB or B * W > MAX_ROWS:
        raise ValueError(f"{B} x {W} beams, vocabulary {V}: at most {MAX_BEAMS} beams, {MAX_ROWS} rows, {MAX_VOCAB} tokens")
    if not 1 <= n <= min(MAX_N, W * V):
        raise ValueError(f"n={n} (1 to {min(MAX_N, W * V)})")
    if logits.dim() == 3:
        logits = logits.reshape(B * W, V)
    ld = logits.stride(0) if B * W > 1 else V
    if (V > 1 and logits.stride(1) != 1) or ld < V:
        logits, ld = logits.contiguous(), V
    scores = scores.contiguous()
    out_scores = torch.empty((B, n), device=logits.device, dtype=torch.float32)
    out = torch.empty((2, B, n), device=logits.device, dtype=torch.int64)
    if B:
        fp32 = logits.dtype is torch.float32
        nbytes = L.lib().krq_beam_select_ws_bytes(B, W, V, n, fp32)
        ws = torch.empty((nbytes,), device=logits.device, dtype=torch.uint8)
        _mx._call(logits.get_device(), "krq_beam_select", logits.data_ptr(), fp32, ld, scores.data_ptr(), B, W, V, n, ws.data_ptr(), nbytes,
                  out_scores.data_ptr(), out[0].data_ptr(), out[1].data_ptr())
    return out_scores, out[0], out[1]


def reorder(states, beams, dim=0, lengths=None, length_dim=None):
    """Put states in the order of the chosen beams, in place: row b W + w along `dim` of every state becomes what row
    b W + beams[b, w] was. states: a contiguous tensor of any type, or a list of them that do not overlap, with the same B W rows along dim; beams
    int64 or int32 [B, W] (the first W columns of what select gave, or the W that stayed; repeats are the rule). lengths int32 or int64
    [B] with length_dim (after dim): of each entry only the positions before its length move, those behind stay as they are.
    A beam outside [0, W) leaves its row as it is. Rows whose beam is their own are neither read nor written. One launch for all states
    of a shape (of up to 64). Returns states."""
    many = [states] if isinstance(states, torch.Tensor) else list(states)
    if beams.dtype not in (torch.int64, torch.int32) or beams.dim() != 2:
        raise ValueError(f"beams must be int64 or int32 [B, W], got {beams.dtype} {tuple(beams.shape)}")
    if (lengths is None) != (length_dim is None):
        raise ValueError("lengths and length_dim go together")
    _same_device(beams, lengths, *many)
    B, W = beams.shape
    if W > MAX_BEAMS or B > 1 << 20:
        raise ValueError(f"{B} x {W} beams (at most {MAX_BEAMS} beams, 2^20 entries)")
    if lengths is not None and (lengths.dtype not in (torch.int64, torch.int32) or tuple(lengths.shape) != (B,)):
        raise ValueError(f"lengths must be int64 or int32 [{B}], got {lengths.dtype} {tuple(lengths.shape)}")
    groups, spans = {}, []
    for t in many:
        d = dim + t.dim() if dim < 0 else dim
        s = t.dim() if length_dim is None else length_dim + t.dim() if length_dim < 0 else length_dim
        if not 0 <= d < t.dim() or t.shape[d] != B * W or (length_dim is not None and not d < s < t.dim()):
            raise ValueError(f"state {tuple(t.shape)}: {B} x {W} rows along dim={dim}, positions along length_dim={length_dim} after it")
        if not t.is_contiguous():
            raise ValueError(f"state {tuple(t.shape)} strides {t.stride()}: states are reordered in place and must be contiguous")
        if t.numel() == 0:
            continue
        outer = mid = 1
        for k in t.shape[:d]:
            outer *= k
        for k in t.shape[d + 1:s]:
            mid *= k
        if length_dim is None:
            outer, mid, S, size = outer, 1, 1, mid * t.element_size()
        else:
            S, size = t.shape[s], t.element_size()
            for k in t.shape[s + 1:]:
                size *= k
        groups.setdefault((outer, mid, S, size), []).append(t.data_ptr())
        spans.append((t.data_ptr(), t.numel() * t.element_size()))
    spans.sort()
    for (a, size), (b, _) in zip(spans, spans[1:]):
        if a + size > b:
            raise ValueError("states overlap: each would be reordered more than once")
    beams = beams.contiguous()
    lengths = lengths if lengths is None else lengths.contiguous()
    for (outer, mid, S, size), ptrs in groups.items():
        for i in range(0, len(ptrs), MAX_STATES):
            part = ptrs[i:i + MAX_STATES]
            _mx._call(beams.get_device(), "krq_beam_reorder", (L.ctypes.c_void_p * len(part))(*part), len(part), outer, B, W, mid, S, size,
                      beams.data_ptr(), beams.dtype is torch.int64, L.ptr(lengths), lengths is not None and lengths.dtype is torch.int64)
    return states

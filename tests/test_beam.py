"""Calls of kernels.beam and its entry points that end before anything is launched, without a GPU."""

import ctypes

import pytest
import torch

from kernels import _lib as L
from kernels import beam, mxfp4

BF = torch.bfloat16


class OnDevice(torch.Tensor):
    """A host tensor that the checks take for one on device `dev`."""

    dev = 0

    @property
    def is_cuda(self):
        return True

    def get_device(self):
        return self.dev


def on(t, dev=0):
    t = t.as_subclass(OnDevice)
    t.dev = dev
    return t


@pytest.fixture
def launched(monkeypatch):
    seen = []
    monkeypatch.setattr(mxfp4, "_call", lambda dev, name, *args: seen.append((dev, name, args)))
    return seen


def test_select_refuses(launched):
    l, s = torch.zeros(6, 50, dtype=BF), torch.zeros(2, 3)
    for a, b in ((l, on(s)), (on(l), s)):
        with pytest.raises(RuntimeError, match="ROCm device"):
            beam.select(a, b)
    with pytest.raises(ValueError, match="tensors on"):
        beam.select(on(l), on(s, 1))
    for a, b, n, match in [
        (l.half(), s, None, "logits must be"), (l[0], s, None, "logits must be"), (l, s.double(), None, "scores must be"),
        (l, s[0], None, "scores must be"), (l[:5], s, None, "do not match"), (l.view(3, 2, 50), s, None, "do not match"),
        (l, s, 0, "n=0"), (l, s, -1, "n=-1"), (l, s, 65, "n=65"), (l[:, :2], s, 7, "n=7"), (torch.zeros(65, 9), torch.zeros(1, 65), 4, "at most"),
        (torch.zeros(6, 0), s, None, "at most"), (torch.zeros(2, (1 << 20) + 1, dtype=BF), torch.zeros(1, 2), None, "at most"),
        (torch.zeros(65536, 1), torch.zeros(65536, 1), 1, "at most"), (torch.zeros(0, 9), torch.zeros(3, 0), None, "at most"),
    ]:
        with pytest.raises(ValueError, match=match):
            beam.select(on(a), on(b), n)
    assert not launched


def test_reorder_refuses(launched):
    s, b, n = torch.zeros(2, 6, 4, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm device"):
        beam.reorder(s, on(b), 1)
    with pytest.raises(RuntimeError, match="ROCm device"):
        beam.reorder(on(s), on(b), 1, n, 2)
    with pytest.raises(ValueError, match="tensors on"):
        beam.reorder([on(s), on(s, 1)], on(b), 1)
    for state, beams, args, match in [
        (s, b.float(), (1,), "beams must be"), (s, b[0], (1,), "beams must be"), (s, b, (1, n), "go together"), (s, b, (1, None, 2), "go together"),
        (s, b, (1, n.float(), 2), "lengths must be"), (s, b, (1, n[:1], 2), "lengths must be"), (s, b, (0,), "rows along"), (s, b, (4,), "rows along"),
        (s, b, (-5,), "rows along"), (s, b, (1, n, 1), "rows along"), (s, b, (1, n, 0), "rows along"), (s, b, (1, n, 4), "rows along"),
        (s[..., ::2], b, (1,), "contiguous"), (s.transpose(2, 3), b, (1,), "contiguous"),
        (torch.zeros(65, 2), torch.zeros(1, 65, dtype=torch.int64), (0,), "at most"),
    ]:
        with pytest.raises(ValueError, match=match):
            beam.reorder(on(state), on(beams), *(on(a) if isinstance(a, torch.Tensor) else a for a in args))
    for many in ([s, s], [s[:1], s[:1]], [s, s[1:]], [s[1:], s]):
        with pytest.raises(ValueError, match="overlap"):
            beam.reorder([on(t) for t in many], on(b), 1)
    assert not launched
    beam.reorder([on(s[:1]), on(s[1:])], on(b), 1)  # (side by side is no overlap)
    assert len(launched) == 1


def test_entry_points_refuse():
    lib, p = L.lib(), ctypes.c_void_p(4096)  # (never dereferenced: the checks end the call first)

    def select(logits=p, fp32=0, ld=50, scores=p, B=2, W=3, V=50, n=6, ws=p, nbytes=1 << 30, s=p, b=p, t=p):
        return lib.krq_beam_select(logits, fp32, ld, scores, B, W, V, n, ws, nbytes, s, b, t, None)

    bad = [dict([(k, None)]) for k in ("logits", "scores", "ws", "s", "b", "t")]
    bad += [dict(B=0), dict(W=0), dict(W=65), dict(V=0), dict(V=(1 << 20) + 1, ld=1 << 21), dict(n=0), dict(n=65), dict(V=1, n=4), dict(ld=49),
            dict(B=1 << 16), dict(logits=ctypes.c_void_p(4097)), dict(fp32=1, logits=ctypes.c_void_p(4098)), dict(ws=ctypes.c_void_p(4104)),
            dict(nbytes=lib.krq_beam_select_ws_bytes(2, 3, 50, 6, 0) - 1)]
    for kw in bad:
        assert select(**kw) == L.KRQ_EINVAL, kw
        assert b"beam_select" in lib.krq_last_error(), kw
    assert lib.krq_beam_select_ws_bytes(0, 3, 50, 6, 0) == -1 and lib.krq_beam_select_ws_bytes(2, 3, 50, 151, 0) == -1

    def reorder(states=(4096,), count=None, outer=1, B=2, W=3, mid=1, S=1, size=16, beams=p):
        states = (ctypes.c_void_p * max(1, len(states)))(*states)
        return lib.krq_beam_reorder(states, len(states) if count is None else count, outer, B, W, mid, S, size, beams, 1, None, 0, None)

    for kw in [dict(count=0), dict(states=[4096] * 65), dict(states=[None]), dict(beams=None), dict(outer=0), dict(B=0), dict(W=0), dict(W=65),
               dict(mid=0), dict(S=0), dict(size=0), dict(B=(1 << 20) + 1), dict(outer=1 << 20, mid=1 << 20)]:
        assert reorder(**kw) == L.KRQ_EINVAL, kw
        assert b"beam_reorder" in lib.krq_last_error(), kw


def test_more_threads_than_a_launch_has():
    lib, p = L.lib(), ctypes.c_void_p(4096)
    states = (ctypes.c_void_p * 1)(4096)
    for outer, S, size in ((1, 1 << 32, 1), (1 << 10, 1 << 22, 1), (1 << 24, 1, 16), (1, 1 << 36, 16), (1, 1 << 40, 1 << 40)):
        assert lib.krq_beam_reorder(states, 1, outer, 1, 2, 1, S, size, p, 1, None, 0, None) == L.KRQ_EINVAL
        assert b"beam_reorder" in lib.krq_last_error()

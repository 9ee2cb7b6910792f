"""Calls of kernels.lora and krq_lora_add that end before anything is launched, without a GPU."""

import copy
import ctypes
import pickle

import pytest
import torch

from kernels import _lib as L
from kernels import lora, mxfp4

BF = torch.bfloat16


class OnDevice:
    """A stand-in for a tensor on device `dev`, as far as the checks look at one."""

    def __init__(self, t, dev=0):
        self.t, self.dev, self.device, self.is_cuda = t, dev, torch.device("cpu"), True

    def get_device(self):
        return self.dev

    def contiguous(self):
        return self

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.fixture
def launched(monkeypatch):
    seen = []
    monkeypatch.setattr(mxfp4, "_call", lambda dev, name, *args: seen.append((dev, name, args)))
    return seen


def bank():
    ad = lora.Adapters(64, (48, 16), 8, 4, "cpu")
    ad.a = OnDevice(ad.a)
    return ad


def operands(M=3, ydtype=BF):
    return [OnDevice(torch.zeros(M, 64, dtype=ydtype)), OnDevice(torch.zeros(M, 64, dtype=BF)), bank(),
            OnDevice(torch.zeros(M, dtype=torch.int32))]


def test_host_tensors_are_refused(launched):
    for i in (0, 1, 3):
        a = operands()
        a[i] = a[i].t
        with pytest.raises(RuntimeError, match="ROCm device"):
            lora.add(*a)
    assert not launched


def test_other_devices_are_refused(launched):
    for i in (0, 1, 3):
        a = operands()
        a[i].dev = 1
        with pytest.raises(ValueError, match="tensors on"):
            lora.add(*a)
    a = operands()
    a[2].a.dev = 1
    with pytest.raises(ValueError, match="tensors on"):
        lora.add(*a)
    assert not launched


@pytest.mark.parametrize("i,t,match", [
    (0, torch.zeros(3, 63, dtype=BF), "y must be"),
    (0, torch.zeros(3, 64, dtype=torch.float16), "y must be"),
    (0, torch.zeros(2, 64, dtype=BF), "do not match"),
    (0, torch.zeros(1, 3, 64, dtype=BF), "y must be"),
    (1, torch.zeros(3, 32, dtype=BF), "x must be"),
    (1, torch.zeros(3, 64), "x must be"),
    (3, torch.zeros(2, dtype=torch.int32), "do not match"),
    (3, torch.zeros(3, 1, dtype=torch.int32), "do not match"),
    (3, torch.zeros(3, dtype=torch.int16), "do not match"),
])
def test_shapes_and_types(launched, i, t, match):
    a = operands()
    a[i] = OnDevice(t)
    with pytest.raises(ValueError, match=match):
        lora.add(*a)
    assert not launched


def test_out(launched):
    a = operands()
    for bad in (torch.zeros(3, 64), torch.zeros(4, 64, dtype=BF), torch.zeros(64, 3, dtype=BF).t(), torch.zeros(3, 63, dtype=BF)):
        with pytest.raises(ValueError, match="out must be"):
            lora.add(*a, out=OnDevice(bad))
    room = torch.zeros(4 * 64, dtype=BF)
    a[0] = OnDevice(room[:192].view(3, 64))
    with pytest.raises(ValueError, match="overlaps"):
        lora.add(*a, out=OnDevice(room[64:].view(3, 64)))
    with pytest.raises(ValueError, match="overlaps"):
        lora.add(*a, out=a[1])
    a[0] = OnDevice(torch.zeros(64, 3, dtype=BF).t())
    with pytest.raises(ValueError, match="out must be|in place"):
        lora.add(*a, out=a[0])
    assert not launched


@pytest.mark.parametrize("args", [(8, 4, 4, 1), (40, 4, 4, 1), (0, 4, 4, 1), (64, [], 4, 1), (64, [1] * 9, 4, 1), (64, [4, 0], 4, 1), (64, 4, 0, 1),
                                  (64, 4, 257, 1), (64, 4, 4, 0)])
def test_banks_that_cannot_be(args):
    with pytest.raises(ValueError):
        lora.Adapters(*args, "cpu")


def test_load_checks_its_pairs():
    ad = lora.Adapters(64, (48, 16), 20, 4, "cpu")
    assert ad.rank == 32 and ad.a.shape == (4, 2, 2, 1, 2, 4, 16, 8) and ad.b.shape == (4, 64 * 32)

    def pair(r, n=48, K=64, rb=None):
        return torch.ones(r, K), torch.ones(n, rb or r)

    for slot in (-1, 4):
        with pytest.raises(ValueError, match="slot"):
            ad.load(slot, [None, None])
        with pytest.raises(ValueError, match="slot"):
            ad.clear(slot)
    for pairs in ([pair(4)], [pair(4), pair(4, 16), pair(4)], pair(4)[:1]):
        with pytest.raises(ValueError, match="pairs for 2 parts"):
            ad.load(0, pairs)
    for p in (pair(4, K=32), pair(4, n=47), pair(4, rb=5)):
        with pytest.raises(ValueError, match="do not match"):
            ad.load(0, [p, None])
    with pytest.raises(ValueError, match="rank 33"):
        ad.load(0, [pair(33), None])
    assert not ad.ranks.any() and not ad.a.any()


def test_load_packs_a_slot():
    ad = lora.Adapters(32, (3, 2), 40, 2, "cpu")
    g = torch.Generator().manual_seed(0)
    a0, b0, a1, b1 = (torch.randn(*s, generator=g).to(BF) for s in ((17, 32), (3, 17), (5, 32), (2, 5)))
    ad.load(1, [(torch.randn(40, 32), torch.randn(3, 40)), None], 1.0)
    ad.load(1, [(a0, b0), (a1, b1)], 0.5)
    assert ad.ranks.tolist() == [0, 17] and ad.scales.tolist() == [0.0, 0.5]
    want = torch.zeros(2, 32, 64, dtype=BF)  # (tiles past the slot's rank are not read)
    want[0, :17, :32], want[1, :5, :32] = a0, a1
    got = ad.a[1, :, :2].permute(0, 1, 5, 2, 4, 3, 6).reshape(2, 32, 64)  # [part, rank tile, j | step, g, e, 8]
    assert torch.equal(got, want)
    for part, (b, n) in enumerate(((b0, 3), (b1, 2))):  # a tile of 16 columns each: [g, j, 8] of 32 ranks
        want = torch.zeros(16, 32, dtype=BF)
        want[:n, :b.shape[1]] = b
        assert torch.equal(ad.b[1].view(-1)[part * 512:(part + 1) * 512].view(4, 16, 8).permute(1, 0, 2).reshape(16, 32), want)
    ad = lora.Adapters(32, 35, 40, 1, "cpu")  # three tiles; 32 ranks and 16 more
    b0 = torch.randn(35, 40, generator=g).to(BF)
    ad.load(0, (torch.randn(40, 32), b0))
    t = ad.b[0, :3 * 16 * 48].view(3, 16 * 48)
    got = torch.cat([t[:, :512].view(3, 4, 16, 8).permute(0, 2, 1, 3).reshape(48, 32), t[:, 512:].view(3, 2, 16, 8).permute(0, 2, 1, 3).reshape(48, 16)], 1)
    want = torch.zeros(48, 48, dtype=BF)
    want[:35, :40] = b0
    assert torch.equal(got, want)


def test_clear():
    ad = lora.Adapters(32, (3, 2), 40, 2, "cpu")
    ad.load(1, [(torch.randn(17, 32), torch.randn(3, 17)), None])
    ad.clear(1)
    assert ad.ranks.tolist() == [0, 0]


def test_load_without_pairs_empties_a_slot():
    ad = lora.Adapters(32, (3, 2), 40, 2, "cpu")
    ad.load(1, [(torch.randn(17, 32), torch.randn(3, 17)), None])
    ad.load(1, [None, None])
    assert ad.ranks.tolist() == [0, 0]


def test_a_bank_can_be_copied():
    ad = lora.Adapters(32, (3, 2), 40, 2, "cpu")
    ad.load(1, [(torch.randn(17, 32), torch.randn(3, 17)), None], 0.25)
    for other in (copy.deepcopy(ad), pickle.loads(pickle.dumps(ad))):
        assert other.parts == ad.parts and list(other._n) == [3, 2] and other.ranks.tolist() == [0, 17]
        assert torch.equal(other.a, ad.a) and torch.equal(other.b, ad.b) and other.a.data_ptr() != ad.a.data_ptr()


def test_entry_point_refuses():
    lib, p = L.lib(), ctypes.c_void_p(4096)  # (never dereferenced: the checks end the call first)

    def call(x=p, ldx=64, ids=p, a=p, b=p, ranks=p, scales=p, slots=4, M=3, K=64, n=(48, 16), parts=2, rank=16, y=p, ldy=64, out=p,
             ldo=64, fp32=0, ws=p, nbytes=1 << 20):
        n = (ctypes.c_int64 * len(n))(*n)
        return lib.krq_lora_add(x, ldx, ids, 0, a, b, ranks, scales, slots, M, K, n, parts, rank, y, ldy, out, ldo, fp32, ws, nbytes, None)

    odd, q = ctypes.c_void_p(4097), ctypes.c_void_p(8200)
    bad = [dict([(k, None)]) for k in ("x", "ids", "a", "b", "ranks", "scales", "y", "out", "ws")]
    bad += [dict(M=0), dict(M=1 << 25), dict(K=8), dict(K=72), dict(K=1 << 25), dict(parts=0), dict(n=(1,) * 9, parts=9), dict(n=(48, 0)),
            dict(rank=0), dict(rank=8), dict(rank=272), dict(slots=0), dict(slots=1 << 23), dict(ldx=32), dict(ldx=68), dict(x=q), dict(a=q),
            dict(b=q), dict(ws=q), dict(ldy=63), dict(ldo=63), dict(y=odd), dict(out=odd), dict(y=q, fp32=1, out=ctypes.c_void_p(4098)),
            dict(ldy=72), dict(nbytes=3 * 2 * 16 * 4 - 1)]
    for kw in bad:
        assert call(**kw) == L.KRQ_EINVAL, kw
        assert b"lora_add" in lib.krq_last_error(), kw
    assert lib.krq_lora_ws_bytes(3, 64, 2, 16) >= 3 * 2 * 16 * 4
    for args in ((0, 64, 2, 16), (3, 8, 2, 16), (3, 64, 0, 16), (3, 64, 9, 16), (3, 64, 2, 8), (3, 64, 2, 300)):
        assert lib.krq_lora_ws_bytes(*args) == -1


def test_more_threads_than_a_launch_has():
    lib, p = L.lib(), ctypes.c_void_p(4096)
    for M, N, fp32 in ((48, 1 << 27, 0), (384, 1 << 24, 1), (1 << 24, 1 << 14, 0), (1 << 22, 1 << 15, 1)):
        n = (ctypes.c_int64 * 8)(*[N // 8] * 8)
        assert lib.krq_lora_add(p, 64, p, 0, p, p, p, p, 4, M, 64, n, 8, 16, p, N, p, N, fp32, p, 1 << 50, None) == L.KRQ_EINVAL
        assert b"too large" in lib.krq_last_error()


def test_ranks_of_parts():
    ad = lora.Adapters(32, (3, 2), 40, 2, "cpu")
    ad.load(1, [(torch.randn(17, 32), torch.randn(3, 17)), None])
    assert ad.ranks.tolist() == [0, 17] and ad.part_ranks.tolist() == [[0, 0], [17, 0]]
    ad.load(1, [(torch.randn(4, 32), torch.randn(3, 4)), (torch.randn(40, 32), torch.randn(2, 40))])
    assert ad.ranks.tolist() == [0, 40] and ad.part_ranks.tolist() == [[0, 0], [4, 40]]
    ad.load(1, [None, None])
    assert ad.ranks.tolist() == [0, 0] and ad.part_ranks.tolist() == [[0, 0], [0, 0]]
    ad.load(0, [None, (torch.randn(5, 32), torch.randn(2, 5))])
    ad.clear(0)
    assert not ad.ranks.any() and not ad.part_ranks.any()
    state = {k: v for k, v in ad.__getstate__().items() if k != "part_ranks"}  # a bank saved with a rank for each slot only
    old = lora.Adapters.__new__(lora.Adapters)
    old.__setstate__({**state, "ranks": torch.tensor([0, 17], dtype=torch.int32)})
    assert old.part_ranks.tolist() == [[0, 0], [17, 17]] and old.part_ranks.dtype is torch.int32


def test_entry_point_of_parts_refuses():
    lib, p = L.lib(), ctypes.c_void_p(4096)
    n = (ctypes.c_int64 * 2)(48, 16)

    def call(ranks=p, part_ranks=p, M=3):
        return lib.krq_lora_add_parts(p, 64, p, 0, p, p, ranks, part_ranks, p, 4, M, 64, n, 2, 16, p, 64, p, 64, 0, p, 1 << 20, None)

    for kw in (dict(ranks=None), dict(part_ranks=None), dict(M=0)):
        assert call(**kw) == L.KRQ_EINVAL, kw
        assert b"lora_add" in lib.krq_last_error(), kw

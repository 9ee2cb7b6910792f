"""Calls of kernels.mxfp4 that end before anything is launched, without a GPU: the library's entry points are
replaced by a list of what would have been called."""

import copy
import io
import pickle

import pytest
import torch

from kernels import _lib as L
from kernels import lmhead
from kernels import mxfp4 as X
from kernels.mlp import PersistentMLP


def u8(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


def weight(N=64, K=64):
    """An MXFP4Weight of zeros in host memory."""
    return X.MXFP4Weight(u8(N, K // 2), u8(N, K // 32), u8(L.lib().krq_mx_tiled_bytes(N, K, 0)), u8(L.lib().krq_mx_scale_bytes(N, K)))


def rows(M=4, K=64, elem="e4m3"):
    """MXRows of zeros in host memory."""
    at, size = X._rows_bytes(M, K, X.ELEMS[elem])
    return X.MXRows(u8(size), at, (M, K), elem)


@pytest.fixture
def launched(monkeypatch):
    seen = []
    monkeypatch.setattr(X, "_call", lambda dev, name, *args: seen.append((dev, name, args)))
    return seen


class OnDevice:
    """A stand-in for a tensor on device `dev`, as far as the checks look at one."""

    def __init__(self, t, dev):
        self.t, self.dev, self.device, self.is_cuda = t, dev, f"cuda:{dev}", True

    def get_device(self):
        return self.dev

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.mark.parametrize("call", [
    lambda q, r: X.dequantize(q),
    lambda q, r: X.dequantize(r),
    lambda q, r: X.gemv_mxfp4(r, q),
    lambda q, r: X.gemv_mxfp4(r, q, 2),
    lambda q, r: X.gemv_swiglu_mxfp4(r, q),
    lambda q, r: X.gemm_mxfp4(r, q),
    lambda q, r: X.linear_mxfp4(r, q),
    lambda q, r: X.embedding(torch.zeros(2, dtype=torch.int64), q),
])
def test_weights_and_rows_of_the_host_are_refused(launched, call):
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(weight(64, 1024), rows(4, 1024))
    assert not launched


@pytest.mark.parametrize("what", ["tiled", "tiled_scale"])
@pytest.mark.parametrize("where", ["host", "other"])
def test_every_part_of_a_weight_is_on_the_rows_device(launched, what, where):
    """A weight of which one tensor stayed behind, or went to another device."""
    q, r = weight(), rows()
    r.data = OnDevice(r.data, 0)
    for name in ("tiled", "tiled_scale"):
        t = getattr(q, name)
        if name != what:
            setattr(q, name, OnDevice(t, 0))
        elif where == "other":
            setattr(q, name, OnDevice(t, 1))
    err = RuntimeError if where == "host" else ValueError
    for call in (lambda: X.dequantize(q), lambda: X.linear_mxfp4(r, q), lambda: X.gemm_mxfp4(r, q), lambda: X.gemv_swiglu_mxfp4(r, q)):
        with pytest.raises(err, match="ROCm device|tensors on cuda"):
            call()
    assert not launched


@pytest.mark.parametrize("where", ["host", "other"])
def test_the_embeddings_scales_are_on_the_codes_device(launched, where):
    q, ids = weight(), torch.zeros(2, dtype=torch.int64)
    scale = q[1] if where == "host" else OnDevice(q[1], 1)
    moved = X.MXFP4Weight(OnDevice(q[0], 0), scale, q.tiled, q.tiled_scale)
    with pytest.raises(RuntimeError if where == "host" else ValueError, match="ROCm device|tensors on cuda"):
        X.embedding(OnDevice(ids, 0), moved)
    assert not launched


@pytest.mark.parametrize("M", [1, 32])
@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
def test_the_head_takes_rounded_rows(launched, M, elem):
    """MXRows reach the head's checks as every other product's: here those of where they lie and of how many they are."""
    with pytest.raises(RuntimeError, match="ROCm device"):
        lmhead.lm_head_argmax(rows(M, elem=elem), weight())
    with pytest.raises(ValueError, match="33 > 32"):
        lmhead.lm_head_argmax(rows(33, elem=elem), weight())
    with pytest.raises(ValueError, match="ActScale"):
        lmhead.lm_head_argmax(rows(M, elem=elem), weight(), a=object())
    with pytest.raises(ValueError, match="do not match"):
        lmhead.lm_head_argmax(rows(M, 96, elem), weight())
    assert not launched


def _saved(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)  # (written just above)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda q: pickle.loads(pickle.dumps(q)),
                                   lambda q: pickle.loads(pickle.dumps(q, protocol=2)), _saved,
                                   lambda q: copy.deepcopy({"layer": [q]})["layer"][0]])
def test_copies_and_pickles_of_a_weight(again):
    q = weight(17, 544)
    parts = (q[0], q[1], q.tiled, q.tiled_scale)
    for i, t in enumerate(parts):
        t.random_(256, generator=torch.Generator().manual_seed(i))
    p = again(q)
    assert type(p) is X.MXFP4Weight and len(p) == 2 and p.shape == (17, 544)
    for a, b in zip(parts, (p[0], p[1], p.tiled, p.tiled_scale)):
        assert torch.equal(a, b) and (a.data_ptr() == b.data_ptr()) == (again is copy.copy)


@pytest.mark.parametrize("K,split", [(64, 2), (1024, 3), (1024, 0), (1024, -1), (40960, 65), (1 << 20, 1 << 20)])
def test_a_split_without_groups_is_refused_before_its_output_is_made(monkeypatch, launched, K, split):
    """With a tensor on the device the partials would be allocated next: split [M, N] planes of them."""
    r, q = rows(4, K), weight(16, K)
    made = []
    data = OnDevice(r.data, 0)
    data.new_empty = lambda *a, **k: made.append(a)
    r.data, q.tiled, q.tiled_scale = data, OnDevice(q.tiled, 0), OnDevice(q.tiled_scale, 0)
    with pytest.raises(ValueError, match=f"split={split}"):
        X._decode(r, q, split, L.OUT_PARTIAL, "e4m3")
    assert not launched and not made


def test_the_mlp_refuses_a_split_before_its_first_launch(monkeypatch, launched):
    """I = 1,024 is two groups; split = 4 is one that FP8 weights take."""
    H, I = 512, 1024
    mlp = PersistentMLP(1, H, I, "cpu", split=4)
    monkeypatch.setattr(X, "gemv_swiglu_mxfp4", lambda *a: launched.append(a))
    monkeypatch.setattr("kernels.fp8._rows", lambda h: h)
    with pytest.raises(ValueError, match="split=4 of 2 groups"):
        mlp(torch.zeros(1, H, dtype=torch.bfloat16), weight(2 * I, H), weight(H, I))
    assert not launched and mlp.act is None


@pytest.mark.parametrize("M,V,K,asked", [(8, 151936, 2560, 0), (9, 151936, 2560, 0), (16, 16000, 3584, 0), (16, 15984, 2560, 1), (17, 151936, 2560, 1),
                                         (16, 151936, 3616, 1), (2, 16, 5152, 1), (1, 16, 10240, 0), (1, 16, 10272, 1)])
def test_the_head_asks_for_room_for_the_rows_only_where_they_are_rounded_before(M, V, K, asked):
    lib = L.lib()
    for e in (L.MX_E2M1, L.MX_E4M3):
        cands = lib.krq_lmhead_mxfp4_ws_bytes(L.MX_X_TILED, e, M, V, K)
        assert lib.krq_lmhead_mxfp4_ws_bytes(L.MX_X_BF16, e, M, V, K) - cands == asked * X._rows_bytes(M, K, e)[1]


def test_workspaces_are_the_librarys_at_every_size(monkeypatch):
    """The wrapper knows without a call which rows need no workspace, and most sizes of others: as the library says, everywhere."""
    sizes = []
    monkeypatch.setattr(X, "_call", lambda dev, name, *a: sizes.append(a[13]))
    lib = L.lib()
    for K in range(32, 12001, 32):
        q = weight(16, K)
        q.tiled, q.tiled_scale = OnDevice(q.tiled, 0), OnDevice(q.tiled_scale, 0)
        for M in (1, 2, 8, 9, 16, 17, 32):
            x = OnDevice(torch.empty((M, K), dtype=torch.bfloat16), 0)
            for split in {1, 2, 3, -(-K // 512)}:
                if split <= -(-K // 512):
                    X._decode(x, q, split, L.OUT_PARTIAL, "e4m3" if K % 64 else "e2m1")
                    assert sizes.pop() == lib.krq_gemv_mxfp4_ws_bytes(L.MX_X_BF16, int(K % 64 != 0), M, K, split), (M, K, split)


def test_parts_that_do_not_match_make_no_weight():
    """A weight's tiles and codes hold the bytes that its shape says the kernels read, when it is made and when they are replaced."""
    q = weight(17, 544)
    w4, scale, t, ts = q[0], q[1], q.tiled, q.tiled_scale
    for bad in ((w4[:16], scale, t, ts), (w4, scale[:, :16], t, ts), (w4, scale, t[:-1], ts), (w4, scale, t, ts[:256]), (w4, scale, ts, t),
                (w4, scale, t.view(torch.int16), ts), (w4, scale, t, ts.float()), (w4.int(), scale, t, ts), (w4.t().contiguous().t(), scale, t, ts),
                (w4[:1].expand(17, -1), scale, t, ts), (w4, scale, t[:1].expand(t.numel()), ts), (u8(0, 272), u8(0, 17), u8(0), u8(0)),
                (u8(17, 24), u8(17, 1), t, ts)):
        with pytest.raises(ValueError, match="MXFP4Weight"):
            X.MXFP4Weight(*bad)
    for name, value in (("tiled", t[:1024]), ("tiled", t.float()), ("tiled_scale", ts[:-4]), ("tiled_scale", t)):
        with pytest.raises(ValueError, match=name):
            setattr(q, name, value)
    assert q.tiled is t and q.tiled_scale is ts
    q.tiled, q.tiled_scale = t.clone(), ts.clone()

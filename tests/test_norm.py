"""Calls of kernels.norm and krq_add_rmsnorm that end before anything is launched, without a GPU."""

import ctypes

import pytest
import torch

from kernels import _lib as L
from kernels import mxfp4, norm

BF = torch.bfloat16


class OnDevice:
    """A stand-in for a tensor on device `dev`, as far as the checks look at one."""

    def __init__(self, t, dev=0):
        self.t, self.dev, self.device, self.is_cuda = t, dev, torch.device("cpu"), True

    def get_device(self):
        return self.dev

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.fixture
def launched(monkeypatch):
    seen = []
    monkeypatch.setattr(mxfp4, "_call", lambda dev, name, *args: seen.append((dev, name, args)))
    return seen


def x(M=4, K=64, dtype=BF):
    return torch.zeros(M, K, dtype=dtype)


def ln(K=64):
    return torch.zeros(K, dtype=BF)


@pytest.mark.parametrize("call", [norm.add_rmsnorm, norm.add_rmsnorm_fp8, norm.add_rmsnorm_mx])
def test_tensors_of_the_host_are_refused(launched, call):
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(x(), None, ln())
    with pytest.raises(RuntimeError, match="ROCm device"):
        call(OnDevice(x()), x(), OnDevice(ln()))
    assert not launched


@pytest.mark.parametrize("args,match", [
    ((x(dtype=torch.float32), None, ln()), "must be bf16"),
    ((torch.zeros(64, dtype=BF), None, ln()), "must be bf16"),
    ((x(4, 72), None, ln(72)), "multiple of 16"),
    ((x(4, 16400), None, ln(16400)), "multiple of 16 up to"),
    ((x(4, 0), None, ln(0)), "multiple of 16"),
    ((x(), None, ln(32)), "ln must be"),
    ((x(), x(5), ln()), "do not match"),
    ((x(), x(dtype=torch.float32), ln()), "must be bf16"),
    ((x(), torch.zeros(2, 4, 64, dtype=BF), ln()), "partials"),
    ((x(), torch.zeros(0, 4, 64), ln()), "0 partials"),
    ((x(), torch.zeros(65, 4, 64), ln()), "65 partials"),
])
def test_shapes_and_types(launched, args, match):
    args = [t if t is None else OnDevice(t) for t in args]
    with pytest.raises(ValueError, match=match):
        norm.add_rmsnorm(*args)
    assert not launched


def test_other_devices_are_refused(launched):
    for i in (1, 2):
        args = [OnDevice(x()), OnDevice(x()), OnDevice(ln())]
        args[i].dev = 1
        with pytest.raises(ValueError, match="tensors on"):
            norm.add_rmsnorm(*args)
    assert not launched


def test_res_out(launched):
    a = (OnDevice(x()), OnDevice(x()), OnDevice(ln()))
    for bad in (x(5), x(dtype=torch.float32), x(4, 128)[:, ::2]):
        with pytest.raises(ValueError, match="res_out"):
            norm.add_rmsnorm(*a, res_out=OnDevice(bad))
    with pytest.raises(ValueError, match="no new residual"):
        norm.add_rmsnorm(a[0], None, a[2], res_out=OnDevice(x()))
    room = torch.zeros(5, 64, dtype=BF)
    with pytest.raises(ValueError, match="overlaps"):
        norm.add_rmsnorm(OnDevice(room[:4]), a[1], a[2], res_out=OnDevice(room[1:]))
    assert not launched


def test_layouts_that_k_does_not_allow(launched):
    with pytest.raises(ValueError, match="tiled rows"):
        norm.add_rmsnorm_fp8(OnDevice(x(4, 80)), None, OnDevice(ln(80)), tiled=True)
    with pytest.raises(ValueError, match="MX blocks"):
        norm.add_rmsnorm_mx(OnDevice(x(4, 80)), None, OnDevice(ln(80)))
    with pytest.raises(ValueError, match="elem must be"):
        norm.add_rmsnorm_mx(OnDevice(x()), None, OnDevice(ln()), elem="e5m2")
    assert not launched


def test_entry_point_refuses():
    lib, p = L.lib(), ctypes.c_void_p(4096)  # (never dereferenced: the checks end the call first)

    def call(x=p, ldx=64, delta=p, split=0, ldd=64, part=0, ln=p, M=4, K=64, kind=0, inv=None, res=p, h=p, out=None, scale=None):
        return lib.krq_add_rmsnorm(x, ldx, delta, split, ldd, part, ln, 1e-6, M, K, kind, inv, res, h, out, scale, None)

    bad = [dict(x=None), dict(ln=None), dict(M=0), dict(M=-1), dict(K=8), dict(K=72), dict(K=16400), dict(kind=7), dict(kind=-1),
           dict(res=None), dict(split=-1), dict(split=65), dict(ldx=32), dict(ldx=68), dict(ldd=60), dict(ldd=66, split=2),
           dict(split=2, part=6), dict(x=ctypes.c_void_p(4104)), dict(h=ctypes.c_void_p(4100)), dict(h=None), dict(kind=1),
           dict(kind=1, out=p), dict(kind=3, out=p), dict(kind=2, out=p, scale=p, K=80, ldx=80, ldd=80),
           dict(kind=5, out=p, scale=p, K=80, ldx=80, ldd=80), dict(M=1 << 31)]
    for kw in bad:
        assert call(**kw) == L.KRQ_EINVAL, kw
        assert b"add_rmsnorm" in lib.krq_last_error(), kw


def test_more_threads_than_a_launch_has():
    lib, p = L.lib(), ctypes.c_void_p(4096)
    for M, K, split in ((1 << 23, 64, 2), (1 << 26, 64, 0), (1 << 22, 16384, 0)):
        assert lib.krq_add_rmsnorm(p, K, p, split, K, M * K, p, 1e-6, M, K, 0, None, p, p, None, None, None) == L.KRQ_EINVAL
        assert b"too many" in lib.krq_last_error()

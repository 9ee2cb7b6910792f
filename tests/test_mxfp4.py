"""MXFP4 without a GPU: the oracle against the format's definition, the host-side sizes, and every refusal
of the C entry points and of kernels.mxfp4 before anything runs."""

import ctypes

import numpy as np
import pytest
import torch

from kernels import _lib as L
from kernels import mxfp4 as X
from oracle import mx as MX


def bits(x):
    return x.to(torch.bfloat16).view(torch.int16).numpy().view(np.uint16)


def test_tables():
    assert MX.table("e2m1").tolist() == [0, .5, 1, 1.5, 2, 3, 4, 6]
    f8 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(MX.table("e4m3"), f8)


@pytest.mark.parametrize("elem", ["e2m1", "e4m3"])
def test_encode_is_nearest_even(elem):
    t = MX.table(elem)
    mid = (t[1:] + t[:-1]) / 2
    v = np.concatenate([t, mid, np.nextafter(mid, 0), np.nextafter(mid, 9e9), [1.5 * t[-1]], np.linspace(0, t[-1], 999)])
    for sign in (1, -1):
        got = MX.encode(sign * v, elem)
        for x, c in zip(v, got):
            i = c & (7 if elem == "e2m1" else 127)
            d = np.abs(t - min(x, t[-1]))
            best = np.flatnonzero(d == d.min())
            assert i in best and (len(best) == 1 or i % 2 == 0), (x, c)
            assert bool(c & (8 if elem == "e2m1" else 128)) == (sign < 0)


def test_e4m3_elements_match_torch():
    x = (torch.randn(64, 96, generator=torch.Generator().manual_seed(0)) * 3).bfloat16()
    q, c = MX.quantize(bits(x), "e4m3")
    s = torch.from_numpy(2.0 ** (c.astype(np.float64) - 127)).float().repeat_interleave(32, 1)
    ref = (x.float() / s).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(q, ref)


def test_quantize_known_answers():
    x = torch.zeros(1, 192)
    x[0, :4] = torch.tensor([6.0, -0.25, 0.75, 5.0])   # scale 1: 6, -0 (tie to even), 1 (tie), 4 (tie)
    x[0, 32:34] = torch.tensor([7.9, 7.0])             # amax below 8: scale 1, both clamp or round to 6
    x[0, 64:66] = torch.tensor([8.0, 1.0])             # scale 2: 4, 0.5
    x[0, 96] = float("inf")
    x[0, 128] = float("nan")
    x[0, 160] = 1e-39                                  # below the smallest scale's half step
    q, c = MX.quantize(bits(x), "e2m1")
    assert c[0].tolist() == [127, 127, 128, 255, 255, 0]
    assert q[0, :4].tolist() == [7, 8, 2, 6] and q[0, 32:34].tolist() == [7, 7] and q[0, 64:66].tolist() == [6, 1]
    assert not q[0, 96:160].any()
    v = MX.values(q, c, "e2m1")
    assert np.isnan(v[0, 96:160]).all() and v[0, 64] == 8 and v[0, 1] == 0


@pytest.mark.parametrize("elem,M,K", [("e2m1", 17, 160), ("e4m3", 17, 160), ("e2m1", 16, 512), ("e4m3", 3, 1056)])
def test_tile_layout(elem, M, K):
    g = np.random.default_rng(1)
    codes = g.integers(0, 16 if elem == "e2m1" else 256, (M, K)).astype(np.uint8)
    scale = g.integers(0, 256, (M, K // 32)).astype(np.uint8)
    t, s = MX.tile(codes, scale, elem)
    kt, ks = -(-K // 128), -(-K // 512)
    size = 1024 if elem == "e2m1" else 2048
    assert t.size == L.lib().krq_mx_tiled_bytes(M, K, X.ELEMS[elem]) and s.size == L.lib().krq_mx_scale_bytes(M, K)
    seen = np.zeros(t.size, int)
    for m in range(M):
        for k in range(K):
            base = ((m // 16) * kt + k // 128) * size
            kk, r = k % 128, m % 16
            if elem == "e2m1":
                at = base + (16 * (kk // 32) + r) * 16 + (kk % 32) // 2
                assert (t[at] >> (4 * (kk % 2))) & 15 == codes[m, k]
            else:
                at = base + 1024 * (kk // 64) + (16 * ((kk % 64) // 16) + r) * 16 + kk % 16
                assert t[at] == codes[m, k]
            seen[at] += 1
            assert s[(((m // 16) * ks + k // 512) * 64 + 16 * (kk // 32) + r) * 4 + (k % 512) // 128] == scale[m, k // 32]
    assert seen.max() <= (2 if elem == "e2m1" else 1) and not t[seen == 0].any()


def test_sizes_refuse_bad_arguments():
    lib = L.lib()
    assert lib.krq_mx_tiled_bytes(1, 32, 0) == 1024 and lib.krq_mx_tiled_bytes(17, 160, 1) == 2 * 2 * 2048
    assert lib.krq_mx_scale_bytes(17, 544) == 2 * 2 * 256
    for bad in ((0, 32, 0), (1, 0, 0), (1, 32, 2)):
        assert lib.krq_mx_tiled_bytes(*bad) == -1
    assert lib.krq_mx_scale_bytes(0, 32) == -1


def test_c_entry_points_refuse_before_any_launch():
    """Addresses that are never dereferenced: every call is refused by its checks."""
    p, odd, z = ctypes.c_void_p(4096), ctypes.c_void_p(4104), None

    def refuse(name, needle, *args):
        assert getattr(L.lib(), name)(*args) == L.KRQ_EINVAL
        assert needle in L.lib().krq_last_error(), L.lib().krq_last_error()

    refuse("krq_quant_mxfp4", b"null", z, 16, 64, 64, p, p, p, p, z)
    refuse("krq_quant_mxfp4", b"null", p, 16, 64, 64, p, p, p, z, z)
    refuse("krq_quant_mxfp4", b"multiple of 32", p, 16, 48, 48, p, p, p, p, z)
    refuse("krq_quant_mxfp4", b"0 x 64", p, 0, 64, 64, p, p, p, p, z)
    refuse("krq_quant_mxfp4", b"16 bytes", p, 16, 64, 60, p, p, p, p, z)
    refuse("krq_quant_mxfp4", b"16 bytes", odd, 16, 64, 64, p, p, p, p, z)
    refuse("krq_quant_mxfp4", b"too large", p, 1 << 40, 64, 64, p, p, p, p, z)
    refuse("krq_quant_mx_rows", b"element type", p, 16, 64, 64, 2, p, p, z)
    refuse("krq_quant_mx_rows", b"16 bytes", p, 16, 64, 68, 1, p, p, z)
    refuse("krq_quant_mx_rows", b"multiple of 32", p, 16, 0, 64, 1, p, p, z)
    refuse("krq_pack_mxfp4", b"16 bytes", odd, p, 16, 64, p, p, z)
    refuse("krq_pack_mxfp4", b"multiple of 32", p, p, 16, 65, p, p, z)
    refuse("krq_dequant_mx", b"element type", p, p, 5, 16, 64, p, z)
    refuse("krq_dequant_mx", b"16 bytes", p, p, 1, 16, 64, odd, z)
    refuse("krq_embed_mxfp4", b"indices", p, 1, 0, p, p, 16, 64, 1.0, p, z)
    refuse("krq_embed_mxfp4", b"indices", p, 1, 1 << 39, p, p, 16, 64, 1.0, p, z)
    refuse("krq_embed_mxfp4", b"multiple of 32", p, 1, 4, p, p, 16, 40, 1.0, p, z)
    gemv = lambda needle, x=p, xs=p, kind=1, elem=1, ld=0, w=p, M=4, N=64, K=1024, split=1, mode=0, ws=z, nb=0, out=p: refuse(
        "krq_gemv_mxfp4", needle, x, xs, kind, elem, ld, w, p, M, N, K, split, mode, ws, nb, out, z)
    gemv(b"null", x=z)
    gemv(b"null", out=z)
    gemv(b"element type", elem=3)
    gemv(b"x_kind", kind=2)
    gemv(b"outside 1..32", M=0)
    gemv(b"outside 1..32", M=33)
    gemv(b"multiple of 32", K=1000)
    gemv(b"N=0", N=0)
    gemv(b"their scales", xs=z)
    gemv(b"bf16 rows", kind=0, M=9, ld=1024)
    gemv(b"bf16 rows", kind=0, M=9, ld=1024, ws=p, nb=100)
    gemv(b"16 bytes", kind=0, ld=1000)
    gemv(b"16 bytes", kind=0, ld=1028)
    gemv(b"16 bytes", ws=odd)
    gemv(b"16 bytes", x=odd)
    gemv(b"16 bytes", w=odd)
    gemv(b"split=3 of 2", split=3, mode=1)
    gemv(b"split=0", split=0, mode=1)
    gemv(b"partials", split=2)
    gemv(b"I % 16", mode=2, N=48)
    gemv(b"bad mode", mode=3)
    gemm = lambda needle, x=p, xs=p, kind=1, elem=1, ld=1024, w=p, M=40, N=64, K=1024, ws=z, nb=0, out=p: refuse(
        "krq_gemm_mxfp4", needle, x, xs, kind, elem, ld, w, p, M, N, K, ws, nb, out, z)
    gemm(b"null", out=z)
    gemm(b"element type", elem=2)
    gemm(b"x_kind", kind=-1)
    gemm(b"their scales", xs=z)
    gemm(b"16 bytes", x=odd)
    gemm(b"16 bytes", ws=odd)
    gemm(b"multiple of 32", K=16)
    gemm(b"at most 2^22", K=(1 << 22) + 32)
    gemm(b"M=0", M=0)
    gemm(b"too large", M=0x3fffffff, N=0x3fffffff)
    head = lambda needle, V=1024, M=1, ws=p, nb=1 << 20, idx=p: refuse(
        "krq_lmhead_argmax_mxfp4", needle, p, z, 0, 1, 64, p, p, M, V, 64, z, ws, nb, idx, z)
    head(b"null", ws=z)
    head(b"null", idx=z)
    head(b"multiple of 16", V=1000)
    head(b"workspace", nb=8)
    head(b"workspace", M=33)
    lib = L.lib()
    assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, 8, 5120, 1) == lib.krq_gemv_mxfp4_ws_bytes(1, 1, 32, 64, 1) == 0
    assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, 9, 64, 1) == 2048 + 256 and lib.krq_gemv_mxfp4_ws_bytes(0, 0, 32, 64, 1) == 2 * 1024 + 512
    assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, 1, 10240, 1) == lib.krq_gemv_mxfp4_ws_bytes(0, 1, 8, 10240, 2) == 0
    assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, 2, 5152, 1) > 0
    assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, 1, 10272, 1) > 0 and lib.krq_gemv_mxfp4_ws_bytes(0, 1, 1, 64, 0) == -1
    assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, 33, 64, 1) == lib.krq_gemm_mxfp4_ws_bytes(0, 3, 40, 64, 64) == -1
    assert lib.krq_lmhead_mxfp4_ws_bytes(0, 1, 1, 1024, 64) == 768 and lib.krq_lmhead_mxfp4_ws_bytes(0, 1, 0, 1024, 64) == -1


def test_tiles_and_scales_off_their_alignment_are_refused():
    p, odd, z = ctypes.c_void_p(4096), ctypes.c_void_p(4100), None
    one_odd = lambda n: [[odd if i == j else p for i in range(n)] for j in range(n)]
    calls = [("krq_quant_mxfp4", [p, 16, 64, 64, w4, p, t, ts, z]) for w4, t, ts in one_odd(3)]
    calls += [("krq_quant_mx_rows", [p, 16, 64, 64, 1, t, ts, z]) for t, ts in one_odd(2)]
    calls += [("krq_pack_mxfp4", [w4, p, 16, 64, t, ts, z]) for w4, t, ts in one_odd(3)]
    calls += [("krq_dequant_mx", [t, ts, 1, 16, 64, out, z]) for t, ts, out in one_odd(3)]
    calls += [("krq_gemv_mxfp4", [x, xs, 1, 1, 0, w, ws, 4, 64, 1024, 1, 0, z, 0, p, z]) for x, xs, w, ws in one_odd(4)]
    calls += [("krq_gemm_mxfp4", [x, xs, 1, 1, 0, w, ws, 40, 64, 1024, z, 0, p, z]) for x, xs, w, ws in one_odd(4)]
    calls += [("krq_lmhead_argmax_mxfp4", [x, xs, 1, 1, 0, w, ws, 4, 64, 1024, z, p, 1 << 20, p, z]) for x, xs, w, ws in one_odd(4)]
    for name, args in calls:
        assert getattr(L.lib(), name)(*args) == L.KRQ_EINVAL, (name, args)
        assert b"16 bytes" in L.lib().krq_last_error(), (name, args)


def test_sizes_known_without_a_call():
    lib = L.lib()
    for M, K in [(1, 32), (16, 512), (17, 544), (32, 9728), (1000, 2560)]:
        for e in (0, 1):
            at, n = X._rows_bytes(M, K, e)
            assert at == lib.krq_mx_tiled_bytes(M, K, e) and n - at == lib.krq_mx_scale_bytes(M, K)
            if L.MX_BF16_ROWS < M <= 32:
                assert n == lib.krq_gemv_mxfp4_ws_bytes(0, e, M, K, 1) == lib.krq_gemv_mxfp4_ws_bytes(0, e, M, K, 2)
    for split in (1, 2, 3):
        assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, L.MX_BF16_ROWS, X.ROWS_MAX_K, split) == 0
        assert lib.krq_gemv_mxfp4_ws_bytes(0, 1, 1, X.ROW_MAX_K, split) == 0


def _q(N=64, K=64, device="cpu"):
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8, device=device)
    return X.MXFP4Weight(u8(N, K // 2), u8(N, K // 32), u8(L.lib().krq_mx_tiled_bytes(N, K, 0)), u8(L.lib().krq_mx_scale_bytes(N, K)))


def test_wrappers_refuse():
    """Wrong shapes and types, and tensors of the CPU, before a launch."""
    from kernels import fp8, lmhead
    from kernels.mlp import PersistentMLP
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    for fn in (X.quantize, X.quant_rows, lambda x: X.linear_mxfp4(x, _q()), lambda x: X.gemm_mxfp4(x, _q()),
               lambda x: X.gemv_swiglu_mxfp4(x, _q()), lambda x: lmhead.lm_head_argmax(x, _q())):
        with pytest.raises(RuntimeError, match="ROCm device"):
            fn(bf(4, 64))
    with pytest.raises(RuntimeError, match="ROCm device"):
        X.embedding(torch.zeros(2, dtype=torch.int64), _q())
    with pytest.raises(RuntimeError, match="ROCm device"):
        X.pack(_q()[0], _q()[1])
    with pytest.raises(ValueError, match="int64 or int32"):
        X.embedding(torch.zeros(2), _q())
    with pytest.raises(ValueError, match="MXFP4Weight"):
        X.linear_mxfp4(bf(4, 64), (bf(4, 64), bf(4)))
    with pytest.raises(ValueError, match="do not match"):
        X.gemm_mxfp4(bf(4, 96), _q())
    with pytest.raises(ValueError, match="elem"):
        X._elem("e5m2")
    with pytest.raises(ValueError, match="weight scale"):  # what every FP8 call checks first of a weight
        fp8._check_weight_scale(_q()[1], 64)
    q = _q()
    assert isinstance(q, tuple) and q.shape == (64, 64) and q[0].shape == (64, 32) and q[1].shape == (64, 2)
    pm = PersistentMLP(1, 512, 1024, "cpu", split=2)
    with pytest.raises(ValueError):
        pm(bf(1, 512), _q(), torch.zeros(1))

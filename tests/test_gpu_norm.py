"""kernels.norm on the GPU: the residual, the normalized rows and their 8-bit forms against the formula in 64 bits on the
CPU, rounded where it rounds. The kernel's only inexact steps before those roundings are an fp64 sum (relative error below
2^-49 for K <= 16384) and an fp64 root and division, so rstd in fp32 differs from the reference's only where that lies
within 2^-48 of a rounding border, one row in 2^23: rows are compared for equality."""

import pytest
import torch

from kernels import fp8, mxfp4, norm
from kernels import gemv as G

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def same(a, b):
    """Equal values, NaN where the other has NaN."""
    a, b = a.float().cpu(), b.float().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def reference(x, delta, ln, eps=1e-6):
    x, ln = x.cpu(), ln.cpu()
    r = x
    if delta is not None:
        d = delta.cpu()
        if d.dim() == 3:
            s = d[0]
            for p in d[1:]:
                s = s + p
            d = s.to(BF)
        r = (x.float() + d.float()).to(BF)
    rstd = (1 / torch.sqrt(r.double().square().sum(-1, keepdim=True) / x.shape[1] + eps)).float()
    return r, ((r.float() * rstd).to(BF).float() * ln.float()).to(BF)


def make(dev, M, K, src, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(M, K, generator=g, device=dev) * 3).to(BF)
    ln = (1 + 0.3 * torch.randn(K, generator=g, device=dev)).to(BF)
    delta = None
    if src == "bf16":
        delta = torch.randn(M, K, generator=g, device=dev).to(BF)
    elif src:
        delta = torch.randn(src, M, K, generator=g, device=dev)
    return x, delta, ln


SIZES = [(1, 16), (1, 2560), (2, 48), (3, 4096), (5, 4112), (16, 320), (17, 2560), (33, 5120), (77, 2560), (1, 16384),
         (19, 8208), (130, 192), (1027, 2560), (1025, 4096), (1030, 2624)]


@pytest.mark.parametrize("src", [None, "bf16", 1, 4, 7])
@pytest.mark.parametrize("M,K", SIZES)
def test_rows(dev, M, K, src):
    x, delta, ln = make(dev, M, K, src)
    keep = x.clone()
    res, h = norm.add_rmsnorm(x, delta, ln)
    r, want = reference(keep, delta, ln)
    assert same(x, keep) and same(res, r) and same(h, want)
    assert (res is x) == (src is None)


def check_outputs(x, delta, ln, eps=1e-6):
    """The 8-bit forms are the package's quantizers of h, byte for byte; h and res are the same in every call."""
    M, K = x.shape
    res, h = norm.add_rmsnorm(x, delta, ln, eps)
    res2, x8, xs, h2 = norm.add_rmsnorm_fp8(x, delta, ln, eps, with_h=True)
    assert same(res, res2) and same(h, h2)
    q8, qs = fp8.quant_rows(h)
    assert torch.equal(x8.view(torch.uint8), q8.view(torch.uint8)) and same(xs, qs) and xs.shape == qs.shape
    a = fp8.SharedScale(torch.full((1,), 37.5, device=x.device), torch.full((1,), 1 / 37.5, device=x.device))
    _, x8, xs = norm.add_rmsnorm_fp8(x, delta, ln, eps, a=a)
    assert torch.equal(x8.view(torch.uint8), fp8._cast_hip(h, a).view(torch.uint8)) and xs is a.scale
    if K % 64 == 0:
        _, x8, xs = norm.add_rmsnorm_fp8(x, delta, ln, eps, tiled=True)
        q8, qs = fp8.quant_rows_tiled(h)
        assert torch.equal(x8, q8) and same(xs, qs)
        _, x8, _ = norm.add_rmsnorm_fp8(x, delta, ln, eps, a=a, tiled=True)
        assert torch.equal(x8, fp8.cast_tiled(h, a))
    if K % 32 == 0:
        for elem in ("e4m3", "e2m1"):
            res3, rows, h3 = norm.add_rmsnorm_mx(x, delta, ln, eps, elem, with_h=True)
            want = mxfp4.quant_rows(h, elem)
            assert same(res, res3) and same(h, h3)
            assert rows.shape == (M, K) and rows.scale_at == want.scale_at and torch.equal(rows.data, want.data)
    return res, h


@pytest.mark.parametrize("src", [None, "bf16", 3])
@pytest.mark.parametrize("M,K", SIZES)
def test_outputs_are_the_quantizers_of_h(dev, M, K, src):
    check_outputs(*make(dev, M, K, src, seed=1))


@pytest.mark.parametrize("M,K", [(20, 320), (1040, 2560)])
def test_nan_inf_and_zero_rows(dev, M, K):
    x, delta, ln = make(dev, M, K, "bf16", seed=2)
    x[1, 7], x[3, 0], x[4, 5], delta[4, 5] = float("nan"), float("inf"), float("inf"), float("-inf")
    x[6], delta[6] = 0.0, 0.0
    x[7], delta[7] = 3e38, 3e38   # the addition passes bf16's range
    x[8], delta[8] = 1e-38, 0.0
    x[9], x[10] = 3e38, -3e38     # squares past fp32's range
    r, want = reference(x, delta, ln)
    res, h = check_outputs(x, delta, ln)
    assert same(res, r) and same(h, want)
    assert h[1].isnan().all() and not h[0].isnan().any() and not h[6].any() and h[9].abs().max() > 0.5
    res, h = check_outputs(x, delta, ln, eps=0.0)  # (a row of zeros has no norm then)
    assert h[6].isnan().all()


def test_partials_of_a_product(dev):
    """The producer's own partials: one call in place of their sum, the addition and the norm."""
    g = torch.Generator(device=dev).manual_seed(3)
    w = torch.randn(2560, 512, generator=g, device=dev).to(BF)
    y = torch.randn(5, 512, generator=g, device=dev).to(BF)
    x, _, ln = make(dev, 5, 2560, None)
    p = G.gemv(y, w, 4)
    res, h = norm.add_rmsnorm(x, p, ln)
    r, want = reference(x, p, ln)
    assert same(res, r) and same(h, want)


def test_strides_alignment_and_in_place(dev):
    M, K = 37, 640
    x, delta, ln = make(dev, M, K, "bf16", seed=4)
    _, parts, _ = make(dev, M, K, 3, seed=5)
    for d in (delta, parts):
        r, want = reference(x, d, ln)
        wide = torch.zeros(M, K + 72, device=dev, dtype=BF)
        wide[:, 8:8 + K] = x
        odd = torch.zeros(M * K + 1, device=dev, dtype=BF)[1:].view(M, K)  # rows that start on 2 bytes
        odd.copy_(x)
        dw = torch.zeros(*d.shape[:-1], K + 40, device=dev, dtype=d.dtype)[..., 16:16 + K]
        dw.copy_(d)
        dt = d.transpose(-1, -2).contiguous().transpose(-1, -2)
        lw = torch.zeros(2 * K, device=dev, dtype=BF)[::2]
        lw.copy_(ln)
        for xx in (wide[:, 8:8 + K], odd, x.t().contiguous().t()):
            for dd in (dw, dt):
                res, h = norm.add_rmsnorm(xx, dd, lw)
                assert same(res, r) and same(h, want)
        xx = x.clone()
        res, h = norm.add_rmsnorm(xx, d, ln, res_out=xx)
        assert res is xx and same(xx, r) and same(h, want)
    dd = delta.clone()
    res, h = norm.add_rmsnorm(x, dd, ln, res_out=dd)
    r, want = reference(x, delta, ln)
    assert res is dd and same(dd, r) and same(h, want)
    wide = torch.ones(M, K + 72, device=dev, dtype=BF)
    with pytest.raises(ValueError, match="overlaps"):
        norm.add_rmsnorm(wide[:, :K], delta, ln, res_out=wide.view(-1)[:M * K].view(M, K))
    with pytest.raises(ValueError, match="overlaps"):
        norm.add_rmsnorm(x, parts, ln, res_out=parts.view(-1).view(BF)[:M * K].view(M, K))


def test_rows_around_the_outputs_are_left(dev):
    M, K = 21, 320
    x, delta, ln = make(dev, M, K, "bf16", seed=6)
    room = torch.full((M + 2, K), 7.0, device=dev, dtype=BF)
    norm.add_rmsnorm(x, delta, ln, res_out=room[1:M + 1])
    assert (room[0] == 7).all() and (room[-1] == 7).all()


def test_no_rows(dev):
    x = torch.empty(0, 320, device=dev, dtype=BF)
    ln = torch.ones(320, device=dev, dtype=BF)
    for d in (None, x, torch.empty(2, 0, 320, device=dev)):
        res, h = norm.add_rmsnorm(x, d, ln)
        assert res.shape == h.shape == (0, 320)
    _, x8, xs = norm.add_rmsnorm_fp8(x, x, ln)
    assert x8.shape == (0, 320) and xs.shape == (0, 1)
    _, rows = norm.add_rmsnorm_mx(x, x, ln)
    assert rows.shape == (0, 320) and rows.data.numel() == 0


def test_graph_and_streams(dev):
    x, delta, ln = make(dev, 18, 2560, 4, seed=7)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm.add_rmsnorm_mx(x, delta, ln)
        eager = norm.add_rmsnorm_fp8(x, delta, ln, with_h=True)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = norm.add_rmsnorm_fp8(x, delta, ln, with_h=True)
    for i in range(3):
        x.copy_(make(dev, 18, 2560, None, seed=20 + i)[0])
        graph.replay()
        eager = norm.add_rmsnorm_fp8(x, delta, ln, with_h=True)
        for a, b in zip(out, eager):
            assert same(a, b)


# Both sides of every border between the thread layouts: rows 600 and 1,536, K 2,560, 4,096, 5,120 and 8,192, and what is left of 16 rows and of
# a wave's chunks. (M, K): <4 waves a workgroup, 1 a row, 5 chunks a lane>, <4, 1, 8>, <2, 2, 5>, <8, 8, 1>, <8, 8, 2>, <16, 16, 2>
BORDERS = [(600, 2560), (599, 2560), (613, 16), (600, 2576), (1537, 4096), (1541, 2624), (1536, 2592), (1535, 2592), (1535, 4096),
           (601, 5120), (613, 4112), (600, 4608), (1600, 4160), (599, 5120), (600, 5136), (1550, 8192), (603, 8208)]


@pytest.mark.parametrize("src", [None, "bf16", 2])
@pytest.mark.parametrize("M,K", BORDERS)
def test_layouts(dev, M, K, src):
    """Against the formula and the quantizers, and the same bytes as a few rows that go alone, eight or sixteen waves to a row."""
    x, delta, ln = make(dev, M, K, src, seed=8)
    r, want = reference(x, delta, ln)
    res, h = check_outputs(x, delta, ln)
    assert same(res, r) and same(h, want)
    for rows in (slice(0, 3), slice(M // 2, M // 2 + 17), slice(M - 5, M)):
        d = delta if delta is None else delta[..., rows, :].contiguous()
        for few, many in zip(norm.add_rmsnorm_fp8(x[rows].contiguous(), d, ln, with_h=True), norm.add_rmsnorm_fp8(x, delta, ln, with_h=True)):
            assert same(few, many[rows])


@pytest.mark.parametrize("M,K", [(1541, 4096), (1539, 2656), (605, 5120), (613, 4160)])
def test_layouts_with_nan_inf_and_zero_rows(dev, M, K):
    test_nan_inf_and_zero_rows(dev, M, K)


@pytest.mark.parametrize("M,K", [(1541, 4096), (605, 5120), (700, 2560)])
def test_layouts_in_place_and_strided(dev, M, K):
    x, delta, ln = make(dev, M, K, "bf16", seed=9)
    r, want = reference(x, delta, ln)
    wide = torch.full((M, K + 40), 7.0, device=dev, dtype=BF)
    wide[:, 16:16 + K] = x
    res, h = norm.add_rmsnorm(wide[:, 16:16 + K], delta, ln)
    assert same(res, r) and same(h, want) and (wide[:, :16] == 7).all() and (wide[:, 16 + K:] == 7).all()
    for own in (x, delta):
        xx, dd = x.clone(), delta.clone()
        out = xx if own is x else dd
        res, x8, xs = norm.add_rmsnorm_fp8(xx, dd, ln, res_out=out)
        q8, qs = fp8.quant_rows(h)
        assert res is out and same(out, r) and torch.equal(x8.view(torch.uint8), q8.view(torch.uint8)) and same(xs, qs)


def test_more_than_2_31_elements(dev):
    """Rows behind 2^31 elements, and 2^32 bytes of 8-bit rows in tiles: the last ones against the same rows alone."""
    M, K = (1 << 31) // 16384 + 21, 16384
    g = torch.Generator(device=dev).manual_seed(10)
    x, delta = (torch.empty(M, K, device=dev, dtype=BF).normal_(generator=g) for _ in range(2))
    ln = (1 + 0.3 * torch.randn(K, generator=g, device=dev)).to(BF)
    at = M // 16 * 16 - 16
    for call in (lambda a, b: norm.add_rmsnorm_fp8(a, b, ln, with_h=True), lambda a, b: norm.add_rmsnorm_fp8(a, b, ln, tiled=True),
                 lambda a, b: norm.add_rmsnorm_mx(a, b, ln)):
        out, tail = call(x, delta), call(x[at:].contiguous(), delta[at:].contiguous())
        assert same(out[0][at:], tail[0])
        if isinstance(out[1], mxfp4.MXRows):  # (data, then scales, each in blocks of sixteen rows)
            a, b = out[1], tail[1]
            size = b.scale_at
            assert torch.equal(a.data[a.scale_at - size:a.scale_at], b.data[:size])
            rest = b.data.numel() - size
            assert torch.equal(a.data[-rest:], b.data[-rest:])
        elif out[1].dtype is torch.uint8:
            assert torch.equal(out[1][at * K:], tail[1]) and same(out[2][at:], tail[2])
        else:
            assert all(same(a[at:], b) for a, b in zip(out[1:], tail[1:]))
        del out, tail

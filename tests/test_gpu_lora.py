"""kernels.lora on the GPU against the formula in 64 bits.

Tolerance, element by element. h is an fp32 sum of K products that are exact in fp32: off by at most K 2^-24 sum_k |A x|,
whatever its order. It enters the second product as two bf16, off by at most 2^-16 |h| (the rest of a rounding to 2^-8,
rounded to 2^-8), scaled with one rounding and summed over r ranks and two terms in fp32: 2 r 2^-24 sum_r |B h|. Then y is
added and rounded once to the result's type: eps / 2 of the result, and 2^-24 of it for the fp32 addition before.
By the 2-norm over all outputs, with y = 0 and fp32 results, roundings of either sign add as their root: the split's,
whose mean square is a small part of 2^-16, and sqrt(K) 2^-24 stay under 2^-16."""

import pytest
import torch

from kernels import _lib as L
from kernels import gemv as G
from kernels import lora

pytestmark = pytest.mark.gpu
BF, INF, NAN = torch.bfloat16, float("inf"), float("nan")


def factors(g, K, parts, ranks, dev):
    def randn(*s):
        return torch.randn(*s, generator=g, device=dev)

    return [[((randn(r, K) * K ** -0.5).to(BF), randn(n, r).to(BF)) for n in parts] for r in ranks]


def bank(dev, K, parts, rank, pairs, scales, slots=None):
    ad = lora.Adapters(K, parts if len(parts) > 1 else parts[0], rank, slots or max(1, len(pairs)), dev)
    for i, (p, s) in enumerate(zip(pairs, scales)):
        if p is not None:
            ad.load(i, p, s)
    return ad


def reference(y, x, pairs, scales, ids, parts):
    """(the result in 64 bits, the tolerance of every element before the last rounding)."""
    out, tol, at = y.double().clone(), torch.zeros_like(y, dtype=torch.float64), 0
    xd, K = x.double(), x.shape[1]
    for p, n in enumerate(parts):
        for i, pair in enumerate(pairs):
            rows = torch.nonzero(ids == i)[:, 0]
            if pair is None or pair[p] is None or not len(rows):
                continue
            a, b = pair[p][0].double(), pair[p][1].double()
            h, ha = xd[rows] @ a.t(), xd[rows].abs() @ a.abs().t()
            out[rows, at:at + n] += scales[i] * (h @ b.t())
            off = K * 2.0 ** -24 * ha + (2.0 ** -16 + (2 * a.shape[0] + 2) * 2.0 ** -24) * h.abs()
            tol[rows, at:at + n] = abs(scales[i]) * (off @ b.abs().t())
        at += n
    return out, tol


def check(got, y, x, pairs, scales, ids, parts):
    want, tol = reference(y, x, pairs, scales, ids, parts)
    assert got.dtype == y.dtype and got.shape == y.shape
    tol = tol + (torch.finfo(y.dtype).eps / 2 + 2.0 ** -24) * (want.abs() + tol) + 1e-37
    bad = ((got.double() - want).abs() > tol) | got.isnan()
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:3].tolist())


def make(dev, M, K, parts, ranks, dtype, seed=0, order="each", none=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    pairs = factors(g, K, parts, ranks, dev)
    scales = [0.5 + 0.25 * i for i in range(len(ranks))]
    x = torch.randn(M, K, generator=g, device=dev).to(BF)
    y = (torch.randn(M, sum(parts), generator=g, device=dev) * 2).to(dtype)
    if order == "each":
        ids = torch.randint(-1 if none else 0, len(ranks), (M,), generator=g, device=dev)
    else:
        ids = torch.arange(M, device=dev) * len(ranks) // M
    return pairs, scales, x, y, ids


CASES = [
    # M, K, parts, ranks, the bank's rank
    (1, 16, [1], [1], 1),
    (1, 2560, [2560], [16], 16),
    (2, 48, [16], [8, 3], 8),
    (5, 2560, [4096, 1024, 1024], [64, 32, 16, 8], 64),
    (16, 4096, [2560], [16] * 16, 16),
    (17, 80, [65, 3, 130], [17, 40, 200], 200),
    (33, 2576, [100], [256], 256),
    (64, 9728, [2560], [16, 32], 32),
    (65, 320, [64, 64], [24, 24, 24, 24, 24], 24),
    (77, 2560, [6144], [8, 16, 32, 64, 128], 128),
    (256, 640, [300, 20], [16, 16], 16),
    (257, 640, [300, 20], [16, 16], 16),
    (300, 2560, [4096, 1024, 1024], [8, 48, 16], 48),
    (1000, 1040, [333, 1], [32, 5, 250], 256),
    (515, 64, [1, 2, 3, 4, 5, 6, 7, 8], [16, 1], 16),
    (2049, 512, [9728, 72], [16] * 5, 16),
]


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("order", ["each", "runs"])
@pytest.mark.parametrize("M,K,parts,ranks,rank", CASES)
def test_against_the_formula(dev, M, K, parts, ranks, rank, order, dtype):
    pairs, scales, x, y, ids = make(dev, M, K, parts, ranks, dtype, order=order)
    ad = bank(dev, K, parts, rank, pairs, scales)
    keep = y.clone()
    got = lora.add(y, x, ad, ids)
    assert torch.equal(y, keep)
    check(got, y, x, pairs, scales, ids, parts)
    assert torch.equal(got, lora.add(y, x, ad, ids.int()))  # the same values again, for the other type of ids
    assert lora.add(y, x, ad, ids, out=y) is y and torch.equal(got, y)


@pytest.mark.parametrize("M,K,parts,ranks,rank", [
    (777, 2576, [90, 30, 17], [32, 16, 8], 32),      # 16 places, three tiles of ranks of six
    (1100, 320, [64, 70], [32, 20], 32),             # 16 places, all four
    (6700, 2064, [66], [16, 9, 3], 16),              # 32 places, one tile of ranks
    (3400, 1040, [40, 24], [16, 5], 16),             # 32 places, two
    (2250, 2128, [33, 8, 60], [16, 16, 16, 16], 16),  # three
    (1700, 6144, [50], [64, 48], 64),                # four, K in two parts
])
@pytest.mark.parametrize("order", ["each", "runs"])
def test_tiles_of_places_and_ranks(dev, M, K, parts, ranks, rank, order):
    pairs, scales, x, y, ids = make(dev, M, K, parts, ranks, BF, order=order)
    ad = bank(dev, K, parts, rank, pairs, scales)
    got = lora.add(y, x, ad, ids)
    check(got, y, x, pairs, scales, ids, parts)
    assert torch.equal(got, lora.add(y, x, ad, ids))


@pytest.mark.parametrize("M,K,N,r", [(9, 2560, 2560, 16), (400, 4096, 1024, 64)])
def test_norm_of_the_error(dev, M, K, N, r):
    pairs, scales, x, _, ids = make(dev, M, K, [N], [r] * 3, BF, none=False)
    y = torch.zeros(M, N, device=dev)
    got = lora.add(y, x, bank(dev, K, [N], r, pairs, scales), ids).double()
    want, _ = reference(y, x, pairs, scales, ids, [N])
    assert float((got - want).norm() / want.norm()) < 2.0 ** -16


@pytest.mark.parametrize("M", [6, 300])
def test_rows_without_an_adapter_and_empty_slots(dev, M):
    pairs, scales, x, y, ids = make(dev, M, 640, [96, 40], [16, 8, 24], BF)
    pairs[1] = None                       # an empty slot
    pairs[2] = [None, pairs[2][1]]        # a part left alone
    ad = bank(dev, 640, [96, 40], 24, pairs, scales)
    got = lora.add(y, x, ad, ids)
    check(got, y, x, pairs, scales, ids, [96, 40])
    still = (ids < 0) | (ids == 1)
    assert torch.equal(got[still], y[still]) and torch.equal(got[ids == 2][:, :96], y[ids == 2][:, :96])
    ids.fill_(-7)
    assert torch.equal(lora.add(y, x, ad, ids), y)
    ids[M // 2] = 3                       # past the last slot
    got = lora.add(y, x, ad, ids)
    assert got[M // 2].isnan().all() and torch.equal(got[ids < 0], y[ids < 0])


@pytest.mark.parametrize("M", [7, 290])
def test_nan_and_infinities_stay_in_their_rows(dev, M):
    pairs, scales, x, y, ids = make(dev, M, 320, [80], [16, 8], BF, none=False)
    ad = bank(dev, 320, [80], 16, pairs, scales, slots=3)
    clean = lora.add(y, x, ad, ids)
    x2, y2 = x.clone(), y.clone()
    x2[2, 5], x2[4, 0], y2[5, 7] = float("nan"), float("inf"), float("-inf")
    got = lora.add(y2, x2, ad, ids)
    fine = torch.ones(M, dtype=torch.bool, device=dev)
    fine[[2, 4, 5]] = False
    assert torch.equal(got[fine], clean[fine])
    assert got[2].isnan().all() and not got[4].isfinite().any() and got[5, 7] == float("-inf")
    nan = [(torch.full((16, 320), float("nan"), dtype=BF, device=dev), torch.full((80, 16), float("inf"), dtype=BF, device=dev))]
    ad.load(2, nan)
    assert torch.equal(lora.add(y, x, ad, ids), clean)
    # ranks that a slot does not have stay out of the sum: an infinity of x meets no zero row of A
    one = [(torch.ones(1, 320, dtype=BF, device=dev), torch.ones(80, 1, dtype=BF, device=dev))]
    ad.load(2, one)
    ids2 = torch.full_like(ids, 2)
    assert (lora.add(y, x2, ad, ids2)[4] == float("inf")).all()


@pytest.mark.parametrize("M", [5, 270])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_strides_and_alignment(dev, M, dtype):
    K, N = 160, 200
    pairs, scales, x, y, ids = make(dev, M, K, [N], [16, 8], dtype)
    ad = bank(dev, K, [N], 16, pairs, scales)
    want = lora.add(y, x, ad, ids)
    for pad, off in ((56, 8), (7, 3), (1, 1)):
        wide = torch.full((M, N + pad), 9.0, device=dev, dtype=dtype)
        wide[:, off:off + N] = y
        view = wide[:, off:off + N]
        wx = torch.zeros(M, K + pad, device=dev, dtype=BF)
        wx[:, off:off + K] = x
        room = torch.full((M, N + pad), 9.0, device=dev, dtype=dtype)
        lora.add(view, wx[:, off:off + K], ad, ids, out=room[:, off:off + N])
        assert torch.equal(room[:, off:off + N], want)
        lora.add(view, x, ad, ids, out=view)
        for t in (wide, room):
            assert torch.equal(t[:, off:off + N], want) and (t[:, :off] == 9).all() and (t[:, off + N:] == 9).all()
    assert torch.equal(lora.add(y.t().contiguous().t(), x.t().contiguous().t(), ad, ids), want)
    ids2 = torch.stack([ids, ids], 1)[:, 0]
    assert torch.equal(lora.add(y, x, ad, ids2), want)
    with pytest.raises(ValueError, match="overlaps"):
        room = torch.zeros(M * N + 8, device=dev, dtype=dtype)
        lora.add(room[:M * N].view(M, N), x, ad, ids, out=room[8:].view(M, N))


def test_partials(dev):
    """Adapters into a split-K product's partials: their sum is the product with the adapters."""
    K, N = 512, 640
    pairs, scales, x, _, ids = make(dev, 6, K, [N], [16, 32], BF)
    g = torch.Generator(device=dev).manual_seed(9)
    w = (torch.randn(N, K, generator=g, device=dev) * 0.05).to(BF)
    p = G.gemv(x, w, 4)
    rest, first = p[1:].clone(), p[0].clone()
    ad = bank(dev, K, [N], 32, pairs, scales)
    lora.add(p[0], x, ad, ids, out=p[0])
    assert torch.equal(p[1:], rest)
    check(p[0], first, x, pairs, scales, ids, [N])


def test_loading_and_clearing(dev):
    K, N = 320, 72
    pairs, scales, x, y, ids = make(dev, 8, K, [N], [32, 8], BF, none=False)
    ad = bank(dev, K, [N], 32, pairs, scales)
    lora.add(y, x, ad, ids)
    ad.load(0, [pairs[1][0]], 2.0)  # a smaller rank over a larger one
    check(lora.add(y, x, ad, ids), y, x, [pairs[1], pairs[1]], [2.0, scales[1]], ids, [N])
    ad.clear(1)
    check(lora.add(y, x, ad, ids), y, x, [pairs[1], None], [2.0, 0], ids, [N])
    ad.load(1, pairs[0][0], 1.0)    # one pair as such
    check(lora.add(y, x, ad, ids), y, x, [pairs[1], pairs[0]], [2.0, 1.0], ids, [N])


def test_no_rows(dev):
    ad = lora.Adapters(32, 8, 4, 1, dev)
    y = torch.empty(0, 8, device=dev, dtype=BF)
    assert lora.add(y, torch.empty(0, 32, device=dev, dtype=BF), ad, torch.empty(0, dtype=torch.int32, device=dev)).shape == (0, 8)


@pytest.mark.parametrize("M", [12, 300])
def test_graph_with_new_ids_and_adapters(dev, M):
    K, parts = 640, [128, 64]
    pairs, scales, x, y, ids = make(dev, M, K, parts, [16, 8, 32], BF)
    ad = bank(dev, K, parts, 32, pairs, scales)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lora.add(y, x, ad, ids)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lora.add(y, x, ad, ids)
    for i in range(4):
        ids.copy_(make(dev, M, K, parts, [16, 8, 32], BF, seed=30 + i)[4])
        if i == 2:
            pairs[0], scales[0] = pairs[2], 3.0
            ad.load(0, pairs[0], 3.0)
        graph.replay()
        check(out, y, x, pairs, scales, ids, parts)
        assert torch.equal(out, lora.add(y, x, ad, ids))


def test_calls_on_two_streams(dev):
    K, N = 2560, 2560
    pairs, scales, x, y, ids = make(dev, 40, K, [N], [16] * 4, BF)
    ad = bank(dev, K, [N], 16, pairs, scales)
    want, perm = lora.add(y, x, ad, ids), torch.randperm(40, device=dev)
    want2 = lora.add(y[perm], x[perm], ad, ids[perm])
    y2, x2, ids2 = y[perm].contiguous(), x[perm].contiguous(), ids[perm].contiguous()
    torch.cuda.synchronize()
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), ([], [])
    for _ in range(8):
        for s, (yy, xx, ii), o in zip(streams, ((y, x, ids), (y2, x2, ids2)), got):
            with torch.cuda.stream(s):
                o.append(lora.add(yy, xx, ad, ii))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got[0]) and all(torch.equal(o, want2) for o in got[1])


def test_a_bank_past_32_bit_offsets(dev):
    """The last slot of a bank whose factors span more than 2^31 elements."""
    K, N, r, slots = 16384, 16384, 256, 513
    ad = lora.Adapters(K, N, r, slots, dev)
    assert ad.a.numel() > 2 ** 31 and ad.b.numel() > 2 ** 31
    pairs, scales, x, y, _ = make(dev, 3, K, [N], [r], BF)
    ad.load(slots - 1, pairs[0], scales[0])
    ids = torch.tensor([slots - 1, -1, slots - 1], device=dev)
    check(lora.add(y, x, ad, ids), y, x, [pairs[0]], scales, torch.where(ids < 0, -1, 0), [N])


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("M", [7, 40, 390, 2100])
def test_parts_of_their_own_ranks(dev, M, dtype):
    """A part that an adapter leaves alone, or in which it has fewer ranks than in another, takes part with its own: what is not
    finite in x meets no rank that the part does not have. Positive factors, so that an infinity stays one."""
    K, parts = 160, [96, 40, 33]
    pairs, scales, x, y, ids = make(dev, M, K, parts, [40, 17, 33, 16], dtype, seed=11)
    for i, own in enumerate(([None, 20, 5], [3, None, 17], [16, 33, None], [None, None, 7])):
        pairs[i] = [None if r is None else (a[:r].abs().contiguous(), b[:, :r].abs().contiguous()) for r, (a, b) in zip(own, pairs[i])]
    ad = bank(dev, K, parts, 40, pairs, scales)
    check(lora.add(y, x, ad, ids), y, x, pairs, scales, ids, parts)
    bad = torch.arange(M, device=dev) % 3 == 0
    x[bad, 5] = torch.where(torch.arange(M, device=dev) % 2 == 0, INF, NAN).to(BF)[bad]
    got = lora.add(y, x, ad, ids)
    want, at = y.clone(), 0
    for p, n in enumerate(parts):
        for i, pair in enumerate(pairs):
            if pair[p] is not None:
                rows = torch.nonzero((ids == i) & bad)[:, 0]
                want[rows, at:at + n] = x[rows, 5:6].to(dtype)
        at += n
    assert torch.equal(got[bad].isnan(), want[bad].isnan())
    fine = bad[:, None] & ~want.isnan()
    assert torch.equal(got[fine], want[fine])
    check(got[~bad], y[~bad], x[~bad], pairs, scales, ids[~bad], parts)
    assert lora.add(y, x, ad, ids, out=y) is y and torch.equal(y[fine], want[fine]) and torch.equal(y[~bad], got[~bad])


@pytest.mark.parametrize("M", [9, 400])
def test_entry_point_with_one_rank_for_a_slot(dev, M):
    """krq_lora_add: every part has the slot's rank, as where a bank's parts have the same."""
    K, parts = 160, [96, 40]
    pairs, scales, x, y, ids = make(dev, M, K, parts, [40, 17], BF, seed=12)
    ad = bank(dev, K, parts, 40, pairs, scales)
    want, got, lib = lora.add(y, x, ad, ids), torch.empty_like(y), L.lib()
    nbytes = lib.krq_lora_ws_bytes(M, K, 2, ad.rank)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    L.call("krq_lora_add", L.ptr(x), K, L.ptr(ids), True, L.ptr(ad.a), L.ptr(ad.b), L.ptr(ad.ranks), L.ptr(ad.scales), ad.slots, M, K, ad._n, 2,
           ad.rank, L.ptr(y), sum(parts), L.ptr(got), sum(parts), False, L.ptr(ws), nbytes, L.stream(x))
    assert torch.equal(got, want)


def test_the_most_rows_and_slots(dev):
    """2^24 rows, and a bank of 2^23 - 1 slots: places and ids as long as the kernels keep them."""
    M, K, N = 1 << 24, 16, 3
    pairs, scales, x, y, ids = make(dev, 64, K, [N], [16, 5], BF, seed=13)
    ad = bank(dev, K, [N], 16, pairs, scales)
    want = lora.add(y, x, ad, ids)
    got = lora.add(y.repeat(M // 64, 1), x.repeat(M // 64, 1), ad, ids.repeat(M // 64))
    assert torch.equal(got.view(M // 64, 64, N), want.expand(M // 64, 64, N))
    del ad, got
    slots = (1 << 23) - 1
    ad = lora.Adapters(K, N, 5, slots, dev)
    for i, s in enumerate((slots - 1, 0)):
        ad.load(s, pairs[1], scales[i])
    ids = torch.tensor([slots - 1, 0, -1, slots, 1 << 40] * 80, device=dev)
    x, y = x[:40].repeat(10, 1), y[:40].repeat(10, 1)
    got = lora.add(y, x, ad, ids)
    fine = ids < slots
    check(got[fine], y[fine], x[fine], [pairs[1], pairs[1]], scales, torch.where(ids < 0, -1, torch.where(ids == 0, 1, 0))[fine], [N])
    assert got[~fine].isnan().all()

"""kernels.beam on the GPU. Selection against its definition in 64 bits with a stable sort; reordering against indexing.

Tolerance of the selection: the kernel's lse sums exponentials in fp32, each off by at most (1.5 |x| + 4) 2^-24 of itself for
an exponent x, of which only |x| < 32 matter, and adds them in less than 64 steps: off by less than 2^-17 in all. Two candidates of
different beams may change places where their values in 64 bits are within twice that (within a beam they are ordered by
their logits); a score is a rounding of v to fp32 beside it."""

import pytest
import torch

from kernels import beam, fp8, lmhead
from kernels import gemv as G

pytestmark = pytest.mark.gpu
BF, INF, NAN = torch.bfloat16, float("inf"), float("nan")
OFF = 2.0 ** -17


def values(logits, scores):
    """v [B, W V] in 64 bits on the CPU; NaN as the largest (inf), which no other v is."""
    B, W = scores.shape
    l, s = logits.double().cpu().reshape(B, W, -1), scores.double().cpu()[..., None]
    v = s + (l - torch.logsumexp(l, -1, keepdim=True))
    dead = (l == -INF).all(-1, keepdim=True) | (s == -INF)
    bad = (l.isnan() | (l == INF)).any(-1, keepdim=True) | s.isnan() | (s == INF)
    v = torch.where(dead, -INF, v)
    return torch.where(bad, INF, v).reshape(B, -1)


def check(logits, scores, n=None):
    got, beams, tokens = beam.select(logits, scores, n)
    B, W = scores.shape
    n = 2 * W if n is None else n
    assert got.shape == beams.shape == tokens.shape == (B, n) and got.dtype == torch.float32
    assert beams.dtype == tokens.dtype == torch.int64
    v = values(logits, scores)
    V = v.shape[1] // W
    best, at = torch.sort(v, dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    flat = (beams * V + tokens).cpu()
    assert ((tokens >= 0) & (tokens < V) & (beams >= 0) & (beams < W)).all()
    assert all(len(set(r)) == n for r in flat.tolist())
    mine = torch.gather(v, 1, flat)
    other = flat != at
    if other.any():  # only near candidates of different beams
        assert ((mine - best).abs()[other] <= 2 * OFF).all(), (flat[other][:5], at[other][:5])
        assert (other.sum(1) <= 2).all()
    g = got.double().cpu()
    assert torch.equal(g.isnan(), mine == INF) and torch.equal(g == -INF, mine == -INF)
    fine = mine.isfinite()
    assert ((g - mine).abs()[fine] <= OFF + 2.0 ** -24 * mine.abs()[fine]).all()
    return got, beams, tokens


def make(dev, B, W, V, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    logits = torch.randn(B * W, V, generator=g, device=dev) * 3
    logits.scatter_(1, torch.randint(V, (B * W, 6), generator=g, device=dev), 12.0 + torch.rand(B * W, 6, generator=g, device=dev))
    return logits.to(dtype), -5 * torch.rand(B, W, generator=g, device=dev)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,W,V,n", [(1, 1, 1, 1), (1, 1, 5, 5), (1, 2, 1, 2), (2, 3, 7, 21), (3, 4, 64, 8), (1, 4, 151936, 8), (8, 8, 1000, 16),
                                     (3, 5, 8191, 10), (1, 64, 300, 64), (2, 16, 20001, 32), (1, 2, 1 << 20, 64), (70, 1, 999, 2),
                                     (1, 64, 151936, 64), (16, 32, 2048, 64), (4, 8, 32768, 1), (300, 3, 257, 6)])
def test_against_the_definition(dev, B, W, V, n, dtype):
    check(*make(dev, B, W, V, dtype), n)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("V", [5, 8, 2047, 2048, 2049, 8192, 40000])
def test_ties_go_to_the_lowest_beam_and_token(dev, V, dtype):
    """Equal logits and equal beams: exactly the stable order, for every n."""
    logits = torch.zeros(12, V, device=dev, dtype=dtype)
    scores = torch.zeros(3, 4, device=dev)
    for n in (1, 4, 17, 64):
        n = min(n, 4 * V)
        got, beams, tokens = beam.select(logits, scores, n)
        at = torch.arange(n, device=dev).expand(3, n)
        assert torch.equal(beams, at // V) and torch.equal(tokens, at % V)
    g = torch.Generator(device=dev).manual_seed(V)
    row = torch.randint(-3, 4, (1, V), generator=g, device=dev).to(dtype)  # seven levels; -0 beside 0
    row = torch.where((row == 0) & (torch.rand(1, V, generator=g, device=dev) < 0.5), -row, row)
    logits = row.expand(12, V).contiguous()
    n = min(64, 4 * V)
    _, beams, tokens = beam.select(logits, scores, n)
    order = torch.sort(row.float().expand(4, V).reshape(-1).cpu(), descending=True, stable=True).indices
    # equal beams: each level's tokens of beam 0, then of beam 1, ..
    flat = (beams * V + tokens).cpu()
    assert torch.equal(flat, order[:n].expand(3, n))
    sorted_row = torch.sort(row, descending=True, stable=True).values  # few lanes hold the largest
    _, beams, tokens = beam.select(sorted_row.expand(12, V).contiguous(), scores, n)
    order = torch.sort(sorted_row.float().expand(4, V).reshape(-1).cpu(), descending=True, stable=True).indices
    assert torch.equal((beams * V + tokens).cpu(), order[:n].expand(3, n))


@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_masks(dev, dtype):
    for V in (40, 3000, 70001):
        logits, scores = make(dev, 6, 4, V, dtype, seed=V)
        logits[0] = -INF                         # a beam with nothing allowed
        logits[4:8] = -INF                       # an entry with nothing allowed
        logits[8:12] = -INF
        logits[9, V - 1], logits[10, 3] = 1.0, -2.0   # two continuations for eight places
        scores[3, 1:] = -INF                     # a first step: copies of one beam
        logits[16, V // 2], logits[17, 1], logits[18, 2] = NAN, INF, -INF
        scores[5] = torch.tensor([NAN, INF, -INF, -1.0], device=dev)
        check(logits, scores)
        check(logits, scores, 30)
    got, beams, tokens = beam.select(logits, scores)
    assert (got[1] == -INF).all() and (beams[1] == 0).all() and torch.equal(tokens[1], torch.arange(8, device=dev))
    assert beams[2, :2].tolist() in ([1, 2], [2, 1]) and (got[2, 2:] == -INF).all()
    assert got[4].isnan().all() and (beams[4] == 0).all() and got[5].isnan().all()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("V,n", [(5000, 64), (5000, 9), (20000, 33)])
def test_few_tokens_allowed(dev, V, n, dtype):
    """Masks that leave some tokens, fewer and more than a chunk's threshold needs, among them whole chunks without one."""
    g = torch.Generator(device=dev).manual_seed(V + n)
    allowed = (1, 5, n - 1, n, n + 1, 100, 520, 2047)
    logits = torch.full((len(allowed) * 2, V), -INF, device=dev)
    for i, k in enumerate(allowed):
        for row in (2 * i, 2 * i + 1):
            where = torch.randperm(V if row % 2 else min(V, 2100), generator=g, device=dev)[:k]
            logits[row, where] = torch.randn(k, generator=g, device=dev) * 2
    check(logits.to(dtype), -torch.rand(len(allowed), 2, generator=g, device=dev), n)
    check(logits[4:].to(dtype), torch.zeros(2 * len(allowed) - 4, 1, device=dev), n)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("left", [1, 20, 130, 255, 256, 511, 512])
def test_short_last_chunk(dev, left, dtype):
    """A row's last tokens, behind whole chunks: distinct, equal, masked in part, the largest of the row or none of them."""
    V = 3 * 8192 + left
    for n in (1, 19, 64):
        logits, scores = make(dev, 2, 3, V, dtype, seed=left)
        logits[0, -left:] += 20
        logits[1, -left:] = 25
        logits[2, :-left] = -INF
        logits[3, -left // 2:] = -INF
        logits[4, -left:] = -INF
        check(logits, scores, n)


def test_extreme_values(dev):
    big = torch.finfo(torch.float32).max
    logits = torch.zeros(2, 3000, device=dev)
    logits[0, 5], logits[0, 6], logits[1] = big, -big, -big
    logits[1, 2999] = -big / 2
    check(logits, torch.tensor([[-big, 0.0]], device=dev), 4)
    logits = torch.full((2, 2000), torch.finfo(BF).min, device=dev, dtype=BF)  # a mask of the type's lowest value
    logits[0, 1999] = 3.0
    check(logits, torch.tensor([[0.0, -1.0]], device=dev), 8)


def test_views(dev):
    logits, scores = make(dev, 3, 4, 501, BF)
    want = beam.select(logits, scores)
    wide = torch.full((12, 517), INF, device=dev, dtype=BF)
    for off in (0, 1, 9):
        view = wide[:, off:off + 501]
        view.copy_(logits)
        assert all(torch.equal(a, b) for a, b in zip(want, beam.select(view, scores)))
        wide.fill_(INF)
    wide_scores = torch.zeros(3, 9, device=dev)
    wide_scores[:, ::2][:, :4] = scores
    for l in (logits.view(3, 4, 501), logits.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(want, beam.select(l, wide_scores[:, ::2][:, :4])))
    assert [t.shape for t in beam.select(logits[:0], scores[:0])] == [(0, 8)] * 3


def test_graph_and_two_streams(dev):
    logits, scores = make(dev, 4, 4, 30000, BF)
    logits2, scores2 = make(dev, 4, 4, 30000, BF, seed=5)
    want, want2 = beam.select(logits, scores), beam.select(logits2, scores2)
    torch.cuda.synchronize()
    streams, got = (torch.cuda.Stream(), torch.cuda.Stream()), ([], [])
    for _ in range(8):
        for s, (l, sc), o in zip(streams, ((logits, scores), (logits2, scores2)), got):
            with torch.cuda.stream(s):
                o.append(beam.select(l, sc))
    torch.cuda.synchronize()
    for o, w in zip(got, (want, want2)):
        assert all(torch.equal(a, b) for r in o for a, b in zip(r, w))
    graph = torch.cuda.CUDAGraph()
    caches = [torch.zeros(2, 16, 3, 10, 8, device=dev, dtype=BF) for _ in range(3)]
    lengths = torch.tensor([10, 3, 0, 7], device=dev)
    with torch.cuda.graph(graph):
        out = beam.select(logits, scores)
        beam.reorder(caches, out[1][:, :4], dim=1, lengths=lengths, length_dim=3)
    for i in range(4):
        l, s = make(dev, 4, 4, 30000, BF, seed=40 + i)
        logits.copy_(l)
        scores.copy_(s)
        for c in caches:
            c.copy_(torch.randn(c.shape, device=dev))
        before = [c.clone() for c in caches]
        graph.replay()
        eager = beam.select(l, s)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        for c, b in zip(caches, before):
            assert torch.equal(c, expected(b, eager[1][:, :4], 1, lengths, 3))


def test_behind_the_lm_head(dev):
    """The head's own logits: the first candidate of a single beam is its argmax."""
    g = torch.Generator(device=dev).manual_seed(2)
    w = torch.randn(4096, 256, generator=g, device=dev).to(BF)
    h = torch.randn(6, 256, generator=g, device=dev).to(BF)
    for head in (w, fp8.quantize(w)):
        ids, logits = lmhead.lm_head_argmax(h, head, return_logits=True)
        _, beams, tokens = check(logits, torch.zeros(6, 1, device=dev), 3)
        assert torch.equal(tokens[:, 0], ids) and not beams.any()
        check(logits, torch.zeros(2, 3, device=dev))
    check(G.gemv(h, w, 1), torch.zeros(3, 2, device=dev))


# ---------------------------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------------------------
def expected(state, beams, dim, lengths=None, length_dim=None):
    B, W = beams.shape
    own = torch.arange(W, device=beams.device)
    p = torch.where((beams < 0) | (beams >= W), own, beams.long())
    src = (p + W * torch.arange(B, device=beams.device)[:, None]).reshape(-1)
    new = state.index_select(dim, src)
    if lengths is None:
        return new
    S = state.shape[length_dim]
    valid = torch.arange(S, device=beams.device) < lengths.long().repeat_interleave(W)[:, None]
    shape = [1] * state.dim()
    shape[dim], shape[length_dim] = B * W, S
    return torch.where(valid.view(shape), new, state)


def random_state(shape, dtype, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    bits = torch.randint(0, 256, (*shape, torch.empty(0, dtype=dtype).element_size()), generator=g, device=dev, dtype=torch.uint8)
    return bits.view(dtype).reshape(shape)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dtype", [BF, torch.uint8, torch.float32, torch.int64])
@pytest.mark.parametrize("B,W,shape,dim,length_dim", [
    (1, 1, (1, 8), 0, None), (1, 4, (4,), 0, None), (2, 3, (6, 5), 0, None), (3, 2, (2, 6, 7, 3), 1, None), (2, 4, (3, 8, 2, 33, 16), 1, 3),
    (2, 4, (8, 33, 2, 16), 0, 1), (1, 5, (5, 2, 9, 7), 0, 2), (4, 16, (64, 3, 40, 8), 0, 2), (2, 17, (34, 5, 8), 0, 1), (1, 64, (2, 64, 2, 9, 32), 1, 3),
    (2, 8, (2, 16, 2, 700, 64), 1, 3), (7, 33, (231, 3), 0, 1), (2, 2, (4, 6, 5), -3, -1)])
def test_reorder(dev, B, W, shape, dim, length_dim, dtype):
    g = torch.Generator(device=dev).manual_seed(1)
    d = dim % len(shape)
    for kind in ("any", "cycle", "same", "first", "out"):
        beams = torch.randint(W, (B, W), generator=g, device=dev)
        if kind == "cycle":
            beams = ((torch.arange(W, device=dev) + 1) % W).expand(B, W)
        elif kind == "same":
            beams = torch.arange(W, device=dev).expand(B, W)
        elif kind == "first":
            beams = torch.zeros_like(beams)
        elif kind == "out":
            beams[0, W // 2], beams[-1, -1] = -1, W
        state = random_state(shape, dtype, dev)
        if length_dim is None:
            lens = [None]
        else:
            S = shape[length_dim]
            lens = [torch.randint(0, S + 1, (B,), generator=g, device=dev), torch.full((B,), S, device=dev, dtype=torch.int32),
                    torch.tensor([0, S + 9, -5, 1] * B, device=dev)[:B], torch.ones(B, device=dev, dtype=torch.int32)]
        for lengths in lens:
            for b in (beams, beams.int()):
                s = state.clone()
                assert beam.reorder(s, b, dim, lengths, length_dim) is s
                ld = None if length_dim is None else length_dim % len(shape)
                assert same_bits(s, expected(state, b, d, lengths, ld)), kind


def test_reorder_of_many_states(dev):
    """One call for all layers, of two shapes, more than a launch takes."""
    beams = torch.tensor([[2, 0, 0], [1, 1, 2]], device=dev)
    lengths = torch.tensor([5, 9], device=dev)
    states = [random_state((6, 2, 12, 8 if i % 3 else 5), BF, dev, seed=i) for i in range(140)]
    before = [s.clone() for s in states]
    assert beam.reorder(states, beams, 0, lengths, 2) is states
    for s, b in zip(states, before):
        assert same_bits(s, expected(b, beams, 0, lengths, 2))


def test_reorder_of_unaligned_states_and_what_lies_around(dev):
    beams = torch.tensor([[1, 2, 0]], device=dev)
    room = random_state((2 + 3 * 4 * 10,), BF, dev)
    for off in (0, 1, 2):
        before = room.clone()
        state = room[off:off + 120].view(3, 4, 10)
        want = expected(state, beams, 0)
        beam.reorder(state, beams)
        assert same_bits(state, want)
        assert same_bits(room[:off], before[:off]) and same_bits(room[off + 120:], before[off + 120:])
    empty = torch.empty(3, 0, device=dev)
    beam.reorder([empty], beams)


def test_reorder_past_32_bit_offsets(dev):
    """A state of more than 2^32 bytes: its last layer."""
    state = torch.zeros(260, 4, 8, 2048, 128, device=dev, dtype=BF)
    assert state.numel() * 2 > 2 ** 32
    state[-1].copy_(torch.randn(4, 8, 2048, 128, device=dev))
    last = state[-1].clone()
    beams = torch.tensor([[3, 3, 0, 1]], device=dev)
    lengths = torch.tensor([2000], device=dev)
    beam.reorder(state, beams, 1, lengths, 3)
    assert same_bits(state[-1], expected(last, beams, 0, lengths, 2)) and not state[:-1].any()


# ---------------------------------------------------------------------------------------------
# how far lse may be off, and the order between beams with it
# ---------------------------------------------------------------------------------------------
LSE_OFF = 2.0 ** -18
"""With u = 2^-24 and V up to 2^20. A term exp(t), t the distance to its chunk's largest and that chunk's to the row's: t, its product with log2 e and that
constant are rounded, 2.23 u |t|, and the mean of |t| weighed by the terms is at most the w with w e^(w + 1) = V, 10.6: 23.7 u. Two exponentials of 1 ulp, 2 u
each, and their product: 5 u. Sums of 8 in a lane and of four such, then of 64 lanes and 4 waves: 9 + 8 u. 46 u in all, below 64 u = 2^-18."""


def check_bounds(logits, scores, n):
    """Candidates of two beams within 2 LSE_OFF may come in either order, all others and those of one beam may not."""
    got, beams, tokens = beam.select(logits, scores, n)
    v, W = values(logits, scores), scores.shape[1]
    best, at = torch.sort(v, dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    flat = (beams * (v.shape[1] // W) + tokens).cpu()
    mine, other = torch.gather(v, 1, flat), flat != at
    assert ((mine - best).abs()[other] <= 2 * LSE_OFF).all()
    assert all(len(set(r)) == n for r in flat.tolist())
    for row, b in zip(mine, beams.cpu()):
        for w in range(W):
            assert (row[b == w].diff() <= 0).all()
    g, fine = got.double().cpu(), mine.isfinite()
    assert ((g - mine).abs()[fine] <= LSE_OFF + 2.0 ** -24 * mine.abs()[fine]).all()
    assert (got[:, :-1] >= got[:, 1:]).all()
    return got, beams, tokens


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("V", [700, 20001, 151936, 1 << 20])
@pytest.mark.parametrize("B,W,n", [(6, 2, 4), (5, 6, 3), (3, 6, 12), (2, 17, 20)])
def test_one_peak_over_a_floor(dev, B, W, n, V, dtype):
    """Equal logits 11 to 12 below the largest, another floor for every beam: the errors of their exponentials are the same and add up.
    Scores that put all beams' peaks next to each other."""
    g = torch.Generator(device=dev).manual_seed(V + W)
    for i in range(3):
        logits = (torch.randint(0, 17, (B * W, 1), generator=g, device=dev) / 16).expand(B * W, V).contiguous()
        if i == 2:  # a beam's own noise over its floor
            logits += torch.randn(B * W, V, generator=g, device=dev) * 0.25
        logits[torch.arange(B * W, device=dev), torch.randint(V, (B * W,), generator=g, device=dev)] = 12.0
        logits = logits.to(dtype)
        lse = torch.logsumexp(logits.double().cpu(), -1).view(B, W)
        check_bounds(logits, (lse - 12.5 - torch.rand(B, 1, dtype=torch.float64)).float().to(dev), n)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("B,W,V,n", [(1, 4, 151936, 8), (8, 8, 151936, 16), (3, 5, 8191, 10), (16, 32, 2048, 64), (1, 64, 40000, 64), (64, 4, 999, 8)])
def test_drawn_logits_within_the_bound(dev, B, W, V, n, dtype):
    for seed in range(4):
        check_bounds(*make(dev, B, W, V, dtype, seed=100 + seed), n)


def test_equal_beams_beside_others(dev):
    """Copies of a beam with its score: equal sums, so each token's candidates in the order of the beams."""
    logits, scores = make(dev, 3, 6, 9000, torch.float32, seed=70)
    logits = logits.view(3, 6, -1)
    logits[:, 3], logits[:, 5] = logits[:, 1], logits[:, 1]
    scores[:, 3], scores[:, 5] = scores[:, 1], scores[:, 1]
    _, beams, tokens = check_bounds(logits, scores, 18)
    for b, t in zip(beams.tolist(), tokens.tolist()):
        first = [t[i] for i in range(18) if b[i] == 1]
        copies = [(t[i], b[i]) for i in range(18) if b[i] in (1, 3, 5)]
        want = [(x, w) for x in first for w in (1, 3, 5)]
        assert copies == want[:len(copies)]


def test_reorder_of_short_lengths_in_a_large_room(dev):
    """A static cache of 32,768 positions of which a few hundred are in use: only those move."""
    for W in (4, 8, 16, 20):
        state = random_state((2 * W, 2, 32768, 64), BF, dev, seed=W)
        beams = torch.randint(W, (2, W), device=dev, generator=torch.Generator(device=dev).manual_seed(W))
        lengths = torch.tensor([512, 3], device=dev)
        want = expected(state, beams, 0, lengths, 2)
        beam.reorder(state, beams, 0, lengths, 2)
        assert same_bits(state, want)

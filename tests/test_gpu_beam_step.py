"""A decode step of several requests with beams, each request with its own adapter, as a server would run it on these
kernels: norm -> projection + adapters -> ... -> final norm -> lm head -> selection -> caches reordered. Each operator's
result is checked against the package's separate calls or its own formula on the same operands, then the whole step is
captured and its replays, with new tokens and caches, are compared with eager steps."""

import pytest
import torch

from kernels import beam, fp8, lmhead, lora, mxfp4, norm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
H, I, V, B, W, S = 512, 768, 2048, 3, 4, 9  # hidden, intermediate, vocabulary, requests, beams, cache positions
PARTS = [H, 128, 128]
M = B * W


class Model:
    """One layer (no attention: its rows of V stand for it) and a head, on FP8 or MXFP4 weights."""

    def __init__(self, dev, kind):
        g = torch.Generator(device=dev).manual_seed(0)

        def w(n, k):
            return (torch.randn(n, k, generator=g, device=dev) * k ** -0.5).to(BF)

        quantize = fp8.quantize if kind == "fp8" else mxfp4.quantize
        self.kind = kind
        self.embed = w(V, H)
        self.qkv, self.o, self.gu, self.down = (quantize(w(n, k)) for n, k in ((sum(PARTS), H), (H, 128), (2 * I, H), (H, I)))
        self.head = quantize(self.embed)
        self.ln = [(1 + 0.1 * torch.randn(H, generator=g, device=dev)).to(BF) for _ in range(3)]
        self.ranks, self.scales = [16, 8], [0.5, 1.25]
        self.sets, self.pairs = {}, {}
        for name, k, parts in (("qkv", H, PARTS), ("gu", H, [I, I]), ("down", I, [H])):
            self.sets[name] = lora.Adapters(k, parts, 16, 2, dev)
            self.pairs[name] = []
            for i, r in enumerate(self.ranks):
                pairs = [(w(r, k), w(n, r)) for n in parts]
                self.sets[name].load(i, pairs, self.scales[i])
                self.pairs[name].append(pairs)

    def norm(self, x, delta, i):
        if self.kind == "fp8":
            res, x8, xs, h = norm.add_rmsnorm_fp8(x, delta, self.ln[i], with_h=True)
            return res, (x8, xs), h
        res, rows, h = norm.add_rmsnorm_mx(x, delta, self.ln[i], with_h=True)
        return res, rows, h

    def product(self, rows, q, split=1):
        if self.kind == "fp8":
            return fp8.gemv_fp8(rows[0], q, split, xs=rows[1])
        return mxfp4.gemv_mxfp4(rows, q, split)

    def rows(self, x):
        return fp8.quant_rows(x) if self.kind == "fp8" else mxfp4.quant_rows(x)

    def step(self, tokens, ids, scores, caches, lengths, seen=None):
        x = self.embed[tokens]
        x, rows, h = self.norm(x, None, 0)
        y = self.product(rows, self.qkv)
        qkv = lora.add(y, h, self.sets["qkv"], ids)
        v = qkv[:, H + 128:].contiguous()
        caches[0][torch.arange(M, device=x.device), lengths.repeat_interleave(W)] = qkv[:, H:H + 128]
        caches[1][torch.arange(M, device=x.device), lengths.repeat_interleave(W)] = v
        p = self.product(self.rows(v), self.o)[None].float()  # (K = 128: one partial)
        res, rows, h2 = self.norm(x, p, 1)
        gu = lora.add(self.product(rows, self.gu), h2, self.sets["gu"], ids)
        act = (torch.nn.functional.silu(gu[:, :I].float()).to(BF).float() * gu[:, I:].float()).to(BF)
        parts = self.product(self.rows(act), self.down, 2)  # split-K partials; the adapters go into the first
        before = parts[0].clone()
        lora.add(parts[0], act, self.sets["down"], ids, out=parts[0])
        res2, rows, h3 = self.norm(res, parts, 2)
        if self.kind == "fp8":
            _, logits = lmhead.lm_head_argmax(h3, self.head, return_logits=True)
        else:
            _, logits = lmhead.lm_head_argmax(rows, self.head, return_logits=True)
        new, beams, tokens = beam.select(logits, scores)
        kept = beams[:, :W]
        beam.reorder(caches, kept, dim=0, lengths=lengths + 1, length_dim=1)
        if seen is not None:
            seen.update(x=x, y=y, h=h, qkv=qkv, p=p, res=res, h2=h2, gu=gu, act=act, before=before, parts=parts, res2=res2, h3=h3, logits=logits,
                        beams=beams, rows=rows)
        return new[:, :W], kept, tokens[:, :W].reshape(-1)


def state(dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    tokens = torch.randint(V, (M,), generator=g, device=dev)
    ids = torch.tensor([0, -1, 1], device=dev).repeat_interleave(W)
    scores = -torch.rand(B, W, generator=g, device=dev)
    caches = [torch.randn(M, S, 128, generator=g, device=dev).to(BF) for _ in range(2)]
    lengths = torch.tensor([2, 5, 0], device=dev)
    return tokens, ids, scores, caches, lengths


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def low_rank(m, name, x, ids, y):
    """y with the adapters' products, in 64 bits."""
    out = y.double().clone()
    for i, pairs in enumerate(m.pairs[name]):
        rows, at = torch.nonzero(ids == i)[:, 0], 0
        for a, b in pairs:
            out[rows, at:at + b.shape[0]] += m.scales[i] * ((x[rows].double() @ a.double().t()) @ b.double().t())
            at += b.shape[0]
    return out


@pytest.mark.parametrize("kind", ["fp8", "mxfp4"])
def test_each_link(dev, kind):
    m, t = Model(dev, kind), {}
    tokens, ids, scores, caches, lengths = state(dev, 1)
    before = [c.clone() for c in caches]
    new, beams, chosen = m.step(tokens, ids, scores, caches, lengths, t)
    # the norms: the separate calls on their rows, bit for bit
    for x, d, i, h in ((t["x"], None, 0, "h"), (t["x"], t["p"], 1, "h2"), (t["res"], t["parts"], 2, "h3")):
        res, want = norm.add_rmsnorm(x, d, m.ln[i])
        assert same(want, t[h])
    assert same(t["res2"], (t["res"].float() + (t["parts"][0] + t["parts"][1]).to(BF).float()).to(BF))
    if kind == "fp8":
        x8, xs = fp8.quant_rows(t["h3"])
        assert same(t["rows"][0], x8) and same(t["rows"][1], xs)
        assert same(t["y"], fp8.gemv_fp8(t["h"], m.qkv))  # the product of the bf16 rows
    else:
        assert same(t["rows"].data, mxfp4.quant_rows(t["h3"]).data)
        assert same(t["y"], mxfp4.gemv_mxfp4(t["h"], m.qkv))
    # the adapters: half a step of bf16 and the sums' 2^-16 beside it; fp32: 2^-16 of the delta
    for name, x, y, out in (("qkv", t["h"], t["y"], t["qkv"]), ("gu", t["h2"], None, t["gu"]), ("down", t["act"], t["before"], t["parts"][0])):
        if y is None:
            continue
        want = low_rank(m, name, x, ids, y)
        step = 2.0 ** -8 if out.dtype is BF else 2.0 ** -23
        assert ((out.double() - want).abs() <= step * want.abs() + 2.0 ** -14 * (want - y.double()).abs().amax(1, keepdim=True)).all()
        assert same(out[ids < 0], y[ids < 0])
    # the choice: every kept continuation's score is its beam's plus its log probability, and the caches follow it
    lp = torch.log_softmax(t["logits"].double(), -1).view(B, W, V)
    tok = chosen.view(B, W)
    want = torch.gather(scores.double(), 1, beams) + lp[torch.arange(B, device=dev)[:, None], beams, tok]
    assert (new.double() - want).abs().max() < 2.0 ** -16
    assert (new[:, :-1] >= new[:, 1:]).all()
    best = (scores.double()[..., None] + lp).view(B, -1).amax(1)
    assert (new[:, 0].double() - best).abs().max() < 2.0 ** -16
    for c, b, row in zip(caches, before, (t["qkv"][:, H:H + 128], t["qkv"][:, H + 128:])):
        b[torch.arange(M, device=dev), lengths.repeat_interleave(W)] = row
        src = (beams + W * torch.arange(B, device=dev)[:, None]).reshape(-1)
        valid = torch.arange(S, device=dev) < (lengths + 1).repeat_interleave(W)[:, None]
        assert same(c, torch.where(valid[..., None], b[src], b))


@pytest.mark.parametrize("kind", ["fp8", "mxfp4"])
def test_captured_step(dev, kind):
    m = Model(dev, kind)
    tokens, ids, scores, caches, lengths = state(dev, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.step(tokens, ids, scores, [c.clone() for c in caches], lengths)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(tokens, ids, scores, caches, lengths)
    for seed in range(3, 7):
        new = state(dev, seed)
        perm = torch.randperm(B, device=dev)
        new[1].copy_(new[1].view(B, W)[perm].reshape(-1))
        for a, b in zip((tokens, ids, scores, *caches, lengths), (*new[:3], *new[3], new[4])):
            a.copy_(b)
        graph.replay()
        want = m.step(*new)
        for a, b in zip((*out, *caches), (*want, *new[3])):
            assert same(a, b)


@pytest.mark.parametrize("kind", ["fp8", "mxfp4"])
def test_first_residual_and_gate_up(dev, kind):
    """The links between the attention's output and the activation: the residual by its formula, gate_up's adapters in 64 bits beside the
    product of the same rows."""
    m, t = Model(dev, kind), {}
    tokens, ids, scores, caches, lengths = state(dev, 3)
    m.step(tokens, ids, scores, caches, lengths, t)
    assert same(t["res"], (t["x"].float() + t["p"][0].to(BF).float()).to(BF))
    y = m.product(m.rows(t["h2"]), m.gu)
    want, got = low_rank(m, "gu", t["h2"], ids, y), t["gu"]
    assert not torch.equal(got, y) and same(got[ids < 0], y[ids < 0])
    assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * (want - y.double()).abs().amax(1, keepdim=True)).all()
    act = (torch.nn.functional.silu(got[:, :I].float()).to(BF).float() * got[:, I:].float()).to(BF)
    assert same(t["act"], act)

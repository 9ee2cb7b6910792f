"""Low-rank adapters of many requests at once, beside one shared projection (HIP kernels k_lora_down and k_lora_up of
libkrq.so; the reference has no counterpart):

  out[m] = y[m] + s_i B_i (A_i x[m]),   i = ids[m]

y [M, N] is what linear_fp8, gemv, gemv_fp8 or linear_mxfp4 gave for the rows x [M, K] (the bf16 rows, as norm.add_rmsnorm
or add_rmsnorm_fp8(with_h=True) writes them), bf16 or fp32; a split-K product's partials take the adapters in one of
them: add(p[0], x, adapters, ids, out=p[0]). Every row names its adapter, in any order, or none; sums are fp32, the result
is rounded once. A projection fused from several (QKV, [gate; up]) has one pair of factors per part. Decode and
prefill take the same call, two launches; rows and ids may change between replays of a captured one.
"""

import functools

import torch

from . import _lib as L
from . import mxfp4 as _mx

MAX_PARTS, MAX_RANK, MAX_ROW = 8, 256, 1 << 22


class Adapters:
    """The adapters of one projection [N, K], in `slots` slots of up to `rank` ranks (rounded up to 16).
    K % 16 == 0; n: N, or the columns of each part of a fused projection in order (at most 8 parts).
    A slot holds a pair of factors for every part, with a rank of its own: a call reads what the slots in use hold, not
    `rank`. Slots start empty (rank 0), and an empty slot adds nothing. load and clear write into the same memory on the current stream, so
    that captured calls see them; they must not run beside a call that reads the slot."""

    def __init__(self, K, n, rank, slots, device):
        self.parts = [int(n)] if isinstance(n, int) else [int(p) for p in n]
        self.K, self.N, self.slots = int(K), sum(self.parts), int(slots)
        if not 16 <= self.K < MAX_ROW or self.K % 16:
            raise ValueError(f"K={K} must be a positive multiple of 16 under 2^22")
        if not 1 <= len(self.parts) <= MAX_PARTS or min(self.parts) < 1:
            raise ValueError(f"n={n}: 1 to {MAX_PARTS} parts of positive size")
        if not 1 <= rank <= MAX_RANK:
            raise ValueError(f"rank={rank} (1 to {MAX_RANK})")
        if not 1 <= self.slots < 1 << 23:
            raise ValueError(f"slots={slots}")
        self.rank = (int(rank) + 15) // 16 * 16
        # a slot's A: for each part, 16 ranks and 64 k the kernel's operands in lane order (lane 16 g + j: rank j, k = 16 g + 8 e
        # .. + 7), zeros past its rank and past K; its B: for each 16 columns of a part and 32 ranks the same (lane 16 g + j:
        # column j, ranks 8 g .. + 7; 32 lanes of an odd last 16 ranks), zeros past its rank and past the part
        self.a = torch.zeros((self.slots, len(self.parts), self.rank // 16, -(-self.K // 64), 2, 4, 16, 8), device=device,
                             dtype=torch.bfloat16)
        self._tiles = [-(-p // 16) for p in self.parts]
        self.b = torch.zeros((self.slots, sum(self._tiles) * 16 * self.rank), device=device, dtype=torch.bfloat16)
        self.ranks = torch.zeros((self.slots,), device=device, dtype=torch.int32)  # the parts' largest, by which a slot's factors lie
        self.part_ranks = torch.zeros((self.slots, len(self.parts)), device=device, dtype=torch.int32)
        self.scales = torch.zeros((self.slots,), device=device, dtype=torch.float32)
        self._set_n()

    def _set_n(self):
        self._n = (L.ctypes.c_int64 * len(self.parts))(*self.parts)  # the entry point's argument

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k != "_n"}

    def __setstate__(self, state):
        self.__dict__.update(state)
        if "part_ranks" not in state:  # (saved with one rank for all parts of a slot)
            self.part_ranks = self.ranks[:, None].repeat(1, len(self.parts))
        self._set_n()

    def _slot(self, slot):
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} of {self.slots}")
        return slot

    @torch.no_grad()
    def load(self, slot, pairs, scale=1.0):
        """Put an adapter into a slot: pairs, for each part its (A [r, K], B [part's columns, r]), rounded to bf16, or None where the
        adapter leaves the part alone; a single (A, B) for a projection of one part. Parts may differ in r, which is at most
        the rank the Adapters were made for (each then takes the largest's memory; its sum is over its own ranks). scale: the adapter's alpha / r."""
        slot = self._slot(slot)
        if len(self.parts) == 1 and len(pairs) == 2 and all(isinstance(t, torch.Tensor) for t in pairs):
            pairs = [pairs]
        if len(pairs) != len(self.parts):
            raise ValueError(f"{len(pairs)} pairs for {len(self.parts)} parts")
        own = []
        for p, n in zip(pairs, self.parts):
            if p is not None:
                a, b = p
                if a.dim() != 2 or b.dim() != 2 or a.shape[1] != self.K or b.shape[0] != n or a.shape[0] != b.shape[1]:
                    raise ValueError(f"A {tuple(a.shape)} and B {tuple(b.shape)} do not match [r, {self.K}] and [{n}, r]")
                if not 1 <= a.shape[0] <= self.rank:
                    raise ValueError(f"rank {a.shape[0]} (1 to {self.rank})")
            own.append(0 if p is None else p[0].shape[0])
        rank = max(own)
        if rank == 0:  # (no part has a pair)
            self.clear(slot)
            return
        r16 = (rank + 15) // 16 * 16
        packed = self.b[slot, :sum(self._tiles) * 16 * r16].view(-1, 16 * r16)
        full = r16 // 32 * 32  # ranks of whole steps
        for i, (p, n, cols) in enumerate(zip(pairs, self.parts, packed.split(self._tiles))):
            tiles = self.a[slot, i, :r16 // 16]
            if p is None:
                tiles.zero_()
                cols.zero_()
                continue
            # [rank tile, j, step, g, e, 8] -> [rank tile, step, e, g, j, 8]
            a = self._whole(p[0], r16, tiles.shape[1] * 64).view(r16 // 16, 16, -1, 4, 2, 8)
            tiles.copy_(a.permute(0, 2, 4, 3, 1, 5))
            # [tile, j, step, g, 8] -> [tile, step, g, j, 8]
            b = self._whole(p[1], cols.shape[0] * 16, r16).view(-1, 16, r16)
            if full:
                cols[:, :16 * full].view(-1, full // 32, 4, 16, 8).copy_(b[:, :, :full].view(-1, 16, full // 32, 4, 8).permute(0, 2, 3, 1, 4))
            if full < r16:
                cols[:, 16 * full:].view(-1, 2, 16, 8).copy_(b[:, :, full:].view(-1, 16, 2, 8).permute(0, 2, 1, 3))
        self.scales[slot] = float(scale)
        self.ranks[slot] = rank
        for i, r in enumerate(own):
            self.part_ranks[slot, i] = r

    def _whole(self, t, rows, cols):
        """t in bf16 on the slots' device, with zeros up to [rows, cols]."""
        if t.shape == (rows, cols):
            return t.to(self.a.device, torch.bfloat16).contiguous()
        w = torch.zeros((rows, cols), device=self.a.device, dtype=torch.bfloat16)
        w[:t.shape[0], :t.shape[1]] = t
        return w

    @torch.no_grad()
    def clear(self, slot):
        """Empty a slot."""
        self.ranks[self._slot(slot)] = 0
        self.part_ranks[slot] = 0


def _ld(t, cols):
    """The row stride of t [M, cols], None where its rows are not of consecutive values."""
    ld = t.stride(0) if t.shape[0] > 1 else cols
    return ld if (cols == 1 or t.stride(1) == 1) and ld >= cols else None


def _extent(t, ld):
    return t.data_ptr(), t.data_ptr() + ((t.shape[0] - 1) * ld + t.shape[1]) * t.element_size()


@functools.lru_cache(maxsize=4096)
def _ws_bytes(M, K, parts, rank):
    return L.lib().krq_lora_ws_bytes(M, K, parts, rank)


def add(y, x, adapters, ids, out=None):
    """y [M, N] bf16 or fp32, x [M, K] bf16, ids [M] int32 or int64 (a slot of adapters for each row; negative: none) ->
    y plus every row's adapter's product, in y's type. out: where it goes (default a new tensor; y itself adds in place).
    An id past the last slot gives a row of NaN. Rows of y, x and out may lie apart; x's are copied where they do not start on 16 bytes."""
    ad, dev = adapters, x.get_device()
    if dev < 0 or y.get_device() != dev or ids.get_device() != dev or ad.a.get_device() != dev or (
            out is not None and out.get_device() != dev):
        L.require_device(y, x, ids, out)
        raise ValueError(f"tensors on {x.device}, {y.device}, {ids.device}, {ad.a.device}" + ("" if out is None else f", {out.device}"))
    K, N, M = ad.K, ad.N, x.shape[0]
    if x.dtype is not torch.bfloat16 or x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"x must be bf16 [M, {K}], got {x.dtype} {tuple(x.shape)}")
    fp32 = y.dtype is torch.float32
    shape = y.shape
    if not (fp32 or y.dtype is torch.bfloat16) or len(shape) != 2 or shape[1] != N:
        raise ValueError(f"y must be bf16 or fp32 [M, {N}], got {y.dtype} {tuple(y.shape)}")
    wide = ids.dtype is torch.int64
    if not (wide or ids.dtype is torch.int32) or ids.dim() != 1 or ids.shape[0] != M or shape[0] != M:
        raise ValueError(f"ids {ids.dtype} {tuple(ids.shape)}, x {tuple(x.shape)} and y {tuple(y.shape)} do not match")
    ldx = K if x.is_contiguous() else _ld(x, K)
    ldy = N if y.is_contiguous() else _ld(y, N)
    px = x.data_ptr()
    if px & 15 or ldx is None or ldx & 7 or ldx >= MAX_ROW:
        x, ldx = x.clone(memory_format=torch.contiguous_format), K
        px = x.data_ptr()
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if out is None:
        if ldy is None:
            y, ldy = y.contiguous(), N
        out, ldo = torch.empty_like(y) if ldy == N else y.new_empty((M, N)), N
    else:
        ldo = _ld(out, N) if out.dim() == 2 and out.dtype is y.dtype and out.shape == (M, N) else None
        if ldo is None:
            raise ValueError(f"out must be {y.dtype} [{M}, {N}] with rows of consecutive values, got {out.dtype} {tuple(out.shape)} "
                             f"strides {out.stride()}")
        if ldy is None:
            y, ldy = y.contiguous(), N
        if M:
            o0, o1 = _extent(out, ldo)
            for t, ld in ((y, ldy), (x, ldx)):
                if t is y and o0 == y.data_ptr() and ldo == ldy:
                    continue
                a, b = _extent(t, ld)
                if o0 < b and a < o1:
                    raise ValueError("out overlaps an input (it may be y itself)")
    if M == 0:
        return out
    parts = len(ad.parts)
    nbytes = _ws_bytes(M, K, parts, ad.rank)
    ws = x.new_empty((nbytes + 1) // 2)
    _mx._call(dev, "krq_lora_add_parts", px, ldx, ids.data_ptr(), wide, ad.a.data_ptr(), ad.b.data_ptr(), ad.ranks.data_ptr(),
              ad.part_ranks.data_ptr(), ad.scales.data_ptr(), ad.slots, M, K, ad._n, parts, ad.rank, y.data_ptr(), ldy, out.data_ptr(), ldo, fp32, ws.data_ptr(), nbytes)
    return out

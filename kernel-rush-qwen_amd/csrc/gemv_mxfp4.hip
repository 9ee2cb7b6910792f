// MXFP4 skinny GEMM / GEMV (M <= 32): y = x . w^T on microscaled blocks, w e2m1 in the operand tiles of
// mx_common.h, x in e4m3 or e2m1 blocks, fp32 accumulation in v_mfma_scale_f32_16x16x128_f8f6f4.
//
// The unit of work is a (row block, group): 16 weight rows x 512 k, four 1 KiB tiles and one dword of
// scales per lane, 4.25 KiB that a wave loads with five contiguous loads. A workgroup's waves deal the groups of its K split
// among them (wave, wave + waves, ...) and their sums meet in LDS in wave order, so a result does not depend on timing.
//
// k_gemv_mx_held: each wave holds its groups' activation operands in registers (GW groups, MT row tiles) for the whole launch, and the
// workgroup walks over sets of P row blocks (SwiGLU: a gate block and its up block), the next set's weights in flight.
// k_gemv_mx_stream: longer rows, more of them; activation tiles are loaded beside the weights.
// k_gemv_mx_wide: many row blocks of not too long rows; the operands lie in LDS, a wave takes whole row blocks.
//
// Large launches are bound by the weights' read (the head at one row, 151,936 x 2,560: 33.4 us, 6.2 TB/s, the card's read rate;
// at 16 36.6), small ones by a launch and a round trip to memory (2,560 x 4,096, M = 1: 3.4 us; SwiGLU over 19,456 x 2,560, M = 5:
// 8.7, of which 1.3 round the rows), the streaming ones by the rows that every workgroup reads again from L2 (2,560 x
// 9,728, M = 32: 8.5 us, 311 KB of rows beside 83 KB of weights).
#include <algorithm>

#include "mx_common.h"

using namespace krq;

namespace {

constexpr int kHeldWaves = 10, kStreamWaves = 8;
// the held kernel's waves with MT row tiles of operands (two: 64 registers of e4m3 operands a group)
constexpr int held_waves(int MT) { return MT == 1 ? kHeldWaves : 8; }
constexpr int kMxSplitMax = 64;
// A held launch has a workgroup per set up to 512 sets, above that at most one per compute unit (a few more sets each than
// units would leave some units with twice the work). us, M = 1 on cold weights: 6,144 x 2,560 (384 sets) in 192 workgroups
// 4.58, 384 4.14; SwiGLU over 19,456 x 2,560 (608) in 203 7.57, 304 10.4, 608 9.3; 18,000 x 6,400 (563) in 188 13.7, 282 17.0,
// 563 15.4; the lm head (4,748) in 250 39.5, 475 40.6, 950 45.0.
// One over the units, 257 against 171 (513 sets) or 205 (1,025): the head over 16,416 x 2,560, M = 4 13.4 / 10.8, over 32,800 19.3 /
// 14.3, SwiGLU over 32,800 x 2,560 13.8 / 10.3, 8,208 x 10,240 in two splits 12.3 / 9.8; a plain product, whose workgroups are small
// enough for two to a unit, 8,208 x 2,560 5.0 / 5.3.
constexpr int kHeldOnce = 512, kHeldMost = 256;

// acc += A (16 rows) . B (16 weight rows) over 128 k, scale byte t of sa and sb (t a constant after unrolling). A: e2m1 or
// e4m3, B: e2m1.
template <int ELEM, int T>
KRQ_DEV v4f mx_mfma(v8i a, uint4 b, v4f acc, uint32_t sa, uint32_t sb) {
  constexpr int fa = ELEM == KRQ_MX_E2M1 ? 4 : 0;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, pack_v8i(b, zero4()), acc, fa, 4, T, static_cast<int>(sa), T,
                                                          static_cast<int>(sb));
}
template <int ELEM>
KRQ_DEV v4f mx_mfma(int t, v8i a, uint4 b, v4f acc, uint32_t sa, uint32_t sb) {
  return t == 0 ? mx_mfma<ELEM, 0>(a, b, acc, sa, sb) : t == 1 ? mx_mfma<ELEM, 1>(a, b, acc, sa, sb)
         : t == 2 ? mx_mfma<ELEM, 2>(a, b, acc, sa, sb) : mx_mfma<ELEM, 3>(a, b, acc, sa, sb);
}

// The same with the weights first: a lane's sums are four columns of a row.
template <int ELEM, int T>
KRQ_DEV v4f mx_mfma_w(uint4 w, v8i x, v4f acc, uint32_t sw, uint32_t sx) {
  constexpr int fx = ELEM == KRQ_MX_E2M1 ? 4 : 0;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(pack_v8i(w, zero4()), x, acc, 4, fx, T, static_cast<int>(sw), T,
                                                          static_cast<int>(sx));
}
template <int ELEM>
KRQ_DEV v4f mx_mfma_w(int t, uint4 w, v8i x, v4f acc, uint32_t sw, uint32_t sx) {
  return t == 0 ? mx_mfma_w<ELEM, 0>(w, x, acc, sw, sx) : t == 1 ? mx_mfma_w<ELEM, 1>(w, x, acc, sw, sx)
         : t == 2 ? mx_mfma_w<ELEM, 2>(w, x, acc, sw, sx) : mx_mfma_w<ELEM, 3>(w, x, acc, sw, sx);
}

struct MxArgs {
  const uint8_t* x;    // bf16 rows, or tiles
  const uint8_t* xs;   // the tiles' scales
  const uint8_t* w;    // tiles
  const uint8_t* ws;   // their scales
  void* out;           // bf16 [M, NO], fp32 [splits][M][NO], or the logits (may be null)
  Best* cand;          // argmax candidates [M][workgroups][row blocks of a set]
  int64_t ldx;         // bf16 rows' stride
  int64_t NO;          // output columns
  int M, K, KT, groups, nrb, sets, nw;  // nrb: row blocks of the output; sets of P of them; waves (the block's size, which
                                        // the compiler would load from memory behind every load in flight)
};

// MODE: KRQ_OUT_BF16, KRQ_OUT_PARTIAL (blockIdx.y: the split), KRQ_OUT_SWIGLU, kOutArgmax.
// The row blocks of a set: P adjacent ones (past the last: the last again), or SwiGLU's gate block and its up block.
template <int MODE, int P>
KRQ_DEV int row_block(const MxArgs& a, int set, int p) {
  return MODE == KRQ_OUT_SWIGLU ? set + p * a.nrb : min(set * P + p, a.nrb - 1);
}

// Sums the waves' accumulators of a set, red [nw][P][MT][256], in wave order and writes its outputs; every thread of the
// workgroup calls it, and takes the same rows and columns of each set. kOutArgmax: best holds the thread's largest
// logits so far (its columns come in rising order), for at least kArgmaxWaves waves.
constexpr int kArgmaxWaves = 4;
template <int MT, int MODE, int P>
constexpr int best_count() { return MODE == kOutArgmax ? P * MT * 256 / (64 * kArgmaxWaves) : 1; }

template <int MT, int MODE, int P>
KRQ_DEV void finish(const MxArgs& a, const float* red, int set, int sp, Best* best) {
  constexpr int PO = MODE == KRQ_OUT_SWIGLU ? 1 : P;  // output row blocks
  static_assert(PO <= 2, "sets of one or two row blocks");
  const int rows = 16 * a.M;  // values of a row block: row v / 16, column v % 16
  auto one = [&](int v, Best* bst) {
    const int p = PO == 2 && v >= rows ? 1 : 0, w = v - p * rows, m = w >> 4;
    const int e = 256 * (m >> 4) + 64 * (m & 3) + 16 * ((m >> 2) & 3) + (w & 15);  // its place in an accumulator
    const int64_t n = ((int64_t)set * PO + p) * 16 + (w & 15);
    if (n >= a.NO) return;
    float y = 0.0f, up = 0.0f;
    for (int i = 0; i < a.nw; ++i) {
      y += red[(i * P + p) * MT * 256 + e];
      if (MODE == KRQ_OUT_SWIGLU) up += red[(i * P + 1) * MT * 256 + e];
    }
    if constexpr (MODE == kOutArgmax) {
      const uint16_t yb = f32_to_bf16(y);
      if (a.out) static_cast<uint16_t*>(a.out)[(int64_t)m * a.NO + n] = yb;
      const float l = bf16_to_f32(yb);
      if (better(l, static_cast<int>(n), bst->v, bst->i)) *bst = Best{l, static_cast<int>(n)};
    } else {
      if constexpr (MODE == KRQ_OUT_SWIGLU) y = y / (1.0f + expf(-y)) * up;
      if constexpr (MODE == KRQ_OUT_PARTIAL) static_cast<float*>(a.out)[((int64_t)sp * a.M + m) * a.NO + n] = y;
      else static_cast<uint16_t*>(a.out)[(int64_t)m * a.NO + n] = f32_to_bf16(y);
    }
  };
  if constexpr (MODE == kOutArgmax) {
#pragma unroll
    for (int q = 0; q < best_count<MT, MODE, P>(); ++q) {
      const int v = static_cast<int>(threadIdx.x) + q * 64 * a.nw;
      if (v < PO * rows) one(v, &best[q]);
    }
  } else {
    for (int v = threadIdx.x; v < PO * rows; v += 64 * a.nw) one(v, nullptr);
  }
}

template <int MT, int MODE, int P>
KRQ_DEV void no_best(Best* best) {
#pragma unroll
  for (int q = 0; q < best_count<MT, MODE, P>(); ++q) best[q] = Best{-INFINITY, 0x7fffffff};
}

// the threads' largest logits, folded over the sixteen lanes of a row (which share it: 16 divides a row block's values)
template <int MT, int MODE, int P>
KRQ_DEV void write_best(const MxArgs& a, Best* best) {
  if constexpr (MODE == kOutArgmax) {
#pragma unroll
    for (int q = 0; q < best_count<MT, MODE, P>(); ++q) {
      Best b = best[q];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        const Best c = shfl_best(b, o);
        if (better(c.v, c.i, b.v, b.i)) b = c;
      }
      const int v = static_cast<int>(threadIdx.x) + q * 64 * a.nw, rows = 16 * a.M;
      if (v < P * rows && (v & 15) == 0)
        a.cand[((int64_t)((v >= rows ? v - rows : v) >> 4) * gridDim.x + blockIdx.x) * P + (v >= rows ? 1 : 0)] = b;
    }
  }
}

// XSRC: where the activations come from. 0: tiles (MT of them). 1 or 4: bf16 rows (one; at most KRQ_MX_BF16_ROWS, in
// chunks of four), rounded here: the 512 k of a group are one 16-byte load per row, the four lanes of a quad hold a
// block, and the wave's own region of LDS turns them into operands, without a launch or a barrier before the product.
// Lanes of rows past the last hold zeros (or, XSRC 1, the row: nobody reads their sums).
template <int ELEM, int XSRC, int MT, int MODE, int P, int GW>
__global__ __launch_bounds__(held_waves(MT) * 64) void k_gemv_mx_held(const MxArgs a) {
  static_assert(XSRC == 0 || MT == 1, "rows rounded here: one row tile");
  static_assert(MODE != KRQ_OUT_SWIGLU || P == 2, "SwiGLU: a gate and an up row block");
  constexpr int AB = ELEM == KRQ_MX_E2M1 ? 1 : 2;  // 16-byte loads per activation tile
  constexpr int D = P * GW <= 2 ? 2 : 1;           // sets in flight
  constexpr int kEl = ELEM == KRQ_MX_E2M1 ? 256 : 512, kRow = kEl + 16, kRows = XSRC == 4 ? 4 : 1;
  // sums [2][waves][P][MT][256]; at first the rows' regions, per wave kRows x (a group's elements, linear in k; 16 scale bytes)
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)), nw = a.nw;
  const int splits = gridDim.y, sp = blockIdx.y;
  const int g0 = a.groups * sp / splits, g1 = a.groups * (sp + 1) / splits;  // this split's groups
  const int n = (a.sets - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  // group j of the wave (past the split's last: it again, to load from; its products are skipped)
  auto group_of = [&](int j) { return min(g0 + wave + j * nw, g1 - 1); };

  uint4 av[GW][MT][4 * AB];
  uint32_t asc[GW][MT];
  uint4 xv[GW][XSRC == 4 ? KRQ_MX_BF16_ROWS : 1];
  if constexpr (XSRC > 0) {
#pragma unroll
    for (int j = 0; j < GW; ++j) {
      const int k = min(group_of(j) * kMxGroup + 8 * lane, a.K - 8);
#pragma unroll
      for (int m = 0; m < (XSRC == 4 ? KRQ_MX_BF16_ROWS : 1); ++m)
        if (m < 4 || a.M > 4) xv[j][m] = ld16(a.x + 2 * (min(m, a.M - 1) * a.ldx + k));
    }
  } else {
#pragma unroll
    for (int j = 0; j < GW; ++j)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int s = group_of(j);
        asc[j][mt] = *reinterpret_cast<const uint32_t*>(a.xs + (((int64_t)mt * a.groups + s) * 64 + lane) * 4);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint8_t* q = a.x + (((int64_t)mt * a.KT + min(4 * s + t, a.KT - 1)) * (64 * AB) + lane) * 16;
#pragma unroll
          for (int h = 0; h < AB; ++h) av[j][mt][t * AB + h] = ld16(q + 1024 * h);
        }
      }
  }
  __builtin_amdgcn_sched_barrier(0);

  uint4 wv[D][GW][P][4];
  uint32_t wsc[D][GW][P];
  auto load = [&](int d, int i) {
    const int set = static_cast<int>(blockIdx.x + i * gridDim.x);
#pragma unroll
    for (int j = 0; j < GW; ++j) {
      const int s = group_of(j);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t rb = row_block<MODE, P>(a, set, p);
        wsc[d][j][p] = *reinterpret_cast<const uint32_t*>(a.ws + ((rb * a.groups + s) * 64 + lane) * 4);
#pragma unroll
        for (int t = 0; t < 4; ++t) wv[d][j][p][t] = ld16nt(a.w + ((rb * a.KT + min(4 * s + t, a.KT - 1)) * 64 + lane) * 16);
      }
    }
  };
  load(0, 0);
  if (D == 2 && n > 1) load(1, 1);
  __builtin_amdgcn_sched_barrier(0);

  if constexpr (XSRC > 0) {
    uint8_t* reg = smem + wave * (kRows * kRow);
#pragma unroll
    for (int j = 0; j < GW; ++j) {
#pragma unroll
      for (int t = 0; t < 4 * AB; ++t) av[j][0][t] = zero4();
      asc[j][0] = 0;
#pragma unroll
      for (int c = 0; c < (XSRC == 4 ? KRQ_MX_BF16_ROWS / 4 : 1); ++c) {
        if (4 * c >= a.M) break;
#pragma unroll
        for (int m = 0; m < kRows; ++m) {
          const uint4 v = sel4(group_of(j) * kMxGroup + 8 * lane < a.K, xv[j][4 * c + m]);
          const uint32_t code = mx_code<ELEM>(quad_absmax(v));
          uint8_t* p = reg + m * kRow;
          if constexpr (ELEM == KRQ_MX_E2M1) *reinterpret_cast<uint32_t*>(p + 4 * lane) = mx_quant8_e2m1(v, code);
          else *reinterpret_cast<uint2*>(p + 8 * lane) = mx_quant8_e4m3(v, code);
          // block lane / 4 = 4 t + g of the row: byte t of dword g
          if ((lane & 3) == 0) p[kEl + 4 * ((lane >> 2) & 3) + (lane >> 4)] = static_cast<uint8_t>(code);
        }
        // the wave reads only what it wrote: a wave's LDS operations complete in order
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        if (XSRC == 1 || ((r >> 2) == c && r < a.M)) {
          const uint8_t* p = reg + (r & (kRows - 1)) * kRow;
          asc[j][0] = *reinterpret_cast<const uint32_t*>(p + kEl + 4 * g);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            if constexpr (AB == 1) {
              av[j][0][t] = *reinterpret_cast<const uint4*>(p + 64 * t + 16 * g);
            } else {
              av[j][0][2 * t] = *reinterpret_cast<const uint4*>(p + 128 * t + 16 * g);
              av[j][0][2 * t + 1] = *reinterpret_cast<const uint4*>(p + 128 * t + 64 + 16 * g);
            }
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      }
    }
    barrier_lds();  // (the sums lie where the regions are)
  }

  float* red = reinterpret_cast<float*>(smem);
  Best best[best_count<MT, MODE, P>()];
  no_best<MT, MODE, P>(best);
  auto consume = [&](int d, int i) __attribute__((always_inline)) {
    v4f acc[P][MT];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[p][mt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < GW; ++j)
      if (g0 + wave + j * nw < g1) {
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (4 * group_of(j) + t < a.KT) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              const v8i A = pack_v8i(av[j][mt][t * AB], AB == 2 ? av[j][mt][t * AB + AB - 1] : zero4());
#pragma unroll
              for (int p = 0; p < P; ++p) acc[p][mt] = mx_mfma<ELEM>(t, A, wv[d][j][p][t], acc[p][mt], asc[j][mt], wsc[d][j][p]);
            }
          }
      }
    float* buf = red + (i & 1) * nw * P * MT * 256;  // (two: one barrier per set)
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int q = 0; q < 4; ++q) buf[((wave * P + p) * MT + mt) * 256 + q * 64 + lane] = acc[p][mt][q];
  };
  auto sums = [&](int i) {
    barrier_lds();
    finish<MT, MODE, P>(a, red + (i & 1) * nw * P * MT * 256, static_cast<int>(blockIdx.x + i * gridDim.x), sp, best);
  };
  int i = 0;
  if constexpr (D == 2) {
    for (; i + 3 < n; i += 2) {
      consume(0, i);
      load(0, i + 2);
      sums(i);
      consume(1, i + 1);
      load(1, i + 3);
      sums(i + 1);
    }
    if (n - i == 3) {
      consume(0, i);
      load(0, i + 2);
      sums(i);
      consume(1, i + 1);
      sums(i + 1);
      i += 2;
    }
    consume(0, i);
    sums(i);
    if (n - i == 2) {
      consume(1, i + 1);
      sums(i + 1);
    }
  } else {
    for (; i + 1 < n; ++i) {
      consume(0, i);
      load(0, i + 1);
      sums(i);
    }
    consume(0, i);
    sums(i);
  }
  write_best<MT, MODE, P>(a, best);
}

// MT row tiles of activations beside every set's weights; U groups of a wave in flight.
template <int ELEM, int MT, int MODE, int P, int U>
__global__ __launch_bounds__(kStreamWaves * 64) void k_gemv_mx_stream(const MxArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];  // sums [waves][P][MT][256]
  constexpr int AB = ELEM == KRQ_MX_E2M1 ? 1 : 2;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)), nw = a.nw;
  const int splits = gridDim.y, sp = blockIdx.y;
  const int g0 = a.groups * sp / splits, g1 = a.groups * (sp + 1) / splits;
  const int jc = g0 + wave < g1 ? (g1 - g0 - wave + nw - 1) / nw : 0;  // this wave's groups
  uint4 wv[U][P][4], av[U][MT][4 * AB];
  uint32_t wsc[U][P], asc[U][MT];
  // (loads past the wave's last group repeat it: every load is unconditional, the products are not)
  auto load = [&](int u, int j) {
    const int s = jc > 0 ? g0 + wave + min(j, jc - 1) * nw : g0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      asc[u][mt] = *reinterpret_cast<const uint32_t*>(a.xs + (((int64_t)mt * a.groups + s) * 64 + lane) * 4);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint8_t* q = a.x + (((int64_t)mt * a.KT + min(4 * s + t, a.KT - 1)) * (64 * AB) + lane) * 16;
#pragma unroll
        for (int h = 0; h < AB; ++h) av[u][mt][t * AB + h] = ld16(q + 1024 * h);
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int64_t rb = row_block<MODE, P>(a, blockIdx.x, p);
      wsc[u][p] = *reinterpret_cast<const uint32_t*>(a.ws + ((rb * a.groups + s) * 64 + lane) * 4);
#pragma unroll
      for (int t = 0; t < 4; ++t) wv[u][p][t] = ld16nt(a.w + ((rb * a.KT + min(4 * s + t, a.KT - 1)) * 64 + lane) * 16);
    }
  };
  v4f acc[P][MT];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[p][mt] = v4f{0.f, 0.f, 0.f, 0.f};
  auto consume = [&](int u, int j) {
    if (j >= jc) return;
    const int s = g0 + wave + j * nw;
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (4 * s + t < a.KT) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const v8i A = pack_v8i(av[u][mt][t * AB], AB == 2 ? av[u][mt][t * AB + AB - 1] : zero4());
#pragma unroll
          for (int p = 0; p < P; ++p) acc[p][mt] = mx_mfma<ELEM>(t, A, wv[u][p][t], acc[p][mt], asc[u][mt], wsc[u][p]);
        }
      }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, u);
  __builtin_amdgcn_sched_barrier(0);
  int j = 0;
  for (; j + U < jc; j += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      consume(u, j + u);
      load(u, j + U + u);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) consume(u, j + u);
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int q = 0; q < 4; ++q) red[((wave * P + p) * MT + mt) * 256 + q * 64 + lane] = acc[p][mt][q];
  barrier_lds();
  Best best[best_count<MT, MODE, P>()];
  no_best<MT, MODE, P>(best);
  finish<MT, MODE, P>(a, red, blockIdx.x, sp, best);
  write_best<MT, MODE, P>(a, best);
}

int sets_of(const MxArgs& a, int mode, int P) { return mode == KRQ_OUT_SWIGLU ? a.nrb : (a.nrb + P - 1) / P; }

typedef uint32_t v2u_any __attribute__((ext_vector_type(2), aligned(2)));  // 8 bytes at any element's address

// Many row blocks: the rows (bf16 ones rounded by every workgroup for itself) stay in LDS as operands, and a wave takes whole row
// blocks, so that it waits for nothing but its own weights, of which four groups are in flight on from row block to row block;
// no sums meet and no barrier holds the stream. Padding to whole groups is zero. Weights are the first operand here: a lane ends
// with four adjacent columns of row lane % 16. One workgroup per compute unit. us a call: 65,536 x 2,560, M = 16 21.6 (held) -> 17.8,
// M = 32 26.0 -> 22.4; 151,936 x 2,560, M = 1 42.3 -> 35.3 (5.9 TB/s); the head, M = 16 46.8 -> 42.4, M = 32 58.5 -> 50.2. Pairs of
// row blocks 45.4 and 53.4, sixteen waves with two groups each 45.0 and 51.7.
constexpr int kWideWaves = 8, kWideFlight = 4, kWideGroups = 7;  // (more groups: takes_wide)
template <int ELEM, bool BF16, int MT, int MODE>
__global__ __launch_bounds__(kWideWaves * 64) void k_gemv_mx_wide(const MxArgs a) {
  static_assert(!BF16 || MT == 1, "more than sixteen rows come rounded");
  static_assert(MODE == KRQ_OUT_BF16 || MODE == kOutArgmax, "outputs of a row block are final");
  constexpr int AB = ELEM == KRQ_MX_E2M1 ? 1 : 2, TB = 1024 * AB, W = kWideWaves, U = kWideFlight, B = 4;
  __shared__ __align__(16) uint8_t lx[MT * kWideGroups * 4 * TB];
  __shared__ __align__(16) uint8_t lsc[MT * kWideGroups * 256];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int G = a.groups, tiles = MT * G * 4;
  const int first = static_cast<int>(blockIdx.x) * W + wave, stride = static_cast<int>(gridDim.x) * W;
  const int total = first < a.nrb ? ((a.nrb - first + stride - 1) / stride) * G : 0;  // this wave's groups

  // tile i of the rows: row tile i / (4 G), tile i % (4 G) of it; lanes as k_mx_quant's
  const int kc = 8 * r, b = kc >> 5;
  uint4 xv[B][BF16 ? 4 : AB];
  auto load_rows = [&](int i0) {
#pragma unroll
    for (int q = 0; q < B; ++q) {
      const int i = min(i0 + q * W, tiles - 1), mt = i / (4 * G), t = i - mt * 4 * G;
      if constexpr (BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xv[q][j] = ld16(a.x + 2 * (min(16 * mt + 4 * j + g, a.M - 1) * a.ldx + min(kMxTile * t + kc, a.K - 8)));
      } else {
#pragma unroll
        for (int h = 0; h < AB; ++h) xv[q][h] = ld16(a.x + (((int64_t)mt * a.KT + min(t, a.KT - 1)) * (64 * AB) + lane) * 16 + 1024 * h);
      }
    }
  };
  auto keep_rows = [&](int i0) {
#pragma unroll
    for (int q = 0; q < B; ++q) {
      const int i = i0 + q * W;
      if (i >= tiles) break;
      const int mt = i / (4 * G), t = i - mt * 4 * G;
      if constexpr (BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 4 * j + g;
          const uint4 v = sel4(16 * mt + row < a.M && kMxTile * t + kc < a.K, xv[q][j]);
          const uint32_t code = mx_code<ELEM>(quad_absmax(v));
          if ((lane & 3) == 0) lsc[(((i >> 2) * 64) + 16 * b + row) * 4 + (i & 3)] = static_cast<uint8_t>(code);
          if constexpr (ELEM == KRQ_MX_E2M1)
            *reinterpret_cast<uint32_t*>(lx + i * TB + 16 * (16 * b + row) + 4 * (lane & 3)) = mx_quant8_e2m1(v, code);
          else
            *reinterpret_cast<uint2*>(lx + i * TB + 1024 * (kc >> 6) + 16 * (16 * ((kc & 63) >> 4) + row) + (kc & 15)) =
                mx_quant8_e4m3(v, code);
        }
      } else {
#pragma unroll
        for (int h = 0; h < AB; ++h) *reinterpret_cast<uint4*>(lx + i * TB + 1024 * h + 16 * lane) = sel4(t < a.KT, xv[q][h]);
      }
    }
  };

  uint4 wv[U][4];
  uint32_t wsc[U];
  int lrb = first, lg = 0;  // the loading end
  auto load = [&](int u) {
    const int64_t rb = min(lrb, a.nrb - 1);
    wsc[u] = *reinterpret_cast<const uint32_t*>(a.ws + ((rb * G + lg) * 64 + lane) * 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) wv[u][t] = ld16nt(a.w + ((rb * a.KT + min(4 * lg + t, a.KT - 1)) * 64 + lane) * 16);
    if (++lg == G) {
      lg = 0;
      lrb += stride;
    }
  };
  load_rows(wave);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < U; ++u) load(u);  // (past the last: the last row block)
  __builtin_amdgcn_sched_barrier(0);
  keep_rows(wave);
  for (int i = wave + B * W; i < tiles; i += B * W) {
    load_rows(i);
    keep_rows(i);
  }
  if constexpr (!BF16)
    for (int i = threadIdx.x; i < MT * G * 64; i += 64 * W)
      *reinterpret_cast<uint32_t*>(lsc + 4 * i) = *reinterpret_cast<const uint32_t*>(a.xs + (int64_t)4 * i);
  barrier_lds();

  v4f acc[MT];
  Best best[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    acc[mt] = v4f{0.f, 0.f, 0.f, 0.f};
    best[mt] = Best{-INFINITY, 0x7fffffff};
  }
  int crb = first, cg = 0;  // the consuming end
  auto consume = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const uint32_t sx = *reinterpret_cast<const uint32_t*>(lsc + ((mt * G + cg) * 64 + lane) * 4);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint8_t* q = lx + ((mt * G + cg) * 4 + t) * TB + 16 * lane;
        const v8i x = pack_v8i(*reinterpret_cast<const uint4*>(q), AB == 2 ? *reinterpret_cast<const uint4*>(q + 1024 * (AB - 1)) : zero4());
        acc[mt] = mx_mfma_w<ELEM>(t, wv[u][t], x, acc[mt], wsc[u], sx);
      }
    }
    if (++cg < G) return;
    cg = 0;
    const int64_t n = (int64_t)crb * 16 + 4 * g;
    crb += stride;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int m = 16 * mt + r;
      const uint32_t y[2] = {pack_bf16x2(acc[mt][0], acc[mt][1]), pack_bf16x2(acc[mt][2], acc[mt][3])};
      acc[mt] = v4f{0.f, 0.f, 0.f, 0.f};
      uint16_t* o = static_cast<uint16_t*>(a.out) + m * a.NO + n;
      if (m < a.M && n + 4 <= a.NO) {
        if (MODE == KRQ_OUT_BF16 || a.out) *reinterpret_cast<v2u_any*>(o) = v2u_any{y[0], y[1]};
        if constexpr (MODE == kOutArgmax) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float l = as_f32(e & 1 ? y[e >> 1] & 0xffff0000u : y[e >> 1] << 16);
            if (better(l, static_cast<int>(n) + e, best[mt].v, best[mt].i)) best[mt] = Best{l, static_cast<int>(n) + e};
          }
        }
      } else if (MODE == KRQ_OUT_BF16 && m < a.M) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < a.NO) o[e] = static_cast<uint16_t>(y[e >> 1] >> (16 * (e & 1)));
      }
    }
  };
  int i = 0;
  for (; i + 2 * U <= total; i += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      consume(u);
      load(u);
    }
  }
  const int rem = total - i;  // fewer than 2 U groups
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < rem) {
      consume(u);
      if (U + u < rem) load(u);
    }
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (U + u < rem) consume(u);

  if constexpr (MODE == kOutArgmax) {  // over the lanes of a row, then over the waves
    __syncthreads();
    Best* red = reinterpret_cast<Best*>(lx);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      Best t = best[mt];
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) {
        const Best c = shfl_best(t, o);
        if (better(c.v, c.i, t.v, t.i)) t = c;
      }
      if (lane < 16) red[wave * (16 * MT) + 16 * mt + lane] = t;
    }
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < a.M) {
      Best t = red[threadIdx.x];
      for (int w = 1; w < W; ++w) {
        const Best c = red[w * (16 * MT) + threadIdx.x];
        if (better(c.v, c.i, t.v, t.i)) t = c;
      }
      a.cand[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = t;
    }
  }
}

// Row blocks of a set: the head takes pairs (151,936 x 2,560, single / pairs, us a call: M = 1 44.5 / 37.9, M = 16 55.3 / 46.3,
// M = 32 101 / 58), the other outputs single ones (19,456 x 2,560, M = 16 7.5 / 8.5; 65,536 x 2,560, M = 1 17.1 / 17.0).
constexpr int set_blocks(int mode) { return mode == KRQ_OUT_SWIGLU || mode == kOutArgmax ? 2 : 1; }

template <int ELEM, int XSRC, int MT, int MODE, int P, int GW>
int launch_held(MxArgs a, int splits, int nw, hipStream_t s) {
  a.sets = sets_of(a, MODE, P);
  a.nw = nw;
  const int most = (int64_t)a.sets * splits <= kHeldOnce ? a.sets : std::max(1, kHeldMost / splits);
  const int rounds = (a.sets + most - 1) / most, blocks = (a.sets + rounds - 1) / rounds;  // as many sets for each
  constexpr size_t row = (ELEM == KRQ_MX_E2M1 ? 256 : 512) + 16;
  const size_t smem = std::max((size_t)2 * nw * P * MT * 1024, XSRC > 0 ? nw * (XSRC == 4 ? 4 : 1) * row : 0);
  hipLaunchKernelGGL((k_gemv_mx_held<ELEM, XSRC, MT, MODE, P, GW>), dim3(blocks, splits), dim3(64 * nw), smem, s, a);
  return blocks * P;
}

template <int ELEM, int MT, int MODE, int P, int U>
int launch_stream(MxArgs a, int splits, int nw, hipStream_t s) {
  a.sets = sets_of(a, MODE, P);
  a.nw = nw;
  hipLaunchKernelGGL((k_gemv_mx_stream<ELEM, MT, MODE, P, U>), dim3(a.sets, splits), dim3(64 * nw), (size_t)nw * P * MT * 1024, s, a);
  return a.sets * P;
}

// Launches a mode; returns the row blocks that a split's workgroups take at a time (the head's candidates of a row). One row tile of
// at most 20 groups a split is held, more streams (stream / held, us a call: 2,560 x 9,728, M = 1 9.3 / 5.2, M = 16 9.4 / 9.1;
// SwiGLU over 19,456 x 6,400, M = 1 21.0 / 14.2).
template <int ELEM, int MODE>
int launch_mode(const MxArgs& a, bool bf16, int splits, hipStream_t s) {
  const int per = (a.groups + splits - 1) / splits;  // groups of the longest split
  const int gw = (per + kHeldWaves - 1) / kHeldWaves, least = MODE == kOutArgmax ? kArgmaxWaves : 1;
  const int nw = std::max((per + gw - 1) / gw, least);
  constexpr int P = set_blocks(MODE);
  // the head with two groups a wave: single row blocks, of which two sets are in flight (50,000 x 6,400, pairs / single, us a
  // call: M = 1 37.6 / 32.4, M = 16 45.8 / 38.3)
  constexpr int P2 = MODE == kOutArgmax ? 1 : P;
  if (a.M > 16 && per <= held_waves(2)) return launch_held<ELEM, 0, 2, MODE, P, 1>(a, splits, nw, s);
  if (gw <= 2 && a.M <= 16) {
    if (bf16 && a.M == 1)
      return gw == 1 ? launch_held<ELEM, 1, 1, MODE, P, 1>(a, splits, nw, s) : launch_held<ELEM, 1, 1, MODE, P2, 2>(a, splits, nw, s);
    if (bf16) return launch_held<ELEM, 4, 1, MODE, P, 1>(a, splits, nw, s);
    return gw == 1 ? launch_held<ELEM, 0, 1, MODE, P, 1>(a, splits, nw, s) : launch_held<ELEM, 0, 1, MODE, P2, 2>(a, splits, nw, s);
  }
  const int ns = std::max(std::min(per, kStreamWaves), least);
  // (two row tiles and single row blocks: two groups in flight 12.45 -> 11.1 us at 2,560 x 16,384, M = 32; with pairs of row
  // blocks registers run out, 15.2 -> 16.7 for SwiGLU over 16,384 x 6,144)
  return a.M <= 16 ? launch_stream<ELEM, 1, MODE, P, 2>(a, splits, ns, s) : launch_stream<ELEM, 2, MODE, P, P == 1 ? 2 : 1>(a, splits, ns, s);
}

// Where k_gemv_mx_wide takes a product: up to seven groups (65,536 x 4,096, held / wide, us a call: M = 5 27.0 / 28.1, M = 16
// 29.6 / 28.7, M = 32 32.6 / 35.4; the head over 64,000 x 3,584, M = 16 31.3 / 27.4), plain outputs from 32,768 columns (M = 5,
// K = 2,560: 16,384 8.4 / 8.6, 32,768 12.0 / 10.7), for a few rows from 65,536 (M = 4, K = 2,048: 32,768 9.4 / 9.7, 65,536
// 15.3 / 14.7), the head from 9 rows and 16,000 columns (16,000 x 2,560, M = 16 16.9 / 13.4, M = 32 22.0 / 18.4; fewer rows:
// 65,536 x 2,048, M = 4 17.8 / 18.5).
bool takes_wide(int64_t M, int64_t N, int64_t K, int mode) {
  if (mx_groups(K) > kWideGroups) return false;
  return mode == kOutArgmax ? M > 8 && N >= 16000 : mode == KRQ_OUT_BF16 && N >= (M > 4 ? 32768 : 65536);
}

template <int ELEM, int MODE>
int launch_wide(const MxArgs& a, bool bf16, hipStream_t s) {
  const int blocks = std::min((a.nrb + kWideWaves - 1) / kWideWaves, kHeldMost);
  const dim3 block(64 * kWideWaves);
  if (a.M > 16) hipLaunchKernelGGL((k_gemv_mx_wide<ELEM, false, 2, MODE>), dim3(blocks), block, 0, s, a);
  else if (bf16) hipLaunchKernelGGL((k_gemv_mx_wide<ELEM, true, 1, MODE>), dim3(blocks), block, 0, s, a);
  else hipLaunchKernelGGL((k_gemv_mx_wide<ELEM, false, 1, MODE>), dim3(blocks), block, 0, s, a);
  return blocks;
}

template <int MODE>
int launch_elem(const MxArgs& a, int elem, bool bf16, bool wide, int splits, hipStream_t s) {
  if constexpr (MODE == KRQ_OUT_BF16 || MODE == kOutArgmax)
    if (wide) return elem == KRQ_MX_E2M1 ? launch_wide<KRQ_MX_E2M1, MODE>(a, bf16, s) : launch_wide<KRQ_MX_E4M3, MODE>(a, bf16, s);
  return elem == KRQ_MX_E2M1 ? launch_mode<KRQ_MX_E2M1, MODE>(a, bf16, splits, s) : launch_mode<KRQ_MX_E4M3, MODE>(a, bf16, splits, s);
}

// bf16 rows that a launch of any N rounds itself (k_gemv_mx_wide: up to sixteen): one whose groups its waves hold, or a few over
// one group per wave. Rounded before /
// in the launch, us: SwiGLU over 19,456 x 2,560, M = 5 10.4 / 8.8, M = 8 10.4 / 8.8; 2,560 x 9,728, M = 1 9.0 / 5.2, M = 5
// (two groups per wave) 9.2 / 11.3.
bool rounds_rows(int64_t M, int64_t K, int split) {
  const int64_t per = (mx_groups(K) + split - 1) / split;
  return M == 1 ? per <= 2 * kHeldWaves : M <= KRQ_MX_BF16_ROWS && per <= kHeldWaves;
}

}  // namespace

namespace krq {

int64_t gemv_mx_rows_bytes(int x_kind, int elem, int64_t M, int64_t N, int64_t K, int split, int mode) {
  const bool in_launch = rounds_rows(M, K, split) || (M <= 16 && takes_wide(M, N, K, mode));
  return x_kind == KRQ_MX_X_BF16 && !in_launch ? mx_rows_bytes(elem, M, K) : 0;
}

// The checks and the launch of every product on MXFP4 weights of at most 32 rows (kOutArgmax: the head's).
int gemv_mx_run(const char* what, const void* x, const void* x_scale, int x_kind, int elem, int64_t ldx, const void* w,
                const void* w_scale, int64_t M, int64_t N, int64_t K, int split, int mode, void* ws, int64_t ws_bytes, void* out,
                Best* cand, int64_t* cands, void* stream) {
  KRQ_REQUIRE(x && w && w_scale && (out || mode == kOutArgmax), "%s: null pointer", what);
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "%s: bad element type %d", what, elem);
  KRQ_REQUIRE(x_kind == KRQ_MX_X_BF16 || x_kind == KRQ_MX_X_TILED, "%s: bad x_kind %d", what, x_kind);
  KRQ_REQUIRE(M >= 1 && M <= 32, "%s: M=%lld outside 1..32", what, (long long)M);
  KRQ_REQUIRE(N >= 1 && N <= 0x7fffffff - 64 && K >= kMxBlock && K % kMxBlock == 0 && K <= 0x3fffffff, "%s: shape N=%lld K=%lld (K a multiple of 32)", what,
              (long long)N, (long long)K);
  const int64_t rows = gemv_mx_rows_bytes(x_kind, elem, M, N, K, std::max(split, 1), mode);
  KRQ_REQUIRE(x_kind == KRQ_MX_X_BF16 || x_scale, "%s: tiled rows need their scales", what);
  KRQ_REQUIRE(x_kind != KRQ_MX_X_BF16 || (ldx >= K && ldx % 8 == 0), "%s: rows of x must start on 16 bytes (ldx=%lld)", what, (long long)ldx);
  KRQ_REQUIRE(aligned16(x) && aligned16(x_scale) && aligned16(w) && aligned16(w_scale) && aligned16(ws),
              "%s: x, w, their scales and ws must start on 16 bytes", what);
  KRQ_REQUIRE(rows == 0 || (ws && ws_bytes >= rows), "%s: bf16 rows need a workspace of %lld bytes", what, (long long)rows);
  const int groups = static_cast<int>(mx_groups(K));
  KRQ_REQUIRE(split >= 1 && split <= groups && split <= kMxSplitMax, "%s: split=%d of %d groups of 512", what, split, groups);
  KRQ_REQUIRE(split == 1 || mode == KRQ_OUT_PARTIAL, "%s: split=%d needs the partials output", what, split);
  const bool swiglu = mode == KRQ_OUT_SWIGLU;
  KRQ_REQUIRE(!swiglu || N % 32 == 0, "%s: SwiGLU needs N=%lld = 2 I with I %% 16 == 0", what, (long long)N);
  const bool wide = takes_wide(M, N, K, mode), bf16 = x_kind == KRQ_MX_X_BF16 && rows == 0;
  if (rows) {
    uint8_t* sc = (uint8_t*)ws + mx_rows_scale_at(elem, M, K);
    if (const int rc = krq_quant_mx_rows(x, M, K, ldx, elem, ws, sc, stream)) return rc;
    x = ws;
    x_scale = sc;
  }
  MxArgs a;
  a.x = (const uint8_t*)x;
  a.xs = (const uint8_t*)x_scale;
  a.w = (const uint8_t*)w;
  a.ws = (const uint8_t*)w_scale;
  a.out = out;
  a.cand = cand;
  a.ldx = ldx;
  a.NO = swiglu ? N / 2 : N;
  a.M = static_cast<int>(M);
  a.K = static_cast<int>(K);
  a.KT = static_cast<int>(mx_tiles(K));
  a.groups = groups;
  a.nrb = static_cast<int>((a.NO + 15) / 16);
  a.sets = a.nw = 0;
  hipStream_t s = (hipStream_t)stream;
  if (mode == KRQ_OUT_SWIGLU) launch_elem<KRQ_OUT_SWIGLU>(a, elem, bf16, wide, split, s);
  else if (mode == KRQ_OUT_PARTIAL) launch_elem<KRQ_OUT_PARTIAL>(a, elem, bf16, wide, split, s);
  else if (mode == kOutArgmax) *cands = launch_elem<kOutArgmax>(a, elem, bf16, wide, split, s);
  else launch_elem<KRQ_OUT_BF16>(a, elem, bf16, wide, split, s);
  return krq_check_launch(what);
}

}  // namespace krq

extern "C" int64_t krq_gemv_mxfp4_ws_bytes(int x_kind, int elem, int64_t M, int64_t K, int split) {
  if (M < 1 || M > 32 || K < 1 || split < 1 || (elem != KRQ_MX_E2M1 && elem != KRQ_MX_E4M3)) return -1;
  return x_kind == KRQ_MX_X_BF16 && !rounds_rows(M, K, split) ? mx_rows_bytes(elem, M, K) : 0;
}

extern "C" int krq_gemv_mxfp4(const void* x, const void* x_scale, int x_kind, int elem, int64_t ldx, const void* w_tiled,
                              const void* w_scale, int64_t M, int64_t N, int64_t K, int split, int mode, void* ws, int64_t ws_bytes,
                              void* out, void* stream) {
  KRQ_REQUIRE(mode == KRQ_OUT_BF16 || mode == KRQ_OUT_PARTIAL || mode == KRQ_OUT_SWIGLU, "gemv_mxfp4: bad mode %d", mode);
  return gemv_mx_run("gemv_mxfp4", x, x_scale, x_kind, elem, ldx, w_tiled, w_scale, M, N, K, split, mode, ws, ws_bytes, out, nullptr,
                     nullptr, stream);
}

// MXFP4 GEMM for prefill: out = bf16(x . w^T), x in e4m3 or e2m1 blocks, w in e2m1 blocks, both in the operand
// tiles of mx_common.h, fp32 accumulation on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// Persistent workgroups of W waves own BM x BN outputs, each wave BM / 2 x 2 BN / W of them, in 32 x 32 pieces. The
// stream of stages (a stage: T times 128 k, T tiles of every row block) runs on from one output tile into the next:
// direct loads bring a stage into one of NB LDS buffers, NB stages ahead of its use. A tile is stored in
// lane order, so each load copies one whole KiB, and each 16-byte LDS read takes runs of 256 bytes: no padding, no
// swizzle, no bank conflict of the elements, and no address arithmetic per lane. The scale bytes come a group of four
// stages at a time into a ring of their own, from which every product reads its byte (or two): sixteen lanes' rows of two row
// blocks lie 256 bytes apart there and conflict, 17 to 19% of the cycles that LDS is busy (27 to 32% of all).
//
// Fragment of 32 rows, half h of a tile (64 k): lane l holds row l % 32, that is row r = l % 16 of row block
// (l / 16) % 2, with c = l / 32
//   e2m1: k = 64 h + 32 c + 0..31, the 16 bytes of tile lane 16 (2 h + c) + r;
//   e4m3: k = 64 h + 16 c + 0..15 and 32 more, the bytes of tile lanes 16 c + r and 16 (c + 2) + r of KiB h;
// its scale byte is that of block 2 h + c. Weights are the instruction's first operand, so a lane ends with four
// adjacent columns of one row: element e of lane l is column 8 (e / 4) + 4 c + e % 4 of row l % 32.
//
// Large products are bound by the matrix cores at the card's power and by the burst of every round's stores: 4,096 x 19,456 x
// 2,560 with e4m3 rows takes 158 to 183 us (the cores 64% busy; 128 without loads, LDS reads and stores), 8,192^3 392 us (2.8
// PFLOP/s; e2m1 rows 251). Small ones are bound by their loads (1,000 x 2,560 x 9,728, e2m1 rows: 160 tiles on 256 units,
// 25.4 us, 19 without loads; 77 x 6,144 x 2,560: 7.9).
#include <algorithm>
#include <type_traits>

#include "mx_common.h"

using namespace krq;

namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
// 16 bytes at any element's address (rows of an odd N start anywhere; global stores take any address)
typedef v4u v4u_any __attribute__((aligned(2)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));

// 32-bit LDS address of a pointer into a __shared__ array, wave-uniform
KRQ_DEV uint32_t lds_at(const uint8_t* p) {
  return __builtin_amdgcn_readfirstlane(
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t*)p)));
}

// Direct loads and their waits are assembly, so that the compiler, which does not know the ring's buffers apart, waits for
// none of them by itself, and (the two that branch) so that a stage of the stream stays one basic block, within which
// products, LDS reads and loads can be interleaved.
KRQ_DEV uint64_t uniform(const uint8_t* p) {
  const uint64_t b = reinterpret_cast<uint64_t>(p);
  return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b))) |
         static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b >> 32)))) << 32;
}

// a wave-uniform value that a division or a conversion left in vector registers, as a scalar
KRQ_DEV int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }

// 16 bytes per lane from base + off (base wave-uniform) to LDS at l + 16 lane (s_nop: M0 is read right after its scalar write)
KRQ_DEV void load_lds(const uint8_t* base, uint32_t off, uint32_t l) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(l)), "v"(off),
               "s"(uniform(base))
               : "memory", "m0");
}

// the same, if on != 0 (wave-uniform)
KRQ_DEV void load_lds_if(int on, const uint8_t* base, uint32_t off, uint32_t l) {
  asm volatile(
      "s_cmp_eq_u32 %3, 0\n\ts_cbranch_scc1 .Lkrq_no_load%=\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, "
      "%2\n.Lkrq_no_load%=:" ::"s"(__builtin_amdgcn_readfirstlane(l)),
      "v"(off), "s"(uniform(base)), "s"(__builtin_amdgcn_readfirstlane(on))
      : "memory", "m0", "scc");
}

template <int N>
KRQ_DEV void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N < 63 ? N : 63) : "memory");
}

// at most N operations in flight, or at most N + S where more != 0 (wave-uniform)
template <int N, int S>
KRQ_DEV void wait_loads_or(int more) {
  asm volatile(
      "s_cmp_eq_u32 %2, 0\n\ts_cbranch_scc0 .Lkrq_more%=\n\ts_waitcnt vmcnt(%0)\n.Lkrq_more%=:\n\ts_waitcnt vmcnt(%1)" ::"n"(N < 63 ? N : 63),
      "n"(N + S < 63 ? N + S : 63), "s"(__builtin_amdgcn_readfirstlane(more))
      : "memory", "scc");
}

// LDS reads issued up to product U of NP, of NR in all: spread over the first half of the products, so that the rest of
// them cover the last reads' latency
template <int NP, int NR>
constexpr int reads_to(int u) {
  constexpr int over = NP > 1 ? NP / 2 : 1;
  return u >= over ? NR : u * NR / over;
}
template <int U, int NP, int NR>
KRQ_DEV void interleave() {
  if constexpr (U < NP) {
    constexpr int c = reads_to<NP, NR>(U + 1) - reads_to<NP, NR>(U);
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (c > 0) __builtin_amdgcn_sched_group_barrier(0x100, c, 0);
    interleave<U + 1, NP, NR>();
  }
}

struct GemmArgs {
  const uint8_t *x, *xs, *w, *ws;
  int M, N, KT, KS, groups, mbs, nbs;  // KT tiles of K in KS stages; mbs, nbs: row blocks of x and w
  int tiles_m, tiles, splits;
  float* part;                     // fp32 [splits][M][N] (PART)
  uint16_t* out;
};

// PART: a work unit is (tile, split) and writes its fp32 sums to plane `split` of part; else bf16 to out.
template <int ELEM, int BM, int BN, int W, int OCC, int NB, int T, bool PART>
__global__ __launch_bounds__(64 * W, OCC * W / 4) void k_gemm_mx(const GemmArgs a) {
  constexpr int AB = ELEM == KRQ_MX_E2M1 ? 1 : 2;          // KiB per activation tile
  constexpr int kA = BM / 16 * AB * 1024, kB = BN / 16 * 1024, kTile = kA + kB, kStage = T * kTile;
  constexpr int QA = (kA / 1024 + W - 1) / W, QB = (kB / 1024 + W - 1) / W, kLoads = T * (QA + QB);  // loads per wave per stage
  constexpr int kScale = (BM + BN) / 16 * 256;             // scale bytes of a group
  constexpr int kSl = (kScale / 1024 + W - 1) / W;             // loads per wave per group (some twice)
  constexpr int FI = BM / 64, FJ = BN / (16 * W);          // 32-row fragments of a wave
  constexpr int NP = FI * FJ, NF = FI * AB + FJ;           // products of a half tile, LDS reads of its elements
  constexpr int HT = 2 * T, kG = 4 / T;                    // half tiles of a stage; stages of a scale group
  typedef std::conditional_t<T == 1, uint8_t, uint16_t> scale_t;  // a block's scales in a stage
  constexpr int kStores = PART ? NP * 4 : NP * 2, JP = FJ % 2 == 0 ? 2 : 1;
  static_assert(NB >= 2 && NB <= 4 && (T == 1 || T == 2) && BM % 64 == 0 && BN % (16 * W) == 0, "tile shape");
  // Scales are loaded for the stage kLag before the tiles' (three buffers and more: they still come a whole stage early),
  // so that a slot can be filled again when all of the next kSlots groups (of one stage at least each) lie ahead of it.
  constexpr int kLag = NB > 2 ? 1 : 0, kSlots = NB - kLag;
  __shared__ __align__(1024) uint8_t ring[NB * kStage + kSlots * kScale];
  uint8_t* const sring = ring + NB * kStage;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int c = lane >> 5, hi = (lane >> 4) & 1, r = lane & 15;
  const int wmb = (wave & 1) * (BM / 32), wnb = (wave >> 1) * (2 * FJ);  // this wave's first row blocks
  const int G = gridDim.x, bid = blockIdx.x, units = a.tiles * a.splits;

  // the workgroup's k-th unit: units in order, M-fastest; in a whole round of G units the workgroups of one XCD
  // (b, b + 8, ...) take a contiguous run
  auto unit_of = [&](int k) {
    const int base = k * G;
    if (base + bid >= units) return -1;
    if ((G & 7) == 0 && units - base >= G) return base + (bid & 7) * (G >> 3) + (bid >> 3);
    return base + bid;
  };

  // tile row, tile column (in tiles), first stage and end of unit u
  struct Unit {
    int tm, tn, s0, s1;
  };
  auto unit = [&](int u) {
    const int sp = scalar(u / a.tiles), p = u - sp * a.tiles, tn = scalar(p / a.tiles_m);
    return Unit{p - tn * a.tiles_m, tn, PART ? scalar(static_cast<int>((int64_t)a.KS * sp / a.splits)) : 0,
                PART ? scalar(static_cast<int>((int64_t)a.KS * (sp + 1) / a.splits)) : a.KS};
  };

  // ---- the stream's loading end: stage ls of ls1 of unit lk, into buffer lb ----
  int lk = 0, ls = 0, ls1 = 0, lstep = 1, lb = 0;
  int cs = 0, cstep = 1, cslot = kSlots - 1, cnew = 1;  // the scales' stage; cnew: the first of a unit
  const uint8_t *xb = a.x, *wb = a.w, *xsb = a.xs, *wsb = a.ws;  // the unit's tiles, at stage ls; its scales
  uint32_t off[QA + QB], soff[kSl];
  auto load_unit = [&](int u) {
    const Unit un = unit(u);
    const int mb0 = un.tm * (BM / 16), nb0 = un.tn * (BN / 16);
    ls = un.s0;
    ls1 = un.s1;
    xb = a.x + ((int64_t)mb0 * a.KT + ls * T) * (1024 * AB);
    wb = a.w + ((int64_t)nb0 * a.KT + ls * T) * 1024;
    int ln = lane;  // (opaque: computed here per unit, not kept live across units)
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int q = 0; q < QA; ++q) {
      const int i = (wave + W * q) % (kA / 1024), rb = min(mb0 + i / AB, a.mbs - 1) - mb0;
      off[q] = static_cast<uint32_t>(rb * a.KT * (1024 * AB) + (i % AB) * 1024 + 16 * ln);
    }
#pragma unroll
    for (int q = 0; q < QB; ++q)
      off[QA + q] = static_cast<uint32_t>((min(nb0 + (wave + W * q) % (kB / 1024), a.nbs - 1) - nb0) * a.KT * 1024 + 16 * ln);
  };
  auto scale_unit = [&](int u) {
    const Unit un = unit(u);
    const int mb0 = un.tm * (BM / 16), nb0 = un.tn * (BN / 16);
    cs = un.s0;
    cnew = 1;
    xsb = a.xs + (int64_t)mb0 * a.groups * 256;
    wsb = a.ws + (int64_t)nb0 * a.groups * 256;
    int ln = lane;
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int q = 0; q < kSl; ++q) {  // four row blocks' scales per load
      const int rb = (wave + W * q) % (kScale / 1024) * 4 + (ln >> 4);
      const int at = rb < BM / 16 ? min(mb0 + rb, a.mbs - 1) - mb0 : min(nb0 + rb - BM / 16, a.nbs - 1) - nb0;
      soff[q] = static_cast<uint32_t>(at * a.groups * 256 + 16 * (ln & 15));
    }
  };
  const uint32_t l0 = lds_at(ring), sl0 = lds_at(sring);
  // the scales of the scales' stage, where it begins a group
  auto load_scales = [&]() {
    const int on = cstep & (cnew | ((cs & (kG - 1)) == 0 ? 1 : 0));
    cslot += on;
    cslot = cslot == kSlots ? 0 : cslot;
#pragma unroll
    for (int q = 0; q < kSl; ++q) {
      const int li = (wave + W * q) % (kScale / 1024);
      load_lds_if(on, (li < BM / 64 ? xsb : wsb) + (int64_t)(cs / kG) * 256, soff[q], sl0 + cslot * kScale + li * 1024);
    }
    cnew = 0;
    cs += cstep;
  };
  auto load_tile = [&](int i) {
    const int t = i / (QA + QB), q = i % (QA + QB);
    load_lds(q < QA ? xb + t * (1024 * AB) : wb + t * 1024, off[q],
             l0 + lb * kStage + t * kTile +
                 (q < QA ? (wave + W * q) % (kA / 1024) * 1024 : kA + (wave + W * (q - QA)) % (kB / 1024) * 1024));
  };
  auto advance = [&]() {  // past the loaded stage
    lb = lb + 1 == NB ? 0 : lb + 1;
    ls += lstep;
    xb += lstep * (T * 1024 * AB);
    wb += lstep * (T * 1024);
  };
  // Behind the stream's last stage its loads repeat (lstep 0), into buffers that nobody reads any more, so that every stage
  // issues as many.
  auto next_unit = [&]() {
    const int u = unit_of(++lk);
    if (u >= 0) {
      load_unit(u);
    } else {
      lstep = 0;
      --ls;
      ls1 = 0x7fffffff;
      xb -= T * 1024 * AB;
      wb -= T * 1024;
    }
  };
  auto next_scale_unit = [&]() {  // (after next_unit)
    const int u = unit_of(lk);
    if (u >= 0) scale_unit(u);
    else cstep = 0;
  };
  if (unit_of(0) < 0) return;
  load_unit(unit_of(0));
  scale_unit(unit_of(0));
  for (int b = 0; b < NB; ++b) {
    if (b < NB - kLag) load_scales();
#pragma unroll
    for (int q = 0; q < kLoads; ++q) load_tile(q);
    advance();
  }

  // ---- the consuming end ----
  const int lo = hi * 1024 + c * 256 + r * 16;  // e2m1 tile: this lane's 16 bytes of half 0
  const int loa = hi * (1024 * AB) + c * 256 + r * 16;
  const int los = (hi * 64 + 16 * c + r) * 4;
  uint4 fa[2][FI][AB], fb[2][FJ];
  uint32_t sa[2][FI], sb[2][FJ];
  // read n of half tile H of the stage in buffer b, its scales in slot sl at byte t: elements, then (tile 0: the stage's) scales,
  // into register set H % 2
  auto read = [&](auto H_c, int n, int b, int sl, int t) __attribute__((always_inline)) {
    constexpr int H = decltype(H_c)::value, h = H & 1;
    const uint8_t* pa = ring + b * kStage + (H >> 1) * kTile + wmb * (1024 * AB) + loa;
    const uint8_t* pb = ring + b * kStage + (H >> 1) * kTile + kA + wnb * 1024 + lo;
    const uint8_t* ps = sring + sl * kScale + los + t + 128 * h;  // (block 2 h + c)
    if (n < FI * AB) {
      const int f = n / AB, e = n % AB;
      fa[h][f][e] = *reinterpret_cast<const uint4*>(pa + f * (2048 * AB) + (AB == 2 ? 1024 * h + 512 * e : 512 * h));
    } else if (n < NF) {
      const int f = n - FI * AB;
      fb[h][f] = *reinterpret_cast<const uint4*>(pb + f * 2048 + 512 * h);
    } else if (n < NF + FI) {
      const int f = n - NF;
      sa[h][f] = *reinterpret_cast<const scale_t*>(ps + (wmb + 2 * f) * 256);
    } else {
      const int f = n - NF - FI;
      sb[h][f] = *reinterpret_cast<const scale_t*>(ps + (BM / 16 + wnb + 2 * f) * 256);
    }
  };
  v16f acc[FI][FJ];
  auto zero = [&]() {
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  };
  // half tile H of a stage: its products, each followed by its share of the reads of the next half tile (of buffer b, ...; behind
  // the stream's last stage they read what nobody uses) and, the stage's last, of the loads of the stage at the loading end
  auto half = [&](auto H_c, int b, int sl, int t) __attribute__((always_inline)) {
    constexpr int H = decltype(H_c)::value, h = H & 1, next = (H + 1) % HT;
    constexpr int NR = NF + (next < 2 ? FI + FJ : 0);
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int i = u / FJ, j = u % FJ;
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
          pack_v8i(fb[h][j], zero4()), AB == 2 ? pack_v8i(fa[h][i][0], fa[h][i][AB - 1]) : pack_v8i(fa[h][i][0], zero4()),
          acc[i][j], 4, ELEM == KRQ_MX_E2M1 ? 4 : 0, H >> 1, static_cast<int>(sb[h][j]), H >> 1, static_cast<int>(sa[h][i]));
      if (H == HT - 1) {
        if (u == 0) load_scales();
#pragma unroll
        for (int q = u * kLoads / NP; q < (u + 1) * kLoads / NP; ++q) load_tile(q);
      }
#pragma unroll
      for (int n = reads_to<NP, NR>(u); n < reads_to<NP, NR>(u + 1); ++n)
        read(std::integral_constant<int, next>{}, n, b, sl, t);
    }
    interleave<0, NP, NR>();
  };
  using yes = std::true_type;
  using no = std::false_type;

  // A lane ends with four adjacent columns (8 bytes in bf16) of row l % 32 in every eighth column. Exchanges turn that into
  // whole lines: lanes l and l + 32 (v_permlane32_swap) make 16 bytes each, odd and even sixteens (v_permlane16_swap) 64 bytes of
  // sixteen rows per store, and lanes l and l ^ 8 of two 32-column pieces (DPP) 128 bytes of eight rows (against
  // stores of 32 bytes of thirty-two rows: 4,096 x 19,456 x 2,560, e2m1 rows, 117.2 -> 114.4 us; without its stores, whose
  // 159 MB all units write at once, it takes 92). FULL: every row and column lies in the output.
  auto store = [&](auto full_c, int m0, int n0, int sp) {
    constexpr bool FULL = decltype(full_c)::value;
    int le = lane;  // (opaque: addresses are computed here, not hoisted out of the stream and kept)
    asm volatile("" : "+v"(le));
    const int ce = le >> 5, mrow = m0 + 16 * wmb + (le & 31);
#pragma unroll
    for (int i = 0; i < FI; ++i) {
      const int m = mrow + 32 * i;
#pragma unroll
      for (int j = 0; j < FJ; ++j) {
        const int n = n0 + 16 * wnb + 32 * j;
        if constexpr (PART) {
          float* p = a.part + ((int64_t)sp * a.M + m) * a.N + n + 4 * ce;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int left = a.N - (n + 8 * g + 4 * ce);  // columns from here on
            if (FULL || (m < a.M && left >= 4)) {
              *reinterpret_cast<v4f_any*>(p + 8 * g) =
                  v4f{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            } else if (m < a.M) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (e < left) p[8 * g + e] = acc[i][j][4 * g + e];
            }
          }
        } else {
          if (j % JP == 0) {
            uint32_t x[JP][4], y[JP][4];  // rows 0 .. 15 and 16 .. 31 of the pieces
#pragma unroll
            for (int q = 0; q < JP; ++q) {
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const v16f& c16 = acc[i][j + q];
                const auto lo = __builtin_amdgcn_permlane32_swap(pack_bf16x2(c16[8 * g], c16[8 * g + 1]),
                                                                 pack_bf16x2(c16[8 * g + 4], c16[8 * g + 5]), false, false);
                const auto hi = __builtin_amdgcn_permlane32_swap(pack_bf16x2(c16[8 * g + 2], c16[8 * g + 3]),
                                                                 pack_bf16x2(c16[8 * g + 6], c16[8 * g + 7]), false, false);
                uint32_t* o = g == 0 ? x[q] : y[q];
                o[0] = lo[0];
                o[1] = hi[0];
                o[2] = lo[1];
                o[3] = hi[1];
              }
#pragma unroll
              for (int d = 0; d < 4; ++d) {
                const auto w = __builtin_amdgcn_permlane16_swap(x[q][d], y[q][d], false, false);
                x[q][d] = w[0];
                y[q][d] = w[1];
              }
            }
            // sixteen l / 16 now holds columns 8 ((l / 32) + 2 ((l / 16) % 2)) .. + 7
            const int r16 = le & 15, col = n + 8 * (ce + 2 * ((le >> 4) & 1));
            auto put = [&](int row, int cc, const uint32_t* v) {
              uint16_t* o = a.out + (int64_t)row * a.N + cc;
              if (FULL || (row < a.M && cc + 8 <= a.N)) {
                *reinterpret_cast<v4u_any*>(o) = v4u{v[0], v[1], v[2], v[3]};
              } else if (row < a.M) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (cc + e < a.N) o[e] = static_cast<uint16_t>(v[e >> 1] >> (16 * (e & 1)));
              }
            };
            const int row0 = m0 + 16 * wmb + 32 * i;
            if constexpr (JP == 2) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t u[4], v[4];
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                  const uint32_t p0 = h == 0 ? x[0][d] : y[0][d], p1 = h == 0 ? x[JP - 1][d] : y[JP - 1][d];
                  u[d] = take_ror8<0xc>(p0, p1);
                  v[d] = take_ror8<0x3>(p1, p0);
                }
                const int row = row0 + 16 * h + (r16 & 7), cc = col + 32 * (r16 >> 3);
                put(row, cc, u);
                put(row + 8, cc, v);
              }
            } else {
              put(row0 + r16, col, x[0]);
              put(row0 + 16 + r16, col, y[0]);
            }
          }
        }
      }
    }
  };

  // in flight: NB stages. Stage 0's loads are the oldest
  wait_loads<(NB - 1) * kLoads>();
  barrier_lds();
#pragma unroll
  for (int n = 0; n < NF + FI + FJ; ++n) read(std::integral_constant<int, 0>{}, n, 0, 0, unit(unit_of(0)).s0 % kG * T);
  int buf = 0, slot = 0;
  int stores = 0;  // the last tile's kStores stores per lane are younger than the next stage's loads
  for (int k = 0, u = unit_of(0), un; u >= 0; ++k, u = un) {
    un = unit_of(k + 1);
    const Unit cur = unit(u);
    int s = cur.s0;
    const int s1 = cur.s1, sfirst = un < 0 ? 0 : unit(un).s0;
    zero();
    // stage s; the loading end is NB stages ahead
    auto stage = [&](bool last) __attribute__((always_inline)) {
      const int t = s % kG * T;
      half(std::integral_constant<int, 0>{}, buf, slot, t);
      if constexpr (T == 2) {
        half(std::integral_constant<int, 1>{}, buf, slot, t);
        half(std::integral_constant<int, 2>{}, buf, slot, t);
      }
      ++s;
      const int sn = last ? sfirst : s;  // the next stage: of this unit, or the next one's first
      const int on = last || sn % kG == 0 ? 1 : 0;
      buf = buf + 1 == NB ? 0 : buf + 1;
      slot = slot + on == kSlots ? 0 : slot + on;
      // the next stage has landed, and once every wave is here none reads this one's buffer any more: refill it
      wait_loads_or<(NB - 2) * kLoads, kStores>(stores);
      stores = 0;
      barrier_lds();
      half(std::integral_constant<int, HT - 1>{}, buf, slot, sn % kG * T);
      advance();
    };
#pragma clang loop unroll(disable)
    while (s < s1 - NB) stage(false);
    next_unit();  // the loading end goes on into the next unit
#pragma clang loop unroll(disable)
    while (s < s1 - NB + kLag) stage(false);
    next_scale_unit();
#pragma clang loop unroll(disable)
    while (s < s1) stage(s + 1 == s1);
    const int m0 = cur.tm * BM, n0 = cur.tn * BN, sp = PART ? scalar(u / a.tiles) : 0;
    if (m0 + BM <= a.M && n0 + BN <= a.N) {
      store(yes{}, m0, n0, sp);
      stores = 1;
    } else {
      store(no{}, m0, n0, sp);
    }
  }
  wait_loads<0>();  // no load into LDS outlives the workgroup
}

// K of fewer stages than the stream holds: 128 x 128 outputs per workgroup, four waves of 64 x 64, operands straight
// from memory, v_mfma_scale_f32_16x16x128_f8f6f4 (element e of lane l: row 4 (l / 16) + e of x, column l % 16). A launch and its
// writes: 4,096 x 2,560 x 384 13.3 us (the stream at K = 512 13.2), 4,096 x 19,456 x 128 47 (159 MB at 3.4 TB/s).
constexpr int kMinStages = 4;
template <int ELEM>
__global__ __launch_bounds__(256) void k_gemm_mx_short(const GemmArgs a, int tiles_m) {
  constexpr int AB = ELEM == KRQ_MX_E2M1 ? 1 : 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = static_cast<int>(blockIdx.x % tiles_m) * 8 + 4 * (wave & 1);  // in row blocks of 16
  const int n0 = static_cast<int>(blockIdx.x / tiles_m) * 8 + 4 * (wave >> 1);
  v4f acc[4][4];
  uint32_t sa[4], sb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // (one group of scales: KT < 4)
    sa[i] = *reinterpret_cast<const uint32_t*>(a.xs + ((int64_t)min(m0 + i, a.mbs - 1) * 64 + lane) * 4);
    sb[i] = *reinterpret_cast<const uint32_t*>(a.ws + ((int64_t)min(n0 + i, a.nbs - 1) * 64 + lane) * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  for (int t = 0; t < a.KT; ++t) {
    v8i x[4], w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* p = a.x + (((int64_t)min(m0 + i, a.mbs - 1) * a.KT + t) * (64 * AB) + lane) * 16;
      x[i] = pack_v8i(ld16(p), AB == 2 ? ld16(p + 1024) : zero4());
      w[i] = pack_v8i(ld16(a.w + (((int64_t)min(n0 + i, a.nbs - 1) * a.KT + t) * 64 + lane) * 16), zero4());
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x[i], w[j], acc[i][j], ELEM == KRQ_MX_E2M1 ? 4 : 0, 4, 0,
                                                                     static_cast<int>(sa[i] >> (8 * t)), 0,
                                                                     static_cast<int>(sb[j] >> (8 * t)));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t m = 16 * (m0 + i) + 4 * (lane >> 4) + e, n = 16 * (n0 + j) + (lane & 15);
        if (m < a.M && n < a.N) a.out[m * a.N + n] = f32_to_bf16(acc[i][j][e]);
      }
}

// out[m][n] = bf16(sum over s of part[s][m][n], s in order), V columns per thread
template <int V>
__global__ __launch_bounds__(256) void k_gemm_mx_reduce(const float* __restrict__ part, int splits, int64_t plane,
                                                        uint16_t* __restrict__ out) {
  const int64_t e = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * V;
  if (e >= plane) return;
  if constexpr (V == 4) {
    float4 v = *reinterpret_cast<const float4*>(part + e);
    for (int s = 1; s < splits; ++s) {
      const float4 o = *reinterpret_cast<const float4*>(part + s * plane + e);
      v.x += o.x;
      v.y += o.y;
      v.z += o.z;
      v.w += o.w;
    }
    *reinterpret_cast<uint2*>(out + e) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  } else {
    float v = part[e];
    for (int s = 1; s < splits; ++s) v += part[s * plane + e];
    out[e] = f32_to_bf16(v);
  }
}

// The output tile and the parts of K. A tile's time for a given K in a whole round of the chip, in that of 256 x 256 tiles (one
// workgroup per compute unit); the smaller ones run two per unit, the second figure is for a unit with one. Measured
// (us, e4m3 / e2m1 rows): 4,096 x 19,456 x 2,560, 5 rounds of 256 x 256 159 / 115, 7 of 192 x 256 176 / 131, 128 x 256
// 176 / 128, 128 x 128 217 / 148; 4,096 x 2,560 x 9,728 in one round of 160 256 x 256 tiles 88 / 60, of 220 192 x 256
// ones 81 / 58; 4,096 x 6,144 x 2,560 256 x 256 63 / 46, 128 x 256 52 / 43; 1,000 x 2,560 x 9,728 128 x 128 32 / 27, 64 x 64
// 45 / 43; 77 x 6,144 x 2,560 64 x 64 8.4 / 8.3, 128 x 128 11 / 10; 77 x 19,456 x 2,560 128 x 128 11.6 / 10.5, 64 x 64 15.5 / 15.
// K is split only where 64 x 64 tiles would leave half the chip idle for 64 stages and more (77 x 2,560 x 9,728, 80 tiles,
// in 4 parts 15.1 / 14.9 with their sum, whole 24.8 / 22.1; 256 x 2,560 x 4,096, 160 tiles of 32 stages, whole 12.9 / 11.7,
// in 2 15.4 / 15.0).
struct GemmPlan {
  int bm, bn, splits;
};
GemmPlan plan_of(int64_t M, int64_t N, int64_t KT, int cus) {
  auto tiles = [&](int64_t bm, int64_t bn) { return (M + bm - 1) / bm * ((N + bn - 1) / bn); };
  auto cost = [&](int64_t t, double pair, double one) {
    return pair * (double)(t / (2 * cus)) + (t % (2 * cus) == 0 ? 0.0 : t % (2 * cus) <= cus ? one : pair);
  };
  const int shape[5][2] = {{256, 256}, {192, 256}, {128, 256}, {128, 128}, {64, 64}};
  const double c[5] = {cost(tiles(256, 256), 2.0, 1.0), cost(tiles(192, 256), 1.66, 0.83), cost(tiles(128, 256), 1.09, 0.58),
                       cost(tiles(128, 128), 0.62, 0.36), cost(tiles(64, 64), 0.30, 0.22)};
  const int best = static_cast<int>(std::min_element(c, c + 5) - c);
  int splits = 1;
  if (best == 4 && KT >= 64 && tiles(64, 64) <= cus / 2)
    while (splits < 8 && tiles(64, 64) * splits <= cus && KT / (2 * splits) >= 16) splits *= 2;
  return {shape[best][0], shape[best][1], splits};
}

int cu_count(int* cus) {
  int dev = 0;
  return hipGetDevice(&dev) == hipSuccess &&
                 hipDeviceGetAttribute(cus, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && *cus > 0
             ? KRQ_OK
             : KRQ_EHIP;
}

template <int ELEM, int BM, int BN, int W, int OCC, int NB, int T, bool PART>
void launch(const GemmArgs& g, int cus, hipStream_t s) {
  GemmArgs a = g;
  a.KS = a.KT / T;
  a.tiles_m = (a.M + BM - 1) / BM;
  a.tiles = a.tiles_m * ((a.N + BN - 1) / BN);
  const int64_t units = (int64_t)a.tiles * a.splits, slots = (int64_t)cus * OCC;
  hipLaunchKernelGGL((k_gemm_mx<ELEM, BM, BN, W, OCC, NB, T, PART>), dim3(static_cast<unsigned>(std::min(units, slots))), dim3(64 * W),
                     0, s, a);
}

// Two tiles a stage (an even number of tiles, and stages for the buffers) where a stage of one is too short for its
// barrier and its scalar work: 64 x 64 outputs (us, one / two: 77 x 6,144 x 2,560 8.5 / 7.8, 256 x 2,560 x 4,096 11.4 / 9.3),
// and e2m1 rows in 256 x 256 (4,096 x 19,456 x 2,560 117.9 / 114.1) and in 128 x 128 with one workgroup per unit, which
// then takes the unit's whole LDS (1,000 x 2,560 x 9,728 29.7 / 25.0; e4m3 rows 35.2 / 37.4).
template <int ELEM>
void launch_plan(const GemmArgs& a, const GemmPlan& p, int cus, hipStream_t s) {
  constexpr bool E2 = ELEM == KRQ_MX_E2M1;
  constexpr int D = E2 ? 1 : 0;  // e2m1 stages are smaller: one buffer more
  const bool pairs = a.KT % 2 == 0 && a.KT / 2 / p.splits >= 4;
  const int64_t tiles = (int64_t)((a.M + p.bm - 1) / p.bm) * ((a.N + p.bn - 1) / p.bn);
  if (a.KT < kMinStages) {
    const int tm = (a.M + 127) / 128;
    hipLaunchKernelGGL((k_gemm_mx_short<ELEM>), dim3(static_cast<unsigned>(tm * ((a.N + 127) / 128))), dim3(256), 0, s, a, tm);
  } else if (p.bm == 256) {
    if constexpr (E2)
      if (pairs) return launch<ELEM, 256, 256, 8, 1, 2, 2, false>(a, cus, s);
    launch<ELEM, 256, 256, 8, 1, 3 + D, 1, false>(a, cus, s);
  } else if (p.bm == 192) {
    launch<ELEM, 192, 256, 8, 1, 3 + D, 1, false>(a, cus, s);
  } else if (p.bm == 128 && p.bn == 256) {
    launch<ELEM, 128, 256, 4, 2, 2, 1, false>(a, cus, s);
  } else if (p.bm == 128) {
    if constexpr (E2)
      if (pairs && tiles <= cus) return launch<ELEM, 128, 128, 4, 1, 4, 2, false>(a, cus, s);
    launch<ELEM, 128, 128, 4, 2, 3 + D, 1, false>(a, cus, s);
  } else if (p.splits == 1) {
    if (pairs) launch<ELEM, 64, 64, 4, 2, 3 + D, 2, false>(a, cus, s);
    else launch<ELEM, 64, 64, 4, 2, 4, 1, false>(a, cus, s);
  } else {
    if (pairs) launch<ELEM, 64, 64, 4, 2, 3 + D, 2, true>(a, cus, s);
    else launch<ELEM, 64, 64, 4, 2, 4, 1, true>(a, cus, s);
  }
}

}  // namespace

extern "C" int64_t krq_gemm_mxfp4_ws_bytes(int x_kind, int elem, int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1 || K % kMxBlock != 0 || (elem != KRQ_MX_E2M1 && elem != KRQ_MX_E4M3)) return -1;
  int cus = 0;
  if (cu_count(&cus) != KRQ_OK) return -1;
  const GemmPlan p = plan_of(M, N, mx_tiles(K), cus);
  return (x_kind == KRQ_MX_X_BF16 ? mx_rows_bytes(elem, M, K) : 0) + (p.splits > 1 ? p.splits * M * N * 4 : 0);
}

extern "C" int krq_gemm_mxfp4(const void* x, const void* x_scale, int x_kind, int elem, int64_t ldx, const void* w_tiled,
                              const void* w_scale, int64_t M, int64_t N, int64_t K, void* ws, int64_t ws_bytes, void* out,
                              void* stream) {
  KRQ_REQUIRE(x && w_tiled && w_scale && out, "gemm_mxfp4: null pointer");
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "gemm_mxfp4: bad element type %d", elem);
  KRQ_REQUIRE(x_kind == KRQ_MX_X_BF16 || x_kind == KRQ_MX_X_TILED, "gemm_mxfp4: bad x_kind %d", x_kind);
  KRQ_REQUIRE(x_kind == KRQ_MX_X_BF16 || x_scale, "gemm_mxfp4: tiled rows need their scales");
  KRQ_REQUIRE(aligned16(x) && aligned16(x_scale) && aligned16(w_tiled) && aligned16(w_scale) && aligned16(ws),
              "gemm_mxfp4: x, w, their scales and ws must start on 16 bytes");
  KRQ_REQUIRE(M >= 1 && M <= 0x3fffffff && N >= 1 && N <= 0x3fffffff && K >= kMxBlock && K % kMxBlock == 0 && K <= (1 << 22),
              "gemm_mxfp4: shape M=%lld N=%lld K=%lld (K a multiple of 32, at most 2^22)", (long long)M, (long long)N, (long long)K);
  KRQ_REQUIRE(((M + 63) / 64) * ((N + 63) / 64) <= 0x0fffffff, "gemm_mxfp4: M=%lld N=%lld are too large", (long long)M, (long long)N);
  int cus = 0;
  if (cu_count(&cus) != KRQ_OK) {
    krq_set_error("gemm_mxfp4: device query failed");
    return KRQ_EHIP;
  }
  GemmPlan p = plan_of(M, N, mx_tiles(K), cus);
  const int64_t rows = (x_kind == KRQ_MX_X_BF16 ? mx_rows_bytes(elem, M, K) : 0);
  KRQ_REQUIRE(rows == 0 || (ws && ws_bytes >= rows), "gemm_mxfp4: bf16 rows need a workspace of %lld bytes", (long long)rows);
  if (p.splits > 1 && (!ws || ws_bytes < rows + p.splits * M * N * 4)) p.splits = 1;
  GemmArgs a;
  if (rows) {
    a.x = (const uint8_t*)ws;
    a.xs = (const uint8_t*)ws + mx_rows_scale_at(elem, M, K);
    if (const int rc = krq_quant_mx_rows(x, M, K, ldx, elem, ws, (uint8_t*)ws + mx_rows_scale_at(elem, M, K), stream)) return rc;
  } else {
    a.x = (const uint8_t*)x;
    a.xs = (const uint8_t*)x_scale;
  }
  a.w = (const uint8_t*)w_tiled;
  a.ws = (const uint8_t*)w_scale;
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.KT = static_cast<int>(mx_tiles(K));
  a.groups = static_cast<int>(mx_groups(K));
  a.mbs = static_cast<int>((M + 15) / 16);
  a.nbs = static_cast<int>((N + 15) / 16);
  a.splits = p.splits;
  a.part = (float*)((uint8_t*)ws + rows);
  a.out = (uint16_t*)out;
  hipStream_t s = (hipStream_t)stream;
  if (elem == KRQ_MX_E2M1) launch_plan<KRQ_MX_E2M1>(a, p, cus, s);
  else launch_plan<KRQ_MX_E4M3>(a, p, cus, s);
  if (p.splits > 1) {
    const int64_t plane = M * N;
    if (plane % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 7) == 0)
      hipLaunchKernelGGL(k_gemm_mx_reduce<4>, dim3(static_cast<unsigned>((plane / 4 + 255) / 256)), dim3(256), 0, s, a.part, p.splits,
                         plane, a.out);
    else
      hipLaunchKernelGGL(k_gemm_mx_reduce<1>, dim3(static_cast<unsigned>((plane + 255) / 256)), dim3(256), 0, s, a.part, p.splits,
                         plane, a.out);
  }
  return krq_check_launch("gemm_mxfp4");
}

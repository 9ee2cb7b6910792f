// Low-rank adapters of many requests beside one shared projection:
//
//   out[m, n] = y[m, n] + s_i sum_r B_i[n, r] h[m, r],   h[m, r] = sum_k A_i,p(n)[r, k] x[m, k],   i = ids[m]
//
// for the P parts of a fused projection (part p(n) of column n), each with its own factors. Two launches: k_lora_down
// makes h, k_lora_up adds. A tile of rows may name any adapters in any order: a wave takes the distinct ones of its tile
// one after the other (or, where rows are few, each by a workgroup of its own), multiplies the whole tile and writes the
// rows that name it. The rows of a matrix-core operand do not mix, so rows of other adapters cost nothing but the idle
// columns, and a NaN stays in its row.
//
// What bounds it: the factors of the adapters in use, read once each, at few rows; x, y and out at many. The products
// are a few percent of the matrix cores' rate.
//
// k order. v_mfma_f32_16x16x32_bf16 adds products over 32 k of which lane group g = lane / 16 holds eight; which eight is
// free as long as both operands agree. In steps of 64 k, group g takes k = 16 g .. 16 g + 15 of each row: 32 contiguous
// bytes, so that the four groups read whole 128-byte lines of row-major factors and rows.
//
// h is kept in fp32 and enters the second product as the sum of two bf16 (h to 2^-16 at most), so that the sum is rounded once,
// at the end: the second product takes twice the matrix instructions, which it has to spare.
#include <algorithm>

#include "mx_common.h"

using namespace krq;

namespace {

constexpr int kMaxParts = 8, kMaxRank = 256, kMaxSplit = 8;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

struct LoraArgs {
  const uint16_t* x;
  const void* ids;
  const uint16_t* a;     // [slots][P][R][K]
  const uint16_t* b;     // [slots][N R], a slot's factors as [N][its rank, rounded up to 16]
  const int32_t* ranks;  // [slots], up to R; 0: none
  const float* scales;   // [slots]
  const void* y;
  void* out;
  float* h;              // [split][M][P R]
  int64_t M, K, ldx, ldy, ldo;
  int slots, P, R, N, split, ids64, slot_ways;
  int part[kMaxParts + 1], block[kMaxParts + 1];  // first column of each part; first group of column blocks
};

KRQ_DEV int load_id(const LoraArgs& a, int64_t m) {  // -1: none; slots: out of range
  int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[m] : static_cast<const int32_t*>(a.ids)[m];
  return id < 0 ? -1 : id >= a.slots ? a.slots : static_cast<int>(id);
}

KRQ_DEV int rank_of(const LoraArgs& a, int id) {
  return id < 0 || id >= a.slots ? 0 : min(max(a.ranks[id], 0), a.R);
}

KRQ_DEV v4f mfma32(uint4 a, uint4 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
KRQ_DEV v4f mfma16(uint2 a, uint2 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a), __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}

// The distinct ids of up to 64 rows, one at a time: `id` is each lane's row's, `left` the lanes not yet taken.
KRQ_DEV int next_id(int id, uint64_t& left, uint64_t& same) {
  const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
  same = __ballot(id == cur) & left;
  left &= ~same;
  return cur;
}

// h. A workgroup takes MT tiles of 16 rows, TC tiles of 16 ranks (of the P r of the row's adapter) and one of the
// `split` parts of K, its four waves a quarter of that each, summed in LDS in wave order.
template <int MT, int TC>
__global__ __launch_bounds__(256) void k_lora_down(LoraArgs a) {
  __shared__ float red[4][MT * TC][64 * 4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, j = lane & 15;
  const int ways = a.slot_ways;
  const int64_t m0 = (blockIdx.x / ways) * (int64_t)(16 * MT);
  const int way = blockIdx.x % ways;
  const int64_t mine = m0 + (lane & (16 * MT - 1));
  const int id = load_id(a, min(mine, a.M - 1));
  uint64_t left = __ballot(mine < a.M && lane < 16 * MT);
  // this wave's part of K, in steps of 64
  const int64_t steps = (a.K + 63) >> 6;
  const int64_t q0 = blockIdx.z * 4 + w, qn = a.split * 4;
  const int64_t s0 = steps * q0 / qn, s1 = steps * (q0 + 1) / qn;
  for (int turn = 0; left; ++turn) {
    uint64_t same;
    const int cur = next_id(id, left, same);
    if (ways > 1 && turn % ways != way) continue;
    const int per = (rank_of(a, cur) + 15) >> 4, T = a.P * per;
    const int t0 = blockIdx.y * TC;
    if (t0 >= T) continue;
    const uint16_t* ar[TC];
#pragma unroll
    for (int t = 0; t < TC; ++t) {
      const int tt = min(t0 + t, T - 1);
      ar[t] = a.a + (((int64_t)cur * a.P + tt / per) * a.R + 16 * (tt % per) + j) * a.K + 16 * g;
    }
    const uint16_t* xr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xr[i] = a.x + min(m0 + 16 * i + j, a.M - 1) * a.ldx + 16 * g;
    v4f acc[MT][TC] = {};
#pragma unroll 2
    for (int64_t s = s0; s < s1; ++s) {
      const bool in = 64 * s + 16 * g < a.K;  // (K is a multiple of 16)
      uint4 av[TC][2], xv[MT][2];
#pragma unroll
      for (int t = 0; t < TC; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) av[t][e] = in ? ld16(reinterpret_cast<const uint8_t*>(ar[t] + 64 * s + 8 * e)) : zero4();
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) xv[i][e] = in ? ld16(reinterpret_cast<const uint8_t*>(xr[i] + 64 * s + 8 * e)) : zero4();
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int t = 0; t < TC; ++t) acc[i][t] = mfma32(av[t][e], xv[i][e], acc[i][t]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < TC; ++t) *reinterpret_cast<v4f*>(&red[w][i * TC + t][4 * lane]) = acc[i][t];
    __syncthreads();
    // lane: row j of a tile, ranks 4 g .. 4 g + 3
    for (int p = w; p < MT * TC; p += 4) {
      v4f v = *reinterpret_cast<v4f*>(&red[0][p][4 * lane]);
#pragma unroll
      for (int q = 1; q < 4; ++q) v += *reinterpret_cast<v4f*>(&red[q][p][4 * lane]);
      const int i = p / TC, t = t0 + p % TC;
      if (t < T && (same >> (16 * i + j) & 1)) {
        const int64_t m = m0 + 16 * i + j;
        *reinterpret_cast<v4f*>(a.h + (blockIdx.z * a.M + m) * (a.P * a.R) + (t / per) * a.R + 16 * (t % per) + 4 * g) = v;
      }
    }
    __syncthreads();
  }
}

KRQ_DEV float lo_of(float v, float hi) { return finite_f32(hi) ? v - hi : 0.0f; }

// fp32 as the sum of two bf16: hi rounded, lo the rest rounded (none beside an infinity or a NaN)
KRQ_DEV void split_bf16(const float* v, int n, uint32_t* hi, uint32_t* lo) {
#pragma unroll
  for (int i = 0; i < n / 2; ++i) {
    hi[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    lo[i] = pack_bf16x2(lo_of(v[2 * i], as_f32(hi[i] << 16)), lo_of(v[2 * i + 1], as_f32(hi[i] & 0xffff0000u)));
  }
}

// Sixteen values of a row at `at`, of which `n` lie in the part (n >= 16: all).
template <typename T>
KRQ_DEV void load16(const T* at, int n, bool wide, float* v) {
  if (wide) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint4 u = ld16(reinterpret_cast<const uint8_t*>(at) + 16 * q);
        const uint32_t e[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[8 * q + 2 * i] = as_f32(e[i] << 16), v[8 * q + 2 * i + 1] = as_f32(e[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 u = reinterpret_cast<const float4*>(at)[q];
        v[4 * q] = u.x, v[4 * q + 1] = u.y, v[4 * q + 2] = u.z, v[4 * q + 3] = u.w;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = i < n ? bf16_to_f32(at[i]) : 0.0f;
      else v[i] = i < n ? at[i] : 0.0f;
    }
  }
}

template <typename T>
KRQ_DEV void store16(T* at, int n, bool wide, const float* v) {
  if (wide) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        *reinterpret_cast<uint4*>(at + 8 * q) =
            make_uint4(pack_bf16x2(v[8 * q], v[8 * q + 1]), pack_bf16x2(v[8 * q + 2], v[8 * q + 3]),
                       pack_bf16x2(v[8 * q + 4], v[8 * q + 5]), pack_bf16x2(v[8 * q + 6], v[8 * q + 7]));
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) reinterpret_cast<float4*>(at)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 2) at[i] = static_cast<uint16_t>(pack_bf16x2(v[i], v[i]));
        else at[i] = v[i];
      }
  }
}

// y + the delta. A wave takes 16 rows and NI blocks of 64 columns of one part; a lane finishes 16 consecutive columns
// of one row: tile t of a block multiplies the columns 16 (i / 4) + 4 t + i % 4, i = 0 .. 15, so that the four
// accumulators of a lane are neighbours. ROWS: the workgroup's waves take four row tiles, else four groups of columns.
template <typename T, int NI, bool ROWS>
__global__ __launch_bounds__(256) void k_lora_up(LoraArgs a) {
  extern __shared__ uint4 stage[];  // h as operands: [wave][R / 32 or less][hi, lo][lane]
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, j = lane & 15;
  const int ways = a.slot_ways;
  const int units = a.block[a.P], wide_units = ROWS ? units : (units + 3) >> 2;  // (the columns of a row tile first)
  const int64_t at = blockIdx.x / wide_units;
  const int64_t m0 = ROWS ? (at * 4 + w) * 16 : at / ways * 16;
  const int way = ROWS ? 0 : static_cast<int>(at % ways);
  const int unit = ROWS ? blockIdx.x % wide_units : blockIdx.x % wide_units * 4 + w;
  if (m0 >= a.M || unit >= units) return;
  int p = 0;
  while (unit >= a.block[p + 1]) ++p;
  const int n0 = a.part[p] + (unit - a.block[p]) * 64 * NI, n1 = a.part[p + 1];
  const int64_t m = m0 + j;
  const int id = load_id(a, min(m, a.M - 1));
  uint64_t left = __ballot(m < a.M) & 0xffff;
  uint4* st = stage + w * ((a.R + 31) / 32) * 128;
  const T* yr = static_cast<const T*>(a.y) + min(m, a.M - 1) * a.ldy;
  T* orow = static_cast<T*>(a.out) + min(m, a.M - 1) * a.ldo;
  constexpr int kVec = 16 / sizeof(T);
  const bool even = a.ldy % kVec == 0 && a.ldo % kVec == 0 && n0 % kVec == 0 &&
                    (reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.out)) % 16 == 0;
  for (int turn = 0; left; ++turn) {
    uint64_t same;
    const int cur = next_id(id, left, same);
    if (ways > 1 && turn % ways != way) continue;
    const bool me = same >> j & 1;
    const int rank = rank_of(a, cur), r16 = (rank + 15) & ~15, full = r16 >> 5;
    const bool tail = r16 & 16;
    if (r16 == 0 && cur < a.slots && a.out == a.y) continue;
    // this row's h, summed over the parts of K in order, times the adapter's scale
    if (r16) {
      const float scale = a.scales[cur];
      const int64_t slice = a.M * (a.P * a.R);
      const float* hr = a.h + m * (a.P * a.R) + p * a.R;
      for (int s = 0; s < full; ++s) {
        float v[8] = {};
        if (me) {
          for (int q = 0; q < a.split; ++q) {
            const float4* f = reinterpret_cast<const float4*>(hr + q * slice + 32 * s + 8 * g);
            const float4 f0 = f[0], f1 = f[1];
            v[0] += f0.x; v[1] += f0.y; v[2] += f0.z; v[3] += f0.w;
            v[4] += f1.x; v[5] += f1.y; v[6] += f1.z; v[7] += f1.w;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 32 * s + 8 * g + i < rank ? v[i] * scale : 0.0f;
        }
        uint32_t hi[4], lo[4];
        split_bf16(v, 8, hi, lo);
        st[s * 128 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        st[s * 128 + 64 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      if (tail) {
        float v[4] = {};
        if (me) {
          for (int q = 0; q < a.split; ++q) {
            const float4 f = *reinterpret_cast<const float4*>(hr + q * slice + 32 * full + 4 * g);
            v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = 32 * full + 4 * g + i < rank ? v[i] * scale : 0.0f;
        }
        uint32_t hi[2], lo[2];
        split_bf16(v, 4, hi, lo);
        st[full * 128 + lane] = make_uint4(hi[0], hi[1], lo[0], lo[1]);
      }
    }
    const uint16_t* bs = r16 ? a.b + (int64_t)cur * a.N * a.R : a.b;
#pragma unroll 1
    for (int blk = 0; blk < NI; ++blk) {
      const int nb = n0 + 64 * blk;
      if (nb >= n1) break;
      const int nl = nb + 16 * g, have = n1 - nl;
      const bool wide = even && have >= 16;
      float v[16];
      if (me) load16(yr + nl, have, wide, v);
      if (r16) {
        v4f acc[4] = {};
        const uint16_t* br[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) br[t] = bs + (int64_t)min(nb + 16 * (j >> 2) + 4 * t + (j & 3), n1 - 1) * r16;
        for (int s = 0; s < full; ++s) {
          const uint4 hi = st[s * 128 + lane], lo = st[s * 128 + 64 + lane];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint4 bv = ld16(reinterpret_cast<const uint8_t*>(br[t] + 32 * s + 8 * g));
            acc[t] = mfma32(bv, hi, acc[t]);
            acc[t] = mfma32(bv, lo, acc[t]);
          }
        }
        if (tail) {
          const uint4 hl = st[full * 128 + lane];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint2 bv = *reinterpret_cast<const uint2*>(br[t] + 32 * full + 4 * g);
            acc[t] = mfma16(bv, make_uint2(hl.x, hl.y), acc[t]);
            acc[t] = mfma16(bv, make_uint2(hl.z, hl.w), acc[t]);
          }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) v[4 * t + i] += acc[t][i];
      }
      if (cur >= a.slots) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = as_f32(0x7fc00000u);
      }
      if (me && have > 0) store16(orow + nl, have, wide, v);
    }
  }
}

struct LoraPlan {
  int split, mt, ways;
};

// Few rows: 16-row tiles, K in up to eight parts, the adapters of a tile each in a workgroup of its own (every row may
// name another one). Many: 64-row tiles, so that a factor is read once for 64 rows, K in as many parts as fill the chip.
LoraPlan lora_plan(int64_t M, int64_t K, int P, int R) {
  LoraPlan p;
  p.mt = M <= 256 ? 1 : 4;
  const int64_t tiles = (M + 16 * p.mt - 1) / (16 * p.mt);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kMaxSplit, K / 512));
  if (p.mt == 1) {
    p.ways = M <= 64 ? 16 : 4;
    p.split = static_cast<int>(most);
  } else {
    p.ways = 1;
    p.split = static_cast<int>(std::max<int64_t>(1, std::min(most, 512 / tiles)));
  }
  return p;
}

template <typename T, int NI, bool ROWS>
void launch_up(const LoraArgs& a, hipStream_t s) {
  LoraArgs u = a;
  u.block[0] = 0;
  for (int p = 0; p < a.P; ++p) u.block[p + 1] = u.block[p] + (a.part[p + 1] - a.part[p] + 64 * NI - 1) / (64 * NI);
  const int64_t units = u.block[a.P];
  const int64_t tiles = (a.M + 15) / 16;
  const dim3 grid(static_cast<unsigned>(ROWS ? units * ((tiles + 3) / 4) : (units + 3) / 4 * tiles * a.slot_ways));
  const size_t smem = static_cast<size_t>(4) * ((a.R + 31) / 32) * 128 * 16;
  hipLaunchKernelGGL((k_lora_up<T, NI, ROWS>), grid, dim3(256), smem, s, u);
}

}  // namespace

extern "C" int64_t krq_lora_ws_bytes(int64_t M, int64_t K, int parts, int rank) {
  if (M < 1 || K < 16 || parts < 1 || parts > kMaxParts || rank < 16 || rank > kMaxRank) return -1;
  return lora_plan(M, K, parts, rank).split * M * parts * rank * (int64_t)sizeof(float);
}

extern "C" int krq_lora_add(const void* x, int64_t ldx, const void* ids, int ids_64, const void* a, const void* b, const int32_t* ranks,
                            const float* scales, int64_t slots, int64_t M, int64_t K, const int64_t* parts_n, int parts, int rank,
                            const void* y, int64_t ldy, void* out, int64_t ldo, int fp32, void* ws, int64_t ws_bytes, void* stream) {
  KRQ_REQUIRE(x && ids && a && b && ranks && scales && parts_n && y && out && ws, "lora_add: null pointer");
  KRQ_REQUIRE(M >= 1 && M <= (1 << 24) && K >= 16 && K % 16 == 0 && K <= (1 << 24), "lora_add: bad shape M=%lld K=%lld (K a multiple of 16)",
              (long long)M, (long long)K);
  KRQ_REQUIRE(parts >= 1 && parts <= kMaxParts, "lora_add: %d parts (at most %d)", parts, kMaxParts);
  KRQ_REQUIRE(rank >= 16 && rank % 16 == 0 && rank <= kMaxRank, "lora_add: rank=%d (a multiple of 16, at most %d)", rank, kMaxRank);
  KRQ_REQUIRE(slots >= 1 && slots < (1 << 24), "lora_add: %lld slots", (long long)slots);
  KRQ_REQUIRE(ldx >= K && ldx % 8 == 0 && aligned16(x), "lora_add: rows of x must start on 16 bytes (ldx=%lld)", (long long)ldx);
  KRQ_REQUIRE(aligned16(a) && aligned16(b) && aligned16(ws), "lora_add: the factors and ws must start on 16 bytes");
  LoraArgs l{};
  int64_t n = 0;
  for (int p = 0; p < parts; ++p) {
    KRQ_REQUIRE(parts_n[p] >= 1 && parts_n[p] <= (1 << 24), "lora_add: part %d of %lld columns", p, (long long)parts_n[p]);
    l.part[p] = static_cast<int>(n);
    n += parts_n[p];
  }
  l.part[parts] = static_cast<int>(n);
  KRQ_REQUIRE(ldy >= n && ldo >= n, "lora_add: rows of %lld columns %lld and %lld apart", (long long)n, (long long)ldy, (long long)ldo);
  const int esize = fp32 ? 4 : 2;
  KRQ_REQUIRE((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out)) % esize == 0, "lora_add: y and out must start on a value");
  KRQ_REQUIRE(y != out || ldy == ldo, "lora_add: out is y with other rows");
  KRQ_REQUIRE((M + 15) / 16 * (n / 64 + parts) < 0x7fffffff, "lora_add: %lld x %lld is too large", (long long)M, (long long)n);
  const LoraPlan plan = lora_plan(M, K, parts, rank);
  KRQ_REQUIRE(ws_bytes >= krq_lora_ws_bytes(M, K, parts, rank), "lora_add: ws of %lld bytes is too small", (long long)ws_bytes);
  l.x = (const uint16_t*)x;
  l.ids = ids;
  l.a = (const uint16_t*)a;
  l.b = (const uint16_t*)b;
  l.ranks = ranks;
  l.scales = scales;
  l.y = y;
  l.out = out;
  l.h = (float*)ws;
  l.M = M;
  l.K = K;
  l.ldx = ldx;
  l.ldy = ldy;
  l.ldo = ldo;
  l.slots = (int)slots;
  l.P = parts;
  l.R = rank;
  l.N = (int)n;
  l.split = plan.split;
  l.ids64 = ids_64 != 0;
  l.slot_ways = plan.ways;
  hipStream_t s = (hipStream_t)stream;
  const int T = parts * rank / 16;
  const int64_t tiles = (M + 16 * plan.mt - 1) / (16 * plan.mt);
  if (plan.mt == 1)
    hipLaunchKernelGGL((k_lora_down<1, 1>), dim3((unsigned)(tiles * plan.ways), T, plan.split), dim3(256), 0, s, l);
  else
    hipLaunchKernelGGL((k_lora_down<4, 4>), dim3((unsigned)tiles, (T + 3) / 4, plan.split), dim3(256), 0, s, l);
  if (const int rc = krq_check_launch("lora_add")) return rc;
  if (plan.mt == 1) {
    if (fp32) launch_up<float, 1, false>(l, s);
    else launch_up<uint16_t, 1, false>(l, s);
  } else {
    if (fp32) launch_up<float, 4, true>(l, s);
    else launch_up<uint16_t, 4, true>(l, s);
  }
  return krq_check_launch("lora_add");
}

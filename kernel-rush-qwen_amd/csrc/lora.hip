// Low-rank adapters of many requests beside one shared projection:
//
//   out[m, n] = y[m, n] + s_i sum_r B_i[n, r] h[m, r],   h[m, r] = sum_k A_i,p(n)[r, k] x[m, k],   i = ids[m]
//
// for the P parts of a fused projection (part p(n) of column n), each with its own factors. Two launches: k_lora_down
// makes h, k_lora_up adds. Rows may name any adapters in any order: a tile of 16 takes its distinct ones one after the
// other (or, where rows are few, each in a workgroup of its own), multiplies the whole tile and writes the rows that
// name it; from 17 rows, windows of up to 256 are put in the order of their adapters first. The rows of a matrix-core
// operand do not mix, so rows of other adapters cost nothing but the idle columns, and a NaN stays in its row.
//
// What bounds it: the factors of the adapters in use, read once each, at few rows; x, y and out at many. The products
// are a few percent of the matrix cores' rate.
//
// The operands of the factors. v_mfma_f32_16x16x32_bf16 takes 16 bytes of one row per lane; sixteen consecutive lanes have
// sixteen rows, so that loads of row-major operands touch a line per lane (a launch of 4,096 x 2,560 rows took 11.5 us bound
// by that). A is kept in lane order, [K / 64][2][64 lanes][8] per 16 ranks, lane 16 g + j its rank j, k = 16 g + 8 e .. + 7 of a
// step's 64; rows of x are loaded eight lanes to a line and turned through LDS, each wave its own. B is kept as [r / 32][64 lanes][8]
// per 16 columns, lane 16 g + j column j, ranks 8 g .. + 7 of 32, and an odd last 16 ranks in 32 lanes (row-major, 4,096 rows of
// gate_up with rank 64 took 151 us, 119 this way).
//
// h is kept in fp32 and enters the second product as the sum of two bf16 (to 2^-16; three, to 2^-24, beside an fp32 y), so
// that the sum is rounded once, at the end: the second product takes two or three times the matrix instructions, which
// it has to spare.
#include <algorithm>

#include "mx_common.h"

using namespace krq;

namespace {

constexpr int kMaxParts = 8, kMaxRank = 256, kWindow = 256;
constexpr int kSplitFew = 4, kSplitMany = 2;  // parts of K at most, for up to kFewRows rows and for more

// What k_lora_down found at a place, in the 16 bytes that k_lora_up waits for: the row (24 bits) and id + 1 (24), under each the ranks
// of four parts (9 bits each), and above the row the 16 ranks past the first by which the slot's factors lie.
typedef ulonglong2 Place;
static_assert(kMaxParts <= 8 && kMaxRank <= 256);
KRQ_DEV int place_row(Place p) { return static_cast<int>(p.x & 0xffffff); }
KRQ_DEV int place_id(Place p) { return static_cast<int>(p.y & 0xffffff) - 1; }
KRQ_DEV int place_r16(Place p) { return 16 * static_cast<int>(p.x >> 60) + 16; }
KRQ_DEV int place_rank(Place p, int part) { return static_cast<int>((part < 4 ? p.x : p.y) >> (24 + 9 * (part & 3))) & 511; }

struct LoraArgs {
  const uint16_t* x;
  const void* ids;
  const uint16_t* a;     // [slots][P][R / 16][steps][2][64][8]: lane order, zeros past K
  const uint16_t* b;     // [slots][tiles 16 R]: for each tile of 16 columns and the slot's rank, rounded up to 16, lane order
  const int32_t* ranks;  // [slots], up to R; 0: none
  const int32_t* part_ranks;  // [slots][P], up to the slot's rank; null: the slot's for every part
  const float* scales;   // [slots]
  const void* y;
  void* out;
  Place* place;          // [M]
  float* h;              // [split][M][P R] by place, times the scale
  int64_t M, K, ldx, ldy, ldo;
  int slots, P, R, split, ids64, ways, window;
  int part[kMaxParts + 1], block[kMaxParts + 1];  // first column of each part; first group of column blocks
  int tile[kMaxParts + 1];                        // first tile of 16 columns: every part starts a new one
};

KRQ_DEV int load_id(const LoraArgs& a, int64_t m) {  // -1: none; slots: out of range
  const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[m] : static_cast<const int32_t*>(a.ids)[m];
  return id < 0 ? -1 : id >= a.slots ? a.slots : static_cast<int>(id);
}

KRQ_DEV int rank_of(const LoraArgs& a, int id) {
  return id < 0 || id >= a.slots ? 0 : min(max(a.ranks[id], 0), a.R);
}

KRQ_DEV v4f mfma32(uint4 a, uint4 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// The rows of a workgroup's window (up to 256 rows from w0) by adapter: the key of place i, id + 1 and the row in the
// window. A window of few runs of the same id, as requests that follow each other make, stays as it is; another is
// sorted (each row counts the rows before it, half of them in each of two threads), so that a tile of 16 places meets few
// adapters in whatever order the rows name them. Rows past M are last.
constexpr int kRunsMax = 12;
KRQ_DEV void sort_window(const LoraArgs& a, int64_t w0, uint32_t* raw, uint32_t* sorted) {
  const uint32_t t = threadIdx.x & (kWindow - 1), half = threadIdx.x / kWindow;
  const bool real = t < a.window && w0 + t < a.M;
  const uint32_t key = real ? static_cast<uint32_t>(load_id(a, w0 + t) + 1) << 8 | t : 0xffffffffu;
  if (half == 0) raw[t] = key;
  __syncthreads();
  const int runs = __syncthreads_count(half == 0 && t > 0 && raw[t - 1] >> 8 != key >> 8);
  uint32_t place = t;
  if (runs > kRunsMax) {
    uint32_t before = 0;
#pragma unroll 8
    for (int j = 0; j < kWindow / 2; j += 4) {
      const uint4 o = *reinterpret_cast<const uint4*>(raw + half * (kWindow / 2) + j);
      before += o.x < key;
      before += o.y < key;
      before += o.z < key;
      before += o.w < key;
    }
    if (half) sorted[t] = before;
    __syncthreads();
    if (!half) place = real ? before + sorted[t] : t;  // (past M: equal keys, each stays, behind the others)
    __syncthreads();
  }
  if (half == 0) sorted[place] = key;
  __syncthreads();
}

// The distinct ids of up to 64 places, one at a time: `id` is each lane's place's, `left` the lanes not yet taken.
KRQ_DEV int next_id(int id, uint64_t& left, uint64_t& same) {
  const int cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
  same = __ballot(id == cur) & left;
  left &= ~same;
  return cur;
}

// h. A workgroup takes MT tiles of 16 places, TC tiles of 16 ranks (of the P r of the adapter) and one of the `split`
// parts of K, its NW waves a part of that each, summed in LDS in wave order. A wave has few steps of 64 k, so that a launch is
// as long as its chain of loads, ids, ranks, the first NB steps: those of x wait for the row alone, and with TC = 1 those of
// A for the id alone.
template <int MT, int TC, int NW, int NB, bool SORT>
__global__ __launch_bounds__(64 * NW, TC <= 2 ? 4 : 2) void k_lora_down(LoraArgs a) {
  static_assert(64 * NW == 2 * kWindow);
  constexpr int kOwn = (TC > 2 ? TC : 2) * MT * 64;  // a wave's LDS: a step of x, then its sums
  __shared__ uint4 own[NW][kOwn];
  __shared__ uint32_t sorted[SORT ? kWindow : 1];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, j = lane & 15;
  // (the tiles' first workgroups before their second ones, which often have nothing to do: blocks go round the XCDs)
  const uint32_t tiles = gridDim.x / a.ways;
  const int64_t m0 = (blockIdx.x % tiles) * (int64_t)(16 * MT), w0 = SORT ? m0 / a.window * a.window : m0;
  const int way = blockIdx.x / tiles, slot = lane & (16 * MT - 1);
  // this wave's part of K, in steps of 64
  const int steps = static_cast<int>((a.K + 63) >> 6), q0 = blockIdx.z * NW + w, qn = a.split * NW;
  const int s0 = static_cast<int>((int64_t)steps * q0 / qn), s1 = static_cast<int>((int64_t)steps * (q0 + 1) / qn);
  int id;
  if constexpr (SORT) {
    sort_window(a, w0, reinterpret_cast<uint32_t*>(&own[0][0]), sorted);
    id = static_cast<int>(sorted[m0 - w0 + slot] >> 8) - 1;
  } else {
    id = load_id(a, min(m0 + slot, a.M - 1));
  }
  const int most = static_cast<int>(min(a.M - w0, (int64_t)(SORT ? a.window : 16))) - 1;
  auto row_of = [&](int place) {  // the row in the window of a place of the tile
    return min(SORT ? static_cast<int>(sorted[m0 - w0 + place] & 255u) : place, most);
  };
  // x: lane l takes 16 bytes l % 8 of rows l / 8 and 8 + l / 8 of a tile's 128 of a step
  const int c = lane & 7, last = static_cast<int>(a.K) - 8 - 8 * c;  // the last 8 k, from this lane's
  const uint8_t* xw = reinterpret_cast<const uint8_t*>(a.x + w0 * a.ldx);
  uint32_t xr[MT][2];  // (a window's rows lie within 4 GiB)
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) xr[i][e] = 2u * (row_of(16 * i + 8 * e + (lane >> 3)) * static_cast<uint32_t>(a.ldx) + 8 * c);
  uint4 av[NB][TC][2], xv[NB][MT][2];
  const uint4* ar[TC];
  auto load_x = [&](int s, int at) {
    if (s < s1) {
      const int k = min(64 * s, last);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          xv[at][i][e] = ld16(xw + (xr[i][e] + 2 * k));
        }
    }
  };
  auto load_a = [&](int s, int at) {
    if (s < s1) {
#pragma unroll
      for (int t = 0; t < TC; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) av[at][t][e] = ar[t][(2 * s + e) * 64];
    }
  };
  const bool real = m0 + slot < a.M && lane < 16 * MT;
  uint64_t left = __ballot(real);
  const int rank = real ? rank_of(a, id) : 0;
  const float scale = real && id >= 0 && id < a.slots ? a.scales[id] : 0.0f;
  auto write_place = [&]() {
    if (!real || w != 0 || way != 0 || blockIdx.y != 0 || blockIdx.z != 0) return;
    int own_rank[kMaxParts];  // (a last part again for those past it: loads without branches, all in flight)
    const bool known = a.part_ranks && id >= 0 && id < a.slots;
    const int32_t* from = known ? a.part_ranks + id * (int64_t)a.P : a.ranks;
#pragma unroll
    for (int p = 0; p < kMaxParts; ++p) own_rank[p] = from[known ? min(p, a.P - 1) : 0];
    auto four = [&](int p) {
      uint64_t v = 0;
#pragma unroll
      for (int i = 3; i >= 0; --i) v = v << 9 | static_cast<uint32_t>(known ? min(max(own_rank[p + i], 0), rank) : rank);
      return v << 24;
    };
    Place place;
    place.x = static_cast<uint32_t>(static_cast<int>(w0) + row_of(slot)) | four(0) | static_cast<uint64_t>(max(rank - 1, 0) >> 4) << 60;
    place.y = static_cast<uint32_t>(id + 1) | four(4);
    a.place[m0 + slot] = place;
  };
  // this workgroup's adapters of the tile: every `ways`-th, from the way-th
  int turn = -1, first, cur;
  uint64_t same;
  auto next = [&]() {
    if constexpr (!SORT) {  // one tile and a workgroup for each row: the first row of an adapter takes it
      const bool mine = left != 0;
      left = 0;
      first = way;
      cur = __builtin_amdgcn_readlane(id, way);
      same = __ballot(real && id == cur);
      return mine && cur >= 0 && cur < a.slots && __builtin_ctzll(same) == way;
    }
    while (left) {
      first = __builtin_ctzll(left);
      cur = next_id(id, left, same);
      if (cur >= 0 && cur < a.slots && ++turn % a.ways == way) return true;
    }
    return false;
  };
  if (!next()) return write_place();
#pragma unroll
  for (int u = 0; u < NB; ++u) load_x(s0 + u, u);
  write_place();
  bool fresh = true;
  do {
    const int R16 = a.R >> 4;
    int per = 1, T, t0 = blockIdx.y * TC;
    auto tile_at = [&](int tile) { return reinterpret_cast<const uint4*>(a.a) + ((int64_t)cur * a.P * R16 + tile) * steps * 128 + lane; };
    if constexpr (TC == 1) {  // tile blockIdx.y of the bank's, whatever the rank
      ar[0] = tile_at(t0);
#pragma unroll
      for (int u = 0; u < NB; ++u) load_a(s0 + u, u);
      per = (__builtin_amdgcn_readlane(rank, first) + 15) >> 4;
      if (t0 % R16 >= per) continue;
      t0 = t0 / R16 * per + t0 % R16;
      T = t0 + 1;
    } else {
      per = (__builtin_amdgcn_readlane(rank, first) + 15) >> 4;
      T = a.P * per;
      if (t0 >= T) continue;
#pragma unroll
      for (int t = 0; t < TC; ++t) {
        const int tt = min(t0 + t, T - 1);
        ar[t] = tile_at(tt / per * R16 + tt % per);
      }
#pragma unroll
      for (int u = 0; u < NB; ++u) load_a(s0 + u, u);
    }
    if (!fresh) {
#pragma unroll
      for (int u = 0; u < NB; ++u) load_x(s0 + u, u);
    }
    fresh = false;
    v4f acc[MT][TC] = {};
    auto multiply = [&](int s, int at) {
      // slot (row, chunk ^ row % 8): neither the writes nor the reads of a chunk of sixteen rows meet in a bank
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          own[w][i * 128 + (8 * e + (lane >> 3)) * 8 + (c ^ (lane >> 3))] = sel4(64 * s <= last, xv[at][i][e]);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const uint4 xo = own[w][i * 128 + j * 8 + ((2 * g + e) ^ (j & 7))];
#pragma unroll
          for (int t = 0; t < TC; ++t) acc[i][t] = mfma32(av[at][t][e], xo, acc[i][t]);
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    for (int s = s0; s < s1; s += NB) {
#pragma unroll
      for (int u = 0; u < NB; ++u)
        if (s + u < s1) {
          multiply(s + u, u);
          load_a(s + u + NB, u);
          load_x(s + u + NB, u);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < TC; ++t) own[w][(i * TC + t) * 64 + lane] = __builtin_bit_cast(uint4, acc[i][t]);
    __syncthreads();
    // lane: place j of a tile, ranks 4 g .. 4 g + 3
    const float sc = as_f32(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(as_u32(scale)), first)));
    for (int p = w; p < MT * TC; p += NW) {
      v4f v = __builtin_bit_cast(v4f, own[0][p * 64 + lane]);
#pragma unroll
      for (int q = 1; q < NW; ++q) v += __builtin_bit_cast(v4f, own[q][p * 64 + lane]);
      v *= sc;
      const int i = p / TC, t = t0 + p % TC;
      if (t < T && (same >> (16 * i + j) & 1))
        *reinterpret_cast<v4f*>(a.h + (blockIdx.z * a.M + m0 + 16 * i + j) * (a.P * a.R) + (t / per) * a.R + 16 * (t % per) + 4 * g) = v;
    }
    __syncthreads();
  } while (next());
}

// fp32 as the sum of NT bf16: each the rounded rest of those before it (none beside an infinity or a NaN)
template <int NT>
KRQ_DEV void split_bf16(float x, float y, uint32_t (&o)[NT]) {
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    o[i] = pack_bf16x2(x, y);
    const float hx = as_f32(o[i] << 16), hy = as_f32(o[i] & 0xffff0000u);
    x = finite_f32(hx) ? x - hx : 0.0f;
    y = finite_f32(hy) ? y - hy : 0.0f;
  }
}

// A lane's piece of a row: 16 bytes, VEC values, on any address that holds one (rows of an odd number of columns).
typedef unsigned int v4u_on2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int v4u_on4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T>
struct Piece {
  static constexpr int VEC = 16 / sizeof(T);
  v4u u;
  KRQ_DEV void load(const uint16_t* at) { u = *reinterpret_cast<const v4u_on2*>(at); }
  KRQ_DEV void load(const float* at) { u = *reinterpret_cast<const v4u_on4*>(at); }
  KRQ_DEV void store(uint16_t* at) const { *reinterpret_cast<v4u_on2*>(at) = u; }
  KRQ_DEV void store(float* at) const { *reinterpret_cast<v4u_on4*>(at) = u; }
  KRQ_DEV void load(const T* at, int n) {  // the first n values
    if (n >= VEC) return load(at);
    if (n <= 0) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2)
        u[i] = (2 * i < n ? at[2 * i] : 0u) | (2 * i + 1 < n ? static_cast<uint32_t>(at[2 * i + 1]) << 16 : 0u);
      else
        u[i] = i < n ? as_u32(at[i]) : 0u;
    }
  }
  KRQ_DEV void store(T* at, int n) const {
    if (n >= VEC) return store(at);
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i < n) {
        if constexpr (sizeof(T) == 2) at[i] = static_cast<uint16_t>(u[i >> 1] >> (16 * (i & 1)));
        else at[i] = as_f32(u[i]);
      }
  }
  KRQ_DEV void add(const v4f* acc) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2)
        u[i] = pack_bf16x2(as_f32(u[i] << 16) + acc[i >> 1][2 * (i & 1)], as_f32(u[i] & 0xffff0000u) + acc[i >> 1][2 * (i & 1) + 1]);
      else
        u[i] = as_u32(as_f32(u[i]) + acc[0][i]);
    }
  }
};

// y + the delta. A wave takes 16 places and NI blocks of 64 columns of one part; a lane finishes pieces of 16 bytes of
// one row, the four lanes of a row 64 contiguous bytes at a time. Of bf16, tile t of a block multiplies the columns
// 32 (t / 2) + 8 (i / 4) + 4 (t % 2) + i % 4, i = 0 .. 15, so that two accumulators make a piece; of fp32 the columns 16 t + i.
// ROWS: the workgroup's waves take four tiles of places, else four groups of columns.
template <typename T, int NI, bool ROWS>
__global__ __launch_bounds__(256, 4) void k_lora_up(LoraArgs a) {
  constexpr int SP = ROWS ? kSplitMany : kSplitFew;
  constexpr int NT = sizeof(T) == 2 ? 2 : 3;  // bf16 terms of h: to 2^-16 or 2^-24
  constexpr int VEC = Piece<T>::VEC, NP = 16 / VEC, TP = 4 / NP;  // pieces of a block, accumulators of a piece
  extern __shared__ uint4 stage[];  // h as operands: [wave][steps of 32 ranks][NT][lane]
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, j = lane & 15;
  const int units = a.block[a.P], wide_units = ROWS ? units : (units + 3) >> 2;  // (the columns of a row tile first)
  const int64_t at = blockIdx.x / wide_units;
  const int64_t m0 = ROWS ? (at * 4 + w) * 16 : at / a.ways * 16;
  const int way = ROWS ? 0 : static_cast<int>(at % a.ways);
  const int unit = ROWS ? blockIdx.x % wide_units : blockIdx.x % wide_units * 4 + w;
  if (m0 >= a.M || unit >= units) return;
  int p = 0;
  while (unit >= a.block[p + 1]) ++p;
  const int n0 = a.part[p] + (unit - a.block[p]) * 64 * NI, n1 = a.part[p + 1];
  const int64_t pc = min(m0 + j, a.M - 1);  // the lane's place
  const float* hr = a.h + pc * (a.P * a.R) + p * a.R;
  const int64_t slice = a.M * (a.P * a.R);
  // a step of 32 ranks of h, 8 g .. 8 g + 7 of them in this lane; the first waits for nothing
  // (an odd last 16 ranks: the lanes 32 .. 63 have the same as those 32 before them)
  auto load_h = [&](int s, bool odd, v4f (&f)[SP][2]) {
    const int r = min(32 * s + 8 * (odd ? g & 1 : g), a.R - 8);
#pragma unroll
    for (int q = 0; q < SP; ++q)
      if (q < a.split)
#pragma unroll
        for (int e = 0; e < 2; ++e) f[q][e] = *reinterpret_cast<const v4f*>(hr + q * slice + r + 4 * e);
  };
  v4f f[SP][2];
  load_h(0, a.R == 16, f);
  const Place place = a.place[pc];
  const int id = place_id(place), slot_r16 = place_r16(place), own_rank = place_rank(place, p);
  uint64_t left = __ballot(m0 + j < a.M) & 0xffff;
  uint4* st = stage + w * ((a.R + 31) / 32) * NT * 64 + lane;
  const T* yr = static_cast<const T*>(a.y) + (int64_t)place_row(place) * a.ldy;
  T* orow = static_cast<T*>(a.out) + (int64_t)place_row(place) * a.ldo;
  bool fresh = true;  // f holds the first step
  for (int turn = 0; left; ++turn) {
    uint64_t same;
    int first = __builtin_ctzll(left), cur;
    if (!ROWS && a.M <= 16) {  // one tile and a workgroup for each row
      first = way;
      cur = __builtin_amdgcn_readlane(id, way);
      same = __ballot(id == cur) & left;
      left = 0;
      if (__builtin_ctzll(same) != way) return;
    } else {
      cur = next_id(id, left, same);
      if (!ROWS && turn % a.ways != way) continue;
    }
    const bool me = same >> j & 1;
    // the factors lie by the slot's rank; the sum is over the part's own, past which they hold zeros for which an h may not be finite
    const int r16 = __builtin_amdgcn_readlane(slot_r16, first), rank = __builtin_amdgcn_readlane(own_rank, first);
    if (rank == 0 && cur < a.slots && a.out == a.y) continue;
    // whole blocks of the wave, all their y in flight before anything else; a last block that the part ends in by itself
    const int whole = min(NI, (n1 - n0) >> 6);
    Piece<T> v[NI][NP];
    if (me) {
#pragma unroll
      for (int blk = 0; blk < NI; ++blk)
        if (blk < whole)
#pragma unroll
          for (int q = 0; q < NP; ++q) v[blk][q].load(yr + n0 + VEC * g + 64 * blk + 4 * VEC * q);
    }
    // this place's h, summed over the parts of K in order, in NT terms
    for (int s = 0; 32 * s < rank; ++s) {
      const bool odd = 32 * s + 16 == r16;
      if (!(fresh && s == 0 && odd == (a.R == 16))) load_h(s, odd, f);
      v4f v2[2] = {f[0][0], f[0][1]};
#pragma unroll
      for (int q = 1; q < SP; ++q)
        if (q < a.split) v2[0] += f[q][0], v2[1] += f[q][1];
#pragma unroll
      for (int i = 0; i < 8; ++i) v2[i >> 2][i & 3] = me && 32 * s + 8 * (odd ? g & 1 : g) + i < rank ? v2[i >> 2][i & 3] : 0.0f;
      uint32_t o[4][NT];
#pragma unroll
      for (int i = 0; i < 4; ++i) split_bf16<NT>(v2[i >> 1][2 * (i & 1)], v2[i >> 1][2 * (i & 1) + 1], o[i]);
#pragma unroll
      for (int e = 0; e < NT; ++e) {
        uint4 u = make_uint4(o[0][e], o[1][e], o[2][e], o[3][e]);
        if (odd && g >= 2) u = e + 1 < NT ? make_uint4(o[0][e + 1 < NT ? e + 1 : e], o[1][e + 1 < NT ? e + 1 : e], o[2][e + 1 < NT ? e + 1 : e], o[3][e + 1 < NT ? e + 1 : e]) : zero4();
        st[(s * NT + e) * 64] = u;
      }
      fresh = false;
    }
    const uint8_t* bs = reinterpret_cast<const uint8_t*>(a.b) + (int64_t)(rank ? cur : 0) * a.tile[a.P] * (32 * a.R);
    // the products of the 64 columns of block nb of the part. Column j of the operand of tile t: see above; of fp32 it is the
    // column j of the factor's tile t, of bf16 it lies in tile 2 (t / 2) + j / 8, there 8 (j / 4 % 2) + 4 (t % 2) + j % 4
    const int first_tile = a.tile[p] + ((n0 - a.part[p]) >> 4), last_tile = a.tile[p + 1] - 1;
    const int row = sizeof(T) == 2 ? 8 * ((j >> 2) & 1) + (j & 3) : j, over = sizeof(T) == 2 ? j >> 3 : 0;
    auto product = [&](int blk, bool edge, v4f* acc) {
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t] = v4f{};
      const int64_t size = 32 * r16;  // bytes of a tile
      const uint8_t* base = bs + (first_tile + 4 * blk) * size;
      const int most = last_tile - (first_tile + 4 * blk);
      for (int s = 0; 32 * s < rank; ++s) {
        const bool odd = 32 * s + 16 == r16;
        const uint32_t lane_at = 16u * (16 * (odd ? g & 1 : g) + row);
        uint4 bv[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int tile = sizeof(T) == 2 ? 2 * (t >> 1) : t, sub = sizeof(T) == 2 ? 64 * (t & 1) : 0;
          bv[t] = ld16(edge ? base + min(tile + over, most) * size + (1024 * s + sub + lane_at)
                            : base + tile * size + 1024 * s + sub + (static_cast<uint32_t>(over * size) + lane_at));
        }
#pragma unroll
        for (int e = 0; e < NT; ++e) {
          if (odd && e % 2) continue;  // (two terms of 16 ranks in one operand)
          const uint4 h = st[(s * NT + e) * 64];
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[t] = mfma32(bv[t], h, acc[t]);
        }
      }
    };
    auto finish = [&](Piece<T>& u, const v4f* acc) {
      if (rank) u.add(acc);
      if (cur >= a.slots) {
        constexpr uint32_t nan = sizeof(T) == 2 ? 0x7fc07fc0u : 0x7fc00000u;
        u.u = v4u{nan, nan, nan, nan};
      }
    };
    v4f acc[4];
#pragma unroll
    for (int blk = 0; blk < NI; ++blk) {
      if (blk < whole) {
        if (rank) product(blk, false, acc);
#pragma unroll
        for (int q = 0; q < NP; ++q) {
          finish(v[blk][q], acc + TP * q);
          if (me) v[blk][q].store(orow + n0 + VEC * g + 64 * blk + 4 * VEC * q);
        }
      }
    }
    const int ne = n0 + 64 * whole;
    if (whole < NI && ne < n1) {
      if (rank) product(whole, true, acc);
#pragma unroll
      for (int q = 0; q < NP; ++q) {
        const int n = ne + VEC * g + 4 * VEC * q;
        Piece<T> u;
        if (me) u.load(yr + n, n1 - n);
        finish(u, acc + TP * q);
        if (me) u.store(orow + n, n1 - n);
      }
    }
  }
}

struct LoraPlan {
  int split, mt, tc, ways;
};

constexpr int kDownWaves = 8, kFewRows = 384, kShortTiles = 6600;
constexpr int64_t kUpGroups = 2000;

// The most parts of K: two steps of 64 k for a wave at the least.
int64_t most_parts(int64_t M, int64_t K) {
  return std::max<int64_t>(1, std::min<int64_t>(K / (64 * 2 * kDownWaves), M <= kFewRows ? kSplitFew : kSplitMany));
}

// The first launch's tiles. Rows: 16 at a time; 32 from kShortTiles products of a row and 16 ranks on, so that the factors are read half as
// often (both launches, us, 16 / 32 rows: 1,715 x 4,976, rank 32, 23.5 / 27.9; 3,744 x 464, two parts of rank 24, 21.0 / 18.1).
// Ranks: up to two tiles of 16 together, or four from kFewRows rows on, so that the rows are read fewer times; one where
// there would be less than 64 workgroups with work, a quarter of the CUs (186 x 7,056, two parts of rank 32, one / two / four:
// 18.4 / 17.0 / 18.9). The adapters that a tile meets go to `ways` workgroups: the mean, slots 16 mt / window, of a bank whose slots
// are all in use, and two more (75 rows of 14 adapters, 1,984 x three parts of rank 32: 14.2, with one way less 16.9). K in as many
// parts as keep the workgroups with work to 192 at few rows, three quarters of the CUs, so that there is no second round of them
// (85 x 8,592, 13 adapters, three parts of rank 24, one / two / four: 22.1 / 18.1 / 19.9), and to 5 K / 64 at many: the more
// steps of 64 a wave has, the more of a second round its halving is worth.
// kShortTiles, the 64, the 192 and the 5 are fits to this card, over 140 drawn calls of 17 to 4,096 rows: at the mean 2 % behind
// the best of 16 plans each. Another count of CUs or another kernel needs them again.
LoraPlan lora_plan(int64_t M, int64_t K, int P, int R, int64_t slots) {
  LoraPlan p;
  const int T = P * R / 16;
  const int64_t most = most_parts(M, K), window = std::min<int64_t>(M, kWindow);
  if (M <= 16) {  // a workgroup for each row
    p.mt = p.tc = 1;
    p.ways = static_cast<int>(M);
    p.split = static_cast<int>(std::min<int64_t>(most, (512 + M * T - 1) / (M * T)));
    return p;
  }
  const bool few = M <= kFewRows;
  p.mt = few || M * T <= kShortTiles ? 1 : 2;
  p.ways = static_cast<int>(std::min<int64_t>({few ? 16 : 4, slots, (slots * 32 * p.mt + 5 * window) / (2 * window)}));
  // 16 times the adapters that a tile meets at the mean
  const int64_t tiles = (M + 16 * p.mt - 1) / (16 * p.mt), met = std::min<int64_t>({16 * slots, 256 * p.mt, 16 + slots * 256 * p.mt / window});
  const int wide = tiles * T * met < 16 * 64 ? 1 : few ? 2 : 4, groups = (T + wide - 1) / wide;
  p.tc = (T + groups - 1) / groups;
  p.split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(most, 16 * (few ? 192 : 5 * K / 64) / (tiles * groups * met))));
  return p;
}

template <int MT, int TC, bool SORT>
void launch_down(const LoraArgs& a, hipStream_t s) {
  const int64_t tiles = (a.M + 16 * MT - 1) / (16 * MT);
  const int T = a.P * a.R / 16;
  hipLaunchKernelGGL((k_lora_down<MT, TC, kDownWaves, MT * TC == 1 ? 3 : 2, SORT>), dim3((unsigned)(tiles * a.ways), (T + TC - 1) / TC, a.split),
                     dim3(64 * kDownWaves), 0, s, a);
}

template <typename T, int NI, bool ROWS>
void launch_up(const LoraArgs& a, hipStream_t s) {
  LoraArgs u = a;
  u.block[0] = 0;
  for (int p = 0; p < a.P; ++p) u.block[p + 1] = u.block[p] + (a.part[p + 1] - a.part[p] + 64 * NI - 1) / (64 * NI);
  const int64_t units = u.block[a.P], tiles = (a.M + 15) / 16;
  const dim3 grid(static_cast<unsigned>(ROWS ? units * ((tiles + 3) / 4) : (units + 3) / 4 * tiles * a.ways));
  const size_t smem = static_cast<size_t>(4) * ((a.R + 31) / 32) * (sizeof(T) == 2 ? 2 : 3) * 64 * 16;
  hipLaunchKernelGGL((k_lora_up<T, NI, ROWS>), grid, dim3(256), smem, s, u);
}

// Column blocks of 64 that a wave of the many-row form takes: one where that leaves few workgroups, else 512 bytes of a row. Both launches
// of a graph, us, one / four: 777 rows of QKV 19.2 / 20.8, 2,048 24.1 / 22.7, 4,096 rows of gate_up 126 / 91.6.
template <typename T>
void launch_up_any(const LoraArgs& a, hipStream_t s) {
  if (a.M <= kFewRows) return launch_up<T, 1, false>(a, s);
  int64_t blocks = 0;
  for (int p = 0; p < a.P; ++p) blocks += (a.part[p + 1] - a.part[p] + 63) / 64;
  if (blocks * ((a.M + 63) / 64) < kUpGroups) launch_up<T, 1, true>(a, s);
  else launch_up<T, sizeof(T) == 2 ? 4 : 2, true>(a, s);
}

// places, then h
int64_t place_bytes(int64_t M) { return (M * (int64_t)sizeof(Place) + 255) / 256 * 256; }

}  // namespace

extern "C" int64_t krq_lora_ws_bytes(int64_t M, int64_t K, int parts, int rank) {
  if (M < 1 || K < 16 || parts < 1 || parts > kMaxParts || rank < 16 || rank > kMaxRank) return -1;
  return place_bytes(M) + most_parts(M, K) * M * parts * rank * (int64_t)sizeof(float);
}

namespace {

int lora_add(const void* x, int64_t ldx, const void* ids, int ids_64, const void* a, const void* b, const int32_t* ranks,
                    const int32_t* part_ranks, const float* scales, int64_t slots, int64_t M, int64_t K, const int64_t* parts_n,
                    int parts, int rank, const void* y, int64_t ldy, void* out, int64_t ldo, int fp32, void* ws, int64_t ws_bytes,
                    void* stream) {
  KRQ_REQUIRE(x && ids && a && b && ranks && scales && parts_n && y && out && ws, "lora_add: null pointer");
  KRQ_REQUIRE(M >= 1 && M <= (1 << 24) && K >= 16 && K % 16 == 0 && K < (1 << 22), "lora_add: bad shape M=%lld K=%lld (K a multiple of 16)",
              (long long)M, (long long)K);
  KRQ_REQUIRE(parts >= 1 && parts <= kMaxParts, "lora_add: %d parts (at most %d)", parts, kMaxParts);
  KRQ_REQUIRE(rank >= 16 && rank % 16 == 0 && rank <= kMaxRank, "lora_add: rank=%d (a multiple of 16, at most %d)", rank, kMaxRank);
  KRQ_REQUIRE(slots >= 1 && slots < (1 << 23), "lora_add: %lld slots", (long long)slots);
  KRQ_REQUIRE(ldx >= K && ldx % 8 == 0 && ldx < (1 << 22) && aligned16(x), "lora_add: rows of x must start on 16 bytes, less than 2^22 apart (ldx=%lld)",
              (long long)ldx);
  KRQ_REQUIRE(aligned16(a) && aligned16(b) && aligned16(ws), "lora_add: the factors and ws must start on 16 bytes");
  LoraArgs l{};
  int64_t n = 0;
  for (int p = 0; p < parts; ++p) {
    KRQ_REQUIRE(parts_n[p] >= 1 && parts_n[p] <= (1 << 24), "lora_add: part %d of %lld columns", p, (long long)parts_n[p]);
    l.part[p] = static_cast<int>(n);
    n += parts_n[p];
    l.part[p + 1] = static_cast<int>(n);
    l.tile[p + 1] = l.tile[p] + static_cast<int>((parts_n[p] + 15) / 16);
  }
  KRQ_REQUIRE(ldy >= n && ldo >= n, "lora_add: rows of %lld columns %lld and %lld apart", (long long)n, (long long)ldy, (long long)ldo);
  const int esize = fp32 ? 4 : 2;
  KRQ_REQUIRE((reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out)) % esize == 0, "lora_add: y and out must start on a value");
  KRQ_REQUIRE(y != out || ldy == ldo, "lora_add: out is y with other rows");
  // (the second launch's workgroups at the most: of few rows one for each way, of many a wave has 512 bytes of a row)
  KRQ_REQUIRE((M <= kFewRows ? (M + 15) / 16 * 16 * (n / 256 + parts) : (M + 63) / 64 * (n / (fp32 ? 128 : 256) + parts)) < (1 << 24), "lora_add: %lld x %lld is too large", (long long)M, (long long)n);
  const LoraPlan plan = lora_plan(M, K, parts, rank, slots);
  KRQ_REQUIRE(ws_bytes >= krq_lora_ws_bytes(M, K, parts, rank), "lora_add: ws of %lld bytes is too small", (long long)ws_bytes);
  l.x = (const uint16_t*)x;
  l.ids = ids;
  l.a = (const uint16_t*)a;
  l.b = (const uint16_t*)b;
  l.ranks = ranks;
  l.part_ranks = part_ranks;
  l.scales = scales;
  l.y = y;
  l.out = out;
  l.place = (Place*)ws;
  l.h = (float*)((uint8_t*)ws + place_bytes(M));
  l.M = M;
  l.K = K;
  l.ldx = ldx;
  l.ldy = ldy;
  l.ldo = ldo;
  l.slots = (int)slots;
  l.P = parts;
  l.R = rank;
  l.split = plan.split;
  l.ids64 = ids_64 != 0;
  l.ways = plan.ways;
  // windows of one size, so that a short last one has no tile of many adapters
  const int64_t windows = (M + kWindow - 1) / kWindow;
  l.window = static_cast<int>(((M + windows - 1) / windows + 31) / 32 * 32);
  hipStream_t s = (hipStream_t)stream;
  if (M <= 16) launch_down<1, 1, false>(l, s);
  else if (plan.mt == 1 && plan.tc == 1) launch_down<1, 1, true>(l, s);
  else if (plan.mt == 1 && plan.tc == 2) launch_down<1, 2, true>(l, s);
  else if (plan.mt == 1 && plan.tc == 3) launch_down<1, 3, true>(l, s);
  else if (plan.mt == 1) launch_down<1, 4, true>(l, s);
  else if (plan.tc == 1) launch_down<2, 1, true>(l, s);
  else if (plan.tc == 2) launch_down<2, 2, true>(l, s);
  else if (plan.tc == 3) launch_down<2, 3, true>(l, s);
  else launch_down<2, 4, true>(l, s);
  if (const int rc = krq_check_launch("lora_add")) return rc;
  if (fp32) launch_up_any<float>(l, s);
  else launch_up_any<uint16_t>(l, s);
  return krq_check_launch("lora_add");
}

}  // namespace

extern "C" int krq_lora_add(const void* x, int64_t ldx, const void* ids, int ids_64, const void* a, const void* b, const int32_t* ranks,
                            const float* scales, int64_t slots, int64_t M, int64_t K, const int64_t* parts_n, int parts, int rank,
                            const void* y, int64_t ldy, void* out, int64_t ldo, int fp32, void* ws, int64_t ws_bytes, void* stream) {
  return lora_add(x, ldx, ids, ids_64, a, b, ranks, nullptr, scales, slots, M, K, parts_n, parts, rank, y, ldy, out, ldo, fp32, ws,
                  ws_bytes, stream);
}

extern "C" int krq_lora_add_parts(const void* x, int64_t ldx, const void* ids, int ids_64, const void* a, const void* b,
                                  const int32_t* ranks, const int32_t* part_ranks, const float* scales, int64_t slots, int64_t M,
                                  int64_t K, const int64_t* parts_n, int parts, int rank, const void* y, int64_t ldy, void* out,
                                  int64_t ldo, int fp32, void* ws, int64_t ws_bytes, void* stream) {
  KRQ_REQUIRE(part_ranks, "lora_add: null pointer");
  return lora_add(x, ldx, ids, ids_64, a, b, ranks, part_ranks, scales, slots, M, K, parts_n, parts, rank, y, ldy, out, ldo, fp32, ws,
                  ws_bytes, stream);
}

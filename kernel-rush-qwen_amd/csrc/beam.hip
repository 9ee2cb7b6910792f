// Beam search's step behind the lm head: the n best continuations of every batch entry's beams, and the states put in
// their order.
//
// Selection. v[w, t] = score[w] + (logit[w, t] - lse[w]), lse[w] = log sum_t exp(logit[w, t]); the n largest v of an
// entry's W beams, ties to the lower beam, then to the lower token. Within a beam v goes as the logit, so the logits are
// read once, by k_beam_rows: a workgroup takes a chunk of a row, keeps it in registers, and leaves the chunk's largest
// value, its sum of exponentials and its n largest logits (with tokens, in order). k_beam_pick then takes a batch
// entry: lse and the merged n of every row, and the merge of the rows by v, added and compared in fp64.
//
// lse is as good as the fp32 exponentials and sums behind it, off by less than 64 u = 2^-18 (u = 2^-24, vocabularies up to 2^20): a term's
// distance t to the chunk's largest and on to the row's takes three roundings, 2.3 u |t|, whose mean over the terms is at most
// 24 u (the weighed mean of |t| is W(V / e) at most); two exponentials and a product 5 u; 17 additions 17 u. Candidates of
// one beam are in the order of their logits; those of two beams within 2^-17 may come in either order. (Exponentials in fp64 settle that: 8 x 8
// beams 16.1 -> 21.1 us, 1 x 4 9.2 -> 9.9; the fp32 argument's rest carried to first order halves the bound: 17.9.)
//
// The n largest of a chunk. The n-th largest of 64 groups' largest values, found by its upper 16 bits with ballots, has n
// values at or above it, and few more: those go to LDS, and each finds its place by counting the larger ones. Logit and
// token make one 64-bit key for that, all of them different: the logit's bits in an order that compares as unsigned (NaN over
// everything), then the token's complement. Where equal logits leave too many (a mask, a coarse type), the n-th largest
// is taken of the lanes' largest keys instead, which only n lanes of a wave reach.
//
// Bound by the read of the logits from a few rows on; by the two launches' latencies below.
#include <algorithm>

#include "gemv_common.h"

using namespace krq;

namespace {

constexpr int kBeamMax = 64, kBeamThreads = 256, kPickThreads = 1024, kPickWaves = kPickThreads / 64;
constexpr uint32_t kOrdInf = 0xff800000u, kOrdNegInf = 0x007fffffu;

// fp32 bits in an order that compares as unsigned: NaN on top, -0 as +0
KRQ_DEV uint32_t ord_of(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = as_u32(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
KRQ_DEV float of_ord(uint32_t o) { return as_f32(o & 0x80000000u ? o & 0x7fffffffu : ~o); }  // (not of a NaN's)
KRQ_DEV uint64_t ord_of_f64(double f) {
  if (f != f) return ~0ull;
  const uint64_t u = __builtin_bit_cast(uint64_t, f + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}
KRQ_DEV uint32_t hi32(uint64_t k) { return static_cast<uint32_t>(k >> 32); }

// The n-th largest of the wave's 64 keys (different but for zeros): its upper half bit by bit, then among the lanes that
// share that the lower.
KRQ_DEV uint64_t nth_key(uint64_t key, int n) {
  const uint32_t hi = hi32(key), lo = static_cast<uint32_t>(key);
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 0; --b) {
    const uint32_t c = t | 1u << b;
    if (__popcll(__ballot(hi >= c)) >= n) t = c;
  }
  const int more = __popcll(__ballot(hi > t));
  const uint64_t tied = __ballot(hi == t);
  uint32_t u = 0;
  if (__popcll(tied) > 1) {
#pragma unroll
    for (int b = 31; b >= 0; --b) {
      const uint32_t c = u | 1u << b;
      if (more + __popcll(__ballot(hi == t && lo >= c)) >= n) u = c;
    }
  } else {
    u = __builtin_amdgcn_readlane(static_cast<int>(lo), __builtin_ctzll(tied | 1ull << 63));
  }
  return static_cast<uint64_t>(t) << 32 | u;
}

struct RowStat {
  uint32_t top;  // ord_of the chunk's largest value, a NaN's where one is among them
  float sum;     // sum of exp(value - largest)
};

// 16 bytes of logits that start on any of them (an odd vocabulary's rows): chunks and threads take the same tokens wherever
// a row starts, so that equal rows have equal sums.
typedef unsigned int v4u_on2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int v4u_on4 __attribute__((ext_vector_type(4), aligned(4)));
KRQ_DEV v4u ld16_any(const uint16_t* p) { return *reinterpret_cast<const v4u_on2*>(p); }
KRQ_DEV v4u ld16_any(const float* p) { return *reinterpret_cast<const v4u_on4*>(p); }

// The largest threshold of 16 upper bits that n of the wave's values reach.
KRQ_DEV uint32_t nth_upper(uint32_t ord, int n) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t c = t | 1u << b;
    if (__popcll(__ballot(ord >= c)) >= n) t = c;
  }
  return t;
}

// Sum over the lanes before this one, and over all.
KRQ_DEV int wave_before(int v, int& all) {
  const int lane = threadIdx.x & 63;
  int s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(s, d, 64);
    if (lane >= d) s += o;
  }
  all = __builtin_amdgcn_readlane(s, 63);
  return s - v;
}

constexpr int kFewKeys = 512, kSegKeys = kFewKeys / 4;  // keys that are ranked as they come; of a wave

template <typename T, int NV>
__global__ __launch_bounds__(kBeamThreads) void k_beam_rows(const T* __restrict__ logits, int64_t ld, int64_t V, int n, int chunks,
                                                            RowStat* __restrict__ stat, uint64_t* __restrict__ cand) {
  constexpr int VEC = 16 / sizeof(T), P = NV * VEC, CH = P * kBeamThreads;
  extern __shared__ __attribute__((aligned(16))) uint64_t list[];  // [max(4 n P, kFewKeys)]
  __shared__ float tops[kBeamThreads], sums[4];
  __shared__ uint64_t nth[4];
  __shared__ int counts[4];
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63, c = blockIdx.x;
  const int64_t row = blockIdx.y;
  const T* r = logits + row * ld;
  const int64_t base = (int64_t)c * CH;
  const int left = static_cast<int>(min(V - base, (int64_t)CH));  // tokens of the chunk
  float f[P];  // (places past V hold -inf)
  auto unpack = [](v4u a, float* o) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 2) o[2 * i] = as_f32(a[i] << 16), o[2 * i + 1] = as_f32(a[i] & 0xffff0000u);
      else o[i] = as_f32(a[i]);
    }
  };
  // Place i of the thread's vector v: 16 bytes of a row to a thread, but token by token in a chunk of so few that they
  // would be in one wave (a row's last 130 tokens, n = 19: all reached, past that wave's list, 11.3 us for 4.5).
  const bool spread = left < 64 * VEC;
  auto token = [&](int v, int i) { return spread ? (v * VEC + i) * kBeamThreads + tid : (v * kBeamThreads + tid) * VEC + i; };
  auto load = [&](int v, float* o) {
    const int e = token(v, 0);
    if (!spread && e + VEC <= left) {
      unpack(ld16_any(r + base + e), o);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        o[i] = -__builtin_inff();
        const int at = token(v, i);
        if (at < left) {
          if constexpr (sizeof(T) == 2) o[i] = bf16_to_f32(r[base + at]);
          else o[i] = r[base + at];
        }
      }
    }
  };
  if (left == CH) {  // (all loads in flight at once: a branch around each would wait for it)
    v4u a[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) a[v] = ld16_any(r + base + (v * kBeamThreads + tid) * VEC);
#pragma unroll
    for (int v = 0; v < NV; ++v) unpack(a[v], f + v * VEC);
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) load(v, f + v * VEC);
  }
  auto key_of = [&](int v, int i, float value) {  // of place i of the thread's vector v; 0 past V
    const int e = token(v, i);
    return e < left ? static_cast<uint64_t>(ord_of(value)) << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(base + e)) : 0;
  };
  float top = f[0];
#pragma unroll
  for (int i = 1; i < P; ++i) top = fmaxf(top, f[i]);  // (a NaN shows in the sum)
  // the largest of the four waves' lanes of a number: the n-th largest of those 64 is reached by n values, and by few more
  // (of 8,192, for n = 16, by 18 at the mean; the n-th of a wave's own lanes by 70)
  tops[tid] = top == top ? top : -__builtin_inff();
  __syncthreads();
  top = fmaxf(fmaxf(tops[lane], tops[lane + 64]), fmaxf(tops[lane + 128], tops[lane + 192]));
  const uint32_t ord = ord_of(top), t = nth_upper(ord, n);
  const float m = of_ord(wave_max_u32_dpp(ord));
  uint64_t* out = cand + (row * chunks + c) * n;
  if (m == -__builtin_inff()) {  // masked altogether: its first tokens (with a NaN, its row's candidates are not read)
    bool nan = false;
#pragma unroll
    for (int i = 0; i < P; ++i) nan |= f[i] != f[i];
    nan = __syncthreads_or(nan);
    if (tid < n) out[tid] = tid < left ? static_cast<uint64_t>(kOrdNegInf) << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(base + tid)) : 0;
    if (tid == 0) stat[row * chunks + c] = RowStat{nan ? 0xffffffffu : kOrdNegInf, 0.0f};
    return;
  }
  // Fewer than n groups with a finite value (a mask that ends in the chunk): the finite ones are taken, and then the first
  // masked tokens.
  const bool few = t <= kOrdNegInf;
  const float tf = few ? -3.40282347e38f : of_ord(t);
  // every wave its own part of the list, as far as that goes; the count tells whether it did
  uint64_t* seg = list + w * kSegKeys;
  int mine = 0;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const bool in = f[i] >= tf;
    const uint64_t mask = __ballot(in);
    if (mask) {
      const int at = mine + static_cast<int>(__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                                                       __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0)));
      if (in && at < kSegKeys) seg[at] = key_of(i / VEC, i % VEC, f[i]);  // (0 past V)
      mine += __popcll(mask);
    }
  }
  if (lane == 0 && (mine & 1) && mine < kSegKeys) seg[mine] = 0;  // (read in pairs)
  float s4[4] = {};  // (four sums: fewer roundings behind each other)
#pragma unroll
  for (int i = 0; i < P; ++i) s4[i & 3] += __builtin_amdgcn_exp2f((f[i] - m) * 1.44269504f);
  const float s = wave_sum((s4[0] + s4[1]) + (s4[2] + s4[3]));
  if (lane == 0) sums[w] = s, counts[w] = mine;
  __syncthreads();
  const int most = max(max(counts[0], counts[1]), max(counts[2], counts[3]));
  int have = counts[0] + counts[1] + counts[2] + counts[3];
  // (a NaN gives a sum of NaN, and +inf does)
  if (tid == 0) {
    const float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    stat[row * chunks + c] = RowStat{sum != sum ? 0xffffffffu : ord_of(m), sum};
  }
  if (most <= kSegKeys) {
    // sixteen of the wave's keys at a time, a quarter of the lanes for each wave's list
    const int q = lane >> 4, others = counts[q];
    const ulonglong2* from = reinterpret_cast<const ulonglong2*>(list + q * kSegKeys);
    for (int i0 = 0; i0 < mine; i0 += 16) {
      const int i = i0 + (lane & 15);
      const uint64_t key = i < mine ? seg[i] : 0;
      int rank = 0;
#pragma unroll 4
      for (int j = 0; 2 * j < others; ++j) {
        const ulonglong2 k2 = from[j];
        rank += k2.x > key;
        rank += k2.y > key;
      }
      rank += __shfl_xor(rank, 16, 64);
      rank += __shfl_xor(rank, 32, 64);
      if (q == 0 && rank < n && key) out[rank] = key;
    }
    if (few && have < n) {  // n - have masked tokens more, which lie among the first have + n, if the chunk has them
      __syncthreads();      // (counts are written again)
      const int span = min(left, have + n);
      int found = have;
      for (int i0 = 0; i0 < span; i0 += kBeamThreads) {
        const int i = i0 + tid;
        float v = 0.0f;
        if (i < span) {
          if constexpr (sizeof(T) == 2) v = bf16_to_f32(r[base + i]);
          else v = r[base + i];
        }
        const bool masked = v == -__builtin_inff();
        const uint64_t mask = __ballot(masked);
        if (lane == 0) counts[w] = __popcll(mask);
        __syncthreads();
        int at = found + __popcll(mask & ((1ull << lane) - 1));
        for (int q = 0; q < w; ++q) at += counts[q];
        if (masked && at < n)
          out[at] = static_cast<uint64_t>(kOrdNegInf) << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(base + i));
        found += counts[0] + counts[1] + counts[2] + counts[3];
        __syncthreads();
      }
      have = found;
    }
    for (int i = have + tid; i < n; i += kBeamThreads) out[i] = 0;  // (the chunk has fewer)
  } else {  // by keys, the logits read again (a launch of equal logits: few registers for it)
    float o[VEC];
    uint64_t best = 0;
#pragma unroll 1
    for (int v = 0; v < NV; ++v) {
      load(v, o);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const uint64_t k = key_of(v, i, o[i]);
        best = k > best ? k : best;
      }
    }
    const uint64_t exact = nth_key(best, n);
    if (lane == 0) nth[w] = exact;
    __syncthreads();
    uint64_t lk = nth[0];
#pragma unroll
    for (int q = 1; q < 4; ++q) lk = nth[q] > lk ? nth[q] : lk;
    mine = 0;
#pragma unroll 1
    for (int v = 0; v < NV; ++v) {
      load(v, o);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const uint64_t k = key_of(v, i, o[i]);
        mine += k >= lk && k;
      }
    }
    int all, at = wave_before(mine, all);
    if (lane == 0) counts[w] = all;
    __syncthreads();
    have = counts[0] + counts[1] + counts[2] + counts[3];
    for (int q = 0; q < w; ++q) at += counts[q];
#pragma unroll 1
    for (int v = 0; v < NV; ++v) {
      load(v, o);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const uint64_t k = key_of(v, i, o[i]);
        if (k >= lk && k) list[at++] = k;  // (at most n lanes of a wave, P keys each)
      }
    }
    __syncthreads();
    for (int i = tid; i < have; i += kBeamThreads) {
      const uint64_t key = list[i];
      int rank = 0;
      for (int j = 0; j < have; ++j) rank += list[j] > key;
      if (rank < n) out[rank] = key;
    }
    for (int i = have + tid; i < n; i += kBeamThreads) out[i] = 0;
  }
}

// One batch entry. A wave merges a row at a time, its keys in registers where they are up to KR a lane; then every row's
// sorted candidates meet in LDS, where each finds its place by binary searches in the other rows, by several threads for
// each where there are (counting all of 260 took 10 us, of 450 19).
template <int KR>
__global__ __launch_bounds__(kPickThreads) void k_beam_pick(const RowStat* __restrict__ stat, const uint64_t* __restrict__ cand,
                                                            const float* __restrict__ scores, int64_t V, int W, int n, int chunks,
                                                            int lists, float* __restrict__ out_scores,
                                                            int64_t* __restrict__ out_beams, int64_t* __restrict__ out_tokens) {
  __shared__ int ranks[kPickThreads];
  extern __shared__ uint64_t mem[];  // values [W][n], tokens [W][n] (32 bits), a list for each of `lists` waves [n * per]
  const int tid = threadIdx.x, threads = blockDim.x, wave = tid >> 6, lane = tid & 63;
  const int64_t b = blockIdx.x;
  const int total = chunks * n, per = (total + 63) >> 6, len = static_cast<int>(min((int64_t)n, V));
  uint64_t* vals = mem;
  uint32_t* toks = reinterpret_cast<uint32_t*>(mem + W * n);
  uint64_t* list = mem + W * n + (W * n + 1) / 2 + (int64_t)wave * n * per;
  for (int w = wave; wave < lists && w < W; w += lists) {
    const int64_t row = b * W + w;
    const RowStat* st = stat + row * chunks;
    const uint64_t* rc = cand + row * total;
    uint64_t k[KR > 0 ? KR : 1];
    if constexpr (KR > 0) {
#pragma unroll
      for (int i = 0; i < KR; ++i) k[i] = lane + 64 * i < total ? rc[lane + 64 * i] : 0;
    }
    auto each = [&](auto visit) {  // every key of the row, all lanes together; 0: none
      if constexpr (KR > 0) {
#pragma unroll
        for (int i = 0; i < KR; ++i) visit(k[i]);
      } else {
        for (int i = 0; i < total; i += 64) visit(i + lane < total ? rc[i + lane] : 0);
      }
    };
    const float score = scores[row];
    const RowStat q = lane < chunks ? st[lane] : RowStat{0, 0.0f};
    uint32_t top = q.top;
    for (int c = lane + 64; c < chunks; c += 64) top = umax32(top, st[c].top);
    top = wave_max_u32_dpp(top);
    // the kind of the row: v of all its candidates, where that is one value
    const bool bad = top >= kOrdInf || !(score < __builtin_inff());
    const bool dead = top == kOrdNegInf || score == -__builtin_inff();
    if (bad || dead) {
      for (int i = lane; i < len; i += 64) vals[w * n + i] = bad ? ~0ull : ord_of_f64(-__builtin_inf()), toks[w * n + i] = i;
      continue;
    }
    const float mx = of_ord(top);
    // (as exact as the sums are: the chunks that matter have small exponents)
    auto part = [&](RowStat r) {
      return r.top > kOrdNegInf ? (double)(r.sum * __builtin_amdgcn_exp2f((of_ord(r.top) - mx) * 1.44269504f)) : 0.0;
    };
    double s = part(q);
    for (int c = lane + 64; c < chunks; c += 64) s += part(st[c]);
    const double lse = (double)mx + log(wave_sum_f64(s));
    uint64_t best = 0;
    each([&](uint64_t key) { best = key > best ? key : best; });
    uint64_t least = static_cast<uint64_t>(nth_upper(hi32(best), n)) << 32;
    int have = 0;
    each([&](uint64_t key) { have += __popcll(__ballot(key && key >= least)); });
    if (have > min(n * per, kFewKeys)) least = nth_key(best, n);  // (reached by n lanes' keys, n * per)
    have = 0;
    each([&](uint64_t key) {
      const bool in = key && key >= least;
      const uint64_t mask = __ballot(in);
      if (in) list[have + __popcll(mask & ((1ull << lane) - 1))] = key;
      have += __popcll(mask);
    });
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int i = lane; i < have; i += 64) {
      const uint64_t key = list[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < have; ++j) rank += list[j] > key;
      if (rank < len) {
        vals[w * n + rank] = ord_of_f64((double)score + ((double)of_ord(hi32(key)) - lse));
        toks[w * n + rank] = ~static_cast<uint32_t>(key);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // the place of a candidate: those of larger v before it, and of equal v those of lower beams and before it in its own,
  // the order that the rows lie in
  const int all = W * len;
  auto put = [&](int i, int rank) {
    const int w = i / len, p = i % len;
    if (rank < n) {
      const int64_t at = b * n + rank;
      const uint64_t v = vals[w * n + p];
      out_scores[at] = v == ~0ull ? __builtin_nanf("")
                                  : static_cast<float>(__builtin_bit_cast(double, v >> 63 ? v & ~(1ull << 63) : ~v));
      out_beams[at] = w;
      out_tokens[at] = toks[w * n + p];
    }
  };
  const int ways = min(max(threads / all, 1), W);
  auto before = [&](int i, int k) {  // how many come before candidate i in the k-th of `ways` parts of the rows
    const int w = i / len, p = i % len;
    const uint64_t v = vals[w * n + p];
    int rank = 0;
    for (int q = k; q < W && rank < n; q += ways) {
      int lo = q == w ? p : 0, hi = q == w ? p : len;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const uint64_t u = vals[q * n + mid];
        if (u > v || (u == v && q < w)) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    return rank;
  };
  if (ways > 1) {  // (all < threads <= kPickThreads)
    for (int i = tid; i < all; i += threads) ranks[i] = 0;
    __syncthreads();
    for (int k = tid; k < all * ways; k += threads) atomicAdd(&ranks[k % all], before(k % all, k / all));
    __syncthreads();
    for (int i = tid; i < all; i += threads) put(i, ranks[i]);
  } else {
    __syncthreads();
    for (int i = tid; i < all; i += threads) put(i, before(i, 0));
  }
}

struct SelectPlan {
  int nv, chunks;
  int64_t stat_bytes, bytes;
};

// Chunks of 32 values a thread; of 8 or 16 where the rows would not fill the chip and the keys that are left still fit
// k_beam_pick's registers.
constexpr int kKeysShort = 10 * 64, kKeysLong = 20 * 64;
SelectPlan select_plan(int64_t rows, int64_t V, int n, int esize) {
  SelectPlan p;
  const int vec = 16 / esize;
  auto chunks = [&](int values) { return (V + values * kBeamThreads - 1) / (values * kBeamThreads); };
  const bool many = rows * chunks(32) >= 512;
  const int values = !many && chunks(8) * n <= kKeysShort ? 8 : !many && chunks(16) * n <= kKeysLong ? 16 : 32;
  p.nv = values / vec;
  p.chunks = static_cast<int>(chunks(values));
  p.stat_bytes = (rows * p.chunks * (int64_t)sizeof(RowStat) + 15) / 16 * 16;
  p.bytes = p.stat_bytes + rows * p.chunks * n * (int64_t)sizeof(uint64_t);
  return p;
}

// The waves of k_beam_pick that merge rows side by side, by the LDS that their lists take beside the rows', and that LDS.
constexpr size_t kPickLds = 128 * 1024;
int pick_lists(int W, int n, int chunks, size_t* lds) {
  const size_t rows = sizeof(uint64_t) * (W * n + (W * n + 1) / 2), list = sizeof(uint64_t) * n * ((chunks * n + 63) / 64);
  const int lists = static_cast<int>(std::min<size_t>((kPickLds - rows) / list, std::min(W, kPickWaves)));
  *lds = rows + lists * list;
  return lists;
}
// (48 KiB of rows and a list of 66 KiB at the most: the largest W, n and vocabulary)
constexpr int64_t kVocabMax = 1 << 20;

bool select_fits(int64_t B, int64_t W, int64_t V, int64_t n) {
  return B >= 1 && W >= 1 && W <= kBeamMax && n >= 1 && n <= kBeamMax && V >= 1 && V <= kVocabMax && n <= W * V && B * W <= 65535;
}

// ---------------------------------------------------------------------------------------------
// Reordering. States are [outer][B W][mid][S][d] in memory; row b W + w takes the positions s < length[b] of row b W +
// beams[b, w]. A thread owns the same unit of bytes in all W rows of an entry: it reads the sources of the rows that
// change, then writes those, so that the work is done in place with no second copy, whatever the order.
// ---------------------------------------------------------------------------------------------
constexpr int kReorderStates = 64, kReorderThreads = 256;

struct ReorderArgs {
  void* state[kReorderStates];
  const void* beams;
  const void* lengths;
  int64_t outer, mid, span, dbytes, S;  // span: S * dbytes
  int B, W, blocks, beams64, lengths64;
};

template <typename U, int WM>
__global__ __launch_bounds__(kReorderThreads) void k_beam_reorder(ReorderArgs a) {
  const int64_t block = blockIdx.x % a.blocks;
  int64_t at = blockIdx.x / a.blocks;
  const int64_t h = at % a.mid;
  at /= a.mid;
  const int b = static_cast<int>(at % a.B);
  const int64_t o = at / a.B;
  int64_t len = a.span;
  if (a.lengths) {
    const int64_t l = a.lengths64 ? static_cast<const int64_t*>(a.lengths)[b] : static_cast<const int32_t*>(a.lengths)[b];
    len = min(max(l, (int64_t)0), a.S) * a.dbytes;
  }
  const int64_t byte = (block * kReorderThreads + threadIdx.x) * (int64_t)sizeof(U);
  if (byte >= len) return;
  const int64_t row = a.mid * a.span;  // bytes between two rows
  uint8_t* base = static_cast<uint8_t*>(a.state[blockIdx.y]) + ((o * a.B + b) * a.W * a.mid + h) * a.span + byte;
  U v[WM];
  uint64_t moved = 0;
#pragma unroll
  for (int w = 0; w < WM; ++w) {
    if (w < a.W) {
      const int64_t p = a.beams64 ? static_cast<const int64_t*>(a.beams)[b * a.W + w] : static_cast<const int32_t*>(a.beams)[b * a.W + w];
      if (p != w && p >= 0 && p < a.W) {
        v[w] = *reinterpret_cast<const U*>(base + p * row);
        moved |= 1ull << w;
      }
    }
  }
#pragma unroll
  for (int w = 0; w < WM; ++w)
    if (moved >> w & 1) *reinterpret_cast<U*>(base + w * row) = v[w];
}

template <typename U>
void launch_reorder(const ReorderArgs& a, int states, hipStream_t s) {
  ReorderArgs r = a;
  const int64_t unit = (int64_t)kReorderThreads * sizeof(U);
  r.blocks = static_cast<int>((a.span + unit - 1) / unit);
  const dim3 grid(static_cast<unsigned>(r.blocks * a.outer * a.B * a.mid), states);
  if (a.W <= 4) hipLaunchKernelGGL((k_beam_reorder<U, 4>), grid, dim3(kReorderThreads), 0, s, r);
  else if (a.W <= 8) hipLaunchKernelGGL((k_beam_reorder<U, 8>), grid, dim3(kReorderThreads), 0, s, r);
  else if (a.W <= 16) hipLaunchKernelGGL((k_beam_reorder<U, 16>), grid, dim3(kReorderThreads), 0, s, r);
  else if constexpr (sizeof(U) <= 4) hipLaunchKernelGGL((k_beam_reorder<U, kBeamMax>), grid, dim3(kReorderThreads), 0, s, r);
}

}  // namespace

extern "C" int64_t krq_beam_select_ws_bytes(int64_t B, int64_t W, int64_t V, int64_t n, int fp32) {
  if (!select_fits(B, W, V, n)) return -1;
  return select_plan(B * W, V, static_cast<int>(n), fp32 ? 4 : 2).bytes;
}

extern "C" int krq_beam_select(const void* logits, int fp32, int64_t ld, const float* scores, int64_t B, int64_t W, int64_t V, int64_t n,
                               void* ws, int64_t ws_bytes, float* out_scores, int64_t* out_beams, int64_t* out_tokens, void* stream) {
  KRQ_REQUIRE(logits && scores && ws && out_scores && out_beams && out_tokens, "beam_select: null pointer");
  KRQ_REQUIRE(select_fits(B, W, V, n), "beam_select: %lld x %lld beams, vocabulary %lld, n=%lld (beams and n up to %d, n <= beams * "
              "vocabulary, rows up to 65535, vocabulary up to 2^20)", (long long)B, (long long)W, (long long)V, (long long)n, kBeamMax);
  KRQ_REQUIRE(ld >= V, "beam_select: rows of %lld logits %lld apart", (long long)V, (long long)ld);
  const int esize = fp32 ? 4 : 2;
  KRQ_REQUIRE(reinterpret_cast<uintptr_t>(logits) % esize == 0 && aligned16(ws), "beam_select: logits or ws not on their alignment");
  const SelectPlan p = select_plan(B * W, V, static_cast<int>(n), esize);
  KRQ_REQUIRE(ws_bytes >= p.bytes, "beam_select: ws of %lld bytes, needs %lld", (long long)ws_bytes, (long long)p.bytes);
  size_t lds;
  const int lists = pick_lists(static_cast<int>(W), static_cast<int>(n), p.chunks, &lds);
  RowStat* stat = (RowStat*)ws;
  uint64_t* cand = (uint64_t*)((uint8_t*)ws + p.stat_bytes);
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid(p.chunks, static_cast<unsigned>(B * W));
  const size_t list = sizeof(uint64_t) * std::max<int64_t>(4 * n * (p.nv * 16 / esize), kFewKeys);
#define KRQ_ROWS(T, NV)                                                                                                       \
  hipLaunchKernelGGL((k_beam_rows<T, NV>), grid, dim3(kBeamThreads), list, s, (const T*)logits, ld, V, (int)n, p.chunks, stat, cand)
  if (fp32) {
    if (p.nv == 8) KRQ_ROWS(float, 8);
    else if (p.nv == 4) KRQ_ROWS(float, 4);
    else KRQ_ROWS(float, 2);
  } else {
    if (p.nv == 4) KRQ_ROWS(uint16_t, 4);
    else if (p.nv == 2) KRQ_ROWS(uint16_t, 2);
    else KRQ_ROWS(uint16_t, 1);
  }
#undef KRQ_ROWS
  if (const int rc = krq_check_launch("beam_select")) return rc;
  const int waves = static_cast<int>(std::max<int64_t>(4, std::min<int64_t>(W, kPickWaves)));
#define KRQ_PICK(KR)                                                                                                          \
  hipLaunchKernelGGL(k_beam_pick<KR>, dim3(static_cast<unsigned>(B)), dim3(64 * waves), lds, s, stat, cand, scores, V, (int)W, \
                     (int)n, p.chunks, lists, out_scores, out_beams, out_tokens)
  const int64_t keys = p.chunks * n;
  if (keys <= 5 * 64) KRQ_PICK(5);
  else if (keys <= kKeysShort) KRQ_PICK(10);
  else if (keys <= kKeysLong) KRQ_PICK(20);
  else KRQ_PICK(0);
#undef KRQ_PICK
  return krq_check_launch("beam_select");
}

extern "C" int krq_beam_reorder(void* const* states, int count, int64_t outer, int64_t B, int64_t W, int64_t mid, int64_t S,
                                int64_t dbytes, const void* beams, int beams_64, const void* lengths, int lengths_64, void* stream) {
  KRQ_REQUIRE(states && beams && count >= 1 && count <= kReorderStates, "beam_reorder: %d states (1 to %d)", count, kReorderStates);
  KRQ_REQUIRE(outer >= 1 && B >= 1 && W >= 1 && W <= kBeamMax && mid >= 1 && S >= 1 && dbytes >= 1 && B <= (1 << 20) && S <= ((int64_t)1 << 40) / dbytes,
              "beam_reorder: bad shape [%lld][%lld x %lld][%lld][%lld][%lld bytes] (at most %d beams)", (long long)outer, (long long)B,
              (long long)W, (long long)mid, (long long)S, (long long)dbytes, kBeamMax);
  ReorderArgs a{};
  uintptr_t bits = static_cast<uintptr_t>(dbytes);
  for (int i = 0; i < count; ++i) {
    KRQ_REQUIRE(states[i], "beam_reorder: null state");
    a.state[i] = states[i];
    bits |= reinterpret_cast<uintptr_t>(states[i]);
  }
  a.beams = beams;
  a.lengths = lengths;
  a.outer = outer;
  a.mid = mid;
  a.span = S * dbytes;
  a.dbytes = dbytes;
  a.S = S;
  a.B = static_cast<int>(B);
  a.W = static_cast<int>(W);
  a.beams64 = beams_64 != 0;
  a.lengths64 = lengths_64 != 0;
  const int unit = bits % 16 == 0 && W <= 16 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  const double blocks = (double)((a.span + (int64_t)kReorderThreads * unit - 1) / ((int64_t)kReorderThreads * unit)) * outer * B * mid;
  KRQ_REQUIRE(blocks * kReorderThreads < 4294967296.0, "beam_reorder: a state is too large for one launch");
  hipStream_t s = (hipStream_t)stream;
  if (unit == 16) launch_reorder<v4u>(a, count, s);
  else if (unit == 4) launch_reorder<uint32_t>(a, count, s);
  else if (unit == 2) launch_reorder<uint16_t>(a, count, s);
  else launch_reorder<uint8_t>(a, count, s);
  return krq_check_launch("beam_reorder");
}

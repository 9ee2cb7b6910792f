// Residual addition and RMSNorm with the rows rounded for the next product, one launch between two projections.
//
//   d    = bf16(p_0 + p_1 + .. + p_{S-1})   the addend: split-K partials summed in order in fp32, or bf16 rows
//   r    = bf16(x + d)                      the new residual row (written where there is an addend)
//   rstd = fp32(1 / sqrt(sum(r^2) / K + eps))
//   h    = bf16(bf16(r * rstd) * ln)
//   out  = h, and/or e4m3 rows with a per-token or a given scale (the arithmetic of krq_quant_rows and krq_cast_fp8,
//          their bytes), or MX blocks of 32 (krq_quant_mx_rows' bytes)
// The sum of squares is held in fp64: a square of a bf16 is exact in fp32, and its 70 additions of a lane and across lanes at the
// most leave the sum off by less than 2^-46 and rstd, before its rounding to fp32, by less than 2^-47: it is the rounding of
// the exact value, whatever the order of the sum, but for at most one row in some 2^22 that lies so near a border; the
// roundings to bf16 and e4m3 behind it, which have borders of their own, come out the same for every thread layout
// below. It costs two fp64 operations per value, hidden under the loads.
//
// A row is held in registers between the passes over it: W waves, C chunks of 8 values per lane, so that every value
// is read once and written once. W = 1 needs no barrier.
#include "mx_common.h"

using namespace krq;

namespace {

constexpr int kNormMaxK = 16384, kPartials = 4;  // partials of a split in flight

enum Src { kSrcNone, kSrcBf16, kSrcPartials };
enum Out { kOutRows, kOutToken, kOutGiven, kOutMxE4, kOutMxE2 };

struct NormArgs {
  const uint16_t* x;
  const void* delta;
  const uint16_t* ln;
  uint16_t* res;
  uint16_t* h;
  uint8_t* out;
  float* scale;        // per token
  const float* inv;    // given
  uint8_t* mx_scale;
  int64_t M, rows, ldx, ldd, slice;
  float eps;
  int K, split, tiled, spread;
};

KRQ_DEV uint4 add8(uint4 x, uint4 d) {
  const uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {d.x, d.y, d.z, d.w};
  uint32_t o[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    o[q] = pack_bf16x2(as_f32(a[q] << 16) + as_f32(b[q] << 16), as_f32(a[q] & 0xffff0000u) + as_f32(b[q] & 0xffff0000u));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

KRQ_DEV double sumsq8_f64(uint4 v, double s) {
  const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float lo = as_f32(a[q] << 16), hi = as_f32(a[q] & 0xffff0000u);
    s = fma((double)lo, (double)lo, s);
    s = fma((double)hi, (double)hi, s);
  }
  return s;
}

KRQ_DEV bool has_nonfinite(uint4 v) { return bits_max_to_u32(absmax8_bits(v, u16x2{0, 0})) >= 0x7f800000u; }

KRQ_DEV uint2 quant8_given(uint4 v, float s) {
  if (has_nonfinite(v) || !finite_f32(s)) return quant8(v, s);
  const uint32_t a[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    auto q = [&](float f) { return __builtin_amdgcn_fmed3f(f * s, -kFp8Max, kFp8Max); };
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(q(as_f32(a[2 * i] << 16)), q(as_f32(a[2 * i] & 0xffff0000u)), 0, false);
    o[i] = static_cast<uint32_t>(
        __builtin_amdgcn_cvt_pk_fp8_f32(q(as_f32(a[2 * i + 1] << 16)), q(as_f32(a[2 * i + 1] & 0xffff0000u)), p, true));
  }
  return make_uint2(o[0], o[1]);
}

// W waves of a workgroup of NW take a row, C chunks of 8 values per lane (chunk lane + 64 (w + W c)).
template <int NW, int W, int C, int SRC, int OUT>
__global__ __launch_bounds__(64 * NW) void k_add_rmsnorm(NormArgs a) {
  constexpr bool kMx = OUT == kOutMxE4 || OUT == kOutMxE2;
  __shared__ double ssum[W > 1 ? NW : 1];
  __shared__ uint32_t smax[W > 1 && OUT == kOutToken ? NW : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, K = a.K;
  int64_t b = blockIdx.x;
  constexpr int kTile = 16 / (NW / W);  // blocks to sixteen rows
  if (a.spread) {  // sixteen rows share a tile's lines: blocks of one XCD (blockIdx % 8) take them
    const int64_t q = b / (8 * kTile);
    const int in = static_cast<int>(b % (8 * kTile));
    b = q * (8 * kTile) + kTile * (in & 7) + (in >> 3);
  }
  const int64_t m = b * (NW / W) + wave / W;
  if (m >= a.rows) return;  // (whole rows' waves: with W > 1 a workgroup has one row)
  const int first = lane + 64 * (wave % W);  // chunk
  const int n8 = K >> 3;
  const bool pad = m >= a.M;
  uint4 v[C];
  const int KT = kMx ? static_cast<int>(mx_tiles(K)) : 0, groups = kMx ? static_cast<int>(mx_groups(K)) : 0;
  const int64_t mb = m >> 4;
  const int r16 = static_cast<int>(m & 15);

  auto put8 = [&](int i, uint2 o) {  // e4m3 bytes of chunk i
    const int64_t at = a.tiled ? tiled_offset(m, 8 * i, K) : m * K + 8 * i;
    *reinterpret_cast<uint2*>(a.out + at) = o;
  };
  auto put_mx = [&](int i, uint4 h8, bool real) {  // chunk i as part of a block: a quad of lanes holds one
    const uint32_t c = mx_code<OUT == kOutMxE2 ? KRQ_MX_E2M1 : KRQ_MX_E4M3>(quad_absmax(h8));
    const int k = 8 * i, kc = k & 127, tile = k >> 7, s = k >> 9;
    if (tile < KT) {
      if constexpr (OUT == kOutMxE2) {
        *reinterpret_cast<uint32_t*>(a.out + ((mb * KT + tile) * 64 + 16 * (kc >> 5) + r16) * 16 + 4 * (i & 3)) =
            real ? mx_quant8_e2m1(h8, c) : 0u;
      } else {
        *reinterpret_cast<uint2*>(a.out + (mb * KT + tile) * 2048 + 1024 * (kc >> 6) + 16 * (16 * ((kc & 63) >> 4) + r16) +
                                  (kc & 15)) = real ? mx_quant8_e4m3(h8, c) : make_uint2(0u, 0u);
      }
    }
    if ((i & 3) == 0 && s < groups)
      a.mx_scale[((mb * groups + s) * 64 + 16 * (kc >> 5) + r16) * 4 + (tile & 3)] = real ? static_cast<uint8_t>(c) : 0;
  };

  if (pad) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = first + 64 * W * c;
      if constexpr (kMx) put_mx(i, zero4(), false);
      else if (OUT != kOutRows && i < n8) put8(i, make_uint2(0u, 0u));
    }
    return;
  }

  // the row, read once: every load at once, at a clamped address (chunks past K repeat the last and count as zeros)
  auto chunk = [&](int c) { return min(first + 64 * W * c, n8 - 1); };
  const uint8_t* xr = reinterpret_cast<const uint8_t*>(a.x + m * a.ldx);
  uint4 l[C];
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = ld16(xr + 16 * chunk(c));
  if constexpr (SRC == kSrcBf16) {
    const uint8_t* dr = reinterpret_cast<const uint8_t*>(static_cast<const uint16_t*>(a.delta) + m * a.ldd);
    uint4 d[C];
#pragma unroll
    for (int c = 0; c < C; ++c) d[c] = ld16(dr + 16 * chunk(c));
#pragma unroll
    for (int c = 0; c < C; ++c) l[c] = ld16(reinterpret_cast<const uint8_t*>(a.ln) + 16 * chunk(c));
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = add8(v[c], d[c]);
  } else if constexpr (SRC == kSrcPartials) {
    const float* dr = static_cast<const float*>(a.delta) + m * a.ldd;
    v4f sum[C][2];
#pragma unroll
    for (int c = 0; c < C; ++c) l[c] = ld16(reinterpret_cast<const uint8_t*>(a.ln) + 16 * chunk(c));
    for (int s = 0; s < a.split; s += kPartials) {  // (past the last: loaded again, not added)
      v4f t[kPartials][C][2];
#pragma unroll
      for (int u = 0; u < kPartials; ++u)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            t[u][c][e] = *reinterpret_cast<const v4f*>(dr + min(s + u, a.split - 1) * a.slice + 8 * chunk(c) + 4 * e);
#pragma unroll
      for (int u = 0; u < kPartials; ++u)
        if (s + u < a.split)
#pragma unroll
          for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) sum[c][e] = s + u == 0 ? t[u][c][e] : sum[c][e] + t[u][c][e];
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
      v[c] = add8(v[c], make_uint4(pack_bf16x2(sum[c][0][0], sum[c][0][1]), pack_bf16x2(sum[c][0][2], sum[c][0][3]),
                                   pack_bf16x2(sum[c][1][0], sum[c][1][1]), pack_bf16x2(sum[c][1][2], sum[c][1][3])));
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) l[c] = ld16(reinterpret_cast<const uint8_t*>(a.ln) + 16 * chunk(c));
  }
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = sel4(first + 64 * W * c < n8, v[c]);
  double ss = 0.0;
  if (SRC != kSrcNone) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = first + 64 * W * c;
      if (i < n8) *reinterpret_cast<uint4*>(a.res + m * K + 8 * i) = v[c];
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) ss = sumsq8_f64(v[c], ss);  // (chunks past K hold zeros)
  ss = wave_sum_f64(ss);
  if constexpr (W > 1) {
    if (lane == 0) ssum[wave] = ss;
    __syncthreads();
    ss = ssum[0];
#pragma unroll
    for (int w = 1; w < W; ++w) ss += ssum[w];
  }
  const float rstd = static_cast<float>(1.0 / sqrt(ss / K + (double)a.eps));

  uint32_t am = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int i = first + 64 * W * c;
    v[c] = sel4(i < n8, norm8(v[c], l[c], rstd));
    if (a.h && i < n8) *reinterpret_cast<uint4*>(a.h + m * K + 8 * i) = v[c];
    if constexpr (OUT == kOutToken) am = absmax8(v[c], am);
  }
  if constexpr (OUT == kOutToken) {
    am = wave_max_u32_dpp(am);
    if constexpr (W > 1) {
      if (lane == 0) smax[wave] = am;
      __syncthreads();
      am = smax[0];
#pragma unroll
      for (int w = 1; w < W; ++w) am = umax32(am, smax[w]);
    }
    const float amax = clamp_min_nan(as_f32(am), 1e-6f), inv = inv_from_amax(amax);
    if (first == 0) a.scale[m] = scale_from_amax(amax);
    const bool fine = finite_f32(amax);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = first + 64 * W * c;
      if (i < n8) put8(i, fine ? quant8_own_amax(v[c], inv) : quant8(v[c], inv));
    }
  } else if constexpr (OUT == kOutGiven) {
    const float inv = a.inv[0];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = first + 64 * W * c;
      if (i < n8) put8(i, quant8_given(v[c], inv));
    }
  } else if constexpr (kMx) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int i = first + 64 * W * c;
      put_mx(i, v[c], true);
    }
  }
}

template <int NW, int W, int C, int SRC, int OUT>
int launch(const NormArgs& a, hipStream_t s) {
  constexpr int per = NW / W;
  NormArgs b = a;
  int64_t blocks = (a.rows + per - 1) / per;
  b.spread = (a.tiled || OUT == kOutMxE4 || OUT == kOutMxE2) && a.rows >= 128;
  if (b.spread) blocks = (blocks + 128 / per - 1) / (128 / per) * (128 / per);
  KRQ_REQUIRE(blocks * (64 * NW) < (int64_t)1 << 32, "add_rmsnorm: %lld rows of K=%d are too many for a launch", (long long)a.M, a.K);
  hipLaunchKernelGGL((k_add_rmsnorm<NW, W, C, SRC, OUT>), dim3(static_cast<unsigned>(blocks)), dim3(64 * NW), 0, s, b);
  return krq_check_launch("add_rmsnorm");
}

// Rows by one or two waves each where there are enough rows to fill the chip that way, else by eight or sixteen waves, whose loads
// are all in flight at once. Calls of a graph, per-token scales, a bf16 addend, us, few waves / many: 2,560 x 512 rows 5.0 / 4.9, 601 rows
// 5.1 / 5.7, 1,001 6.4 / 7.4, 2,048 9.2 / 11.3, 4,096 14.0 / 18.1; 4,096 x 1,001 8.7 / 8.5; 5,120 x 1,001 9.6 / 10.6, 4,096 rows 27.4 / 31.2; 8,192 x 1,001
// 13.1 / 12.6 and 16,384 x 1,001 (four waves) 22.9 / 22.7. One wave has five chunks a lane for every K up to 2,560, of which a smaller K leaves
// some idle (loaded again at the row's end, squared as zeros): 256 x 601 rows 3.9 / 4.9, 4,096 rows 7.8 / 14.9; 1,024 x 601 4.0 / 4.9, 4,096
// rows 9.8 / 16.4.
constexpr int64_t kManyRows = 600, kMoreRows = 1536;

template <int SRC, int OUT>
int pick(const NormArgs& a, hipStream_t s) {
  const int K = OUT == kOutMxE4 || OUT == kOutMxE2 ? static_cast<int>(mx_groups(a.K)) * kMxGroup : a.K;  // chunks written
  if constexpr (SRC != kSrcPartials) {  // (partials of many rows: too many registers)
    if (a.rows >= kManyRows && K <= 2560) return launch<4, 1, 5, SRC, OUT>(a, s);
    if (a.rows >= kMoreRows && K <= 4096) return launch<4, 1, 8, SRC, OUT>(a, s);
    if (a.rows >= kManyRows && K > 4096 && K <= 5120) return launch<2, 2, 5, SRC, OUT>(a, s);
  }
  if (K <= 4096) return launch<8, 8, 1, SRC, OUT>(a, s);
  if (K <= 8192) return launch<8, 8, 2, SRC, OUT>(a, s);
  return launch<16, 16, 2, SRC, OUT>(a, s);
}

template <int OUT>
int pick_src(const NormArgs& a, hipStream_t s) {
  if (!a.delta) return pick<kSrcNone, OUT>(a, s);
  return a.split == 0 ? pick<kSrcBf16, OUT>(a, s) : pick<kSrcPartials, OUT>(a, s);
}

}  // namespace

extern "C" int krq_add_rmsnorm(const void* x, int64_t ldx, const void* delta, int split, int64_t ldd, int64_t slice,
                               const void* ln, float eps, int64_t M, int64_t K, int out_kind, const float* inv, void* res,
                               void* h, void* out, void* out_scale, void* stream) {
  KRQ_REQUIRE(x && ln, "add_rmsnorm: null pointer");
  KRQ_REQUIRE(M >= 1 && M <= 0x7fffffff - 127 && K >= 16 && K % 16 == 0 && K <= kNormMaxK,
              "add_rmsnorm: bad shape M=%lld K=%lld (K a multiple of 16, at most %d)", (long long)M, (long long)K, kNormMaxK);
  KRQ_REQUIRE(out_kind >= KRQ_NORM_ROWS && out_kind <= KRQ_NORM_MX_E2M1, "add_rmsnorm: bad output %d", out_kind);
  KRQ_REQUIRE(!delta || res, "add_rmsnorm: an addend needs res");
  KRQ_REQUIRE(split >= 0 && split <= 64, "add_rmsnorm: split=%d (0 for bf16 rows, at most 64)", split);
  KRQ_REQUIRE(ldx >= K && ldx % 8 == 0, "add_rmsnorm: rows of x must start on 16 bytes (ldx=%lld)", (long long)ldx);
  KRQ_REQUIRE(!delta || (ldd >= K && ldd % (split ? 4 : 8) == 0 && (split < 2 || slice % 4 == 0)),
              "add_rmsnorm: rows of the addend must start on 16 bytes (ldd=%lld, slice=%lld)", (long long)ldd, (long long)slice);
  KRQ_REQUIRE(aligned16(x) && aligned16(delta) && aligned16(ln) && aligned16(res) && aligned16(h) && aligned16(out),
              "add_rmsnorm: every operand must start on 16 bytes");
  const bool tiled = out_kind == KRQ_NORM_FP8_TOKEN_TILED || out_kind == KRQ_NORM_FP8_GIVEN_TILED;
  const bool given = out_kind == KRQ_NORM_FP8_GIVEN || out_kind == KRQ_NORM_FP8_GIVEN_TILED;
  const bool mx = out_kind == KRQ_NORM_MX_E4M3 || out_kind == KRQ_NORM_MX_E2M1;
  KRQ_REQUIRE(out_kind == KRQ_NORM_ROWS ? h != nullptr : out != nullptr, "add_rmsnorm: null output");
  KRQ_REQUIRE(out_kind == KRQ_NORM_ROWS || (given ? inv != nullptr : out_scale != nullptr), "add_rmsnorm: null scale");
  KRQ_REQUIRE(!tiled || K % 64 == 0, "add_rmsnorm: tiled rows need K=%lld a multiple of 64", (long long)K);
  KRQ_REQUIRE(!mx || K % kMxBlock == 0, "add_rmsnorm: MX blocks need K=%lld a multiple of 32", (long long)K);
  NormArgs a{};
  a.x = (const uint16_t*)x;
  a.delta = delta;
  a.ln = (const uint16_t*)ln;
  a.res = (uint16_t*)res;
  a.h = (uint16_t*)h;
  a.out = (uint8_t*)out;
  a.scale = (float*)out_scale;
  a.inv = inv;
  a.mx_scale = (uint8_t*)out_scale;
  a.M = M;
  a.rows = tiled || mx ? (M + 15) / 16 * 16 : M;
  a.ldx = ldx;
  a.ldd = ldd;
  a.slice = slice;
  a.eps = eps;
  a.K = (int)K;
  a.split = split;
  a.tiled = tiled;
  hipStream_t s = (hipStream_t)stream;
  if (out_kind == KRQ_NORM_ROWS) return pick_src<kOutRows>(a, s);
  if (given) return pick_src<kOutGiven>(a, s);
  if (out_kind == KRQ_NORM_MX_E4M3) return pick_src<kOutMxE4>(a, s);
  if (out_kind == KRQ_NORM_MX_E2M1) return pick_src<kOutMxE2>(a, s);
  return pick_src<kOutToken>(a, s);
}

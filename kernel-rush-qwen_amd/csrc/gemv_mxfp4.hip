// MXFP4 skinny GEMM / GEMV (M <= 32): y = x . w^T on microscaled blocks, w e2m1 in the operand tiles of
// mx_common.h, x in e4m3 or e2m1 blocks, fp32 accumulation in v_mfma_scale_f32_16x16x128_f8f6f4.
//
// The unit of work is a (row block, group): 16 weight rows x 512 k, four 1 KiB tiles and one dword of
// scales per lane, 4.25 KiB that a wave loads with five contiguous loads. A workgroup owns P row blocks (SwiGLU: a gate
// block and its up block) over a K split; its waves take the groups wave, wave + waves, ... and their sums meet in
// LDS, in wave order, so the result does not depend on timing.
//
// Activations. XR > 0: bf16 rows, at most XR, quantised here: the 512 k of a group are one 16-byte load per
// row, the four lanes of a quad hold a block, and the wave's own region of LDS turns them into operands (lanes of
// rows past the last read the last one's; their products land in accumulator rows nobody writes). No launch and no
// barrier before the product. XR = 0: rows quantised before by krq_quant_mx_rows, MT row tiles of them.
#include "mx_common.h"

using namespace krq;

namespace {

constexpr int kMaxWaves = 8;
constexpr int kMxSplitMax = 64;

template <int ELEM, int XR>
struct XLds {  // a wave's region for one group of its bf16 rows: elements linear in k, then 16 scale bytes [g][t]
  static constexpr int kBytes = ELEM == KRQ_MX_E2M1 ? 256 : 512;
  static constexpr int kRow = kBytes + 16;  // rows start in different banks
  static constexpr int kWave = XR * kRow;
};

// the A operand of tile t (of the group) for this lane's row, at p = row base in LDS
template <int ELEM>
KRQ_DEV v8i lds_operand(const uint8_t* p, int t, int g) {
  if constexpr (ELEM == KRQ_MX_E2M1) {
    return pack_v8i(*reinterpret_cast<const uint4*>(p + 64 * t + 16 * g), zero4());
  } else {
    const uint8_t* q = p + 128 * t + 16 * g;
    return pack_v8i(*reinterpret_cast<const uint4*>(q), *reinterpret_cast<const uint4*>(q + 64));
  }
}

// acc += A (16 rows) . B (16 weight rows) over 128 k, scale bytes T of sa and sb. A: e2m1 or e4m3, B: e2m1.
template <int ELEM, int T>
KRQ_DEV v4f mx_mfma(v8i a, v8i b, v4f acc, uint32_t sa, uint32_t sb) {
  constexpr int fa = ELEM == KRQ_MX_E2M1 ? 4 : 0;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, fa, 4, T, static_cast<int>(sa), T, static_cast<int>(sb));
}
template <int ELEM>
KRQ_DEV v4f mx_mfma(int t, v8i a, v8i b, v4f acc, uint32_t sa, uint32_t sb) {  // (t a constant after unrolling)
  return t == 0 ? mx_mfma<ELEM, 0>(a, b, acc, sa, sb) : t == 1 ? mx_mfma<ELEM, 1>(a, b, acc, sa, sb)
         : t == 2 ? mx_mfma<ELEM, 2>(a, b, acc, sa, sb) : mx_mfma<ELEM, 3>(a, b, acc, sa, sb);
}

struct MxArgs {
  const uint8_t* x;    // bf16 rows, or tiles
  const uint8_t* xs;   // the tiles' scales
  const uint8_t* w;    // tiles
  const uint8_t* ws;   // their scales
  void* out;           // bf16 [M, NO], fp32 [splits][M][NO], or the logits (may be null)
  Best* cand;          // argmax candidates [M][row blocks]
  int64_t ldx;         // bf16 rows' stride
  int64_t NO;          // output columns
  int M, K, KT, groups, nrb;  // nrb: row blocks of the output
};

// MODE: KRQ_OUT_BF16, KRQ_OUT_PARTIAL (blockIdx.y: the split), KRQ_OUT_SWIGLU, kOutArgmax
template <int ELEM, int XR, int MT, int MODE, int P, int U>
__global__ __launch_bounds__(kMaxWaves * 64) void k_gemv_mx(const MxArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];  // sums [waves][P][MT][256], or before them the bf16 rows' regions
  static_assert(XR == 0 || MT == 1, "rows quantised here: one row tile");
  static_assert(MODE != KRQ_OUT_SWIGLU || P == 2, "SwiGLU: a gate and an up row block");
  using X = XLds<ELEM, XR>;
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6)), nw = blockDim.x >> 6;
  const int splits = gridDim.y, sp = blockIdx.y;
  const int g0 = a.groups * sp / splits, g1 = a.groups * (sp + 1) / splits;  // this split's groups
  const int jc = g0 + wave < g1 ? (g1 - g0 - wave + nw - 1) / nw : 0;         // this wave's
  int rbs[P];
#pragma unroll
  for (int p = 0; p < P; ++p)
    rbs[p] = MODE == KRQ_OUT_SWIGLU ? static_cast<int>(blockIdx.x) + p * a.nrb
                                    : min(static_cast<int>(blockIdx.x) * P + p, a.nrb - 1);

  constexpr int AB = ELEM == KRQ_MX_E2M1 ? 1 : 2;  // 16-byte loads per activation tile
  uint4 xv[U][XR > 0 ? XR : 1];
  uint4 wv[U][P][4], av[U][XR > 0 ? 1 : MT][4 * AB];
  uint32_t wsc[U][P], asc[U][MT];
  auto group_of = [&](int j) { return jc > 0 ? g0 + wave + min(j, jc - 1) * nw : g0; };
  // (loads past the wave's last group repeat it: every load is unconditional, the products are not)
  auto load_x = [&](int u, int j) {
    const int s = group_of(j);
    if constexpr (XR > 0) {
      const int k = min(s * kMxGroup + 8 * lane, a.K - 8);
#pragma unroll
      for (int m = 0; m < XR; ++m) xv[u][m] = ld16(a.x + 2 * (min(m, a.M - 1) * a.ldx + k));
    } else {
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
    }
  };
  auto load_w = [&](int u, int j) {
    const int s = group_of(j);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      wsc[u][p] = *reinterpret_cast<const uint32_t*>(a.ws + (((int64_t)rbs[p] * a.groups + s) * 64 + lane) * 4);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        wv[u][p][t] = ld16nt(a.w + (((int64_t)rbs[p] * a.KT + min(4 * s + t, a.KT - 1)) * 64 + lane) * 16);
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
    if constexpr (XR > 0) {
      uint8_t* reg = smem + wave * X::kWave;
#pragma unroll
      for (int m = 0; m < XR; ++m) {
        const uint4 v = sel4(s * kMxGroup + 8 * lane < a.K, xv[u][m]);
        const uint32_t c = mx_code<ELEM>(quad_absmax(v));
        uint8_t* p = reg + m * X::kRow;
        if constexpr (ELEM == KRQ_MX_E2M1) *reinterpret_cast<uint32_t*>(p + 4 * lane) = mx_quant8_e2m1(v, c);
        else *reinterpret_cast<uint2*>(p + 8 * lane) = mx_quant8_e4m3(v, c);
        // block lane / 4 = 4 t + g of the row: byte t of dword g
        if ((lane & 3) == 0) p[X::kBytes + 4 * ((lane >> 2) & 3) + (lane >> 4)] = static_cast<uint8_t>(c);
      }
      // the wave reads only what it wrote: LDS operations of a wave complete in order
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
      const uint8_t* p = reg + min(r, XR - 1) * X::kRow;
      asc[u][0] = *reinterpret_cast<const uint32_t*>(p + X::kBytes + 4 * g);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const v8i A = lds_operand<ELEM>(p, t, g);
        if (4 * s + t < a.KT)
#pragma unroll
          for (int q = 0; q < P; ++q) acc[q][0] = mx_mfma<ELEM>(t, A, pack_v8i(wv[u][q][t], zero4()), acc[q][0], asc[u][0], wsc[u][q]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (4 * s + t < a.KT)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const v8i A = pack_v8i(av[u][mt][t * AB], AB == 2 ? av[u][mt][t * AB + AB - 1] : zero4());
#pragma unroll
            for (int q = 0; q < P; ++q)
              acc[q][mt] = mx_mfma<ELEM>(t, A, pack_v8i(wv[u][q][t], zero4()), acc[q][mt], asc[u][mt], wsc[u][q]);
          }
    }
  };

#pragma unroll
  for (int u = 0; u < U; ++u) load_x(u, u);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < U; ++u) load_w(u, u);
  __builtin_amdgcn_sched_barrier(0);
  int j = 0;
  for (; j + U < jc; j += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      consume(u, j + u);
      load_x(u, j + U + u);
      load_w(u, j + U + u);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) consume(u, j + u);

  // ---- the waves' sums, in wave order ----
  float* red = reinterpret_cast<float*>(smem);
  if (XR > 0) __syncthreads();  // (the rows' regions lie there)
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[((wave * P + p) * MT + mt) * 256 + i * 64 + lane] = acc[p][mt][i];
  __syncthreads();
  constexpr int PO = MODE == KRQ_OUT_SWIGLU ? 1 : P;  // output row blocks
  for (int v = threadIdx.x; v < PO * MT * 256; v += blockDim.x) {
    const int p = v / (MT * 256), e = v % (MT * 256);
    const int m = 16 * (e >> 8) + 4 * ((e >> 4) & 3) + ((e >> 6) & 3);
    const int64_t n = ((int64_t)blockIdx.x * PO + p) * 16 + (e & 15);
    const bool real = m < a.M && n < a.NO;
    float y = 0.0f, up = 0.0f;
    for (int w = 0; w < nw; ++w) {
      y += red[(w * P + p) * MT * 256 + e];
      if (MODE == KRQ_OUT_SWIGLU) up += red[(w * P + 1) * MT * 256 + e];
    }
    if constexpr (MODE == kOutArgmax) {
      Best b{-INFINITY, 0x7fffffff};
      if (real) {
        const uint16_t yb = f32_to_bf16(y);
        if (a.out) static_cast<uint16_t*>(a.out)[(int64_t)m * a.NO + n] = yb;
        b = Best{bf16_to_f32(yb), static_cast<int>(n)};
      }
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) {
        const Best c = shfl_best(b, o);
        if (better(c.v, c.i, b.v, b.i)) b = c;
      }
      if (real && (e & 15) == 0) a.cand[(int64_t)m * a.nrb + (int64_t)blockIdx.x * PO + p] = b;
    } else if (real) {
      if constexpr (MODE == KRQ_OUT_SWIGLU) y = y / (1.0f + expf(-y)) * up;
      if constexpr (MODE == KRQ_OUT_PARTIAL) static_cast<float*>(a.out)[((int64_t)sp * a.M + m) * a.NO + n] = y;
      else static_cast<uint16_t*>(a.out)[(int64_t)m * a.NO + n] = f32_to_bf16(y);
    }
  }
}

template <int ELEM, int XR, int MT, int MODE, int P, int U>
void launch(const MxArgs& a, int blocks, int splits, int nw, hipStream_t s) {
  size_t smem = (size_t)nw * P * MT * 1024;
  if (XR > 0) smem = std::max(smem, (size_t)nw * XLds<ELEM, XR>::kWave);
  hipLaunchKernelGGL((k_gemv_mx<ELEM, XR, MT, MODE, P, U>), dim3(blocks, splits), dim3(64 * nw), smem, s, a);
}

template <int ELEM, int MODE, int P>
void launch_rows(const MxArgs& a, bool bf16, int blocks, int splits, int nw, hipStream_t s) {
  if (bf16) {
    if (a.M == 1) launch<ELEM, 1, 1, MODE, P, 2>(a, blocks, splits, nw, s);
    else if (a.M <= 4) launch<ELEM, 4, 1, MODE, P, 2>(a, blocks, splits, nw, s);
    else launch<ELEM, 8, 1, MODE, P, 2>(a, blocks, splits, nw, s);
  } else if (a.M <= 16) {
    launch<ELEM, 0, 1, MODE, P, 2>(a, blocks, splits, nw, s);
  } else {
    launch<ELEM, 0, 2, MODE, P, 1>(a, blocks, splits, nw, s);
  }
}

}  // namespace

namespace krq {

// The checks and the launch of every product on MXFP4 weights of at most 32 rows (kOutArgmax: the head's).
int gemv_mx_run(const char* what, const void* x, const void* x_scale, int x_kind, int elem, int64_t ldx, const void* w,
                const void* w_scale, int64_t M, int64_t N, int64_t K, int split, int mode, void* ws, int64_t ws_bytes, void* out,
                Best* cand, void* stream) {
  KRQ_REQUIRE(x && w && w_scale && (out || mode == kOutArgmax), "%s: null pointer", what);
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "%s: bad element type %d", what, elem);
  KRQ_REQUIRE(x_kind == KRQ_MX_X_BF16 || x_kind == KRQ_MX_X_TILED, "%s: bad x_kind %d", what, x_kind);
  KRQ_REQUIRE(M >= 1 && M <= 32, "%s: M=%lld outside 1..32", what, (long long)M);
  KRQ_REQUIRE(N >= 1 && N <= 0x7fffffff - 64 && K >= kMxBlock && K % kMxBlock == 0 && K <= 0x3fffffff, "%s: shape N=%lld K=%lld (K a multiple of 32)", what,
              (long long)N, (long long)K);
  const bool bf16 = x_kind == KRQ_MX_X_BF16 && M <= KRQ_MX_BF16_ROWS;  // rounded in the kernel
  const int64_t rows = x_kind == KRQ_MX_X_BF16 && !bf16 ? mx_rows_bytes(elem, M, K) : 0;
  KRQ_REQUIRE(x_kind == KRQ_MX_X_BF16 || x_scale, "%s: tiled rows need their scales", what);
  KRQ_REQUIRE(x_kind != KRQ_MX_X_BF16 || (ldx >= K && ldx % 8 == 0), "%s: rows of x must start on 16 bytes (ldx=%lld)", what, (long long)ldx);
  KRQ_REQUIRE(aligned16(x) && aligned16(w) && aligned16(ws), "%s: x, w and ws must start on 16 bytes", what);
  KRQ_REQUIRE(rows == 0 || (ws && ws_bytes >= rows), "%s: bf16 rows need a workspace of %lld bytes", what, (long long)rows);
  const int groups = static_cast<int>(mx_groups(K));
  KRQ_REQUIRE(split >= 1 && split <= groups && split <= kMxSplitMax, "%s: split=%d of %d groups of 512", what, split, groups);
  KRQ_REQUIRE(split == 1 || mode == KRQ_OUT_PARTIAL, "%s: split=%d needs the partials output", what, split);
  const bool swiglu = mode == KRQ_OUT_SWIGLU;
  KRQ_REQUIRE(!swiglu || N % 32 == 0, "%s: SwiGLU needs N=%lld = 2 I with I %% 16 == 0", what, (long long)N);
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
  hipStream_t s = (hipStream_t)stream;
  const int per = (groups + split - 1) / split;  // groups of the longest split
  const int nw = std::min(per, kMaxWaves);
#define KRQ_MX_GO(MODE_, P_)                                                                            \
  do {                                                                                                  \
    const int blocks = (a.nrb + (MODE_ == KRQ_OUT_SWIGLU ? 1 : (P_)) - 1) / (MODE_ == KRQ_OUT_SWIGLU ? 1 : (P_)); \
    if (elem == KRQ_MX_E2M1) launch_rows<KRQ_MX_E2M1, MODE_, P_>(a, bf16, blocks, split, nw, s);        \
    else launch_rows<KRQ_MX_E4M3, MODE_, P_>(a, bf16, blocks, split, nw, s);                            \
  } while (0)
  if (mode == KRQ_OUT_SWIGLU) KRQ_MX_GO(KRQ_OUT_SWIGLU, 2);
  else if (mode == KRQ_OUT_PARTIAL) KRQ_MX_GO(KRQ_OUT_PARTIAL, 1);
  else if (mode == kOutArgmax) KRQ_MX_GO(kOutArgmax, 2);
  else if (mode == KRQ_OUT_BF16) KRQ_MX_GO(KRQ_OUT_BF16, 1);
  else KRQ_REQUIRE(false, "%s: bad mode %d", what, mode);
#undef KRQ_MX_GO
  return krq_check_launch(what);
}

}  // namespace krq

extern "C" int64_t krq_gemv_mxfp4_ws_bytes(int x_kind, int elem, int64_t M, int64_t K) {
  if (M < 1 || M > 32 || K < 1 || (elem != KRQ_MX_E2M1 && elem != KRQ_MX_E4M3)) return -1;
  return x_kind == KRQ_MX_X_BF16 && M > KRQ_MX_BF16_ROWS ? mx_rows_bytes(elem, M, K) : 0;
}

extern "C" int krq_gemv_mxfp4(const void* x, const void* x_scale, int x_kind, int elem, int64_t ldx, const void* w_tiled,
                              const void* w_scale, int64_t M, int64_t N, int64_t K, int split, int mode, void* ws, int64_t ws_bytes,
                              void* out, void* stream) {
  KRQ_REQUIRE(mode == KRQ_OUT_BF16 || mode == KRQ_OUT_PARTIAL || mode == KRQ_OUT_SWIGLU, "gemv_mxfp4: bad mode %d", mode);
  return gemv_mx_run("gemv_mxfp4", x, x_scale, x_kind, elem, ldx, w_tiled, w_scale, M, N, K, split, mode, ws, ws_bytes, out, nullptr,
                     stream);
}

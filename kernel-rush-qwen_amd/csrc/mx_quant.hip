// Microscaled (OCP MX) quantisation and what undoes it: bf16 rows to e2m1 or e4m3 blocks in the operand
// tiles of mx_common.h (weights also row-major), packed codes to tiles, tiles to bf16, and rows of a packed
// table by index. Every kernel moves each byte once; all are bound by memory, the small ones by one round
// trip to it. us: weights 19,456 x 2,560 28.0 (153 MB, 5.4 TB/s), back to bf16 19.4 (126 MB, 6.5 TB/s), 4,096 rows of 2,560 to
// e4m3 8.1 and 16 rows 3.4, 4,095 rows of a table 7.3 (27 MB) and 16 rows 2.2.
#include <algorithm>

#include "mx_common.h"

using namespace krq;

namespace {

// One workgroup takes 16 rows x 512 k, a scale group, its wave t the tile t: load i gives lane l eight values of row
// 4 i + l / 16 at k = 8 (l % 16) of the tile, so that each load reads four runs of 256 bytes, the four lanes of a quad
// hold one block, and a store of four rows fills runs of 64 bytes of the tile. All four loads are in flight before the
// first is used. The 256 scale bytes meet in LDS and leave as one dword per lane.
template <int ELEM, bool ROWMAJOR>
__global__ __launch_bounds__(256) void k_mx_quant(const uint16_t* __restrict__ x, uint8_t* __restrict__ tiled,
                                                  uint32_t* __restrict__ tscale, int64_t M, int64_t ldx, int K, int mbs,
                                                  uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  __shared__ __align__(16) uint8_t sc[256];  // byte 4 (16 g + r) + t: block 4 t + g of row r
  const int lane = threadIdx.x & 63, t = threadIdx.x >> 6, kc = 8 * (lane & 15), rl = lane >> 4, b = kc >> 5;
  const int s = blockIdx.x, tile = 4 * s + t, k = kMxTile * tile + kc, KT = static_cast<int>(mx_tiles(K));
  for (int64_t mb = blockIdx.y; mb < mbs; mb += gridDim.y) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = min(mb * 16 + 4 * i + rl, M - 1);
      v[i] = ld16(reinterpret_cast<const uint8_t*>(x + row * ldx + min(k, K - 8)));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + rl;
      const bool real = mb * 16 + r < M && k < K;
      const uint4 a = sel4(real, v[i]);
      const uint32_t c = mx_code<ELEM>(quad_absmax(a));
      if ((lane & 3) == 0) sc[4 * (16 * b + r) + t] = static_cast<uint8_t>(c);
      if constexpr (ELEM == KRQ_MX_E2M1) {
        const uint32_t o = mx_quant8_e2m1(a, c);
        if (tile < KT)
          *reinterpret_cast<uint32_t*>(tiled + ((mb * KT + tile) * 64 + 16 * b + r) * 16 + 4 * (lane & 3)) = o;
        if (ROWMAJOR && real) *reinterpret_cast<uint32_t*>(q + (mb * 16 + r) * (K >> 1) + (k >> 1)) = o;
      } else {
        const uint2 o = mx_quant8_e4m3(a, c);
        if (tile < KT)
          *reinterpret_cast<uint2*>(tiled + (mb * KT + tile) * 2048 + 1024 * (kc >> 6) + 16 * (16 * ((kc & 63) >> 4) + r) +
                                    (kc & 15)) = o;
      }
    }
    __syncthreads();
    if (t == 0) tscale[(mb * gridDim.x + s) * 64 + lane] = *reinterpret_cast<const uint32_t*>(sc + 4 * lane);
    if (ROWMAJOR && t == 1) {  // lane: row lane / 4, blocks 4 u .. 4 u + 3 of tile u = lane % 4
      const int r = lane >> 2, u = lane & 3;
      const int64_t row = mb * 16 + r;
      const int kb = K >> 5, b0 = 16 * s + 4 * u;
      if (row < M) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (b0 + g < kb) scale[row * kb + b0 + g] = sc[4 * (16 * g + r) + u];
      }
    }
    __syncthreads();
  }
}

// Row-major codes and scales to tiles: one wave per scale group, lane l a row's 16 bytes of each tile.
__global__ __launch_bounds__(64) void k_mx_pack(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                uint8_t* __restrict__ tiled, uint32_t* __restrict__ tscale, int64_t N, int K,
                                                int nbs) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4, s = blockIdx.x;
  const int KT = static_cast<int>(mx_tiles(K)), kb = K >> 5;
  for (int64_t nb = blockIdx.y; nb < nbs; nb += gridDim.y) {
    const int64_t n = nb * 16 + r, row = min(n, N - 1);
    uint4 v[4];
    uint32_t c[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int b = min(16 * s + 4 * t + g, kb - 1);
      v[t] = ld16(q + row * (K >> 1) + 16 * b);
      c[t] = scale[row * kb + b];
    }
    uint32_t w = 0;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const bool real = n < N && 16 * s + 4 * t + g < kb;
      if (real) w |= c[t] << (8 * t);
      if (4 * s + t < KT) *reinterpret_cast<uint4*>(tiled + ((nb * KT + 4 * s + t) * 64 + lane) * 16) = sel4(real, v[t]);
    }
    tscale[(nb * gridDim.x + s) * 64 + lane] = w;
  }
}

KRQ_DEV uint4 mx_dequant8_e2m1(uint32_t o, float s) {
  uint4 v;
  v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(o, s, 0));
  v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(o, s, 1));
  v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(o, s, 2));
  v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(o, s, 3));
  return v;
}
KRQ_DEV uint4 mx_dequant8_e4m3(uint2 o, float s) {
  uint4 v;
  v.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(o.x, s, false));
  v.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(o.x, s, true));
  v.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(o.y, s, false));
  v.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(o.y, s, true));
  return v;
}
constexpr uint4 kNaN8{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};

// Tiles to bf16, k_mx_quant's lanes in reverse.
template <int ELEM>
__global__ __launch_bounds__(256) void k_mx_dequant(const uint8_t* __restrict__ tiled, const uint8_t* __restrict__ tscale,
                                                    uint16_t* __restrict__ out, int64_t M, int K, int mbs) {
  const int lane = threadIdx.x & 63, t = threadIdx.x >> 6, kc = 8 * (lane & 15), rl = lane >> 4;
  const int s = blockIdx.x, k = kMxGroup * s + kMxTile * t + kc, KT = static_cast<int>(mx_tiles(K)), tile = min(4 * s + t, KT - 1);
  for (int64_t mb = blockIdx.y; mb < mbs; mb += gridDim.y) {
    uint2 v[4];
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + rl;
      c[i] = tscale[((mb * gridDim.x + s) * 64 + 16 * (kc >> 5) + r) * 4 + t];
      if constexpr (ELEM == KRQ_MX_E2M1)
        v[i].x = *reinterpret_cast<const uint32_t*>(tiled + ((mb * KT + tile) * 64 + 16 * (kc >> 5) + r) * 16 + 4 * (lane & 3));
      else
        v[i] = *reinterpret_cast<const uint2*>(tiled + (mb * KT + tile) * 2048 + 1024 * (kc >> 6) +
                                               16 * (16 * ((kc & 63) >> 4) + r) + (kc & 15));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = mb * 16 + 4 * i + rl;
      const float f = mx_scale(c[i]);
      uint4 o;
      if constexpr (ELEM == KRQ_MX_E2M1) o = mx_dequant8_e2m1(v[i].x, f);
      else o = mx_dequant8_e4m3(v[i], f);
      if (c[i] == 255u) o = kNaN8;
      if (row < M && k < K) *reinterpret_cast<uint4*>(out + row * K + k) = o;
    }
  }
}

// Rows of a packed table: out[i] = bf16(w[ids[i]] * mult), the product in fp32 (w is exact in it). A wave takes 512 k of a
// row, eight values per lane, and a workgroup four rows; an index outside the table gives a row of NaN.
template <typename ID>
__global__ __launch_bounds__(256) void k_mx_embed(const ID* __restrict__ ids, const uint8_t* __restrict__ q,
                                                  const uint8_t* __restrict__ scale, uint16_t* __restrict__ out, int64_t N,
                                                  int64_t T, int K, float mult) {
  const int c = blockIdx.x * 64 + (threadIdx.x & 63);  // the row's eight values 8 c .. 8 c + 7
  if (8 * c >= K) return;
  for (int64_t i = blockIdx.y * (int64_t)4 + (threadIdx.x >> 6); i < T; i += (int64_t)gridDim.y * 4) {
    const int64_t id = ids[i];
    const bool real = id >= 0 && id < N;
    const int64_t row = real ? id : 0;
    const uint32_t o = *reinterpret_cast<const uint32_t*>(q + row * (K >> 1) + 4 * c);
    // Codes 253 and 254: 4 (or 2) times the scale passes fp32 where its product with mult need not. 2^8 of the scale is kept back
    // until then; the product before is normal for every mult, so that it is rounded as the whole one.
    const uint32_t code = scale[row * (K >> 5) + (c >> 2)];
    const bool far = code == 253u || code == 254u;
    const float s = mx_scale(far ? code - 8 : code), rest = far ? 256.0f : 1.0f;
    const uint4 v = mx_dequant8_e2m1(o, 1.0f);
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = pack_bf16x2(as_f32(w[j] << 16) * s * mult * rest, as_f32(w[j] & 0xffff0000u) * s * mult * rest);
    *reinterpret_cast<uint4*>(out + i * K + 8 * c) = real ? make_uint4(w[0], w[1], w[2], w[3]) : kNaN8;
  }
}

constexpr int64_t kGridY = 65535;

int mx_shape(const char* what, int64_t M, int64_t K) {
  KRQ_REQUIRE(M >= 1 && K >= kMxBlock && K % kMxBlock == 0, "%s: shape %lld x %lld (K a multiple of 32)", what, (long long)M,
              (long long)K);
  KRQ_REQUIRE(M <= 0x7fffffff && K <= 0x1ffffff, "%s: %lld x %lld is too large", what, (long long)M, (long long)K);
  return KRQ_OK;
}
int mx_mbs(int64_t M) { return static_cast<int>((M + 15) / 16); }
// a workgroup per scale group and row block, groups first (row blocks past the grid's second axis by a loop)
dim3 mx_grid(int64_t M, int64_t K) {
  return dim3(static_cast<unsigned>(mx_groups(K)), static_cast<unsigned>(std::min<int64_t>(mx_mbs(M), kGridY)));
}

}  // namespace

extern "C" int64_t krq_mx_tiled_bytes(int64_t M, int64_t K, int elem) {
  if (M < 1 || K < 1 || (elem != KRQ_MX_E2M1 && elem != KRQ_MX_E4M3)) return -1;
  return (M + 15) / 16 * mx_tiles(K) * mx_tile_bytes(elem);
}

extern "C" int64_t krq_mx_scale_bytes(int64_t M, int64_t K) {
  return M < 1 || K < 1 ? -1 : (M + 15) / 16 * mx_groups(K) * 256;
}

extern "C" int krq_quant_mxfp4(const void* w_bf16, int64_t N, int64_t K, int64_t ldw, void* w4, void* scale, void* tiled,
                               void* tiled_scale, void* stream) {
  KRQ_REQUIRE(w_bf16 && w4 && scale && tiled && tiled_scale, "quant_mxfp4: null pointer");
  if (const int rc = mx_shape("quant_mxfp4", N, K)) return rc;
  KRQ_REQUIRE(ldw >= K && ldw % 8 == 0 && aligned16(w_bf16), "quant_mxfp4: rows of w must start on 16 bytes (ldw=%lld)", (long long)ldw);
  KRQ_REQUIRE(aligned16(w4) && aligned16(tiled) && aligned16(tiled_scale), "quant_mxfp4: w4 and the tiles must start on 16 bytes");
  hipLaunchKernelGGL((k_mx_quant<KRQ_MX_E2M1, true>), mx_grid(N, K), dim3(256), 0, (hipStream_t)stream, (const uint16_t*)w_bf16,
                     (uint8_t*)tiled, (uint32_t*)tiled_scale, N, ldw, (int)K, mx_mbs(N), (uint8_t*)w4, (uint8_t*)scale);
  return krq_check_launch("quant_mxfp4");
}

extern "C" int krq_quant_mx_rows(const void* x_bf16, int64_t M, int64_t K, int64_t ldx, int elem, void* tiled, void* tiled_scale,
                                 void* stream) {
  KRQ_REQUIRE(x_bf16 && tiled && tiled_scale, "quant_mx_rows: null pointer");
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "quant_mx_rows: bad element type %d", elem);
  if (const int rc = mx_shape("quant_mx_rows", M, K)) return rc;
  KRQ_REQUIRE(ldx >= K && ldx % 8 == 0 && aligned16(x_bf16), "quant_mx_rows: rows of x must start on 16 bytes (ldx=%lld)", (long long)ldx);
  KRQ_REQUIRE(aligned16(tiled) && aligned16(tiled_scale), "quant_mx_rows: the tiles must start on 16 bytes");
  const dim3 grid = mx_grid(M, K);
  if (elem == KRQ_MX_E2M1)
    hipLaunchKernelGGL((k_mx_quant<KRQ_MX_E2M1, false>), grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t*)x_bf16,
                       (uint8_t*)tiled, (uint32_t*)tiled_scale, M, ldx, (int)K, mx_mbs(M), nullptr, nullptr);
  else
    hipLaunchKernelGGL((k_mx_quant<KRQ_MX_E4M3, false>), grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t*)x_bf16,
                       (uint8_t*)tiled, (uint32_t*)tiled_scale, M, ldx, (int)K, mx_mbs(M), nullptr, nullptr);
  return krq_check_launch("quant_mx_rows");
}

extern "C" int krq_pack_mxfp4(const void* w4, const void* scale, int64_t N, int64_t K, void* tiled, void* tiled_scale, void* stream) {
  KRQ_REQUIRE(w4 && scale && tiled && tiled_scale, "pack_mxfp4: null pointer");
  if (const int rc = mx_shape("pack_mxfp4", N, K)) return rc;
  KRQ_REQUIRE(aligned16(w4) && aligned16(tiled) && aligned16(tiled_scale), "pack_mxfp4: w4 and the tiles must start on 16 bytes");
  hipLaunchKernelGGL(k_mx_pack, mx_grid(N, K), dim3(64), 0, (hipStream_t)stream, (const uint8_t*)w4, (const uint8_t*)scale,
                     (uint8_t*)tiled, (uint32_t*)tiled_scale, N, (int)K, mx_mbs(N));
  return krq_check_launch("pack_mxfp4");
}

extern "C" int krq_dequant_mx(const void* tiled, const void* tiled_scale, int elem, int64_t M, int64_t K, void* out, void* stream) {
  KRQ_REQUIRE(tiled && tiled_scale && out, "dequant_mx: null pointer");
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "dequant_mx: bad element type %d", elem);
  if (const int rc = mx_shape("dequant_mx", M, K)) return rc;
  KRQ_REQUIRE(aligned16(out) && aligned16(tiled) && aligned16(tiled_scale), "dequant_mx: out and the tiles must start on 16 bytes");
  const dim3 grid = mx_grid(M, K);
  if (elem == KRQ_MX_E2M1)
    hipLaunchKernelGGL((k_mx_dequant<KRQ_MX_E2M1>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)tiled,
                       (const uint8_t*)tiled_scale, (uint16_t*)out, M, (int)K, mx_mbs(M));
  else
    hipLaunchKernelGGL((k_mx_dequant<KRQ_MX_E4M3>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)tiled,
                       (const uint8_t*)tiled_scale, (uint16_t*)out, M, (int)K, mx_mbs(M));
  return krq_check_launch("dequant_mx");
}

extern "C" int krq_embed_mxfp4(const void* ids, int ids_64, int64_t T, const void* w4, const void* scale, int64_t N, int64_t K, float mult,
                               void* out, void* stream) {
  KRQ_REQUIRE(ids && w4 && scale && out, "embed_mxfp4: null pointer");
  if (const int rc = mx_shape("embed_mxfp4", N, K)) return rc;
  KRQ_REQUIRE(T >= 1 && T <= 0x7fffffffffll, "embed_mxfp4: %lld indices", (long long)T);
  KRQ_REQUIRE(aligned16(w4) && aligned16(out), "embed_mxfp4: w4 and out must start on 16 bytes");
  const dim3 grid(static_cast<unsigned>(mx_groups(K)), static_cast<unsigned>(std::min<int64_t>((T + 3) / 4, kGridY)));
  if (ids_64)
    hipLaunchKernelGGL((k_mx_embed<int64_t>), grid, dim3(256), 0, (hipStream_t)stream, (const int64_t*)ids, (const uint8_t*)w4,
                       (const uint8_t*)scale, (uint16_t*)out, N, T, (int)K, mult);
  else
    hipLaunchKernelGGL((k_mx_embed<int32_t>), grid, dim3(256), 0, (hipStream_t)stream, (const int32_t*)ids, (const uint8_t*)w4,
                       (const uint8_t*)scale, (uint16_t*)out, N, T, (int)K, mult);
  return krq_check_launch("embed_mxfp4");
}

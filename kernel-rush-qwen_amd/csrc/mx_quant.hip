// Microscaled (OCP MX) quantisation and what undoes it: bf16 rows to e2m1 or e4m3 blocks in the operand
// tiles of mx_common.h (weights also row-major), packed codes to tiles, tiles to bf16, and rows of a packed
// table by index. Every kernel moves each byte once; all are bound by memory, the small ones by one round
// trip to it.
#include "mx_common.h"

using namespace krq;

namespace {

// One wave takes 16 rows x 512 k, a scale group of four tiles: load i of tile t gives lane l eight values
// of row 4 i + l / 16 at k = 128 t + 8 (l % 16), so each load reads four runs of 256 bytes, the four lanes of a quad
// hold one block, and a store of four rows fills runs of 64 bytes of the tile. All sixteen loads are in flight before the
// first is used. The 256 scale bytes meet in LDS and leave as one dword per lane.
template <int ELEM, bool ROWMAJOR>
__global__ __launch_bounds__(64) void k_mx_quant(const uint16_t* __restrict__ x, int64_t M, int K, int64_t ldx,
                                                 int groups, uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                                                 uint8_t* __restrict__ tiled, uint32_t* __restrict__ tscale) {
  __shared__ __align__(16) uint8_t sc[256];  // byte 4 (16 g + r) + t: block 4 t + g of row r
  const int lane = threadIdx.x, kc = 8 * (lane & 15), rl = lane >> 4;
  const int64_t mb = blockIdx.x / groups;
  const int s = static_cast<int>(blockIdx.x - mb * groups), k0 = s * kMxGroup;
  const int KT = static_cast<int>(mx_tiles(K));
  uint4 v[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = min(mb * 16 + 4 * i + rl, M - 1);
      const int k = min(k0 + 128 * t + kc, K - 8);
      v[t][i] = ld16(reinterpret_cast<const uint8_t*>(x + row * ldx + k));
    }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int tile = 4 * s + t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + rl;
      const bool real = mb * 16 + r < M && k0 + 128 * t + kc < K;
      const uint4 a = sel4(real, v[t][i]);
      const uint32_t c = mx_code<ELEM>(quad_absmax(a));
      const int b = kc >> 5;  // block of the tile
      if ((lane & 3) == 0) sc[4 * (16 * b + r) + t] = static_cast<uint8_t>(c);
      if constexpr (ELEM == KRQ_MX_E2M1) {
        const uint32_t o = mx_quant8_e2m1(a, c);
        if (tile < KT)
          *reinterpret_cast<uint32_t*>(tiled + ((mb * KT + tile) * 64 + 16 * b + r) * 16 + 4 * (lane & 3)) = o;
        if (ROWMAJOR && real) *reinterpret_cast<uint32_t*>(q + (mb * 16 + r) * (K >> 1) + ((k0 + 128 * t + kc) >> 1)) = o;
      } else {
        const uint2 o = mx_quant8_e4m3(a, c);
        if (tile < KT)
          *reinterpret_cast<uint2*>(tiled + (mb * KT + tile) * 2048 + 1024 * (kc >> 6) + 16 * (16 * ((kc & 63) >> 4) + r) +
                                    (kc & 15)) = o;
      }
    }
  }
  __syncthreads();
  tscale[(mb * groups + s) * 64 + lane] = *reinterpret_cast<const uint32_t*>(sc + 4 * lane);
  if (ROWMAJOR) {  // lane: row lane / 4, blocks 4 t .. 4 t + 3 of tile t = lane % 4
    const int r = lane >> 2, t = lane & 3;
    const int64_t row = mb * 16 + r;
    const int kb = K >> 5, b0 = 16 * s + 4 * t;
    if (row < M)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (b0 + g < kb) scale[row * kb + b0 + g] = sc[4 * (16 * g + r) + t];
  }
}

// Row-major codes and scales to tiles: one wave per scale group, lane l a row's 16 bytes of each tile.
__global__ __launch_bounds__(64) void k_mx_pack(const uint8_t* __restrict__ q, const uint8_t* __restrict__ scale,
                                                int64_t N, int K, int groups, uint8_t* __restrict__ tiled,
                                                uint32_t* __restrict__ tscale) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
  const int64_t nb = blockIdx.x / groups;
  const int s = static_cast<int>(blockIdx.x - nb * groups);
  const int KT = static_cast<int>(mx_tiles(K)), kb = K >> 5;
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
    if (4 * s + t < KT)
      *reinterpret_cast<uint4*>(tiled + ((nb * KT + 4 * s + t) * 64 + lane) * 16) = sel4(real, v[t]);
  }
  tscale[(nb * groups + s) * 64 + lane] = w;
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

// Tiles to bf16, k_mx_quant's lanes in reverse: one wave per 16 rows x 512 k, every load first.
template <int ELEM>
__global__ __launch_bounds__(64) void k_mx_dequant(const uint8_t* __restrict__ tiled, const uint8_t* __restrict__ tscale,
                                                   int64_t M, int K, int groups, uint16_t* __restrict__ out) {
  const int lane = threadIdx.x, kc = 8 * (lane & 15), rl = lane >> 4;
  const int64_t mb = blockIdx.x / groups;
  const int s = static_cast<int>(blockIdx.x - mb * groups), k0 = s * kMxGroup;
  const int KT = static_cast<int>(mx_tiles(K));
  uint2 v[4][4];
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = *reinterpret_cast<const uint32_t*>(tscale + ((mb * groups + s) * 64 + 16 * (kc >> 5) + 4 * i + rl) * 4);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int tile = min(4 * s + t, KT - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * i + rl;
      if constexpr (ELEM == KRQ_MX_E2M1)
        v[t][i].x =
            *reinterpret_cast<const uint32_t*>(tiled + ((mb * KT + tile) * 64 + 16 * (kc >> 5) + r) * 16 + 4 * (lane & 3));
      else
        v[t][i] = *reinterpret_cast<const uint2*>(tiled + (mb * KT + tile) * 2048 + 1024 * (kc >> 6) +
                                                  16 * (16 * ((kc & 63) >> 4) + r) + (kc & 15));
    }
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = mb * 16 + 4 * i + rl;
      const int k = k0 + 128 * t + kc;
      const uint32_t cc = (c[i] >> (8 * t)) & 255u;
      const float f = mx_scale(cc);
      uint4 o;
      if constexpr (ELEM == KRQ_MX_E2M1) o = mx_dequant8_e2m1(v[t][i].x, f);
      else o = mx_dequant8_e4m3(v[t][i], f);
      if (cc == 255u) o = kNaN8;
      if (row < M && k < K) *reinterpret_cast<uint4*>(out + row * K + k) = o;
    }
}

// Rows of a packed table: out[i] = bf16(w[ids[i]] * mult), the product in fp32 (w is exact in it). Eight values
// per thread; an index outside the table gives a row of NaN. One wave per 512 k of a row.
template <typename ID>
__global__ __launch_bounds__(256) void k_mx_embed(const ID* __restrict__ ids, const uint8_t* __restrict__ q,
                                                  const uint8_t* __restrict__ scale, int64_t N, int K, float mult,
                                                  int64_t chunks, uint16_t* __restrict__ out) {
  const int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;  // eight values: row e / (K / 8)
  if (e >= chunks) return;
  const int per = K >> 3;
  const int64_t i = e / per;
  const int c = static_cast<int>(e - i * per);
  const int64_t id = ids[i];
  const bool real = id >= 0 && id < N;
  const int64_t row = real ? id : 0;
  const uint32_t o = *reinterpret_cast<const uint32_t*>(q + row * (K >> 1) + 4 * c);
  const uint32_t cc = scale[row * (K >> 5) + (c >> 2)];
  const uint4 v = mx_dequant8_e2m1(o, 1.0f);
  const float s = mx_scale(cc);
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = as_f32(w[j] << 16) * s * mult, b = as_f32(w[j] & 0xffff0000u) * s * mult;
    w[j] = static_cast<uint32_t>(f32_to_bf16(a)) | (static_cast<uint32_t>(f32_to_bf16(b)) << 16);
  }
  *reinterpret_cast<uint4*>(out + i * K + 8 * c) = real ? make_uint4(w[0], w[1], w[2], w[3]) : kNaN8;
}

int mx_shape(const char* what, int64_t M, int64_t K) {
  KRQ_REQUIRE(M >= 1 && K >= kMxBlock && K % kMxBlock == 0 && K <= 0x3fffffff, "%s: shape %lld x %lld (K a multiple of 32)", what,
              (long long)M, (long long)K);
  KRQ_REQUIRE((M + 15) / 16 <= 0x3ffffff / mx_groups(K), "%s: %lld x %lld is too large", what, (long long)M, (long long)K);
  return KRQ_OK;
}
unsigned mx_grid(int64_t M, int64_t K) { return static_cast<unsigned>((M + 15) / 16 * mx_groups(K)); }

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
  hipLaunchKernelGGL((k_mx_quant<KRQ_MX_E2M1, true>), dim3(mx_grid(N, K)), dim3(64), 0, (hipStream_t)stream,
                     (const uint16_t*)w_bf16, N, (int)K, ldw, (int)mx_groups(K), (uint8_t*)w4, (uint8_t*)scale, (uint8_t*)tiled,
                     (uint32_t*)tiled_scale);
  return krq_check_launch("quant_mxfp4");
}

extern "C" int krq_quant_mx_rows(const void* x_bf16, int64_t M, int64_t K, int64_t ldx, int elem, void* tiled, void* tiled_scale,
                                 void* stream) {
  KRQ_REQUIRE(x_bf16 && tiled && tiled_scale, "quant_mx_rows: null pointer");
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "quant_mx_rows: bad element type %d", elem);
  if (const int rc = mx_shape("quant_mx_rows", M, K)) return rc;
  KRQ_REQUIRE(ldx >= K && ldx % 8 == 0 && aligned16(x_bf16), "quant_mx_rows: rows of x must start on 16 bytes (ldx=%lld)", (long long)ldx);
  const dim3 grid(mx_grid(M, K));
  if (elem == KRQ_MX_E2M1)
    hipLaunchKernelGGL((k_mx_quant<KRQ_MX_E2M1, false>), grid, dim3(64), 0, (hipStream_t)stream, (const uint16_t*)x_bf16, M,
                       (int)K, ldx, (int)mx_groups(K), nullptr, nullptr, (uint8_t*)tiled, (uint32_t*)tiled_scale);
  else
    hipLaunchKernelGGL((k_mx_quant<KRQ_MX_E4M3, false>), grid, dim3(64), 0, (hipStream_t)stream, (const uint16_t*)x_bf16, M,
                       (int)K, ldx, (int)mx_groups(K), nullptr, nullptr, (uint8_t*)tiled, (uint32_t*)tiled_scale);
  return krq_check_launch("quant_mx_rows");
}

extern "C" int krq_pack_mxfp4(const void* w4, const void* scale, int64_t N, int64_t K, void* tiled, void* tiled_scale, void* stream) {
  KRQ_REQUIRE(w4 && scale && tiled && tiled_scale, "pack_mxfp4: null pointer");
  if (const int rc = mx_shape("pack_mxfp4", N, K)) return rc;
  KRQ_REQUIRE(aligned16(w4), "pack_mxfp4: w4 must start on 16 bytes");
  hipLaunchKernelGGL(k_mx_pack, dim3(mx_grid(N, K)), dim3(64), 0, (hipStream_t)stream, (const uint8_t*)w4, (const uint8_t*)scale, N,
                     (int)K, (int)mx_groups(K), (uint8_t*)tiled, (uint32_t*)tiled_scale);
  return krq_check_launch("pack_mxfp4");
}

extern "C" int krq_dequant_mx(const void* tiled, const void* tiled_scale, int elem, int64_t M, int64_t K, void* out, void* stream) {
  KRQ_REQUIRE(tiled && tiled_scale && out, "dequant_mx: null pointer");
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "dequant_mx: bad element type %d", elem);
  if (const int rc = mx_shape("dequant_mx", M, K)) return rc;
  KRQ_REQUIRE(aligned16(out), "dequant_mx: out must start on 16 bytes");
  const dim3 grid(mx_grid(M, K));
  if (elem == KRQ_MX_E2M1)
    hipLaunchKernelGGL((k_mx_dequant<KRQ_MX_E2M1>), grid, dim3(64), 0, (hipStream_t)stream, (const uint8_t*)tiled,
                       (const uint8_t*)tiled_scale, M, (int)K, (int)mx_groups(K), (uint16_t*)out);
  else
    hipLaunchKernelGGL((k_mx_dequant<KRQ_MX_E4M3>), grid, dim3(64), 0, (hipStream_t)stream, (const uint8_t*)tiled,
                       (const uint8_t*)tiled_scale, M, (int)K, (int)mx_groups(K), (uint16_t*)out);
  return krq_check_launch("dequant_mx");
}

extern "C" int krq_embed_mxfp4(const void* ids, int ids_64, int64_t T, const void* w4, const void* scale, int64_t N, int64_t K, float mult,
                               void* out, void* stream) {
  KRQ_REQUIRE(ids && w4 && scale && out, "embed_mxfp4: null pointer");
  if (const int rc = mx_shape("embed_mxfp4", N, K)) return rc;
  KRQ_REQUIRE(T >= 1 && T <= 0xffffff00ll / (K / 8), "embed_mxfp4: %lld indices", (long long)T);
  KRQ_REQUIRE(aligned16(w4) && aligned16(out), "embed_mxfp4: w4 and out must start on 16 bytes");
  const int64_t chunks = T * (K / 8);
  const dim3 grid(static_cast<unsigned>((chunks + 255) / 256));
  if (ids_64)
    hipLaunchKernelGGL((k_mx_embed<int64_t>), grid, dim3(256), 0, (hipStream_t)stream, (const int64_t*)ids, (const uint8_t*)w4,
                       (const uint8_t*)scale, N, (int)K, mult, chunks, (uint16_t*)out);
  else
    hipLaunchKernelGGL((k_mx_embed<int32_t>), grid, dim3(256), 0, (hipStream_t)stream, (const int32_t*)ids, (const uint8_t*)w4,
                       (const uint8_t*)scale, N, (int)K, mult, chunks, (uint16_t*)out);
  return krq_check_launch("embed_mxfp4");
}

// MXFP4 GEMM for prefill: out = bf16(x . w^T), x e4m3 or e2m1 blocks and w e2m1 blocks, both in the operand
// tiles of mx_common.h, fp32 accumulation.
//
// A workgroup owns 128 x 128 outputs, its four waves 64 x 64 each: per 128 k four activation and four weight
// tiles straight from memory and sixteen v_mfma_scale_f32_16x16x128_f8f6f4.
#include "mx_common.h"

using namespace krq;

namespace {

template <int ELEM>
__global__ __launch_bounds__(256) void k_gemm_mx(const uint8_t* __restrict__ x, const uint8_t* __restrict__ xs,
                                                 const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws, int M, int N,
                                                 int KT, int groups, int tiles_m, uint16_t* __restrict__ out) {
  constexpr int AB = ELEM == KRQ_MX_E2M1 ? 1 : 2;
  constexpr int fa = ELEM == KRQ_MX_E2M1 ? 4 : 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int m0 = static_cast<int>(blockIdx.x % tiles_m) * 8 + 4 * (wave & 1);  // in row blocks of 16
  const int n0 = static_cast<int>(blockIdx.x / tiles_m) * 8 + 4 * (wave >> 1);
  const int mbs = (M + 15) >> 4, nbs = (N + 15) >> 4;
  v4f acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < groups; ++s) {
    uint32_t sa[4], sb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sa[i] = *reinterpret_cast<const uint32_t*>(xs + (((int64_t)min(m0 + i, mbs - 1) * groups + s) * 64 + lane) * 4);
      sb[i] = *reinterpret_cast<const uint32_t*>(ws + (((int64_t)min(n0 + i, nbs - 1) * groups + s) * 64 + lane) * 4);
    }
    for (int t = 0; t < min(4, KT - 4 * s); ++t) {
      v8i a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* p = x + (((int64_t)min(m0 + i, mbs - 1) * KT + 4 * s + t) * (64 * AB) + lane) * 16;
        a[i] = pack_v8i(ld16(p), AB == 2 ? ld16(p + 1024) : zero4());
        b[i] = pack_v8i(ld16(w + (((int64_t)min(n0 + i, nbs - 1) * KT + 4 * s + t) * 64 + lane) * 16), zero4());
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a[i], b[j], acc[i][j], fa, 4, 0,
                                                                       static_cast<int>(sa[i] >> (8 * t)), 0,
                                                                       static_cast<int>(sb[j] >> (8 * t)));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t m = 16 * (m0 + i) + 4 * (lane >> 4) + e, n = 16 * (n0 + j) + (lane & 15);
        if (m < M && n < N) out[m * N + n] = f32_to_bf16(acc[i][j][e]);
      }
}

}  // namespace

extern "C" int krq_gemm_mxfp4(const void* x_tiled, const void* x_scale, int elem, const void* w_tiled, const void* w_scale,
                              int64_t M, int64_t N, int64_t K, void* out, void* stream) {
  KRQ_REQUIRE(x_tiled && x_scale && w_tiled && w_scale && out, "gemm_mxfp4: null pointer");
  KRQ_REQUIRE(elem == KRQ_MX_E2M1 || elem == KRQ_MX_E4M3, "gemm_mxfp4: bad element type %d", elem);
  KRQ_REQUIRE(aligned16(x_tiled) && aligned16(w_tiled), "gemm_mxfp4: x and w must start on 16 bytes");
  KRQ_REQUIRE(M >= 1 && M <= 0x3fffffff && N >= 1 && N <= 0x3fffffff && K >= kMxBlock && K % kMxBlock == 0 && K <= 0x3fffffff,
              "gemm_mxfp4: shape M=%lld N=%lld K=%lld (K a multiple of 32)", (long long)M, (long long)N, (long long)K);
  const int64_t tiles_m = (M + 127) / 128, blocks = tiles_m * ((N + 127) / 128);
  KRQ_REQUIRE(blocks <= 0xffffff, "gemm_mxfp4: M=%lld N=%lld are too large", (long long)M, (long long)N);
  const dim3 grid(static_cast<unsigned>(blocks));
  if (elem == KRQ_MX_E2M1)
    hipLaunchKernelGGL((k_gemm_mx<KRQ_MX_E2M1>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)x_tiled,
                       (const uint8_t*)x_scale, (const uint8_t*)w_tiled, (const uint8_t*)w_scale, (int)M, (int)N,
                       (int)mx_tiles(K), (int)mx_groups(K), (int)tiles_m, (uint16_t*)out);
  else
    hipLaunchKernelGGL((k_gemm_mx<KRQ_MX_E4M3>), grid, dim3(256), 0, (hipStream_t)stream, (const uint8_t*)x_tiled,
                       (const uint8_t*)x_scale, (const uint8_t*)w_tiled, (const uint8_t*)w_scale, (int)M, (int)N,
                       (int)mx_tiles(K), (int)mx_groups(K), (int)tiles_m, (uint16_t*)out);
  return krq_check_launch("gemm_mxfp4");
}

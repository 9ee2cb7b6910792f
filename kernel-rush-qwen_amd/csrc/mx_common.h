// Helpers shared by the microscaled kernels (OCP MX v1.0): blocks of 32 consecutive k of a row, each with
// one E8M0 scale byte c standing for 2^(c - 127) (255: NaN), elements e2m1 (4 bits: 0, .5, 1, 1.5, 2, 3, 4,
// 6 and their negatives) or e4m3.
//
// Quantisation of a block with largest magnitude a: c = max(0, floor(log2 a) + 127 - emax), emax the exponent
// of the format's largest value (2 for e2m1, 8 for e4m3), then every value / 2^(c - 127), which is exact,
// rounded to the nearest element, ties to even, and clamped to the largest (6 or 448; a / scale lies below
// 8 or 512). A block with a NaN or an infinity has c = 255 and elements 0: the format has no infinity.
//
// Operand tiles. A tile is 16 rows x 128 k, the operand of one v_mfma_scale_f32_16x16x128_f8f6f4, stored in
// lane order so that a wave's 16-byte-per-lane load is one contiguous KiB. Lane l = 16 g + r holds of row r
//   e2m1 (1 KiB): k = 32 g + 0..31, element 2i in the low half of byte i;
//   e4m3 (2 KiB): k = 16 g + 0..15 in the first KiB, 64 + 16 g + 0..15 in the second,
// the k orders of that instruction (its scale byte in lane l is that of row r, k = 32 g + 0..31 for both).
// Tiles are row-block-major, [rows / 16][KT] with KT = ceil(K / 128). Scales lie in groups of four tiles,
// [rows / 16][ceil(KT / 4)][64 lanes], 4 bytes per lane, byte t for tile 4 s + t: one dword load serves four
// instructions, which pick their byte by op_sel. Rows past the last and k past K have elements 0, scales 0.
#pragma once

#include "gemv_common.h"

namespace krq {

constexpr int kMxBlock = 32, kMxTile = 128, kMxGroup = 512;  // k per block, operand tile, scale group

KRQ_HD int64_t mx_tiles(int64_t K) { return (K + kMxTile - 1) / kMxTile; }
KRQ_HD int64_t mx_groups(int64_t K) { return (K + kMxGroup - 1) / kMxGroup; }
KRQ_HD int mx_tile_bytes(int elem) { return elem == KRQ_MX_E2M1 ? 1024 : 2048; }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// the scale code of a block from its largest magnitude, given as bf16 bits without the sign
template <int ELEM>
KRQ_DEV uint32_t mx_code(uint32_t mag) {
  constexpr uint32_t emax = ELEM == KRQ_MX_E2M1 ? 2 : 8;
  const uint32_t e = mag >> 7;
  return e == 255u ? 255u : e > emax ? e - emax : 0u;
}

// 2^(c - 127) for c < 255 (c = 0: the subnormal 2^-127); NaN for c = 255
KRQ_DEV float mx_scale(uint32_t c) { return as_f32(c == 0u ? 0x00400000u : c == 255u ? 0x7fc00000u : c << 23); }

// the largest magnitude (bf16 bits) of the 32 values held eight each by the four lanes of a quad
KRQ_DEV uint32_t quad_absmax(uint4 v) {
  uint32_t m = __builtin_bit_cast(uint32_t, absmax8_bits(v, u16x2{0, 0}));
  auto step = [](uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
  };
  m = step(m, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(m), 0xB1, 0xf, 0xf, false)));
  m = step(m, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(m), 0x4E, 0xf, 0xf, false)));
  const uint32_t hi = m >> 16, lo = m & 0xffffu;
  return hi > lo ? hi : lo;
}

// 8 bf16 of a block with scale code c -> 8 e2m1 elements. The convert divides by the scale, rounds to nearest
// even and saturates.
KRQ_DEV uint32_t mx_quant8_e2m1(uint4 v, uint32_t c) {
  const float s = mx_scale(c);
  uint32_t o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, v.x), s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, v.y), s, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, v.z), s, 2);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, __builtin_bit_cast(bf16x2, v.w), s, 3);
  return c == 255u ? 0u : o;
}

// 8 bf16 of a block with scale code c -> 8 e4m3 bytes. This convert turns what it would round past 448 into
// NaN, so the values are clamped first.
KRQ_DEV uint2 mx_quant8_e4m3(uint4 v, uint32_t c) {
  const float s = mx_scale(c), top = kFp8Max * s;
  auto pair = [&](uint32_t a, s16x2 o, bool hi) {
    const float x = __builtin_amdgcn_fmed3f(as_f32(a << 16), -top, top);
    const float y = __builtin_amdgcn_fmed3f(as_f32(a & 0xffff0000u), -top, top);
    return hi ? __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, x, y, s, true)
              : __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, x, y, s, false);
  };
  s16x2 lo = {0, 0}, hi = {0, 0};
  lo = pair(v.y, pair(v.x, lo, false), true);
  hi = pair(v.w, pair(v.z, hi, false), true);
  if (c == 255u) return make_uint2(0u, 0u);
  return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// workgroup barrier for LDS accesses alone: loads from memory stay in flight across it
KRQ_DEV void barrier_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Rows rounded into a workspace: elements, then scales, each on 256 bytes.
inline int64_t mx_rows_scale_at(int elem, int64_t M, int64_t K) { return (krq_mx_tiled_bytes(M, K, elem) + 255) & ~(int64_t)255; }
inline int64_t mx_rows_bytes(int elem, int64_t M, int64_t K) { return mx_rows_scale_at(elem, M, K) + krq_mx_scale_bytes(M, K); }

// Bytes of workspace that gemv_mx_run takes: room for the rounded rows where they are not rounded in the launch.
int64_t gemv_mx_rows_bytes(int x_kind, int elem, int64_t M, int64_t N, int64_t K, int split, int mode);

// The checks and the launch of every product on MXFP4 weights of at most 32 rows (gemv_mxfp4.hip; kOutArgmax:
// the lm head's, *cands candidates of each row to cand [M][*cands], at most 2 more than row blocks).
int gemv_mx_run(const char* what, const void* x, const void* x_scale, int x_kind, int elem, int64_t ldx, const void* w,
                const void* w_scale, int64_t M, int64_t N, int64_t K, int split, int mode, void* ws, int64_t ws_bytes, void* out,
                Best* cand, int64_t* cands, void* stream);

}  // namespace krq

// Layout and device helpers of MXFP4 matrices: 4-bit floating point (e2m1) in
// blocks of 32 along k with one shared power of two (e8m0) each, after the OCP
// Microscaling Formats (MX) v1.0.
//
// A matrix [rows][k] is kept in tiles of 16 rows x 128 k in the operand order of
// the 16x16 matrix instructions, so that a wave's load of a tile is 1,024
// contiguous bytes and is an operand as it stands:
//   codes  [row tile][k slab of 128][lane][16 bytes]: lane l holds row l % 16, the
//          block l / 16 of the slab; element j of the block in byte j / 2, the even
//          one in the lower half
//   scales [row tile][4 slabs][lane][4]: byte s of lane l is the scale of the block
//          that lane l holds of slab s
// Rows and k past the matrix are zero codes with scale byte 0.
#pragma once

#include "mi_common.h"

namespace mi::mx4 {

constexpr int kBlock = 32;
constexpr int kTileRows = 16;
constexpr int kSlab = 128;      // k per tile
constexpr int kTileBytes = 1024;
constexpr int kQuadBytes = 256;  // scales of a row tile over 4 slabs
constexpr int kMaxK = 1 << 20;

inline __host__ __device__ int64_t row_tiles(int64_t rows) { return (rows + kTileRows - 1) / kTileRows; }
inline __host__ __device__ int64_t slabs(int64_t k) { return (k + kSlab - 1) / kSlab; }
inline __host__ __device__ int64_t quads(int64_t k) { return (k + 4 * kSlab - 1) / (4 * kSlab); }

typedef __attribute__((ext_vector_type(4))) unsigned int u32x4_t;
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;
typedef __attribute__((ext_vector_type(8))) int i32x8_t;
typedef __attribute__((address_space(3))) char lds_t;

constexpr int kBufferWord3 = 0x00020000;
constexpr int kCacheNT = 2;

__device__ __forceinline__ u32x4_t lds_load16(const lds_t* p) {
  return *(const __attribute__((address_space(3))) u32x4_t*)p;
}
__device__ __forceinline__ uint32_t lds_load4(const lds_t* p) { return *(const __attribute__((address_space(3))) uint32_t*)p; }
__device__ __forceinline__ void lds_store16(lds_t* p, u32x4_t v) { *(__attribute__((address_space(3))) u32x4_t*)p = v; }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, kBufferWord3);
}

// The power of two of a scale byte as the conversions take it: they read the
// exponent field alone (0 is 2^-127, 255 NaN).
__device__ __forceinline__ float scale_f32(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight codes to bf16, exactly: three significant bits and a power of two.
__device__ __forceinline__ bf16x8_t to_bf16(uint32_t codes, float scale) {
  typedef __attribute__((ext_vector_type(2))) __bf16 pair_t;
  pair_t v[4];
  v[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  v[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  v[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  v[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return __builtin_bit_cast(bf16x8_t, v);
}

// D(16x16 fp32) += A(16x128) * B(128x16), both fp4 with a scale byte per lane (row
// or column l % 16, block l / 16).
template <int SA, int SB>
__device__ __forceinline__ f32x4_t mfma_fp4(u32x4_t a, uint32_t sa, u32x4_t b, uint32_t sb, f32x4_t c) {
  const i32x8_t x = {int(a[0]), int(a[1]), int(a[2]), int(a[3]), 0, 0, 0, 0};
  const i32x8_t y = {int(b[0]), int(b[1]), int(b[2]), int(b[3]), 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, SA, int(sa), SB, int(sb));
}

}  // namespace mi::mx4

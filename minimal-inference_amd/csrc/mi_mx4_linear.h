// What the launches of MXFP4 projections share: arguments, the rows of W that a
// lane reads, and the end of a product.
#pragma once

#include "mi_mx4.h"

namespace mi::mx4 {

struct LinearParams {
  const char* x;     // bf16 rows, or tiles of codes
  int64_t x_stride;  // of bf16 rows
  const char* xs;    // scales of x's tiles; null: x is bf16
  const char* w;
  const char* ws;
  const uint16_t* bias;  // null: none
  uint16_t* out;
  int64_t o_stride;
  int64_t rows;
  int n, k;  // n: columns of out; with the gated product W holds n gate rows, then n up rows
  int slabs, quads;
  int w_tiles;  // row tiles of W
  f32x4_t* parts;   // sums of workgroups that share k
  int split_slabs;  // slabs that one of them takes
  bool vec;     // out and bias take 8-byte accesses,
  bool wide;    // out 16-byte ones
};

// Row h n + first + i of W (i the lane's row of 16): its 16 codes' place from the
// tile of row h n + first on.  n need not be a multiple of 16, so a lane's up row may
// lie in another tile than its neighbour's.
struct LaneRow {
  int codes, scales;
};
__device__ __forceinline__ LaneRow lane_row(const LinearParams& p, int base_row, int row, int g) {
  const int tile = row / kTileRows - base_row / kTileRows, at = row % kTileRows + 16 * g;
  return {tile * p.slabs * kTileBytes + at * 16, tile * p.quads * kQuadBytes + at * 4};
}

// The bias of columns col .. col + 3.
__device__ __forceinline__ f32x4_t bias4(const LinearParams& p, int col) {
  f32x4_t v = {0.f, 0.f, 0.f, 0.f};
  if (!p.bias || col >= p.n) return v;
  if (p.vec) {
    const u32x2_t b = *reinterpret_cast<const u32x2_t*>(p.bias + col);
    return f32x4_t{bf16_lo(b.x), bf16_hi(b.x), bf16_lo(b.y), bf16_hi(b.y)};
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < p.n) v[i] = bf16_to_f32(p.bias[col + i]);
  return v;
}

// A lane's sums (and, gated, those of the up rows): bias or silu(gate) * up in fp32, one
// rounding.
template <bool GLU>
__device__ __forceinline__ u32x2_t round4(f32x4_t sum, f32x4_t up, f32x4_t bias) {
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] = GLU ? silu(sum[i]) * up[i] : sum[i] + bias[i];
  return u32x2_t{cvt_pk_bf16(sum[0], sum[1]), cvt_pk_bf16(sum[2], sum[3])};
}
// They are columns col .. col + 3 of out's row m.
template <bool GLU>
__device__ __forceinline__ void store4(const LinearParams& p, int64_t m, int col, f32x4_t sum, f32x4_t up, f32x4_t bias) {
  uint16_t* const out = p.out + m * p.o_stride + col;
  const u32x2_t v = round4<GLU>(sum, up, bias);
  if (p.vec) {
    *reinterpret_cast<u32x2_t*>(out) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < p.n) out[i] = uint16_t(v[i / 2] >> (16 * (i & 1)));
}

// Slot of 16-byte chunk c in a staged row of 256 bytes: the 8 rows that an operand
// read touches together at one chunk fall on distinct banks.
__device__ __forceinline__ int chunk_slot(int r, int c) { return c ^ ((r & 7) << 1); }

constexpr int64_t kMaxRows = 1 << 22, kMaxN = 1 << 24, kMaxStride = 1 << 22;

// The rows that a workgroup of the few-row kernel takes at most.
constexpr int64_t few_group(bool mx) { return mx ? 64 : 32; }

// Whether the few-row kernel is the faster one in any case.  (Two blocks of bf16 rows along a long k
// are read by every one of its workgroups: 32 x 14,336 x 4,096 19.1 us, the blocks of
// 128 rows of W with k in parts 14.5; 32 x 4,096 x 4,096 7.6, 10.0.)
inline bool few(bool mx, int64_t rows, int64_t w_rows, int64_t k) {
  return mx ? rows <= 64 : rows <= 16 || (rows <= 32 && (w_rows > 4096 || k < 8192));
}
void launch_few(const LinearParams& p, bool glu, hipStream_t stream);
void launch_many(const LinearParams& p, bool glu, size_t room, hipStream_t stream);

}  // namespace mi::mx4

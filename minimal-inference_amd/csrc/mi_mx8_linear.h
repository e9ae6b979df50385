// What the launches of MXFP8 projections share: arguments and the end of a product.
#pragma once

#include "mi_mx8.h"

namespace mi::mx8 {

struct LinearParams {
  const char* x;
  int64_t x_stride;  // bytes
  const char* xs;
  int64_t xs_stride;
  const char* w;
  int64_t w_stride;
  const char* ws;
  int64_t ws_stride;
  const uint16_t* bias;  // null: none
  char* out;             // bf16, or codes where scales is not null
  int64_t o_stride;      // elements
  uint8_t* scales;
  int64_t s_stride;
  int64_t rows;
  int n, k;       // n: columns of out; with the gated product W holds n gate rows, then n up rows
  int w_rows;
  int slabs;
  f32x4_t* parts;   // sums of workgroups that share k
  int split_slabs;  // slabs that one of them takes
  bool vec;   // out and bias take 8-byte accesses,
  bool wide;  // out 16-byte ones
  float* sums;  // of the gated product: where gate's and, n columns on, up's sums go as they are; null: silu and out
  int64_t sums_stride;
};

// Columns col .. col + 3 of a row's gate and up sums in fp32; NT: stores that L2 need not keep.
template <bool NT = false>
__device__ __forceinline__ void store_sums(const LinearParams& p, int64_t m, int col, f32x4_t gate, f32x4_t up) {
  f32x4_t* const to = reinterpret_cast<f32x4_t*>(p.sums + m * p.sums_stride + col);
  f32x4_t* const to_up = reinterpret_cast<f32x4_t*>(p.sums + m * p.sums_stride + col + p.n);
  if constexpr (NT) {
    __builtin_nontemporal_store(gate, to);
    __builtin_nontemporal_store(up, to_up);
  } else {
    *to = gate;
    *to_up = up;
  }
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

// A lane's sums (and, gated, those of the up rows): bias or silu(gate) * up in fp32.
template <bool GLU>
__device__ __forceinline__ f32x4_t finish(f32x4_t sum, f32x4_t up, f32x4_t bias) {
#pragma unroll
  for (int i = 0; i < 4; ++i) sum[i] = GLU ? silu20(sum[i]) * up[i] : sum[i] + bias[i];
  return sum;
}
__device__ __forceinline__ u32x2_t round4(f32x4_t v) { return u32x2_t{cvt_pk_bf16(v[0], v[1]), cvt_pk_bf16(v[2], v[3])}; }
// Columns col .. col + 3 of out's row m in bf16, one rounding.
__device__ __forceinline__ void store4(const LinearParams& p, int64_t m, int col, f32x4_t sum) {
  uint16_t* const out = reinterpret_cast<uint16_t*>(p.out) + m * p.o_stride + col;
  const u32x2_t v = round4(sum);
  if (p.vec) {
    *reinterpret_cast<u32x2_t*>(out) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < p.n) out[i] = uint16_t(v[i / 2] >> (16 * (i & 1)));
}
__device__ __forceinline__ uint32_t magnitude4(f32x4_t v) {
  return max(max(magnitude(v[0]), magnitude(v[1])), max(magnitude(v[2]), magnitude(v[3])));
}
// A block's 32 columns from `first` on of out's row m in 8 bits: lane (g, n) holds columns
// 4 g .. 4 g + 3 (a) and 16 + 4 g .. (b) of row n.  All 64 lanes come here.
__device__ __forceinline__ void store_block(const LinearParams& p, int64_t m, bool in, int first, int g, f32x4_t a, f32x4_t b) {
  uint32_t top = max(magnitude4(a), magnitude4(b));
  top = max(top, uint32_t(lane_shuffle_i(int(top), (threadIdx.x & 63) ^ 16)));
  top = max(top, uint32_t(lane_shuffle_i(int(top), (threadIdx.x & 63) ^ 32)));
  const uint32_t byte = scale_byte(top);
  // two lanes change places, so that each holds eight columns
  const auto s = __builtin_amdgcn_permlane16_swap(to_codes(a[0], a[1], a[2], a[3], byte), to_codes(b[0], b[1], b[2], b[3], byte),
                                                  false, false);
  if (!in) return;
  *reinterpret_cast<u32x2_t*>(p.out + m * p.o_stride + first + (g & 1) * 16 + (g >> 1) * 8) = u32x2_t{s[0], s[1]};
  if (g == 0) p.scales[m * p.s_stride + first / kBlock] = uint8_t(byte);
}

// The rows that the few-row kernel takes.
constexpr int64_t kFewRows = 64;
constexpr int64_t kMaxRows = 1 << 22, kMaxN = 1 << 24, kMaxStride = 1 << 22;

// (rows at most kFewRows; `room` bytes for parts)
size_t few_workspace(bool glu, int64_t rows, int64_t n, int slabs, size_t room);
void launch_few(const LinearParams& p, bool glu, size_t room, hipStream_t stream);
// The sum of parts [part][half][row][columns in fours], and the end of the product.
void launch_combine(const LinearParams& p, bool glu, int parts, hipStream_t stream);

}  // namespace mi::mx8

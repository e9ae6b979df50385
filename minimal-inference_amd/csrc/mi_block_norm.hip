// The norms after a block and before the next one in one pass, for layers that
// normalise a block's output before it joins the residual stream:
//   s = x + scale * gate * (y * rsqrt(mean(y^2) + eps) * post)
//   x_out = bf16(s),  h = bf16(s * rsqrt(mean(s^2) + eps) * pre)
// in fp32, h from s before its rounding, one rounding per output.  gate: none, one
// value per channel, per row, or per element.
//
// Bound: HBM, 8 bytes per element (10 with a full gate), half of them writes: 18,240 x
// 4,096 107 us = 5.6 TB/s, where a copy of 1 GiB reaches 5.2.  One workgroup per row,
// one, two or four 16-byte chunks per thread; every load of the row is issued before anything
// is computed or stored, and the row stays in registers over both sums.
#include "mi_common.h"
#include "mi_overlap.h"

namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxHidden = 16384;
constexpr int64_t kMaxRows = 1 << 22;  // (a launch counts its threads in 32 bits)

struct BlockNormParams {
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* y;
  int64_t y_stride;
  const uint16_t* post;
  const uint16_t* pre;
  const uint16_t* gate;  // null: none
  int64_t g_stride;      // of rows; 0: the same for every row
  int g_column;          // 1: a value per column, 0: one per row
  uint16_t* x_out;
  int64_t xo_stride;
  uint16_t* h_out;
  int64_t h_stride;
  int hidden;
  float eps, scale;
};

// Sum over the workgroup, in wave order; every thread gets it.
__device__ __forceinline__ float block_sum(float v, float* red, int waves) {
  v = mi::wave_sum(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float sum = 0.f;
  for (int w = 0; w < waves; ++w) sum += red[w];
  return sum;
}

// CH chunks per thread.
template <int CH>
__global__ __launch_bounds__(kMaxThreads) void block_norm_kernel(BlockNormParams p) {
  __shared__ float red[2][kMaxThreads / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, nt = blockDim.x, nch = p.hidden / 8;
  uint4 xv[CH], yv[CH], gv[CH], pv[CH], nv[CH];
  float row_gate = p.scale;
  if (p.gate && !p.g_column) row_gate *= mi::bf16_to_f32(p.gate[row * p.g_stride]);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int ch = tid + c * nt;
    xv[c] = yv[c] = pv[c] = nv[c] = make_uint4(0u, 0u, 0u, 0u);
    gv[c] = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);  // ones
    if (ch < nch) {
      yv[c] = mi::load16_nt(p.y + row * p.y_stride + ch * 8);
      xv[c] = mi::load16_nt(p.x + row * p.x_stride + ch * 8);
      pv[c] = mi::load16(p.post + ch * 8);
      nv[c] = mi::load16(p.pre + ch * 8);
      if (p.gate && p.g_column) gv[c] = mi::load16(p.gate + row * p.g_stride + ch * 8);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t yw[4] = {yv[c].x, yv[c].y, yv[c].z, yv[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = mi::bf16_lo(yw[k]), b = mi::bf16_hi(yw[k]);
      ss = fmaf(a, a, ss);
      ss = fmaf(b, b, ss);
    }
  }
  const float by = rsqrtf(block_sum(ss, red[0], nt / 64) / float(p.hidden) + p.eps) * row_gate;
  float s[CH][8];
  ss = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t xw[4] = {xv[c].x, xv[c].y, xv[c].z, xv[c].w}, yw[4] = {yv[c].x, yv[c].y, yv[c].z, yv[c].w};
    const uint32_t gw[4] = {gv[c].x, gv[c].y, gv[c].z, gv[c].w}, pw[4] = {pv[c].x, pv[c].y, pv[c].z, pv[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = fmaf(mi::bf16_lo(yw[k]) * by, mi::bf16_lo(pw[k]) * mi::bf16_lo(gw[k]), mi::bf16_lo(xw[k]));
      const float b = fmaf(mi::bf16_hi(yw[k]) * by, mi::bf16_hi(pw[k]) * mi::bf16_hi(gw[k]), mi::bf16_hi(xw[k]));
      s[c][2 * k] = a;
      s[c][2 * k + 1] = b;
      ss = fmaf(a, a, ss);
      ss = fmaf(b, b, ss);
    }
  }
  const float bs = rsqrtf(block_sum(ss, red[1], nt / 64) / float(p.hidden) + p.eps);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int ch = tid + c * nt;
    if (ch >= nch) break;
    const uint32_t nw[4] = {nv[c].x, nv[c].y, nv[c].z, nv[c].w};
    uint32_t xw[4], hw[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = s[c][2 * k], b = s[c][2 * k + 1];
      xw[k] = mi::cvt_pk_bf16(a, b);
      hw[k] = mi::cvt_pk_bf16(a * bs * mi::bf16_lo(nw[k]), b * bs * mi::bf16_hi(nw[k]));
    }
    mi::store16(p.x_out + row * p.xo_stride + ch * 8, make_uint4(xw[0], xw[1], xw[2], xw[3]));
    mi::store16(p.h_out + row * p.h_stride + ch * 8, make_uint4(hw[0], hw[1], hw[2], hw[3]));
  }
}

}  // namespace

extern "C" int mi_post_norm_add_rms_norm(const void* x, int64_t x_stride, const void* y, int64_t y_stride,
                                         const void* post_weight, const void* weight, const void* gate,
                                         int64_t gate_row_stride, int32_t gate_per_column, void* x_out,
                                         int64_t x_out_stride, void* h_out, int64_t h_stride, int64_t rows,
                                         int32_t hidden, float eps, float scale, mi_stream_t stream) {
  mi::clear_error();
  if (rows < 0 || rows > kMaxRows || hidden <= 0 || hidden % 8 || hidden > kMaxHidden)
    return mi::fail(MI_ERR_INVALID, "post_norm_add_rms_norm: %lld rows (0..2^22), hidden %d (multiple of 8, <= %d)",
                    (long long)rows, hidden, kMaxHidden);
  if (rows == 0) return MI_OK;
  if (!x || !y || !post_weight || !weight || !x_out || !h_out)
    return mi::fail(MI_ERR_INVALID, "post_norm_add_rms_norm: null pointer argument");
  uintptr_t aligned = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) |
                      reinterpret_cast<uintptr_t>(post_weight) | reinterpret_cast<uintptr_t>(weight) |
                      reinterpret_cast<uintptr_t>(x_out) | reinterpret_cast<uintptr_t>(h_out);
  if (rows == 1) x_stride = y_stride = x_out_stride = h_stride = hidden;  // (nothing lies at a row stride)
  if (rows == 1 && gate) gate_row_stride = 0;
  int64_t strides = x_stride | y_stride | x_out_stride | h_stride;
  if (gate && gate_per_column) aligned |= reinterpret_cast<uintptr_t>(gate), strides |= gate_row_stride;
  if ((aligned & 15) || (strides & 7) || (reinterpret_cast<uintptr_t>(gate) & 1))
    return mi::fail(MI_ERR_INVALID, "post_norm_add_rms_norm: rows must be 16-byte aligned");
  if (x_out_stride < hidden || h_stride < hidden)
    return mi::fail(MI_ERR_INVALID, "post_norm_add_rms_norm: output row strides %lld, %lld for hidden %d",
                    (long long)x_out_stride, (long long)h_stride, hidden);
  // (a row's workgroup has read all of x, y and gate that it takes when it writes; the other
  // rows' have not, nor has anyone the weights)
  const int64_t width = int64_t(hidden) * 2;
  const mi::Rows xo = {x_out, x_out_stride * 2, rows, width}, ho = {h_out, h_stride * 2, rows, width};
  const mi::Rows in[] = {{x, x_stride * 2, rows, width}, {y, y_stride * 2, rows, width},
                         {gate, gate_row_stride * 2, gate ? rows : 0, gate_per_column ? width : 2}};
  const mi::Rows w[] = {{post_weight, 0, 1, width}, {weight, 0, 1, width}};
  bool meet = mi::rows_meet(xo, ho);
  for (const mi::Rows& r : in) meet = meet || mi::rows_meet(xo, r, true) || mi::rows_meet(ho, r, true);
  for (const mi::Rows& r : w) meet = meet || mi::rows_meet(xo, r) || mi::rows_meet(ho, r);
  if (meet)
    return mi::fail(MI_ERR_INVALID, "post_norm_add_rms_norm: an output overlaps the other, a weight or another row's input");
  BlockNormParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.x_stride = x_stride;
  p.y = static_cast<const uint16_t*>(y);
  p.y_stride = y_stride;
  p.post = static_cast<const uint16_t*>(post_weight);
  p.pre = static_cast<const uint16_t*>(weight);
  p.gate = static_cast<const uint16_t*>(gate);
  p.g_stride = gate_row_stride;
  p.g_column = gate_per_column;
  p.x_out = static_cast<uint16_t*>(x_out);
  p.xo_stride = x_out_stride;
  p.h_out = static_cast<uint16_t*>(h_out);
  p.h_stride = h_stride;
  p.hidden = hidden;
  p.eps = eps;
  p.scale = scale;
  // One chunk per thread up to 512 threads, then two and four (us, 32 x 8,192: 1,024
  // threads 4.6, 512 4.5; 5,000 x 16,384: 1,024 threads 148, 512 121, 256 with eight
  // chunks, which leave the registers, 314; 18,240 x 4,096: 512 threads 107, 256 109,
  // 128 110).
  const int chunks = hidden / 8, each = chunks <= kMaxThreads ? 1 : chunks <= 2 * kMaxThreads ? 2 : 4;
  const int threads = (chunks + 64 * each - 1) / (64 * each) * 64;
  const auto kernel = each == 1 ? block_norm_kernel<1> : each == 2 ? block_norm_kernel<2> : block_norm_kernel<4>;
  hipLaunchKernelGGL(kernel, dim3(uint32_t(rows)), dim3(threads), 0, static_cast<hipStream_t>(stream), p);
  return mi::check_launch("block_norm_kernel");
}

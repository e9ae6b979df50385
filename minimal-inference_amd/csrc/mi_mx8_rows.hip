// Rows in MXFP8: quantisation of bf16 rows, their return to bf16, and the residual sum
// with the root-mean-square norm that leaves 8-bit rows.
//
//   quantise : per block of 32 the least power of two u with max|x| <= 448 u, each code
//              the e4m3 value nearest to x / u (ties to even), scale byte log2 u + 127, at
//              least 0.  A block that holds an infinity or a NaN gets byte 255, the
//              format's NaN, and zero codes: all of it reads back as NaN.
//   add_rms  : x' = bf16(x + d), stored when asked; h = x' rsqrt(mean(x'^2) + eps) w, quantised.
//              The sum and the root are taken in 64 bits and the product x' w (exact in
//              fp32 where that holds it: weights within 2^+-60) times the root is rounded to odd, so that the codes are those of the exact
//              norm (in fp32 alone some 4e-7 of them fall on the other side of a border).
//
// Bound: HBM.  add_rms reads x and d once, writes x' and 1.03 bytes of h per element.
#include "mi_mx8.h"
#include "mi_overlap.h"

namespace {

using namespace mi::mx8;

constexpr int64_t kMaxRows = 1 << 22;

struct MatrixParams {
  const uint16_t* x;  // rows of bf16: read (quantise) or written (dequantise)
  uint16_t* y;
  int64_t stride;
  uint8_t* codes;
  int64_t c_stride;
  uint8_t* scales;
  int64_t s_stride;
  int64_t rows;
  int cols;
};

// Eight values of a lane, a block's by four neighbouring lanes: its 8 codes and byte.
__device__ __forceinline__ u32x2_t quantize8(const float (&v)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[j]));
  byte = scale_byte(max4(top));
  return u32x2_t{to_codes(v[0], v[1], v[2], v[3], byte), to_codes(v[4], v[5], v[6], v[7], byte)};
}

// A thread per 8 values; blockDim.y rows of blockDim.x chunks, the grid's second axis
// walks the rows.
__global__ __launch_bounds__(256) void quantize_kernel(MatrixParams p) {
  const int ch = int(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t step = int64_t(gridDim.y) * blockDim.y;
  for (int64_t row = int64_t(blockIdx.y) * blockDim.y + threadIdx.y; row < p.rows; row += step) {
    const bool in = ch * 8 < p.cols;  // (whole blocks: the lanes of a block agree)
    const uint4 v = in ? mi::load16_nt(p.x + row * p.stride + ch * 8) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[2 * j] = mi::bf16_lo(w[j]), f[2 * j + 1] = mi::bf16_hi(w[j]);
    uint32_t byte;
    const u32x2_t c = quantize8(f, byte);
    if (!in) continue;
    *reinterpret_cast<u32x2_t*>(p.codes + row * p.c_stride + ch * 8) = c;
    if ((ch & 3) == 0) p.scales[row * p.s_stride + ch / 4] = uint8_t(byte);
  }
}

// The same shape backwards.
__global__ __launch_bounds__(256) void dequantize_kernel(MatrixParams p) {
  const int ch = int(blockIdx.x) * blockDim.x + threadIdx.x;
  if (ch * 8 >= p.cols) return;
  const int64_t step = int64_t(gridDim.y) * blockDim.y;
  for (int64_t row = int64_t(blockIdx.y) * blockDim.y + threadIdx.y; row < p.rows; row += step) {
    const u32x2_t c = *reinterpret_cast<const u32x2_t*>(p.codes + row * p.c_stride + ch * 8);
    const float s = scale_f32(p.scales[row * p.s_stride + ch / 4]);
    const u32x2_t a = to_bf16(c.x, s), b = to_bf16(c.y, s);
    mi::store16(p.y + row * p.stride + ch * 8, make_uint4(a.x, a.y, b.x, b.y));
  }
}

constexpr int kMaxThreads = 512;
constexpr int kMaxHidden = 16384;

struct AddRmsParams {
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* delta;  // null: no sum
  int64_t d_stride;
  const uint16_t* weight;
  uint16_t* x_out;  // null: the sum is not stored
  int64_t xo_stride;
  uint8_t* codes;
  int64_t c_stride;
  uint8_t* scales;
  int64_t s_stride;
  int hidden;
  float eps;
};

// Sum over the wave in 64 bits; every lane gets it.
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u)), CTRL, 0xf, 0xf, false));
  const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u >> 32)), CTRL, 0xf, 0xf, false));
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) {
  v += dpp<mi::kDppQuadSwap1>(v);
  v += dpp<mi::kDppQuadSwap2>(v);
  v += dpp<mi::kDppRowHalfMirror>(v);
  v += dpp<mi::kDppRowMirror>(v);
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// a (hi + lo), rounded to odd: cut, with the last bit set where something was cut off.  Rounded
// again to the four bits of a code this is the exact product's rounding.  So is all of a (hi + lo) rounded to
// nearest (a hi alone may be an ulp off and pass the middle), unless that lies halfway between two codes, with 19
// zeros behind its leading bits.
__device__ __forceinline__ float nearest_product(float a, float hi, float lo) { return fmaf(a, hi, a * lo); }
__device__ __forceinline__ float product_to_odd(float a, float hi, float lo) {
  const float h = nearest_product(a, hi, lo), rest = fmaf(a, lo, fmaf(a, hi, -h));
  const uint32_t u = __float_as_uint(h);
  // (an infinity or a NaN leaves a NaN)
  return !(rest < 0.f || rest > 0.f) ? h : __uint_as_float((u - ((u ^ __float_as_uint(rest)) >> 31)) | 1u);
}

// One workgroup per row, CH 16-byte chunks per thread; every load of the row is issued
// before anything is computed, all of it is read before any of it is written (x_out may
// lie over x or delta), and the row stays in registers between the sum of squares and the codes.
template <int CH>
__global__ __launch_bounds__(kMaxThreads) void add_rms_kernel(AddRmsParams p) {
  __shared__ double red[kMaxThreads / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, nt = blockDim.x, nch = p.hidden / 8;
  uint4 xv[CH], dv[CH], wv[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int ch = tid + c * nt;
    xv[c] = dv[c] = wv[c] = make_uint4(0u, 0u, 0u, 0u);
    if (ch < nch) {
      xv[c] = mi::load16_nt(p.x + row * p.x_stride + ch * 8);
      if (p.delta) dv[c] = mi::load16_nt(p.delta + row * p.d_stride + ch * 8);
      wv[c] = mi::load16(p.weight + ch * 8);
    }
  }
  float v[CH][8];
  uint32_t xo[CH][4];
  double ss = 0.;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const uint32_t xw[4] = {xv[c].x, xv[c].y, xv[c].z, xv[c].w}, dw[4] = {dv[c].x, dv[c].y, dv[c].z, dv[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t o = xo[c][k] = p.delta ? mi::cvt_pk_bf16(mi::bf16_lo(xw[k]) + mi::bf16_lo(dw[k]), mi::bf16_hi(xw[k]) + mi::bf16_hi(dw[k]))
                                 : xw[k];
      const float a = mi::bf16_lo(o), b = mi::bf16_hi(o);
      v[c][2 * k] = a;
      v[c][2 * k + 1] = b;
      ss = fma(double(a), double(a), ss);
      ss = fma(double(b), double(b), ss);
    }
  }
  ss = wave_sum(ss);
  if ((tid & 63) == 0) red[tid >> 6] = ss;
  __syncthreads();
  double tot = 0.;
  for (int w = 0; w < nt / 64; ++w) tot += red[w];
  // 1 / sqrt(m) from an estimate and a step in 64 bits, of m's mantissa where fp32 does not hold m: the
  // row takes the power of two then
  double m = tot / p.hidden + p.eps;
  if (!(m > 0x1p-100 && m < 0x1p100) && m < 1e300) {
    const int e = (__builtin_amdgcn_frexp_exp(m) - 1) & ~1;
    m = ldexp(m, -e);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = ldexpf(v[c][k], -e / 2);
  }
  const double r0 = rsqrtf(float(m)), off = fma(-m * r0, r0, 1.);
  const double r = m < 1e300 ? fma(r0 * off, fma(0.375, off, 0.5), r0) : r0;  // (else 0 or NaN)
  const float hi = float(r), lo = float(r - double(hi));
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int ch = tid + c * nt;
    const uint32_t ww[4] = {wv[c].x, wv[c].y, wv[c].z, wv[c].w};
    if (ch >= nch) break;
    if (p.x_out)
      mi::store16(p.x_out + row * p.xo_stride + ch * 8, make_uint4(xo[c][0], xo[c][1], xo[c][2], xo[c][3]));
    float h[8];
    uint32_t zeros = ~0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t w16 = ww[k / 2];
      v[c][k] *= k % 2 ? mi::bf16_hi(w16) : mi::bf16_lo(w16);
      h[k] = nearest_product(v[c][k], hi, lo);
      zeros = min(zeros, __float_as_uint(h[k]) & 0x7ffffu);
    }
    if (zeros == 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) h[k] = product_to_odd(v[c][k], hi, lo);
    }
    uint32_t byte;
    const u32x2_t code = quantize8(h, byte);
    *reinterpret_cast<u32x2_t*>(p.codes + row * p.c_stride + ch * 8) = code;
    if ((ch & 3) == 0) p.scales[row * p.s_stride + ch / 4] = uint8_t(byte);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Checks of an MXFP8 matrix's parts.
int check_parts(const char* name, const void* codes, int64_t& c_stride, const void* scales, int64_t& s_stride, int64_t rows,
                int64_t cols) {
  if (!codes || !scales) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if (rows == 1) c_stride = cols, s_stride = cols / kBlock;  // (nothing lies at a row stride)
  if (!aligned16(codes) || (rows > 1 && c_stride % 16) || c_stride < cols || s_stride < cols / kBlock)
    return mi::fail(MI_ERR_INVALID, "%s: rows of codes must be 16-byte aligned; row strides %lld, %lld for %lld columns",
                    name, (long long)c_stride, (long long)s_stride, (long long)cols);
  return MI_OK;
}

int run_matrix(const char* name, bool quantize, const void* x, int64_t stride, void* codes, int64_t c_stride, void* scales,
               int64_t s_stride, int64_t rows, int64_t cols, mi_stream_t stream) {
  mi::clear_error();
  if (rows < 0 || rows > (int64_t(1) << 31) || cols <= 0 || cols % kBlock || cols > kMaxK)
    return mi::fail(MI_ERR_INVALID, "%s: %lld rows (0..2^31) of %lld columns (multiple of %d, at most %d)", name,
                    (long long)rows, (long long)cols, kBlock, kMaxK);
  if (rows == 0) return MI_OK;
  if (!x) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if (int rc = check_parts(name, codes, c_stride, scales, s_stride, rows, cols)) return rc;
  if (rows == 1) stride = cols;
  if (!aligned16(x) || stride % 8 || stride < cols)
    return mi::fail(MI_ERR_INVALID, "%s: rows must be 16-byte aligned, row stride at least the columns", name);
  // (rows are read by one workgroup while others write theirs)
  const mi::Rows bf = {x, stride * 2, rows, cols * 2}, cd = {codes, c_stride, rows, cols},
                 sc = {scales, s_stride, rows, cols / kBlock};
  if (mi::rows_meet(bf, cd) || mi::rows_meet(bf, sc) || mi::rows_meet(cd, sc))
    return mi::fail(MI_ERR_INVALID, "%s: an output overlaps an input or the other output", name);
  MatrixParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.y = static_cast<uint16_t*>(const_cast<void*>(x));
  p.stride = stride;
  p.codes = static_cast<uint8_t*>(codes);
  p.c_stride = c_stride;
  p.scales = static_cast<uint8_t*>(scales);
  p.s_stride = s_stride;
  p.rows = rows;
  p.cols = int(cols);
  // rows of up to a workgroup's chunks share one (a row's chunks in whole blocks of four lanes)
  const int chunks = int(cols / 8), bx = chunks >= 256 ? 256 : chunks, by = 256 / bx;
  const int64_t y = (rows + by - 1) / by;
  const dim3 grid(uint32_t((chunks + bx - 1) / bx), uint32_t(y < 65535 ? y : 65535));
  hipLaunchKernelGGL(quantize ? quantize_kernel : dequantize_kernel, grid, dim3(bx, by), 0, static_cast<hipStream_t>(stream), p);
  return mi::check_launch(name);
}

}  // namespace

extern "C" int mi_mxfp8_quantize(const void* x, int64_t x_stride, void* codes, int64_t codes_stride, void* scales,
                                 int64_t scales_stride, int64_t rows, int64_t cols, mi_stream_t stream) {
  return run_matrix("mxfp8_quantize", true, x, x_stride, codes, codes_stride, scales, scales_stride, rows, cols, stream);
}

extern "C" int mi_mxfp8_dequantize(const void* codes, int64_t codes_stride, const void* scales, int64_t scales_stride,
                                   void* out, int64_t out_stride, int64_t rows, int64_t cols, mi_stream_t stream) {
  return run_matrix("mxfp8_dequantize", false, out, out_stride, const_cast<void*>(codes), codes_stride,
                    const_cast<void*>(scales), scales_stride, rows, cols, stream);
}

extern "C" int mi_add_rms_norm_mxfp8(const void* x, int64_t x_stride, const void* delta, int64_t delta_stride,
                                     const void* weight, void* x_out, int64_t x_out_stride, void* codes,
                                     int64_t codes_stride, void* scales, int64_t scales_stride, int64_t rows,
                                     int32_t hidden, float eps, mi_stream_t stream) {
  const char* const name = "add_rms_norm_mxfp8";
  mi::clear_error();
  if (rows < 0 || rows > kMaxRows || hidden <= 0 || hidden % kBlock || hidden > kMaxHidden)
    return mi::fail(MI_ERR_INVALID, "%s: %lld rows (0..2^22), hidden %d (multiple of %d, at most %d)", name, (long long)rows,
                    hidden, kBlock, kMaxHidden);
  if (rows == 0) return MI_OK;
  if (!x || !weight) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if (int rc = check_parts(name, codes, codes_stride, scales, scales_stride, rows, hidden)) return rc;
  if (rows == 1) x_stride = x_out_stride = hidden, delta_stride = hidden;
  if (!delta) delta_stride = 0;
  if (!x_out) x_out_stride = 0;
  if (!aligned16(x) || !aligned16(delta) || !aligned16(weight) || !aligned16(x_out) ||
      ((x_stride | delta_stride | x_out_stride) & 7))
    return mi::fail(MI_ERR_INVALID, "%s: rows must be 16-byte aligned", name);
  if (x_out && x_out_stride < hidden)
    return mi::fail(MI_ERR_INVALID, "%s: output row stride %lld for hidden %d", name, (long long)x_out_stride, hidden);
  // (a row's workgroup has read its x and delta when it writes; the other rows' have not, nor
  // has anyone the weight)
  const int64_t width = int64_t(hidden) * 2;
  const mi::Rows out[] = {{x_out, x_out_stride * 2, x_out ? rows : 0, width},
                          {codes, codes_stride, rows, hidden},
                          {scales, scales_stride, rows, hidden / kBlock}};
  const mi::Rows in[] = {{x, x_stride * 2, rows, width}, {delta, delta_stride * 2, delta ? rows : 0, width}};
  const mi::Rows w = {weight, 0, 1, width};
  bool meet = mi::rows_meet(out[0], out[1]) || mi::rows_meet(out[0], out[2]) || mi::rows_meet(out[1], out[2]);
  for (const mi::Rows& o : out) {
    meet = meet || mi::rows_meet(o, w);
    for (const mi::Rows& r : in) meet = meet || mi::rows_meet(o, r, true);
  }
  if (meet) return mi::fail(MI_ERR_INVALID, "%s: an output overlaps another, the weight or another row's input", name);
  AddRmsParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.x_stride = x_stride;
  p.delta = static_cast<const uint16_t*>(delta);
  p.d_stride = delta_stride;
  p.weight = static_cast<const uint16_t*>(weight);
  p.x_out = static_cast<uint16_t*>(x_out);
  p.xo_stride = x_out_stride;
  p.codes = static_cast<uint8_t*>(codes);
  p.c_stride = codes_stride;
  p.scales = static_cast<uint8_t*>(scales);
  p.s_stride = scales_stride;
  p.hidden = hidden;
  p.eps = eps;
  const int chunks = hidden / 8, each = chunks <= kMaxThreads ? 1 : chunks <= 2 * kMaxThreads ? 2 : 4;
  const int threads = (chunks + 64 * each - 1) / (64 * each) * 64;
  const auto kernel = each == 1 ? add_rms_kernel<1> : each == 2 ? add_rms_kernel<2> : add_rms_kernel<4>;
  hipLaunchKernelGGL(kernel, dim3(uint32_t(rows)), dim3(threads), 0, static_cast<hipStream_t>(stream), p);
  return mi::check_launch("add_rms_norm_mxfp8");
}

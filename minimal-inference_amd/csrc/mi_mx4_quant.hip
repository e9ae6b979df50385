// MXFP4 quantisation, its return to bf16, and the exchange with row-major codes
// (the layout of checkpoints: codes [rows][k / 2], scale bytes [rows][k / 32]).
//
//   quantise: per block of 32, e = max(floor(log2 max|x|) - 2, -127), each code the
//             e2m1 value nearest to x / 2^e (ties to the even code, at most 6), scale
//             byte e + 127.  A block that holds an infinity or a NaN gets byte 255,
//             the format's NaN, and zero codes: all of it reads back as NaN.
//
// Bound: HBM.  A workgroup takes 16 rows x 512 k, a wave one slab of 128 k of it in
// four loads of 4 rows x 256 contiguous bytes; a block is four neighbouring lanes,
// whose maximum takes two lane swaps, and their four dwords of codes are the 16
// bytes of the block's place in the tile.
#include "mi_mx4.h"

namespace {

using namespace mi::mx4;

constexpr int kWaves = 4;
typedef __attribute__((ext_vector_type(2))) __bf16 pair_t;

struct MatrixParams {
  const uint16_t* x;  // rows of bf16: read (quantise) or written (dequantise)
  uint16_t* y;
  int64_t stride;
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows;
  int cols, slabs, quads;
};

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
  return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xf, 0xf, false)));
}

__global__ __launch_bounds__(64 * kWaves) void quantize_kernel(MatrixParams p) {
  __shared__ uint8_t scale[kQuadBytes];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t rt = blockIdx.y + int64_t(blockIdx.z) * gridDim.y;
  if (rt >= row_tiles(p.rows)) return;
  const int q = blockIdx.x, slab = 4 * q + w;
  const int c = lane & 15, r4 = lane >> 4;  // chunk of 8 values, row of four
  const int col = slab * kSlab + c * 8;
  uint4 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = rt * kTileRows + 4 * i + r4;
    v[i] = row < p.rows && col < p.cols ? mi::load16_nt(p.x + row * p.stride + col) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 4 * i + r4;
    const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    // magnitudes of bf16 compare as whole numbers
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, max(x[j] & 0x7fffu, x[j] >> 16 & 0x7fffu));
    top = max_dpp<mi::kDppQuadSwap2>(max_dpp<mi::kDppQuadSwap1>(top));
    const uint32_t field = top >> 7;  // 0: below 2^-126, where e is at its least
    const bool nan = field == 255;
    const uint32_t byte = nan ? 255u : max(field, 2u) - 2u;
    const float s = scale_f32(byte);
    uint32_t code = 0;
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(pair_t, x[0]), s, 0);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(pair_t, x[1]), s, 1);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(pair_t, x[2]), s, 2);
    code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(pair_t, x[3]), s, 3);
    if (nan) code = 0;
    const int at = row + 16 * (c >> 2);  // the lane of the tile that holds the block
    if (slab < p.slabs)
      *reinterpret_cast<uint32_t*>(p.codes + (rt * p.slabs + slab) * kTileBytes + at * 16 + (c & 3) * 4) = code;
    if ((c & 3) == 0) scale[at * 4 + w] = uint8_t(byte);
  }
  __syncthreads();
  if (threadIdx.x < 64)
    reinterpret_cast<uint32_t*>(p.scales + (rt * p.quads + q) * kQuadBytes)[lane] =
        reinterpret_cast<const uint32_t*>(scale)[lane];
}

// The same shape backwards: each lane turns four bytes of codes into 16 of bf16.
__global__ __launch_bounds__(64 * kWaves) void dequantize_kernel(MatrixParams p) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t rt = blockIdx.y + int64_t(blockIdx.z) * gridDim.y;
  const int q = blockIdx.x, slab = 4 * q + w;
  const int c = lane & 15, r4 = lane >> 4;
  const int col = slab * kSlab + c * 8;
  if (rt >= row_tiles(p.rows) || col >= p.cols) return;
  uint32_t code[4], byte[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = 4 * i + r4 + 16 * (c >> 2);
    code[i] = *reinterpret_cast<const uint32_t*>(p.codes + (rt * p.slabs + slab) * kTileBytes + at * 16 + (c & 3) * 4);
    byte[i] = p.scales[(rt * p.quads + q) * kQuadBytes + at * 4 + w];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = rt * kTileRows + 4 * i + r4;
    if (row < p.rows)
      mi::store16(p.y + row * p.stride + col, __builtin_bit_cast(uint4, to_bf16(code[i], scale_f32(byte[i]))));
  }
}

struct PackParams {
  uint8_t* row_codes;   // [rows][k / 2]
  uint8_t* row_scales;  // [rows][k / 32]
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows;
  int cols, slabs, quads;
};

// One thread per block of 32 (16 bytes of codes); done once per weight.  A wave
// takes four rows x 16 blocks, so the row-major side moves 256-byte runs.
template <bool PACK>
__global__ __launch_bounds__(256) void pack_kernel(PackParams p) {
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t rt = blockIdx.y + int64_t(blockIdx.z) * gridDim.y;
  if (rt >= row_tiles(p.rows)) return;
  const int q = blockIdx.x, row = 4 * w + (lane >> 4), b = lane & 15;  // block b of the four slabs
  const int slab = 4 * q + (b >> 2), at = row + 16 * (b & 3);
  const int64_t r = rt * kTileRows + row;
  const int64_t blocks = p.cols / kBlock, block = int64_t(q) * 16 + b;
  const bool in = r < p.rows && block < blocks;
  uint8_t* const tile = p.codes + (rt * p.slabs + slab) * kTileBytes + at * 16;
  uint8_t* const scale = p.scales + (rt * p.quads + q) * kQuadBytes + at * 4 + (b >> 2);
  if constexpr (PACK) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (in) v = mi::load16(p.row_codes + (r * blocks + block) * 16);
    if (slab < p.slabs) mi::store16(tile, v);
    *scale = in ? p.row_scales[r * blocks + block] : 0;
  } else if (in) {
    mi::store16(p.row_codes + (r * blocks + block) * 16, mi::load16(tile));
    p.row_scales[r * blocks + block] = *scale;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_shape(const char* name, int64_t rows, int64_t cols) {
  if (rows < 0 || rows > (int64_t(1) << 31) || cols <= 0 || cols % kBlock || cols > kMaxK)
    return mi::fail(MI_ERR_INVALID, "%s: %lld rows (0..2^31) of %lld columns (multiple of %d, at most %d)", name,
                    (long long)rows, (long long)cols, kBlock, kMaxK);
  return MI_OK;
}

dim3 tile_grid(int64_t rows, int64_t cols) {
  const int64_t rt = row_tiles(rows), y = rt < 32768 ? rt : 32768;
  return dim3(uint32_t(quads(cols)), uint32_t(y), uint32_t((rt + y - 1) / y));
}

int run_matrix(const char* name, bool quantize, const void* x, int64_t stride, void* codes, void* scales, int64_t rows,
               int64_t cols, mi_stream_t stream) {
  mi::clear_error();
  if (int rc = check_shape(name, rows, cols)) return rc;
  if (rows == 0) return MI_OK;
  if (rows == 1) stride = cols;  // (nothing lies at a row stride)
  if (!x || !codes || !scales) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if (!aligned16(x) || !aligned16(codes) || !aligned16(scales) || stride % 8 || stride < cols)
    return mi::fail(MI_ERR_INVALID, "%s: rows, codes and scales must be 16-byte aligned, row stride at least the columns",
                    name);
  MatrixParams p;
  p.x = static_cast<const uint16_t*>(x);
  p.y = static_cast<uint16_t*>(const_cast<void*>(x));
  p.stride = stride;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  p.rows = rows;
  p.cols = int(cols);
  p.slabs = int(slabs(cols));
  p.quads = int(quads(cols));
  hipLaunchKernelGGL(quantize ? quantize_kernel : dequantize_kernel, tile_grid(rows, cols), dim3(64 * kWaves), 0,
                     static_cast<hipStream_t>(stream), p);
  return mi::check_launch(name);
}

int run_pack(const char* name, bool pack, const void* row_codes, const void* row_scales, const void* codes,
             const void* scales, int64_t rows, int64_t cols, mi_stream_t stream) {
  mi::clear_error();
  if (int rc = check_shape(name, rows, cols)) return rc;
  if (rows == 0) return MI_OK;
  if (!row_codes || !row_scales || !codes || !scales) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if (!aligned16(row_codes) || !aligned16(codes) || !aligned16(scales))
    return mi::fail(MI_ERR_INVALID, "%s: codes must be 16-byte aligned", name);
  PackParams p;
  p.row_codes = static_cast<uint8_t*>(const_cast<void*>(row_codes));
  p.row_scales = static_cast<uint8_t*>(const_cast<void*>(row_scales));
  p.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
  p.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  p.rows = rows;
  p.cols = int(cols);
  p.slabs = int(slabs(cols));
  p.quads = int(quads(cols));
  hipLaunchKernelGGL(pack ? pack_kernel<true> : pack_kernel<false>, tile_grid(rows, cols), dim3(256), 0,
                     static_cast<hipStream_t>(stream), p);
  return mi::check_launch(name);
}

}  // namespace

extern "C" size_t mi_mxfp4_codes_size(int64_t rows, int64_t cols) {
  if (check_shape("mxfp4_codes_size", rows, cols)) return 0;
  return size_t(row_tiles(rows)) * size_t(slabs(cols)) * kTileBytes;
}

extern "C" size_t mi_mxfp4_scales_size(int64_t rows, int64_t cols) {
  if (check_shape("mxfp4_scales_size", rows, cols)) return 0;
  return size_t(row_tiles(rows)) * size_t(quads(cols)) * kQuadBytes;
}

extern "C" int mi_mxfp4_quantize(const void* x, int64_t x_stride, void* codes, void* scales, int64_t rows,
                                 int64_t cols, mi_stream_t stream) {
  return run_matrix("mxfp4_quantize", true, x, x_stride, codes, scales, rows, cols, stream);
}

extern "C" int mi_mxfp4_dequantize(const void* codes, const void* scales, void* out, int64_t out_stride, int64_t rows,
                                   int64_t cols, mi_stream_t stream) {
  return run_matrix("mxfp4_dequantize", false, out, out_stride, const_cast<void*>(codes), const_cast<void*>(scales),
                    rows, cols, stream);
}

extern "C" int mi_mxfp4_pack(const void* row_codes, const void* row_scales, void* codes, void* scales, int64_t rows,
                             int64_t cols, mi_stream_t stream) {
  return run_pack("mxfp4_pack", true, row_codes, row_scales, codes, scales, rows, cols, stream);
}

extern "C" int mi_mxfp4_unpack(const void* codes, const void* scales, void* row_codes, void* row_scales, int64_t rows,
                               int64_t cols, mi_stream_t stream) {
  return run_pack("mxfp4_unpack", false, row_codes, row_scales, codes, scales, rows, cols, stream);
}

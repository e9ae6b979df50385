// Projections of many rows with an MXFP4 weight (prompts): out = x W^T (+ bias) or
// silu(x Wg^T) * (x Wu^T), fp32 accumulation and one rounding; x bf16 or MXFP4.
//
// Bound: the matrix instructions.  A workgroup of WM x WN waves owns a block of out;
// per slab of 128 k its tiles of W and of x go straight from memory to LDS (one of two
// buffers, the next slab's while this one is multiplied) and from there, as operands,
// to the waves.  MXFP4 tiles are operands as they lie; the codes of W become bf16 in
// registers, exactly, where x is bf16, whose rows are staged with permuted chunks.
#include "mi_mx4_linear.h"

namespace mi::mx4 {
namespace {

__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t rs, lds_t* dst, int voffset) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, voffset, 0, 0, 0);
#endif
}

// MB blocks of 16 rows of x and NT tiles of W per wave.
template <int WM, int WN, int MB, int NT, bool MX, bool GLU>
__global__ __launch_bounds__(64 * WM * WN) void many_kernel(LinearParams p) {
  constexpr int WAVES = WM * WN, HALVES = GLU ? 2 : 1;
  constexpr int XBLK = MX ? kTileBytes : 16 * kSlab * 2;  // 16 rows of x of a slab
  constexpr int BM = WM * MB * 16, TILES = WN * NT, COLS = TILES * 16 / HALVES;
  constexpr int XBYTES = WM * MB * XBLK, STAGE = XBYTES + TILES * kTileBytes;
  constexpr int XLOADS = XBYTES / 1024 / WAVES, WLOADS = TILES / WAVES;
  static_assert(XBYTES / 1024 % WAVES == 0 && TILES % WAVES == 0 && NT % HALVES == 0, "even shares");
  __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
  lds_t* const lds = (lds_t*)smem;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int wm = w / WN, wn = w % WN;
  const int g = lane >> 4, n = lane & 15;
  const int col0 = int(blockIdx.x) * COLS;
  const int64_t m0 = int64_t(blockIdx.y) * BM;
  const int rows = int(min(int64_t(BM), p.rows - m0));

  const char *wbase[HALVES], *sbase[HALVES];
  int wsize[HALVES], ssize[HALVES];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
    const int tile = (h * p.n + col0) / kTileRows, tiles = min(TILES / HALVES + 1, p.w_tiles - tile);
    wbase[h] = p.w + int64_t(tile) * p.slabs * kTileBytes;
    sbase[h] = p.ws + int64_t(tile) * p.quads * kQuadBytes;
    wsize[h] = tiles * p.slabs * kTileBytes;
    ssize[h] = tiles * p.quads * kQuadBytes;
  }
  auto row_of = [&](int t) {  // tile t of the workgroup's, this lane's row of W
    const int base = t % HALVES * p.n + col0;
    return lane_row(p, base, base + t / HALVES * 16 + n, g);
  };
  int wv[WLOADS], xv[XLOADS], wsv[NT];
#pragma unroll
  for (int i = 0; i < WLOADS; ++i) wv[i] = row_of(w * WLOADS + i).codes;
#pragma unroll
  for (int t = 0; t < NT; ++t) wsv[t] = row_of(wn * NT + t).scales;
  const char* xbase;
  const char* xsbase = nullptr;
  int xsize, xssize = 0;
  if constexpr (MX) {
    const int tiles = (rows + 15) / 16;
    xbase = p.x + m0 / 16 * p.slabs * kTileBytes;
    xsbase = p.xs + m0 / 16 * p.quads * kQuadBytes;
    xsize = tiles * p.slabs * kTileBytes;
    xssize = tiles * p.quads * kQuadBytes;
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) xv[i] = (w * XLOADS + i) * p.slabs * kTileBytes + lane * 16;
  } else {
    const int stride = int(p.x_stride * 2);
    xbase = p.x + m0 * p.x_stride * 2;
    xsize = (rows - 1) * stride + p.k * 2;
    // load i: 4 rows, lane l slot l % 16 of row l / 16.  A row's permutation depends
    // on the row modulo 8: one chunk for even i, one for odd (two chunks to test)
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) {
      const int row = (w * XLOADS + i) * 4 + (lane >> 4);
      xv[i] = row * stride + chunk_slot(row, lane & 15) * 16;
    }
  }
  auto load = [&](int slab, int buf) {
    lds_t* const stage = lds + buf * STAGE;
    const int off = MX ? slab * kTileBytes : slab * kSlab * 2;
    const __amdgpu_buffer_rsrc_t rx = buffer(xbase + off, xsize - off);
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) {
      int v = xv[i];
      if constexpr (!MX) {
        const int row = (w * XLOADS + i) * 4 + (lane >> 4);
        if (off + chunk_slot(row, lane & 15) * 16 >= p.k * 2) v = 0x7ffffff0;  // past the row's end lies the next row
      }
      lds_dma16(rx, stage + (w * XLOADS + i) * 1024, v);
    }
#pragma unroll
    for (int i = 0; i < WLOADS; ++i) {
      const int h = (w * WLOADS + i) % HALVES;
      lds_dma16(buffer(wbase[h] + slab * kTileBytes, wsize[h] - slab * kTileBytes),
                stage + XBYTES + (w * WLOADS + i) * kTileBytes, wv[i]);
    }
  };
  uint32_t wscale[NT], xscale[MB], wnext[NT], xnext[MB];
  auto load_scales = [&](int quad) {
    const int off = quad * kQuadBytes;
#pragma unroll
    for (int t = 0; t < NT; ++t)
      wnext[t] = __builtin_amdgcn_raw_buffer_load_b32(buffer(sbase[t % HALVES] + off, ssize[t % HALVES] - off), wsv[t], 0, 0);
    if constexpr (MX) {
#pragma unroll
      for (int b = 0; b < MB; ++b)
        xnext[b] = __builtin_amdgcn_raw_buffer_load_b32(buffer(xsbase + off, xssize - off),
                                                        (wm * MB + b) * p.quads * kQuadBytes + lane * 4, 0, 0);
    }
  };

  f32x4_t acc[NT][MB];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[t][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  int ro[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) ro[s] = n * 256 + chunk_slot(n, 4 * g + s) * 16;

  load(0, 0);
  load_scales(0);
  for (int slab = 0; slab < p.slabs; ++slab) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
    if ((slab & 3) == 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t) wscale[t] = wnext[t];
#pragma unroll
      for (int b = 0; b < MB; ++b) xscale[b] = xnext[b];
    }
    if (slab + 1 < p.slabs) {
      load(slab + 1, (slab + 1) & 1);
      if ((slab & 3) == 3) load_scales((slab + 1) >> 2);
    }
    const lds_t* const xl = lds + (slab & 1) * STAGE + wm * MB * XBLK;
    const lds_t* const wl = lds + (slab & 1) * STAGE + XBYTES + wn * NT * kTileBytes + lane * 16;
    const int shift = 8 * (slab & 3);
    u32x4_t a[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) a[t] = lds_load16(wl + t * kTileBytes);
    if constexpr (MX) {
      u32x4_t x[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) x[b] = lds_load16(xl + b * XBLK + lane * 16);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b)
          acc[t][b] = mfma_fp4<0, 0>(a[t], wscale[t] >> shift, x[b], xscale[b] >> shift, acc[t][b]);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        bf16x8_t x[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) x[b] = __builtin_bit_cast(bf16x8_t, lds_load16(xl + b * XBLK + ro[s]));
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const bf16x8_t v = to_bf16(a[t][s], scale_f32(wscale[t] >> shift & 255u));
#pragma unroll
          for (int b = 0; b < MB; ++b) acc[t][b] = mfma_16x16x32_bf16(v, x[b], acc[t][b]);
        }
      }
    }
  }

  // Lane (g, n) holds columns 4 g .. 4 g + 3 of a tile for row n of a block.
#pragma unroll
  for (int t = 0; t < NT; t += HALVES) {
    const int col = col0 + (wn * NT + t) / HALVES * 16 + 4 * g;
    if (col >= p.n) continue;
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const int m = (wm * MB + b) * 16 + n;
      if (m < rows) store4<GLU>(p, m0 + m, col, acc[t][b], acc[t + HALVES - 1][b]);
    }
  }
}

template <bool MX, bool GLU>
void launch(const LinearParams& p, hipStream_t stream) {
  const int cols = 128 / (GLU ? 2 : 1);
  const dim3 grid((p.n + cols - 1) / cols, uint32_t((p.rows + 127) / 128));
  hipLaunchKernelGGL((many_kernel<2, 2, 4, 4, MX, GLU>), grid, dim3(256), 0, stream, p);
}

}  // namespace

void launch_many(const LinearParams& p, bool glu, hipStream_t stream) {
  if (p.xs) glu ? launch<true, true>(p, stream) : launch<true, false>(p, stream);
  else glu ? launch<false, true>(p, stream) : launch<false, false>(p, stream);
}

}  // namespace mi::mx4

extern "C" int mi_linear_mxfp4(const void* x, int64_t x_stride, const void* x_scales, const void* codes,
                               const void* scales, const void* bias, void* out, int64_t out_stride, int64_t rows,
                               int64_t n, int64_t k, int32_t silu, mi_stream_t stream) {
  using namespace mi::mx4;
  mi::clear_error();
  constexpr int64_t kMaxRows = 1 << 22, kMaxN = 1 << 24, kMaxStride = 1 << 22;
  if (rows < 0 || rows > kMaxRows || n <= 0 || n > kMaxN || k <= 0 || k % kBlock || k > kMaxK)
    return mi::fail(MI_ERR_INVALID, "linear_mxfp4: rows %lld (0..2^22), n %lld (1..2^24), k %lld (multiple of %d, at most %d)",
                    (long long)rows, (long long)n, (long long)k, kBlock, kMaxK);
  if (silu && bias) return mi::fail(MI_ERR_INVALID, "linear_mxfp4: no bias with the gated product");
  if (rows == 0) return MI_OK;
  if (!x || !codes || !scales || !out) return mi::fail(MI_ERR_INVALID, "linear_mxfp4: null pointer argument");
  const uintptr_t aligned = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) |
                            reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(x_scales);
  if ((aligned & 15) || ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 1) ||
      (!x_scales && x_stride % 8))
    return mi::fail(MI_ERR_INVALID, "linear_mxfp4: x rows, codes and scales must be 16-byte aligned");
  if (out_stride < n || (!x_scales && (x_stride < k || x_stride > kMaxStride)))
    return mi::fail(MI_ERR_INVALID, "linear_mxfp4: row strides %lld (at most 2^22) / %lld for k %lld, n %lld",
                    (long long)x_stride, (long long)out_stride, (long long)k, (long long)n);
  LinearParams p;
  p.x = static_cast<const char*>(x);
  p.x_stride = x_stride;
  p.xs = static_cast<const char*>(x_scales);
  p.w = static_cast<const char*>(codes);
  p.ws = static_cast<const char*>(scales);
  p.bias = static_cast<const uint16_t*>(bias);
  p.out = static_cast<uint16_t*>(out);
  p.o_stride = out_stride;
  p.rows = rows;
  p.n = int(n);
  p.k = int(k);
  p.slabs = int(slabs(k));
  p.quads = int(quads(k));
  p.w_tiles = int(row_tiles(silu ? 2 * n : n));
  p.vec = n % 4 == 0 && out_stride % 4 == 0 &&
          ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 7) == 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows <= kFewRows) launch_few(p, silu != 0, s);
  else launch_many(p, silu != 0, s);
  return mi::check_launch("linear_mxfp4");
}

// Projections of few rows with both operands in MXFP8 (decode steps): out = x W^T (+ bias)
// or silu(x Wg^T) * (x Wu^T), fp32 accumulation and one rounding.
//
// Bound: HBM, the one read of W, 1.03 bytes per weight.  A workgroup of 4 or 8 waves owns
// 16 R rows of W over all of k and the waves split k: wave w takes the slabs of 128 k
// w, w + WAVES, ...  A lane's two chunks of a slab and its scale byte go from memory to
// the matrix instructions through registers alone, D slabs ahead.  The waves meet once, at
// the end, where their accumulators are added in wave order: the result does not depend on
// timing.  More rows than the accumulators hold (64) are groups of their own workgroups, which read
// W again, from the caches.
#include <algorithm>

#include "mi_mx8_linear.h"

namespace mi::mx8 {
namespace {

template <int R, int MB, int D, bool GLU, bool OUT8, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(LinearParams p) {
  constexpr int HALVES = GLU ? 2 : 1, COLS = 16 * R / HALVES;
  static_assert(R % HALVES == 0 && (!OUT8 || COLS % kBlock == 0), "gate and up tiles in pairs, whole blocks");
  __shared__ __attribute__((aligned(16))) char smem[WAVES * R * MB * 1024];
  lds_t* const lds = (lds_t*)smem;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const int col0 = int(blockIdx.x) * COLS;
  const int steps = (p.slabs - w + WAVES - 1) / WAVES;  // this wave's slabs: w, w + WAVES, ...
  const int blocks = p.k / kBlock;

  // tile r of W's rows, and a lane's place in it
  const char *wbase[HALVES], *sbase[HALVES];
  int wsize[HALVES], ssize[HALVES], wv[R], sv[R];
  const int wstride = int(p.w_stride), wsstride = int(p.ws_stride);
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
    const int row = h * p.n + col0, rows = min(COLS, p.w_rows - row);
    wbase[h] = p.w + row * p.w_stride;
    sbase[h] = p.ws + row * p.ws_stride;
    wsize[h] = (rows - 1) * wstride + p.k;
    ssize[h] = (rows - 1) * wsstride + blocks;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    wv[r] = (r / HALVES * 16 + n) * wstride + g * 16;
    sv[r] = (r / HALVES * 16 + n) * wsstride + g;
  }
  const int64_t m0 = int64_t(blockIdx.y) * (16 * MB);
  const int rows = int(min(p.rows - m0, int64_t(16 * MB))), xstride = int(p.x_stride), xsstride = int(p.xs_stride);
  const char* const x = p.x + m0 * p.x_stride;
  const char* const xs = p.xs + m0 * p.xs_stride;
  const int xsize = (rows - 1) * xstride + p.k, xssize = (rows - 1) * xsstride + blocks;

  u32x4_t wr[D][R][2], xr[D][MB][2];
  uint32_t wscale[D][R], xscale[D][MB];
  auto load = [&](int d, int step) {
    const int slab = step * WAVES + w, off = slab * kSlab, soff = slab * (kSlab / kBlock);
    const bool ok = step < steps;
    __amdgpu_buffer_rsrc_t rw[HALVES], rs[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      rw[h] = buffer(wbase[h] + off, ok ? wsize[h] - off : 0);
      rs[h] = buffer(sbase[h] + soff, ok ? ssize[h] - soff : 0);
    }
    // past a row's end lies the next row: out of range instead
    const bool lo = off + g * 16 < p.k, hi = off + 64 + g * 16 < p.k, sc = soff + g < blocks;
    // W is read once: non-temporal
#pragma unroll
    for (int r = 0; r < R; ++r) {
      wr[d][r][0] = __builtin_amdgcn_raw_buffer_load_b128(rw[r % HALVES], lo ? wv[r] : kOutOfRange, 0, kCacheNT);
      wr[d][r][1] = __builtin_amdgcn_raw_buffer_load_b128(rw[r % HALVES], hi ? wv[r] + 64 : kOutOfRange, 0, kCacheNT);
      wscale[d][r] = uint8_t(__builtin_amdgcn_raw_buffer_load_b8(rs[r % HALVES], sc ? sv[r] : kOutOfRange, 0, 0));
    }
    const __amdgpu_buffer_rsrc_t rx = buffer(x + off, ok ? xsize - off : 0);
    const __amdgpu_buffer_rsrc_t rxs = buffer(xs + soff, ok ? xssize - soff : 0);
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const int v = (b * 16 + n) * xstride + g * 16, s = (b * 16 + n) * xsstride + g;
      xr[d][b][0] = __builtin_amdgcn_raw_buffer_load_b128(rx, lo ? v : kOutOfRange, 0, 0);
      xr[d][b][1] = __builtin_amdgcn_raw_buffer_load_b128(rx, hi ? v + 64 : kOutOfRange, 0, 0);
      xscale[d][b] = uint8_t(__builtin_amdgcn_raw_buffer_load_b8(rxs, sc ? s : kOutOfRange, 0, 0));
    }
  };

  f32x4_t acc[R][MB];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[r][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < D; ++d) {
    load(d, d);
    __builtin_amdgcn_sched_barrier(0);
  }
  // (no branch inside a round of D steps: the steps past the last one add zeros)
  for (int s0 = 0; s0 < steps; s0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      u32x4_t a[R][2], xc[MB][2];
      uint32_t as[R], xsc[MB];
#pragma unroll
      for (int r = 0; r < R; ++r) a[r][0] = wr[d][r][0], a[r][1] = wr[d][r][1], as[r] = wscale[d][r];
#pragma unroll
      for (int b = 0; b < MB; ++b) xc[b][0] = xr[d][b][0], xc[b][1] = xr[d][b][1], xsc[b] = xscale[d][b];
      load(d, s0 + d + D);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[r][b] = mfma_fp8(a[r][0], a[r][1], as[r], xc[b][0], xc[b][1], xsc[b], acc[r][b]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Lane (g, n) holds columns 4 g .. 4 g + 3 of the output of row 16 b + n.
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < MB; ++b)
      lds_store16(lds + (w * R * MB + r * MB + b) * 1024 + lane * 16, __builtin_bit_cast(u32x4_t, acc[r][b]));
  __syncthreads();
  auto total = [&](int q) {
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < WAVES; ++o)
      sum += __builtin_bit_cast(f32x4_t, lds_load16(lds + (o * R * MB + q) * 1024 + lane * 16));
    return sum;
  };
  auto result = [&](int r, int b) {  // of tile (or pair of tiles) r
    const f32x4_t sum = total(HALVES * r * MB + b);
    f32x4_t up = {0.f, 0.f, 0.f, 0.f};
    if constexpr (GLU) up = total((HALVES * r + 1) * MB + b);
    return finish<GLU>(sum, up, bias4(p, col0 + r * 16 + 4 * g));
  };
  constexpr int STEP = OUT8 ? 2 : 1;
  for (int q = w; q < COLS / 16 / STEP * MB; q += WAVES) {
    const int r = q / MB * STEP, b = q % MB, m = b * 16 + n, col = col0 + r * 16;
    if constexpr (OUT8) {
      store_block(p, m0 + m, m < rows && col < p.n, col, g, result(r, b), result(r + 1, b));
    } else {
      const f32x4_t v = result(r, b);
      if (m < rows && col + 4 * g < p.n) store4(p, m0 + m, col + 4 * g, v);
    }
  }
}

template <int R, int MB, int D, bool GLU, bool OUT8, int WAVES>
void run(const LinearParams& p, hipStream_t stream) {
  constexpr int COLS = 16 * R / (GLU ? 2 : 1);
  const dim3 grid((p.n + COLS - 1) / COLS, uint32_t((p.rows + 16 * MB - 1) / (16 * MB)));
  hipLaunchKernelGGL((few_kernel<R, MB, D, GLU, OUT8, WAVES>), grid, dim3(64 * WAVES), 0, stream, p);
}

template <int MB, bool GLU, bool OUT8>
void pick(const LinearParams& p, hipStream_t stream) {
  if constexpr (OUT8) run<4, MB, 1, GLU, OUT8, 4>(p, stream);
  else run<2, MB, 1, GLU, OUT8, 8>(p, stream);
}

template <bool GLU, bool OUT8>
void launch(const LinearParams& p, hipStream_t stream) {
  const int blocks = int((std::min<int64_t>(p.rows, 64) + 15) / 16);
  if (blocks == 1) pick<1, GLU, OUT8>(p, stream);
  else if (blocks == 2) pick<2, GLU, OUT8>(p, stream);
  else if (blocks == 3) pick<3, GLU, OUT8>(p, stream);
  else pick<4, GLU, OUT8>(p, stream);
}

}  // namespace

void launch_few(const LinearParams& p, bool glu, hipStream_t stream) {
  if (!glu) launch<false, false>(p, stream);
  else p.scales ? launch<true, true>(p, stream) : launch<true, false>(p, stream);
}

}  // namespace mi::mx8

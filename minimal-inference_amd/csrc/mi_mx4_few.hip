// Projections of few rows with an MXFP4 weight (decode steps): out = x W^T (+ bias)
// or silu(x Wg^T) * (x Wu^T), fp32 accumulation and one rounding; x bf16 or MXFP4.
//
// Bound: HBM, the one read of W, 0.53 bytes per weight (a launch starts and ends in 3 to
// 4 us; beyond that 62 MB, one row, stream at 6.3 TB/s).  A workgroup of 4 or 8 waves owns
// 16 R rows of W over all of k and the waves split k: wave w takes the slabs of 128 k
// w, w + WAVES, ...  A tile of W is an operand as it is loaded, so it goes from memory to
// the matrix instructions through registers alone, D slabs ahead.  With bf16 rows
// its codes become bf16 by one instruction per pair, exactly, and x passes through a
// wave-private LDS slot into operand order; with MXFP4 rows x's tiles are operands
// too and one scaled instruction does a slab.  The waves meet once, at the end, where
// their accumulators are added in wave order: the result does not depend on timing.
// More rows than the accumulators hold (64 of MXFP4, 32 of bf16) are groups of their own
// workgroups, which read W again, from the caches.
#include <algorithm>

#include "mi_mx4_linear.h"

namespace mi::mx4 {
namespace {

constexpr int kXSlot = 16 * kSlab * 2;  // a block of 16 bf16 rows of a slab

template <int R, int MB, int D, bool MX, bool GLU, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(LinearParams p) {
  constexpr int HALVES = GLU ? 2 : 1, COLS = 16 * R / HALVES;
  static_assert(R % HALVES == 0, "gate and up tiles in pairs");
  constexpr int SLOT = MX ? 0 : MB * kXSlot, RED = R * MB * 1024;
  __shared__ __attribute__((aligned(16))) char smem[WAVES * (SLOT > RED ? SLOT : RED)];
  lds_t* const lds = (lds_t*)smem;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const int col0 = int(blockIdx.x) * COLS;
  const int steps = (p.slabs - w + WAVES - 1) / WAVES;  // this wave's slabs: w, w + WAVES, ...

  const char *wbase[HALVES], *sbase[HALVES];
  int wsize[HALVES], ssize[HALVES];
  LaneRow at[R];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
    const int row = h * p.n + col0, tile = row / kTileRows, tiles = min(R / HALVES + 1, p.w_tiles - tile);
    wbase[h] = p.w + int64_t(tile) * p.slabs * kTileBytes;
    sbase[h] = p.ws + int64_t(tile) * p.quads * kQuadBytes;
    wsize[h] = tiles * p.slabs * kTileBytes;
    ssize[h] = tiles * p.quads * kQuadBytes;
#pragma unroll
    for (int r = h; r < R; r += HALVES) at[r] = lane_row(p, row, row + r / HALVES * 16 + n, g);
  }
  // bf16: load i of block b takes 4 rows, lane l chunk l % 16 of row l / 16
  const int lr = lane >> 4, lc = lane & 15;
  const int64_t m0 = int64_t(blockIdx.y) * (16 * MB);
  const int rows = int(min(p.rows - m0, int64_t(16 * MB))), stride = int(p.x_stride * 2);
  const char* const x = p.x + (MX ? m0 / kTileRows * p.slabs * kTileBytes : m0 * stride);
  const char* const xs = p.xs + (MX ? m0 / kTileRows * p.quads * kQuadBytes : 0);
  const int xsize = MX ? (rows + 15) / 16 * p.slabs * kTileBytes : (rows - 1) * stride + p.k * 2;
  const int xssize = (rows + 15) / 16 * p.quads * kQuadBytes;

  u32x4_t wr[D][R], xr[D][MX ? MB : 4 * MB];
  uint32_t wscale[D][R], xscale[D][MB];
  auto load = [&](int d, int step) {
    const int slab = step * WAVES + w, quad = (slab >> 2) * kQuadBytes;
    const bool ok = step < steps;
    __amdgpu_buffer_rsrc_t rw[HALVES], rs[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
      rw[h] = buffer(wbase[h] + slab * kTileBytes, ok ? wsize[h] - slab * kTileBytes : 0);
      rs[h] = buffer(sbase[h] + quad, ok ? ssize[h] - quad : 0);
    }
    // W is read once: non-temporal
#pragma unroll
    for (int r = 0; r < R; ++r) {
      wr[d][r] = __builtin_amdgcn_raw_buffer_load_b128(rw[r % HALVES], at[r].codes, 0, kCacheNT);
      wscale[d][r] = __builtin_amdgcn_raw_buffer_load_b32(rs[r % HALVES], at[r].scales, 0, 0);
    }
    if constexpr (MX) {
      const __amdgpu_buffer_rsrc_t rx = buffer(x + slab * kTileBytes, ok ? xsize - slab * kTileBytes : 0);
      const __amdgpu_buffer_rsrc_t rxs = buffer(xs + quad, ok ? xssize - quad : 0);
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        xr[d][b] = __builtin_amdgcn_raw_buffer_load_b128(rx, b * p.slabs * kTileBytes + lane * 16, 0, 0);
        xscale[d][b] = __builtin_amdgcn_raw_buffer_load_b32(rxs, b * p.quads * kQuadBytes + lane * 4, 0, 0);
      }
    } else {
      const int off = slab * kSlab * 2;
      const __amdgpu_buffer_rsrc_t rx = buffer(x + off, ok ? xsize - off : 0);
      // past a row's end lies the next row: out of range instead
      const bool in = off + lc * 16 < p.k * 2;
#pragma unroll
      for (int i = 0; i < 4 * MB; ++i)
        xr[d][i] = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? (4 * i + lr) * stride + lc * 16 : 0x7ffffff0, 0, 0);
    }
  };

  static_assert(WAVES % 4 == 0, "a wave's slabs lie at one place of their groups of four");
  const int shift = 8 * (w & 3);
  f32x4_t acc[R][MB];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[r][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  lds_t* const slot = lds + w * SLOT;
  // row 4 i + lr, whose place in a row depends on the row modulo 8
  const int so[2] = {lr * 256 + chunk_slot(lr, lc) * 16, lr * 256 + chunk_slot(4 + lr, lc) * 16};
  int ro[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) ro[s] = n * 256 + chunk_slot(n, 4 * g + s) * 16;

#pragma unroll
  for (int d = 0; d < D; ++d) {
    load(d, d);
    __builtin_amdgcn_sched_barrier(0);
  }
  // (no branch inside a round of D steps: the steps past the last one add zeros)
  for (int s0 = 0; s0 < steps; s0 += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if constexpr (MX) {
        u32x4_t a[R], xc[MB];
        uint32_t as[R], xsc[MB];
#pragma unroll
        for (int r = 0; r < R; ++r) a[r] = wr[d][r], as[r] = wscale[d][r] >> shift;
#pragma unroll
        for (int b = 0; b < MB; ++b) xc[b] = xr[d][b], xsc[b] = xscale[d][b] >> shift;
        load(d, s0 + d + D);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int b = 0; b < MB; ++b) acc[r][b] = mfma_fp4<0, 0>(a[r], as[r], xc[b], xsc[b], acc[r][b]);
      } else {
#pragma unroll
        for (int i = 0; i < 4 * MB; ++i) lds_store16(slot + i * 1024 + so[i & 1], xr[d][i]);
        u32x4_t a[R];
        float as[R];
#pragma unroll
        for (int r = 0; r < R; ++r) a[r] = wr[d][r], as[r] = scale_f32(wscale[d][r] >> shift & 255u);
        load(d, s0 + d + D);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          bf16x8_t xv[MB];
#pragma unroll
          for (int b = 0; b < MB; ++b)
            xv[b] = __builtin_bit_cast(bf16x8_t, lds_load16(slot + b * kXSlot + ro[s]));
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const bf16x8_t v = to_bf16(a[r][s], as[r]);
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[r][b] = mfma_16x16x32_bf16(v, xv[b], acc[r][b]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // Lane (g, n) holds columns 4 g .. 4 g + 3 of the output of row 16 b + n.
  __syncthreads();
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
  for (int q = w; q < R / HALVES * MB; q += WAVES) {
    const int r = q / MB, b = q - r * MB;  // r: the tile (or pair of tiles)
    const f32x4_t sum = total(HALVES * r * MB + b);
    f32x4_t up = {0.f, 0.f, 0.f, 0.f};
    if constexpr (GLU) up = total((HALVES * r + 1) * MB + b);
    const int m = b * 16 + n, col = col0 + r * 16 + 4 * g;
    if (m < rows && col < p.n) store4<GLU>(p, m0 + m, col, sum, up, bias4(p, col));
  }
}

template <int R, int MB, int D, bool MX, bool GLU, int WAVES>
void run(const LinearParams& p, hipStream_t stream) {
  constexpr int COLS = 16 * R / (GLU ? 2 : 1);
  const dim3 grid((p.n + COLS - 1) / COLS, uint32_t((p.rows + 16 * MB - 1) / (16 * MB)));
  hipLaunchKernelGGL((few_kernel<R, MB, D, MX, GLU, WAVES>), grid, dim3(64 * WAVES), 0, stream, p);
}

// The form of a launch, from the tiles of W, the slabs and the 16-row blocks of x (us,
// weights rotated through 600 MB; R tiles and 4 or 8 waves per workgroup, 1 slab ahead, 2
// where marked):
//                             waves:      4                                  8
//                              rows   R 2*   R 3   R 4   R 5   R 7   R 8   R 1   R 2   R 3   R 4   R 5   R 6
//   N  1152 K   896               8   3.1                                  3.1   3.2         3.8
//   N  4096 K  4096               1   6.1                                  5.1   5.4         6.5
//   N  4096 K  4096              32   8.1                                  7.2   8.3         9.2
//   N  6144 K  4096               8   6.5                                  6.7   5.6         6.7
//   N  8192 K  8192              32  13.6                                       13.0        16.2
//   N 10240 K   896               8          3.8   3.9                                 3.9   4.1
//   N 10240 K  2048              32          6.4   6.6                                 6.7   6.9
//   N 10240 K  8192               8  13.1                     18.1  19.7       14.7  10.7  11.7  13.4  14.3
//   N 10240 K  8192              32  22.2                     21.7  25.1       23.6  15.4  16.9  18.4  19.6
//   N 18432 K  4096              32                           13.6  15.4             15.9  17.9  12.3  12.9
//   N 28672 K  4096               8                     13.7  16.0                   14.7  13.2  14.9  17.6
//   N 28672 K  2048               8                7.7         8.5                         8.7
//   N 28672 K  4096              32                           15.3  17.9             21.2  18.9  21.2  23.1
//   N 59136 K  8192               8               46.0  41.1        49.0                   46.2  40.4
//   N 59136 K  8192              32               59.5              53.4                   62.7
//   gated 2 x 11008, K 4096      32                                 15.4                   19.2        14.1
//   gated 2 x 14336, K 4096       1               12.9              14.7                   13.8
//   gated 2 x 14336, K 4096      32                                 16.3                   19.4
//   MXFP4 x: N 10240 K 8192      64                           19.1  20.6             13.0  14.7  16.4
//   MXFP4 x: N 18432 K 4096      48                           11.5  13.2             12.5  14.7  10.5  11.2
//   MXFP4 x: N 28672 K 4096      48                           13.8  16.4             17.1  15.9  18.3  20.0
// Every workgroup reads x, so as many tiles as make one round of workgroups; eight waves
// while k is long enough to feed them and their sums fit in LDS.  Seven and eight tiles
// pay from two blocks of x on; beyond one round of eight, a single block takes three
// rounds and more blocks two.  (More slabs ahead are slower: gated 2 x 14,336, 32 rows 18.1.)
template <int R, int MB, bool MX, bool GLU>
void waves(const LinearParams& p, hipStream_t stream) {
  if constexpr (R == (GLU ? 2 : 1) && MB == 1) {
    if (p.w_tiles <= mi::num_cus() && p.slabs >= 32) return run<R, MB, 2, MX, GLU, 8>(p, stream);
  }
  if constexpr (R <= 6 && R * MB * 8 <= 160) {
    if (R <= 2 || p.slabs >= 28) return run<R, MB, 1, MX, GLU, 8>(p, stream);
  }
  run<R, MB, 1, MX, GLU, 4>(p, stream);
}
template <int MB, bool MX, bool GLU>
void pick(const LinearParams& p, hipStream_t stream) {
  const int cus = mi::num_cus();
  auto rounds = [&](int n) { return (p.w_tiles + n * cus - 1) / (n * cus); };
  int tiles = rounds(1);
  if (MB == 1 && tiles > 6) tiles = tiles <= 8 ? 4 : std::min(rounds(3), 6);
  else if (tiles > 8) tiles = std::min(rounds(2), 8);
  if constexpr (!GLU) {
    if (tiles == 1) return waves<1, MB, MX, GLU>(p, stream);
    if (tiles == 3) return waves<3, MB, MX, GLU>(p, stream);
    if (tiles == 5) return waves<5, MB, MX, GLU>(p, stream);
    if constexpr (MB > 1) {
      if (tiles == 7) return waves<7, MB, MX, GLU>(p, stream);
    }
  }
  if (tiles <= 2) return waves<2, MB, MX, GLU>(p, stream);
  if (tiles <= 4) return waves<4, MB, MX, GLU>(p, stream);
  if (MB == 1 || tiles <= 6) return waves<6, MB, MX, GLU>(p, stream);
  if constexpr (MB > 1) waves<8, MB, MX, GLU>(p, stream);
}

template <bool GLU>
void launch(const LinearParams& p, hipStream_t stream) {
  const int blocks = int((std::min(p.rows, few_group(p.xs != nullptr)) + 15) / 16);
  if (p.xs) {
    if (blocks == 1) pick<1, true, GLU>(p, stream);
    else if (blocks == 2) pick<2, true, GLU>(p, stream);
    else if (blocks == 3) pick<3, true, GLU>(p, stream);
    else pick<4, true, GLU>(p, stream);
  } else {
    if (blocks == 1) pick<1, false, GLU>(p, stream);
    else pick<2, false, GLU>(p, stream);
  }
}

}  // namespace

void launch_few(const LinearParams& p, bool glu, hipStream_t stream) {
  glu ? launch<true>(p, stream) : launch<false>(p, stream);
}

}  // namespace mi::mx4

// Projections of few rows with both operands in MXFP8 (decode steps): out = x W^T (+ bias)
// or silu(x Wg^T) * (x Wu^T), fp32 accumulation and one rounding.
//
// Bound: HBM, the one read of W, 1.03 bytes per weight.  A workgroup of 1 to 8 waves owns
// 16 R rows of W over all of k and the waves split k: wave w takes the groups of four slabs
// w, w + WAVES, ...  Its rows of a slab (of W and of x) go from memory into a ring of its own in
// LDS, DEPTH slabs ahead, eight rows of 128 bytes by an instruction, and from there, as
// operands, to the matrix instructions: no wave waits for another.  (Operands read from the rows
// directly are 64 separate places an instruction, and the address unit takes them one by
// one: 32 x 14,336 x 4,096 32 us.)  The waves meet once, at the end, where their
// accumulators are added in wave order: the result does not depend on timing.
// SPLIT: the workgroup takes p.split_slabs slabs (a multiple of four) and leaves its sums for launch_combine.
#include <algorithm>

#include "mi_mx8_linear.h"

namespace mi::mx8 {
namespace {

constexpr int few_lds(int r, int mb, int depth, int waves) {
  const int ring = depth * (r + mb) * 2048 + 2 * (((r + mb) * 16 + 63) / 64) * 1024;
  const int sums = r * mb * 1024;
  return waves * (ring > sums ? ring : sums);
}

template <int R, int MB, int DEPTH, bool GLU, bool OUT8, int WAVES, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES) void few_kernel(LinearParams p) {
  constexpr int HALVES = GLU ? 2 : 1, COLS = 16 * R / HALVES, TILES = R + MB;
  constexpr int SLOT = TILES * 2048, SLOADS = (TILES * 16 + 63) / 64, SBYTES = SLOADS * 1024, LOADS = 2 * TILES;
  constexpr int WAVE = few_lds(R, MB, DEPTH, 1);
  static_assert(!SPLIT || (!GLU && !OUT8), "parts are of plain products");
  static_assert(R % HALVES == 0 && (!OUT8 || COLS % kBlock == 0), "gate and up tiles in pairs, whole blocks");
  static_assert(4 % DEPTH == 0 && DEPTH * SLOT + 2 * SBYTES <= WAVE && WAVES * WAVE <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[WAVES * WAVE];
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  lds_t* const lds = (lds_t*)smem + w * WAVE;
  lds_t* const scales = lds + DEPTH * SLOT;
  const int g = lane >> 4, n = lane & 15;
  const int col0 = int(blockIdx.x) * COLS, blocks = p.k / kBlock;
  const int rows = int(p.rows);
  const int slab0 = SPLIT ? int(blockIdx.y) * p.split_slabs : 0, slab_end = SPLIT ? min(slab0 + p.split_slabs, p.slabs) : p.slabs;
  const int wstride = int(p.w_stride), xstride = int(p.x_stride);
  const char* const xbase = p.x;
  const char* const wbase = p.w + col0 * p.w_stride;
  const char* const ubase = p.w + (int64_t(p.n) + col0) * p.w_stride;
  const int xsize = (rows - 1) * xstride + p.k, wsize = (min(COLS, p.w_rows - col0) - 1) * wstride + p.k;
  const int usize = GLU ? (min(COLS, p.n - col0) - 1) * wstride + p.k : 0;
  // a load: 8 rows, lane l chunk slot l % 8 of row l / 8
  const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 16;
  auto load = [&](int slab, int slot) {
    const int xlane = r8 * xstride + chunk, wlane = r8 * wstride + chunk;
    const int off = slab * kSlab;
    const bool ok = slab < slab_end;
    const int past = off + chunk < p.k ? 0 : kOutOfRange;  // past the row's end lies the next row
    const __amdgpu_buffer_rsrc_t rw = buffer(wbase + off, ok ? wsize - off : 0), rx = buffer(xbase + off, ok ? xsize - off : 0);
    const __amdgpu_buffer_rsrc_t ru = GLU ? buffer(ubase + off, ok ? usize - off : 0) : rw;
    lds_t* const to = lds + slot * SLOT;
    // W is read once: non-temporal
#pragma unroll
    for (int i = 0; i < 2 * R; ++i)
      lds_dma16<kCacheNT>(i / 2 % HALVES ? ru : rw, to + i * 1024, (wlane + (i / 2 / HALVES * 16 + i % 2 * 8) * wstride) | past);
#pragma unroll
    for (int i = 0; i < 2 * MB; ++i)
      lds_dma16(rx, to + (2 * R + i) * 1024, (xlane + i * 8 * xstride) | past);
  };
  const int quad0 = slab0 / 4, first = quad0 + w;
  // The scale bytes of four slabs, 16 a row: the tiles' rows of W, then x's.
  auto load_scales = [&](int quad) {
#if defined(__HIP_DEVICE_COMPILE__)
    lds_t* const to = scales + ((quad - quad0) / WAVES & 1) * SBYTES;
#pragma unroll
    for (int i = 0; i < SLOADS; ++i) {
      const int at = i * 64 + lane, tile = at / 16, r = at % 16;
      const int row = tile < R ? tile / HALVES * 16 + r : (tile - R) * 16 + r;
      const char* from = tile < R ? p.ws + (int64_t(tile % HALVES) * p.n + col0 + row) * p.ws_stride
                                  : p.xs + row * p.xs_stride;
      // (anything readable in the place of rows past the matrix's and of blocks past a row's)
      if (quad * 16 >= blocks || tile >= TILES || (tile < R ? col0 + row >= p.n : row >= rows)) from = p.ws;
      else from += quad * 16;
      __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)const_cast<char*>(from),
                                       (__attribute__((address_space(3))) void*)(to + i * 1024), 16, 0, 0);
    }
#endif
  };

  f32x4_t acc[R][MB];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[r][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int lo = n * kSlab + (g ^ (n & 7)) * 16, hi = n * kSlab + ((4 + g) ^ (n & 7)) * 16;
  auto slab_at = [&](int quad, int s) { return 4 * (quad + s / 4 * WAVES) + s % 4; };  // s steps into a group

  if (4 * first < slab_end) {
    load_scales(first);
    load_scales(first + WAVES);
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(slab_at(first, d), d);
  }
  constexpr int kInFlight = (DEPTH - 1) * LOADS;
  static_assert(kInFlight < 64, "vmcnt");
  for (int quad = first; 4 * quad < slab_end; quad += WAVES) {
    // (a group ahead: done by the waits of the four steps before it)
    if (quad != first) load_scales(quad + WAVES);
    const lds_t* const sl = scales + ((quad - quad0) / WAVES & 1) * SBYTES + n * 16 + g;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int slab = 4 * quad + s;
      __builtin_amdgcn_s_waitcnt(0x0f70 | (kInFlight & 15) | (kInFlight >> 4 << 14));
      __builtin_amdgcn_sched_barrier(0);
      const lds_t* const from = lds + s % DEPTH * SLOT;
      const bool known = slab * 4 + g < blocks;  // (a row's padding may hold anything)
      u32x4_t v[TILES][2];
      uint32_t sc[TILES];
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        v[t][0] = lds_load16(from + t * 2048 + lo);
        v[t][1] = lds_load16(from + t * 2048 + hi);
        sc[t] = lds_load1(sl + t * 256 + s * 4);
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);  // read: the place may be filled again
      __builtin_amdgcn_sched_barrier(0);
      load(slab_at(quad, s + DEPTH), s % DEPTH);
#pragma unroll
      for (int t = 0; t < TILES; ++t) sc[t] = known ? sc[t] : 0u;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int b = 0; b < MB; ++b)
          acc[r][b] = mfma_fp8(v[r][0], v[r][1], sc[r], v[R + b][0], v[R + b][1], sc[R + b], acc[r][b]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);  // (the loads past the end write to LDS)

  // Lane (g, n) holds columns 4 g .. 4 g + 3 of the output of row 16 b + n.
  lds_t* const sums = (lds_t*)smem;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < MB; ++b)
      lds_store16(sums + (w * R * MB + r * MB + b) * 1024 + lane * 16, __builtin_bit_cast(u32x4_t, acc[r][b]));
  __syncthreads();
  auto total = [&](int q) {
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < WAVES; ++o)
      sum += __builtin_bit_cast(f32x4_t, lds_load16(sums + (o * R * MB + q) * 1024 + lane * 16));
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
    if constexpr (SPLIT) {
      // [part][row][columns, in fours]
      if (m < rows && col + 4 * g < p.n)
        p.parts[(int64_t(blockIdx.y) * rows + m) * ((p.n + 3) / 4) + col / 4 + g] = total(q);
    } else if constexpr (OUT8) {
      if (p.sums) {
#pragma unroll
        for (int i = 0; i < STEP; ++i)
          if (const int at = col + 16 * i + 4 * g; m < rows && at < p.n)
            store_sums(p, m, at, total(HALVES * (r + i) * MB + b), total((HALVES * (r + i) + 1) * MB + b));
        continue;
      }
      store_block(p, m, m < rows && col < p.n, col, g, result(r, b), result(r + 1, b));
    } else {
      const f32x4_t v = result(r, b);
      if (m < rows && col + 4 * g < p.n) store4(p, m, col + 4 * g, v);
    }
  }
}

template <int R, int MB, int DEPTH, bool GLU, bool OUT8, int WAVES, bool SPLIT = false>
void run(const LinearParams& p, hipStream_t stream) {
  constexpr int COLS = 16 * R / (GLU ? 2 : 1);
  const dim3 grid((p.n + COLS - 1) / COLS, SPLIT ? (p.slabs + p.split_slabs - 1) / p.split_slabs : 1);
  hipLaunchKernelGGL((few_kernel<R, MB, DEPTH, GLU, OUT8, WAVES, SPLIT>), grid, dim3(64 * WAVES), 0, stream, p);
}

// The form of a launch, from the tiles of W and the 16-row blocks of x (us, weights rotated
// through 600 MB, calls in a graph; R tiles by 4 or 8 waves, 2 or 4 slabs deep):
//                            rows  1 4x8  1 4x4  1 2x4  2 2x8  2 2x4  3 2x8  3 2x4  4 2x4  6 2x4
//   N   896 K   896             8    3.2    3.2    3.7           3.9
//   N   896 K  4864             8    5.7    5.4    7.1    7.3
//   N  4096 K  4096             1    6.5    6.0    6.6    6.7
//   N  3584 K 18944             1   15.5   14.6   19.1   19.4
//   N  4096 K 14336            16   14.3   13.9   15.0   18.6
//   N  4096 K 14336            32          19.6   20.4   22.4   24.0         27.6
//   N  4096 K 14336            64                 25.3          29.8         35.3   40.6
//   N  6144 K  4096             1           8.8    8.2    7.6    8.2    8.7    8.6
//   N  6144 K  4096            32                 11.5    9.6    9.5         10.5   11.2
//   N  6144 K  4096            64                 16.7          11.3         12.9   14.0
//   N  8192 K 29568            16   54.2   53.3   52.2   46.3   48.0
//   N 10240 K  8192            16                 21.2                 17.8  18.7   19.9
//   N 10240 K  8192            48                 33.0          31.9         21.9   24.5
//   gated 2 x 4864, K 896       8                         7.9    5.4                 4.8    5.4
//   gated 2 x 14336, K 4096     1                        30.1   26.3                27.0   33.8
//   gated 2 x 14336, K 4096    32                        37.2   31.1                30.2   37.3
//   gated 2 x 18944, K 3584    64                               48.7                39.3
//   gated 2 x 29568, K 8192     1                        99.0   84.1                89.4   94.6
//   gated 2 x 29568, K 8192    64                              141.2               116.8
// Every workgroup reads x, so as many tiles as make one round of workgroups, four at most;
// eight waves with a single block of x and two or three.  Beyond three rounds a single
// block takes two, whose workgroups run side by side.
// Four tiles by as many waves as leave room for all workgroups at once: no round starts with empty rings
// (us, gated, 4 / 2 / 1 waves, * where all fit):
//   2 x 14336, K 4096  32 rows 30.7 / 27.3* / 28.6*   64 rows 34.5 / 31.0* / 32.9*
//   2 x 18944, K 3584   1 row  28.8 / 27.2* / 26.0*   64 rows 39.0 / 45.1 / 36.7*
//   2 x 29568, K 8192  32 rows 99.4 / 100.6 / 100.2*  64 rows 116.5 / 114.1 / 110.2*
template <int MB, bool GLU, bool OUT8>
void run_four(const LinearParams& p, hipStream_t stream) {
  constexpr int COLS = 64 / (GLU ? 2 : 1), kLds = 160 * 1024, kWave = few_lds(4, MB, 2, 1);
  const int64_t workgroups = (p.n + COLS - 1) / COLS, cus = mi::num_cus();
  if (workgroups <= cus * (kLds / (4 * kWave))) run<4, MB, 2, GLU, OUT8, 4>(p, stream);
  else if (workgroups <= cus * (kLds / (2 * kWave))) run<4, MB, 2, GLU, OUT8, 2>(p, stream);
  else if (workgroups <= cus * (kLds / kWave)) run<4, MB, 2, GLU, OUT8, 1>(p, stream);
  else run<4, MB, 2, GLU, OUT8, 4>(p, stream);
}

template <int MB, bool GLU, bool OUT8>
void pick(const LinearParams& p, hipStream_t stream) {
  if constexpr (OUT8) {
    run_four<MB, GLU, OUT8>(p, stream);  // (whole blocks of out)
  } else {
    const int tiles = (p.w_rows + 15) / 16, cus = mi::num_cus(), rounds = (tiles + cus - 1) / cus;
    if constexpr (!GLU) {
      if (rounds <= 1) {
        if constexpr (MB == 1) return run<1, MB, 4, GLU, OUT8, 4>(p, stream);
        else return run<1, MB, MB == 2 ? 4 : 2, GLU, OUT8, 4>(p, stream);
      }
      if (rounds == 3) return run<3, MB, 2, GLU, OUT8, MB == 1 ? 8 : 4>(p, stream);
      if constexpr (MB == 1) {
        if (rounds == 2) return run<2, MB, 2, GLU, OUT8, 8>(p, stream);
      }
    }
    if (rounds <= 2 || (MB == 1 && rounds > 3)) run<2, MB, 2, GLU, OUT8, 4>(p, stream);
    else run_four<MB, GLU, OUT8>(p, stream);
  }
}

template <bool GLU, bool OUT8>
void launch(const LinearParams& p, hipStream_t stream) {
  const int blocks = int((p.rows + 15) / 16);
  if (blocks == 1) pick<1, GLU, OUT8>(p, stream);
  else if (blocks == 2) pick<2, GLU, OUT8>(p, stream);
  else if (blocks == 3) pick<3, GLU, OUT8>(p, stream);
  else pick<4, GLU, OUT8>(p, stream);
}

// Workgroups that share k (S of them, four tiles each) read an S-th of x's bytes where
// one by itself reads all; their sums go through memory in fp32, and another launch adds them in
// order. The count, in us: the way into LDS of a CU (56.6 GB/s, half of it hidden behind
// HBM) against the launch and the sums' way. Measured (calls in a graph, alone / shared):
//   N  4096 K 14336   16 rows 17.4 / 17.5 (S 4)   32 rows 20.5 / 18.7 (4)   64 rows 25.7 / 21.3 (4)
//   N  3584 K 18944   32 rows 24.6 / 22.1 (4)     64 rows 32.6 / 25.6 (4)
//   N  8192 K 29568   32 rows 62.4 / 57.6 (2)     64 rows 72.6 / 64.3 (2)
//   N  4096 K  4096   64 rows  9.8 / 11.5 (4)     N 6144 K 4096   64 rows 12.1 / 13.7 (2)
//   N  8192 K  8192   64 rows 22.6 / 24.9 (2)
// (other tiles and S were slower than the better of the two; a single block of x gains nothing)
int split_slabs_of(bool glu, int64_t rows, int64_t n, int slabs, size_t room) {
  const int tiles = int((n + 15) / 16), blocks = int((rows + 15) / 16), cus = mi::num_cus();
  if (glu || blocks == 1) return slabs;
  const int rounds = std::min((tiles + cus - 1) / cus, 4);
  const float k = float(slabs) * kSlab, per_us = 2 * 56.6e3f;
  float best = (rounds + blocks) * 16 * k / per_us;
  int found = slabs;
  for (int s = 2; s <= 4; s += 2) {
    const int each = ((slabs + s - 1) / s + 3) / 4 * 4;
    if ((tiles + 3) / 4 * s > cus || each * (s - 1) >= slabs || room < size_t(s) * rows * ((n + 3) / 4) * 16) continue;
    const float us = (4 + blocks) * 16 * float(each) * kSlab / per_us + 1.f + 2.f * 4 * s * float(rows) * float(n) / 4.4e6f;
    if (us < best) best = us, found = each;
  }
  return found;
}

template <int MB>
void run_shared(const LinearParams& p, hipStream_t stream) {
  run<4, MB, 2, false, false, 4, true>(p, stream);
}

}  // namespace

size_t few_workspace(bool glu, int64_t rows, int64_t n, int slabs, size_t room) {
  const int each = split_slabs_of(glu, rows, n, slabs, room);
  return each < slabs ? size_t((slabs + each - 1) / each) * rows * ((n + 3) / 4) * 16 : 0;
}

void launch_few(const LinearParams& p, bool glu, size_t room, hipStream_t stream) {
  LinearParams q = p;
  q.split_slabs = split_slabs_of(glu, p.rows, p.n, p.slabs, room);
  if (q.split_slabs < p.slabs) {
    const int blocks = int((p.rows + 15) / 16);
    if (blocks == 2) run_shared<2>(q, stream);
    else if (blocks == 3) run_shared<3>(q, stream);
    else run_shared<4>(q, stream);
    launch_combine(q, false, (p.slabs + q.split_slabs - 1) / q.split_slabs, stream);
    return;
  }
  if (!glu) launch<false, false>(p, stream);
  else p.scales || p.sums ? launch<true, true>(p, stream) : launch<true, false>(p, stream);
}

}  // namespace mi::mx8

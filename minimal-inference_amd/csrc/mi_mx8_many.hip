// Projections of many rows with both operands in MXFP8 (prompts): out = x W^T (+ bias) or
// silu(x Wg^T) * (x Wu^T), fp32 accumulation and one rounding.
//
// Bound: the matrix instructions.  A workgroup of WM x WN waves owns a block of out; per
// slab of 128 k its rows of W and of x go straight from memory to LDS (one of STAGES
// buffers, the later slabs' while this one is multiplied) and from there, as operands, to the
// waves.  A row of a slab is 128 bytes, eight chunks whose places are permuted by the row,
// so that the rows an operand read touches together fall on distinct banks.  The scale
// bytes of four slabs (16 bytes a row) are staged alike.
#include <algorithm>

#include "mi_mx8_linear.h"
#include "mi_overlap.h"

namespace mi::mx8 {
namespace {

__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t rs, lds_t* dst, int voffset) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, voffset, 0, 0, 0);
#endif
}

constexpr int kGroupM = 4;

// Which block of out a workgroup owns.  Workgroups go to the eight XCDs in turn.  Each XCD
// gets a run of tiles, in groups of kGroupM down the rows of x, so that those it holds at a
// time share rows of x and of W in its L2.
__device__ __forceinline__ void place(const LinearParams& p, int bm, int cols, int& col0, int64_t& m0) {
  const int mt = int((p.rows + bm - 1) / bm), nt = (p.n + cols - 1) / cols, all = mt * nt;
  const int id = int(blockIdx.x), xcd = id & 7, each = all / 8, more = all % 8;
  const int tile_id = xcd * each + min(xcd, more) + (id >> 3);
  const int group = tile_id / (kGroupM * nt), in = tile_id - group * kGroupM * nt;
  const int high = min(kGroupM, mt - group * kGroupM);
  col0 = in / high * cols;
  m0 = int64_t(group * kGroupM + in % high) * bm;
}

// Scales of four slabs: 64 rows a load, XS loads of x's and the rest of W's rows (16 of
// each half in turn).
template <int WAVES, int BM, int BN, bool GLU>
__device__ __forceinline__ void load_scales(const LinearParams& p, lds_t* to, int quad, int w, int col0, int64_t m0, int rows) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int HALVES = GLU ? 2 : 1, XS = (BM + 63) / 64, LOADS = XS + (BN + 63) / 64;
  const char *const xsbase = p.xs + m0 * p.xs_stride, *const wsbase = p.ws + col0 * p.ws_stride;
  const int off = quad * 16, lane = threadIdx.x & 63;
  for (int i = w; i < LOADS; i += WAVES) {
    const bool of_x = i < XS;
    const int at = (of_x ? i : i - XS) * 64 + lane, tile = at / 16;
    const int row = of_x ? at : tile / HALVES * 16 + at % 16;
    const char* from = of_x ? xsbase + row * p.xs_stride : wsbase + (tile % HALVES * int64_t(p.n) + row) * p.ws_stride;
    // (anything readable in the place of rows past the matrix's and of blocks past a row's)
    if (off * kBlock >= p.k || (of_x ? at >= rows : at >= BN || col0 + row >= p.n)) from = p.ws;
    else from += off;
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)const_cast<char*>(from),
                                     (__attribute__((address_space(3))) void*)(to + i * 1024), 16, 0, 0);
  }
#endif
}

// A wave's sums to memory: tile t of W's rows is columns col0 + 16 (first_tile + t) / HALVES
// on, block b rows m0 + row0 + 16 b on.  Lane (g, n) holds columns 4 g .. 4 g + 3 of a tile for row n of a block.
template <int MB, int NT, bool GLU, bool OUT8, bool SPLIT>
__device__ __forceinline__ void end_of_product(const LinearParams& p, const f32x4_t (&acc)[NT][MB], int col0, int first_tile,
                                               int64_t m0, int row0, int rows) {
  constexpr int HALVES = GLU ? 2 : 1;
  const int g = (threadIdx.x & 63) >> 4, n = threadIdx.x & 15;
  if constexpr (OUT8 && !SPLIT) {
#pragma unroll
    for (int t = 0; t < NT; t += 4) {
      const int first = col0 + (first_tile + t) / 2 * 16;
      const f32x4_t none = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        const int m = row0 + b * 16 + n;
        store_block(p, m0 + m, m < rows && first < p.n, first, g, finish<true>(acc[t][b], acc[t + 1][b], none),
                    finish<true>(acc[t + 2][b], acc[t + 3][b], none));
      }
    }
    return;
  }
  // Two tiles' lanes change places, so that a lane has eight columns and four lanes 64
  // bytes of a row.
  if constexpr (!SPLIT && !OUT8 && NT / HALVES % 2 == 0) {
    if (p.wide) {
#pragma unroll
      for (int t = 0; t < NT; t += 2 * HALVES) {
        const int first = col0 + (first_tile + t) / HALVES * 16, col = first + (g & 1) * 16 + (g >> 1) * 8;
        const f32x4_t bias0 = bias4(p, first + 4 * g), bias1 = bias4(p, first + 16 + 4 * g);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          const u32x2_t u = round4(finish<GLU>(acc[t][b], acc[t + HALVES - 1][b], bias0));
          const u32x2_t v = round4(finish<GLU>(acc[t + HALVES][b], acc[t + 2 * HALVES - 1][b], bias1));
          const auto s0 = __builtin_amdgcn_permlane16_swap(u.x, v.x, false, false);
          const auto s1 = __builtin_amdgcn_permlane16_swap(u.y, v.y, false, false);
          const int m = row0 + b * 16 + n;
          if (m < rows && col < p.n)
            *reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(p.out) + (m0 + m) * p.o_stride + col) =
                u32x4_t{s0[0], s1[0], s0[1], s1[1]};
        }
      }
      return;
    }
  }
#pragma unroll
  for (int t = 0; t < NT; t += HALVES) {
    const int col = col0 + (first_tile + t) / HALVES * 16 + 4 * g;
    if (col >= p.n) continue;
    const f32x4_t bias = SPLIT ? f32x4_t{0.f, 0.f, 0.f, 0.f} : bias4(p, col);
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const int m = row0 + b * 16 + n;
      if (m >= rows) continue;
      if constexpr (SPLIT) {
        // [part][half][row][columns, in fours]
        const int64_t fours = (p.n + 3) / 4;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          p.parts[((int64_t(blockIdx.y) * HALVES + h) * p.rows + m0 + m) * fours + col / 4] = acc[t + h][b];
      } else if constexpr (!OUT8) {
        store4(p, m0 + m, col, finish<GLU>(acc[t][b], acc[t + HALVES - 1][b], bias));
      }
    }
  }
}

// MB blocks of 16 rows of x and NT tiles of 16 rows of W per wave.  Slabs are staged STAGES
// deep: before slab s is multiplied the loads of the STAGES - 2 slabs behind it may be in
// flight, and after the barrier its predecessor's buffer is filled again.  Loads past the last slab
// are out of range, so that every wait counts the same loads.
//
// SPLIT: the workgroup takes p.split_slabs slabs and leaves its sums, in fp32, for
// combine_kernel.
template <int WM, int WN, int MB, int NT, int STAGES, bool GLU, bool OUT8, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN) void many_kernel(LinearParams p) {
  constexpr int WAVES = WM * WN, HALVES = GLU ? 2 : 1;
  constexpr int BM = WM * MB * 16, BN = WN * NT * 16, COLS = BN / HALVES;  // BN rows of W
  constexpr int XBYTES = BM * kSlab, STAGE = XBYTES + BN * kSlab;
  constexpr int XLOADS = XBYTES / 1024 / WAVES, WLOADS = BN * kSlab / 1024 / WAVES;
  constexpr int XS = (BM + 63) / 64, SLOADS = XS + (BN + 63) / 64, SBYTES = SLOADS * 1024;
  static_assert(XBYTES / 1024 % WAVES == 0 && BN * kSlab / 1024 % WAVES == 0 && NT % HALVES == 0, "even shares");
  static_assert(!OUT8 || (GLU && NT % 4 == 0), "whole blocks");
  static_assert(STAGES * STAGE + 2 * SBYTES <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[STAGES * STAGE + 2 * SBYTES];
  lds_t* const lds = (lds_t*)smem;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int wm = w / WN, wn = w % WN;
  const int g = lane >> 4, n = lane & 15;
  int col0;
  int64_t m0;
  place(p, BM, COLS, col0, m0);
  const int rows = int(min(int64_t(BM), p.rows - m0));
  const int slab0 = SPLIT ? int(blockIdx.y) * p.split_slabs : 0;
  const int slab_end = SPLIT ? min(slab0 + p.split_slabs, p.slabs) : p.slabs;
  const int blocks = p.k / kBlock;

  // Row r of the workgroup's rows of W: 16 of each half in turn (gate, up, gate, ...).
  const int wstride = int(p.w_stride), xstride = int(p.x_stride);
  const char* wbase[HALVES];
  int wsize[HALVES];
#pragma unroll
  for (int h = 0; h < HALVES; ++h) {
    const int row = h * p.n + col0, count = min(COLS, p.w_rows - row);
    wbase[h] = p.w + row * p.w_stride;
    wsize[h] = (count - 1) * wstride + p.k;
  }
  const char* const xbase = p.x + m0 * p.x_stride;
  const int xsize = (rows - 1) * xstride + p.k;
  // load i: 8 rows, lane l chunk slot l % 8 of row l / 8
  const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 16;
  int xv[XLOADS], wv[WLOADS];
#pragma unroll
  for (int i = 0; i < XLOADS; ++i) xv[i] = ((w * XLOADS + i) * 8 + r8) * xstride + chunk;
#pragma unroll
  for (int i = 0; i < WLOADS; ++i) {
    const int at = (w * WLOADS + i) * 8 + r8, tile = at / 16;
    wv[i] = (tile / HALVES * 16 + at % 16) * wstride + chunk;
  }
  auto load = [&](int slab, int buf) {
    lds_t* const stage = lds + buf * STAGE;
    const int off = slab * kSlab;
    const bool ok = slab < slab_end, inside = off + chunk < p.k;  // past the row's end lies the next row
    const __amdgpu_buffer_rsrc_t rx = buffer(xbase + off, ok ? xsize - off : 0);
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) lds_dma16(rx, stage + (w * XLOADS + i) * 1024, inside ? xv[i] : kOutOfRange);
    __amdgpu_buffer_rsrc_t rw[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) rw[h] = buffer(wbase[h] + off, ok ? wsize[h] - off : 0);
#pragma unroll
    for (int i = 0; i < WLOADS; ++i)
      lds_dma16(rw[(w * WLOADS + i) / 2 % HALVES], stage + XBYTES + (w * WLOADS + i) * 1024, inside ? wv[i] : kOutOfRange);
  };
  lds_t* const scales = lds + STAGES * STAGE;
  auto stage_scales = [&](int quad) {
    load_scales<WAVES, BM, BN, GLU>(p, scales + (quad & 1) * SBYTES, quad, w, col0, m0, rows);
  };

  f32x4_t acc[NT][MB];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[t][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // a lane's two chunks of row n of 16
  const int lo = n * kSlab + (g ^ (n & 7)) * 16, hi = n * kSlab + ((4 + g) ^ (n & 7)) * 16;

  constexpr int kInFlight = (STAGES - 2) * (XLOADS + WLOADS);
  static_assert(kInFlight < 64, "vmcnt");
  stage_scales(slab0 >> 2);
  stage_scales((slab0 >> 2) + 1);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(slab0 + i, i);
  int buf = 0, before = STAGES - 1;
  for (int slab = slab0; slab < slab_end; ++slab) {
    // vmcnt: this slab (and the scales, older than its successors') is in LDS; lgkmcnt: this
    // wave has read the one before
    __builtin_amdgcn_s_waitcnt(0x0070 | (kInFlight & 15) | (kInFlight >> 4 << 14));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    const int quad = slab >> 2;
    if ((slab & 3) == 0 && slab != slab0) stage_scales(quad + 1);  // (four slabs ahead: done by any wait before them)
    load(slab + STAGES - 1, before);
    const lds_t* const xl = lds + buf * STAGE + wm * MB * 16 * kSlab;
    const lds_t* const wl = lds + buf * STAGE + XBYTES + wn * NT * 16 * kSlab;
    const lds_t* const sl = scales + (quad & 1) * SBYTES + n * 16 + (slab & 3) * 4 + g;
    const bool known = slab * 4 + g < blocks;  // (a row's padding may hold anything)
    u32x4_t a[NT][2], x[MB][2];
    uint32_t as[NT], xs[MB];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      a[t][0] = lds_load16(wl + t * 16 * kSlab + lo);
      a[t][1] = lds_load16(wl + t * 16 * kSlab + hi);
      as[t] = known ? lds_load1(sl + (XS * 64 + (wn * NT + t) * 16) * 16) : 0u;
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      x[b][0] = lds_load16(xl + b * 16 * kSlab + lo);
      x[b][1] = lds_load16(xl + b * 16 * kSlab + hi);
      xs[b] = known ? lds_load1(sl + (wm * MB + b) * 16 * 16) : 0u;
    }
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[t][b] = mfma_fp8(a[t][0], a[t][1], as[t], x[b][0], x[b][1], xs[b], acc[t][b]);
    before = buf;
    buf = buf + 1 == STAGES ? 0 : buf + 1;
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);  // (the loads past the end write to LDS)

  end_of_product<MB, NT, GLU, OUT8, SPLIT>(p, acc, col0, wn * NT, m0, wm * MB * 16, rows);
}

// The product into accumulation registers that stay where they are: 64 sums fill all of them, and
// left to choose, the compiler moves a quarter of the sums about in every slab.  The sums may be read 18
// cycles after the last of these at the earliest.
__device__ __forceinline__ void mfma_in_place(u32x4_t alo, u32x4_t ahi, uint32_t sa, u32x4_t blo, u32x4_t bhi, uint32_t sb,
                                              f32x4_t& c) {
#if defined(__HIP_DEVICE_COMPILE__)
  const i32x8_t x = {int(alo[0]), int(alo[1]), int(alo[2]), int(alo[3]), int(ahi[0]), int(ahi[1]), int(ahi[2]), int(ahi[3])};
  const i32x8_t y = {int(blo[0]), int(blo[1]), int(blo[2]), int(blo[3]), int(bhi[0]), int(bhi[1]), int(bhi[2]), int(bhi[3])};
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0]" : "+a"(c) : "v"(x), "v"(y), "v"(sa), "v"(sb));
#endif
}

// The largest blocks: 256 rows of x by 256 of W, four waves of 128 x 128, whose sums are half of
// a SIMD's registers.  One wave per SIMD hides nothing, so everything is read before its turn.
// A slab is four units of 128 rows (16 KB): the first and the second 64 of every wave's rows
// of W (W0, W1) and of x (X0, X1), and its products four phases of 16 instructions:
//   even slabs  X0 W0, X1 W0, X1 W1, X0 W1     odd slabs  X1 W0, X0 W0, X0 W1, X1 W1
// so that a unit's registers are free two phases before the next slab needs them, and each
// phase reads one unit from LDS for the next phase or the one after.  Units go through a ring of
// eight buffers, two slabs', in the order in which they are read (W0, X, X, W1): a phase
// waits for its unit, and after the barrier fills the buffer that the phase before has read,
// seven phases before that unit's turn.  Between two matrix instructions stands one read or load:
// an instruction leaves a wave seven issue slots, and what does not fit in them is lost.
template <bool GLU, bool OUT8>
__global__ __launch_bounds__(256) void wide_kernel(LinearParams p) {
  constexpr int HALVES = GLU ? 2 : 1, BM = 256, BN = 256, COLS = BN / HALVES;
  constexpr int UNITS = 8, UNIT = 128 * kSlab, SBYTES = 8 * 1024, LOADS = UNIT / 1024 / 4;
  static_assert(UNITS * UNIT + 2 * SBYTES <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[UNITS * UNIT + 2 * SBYTES];
  lds_t* const lds = (lds_t*)smem;
  lds_t* const scales = lds + UNITS * UNIT;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int wm = w / 2, wn = w % 2;
  const int g = lane >> 4, n = lane & 15;
  int col0;
  int64_t m0;
  place(p, BM, COLS, col0, m0);
  const int rows = int(min(int64_t(BM), p.rows - m0)), blocks = p.k / kBlock;
  const int wstride = int(p.w_stride), xstride = int(p.x_stride);
  const char* const xbase = p.x + m0 * p.x_stride;
  const char* const wbase = p.w + col0 * p.w_stride;
  const char* const ubase = p.w + (int64_t(p.n) + col0) * p.w_stride;
  const int xsize = (rows - 1) * xstride + p.k, wsize = (min(COLS, p.w_rows - col0) - 1) * wstride + p.k;
  const int usize = GLU ? (min(COLS, p.n - col0) - 1) * wstride + p.k : 0;
  // load i of a wave: 8 rows of a unit, lane l chunk slot l % 8 of row l / 8; rows r on of
  // wave `of`'s 64 of the unit
  const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 16;
  int xv[2][LOADS], wv[2][LOADS];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int of = w >> 1, r = (w & 1) * 32 + i * 8, tile = j * 4 + r / 16;
      xv[j][i] = (of * 128 + j * 64 + r + r8) * xstride + chunk;
      wv[j][i] = (of * (128 / HALVES) + tile / HALVES * 16 + r % 16 + r8) * wstride + chunk;
    }
  // The loads of a unit: of slab u / 4, W0, X, X, W1 (`part`).
  auto loads = [&](int slab, int part, int odd, int slot, auto each) {
    const int off = slab * kSlab;
    const bool ok = slab < p.slabs;
    lds_t* const to = lds + slot * UNIT + w * LOADS * 1024;
    const int past = off + chunk < p.k ? 0 : kOutOfRange;  // past the row's end lies the next row
    const bool of_x = part == 1 || part == 2;
    const int j = part == 1 ? odd : part == 2 ? 1 - odd : part == 3;
    const __amdgpu_buffer_rsrc_t rs = of_x ? buffer(xbase + off, ok ? xsize - off : 0) : buffer(wbase + off, ok ? wsize - off : 0);
    const __amdgpu_buffer_rsrc_t ru = GLU && !of_x ? buffer(ubase + off, ok ? usize - off : 0) : rs;
    each([=, &xv, &wv](int i) {
      lds_dma16(GLU && i / 2 ? ru : rs, to + i * 1024, (of_x ? xv[j][i] : wv[j][i]) | past);
    });
  };
  struct Set {
    u32x4_t v[4][2];
    uint32_t s[4];
  };
  // a lane's two chunks of row n of 16 (and 64 of `wave`'s rows of a unit)
  const lds_t* const xread = lds + wm * 64 * kSlab + n * kSlab;
  const lds_t* const wread = lds + wn * 64 * kSlab + n * kSlab;
  const int lo = (g ^ (n & 7)) * 16, hi = ((4 + g) ^ (n & 7)) * 16;
  const lds_t* const xr[2] = {xread + lo, xread + hi};
  const lds_t* const wr[2] = {wread + lo, wread + hi};
  const lds_t* const xsr = scales + (wm * 128 + n) * 16;
  const lds_t* const wsr = scales + (BM + wn * 128 + n) * 16;
  // Where a slab's scale bytes lie in a staged row: behind the last block (whose codes are
  // zeros) the last one's, since a row's padding may hold anything.
  auto scale_at = [&](int slab) { return (slab >> 2 & 1) * SBYTES + (slab & 3) * 4 + min(g, max(blocks - 1 - slab * 4, 0)); };

  f32x4_t acc[8][8];
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int b = 0; b < 8; ++b) acc[t][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  Set x[2], a[2];
  load_scales<4, BM, BN, GLU>(p, scales, 0, w, col0, m0, rows);
  load_scales<4, BM, BN, GLU>(p, scales + SBYTES, 1, w, col0, m0, rows);
#pragma unroll
  for (int u = 0; u < UNITS; ++u)
    loads(u / 4, u & 3, u / 4, u, [&](auto load) { for (int i = 0; i < LOADS; ++i) load(i); });
  constexpr int kFirst = (UNITS - 2) * LOADS;
  __builtin_amdgcn_s_waitcnt(0x0070 | (kFirst & 15) | (kFirst >> 4 << 14));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  const int s0 = scale_at(0);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      a[0].v[t][h] = lds_load16(wr[h] + t * 16 * kSlab);
      x[0].v[t][h] = lds_load16(xr[h] + UNIT + t * 16 * kSlab);
    }
    a[0].s[t] = lds_load1(wsr + s0 + t * 256);
    x[0].s[t] = lds_load1(xsr + s0 + t * 256);
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt: the first buffer is read
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  loads(2, 0, 0, 0, [&](auto load) { for (int i = 0; i < LOADS; ++i) load(i); });

  constexpr int kInFlight = (UNITS - 2) * LOADS;
  static_assert(kInFlight < 64, "vmcnt");
  // Phase P of a slab of parity ODD; `at`: the scales of the slab whose unit it reads.
  auto phase = [&]<int P, int ODD>(int slab, int at) {
    constexpr int XH = (P == 0 || P == 3) ? ODD : 1 - ODD, WH = P < 2 ? 0 : 1;  // halves multiplied
    // halves read: the slab's other x, its W1, the next slab's W0 and first x (by its parity)
    constexpr bool READ_X = P == 0 || P == 3;
    constexpr int HALF = P == 0 ? 1 - ODD : P == 1 ? 1 : P == 2 ? 0 : 1 - ODD;
    constexpr int SLOT = (4 * ODD + P + 2) % UNITS, BEFORE = (SLOT + UNITS - 1) % UNITS;
    // the unit seven behind: the part before this one's, two slabs on or, from its W0 back, one
    constexpr int PART = (P + 1) & 3, ON = P + 2 + UNITS - 1;
    __builtin_amdgcn_s_waitcnt(0x0070 | (kInFlight & 15) | (kInFlight >> 4 << 14));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    loads(slab + ON / 4, PART, ODD ^ (ON / 4 & 1), BEFORE, [&](auto load) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int t = e / 4, b = e % 4;
        mfma_in_place(a[WH].v[t][0], a[WH].v[t][1], a[WH].s[t], x[XH].v[b][0], x[XH].v[b][1], x[XH].s[b],
                      acc[WH * 4 + t][XH * 4 + b]);
        Set& to = READ_X ? x[HALF] : a[HALF];
        if (e < 8) to.v[e / 2][e % 2] = lds_load16((READ_X ? xr : wr)[e % 2] + SLOT * UNIT + e / 2 * 16 * kSlab);
        else if (e < 12) to.s[e - 8] = lds_load1((READ_X ? xsr : wsr) + at + (HALF * 64 + (e - 8) * 16) * 16);
        else load(e - 12);
        __builtin_amdgcn_sched_barrier(0);
      }
    });
  };
  auto slab_of = [&]<int ODD>(int slab) {
    if ((slab & 3) == 0 && slab)
      load_scales<4, BM, BN, GLU>(p, scales + ((slab >> 2) + 1 & 1) * SBYTES, (slab >> 2) + 1, w, col0, m0, rows);
    const int at = scale_at(slab), next = scale_at(slab + 1);
    phase.template operator()<0, ODD>(slab, at);
    phase.template operator()<1, ODD>(slab, at);
    phase.template operator()<2, ODD>(slab, next);
    phase.template operator()<3, ODD>(slab, next);
  };
  int slab = 0;
  for (; slab + 1 < p.slabs; slab += 2) {
    slab_of.template operator()<0>(slab);
    slab_of.template operator()<1>(slab + 1);
  }
  if (slab < p.slabs) slab_of.template operator()<0>(slab);
  __builtin_amdgcn_s_waitcnt(0x0070);  // (the loads past the end write to LDS)
  // (the last products' sums are written some cycles after their issue)
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int b = 0; b < 8; ++b) asm volatile("" : "+a"(acc[t][b]));
  end_of_product<8, 8, GLU, OUT8, false>(p, acc, col0, wn * 8, m0, wm * 128, rows);
}

// The sum of the parts in their order, and the end of the product.
template <bool GLU, bool OUT8>
__global__ __launch_bounds__(256) void combine_kernel(LinearParams p, int parts) {
  constexpr int HALVES = GLU ? 2 : 1;
  const int fours = (p.n + 3) / 4;
  const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x, one = p.rows * fours;
  if (at >= one) return;  // (8-bit: whole blocks of eight threads)
  f32x4_t sum = p.parts[at], up = {0.f, 0.f, 0.f, 0.f};
  if constexpr (GLU) up = p.parts[one + at];
#pragma unroll 4
  for (int i = 1; i < parts; ++i) {
    sum += p.parts[i * HALVES * one + at];
    if constexpr (GLU) up += p.parts[(i * HALVES + 1) * one + at];
  }
  const int col = int(at % fours) * 4;
  const int64_t row = at / fours;
  const f32x4_t v = finish<GLU>(sum, up, bias4(p, col));
  if constexpr (OUT8) {
    const uint32_t byte = scale_byte(max8(magnitude4(v)));
    *reinterpret_cast<uint32_t*>(p.out + row * p.o_stride + col) = to_codes(v[0], v[1], v[2], v[3], byte);
    if (col % kBlock == 0) p.scales[row * p.s_stride + col / kBlock] = uint8_t(byte);
  } else {
    store4(p, row, col, v);
  }
}

// ---------------------------------------------------------------- which form
struct Form {
  int rows, w_rows;
  float one_us, more_us;
  bool split;
};
constexpr Form kForms[] = {{64, 128, 0.45f, 0.45f, true}, {128, 128, 0.6f, 0.5f, true}, {256, 256, 1.5f, 1.5f, false}};
constexpr float kStartUs = 3.5f, kCombineUs = 2.5f, kBytesPerUs = 4.4e6f;
constexpr int kMaxParts = 32;

struct Choice {
  float us;
  int form, parts, split_slabs;
  size_t bytes;  // of the parts
};

// The fastest by that count within `room` bytes for parts.
Choice choose(bool glu, int64_t rows, int64_t n, int slabs, size_t room) {
  Choice best = {1e30f, 0, 1, slabs, 0};
  const int cus = mi::num_cus();
  for (int f = 0; f < int(sizeof(kForms) / sizeof(kForms[0])); ++f) {
    const Form& form = kForms[f];
    const int64_t cols = form.w_rows / (glu ? 2 : 1);
    const int64_t tiles = (rows + form.rows - 1) / form.rows * ((n + cols - 1) / cols);
    for (int want = 1; want <= (form.split ? kMaxParts : 1); ++want) {
      const int each = (slabs + want - 1) / want, parts = (slabs + each - 1) / each;
      if (parts != want || (want > 1 && (each < 2 || tiles * (want - 1) >= 2 * cus))) continue;
      const size_t bytes = want > 1 ? size_t(want) * (glu ? 2 : 1) * rows * ((n + 3) / 4) * 16 : 0;
      if (bytes > room) continue;
      const int64_t per_cu = (tiles * want + cus - 1) / cus;
      float us = kStartUs + each * (per_cu == 1 ? form.one_us : float(per_cu) * form.more_us);
      us += want > 1 ? kCombineUs + 2 * float(bytes) / kBytesPerUs : 2 * float(rows) * float(n) / kBytesPerUs;
      if (us < best.us) best = {us, f, want, each, bytes};
    }
  }
  return best;
}

template <int WM, int WN, int MB, int NT, int STAGES, bool GLU, bool OUT8, bool SPLIT>
void run(const LinearParams& p, int parts, hipStream_t stream) {
  constexpr int BM = WM * MB * 16, COLS = WN * NT * 16 / (GLU ? 2 : 1);
  const dim3 grid(uint32_t((p.rows + BM - 1) / BM * ((p.n + COLS - 1) / COLS)), parts);
  hipLaunchKernelGGL((many_kernel<WM, WN, MB, NT, STAGES, GLU, OUT8, SPLIT>), grid, dim3(64 * WM * WN), 0, stream, p);
}

template <bool GLU, bool OUT8, bool SPLIT>
void run_form(const LinearParams& p, int form, int parts, hipStream_t stream) {
  if (form == 0) run<1, 2, 4, 4, 4, GLU, OUT8, SPLIT>(p, parts, stream);
  else if (SPLIT || form == 1) run<2, 2, 4, 4, 4, GLU, OUT8, SPLIT>(p, parts, stream);
  else {
    constexpr int COLS = GLU ? 128 : 256;
    hipLaunchKernelGGL((wide_kernel<GLU, OUT8>), dim3(uint32_t((p.rows + 255) / 256 * ((p.n + COLS - 1) / COLS))), dim3(256), 0,
                       stream, p);
  }
}

template <bool GLU, bool OUT8>
void launch(const LinearParams& p, const Choice& c, hipStream_t stream) {
  LinearParams q = p;
  q.split_slabs = c.split_slabs;
  if (c.parts == 1) {
    run_form<GLU, OUT8, false>(q, c.form, 1, stream);
    return;
  }
  run_form<GLU, false, true>(q, c.form, c.parts, stream);
  const int64_t fours = p.rows * ((p.n + 3) / 4);
  hipLaunchKernelGGL((combine_kernel<GLU, OUT8>), dim3(uint32_t((fours + 255) / 256)), dim3(256), 0, stream, q, c.parts);
}

}  // namespace

// Whether the few-row kernel is the faster one.
bool few(int64_t rows) { return rows <= 64; }

size_t many_workspace(bool glu, int64_t rows, int64_t n, int slabs) {
  return choose(glu, rows, n, slabs, size_t(1) << 28).bytes;
}

void launch_many(const LinearParams& p, bool glu, size_t room, hipStream_t stream) {
  const Choice c = choose(glu, p.rows, p.n, p.slabs, room);
  if (!glu) launch<false, false>(p, c, stream);
  else p.scales ? launch<true, true>(p, c, stream) : launch<true, false>(p, c, stream);
}

}  // namespace mi::mx8

extern "C" size_t mi_linear_mxfp8_workspace_size(int64_t rows, int64_t n, int64_t k, int32_t silu) {
  using namespace mi::mx8;
  if (rows <= 0 || rows > kMaxRows || n <= 0 || n > kMaxN || k <= 0 || k % kBlock || k > kMaxK || few(rows)) return 0;
  return many_workspace(silu != 0, rows, n, int(slabs(k)));
}

extern "C" int mi_linear_mxfp8(const void* x_codes, int64_t x_stride, const void* x_scales, int64_t x_scales_stride,
                               const void* w_codes, int64_t w_stride, const void* w_scales, int64_t w_scales_stride,
                               const void* bias, void* out, int64_t out_stride, void* out_scales,
                               int64_t out_scales_stride, int64_t rows, int64_t n, int64_t k, int32_t silu,
                               void* workspace, size_t workspace_bytes, mi_stream_t stream) {
  using namespace mi::mx8;
  const char* const name = "linear_mxfp8";
  mi::clear_error();
  if (rows < 0 || rows > kMaxRows || n <= 0 || n > kMaxN || k <= 0 || k % kBlock || k > kMaxK)
    return mi::fail(MI_ERR_INVALID, "%s: rows %lld (0..2^22), n %lld (1..2^24), k %lld (multiple of %d, at most %d)", name,
                    (long long)rows, (long long)n, (long long)k, kBlock, kMaxK);
  if (silu && bias) return mi::fail(MI_ERR_INVALID, "%s: no bias with the gated product", name);
  if (out_scales && (!silu || n % kBlock))
    return mi::fail(MI_ERR_INVALID, "%s: rows in 8 bits are the gated product's, n a multiple of %d; got %lld", name, kBlock,
                    (long long)n);
  if (rows == 0) return MI_OK;
  const int64_t w_rows = silu ? 2 * n : n, blocks = k / kBlock, padded = (blocks + 15) & ~int64_t(15);
  // (nothing lies at a single row's stride)
  if (rows == 1) x_stride = (k + 15) & ~int64_t(15), x_scales_stride = padded, out_stride = n, out_scales_stride = n / kBlock;
  if (w_rows == 1) w_stride = (k + 15) & ~int64_t(15), w_scales_stride = padded;
  if (!x_codes || !x_scales || !w_codes || !w_scales || !out)
    return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  const uintptr_t aligned = reinterpret_cast<uintptr_t>(x_codes) | reinterpret_cast<uintptr_t>(x_scales) |
                            reinterpret_cast<uintptr_t>(w_codes) | reinterpret_cast<uintptr_t>(w_scales) |
                            reinterpret_cast<uintptr_t>(workspace);
  if ((aligned & 15) || ((x_stride | x_scales_stride | w_stride | w_scales_stride) & 15) ||
      ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 1) ||
      (out_scales && ((reinterpret_cast<uintptr_t>(out) & 15) || out_stride % 16)))
    return mi::fail(MI_ERR_INVALID, "%s: rows of codes and scales, and the workspace, must be 16-byte aligned", name);
  if (x_stride < k || w_stride < k || x_stride > kMaxStride || w_stride > kMaxStride || x_scales_stride < padded ||
      w_scales_stride < padded || x_scales_stride > kMaxStride || w_scales_stride > kMaxStride || out_stride < n ||
      (out_scales && out_scales_stride < n / kBlock))
    return mi::fail(MI_ERR_INVALID, "%s: row strides %lld, %lld, %lld, %lld (at most 2^22), %lld, %lld for k %lld, n %lld", name,
                    (long long)x_stride, (long long)x_scales_stride, (long long)w_stride, (long long)w_scales_stride,
                    (long long)out_stride, (long long)out_scales_stride, (long long)k, (long long)n);
  // (a workgroup's rows of out are written while others still read all of x, W and bias)
  const int64_t each = out_scales ? 1 : 2;
  const mi::Rows to[] = {{out, out_stride * each, rows, n * each},
                         {out_scales, out_scales_stride, out_scales ? rows : 0, n / kBlock}};
  const mi::Rows from[] = {{x_codes, x_stride, rows, k}, {x_scales, x_scales_stride, rows, blocks},
                           {w_codes, w_stride, w_rows, k}, {w_scales, w_scales_stride, w_rows, blocks},
                           {bias, 0, bias ? 1 : 0, n * 2}};
  bool meet = mi::rows_meet(to[0], to[1]);
  for (const mi::Rows& o : to)
    for (const mi::Rows& r : from) meet = meet || mi::rows_meet(o, r);
  if (meet) return mi::fail(MI_ERR_INVALID, "%s: out overlaps x, the weight, the bias or its own scales", name);
  LinearParams p;
  p.x = static_cast<const char*>(x_codes);
  p.x_stride = x_stride;
  p.xs = static_cast<const char*>(x_scales);
  p.xs_stride = x_scales_stride;
  p.w = static_cast<const char*>(w_codes);
  p.w_stride = w_stride;
  p.ws = static_cast<const char*>(w_scales);
  p.ws_stride = w_scales_stride;
  p.bias = static_cast<const uint16_t*>(bias);
  p.out = static_cast<char*>(out);
  p.o_stride = out_stride;
  p.scales = static_cast<uint8_t*>(out_scales);
  p.s_stride = out_scales_stride;
  p.rows = rows;
  p.n = int(n);
  p.k = int(k);
  p.w_rows = int(w_rows);
  p.slabs = int(slabs(k));
  p.parts = static_cast<mi::f32x4_t*>(workspace);
  p.split_slabs = p.slabs;
  p.vec = n % 4 == 0 && out_stride % 4 == 0 &&
          ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 7) == 0;
  p.wide = p.vec && n % 8 == 0 && out_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (few(rows)) launch_few(p, silu != 0, s);
  else launch_many(p, silu != 0, workspace ? workspace_bytes : 0, s);
  return mi::check_launch(name);
}

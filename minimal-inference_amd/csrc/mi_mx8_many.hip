// Projections of many rows with both operands in MXFP8 (prompts): out = x W^T (+ bias) or
// silu(x Wg^T) * (x Wu^T), fp32 accumulation and one rounding.
//
// Bound: the matrix instructions.  A workgroup of four waves owns a block of out; per slab
// of 128 k its rows of W and of x go straight from memory to LDS, into a ring of buffers,
// and from there, as operands, to the waves.  A row of a slab is 128 bytes, eight chunks whose
// places are permuted by the row, so that the rows an operand read touches together fall on
// distinct banks.  The scale bytes of four slabs (16 bytes a row) are staged alike.
#include <algorithm>

#include "mi_mx8_linear.h"
#include "mi_overlap.h"

namespace mi::mx8 {
namespace {

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
    // (non-temporal, us: 16,384 x 4,096 x 2 x 14,336 1,807 -> 1,602, with the adapters that read them 2,340 -> 2,247;
    // 512 rows 92 -> 96, 100 rows the same)
    if (p.sums) {
#pragma unroll
      for (int t = 0; t < NT; t += 2)
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          const int m = row0 + b * 16 + n, col = col0 + (first_tile + t) / 2 * 16 + 4 * g;
          if (m < rows && col < p.n) store_sums<true>(p, m0 + m, col, acc[t][b], acc[t + 1][b]);
        }
      return;
    }
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
  // bytes of a row.  All CUs come here at once and out is not read before the launch's end: stores
  // that L2 need not keep (us, 40,960 x 4,096 x 4,096 537 -> 512, none at all 477; 1,024 x 4,096 x 4,096 24.5 -> 23.5).
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
            __builtin_nontemporal_store(
                u32x4_t{s0[0], s1[0], s0[1], s1[1]},
                reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(p.out) + (m0 + m) * p.o_stride + col));
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
// eight buffers, two slabs', in the order in which they are read (W0, X, X, W1): every
// second phase waits for its unit and the next, and after the barrier the two phases fill
// the buffers that the two before have read, six phases before those units' turn.  Between
// two matrix instructions stand two reads or a load: an instruction leaves a wave seven issue
// slots, and what does not fit in them is lost.
// (us, 8,192 x 8,192 x 10,240 of normal values: two whole slabs staged and read at once 649;
// these phases with addresses computed in place 649, with constants and pinned sums 503, a
// barrier in every second phase 485; all of it in L2 462, without the reads from LDS 459, without the loads
// 421, without both 379, where products alone would take 314.  Zeros 413: the clock follows the power
// that products and data take.  Workgroups that go from block to block, the next one's first loads under the
// last one's stores, were no faster: 500 / 498.)
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

  constexpr int kInFlight = (UNITS - 4) * LOADS;
  static_assert(kInFlight < 64, "vmcnt");
  // Phase P of a slab of parity ODD; `at`: the scales of the slab whose unit it reads.
  auto phase = [&]<int P, int ODD>(int slab, int at) {
    constexpr int XH = (P == 0 || P == 3) ? ODD : 1 - ODD, WH = P < 2 ? 0 : 1;  // halves multiplied
    // halves read: the slab's other x, its W1, the next slab's W0 and first x (by its parity)
    constexpr bool READ_X = P == 0 || P == 3;
    constexpr int HALF = P == 0 ? 1 - ODD : P == 1 ? 1 : P == 2 ? 0 : 1 - ODD;
    constexpr int SLOT = (4 * ODD + P + 2) % UNITS, BEFORE = (SLOT + UNITS - 2) % UNITS;
    if constexpr (P % 2 == 0) {
      __builtin_amdgcn_s_waitcnt(0x0070 | (kInFlight & 15) | (kInFlight >> 4 << 14));
      __builtin_amdgcn_s_barrier();
    }
    __builtin_amdgcn_sched_barrier(0);
    loads(slab + 2, P, ODD, BEFORE, [&](auto load) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int t = e / 4, b = e % 4;
        mfma_in_place(a[WH].v[t][0], a[WH].v[t][1], a[WH].s[t], x[XH].v[b][0], x[XH].v[b][1], x[XH].s[b],
                      acc[WH * 4 + t][XH * 4 + b]);
        Set& to = READ_X ? x[HALF] : a[HALF];
        if (e < 4) {
          to.v[e][0] = lds_load16((READ_X ? xr : wr)[0] + SLOT * UNIT + e * 16 * kSlab);
          to.v[e][1] = lds_load16((READ_X ? xr : wr)[1] + SLOT * UNIT + e * 16 * kSlab);
        } else if (e < 8) to.s[e - 4] = lds_load1((READ_X ? xsr : wsr) + at + (HALF * 64 + (e - 4) * 16) * 16);
        else if (e < 12) load(e - 8);
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

// Blocks of 128 rows of x by 128 of W, four waves of 64 x 64: as wide_kernel, with one unit of x and
// one of W to a slab, one phase, and one barrier.  The products of slab s read from LDS the
// units of s + 1, into registers of their own; after the barrier of slab s the buffers are
// filled again that slab s - 1 has read, four slabs ahead.
//
// Bound: the operands' way, 32 KB for 16 products a wave, and what lies beyond L2 of it: 0.61 us a slab, with
// all of it in L2 0.42 (1,024 x 4,096 x 4,096 24.0 and 18.3 us; 2,048 x 8,192 x 10,240 212, without the
// loads 133, without the reads from LDS 208).  LDS has no room for more slabs ahead.
//
// SPLIT: the workgroup takes p.split_slabs slabs (a multiple of four) and leaves its sums, in
// fp32, for combine_kernel.
template <bool GLU, bool OUT8, bool SPLIT>
__global__ __launch_bounds__(256) void block_kernel(LinearParams p) {
  constexpr int HALVES = GLU ? 2 : 1, BM = 128, BN = 128, COLS = BN / HALVES;
  constexpr int RING = 4, UNIT = 128 * kSlab, SBYTES = (BM + BN) * 16, LOADS = UNIT / 1024 / 4;
  static_assert(RING * 2 * UNIT + 2 * SBYTES <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[RING * 2 * UNIT + 2 * SBYTES];
  lds_t* const lds = (lds_t*)smem;
  lds_t* const scales = lds + RING * 2 * UNIT;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int wm = w / 2, wn = w % 2;
  const int g = lane >> 4, n = lane & 15;
  int col0;
  int64_t m0;
  place(p, BM, COLS, col0, m0);
  const int rows = int(min(int64_t(BM), p.rows - m0)), blocks = p.k / kBlock;
  const int slab0 = SPLIT ? int(blockIdx.y) * p.split_slabs : 0;
  const int slab_end = SPLIT ? min(slab0 + p.split_slabs, p.slabs) : p.slabs;
  const int wstride = int(p.w_stride), xstride = int(p.x_stride);
  // load i of a wave: 8 rows of a unit, lane l chunk slot l % 8 of row l / 8
  const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 16;
  int xv[LOADS], wv[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int of = w >> 1, r = (w & 1) * 32 + i * 8;
    xv[i] = (of * 64 + r + r8) * xstride + chunk;
    wv[i] = (of * (64 / HALVES) + r / 16 / HALVES * 16 + r % 16 + r8) * wstride + chunk;
  }
  const char* const xbase = p.x + m0 * p.x_stride;
  const char* const wbase = p.w + col0 * p.w_stride;
  const char* const ubase = p.w + (int64_t(p.n) + col0) * p.w_stride;
  const int xsize = (rows - 1) * xstride + p.k, wsize = (min(COLS, p.w_rows - col0) - 1) * wstride + p.k;
  const int usize = GLU ? (min(COLS, p.n - col0) - 1) * wstride + p.k : 0;
  struct Source {
    __amdgpu_buffer_rsrc_t first, second;  // the rows of a unit's first two loads and of the others
    int past;
  };
  auto source = [&](int slab, bool of_x) {
    const int off = slab * kSlab;
    const bool ok = slab < slab_end;
    const __amdgpu_buffer_rsrc_t r = of_x ? buffer(xbase + off, ok ? xsize - off : 0) : buffer(wbase + off, ok ? wsize - off : 0);
    const __amdgpu_buffer_rsrc_t u = GLU && !of_x ? buffer(ubase + off, ok ? usize - off : 0) : r;
    return Source{r, u, off + chunk < p.k ? 0 : kOutOfRange};  // past the row's end lies the next row
  };
  // Load i of a slab's unit (0: x, 1: W) into place `ring` of the ring.
  auto load = [&](const Source& s, int unit, int ring, int i) {
    lds_dma16(i / 2 ? s.second : s.first, lds + (ring * 2 + unit) * UNIT + (w * LOADS + i) * 1024, (unit ? wv[i] : xv[i]) | s.past);
  };
  auto load_slab = [&](int slab, int ring) {
    const Source sx = source(slab, true), sw = source(slab, false);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(sx, 0, ring, i);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(sw, 1, ring, i);
  };
  struct Set {
    u32x4_t v[4][2];
    uint32_t s[4];
  };
  const int lo = n * kSlab + (g ^ (n & 7)) * 16, hi = n * kSlab + ((4 + g) ^ (n & 7)) * 16;
  const lds_t* const xr[2] = {lds + wm * 64 * kSlab + lo, lds + wm * 64 * kSlab + hi};
  const lds_t* const wr[2] = {lds + wn * 64 * kSlab + lo, lds + wn * 64 * kSlab + hi};
  const lds_t* const xsr = scales + (wm * 64 + n) * 16;
  const lds_t* const wsr = scales + (BM + wn * 64 + n) * 16;
  // Where a slab's scale bytes lie in a staged row: behind the last block (whose codes are
  // zeros) the last one's, since a row's padding may hold anything.
  auto scale_at = [&](int slab) { return (slab >> 2 & 1) * SBYTES + (slab & 3) * 4 + min(g, max(blocks - 1 - slab * 4, 0)); };
  // Read e of 12 of a unit: eight of operands, four of scales.
  auto read = [&](Set& to, int unit, int ring, int at, int e) {
    if (e < 8) to.v[e / 2][e % 2] = lds_load16((unit ? wr : xr)[e % 2] + (ring * 2 + unit) * UNIT + e / 2 * 16 * kSlab);
    else to.s[e - 8] = lds_load1((unit ? wsr : xsr) + at + (e - 8) * 256);
  };

  f32x4_t acc[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[t][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  Set x[2], a[2];
  load_scales<4, BM, BN, GLU>(p, scales + (slab0 >> 2 & 1) * SBYTES, slab0 >> 2, w, col0, m0, rows);
  load_scales<4, BM, BN, GLU>(p, scales + ((slab0 >> 2) + 1 & 1) * SBYTES, (slab0 >> 2) + 1, w, col0, m0, rows);
#pragma unroll
  for (int i = 0; i < RING; ++i) load_slab(slab0 + i, i);
  constexpr int kFirst = (RING - 1) * 2 * LOADS, kInFlight = (RING - 2) * 2 * LOADS;
  static_assert(kFirst < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt(0x0070 | (kFirst & 15) | (kFirst >> 4 << 14));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  int at = scale_at(slab0);
#pragma unroll
  for (int e = 0; e < 12; ++e) {
    read(x[0], 0, 0, at, e);
    read(a[0], 1, 0, at, e);
  }
  auto slab_of = [&]<int I>(int slab) {
    constexpr int HERE = I & 1, NEXT = 1 - HERE, RNEXT = (I + 1) % RING;
    __builtin_amdgcn_s_waitcnt(0x0070 | (kInFlight & 15) | (kInFlight >> 4 << 14));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    int at_next = 0;
    Source sx, sw;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int t = e / 4, b = e % 4;
      mfma_in_place(a[HERE].v[t][0], a[HERE].v[t][1], a[HERE].s[t], x[HERE].v[b][0], x[HERE].v[b][1], x[HERE].s[b], acc[t][b]);
      if (e == 2) sx = source(slab + RING, true);
      if (e == 4) sw = source(slab + RING, false);
      if (e == 6) at_next = scale_at(slab + 1);
      if (e < 12) {
        read(x[NEXT], 0, RNEXT, at_next, e);
        read(a[NEXT], 1, RNEXT, at_next, e);
      }
      if (e >= 8 && e < 12) load(sx, 0, I, e - 8);
      if (e >= 12) load(sw, 1, I, e - 12);
      __builtin_amdgcn_sched_barrier(0);
    }
    if ((slab & 3) == 0 && slab != slab0)  // (three slabs ahead: done by the waits before them)
      load_scales<4, BM, BN, GLU>(p, scales + ((slab >> 2) + 1 & 1) * SBYTES, (slab >> 2) + 1, w, col0, m0, rows);
    at = at_next;
  };
  for (int slab = slab0;;) {
    slab_of.template operator()<0>(slab);
    if (++slab >= slab_end) break;
    slab_of.template operator()<1>(slab);
    if (++slab >= slab_end) break;
    slab_of.template operator()<2>(slab);
    if (++slab >= slab_end) break;
    slab_of.template operator()<3>(slab);
    if (++slab >= slab_end) break;
  }
  __builtin_amdgcn_s_waitcnt(0x0070);  // (the loads past the end write to LDS)
  // (the last products' sums are written some cycles after their issue)
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int b = 0; b < 4; ++b) asm volatile("" : "+a"(acc[t][b]));
  end_of_product<4, 4, GLU, OUT8, SPLIT>(p, acc, col0, wn * 4, m0, wm * 64, rows);
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
    if (p.sums) return store_sums(p, row, col, sum, up);
    const uint32_t byte = scale_byte(max8(magnitude4(v)));
    *reinterpret_cast<uint32_t*>(p.out + row * p.o_stride + col) = to_codes(v[0], v[1], v[2], v[3], byte);
    if (col % kBlock == 0) p.scales[row * p.s_stride + col / kBlock] = uint8_t(byte);
  } else {
    store4(p, row, col, v);
  }
}

// ---------------------------------------------------------------- which form
// The time of a launch, counted: its start, and for every round of workgroups their own start and end
// and a slab's time for every slab; of the largest blocks the last round is the faster, the fewer CUs it
// takes (they share the power), of the others where another round has left W in the caches.  Workgroups
// that share k add the combining launch with the parts' way to memory and back.  Counted and measured (us,
// calls in a graph): 8,192 x 8,192 x 10,240 wide 482 / 491, 2,048 x 8,192 x 10,240 wide 178 / 173, block 209 / 207;
// 18,240 x 4,096 x 6,144 wide 356 / 349; 1,000 x 4,096 x 6,144 wide 47 / 45, block 43 / 45; 700 rows of it block
// 41 / 37, wide 46 / 45; 600 x 14,336 x 4,096 block 74 / 74, in 3 parts 71 / 70, wide 137 / 131; 512 x 3,584 x
// 4,608 block 23 / 23; 200 x 4,096 x 6,144 block 25 / 23, in 2 parts 22 / 21; 77 x 18,944 x 3,584 in 8 parts
// 24 / 27, whole 96 / 89; 128 x 4,096 x 4,096 in 4 parts 17 / 19.  (Blocks of 128 x 256 were no faster than
// either in any of these, nor two workgroups of 128 x 128 on a CU.)
constexpr float kStartUs = 3.5f, kCombineUs = 2.5f, kBytesPerUs = 4.4e6f;
constexpr int kMaxParts = 32;
enum class Form { few, block, wide };

struct Choice {
  float us;
  Form form;
  int parts, split_slabs;
  size_t bytes;  // of the parts
  int64_t rest;  // rows behind the last whole block, for a launch of their own
};

// A slab of a round on every CU takes least + more.
float rounds_us(int64_t workgroups, int slabs, float own, float least, float more, bool first_is_whole) {
  const int cus = mi::num_cus();
  const int64_t whole = workgroups / cus, last = workgroups % cus;
  const float part = first_is_whole && !whole ? 1.f : float(last) / float(cus);
  return kStartUs + float(whole) * (own + slabs * (least + more)) + (last ? own + slabs * (least + more * part) : 0.f);
}
float wide_us(int64_t workgroups, int slabs) { return rounds_us(workgroups, slabs, 6.f, 1.05f, 0.35f, false); }
float block_us(int64_t workgroups, int slabs) { return rounds_us(workgroups, slabs, 2.f, 0.41f, 0.2f, true); }
// The few-row kernel's (up to 64 rows): W's bytes from memory, x's into every workgroup.
float few_us(int64_t rows, int64_t w_rows, int slabs) {
  const float k = float(slabs) * kSlab, workgroups = std::max(1.f, float(w_rows) / 64);
  return kStartUs + float(w_rows) * k * 33 / 32 / 5.2e6f + float(rows) * k * workgroups / 15e6f;
}

// The fastest by that count within `room` bytes for parts.
Choice choose(bool glu, int64_t rows, int64_t n, int slabs, size_t room) {
  if (rows <= kFewRows) return {0.f, Form::few, 1, slabs, 0, 0};
  const int64_t w_rows = glu ? 2 * n : n, across = (w_rows + 255) / 256;
  Choice best = {wide_us((rows + 255) / 256 * across, slabs), Form::wide, 1, slabs, 0, 0};
  // (8,201 x 8,192 x 10,240: 33 rows of blocks are a round more than 32 and a launch of nine rows)
  if (const int64_t rest = rows % 256; rest && rest <= kFewRows && rest < rows) {
    const float us = wide_us(rows / 256 * across, slabs) + few_us(rest, w_rows, slabs);
    if (us < best.us) best.us = us, best.rest = rest;
  }
  const int64_t block = (rows + 127) / 128 * ((w_rows + 127) / 128);
  for (int want = 1; want <= kMaxParts; ++want) {
    const int each = want == 1 ? slabs : ((slabs + want - 1) / want + 3) / 4 * 4, parts = (slabs + each - 1) / each;
    if (parts != want || (want > 1 && block * (want - 1) >= 2 * mi::num_cus())) continue;
    const size_t bytes = want > 1 ? size_t(want) * (glu ? 2 : 1) * rows * ((n + 3) / 4) * 16 : 0;
    if (bytes > room) continue;
    const float us = block_us(block * want, each) + (want > 1 ? kCombineUs + 2 * float(bytes) / kBytesPerUs : 0.f);
    if (us < best.us) best = {us, Form::block, want, each, bytes, 0};
  }
  return best;
}

template <bool GLU, bool OUT8>
void launch(const LinearParams& p, const Choice& c, hipStream_t stream) {
  const int size = c.form == Form::wide ? 256 : 128, cols = size / (GLU ? 2 : 1);
  const dim3 grid(uint32_t((p.rows + size - 1) / size * ((p.n + cols - 1) / cols)), c.parts), block(256);
  LinearParams q = p;
  q.split_slabs = c.split_slabs;
  if (c.form == Form::wide) {
    hipLaunchKernelGGL((wide_kernel<GLU, OUT8>), grid, block, 0, stream, q);
  } else if (c.parts == 1) {
    hipLaunchKernelGGL((block_kernel<GLU, OUT8, false>), grid, block, 0, stream, q);
  } else {
    hipLaunchKernelGGL((block_kernel<GLU, false, true>), grid, block, 0, stream, q);
    launch_combine(q, GLU, c.parts, stream);
  }
}

}  // namespace

void launch_combine(const LinearParams& p, bool glu, int parts, hipStream_t stream) {
  const int64_t fours = p.rows * ((p.n + 3) / 4);
  const dim3 grid(uint32_t((fours + 255) / 256)), block(256);
  if (!glu) hipLaunchKernelGGL((combine_kernel<false, false>), grid, block, 0, stream, p, parts);
  else if (p.scales || p.sums) hipLaunchKernelGGL((combine_kernel<true, true>), grid, block, 0, stream, p, parts);
  else hipLaunchKernelGGL((combine_kernel<true, false>), grid, block, 0, stream, p, parts);
}

void launch_many(const LinearParams& p, bool glu, const Choice& c, hipStream_t stream) {
  LinearParams q = p;
  q.rows = p.rows - c.rest;
  if (!glu) launch<false, false>(q, c, stream);
  else p.scales || p.sums ? launch<true, true>(q, c, stream) : launch<true, false>(q, c, stream);
  if (!c.rest) return;
  LinearParams rest = p;
  rest.rows = c.rest;
  rest.x += q.rows * p.x_stride;
  rest.xs += q.rows * p.xs_stride;
  rest.out += q.rows * p.o_stride * (p.scales ? 1 : 2);
  if (p.scales) rest.scales += q.rows * p.s_stride;
  if (p.sums) rest.sums += q.rows * p.sums_stride;
  launch_few(rest, glu, 0, stream);
}

}  // namespace mi::mx8

extern "C" size_t mi_linear_mxfp8_workspace_size(int64_t rows, int64_t n, int64_t k, int32_t silu) {
  using namespace mi::mx8;
  if (rows <= 0 || rows > kMaxRows || n <= 0 || n > kMaxN || k <= 0 || k % kBlock || k > kMaxK) return 0;
  const size_t room = size_t(1) << 28;
  if (rows <= kFewRows) return few_workspace(silu != 0, rows, n, int(slabs(k)), room);
  return choose(silu != 0, rows, n, int(slabs(k)), room).bytes;
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
  const bool sums = silu == MI_SILU_SUMS;
  if (sums && (out_scales || n % 4))
    return mi::fail(MI_ERR_INVALID, "%s: sums are fp32, a multiple of 4 columns each; got %lld", name, (long long)n);
  if (out_scales && (!silu || n % kBlock))
    return mi::fail(MI_ERR_INVALID, "%s: rows in 8 bits are the gated product's, n a multiple of %d; got %lld", name, kBlock,
                    (long long)n);
  if (rows == 0) return MI_OK;
  const int64_t w_rows = silu ? 2 * n : n, blocks = k / kBlock, padded = (blocks + 15) & ~int64_t(15);
  // (nothing lies at a single row's stride)
  const int64_t out_n = sums ? 2 * n : n;
  if (rows == 1) x_stride = (k + 15) & ~int64_t(15), x_scales_stride = padded, out_stride = out_n, out_scales_stride = n / kBlock;
  if (w_rows == 1) w_stride = (k + 15) & ~int64_t(15), w_scales_stride = padded;
  if (!x_codes || !x_scales || !w_codes || !w_scales || !out)
    return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  const uintptr_t aligned = reinterpret_cast<uintptr_t>(x_codes) | reinterpret_cast<uintptr_t>(x_scales) |
                            reinterpret_cast<uintptr_t>(w_codes) | reinterpret_cast<uintptr_t>(w_scales) |
                            reinterpret_cast<uintptr_t>(workspace);
  if ((aligned & 15) || ((x_stride | x_scales_stride | w_stride | w_scales_stride) & 15) ||
      ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 1) ||
      (out_scales && ((reinterpret_cast<uintptr_t>(out) & 15) || out_stride % 16)) ||
      (sums && ((reinterpret_cast<uintptr_t>(out) & 15) || out_stride % 4)))
    return mi::fail(MI_ERR_INVALID, "%s: rows of codes and scales, and the workspace, must be 16-byte aligned", name);
  if (x_stride < k || w_stride < k || x_stride > kMaxStride || w_stride > kMaxStride || x_scales_stride < padded ||
      w_scales_stride < padded || x_scales_stride > kMaxStride || w_scales_stride > kMaxStride || out_stride < out_n ||
      (out_scales && out_scales_stride < n / kBlock))
    return mi::fail(MI_ERR_INVALID, "%s: row strides %lld, %lld, %lld, %lld (at most 2^22), %lld, %lld for k %lld, n %lld", name,
                    (long long)x_stride, (long long)x_scales_stride, (long long)w_stride, (long long)w_scales_stride,
                    (long long)out_stride, (long long)out_scales_stride, (long long)k, (long long)n);
  // (a workgroup's rows of out are written while others still read all of x, W and bias)
  const int64_t each = out_scales ? 1 : sums ? 4 : 2;
  const mi::Rows to[] = {{out, out_stride * each, rows, out_n * each},
                         {out_scales, out_scales_stride, out_scales ? rows : 0, n / kBlock}};
  const mi::Rows from[] = {{x_codes, x_stride, rows, k}, {x_scales, x_scales_stride, rows, blocks},
                           {w_codes, w_stride, w_rows, k}, {w_scales, w_scales_stride, w_rows, blocks},
                           {bias, 0, bias ? 1 : 0, n * 2}};
  bool meet = mi::rows_meet(to[0], to[1]);
  for (const mi::Rows& o : to)
    for (const mi::Rows& r : from) meet = meet || mi::rows_meet(o, r);
  if (meet) return mi::fail(MI_ERR_INVALID, "%s: out overlaps x, the weight, the bias or its own scales", name);
  // (parts are written while others still read x and W, and read while out is written)
  const size_t room = workspace ? workspace_bytes : 0;
  const Choice choice = choose(silu != 0, rows, n, int(slabs(k)), room);
  if (const size_t bytes = choice.form == Form::few ? few_workspace(silu != 0, rows, n, int(slabs(k)), room) : choice.bytes) {
    const mi::Rows parts = {workspace, 0, 1, int64_t(bytes)};
    for (const mi::Rows& r : to) meet = meet || mi::rows_meet(parts, r);
    for (const mi::Rows& r : from) meet = meet || mi::rows_meet(parts, r);
    if (meet) return mi::fail(MI_ERR_INVALID, "%s: the workspace overlaps another argument", name);
  }
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
  p.sums = sums ? static_cast<float*>(out) : nullptr;
  p.sums_stride = out_stride;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (choice.form == Form::few) launch_few(p, silu != 0, room, s);
  else launch_many(p, silu != 0, choice, s);
  return mi::check_launch(name);
}

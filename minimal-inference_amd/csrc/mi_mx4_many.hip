// Projections of many rows with an MXFP4 weight (prompts): out = x W^T (+ bias) or
// silu(x Wg^T) * (x Wu^T), fp32 accumulation and one rounding; x bf16 or MXFP4.
//
// Bound: the matrix instructions.  A workgroup of WM x WN waves owns a block of out;
// per slab of 128 k its tiles of W and of x go straight from memory to LDS (one of two
// buffers, the next slab's while this one is multiplied) and from there, as operands,
// to the waves.  MXFP4 tiles are operands as they lie; the codes of W become bf16 in
// registers, exactly, where x is bf16, whose rows are staged with permuted chunks.
#include <algorithm>

#include "mi_mx4_linear.h"
#include "mi_overlap.h"

namespace mi::mx4 {
namespace {

__device__ __forceinline__ void lds_dma16(__amdgpu_buffer_rsrc_t rs, lds_t* dst, int voffset) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, voffset, 0, 0, 0);
#endif
}

constexpr int kGroupM = 4;

// MB blocks of 16 rows of x and NT tiles of W per wave.  Slabs are staged STAGES deep:
// before slab s is multiplied the loads of the STAGES - 2 slabs behind it may be in
// flight, and after the barrier its predecessor's buffer is filled again.  Loads past
// the last slab are out of range, so that every wait counts the same loads.
//
// AHEAD (the largest blocks of MXFP4 rows): four waves of 128 x 128 read 16 operands for 64
// products, where eight of 128 x 64 read 12 for 32 and LDS could feed no more; the next
// slab's tiles of W, and tiles of x AHEAD blocks before their turn, are read between the
// products, whose sums fill the half of a SIMD's registers that the operands leave free.
// (8,192 x 8,192 x 10,240, operands read at a slab's begin: eight waves 346 us, four 342; so
// 316.)
//
// SPLIT: the workgroup takes p.split_slabs slabs and leaves its sums, in fp32, for
// combine_kernel.
template <int WM, int WN, int MB, int NT, int STAGES, bool MX, bool GLU, bool SPLIT, int AHEAD = 0>
__global__ __launch_bounds__(64 * WM * WN) void many_kernel(LinearParams p) {
  constexpr int WAVES = WM * WN, HALVES = GLU ? 2 : 1;
  constexpr int XBLK = MX ? kTileBytes : 16 * kSlab * 2;  // 16 rows of x of a slab
  constexpr int BM = WM * MB * 16, TILES = WN * NT, COLS = TILES * 16 / HALVES;
  constexpr int XBYTES = WM * MB * XBLK, STAGE = XBYTES + TILES * kTileBytes;
  constexpr int XLOADS = XBYTES / 1024 / WAVES, WLOADS = TILES / WAVES;
  static_assert(XBYTES / 1024 % WAVES == 0 && TILES % WAVES == 0 && NT % HALVES == 0, "even shares");
  static_assert(STAGES * STAGE <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[STAGES * STAGE];
  lds_t* const lds = (lds_t*)smem;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int wm = w / WN, wn = w % WN;
  const int g = lane >> 4, n = lane & 15;
  // Workgroups go to the eight XCDs in turn.  Each XCD gets a run of tiles, in groups of
  // kGroupM down the rows of x, so that those it holds at a time share tiles of x and of
  // W in its L2.  (us, 8,192 x 8,192 x 10,240 in 4 bits: groups of 64 376, 16 354, 8 344,
  // 4 345; 4,096 x 4,096 x 6,144 bf16 169, 164, 161, 157.)
  const int mt = int((p.rows + BM - 1) / BM), nt = (p.n + COLS - 1) / COLS, all = mt * nt;
  const int id = int(blockIdx.x), xcd = id & 7, each = all / 8, more = all % 8;
  const int tile_id = xcd * each + min(xcd, more) + (id >> 3);
  const int group = tile_id / (kGroupM * nt), in = tile_id - group * kGroupM * nt;
  const int high = min(kGroupM, mt - group * kGroupM);
  const int col0 = in / high * COLS;
  const int64_t m0 = int64_t(group * kGroupM + in % high) * BM;
  const int rows = int(min(int64_t(BM), p.rows - m0));
  const int slab0 = SPLIT ? int(blockIdx.y) * p.split_slabs : 0;
  const int slab_end = SPLIT ? min(slab0 + p.split_slabs, p.slabs) : p.slabs;

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
    // load i: 4 rows, lane l slot l % 16 of row l / 16
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) {
      const int row = (w * XLOADS + i) * 4 + (lane >> 4);
      xv[i] = row * stride + chunk_slot(row, lane & 15) * 16;
    }
  }
  // a lane's k of its even and odd loads: a row's permutation depends on it modulo 8
  const int xk[2] = {chunk_slot(w * XLOADS * 4 + (lane >> 4), lane & 15) * 16,
                     chunk_slot(w * XLOADS * 4 + 4 + (lane >> 4), lane & 15) * 16};
  auto load = [&](int slab, int buf) {
    lds_t* const stage = lds + buf * STAGE;
    const bool ok = slab < slab_end;
    const int off = MX ? slab * kTileBytes : slab * kSlab * 2;
    const __amdgpu_buffer_rsrc_t rx = buffer(xbase + off, ok ? xsize - off : 0);
#pragma unroll
    for (int i = 0; i < XLOADS; ++i) {
      int v = xv[i];
      if constexpr (!MX) v = off + xk[i & 1] < p.k * 2 ? v : 0x7ffffff0;  // past the row's end lies the next row
      lds_dma16(rx, stage + (w * XLOADS + i) * 1024, v);
    }
    __amdgpu_buffer_rsrc_t rw[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h)
      rw[h] = buffer(wbase[h] + slab * kTileBytes, ok ? wsize[h] - slab * kTileBytes : 0);
#pragma unroll
    for (int i = 0; i < WLOADS; ++i)
      lds_dma16(rw[(w * WLOADS + i) % HALVES], stage + XBYTES + (w * WLOADS + i) * kTileBytes, wv[i]);
  };
  uint32_t wnext[NT], xnext[MX ? MB : 1];
  auto load_scales = [&](int quad) {
    const bool ok = quad < p.quads;
    const int off = quad * kQuadBytes;
    __amdgpu_buffer_rsrc_t rs[HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) rs[h] = buffer(sbase[h] + off, ok ? ssize[h] - off : 0);
#pragma unroll
    for (int t = 0; t < NT; ++t) wnext[t] = __builtin_amdgcn_raw_buffer_load_b32(rs[t % HALVES], wsv[t], 0, 0);
    if constexpr (MX) {
      const __amdgpu_buffer_rsrc_t rx = buffer(xsbase + off, ok ? xssize - off : 0);
#pragma unroll
      for (int b = 0; b < MB; ++b)
        xnext[b] = __builtin_amdgcn_raw_buffer_load_b32(rx, (wm * MB + b) * p.quads * kQuadBytes + lane * 4, 0, 0);
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

  constexpr int kInFlight = (STAGES - (AHEAD ? 3 : 2)) * (XLOADS + WLOADS);
  static_assert(kInFlight < 64, "vmcnt");
  load_scales(slab0 >> 2);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) load(slab0 + i, i);
  int buf = 0, before = STAGES - 1;
  if constexpr (AHEAD) {
    static_assert(MX && !SPLIT && NT == MB && STAGES > 3);
    u32x4_t a[2][NT], x[MB];
    auto w_tile = [&](int at, int t) {
      return lds_load16(lds + at * STAGE + XBYTES + (wn * NT + t) * kTileBytes + lane * 16);
    };
    auto x_tile = [&](int at, int b) { return lds_load16(lds + at * STAGE + (wm * MB + b) * XBLK + lane * 16); };
    constexpr int kFirst = (STAGES - 2) * (XLOADS + WLOADS);
    __builtin_amdgcn_s_waitcnt(0x0070 | (kFirst & 15) | (kFirst >> 4 << 14));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int t = 0; t < NT; ++t) a[0][t] = w_tile(0, t);
#pragma unroll
    for (int b = 0; b < AHEAD; ++b) x[b] = x_tile(0, b);
    for (int quad = 0; 4 * quad < slab_end; ++quad) {
      uint32_t wscale[NT], xscale[MB];
#pragma unroll
      for (int t = 0; t < NT; ++t) wscale[t] = wnext[t];
#pragma unroll
      for (int b = 0; b < MB; ++b) xscale[b] = xnext[b];
      auto step = [&]<int S>() {
        const int slab = 4 * quad + S;
        __builtin_amdgcn_s_waitcnt(0x0f70 | (kInFlight & 15) | (kInFlight >> 4 << 14));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (S == 0) load_scales(quad + 1);
        load(slab + STAGES - 1, before);
        const int next = buf + 1 == STAGES ? 0 : buf + 1;
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          x[(b + AHEAD) % MB] = x_tile(b + AHEAD < MB ? buf : next, (b + AHEAD) % MB);
          a[(S + 1) & 1][b] = w_tile(next, b);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t][b] = mfma_fp4<S, S>(a[S & 1][t], wscale[t], x[b], xscale[b], acc[t][b]);
          __builtin_amdgcn_sched_barrier(0);
        }
        before = buf;
        buf = next;
      };
      step.template operator()<0>();
      step.template operator()<1>();
      step.template operator()<2>();
      step.template operator()<3>();
    }
  } else
  for (int quad = slab0 >> 2; 4 * quad < slab_end; ++quad) {
    uint32_t wscale[NT], xscale[MX ? MB : 1];
#pragma unroll
    for (int t = 0; t < NT; ++t) wscale[t] = wnext[t];
#pragma unroll
    for (int b = 0; b < (MX ? MB : 1); ++b) xscale[b] = xnext[b];
    auto slab_of = [&]<int S>(int at) {  // the slab in buffer `at`
      const lds_t* const xl = lds + at * STAGE + wm * MB * XBLK;
      const lds_t* const wl = lds + at * STAGE + XBYTES + wn * NT * kTileBytes + lane * 16;
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
          for (int b = 0; b < MB; ++b) acc[t][b] = mfma_fp4<S, S>(a[t], wscale[t], x[b], xscale[b], acc[t][b]);
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          bf16x8_t x[MB];
#pragma unroll
          for (int b = 0; b < MB; ++b) x[b] = __builtin_bit_cast(bf16x8_t, lds_load16(xl + b * XBLK + ro[s]));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const bf16x8_t v = to_bf16(a[t][s], scale_f32(wscale[t] >> (8 * S) & 255u));
#pragma unroll
            for (int b = 0; b < MB; ++b) acc[t][b] = mfma_16x16x32_bf16(v, x[b], acc[t][b]);
          }
        }
      }
    };
    auto step = [&]<int S>() {
      const int slab = 4 * quad + S;
      if ((SPLIT && slab < slab0) || slab >= slab_end) return;
      // vmcnt: this slab is in LDS; lgkmcnt: this wave has read the one before
      __builtin_amdgcn_s_waitcnt(0x0070 | (kInFlight & 15) | (kInFlight >> 4 << 14));
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      if (S == 0 || (SPLIT && slab == slab0)) load_scales(quad + 1);
      load(slab + STAGES - 1, before);
      slab_of.template operator()<S>(buf);
      before = buf;
      buf = buf + 1 == STAGES ? 0 : buf + 1;
      __builtin_amdgcn_sched_barrier(0);
    };
    step.template operator()<0>();
    step.template operator()<1>();
    step.template operator()<2>();
    step.template operator()<3>();
  }

  __builtin_amdgcn_s_waitcnt(0x0f70);  // (the loads past the end write zeros to LDS)

  // Lane (g, n) holds columns 4 g .. 4 g + 3 of a tile for row n of a block.  Two tiles'
  // lanes change places, so that a lane has eight columns and four lanes 64 bytes of a row
  // (in 4 bits 8,192 x 8,192 x 10,240 317 -> 299 us, 2,048 x 4,096 x 28,672 147 -> 131).
  if constexpr (!SPLIT && NT / HALVES % 2 == 0) {
    if (p.wide) {
#pragma unroll
      for (int t = 0; t < NT; t += 2 * HALVES) {
        const int first = col0 + (wn * NT + t) / HALVES * 16, col = first + (g & 1) * 16 + (g >> 1) * 8;
        const f32x4_t bias0 = bias4(p, first + 4 * g), bias1 = bias4(p, first + 16 + 4 * g);
#pragma unroll
        for (int b = 0; b < MB; ++b) {
          const u32x2_t u = round4<GLU>(acc[t][b], acc[t + HALVES - 1][b], bias0);
          const u32x2_t v = round4<GLU>(acc[t + HALVES][b], acc[t + 2 * HALVES - 1][b], bias1);
          const auto s0 = __builtin_amdgcn_permlane16_swap(u.x, v.x, false, false);
          const auto s1 = __builtin_amdgcn_permlane16_swap(u.y, v.y, false, false);
          const int m = (wm * MB + b) * 16 + n;
          if (m < rows && col < p.n)
            *reinterpret_cast<u32x4_t*>(p.out + (m0 + m) * p.o_stride + col) = u32x4_t{s0[0], s1[0], s0[1], s1[1]};
        }
      }
      return;
    }
  }
#pragma unroll
  for (int t = 0; t < NT; t += HALVES) {
    const int col = col0 + (wn * NT + t) / HALVES * 16 + 4 * g;
    if (col >= p.n) continue;
    const f32x4_t bias = SPLIT ? f32x4_t{0.f, 0.f, 0.f, 0.f} : bias4(p, col);
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      const int m = (wm * MB + b) * 16 + n;
      if (m >= rows) continue;
      if constexpr (SPLIT) {
        // [part][half][row][columns, in fours]
        const int64_t fours = (p.n + 3) / 4;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
          p.parts[((int64_t(blockIdx.y) * HALVES + h) * p.rows + m0 + m) * fours + col / 4] = acc[t + h][b];
      } else {
        store4<GLU>(p, m0 + m, col, acc[t][b], acc[t + HALVES - 1][b], bias);
      }
    }
  }
}

// The sum of the parts in their order, and the end of the product.
template <bool GLU>
__global__ __launch_bounds__(256) void combine_kernel(LinearParams p, int parts) {
  constexpr int HALVES = GLU ? 2 : 1;
  const int fours = (p.n + 3) / 4;
  const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x, one = p.rows * fours;
  if (at >= one) return;
  f32x4_t sum = p.parts[at], up = {0.f, 0.f, 0.f, 0.f};
  if constexpr (GLU) up = p.parts[one + at];
#pragma unroll 4
  for (int i = 1; i < parts; ++i) {
    sum += p.parts[i * HALVES * one + at];
    if constexpr (GLU) up += p.parts[(i * HALVES + 1) * one + at];
  }
  const int col = int(at % fours) * 4;
  store4<GLU>(p, at / fours, col, sum, up, bias4(p, col));
}

// ---------------------------------------------------------------- which form
// Forms of the kernel: rows of x and of W per workgroup, and the time of a slab (us,
// measured) with one workgroup on a CU and, per workgroup, with more of them in turn or
// side by side.  The larger the block, the fewer the bytes that each product needs and
// the fewer the workgroups.  A launch takes its start, a slab's time for every slab of
// every workgroup of a CU, the way of its output to memory, and, where workgroups share
// k, the combining launch with the parts' way there and back.  Model and measured (us):
// 77 x 18,944 x 3,584, 80-row blocks, 9 parts 22.0 / 22.5, whole 96.9 / 95.5;
// 128 x 8,192 x 10,240, 128 x 128, 3 parts 31.7 / 32.2; bf16 1,024 x 8,192 x 10,240,
// 128 x 128 in fours of waves 153 / 154, 128 x 256 190 / 179; in 4 bits 2,048 x 8,192 x
// 10,240, 128 x 128 98 / 100, 128 x 256 99 / 98, 256 x 256 122 / 112; 8,192 rows of it 381 /
// 378, 326 / 321, 314 / 312: most within 3 %, some blocks of 256 columns counted 6 to 9 % slow.
//
// Blocks of bf16 rows: 32, 64 and 128 rows, and one rung between the last two, of 80, for 65 to
// 80 rows and for twice as many and more where 128 would leave a block half empty (us, with
// that rung and without: 72 x 3,584 x 18,944 21.9 and 24.5, 72 x 10,240 x 8,192 24.4 and 27.8,
// 72 x 8,192 x 29,568 51 and 60, 144 x 4,096 x 14,336 28.8 and 34.2, 144 x 8,192 x 29,568 88
// and 112; along a short k it gains nothing: 72 x 6,144 x 4,096 16.0 and 15.6).  81 to 96 rows
// have no rung of their own: they take blocks of 128 (96 x 10,240 x 8,192 29.8; 80 rows 25.1).
struct Form {
  int rows, tiles;  // 16-row tiles of W
  float one_us, more_us;
  bool split;
};
constexpr Form kBf16Forms[] = {{32, 8, 0.45f, 0.45f, true}, {64, 8, 0.56f, 0.56f, true}, {80, 8, 0.63f, 0.63f, true},
                               {128, 8, 0.84f, 0.885f, true}, {128, 8, 0.96f, 0.755f, false}, {128, 16, 1.35f, 1.42f, false}};
constexpr Form kMxForms[] = {{128, 8, 0.345f, 0.265f, true}, {128, 16, 0.51f, 0.445f, false}, {256, 16, 0.78f, 0.85f, false}};
constexpr float kStartUs = 3.5f, kCombineUs = 2.5f, kBytesPerUs = 4.4e6f;
constexpr int kMaxParts = 32;

struct Choice {
  float us;
  int form, parts, split_slabs;
  size_t bytes;  // of the parts
};

// The fastest by that count within `room` bytes for parts.
Choice choose(bool mx, bool glu, int64_t rows, int64_t n, int slabs, size_t room) {
  Choice best = {1e30f, 0, 1, slabs, 0};
  const int cus = mi::num_cus(), forms = mx ? 3 : 6;
  for (int f = 0; f < forms; ++f) {
    const Form& form = mx ? kMxForms[f] : kBf16Forms[f];
    const int64_t cols = form.tiles * kTileRows / (glu ? 2 : 1);
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

// The few-row kernel's time: W's bytes once for every group of rows, beyond the first
// from the caches, or where that is longer the rows of x into each of its workgroups.
// More groups than one are faster than blocks of 128 rows where W is small (128 x 4,096 x
// 4,096 in 4 bits 6.0 us, in blocks 13; 64 x 4,096 x 6,144 of bf16 rows 11 and 13; the
// count's 8.4 and 13, 11.6 and 13); one is slower along a long k (32 x 18,944 x 3,584 21,
// in blocks 17; the count's 19 and 17).  More than 512 rows are not measured and not asked
// for.
float few_us(bool mx, int64_t rows, int w_tiles, int slabs) {
  if (rows > 512) return 1e30f;
  const int64_t group = few_group(mx), groups = (rows + group - 1) / group;
  const int cus = mi::num_cus(), each = (w_tiles + cus - 1) / cus, wgs = (w_tiles + each - 1) / each;
  const float w = float(groups * w_tiles) * slabs * (kTileBytes + kQuadBytes / 4) / (mx ? 4e6f : 3.5e6f);
  const float x = float(std::min(rows, group) * slabs * (mx ? kSlab / 2 : 2 * kSlab)) / 8e4f;
  return 4.f + std::max(w, x * float((wgs * groups + cus - 1) / cus));
}

template <int WM, int WN, int MB, int NT, int STAGES, bool MX, bool GLU, bool SPLIT, int AHEAD = 0>
void run(const LinearParams& p, int parts, hipStream_t stream) {
  constexpr int BM = WM * MB * 16, COLS = WN * NT * 16 / (GLU ? 2 : 1);
  const dim3 grid(uint32_t((p.rows + BM - 1) / BM * ((p.n + COLS - 1) / COLS)), parts);
  hipLaunchKernelGGL((many_kernel<WM, WN, MB, NT, STAGES, MX, GLU, SPLIT, AHEAD>), grid, dim3(64 * WM * WN), 0, stream, p);
}

template <bool MX, bool GLU, bool SPLIT>
void run_form(const LinearParams& p, int form, int parts, hipStream_t stream) {
  if constexpr (MX) {
    if (SPLIT || form == 0) run<2, 2, 4, 4, 4, true, GLU, SPLIT>(p, parts, stream);
    else if (form == 1) run<2, 4, 4, 4, 3, true, GLU, false>(p, 1, stream);
    else run<2, 2, 8, 8, 4, true, GLU, false, 3>(p, 1, stream);
  } else {
    if (form == 0) run<1, 4, 2, 2, 4, false, GLU, SPLIT>(p, parts, stream);
    else if (form == 1) run<2, 4, 2, 2, 4, false, GLU, SPLIT>(p, parts, stream);
    else if (form == 2) run<1, 4, 5, 2, 4, false, GLU, SPLIT>(p, parts, stream);
    else if (SPLIT || form == 3) run<2, 4, 4, 2, 3, false, GLU, SPLIT>(p, parts, stream);
    else if (form == 4) run<2, 2, 4, 4, 2, false, GLU, false>(p, 1, stream);
    else run<2, 4, 4, 4, 3, false, GLU, false>(p, 1, stream);
  }
}

template <bool MX, bool GLU>
void launch(const LinearParams& p, const Choice& c, hipStream_t stream) {
  LinearParams q = p;
  q.split_slabs = c.split_slabs;
  if (c.parts == 1) {
    run_form<MX, GLU, false>(q, c.form, 1, stream);
    return;
  }
  run_form<MX, GLU, true>(q, c.form, c.parts, stream);
  const int64_t fours = p.rows * ((p.n + 3) / 4);
  hipLaunchKernelGGL((combine_kernel<GLU>), dim3(uint32_t((fours + 255) / 256)), dim3(256), 0, stream, q, c.parts);
}

// The rows behind the last whole block of 128, where they are few enough for the
// few-row kernel.
int64_t rest_of(bool mx, int64_t rows) {
  const int64_t rest = rows % (mx ? 256 : 128);
  return rest <= (mx ? 64 : 16) && rest < rows ? rest : 0;
}

}  // namespace

size_t many_workspace(bool mx, bool glu, int64_t rows, int64_t n, int slabs) {
  const Choice c = choose(mx, glu, rows, n, slabs, size_t(1) << 28);
  return few_us(mx, rows, int(row_tiles(glu ? 2 * n : n)), slabs) < c.us ? 0 : c.bytes;
}

// How a call with `room` bytes for parts goes: rows by blocks, the others by the few-row kernel.
struct Way {
  Choice c;
  int64_t blocks;  // rows
};
Way way_of(bool mx, bool glu, int64_t rows, int64_t n, int slabs, size_t room) {
  const int w_tiles = int(row_tiles(glu ? 2 * n : n));
  const Choice c = choose(mx, glu, rows, n, slabs, room);
  if (few_us(mx, rows, w_tiles, slabs) < c.us) return {c, 0};
  // (4,105 x 4,096 x 6,144: 792 blocks are four rounds; 768 and nine rows of the few-row
  // kernel three and 7 us)
  if (const int64_t rest = rest_of(mx, rows)) {
    const Choice whole = choose(mx, glu, rows - rest, n, slabs, room);
    if (whole.us + few_us(mx, rest, w_tiles, slabs) < c.us) return {whole, rows - rest};
  }
  return {c, rows};
}

void launch_way(const LinearParams& p, bool glu, const Way& way, hipStream_t stream) {
  const bool mx = p.xs != nullptr;
  LinearParams q = p;
  if (!way.blocks) return launch_few(p, glu, stream);
  const Choice& c = way.c;
  q.rows = way.blocks;
  if (mx) glu ? launch<true, true>(q, c, stream) : launch<true, false>(q, c, stream);
  else glu ? launch<false, true>(q, c, stream) : launch<false, false>(q, c, stream);
  if (q.rows == p.rows) return;
  LinearParams rest = p;
  rest.rows = p.rows - q.rows;
  rest.x += mx ? q.rows / kTileRows * p.slabs * kTileBytes : q.rows * p.x_stride * 2;
  if (mx) rest.xs += q.rows / kTileRows * p.quads * kQuadBytes;
  rest.out += q.rows * p.o_stride;
  if (p.sums) rest.sums += q.rows * p.sums_stride;
  launch_few(rest, glu, stream);
}

}  // namespace mi::mx4

extern "C" size_t mi_linear_mxfp4_workspace_size(int64_t rows, int64_t n, int64_t k, int32_t silu, int32_t x_mxfp4) {
  using namespace mi::mx4;
  if (rows <= 0 || rows > kMaxRows || n <= 0 || n > kMaxN || k <= 0 || k % kBlock || k > kMaxK ||
      few(x_mxfp4 != 0, rows, silu ? 2 * n : n, k))
    return 0;
  return many_workspace(x_mxfp4 != 0, silu != 0, rows, n, int(slabs(k)));
}

extern "C" int mi_linear_mxfp4(const void* x, int64_t x_stride, const void* x_scales, const void* codes,
                               const void* scales, const void* bias, void* out, int64_t out_stride, int64_t rows,
                               int64_t n, int64_t k, int32_t silu, void* workspace, size_t workspace_bytes,
                               mi_stream_t stream) {
  using namespace mi::mx4;
  mi::clear_error();
  if (rows < 0 || rows > kMaxRows || n <= 0 || n > kMaxN || k <= 0 || k % kBlock || k > kMaxK)
    return mi::fail(MI_ERR_INVALID, "linear_mxfp4: rows %lld (0..2^22), n %lld (1..2^24), k %lld (multiple of %d, at most %d)",
                    (long long)rows, (long long)n, (long long)k, kBlock, kMaxK);
  if (silu && bias) return mi::fail(MI_ERR_INVALID, "linear_mxfp4: no bias with the gated product");
  const bool sums = silu == MI_SILU_SUMS;
  if (sums && n % 4)
    return mi::fail(MI_ERR_INVALID, "linear_mxfp4: sums are fp32, a multiple of 4 columns each; got %lld", (long long)n);
  const int64_t out_n = sums ? 2 * n : n;
  if (rows == 0) return MI_OK;
  if (rows == 1) x_stride = k, out_stride = out_n;  // (nothing lies at a row stride)
  if (!x || !codes || !scales || !out) return mi::fail(MI_ERR_INVALID, "linear_mxfp4: null pointer argument");
  const uintptr_t aligned = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(codes) |
                            reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(x_scales) |
                            reinterpret_cast<uintptr_t>(workspace);
  if ((aligned & 15) || ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(bias)) & 1) ||
      (!x_scales && x_stride % 8) || (sums && ((reinterpret_cast<uintptr_t>(out) & 15) || out_stride % 4)))
    return mi::fail(MI_ERR_INVALID, "linear_mxfp4: x rows, codes, scales and workspace must be 16-byte aligned");
  if (out_stride < out_n || (!x_scales && (x_stride < k || x_stride > kMaxStride)))
    return mi::fail(MI_ERR_INVALID, "linear_mxfp4: row strides %lld (at most 2^22) / %lld for k %lld, n %lld",
                    (long long)x_stride, (long long)out_stride, (long long)k, (long long)n);
  // (a workgroup's rows of out are written while others still read all of x, W and bias)
  const int64_t w_rows = silu ? 2 * n : n;
  const int64_t each = sums ? 4 : 2;
  const mi::Rows to = {out, out_stride * each, rows, out_n * each};
  const mi::Rows from[] = {
      x_scales ? mi::Rows{x, 0, 1, row_tiles(rows) * slabs(k) * kTileBytes} : mi::Rows{x, x_stride * 2, rows, k * 2},
      {x_scales, 0, x_scales ? 1 : 0, row_tiles(rows) * quads(k) * kQuadBytes},
      {codes, 0, 1, row_tiles(w_rows) * slabs(k) * kTileBytes},
      {scales, 0, 1, row_tiles(w_rows) * quads(k) * kQuadBytes},
      {bias, 0, bias ? 1 : 0, n * 2}};
  for (const mi::Rows& r : from)
    if (mi::rows_meet(to, r)) return mi::fail(MI_ERR_INVALID, "linear_mxfp4: out overlaps x, the weight or the bias");
  // (parts are written while others still read x and W, and read while out is written)
  Way way = {};
  if (!few(x_scales != nullptr, rows, w_rows, k))
    way = way_of(x_scales != nullptr, silu != 0, rows, n, int(slabs(k)), workspace ? workspace_bytes : 0);
  if (way.blocks && way.c.parts > 1) {
    const mi::Rows parts = {workspace, 0, 1, int64_t(way.c.bytes)};
    bool meet = mi::rows_meet(parts, to);
    for (const mi::Rows& r : from) meet = meet || mi::rows_meet(parts, r);
    if (meet) return mi::fail(MI_ERR_INVALID, "linear_mxfp4: the workspace overlaps another argument");
  }
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
  p.wide = p.vec && !sums && n % 8 == 0 && out_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  p.sums = sums ? static_cast<float*>(out) : nullptr;
  p.sums_stride = out_stride;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  p.parts = static_cast<mi::f32x4_t*>(workspace);
  launch_way(p, silu != 0, way, s);
  return mi::check_launch("linear_mxfp4");
}

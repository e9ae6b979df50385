// Low-rank adapters of many requests beside a shared projection: out = y + scale B (A x),
// A [r][k] and B [n][r] of the row's own adapter.  The projection's outputs are one to
// eight pieces (q, k, v), each with r rows of A of its own.
//
//   plan   : rows sorted by adapter into tiles of up to 16 or 64 rows of one adapter, once
//            per batch.  Which row comes where in its adapter's tiles is of no matter: a row's
//            result depends on its own operands alone.
//   shrink : v = A x of a tile, k in parts over workgroups; sums in fp32.
//   (few rows and a short A: both products in one launch)
//   expand : the parts' sum, times scale, as a pair of bf16 (v and what its rounding left: 16
//            bits of v), times B in fp32, plus y, one rounding; or SiLU(gate) * up of the sums of a
//            gate and an up piece.  Rows without an adapter get the bits that the projection's own
//            gated form leaves them, whatever rows stand beside them.
//
// Bound: for prompts HBM, one read of x, one of y and the write of out; A and B come from the
// caches.  For decode steps the two launches' start and end, and the read of the adapters.
#include <algorithm>
#include <cmath>

#include "mi_adapter_ring.h"
#include "mi_mx8.h"
#include "mi_overlap.h"

namespace {

using mi::bf16x8_t;
using mi::f32x4_t;
using mi::mx8::u32x2_t;
using mi::mx8::u32x4_t;

// Rows of a tile: 16 up to 320 rows, 64 beyond, which read A a quarter as often (us in a graph, 16 / 64, with 1,
// 8 and 64 adapters at 512 rows, 4 and 32 at the others, one launch for none):
//                           256 rows               512 rows                            1,024 rows
//   k  4,096 ->  6,144, 16  11.4 / 13.1 15.8 / 18.0  16.9 / 15.4 17.3 / 18.2 23.8 / 24.6  24.3 / 23.0 25.2 / 20.5
//   k  4,096 -> 28,672, 16  19.0 / 18.7 29.7 / 30.1  31.3 / 24.5 30.3 / 24.8 50.8 / 52.0  53.7 / 38.0 56.2 / 44.5
//   k 14,336 ->  4,096, 64  21.2 / 20.6 35.5 / 34.7  29.6 / 24.5 31.7 / 25.6 57.1 / 50.3  44.7 / 32.5 56.3 / 41.6
constexpr int64_t kFewRows = 320;
constexpr int tile_rows(int64_t rows) { return rows <= kFewRows ? 16 : 64; }
constexpr int kMaxSlots = 1023;  // (and one more count for the rows without)
constexpr int kMaxRank = 128;
constexpr int kMaxPieces = 8;
constexpr int64_t kMaxRows = 1 << 22;
constexpr int kWaves = 4;
constexpr int kManyWaves = 2;  // of a shrink workgroup of 64 rows: two of them share a CU's LDS
constexpr int kStep = 64;  // k of a wave's step
constexpr int kMaxParts = 16;
constexpr int kGroup = 4;  // 16-rank tiles of a workgroup; of 8-bit rows in tiles of 64 half as many

struct Tile {
  int slot, count;  // slot -1: rows without an adapter
};

// A plan: the number of tiles and what it is a plan of in 16 bytes, each tile's rows (in a place of their own,
// so that they are read at once with the tile: a launch of few rows is a chain of such reads), the tiles.
int64_t max_tiles(int64_t rows, int64_t slots) { return std::min(rows, slots + 1) + rows / tile_rows(rows); }
size_t plan_size(int64_t rows, int64_t slots) {
  return 16 + size_t(max_tiles(rows, slots)) * (sizeof(Tile) + 4 * size_t(tile_rows(rows)));
}
struct PlanView {
  int* count;
  int* rows;
  Tile* tiles;
};
PlanView view(void* plan, int64_t rows, int64_t slots) {
  char* const p = static_cast<char*>(plan);
  return {reinterpret_cast<int*>(p), reinterpret_cast<int*>(p + 16),
          reinterpret_cast<Tile*>(p + 16 + 4 * tile_rows(rows) * max_tiles(rows, slots))};
}

constexpr int kPlanThreads = 1024;

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const int* slot_of_row, int rows, int slots, int tile_rows, PlanView p) {
  __shared__ int count[kPlanThreads], tiles[kPlanThreads];
  const int tid = threadIdx.x, lane = tid & 63;
  count[tid] = 0;
  __syncthreads();
  auto at = [&](int row) {
    const int s = slot_of_row[row];
    return uint32_t(s) < uint32_t(slots) ? s : slots;
  };
  // Places of a wave's rows in their slots' lists: one addition where they share the slot,
  // as the rows of a prompt do.
  auto places = [&](int s, int* counts) {
    const int same = __builtin_amdgcn_readfirstlane(s);
    const uint64_t active = __ballot(1), mine = __ballot(s == same);
    if (active != mine) return atomicAdd(&counts[s], 1);
    const int ahead = __popcll(active & ((uint64_t(1) << lane) - 1));
    int base = 0;
    if (ahead == 0) base = atomicAdd(&counts[s], __popcll(active));
    return __builtin_amdgcn_readfirstlane(base) + ahead;
  };
  for (int row = tid; row < rows; row += kPlanThreads) places(at(row), count);
  __syncthreads();
  const int mine = count[tid], need = (mine + tile_rows - 1) / tile_rows;
  tiles[tid] = need;
  __syncthreads();
  for (int d = 1; d < kPlanThreads; d *= 2) {  // sums up to and with each slot
    const int a = tid >= d ? tiles[tid - d] : 0;
    __syncthreads();
    tiles[tid] += a;
    __syncthreads();
  }
  const int tile = tiles[tid] - need;
  for (int i = 0; i < need; ++i) p.tiles[tile + i] = {tid < slots ? tid : -1, min(tile_rows, mine - i * tile_rows)};
  if (tid == kPlanThreads - 1) p.count[0] = tiles[tid], p.count[1] = rows, p.count[2] = slots;
  count[tid] = tile * tile_rows;  // (a slot's tiles lie one behind the other, so its rows do)
  __syncthreads();
  for (int row = tid; row < rows; row += kPlanThreads) p.rows[places(at(row), count)] = row;
}

struct AdapterParams {
  const char* x;      // bf16 rows, or codes
  int64_t x_stride;   // bytes
  const char* xs;     // scale bytes, rows of whole 16 bytes; null: x is bf16
  int64_t xs_stride;
  const uint16_t* a;  // [slots][pieces * rank][k]
  const uint16_t* b;  // [slots][n][rank]
  const float* scale;
  const uint16_t* y;
  int64_t y_stride;
  uint16_t* out;
  int64_t o_stride;
  PlanView plan;
  float* parts;  // [part][tile][row of the tile][ranks, padded]
  int rows, slots;
  int eighths, per_eighths;  // rank / 8; 2^16 over it, rounded up
  int k, n, rank, ranks, padded;  // ranks = pieces * rank, padded to 16
  int n_parts, part_steps, max_tiles, group_ranks;
  int pieces, chunk;  // columns of an expand workgroup
  int up;             // the first of the up columns, with SiLU
  uint8_t* scales;    // of out in 8 bits
  int64_t s_stride;
  int end[kMaxPieces];       // columns,
  int end_chunk[kMaxPieces]; // chunks up to and with each piece
};

// The tiles of a plan, -1 where it is of another batch than the launch (a captured one replayed after another plan).
__device__ __forceinline__ int plan_tiles(const AdapterParams& p) {
  return p.plan.count[1] == p.rows && p.plan.count[2] == p.slots ? p.plan.count[0] : -1;
}

// A workgroup's columns: a chunk of one piece.
struct Columns {
  int piece, begin, end;
};
__device__ __forceinline__ Columns columns_of(const AdapterParams& p) {
  int piece = 0;
  while (int(blockIdx.y) >= p.end_chunk[piece]) ++piece;
  const int start = piece ? p.end[piece - 1] : 0, before = piece ? p.end_chunk[piece - 1] : 0;
  const int begin = start + (int(blockIdx.y) - before) * p.chunk;
  return {piece, begin, min(begin + p.chunk, p.end[piece])};
}
// What becomes of the sums: out's bf16, or, of gate and up columns, SiLU(gate) * up in bf16 or 8 bits; `steps`: each
// step rounded to bf16, as mi_silu_mul is; `sums`: y is fp32, SiLU as linear_mxfp4's gated form takes
// it (sums) and as linear_mxfp8's (sums8).
enum class End { plain, silu, silu8, steps, sums, sums8 };
constexpr bool in_8_bits(End end) { return end == End::silu8 || end == End::sums8; }
constexpr bool y_is_fp32(End end) { return end == End::sums || end == End::sums8; }

// Eight columns of a row of y.
template <End END>
struct Eight {
  uint4 v[y_is_fp32(END) ? 2 : 1];
  __device__ __forceinline__ void load(const AdapterParams& p, int64_t row, int col, bool in) {
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (y_is_fp32(END)) {
      const float* const from = reinterpret_cast<const float*>(p.y) + row * p.y_stride + col;
      v[0] = in ? mi::load16_nt(from) : none;
      v[1] = in ? mi::load16_nt(from + 4) : none;
    } else {
      v[0] = in ? mi::load16_nt(p.y + row * p.y_stride + col) : none;
    }
  }
  __device__ __forceinline__ float operator[](int t) const {
    if constexpr (y_is_fp32(END)) {
      const uint32_t words[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
      return __uint_as_float(words[t]);
    } else {
      const uint32_t pairs[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
      return t % 2 ? mi::bf16_hi(pairs[t / 2]) : mi::bf16_lo(pairs[t / 2]);
    }
  }
};

// What a unit's sums start from: y where that is fp32 (which frees its registers while they grow), else zeros.
template <End END>
__device__ __forceinline__ void begin_sums(f32x4_t (&d)[8], const Eight<END> (&y)[4]) {
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) d[t][i] = y_is_fp32(END) ? y[i][t] : 0.f;
}

// Where no row's adapter is known: NaN (the tiles are as many as the rows' at least).
template <End END>
__device__ __forceinline__ void write_nan(const AdapterParams& p, int tile_rows, const Columns& c) {
  for (int i = 0; i < tile_rows && int(blockIdx.x) * tile_rows + i < p.rows; ++i)
    for (int col = c.begin + int(threadIdx.x); col < c.end; col += int(blockDim.x)) {
      const int64_t row = int64_t(blockIdx.x) * tile_rows + i;
      if constexpr (in_8_bits(END)) {
        reinterpret_cast<uint8_t*>(p.out)[row * p.o_stride + col] = 0;
        if (col % mi::mx8::kBlock == 0) p.scales[row * p.s_stride + col / mi::mx8::kBlock] = 255;
      } else {
        p.out[row * p.o_stride + col] = 0x7fc0;
      }
    }
}
// Piece e of B's rows of a unit, 16 bytes each: its row.  (e is 128 times 16 at most, where this is exact.)
__device__ __forceinline__ int row_of_piece(const AdapterParams& p, int e) { return e * p.per_eighths >> 16; }

// Four sums times scale as pairs of bf16: the values and what their rounding left.
__device__ __forceinline__ uint4 bf16_pair(f32x4_t sum, float scale) {
  uint32_t hi[2], lo[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float s = sum[2 * j] * scale, t = sum[2 * j + 1] * scale;
    hi[j] = mi::cvt_pk_bf16(s, t);
    const float ds = s - mi::bf16_lo(hi[j]), dt = t - mi::bf16_hi(hi[j]);
    // (an infinity leaves nothing)
    lo[j] = mi::cvt_pk_bf16(isfinite(mi::bf16_lo(hi[j])) ? ds : 0.f, isfinite(mi::bf16_hi(hi[j])) ? dt : 0.f);
  }
  return make_uint4(hi[0], hi[1], lo[0], lo[1]);
}
// y's eight columns with row i of eight products' sums.
__device__ __forceinline__ uint4 add_rounded(uint4 y, const f32x4_t (&d)[8], int i) {
  return make_uint4(mi::cvt_pk_bf16(mi::bf16_lo(y.x) + d[0][i], mi::bf16_hi(y.x) + d[1][i]),
                    mi::cvt_pk_bf16(mi::bf16_lo(y.y) + d[2][i], mi::bf16_hi(y.y) + d[3][i]),
                    mi::cvt_pk_bf16(mi::bf16_lo(y.z) + d[4][i], mi::bf16_hi(y.z) + d[5][i]),
                    mi::cvt_pk_bf16(mi::bf16_lo(y.w) + d[6][i], mi::bf16_hi(y.w) + d[7][i]));
}

// 64 k of a wave's 16 rows of x and of RT tiles of A, straight from memory to registers.  Lane (g, n)
// holds row n's k from 16 g on: its first eight are one product's operand, the other eight the next
// one's.  (Which k comes where is of no matter as long as both operands agree.)
template <bool X8, int RT>
struct Step {
  uint4 a[RT][2], x[2];
  float s;
  __device__ __forceinline__ void load(const AdapterParams& p, const uint16_t* const (&from)[RT], const char* row, const char* scales,
                                       int step, int end) {
    const int k0 = step * kStep, g = (threadIdx.x & 63) >> 4;
    const bool in = step < end && k0 + 16 * g < p.k;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      a[t][0] = in ? mi::load16(from[t] + k0) : none;
      a[t][1] = in ? mi::load16(from[t] + k0 + 8) : none;
    }
    x[0] = in ? mi::load16(row + (X8 ? 1 : 2) * k0) : none;
    if constexpr (X8) s = in ? mi::mx8::scale_f32(uint8_t(scales[k0 / 32])) : 0.f;
    else x[1] = in ? mi::load16(row + 2 * k0 + 16) : none;
  }
  __device__ __forceinline__ void multiply(f32x4_t (&acc)[RT][1]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bf16x8_t v;
      if constexpr (X8) {
        const u32x2_t lo = mi::mx8::to_bf16(h ? x[0].z : x[0].x, s);
        const u32x2_t hi = mi::mx8::to_bf16(h ? x[0].w : x[0].y, s);
        v = mi::as_bf16x8(make_uint4(lo.x, lo.y, hi.x, hi.y));
      } else {
        v = mi::as_bf16x8(x[h]);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[t][0] = mi::mfma_16x16x32_bf16(mi::as_bf16x8(a[t][h]), v, acc[t][0]);
    }
  }
};

// The waves' sums of a tile's ranks to memory: lane (g, n) holds ranks 4 g .. 4 g + 3 of
// tile t for row n of block b.
template <int WAVES, int RT, int NB>
__device__ __forceinline__ void store_ranks(const AdapterParams& p, const f32x4_t (&acc)[RT][NB], f32x4_t* red, int count,
                                            int rank0) {
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int b = 0; b < NB; ++b) red[(w * RT * NB + t * NB + b) * 64 + lane] = acc[t][b];
  __syncthreads();
  for (int q = w; q < RT * NB; q += WAVES) {
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < WAVES; ++o) sum += red[(o * RT * NB + q) * 64 + lane];
    const int row = q % NB * 16 + n, r = rank0 + q / NB * 16 + 4 * g;
    if (row < count && r < p.padded)
      *reinterpret_cast<f32x4_t*>(p.parts + ((int64_t(blockIdx.y) * p.max_tiles + blockIdx.x) * (16 * NB) + row) * p.padded + r) = sum;
  }
}

// Tiles of 16 rows: a wave takes steps in turn, the next one's on their way while this one is multiplied.
template <bool X8, int RT>
__global__ __launch_bounds__(64 * kWaves) void shrink_few_kernel(AdapterParams p) {
  __shared__ __attribute__((aligned(16))) f32x4_t red[kWaves * RT * 64];
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const int tiles = plan_tiles(p);
  const Tile tile = p.plan.tiles[blockIdx.x];
  const int* const order = p.plan.rows + blockIdx.x * 16;
  const int own = order[n], any = order[0];
  if (int(blockIdx.x) >= tiles || tile.slot < 0) return;
  const int rank0 = int(blockIdx.z) * p.group_ranks;
  const int64_t row = n < tile.count ? own : any;  // (past the tile's last row any will do)
  const char* const x = p.x + row * p.x_stride + (X8 ? 16 : 32) * g;
  const char* const xs = X8 ? p.xs + row * p.xs_stride + g / 2 : nullptr;
  const uint16_t* a[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = rank0 + t * 16 + n;  // (past the last rank any row will do: its sums are not kept)
    a[t] = p.a + (int64_t(tile.slot) * p.ranks + (r < p.ranks ? r : 0)) * p.k + 16 * g;
  }
  const int end = min((p.k + kStep - 1) / kStep, int(blockIdx.y + 1) * p.part_steps);
  f32x4_t acc[RT][1];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t][0] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  Step<X8, RT> cur, next;
  int step = int(blockIdx.y) * p.part_steps + w;
  cur.load(p, a, x, xs, step, end);
  for (; step < end; step += kWaves) {
    next.load(p, a, x, xs, step + kWaves, end);
    cur.multiply(acc);
    cur = next;
  }
  store_ranks<kWaves, RT, 1>(p, acc, red, tile.count, rank0);
}

// A wave's part of 16 RT ranks from rank0 on times a tile of 16 NB rows: as in the few-row projections, its
// rows go through a ring of its own in LDS, two steps deep, eight rows of 128 bytes by an
// instruction (rows read as operands straight from memory are 64 places an instruction, which
// the address unit takes one by one).  A step is 128 bytes of x: 64 k of bf16, 128 of 8 bits, which
// take two lots of A.  Steps first .. end - 1, the waves' in turn.
constexpr int ring_bytes(bool x8, int rt, int nb) { return 2 * (nb + rt * (x8 ? 2 : 1)) * 2048 + (x8 ? 2048 : 0); }
template <bool X8, int RT, int NB, int WAVES>
__device__ __forceinline__ void multiply_ring(const AdapterParams& p, const Tile& tile, const int* order, mi::mx8::lds_t* lds, int rank0,
                                              int first, int end, f32x4_t (&acc)[RT][NB]) {
  using namespace mi::mx8;
  constexpr int LOTS = X8 ? 2 : 1, DEPTH = 2;
  constexpr int XBYTES = NB * 2048, SLOT = XBYTES + RT * LOTS * 2048, SBYTES = X8 ? 1024 : 0;
  constexpr int LOADS = SLOT / 1024;
  static_assert(DEPTH * SLOT + 2 * SBYTES == ring_bytes(X8, RT, NB), "LDS");
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  lds_t* const scales = lds + DEPTH * SLOT;
  const int g = lane >> 4, n = lane & 15, width = X8 ? p.k : 2 * p.k;  // bytes of a row of x
  // a load: 8 rows, lane l chunk slot l % 8 of row l / 8
  const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 16;
  const char* x[2 * NB];
#pragma unroll
  for (int i = 0; i < 2 * NB; ++i) {
    const int at = i * 8 + r8;
    x[i] = p.x + int64_t(order[at < tile.count ? at : 0]) * p.x_stride;
  }
  const char* a[2 * RT];
#pragma unroll
  for (int i = 0; i < 2 * RT; ++i) {
    const int r = rank0 + i * 8 + r8;  // (past the last rank any row will do: its sums are not kept)
    a[i] = reinterpret_cast<const char*>(p.a + (int64_t(tile.slot) * p.ranks + (r < p.ranks ? r : 0)) * p.k);
  }
  const char* const xs = X8 ? p.xs + int64_t(order[lane < tile.count ? lane : 0]) * p.xs_stride : nullptr;
  auto dma = [&](const char* from, lds_t* to) {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)const_cast<char*>(from),
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
#endif
  };
  // (behind the last k the row's start: it meets zeros, below)
  auto load = [&](int step, int slot) {
    lds_t* const to = lds + slot * SLOT;
    const int off = step < end ? step * 128 : 0;
    const int xo = mi::adapter::ring_place(off, chunk, width);
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) dma(x[i] + xo, to + i * 1024);
#pragma unroll
    for (int l = 0; l < LOTS; ++l) {
      const int ao = mi::adapter::ring_place(off * LOTS + l * 128, chunk, 2 * p.k);
#pragma unroll
      for (int i = 0; i < 2 * RT; ++i) dma(a[i] + ao, to + XBYTES + (l * 2 * RT + i) * 1024);
    }
  };
  // (8 bits: the scale bytes of four steps, 16 a row; a wave takes groups of four in turn)
  auto load_scales = [&](int quad) { dma(xs + (quad * 512 < p.k ? quad * 16 : 0), scales + (quad / WAVES & 1) * SBYTES); };
  auto step_at = [&](int i) { return X8 ? first + 4 * (w + i / 4 * WAVES) + i % 4 : first + w + i * WAVES; };
  const int lo = n * 128 + (g ^ (n & 7)) * 16, hi = n * 128 + ((4 + g) ^ (n & 7)) * 16;
  const int even = n * 128 + ((2 * g) ^ (n & 7)) * 16, odd = n * 128 + ((2 * g + 1) ^ (n & 7)) * 16;

#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[t][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  constexpr int kInFlight = (DEPTH - 1) * LOADS;
  static_assert(kInFlight < 64, "vmcnt");
  const int quad0 = first / 4 + w;
  if constexpr (X8) {
    load_scales(quad0);
    load_scales(quad0 + WAVES);
  }
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) load(step_at(i), i);
  for (int i = 0; X8 ? step_at(i & ~3) < end : step_at(i) < end; i += DEPTH) {
    if constexpr (X8) {  // (a group ahead: done by the waits before it)
      if (i && (i & 3) == 0) load_scales(quad0 + (i / 4 + 1) * WAVES);
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int step = step_at(i + d);
      __builtin_amdgcn_s_waitcnt(0x0f70 | (kInFlight & 15) | (kInFlight >> 4 << 14));
      __builtin_amdgcn_sched_barrier(0);
      const lds_t* const xl = lds + d * SLOT;
      const lds_t* const al = xl + XBYTES;
      u32x4_t v[NB][2], f[LOTS][RT][2];
      float s[NB][2];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        v[b][0] = lds_load16(xl + b * 2048 + lo);
        v[b][1] = lds_load16(xl + b * 2048 + hi);
        if constexpr (X8) {
          const lds_t* const sl = scales + (((first / 4 + w + i / 4 * WAVES) / WAVES) & 1) * SBYTES + (b * 16 + n) * 16 + (i + d) % 4 * 4;
          s[b][0] = scale_f32(lds_load1(sl + g / 2));
          s[b][1] = scale_f32(lds_load1(sl + 2 + g / 2));
        }
      }
#pragma unroll
      for (int l = 0; l < LOTS; ++l)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          f[l][t][0] = lds_load16(al + (l * RT + t) * 2048 + (X8 ? even : lo));
          f[l][t][1] = lds_load16(al + (l * RT + t) * 2048 + (X8 ? odd : hi));
        }
      __builtin_amdgcn_s_waitcnt(0xc07f);  // read: the place may be filled again
      __builtin_amdgcn_sched_barrier(0);
      load(step_at(i + d + DEPTH), d);
      // the operands' k of x's two chunks; A's behind the last k (and in no step) are made zeros
      const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = step < end && step * 128 + h * 64 + g * 16 < width;
#pragma unroll
        for (int l = 0; l < LOTS; ++l) {
          bf16x8_t u[NB];
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            uint4 q = __builtin_bit_cast(uint4, v[b][h]);
            if constexpr (X8) {
              const u32x2_t c = to_bf16(l ? q.z : q.x, s[b][h]), d2 = to_bf16(l ? q.w : q.y, s[b][h]);
              q = make_uint4(c.x, c.y, d2.x, d2.y);
            }
            u[b] = mi::as_bf16x8(in ? q : none);
          }
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            // 8 bits: chunk h of x is lot h of A, its halves A's even and odd chunks
            const u32x4_t fa = X8 ? f[X8 ? h : 0][t][l] : f[0][t][h];
            const bf16x8_t m = mi::as_bf16x8(in ? __builtin_bit_cast(uint4, fa) : none);
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[t][b] = mi::mfma_16x16x32_bf16(m, u[b], acc[t][b]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_s_waitcnt(0x0070);  // (the loads past the end write to LDS)
}

template <bool X8, int RT>
__global__ __launch_bounds__(64 * kManyWaves) void shrink_many_kernel(AdapterParams p) {
  constexpr int WAVES = kManyWaves, NB = 4, WAVE = ring_bytes(X8, RT, NB);
  static_assert(WAVES * WAVE <= 80 * 1024 && RT * NB * 1024 <= WAVE, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[WAVES * WAVE];
  const int tiles = plan_tiles(p);
  const Tile tile = p.plan.tiles[blockIdx.x];
  if (int(blockIdx.x) >= tiles || tile.slot < 0) return;
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int rank0 = int(blockIdx.z) * p.group_ranks, steps = ((X8 ? p.k : 2 * p.k) + 127) / 128;
  const int first = int(blockIdx.y) * p.part_steps, end = min(steps, first + p.part_steps);
  f32x4_t acc[RT][NB];
  multiply_ring<X8, RT, NB, WAVES>(p, tile, p.plan.rows + int64_t(blockIdx.x) * (16 * NB), (mi::mx8::lds_t*)smem + w * WAVE, rank0,
                                   first, end, acc);
  __syncthreads();
  store_ranks<WAVES, RT, NB>(p, acc, reinterpret_cast<f32x4_t*>(smem), tile.count, rank0);
}


// What a lane makes of its four rows' y and of its sums for columns col .. col + 7 of them, the first `count` of
// which are the tile's: out, or, of gate columns, the values that the up columns' turn takes.
template <End END, int HALF>
__device__ __forceinline__ void end_of_unit(const AdapterParams& p, bool adds, const Eight<END> (&y)[4], const f32x4_t (&d)[8],
                                            float (&gate)[END == End::plain ? 1 : 4][8], const int64_t (&row)[4], int col, int count) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (END == End::plain) {
      const uint4 o = adds ? add_rounded(y[i].v[0], d, i) : y[i].v[0];
      if (i < count) mi::store16(p.out + row[i] * p.o_stride + col, o);
    } else {
      float v[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        if constexpr (y_is_fp32(END)) v[t] = d[t][i];
        else v[t] = adds ? y[i][t] + d[t][i] : y[i][t];
        if constexpr (END == End::steps) v[t] = mi::bf16_lo(mi::cvt_pk_bf16(v[t], 0.f));
        if constexpr (HALF == 1) v[t] *= gate[i][t];
        else if constexpr (END == End::steps) gate[i][t] = mi::bf16_lo(mi::cvt_pk_bf16(mi::silu(v[t]), 0.f));
        else if constexpr (END == End::sums) gate[i][t] = mi::silu(v[t]);
        else gate[i][t] = mi::mx8::silu20(v[t]);
      }
      if constexpr (HALF == 1 && !in_8_bits(END)) {
        if (i < count)
          mi::store16(p.out + row[i] * p.o_stride + col, make_uint4(mi::cvt_pk_bf16(v[0], v[1]), mi::cvt_pk_bf16(v[2], v[3]),
                                                                   mi::cvt_pk_bf16(v[4], v[5]), mi::cvt_pk_bf16(v[6], v[7])));
      } else if constexpr (HALF == 1) {  // (a block's 32 columns are four lanes')
        uint32_t top = 0;
#pragma unroll
        for (int t = 0; t < 8; ++t) top = max(top, mi::mx8::magnitude(v[t]));
        const uint32_t byte = mi::mx8::scale_byte(mi::mx8::max4(top));
        if (i < count) {
          *reinterpret_cast<u32x2_t*>(reinterpret_cast<uint8_t*>(p.out) + row[i] * p.o_stride + col) =
              u32x2_t{mi::mx8::to_codes(v[0], v[1], v[2], v[3], byte), mi::mx8::to_codes(v[4], v[5], v[6], v[7], byte)};
          if (col % mi::mx8::kBlock == 0) p.scales[row[i] * p.s_stride + col / mi::mx8::kBlock] = uint8_t(byte);
        }
      }
    }
  }
}

// The sum of the parts of four ranks, in their order, eight on their way at once.
__device__ __forceinline__ f32x4_t sum_of_parts(const AdapterParams& p, const float* from, int64_t part) {
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](int first) {
    f32x4_t v[8];
#pragma unroll
    for (int o = 0; o < 8; ++o)
      v[o] = first + o < p.n_parts ? *reinterpret_cast<const f32x4_t*>(from + (first + o) * part) : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < 8; ++o) sum += v[o];
  };
  static_assert(kMaxParts == 16);
  add(0);
  if (p.n_parts > 8) add(8);
  return sum;
}

// out = y + B v of a tile of 16 NB rows and a chunk of columns.  J: products of 32 that the
// pairs of a piece's ranks take.  A unit of work is 16 rows by 128 columns, eight products
// side by side: column c of product t is column 8 c + t of the unit, so that lane (g, n) ends with
// columns 8 n .. 8 n + 7 of rows 4 g .. 4 g + 3, 16 bytes of y and out in the order of the lanes.  With SiLU a
// unit of gate columns and the same of up columns follow each other, and the gate's values wait in fp32.
// (rank 64 with SiLU: two waves a SIMD)
template <int NB, int J, End END>
__global__ __launch_bounds__(64 * kWaves, END != End::plain && J == 4 ? 2 : 1) void expand_kernel(AdapterParams p) {
  constexpr int ROWS = 16 * NB, kPair = 32 * J;  // a row's ranks in bf16, and what the rounding left of them
  constexpr int VSTRIDE = kPair + 8;              // (the rows of an operand on distinct banks)
  constexpr int kMaxWeights = 128 * (kPair / 2) + 128;  // a unit's columns of B: eight of them, then 16 bytes apart
  constexpr int HALVES = END == End::plain ? 1 : 2;
  __shared__ __attribute__((aligned(16))) uint16_t vs[HALVES][ROWS * VSTRIDE];
  __shared__ __attribute__((aligned(16))) uint16_t ws[2][kMaxWeights];
  const int tiles = plan_tiles(p);
  const Columns columns = columns_of(p);
  const int piece = columns.piece, c0 = columns.begin, c1 = columns.end;
  if (tiles < 0) return write_nan<END>(p, ROWS, columns);
  const Tile tile = p.plan.tiles[blockIdx.x];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, n = lane & 15;
  // wave w takes row block w (of a tile of one block the first wave)
  const int* const order = p.plan.rows + int64_t(blockIdx.x) * ROWS;
  int own[4] = {0, 0, 0, 0}, any = order[0];
  if (w < NB) {
#pragma unroll
    for (int i = 0; i < 4; ++i) own[i] = order[w * 16 + 4 * g + i];
  }
  if (int(blockIdx.x) >= tiles || (END == End::plain && tile.slot < 0 && p.out == p.y)) return;
  const bool adds = tile.slot >= 0;
  const int nb = (tile.count + 15) / 16, units = (c1 - c0 + 127) / 128 * HALVES;
  const int eighths = p.eighths;
  const uint16_t* const weights = p.b + int64_t(max(tile.slot, 0)) * p.n * p.rank;

  // the weights of a unit's 128 columns, 16 bytes a thread and lot
  constexpr int LOTS = (128 * (kPair / 2) / 8 + 64 * kWaves - 1) / (64 * kWaves);
  uint4 wv[LOTS];
  auto fetch = [&](int unit) {
    const int up = unit % HALVES * p.up;
#pragma unroll
    for (int i = 0; i < LOTS; ++i) {
      const int e = i * 64 * kWaves + tid, in = row_of_piece(p, e), col = c0 + unit / HALVES * 128 + in;
      wv[i] = adds && e < 128 * eighths && col < c1 ? mi::load16(weights + int64_t(up + col) * p.rank + (e - in * eighths) * 8)
                                                    : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  auto keep = [&](int buf) {
#pragma unroll
    for (int i = 0; i < LOTS; ++i) {
      const int e = i * 64 * kWaves + tid, col = row_of_piece(p, e);
      if (e < 128 * eighths) mi::store16(ws[buf] + col * p.rank + col / 8 * 8 + (e - col * eighths) * 8, wv[i]);
    }
  };
  fetch(0);
  struct Rows {
    Eight<END> y[4];
  };
  int64_t row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = w * 16 + 4 * g + i;
    row[i] = at < tile.count ? own[i] : any;  // (past the tile's last row any will do)
  }
  auto load_rows = [&](Rows& r, int unit) {
    const int col = c0 + unit / HALVES * 128 + 8 * n, up = unit % HALVES * p.up;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.y[i].load(p, row[i], up + col, w < nb && col < c1);
  };
  Rows rows, next_rows;
  load_rows(rows, 0);
  if (adds) {
    const float scale = p.scale[tile.slot];
    const int fours = p.rank / 4;
    const int64_t part = int64_t(p.max_tiles) * ROWS * p.padded;
    for (int i = tid; i < tile.count * fours * HALVES; i += 64 * kWaves) {
      const int row = i / (fours * HALVES), half = i / fours % HALVES, r = i % fours * 4;
      const float* const from = p.parts + (int64_t(blockIdx.x) * ROWS + row) * p.padded + (piece + half) * p.rank + r;
      const f32x4_t sum = sum_of_parts(p, from, part);
      const uint4 pair = bf16_pair(sum, scale);
      *reinterpret_cast<uint2*>(vs[half] + row * VSTRIDE + r) = make_uint2(pair.x, pair.y);
      *reinterpret_cast<uint2*>(vs[half] + row * VSTRIDE + p.rank + r) = make_uint2(pair.z, pair.w);
    }
  }
  int from[J];  // of a lane's eight ranks of product j, -1: past the last pair
#pragma unroll
  for (int j = 0; j < J; ++j) from[j] = 4 * j + g < 2 * eighths ? (4 * j + g < eighths ? 4 * j + g : 4 * j + g - eighths) * 8 : -1;
  float gate[END == End::plain ? 1 : 4][8];
  auto step = [&]<int HALF>(int unit) {
    const int col = c0 + unit / HALVES * 128 + 8 * n, buf = unit & 1;
    keep(buf);
    f32x4_t d[8];
    begin_sums<END>(d, rows.y);
    if (unit + 1 < units) {
      fetch(unit + 1);
      load_rows(next_rows, unit + 1);
    }
    __syncthreads();
    if (w < nb) {
      if (adds) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint4 none = make_uint4(0u, 0u, 0u, 0u);
          const uint4 q = *reinterpret_cast<const uint4*>(vs[HALF] + (w * 16 + n) * VSTRIDE + (4 * j + g) * 8);
          const bf16x8_t v = mi::as_bf16x8(from[j] >= 0 ? q : none);
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            const int at = (8 * n + t) * p.rank + n * 8 + (from[j] >= 0 ? from[j] : 0);
            const uint4 m = *reinterpret_cast<const uint4*>(ws[buf] + at);
            d[t] = mi::mfma_16x16x32_bf16(v, mi::as_bf16x8(from[j] >= 0 ? m : none), d[t]);
          }
          // (with SiLU and all reads ahead a SIMD's registers hold one wave: rank 64 25 us -> 43)
          if constexpr (END != End::plain && J >= 4) __builtin_amdgcn_sched_barrier(0);
        }
      }
      end_of_unit<END, HALF>(p, adds, rows.y, d, gate, row, col, col < c1 ? tile.count - w * 16 - 4 * g : 0);
    }
    rows = next_rows;
  };
  for (int unit = 0; unit < units; unit += HALVES) {
    step.template operator()<0>(unit);
    if constexpr (HALVES == 2) step.template operator()<1>(unit + 1);
  }
}

// The units of a chunk for a tile of 16 rows, each a wave's own.  B's rows of a unit are one piece of memory, which the
// wave reads in the order of its lanes and passes to itself through LDS, eight columns and then 16 bytes
// apart (read as operands straight from memory: a unit of rank 16 1 us more, of rank 64 4).
template <int J>
constexpr int kUnitWeights = 128 * 16 * J + 128;
template <int J, End END, int WAVES>
struct Units {
  static constexpr int HALVES = END == End::plain ? 1 : 2, VSTRIDE = 32 * J + 8, LOTS = 4 * J;
  const AdapterParams& p;
  const Columns& c;
  const Tile& tile;
  const int w, lane, eighths;
  const uint16_t* weights;
  int64_t row[4];
  uint4 b[LOTS];
  Eight<END> y[4];

  __device__ __forceinline__ Units(const AdapterParams& p, const Columns& c, const Tile& tile, const int (&mine)[4], int any)
      : p(p), c(c), tile(tile), w(__builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6)), lane(threadIdx.x & 63), eighths(p.eighths) {
    weights = p.b + int64_t(max(tile.slot, 0)) * p.n * p.rank;
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = 4 * (lane >> 4) + i < tile.count ? mine[i] : any;  // (past the tile's last row any will do)
  }
  // What the wave's unit `i` reads (of gate and up columns in turn).
  __device__ __forceinline__ void load(int i) {
    const int c0 = c.begin + (i / HALVES * WAVES + w) * 128, up = i % HALVES * p.up, col = c0 + 8 * (lane & 15);
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int k = 0; k < LOTS; ++k) {
      const int e = k * 64 + lane, in = row_of_piece(p, e), at = c0 + in;
      b[k] = tile.slot >= 0 && e < 128 * eighths && at < c.end
                 ? mi::load16(weights + int64_t(up + at) * p.rank + (e - in * eighths) * 8) : none;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k].load(p, row[k], up + col, col < c.end);
  }
  // vs: v's pairs, those of the gate and of the up columns; ws: room for a unit's weights, the wave's own.
  template <int HALF>
  __device__ __forceinline__ void step(int i, const uint16_t* vs, uint16_t* ws, float (&gate)[END == End::plain ? 1 : 4][8]) {
    const int g = lane >> 4, n = lane & 15, c0 = c.begin + (i / HALVES * WAVES + w) * 128, col = c0 + 8 * n;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
    f32x4_t d[8];
    begin_sums<END>(d, y);
    const Eight<END> own[4] = {y[0], y[1], y[2], y[3]};
    if (tile.slot >= 0) {
#pragma unroll
      for (int k = 0; k < LOTS; ++k) {
        const int e = k * 64 + lane, at = row_of_piece(p, e);
        if (e < 128 * eighths) mi::store16(ws + at * p.rank + at / 8 * 8 + (e - at * eighths) * 8, b[k]);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    if (c.begin + ((i + 1) / HALVES * WAVES + w) * 128 < c.end) load(i + 1);
    if (tile.slot >= 0) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const bool in = 4 * j + g < 2 * eighths;  // (or past the last pair)
        const int from = in ? (4 * j + g < eighths ? 4 * j + g : 4 * j + g - eighths) * 8 : 0;
        const uint4 q = *reinterpret_cast<const uint4*>(vs + (HALF * 16 + n) * VSTRIDE + (4 * j + g) * 8);
        const bf16x8_t v = mi::as_bf16x8(in ? q : none);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const uint4 m = *reinterpret_cast<const uint4*>(ws + (8 * n + t) * p.rank + n * 8 + from);
          d[t] = mi::mfma_16x16x32_bf16(v, mi::as_bf16x8(in ? m : none), d[t]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    end_of_unit<END, HALF>(p, tile.slot >= 0, own, d, gate, row, col, col < c.end ? tile.count - 4 * g : 0);
  }
  __device__ __forceinline__ void run(const uint16_t* vs, uint16_t* ws) {
    float gate[END == End::plain ? 1 : 4][8];
    for (int i = 0; c.begin + (i / HALVES * WAVES + w) * 128 < c.end; i += HALVES) {
      step<0>(i, vs, ws, gate);
      if constexpr (HALVES == 2) step<1>(i + 1, vs, ws, gate);
    }
  }
};

// expand_kernel's work for tiles of 16 rows, a unit a wave.
template <int J, End END>
__global__ __launch_bounds__(64 * kWaves, END != End::plain ? 2 : 1) void expand_waves_kernel(AdapterParams p) {
  constexpr int HALVES = END == End::plain ? 1 : 2, VSTRIDE = 32 * J + 8;
  __shared__ __attribute__((aligned(16))) uint16_t vs[HALVES * 16 * VSTRIDE];
  __shared__ __attribute__((aligned(16))) uint16_t ws[kWaves][kUnitWeights<J>];
  const int tid = threadIdx.x, g = (tid & 63) >> 4;
  const int tiles = plan_tiles(p);
  const Tile tile = p.plan.tiles[blockIdx.x];
  const int* const order = p.plan.rows + blockIdx.x * 16;
  const int any = order[0];
  int mine[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mine[i] = order[4 * g + i];
  const Columns c = columns_of(p);
  if (tiles < 0) return write_nan<END>(p, 16, c);
  if (int(blockIdx.x) >= tiles || (END == End::plain && tile.slot < 0 && p.out == p.y)) return;
  Units<J, END, kWaves> units(p, c, tile, mine, any);
  units.load(0);
  if (tile.slot >= 0) {
    const float scale = p.scale[tile.slot];
    const int fours = p.rank / 4;
    const int64_t part = int64_t(p.max_tiles) * 16 * p.padded;
    for (int i = tid; i < tile.count * fours * HALVES; i += 64 * kWaves) {
      const int row = i / (fours * HALVES), half = i / fours % HALVES, r = i % fours * 4;
      const f32x4_t sum =
          sum_of_parts(p, p.parts + (int64_t(blockIdx.x) * 16 + row) * p.padded + (c.piece + half) * p.rank + r, part);
      const uint4 pair = bf16_pair(sum, scale);
      *reinterpret_cast<uint2*>(vs + (half * 16 + row) * VSTRIDE + r) = make_uint2(pair.x, pair.y);
      *reinterpret_cast<uint2*>(vs + (half * 16 + row) * VSTRIDE + p.rank + r) = make_uint2(pair.z, pair.w);
    }
  }
  __syncthreads();
  units.run(vs, ws[units.w]);
}

// Both products of a tile of 16 rows in one launch: every workgroup multiplies the whole of x by its
// piece's A, 8 or 16 waves sharing k, and then a chunk of B's columns, units of 128, a
// wave at a time.  A comes from L2 for all workgroups but an XCD's first; what is won is a launch and
// the sums' way through memory.
constexpr int whole_waves(bool x8) { return x8 ? 8 : 16; }
template <bool X8>
__global__ __launch_bounds__(64 * whole_waves(X8)) void whole_kernel(AdapterParams p) {
  constexpr int RT = 1, WAVES = whole_waves(X8), J = RT, VSTRIDE = 32 * J + 8, WAVE = ring_bytes(X8, RT, 1);
  static_assert(WAVES * WAVE <= 150 * 1024 && RT * 1024 <= WAVE && RT <= WAVES && kUnitWeights<J> * 2 <= WAVE, "LDS");
  __shared__ __attribute__((aligned(16))) char smem[WAVES * WAVE];
  __shared__ __attribute__((aligned(16))) uint16_t vs[16 * VSTRIDE];
  f32x4_t* const red = reinterpret_cast<f32x4_t*>(smem);
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, n = lane & 15;
  const int tiles = plan_tiles(p);
  const Tile tile = p.plan.tiles[blockIdx.x];
  const int* const order = p.plan.rows + blockIdx.x * 16;
  const int any = order[0];
  int mine[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) mine[i] = order[4 * g + i];
  const Columns c = columns_of(p);
  if (tiles < 0) return write_nan<End::plain>(p, 16, c);
  if (int(blockIdx.x) >= tiles || (tile.slot < 0 && p.out == p.y)) return;
  const bool adds = tile.slot >= 0;
  if (adds) {
    f32x4_t acc[RT][1];
    multiply_ring<X8, RT, 1, WAVES>(p, tile, order, (mi::mx8::lds_t*)smem + w * WAVE, c.piece * p.rank, 0,
                                    ((X8 ? p.k : 2 * p.k) + 127) / 128, acc);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t) red[(w * RT + t) * 64 + lane] = acc[t][0];
  }
  Units<J, End::plain, WAVES> units(p, c, tile, mine, any);
  units.load(0);
  __syncthreads();
  // lane (g, n) of tile t holds ranks 16 t + 4 g .. + 3 of row n
  if (adds && tid < RT * 64) {
    const int r = w * 16 + 4 * g;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < WAVES; ++o) sum += red[(o * RT + w) * 64 + lane];
    if (r < p.rank) {
      const uint4 pair = bf16_pair(sum, p.scale[tile.slot]);
      *reinterpret_cast<uint2*>(vs + n * VSTRIDE + r) = make_uint2(pair.x, pair.y);
      *reinterpret_cast<uint2*>(vs + n * VSTRIDE + p.rank + r) = make_uint2(pair.z, pair.w);
    }
  }
  __syncthreads();
  units.run(vs, reinterpret_cast<uint16_t*>(smem) + w * kUnitWeights<J>);  // (the ring's and the sums' room)
}

int check_plan(const char* name, int64_t rows, int64_t slots) {
  if (rows < 0 || rows > kMaxRows || slots < 1 || slots > kMaxSlots)
    return mi::fail(MI_ERR_INVALID, "%s: %lld rows (0..2^22), %lld adapters (1..%d)", name, (long long)rows, (long long)slots,
                    kMaxSlots);
  return MI_OK;
}
int check_shape(const char* name, int64_t rows, int64_t slots, int64_t k, int64_t rank, int64_t pieces) {
  if (int rc = check_plan(name, rows, slots)) return rc;
  if (k <= 0 || k % 32 || k > mi::mx8::kMaxK || rank <= 0 || rank % 8 || rank > kMaxRank || pieces < 1 || pieces > kMaxPieces)
    return mi::fail(MI_ERR_INVALID, "%s: k %lld (multiple of 32, at most 2^20), rank %lld (multiple of 8, at most %d), "
                    "%lld pieces (1..%d)", name, (long long)k, (long long)rank, kMaxRank, (long long)pieces, kMaxPieces);
  return MI_OK;
}

// How a shrink launch shares k.  `steps` of a wave and `part_steps` of a workgroup are of 64 k,
// or of 128 bytes of x in tiles of 64 rows, whose workgroups share a CU by two.
struct Split {
  int64_t tiles;
  int groups, parts, part_steps;
  size_t bytes;
};
Split split_of(int64_t rows, int64_t slots, int64_t k, int64_t padded, bool x8) {
  Split s;
  const bool many = tile_rows(rows) == 64;
  const int64_t cus = mi::num_cus(), rank_tiles = padded / 16;
  const int64_t width = many && x8 ? 128 : kStep, unit = many && x8 ? 4 : 1;
  const int64_t steps = (k + width - 1) / width, waves = many ? kManyWaves : kWaves;
  const int64_t each = (steps + unit * waves - 1) / (unit * waves) * unit;
  int64_t best = 1, group = many && x8 ? kGroup / 2 : kGroup;
  s.tiles = max_tiles(rows, slots);
  if (!many) {
    // two steps a wave at least; then ranks apart, until every CU has two workgroups (32 rows, 8
    // adapters of rank 64, k 14,336: 4 rank tiles a workgroup 8.0 us, one 7.1)
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kMaxParts, (each + 1) / 2));
    while (group > 1 && s.tiles * ((rank_tiles + group - 1) / group) * most < 2 * cus) group /= 2;
    s.groups = int((rank_tiles + group - 1) / group);
    best = std::max<int64_t>(1, std::min<int64_t>(most, (2 * cus + s.tiles * s.groups - 1) / (s.tiles * s.groups)));
  } else {
    s.groups = int((rank_tiles + group - 1) / group);
    // rounds of workgroups (a part of one counts two thirds and more of a whole), of their steps and a start of
    // twelve, and the parts' way (us of both launches in a graph, by parts, * taken: the least or within 3 % of
    // it but at 4,105 rows, where two parts would be a tenth faster, which a count that fits the others does not give):
    //   1,031 x  3,584 ->  4,608, rank 16          1 29.0   2 21.1   5 17.7   6 18.1*  12 20.4
    //   4,105 x  4,096 ->  6,144, rank 16          1 50.5   2 44.8   4 49.5*  6 50.8    8 58.2
    //  18,240 x  4,096 ->  6,144, rank 16          1 153*   2 162    3 149    4 154     6 160
    //  the same, an eighth of the rows without     1 137*            3 144
    //  18,240 x 14,336 ->  4,096, rank 16, 8 bits  1 171    2 153    3 151*   6 149    12 152
    //   8,201 x  8,192 -> 10,240, rank 64          1 169*   2 170    3 176    6 189
    float least = 1e30f;
    for (int64_t parts = 1; parts <= std::min<int64_t>(kMaxParts, each / unit); ++parts) {
      const float r = float(s.tiles * s.groups * parts) / float(2 * cus), rounds = r <= 1.f ? 1.f : (2 * std::ceil(r) + r) / 3;
      const float cost = rounds * (float(each) / float(parts) + 12.f) + (0.6f + 0.012f * float(s.tiles)) * float(parts);
      if (cost < least) least = cost, best = parts;
    }
  }
  s.part_steps = int(((steps + best - 1) / best + unit - 1) / unit * unit);
  s.parts = int((steps + s.part_steps - 1) / s.part_steps);
  s.bytes = size_t(s.parts) * size_t(s.tiles) * tile_rows(rows) * size_t(padded) * 4;
  return s;
}

template <End END>
auto expand_of(bool many, bool by_waves, int j) {
  using Kernel = void (*)(AdapterParams);
  const Kernel kernels[2][4] = {
      {expand_kernel<1, 1, END>, expand_kernel<1, 2, END>, expand_kernel<1, 4, END>, expand_kernel<1, 8, END>},
      {expand_kernel<4, 1, END>, expand_kernel<4, 2, END>, expand_kernel<4, 4, END>, expand_kernel<4, 8, END>}};
  if (by_waves) return Kernel(j ? expand_waves_kernel<2, END> : expand_waves_kernel<1, END>);
  return kernels[many][j];
}

// One launch for few rows where its workgroups, which each read their piece's A, are a round at most, and A is
// short (us in a graph, two launches / one; adapters of rank 16):
//   1 row               k 896 -> 1,152 7.1 / 5.9    k 4,096 -> 6,144 7.4 / 6.6    k 8,192 -> 10,240 (16 rows) 8.6 / 10.6
//                       k 14,336 -> 4,096 8.3 / 11.1
//   32 rows, 8 adapters k 4,096 -> 6,144 9.9 / 8.9  k 4,096 -> 28,672 11.6 / 15.8 (more than a round)
//   40 rows, 20         k 896 -> 9,728 10.4 / 8.6
//   48 rows, 24         k 3,584 -> 4,608 11.0 / 8.6 k 18,944 -> 3,584 12.5 / 17.5
//   256 rows, 64        k 4,096 -> 6,144 16.8 / 20.1 (more than a round)
constexpr int kMaxChunk = 1024;
bool in_one_launch(int64_t rows, int64_t slots, int64_t k, int64_t rank, int64_t pieces, int64_t n) {
  return tile_rows(rows) == 16 && rank <= 16 && k <= 4096 && max_tiles(rows, slots) * (n / kMaxChunk + pieces) <= mi::num_cus();
}

}  // namespace

extern "C" size_t mi_adapter_plan_size(int64_t rows, int64_t slots) {
  if (check_plan("adapter_plan_size", rows, slots)) return 0;
  // (of fewer rows too: tiles of 16 may take more)
  return std::max(plan_size(rows, slots), plan_size(std::min(rows, kFewRows), slots));
}

extern "C" int mi_adapter_plan(void* plan, size_t plan_bytes, const int32_t* slot_of_row, int64_t rows, int64_t slots,
                               mi_stream_t stream) {
  const char* const name = "adapter_plan";
  mi::clear_error();
  if (int rc = check_plan(name, rows, slots)) return rc;
  // (no rows: the plan that was there is none either, for graphs that are replayed with it)
  if (rows == 0 && !plan) return MI_OK;
  if (!plan || (rows && !slot_of_row)) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if ((reinterpret_cast<uintptr_t>(plan) & 15) || (reinterpret_cast<uintptr_t>(slot_of_row) & 3))
    return mi::fail(MI_ERR_INVALID, "%s: the plan must be 16-byte aligned, the slots 4-byte", name);
  const size_t need = plan_size(rows, slots);
  if (plan_bytes < need)
    return mi::fail(MI_ERR_WORKSPACE, "%s: the plan takes %zu bytes, %zu given", name, need, plan_bytes);
  const mi::Rows to = {plan, 0, 1, int64_t(need)}, from = {slot_of_row, 0, 1, rows * 4};
  if (mi::rows_meet(to, from)) return mi::fail(MI_ERR_INVALID, "%s: the plan overlaps the slots", name);
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), slot_of_row, int(rows),
                     int(slots), tile_rows(rows), view(plan, rows, slots));
  return mi::check_launch(name);
}

extern "C" size_t mi_add_adapters_workspace_size(int64_t rows, int64_t slots, int64_t k, int64_t rank, int64_t pieces,
                                                int64_t n, int32_t silu) {
  if (check_shape("add_adapters_workspace_size", rows, slots, k, rank, pieces) || rows == 0) return 0;
  if (!silu && in_one_launch(rows, slots, k, rank, pieces, n)) return 0;
  const int64_t padded = (pieces * rank + 15) / 16 * 16;
  return std::max(split_of(rows, slots, k, padded, false).bytes, split_of(rows, slots, k, padded, true).bytes);
}

extern "C" int mi_add_adapters(const void* y, int64_t y_stride, const void* x, int64_t x_stride, const void* x_scales,
                               int64_t x_scales_stride, const void* a, const void* b, const float* scale, int64_t slots,
                               int64_t k, int64_t rank, const int32_t* piece_columns, int64_t pieces, void* out,
                               int64_t out_stride, void* out_scales, int64_t out_scales_stride, const void* plan,
                               int64_t rows, int32_t silu, void* workspace, size_t workspace_bytes, mi_stream_t stream) {
  const char* const name = "add_adapters";
  mi::clear_error();
  if (int rc = check_shape(name, rows, slots, k, rank, pieces)) return rc;
  if (!piece_columns) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  AdapterParams p = {};
  int64_t n = 0;
  for (int i = 0; i < pieces; ++i) {
    if (piece_columns[i] <= 0 || piece_columns[i] % 16 || piece_columns[i] > 1 << 20)
      return mi::fail(MI_ERR_INVALID, "%s: a piece of %d columns (multiples of 16 up to 2^20)", name, piece_columns[i]);
    n += piece_columns[i];
    p.end[i] = int(n);
  }
  const int64_t out_n = silu ? n / 2 : n;
  if (silu && (pieces != 2 || piece_columns[0] != piece_columns[1]))
    return mi::fail(MI_ERR_INVALID, "%s: SiLU is of gate and up, two pieces of as many columns", name);
  const bool sums = silu == MI_SILU_SUMS, steps = silu == MI_SILU_STEPS;
  if (out_scales && (!silu || steps || out_n % mi::mx8::kBlock))
    return mi::fail(MI_ERR_INVALID, "%s: rows in 8 bits are the gated sum's, a multiple of %d columns; got %lld", name,
                    mi::mx8::kBlock, (long long)out_n);
  if (rows == 0) return MI_OK;
  const int64_t each = x_scales ? 1 : 2, out_each = out_scales ? 1 : 2, y_each = sums ? 4 : 2;
  const int64_t scale_bytes = (k / 32 + 15) & ~int64_t(15);
  if (rows == 1) {  // (nothing lies at a single row's stride)
    y_stride = n, out_stride = out_n, out_scales_stride = out_n / 32;
    x_stride = (k + 15) & ~int64_t(15), x_scales_stride = scale_bytes;
  }
  if (!y || !x || !a || !b || !scale || !out || !plan)
    return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  const uintptr_t aligned = reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) |
                            reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(out) |
                            reinterpret_cast<uintptr_t>(plan) | reinterpret_cast<uintptr_t>(workspace) |
                            reinterpret_cast<uintptr_t>(x_scales);
  if ((aligned & 15) || (y_stride * y_each) % 16 || (out_stride * out_each) % 16 || (x_scales && x_scales_stride % 16) || (x_stride * each) % 16 || (reinterpret_cast<uintptr_t>(scale) & 3))
    return mi::fail(MI_ERR_INVALID, "%s: rows, factors, plan and workspace must be 16-byte aligned", name);
  if (out_stride < out_n || (out_scales && out_scales_stride < out_n / 32) || x_stride < 0 || y_stride < 0 || (x_scales && x_scales_stride < scale_bytes))
    return mi::fail(MI_ERR_INVALID, "%s: row strides %lld, %lld, %lld, %lld for %lld columns", name, (long long)y_stride,
                    (long long)x_stride, (long long)x_scales_stride, (long long)out_stride, (long long)n);
  const int64_t padded = (pieces * rank + 15) / 16 * 16;
  const Split split = split_of(rows, slots, k, padded, x_scales != nullptr);
  const int64_t tiles = split.tiles;
  const bool whole = !silu && in_one_launch(rows, slots, k, rank, pieces, n);
  const size_t need = whole ? 0 : split.bytes;
  if (need && !workspace) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if (workspace_bytes < need)
    return mi::fail(MI_ERR_WORKSPACE, "%s: the workspace takes %zu bytes, %zu given", name, need, workspace_bytes);
  // (rows of out are written while others are still read; a row of y only by who writes it)
  const bool in_place = !silu && out == y && out_stride == y_stride;
  const mi::Rows to = {out, out_stride * out_each, rows, out_n * out_each},
                 to_scales = {out_scales, out_scales_stride, out_scales ? rows : 0, out_n / 32};
  const mi::Rows from[] = {{y, y_stride * y_each, in_place ? 0 : rows, n * y_each},
                           {x, x_stride * each, rows, k * each},
                           {x_scales, x_scales_stride, x_scales ? rows : 0, k / 32},
                           {a, 0, 1, slots * pieces * rank * k * 2},
                           {b, 0, 1, slots * n * rank * 2},
                           {scale, 0, 1, slots * 4},
                           {plan, 0, 1, int64_t(plan_size(rows, slots))},
                           {workspace, 0, need ? 1 : 0, int64_t(need)}};
  bool meet = mi::rows_meet(to, to_scales);
  for (const mi::Rows& r : from) meet = meet || mi::rows_meet(to, r) || mi::rows_meet(to_scales, r);
  if (meet) return mi::fail(MI_ERR_INVALID, "%s: out overlaps another argument (without SiLU it may be y itself)", name);
  // (sums are written there while others still read x and A, and read before B and y are)
  if (need) {
    const mi::Rows held = from[7], all_y = {y, y_stride * y_each, rows, n * y_each};
    meet = mi::rows_meet(held, all_y);
    for (int i = 1; i < 7; ++i) meet = meet || mi::rows_meet(held, from[i]);
  }
  if (meet) return mi::fail(MI_ERR_INVALID, "%s: the workspace overlaps another argument", name);
  p.x = static_cast<const char*>(x);
  p.x_stride = x_stride * each;
  p.xs = static_cast<const char*>(x_scales);
  p.xs_stride = x_scales_stride;
  p.a = static_cast<const uint16_t*>(a);
  p.b = static_cast<const uint16_t*>(b);
  p.scale = scale;
  p.y = static_cast<const uint16_t*>(y);
  p.y_stride = y_stride;
  p.out = static_cast<uint16_t*>(out);
  p.o_stride = out_stride;
  p.scales = static_cast<uint8_t*>(out_scales);
  p.s_stride = out_scales_stride;
  p.up = int(out_n);
  p.plan = view(const_cast<void*>(plan), rows, slots);
  p.parts = static_cast<float*>(workspace);
  p.rows = int(rows);
  p.slots = int(slots);
  p.k = int(k);
  p.n = int(n);
  p.rank = int(rank);
  p.eighths = int(rank / 8);
  p.per_eighths = (65536 + p.eighths - 1) / p.eighths;
  p.ranks = int(pieces * rank);
  p.padded = int(padded);
  p.max_tiles = int(tiles);
  p.pieces = int(pieces);
  p.part_steps = split.part_steps;
  p.n_parts = split.parts;
  p.group_ranks = int(((padded / 16 + split.groups - 1) / split.groups) * 16);
  const bool x8 = p.xs != nullptr, many = tile_rows(rows) == 64;
  // columns of a workgroup: few where there are few tiles, so that every CU has some
  // Tiles of 16 rows are a wave's work: a unit a wave where there are units enough for more than two workgroups a CU,
  // and the rank is small; else a workgroup fetches a unit's B for one of its waves (us of both launches in a
  // graph, one unit a workgroup / a wave): 32 rows of 8 adapters, 4,096 -> 2 x 14,336 with SiLU, rank 16 17.9 / 13.5,
  // 32 20.0 / 16.0, 64 24.0 / 26.4; 48 of 24, 3,584 -> 2 x 18,944 35.1 / 16.1; 300 of 8, 14,336 -> 4,096 13.4 / 13.1; 32 of
  // 8, 14,336 -> 4,096 (352 units) 10.9 / 11.2, rank 64 14.6 / 16.7; one row -> 2 x 14,336 8.8 / 9.7.
  const int64_t units = tiles * ((out_n + 127) / 128);
  const bool by_waves = !many && rank <= 32 && units > 2 * mi::num_cus();
  p.chunk = 128;
  const int64_t enough = whole ? mi::num_cus() : by_waves ? 2 * mi::num_cus() : 8 * mi::num_cus();
  while (p.chunk < kMaxChunk && tiles * ((out_n + p.chunk - 1) / p.chunk) > enough) p.chunk *= 2;
  int chunks = 0;
  for (int i = 0; i < (silu ? 1 : pieces); ++i) p.end_chunk[i] = chunks += (piece_columns[i] + p.chunk - 1) / p.chunk;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(uint32_t(tiles), uint32_t(p.n_parts), uint32_t(split.groups)), block(64 * kWaves);
  const int rt = p.group_ranks / 16;
  using Kernel = void (*)(AdapterParams);
  if (whole) {
    hipLaunchKernelGGL(x8 ? whole_kernel<true> : whole_kernel<false>, dim3(uint32_t(tiles), uint32_t(chunks)),
                       dim3(64 * whole_waves(x8)), 0, s, p);
    return mi::check_launch(name);
  }
  const Kernel few[2][kGroup] = {
      {shrink_few_kernel<false, 1>, shrink_few_kernel<false, 2>, shrink_few_kernel<false, 3>, shrink_few_kernel<false, 4>},
      {shrink_few_kernel<true, 1>, shrink_few_kernel<true, 2>, shrink_few_kernel<true, 3>, shrink_few_kernel<true, 4>}};
  const Kernel wide[2][kGroup] = {
      {shrink_many_kernel<false, 1>, shrink_many_kernel<false, 2>, shrink_many_kernel<false, 3>, shrink_many_kernel<false, 4>},
      {shrink_many_kernel<true, 1>, shrink_many_kernel<true, 2>, nullptr, nullptr}};
  hipLaunchKernelGGL((many ? wide : few)[x8][rt - 1], grid, dim3(64 * (many ? kManyWaves : kWaves)), 0, s, p);
  const int j = rank <= 16 ? 0 : rank <= 32 ? 1 : rank <= 64 ? 2 : 3;
  const Kernel expand = !silu   ? expand_of<End::plain>(many, by_waves, j)
                        : steps ? expand_of<End::steps>(many, by_waves, j)
                        : sums  ? (p.scales ? expand_of<End::sums8> : expand_of<End::sums>)(many, by_waves, j)
                                : (p.scales ? expand_of<End::silu8> : expand_of<End::silu>)(many, by_waves, j);
  hipLaunchKernelGGL(expand, dim3(uint32_t(tiles), uint32_t(chunks)), block, 0, s, p);
  return mi::check_launch(name);
}

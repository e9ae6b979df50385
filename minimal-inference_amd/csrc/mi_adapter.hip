// Low-rank adapters of many requests beside a shared projection: out = y + scale B (A x),
// A [r][k] and B [n][r] of the row's own adapter.  The projection's outputs are one to
// eight pieces (q, k, v), each with r rows of A of its own.
//
//   plan   : rows sorted by adapter into tiles of up to 64 rows of one adapter, once per
//            batch.  Which row comes where in its adapter's tiles is of no matter: a row's
//            result depends on its own operands alone.
//   shrink : v = A x of a tile, k in parts over workgroups; sums in fp32.
//   expand : the parts' sum, times scale, as a pair of bf16 (v and what its rounding left: 16
//            bits of v), times B in fp32, plus y, one rounding.
//
// Bound: for prompts HBM, one read of x, one of y and the write of out; A and B come from the
// caches.  For decode steps the two launches' start and end, and the read of the adapters.
#include <algorithm>

#include "mi_mx8.h"
#include "mi_overlap.h"

namespace {

using mi::bf16x8_t;
using mi::f32x4_t;
using mi::mx8::u32x2_t;
using mi::mx8::u32x4_t;

constexpr int kTile = 64;        // rows of a tile
constexpr int kMaxSlots = 1023;  // (and one more count for the rows without)
constexpr int kMaxRank = 128;
constexpr int kMaxPieces = 8;
constexpr int64_t kMaxRows = 1 << 22;
constexpr int kWaves = 4;
constexpr int kStep = 64;  // k of a wave's step
constexpr int kMaxParts = 16;
constexpr int kGroup = 4;  // 16-rank tiles of a workgroup

struct Tile {
  int slot, first, count, unused;  // slot -1: rows without an adapter
};

// A plan: the number of tiles in 16 bytes, the tiles, the rows in their order.
int64_t max_tiles(int64_t rows, int64_t slots) { return std::min(rows, slots + 1) + rows / kTile; }
struct PlanView {
  int* count;
  Tile* tiles;
  int* order;
};
PlanView view(void* plan, int64_t rows, int64_t slots) {
  char* const p = static_cast<char*>(plan);
  return {reinterpret_cast<int*>(p), reinterpret_cast<Tile*>(p + 16),
          reinterpret_cast<int*>(p + 16 + 16 * max_tiles(rows, slots))};
}

constexpr int kPlanThreads = 1024;

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const int* slot_of_row, int rows, int slots, PlanView p) {
  __shared__ int count[kPlanThreads], first[kPlanThreads], tiles[kPlanThreads];
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
  const int mine = count[tid], need = (mine + kTile - 1) / kTile;
  first[tid] = mine;
  tiles[tid] = need;
  __syncthreads();
  for (int d = 1; d < kPlanThreads; d *= 2) {  // sums up to and with each slot
    const int a = tid >= d ? first[tid - d] : 0, b = tid >= d ? tiles[tid - d] : 0;
    __syncthreads();
    first[tid] += a;
    tiles[tid] += b;
    __syncthreads();
  }
  const int begin = first[tid] - mine, tile = tiles[tid] - need;
  for (int i = 0; i < need; ++i)
    p.tiles[tile + i] = {tid < slots ? tid : -1, begin + i * kTile, min(kTile, mine - i * kTile), 0};
  if (tid == kPlanThreads - 1) *p.count = tiles[tid];
  count[tid] = begin;
  __syncthreads();
  for (int row = tid; row < rows; row += kPlanThreads) p.order[places(at(row), count)] = row;
}

struct AdapterParams {
  const char* x;      // bf16 rows, or codes
  int64_t x_stride;   // bytes
  const uint8_t* xs;  // scale bytes; null: x is bf16
  int64_t xs_stride;
  const uint16_t* a;  // [slots][pieces * rank][k]
  const uint16_t* b;  // [slots][n][rank]
  const float* scale;
  const uint16_t* y;
  int64_t y_stride;
  uint16_t* out;
  int64_t o_stride;
  PlanView plan;
  float* parts;  // [part][tile][row of 64][ranks, padded]
  int k, n, rank, ranks, padded;  // ranks = pieces * rank, padded to 16
  int n_parts, part_steps, max_tiles;
  int pieces, chunk;  // columns of an expand workgroup
  int end[kMaxPieces];       // columns,
  int end_chunk[kMaxPieces]; // chunks up to and with each piece
};

// In a step of 64 k, lane (g, n) holds row n's k from 16 g on: its first eight are one
// product's operand, the other eight the next one's.  (Which k comes where is of no matter
// as long as both operands agree.)
template <bool X8, int RT, int NB>
__device__ void shrink(const AdapterParams& p, const Tile& tile, char* smem) {
  const int w = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
  const int g = lane >> 4, n = lane & 15;
  const int rank0 = int(blockIdx.z) * kGroup * 16;
  const uint16_t* a[RT];
  const char* x[NB];
  const uint8_t* xs[NB];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = rank0 + t * 16 + n;  // (past the last rank any row will do: its sums are not kept)
    a[t] = p.a + (int64_t(tile.slot) * p.ranks + (r < p.ranks ? r : 0)) * p.k + 16 * g;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int i = b * 16 + n;
    const int64_t row = p.plan.order[tile.first + (i < tile.count ? i : 0)];
    x[b] = p.x + row * p.x_stride + (X8 ? 16 : 32) * g;
    if constexpr (X8) xs[b] = p.xs + row * p.xs_stride + g / 2;
  }
  const int all = (p.k + kStep - 1) / kStep;
  const int end = min(all, int(blockIdx.y + 1) * p.part_steps);
  struct Set {
    uint4 a[RT][2], x[NB][2];
    float s[NB];
  };
  auto load = [&](Set& s, int step) {
    const int k0 = step * kStep;
    const bool in = step < end && k0 + 16 * g < p.k;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      s.a[t][0] = in ? mi::load16(a[t] + k0) : none;
      s.a[t][1] = in ? mi::load16(a[t] + k0 + 8) : none;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      if constexpr (X8) {
        s.x[b][0] = in ? mi::load16(x[b] + k0) : none;
        s.s[b] = in ? mi::mx8::scale_f32(xs[b][k0 / 32]) : 0.f;
      } else {
        s.x[b][0] = in ? mi::load16(x[b] + 2 * k0) : none;
        s.x[b][1] = in ? mi::load16(x[b] + 2 * k0 + 16) : none;
      }
    }
  };
  f32x4_t acc[RT][NB];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[t][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  Set cur, next;
  int step = int(blockIdx.y) * p.part_steps + w;
  load(cur, step);
  for (; step < end; step += kWaves) {
    load(next, step + kWaves);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        bf16x8_t v;
        if constexpr (X8) {
          const u32x2_t lo = mi::mx8::to_bf16(h ? cur.x[b][0].z : cur.x[b][0].x, cur.s[b]);
          const u32x2_t hi = mi::mx8::to_bf16(h ? cur.x[b][0].w : cur.x[b][0].y, cur.s[b]);
          v = mi::as_bf16x8(make_uint4(lo.x, lo.y, hi.x, hi.y));
        } else {
          v = mi::as_bf16x8(cur.x[b][h]);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t][b] = mi::mfma_16x16x32_bf16(mi::as_bf16x8(cur.a[t][h]), v, acc[t][b]);
      }
    cur = next;
  }
  // Lane (g, n) holds ranks 4 g .. 4 g + 3 of a tile for row n of a block.
  f32x4_t* const red = reinterpret_cast<f32x4_t*>(smem);
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int b = 0; b < NB; ++b) red[(w * RT * NB + t * NB + b) * 64 + lane] = acc[t][b];
  __syncthreads();
  for (int q = w; q < RT * NB; q += kWaves) {
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int o = 0; o < kWaves; ++o) sum += red[(o * RT * NB + q) * 64 + lane];
    const int row = q % NB * 16 + n, r = rank0 + q / NB * 16 + 4 * g;
    if (row < tile.count && r < p.padded)
      *reinterpret_cast<f32x4_t*>(p.parts + ((int64_t(blockIdx.y) * p.max_tiles + blockIdx.x) * kTile + row) * p.padded + r) = sum;
  }
}

template <bool X8, int RT>
__global__ __launch_bounds__(64 * kWaves) void shrink_kernel(AdapterParams p) {
  __shared__ __attribute__((aligned(16))) char smem[kWaves * RT * (kTile / 16) * 1024];
  if (int(blockIdx.x) >= *p.plan.count) return;
  const Tile tile = p.plan.tiles[blockIdx.x];
  if (tile.slot < 0) return;
  if (tile.count <= 16) shrink<X8, RT, 1>(p, tile, smem);
  else shrink<X8, RT, kTile / 16>(p, tile, smem);
}

// J: products of 32 that a piece's pairs of ranks take.
template <int J>
__global__ __launch_bounds__(64 * kWaves) void expand_kernel(AdapterParams p) {
  constexpr int kMaxPair = 4 * J * 8;  // pairs of bf16 of a row, side by side: the roundings, then what they left
  __shared__ __attribute__((aligned(16))) uint16_t vs[kTile * (kMaxPair + 8)];
  if (int(blockIdx.x) >= *p.plan.count) return;
  const Tile tile = p.plan.tiles[blockIdx.x];
  if (tile.slot < 0 && p.out == p.y) return;
  int piece = 0;
  while (int(blockIdx.y) >= p.end_chunk[piece]) ++piece;
  const int begin = piece ? p.end[piece - 1] : 0, before = piece ? p.end_chunk[piece - 1] : 0;
  const int c0 = begin + (int(blockIdx.y) - before) * p.chunk, c1 = min(c0 + p.chunk, p.end[piece]);
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int g = lane >> 4, n = lane & 15;
  const int stride = kMaxPair + 8;  // (the rows of an operand on distinct banks)
  const int nb = (tile.count + 15) / 16;
  if (tile.slot >= 0) {
    const float scale = p.scale[tile.slot];
    const int fours = p.rank / 4;
    const int64_t part = int64_t(p.max_tiles) * kTile * p.padded;
    for (int i = tid; i < tile.count * fours; i += 64 * kWaves) {
      const int row = i / fours, r = i % fours * 4;
      const float* const from = p.parts + (int64_t(blockIdx.x) * kTile + row) * p.padded + piece * p.rank + r;
      f32x4_t sum = *reinterpret_cast<const f32x4_t*>(from);
      for (int o = 1; o < p.n_parts; ++o) sum += *reinterpret_cast<const f32x4_t*>(from + o * part);
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float u = sum[2 * j] * scale, v = sum[2 * j + 1] * scale;
        hi[j] = mi::cvt_pk_bf16(u, v);
        const float du = u - mi::bf16_lo(hi[j]), dv = v - mi::bf16_hi(hi[j]);
        // (an infinity leaves nothing)
        lo[j] = mi::cvt_pk_bf16(isfinite(mi::bf16_lo(hi[j])) ? du : 0.f, isfinite(mi::bf16_hi(hi[j])) ? dv : 0.f);
      }
      *reinterpret_cast<uint2*>(vs + row * stride + r) = make_uint2(hi[0], hi[1]);
      *reinterpret_cast<uint2*>(vs + row * stride + p.rank + r) = make_uint2(lo[0], lo[1]);
    }
    __syncthreads();
  }
  const int eighths = p.rank / 8;
  int from[J];  // of a lane's eight ranks of product j, -1: past the last pair
#pragma unroll
  for (int j = 0; j < J; ++j) from[j] = 4 * j + g < 2 * eighths ? (4 * j + g) % eighths * 8 : -1;
  int64_t row[kTile / 16];
#pragma unroll
  for (int b = 0; b < kTile / 16; ++b) {
    const int i = b * 16 + n;
    row[b] = p.plan.order[tile.first + (i < tile.count ? i : 0)];
  }
  const uint16_t* const weights = p.b + int64_t(max(tile.slot, 0)) * p.n * p.rank;
  for (int c = c0 + w * 32; c < c1; c += 32 * kWaves) {  // two tiles of 16 columns
    const int col = c + (g & 1) * 16 + (g >> 1) * 8;
    const bool mine = col < c1;
    uint4 yv[kTile / 16];
#pragma unroll
    for (int b = 0; b < kTile / 16; ++b)
      if (b < nb && mine) yv[b] = mi::load16_nt(p.y + row[b] * p.y_stride + col);
    bf16x8_t wt[2][J];
    if (tile.slot >= 0) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = c + 16 * t + n;  // (the second tile may lie past the piece: not kept)
#pragma unroll
        for (int j = 0; j < J; ++j)
          wt[t][j] = mi::as_bf16x8(from[j] >= 0 ? mi::load16(weights + int64_t(r < c1 ? r : c) * p.rank + from[j])
                                                : make_uint4(0u, 0u, 0u, 0u));
      }
    }
#pragma unroll
    for (int b = 0; b < kTile / 16; ++b) {
      if (b >= nb) break;
      uint4 o = yv[b];
      if (tile.slot >= 0) {
        f32x4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint4 q = *reinterpret_cast<const uint4*>(vs + (b * 16 + n) * stride + (4 * j + g) * 8);
          const bf16x8_t v = mi::as_bf16x8(from[j] >= 0 ? q : make_uint4(0u, 0u, 0u, 0u));
          s[0] = mi::mfma_16x16x32_bf16(wt[0][j], v, s[0]);
          s[1] = mi::mfma_16x16x32_bf16(wt[1][j], v, s[1]);
        }
        // Lane (g, n) holds columns 4 g .. 4 g + 3 of either tile; lanes change places, so that
        // each has eight columns side by side.
        float d[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const auto e = __builtin_amdgcn_permlane16_swap(__float_as_uint(s[0][i]), __float_as_uint(s[1][i]), false, false);
          d[i] = __uint_as_float(e[0]);
          d[4 + i] = __uint_as_float(e[1]);
        }
        o.x = mi::cvt_pk_bf16(mi::bf16_lo(o.x) + d[0], mi::bf16_hi(o.x) + d[1]);
        o.y = mi::cvt_pk_bf16(mi::bf16_lo(o.y) + d[2], mi::bf16_hi(o.y) + d[3]);
        o.z = mi::cvt_pk_bf16(mi::bf16_lo(o.z) + d[4], mi::bf16_hi(o.z) + d[5]);
        o.w = mi::cvt_pk_bf16(mi::bf16_lo(o.w) + d[6], mi::bf16_hi(o.w) + d[7]);
      }
      if (mine && b * 16 + n < tile.count) mi::store16(p.out + row[b] * p.o_stride + col, o);
    }
  }
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

int parts_of(int64_t tiles, int64_t k, int64_t groups) {
  const int64_t steps = (k + kStep - 1) / kStep, most = std::min<int64_t>(kMaxParts, (steps + kWaves - 1) / kWaves);
  const int64_t want = (2 * mi::num_cus() + tiles * groups - 1) / (tiles * groups);
  return int(std::max<int64_t>(1, std::min(most, want)));
}

}  // namespace

extern "C" size_t mi_adapter_plan_size(int64_t rows, int64_t slots) {
  if (check_plan("adapter_plan_size", rows, slots)) return 0;
  return 16 + 16 * size_t(max_tiles(rows, slots)) + 4 * size_t(rows);
}

extern "C" int mi_adapter_plan(void* plan, size_t plan_bytes, const int32_t* slot_of_row, int64_t rows, int64_t slots,
                               mi_stream_t stream) {
  const char* const name = "adapter_plan";
  mi::clear_error();
  if (int rc = check_plan(name, rows, slots)) return rc;
  if (rows == 0) return MI_OK;
  if (!plan || !slot_of_row) return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  if ((reinterpret_cast<uintptr_t>(plan) & 15) || (reinterpret_cast<uintptr_t>(slot_of_row) & 3))
    return mi::fail(MI_ERR_INVALID, "%s: the plan must be 16-byte aligned, the slots 4-byte", name);
  const size_t need = mi_adapter_plan_size(rows, slots);
  if (plan_bytes < need)
    return mi::fail(MI_ERR_WORKSPACE, "%s: the plan takes %zu bytes, %zu given", name, need, plan_bytes);
  const mi::Rows to = {plan, 0, 1, int64_t(need)}, from = {slot_of_row, 0, 1, rows * 4};
  if (mi::rows_meet(to, from)) return mi::fail(MI_ERR_INVALID, "%s: the plan overlaps the slots", name);
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<hipStream_t>(stream), slot_of_row, int(rows),
                     int(slots), view(plan, rows, slots));
  return mi::check_launch(name);
}

extern "C" size_t mi_add_adapters_workspace_size(int64_t rows, int64_t slots, int64_t k, int64_t rank, int64_t pieces) {
  if (check_shape("add_adapters_workspace_size", rows, slots, k, rank, pieces) || rows == 0) return 0;
  const int64_t tiles = max_tiles(rows, slots), padded = (pieces * rank + 15) / 16 * 16;
  const int64_t groups = (padded / 16 + kGroup - 1) / kGroup;
  return size_t(parts_of(tiles, k, groups)) * size_t(tiles) * kTile * size_t(padded) * 4;
}

extern "C" int mi_add_adapters(const void* y, int64_t y_stride, const void* x, int64_t x_stride, const void* x_scales,
                               int64_t x_scales_stride, const void* a, const void* b, const float* scale, int64_t slots,
                               int64_t k, int64_t rank, const int32_t* piece_columns, int64_t pieces, void* out,
                               int64_t out_stride, const void* plan, int64_t rows, void* workspace,
                               size_t workspace_bytes, mi_stream_t stream) {
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
  if (rows == 0) return MI_OK;
  const int64_t each = x_scales ? 1 : 2;
  if (rows == 1) y_stride = out_stride = n, x_stride = (k + 15) & ~int64_t(15), x_scales_stride = k / 32;
  if (!y || !x || !a || !b || !scale || !out || !plan || !workspace)
    return mi::fail(MI_ERR_INVALID, "%s: null pointer argument", name);
  const uintptr_t aligned = reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) |
                            reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(out) |
                            reinterpret_cast<uintptr_t>(plan) | reinterpret_cast<uintptr_t>(workspace);
  if ((aligned & 15) || ((y_stride | out_stride) & 7) || (x_stride * each) % 16 || (reinterpret_cast<uintptr_t>(scale) & 3))
    return mi::fail(MI_ERR_INVALID, "%s: rows, factors, plan and workspace must be 16-byte aligned", name);
  if (out_stride < n || x_stride < 0 || y_stride < 0 || x_scales_stride < 0)
    return mi::fail(MI_ERR_INVALID, "%s: row strides %lld, %lld, %lld, %lld for %lld columns", name, (long long)y_stride,
                    (long long)x_stride, (long long)x_scales_stride, (long long)out_stride, (long long)n);
  const int64_t tiles = max_tiles(rows, slots), padded = (pieces * rank + 15) / 16 * 16;
  const int groups = int((padded / 16 + kGroup - 1) / kGroup);
  const int parts = parts_of(tiles, k, groups);
  const size_t need = size_t(parts) * size_t(tiles) * kTile * size_t(padded) * 4;
  if (workspace_bytes < need)
    return mi::fail(MI_ERR_WORKSPACE, "%s: the workspace takes %zu bytes, %zu given", name, need, workspace_bytes);
  // (rows of out are written while others are still read; a row of y only by who writes it)
  const bool in_place = out == y && out_stride == y_stride;
  const mi::Rows to = {out, out_stride * 2, rows, n * 2};
  const mi::Rows from[] = {{y, y_stride * 2, in_place ? 0 : rows, n * 2},
                           {x, x_stride * each, rows, k * each},
                           {x_scales, x_scales_stride, x_scales ? rows : 0, k / 32},
                           {a, 0, 1, slots * pieces * rank * k * 2},
                           {b, 0, 1, slots * n * rank * 2},
                           {scale, 0, 1, slots * 4},
                           {plan, 0, 1, int64_t(mi_adapter_plan_size(rows, slots))},
                           {workspace, 0, 1, int64_t(need)}};
  for (const mi::Rows& r : from)
    if (mi::rows_meet(to, r)) return mi::fail(MI_ERR_INVALID, "%s: out overlaps another argument (it may be y itself)", name);
  p.x = static_cast<const char*>(x);
  p.x_stride = x_stride * each;
  p.xs = static_cast<const uint8_t*>(x_scales);
  p.xs_stride = x_scales_stride;
  p.a = static_cast<const uint16_t*>(a);
  p.b = static_cast<const uint16_t*>(b);
  p.scale = scale;
  p.y = static_cast<const uint16_t*>(y);
  p.y_stride = y_stride;
  p.out = static_cast<uint16_t*>(out);
  p.o_stride = out_stride;
  p.plan = view(const_cast<void*>(plan), rows, slots);
  p.parts = static_cast<float*>(workspace);
  p.k = int(k);
  p.n = int(n);
  p.rank = int(rank);
  p.ranks = int(pieces * rank);
  p.padded = int(padded);
  p.max_tiles = int(tiles);
  p.pieces = int(pieces);
  const int steps = int((k + kStep - 1) / kStep);
  p.part_steps = (steps + parts - 1) / parts;
  p.n_parts = (steps + p.part_steps - 1) / p.part_steps;
  // columns of a workgroup: few where there are few tiles, so that every CU has some
  p.chunk = 128;
  while (p.chunk < 1024 && tiles * ((n + p.chunk - 1) / p.chunk) > 8 * mi::num_cus()) p.chunk *= 2;
  int chunks = 0;
  for (int i = 0; i < pieces; ++i) p.end_chunk[i] = chunks += (piece_columns[i] + p.chunk - 1) / p.chunk;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(uint32_t(tiles), uint32_t(p.n_parts), uint32_t(groups)), block(64 * kWaves);
  const int rt = int(std::min<int64_t>(padded / 16, kGroup));
  const auto shrink = p.xs ? (rt == 1 ? shrink_kernel<true, 1> : rt == 2 ? shrink_kernel<true, 2>
                              : rt == 3 ? shrink_kernel<true, 3> : shrink_kernel<true, 4>)
                           : (rt == 1 ? shrink_kernel<false, 1> : rt == 2 ? shrink_kernel<false, 2>
                              : rt == 3 ? shrink_kernel<false, 3> : shrink_kernel<false, 4>);
  hipLaunchKernelGGL(shrink, grid, block, 0, s, p);
  const auto expand = rank <= 16 ? expand_kernel<1> : rank <= 32 ? expand_kernel<2> : rank <= 64 ? expand_kernel<4> : expand_kernel<8>;
  hipLaunchKernelGGL(expand, dim3(uint32_t(tiles), uint32_t(chunks)), block, 0, s, p);
  return mi::check_launch(name);
}

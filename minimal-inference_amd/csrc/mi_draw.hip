// One draw per row from given uniform numbers: temperature, top-k, top-p, min-p.
//
// With w_i = exp((l_i - max l) / t), tokens ordered by descending logit and then
// ascending index: kept are the first top_k; of them those with w_i >= min_p; of those
// the shortest prefix whose mass reaches top_p of theirs; always the first.  The draw is
// the lowest index whose cumulative kept weight, in index order, exceeds u times the
// kept total.
//
// A bf16 logit is one of few values, so a row is a histogram of whole numbers: counts
// per value say all that order and mass need, one exp per value in 64 bits is enough,
// and nothing depends on the order of additions.  One or two launches, no atomics on
// memory and nothing kept between calls:
//   count  one workgroup per 8,192 to 32,768 tokens, on the XCD of the row's draw (its L2
//          then holds the counts: 0.4 us): largest value with its lowest index, and
//          the counts of the 2 x 38 x 128 values of magnitude [2^-30, 2^8) and of zero
//          in LDS, written as 16 bits each.
//   draw   one workgroup per row: the counts' sum over the chunks, ten values to a
//          thread; prefix sums of count and mass give the last kept value and how many
//          tokens of it; each chunk's kept mass gives the chunk of the draw, whose
//          tokens are read once more.
// Values from -2^8 down are left out of a row where all of them together would weigh less
// than the rounding of u times the total does (the total is 1 at least: 66 t below the
// maximum for u from 2^-24 on; at u = 0 only those whose power is 0 in 64 bits).  A row
// that holds other values outside the counted range takes the draw kernel's second path,
// which finds the same boundary by bisection over the 2^16 values, a pass over the row each
// (48 such rows of 152,064: up to 1.1 ms).
//
// Bound: latency.  48 rows x 152,064 (us): count 6.6 to 7.9, of which the LDS atomics take
// 3.5 (16 cycles a wave's, at any spread of values); draw 15.8, a chain on one CU per
// row: 3 until the row's counts are there, 2 for the powers and sums, 1.4 for the
// boundary, 1 for the chunks' masses, 2 for 32,768 tokens' weights out of LDS, 1.5 to the
// token.  One row of 32,768: 3.8 and 10.  The bins of two tokens come from 16-bit
// instructions on both: with a 32-bit one for each, 9.1 + 21.1.
// (In the first form every thread had a contiguous run of bins, sums went through LDS
// shuffles and all waves searched alike: 13 + 45, one row 11 + 23.)
#include <math.h>

#include "mi_common.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kMaxVocab = 1 << 20, kMaxRows = 65535;
constexpr int kMaxChunks = 32;
constexpr int kLoField = 127 - 30, kHiField = 127 + 8;  // exponent fields [2^-30, 2^8)
constexpr int kSide = (kHiField - kLoField) * 128;      // values of one sign
constexpr int kZeroBin = kSide;
constexpr int kPairs = 5;  // pairs of bins per thread of the draw kernel
constexpr int kBins = kThreads * kPairs * 2;  // in descending order of value; the last few unused
constexpr int kGroups = kBins / 128;          // a wave's share of one pair per thread
constexpr int kSpareBin = kBins - 64;
static_assert(2 * kSide + 1 <= kSpareBin && kSpareBin % 2 == 0, "bins");
// What a chunk holds outside the bins: this and up for tiny or high values, else the key
// of its largest finite value from -2^8 down, or 0.
constexpr uint32_t kTinyOrHigh = 0x10000;
// Order-preserving keys: 0x8000 + the magnitude's bits with the sign; NaN 0 (never
// drawn) or, in greedy rows, 0xffff (above +inf).
constexpr uint32_t kMinusInf = 0x8000 - 0x7f80;

__device__ __forceinline__ uint32_t key_of(uint32_t b, uint32_t nan) {
  const uint32_t mag = b & 0x7fffu;
  return mag > 0x7f80u ? nan : (b & 0x8000u) ? 0x8000u - mag : 0x8000u + mag;
}
__device__ __forceinline__ double value_of_key(uint32_t k) {
  const uint32_t b = k >= 0x8000u ? k - 0x8000u : 0x8000u | (0x8000u - k);
  return double(__uint_as_float(b << 16));
}
// A value's bin; as an unsigned number over all of them for values outside.
__device__ __forceinline__ int bin_of(uint32_t b) {
  const int mag = int(b & 0x7fffu);
  const int off = mag ? mag - (kLoField * 128 - 1) : 0;  // 1 .. kSide
  if (unsigned(off) > unsigned(kSide) || (off == 0 && mag)) return -1;
  return (b & 0x8000u) ? kZeroBin + off : kZeroBin - off;
}
__device__ __forceinline__ uint32_t key_of_bin(int bin) {
  if (bin == kZeroBin) return 0x8000u;
  const int mag = (bin < kZeroBin ? kZeroBin - bin : bin - kZeroBin) + kLoField * 128 - 1;
  return uint32_t(bin < kZeroBin ? 0x8000 + mag : 0x8000 - mag);
}

struct DrawParams {
  const uint16_t* logits;
  int64_t stride;
  int batch, vocab, chunks;
  const float* temperature;
  const int32_t* top_k;  // null: off
  const float* top_p;    // null: off
  const float* min_p;    // null: off
  const float* u;
  int64_t* out;
  uint32_t* counts;            // [row][chunk][kBins / 2] pairs of 16 bits
  unsigned long long* winner;  // [row][chunk] key << 32 | ~index of the largest
  uint32_t* outside;           // [row][chunk]
};

constexpr uint32_t kPad = 0x7fff7fffu;
// Eight tokens from `at` on, packed; past the end: NaN bits, which weigh nothing.
__device__ __forceinline__ uint4 load8(const uint16_t* row, int at, int vocab) {
  uint4 v;
  if (at + 8 <= vocab) {
    __builtin_memcpy(&v, row + at, 16);
    return v;
  }
  uint32_t x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    x[j] = (at + 2 * j < vocab ? row[at + 2 * j] : 0x7fffu) | (at + 2 * j + 1 < vocab ? row[at + 2 * j + 1] : 0x7fffu) << 16;
  return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ uint32_t token(const uint4& v, int j) {
  const uint32_t x = j < 2 ? v.x : j < 4 ? v.y : j < 6 ? v.z : v.w;
  return j & 1 ? x >> 16 : x & 0xffffu;
}

// ---------------------------------------------------------------- wave sums
// Every step adds the same two values in both of the lanes that exchange them, so all
// lanes end with the same bits.
constexpr int kRowShr = 0x110, kRowBcast15 = 0x142, kRowBcast31 = 0x143;
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ int lanes(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double lanes(double v) {
  const long long b = __double_as_longlong(v);
  return __longlong_as_double((long long)(uint32_t(lanes<CTRL, ROWS>(int(b)))) |
                              (long long)(lanes<CTRL, ROWS>(int(b >> 32))) << 32);
}
__device__ __forceinline__ int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ double lane_value(double v, int lane) {
  const long long b = __double_as_longlong(v);
  return __longlong_as_double((long long)(uint32_t(lane_value(int(b), lane))) |
                              (long long)(lane_value(int(b >> 32), lane)) << 32);
}
template <typename T>
__device__ __forceinline__ T last_lane(T v) { return lane_value(v, 63); }
// Inclusive prefix sum over the lanes; the last lane's is the wave's sum.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
  v += lanes<kRowShr + 1>(v);
  v += lanes<kRowShr + 2>(v);
  v += lanes<kRowShr + 4>(v);
  v += lanes<kRowShr + 8>(v);
  v += lanes<kRowBcast15, 0xa>(v);
  v += lanes<kRowBcast31, 0xc>(v);
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) { return last_lane(wave_scan(v)); }

// Four sums at once: lane l gets that of value l % 4.
constexpr int kRowRor = 0x120;
__device__ __forceinline__ double wave_sum4(double a, double b, double c, double d) {
  const bool one = threadIdx.x & 1, two = threadIdx.x & 2;
  const double ab = (one ? b : a) + lanes<mi::kDppQuadSwap1>(one ? a : b);
  const double cd = (one ? d : c) + lanes<mi::kDppQuadSwap1>(one ? c : d);
  double v = (two ? cd : ab) + lanes<mi::kDppQuadSwap2>(two ? ab : cd);
  v += lanes<kRowRor + 4>(v);
  v += lanes<kRowRor + 8>(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, uint32_t(__shfl_xor(int(v), o)));
  return v;
}
// Sum over the workgroup in wave order; every thread gets it.
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  T sum = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += red[w];
  return sum;
}

typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
typedef __attribute__((ext_vector_type(2))) short s16x2_t;
// The bins of a pair of tokens, by 16-bit instructions on both at once.  As signed
// numbers in descending order of value over all values, NaN apart and those of a
// magnitude in (0, 2^-30), which come out as zero's; from 2^8 on negative.
__device__ __forceinline__ s16x2_t bin_pair(uint32_t x) {
  const u16x2_t off = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2_t, x & 0x7fff7fffu),
                                                    u16x2_t(kLoField * 128 - 1));
  const s16x2_t flip = __builtin_bit_cast(s16x2_t, ~x) >> 15;
  return (__builtin_bit_cast(s16x2_t, off) ^ flip) - flip + short(kZeroBin);
}

// What a chunk's tokens come to, beside their counts.
struct Seen {
  uint32_t best[kWaves];
  uint32_t outside;
  int first;  // 0x10000 - the first place of the largest
};

// A thread's G groups of eight tokens, wave by wave: a wave has 512 G in a row, group i of
// a lane the eight from 512 i + 8 lane on.  Past the row's end: NaN bits.
template <int G>
__device__ __forceinline__ int place_of(int i) {
  return int(threadIdx.x >> 6) * 512 * G + i * 512 + int(threadIdx.x & 63) * 8;
}
template <int G>
__device__ __forceinline__ void load_tokens(uint32_t (&v)[4 * G], const uint16_t* logits, int base, int vocab) {
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int at = base + place_of<G>(i);
    const uint4 x = at < vocab ? load8(logits, at, vocab) : make_uint4(kPad, kPad, kPad, kPad);
    v[4 * i] = x.x, v[4 * i + 1] = x.y, v[4 * i + 2] = x.z, v[4 * i + 3] = x.w;
  }
}

// The counts of a workgroup's tokens (none of a greedy row's) into `hist`, and the key of
// the largest with NaN 0 (highest where the row is greedy); the workgroup's sums are
// complete behind the last barrier.
template <int G>
__device__ __forceinline__ uint32_t count_tokens(const uint32_t (&v)[4 * G], int base, int vocab, bool greedy, uint32_t* hist,
                                                 Seen& seen) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < kBins / kThreads; ++i) hist[i * kThreads + tid] = 0;
  if (tid == 0) seen.outside = 0, seen.first = 0;
  __syncthreads();
  auto place = [&](int i, int h) { return place_of<G>(i >> 2) + (i & 3) * 2 + h; };
  // Without a branch per token (with one it took twice as long): a value outside the
  // bins counts in one behind them, most often its lane's own, since all of a wave's on
  // one, as masked tokens are, would queue.
  const u16x2_t spare = u16x2_t((unsigned short)(kSpareBin + (tid & 63)));
  u16x2_t mags = {0, 0}, least = {0xffff, 0xffff};  // magnitudes: the largest, and the least less one, zeros apart
  s16x2_t bins = {0x7fff, 0x7fff};
#pragma unroll
  for (int g = 0; g < G; ++g) {
    if (base + place_of<G>(g) >= vocab) break;
#pragma unroll
    for (int i = 4 * g; i < 4 * g + 4; ++i) {
      const u16x2_t mag = __builtin_bit_cast(u16x2_t, v[i] & 0x7fff7fffu);
      const s16x2_t pair = bin_pair(v[i]);
      mags = __builtin_elementwise_max(mags, mag);
      least = __builtin_elementwise_min(least, mag - (unsigned short)1);
      bins = __builtin_elementwise_min(bins, pair);
      if (greedy) continue;
      const u16x2_t bin = __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, pair), spare);
      atomicAdd(&hist[bin.x], 1u);
      atomicAdd(&hist[bin.y], 1u);
    }
  }
  const uint32_t most = max(uint32_t(mags.x), uint32_t(mags.y));
  const bool tiny = min(uint32_t(least.x), uint32_t(least.y)) < kLoField * 128 - 1;
  // NaN, or values whose bins do not say their order
  const bool by_key = most > 0x7f80u || tiny, other = most >= kHiField * 128u || tiny;
  const int top_bin = min(int(bins.x), int(bins.y));
  uint32_t top = top_bin == 0x7fff ? 0u : key_of_bin(top_bin);
  const uint32_t nan = greedy ? 0xffffu : 0u;
  auto key_at = [&](int i, int h) -> uint32_t {
    return base + place(i, h) < vocab ? key_of(h ? v[i] >> 16 : v[i] & 0xffffu, nan) : 0u;
  };
  if (by_key) {
    top = 0;
#pragma unroll
    for (int i = 0; i < 4 * G; ++i) top = max(top, max(key_at(i, 0), key_at(i, 1)));
  }
  const uint32_t mine = top;
  top = wave_max(top);
  if ((tid & 63) == 0) seen.best[tid >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) top = max(top, seen.best[w]);
  if (mine == top) {
    int at = 0;
    if (by_key) {
#pragma unroll
      for (int i = 4 * G - 1; i >= 0; --i)
#pragma unroll
        for (int h = 1; h >= 0; --h)
          if (key_at(i, h) == top && base + place(i, h) < vocab) at = 0x10000 - place(i, h);
    } else {
#pragma unroll
      for (int i = 4 * G - 1; i >= 0; --i) {
        const s16x2_t pair = bin_pair(v[i]);
        if (pair.y == top_bin) at = 0x10000 - place(i, 1);
        if (pair.x == top_bin) at = 0x10000 - place(i, 0);
      }
    }
    if (at) atomicMax(&seen.first, at);
  }
  if (other) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4 * G; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t b = h ? v[i] >> 16 : v[i] & 0xffffu, key = key_of(b, 0);
        if (key > kMinusInf && bin_of(b) < 0)
          out = max(out, key < 0x8000u && (b & 0x7fffu) >= kHiField * 128u ? key : kTinyOrHigh);
      }
    if (out) atomicMax(&seen.outside, out);
  }
  __syncthreads();
  return top;
}
// (what lies in `hist` behind the last bin is nobody's)
__device__ __forceinline__ uint2 pair_of(const uint32_t* hist, int d) {
  uint2 c = *reinterpret_cast<const uint2*>(&hist[2 * d]);
  if (2 * d >= 2 * kSide) c = make_uint2(2 * d == 2 * kSide ? c.x : 0u, 0u);
  return c;
}
__device__ __forceinline__ unsigned long long winner_of(uint32_t top, int base, const Seen& seen) {
  return (unsigned long long)top << 32 | (0xffffffffu - uint32_t(base + 0x10000 - seen.first));
}

// G groups of eight tokens per thread, 8,192 G tokens per workgroup.
template <int G>
__global__ __launch_bounds__(kThreads) void count_kernel(DrawParams p) {
  __shared__ __attribute__((aligned(16))) uint32_t hist[kBins];
  __shared__ Seen seen;
  const int tid = threadIdx.x, chunk = blockIdx.x >> 3;
  const int64_t row = blockIdx.y * 8 + (blockIdx.x & 7);
  if (row >= p.batch) return;
  const int base = chunk * kThreads * 8 * G;
  uint32_t v[4 * G];
  load_tokens<G>(v, p.logits + row * p.stride, base, p.vocab);
  const bool greedy = !(p.temperature[row] > 0.f);
  const uint32_t top = count_tokens<G>(v, base, p.vocab, greedy, hist, seen);
  const int64_t slot = row * p.chunks + chunk;
  if (tid == 0) {
    p.winner[slot] = winner_of(top, base, seen);
    p.outside[slot] = seen.outside;
  }
  if (greedy) return;
  uint32_t* counts = p.counts + slot * (kBins / 2);
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const uint2 c = pair_of(hist, i * kThreads + tid);
    counts[i * kThreads + tid] = c.x | c.y << 16;
  }
}

// 2^y for y <= 0 (y below -1,100 counts as that: 0) to some 2^-52 relative: the whole
// part by the exponent, 2^f for |f| <= 1/2 by the exponential series in f ln 2, whose
// first term left out is 2e-16 at most.
struct Series {
  double c[13];
  constexpr Series() : c() {
    double term = 1.0;
    for (int k = 0; k < 13; ++k) {
      c[k] = term;
      term *= 0.693147180559945309417232121458 / (k + 1);
    }
  }
};
__device__ constexpr Series kSeries;
__device__ __forceinline__ double exp2_f64(double y) {
  y = fmax(y, -1100.0);
  const double n = rint(y), f = y - n;
  double v = kSeries.c[12];
#pragma unroll
  for (int k = 11; k >= 0; --k) v = fma(v, f, kSeries.c[k]);
  return ldexp(v, int(n));
}

// A whole number below 2^32 in 64 bits (the conversion takes four times an addition).
__device__ __forceinline__ double whole(uint32_t n) {
  return __longlong_as_double(0x4330000000000000ll | n) - 0x1p52;
}

// How many of `most` tokens of weight w, the first of them behind the mass `before`,
// lie in the prefix that reaches `target`.
__device__ __forceinline__ int reach(double before, double w, double target, int most) {
  if (!(before < target)) return 0;
  const double m = ceil((target - before) / w);
  return m < double(most) ? max(int(m), 1) : most;  // (w = 0 gives infinity: all)
}

struct Place {
  int bin, kept;  // the last bin, and how many of its tokens
  int count_before;  // tokens, and
  double before;     // mass, of the bins ahead of it
};

struct Shared {
  Seen seen;
  Place last;
  double total;
  double weight[kBins];
  uint32_t count[kBins];  // of tokens that min_p keeps
  double group_mass[kGroups];
  int group_count[kGroups];
  double mass[kMaxChunks][kWaves];
  double chunk_mass[kMaxChunks];
  int chunk_ties[kMaxChunks];
  double redd[kWaves];
  int redi[kWaves];
};

// The first bin at which `reached` holds of the (count, mass) of all bins up to and
// with it -- else the last of the `bins_end` bins that holds a token -- by groups and
// then by pairs, in every wave alike.
template <typename F>
__device__ __forceinline__ Place find_bin(const Shared& s, int bins_end, F reached) {
  const int lane = threadIdx.x & 63;
  int group = 0, count_before = 0, count_ahead = 0;  // ahead: of the group
  double mass_before = 0.0, mass_ahead = 0.0;
#pragma unroll
  for (int part = 0; part < (kGroups + 63) / 64; ++part) {
    const int g = part * 64 + lane;
    const bool in = g < kGroups && 128 * g < bins_end;
    const int c = in ? s.group_count[g] : 0;
    const int ci = count_before + wave_scan(c);
    const double mi = mass_before + wave_scan(in ? s.group_mass[g] : 0.0);
    const unsigned long long hit = __ballot(c && reached(ci, mi)), any = __ballot(c != 0);
    if (any) {
      const int at = hit ? __builtin_ctzll(hit) : 63 - __builtin_clzll(any);
      group = part * 64 + at;
      count_ahead = at ? __builtin_amdgcn_readlane(ci, at - 1) : count_before;
      mass_ahead = at ? lane_value(mi, at - 1) : mass_before;
    }
    if (hit) break;
    count_before = last_lane(ci);
    mass_before = last_lane(mi);
  }
  const int bin = 128 * group + 2 * lane;
  const int c0 = bin < bins_end ? int(s.count[bin]) : 0, c1 = bin + 1 < bins_end ? int(s.count[bin + 1]) : 0;
  const double m0 = c0 * s.weight[bin], m1 = c1 * s.weight[bin + 1];
  const int ci = count_ahead + wave_scan(c0 + c1);
  const double mi = mass_ahead + wave_scan(m0 + m1);
  const bool hit0 = c0 && reached(ci - c1, mi - m1), hit1 = c1 && reached(ci, mi);
  const unsigned long long hit = __ballot(hit0 || hit1), any = __ballot(c0 || c1);
  const int at = hit ? __builtin_ctzll(hit) : any ? 63 - __builtin_clzll(any) : 0;
  const bool second = hit ? !hit0 : c1 != 0;
  Place r;
  r.bin = __builtin_amdgcn_readlane(bin + (second ? 1 : 0), at);
  r.kept = __builtin_amdgcn_readlane(second ? c1 : c0, at);
  r.count_before = __builtin_amdgcn_readlane(second ? ci - c1 : ci - c1 - c0, at);
  r.before = lane_value(second ? mi - m1 : mi - m1 - m0, at);
  return r;
}

// A row's maximum and parameters.
struct Row {
  const uint16_t* logits;
  int vocab, top_k;
  uint32_t kmax;
  double lmax, per_t, top_p, min_p, u;  // per_t: log2 e / temperature
  __device__ __forceinline__ double weigh(uint32_t key) const {
    if (key == kmax) return 1.0;
    if (key <= kMinusInf || lmax == INFINITY) return 0.0;
    return exp2_f64((value_of_key(key) - lmax) * per_t);
  }
};

// (count, mass) of the row's tokens with key >= k, in a fixed order.
__device__ __noinline__ void tokens_from(const Row& r, Shared& s, uint32_t k, int* n, double* m) {
  int c = 0;
  double sum = 0.0;
#pragma unroll 1
  for (int at = threadIdx.x; at < r.vocab; at += kThreads) {
    const uint32_t key = key_of(r.logits[at], 0);
    if (key >= k) ++c, sum += r.weigh(key);
  }
  *n = block_sum(c, s.redi);
  *m = block_sum(sum, s.redd);
}

// The draw of a row with values outside the bins: the boundary by bisection over the
// keys, then the token by a pass over the row, kThreads tokens at a time.
__device__ __noinline__ int draw_outside(const Row& r, Shared& s) {
  // the least key above minus infinity that min_p keeps
  uint32_t lo = kMinusInf, hi = r.kmax;  // lo fails, hi holds
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (r.weigh(mid) >= r.min_p) hi = mid;
    else lo = mid;
  }
  uint32_t least = hi;
  int n;
  double m;
  tokens_from(r, s, least, &n, &m);
  int most = 0x7fffffff;  // tokens with key `least` that are kept
  if (n > r.top_k) {      // the largest key from which on there are top_k
    lo = least, hi = r.kmax + 1;  // lo has them, hi has not
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      tokens_from(r, s, mid, &n, &m);
      if (n >= r.top_k) lo = mid;
      else hi = mid;
    }
    least = lo;
    tokens_from(r, s, least + 1, &n, &m);
    most = r.top_k - n;
    m += most * r.weigh(least);
  }
  if (r.top_p < 1.0) {
    const double target = r.top_p * m;
    lo = least, hi = r.kmax + 1;  // lo reaches the target, hi does not
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      tokens_from(r, s, mid, &n, &m);
      if (m >= target) lo = mid;
      else hi = mid;
    }
    int above;
    double before;
    tokens_from(r, s, lo + 1, &above, &before);
    tokens_from(r, s, lo, &n, &m);
    most = min(lo == least ? most : 0x7fffffff, n - above);
    most = max(reach(before, r.weigh(lo), target, most), lo == r.kmax ? 1 : 0);
    least = lo;
  }
  int above;
  double total;
  tokens_from(r, s, least + 1, &above, &total);
  tokens_from(r, s, least, &n, &m);
  int room = min(most, n - above);
  total += room * r.weigh(least);
  const double target = r.u * total;
  // the first token that takes the sum over the target, or the last with a weight
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  double sum = 0.0;
  int drawn = 0;
#pragma unroll 1
  for (int base = 0; base < r.vocab; base += kThreads) {
    const int at = base + tid;
    const uint32_t key = at < r.vocab ? key_of(r.logits[at], 0) : 0u;
    const int rank = wave_scan(int(key == least));
    __syncthreads();
    if (lane == 63) s.redi[wave] = rank;
    __syncthreads();
    int ahead = 0, ties = 0;
#pragma unroll 1
    for (int w = 0; w < kWaves; ++w) {
      ahead += w < wave ? s.redi[w] : 0;
      ties += s.redi[w];
    }
    const double w0 = key > least || (key == least && ahead + rank <= room) ? r.weigh(key) : 0.0;
    const double run = wave_scan(w0);
    const unsigned long long any = __ballot(w0 > 0.0);
    if (lane == 63) s.redd[wave] = run;
    __syncthreads();
    double before = sum;
#pragma unroll 1
    for (int w = 0; w < wave; ++w) before += s.redd[w];
    const unsigned long long over = __ballot(w0 > 0.0 && before + run > target);
    if (lane == 0) s.redi[wave] = over ? __builtin_ctzll(over) : any ? 64 + 63 - __builtin_clzll(any) : -1;
    __syncthreads();
    bool found = false;
#pragma unroll 1
    for (int w = 0; w < kWaves && !found; ++w) {
      const int in = s.redi[w];
      if (in >= 0) drawn = base + 64 * w + (in & 63);
      found = in >= 0 && in < 64;
      sum += s.redd[w];
    }
    if (found) break;
    room -= min(ties, room);
  }
  return drawn;
}

// ONE: the row is one chunk, whose tokens are counted here.
template <int G, bool ONE>
__global__ __launch_bounds__(kThreads) void draw_kernel(DrawParams p) {
  constexpr int kChunk = kThreads * 8 * G;
  __shared__ __attribute__((aligned(16))) Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const uint32_t* row_counts = p.counts + row * p.chunks * (kBins / 2) + tid;

  // (all of the row's parameters and counts are asked for before any is used)
  const float tf = p.temperature[row], uf = p.u[row];
  const int kf = p.top_k ? p.top_k[row] : 0;
  const float pf = p.top_p ? p.top_p[row] : 1.f, mf = p.min_p ? p.min_p[row] : 0.f;
  unsigned long long top = 0;
  uint32_t outside = 0;
  uint32_t tokens[4 * G];
  if constexpr (ONE) {
    load_tokens<G>(tokens, p.logits + row * p.stride, 0, p.vocab);
    const uint32_t key = count_tokens<G>(tokens, 0, p.vocab, !(tf > 0.f), s.count, s.seen);
    top = winner_of(key, 0, s.seen);
    outside = s.seen.outside;
  } else if (lane < p.chunks) {
    top = p.winner[row * p.chunks + lane];
    outside = p.outside[row * p.chunks + lane];
  }
  constexpr int kTogether = 5;  // chunks whose counts are loaded at once
  uint32_t counts[kTogether][kPairs];
  auto load_counts = [&](int c0) {
#pragma unroll
    for (int q = 0; q < kTogether; ++q)
#pragma unroll
      for (int j = 0; j < kPairs; ++j)
        counts[q][j] = c0 + q < p.chunks ? row_counts[(c0 + q) * (kBins / 2) + j * kThreads] : 0u;
  };
  if constexpr (!ONE) {
    load_counts(0);
    for (int o = 1; o < p.chunks; o <<= 1) {
      top = max(top, (unsigned long long)__shfl_xor((long long)top, o));
      outside = max(outside, uint32_t(__shfl_xor(int(outside), o)));
    }
  }
  top = (unsigned long long)__builtin_amdgcn_readfirstlane(int(top >> 32)) << 32 |
        uint32_t(__builtin_amdgcn_readfirstlane(int(top)));
  outside = uint32_t(__builtin_amdgcn_readfirstlane(int(outside)));
  const bool greedy = !(tf > 0.f);
  Row r;
  r.kmax = uint32_t(top >> 32);
  if (greedy || r.kmax <= kMinusInf) {  // nothing has a weight: the row's argmax
    if (tid == 0) p.out[row] = int64_t(0xffffffffu - uint32_t(top));
    return;
  }
  r.logits = p.logits + row * p.stride;
  r.vocab = p.vocab;
  r.per_t = 1.4426950408889634073599 / double(tf);
  r.lmax = value_of_key(r.kmax);
  r.top_k = kf > 0 ? kf : 0x7fffffff;
  r.top_p = pf < 1.f ? double(pf) : 2.0;
  r.min_p = mf > 0.f ? fmin(double(mf), 1.0) : 0.0;
  r.u = fmax(double(uf), 0.0);
  // (the largest of the low values stands for all; -1,100: from there on a power is 0)
  if (outside >= kTinyOrHigh || (outside && (value_of_key(outside) - r.lmax) * r.per_t > -1100.0 &&
                                 r.weigh(outside) * r.vocab > r.u * 0x1p-53)) {
    const Row copy = r;  // (r itself stays in registers)
    const int drawn = draw_outside(copy, s);
    if (tid == 0) p.out[row] = drawn;
    return;
  }

  // pair d = 1,024 j + tid: this thread's bins 2 d and 2 d + 1, group 16 j + wave
  if constexpr (ONE) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int d = j * kThreads + tid;
      if (d >= kSide) *reinterpret_cast<uint2*>(&s.count[2 * d]) = pair_of(s.count, d);
    }
  } else {
    uint2 cnt[kPairs] = {};
    for (int c0 = 0; c0 < p.chunks; c0 += kTogether) {
      if (c0) load_counts(c0);
#pragma unroll
      for (int q = 0; q < kTogether; ++q)
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          cnt[j].x += counts[q][j] & 0xffffu;
          cnt[j].y += counts[q][j] >> 16;
        }
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) *reinterpret_cast<uint2*>(&s.count[2 * (j * kThreads + tid)]) = cnt[j];
  }
#pragma unroll 1
  for (int j = 0; j < kPairs; ++j) {
    const int bin = 2 * (j * kThreads + tid);
    uint2 c = *reinterpret_cast<const uint2*>(&s.count[bin]);
    double w0 = 0.0, w1 = 0.0, m = 0.0;
    int n = 0;
    if (__ballot(c.x + c.y != 0)) {
      // (a bin above the maximum is empty and its power may be infinite)
      w0 = c.x ? r.weigh(key_of_bin(bin)) : 0.0;
      w1 = c.y ? r.weigh(key_of_bin(bin + 1)) : 0.0;
      if (w0 < r.min_p) c.x = 0, w0 = 0.0;
      if (w1 < r.min_p) c.y = 0, w1 = 0.0;
      *reinterpret_cast<uint2*>(&s.count[bin]) = c;
      n = wave_sum(int(c.x + c.y));
      m = wave_sum(whole(c.x) * w0 + whole(c.y) * w1);
    }
    *reinterpret_cast<double2*>(&s.weight[bin]) = make_double2(w0, w1);
    if (lane == 0) s.group_count[j * kWaves + wave] = n, s.group_mass[j * kWaves + wave] = m;
  }
  __syncthreads();
  if (wave == 0) {  // (in every wave alike it took three times as long)
    int tokens = 0;
    double all = 0.0;
#pragma unroll
    for (int part = 0; part < (kGroups + 63) / 64; ++part) {
      const int g = part * 64 + lane;
      tokens += wave_sum(g < kGroups ? s.group_count[g] : 0);
      all += wave_sum(g < kGroups ? s.group_mass[g] : 0.0);
    }
    Place at = {kBins - 1, 0, 0, 0.0};  // (an unused bin: all that min_p keeps)
    if (tokens > r.top_k) {
      at = find_bin(s, kBins, [&](int n, double) { return n >= r.top_k; });
      at.kept = min(at.kept, r.top_k - at.count_before);
      all = at.before + at.kept * s.weight[at.bin];
    }
    if (r.top_p < 1.0) {
      const double target = r.top_p * all;
      const Place cut = find_bin(s, at.bin + 1, [&](int, double m) { return m >= target; });
      // (the most likely token is kept whatever top_p is)
      const int most = cut.bin == at.bin ? at.kept : cut.kept;
      at.kept = max(reach(cut.before, s.weight[cut.bin], target, most), key_of_bin(cut.bin) == r.kmax ? 1 : 0);
      at.bin = cut.bin;
      all = cut.before + at.kept * s.weight[at.bin];
    }
    if (lane == 0) {
      s.last = at, s.total = all;
      s.weight[min(at.bin, 2 * kSide) + 1] = 0.0;  // the weight of all tokens that are not kept
    }
  }
  __syncthreads();
  // kept: the bins before last_bin and the first `ties` tokens of it
  const int last_bin = s.last.bin, ties = s.last.kept;
  const double target = r.u * s.total, w_last = s.weight[last_bin];
  int chunk = 0, room = ties;
  double cum = 0.0, sum = 0.0;
  bool some = ONE && int(s.count[last_bin]) > ties;  // not all of the chunk's tokens with the last value are kept
  if constexpr (!ONE) {
    // each chunk's mass above the last kept value, and its tokens with it
    for (int c0 = 0; c0 < p.chunks; c0 += kTogether) {
      if (c0 || p.chunks > kTogether) load_counts(c0);
      double m[kTogether] = {};
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int bin = 2 * (j * kThreads + tid), group = j * kWaves + wave;
        if (j * kThreads + tid == last_bin / 2) {
#pragma unroll
          for (int q = 0; q < kTogether; ++q)
            if (c0 + q < p.chunks) s.chunk_ties[c0 + q] = int(counts[q][j] >> (16 * (last_bin & 1)) & 0xffffu);
        }
        if (128 * group > last_bin || s.group_count[group] == 0) continue;
        double2 w = *reinterpret_cast<const double2*>(&s.weight[bin]);
        if (bin >= last_bin) w.x = 0.0;
        if (bin + 1 >= last_bin) w.y = 0.0;
#pragma unroll
        for (int q = 0; q < kTogether; ++q)
          m[q] += whole(counts[q][j] & 0xffffu) * w.x + whole(counts[q][j] >> 16) * w.y;
      }
      const double four = wave_sum4(m[0], m[1], m[2], m[3]);
      if (lane < 4 && c0 + lane < p.chunks) s.mass[c0 + lane][wave] = four;
      if (c0 + 4 < p.chunks) {
        m[4] = wave_sum(m[4]);
        if (lane == 0) s.mass[c0 + 4][wave] = m[4];
      }
    }
    __syncthreads();
    if (tid < p.chunks) {
      double m = 0.0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m += s.mass[tid][w];
      s.chunk_mass[tid] = m;
    }
    __syncthreads();
    // The chunk of the draw: the first whose mass takes the sum over the target, or, with u
    // so near 1 that none does, the last that has any.
    int left = ties;
    for (int c = 0; c < p.chunks; ++c) {
      const int here = min(s.chunk_ties[c], left);
      const double m = s.chunk_mass[c] + here * w_last;
      if (m > 0.0) chunk = c, room = left, cum = sum;
      if (sum + m > target) break;
      sum += m;
      left -= here;
    }
    some = s.chunk_ties[chunk] > room;
  }

  // Its tokens, once more where another workgroup counted them.
  if constexpr (!ONE) load_tokens<G>(tokens, r.logits, chunk * kChunk, p.vocab);
  const int first = chunk * kChunk + place_of<G>(0);
  const u16x2_t past = u16x2_t((unsigned short)(min(last_bin, 2 * kSide) + 1));
  u16x2_t bins[G][4];  // `past` for those that are not kept
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      bins[i][j] = __builtin_elementwise_min(__builtin_bit_cast(u16x2_t, bin_pair(tokens[4 * i + j])), past);
  if (some) {
    int n = 0, inc[G];
    uint32_t same[G];  // of a group's eight, a bit each
#pragma unroll
    for (int i = 0; i < G; ++i) {
      same[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) same[i] |= uint32_t(bins[i][j / 2][j & 1] == last_bin) << j;
      inc[i] = wave_scan(int(__popc(same[i])));
      const int all = last_lane(inc[i]);
      inc[i] += n;
      n += all;
    }
    __syncthreads();
    if (lane == 0) s.redi[wave] = n;
    __syncthreads();
    int ahead = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) ahead += w < wave ? s.redi[w] : 0;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      int rank = ahead + inc[i] - int(__popc(same[i]));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((same[i] >> j & 1) && rank++ >= room) bins[i][j / 2][j & 1] = past.x;
    }
  }
  // a token's kept weight
  auto held = [&](int i, int j) -> double { return s.weight[bins[i][j / 2][j & 1]]; };
  double group[G], mine = 0.0;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    group[i] = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) group[i] += held(i, j);
    mine += group[i];
  }
  mine = wave_sum(mine);
  __syncthreads();
  if (lane == 0) s.redd[wave] = mine;
  __syncthreads();
  // The wave, its group, the lane, the token, each found as the chunk was.
  int the_wave = 0;
  sum = cum;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const double m = s.redd[w];
    if (m > 0.0 && !(cum > target)) the_wave = w, sum = cum;
    cum += m;
  }
  if (wave != the_wave) return;
  int gi = 0;
  double ahead = sum, inc = 0.0;
  bool done = false;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const double run = wave_scan(group[i]);
    const double m = last_lane(run);
    if (!done && m > 0.0) gi = i, ahead = sum, inc = run;
    if (!done && sum + m > target) done = true;
    sum += m;
  }
  double g = group[0];
#pragma unroll
  for (int i = 1; i < G; ++i)
    if (gi == i) g = group[i];
  const unsigned long long over = __ballot(g > 0.0 && ahead + inc > target), any = __ballot(g > 0.0);
  const int the_lane = over ? __builtin_ctzll(over) : any ? 63 - __builtin_clzll(any) : 0;
  // (the lane's own sum less its own weights would lose what is small beside them)
  const double before = the_lane ? lane_value(inc, the_lane - 1) : 0.0;
  if (lane != the_lane) return;
  double at = ahead + before;
  int drawn = first + gi * 512;
  bool stop = false;
#pragma unroll
  for (int i = 0; i < G; ++i) {
    if (gi != i) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double m = held(i, j);
      if (!stop && m > 0.0) drawn = first + i * 512 + j;
      at += m;
      if (m > 0.0 && at > target) stop = true;
    }
  }
  p.out[row] = drawn;
}

// Tokens of a workgroup.  A short row is one chunk, counted and drawn in one launch (us, in
// a graph, against two launches: 1 x 5,000 9.2 and 12.1, 300 x 5,000 18 and 30, 1 x 16,384
// 10.3 and 12.9; 32 x 32,768 15.6 and 15.5, 256 rows of it 16.6 and 22.2, one 15.2 and 14.0).
// Else few enough that a small batch takes more CUs (and a thread looks up fewer weights
// at the end), as long as the counts of a row's chunks, 20 KB each, stay few.
int groups_for(int64_t batch, int64_t vocab) {
  if (vocab <= 16384) return vocab <= 8192 ? 1 : 2;  // one chunk
  if (vocab <= 32768 && batch >= 32) return 4;
  if (vocab <= 8 * 8192 && batch * ((vocab + 8191) / 8192) <= 256) return 1;
  if (vocab <= 32 * 16384 && batch * ((vocab + 16383) / 16384) <= 256) return 2;
  return 4;
}
int64_t chunks_of(int64_t vocab, int groups) { return (vocab + 8192 * groups - 1) / (8192 * groups); }
// The most (row, chunk) places that up to `batch` rows take.
int64_t places(int64_t batch, int64_t vocab) {
  const int64_t fine = batch * chunks_of(vocab, 1), coarse = batch * chunks_of(vocab, 4);
  return coarse > 256 ? coarse : fine < 256 ? fine : 256;
}
constexpr size_t kPlaceBytes = kBins / 2 * 4 + 8 + 4;

}  // namespace

extern "C" size_t mi_draw_workspace_size(int32_t batch_size, int32_t vocab_size) {
  if (batch_size <= 0 || batch_size > kMaxRows || vocab_size <= 0 || vocab_size > kMaxVocab) return 0;
  return size_t(places(batch_size, vocab_size)) * kPlaceBytes;
}

extern "C" int mi_draw(const void* logits, int64_t logits_row_stride, int32_t batch_size, int32_t vocab_size,
                       const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                       const float* uniforms, int64_t* out_tokens, void* workspace, size_t workspace_bytes,
                       mi_stream_t stream) {
  mi::clear_error();
  if (batch_size < 0 || batch_size > kMaxRows || vocab_size <= 0 || vocab_size > kMaxVocab)
    return mi::fail(MI_ERR_INVALID, "draw: %d rows (0..%d) of %d tokens (1..%d)", batch_size, kMaxRows, vocab_size,
                    kMaxVocab);
  if (batch_size == 0) return MI_OK;
  if (!logits || !temperature || !uniforms || !out_tokens)
    return mi::fail(MI_ERR_INVALID, "draw: null pointer argument");
  if (logits_row_stride < vocab_size && batch_size > 1)
    return mi::fail(MI_ERR_INVALID, "draw: row stride %lld for %d tokens", (long long)logits_row_stride, vocab_size);
  const size_t need = mi_draw_workspace_size(batch_size, vocab_size);
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need)
    return mi::fail(MI_ERR_WORKSPACE, "draw: workspace of %zu bytes, 16-byte aligned, is needed (got %zu)", need,
                    workspace_bytes);
  DrawParams p;
  p.logits = static_cast<const uint16_t*>(logits);
  p.stride = logits_row_stride;
  p.batch = batch_size;
  p.vocab = vocab_size;
  const int groups = groups_for(batch_size, vocab_size);
  p.chunks = int(chunks_of(vocab_size, groups));
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.u = uniforms;
  p.out = out_tokens;
  const size_t used = size_t(batch_size) * p.chunks;
  p.counts = static_cast<uint32_t*>(workspace);
  p.winner = reinterpret_cast<unsigned long long*>(p.counts + used * (kBins / 2));
  p.outside = reinterpret_cast<uint32_t*>(p.winner + used);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 chunks(8 * p.chunks, (batch_size + 7) / 8), rows(batch_size), threads(kThreads);
  auto run = [&]<int G>() {
    if (p.chunks == 1) {
      hipLaunchKernelGGL((draw_kernel<G, true>), rows, threads, 0, s, p);
      return;
    }
    hipLaunchKernelGGL(count_kernel<G>, chunks, threads, 0, s, p);
    hipLaunchKernelGGL((draw_kernel<G, false>), rows, threads, 0, s, p);
  };
  if (groups == 1) run.template operator()<1>();
  else if (groups == 2) run.template operator()<2>();
  else run.template operator()<4>();
  return mi::check_launch("draw_kernel");
}

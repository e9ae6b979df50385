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
// and nothing depends on the order of additions.  Two launches, no atomics on memory
// and nothing kept between calls:
//   count  one workgroup per 32,768 tokens: largest value with its lowest index, and
//          the counts of the 2 x 38 x 128 values of magnitude [2^-30, 2^8) and of zero
//          in LDS, written as 16 bits each.
//   draw   one workgroup per row: the counts' sum over the chunks, ten values to a
//          thread; prefix sums of count and mass give the last kept value and how many
//          tokens of it; each chunk's kept mass gives the chunk of the draw, whose
//          tokens are read once more.
// Values below -2^8 weigh nothing beside a maximum that is 45 t above; a row that holds
// other values outside the counted range takes the draw kernel's second path, which
// finds the same boundary by bisection over the 2^16 values, a pass over the row each.
//
// Bound: 48 rows x 152,064: the count launch's LDS atomics and the draw launch's chain.
#include <math.h>

#include "mi_common.h"

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kChunk = 32768;                  // tokens of a workgroup of the count launch
constexpr int kPerThread = kChunk / kThreads;  // contiguous tokens of a thread
constexpr int kMaxVocab = 1 << 20, kMaxChunks = kMaxVocab / kChunk, kMaxRows = 65535;
constexpr int kLoField = 127 - 30, kHiField = 127 + 8;  // exponent fields [2^-30, 2^8)
constexpr int kSide = (kHiField - kLoField) * 128;      // values of one sign
constexpr int kZeroBin = kSide;
constexpr int kPerBinThread = 10;
constexpr int kBins = kThreads * kPerBinThread;  // bins in descending order of value; the last few unused
static_assert(2 * kSide + 1 <= kBins, "bins");
constexpr int kOut = -1;
// what a chunk holds outside the bins
constexpr uint32_t kTinyOrHigh = 1, kLow = 2;
constexpr uint32_t kMinusInf = 0x007F;  // its key

// Order-preserving key of a bf16 value, -0 as +0; a NaN gets `nan`.
__device__ __forceinline__ uint32_t key_of(uint32_t b, uint32_t nan) {
  if ((b & 0x7fffu) > 0x7f80u) return nan;
  if (b == 0x8000u) b = 0;
  return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
}
__device__ __forceinline__ double value_of_key(uint32_t k) {
  const uint32_t b = (k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu);
  return double(__uint_as_float(b << 16));
}
__device__ __forceinline__ int bin_of(uint32_t b) {
  const uint32_t mag = b & 0x7fffu;
  if (mag == 0) return kZeroBin;
  const int off = int(mag) - kLoField * 128;
  if (off < 0 || off >= kSide) return kOut;
  return (b & 0x8000u) ? kZeroBin + 1 + off : kZeroBin - 1 - off;
}
__device__ __forceinline__ uint32_t bits_of_bin(int bin) {
  if (bin == kZeroBin) return 0;
  return bin < kZeroBin ? uint32_t(kZeroBin - 1 - bin + kLoField * 128)
                        : 0x8000u | uint32_t(bin - kZeroBin - 1 + kLoField * 128);
}

struct DrawParams {
  const uint16_t* logits;
  int64_t stride;
  int vocab, chunks;
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

// Eight tokens from `at` on; past the end: NaN bits, which weigh nothing.
__device__ __forceinline__ void load8(const uint16_t* row, int at, int vocab, uint32_t (&b)[8]) {
  if (at + 8 <= vocab) {
    uint4 v;
    __builtin_memcpy(&v, row + at, 16);
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) b[2 * j] = x[j] & 0xffffu, b[2 * j + 1] = x[j] >> 16;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = at + j < vocab ? row[at + j] : 0x7fffu;
}

__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long v) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned long long)__shfl_xor((long long)v, o));
  return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

__global__ __launch_bounds__(kThreads) void count_kernel(DrawParams p) {
  __shared__ uint32_t hist[kBins];
  __shared__ unsigned long long best[kWaves];
  __shared__ uint32_t outside;
  const int tid = threadIdx.x, chunk = blockIdx.x;
  const int64_t row = blockIdx.y;
  const bool greedy = !(p.temperature[row] > 0.f);
  const uint16_t* logits = p.logits + row * p.stride;
  const int base = chunk * kChunk;
  if (!greedy)
    for (int i = tid; i < kBins; i += kThreads) hist[i] = 0;
  if (tid == 0) outside = 0;
  __syncthreads();
  unsigned long long top = 0;
  uint32_t seen = 0;
#pragma unroll
  for (int i = 0; i < kPerThread / 8; ++i) {
    const int at = base + (i * kThreads + tid) * 8;
    if (at >= p.vocab) break;
    uint32_t b[8];
    load8(logits, at, p.vocab, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (at + j >= p.vocab) break;
      // greedy: a NaN ranks highest, as in argmax; a draw never takes one
      const unsigned long long k = key_of(b[j], greedy ? 0x10000u : 0u);
      top = max(top, k << 32 | (0xffffffffu - uint32_t(at + j)));
      if (greedy || k == 0) continue;
      const int bin = bin_of(b[j]);
      if (bin >= 0) atomicAdd(&hist[bin], 1u);
      else if (k != kMinusInf) seen |= (b[j] & 0x8000u) && (b[j] & 0x7fffu) >= kHiField * 128u ? kLow : kTinyOrHigh;
    }
  }
  top = wave_max_u64(top);
  if ((tid & 63) == 0) best[tid >> 6] = top;
  if (seen) atomicOr(&outside, seen);
  __syncthreads();
  const int64_t slot = row * p.chunks + chunk;
  if (tid == 0) {
    for (int w = 1; w < kWaves; ++w) top = max(top, best[w]);
    p.winner[slot] = top;
    p.outside[slot] = outside;
  }
  if (greedy) return;
  uint32_t* counts = p.counts + slot * (kBins / 2);
  for (int i = tid; i < kBins / 2; i += kThreads) counts[i] = hist[2 * i] | hist[2 * i + 1] << 16;
}

// Block-wide sums in a fixed order.  `red` holds one value per wave; every thread
// gets the result.
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  T sum = red[0];
  for (int w = 1; w < kWaves; ++w) sum += red[w];
  return sum;
}
// Exclusive prefix sum over the threads.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T inc = v;
  for (int o = 1; o < 64; o <<= 1) {
    const T up = __shfl_up(inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  T before = 0;
  for (int w = 0; w < wave; ++w) before += red[w];
  T left = __shfl_up(inc, 1);
  return before + (lane ? left : T(0));
}

// How many of `most` tokens of weight w, the first of them behind the mass `before`,
// lie in the prefix that reaches `target`.
__device__ __forceinline__ int reach(double before, double w, double target, int most) {
  if (!(before < target)) return 0;
  const double m = ceil((target - before) / w);
  return m < double(most) ? max(int(m), 1) : most;  // (w = 0 gives infinity: all)
}

__global__ __launch_bounds__(kThreads) void draw_kernel(DrawParams p) {
  __shared__ double weight[kBins];
  __shared__ double mass[kMaxChunks][kWaves];
  __shared__ double redd[kWaves];
  __shared__ int redi[kWaves];
  __shared__ unsigned long long last;  // last kept bin << 32 | how many of its tokens
  __shared__ int drawn, final_kept;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const uint16_t* logits = p.logits + row * p.stride;
  const float tf = p.temperature[row];
  const bool greedy = !(tf > 0.f);

  unsigned long long top = 0;
  uint32_t outside = 0;
  for (int c = 0; c < p.chunks; ++c) {
    top = max(top, p.winner[row * p.chunks + c]);
    outside |= p.outside[row * p.chunks + c];
  }
  const uint32_t kmax = uint32_t(top >> 32);
  if (greedy || kmax <= kMinusInf) {  // nothing has a weight: the row's argmax
    if (tid == 0) p.out[row] = int64_t(0xffffffffu - uint32_t(top));
    return;
  }
  const double t = double(tf), lmax = value_of_key(kmax);
  auto weigh = [&](uint32_t key) -> double {
    if (key == kmax) return 1.0;
    if (key <= kMinusInf || lmax == INFINITY) return 0.0;
    return exp((value_of_key(key) - lmax) / t);
  };
  const int top_k = p.top_k && p.top_k[row] > 0 ? p.top_k[row] : 0x7fffffff;
  const double top_p = p.top_p && p.top_p[row] < 1.f ? double(p.top_p[row]) : 2.0;
  const double min_p = p.min_p && p.min_p[row] > 0.f ? fmin(double(p.min_p[row]), 1.0) : 0.0;
  const double u = double(p.u[row]);
  const bool low_matters = (outside & kLow) && (-256.0 - lmax) / t > -45.0;
  const bool fast = !(outside & kTinyOrHigh) && !low_matters;
  if (tid == 0) last = 0, drawn = 0x7fffffff, final_kept = -1;
  __syncthreads();

  uint32_t key_last;  // kept: keys above it and the first `ties` tokens with it
  int ties;
  double total;
  if (fast) {
    // this thread's bins, in descending order of value
    int cnt[kPerBinThread] = {};
    for (int c = 0; c < p.chunks; ++c) {
      const uint32_t* counts = p.counts + (row * p.chunks + c) * (kBins / 2) + tid * (kPerBinThread / 2);
#pragma unroll
      for (int j = 0; j < kPerBinThread / 2; ++j) {
        cnt[2 * j] += counts[j] & 0xffffu;
        cnt[2 * j + 1] += counts[j] >> 16;
      }
    }
    double w[kPerBinThread];
    int own = 0;
#pragma unroll
    for (int j = 0; j < kPerBinThread; ++j) {
      const int bin = tid * kPerBinThread + j;
      w[j] = cnt[j] ? weigh(key_of(bits_of_bin(bin), 0)) : 0.0;
      if (w[j] < min_p) cnt[j] = 0;
      weight[bin] = w[j];
      own += cnt[j];
    }
    int before = block_prefix(own, redi);
    double held = 0.0;
#pragma unroll
    for (int j = 0; j < kPerBinThread; ++j) {
      const int all = cnt[j];
      cnt[j] = min(all, max(top_k - before, 0));
      before += all;
      held += cnt[j] * w[j];
    }
    double mass_before = block_prefix(held, redd);
    const double target = top_p * block_sum(held, redd);
    held = 0.0;
    unsigned long long mine = 0;
#pragma unroll
    for (int j = 0; j < kPerBinThread; ++j) {
      const int bin = tid * kPerBinThread + j;
      if (cnt[j]) {
        // (the most likely token is kept whatever top_p is)
        const int kept = top_p > 1.0 ? cnt[j] : max(reach(mass_before, w[j], target, cnt[j]),
                                                    key_of(bits_of_bin(bin), 0) == kmax ? 1 : 0);
        mass_before += cnt[j] * w[j];
        held += kept * w[j];
        if (kept) mine = (unsigned long long)bin << 32 | uint32_t(kept);
      }
    }
    mine = wave_max_u64(mine);
    if (lane == 0 && mine) atomicMax(&last, mine);
    total = block_sum(held, redd);  // (its barriers publish `last` too)
    const int last_bin = int(last >> 32);
    ties = int(uint32_t(last));
    key_last = key_of(bits_of_bin(last_bin), 0);
    // each chunk's mass above the last kept value
    for (int c = 0; c < p.chunks; ++c) {
      const uint32_t* counts = p.counts + (row * p.chunks + c) * (kBins / 2) + tid * (kPerBinThread / 2);
      double s = 0.0;
      if (tid * kPerBinThread < last_bin) {
#pragma unroll
        for (int j = 0; j < kPerBinThread; ++j) {
          const uint32_t n = counts[j / 2] >> (16 * (j & 1)) & 0xffffu;
          if (tid * kPerBinThread + j < last_bin) s += n * w[j];
        }
      }
      s = wave_sum_f64(s);
      if (lane == 0) mass[c][wave] = s;
    }
  } else {
    // (count, mass) of the tokens with key >= k, in a fixed order
    auto tokens_from = [&](uint32_t k, int* n, double* m) {
      int c = 0;
      double s = 0.0;
      for (int at = tid * 8; at < p.vocab; at += kThreads * 8) {
        uint32_t b[8];
        load8(logits, at, p.vocab, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t key = key_of(b[j], 0);
          if (key >= k) ++c, s += weigh(key);
        }
      }
      *n = block_sum(c, redi);
      *m = block_sum(s, redd);
    };
    // the least key above minus infinity that min_p keeps
    uint32_t lo = kMinusInf, hi = kmax;  // lo fails, hi holds
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (weigh(mid) >= min_p) hi = mid;
      else lo = mid;
    }
    uint32_t least = hi;
    int n;
    double m;
    tokens_from(least, &n, &m);
    int most = 0x7fffffff;  // tokens with key `least` that are kept
    if (n > top_k) {        // the largest key from which on there are top_k
      lo = least, hi = kmax + 1;  // lo has them, hi has not
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        tokens_from(mid, &n, &m);
        if (n >= top_k) lo = mid;
        else hi = mid;
      }
      least = lo;
      tokens_from(least + 1, &n, &m);
      most = top_k - n;
      m += most * weigh(least);
    }
    const double target = top_p * m;
    if (top_p < 1.0) {
      lo = least, hi = kmax + 1;  // lo reaches the target, hi does not
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        tokens_from(mid, &n, &m);
        if (m >= target && mid > least) lo = mid;
        else hi = mid;
      }
      int above;
      double before;
      tokens_from(lo + 1, &above, &before);
      tokens_from(lo, &n, &m);
      most = min(lo == least ? most : 0x7fffffff, n - above);
      most = max(reach(before, weigh(lo), target, most), lo == kmax ? 1 : 0);
      least = lo;
    }
    tokens_from(least + 1, &n, &total);
    key_last = least;
    int at_least;
    tokens_from(least, &at_least, &m);
    ties = min(most, at_least - n);
    total += ties * weigh(least);
    for (int c = 0; c < p.chunks; ++c) {
      double s = 0.0;
#pragma unroll 1
      for (int i = 0; i < kPerThread / 8; ++i) {
        const int at = c * kChunk + (i * kThreads + tid) * 8;
        if (at >= p.vocab) break;
        uint32_t b[8];
        load8(logits, at, p.vocab, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t key = key_of(b[j], 0);
          if (key > key_last) s += weigh(key);
        }
      }
      s = wave_sum_f64(s);
      if (lane == 0) mass[c][wave] = s;
    }
  }
  __syncthreads();

  // the chunk of the draw
  const double w_last = weigh(key_last);
  const double target = u * total;
  auto tokens_at_last = [&](int c) -> int {  // tokens with the last kept key in a chunk
    if (fast) {
      const int bin = int(last >> 32);
      return int(p.counts[(row * p.chunks + c) * (kBins / 2) + bin / 2] >> (16 * (bin & 1)) & 0xffffu);
    }
    int n = 0;
    for (int i = 0; i < kPerThread / 8; ++i) {
      const int at = c * kChunk + (i * kThreads + tid) * 8;
      if (at >= p.vocab) break;
      uint32_t b[8];
      load8(logits, at, p.vocab, b);
#pragma unroll
      for (int j = 0; j < 8; ++j) n += key_of(b[j], 0) == key_last;
    }
    return block_sum(n, redi);
  };
  int chunk = 0, ties_left = ties;
  double cum = 0.0;
  int last_chunk = 0, last_ties = ties;
  double last_cum = 0.0;
  for (int c = 0; c < p.chunks; ++c) {
    double s = 0.0;
    for (int w = 0; w < kWaves; ++w) s += mass[c][w];
    const int here = min(tokens_at_last(c), ties_left);
    s += here * w_last;
    chunk = c;
    if (s > 0.0) last_chunk = c, last_ties = ties_left, last_cum = cum;
    if (cum + s > target) break;
    cum += s;
    ties_left -= here;
  }
  if (chunk != last_chunk) chunk = last_chunk, ties_left = last_ties, cum = last_cum;  // u so near 1 that no sum exceeds it

  const int first = chunk * kChunk + tid * kPerThread;
  uint32_t keep = 0, tie = 0;  // of this thread's 32 tokens
  uint32_t packed[kPerThread / 2];
#pragma unroll
  for (int i = 0; i < kPerThread / 8; ++i) {
    uint32_t b[8] = {0x7fffu, 0x7fffu, 0x7fffu, 0x7fffu, 0x7fffu, 0x7fffu, 0x7fffu, 0x7fffu};
    if (first + i * 8 < p.vocab) load8(logits, first + i * 8, p.vocab, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t key = key_of(b[j], 0);
      if (key > key_last) keep |= 1u << (i * 8 + j);
      if (key == key_last) tie |= 1u << (i * 8 + j);
      if (j & 1) packed[(i * 8 + j) / 2] |= b[j] << 16;
      else packed[(i * 8 + j) / 2] = b[j];
    }
  }
  int room = ties_left - block_prefix(int(__popc(tie)), redi);  // ties that this thread keeps
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    if (tie >> i & 1) {
      if (room > 0) keep |= 1u << i;
      --room;
    }
    const uint32_t b = packed[i / 2] >> (16 * (i & 1)) & 0xffffu;
    if (keep >> i & 1) s += fast ? weight[bin_of(b)] : weigh(key_of(b, 0));
  }
  double at = cum + block_prefix(s, redd);
  if (keep) {
    atomicMax(&final_kept, first + 31 - int(__clz(keep)));
    if (at + s > target) {
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        const uint32_t b = packed[i / 2] >> (16 * (i & 1)) & 0xffffu;
        if (!(keep >> i & 1)) continue;
        at += fast ? weight[bin_of(b)] : weigh(key_of(b, 0));
        if (at > target) {
          atomicMin(&drawn, first + i);
          break;
        }
      }
    }
  }
  __syncthreads();
  if (tid == 0) p.out[row] = drawn != 0x7fffffff ? drawn : final_kept;
}

size_t counts_bytes(int64_t batch, int64_t chunks) { return size_t(batch) * chunks * (kBins / 2) * 4; }

}  // namespace

extern "C" size_t mi_draw_workspace_size(int32_t batch_size, int32_t vocab_size) {
  if (batch_size <= 0 || batch_size > kMaxRows || vocab_size <= 0 || vocab_size > kMaxVocab) return 0;
  const int64_t chunks = (vocab_size + kChunk - 1) / kChunk;
  return counts_bytes(batch_size, chunks) + size_t(batch_size) * chunks * 12;
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
  p.vocab = vocab_size;
  p.chunks = (vocab_size + kChunk - 1) / kChunk;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.u = uniforms;
  p.out = out_tokens;
  p.counts = static_cast<uint32_t*>(workspace);
  char* at = static_cast<char*>(workspace) + counts_bytes(batch_size, p.chunks);
  p.winner = reinterpret_cast<unsigned long long*>(at);
  p.outside = reinterpret_cast<uint32_t*>(at + size_t(batch_size) * p.chunks * 8);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(count_kernel, dim3(p.chunks, batch_size), dim3(kThreads), 0, s, p);
  hipLaunchKernelGGL(draw_kernel, dim3(batch_size), dim3(kThreads), 0, s, p);
  return mi::check_launch("draw_kernel");
}

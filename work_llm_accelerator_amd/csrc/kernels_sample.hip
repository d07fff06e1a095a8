// Token sampling (semantics: include/qwen_hip_sample.h).
//
// Nothing is sorted.  Tokens are ranked by a 32-bit key of their logit (order_key: larger value, larger key) with
// ties by index, so a kept set is {key > T} and the first n of {key == T}; min-p is a test per token.  Weights are
// 64-bit integers (fixed point), so sums are exact whatever the order of their atomics.
//
// Four launches, each over all rows: the row's maximum and minimum; a histogram (counts and weights) over 2048 equal
// steps of the logit below the maximum (only where top-k or top-p is given); a list of the tokens of the steps in
// which they cut, and of each segment of the row the weight of the tokens in steps that are kept whatever the cut; the
// exact (T, n) from the list, and the draw: the listed tokens that are kept join their segments, the goal is found in
// the segments' running sum and then among the tokens of one segment.  Rows are split over many blocks except in
// the last launch.  A row with a small k and a top-p lists everything down to the step of its cut: its weights are
// those of the list only.
#include <hip/hip_runtime.h>

#include "kernels.hpp"
#include "qwen_device_math.hpp"

namespace qwen {

namespace {

constexpr int kBuckets = 2048;
constexpr int kList = 4096;     // most tokens that are listed (more: radix steps over the whole row; 151936 normal
                                // logits have up to 270 in a step)
// Largest k whose row is decided by its list where there is a top-p too, without weights in the histogram.  151936 tokens
// with a top-p, this way and by the histogram: k = 200 35 us and 36, 64 rows 64 and 80; k = 1000 44 and 41, 73 and 87;
// k = 2000 51 and 42, 82 and 91.  (Without a top-p the list takes longer: k = 200 25.0 and 24.7, k = 2000 35 and 30.)
constexpr int kSmall = 1024;
constexpr int kSegment = 512;   // tokens of a segment (times 2, 3, .. for more than kMaxSegments * 512 tokens)
constexpr int kMaxSegments = 1024;
constexpr int kMaxChunks = 256;
constexpr int kRed = 16;  // words for the waves of a block (and two a wave of the chunks' maxima)
constexpr uint32_t kUnlisted = 0xFFFFFFFFu;
constexpr int kChunkThreads = 256;
constexpr int kHistThreads = 512;
constexpr int kCutThreads = 256;  // (512: one row 1 us more, 64 rows 0.5 less; 1024: 4 and 1.4 more)

__device__ __forceinline__ float logit_at(const float* p, int i) { return p[i]; }
__device__ __forceinline__ float logit_at(const uint16_t* p, int i) { return bits_f32((uint32_t)p[i] << 16); }

typedef unsigned long long u64;

// The logit of a key (the inverse of order_key for non-NaN keys).
__device__ __forceinline__ float logit_of_key(uint32_t key) { return bits_f32(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

struct Cut {       // a kept set: key > key, and the first `ties` tokens with key == key
  uint32_t key;
  uint32_t ties;
};

// The value of the lane that DPP control kCtrl names, 0 where there is none or its row is not in kRows.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, kRows, 0xF, false);
}
template <int kCtrl, int kRows>
__device__ __forceinline__ u64 dpp(u64 x) {
  return ((u64)dpp<kCtrl, kRows>((uint32_t)(x >> 32)) << 32) | dpp<kCtrl, kRows>((uint32_t)x);
}
// Running sum (or maximum) over the wave's lanes, this one included: shifts by 1, 2, 4, 8 within rows of 16, then each
// row's last lane to the rows after it.  (A shuffle through LDS takes several times as long, and these launches
// are chains of such steps.)
template <class V, class F>
__device__ __forceinline__ V wave_running(V x, F&& f) {
  x = f(x, dpp<0x111, 0xF>(x));
  x = f(x, dpp<0x112, 0xF>(x));
  x = f(x, dpp<0x114, 0xF>(x));
  x = f(x, dpp<0x118, 0xF>(x));
  x = f(x, dpp<0x142, 0xA>(x));
  return f(x, dpp<0x143, 0xC>(x));
}
template <class V>
__device__ __forceinline__ V wave_scan(V x) {
  return wave_running(x, [](V a, V b) { return a + b; });
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return (uint32_t)__builtin_amdgcn_readlane((int)x, 63); }
__device__ __forceinline__ u64 last_lane(u64 x) { return ((u64)last_lane((uint32_t)(x >> 32)) << 32) | last_lane((uint32_t)x); }
template <class V>
__device__ __forceinline__ V wave_sum(V x) {
  return last_lane(wave_scan(x));
}
__device__ __forceinline__ u64 wave_max(u64 x) {
  return last_lane(wave_running(x, [](u64 a, u64 b) { return a > b ? a : b; }));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  return last_lane(wave_running(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; }));
}

// Sum over the block's threads (N) and the sum of the threads before (exclusive).
template <int N>
__device__ u64 block_scan(u64 x, u64* red, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 inc = wave_scan(x);
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  u64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) {
    const u64 v = red[w];
    before += w < wave ? v : 0ull;
    total += v;
  }
  return before + inc - x;
}

// One row's workspace.
struct RowSpace {
  u64 weights[kBuckets];      // histogram
  uint32_t counts[kBuckets];
  u64 best[kMaxChunks];       // (key << 32 | ~index) of each chunk's maximum
  uint32_t low[kMaxChunks];   // ~key of the least finite logit
  u64 list[kList];            // (key << 32 | index) of the tokens of the steps with a cut
  uint32_t listed;
  int k_step, p_low, p_high;  // the steps in the list (Needed)
  u64 k_before;
};

struct Sampler {
  SampleArgs a;
  int unit_bits;  // the weight of the largest logit is 2^unit_bits
  float spread;   // logits further than spread * temperature below the maximum have weight 0
  int chunks, per_chunk;            // blocks that share a row: maxima,
  int hist_chunks, hist_per_chunk;  // histogram and list
  int segments, blocks_per_segment;  // of kSegment tokens
  int segments_per_chunk;            // list
  RowSpace* space;
  u64* seg_weight;  // [rows][segments]
};

// 2^(t + bits) for t <= 0, 0 where t is below -110: Taylor's series over half a binade each way, degree 12 (its remainder
// is below 2^-52 of the value), the exponent set by integer addition.  (About a third of the operations of the
// library's exp, a division and a conversion to 64-bit integers, which were most of the histogram's time.)
__device__ __forceinline__ double exp2_falling(double t, int bits) {
  constexpr double kLn2 = 0.693147180559945309417232121458, kMagic = 6755399441055744.0;  // 1.5 * 2^52
  constexpr double c2 = kLn2 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4, c5 = c4 * kLn2 / 5, c6 = c5 * kLn2 / 6,
                   c7 = c6 * kLn2 / 7, c8 = c7 * kLn2 / 8, c9 = c8 * kLn2 / 9, c10 = c9 * kLn2 / 10, c11 = c10 * kLn2 / 11,
                   c12 = c11 * kLn2 / 12;
  const bool tiny = !(t >= -110.0);  // (NaN too: -inf logits at an infinite temperature)
  t = tiny ? -110.0 : t;
  const double m = t + kMagic, f = t - (m - kMagic);  // the low word of m is rint(t)
  double p = fma(c12, f, c11);
  p = fma(p, f, c10);
  p = fma(p, f, c9);
  p = fma(p, f, c8);
  p = fma(p, f, c7);
  p = fma(p, f, c6);
  p = fma(p, f, c5);
  p = fma(p, f, c4);
  p = fma(p, f, c3);
  p = fma(p, f, c2);
  p = fma(p, f, kLn2);
  p = fma(p, f, 1.0);
  const int k = (int)(uint32_t)__double_as_longlong(m) + bits;
  return tiny ? 0.0 : __hiloint2double(__double2hiint(p) + (k << 20), __double2loint(p));
}
// rint(x) for 0 <= x < 2^51.
__device__ __forceinline__ u64 rint_u64(double x) {
  constexpr double kMagic = 4503599627370496.0;  // 2^52
  return (u64)__double_as_longlong(x + kMagic) & 0xFFFFFFFFFFFFFull;
}

// What every launch after the first derives from the chunks' maxima.
struct Row {
  uint32_t top_key;
  int top_index;
  float top, temperature;
  float steps;  // histogram steps per unit of the logit
  double dtop, per_unit;  // per_unit: log2(e) / temperature
  int unit_bits;
  bool greedy;

  // Whole blocks of at least 256 threads (a multiple of 64); red: two words per wave.
  __device__ Row(const Sampler& s, int row, u64* red) {
    u64 best = 0;
    uint32_t low_key = 0;  // (~key: the largest is the least logit; 0: no finite logit)
    const RowSpace& w = s.space[row];
    temperature = s.a.temperature ? s.a.temperature[row] : 1.0f;
    if ((int)threadIdx.x < s.chunks) best = w.best[threadIdx.x], low_key = w.low[threadIdx.x];
    best = wave_max(best);
    low_key = wave_max(low_key);
    if ((threadIdx.x & 63) == 0 && threadIdx.x < kMaxChunks) red[threadIdx.x >> 6] = best, red[kMaxChunks / 64 + (threadIdx.x >> 6)] = low_key;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMaxChunks / 64; ++i) {
      best = red[i] > best ? red[i] : best;
      low_key = max(low_key, (uint32_t)red[kMaxChunks / 64 + i]);
    }
    __syncthreads();
    top_key = (uint32_t)(best >> 32);
    top_index = (int)~(uint32_t)best;
    const float low = low_key ? logit_of_key(~low_key) : __builtin_inff();
    top = logit_of_key(top_key);
    greedy = !(temperature > 0.0f) || top_key == 0xFFFFFFFFu || !(fabsf(top) <= 3.402823466e38f);
    dtop = top, per_unit = 1.44269504088896340735992468100 / (double)temperature, unit_bits = s.unit_bits;
    const float range = fminf(s.spread * temperature, top - low);
    steps = fminf((float)(kBuckets - 2) / range, 1.0e30f);
  }
  __device__ double weight(float v) const { return exp2_falling(((double)v - dtop) * per_unit, unit_bits); }  // unrounded
  __device__ u64 fixed(float v) const { return rint_u64(weight(v)); }
  // Falls with the logit; equal logits share a step.  The last step holds the logits without weight: -inf (also
  // where inf * 0 is NaN) and what is further than 2047 / 2046 of the spread below the maximum.
  __device__ int step(float v) const { return (int)fminf((top - v) * steps, (float)(kBuckets - 1)); }
};

template <class T>
__device__ __forceinline__ const T* row_of(const SampleArgs& a, int row) {
  return static_cast<const T*>(a.logits) + row * a.row_stride;
}

// The logits of 16 bytes.
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
  v[0] = bits_f32(q.x), v[1] = bits_f32(q.y), v[2] = bits_f32(q.z), v[3] = bits_f32(q.w);
}
__device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = bits_f32(w[i] << 16), v[2 * i + 1] = bits_f32(w[i] & 0xFFFF0000u);
}

// f(logit, index) over a block's chunk of `per` tokens of a row, four loads of 16 bytes in flight a thread (N of them);
// the tokens before the first 16-byte boundary and behind the last one come alone.
template <int N, class T, class F>
__device__ __forceinline__ void over_chunk(const T* x, int vocab, int per, F&& f) {
  constexpr int kAhead = 4, kVec = 16 / sizeof(T);
  const int begin = blockIdx.x * per, end = min(vocab, begin + per), tid = threadIdx.x;
  const int head = min(end - begin, (int)((16 - (reinterpret_cast<uintptr_t>(x + begin) & 15)) % 16 / sizeof(T)));
  const int first = begin + head, pieces = (end - first) / kVec, tail = first + pieces * kVec;
  const uint4* at = reinterpret_cast<const uint4*>(x + first);
  for (int p0 = tid; p0 < pieces; p0 += kAhead * N) {
    uint4 q[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) q[j] = at[min(p0 + j * N, pieces - 1)];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (p0 + j * N >= pieces) break;
      float v[kVec];
      unpack(q[j], v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(v[e], first + (p0 + j * N) * kVec + e);
    }
  }
  if (tid < head) f(logit_at(x, begin + tid), begin + tid);
  if (tail + tid < end) f(logit_at(x, tail + tid), tail + tid);
}

// Bound by the read: 64 rows of 151936 fp32 9.4 us, 4.1 TB/s (with 4-byte loads 10.6); one row 3.2 us, the launch.
// grid = (chunks, rows).  Also clears the row's histogram.
template <class T>
__global__ void __launch_bounds__(kChunkThreads) sample_max_kernel(Sampler s) {
  __shared__ u64 red[kRed];
  const int row = blockIdx.y, tid = threadIdx.x;
  const T* x = row_of<T>(s.a, row);
  RowSpace& w = s.space[row];
  for (int i = blockIdx.x * kChunkThreads + tid; i < kBuckets; i += gridDim.x * kChunkThreads) w.weights[i] = 0, w.counts[i] = 0;
  if (blockIdx.x == 0 && tid == 0) w.listed = 0;
  u64 best = 0;
  uint32_t low = 0;
  over_chunk<kChunkThreads>(x, s.a.vocab, s.per_chunk, [&](float v, int i) {
    const uint32_t key = order_key(v);
    const u64 k = ((u64)key << 32) | (u64)(~(uint32_t)i);
    best = k > best ? k : best;
    if (v > -__builtin_inff()) low = max(low, ~key);
  });
  best = wave_max(best);
  low = wave_max(low);
  if ((tid & 63) == 0) red[tid >> 6] = best, red[kMaxChunks / 64 + (tid >> 6)] = low;
  __syncthreads();
  if (tid != 0) return;
  for (int i = 1; i < kChunkThreads / 64; ++i) best = red[i] > best ? red[i] : best, low = max(low, (uint32_t)red[kMaxChunks / 64 + i]);
  w.best[blockIdx.x] = best;
  w.low[blockIdx.x] = low;
}

__device__ __forceinline__ bool wants_top_k(const Sampler& s, int row, int& k) {
  k = s.a.top_k ? s.a.top_k[row] : 0;
  return k > 0 && k < s.a.vocab;
}
__device__ __forceinline__ bool small_k(bool top_k, int k, bool top_p) { return top_k && k <= kSmall && top_p; }
__device__ __forceinline__ bool wants_top_p(const Sampler& s, int row, float& p) {
  p = s.a.top_p ? s.a.top_p[row] : 1.0f;
  return p < 1.0f;
}

// 64 rows of 151936, 8 of them with weights: 18 us; 10 without any weights: what they add is arithmetic in 64 bits.
// grid = (chunks, rows).
template <class T>
__global__ void __launch_bounds__(kHistThreads) sample_hist_kernel(Sampler s) {
  __shared__ u64 weights[kBuckets];
  __shared__ uint32_t counts[kBuckets];
  __shared__ u64 red[kRed];
  const int row = blockIdx.y, tid = threadIdx.x;
  int k;
  float p;
  const bool top_p = wants_top_p(s, row, p), top_k = wants_top_k(s, row, k);
  if (!top_k && !top_p) return;
  const bool weigh = top_p && !small_k(top_k, k, top_p);
  const Row r(s, row, red);
  if (r.greedy) return;
  for (int i = tid; i < kBuckets; i += kHistThreads) weights[i] = 0, counts[i] = 0;
  __syncthreads();
  const T* x = row_of<T>(s.a, row);
  over_chunk<kHistThreads>(x, s.a.vocab, s.hist_per_chunk, [&](float v, int) {
    const int b = r.step(v);
    atomicAdd(&counts[b], 1u);
    if (weigh) {
      const u64 n = r.fixed(v);
      if (n) atomicAdd(&weights[b], n);
    }
  });
  __syncthreads();
  RowSpace& w = s.space[row];
  for (int i = tid; i < kBuckets; i += kHistThreads) {
    if (counts[i]) atomicAdd(&w.counts[i], counts[i]);
    if (weights[i]) atomicAdd(&w.weights[i], weights[i]);
  }
}

// The histogram of a row held by a block of N threads: thread t has kBuckets / N adjacent steps and what is before.
template <int N>
struct Held {
  static constexpr int kPer = kBuckets / N;
  u64 count[kPer], weight[kPer], count_before, weight_before, weight_total;
  __device__ explicit Held(const RowSpace& w) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) count[i] = w.counts[kPer * threadIdx.x + i], weight[i] = w.weights[kPer * threadIdx.x + i];
  }
  __device__ void scan(u64* red) {
    u64 n = 0, x = 0, none;
#pragma unroll
    for (int i = 0; i < kPer; ++i) n += count[i], x += weight[i];
    count_before = block_scan<N>(n, red, none);
    weight_before = block_scan<N>(x, red, weight_total);
  }
  struct Found {
    int step;
    u64 before;  // counts or weight before the step
    u64 at, tokens, tokens_before;  // weight and tokens of the step
  };
  // The step in which a rank ends: the last one with tokens before which there are fewer than `limit` (by weight: the
  // last one with weight before which there is less than `goal`).  Steps behind `last` do not count, and step
  // `last` counts as `last_weight`.
  __device__ Found find(bool by_weight, u64 limit, double goal, int last, u64 last_weight, u64* pick, uint32_t* pick_step) const {
    if (threadIdx.x == 0) *pick_step = 0u;
    __syncthreads();
    u64 run = by_weight ? weight_before : count_before, n = count_before, before = 0, at = 0, tokens = 0, tokens_before = 0;
    int mine = threadIdx.x == 0 ? 0 : -1;
    if (threadIdx.x == 0) at = weight[0], tokens = count[0];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = kPer * threadIdx.x + i;
      const u64 x = !by_weight ? count[i] : b < last ? weight[i] : b == last ? last_weight : 0ull;
      if (x && (by_weight ? (double)run < goal : run < limit))
        mine = b, before = run, at = weight[i], tokens = count[i], tokens_before = n;
      run += by_weight ? weight[i] : x;
      n += count[i];
    }
    if (mine >= 0) atomicMax(pick_step, (uint32_t)mine);
    __syncthreads();
    if (mine >= 0 && *pick_step == (uint32_t)mine) pick[0] = before, pick[1] = at, pick[2] = tokens, pick[3] = tokens_before;
    __syncthreads();
    const Found f{(int)*pick_step, pick[0], pick[1], pick[2], pick[3]};
    __syncthreads();
    return f;
  }
  // Weight before step b.
  __device__ u64 weight_to(int b, u64* pick) const {
    if (b >= kBuckets) return weight_total;
    if (b / kPer == (int)threadIdx.x) {
      u64 x = weight_before;
#pragma unroll
      for (int i = 0; i < kPer; ++i) x += i < b % kPer ? weight[i] : 0ull;
      pick[0] = x;
    }
    __syncthreads();
    const u64 x = pick[0];
    __syncthreads();
    return x;
  }
};

// The steps whose tokens decide the cuts of a row: that of top-k (-1: none, or among tokens without weight) and
// those in which top-p can end, which depends on the part of the top-k step that is kept (empty: high < low).
struct Needed {
  int k_step, low, high;
  u64 k_before;
  bool listed;  // their tokens fit the list
  __device__ bool has(int b) const { return b == k_step || (b >= low && b <= high); }
};
template <int N>
__device__ Needed needed_steps(const Held<N>& h, bool top_k, int k, bool top_p, float p, u64* pick, uint32_t* pick_step) {
  Needed n{-1, 0, -1, 0, false};
  u64 at = 0, tokens = 0;
  if (top_k) {
    const auto f = h.find(false, (u64)k, 0.0, kBuckets, 0, pick, pick_step);
    if (f.step < kBuckets - 1) n.k_step = f.step, n.k_before = f.before, at = f.at, tokens = f.tokens;
    if (small_k(top_k, k, top_p)) {  // everything with weight down to the cut
      n.low = 0, n.high = min(f.step, kBuckets - 2);
      n.listed = f.before + tokens <= (u64)kList;
      return n;
    }
  }
  if (top_p) {
    const int last = n.k_step < 0 ? kBuckets : n.k_step;
    const u64 before = h.weight_to(last, pick);
    const double least = (double)p * (double)before, most = (double)p * (double)(before + at);
    if (most > 0.0) {
      const auto hi = h.find(true, 0, most, last, at, pick, pick_step);
      const auto lo = last == kBuckets ? hi : h.find(true, 0, least, last, at, pick, pick_step);
      n.high = hi.step, n.low = lo.step;
      tokens += hi.tokens_before + hi.tokens - lo.tokens_before;  // (the top-k step may count twice)
    }
  }
  n.listed = tokens <= (u64)kList;
  return n;
}

// A lane's kLane adjacent tokens from `first` on (-inf behind the row): 16-byte loads where they are whole and aligned.
constexpr int kLane = kSegment / 64;
template <class T>
__device__ __forceinline__ void load_lane(const T* x, int first, int vocab, float (&v)[kLane]) {
  constexpr int kVec = 16 / sizeof(T);
  if (first + kLane <= vocab && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
#pragma unroll
    for (int n = 0; n < kLane / kVec; ++n) {
      float part[kVec];
      unpack(reinterpret_cast<const uint4*>(x + first)[n], part);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[kVec * n + e] = part[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kLane; ++j) v[j] = first + j < vocab ? logit_at(x, first + j) : -__builtin_inff();
  }
}

// The kept weight of a logit, without regard to ties.
__device__ __forceinline__ u64 kept_weight(const Row& r, float v, double least) {
  const double w = r.weight(v);
  return w >= least ? rint_u64(w) : 0ull;
}
__device__ __forceinline__ double least_weight(const Sampler& s, int row) {
  const float q = s.a.min_p ? s.a.min_p[row] : 0.0f;
  return q > 0.0f ? (double)fminf(q, 1.0f) * (double)(1ull << s.unit_bits) : 0.0;
}

// Lists the needed steps' tokens, and adds up the weight of those in steps that are kept whatever the cut: a wave per
// segment, in turn.  Every block finds the steps for itself.  64 rows of 151936: 27.5 us, one row 10, of which finding
// the steps takes 5.  grid = (chunks of segments, rows).
template <class T>
__global__ void __launch_bounds__(kHistThreads) sample_list_kernel(Sampler s) {
  __shared__ u64 red[kRed], pick[4];
  __shared__ uint32_t pick_step, found, at;
  __shared__ u64 keys[kList];
  const int row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  int k;
  float p;
  const bool top_k = wants_top_k(s, row, k), top_p = wants_top_p(s, row, p);
  RowSpace& w = s.space[row];
  Held<kHistThreads> held(w);
  const double least = least_weight(s, row);
  const Row r(s, row, red);
  if (r.greedy) return;
  Needed need{-1, kBuckets, -1, 0, true};
  int sure = kBuckets;  // tokens of the steps before it are kept
  if (top_k || top_p) {
    held.scan(red);
    need = needed_steps(held, top_k, k, top_p, p, pick, &pick_step);
    if (top_p)
      sure = need.low;
    else if (need.k_step >= 0)
      sure = need.k_step;
  }
  if (blockIdx.x == 0 && tid == 0) {
    w.k_step = need.k_step, w.p_low = need.low, w.p_high = need.high, w.k_before = need.k_before;
    if (!need.listed) w.listed = kUnlisted;
  }
  if (!need.listed) return;
  if (tid == 0) found = 0u;
  __syncthreads();
  const T* x = row_of<T>(s.a, row);
  const int last = min(s.segments, ((int)blockIdx.x + 1) * s.segments_per_chunk);
  for (int seg = blockIdx.x * s.segments_per_chunk + (tid >> 6); seg < last; seg += kHistThreads / 64) {
    u64 sum = 0;
    for (int blk = 0; blk < s.blocks_per_segment; ++blk) {
      const int first = (seg * s.blocks_per_segment + blk) * kSegment + kLane * lane;
      float v[kLane];
      load_lane(x, first, s.a.vocab, v);
#pragma unroll
      for (int j = 0; j < kLane; ++j) {
        if (first + j >= s.a.vocab) break;
        const int b = r.step(v[j]);
        if (need.has(b))
          keys[atomicAdd(&found, 1u)] = ((u64)order_key(v[j]) << 32) | (u64)(uint32_t)(first + j);
        else if (b < sure)
          sum += kept_weight(r, v[j], least);
      }
    }
    sum = wave_sum(sum);
    if (lane == 0) s.seg_weight[(size_t)row * s.segments + seg] = sum;
  }
  __syncthreads();
  if (tid == 0 && found) at = atomicAdd(&w.listed, found);  // one a block: they are serialized over the row
  __syncthreads();
  for (int i = tid; i < (int)found; i += kHistThreads) w.list[at + i] = keys[i];
}

// The cuts of one row, and its draw: a chain of reductions over one block, bound by their latency (64 rows 22.5 us, one row 15).
// A row with more tokens in the cuts' steps than the list holds (nearly equal logits) is gone through whole here: 0.3 to
// 0.9 ms for 151936 tokens, most of it atomics at the same address.
// grid = rows.
template <class T>
__global__ void __launch_bounds__(kCutThreads) sample_cut_kernel(Sampler s) {
  __shared__ u64 hist[kBuckets];
  __shared__ uint32_t count[kBuckets];
  __shared__ u64 list[kList], list_weight[kList];
  __shared__ u64 seg_weight[kMaxSegments];
  __shared__ uint32_t seg_ties[kMaxSegments];
  __shared__ u64 red[kRed], pick[4];
  __shared__ uint32_t pick_step, differ, sample_key;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, vocab = s.a.vocab;
  Cut cut{0u, 0u};  // everything: every key is above 0 (-inf has key 0x007FFFFF)
  int k;
  float p;
  const bool top_k = wants_top_k(s, row, k), top_p = wants_top_p(s, row, p);
  RowSpace& w = s.space[row];
  const uint32_t listed = w.listed;
  Needed need{w.k_step, w.p_low, w.p_high, w.k_before, listed != kUnlisted};
  const bool small = small_k(top_k, k, top_p);
  const float uf = s.a.uniforms[row];
  const double least = least_weight(s, row);
  Held<kCutThreads> held(w);
  for (int i = tid; i < s.segments; i += kCutThreads) seg_weight[i] = s.seg_weight[(size_t)row * s.segments + i], seg_ties[i] = 0;
  if (need.listed)
    for (int i = tid; i < (int)listed; i += kCutThreads) list[i] = w.list[i];
  const Row r(s, row, red);
  if (r.greedy) {
    if (tid == 0) s.a.token_ids[row] = r.top_index;
    return;
  }
  const T* x = row_of<T>(s.a, row);
  if (top_p && !small) held.scan(red);
  if (top_p && need.listed)  // (each thread the entries that it has copied)
    for (int i = tid; i < (int)listed; i += kCutThreads) list_weight[i] = r.fixed(logit_of_key((uint32_t)(list[i] >> 32)));

  // f(index, key) for the listed tokens (index in the list), and for all tokens of the row (eight loads in flight a thread).
  auto list_key = [&](int i) { return (uint32_t)(list[i] >> 32); };
  auto over_list = [&](auto&& f) {
    for (int i = tid; i < (int)listed; i += kCutThreads) f(i, list_key(i));
  };
  auto over_row = [&](auto&& f) {
    constexpr int kAhead = 8;
    for (int i0 = tid; i0 < vocab; i0 += kAhead * kCutThreads) {
      float v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = logit_at(x, min(i0 + j * kCutThreads, vocab - 1));
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i0 + j * kCutThreads < vocab) f(i0 + j * kCutThreads, order_key(v[j]));
    }
  };
  // Selects in falling order of 32-bit keys among candidates, the (i, key) that `over` goes through and `has` accepts, plus
  // extra.ties more at extra.key, with `above` in front of them: the key T at which a rank ends and the number of
  // candidates at T within it.  The rank takes candidates before which there are fewer than `limit` (kCount), or
  // weight below `goal` (kBelow).  Radix steps of up to 11 bits from the highest bit in which the candidates differ,
  // each a histogram scanned from its largest bucket, until the candidates are equal.
  enum { kCount, kBelow };
  auto select = [&](auto over, auto has, auto weight, u64 above, int rank, u64 limit, double goal, Cut extra, Cut none) {
    int known = 32;  // candidates: key >> known == prefix
    uint32_t prefix = 0;
    auto candidate = [&](int i, uint32_t key) { return has(i, key) && (known == 32 || (key >> known) == prefix); };
    auto within = [&](u64 v) { return rank == kCount ? v < limit : (double)v < goal; };
    for (;;) {
      for (int i = tid; i < kBuckets; i += kCutThreads) hist[i] = 0, count[i] = 0;
      if (tid == 0) differ = 0u, sample_key = 0u, pick_step = 0xFFFFFFFFu;
      __syncthreads();
      const bool extra_now = extra.ties && (known == 32 || (extra.key >> known) == prefix);
      uint32_t mine = 0, lo = 0xFFFFFFFFu;
      over([&](int i, uint32_t key) {
        if (candidate(i, key)) mine = max(mine, key), lo = min(lo, key);
      });
      if (extra_now && tid == 0) mine = max(mine, extra.key), lo = min(lo, extra.key);
      if (mine) atomicMax(&sample_key, mine);
      __syncthreads();
      const uint32_t top = sample_key;  // the largest candidate
      if (top == 0u) return none;
      if (mine && (lo ^ top) != 0u) atomicMax(&differ, lo ^ top);  // its highest bit: the highest that differs
      __syncthreads();
      const uint32_t bits_off = differ;
      const int hb = bits_off ? 31 - __clz((int)bits_off) : -1, shift = max(0, hb - 10), bits = hb + 1 - shift;
      const uint32_t mask = bits ? (1u << bits) - 1u : 0u;
      over([&](int i, uint32_t key) {
        if (!candidate(i, key)) return;
        const uint32_t bucket = (key >> shift) & mask;
        atomicAdd(&count[bucket], 1u);
        if (rank != kCount) atomicAdd(&hist[bucket], weight(i, key));
      });
      __syncthreads();
      if (extra_now && tid == 0) {
        const uint32_t bucket = (extra.key >> shift) & mask;
        count[bucket] += extra.ties;
        hist[bucket] += extra.ties * r.fixed(logit_of_key(extra.key));
      }
      __syncthreads();
      if (hb < 0) {  // all equal (bucket 0)
        const u64 have = count[0], one = rank == kCount ? 0ull : hist[0] / have;
        Cut c{top, 1};
        if (rank == kCount) {
          c.ties = (uint32_t)min(have, limit - above);
        } else {
          u64 j = 1;  // the first one is within the rank
          const double guess = (goal - (double)above) / (double)one;
          if (guess > 2.0) j = guess < (double)have ? (u64)guess - 1u : have;
          while (j > 1 && !within(above + (j - 1) * one)) --j;
          while (j < have && within(above + j * one)) ++j;
          c.ties = (uint32_t)j;
        }
        __syncthreads();
        return c;
      }
      // this thread's adjacent buckets, the largest first; the smallest non-empty one that starts within the rank
      constexpr int kPer = kBuckets / kCutThreads;
      const int hi = kBuckets - 1 - kPer * tid;
      u64 b[kPer], sum = 0, total, my_before = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) b[i] = rank == kCount ? count[hi - i] : hist[hi - i], sum += b[i];
      u64 run = above + block_scan<kCutThreads>(sum, red, total);
      uint32_t my = 0xFFFFFFFFu;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (b[i] && within(run)) my = hi - i, my_before = run;
        run += b[i];
      }
      if (my != 0xFFFFFFFFu) atomicMin(&pick_step, my);
      __syncthreads();
      const uint32_t got = pick_step;
      if (got == 0xFFFFFFFFu) return none;
      if (got == my) pick[0] = my_before;
      __syncthreads();
      above = pick[0];
      prefix = shift + bits < 32 ? ((top >> (shift + bits)) << bits) | got : got;
      known = shift;
      __syncthreads();
    }
  };
  auto key_weight = [&](int i, uint32_t key) { return need.listed ? list_weight[i] : r.fixed(logit_of_key(key)); };
  // by counts: the first k of the tokens of the cut's step (the whole row without a list)
  auto top_k_cut = [&]() {
    const int step = need.k_step;
    if (need.listed)
      return select(over_list, [&](int, uint32_t key) { return r.step(logit_of_key(key)) == step; }, key_weight, need.k_before,
                    kCount, (u64)k, 0.0, Cut{0u, 0u}, cut);
    return select(over_row, [](int, uint32_t) { return true; }, key_weight, 0, kCount, (u64)k, 0.0, Cut{0u, 0u}, cut);
  };
  // by weight: what is below `goal` of the tokens within `in` of a step (step < 0: of all listed, of the row without a list)
  auto top_p_cut = [&](int step, u64 before, double goal, Cut in) {
    if (need.listed)
      return select(over_list, [&](int, uint32_t key) { return key > in.key && (step < 0 || r.step(logit_of_key(key)) == step); },
                    key_weight, before, kBelow, 0, goal, in, in);
    return select(over_row, [&](int, uint32_t key) { return key > in.key; }, key_weight, 0, kBelow, 0, goal, in, in);
  };
  // weight of the listed tokens (of the row without a list) above the cut in a step (< 0: in all), and of its ties
  auto weight_of = [&](int step) {
    u64 part = 0, total;
    auto add = [&](int i, uint32_t key) {
      if (key > cut.key && (step < 0 || r.step(logit_of_key(key)) == step)) part += key_weight(i, key);
    };
    if (need.listed)
      over_list(add);
    else
      over_row(add);
    if (tid == 0 && cut.ties) part += cut.ties * r.fixed(logit_of_key(cut.key));
    block_scan<kCutThreads>(part, red, total);
    return total;
  };

  __syncthreads();
  if (need.k_step >= 0) cut = top_k_cut();
  if (top_p) {
    // weight of what is kept so far: whole steps, and the kept part of the cut one
    const int last = need.k_step < 0 ? kBuckets : need.k_step;
    u64 total, last_weight = 0;
    if (small || !need.listed) {
      total = weight_of(-1);
    } else {
      total = held.weight_to(last, pick);
      if (need.k_step >= 0) last_weight = weight_of(last);
      total += last_weight;
    }
    const double goal = (double)p * (double)total;
    if (!(goal > 0.0)) {  // (p <= 0: the first token alone)
      if (tid == 0) s.a.token_ids[row] = r.top_index;
      return;
    }
    if (small || !need.listed) {
      cut = top_p_cut(-1, 0, goal, cut);
    } else {
      const auto f = held.find(true, 0, goal, last, last_weight, pick, &pick_step);
      cut = top_p_cut(f.step, f.before, goal, f.step == last ? cut : Cut{0u, 0u});
    }
  }

  // Each segment's kept weight above the cut, and its tokens at it
  if (need.listed) {
    for (int i = tid; i < (int)listed; i += kCutThreads) {
      const uint32_t key = list_key(i);
      const int seg = (int)(uint32_t)list[i] / (kSegment * s.blocks_per_segment);
      if (key > cut.key) {
        const u64 n = kept_weight(r, logit_of_key(key), least);
        if (n) atomicAdd(&seg_weight[seg], n);
      } else if (key == cut.key) {
        atomicAdd(&seg_ties[seg], 1u);
      }
    }
  } else {
    for (int seg = tid >> 6; seg < s.segments; seg += kCutThreads / 64) {
      u64 sum = 0;
      uint32_t n = 0;
      for (int blk = 0; blk < s.blocks_per_segment; ++blk) {
        const int first = (seg * s.blocks_per_segment + blk) * kSegment + kLane * lane;
        float v[kLane];
        load_lane(x, first, vocab, v);
#pragma unroll
        for (int j = 0; j < kLane; ++j) {
          const uint32_t key = order_key(v[j]);
          if (key > cut.key) sum += kept_weight(r, v[j], least);
          if (first + j < vocab && key == cut.key) ++n;
        }
      }
      sum = wave_sum(sum);
      n = wave_sum(n);
      if (lane == 0) seg_weight[seg] = sum, seg_ties[seg] = n;
    }
  }
  if (tid == 0) pick_step = 0u;
  __syncthreads();
  // The last segment with kept weight that starts at or below the goal; a thread has kPer adjacent ones
  constexpr int kPer = kMaxSegments / kCutThreads;
  const u64 tie = cut.ties ? kept_weight(r, logit_of_key(cut.key), least) : 0ull;
  u64 weight[kPer], sum = 0, none, total, my_above = 0, my_seen = 0;
  uint32_t ties[kPer], all_ties = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const bool live = kPer * tid + i < s.segments;
    ties[i] = live ? seg_ties[kPer * tid + i] : 0u, weight[i] = live ? seg_weight[kPer * tid + i] : 0ull;
    all_ties += ties[i];
  }
  u64 seen = block_scan<kCutThreads>(all_ties, red, none);
  const u64 seen_first = seen;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    weight[i] += (seen >= cut.ties ? 0ull : min((u64)ties[i], (u64)cut.ties - seen)) * tie;
    seen += ties[i];
    sum += weight[i];
  }
  u64 run = block_scan<kCutThreads>(sum, red, total);
  const double goal = (uf > 0.0f ? (double)fminf(uf, 1.0f) : 0.0) * (double)total;
  int mine = -1;
  seen = seen_first;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (weight[i] && !((double)run > goal)) mine = kPer * tid + i, my_above = run, my_seen = seen;
    run += weight[i];
    seen += ties[i];
  }
  if (mine >= 0) atomicMax(&pick_step, (uint32_t)mine);
  __syncthreads();
  const int segment = (int)pick_step;
  if (mine == segment) pick[0] = my_above, pick[1] = my_seen;
  __syncthreads();
  if (tid >= 64) return;
  // The token: one wave, each lane eight adjacent tokens
  u64 above = pick[0];
  uint32_t rank0 = (uint32_t)pick[1];
  int token = 0;
  for (int blk = 0; blk < s.blocks_per_segment; ++blk) {
    const int first = (segment * s.blocks_per_segment + blk) * kSegment + kLane * tid;
    float v[kLane];
    load_lane(x, first, vocab, v);
    uint32_t at_cut = 0;
#pragma unroll
    for (int j = 0; j < kLane; ++j) at_cut += first + j < vocab && order_key(v[j]) == cut.key ? 1u : 0u;
    uint32_t rank = wave_scan(at_cut);
    const uint32_t rank_next = rank0 + last_lane(rank);
    rank += rank0 - at_cut;
    u64 here[kLane], part = 0;
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      const uint32_t key = order_key(v[j]);
      here[j] = key > cut.key ? kept_weight(r, v[j], least) : 0ull;
      if (first + j < vocab && key == cut.key && rank++ < cut.ties) here[j] = tie;
      part += here[j];
    }
    u64 upto = wave_scan(part);
    const u64 above_next = above + last_lane(upto);
    upto += above - part;
    int past = -1, some = -1;  // the lane's first token beyond the goal, and its last one with weight
#pragma unroll
    for (int j = 0; j < kLane; ++j) {
      upto += here[j];
      if (here[j]) {
        some = j;
        if (past < 0 && (double)upto > goal) past = j;
      }
    }
    const u64 beyond = __ballot(past >= 0), any = __ballot(some >= 0);
    if (any) {
      const int from = beyond ? __ffsll(beyond) - 1 : 63 - __clzll(any);
      token = __shfl(first + (beyond ? past : some), from, 64);
    }
    if (beyond) break;
    above = above_next;
    rank0 = rank_next;
  }
  if (tid == 0) s.a.token_ids[row] = token;
}

template <class T>
void run_sample(const Sampler& s, hipStream_t st) {
  const int rows = s.a.rows;
  hipLaunchKernelGGL(sample_max_kernel<T>, dim3(s.chunks, rows), dim3(kChunkThreads), 0, st, s);
  if (s.a.top_k || s.a.top_p)
    hipLaunchKernelGGL(sample_hist_kernel<T>, dim3(s.hist_chunks, rows), dim3(kHistThreads), 0, st, s);
  const int list_chunks = (s.segments + s.segments_per_chunk - 1) / s.segments_per_chunk;
  hipLaunchKernelGGL(sample_list_kernel<T>, dim3(list_chunks, rows), dim3(kHistThreads), 0, st, s);
  hipLaunchKernelGGL(sample_cut_kernel<T>, dim3(rows), dim3(kCutThreads), 0, st, s);
}

}  // namespace

static int blocks_per_segment(int vocab) { return (vocab + kMaxSegments * kSegment - 1) / (kMaxSegments * kSegment); }
static int segments_of(int vocab) {
  const int tokens = blocks_per_segment(vocab) * kSegment;
  return (vocab + tokens - 1) / tokens;
}

size_t sample_workspace_bytes(int rows, int vocab) {
  return (size_t)rows * (sizeof(RowSpace) + segments_of(vocab) * sizeof(u64));
}

void launch_sample(const SampleArgs& a, void* workspace, hipStream_t st) {
  Sampler s{};
  s.a = a;
  int bits = 0;  // weights of up to 2^24 tokens sum to less than 2^62
  while ((1 << bits) < a.vocab) ++bits;
  s.unit_bits = 62 - bits < 50 ? 62 - bits : 50;
  s.spread = (float)(s.unit_bits + 1) * 0.6931472f;
  auto split = [&](int blocks, int least, int threads, int& chunks, int& per) {
    chunks = blocks / a.rows;
    const int most = (a.vocab + least - 1) / least;
    chunks = chunks > most ? most : chunks;
    chunks = chunks < 1 ? 1 : chunks > kMaxChunks ? kMaxChunks : chunks;
    per = ((a.vocab + chunks - 1) / chunks + threads - 1) / threads * threads;
    chunks = (a.vocab + per - 1) / per;
  };
  split(1024, 1024, kChunkThreads, s.chunks, s.per_chunk);  // about four a CU over all rows, of 1024 tokens at least
  // histogram: two of 512 threads a CU (64 rows of 151936: 18 us, and so with four or eight; one of 1024 threads the same, but
  // one row 7 us instead of 6; four of 256 threads 1 and 2 us more; two of 1024 4 more)
  split(512, 4 * kHistThreads, kHistThreads, s.hist_chunks, s.hist_per_chunk);
  s.segments = segments_of(a.vocab);
  s.blocks_per_segment = blocks_per_segment(a.vocab);
  // list: four blocks a CU (64 rows of 151936: 27.5 us; with two or eight 30, with one 33), a segment a wave at least
  s.segments_per_chunk = (int)(((long long)s.segments * a.rows + 1023) / 1024);
  if (s.segments_per_chunk < kHistThreads / 64) s.segments_per_chunk = kHistThreads / 64;
  s.space = static_cast<RowSpace*>(workspace);
  s.seg_weight = reinterpret_cast<u64*>(s.space + a.rows);
  if (a.type == QWEN_TYPE_F32)
    run_sample<float>(s, st);
  else
    run_sample<uint16_t>(s, st);
}

}  // namespace qwen

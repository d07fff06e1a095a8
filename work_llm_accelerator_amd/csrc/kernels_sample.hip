// Token sampling (semantics: include/qwen_hip_sample.h).
//
// Nothing is sorted.  Tokens are ranked by a 32-bit key of their logit (order_key: larger value, larger key) with
// ties by index, so a kept set is {key > T} and the first n of {key == T}: top-k and top-p each find their (T, n)
// by three radix steps (11, 11 and 10 bits) over histograms of counts or weights, min-p is a test per token.
// Weights are 64-bit integers (fixed point), so histogram sums are exact whatever the order of their atomics.
#include <hip/hip_runtime.h>

#include "kernels.hpp"
#include "qwen_device_math.hpp"

namespace qwen {

namespace {

constexpr int kThreads = 1024;
constexpr int kBuckets = 2048;
constexpr int kSegments = 1024;  // most index ranges of a row in the draw

__device__ __forceinline__ float logit_at(const float* p, int i) { return p[i]; }
__device__ __forceinline__ float logit_at(const uint16_t* p, int i) { return bits_f32((uint32_t)p[i] << 16); }

typedef unsigned long long u64;

// The logit of a key (the inverse of order_key for non-NaN keys).
__device__ __forceinline__ float logit_of_key(uint32_t key) { return bits_f32(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key); }

struct Cut {       // a kept set: key > key, and the first `ties` tokens with key == key
  uint32_t key;
  uint32_t ties;
};

// Sum over the block's 1024 threads and the sums of the threads before (exclusive).
__device__ u64 block_scan(u64 x, u64* red, u64& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  u64 inc = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const u64 o = __shfl_up(inc, off, 64);
    if (lane >= off) inc += o;
  }
  __syncthreads();
  if (lane == 63) red[wave] = inc;
  __syncthreads();
  u64 before = 0;
  total = 0;
  for (int w = 0; w < kThreads / 64; ++w) {
    const u64 v = red[w];
    before += w < wave ? v : 0ull;
    total += v;
  }
  return before + inc - x;
}

// One block per row.
template <class T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a, double unit) {
  __shared__ u64 hist[kBuckets];
  __shared__ uint32_t count[kBuckets];
  __shared__ u64 red[kThreads / 64];
  __shared__ u64 pick_above;
  __shared__ uint32_t pick_bucket, pick_count_above;
  const int row = blockIdx.x, tid = threadIdx.x, vocab = a.vocab;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;

  // maximum and its first index
  u64 best = 0;
  for (int i = tid; i < vocab; i += kThreads) {
    const u64 k = ((u64)order_key(logit_at(x, i)) << 32) | (u64)(~(uint32_t)i);
    best = k > best ? k : best;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const u64 o = __shfl_xor(best, off, 64);
    best = o > best ? o : best;
  }
  if ((tid & 63) == 0) red[tid >> 6] = best;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) best = red[w] > best ? red[w] : best;
  const uint32_t top_key = (uint32_t)(best >> 32);
  const float top = logit_of_key(top_key);
  const float temperature = a.temperature ? a.temperature[row] : 1.0f;
  const bool finite = top_key != 0xFFFFFFFFu && fabsf(top) <= 3.402823466e38f;
  if (!(temperature > 0.0f) || !finite) {
    if (tid == 0) a.token_ids[row] = (int)~(uint32_t)best;
    return;
  }
  const double dtop = top, dtemp = temperature;
  const float qmin = a.min_p ? a.min_p[row] : 0.0f;
  const double least = qmin > 0.0f ? (double)fminf(qmin, 1.0f) : 0.0;
  auto real_weight = [&](float v) { return exp(((double)v - dtop) / dtemp); };
  auto fixed = [&](double w) { return (u64)rint(w * unit); };

  // The (T, n) of a rank by counts (`by_weight` false: the first `k` tokens) or by weight within `in` (tokens
  // before which the weight is below `goal`).  One histogram per radix step, scanned from the largest bucket.
  auto select = [&](bool by_weight, uint32_t k, double goal, Cut in) {
    uint32_t prefix = 0, above_n = 0;
    u64 above = 0;
    for (int step = 0; step < 3; ++step) {
      const int shift = step == 0 ? 21 : step == 1 ? 10 : 0, bits = step == 2 ? 10 : 11;
      for (int i = tid; i < kBuckets; i += kThreads) hist[i] = 0, count[i] = 0;
      __syncthreads();
      for (int i = tid; i < vocab; i += kThreads) {
        const float v = logit_at(x, i);
        const uint32_t key = order_key(v);
        if (step > 0 && (key >> (shift + bits)) != prefix) continue;
        if (by_weight && key <= in.key) continue;
        const uint32_t bucket = (key >> shift) & ((1u << bits) - 1u);
        atomicAdd(&count[bucket], 1u);
        if (by_weight) atomicAdd(&hist[bucket], fixed(real_weight(v)));
      }
      __syncthreads();
      if (by_weight && tid == 0 && in.ties && (step == 0 || (in.key >> (shift + bits)) == prefix)) {
        const uint32_t bucket = (in.key >> shift) & ((1u << bits) - 1u);
        count[bucket] += in.ties;
        hist[bucket] += in.ties * fixed(real_weight(logit_of_key(in.key)));
      }
      __syncthreads();
      const int hi = kBuckets - 1 - 2 * tid, lo = hi - 1;  // this thread's two buckets, the largest first
      u64 total, none;
      const u64 n_before = block_scan((u64)count[hi] + count[lo], red, total);
      const u64 w_before = by_weight ? block_scan(hist[hi] + hist[lo], red, none) : 0;
      if (tid == 0) pick_bucket = 0xFFFFFFFFu;
      __syncthreads();
      // the last bucket that holds a token of the rank: those before it hold fewer than asked for
      u64 n = above_n + n_before, w = above + w_before;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int bucket = j ? lo : hi;
        const u64 n_next = n + count[bucket], w_next = w + hist[bucket];
        const bool starts = by_weight ? hist[bucket] && (double)w < goal : count[bucket] && n < k;
        const bool ends = by_weight ? !((double)w_next < goal) : n_next >= k;
        if (starts && ends) pick_bucket = bucket, pick_above = w, pick_count_above = (uint32_t)n;
        n = n_next, w = w_next;
      }
      __syncthreads();
      if (pick_bucket == 0xFFFFFFFFu) return in;  // everything is kept
      prefix = (prefix << bits) | pick_bucket;
      above = pick_above;
      above_n = pick_count_above;
      const uint32_t held = count[pick_bucket];
      __syncthreads();
      if (step == 2) {
        Cut c{prefix, 0};
        if (!by_weight) {
          c.ties = k - above_n;
        } else {
          const u64 w1 = fixed(real_weight(logit_of_key(prefix)));
          uint32_t j = 1;  // the first tie has less than `goal` before it
          const double guess = (goal - (double)above) / (double)w1;
          if (guess > 2.0) j = guess < (double)held ? (uint32_t)guess - 1u : held;
          while (j > 1 && !((double)(above + (u64)(j - 1) * w1) < goal)) --j;
          while (j < held && (double)(above + (u64)j * w1) < goal) ++j;
          c.ties = j;
        }
        return c;
      }
    }
    return in;
  };

  Cut cut{0u, 0u};  // every key is above 0 (-inf has key 0x007FFFFF)
  const int k = a.top_k ? a.top_k[row] : 0;
  if (k > 0 && k < vocab) cut = select(false, (uint32_t)k, 0.0, cut);
  const float p = a.top_p ? a.top_p[row] : 1.0f;
  if (p < 1.0f) {
    // total weight of what is kept so far
    u64 sum = 0, total;
    for (int i = tid; i < vocab; i += kThreads) {
      const float v = logit_at(x, i);
      if (order_key(v) > cut.key) sum += fixed(real_weight(v));
    }
    block_scan(sum, red, total);
    if (cut.ties) total += cut.ties * fixed(real_weight(logit_of_key(cut.key)));
    const double goal = (double)p * (double)total;
    cut = goal > 0.0 ? select(true, 0, goal, cut) : Cut{top_key, 1u};
  }

  // Draw: weights and ties of index ranges, the range that holds the goal, then the token in it
  const int per = ((vocab + kSegments - 1) / kSegments + 63) / 64 * 64;  // tokens of a range: whole waves
  const int segments = (vocab + per - 1) / per;
  u64* seg_w = hist;
  uint32_t* seg_n = count;
  const int wave = tid >> 6, lane = tid & 63;
  auto kept_weight = [&](float v) {
    const double w = real_weight(v);
    return w >= least ? fixed(w) : 0ull;
  };
  __syncthreads();
  for (int s = wave; s < segments; s += kThreads / 64) {
    u64 w = 0;
    uint32_t n = 0;
    for (int i = s * per + lane; i < min(vocab, (s + 1) * per); i += 64) {
      const float v = logit_at(x, i);
      const uint32_t key = order_key(v);
      if (key > cut.key) w += kept_weight(v);
      if (key == cut.key) ++n;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      w += __shfl_xor(w, off, 64);
      n += __shfl_xor(n, off, 64);
    }
    if (lane == 0) seg_w[s] = w, seg_n[s] = n;
  }
  __syncthreads();
  const u64 tie_w = cut.ties ? kept_weight(logit_of_key(cut.key)) : 0ull;
  const u64 n_mine = tid < segments ? seg_n[tid] : 0u;
  u64 n_all, total;
  const u64 n_before = block_scan(n_mine, red, n_all);
  const u64 ties_mine = n_before >= cut.ties ? 0ull : min(n_mine, (u64)cut.ties - n_before);
  const u64 w_mine = tid < segments ? seg_w[tid] + ties_mine * tie_w : 0ull;
  const u64 w_before = block_scan(w_mine, red, total);
  const float uf = a.uniforms[row];
  const double u = uf > 0.0f ? (double)fminf(uf, 1.0f) : 0.0;
  const double goal = u * (double)total;
  // the first token whose running sum exceeds goal; where rounding leaves none, the last one kept
  if (tid == 0) pick_bucket = 0u;
  __syncthreads();
  if (w_mine && !((double)w_before > goal)) atomicMax(&pick_bucket, (uint32_t)tid);
  __syncthreads();
  if ((uint32_t)tid == pick_bucket) pick_above = w_before, pick_count_above = (uint32_t)n_before;
  __syncthreads();
  if (wave != 0) return;
  const int s = pick_bucket;
  u64 run = pick_above;
  uint32_t seen = pick_count_above;
  int token = 0;
  for (int i0 = s * per; i0 < min(vocab, (s + 1) * per); i0 += 64) {
    const int i = i0 + lane;
    const float v = i < vocab ? logit_at(x, i) : 0.0f;
    const uint32_t key = i < vocab ? order_key(v) : 0u;
    const bool tie = i < vocab && key == cut.key;
    const u64 ties = __ballot(tie);
    const uint32_t rank = seen + __popcll(ties & ((1ull << lane) - 1ull));
    u64 w = key > cut.key ? kept_weight(v) : 0ull;
    if (tie && rank < cut.ties) w = tie_w;
    u64 inc = w;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const u64 o = __shfl_up(inc, off, 64);
      if (lane >= off) inc += o;
    }
    const u64 past = __ballot(w && (double)(run + inc) > goal), some = __ballot(w != 0);
    if (some) token = i0 + 63 - __clzll(some);
    if (past) {
      token = i0 + __ffsll((unsigned long long)past) - 1;
      break;
    }
    run += __shfl(inc, 63, 64);
    seen += __popcll(ties);
  }
  if (lane == 0) a.token_ids[row] = token;
}

}  // namespace

size_t sample_workspace_bytes(int, int) { return 0; }

void launch_sample(const SampleArgs& a, void*, hipStream_t st) {
  // weights of up to 2^24 tokens sum to less than 2^62
  int bits = 0;
  while ((1 << bits) < a.vocab) ++bits;
  const double unit = (double)(1ull << (62 - bits));
  if (a.type == QWEN_TYPE_F32)
    hipLaunchKernelGGL(sample_kernel<float>, dim3(a.rows), dim3(kThreads), 0, st, a, unit);
  else
    hipLaunchKernelGGL(sample_kernel<uint16_t>, dim3(a.rows), dim3(kThreads), 0, st, a, unit);
}

}  // namespace qwen

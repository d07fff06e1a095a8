// K/V cache in 8 bits: store, load and the attention over it (code and layout: include/qwen_hip_kv8.h).
//
// The codes are exact in fp16, so the matrix cores take them as fp16 operands and the scales, powers of two,
// are applied to the products: no rounding beside the code's own.
#include <hip/hip_runtime.h>

#include "kv8_device.hpp"

namespace qwen {

namespace {

// 4 x 4 bytes transposed: byte i of o[j] = byte j of w[i].
__device__ __forceinline__ void transpose4(const uint32_t (&w)[4], uint32_t (&o)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  o[0] = __builtin_amdgcn_perm(c, a, 0x05040100u), o[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  o[2] = __builtin_amdgcn_perm(d, b, 0x05040100u), o[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

__device__ __forceinline__ int code_byte(uint32_t w, int i) { return (int)(int8_t)(w >> (8 * i)); }
__device__ __forceinline__ uint32_t code_of(float x) { return (uint32_t)(int)rintf(x) & 0xFFu; }
// The codes of a dword after their block's scale grew by 1 / ratio.
__device__ __forceinline__ uint32_t regrade(uint32_t w, float ratio) {
  uint32_t o = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) o |= code_of((float)code_byte(w, i) * ratio) << (8 * i);
  return o;
}

// ---- store ----------------------------------------------------------------------------------
// One block of 256 threads per (64-token cache block, head, K or V, sequence): the block's new rows are read once
// into registers, their largest magnitude gives the scale (a maximum of bit patterns: non-finite values come
// out on top), and the codes are written once; V goes through LDS to turn 4 x 4 bytes.  The earlier rows of a
// part-filled block are read only where the scale grows.  Bound by the stream of new rows: 8 x 2048 tokens (bf16, 2 heads
// of 128) 8.5 us for 25 MB, of which the launch takes 3; single tokens (fp32) by the launch and two round trips to memory:
// 4.7 us for one sequence, 5.5 for 64.
// grid = (blocks that `rows` tokens can touch, 2 * kv_heads, batch).
template <class T, int D>
__global__ void __launch_bounds__(256) kv8_store_kernel(qwen_kv8_cache c, qwen_kv8_rows kin, qwen_kv8_rows vin, int rows,
                                                        const int* __restrict__ positions) {
  constexpr int kPer = D / 8;               // threads of a row
  constexpr int kStep = 256 / kPer;         // rows of a pass
  constexpr int kPasses = kKv8Block / kStep;
  __shared__ uint32_t red[4];
  __shared__ uint32_t tile[kKv8Block][D / 4 + 2];
  const int b = blockIdx.z, h = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  const int pos = positions[b];
  if (pos < 0) return;
  const int blk = pos / kKv8Block + (int)blockIdx.x;
  if (blk >= c.blocks) return;
  const long long end = (long long)pos + rows - (long long)blk * kKv8Block;
  if (end <= 0) return;
  const int t0 = blockIdx.x == 0 ? pos % kKv8Block : 0, t1 = end < kKv8Block ? (int)end : kKv8Block;
  const long long first = (long long)blk * kKv8Block - pos;  // row of the block's token 0
  const qwen_kv8_rows in = is_v ? vin : kin;
  const T* src = static_cast<const T*>(in.data) + b * in.seq_stride + h * in.head_stride;
  const int tid = threadIdx.x, d8 = (tid % kPer) * 8;
  float x[kPasses][8];
  uint32_t top = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int t = p * kStep + tid / kPer;
    if (t >= t0 && t < t1) {
      load8(src + (first + t) * in.token_stride + d8, x[p]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, f32_bits(x[p][e]) & 0x7FFFFFFFu);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[p][e] = 0.0f;
    }
  }
  const size_t place = ((size_t)b * c.blocks + blk) * c.kv_heads + h;
  float* scale_at = (is_v ? c.v_scale : c.k_scale) + place;
  const float old = t0 > 0 ? *scale_at : 0.0f;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
  if ((tid & 63) == 0) red[tid >> 6] = top;
  __syncthreads();
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  // 127 = 1.7E0000 (hex mantissa) * 2^6: the exponent of the least power of two, biased by 127
  const int e = max(1, (int)(top >> 23) - ((top & 0x7FFFFFu) > 0x7E0000u ? 5 : 6));
  float s = bits_f32((uint32_t)e << 23);
  if (t0 > 0) s = old > s || old != old ? old : s;
  if (top >= 0x7F800000u) s = f32_nan();
  const bool finite = s == s;
  const float inv = finite ? 1.0f / s : 0.0f;
  const bool grown = t0 > 0 && finite && s != old;
  const float ratio = grown ? old * inv : 1.0f;
  if (tid == 0) *scale_at = s;
  uint2 code[kPasses];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    uint32_t w[2] = {0u, 0u};
    if (finite) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i >> 2] |= code_of(x[p][i] * inv) << (8 * (i & 3));
    }
    code[p] = make_uint2(w[0], w[1]);
  }
  int8_t* dst = (is_v ? c.v : c.k) + place * (size_t)(kKv8Block * D);
  if (!is_v) {
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int t = p * kStep + tid / kPer;
      uint2* at = reinterpret_cast<uint2*>(dst + ((d8 >> 6) * kKv8Block + t) * 64 + (d8 & 63));
      if (t >= t0 && t < t1) {
        *at = code[p];
      } else if (t < t0 && grown) {
        const uint2 w = *at;
        *at = make_uint2(regrade(w.x, ratio), regrade(w.y, ratio));
      }
    }
    return;
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int t = p * kStep + tid / kPer;
    tile[t][d8 / 4] = code[p].x;
    tile[t][d8 / 4 + 1] = code[p].y;
  }
  __syncthreads();
  // thread: dimensions 4 d4 .. + 3, tokens 16 (2 half + u) + 4 g .. + 3 for u = 0, 1 (eight adjacent bytes)
  const int half = tid & 1, g = (tid >> 1) & 3, d4 = tid >> 3;
  if (d4 >= D / 4) return;
  uint32_t o[2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int t = 16 * (2 * half + u) + 4 * g;
    const uint32_t w[4] = {tile[t][d4], tile[t + 1][d4], tile[t + 2][d4], tile[t + 3][d4]};
    transpose4(w, o[u]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t* at = reinterpret_cast<uint32_t*>(dst + (4 * d4 + j) * kKv8Block + 16 * g + 8 * half);
    if (t0 == 0 && t1 == kKv8Block) {
      *reinterpret_cast<uint2*>(at) = make_uint2(o[0][j], o[1][j]);
      continue;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int t = 16 * (2 * half + u) + 4 * g;
      const bool any_new = t < t1 && t + 4 > t0, any_old = t < t0;
      if (!any_new && !(any_old && grown)) continue;
      const uint32_t was = at[u], re = grown ? regrade(was, ratio) : was;
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w |= (t + i < t0 ? re : t + i < t1 ? o[u][j] : was) & (0xFFu << (8 * i));
      at[u] = w;
    }
  }
}

// ---- the model's rows before they are stored ----
// One block per token: 64 rotation pairs (p, p + 64) of each of the 14 q and k heads.
__global__ void __launch_bounds__(256) rope_qk_kernel(float* __restrict__ qkv, int stride, int seq_len,
                                                      const int* __restrict__ positions, const float* __restrict__ rope,
                                                      int limit) {
  const int t = blockIdx.x;
  const long long pos = (long long)positions[t / seq_len] + t % seq_len;
  if (pos < 0 || pos >= limit) return;
  const int p = threadIdx.x & 63;
  const float c = rope[(size_t)pos * 128 + p], s = rope[(size_t)pos * 128 + 64 + p];
  float* row = qkv + (size_t)t * stride;
#pragma unroll
  for (int h = threadIdx.x >> 6; h < QWEN_Q_HEADS + QWEN_KV_HEADS; h += 4) {
    float* x = row + h * QWEN_HEAD_DIM + p;
    const float lo = x[0], hi = x[64];
    x[0] = lo * c - hi * s;
    x[64] = hi * c + lo * s;
  }
}

__global__ void __launch_bounds__(256) fill_i32_kernel(int* __restrict__ p, int n, int value) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = value;
}

// ---- load -----------------------------------------------------------------------------------
// The inverse, one block of 256 threads per (cache block, head, K or V, sequence); bound by the rows written: 4 x 32768
// tokens (fp32, 2 heads of 128) 72 us for 336 MB, 4.7 TB/s where a copy reaches 5.2; with 8-byte stores 80 us, with
// nontemporal ones 76 or 116 from run to run.
// grid = (blocks that `rows` tokens can touch, 2 * kv_heads, batch).
template <class T, int D>
__global__ void __launch_bounds__(256) kv8_load_kernel(qwen_kv8_cache c, qwen_kv8_rows kout, qwen_kv8_rows vout, int rows,
                                                       int zero_outside, const int* __restrict__ positions) {
  constexpr int kVec = 16 / sizeof(T);  // elements of a 16-byte store: a wave writes whole rows at a time
  constexpr int kPer = D / kVec, kStep = 256 / kPer, kPasses = kKv8Block / kStep;
  __shared__ uint32_t tile[kKv8Block][D / 4 + 2];
  const int b = blockIdx.z, h = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  const int pos = positions[b];
  const long long blk = (long long)(pos >> 6) + blockIdx.x;  // rounds down for negative positions too
  const bool inside = blk >= 0 && blk < c.blocks;
  if (!inside && !zero_outside) return;
  const long long first = blk * kKv8Block - pos, last = first + kKv8Block;  // rows of the block's tokens
  if (first >= rows) return;
  const int t0 = first < 0 ? (int)-first : 0, t1 = last > rows ? (int)(rows - first) : kKv8Block;
  const qwen_kv8_rows out = is_v ? vout : kout;
  T* dst = static_cast<T*>(out.data) + b * out.seq_stride + h * out.head_stride;
  const int tid = threadIdx.x, d0 = (tid % kPer) * kVec;
  const size_t place = inside ? ((size_t)b * c.blocks + (size_t)blk) * c.kv_heads + h : 0;
  const int8_t* src = (is_v ? c.v : c.k) + place * (size_t)(kKv8Block * D);
  const float s = inside ? (is_v ? c.v_scale : c.k_scale)[place] : 0.0f;
  if (is_v && inside) {
    const int half = tid & 1, g = (tid >> 1) & 3, d4 = tid >> 3;
    if (d4 < D / 4) {
      uint2 in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        in[j] = *reinterpret_cast<const uint2*>(src + (4 * d4 + j) * kKv8Block + 16 * g + 8 * half);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = 16 * (2 * half + u) + 4 * g;
        const uint32_t w[4] = {u ? in[0].y : in[0].x, u ? in[1].y : in[1].x, u ? in[2].y : in[2].x, u ? in[3].y : in[3].x};
        uint32_t o[4];
        transpose4(w, o);
#pragma unroll
        for (int i = 0; i < 4; ++i) tile[t + i][d4] = o[i];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int t = p * kStep + tid / kPer;
    if (t < t0 || t >= t1) continue;
    uint32_t w[kVec / 4] = {};
    if (inside) {
      const int8_t* at = src + ((d0 >> 6) * kKv8Block + t) * 64 + (d0 & 63);
#pragma unroll
      for (int i = 0; i < kVec / 4; ++i) w[i] = is_v ? tile[t][d0 / 4 + i] : reinterpret_cast<const uint32_t*>(at)[i];
    }
    T* to = dst + (first + t) * out.token_stride + d0;
    if constexpr (kVec == 8) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (float)code_byte(w[i >> 2], i & 3) * s;
      store8(to, x);
    } else {
      store4(to, f32x4{(float)code_byte(w[0], 0), (float)code_byte(w[0], 1), (float)code_byte(w[0], 2), (float)code_byte(w[0], 3)} * s);
    }
  }
}

// ---- attention ------------------------------------------------------------------------------
// The value of the lane whose column differs by 8 (row_ror:8).
__device__ __forceinline__ float other_half(float x) {
  return bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_bits(x), 0x128, 0xF, 0xF, false));
}

// Maximum over the four lanes of a column (16 apart).
__device__ __forceinline__ float column_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(f32_bits(x), f32_bits(x), false, false);
  x = fmaxf(bits_f32(a[0]), bits_f32(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
  return fmaxf(bits_f32(b[0]), bits_f32(b[1]));
}

// 16 bytes of the cache that nothing else reads (64 x 4096 fp32: 26.0 us, with cached loads 25.3 to 28.7).
__device__ __forceinline__ uint4 load_once(const int8_t* p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
  return make_uint4(x[0], x[1], x[2], x[3]);
}

// Attention of CT tiles of 16 query columns over one split of the keys.  Per wave and 64-token block:
//   S^T = K Q^T (16x16x32 fp16, A = the codes of 16 tokens as they lie in the cache, B = query columns), so a lane
//   holds the scores of one column for tokens 16t + 4g + i: exactly the k slots of the B operand of
//   O^T += V P^T, whose A operand is again 16 contiguous cache bytes a lane.  Scores and probabilities never leave
//   their lane; K and V go from HBM to the matrix cores through registers alone, with the next block's loads in
//   flight.  Running maximum and sum per column; the waves of a block take its cache blocks in turn and are
//   joined in LDS.
// fp32 queries take two columns each (hi and lo fp16 terms, 8 apart), whose scores are added across lanes; the
// columns then carry the hi and lo terms of the probabilities.
// Bound by HBM: 64 sequences of 4096 tokens (fp32, 12 / 2 heads of 128) 25.1 us, of which 135 MB take 18 at 7.4 TB/s
// and the rest is ramp, join and the last blocks; one sequence of 578 tokens 8.6 us, latency alone.
// grid = (nsplit * tile groups, kv_heads, batch), block = 256 (with 512 threads, eight waves a block: 64 x 4096 1 us
// more, one sequence of 578 tokens 0.2 us more).
template <class T, int D, int CT>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) kv8_attn_kernel(Kv8AttnArgs a) {
  constexpr bool kTwo = std::is_same<T, float>::value;
  constexpr int NW = 4;  // waves
  constexpr int kRowsPerTile = kTwo ? 8 : 16, kHalves = D / 64, kDimTiles = D / 16;
  __shared__ float2 ml[NW][CT * 16];
  __shared__ f32x4 join[NW][CT][kDimTiles][64];
  const int split = blockIdx.x % a.nsplit, groups = gridDim.x / a.nsplit;
  const int tg = groups - 1 - (int)(blockIdx.x / a.nsplit);  // the longest rows first
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int R = a.rows * a.group, row0 = tg * CT * kRowsPerTile;
  const int pos = a.positions[b];
  const size_t block_bytes = (size_t)kKv8Block * D, head0 = (size_t)b * a.c.blocks * a.c.kv_heads + kvh;
  uint4 kr[4][kHalves], vr[kDimTiles];
  auto load_k = [&](int blk) {
    const int8_t* p = a.c.k + (head0 + (size_t)blk * a.c.kv_heads) * block_bytes + col * 64 + 16 * g;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int s = 0; s < kHalves; ++s) kr[t][s] = load_once(p + (s * kKv8Block + 16 * t) * 64);
  };
  auto load_v = [&](int blk) {
    const int8_t* p = a.c.v + (head0 + (size_t)blk * a.c.kv_heads) * block_bytes + col * 64 + 16 * g;
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) vr[dt] = load_once(p + dt * 16 * kKv8Block);
  };
  // the wave's first block is in flight before the sequence's length is known (a block of the cache in any case)
  int blk = split * a.per_split + wave;
  float sk, sv;
  {
    const int first = min(blk, a.c.blocks - 1);
    load_k(first);
    load_v(first);
    sk = a.c.k_scale[head0 + (size_t)first * a.c.kv_heads];
    sv = a.c.v_scale[head0 + (size_t)first * a.c.kv_heads];
  }
  // keys that the first and the last row of the tile group attend
  const int i_last = min(R - 1, row0 + CT * kRowsPerTile - 1) / a.group;
  auto visible = [&](int i) { return pos < 0 ? 0 : (int)min((long long)pos + i + 1, (long long)a.max_keys); };
  const int kmin = visible(row0 / a.group), kmax = visible(i_last);
  const int nblk = (kmax + kKv8Block - 1) / kKv8Block;
  const int blk0 = split * a.per_split, blk1 = min(nblk, blk0 + a.per_split);
  if (blk0 >= blk1 && a.nsplit > 1) return;  // the merge knows the live splits

  // Query columns
  half8 q[CT][2 * kHalves];
  float factor[CT], m[CT], l[CT];
  int keys[CT];
  f32x4 o[CT][kDimTiles];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int row = row0 + ct * kRowsPerTile + (kTwo ? col & 7 : col);
    const bool live = row < R;
    const int i = live ? row / a.group : 0, h = kvh * a.group + (live ? row % a.group : 0);
    const T* src = static_cast<const T*>(a.q.data) + b * a.q.seq_stride + (long long)i * a.q.token_stride +
                   (long long)h * a.q.head_stride;
    keys[ct] = live ? visible(i) : 0;
    float x[2 * kHalves][8];
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < 2 * kHalves; ++s) {
      load8(src + 64 * (s >> 1) + 16 * g + 8 * (s & 1), x[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, f32_bits(x[s][e]) & 0x7FFFFFFFu);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    // times a power of two that brings the row's largest magnitude to [2^13, 2^14), and the scale's sign
    const int ex = min(253, max(13, 267 - (int)(top >> 23)));
    const float up = bits_f32(((uint32_t)ex << 23) | (f32_bits(a.scale_log2e) & 0x80000000u));
    factor[ct] = top >= 0x7F800000u ? f32_nan() : fabsf(a.scale_log2e) * bits_f32((uint32_t)(254 - ex) << 23);
#pragma unroll
    for (int s = 0; s < 2 * kHalves; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = x[s][e] * up;
        const _Float16 hi = (_Float16)y;
        q[ct][s][e] = kTwo && col >= 8 ? (_Float16)(y - (float)hi) : hi;
      }
    m[ct] = -__builtin_inff();
    l[ct] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) o[ct][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const float low_term = kTwo && col >= 8 ? 1.0f : 0.0f;
  for (; blk < blk1; blk += NW) {
    const int next = min(blk + NW, blk1 - 1);  // past the end: a block of the split again (not used)
    f32x4 s[CT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int u = 0; u < kHalves; ++u) {
        const half8 k0 = codes_to_half(kr[t][u].x, kr[t][u].y), k1 = codes_to_half(kr[t][u].z, kr[t][u].w);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[ct][2 * u], s[ct][t], 0, 0, 0);
          s[ct][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[ct][2 * u + 1], s[ct][t], 0, 0, 0);
        }
      }
    }
    load_k(next);
    const float sk_next = a.c.k_scale[head0 + (size_t)next * a.c.kv_heads];
    const bool edge = (blk + 1) * kKv8Block > kmin;
    half8 p[CT][2];
    float sv_col[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      if constexpr (kTwo)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[ct][t][i] += other_half(s[ct][t][i]);
      if (edge)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (blk * kKv8Block + 16 * t + 4 * g + i >= keys[ct]) s[ct][t][i] = -__builtin_inff();
      float top = s[ct][0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[ct][e >> 2][e & 3]);
      top = column_max(top);
      // a column that attends none of the block's tokens takes nothing from it, whatever its scales hold
      const bool none = top == -__builtin_inff();
      float f = factor[ct] * sk;
      f = none || f < 1.0e-37f ? 1.0e-37f : f;  // (a scale of 0 times a masked -inf would be NaN)
      sv_col[ct] = none ? 0.0f : sv;
      top *= f;
      // the accumulators follow the maximum only once it is more than 2^4 ahead
      if (!__all(top <= m[ct] + kProbLag && m[ct] > -__builtin_inff())) {
        const bool up = top > m[ct] + kProbLag || (m[ct] == -__builtin_inff() && top > m[ct]);
        const float mn = up ? top : m[ct], alpha = up ? __builtin_amdgcn_exp2f(m[ct] - mn) : 1.0f;
        l[ct] *= alpha;
#pragma unroll
        for (int dt = 0; dt < kDimTiles; ++dt) o[ct][dt] *= alpha;
        m[ct] = mn;
      }
      const float base = m[ct] == -__builtin_inff() ? 0.0f : m[ct] - kProbBits;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        f32x2 x = {__builtin_amdgcn_exp2f(fmaf(s[ct][e >> 2][e & 3], f, -base)),
                   __builtin_amdgcn_exp2f(fmaf(s[ct][e >> 2][(e & 3) + 1], f, -base))};
        l[ct] += x[0];
        l[ct] += x[1];
        if constexpr (kTwo) {  // columns from 8 on: what the others' rounding leaves
          const half2v hi = __builtin_convertvector(x, half2v);
          x[0] = fmaf(-(float)hi[0], low_term, x[0]);
          x[1] = fmaf(-(float)hi[1], low_term, x[1]);
        }
        const half2v y = __builtin_convertvector(x, half2v);
        p[ct][e >> 3][e & 7] = y[0];
        p[ct][e >> 3][(e & 7) + 1] = y[1];
      }
    }
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) {
      const half8 v0 = codes_to_half(vr[dt].x, vr[dt].y), v1 = codes_to_half(vr[dt].z, vr[dt].w);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[ct][0], d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[ct][1], d, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[ct][dt][i] = fmaf(d[i], sv_col[ct], o[ct][dt][i]);
      }
    }
    load_v(next);
    sv = a.c.v_scale[head0 + (size_t)next * a.c.kv_heads];
    sk = sk_next;
  }

  // Join the waves: every wave leaves its accumulators in LDS, and each thread adds up four dimensions of a column
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16, 64);
    l[ct] += __shfl_xor(l[ct], 32, 64);
    if (g == 0) ml[wave][ct * 16 + col] = make_float2(m[ct], l[ct]);
#pragma unroll
    for (int dt = 0; dt < kDimTiles; ++dt) join[wave][ct][dt][lane] = o[ct][dt];
  }
  __syncthreads();
  // item: (column tile, row, dimension tile, quarter of it)
  constexpr int kItems = CT * kRowsPerTile * kDimTiles * 4;
  for (int item = threadIdx.x; item < kItems; item += 64 * NW) {
    const int c = item % kRowsPerTile, q4 = item / kRowsPerTile % 4, dt = item / kRowsPerTile / 4 % kDimTiles,
              ct = item / kRowsPerTile / 4 / kDimTiles;
    const int row = row0 + ct * kRowsPerTile + c;
    if (row >= R) continue;
    float mm = -__builtin_inff(), total = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, ml[w][ct * 16 + c].x);
    f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 v = ml[w][ct * 16 + c];
      // (a wave without keys: maximum -inf and sum 0; a sum of NaN stays one)
      const float f = v.x == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(v.x - mm);
      total += v.y * f;
      y += join[w][ct][dt][16 * q4 + c] * f;
      if constexpr (kTwo) y += join[w][ct][dt][16 * q4 + c + 8] * f;
    }
    const int dim = 16 * dt + 4 * q4;
    if (nblk > a.per_split) {  // (else the only live split)
      const size_t at = (((size_t)b * a.c.kv_heads + kvh) * R + row) * a.nsplit + split;
      if (dim == 0) a.pml[at] = make_float2(mm, total);
      store4(a.part + at * D + dim, y);
    } else {
      T* dst = static_cast<T*>(a.out.data) + b * a.out.seq_stride + (long long)(row / a.group) * a.out.token_stride +
               (long long)(kvh * a.group + row % a.group) * a.out.head_stride;
      store4(dst + dim, y * (total == 0.0f ? 0.0f : 1.0f / total));
    }
  }
}

// Joins the key splits of a query row: D / 4 lanes hold four dimensions each.  With many splits a block has one row
// and divides the splits over its lane groups; with few it has a row per lane group (12 rows of 125 splits: 4.7 us and 16;
// 3600 rows of 12 splits: 7.2 and 5.2).
constexpr int kMergeWide = 16;
// A row whose tile has one live split is in the output already.  64 x 4096 of 12 heads, two splits each: 4.2 us, most of
// it the launch.
// grid = (rows * group / rows of a block, kv_heads, batch), block = 256.
template <class T, int D, bool kMany>
__global__ void __launch_bounds__(256) kv8_merge_kernel(Kv8AttnArgs a) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const int row = kMany ? blockIdx.x : blockIdx.x * kGroups + grp, kvh = blockIdx.y, b = blockIdx.z, R = a.rows * a.group;
  if (!kMany && row >= R) return;
  const int pos = a.positions[b];
  // live splits: those of the row's tile group, as the kernel before counts them
  const int i_last = min(R - 1, row / a.tile_rows * a.tile_rows + a.tile_rows - 1) / a.group;
  const int kmax = pos < 0 ? 0 : (int)min((long long)pos + i_last + 1, (long long)a.max_keys);
  const int live = ((kmax + kKv8Block - 1) / kKv8Block + a.per_split - 1) / a.per_split;
  if (live == 1) return;  // already in the output
  const size_t at = (((size_t)b * a.c.kv_heads + kvh) * R + row) * a.nsplit;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.part + at * D) + lane;
  float m = -__builtin_inff(), sum = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = kMany ? grp : 0; s < live; s += kMany ? kGroups : 1) {
    const float2 v = a.pml[at + s];
    const f32x4 x = part[(size_t)s * kLanes];
    // (a split without keys for this row: maximum -inf, sum 0; a sum of NaN stays one)
    const float mn = fmaxf(m, v.x), f0 = m == mn ? 1.0f : exp2f(m - mn), f1 = v.x == mn || v.x == -__builtin_inff() ? 1.0f : exp2f(v.x - mn);
    sum = sum * f0 + v.y * f1;
    o = o * f0 + x * f1;
    m = mn;
  }
  if constexpr (kMany) {
    __shared__ float2 ml[kGroups];
    __shared__ f32x4 os[kGroups][kLanes];
    if (lane == 0) ml[grp] = make_float2(m, sum);
    os[grp][lane] = o;
    __syncthreads();
    if (grp != 0) return;
    float mm = m;
    for (int g = 1; g < kGroups; ++g) mm = fmaxf(mm, ml[g].x);
    sum = 0.0f;
    o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float2 v = ml[g];
      const float f = v.x == -__builtin_inff() ? 1.0f : exp2f(v.x - mm);
      sum += v.y * f;
      o += os[g][lane] * f;
    }
  }
  T* dst = static_cast<T*>(a.out.data) + b * a.out.seq_stride + (long long)(row / a.group) * a.out.token_stride +
           (long long)(kvh * a.group + row % a.group) * a.out.head_stride + 4 * lane;
  store4(dst, o * (sum == 0.0f ? 0.0f : 1.0f / sum));
}

template <class T, int D>
void run_attn(const Kv8AttnArgs& a, const Kv8AttnPlan& p, int batch, hipStream_t st) {
  const dim3 grid(a.nsplit * p.groups, a.c.kv_heads, batch);
  if (p.large)
    launch_kv8_attention_tiles(a, std::is_same<T, float>::value ? QWEN_TYPE_F32 : QWEN_TYPE_BF16, batch, p.groups, p.one_key_group, st);
  else if (p.tiles == 1)
    hipLaunchKernelGGL((kv8_attn_kernel<T, D, 1>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((kv8_attn_kernel<T, D, 2>), grid, dim3(256), 0, st, a);
  const int R = a.rows * a.group, per_block = 1024 / D;
  if (a.nsplit > kMergeWide)
    hipLaunchKernelGGL((kv8_merge_kernel<T, D, true>), dim3(R, a.c.kv_heads, batch), dim3(256), 0, st, a);
  else if (a.nsplit > 1)
    hipLaunchKernelGGL((kv8_merge_kernel<T, D, false>), dim3((R + per_block - 1) / per_block, a.c.kv_heads, batch), dim3(256), 0, st, a);
}

template <class F>
void by_type(int type, int head_dim, F&& f) {
  if (type == QWEN_TYPE_F32) {
    if (head_dim == 64)
      f(float{}, std::integral_constant<int, 64>{});
    else
      f(float{}, std::integral_constant<int, 128>{});
  } else {
    if (head_dim == 64)
      f(Bf16{}, std::integral_constant<int, 64>{});
    else
      f(Bf16{}, std::integral_constant<int, 128>{});
  }
}

}  // namespace

void launch_kv8_store(const qwen_kv8_cache& c, int type, const qwen_kv8_rows& k, const qwen_kv8_rows& v, int batch,
                      int rows, const int* positions, hipStream_t st) {
  const int touched = (rows + kKv8Block - 2) / kKv8Block + 1;
  by_type(type, c.head_dim, [&](auto t, auto d) {
    hipLaunchKernelGGL((kv8_store_kernel<decltype(t), decltype(d)::value>), dim3(touched, 2 * c.kv_heads, batch),
                       dim3(256), 0, st, c, k, v, rows, positions);
  });
}

void launch_kv8_load(const qwen_kv8_cache& c, int type, const qwen_kv8_rows& k, const qwen_kv8_rows& v, int batch,
                     int rows, bool zero_outside, const int* positions, hipStream_t st) {
  const int touched = (rows + kKv8Block - 2) / kKv8Block + 1;
  by_type(type, c.head_dim, [&](auto t, auto d) {
    hipLaunchKernelGGL((kv8_load_kernel<decltype(t), decltype(d)::value>), dim3(touched, 2 * c.kv_heads, batch),
                       dim3(256), 0, st, c, k, v, rows, (int)zero_outside, positions);
  });
}

void launch_rope_qk(float* qkv, int stride, int tokens, int seq_len, const int* positions, const float* rope, int limit,
                    hipStream_t st) {
  hipLaunchKernelGGL(rope_qk_kernel, dim3(tokens), dim3(256), 0, st, qkv, stride, seq_len, positions, rope, limit);
}

void launch_fill_i32(int* p, int n, int value, hipStream_t st) {
  hipLaunchKernelGGL(fill_i32_kernel, dim3((n + 255) / 256), dim3(256), 0, st, p, n, value);
}

// Rows and keys over the workgroups; bf16 in parentheses where both types were timed (12 / 2 heads of 128 unless stated).
// - Up to four tiles of 16 columns go to the kernel that reads the cache into registers, two of them a workgroup, more to
//   the kernel of large tiles: 64 sequences of 4000 tokens with 5 fp32 rows (four tiles) 47 us, as a large tile 68; with 6
//   rows (five) 81 and 70.
// - Few rows: keys split to one workgroup a CU or a few more (twice as many: 64 sequences of 4096 tokens the same, 16 of 8000
//   10 % more, 100 of 50 to 3000 tokens 10 % less), in equal parts (100 sequences of 3000 tokens 31 us; in one part of 40
//   blocks and one of 7, 41) of whole turns of the four waves.  A sequence of up to 12 blocks is not split: three blocks
//   a wave cost less than the second launch.
// - Large tiles: keys split so that the workgroups come to one a CU at most, two blocks or more each (512 rows after 32000
//   tokens of one sequence: 203 us (129); one a CU or a little more, which leaves some CUs two: 242 (158)).
// - Several key groups a workgroup where each workgroup has a CU to itself and 12 blocks or more (28 / 4 heads of 64, 204
//   tiles of 19 blocks: 30 us (24), one key group 34 (27)), or up to two a CU and 24 blocks (384 tiles of 64 blocks: 124 us
//   (80), 155 (107); 264 of 22: 67 (50), 62 (45)); else one (384 tiles of 8 blocks: several 37 us (33), one 31 (22); 768 of
//   64: 229 (152), 206 (140)).
Kv8AttnPlan plan_kv8_attention(const qwen_kv8_cache& c, int type, int q_heads, int batch, int rows, int max_keys) {
  constexpr int kCus = 256;
  const bool two = type == QWEN_TYPE_F32;
  const long long R = (long long)rows * (q_heads / c.kv_heads);
  const long long per_tile = two ? 8 : 16, tiles = (R + per_tile - 1) / per_tile;
  Kv8AttnPlan p{};
  p.large = tiles > 4;
  p.tiles = tiles > 1 ? 2 : 1;
  p.tile_rows = p.large ? kKv8TileRows : (int)(p.tiles * per_tile);
  p.groups = (int)((R + p.tile_rows - 1) / p.tile_rows);
  const long long blocks = (max_keys + kKv8Block - 1) / kKv8Block;
  const long long others = (long long)p.groups * c.kv_heads * batch;
  long long per;
  if (p.large) {
    const long long splits = others < kCus ? kCus / others : 1;
    per = (blocks + splits - 1) / splits;
    if (per < 2) per = 2;
  } else {
    per = (blocks * others + kCus - 1) / kCus;
    if (per < 4) per = blocks <= 12 ? blocks : 4;
    const long long splits = (blocks + per - 1) / per;
    per = ((blocks + splits - 1) / splits + 3) / 4 * 4;
  }
  const long long least = (blocks + kKv8MaxSplits - 1) / kKv8MaxSplits;
  if (per < least) per = least;
  p.per_split = (int)per;
  p.nsplit = (int)((blocks + per - 1) / per);
  const long long workgroups = others * p.nsplit;
  p.one_key_group = per < 12 || workgroups >= 2 * kCus || (per < 24 && workgroups > kCus);
  if (p.nsplit > 1)
    p.workspace = (size_t)batch * q_heads * rows * p.nsplit * (size_t)(c.head_dim + 2) * sizeof(float);
  return p;
}

void launch_kv8_attention(const qwen_kv8_cache& c, int type, const qwen_kv8_rows& q, const qwen_kv8_rows& out, int q_heads,
                          int batch, int rows, const int* positions, int max_keys, float scale, const Kv8AttnPlan& p,
                          void* workspace, hipStream_t st) {
  Kv8AttnArgs a{};
  a.c = c;
  a.q = q;
  a.out = out;
  a.positions = positions;
  a.group = q_heads / c.kv_heads;
  a.rows = rows;
  a.max_keys = max_keys;
  a.scale_log2e = scale * 1.44269504088896340736f;
  a.nsplit = p.nsplit;
  a.per_split = p.per_split;
  a.tile_rows = p.tile_rows;
  a.part = static_cast<float*>(workspace);
  a.pml = reinterpret_cast<float2*>(a.part + (size_t)batch * q_heads * rows * p.nsplit * c.head_dim);
  by_type(type, c.head_dim, [&](auto t, auto d) { run_attn<decltype(t), decltype(d)::value>(a, p, batch, st); });
}

}  // namespace qwen

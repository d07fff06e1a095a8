// Attention of many query rows (prompts, chunks) over the 8-bit K/V cache: tiles of 128 rows.
//
// kv8_attn_kernel feeds each wave its own cache blocks from HBM and converts their codes for 32 columns at most; here the
// work is bound by the softmax's vector instructions and the LDS reads of the products, so the codes of a 64-token cache
// block are converted once for the whole tile and shared through LDS.  Four waves of 32 columns are a key group
// (S^T = K Q^T and O^T += V P^T, 32x32x16 fp16; a lane holds one column and half of the block's tokens).
//
// One key group a workgroup (KG = 1), 256 registers a wave and so two workgroups a CU, which drift half a turn apart by
// themselves: while one has the matrix cores, the other has the vector instructions.  Four causal prompts of 4096
// tokens (12 / 2 heads of 128, bf16): 253 us = 815 TFLOP/s, 74 % of a large library product's rate here; with three
// key groups 287.  fp32: 390 us, 530.
// Where the tiles of a call are too few for that and each has many blocks, its longest tile decides: then two or three key
// groups of a workgroup (KG) take the blocks in turn, kept a part of a turn apart by barriers, and are joined at the
// end.  One such prompt: 83 us, with KG = 1 96 to 108 (also as two splits, or as tiles of 64 rows with two key groups
// of two waves: 98).
//
// Counters at four prompts: vector instructions issue in 54 % of the SIMDs' cycles, the matrix cores are busy in 35 %, LDS
// instructions issue in 10 %: the two waves of a SIMD hide little of each other.  One wave that interleaves the scores of
// its next block with its probabilities, and its products with the conversion (two buffers a tile, one barrier a block):
// 272 us instead of 253.
// fp32 rows enter as hi and lo fp16 terms in two products each, as their probabilities do.
#include "kv8_device.hpp"

namespace qwen {

typedef float f32x16 __attribute__((ext_vector_type(16)));

namespace {

constexpr int kTileFold = 6;  // V scales down to 2^-6 of the accumulator's unit go into the probabilities

__device__ __forceinline__ float swap_max(float x) {  // maximum over the two lanes of a column
  const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
  return fmaxf(bits_f32(r[0]), bits_f32(r[1]));
}
__device__ __forceinline__ float swap_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(f32_bits(x), f32_bits(x), false, false);
  return bits_f32(r[0]) + bits_f32(r[1]);
}

// grid = (kv_heads * batch, tiles, nsplit), block = 256 * KG.  Blocks start in the order of their number: the tiles with the
// longest rows of all heads and sequences first.  Heads rotate from one row of the grid to the next, or those of a long
// sequence would all come to the same XCD.
template <class T, int D, int KG>
__global__ void __launch_bounds__(256 * KG) __attribute__((amdgpu_waves_per_eu(KG == 1 ? 2 : KG))) kv8_attn_tile_kernel(Kv8AttnArgs a) {
  constexpr bool kTwo = std::is_same<T, float>::value;
  constexpr int kLimbs = kTwo ? 2 : 1;
  constexpr int kSteps = D / 16, kDims = D / 32, kChunks = D / 8;
  constexpr int kLoads = D / 64;  // 16-byte pieces of K, and pairs of half of them of V, that a thread stages
  __shared__ uint4 kbuf[KG][kKv8Block * kChunks];  // [key group][token][16-byte chunk ^ swizzle]
  __shared__ uint4 vbuf[KG][D * 8];                // [key group][dimension][chunk ^ swizzle]
  // Query operands: in registers where there is room, else in LDS (the same for all key groups)
  constexpr bool kQInLds = kLimbs * kSteps > (KG == 1 ? 16 : 4);
  __shared__ uint4 qbuf[kQInLds ? 4 * kLimbs * kSteps * 64 : 1];  // [column group][term][k step][lane]
  __shared__ float2 ml[KG > 1 ? KG - 1 : 1][kKv8TileRows];  // of the key groups after the first
  __shared__ int unit_of[KG > 1 ? KG - 1 : 1][kKv8TileRows];

  const int tiles = gridDim.y, split = blockIdx.z, tile = tiles - 1 - (int)blockIdx.y;
  const int head = (blockIdx.x + blockIdx.y + blockIdx.z) % gridDim.x, kvh = head % a.c.kv_heads, b = head / a.c.kv_heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), cg = wave & 3, kg = wave >> 2;
  const int col = lane & 31, hh = lane >> 5;
  const int R = a.rows * a.group, row0 = tile * kKv8TileRows;
  const int pos = a.positions[b];
  auto visible = [&](int i) { return pos < 0 ? 0 : (int)min((long long)pos + i + 1, (long long)a.max_keys); };
  const int kmin = visible(row0 / a.group), kmax = visible(min(R - 1, row0 + kKv8TileRows - 1) / a.group);
  const int nblk = (kmax + kKv8Block - 1) / kKv8Block;
  const int blk0 = split * a.per_split, blk1 = min(nblk, blk0 + a.per_split);
  if (blk0 >= blk1 && a.nsplit > 1) return;  // the merge knows the live splits
  const bool parts = nblk > a.per_split;      // more than one: results to be merged
  const int turns = (max(0, blk1 - blk0) + KG - 1) / KG;  // each key group takes every KG-th block
  const int full = min(blk1, kmin / kKv8Block);       // blocks before it need no mask

  // The wave's query columns: B operands, lane (col, hh) has dimensions 16 s + 8 hh + e
  half8 q[kQInLds ? 1 : kLimbs][kQInLds ? 1 : kSteps];
  uint4* const q_at = qbuf + (cg * kLimbs * kSteps) * 64 + lane;
  float factor, m = -__builtin_inff(), l = 0.0f;
  int unit = 127;  // biased exponent of the column's accumulator unit (a V scale)
  f32x16 o[kDims];
  const int row = row0 + cg * 32 + col;
  const bool live = row < R;
  const int qi = live ? row / a.group : 0, qh = kvh * a.group + (live ? row % a.group : 0);
  const int keys = live ? visible(qi) : 0;
  {
    const T* src = static_cast<const T*>(a.q.data) + b * a.q.seq_stride + (long long)qi * a.q.token_stride +
                   (long long)qh * a.q.head_stride;
    uint32_t top = 0;
    float x[kSteps][8];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      load8(src + 16 * s + 8 * hh, x[s]);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, f32_bits(x[s][e]) & 0x7FFFFFFFu);
    }
    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
    // times a power of two that brings the row's largest magnitude to [2^13, 2^14), and the scale's sign
    const int ex = min(253, max(13, 267 - (int)(top >> 23)));
    const float up = bits_f32(((uint32_t)ex << 23) | (f32_bits(a.scale_log2e) & 0x80000000u));
    factor = top >= 0x7F800000u ? f32_nan() : fabsf(a.scale_log2e) * bits_f32((uint32_t)(254 - ex) << 23);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      half8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = x[s][e] * up;
        hi[e] = (_Float16)y;
        lo[e] = (_Float16)(y - (float)hi[e]);
      }
      if constexpr (kQInLds) {
        if (kg == 0) {
          __builtin_memcpy(q_at + s * 64, &hi, 16);
          if constexpr (kTwo) __builtin_memcpy(q_at + (kSteps + s) * 64, &lo, 16);
        }
      } else {
        q[0][s] = hi;
        if constexpr (kTwo) q[kLimbs - 1][s] = lo;
      }
    }
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  }

  const size_t block_bytes = (size_t)kKv8Block * D, head0 = (size_t)b * a.c.blocks * a.c.kv_heads + kvh;
  const int st = (wave & 3) * 64 + lane;  // thread of the key group
  auto place = [&](int turn) { return head0 + (size_t)min(blk0 + KG * turn + kg, blk1 - 1) * a.c.kv_heads; };
  uint4 kreg[kLoads], vreg[kLoads];
  auto load_k = [&](int turn) {
    const uint4* p = reinterpret_cast<const uint4*>(a.c.k + place(turn) * block_bytes);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) kreg[n] = p[st + 256 * n];
  };
  // thread: dimension st / 2, pieces st % 2 and st % 2 + 2 of it
  auto load_v = [&](int turn) {
    const int8_t* p = a.c.v + place(turn) * block_bytes;
    if constexpr (D == 128) {
      const uint4* at = reinterpret_cast<const uint4*>(p) + (st >> 1) * 4 + (st & 1);
      vreg[0] = at[0];
      vreg[1] = at[2];
    } else {  // dimension st / 4, pieces (st / 2) % 2 and + 2, eight bytes of each
      const uint2* at = reinterpret_cast<const uint2*>(p) + (st >> 2) * 8 + ((st >> 1) & 1) * 2 + (st & 1);
      const uint2 x = at[0], y = at[4];
      vreg[0] = make_uint4(x.x, x.y, y.x, y.y);
    }
  };
  // A row of K has kChunks chunks of 8 dimensions, one of V 8 chunks of 8 tokens (those of one k step and lane half);
  // a chunk's place is its number ^ a function of the row, so that 16 lanes of a read touch 16 different ones.
  // All places of a lane are then one offset ^ a constant (+ a constant); the offsets are made opaque where they are
  // used, or the compiler keeps every one of them in a register of its own and spills.
  constexpr int kRowBytes = D * 2;
  auto opaque = [](uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  char* const k_at = reinterpret_cast<char*>(kbuf[kg]);
  char* const v_at = reinterpret_cast<char*>(vbuf[kg]);
  auto k_swizzle = [](int t) { return D == 128 ? t & 15 : (t >> 1) & 7; };
  const uint32_t k_read = col * kRowBytes + ((hh ^ k_swizzle(col)) << 4), v_read = col * 128 + ((hh ^ ((col >> 1) & 7)) << 4);
  const int wt = st >> 2, wd = D == 128 ? st >> 1 : st >> 2;  // the token of K and the dimension of V it stages
  const uint32_t k_write = wt * kRowBytes + ((((st & 3) * 2) ^ k_swizzle(wt)) << 4);
  const uint32_t v_write = wd * 128 + (((D == 128 ? st & 1 : ((st >> 1) & 1) + (st & 1) * 4) ^ ((wd >> 1) & 7)) << 4);
  auto put = [](char* to, uint32_t lo, uint32_t hi) {
    const half8 h = codes_to_half(lo, hi);
    __builtin_memcpy(__builtin_assume_aligned(to, 16), &h, 16);
  };
  auto write_k = [&]() {
    const uint32_t at = opaque(k_write);
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {  // piece n: the n-th 64 dimensions
      put(k_at + (at ^ (n << 7)), kreg[n].x, kreg[n].y);
      put(k_at + (at ^ (n << 7) ^ 16), kreg[n].z, kreg[n].w);
    }
  };
  auto write_v = [&]() {
    const uint32_t at = opaque(v_write);
    if constexpr (D == 128) {
      put(v_at + at, vreg[0].x, vreg[1].x);
      put(v_at + (at ^ 32), vreg[0].y, vreg[1].y);
      put(v_at + (at ^ 64), vreg[0].z, vreg[1].z);
      put(v_at + (at ^ 96), vreg[0].w, vreg[1].w);
    } else {
      put(v_at + at, vreg[0].x, vreg[0].z);
      put(v_at + (at ^ 32), vreg[0].y, vreg[0].w);
    }
  };
  auto operand = [](const char* from) {
    half8 h;
    __builtin_memcpy(&h, __builtin_assume_aligned(from, 16), 16);
    return h;
  };
  f32x16 s[2];            // scores of the block's 64 tokens
  half8 p[kLimbs][4];     // their probabilities, by k step
  // The products read their LDS operands a few steps ahead; the order is pinned, since the compiler on its own waits for
  // each operand right before its product (the LDS latency 40 times a block).
  constexpr int kSchedMfma = 0x8, kSchedRead = 0x100;
  auto scores = [&]() {
    constexpr int kAhead = 3 < kSteps ? 3 : kSteps, kReads = 2 + (kQInLds ? kLimbs : 0);
    const uint32_t at = opaque(k_read);
    __builtin_amdgcn_sched_barrier(0);
    half8 x[kSteps][2], y[kSteps][kLimbs];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
#pragma unroll
      for (int b2 = 0; b2 < kLimbs; ++b2)
        if constexpr (kQInLds)
          y[k][b2] = operand(reinterpret_cast<const char*>(q_at + (b2 * kSteps + k) * 64));
        else
          y[k][b2] = q[b2][k];
#pragma unroll
      for (int t = 0; t < 2; ++t) x[k][t] = operand(k_at + (at ^ (k << 5)) + t * 32 * kRowBytes);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int b2 = 0; b2 < kLimbs; ++b2)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[k][t], y[k][b2], s[t], 0, 0, 0);
    __builtin_amdgcn_sched_group_barrier(kSchedRead, kAhead * kReads, 0);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2 * kLimbs, 0);
      if (k + kAhead < kSteps) __builtin_amdgcn_sched_group_barrier(kSchedRead, kReads, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto weigh = [&]() {
    const uint32_t at = opaque(v_read);
    __builtin_amdgcn_sched_barrier(0);
    half8 x[4][kDims];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int d = 0; d < kDims; ++d) x[u][d] = operand(v_at + (at ^ (u << 5)) + d * 32 * 128);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int b2 = 0; b2 < kLimbs; ++b2)
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[u][d], p[b2][u], o[d], 0, 0, 0);
    __builtin_amdgcn_sched_group_barrier(kSchedRead, 2 * kDims, 0);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, kDims * kLimbs, 0);
      if (u < 2) __builtin_amdgcn_sched_group_barrier(kSchedRead, kDims, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // Softmax of the block whose scores are in s.  First what its probabilities are relative to, and the accumulators made
  // ready for them; then the probabilities of each half of its tokens into p.
  float f = 0.0f, base = 0.0f, sum = 0.0f;
  int shift = 0;
  bool drop = false;
  auto mask = [&](int key0) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (key0 + 32 * t + 8 * (i >> 2) + 4 * hh + (i & 3) >= keys) s[t][i] = -__builtin_inff();
  };
  auto settle = [&](float sk, int sv) {
    f = factor * sk;
    f = f < 1.0e-37f ? 1.0e-37f : f;  // (a scale of 0 times a masked -inf would be NaN)
    float top[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      top[t] = fmaxf(s[t][0], s[t][1]);
#pragma unroll
      for (int i = 2; i < 16; i += 2) top[t] = fmaxf(fmaxf(top[t], s[t][i]), s[t][i + 1]);
    }
    float most = swap_max(fmaxf(top[0], top[1]));
    // a column that sees none of the tokens takes nothing from them, whatever their scales hold
    f = most == -__builtin_inff() ? 1.0e-37f : f;
    most *= f;
    sum = 0.0f;
    // the block's V scale is folded into the probabilities where it is a little below the accumulator's unit
    shift = unit - sv;
    base = m - kProbBits + (float)shift;
    drop = false;
    const bool usual = most <= m + kProbLag && m > -__builtin_inff() && (uint32_t)shift <= (uint32_t)kTileFold;
    if (__all(usual)) return;
    const bool first = m == -__builtin_inff(), up = most > m + kProbLag || (first && most > m);
    const float mn = up ? most : m;
    const float alpha = up ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
    // else the unit changes to it, unless none of its probabilities is large enough to be more than 0, or its values are
    // below 2^-80 of what the accumulators may hold (a block of zeros: its scale is the least one, or 0): those
    // count in the sum alone
    const bool touched = most > mn - (kProbBits + 25.0f);
    const float lead = (float)shift + (up && !first ? m - mn : 0.0f);
    const bool change = touched && (first || ((uint32_t)shift > (uint32_t)kTileFold && lead <= 80.0f));
    const float grow = change && !first ? __builtin_amdgcn_exp2f(lead) : alpha;
    drop = touched && !change && shift > kTileFold;
    unit = change ? sv : unit;
    shift = change || drop ? 0 : shift < 0 ? 400 : shift;
    base = mn == -__builtin_inff() ? 0.0f : mn - kProbBits + (float)shift;
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < kDims; ++d) o[d] *= grow;
  };
  auto probabilities = [&](auto half) {
    constexpr int t = decltype(half)::value;
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const f32x2 x = {__builtin_amdgcn_exp2f(fmaf(s[t][i], f, -base)), __builtin_amdgcn_exp2f(fmaf(s[t][i + 1], f, -base))};
      const half2v hi = __builtin_convertvector(x, half2v);
      p[0][2 * t + (i >> 3)][i & 7] = hi[0];
      p[0][2 * t + (i >> 3)][(i & 7) + 1] = hi[1];
      if constexpr (kTwo) {
        const f32x2 r = {x[0] - (float)hi[0], x[1] - (float)hi[1]};
        const half2v lo = __builtin_convertvector(r, half2v);
        p[1][2 * t + (i >> 3)][i & 7] = lo[0];
        p[1][2 * t + (i >> 3)][(i & 7) + 1] = lo[1];
        sum += x[0];
        sum += x[1];
      } else {
        sum = __builtin_amdgcn_fdot2(hi, half2v{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
      }
    }
  };

  if (turns > 0) {
    load_k(0);
    write_k();
    float sk = a.c.k_scale[place(0)], svf = a.c.v_scale[place(0)];
    __syncthreads();
    // Key group kg runs kg ticks behind.  A barrier counts the waves that arrive, wherever in the code: every wave
    // comes to max(2, KG) * turns + KG of them.
    auto tick = []() {  // (nothing moves across: the work of a tick is balanced)
      __builtin_amdgcn_sched_barrier(0);
      __syncthreads();
      __builtin_amdgcn_sched_barrier(0);
    };
    for (int i = 0; i < kg; ++i) tick();
    for (int it = 0; it < turns; ++it) {
      scores();
      tick();
      const int blk = blk0 + KG * it + kg;
      const int key0 = blk < blk1 ? blk * kKv8Block : 0x7FFFFF00;  // (past the end: no token is seen)
      if (svf != svf) sk = svf;  // a NaN scale of V shows through the sum, and only in columns that see the block
      const int sv = svf != svf ? unit : (int)(f32_bits(svf) >> 23) & 255;
      load_v(it);
      load_k(it + 1);
      if (blk >= full) mask(key0);
      settle(sk, sv);
      probabilities(std::integral_constant<int, 0>{});
      if constexpr (KG > 2) tick();
      probabilities(std::integral_constant<int, 1>{});
      l += __builtin_amdgcn_ldexpf(sum, shift);
      write_v();
      write_k();
      sk = a.c.k_scale[place(it + 1)];
      svf = a.c.v_scale[place(it + 1)];
      if (__any(drop))
#pragma unroll
        for (int b2 = 0; b2 < kLimbs; ++b2)
#pragma unroll
          for (int u = 0; u < 4; ++u) p[b2][u] = drop ? half8{} : p[b2][u];
      tick();
      weigh();
    }
    for (int i = kg; i < KG; ++i) tick();
  }

  // Join the key groups in LDS, one after the other, and write; accumulators in true units from here on
  f32x4* parked = reinterpret_cast<f32x4*>(kbuf);  // half of the dimensions at a time: [column group][..][quarter][lane]
  constexpr int kPart = kDims / 2;
  static_assert(KG == 1 || sizeof(kbuf) >= sizeof(f32x4) * 4 * kPart * 4 * 64, "the join fits the K buffers");
  l = swap_sum(l);
  if (kg > 0 && hh == 0) ml[kg - 1][cg * 32 + col] = make_float2(m, l), unit_of[kg - 1][cg * 32 + col] = unit;
  __syncthreads();
  // (a group without keys: maximum -inf, sum 0; a sum of NaN stays one)
  float mm = m, sum_all = 0.0f;
  if (kg == 0) {
    for (int g = 0; g < KG - 1; ++g) mm = fmaxf(mm, ml[g][cg * 32 + col].x);
    const float f0 = m == -__builtin_inff() ? 1.0f : exp2f(m - mm);
    sum_all = l * f0;
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = __builtin_amdgcn_ldexpf(o[d][i] * f0, unit - 127);
  }
#pragma unroll
  for (int g = 1; g < KG; ++g)
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      if (kg == g)
#pragma unroll
        for (int d = 0; d < kPart; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const f32x16& x = o[part * kPart + d];
            parked[((cg * kPart + d) * 4 + w) * 64 + lane] = f32x4{x[4 * w], x[4 * w + 1], x[4 * w + 2], x[4 * w + 3]};
          }
      __syncthreads();
      if (kg == 0) {
        const float2 other = ml[g - 1][cg * 32 + col];
        const int u = unit_of[g - 1][cg * 32 + col] - 127;
        const float f1 = other.x == -__builtin_inff() ? 1.0f : exp2f(other.x - mm);
        if (part == 0) sum_all += other.y * f1;
#pragma unroll
        for (int d = 0; d < kPart; ++d)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const f32x4 y = parked[((cg * kPart + d) * 4 + w) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[part * kPart + d][4 * w + e] += __builtin_amdgcn_ldexpf(y[e] * f1, u);
          }
      }
      __syncthreads();
    }
  if (kg != 0 || !live) return;
  const size_t at = (((size_t)b * a.c.kv_heads + kvh) * R + row) * a.nsplit + split;
  T* dst = static_cast<T*>(a.out.data) + b * a.out.seq_stride + (long long)qi * a.out.token_stride +
           (long long)qh * a.out.head_stride;
  if (parts && hh == 0) a.pml[at] = make_float2(mm, sum_all);
  const float inv = parts ? 1.0f : sum_all == 0.0f ? 0.0f : 1.0f / sum_all;
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 z = f32x4{o[d][4 * w], o[d][4 * w + 1], o[d][4 * w + 2], o[d][4 * w + 3]} * inv;
      const int dim = 32 * d + 8 * w + 4 * hh;
      if (parts)
        store4(a.part + at * D + dim, z);
      else
        store4(dst + dim, z);
    }
}

}  // namespace

void launch_kv8_attention_tiles(const Kv8AttnArgs& a, int type, int batch, int groups, bool one_key_group, hipStream_t st) {
  const dim3 grid(a.c.kv_heads * batch, groups, a.nsplit);
  auto run = [&](auto t, auto d, auto groups_of_keys) {
    constexpr int KG = decltype(groups_of_keys)::value;
    hipLaunchKernelGGL((kv8_attn_tile_kernel<decltype(t), decltype(d)::value, KG>), grid, dim3(256 * KG), 0, st, a);
  };
  using One = std::integral_constant<int, 1>;
  auto by_keys = [&](auto t, auto d) {
    // three key groups, two where the fp32 queries' LDS leaves no room for more
    using Some = std::integral_constant<int, std::is_same<decltype(t), float>::value && decltype(d)::value == 128 ? 2 : 3>;
    if (one_key_group)
      run(t, d, One{});
    else
      run(t, d, Some{});
  };
  auto by_dim = [&](auto t) {
    if (a.c.head_dim == 64)
      by_keys(t, std::integral_constant<int, 64>{});
    else
      by_keys(t, std::integral_constant<int, 128>{});
  };
  if (type == QWEN_TYPE_F32)
    by_dim(float{});
  else
    by_dim(Bf16{});
}

}  // namespace qwen

// What the kernels of the 8-bit K/V cache share (kernels_fast_kv8.hip, kernels_fast_kv8_tile.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "kernels.hpp"
#include "qwen_device_math.hpp"

namespace qwen {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Probabilities enter the products times 2^11 relative to a maximum that may lag the true one by a factor of 2^4 (so that
// the accumulators are rescaled rarely): up to 2^15, and normal in fp16 down to 2^-25 of the largest.
constexpr float kProbBits = 11.0f, kProbLag = 4.0f;

struct Bf16 {  // storage of a bf16 element
  uint16_t bits;
};

__device__ __forceinline__ float f32_nan() { return bits_f32(0x7FC00000u); }

// Eight consecutive elements of a 16-byte aligned row.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
__device__ __forceinline__ void load8(const Bf16* p, float (&x)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = bits_f32(w[i] << 16), x[2 * i + 1] = bits_f32(w[i] & 0xFFFF0000u);
}
// Round to nearest even; NaN stays a quiet NaN.
__device__ __forceinline__ uint32_t bf16_of(float x) {
  const uint32_t b = f32_bits(x);
  return (b & 0x7FFFFFFFu) > 0x7F800000u ? 0x7FC0u : (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(Bf16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = bf16_of(x[2 * i]) | (bf16_of(x[2 * i + 1]) << 16);
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store4(float* p, const f32x4& x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void store4(Bf16* p, const f32x4& x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(bf16_of(x[0]) | (bf16_of(x[1]) << 16), bf16_of(x[2]) | (bf16_of(x[3]) << 16));
}

struct Kv8AttnArgs {
  qwen_kv8_cache c;
  qwen_kv8_rows q, out;
  const int* positions;
  int group, rows, max_keys;
  float scale_log2e;
  int nsplit, per_split;  // key splits of `per_split` blocks
  int tile_rows;          // query rows of a block
  float* part;            // [batch][kv_heads][rows * group][nsplit][D], nsplit > 1
  float2* pml;            // [batch][kv_heads][rows * group][nsplit]
};

// Eight codes as fp16: 0x64uu is 1024 + uu, uu = code + 128.
__device__ __forceinline__ half8 codes_to_half(uint32_t lo, uint32_t hi) {
  const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
  const uint32_t w[4] = {
      __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u),
      __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)};
  half8 r;
  __builtin_memcpy(&r, w, 16);
  return r - (_Float16)1152.0f;
}

// Attention by tiles of many rows (kernels_fast_kv8_tile.hip): rows of a block, and the launch without a merge.
constexpr int kKv8TileRows = 128;
void launch_kv8_attention_tiles(const Kv8AttnArgs& a, int type, int batch, int groups, bool one_key_group, hipStream_t st);

}  // namespace qwen

// Entry points of the 8-bit K/V cache (include/qwen_hip_kv8.h): argument checks before the launches.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <exception>
#include <string>

#include "kernels.hpp"
#include "qwen_hip_kv8.h"
#include "runtime.hpp"

using namespace qwen;

namespace {

constexpr int kMaxBatch = 65535;       // grid z
constexpr int kMaxRows = 1 << 24;      // tokens of a call: grids and row counts stay within 32 bits
constexpr int kMaxHeads = 1024;
constexpr int kMaxGroup = 64;
constexpr int64_t kMaxQueryRows = 1 << 22, kMaxHeadRows = 1 << 22;  // of the attention: its grids
constexpr int64_t kMaxStride = int64_t(1) << 40;

int bad(const char* why) {
  set_last_error(why);
  return QWEN_ERR_KERNEL;
}

template <class Fn>
int guarded_kv8(Fn&& fn) {
  try {
    return fn();
  } catch (const HipError& e) {
    set_last_error(std::string(e.what) + ": " + hipGetErrorString(e.code));
  } catch (const std::exception& e) {
    set_last_error(e.what());
  }
  if (std::getenv("QWEN_HIP_VERBOSE")) std::fprintf(stderr, "qwen-mi355x: %s\n", last_error_cstr());
  return QWEN_ERR_DEVICE;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

const char* cache_problem(const qwen_kv8_cache* c, int type) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return "null cache";
  if (type != QWEN_TYPE_F32 && type != QWEN_TYPE_BF16) return "unknown element type";
  if (c->head_dim != 64 && c->head_dim != 128) return "head_dim of an 8-bit cache must be 64 or 128";
  if (c->kv_heads < 1 || c->kv_heads > kMaxHeads) return "kv_heads of an 8-bit cache must be 1 .. 1024";
  if (c->sequences < 1 || c->blocks < 1 || c->blocks > (1 << 24)) return "invalid 8-bit cache size";
  if (!aligned16(c->k) || !aligned16(c->v)) return "the codes of an 8-bit cache must be 16-byte aligned";
  if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3u)
    return "the scales of an 8-bit cache must be 4-byte aligned";
  return nullptr;
}

const char* call_problem(const qwen_kv8_cache* c, int batch, int rows, const int* positions) {
  if (!positions) return "null positions";
  if (batch < 1 || batch > c->sequences || batch > kMaxBatch) return "batch must be 1 .. the cache's sequences (65535 at most)";
  if (rows < 1 || rows > kMaxRows) return "rows must be 1 .. 2^24";
  return nullptr;
}

// Rows [batch][rows][heads][dim]: alignment, strides, and (written) no two rows at the same place.
const char* rows_problem(const qwen_kv8_rows* r, int type, int batch, int rows, int heads, int dim, bool written) {
  if (!r || !r->data) return "null rows";
  const int64_t size = type == QWEN_TYPE_F32 ? 4 : 2;
  struct Axis {
    int64_t stride;
    int n;
  } ax[3] = {{r->seq_stride, batch}, {r->token_stride, rows}, {r->head_stride, heads}};
  if (!aligned16(r->data)) return "rows must be 16-byte aligned";
  for (const Axis& a : ax) {
    if (a.n > 1 && (a.stride < 0 || a.stride > kMaxStride)) return "row strides must be 0 .. 2^40 elements";
    if (a.n > 1 && a.stride * size % 16 != 0) return "row strides must be multiples of 16 bytes";
  }
  if (!written) return nullptr;
  for (int i = 0; i < 2; ++i)  // axes by stride
    for (int j = 0; j < 2 - i; ++j)
      if (ax[j].n > 1 && (ax[j + 1].n <= 1 || ax[j].stride > ax[j + 1].stride)) std::swap(ax[j], ax[j + 1]);
  int64_t extent = dim;  // elements that the inner axes span
  for (const Axis& a : ax) {
    if (a.n <= 1) continue;
    if (a.stride < extent) return "rows that are written must not overlap";
    extent += a.stride * (a.n - 1);
  }
  return nullptr;
}

}  // namespace

extern "C" {

int qwen_hip_kv8_store(const qwen_kv8_cache* cache, int type, const qwen_kv8_rows* k, const qwen_kv8_rows* v, int batch,
                       int rows, const int* positions, void* stream) {
  if (const char* why = cache_problem(cache, type)) return bad(why);
  if (const char* why = call_problem(cache, batch, rows, positions)) return bad(why);
  for (const qwen_kv8_rows* r : {k, v})
    if (const char* why = rows_problem(r, type, batch, rows, cache->kv_heads, cache->head_dim, false)) return bad(why);
  return guarded_kv8([&]() -> int {
    launch_kv8_store(*cache, type, *k, *v, batch, rows, positions, static_cast<hipStream_t>(stream));
    QWEN_HIP(hipGetLastError());
    return QWEN_OK;
  });
}

int qwen_hip_kv8_load(const qwen_kv8_cache* cache, int type, const qwen_kv8_rows* k, const qwen_kv8_rows* v, int batch,
                      int rows, int flags, const int* positions, void* stream) {
  if (const char* why = cache_problem(cache, type)) return bad(why);
  if (const char* why = call_problem(cache, batch, rows, positions)) return bad(why);
  if (flags & ~QWEN_KV8_ZERO_OUTSIDE) return bad("unknown flags of an 8-bit cache load");
  for (const qwen_kv8_rows* r : {k, v})
    if (const char* why = rows_problem(r, type, batch, rows, cache->kv_heads, cache->head_dim, true)) return bad(why);
  return guarded_kv8([&]() -> int {
    launch_kv8_load(*cache, type, *k, *v, batch, rows, (flags & QWEN_KV8_ZERO_OUTSIDE) != 0, positions,
                    static_cast<hipStream_t>(stream));
    QWEN_HIP(hipGetLastError());
    return QWEN_OK;
  });
}

static const char* attention_problem(const qwen_kv8_cache* c, int type, int q_heads, int batch, int rows, int max_keys) {
  if (const char* why = cache_problem(c, type)) return why;
  if (batch < 1 || batch > c->sequences || batch > kMaxBatch) return "batch must be 1 .. the cache's sequences (65535 at most)";
  if (q_heads < 1 || q_heads % c->kv_heads != 0 || q_heads / c->kv_heads > kMaxGroup)
    return "q_heads must be a multiple of kv_heads, at most 64 a KV head";
  if (rows < 1 || rows > kMaxRows) return "rows must be 1 .. 2^24";
  if ((int64_t)rows * (q_heads / c->kv_heads) > kMaxQueryRows) return "rows times query heads a KV head must be at most 2^22";
  if ((int64_t)batch * c->kv_heads > kMaxHeadRows) return "batch times kv_heads must be at most 2^22";
  if (max_keys < 1 || max_keys > (int64_t)c->blocks * QWEN_KV8_BLOCK) return "max_keys must be 1 .. 64 * blocks";
  return nullptr;
}

int qwen_hip_kv8_attention_workspace(const qwen_kv8_cache* cache, int type, int q_heads, int batch, int rows,
                                     int max_keys, uint64_t* bytes) {
  if (!bytes) return bad("null size");
  if (const char* why = attention_problem(cache, type, q_heads, batch, rows, max_keys)) return bad(why);
  *bytes = plan_kv8_attention(*cache, type, q_heads, batch, rows, max_keys).workspace;
  return QWEN_OK;
}

int qwen_hip_kv8_attention(const qwen_kv8_cache* cache, int type, const qwen_kv8_rows* q, const qwen_kv8_rows* out,
                           int q_heads, int batch, int rows, const int* positions, int max_keys, float scale,
                           void* workspace, uint64_t workspace_bytes, void* stream) {
  if (const char* why = attention_problem(cache, type, q_heads, batch, rows, max_keys)) return bad(why);
  if (!positions) return bad("null positions");
  if (!std::isfinite(scale * 1.44269504088896340736f)) return bad("the attention's scale must be finite (times log2 e too)");
  if (const char* why = rows_problem(q, type, batch, rows, q_heads, cache->head_dim, false)) return bad(why);
  if (const char* why = rows_problem(out, type, batch, rows, q_heads, cache->head_dim, true)) return bad(why);
  const Kv8AttnPlan plan = plan_kv8_attention(*cache, type, q_heads, batch, rows, max_keys);
  if (plan.workspace > workspace_bytes || (plan.workspace && (!workspace || !aligned16(workspace))))
    return bad("the attention's workspace is too small or not 16-byte aligned");
  return guarded_kv8([&]() -> int {
    launch_kv8_attention(*cache, type, *q, *out, q_heads, batch, rows, positions, max_keys, scale, plan, workspace,
                         static_cast<hipStream_t>(stream));
    QWEN_HIP(hipGetLastError());
    return QWEN_OK;
  });
}

}  // extern "C"

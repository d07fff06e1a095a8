// Entry points of token sampling (include/qwen_hip_sample.h): argument checks before the launch.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <exception>
#include <string>

#include "kernels.hpp"
#include "qwen_hip_sample.h"
#include "runtime.hpp"

using namespace qwen;

namespace {

int bad(const char* why) {
  set_last_error(why);
  return QWEN_ERR_KERNEL;
}

const char* size_problem(int rows, int vocab) {
  if (rows < 1 || rows > 65535) return "sampling takes 1 .. 65535 rows";  // (grid y)
  if (vocab < 1 || vocab > kSampleMaxVocab) return "sampling takes 1 .. 2^24 tokens";
  return nullptr;
}

}  // namespace

extern "C" {

int qwen_hip_sample_workspace(int rows, int vocab, uint64_t* bytes) {
  if (!bytes) return bad("null size");
  if (const char* why = size_problem(rows, vocab)) return bad(why);
  *bytes = sample_workspace_bytes(rows, vocab);
  return QWEN_OK;
}

int qwen_hip_sample(const void* logits, int type, int64_t row_stride, int rows, int vocab, const float* uniforms,
                    const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                    int* token_ids, void* workspace, uint64_t workspace_bytes, void* stream) {
  if (const char* why = size_problem(rows, vocab)) return bad(why);
  if (type != QWEN_TYPE_F32 && type != QWEN_TYPE_BF16) return bad("unknown element type");
  if (!logits || !uniforms || !token_ids) return bad("null sampling argument");
  if (rows > 1 && (row_stride < 0 || row_stride > (int64_t(1) << 40))) return bad("the logits' row stride must be 0 .. 2^40");
  const uintptr_t size = type == QWEN_TYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size) return bad("logits must be aligned to their type");
  const size_t need = sample_workspace_bytes(rows, vocab);
  if (need > workspace_bytes || (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u))))
    return bad("the sampling workspace is too small or not 16-byte aligned");
  try {
    launch_sample(SampleArgs{logits, type, row_stride, rows, vocab, uniforms, temperature, top_k, top_p, min_p, token_ids},
                  workspace, static_cast<hipStream_t>(stream));
    QWEN_HIP(hipGetLastError());
    return QWEN_OK;
  } catch (const HipError& e) {
    set_last_error(std::string(e.what) + ": " + hipGetErrorString(e.code));
  } catch (const std::exception& e) {
    set_last_error(e.what());
  }
  if (std::getenv("QWEN_HIP_VERBOSE")) std::fprintf(stderr, "qwen-mi355x: %s\n", last_error_cstr());
  return QWEN_ERR_DEVICE;
}

}  // extern "C"

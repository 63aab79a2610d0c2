// Host-visible launch interface of the language-model operators. All pointers
// are device pointers, leading dimensions in elements; sizes and types have
// been checked by the caller (lm_runtime.cpp).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace edsl {
namespace lm {

// EDSL_LM_* of include/edsl_hip_lm.h.
enum Type : int { kF32 = 0, kBf16 = 1, kF16 = 2, kI8 = 3, kE4m3 = 4 };
constexpr int type_bytes(int t) { return t == kF32 ? 4 : t <= kF16 ? 2 : 1; }
constexpr bool is_float_type(int t) { return t >= kF32 && t <= kF16; }

// ------------------------------------------------------------------- norm
struct NormArgs {
  const void* x;
  const void* residual;  // or nullptr
  const void* weight;
  void* total;  // or nullptr
  void* y;
  float* scales;  // 8-bit y only
  float* rstd;    // or nullptr
  int64_t ldx, ldr, ldt, ldy, M, N;
  float eps;
  int type, weight_type, y_type;
};
hipError_t launch_rms_norm(const NormArgs& a, int cus, hipStream_t stream, const char** plan);

struct NormBackwardArgs {
  const void* dy;
  const void* h;
  const void* weight;
  const float* rstd;
  const void* dh;  // or nullptr
  void* dx;
  float* dweight;   // or nullptr
  float* partials;  // [groups][N], where dweight is wanted
  int64_t lddy, ldh, lddh, lddx, M, N;
  int groups;  // workgroups, each with a row of partials
  int type, weight_type;
};
int rms_norm_backward_groups(int64_t M, int64_t N, int type, int cus);
hipError_t launch_rms_norm_backward(const NormBackwardArgs& a, hipStream_t stream);

// -------------------------------------------------------------- log probs
constexpr int kMaxTop = 32;
struct LogprobsArgs {
  const void* x;
  const void* tokens;   // or nullptr
  float* logprobs;      // or nullptr
  float* lse;           // or nullptr
  float* entropy;       // or nullptr
  float* top;           // or nullptr
  void* top_ids;        // with top
  char* partials;       // where a row has more than one chunk
  int64_t ldx, M, V;
  float scale;
  int k;       // 0: no alternatives
  int chunks;  // parts of a row, one workgroup each
  bool many;   // more rows than CUs
  int type;
  bool ids64;
};
int logprobs_chunks(int64_t M, int64_t V, int type, int cus);
size_t logprobs_partial_bytes(int64_t M, int chunks, int k);
hipError_t launch_token_logprobs(const LogprobsArgs& a, hipStream_t stream);

struct LogprobsBackwardArgs {
  const void* x;
  const void* tokens;      // or nullptr
  const float* lse;
  const float* dlogprobs;  // or nullptr
  const float* entropy;    // with dentropy
  const float* dentropy;   // or nullptr
  void* dx;
  int64_t ldx, lddx, M, V;
  float scale;
  int type;
  bool ids64;
};
hipError_t launch_token_logprobs_backward(const LogprobsBackwardArgs& a, hipStream_t stream);

}  // namespace lm
}  // namespace edsl

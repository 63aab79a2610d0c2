// Entry points of include/edsl_hip_lm.h: the checks of their arguments, the
// split of the work over the chip, and the launches.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/edsl_hip_lm.h"
#include "dev_buf.hpp"
#include "lm_kernels.hpp"
#include "runtime_internal.hpp"

namespace edsl {
namespace rt {
namespace {

constexpr int64_t kMostDim = int64_t(1) << 30;
constexpr int64_t kMostVocabulary = int64_t(1) << 21;

void check_sizes(int64_t rows, int64_t cols, const char* rn, const char* cn) {
  if (rows < 0 || cols < 0) fail(kErrShape, "negative dimension");
  if (rows > kMostDim || cols > kMostDim)
    fail(kErrLimit, "dimension beyond 2^30 (%s=%lld %s=%lld)", rn, (long long)rows, cn, (long long)cols);
}

void check_float_type(int type, const char* name) {
  if (!lm::is_float_type(type)) fail(kErrDtype, "%s: type %d is not f32, bf16 or f16", name, type);
}

// A required operand of rows x cols elements (none needed where there are none).
void check_mat(const void* p, int64_t ld, int64_t rows, int64_t cols, const char* name) {
  if (rows > 0 && cols > 0 && !p) fail(kErrArgument, "%s is null", name);
  if (rows > 1 && ld < cols) fail(kErrStride, "%s: row stride %lld < row length %lld", name, (long long)ld, (long long)cols);
}

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

const char* type_name(int t) {
  static const char* const names[] = {"f32", "bf16", "f16", "i8", "e4m3"};
  return names[t];
}

void rms_norm(lm::NormArgs a, void* stream) {
  check_sizes(a.M, a.N, "M", "N");
  check_float_type(a.type, "x");
  if (a.weight_type != a.type && a.weight_type != lm::kF32)
    fail(kErrDtype, "weight: type %d is neither x's nor f32", a.weight_type);
  const bool eight = a.y_type == lm::kI8 || a.y_type == lm::kE4m3;
  if (!eight && a.y_type != a.type) fail(kErrDtype, "y: type %d is neither x's nor of 8 bits", a.y_type);
  if (!(a.eps >= 0.0f) || !std::isfinite(a.eps)) fail(kErrArgument, "eps must be finite and not negative");
  if (eight && a.M > 0 && !a.scales) fail(kErrArgument, "an 8-bit y needs scales");
  if (!eight && a.scales) fail(kErrArgument, "scales are of an 8-bit y");
  if (a.M == 0) return set_plan("empty");
  if (a.N == 0) fail(kErrShape, "rows of no elements have no norm");
  check_mat(a.x, a.ldx, a.M, a.N, "x");
  check_mat(a.weight, a.N, 1, a.N, "weight");
  check_mat(a.y, a.ldy, a.M, a.N, "y");
  if (a.residual) check_mat(a.residual, a.ldr, a.M, a.N, "residual");
  if (a.total) check_mat(a.total, a.ldt, a.M, a.N, "total");
  device_launch(0, stream, [&](char*, int cus) {
    const char* plan = "";
    check_hip(lm::launch_rms_norm(a, cus, as_stream(stream), &plan), "rms_norm launch");
    set_plan("rms_norm %s->%s %s", type_name(a.type), type_name(a.y_type), plan);
  });
}

void rms_norm_backward(lm::NormBackwardArgs a, void* stream) {
  check_sizes(a.M, a.N, "M", "N");
  check_float_type(a.type, "dy");
  if (a.weight_type != a.type && a.weight_type != lm::kF32)
    fail(kErrDtype, "weight: type %d is neither dy's nor f32", a.weight_type);
  if (a.M > 0 && a.N == 0) fail(kErrShape, "rows of no elements have no norm");
  check_mat(a.dy, a.lddy, a.M, a.N, "dy");
  check_mat(a.h, a.ldh, a.M, a.N, "h");
  check_mat(a.dx, a.lddx, a.M, a.N, "dx");
  if (a.dh) check_mat(a.dh, a.lddh, a.M, a.N, "dh");
  if (a.M > 0 && !a.weight) fail(kErrArgument, "weight is null");
  if (a.M > 0 && !a.rstd) fail(kErrArgument, "rstd is null");
  if (a.N == 0 || (a.M == 0 && !a.dweight)) return set_plan("empty");
  int cus = 0;
  device_launch(0, stream, [&](char*, int n) { cus = n; });
  a.groups = lm::rms_norm_backward_groups(a.M, a.N, a.type, cus);
  const size_t bytes = a.dweight ? (size_t)a.groups * a.N * sizeof(float) : 0;
  device_launch(bytes, stream, [&](char* ws, int) {
    a.partials = reinterpret_cast<float*>(ws);
    check_hip(lm::launch_rms_norm_backward(a, as_stream(stream)), "rms_norm_backward launch");
    set_plan("rms_norm_backward %s groups=%d%s", type_name(a.type), a.groups, a.dweight ? " +dweight" : "");
  });
}

void check_logits(int64_t M, int64_t V, int type, float scale) {
  check_sizes(M, V, "M", "V");
  check_float_type(type, "logits");
  if (V > kMostVocabulary) fail(kErrLimit, "V=%lld beyond 2^21", (long long)V);
  if (!(scale > 0.0f) || !std::isfinite(scale)) fail(kErrArgument, "scale must be positive and finite");
  if (M > 0 && V == 0) fail(kErrShape, "rows of no logits have no probabilities");
}

void check_grid(int64_t M, int64_t parts) {
  if (M * parts > 0x7fffffff)
    fail(kErrLimit, "%lld rows of %lld parts are more than one launch takes", (long long)M, (long long)parts);
}

void token_logprobs(lm::LogprobsArgs a, void* stream) {
  check_logits(a.M, a.V, a.type, a.scale);
  if (a.k < 0 || a.k > lm::kMaxTop) fail(kErrLimit, "k=%d is not in 0 .. %d", a.k, lm::kMaxTop);
  if (a.M > 0 && a.k > a.V) fail(kErrShape, "k=%d alternatives of V=%lld", a.k, (long long)a.V);
  if (a.M > 0 && a.k > 0 && (!a.top || !a.top_ids)) fail(kErrArgument, "k alternatives need top_logprobs and top_ids");
  if (a.M > 0 && a.logprobs && !a.tokens) fail(kErrArgument, "logprobs need tokens");
  check_mat(a.x, a.ldx, a.M, a.V, "logits");
  if (a.M == 0 || (a.k == 0 && !a.logprobs && !a.lse && !a.entropy)) return set_plan("empty");
  int cus = 0;
  device_launch(0, stream, [&](char*, int n) { cus = n; });
  a.chunks = lm::logprobs_chunks(a.M, a.V, a.type, cus);
  check_grid(a.M, a.chunks);
  device_launch(lm::logprobs_partial_bytes(a.M, a.chunks, a.k), stream, [&](char* ws, int) {
    a.partials = ws;
    check_hip(lm::launch_token_logprobs(a, as_stream(stream)), "token_logprobs launch");
    set_plan("token_logprobs %s parts=%d top=%d%s", type_name(a.type), a.chunks, a.k, a.chunks > 1 ? " +join" : "");
  });
}

void token_logprobs_backward(lm::LogprobsBackwardArgs a, void* stream) {
  check_logits(a.M, a.V, a.type, a.scale);
  check_mat(a.x, a.ldx, a.M, a.V, "logits");
  check_mat(a.dx, a.lddx, a.M, a.V, "dlogits");
  if (a.M == 0) return set_plan("empty");
  if (!a.lse) fail(kErrArgument, "lse is null");
  if (a.dlogprobs && !a.tokens) fail(kErrArgument, "dlogprobs need tokens");
  if (a.dentropy && !a.entropy) fail(kErrArgument, "dentropy needs entropy");
  check_grid(a.M, (a.V + 4095) / 4096);
  device_launch(0, stream, [&](char*, int) {
    check_hip(lm::launch_token_logprobs_backward(a, as_stream(stream)), "token_logprobs_backward launch");
    set_plan("token_logprobs_backward %s%s", type_name(a.type), a.dentropy ? " +entropy" : "");
  });
}

}  // namespace
}  // namespace rt
}  // namespace edsl

using namespace edsl;

extern "C" {

int edsl_hip_rms_norm_launch(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                             int weight_type, void* total, int64_t ldt, void* y, int64_t ldy, int y_type,
                             float* scales, float* rstd, int64_t M, int64_t N, int type, float eps, void* stream) {
  return rt::guarded([&] {
    lm::NormArgs a{};
    a.x = x, a.residual = residual, a.weight = weight, a.total = total, a.y = y, a.scales = scales, a.rstd = rstd;
    a.ldx = ldx, a.ldr = ldr, a.ldt = ldt, a.ldy = ldy, a.M = M, a.N = N, a.eps = eps;
    a.type = type, a.weight_type = weight_type, a.y_type = y_type;
    rt::rms_norm(a, stream);
  });
}

int edsl_hip_rms_norm_backward_launch(const void* dy, int64_t lddy, const void* h, int64_t ldh, const void* weight,
                                      int weight_type, const float* rstd, const void* dh, int64_t lddh, void* dx,
                                      int64_t lddx, float* dweight, int64_t M, int64_t N, int type, void* stream) {
  return rt::guarded([&] {
    lm::NormBackwardArgs a{};
    a.dy = dy, a.h = h, a.weight = weight, a.rstd = rstd, a.dh = dh, a.dx = dx, a.dweight = dweight;
    a.lddy = lddy, a.ldh = ldh, a.lddh = lddh, a.lddx = lddx, a.M = M, a.N = N;
    a.type = type, a.weight_type = weight_type;
    rt::rms_norm_backward(a, stream);
  });
}

int edsl_hip_token_logprobs_launch(const void* logits, int64_t ldl, int type, const void* tokens, int ids64,
                                   float* logprobs, float* lse, float* entropy, float* top_logprobs, void* top_ids,
                                   int k, int64_t M, int64_t V, float scale, void* stream) {
  return rt::guarded([&] {
    lm::LogprobsArgs a{};
    a.x = logits, a.tokens = tokens, a.logprobs = logprobs, a.lse = lse, a.entropy = entropy, a.top = top_logprobs;
    a.top_ids = top_ids, a.ldx = ldl, a.M = M, a.V = V, a.scale = scale, a.k = k, a.type = type, a.ids64 = ids64 != 0;
    rt::token_logprobs(a, stream);
  });
}

int edsl_hip_token_logprobs_backward_launch(const void* logits, int64_t ldl, int type, const void* tokens, int ids64,
                                            const float* lse, const float* dlogprobs, const float* entropy,
                                            const float* dentropy, void* dlogits, int64_t lddl, int64_t M, int64_t V,
                                            float scale, void* stream) {
  return rt::guarded([&] {
    lm::LogprobsBackwardArgs a{};
    a.x = logits, a.tokens = tokens, a.lse = lse, a.dlogprobs = dlogprobs, a.entropy = entropy, a.dentropy = dentropy;
    a.dx = dlogits, a.ldx = ldl, a.lddx = lddl, a.M = M, a.V = V, a.scale = scale, a.type = type;
    a.ids64 = ids64 != 0;
    rt::token_logprobs_backward(a, stream);
  });
}

}  // extern "C"

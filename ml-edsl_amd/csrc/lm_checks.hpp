// Checks of arguments that the language-model entry points share.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include "lm_kernels.hpp"
#include "runtime_internal.hpp"

namespace edsl {
namespace rt {

constexpr int64_t kMostDim = int64_t(1) << 30;
constexpr int64_t kMostVocabulary = int64_t(1) << 21;

inline void check_sizes(int64_t rows, int64_t cols, const char* rn, const char* cn) {
  if (rows < 0 || cols < 0) fail(kErrShape, "negative dimension");
  if (rows > kMostDim || cols > kMostDim)
    fail(kErrLimit, "dimension beyond 2^30 (%s=%lld %s=%lld)", rn, (long long)rows, cn, (long long)cols);
}

inline void check_float_type(int type, const char* name) {
  if (!lm::is_float_type(type)) fail(kErrDtype, "%s: type %d is not f32, bf16 or f16", name, type);
}

// A required operand of rows x cols elements (none needed where there are none).
inline void check_mat(const void* p, int64_t ld, int64_t rows, int64_t cols, const char* name) {
  if (rows > 0 && cols > 0 && !p) fail(kErrArgument, "%s is null", name);
  if (rows > 1 && ld < cols) fail(kErrStride, "%s: row stride %lld < row length %lld", name, (long long)ld, (long long)cols);
}

inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

inline const char* type_name(int t) {
  static const char* const names[] = {"f32", "bf16", "f16", "i8", "e4m3"};
  return names[t];
}

inline size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

inline void check_grid(int64_t M, int64_t parts) {
  if (M * parts > 0x7fffffff)
    fail(kErrLimit, "%lld rows of %lld parts are more than one launch takes", (long long)M, (long long)parts);
}

inline void check_packed(const void* p, const char* name) {
  if (!p) fail(kErrArgument, "%s is null", name);
  if (reinterpret_cast<uintptr_t>(p) % 256 != 0) fail(kErrArgument, "%s is not 256-byte aligned", name);
}

}  // namespace rt
}  // namespace edsl

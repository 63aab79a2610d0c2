// Entry points of include/edsl_hip_lm.h for the layers on 8-bit weights and on groups
// of rows, and for sampling: the checks of their arguments, the choice of kernels,
// and the launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "../../include/edsl_hip_lm.h"
#include "dev_buf.hpp"
#include "lm_checks.hpp"

namespace edsl {
namespace rt {
namespace {

constexpr int64_t kMostI8Depth = (int64_t(1) << 17) - 1;  // K 2^14 < 2^31: 32-bit sums are exact
constexpr int kMostExperts = 65535;
// The streaming kernels' columns go along one axis of the grid, 512 threads for 16 of them: under 2^32.
constexpr int64_t kMostStreamed = int64_t(1) << 26;

// A tile's rows of `ld` elements within the 31 bits of an asynchronous load's offset.
bool reachable(int64_t rows, int64_t ld, int e) { return rows * ld * e < 0x7fffffff; }
// Whether all of these are multiples of 16.
bool whole16(std::initializer_list<int64_t> values) {
  int64_t all = 0;
  for (const int64_t v : values) all |= v;
  return all % 16 == 0;
}
int64_t address(const void* p) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)); }

void check_epilogue(int epi) {
  if (epi < 0 || epi > 7) fail(kErrArgument, "bad epilogue code %d", epi);
}
void check_bias(int epi, const void* bias) {
  check_epilogue(epi);
  if ((epi & 1) && !bias) fail(kErrArgument, "epilogue adds a bias but bias is null");
}

// ------------------------------------------------------------ 8-bit layer
int64_t i8_bytes(int64_t K, int64_t N) {
  check_sizes(K, N, "K", "N");
  if (K == 0) fail(kErrShape, "K=0: a layer of no inputs");
  if (K > kMostI8Depth) fail(kErrLimit, "K=%lld beyond 2^17 - 1: 32-bit sums would not hold it", (long long)K);
  check_grid((lm::i8_tiles(N) + 3) / 4, lm::i8_blocks(K));
  return lm::i8_scales_at(K, N) + lm::i8_tiles(N) * 16 * (int64_t)sizeof(float);
}

void i8_pack(const lm::I8PackArgs& a, size_t bytes, void* stream) {
  const int64_t need = i8_bytes(a.K, a.N);
  check_float_type(a.scale_type, "scales");
  if (bytes < (size_t)need) fail(kErrArgument, "packed: %zu bytes, %lld are needed", bytes, (long long)need);
  if (a.N == 0) return set_plan("empty");
  check_mat(a.q, a.ldq, a.K, a.N, "q");
  check_mat(a.scales, a.N, 1, a.N, "scales");
  check_packed(a.packed, "packed");
  device_launch(0, stream, [&](char*, int) {
    check_hip(lm::launch_i8_pack(a, as_stream(stream)), "i8_pack launch");
    set_plan("i8_pack");
  });
}

void i8_dense(lm::I8Args a, int64_t M, int64_t N, int64_t K, void* stream) {
  check_sizes(M, N, "M", "N");
  i8_bytes(K, N);
  check_float_type(a.y_type, "Y");
  check_bias(a.epi, a.bias);
  if (a.epi & 1)
    check_float_type(a.bias_type, "bias");
  else
    a.bias = nullptr;
  if (M == 0 || N == 0) return set_plan("empty");
  check_mat(a.x, a.ldx, M, K, "X");
  check_mat(a.y, a.ldy, M, N, "Y");
  check_packed(a.w, "packed");
  if (M <= 1) a.ldx = K;
  a.M = (int)M, a.N = (int)N, a.K = (int)K;
  a.w_scales = reinterpret_cast<const float*>(a.w + lm::i8_scales_at(K, N));
  device_launch(0, stream, [&](char*, int cus) {
    const hipStream_t s = as_stream(stream);
    const int64_t tiles = lm::i8_tiles(N), parts = (M + 63) / 64;
    // Streaming, in parts of up to 64 rows: up to 64 rows (33 x 4096 x 4097 in 12.4 us against 18.3 on tiles), 32 of a layer
    // of more columns than two rounds (64 x 4096 x 16000 in 26 against 17.7; 32 x 4096 x 50256 in 40 against 44), and
    // more rows where all parts together are one round (128 x 8192 x 2048 in 23 against 32; two, 256 rows, in 39 against 32).
    if (N <= kMostStreamed && (M <= (tiles > 2 * (int64_t)cus ? 32 : 64) || (parts <= 64 && parts * tiles <= cus))) {
      // Each workgroup reads all of x: more columns a workgroup where there are many (32 x 4096 x 30000 in 22.8 us on
      // 64 columns, on 32 in 32.4; 1 x 4096 x 30000 in 19.5 and 19.3), and where one more than a round of 16 each would run
      // (33 x 4096 x 4097 in 12.4 us, in 15.8 on 16), but not where CUs would be idle (32 x 4096 x 4096 in 8.4, on 32 in 9.2).
      const int cols = tiles > 4 * (int64_t)cus ? 4 : tiles > (M <= 16 ? 2 : 1) * (int64_t)cus ? 2 : 1;
      const int rows = (int)(((M + parts - 1) / parts + 15) / 16);
      check_hip(lm::launch_i8_skinny(a, rows, cols, s), "i8_skinny launch");
      set_plan("i8_skinny rows=%d cols=%d", 16 * rows, 16 * cols);
      return;
    }
    const bool direct = whole16({address(a.x), a.ldx, K}) && reachable(256, a.ldx, 1);
    check_grid((M + 127) / 128 + 4, (N + 127) / 128 + 4);
    a.cus = cus;
    check_hip(lm::launch_i8_tile(a, direct, s), "i8_tile launch");
    set_plan("i8_tile %s", direct ? "direct" : "any");
  });
}

// --------------------------------------------------- layers on groups of rows
void check_groups(int64_t T, int64_t E, const void* offsets) {
  if (E < 0) fail(kErrShape, "negative number of groups");
  if (E > kMostExperts) fail(kErrLimit, "%lld groups, at most %d", (long long)E, kMostExperts);
  if (T < 0 || T > kMostDim) fail(kErrLimit, "T=%lld is not in 0 .. 2^30", (long long)T);
  if (E > 0 && !offsets) fail(kErrArgument, "offsets is null");
}

// [E][rows][cols], or their transposes where `turned`.
void check_weights(const void* p, int64_t* ld, int64_t* stride, bool turned, int64_t E, int64_t K, int64_t N,
                   const char* name) {
  const int64_t rows = turned ? N : K, cols = turned ? K : N;
  check_mat(p, *ld, rows, cols, name);
  if (rows <= 1) *ld = cols;
  if (E <= 1) *stride = 0;
  if (*stride < 0) fail(kErrStride, "%s: negative stride between groups", name);
}

hipError_t skinny_by_type(const lm::GroupedArgs& a, hipStream_t s) {
  return a.type == lm::kF32    ? lm::launch_grouped_skinny<lm::kF32>(a, s)
         : a.type == lm::kBf16 ? lm::launch_grouped_skinny<lm::kBf16>(a, s)
                               : lm::launch_grouped_skinny<lm::kF16>(a, s);
}
hipError_t rows_by_type(const lm::GroupedArgs& a, bool direct, hipStream_t s) {
  return a.type == lm::kF32    ? lm::launch_grouped_rows<lm::kF32>(a, direct, s)
         : a.type == lm::kBf16 ? lm::launch_grouped_rows<lm::kBf16>(a, direct, s)
                               : lm::launch_grouped_rows<lm::kF16>(a, direct, s);
}
hipError_t weights_by_type(const lm::GroupedWeightArgs& a, bool direct, bool big, hipStream_t s) {
  return a.type == lm::kF32    ? lm::launch_grouped_weights<lm::kF32>(a, direct, big, s)
         : a.type == lm::kBf16 ? lm::launch_grouped_weights<lm::kBf16>(a, direct, big, s)
                               : lm::launch_grouped_weights<lm::kF16>(a, direct, big, s);
}

// y = epi(x @ w_e + b_e), the launches of one product over rows. `plan`: what ran.
void rows_product(lm::GroupedArgs a, int cus, hipStream_t s, char* plan, size_t len) {
  const int e = lm::type_bytes(a.type);
  // Streaming, where no group has more rows than that takes (32 x 4096 x 4096 bf16 in 19 us, on tiles in 32) or most
  // have few (200 rows at 64 of 2048 x 1024 in 56 to 62 us against 59 to 72; 400 rows in 59 to 67 against 60 to 74; 300 at 16 of
  // 2048 x 2048 in 39 against 32 to 38, since groups on both sides of the limit take two launches).
  const bool streams = (a.T <= lm::kGroupedSkinnyRows || a.T < 16 * (int64_t)a.E) && (a.turned || a.N >= 4) &&
                       a.N <= kMostStreamed;
  a.skip = streams ? lm::kGroupedSkinnyRows : 0;
  a.cus = cus;
  if (streams) {
    check_hip(skinny_by_type(a, s), "grouped_skinny launch");
  }
  const char* tiles = "";
  if (a.T > a.skip) {
    const bool direct = whole16({address(a.x), a.ldx * e, address(a.w), a.ldw * e, a.stride_w * e, a.K * e}) &&
                        reachable(256, a.ldx, e) && reachable(256, a.ldw, e);
    check_grid(a.T / 64 + a.E, (a.N + 63) / 64 + 16);
    check_hip(rows_by_type(a, direct, s), "grouped_rows launch");
    tiles = direct ? "+tiles direct" : "+tiles any";
  }
  snprintf(plan, len, "%s%s", streams ? "stream" : "", tiles);
}

void grouped_dense(lm::GroupedArgs a, int64_t E, void* stream) {
  check_groups(a.T, E, a.offsets);
  check_sizes(a.K, a.N, "K", "N");
  check_float_type(a.type, "X");
  check_bias(a.epi, a.bias);
  if (!(a.epi & 1)) a.bias = nullptr;
  if (a.T == 0 || E == 0 || a.N == 0) return set_plan("empty");
  check_mat(a.x, a.ldx, a.T, a.K, "X");
  check_weights(a.w, &a.ldw, &a.stride_w, a.turned, E, a.K, a.N, "W");
  if (a.bias && E > 1 && a.ldbias < a.N && a.ldbias != 0)
    fail(kErrStride, "bias: row stride %lld < row length %lld", (long long)a.ldbias, (long long)a.N);
  check_mat(a.y, a.ldy, a.T, a.N, "Y");
  if (a.T <= 1) a.ldx = a.K;
  a.E = (int)E;
  device_launch(0, stream, [&](char*, int cus) {
    char plan[64];
    rows_product(a, cus, as_stream(stream), plan, sizeof plan);
    set_plan("grouped_dense %s %s", type_name(a.type), plan);
  });
}

struct Backward {
  const void *dy, *x, *w, *offsets, *y;
  void *dx, *dw, *db;
  int64_t lddy, ldx, ldw, stride_w, ldy, lddx, lddw, stride_dw, lddb, T, N, K, E;
  int type, dw_type, db_type, epi;
  float alpha;
  bool ids64, turned, dw_turned;
};

void grouped_backward(Backward a, void* stream) {
  check_groups(a.T, a.E, a.offsets);
  check_sizes(a.K, a.N, "K", "N");
  check_float_type(a.type, "dY");
  check_epilogue(a.epi);
  const int act = (a.epi >> 1) & 3;
  if (act != 0 && a.T > 0 && a.N > 0 && !a.y) fail(kErrArgument, "an activation's gradient needs Y");
  // y > 0 says where z > 0 only so.
  if (act == 2 && !(a.alpha >= 0.0f)) fail(kErrArgument, "the gradient of a leaky epilogue needs alpha >= 0");
  if (a.dw && a.dw_type != a.type && a.dw_type != lm::kF32)
    fail(kErrDtype, "dW: type %d is neither dY's nor f32", a.dw_type);
  if (a.db && a.db_type != a.type && a.db_type != lm::kF32)
    fail(kErrDtype, "db: type %d is neither dY's nor f32", a.db_type);
  if (a.E == 0 || (!a.dx && !a.dw && !a.db)) return set_plan("empty");
  check_mat(a.dy, a.lddy, a.T, a.N, "dY");
  if (act != 0) check_mat(a.y, a.ldy, a.T, a.N, "Y");
  if (a.dx) {
    check_mat(a.dx, a.lddx, a.T, a.K, "dX");
    check_weights(a.w, &a.ldw, &a.stride_w, a.turned, a.E, a.K, a.N, "W");
  }
  if (a.dw) {
    check_mat(a.x, a.ldx, a.T, a.K, "X");
    check_weights(a.dw, &a.lddw, &a.stride_dw, a.dw_turned, a.E, a.K, a.N, "dW");
  }
  if (a.db && a.E > 1 && a.lddb < a.N)
    fail(kErrStride, "db: row stride %lld < row length %lld", (long long)a.lddb, (long long)a.N);
  if (a.N == 0) {
    // dX = 0 for the groups' rows: a product over nothing.
    a.db = nullptr, a.dw = nullptr;
  }
  if (a.T <= 1) a.ldx = a.K, a.lddy = a.N;
  const int e = lm::type_bytes(a.type), chunk = 16 / e;
  const bool masks = act != 0 && a.T > 0 && a.N > 0;
  const int64_t lddz = (a.N + chunk - 1) / chunk * chunk;
  // dW through a slope, in f32 or of f16: of dy's two parts, unrounded. Products with 0, 1 and infinity are what 16 bits
  // hold, and scaling a sum by 0 or infinity is not scaling its terms (0 times an infinite one, infinity times none).
  // f16's steps end at 2^-24: of gradients of 1e-5 times a slope of 0.01 one or two are left, and f16 dW of 256 rows was 7.7 times
  // its own rounding off (1.2 to 1.3 at 1e-4 or a slope of 0.9), 1.00 so; 8192 rows at 8 of 4096 x 4096 take 1045 us, rounded 640.
  // bf16 has the range: dW of the rounded product is 1.00 to 1.21 roundings off (slopes 0.01 to 0.9), in 624 us.
  const bool rounds = act == 2 && a.alpha != 0.0f && a.alpha != 1.0f && std::isfinite(a.alpha);
  const bool split = masks && rounds && a.dw && a.type != lm::kF32 && (a.dw_type == lm::kF32 || a.type == lm::kF16);
  const bool whole = masks && ((a.dx && a.K > 0) || (a.dw && !split));
  const size_t one = masks ? aligned((size_t)a.T * lddz * e) : 0, dz_bytes = one * ((whole ? 1 : 0) + (split ? 2 : 0));
  const size_t sums = a.db ? (size_t)lm::grouped_act_tiles(a.T, (int)a.E) * a.N * sizeof(float) : 0;
  if (masks || a.db) check_grid(a.T / lm::kGroupedActRows + a.E, a.N / 256 + 1);
  device_launch(dz_bytes + sums, stream, [&](char* ws, int cus) {
    const hipStream_t s = as_stream(stream);
    const void *dz = a.dy, *up = nullptr, *down = nullptr;
    int64_t ldz = a.lddy;
    if (masks || a.db) {
      lm::GroupedActArgs g{};
      g.dy = a.dy, g.y = masks ? a.y : nullptr, g.dz = whole ? ws : nullptr;
      g.up = split ? ws + (whole ? one : 0) : nullptr, g.down = split ? static_cast<char*>(g.up) + one : nullptr;
      up = g.up, down = g.down;
      g.partials = reinterpret_cast<float*>(ws + dz_bytes), g.db = a.db, g.offsets = a.offsets;
      g.lddy = a.lddy, g.ldy = a.ldy, g.lddz = lddz, g.lddb = a.lddb, g.T = a.T, g.N = a.N;
      g.slope = act == 2 ? a.alpha : 0.0f;
      g.E = (int)a.E, g.type = a.type, g.db_type = a.db_type, g.ids64 = a.ids64;
      check_hip(lm::launch_grouped_act(g, s), "grouped_act launch");
      if (masks) dz = ws, ldz = lddz;
    }
    char plan[64] = "";
    if (a.dx && a.T > 0 && a.K > 0) {
      lm::GroupedArgs g{};
      g.x = dz, g.ldx = ldz, g.w = a.w, g.ldw = a.ldw, g.stride_w = a.stride_w, g.offsets = a.offsets, g.y = a.dx;
      g.ldy = a.lddx, g.T = a.T, g.K = a.N, g.N = a.K, g.E = (int)a.E, g.type = a.type, g.ids64 = a.ids64;
      g.turned = !a.turned;  // W^T
      rows_product(g, cus, s, plan, sizeof plan);
    }
    const char* tiles = "";
    if (a.dw && a.K > 0) {
      lm::GroupedWeightArgs g{};
      g.a = a.x, g.lda = a.ldx, g.b = split ? up : dz, g.ldb = ldz, g.M = a.K, g.N = a.N;
      g.more = down, g.scale = a.alpha, g.more_is_a = a.dw_turned;
      if (a.dw_turned) std::swap(g.a, g.b), std::swap(g.lda, g.ldb), std::swap(g.M, g.N);
      g.offsets = a.offsets, g.dw = a.dw, g.lddw = a.lddw, g.stride_dw = a.stride_dw, g.T = a.T;
      g.E = (int)a.E, g.type = a.type, g.dw_type = a.dw_type, g.ids64 = a.ids64;
      const bool direct = whole16({address(g.a), g.lda * e, address(g.b), g.ldb * e}) && reachable(64, g.lda, e) &&
                          reachable(64, g.ldb, e);
      const int64_t tiles256 = ((g.M + 255) / 256) * ((g.N + 255) / 256) * a.E;
      // 256 x 256 where they fill the CUs and are deep enough: 8192 rows at 8 bf16 experts of 4096 x 4096 in 283 us, 128 x 128
      // in 333; 2048 rows in 122 and 127, 1024 in 102 and 98. f32 results, twice the bytes, 8192 rows: 379 and 435, 4096: 243
      // and 237, 2048: 200 and 178. Two products spill there: the whole way back through a slope in 1041 with it and 986 without, through ReLU in 622.
      const bool big = !split && direct && a.type != lm::kF32 && tiles256 >= cus &&
                       a.T >= (a.dw_type == lm::kF32 ? 768 : 256) * a.E;
      check_grid((g.M + 127) / 128 * a.E, (g.N + 127) / 128);
      check_hip(weights_by_type(g, direct, big, s), "grouped_weights launch");
      tiles = big ? " dW 256x256" : direct ? " dW 128x128" : " dW any";
    }
    set_plan("grouped_dense_backward %s%s%s%s%s", type_name(a.type), masks ? " mask" : "", *plan ? " dX " : "", plan,
             tiles);
  });
}

// --------------------------------------------------------------- sampling
void sample_tokens(lm::SampleArgs a, void* stream) {
  check_sizes(a.M, a.V, "M", "V");
  check_float_type(a.type, "logits");
  if (a.V > kMostVocabulary) fail(kErrLimit, "V=%lld beyond 2^21", (long long)a.V);
  if (a.M > 0 && a.V == 0) fail(kErrShape, "rows of no logits have no tokens");
  if (!a.temperature && !(a.temperature_all >= 0.0f && std::isfinite(a.temperature_all)))
    fail(kErrArgument, "temperature must be finite and not negative");
  if (!a.top_p && std::isnan(a.top_p_all)) fail(kErrArgument, "top_p is NaN");
  if (!a.min_p && std::isnan(a.min_p_all)) fail(kErrArgument, "min_p is NaN");
  check_mat(a.x, a.ldx, a.M, a.V, "logits");
  if (a.M == 0) return set_plan("empty");
  if (!a.uniforms) fail(kErrArgument, "uniforms is null");
  if (!a.tokens) fail(kErrArgument, "tokens is null");
  check_grid(a.M, 1);
  a.shift = 46;
  while (a.V > int64_t(1) << (62 - a.shift)) --a.shift;
  device_launch(0, stream, [&](char*, int) {
    check_hip(lm::launch_sample_tokens(a, as_stream(stream)), "sample_tokens launch");
    set_plan("sample_tokens %s", type_name(a.type));
  });
}

}  // namespace
}  // namespace rt
}  // namespace edsl

using namespace edsl;

extern "C" {

int64_t edsl_hip_i8_packed_bytes(int64_t K, int64_t N) {
  int64_t bytes = -1;
  rt::guarded([&] { bytes = rt::i8_bytes(K, N); });
  return bytes;
}

int edsl_hip_i8_pack_launch(const int8_t* q, int64_t ldq, const void* scales, int scale_type, int64_t K, int64_t N,
                            void* packed, size_t packed_bytes, void* stream) {
  return rt::guarded([&] {
    lm::I8PackArgs a{};
    a.q = q, a.ldq = ldq, a.scales = scales, a.scale_type = scale_type, a.K = K, a.N = N;
    a.packed = static_cast<char*>(packed);
    rt::i8_pack(a, packed_bytes, stream);
  });
}

int edsl_hip_i8_dense_launch(const int8_t* X, int64_t ldx, const float* x_scales, const void* packed, const void* bias,
                             int bias_type, void* Y, int64_t ldy, int y_type, int64_t M, int64_t N, int64_t K,
                             int epilogue, float alpha, void* stream) {
  return rt::guarded([&] {
    lm::I8Args a{};
    a.x = X, a.ldx = ldx, a.x_scales = x_scales, a.w = static_cast<const char*>(packed), a.bias = bias;
    a.bias_type = bias_type, a.y = Y, a.ldy = ldy, a.y_type = y_type, a.epi = epilogue, a.alpha = alpha;
    rt::i8_dense(a, M, N, K, stream);
  });
}

int edsl_hip_grouped_dense_launch(const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t w_stride,
                                  int w_turned, const void* offsets, int ids64, int64_t E, const void* bias,
                                  int64_t ldbias, void* Y, int64_t ldy, int64_t T, int64_t N, int64_t K, int type,
                                  int epilogue, float alpha, void* stream) {
  return rt::guarded([&] {
    lm::GroupedArgs a{};
    a.x = X, a.ldx = ldx, a.w = W, a.ldw = ldw, a.stride_w = w_stride, a.turned = w_turned != 0, a.offsets = offsets;
    a.ids64 = ids64 != 0, a.bias = bias, a.ldbias = ldbias, a.y = Y, a.ldy = ldy, a.T = T, a.N = N, a.K = K;
    a.type = type, a.epi = epilogue, a.alpha = alpha;
    rt::grouped_dense(a, E, stream);
  });
}

int edsl_hip_grouped_dense_backward_launch(const void* dY, int64_t lddy, const void* X, int64_t ldx, const void* W,
                                           int64_t ldw, int64_t w_stride, int w_turned, const void* offsets, int ids64,
                                           int64_t E, const void* Y, int64_t ldy, void* dX, int64_t lddx, void* dW,
                                           int64_t lddw, int64_t dw_stride, int dw_turned, int dw_type, void* db,
                                           int64_t lddb, int db_type, int64_t T, int64_t N, int64_t K, int type,
                                           int epilogue, float alpha, void* stream) {
  return rt::guarded([&] {
    rt::Backward a{};
    a.dy = dY, a.lddy = lddy, a.x = X, a.ldx = ldx, a.w = W, a.ldw = ldw, a.stride_w = w_stride;
    a.turned = w_turned != 0, a.offsets = offsets, a.ids64 = ids64 != 0, a.E = E, a.y = Y, a.ldy = ldy;
    a.dx = dX, a.lddx = lddx, a.dw = dW, a.lddw = lddw, a.stride_dw = dw_stride, a.dw_turned = dw_turned != 0;
    a.dw_type = dw_type, a.db = db, a.lddb = lddb, a.db_type = db_type, a.T = T, a.N = N, a.K = K, a.type = type;
    a.epi = epilogue, a.alpha = alpha;
    rt::grouped_backward(a, stream);
  });
}

int edsl_hip_sample_tokens_launch(const void* logits, int64_t ldl, int type, const float* uniforms, void* tokens,
                                  int ids64, float* logprobs, const float* temperature, float temperature_all,
                                  const int32_t* top_k, int top_k_all, const float* top_p, float top_p_all,
                                  const float* min_p, float min_p_all, int64_t M, int64_t V, void* stream) {
  return rt::guarded([&] {
    lm::SampleArgs a{};
    a.x = logits, a.ldx = ldl, a.type = type, a.uniforms = uniforms, a.tokens = tokens, a.ids64 = ids64 != 0;
    a.logprobs = logprobs, a.temperature = temperature, a.temperature_all = temperature_all, a.top_k = top_k;
    a.top_k_all = top_k_all, a.top_p = top_p, a.top_p_all = top_p_all, a.min_p = min_p, a.min_p_all = min_p_all;
    a.M = M, a.V = V;
    rt::sample_tokens(a, stream);
  });
}

}  // extern "C"

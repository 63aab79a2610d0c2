// Entry points of include/edsl_hip_lm.h: the checks of their arguments, the
// split of the work over the chip, and the launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/edsl_hip_lm.h"
#include "dev_buf.hpp"
#include "lm_kernels.hpp"
#include "q4.hpp"
#include "runtime_internal.hpp"

namespace edsl {
namespace rt {
namespace {

constexpr int64_t kMostDim = int64_t(1) << 30;
constexpr int64_t kMostDepth = int64_t(1) << 23;  // of a 4-bit layer: 128 rows of x within 32-bit offsets
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
  // Its product with log2(e) has to be finite.
  if (!(scale > 0.0f && scale <= 0x1p127f)) fail(kErrArgument, "scale must be positive and at most 2^127");
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
  a.many = a.M > cus;
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

// ------------------------------------------------------------ 4-bit layer
lm::Q4Layout q4_checked_layout(int64_t K, int64_t N, int group, int scale_type, bool zeros) {
  check_sizes(K, N, "K", "N");
  if (K > kMostDepth) fail(kErrLimit, "K=%lld beyond 2^23", (long long)K);
  check_float_type(scale_type, "scales");
  if (group != 32 && group != 64 && (group <= 0 || group % 128 != 0))
    fail(kErrArgument, "group=%d is not 32, 64 or a multiple of 128", group);
  return lm::q4_layout(K, N, group, scale_type, zeros);
}

void check_packed(const void* p, const char* name) {
  if (!p) fail(kErrArgument, "%s is null", name);
  if (reinterpret_cast<uintptr_t>(p) % 256 != 0) fail(kErrArgument, "%s is not 256-byte aligned", name);
}

void q4_pack(lm::Q4PackArgs a, size_t bytes, void* stream) {
  a.layout = q4_checked_layout(a.K, a.N, a.group, a.scale_type, a.zeros != nullptr);
  if (bytes < (size_t)a.layout.bytes)
    fail(kErrArgument, "packed: %zu bytes, %lld are needed", bytes, (long long)a.layout.bytes);
  if (a.layout.bytes == 0) return set_plan("empty");
  const int64_t groups = (a.K + a.group - 1) / a.group;
  check_mat(a.q, a.ldq, a.K, a.N, "q");
  check_mat(a.scales, a.lds, groups, a.N, "scales");
  if (a.zeros) check_mat(a.zeros, a.ldz, groups, a.N, "zeros");
  check_packed(a.packed, "packed");
  check_grid(a.layout.tiles_n, a.layout.blocks);
  device_launch(0, stream, [&](char*, int) {
    check_hip(lm::launch_q4_pack(a, as_stream(stream)), "q4_pack launch");
    set_plan("q4_pack group=%d", a.group);
  });
}

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

// Up to 32 rows: column tiles of a workgroup, one where that is one workgroup a
// CU at most (1 x 4096 x 4096 in 5.0 us against 7.6 on half the CUs), else two (1 x
// 8192 x 8192 in 9.0 against 9.6); and how many workgroups split K, whose sums
// take a second kernel: up to four where CUs would be idle, from K = 16384 on (1
// x 16384 x 1024 in 8.1 us against 9.7 unsplit; 1 x 8192 x 1024 in 6.4 unsplit
// against 7.2). Eight waves of a workgroup split K's blocks, but four where there
// are no two for each (1 x 1024 x 32064 bf16 in 6.4 us, on eight 9.7), in very wide
// layers (1 x 4096 x 50176 in 26.5, on eight 28.3; but 16 x 8192 x 20000 in 22.9 and
// 22.6), and for f32, where a CU holds one workgroup of eight (1 x 4096 x 50176 in
// 45, on eight 58); and two for up to four blocks of a very wide layer (1 x 448 x
// 50176 in 7.6, on four 9.4, on eight 13.3; but 16 x 448 x 32064 in 6.9 and 6.5).
// More than 16 rows, two row tiles a wave, are on eight waves always.
void q4_small_plan(const lm::Q4Args& a, int cus, int* nt, int* waves, int* ksplit) {
  const int64_t tiles = (a.N + 15) / 16;
  *nt = tiles > cus ? 2 : 1;
  const int64_t wgs = (tiles + *nt - 1) / *nt;
  *waves = 8;
  if (*nt == 2 && a.M <= 16) {
    if (a.blocks <= 4 && wgs > 4 * (int64_t)cus)
      *waves = 2;
    else if (a.blocks <= 8 || (a.x_type == lm::kF32 && wgs > cus) || wgs > 3 * (int64_t)cus)
      *waves = 4;
  }
  *ksplit = a.blocks >= 128 ? (int)std::clamp<int64_t>(cus / wgs, 1, 4) : 1;
}

// Whether the small kernel takes the layer: up to 16 rows, and up to 32 of a
// layer that is not wide (17 x 8192 x 8192 in 12.6 us against 23.6 on tiles, 17 x
// 4096 x 50256 in 44 against 34) nor f32, whose operands do not fit.
bool q4_small_takes(const lm::Q4Args& a, int cus) {
  if (a.M <= 16) return true;
  return a.M <= 32 && a.x_type != lm::kF32 && (a.N + 15) / 16 <= 4 * (int64_t)cus;
}

// Tiles: 64 rows, 32 for up to 32, and 48 where that is fewer rows in all: of f32
// always (48 x 4096 x 50256 in 66 us against 79), of the others under three tiles a
// CU (270 x 4096 x 4096 bf16 in 23.2 against 27.6, 1100 rows in 56 against 61) and
// where it is a fifth fewer (144 x 3968 x 42834 in 78 against 86; but 330 rows of
// that layer in 168 against 163, 2000 x 4096 x 4096 in 98 against 85). Under two
// tiles a CU, two teams in a workgroup take K's blocks in turn (512 x 4096 x 4096 in 29 us against 33; 48 x 4096 x 50256
// f32 in 65 against 66.5), not from there on (2048 x 4096 x 4096 in 88 against 85;
// 1024 x 4096 x 4096 f32 in 106 against 99). Under one a CU (`few`), workgroups split
// K too (33 x 8192 x 8192 bf16 in 40, 25, 18, 20 us on 1, 2, 4, 8 slices), and sum
// their x themselves where they read it in place: the prepared sums' launch costs
// more (128 x 4096 x 4096 in 17.4 us against 19.7; 1024 rows in 54 against 47).
struct Q4TilePlan {
  int config, teams, ksplit;
  bool few;  // fewer tiles than CUs
};
Q4TilePlan q4_tile_plan(const lm::Q4Args& a, int cus) {
  static const int rows[] = {32, 64, 48};
  Q4TilePlan p{a.M <= 32 ? lm::kQ4Tile32x128 : lm::kQ4Tile64x128, 1, 1, false};
  const int64_t rows48 = ((int64_t)a.M + 47) / 48 * 48, rows64 = ((int64_t)a.M + 63) / 64 * 64;
  const int64_t tiles_n = ((int64_t)a.N + 127) / 128;
  if (a.M > 32 && rows48 < rows64 &&
      (a.x_type == lm::kF32 || rows64 / 64 * tiles_n < 3 * (int64_t)cus || 5 * rows48 <= 4 * rows64))
    p.config = lm::kQ4Tile48x128;
  const int64_t wgs = ((int64_t)a.M + rows[p.config] - 1) / rows[p.config] * tiles_n;
  check_grid(wgs, 8);
  p.few = wgs < cus;
  p.teams = wgs < 2 * (int64_t)cus ? 2 : 1;
  if (p.few) p.ksplit = (int)std::clamp<int64_t>(cus / wgs, 1, std::clamp(a.blocks / 4, 1, 8));
  return p;
}

// Even slices of K, none of them empty.
void q4_slices(lm::Q4Args& a) {
  a.slice_blocks = (a.blocks + a.ksplit - 1) / a.ksplit;
  if (a.slice_blocks > 0) a.ksplit = (a.blocks + a.slice_blocks - 1) / a.slice_blocks;
}

void q4_dense(lm::Q4Args a, int64_t M, int64_t N, int64_t K, int group, int scale_type, bool zeros, void* stream) {
  check_sizes(M, K, "M", "K");
  const lm::Q4Layout l = q4_checked_layout(K, N, group, scale_type, zeros);
  a.scale_mask = lm::q4_scale_mask(scale_type);
  if (a.x_type < lm::kF32 || a.x_type > lm::kE4m3) fail(kErrDtype, "X: unknown type %d", a.x_type);
  check_float_type(a.y_type, "Y");
  if (a.epi < 0 || a.epi > 7) fail(kErrArgument, "bad epilogue code %d", a.epi);
  if (M == 0 || N == 0) return set_plan("empty");
  if (a.epi & 1) {
    if (!a.bias) fail(kErrArgument, "epilogue adds a bias but bias is null");
    check_float_type(a.bias_type, "bias");
  } else {
    a.bias = nullptr;
  }
  check_mat(a.x, a.ldx, M, K, "X");
  check_mat(a.y, a.ldy, M, N, "Y");
  if (K > 0) check_packed(a.w, "packed");
  a.M = (int)M, a.N = (int)N, a.K = (int)K;
  a.scales_at = l.scales_at, a.zeros_at = l.zeros_at, a.scale_bytes = l.scale_bytes;
  a.zero_step = zeros ? 1 : 0;
  a.blocks = (int)l.blocks, a.scale_blocks = (int)l.scale_blocks;
  const uint64_t per = l.blocks_per_scale;
  a.scale_magic = per > 1 ? (uint32_t)((0x100000000ull + per - 1) / per) : 0;
  int cus = 0;
  device_launch(0, stream, [&](char*, int n) { cus = n; });
  const hipStream_t s = as_stream(stream);
  lm::Q4PrepArgs p{};
  p.x = a.x, p.ldx = a.ldx, p.M = a.M, p.K = a.K, p.blocks = a.blocks, p.spb = l.spb, p.x_type = a.x_type;
  p.ldp = l.blocks * 128, p.plane = M * p.ldp;
  const size_t planes = aligned((size_t)(a.x_type == lm::kF32 ? 3 : 1) * p.plane * 2);
  if (q4_small_takes(a, cus)) {
    int nt, waves;
    q4_small_plan(a, cus, &nt, &waves, &a.ksplit);
    q4_slices(a);
    const size_t bytes = a.ksplit > 1 ? (size_t)a.ksplit * a.M * a.N * sizeof(float) : 0;
    device_launch(bytes, stream, [&](char* ws, int) {
      a.partials = reinterpret_cast<float*>(ws);
      hipError_t (*const launch)(const lm::Q4Args&, int, int, int, hipStream_t) =
          a.x_type == lm::kF32    ? lm::launch_q4_small<lm::kF32>
          : a.x_type == lm::kBf16 ? lm::launch_q4_small<lm::kBf16>
          : a.x_type == lm::kF16  ? lm::launch_q4_small<lm::kF16>
          : a.x_type == lm::kI8   ? lm::launch_q4_small<lm::kI8>
                                  : lm::launch_q4_small<lm::kE4m3>;
      check_hip(launch(a, nt, waves, l.spb, s), "q4_small launch");
      if (a.ksplit > 1) check_hip(lm::launch_q4_join(a, s), "q4_join launch");
      static const char* const fewer[] = {"", "", " waves=2", "", " waves=4"};
      set_plan("q4_small %s cols=%d ksplit=%d%s%s", type_name(a.x_type), 16 * nt, a.ksplit,
               a.ksplit > 1 ? " +join" : "", waves < 8 ? fewer[waves] : "");
    });
    return;
  }
  const Q4TilePlan plan = q4_tile_plan(a, cus);
  a.ksplit = plan.ksplit;
  q4_slices(a);
  p.factor = zeros ? -1.0f : -8.0f - lm::q4_offset(a.x_type);
  p.xs_ld = (M + 127) / 128 * 128;
  // x itself where the tiles can read it: 16 bits, whole blocks, 16-byte aligned rows.
  const bool copy = !((a.x_type == lm::kBf16 || a.x_type == lm::kF16) && K % 128 == 0 && a.ldx % 8 == 0 &&
                      reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx <= kMostDepth);
  const bool own_sums = !copy && plan.few;
  const size_t sums = own_sums ? 0 : aligned((size_t)l.blocks * l.spb * p.xs_ld * sizeof(float));
  const size_t copied = copy ? planes : 0;
  const size_t parts = a.ksplit > 1 ? (size_t)a.ksplit * M * N * sizeof(float) : 0;
  device_launch(sums + copied + parts, stream, [&](char* ws, int) {
    p.xs = own_sums ? nullptr : reinterpret_cast<float*>(ws);
    p.xp = copy ? ws + sums : nullptr;
    a.xs = p.xs, a.xs_ld = p.xs_ld;
    a.xp = copy ? p.xp : a.x, a.ldp = copy ? p.ldp : a.ldx, a.plane = p.plane;
    a.partials = reinterpret_cast<float*>(ws + sums + copied);
    if (a.blocks > 0 && !own_sums) check_hip(lm::launch_q4_prep(p, s), "q4_prep launch");
    check_hip(lm::launch_q4_tile(a, plan.config, l.spb, plan.teams, zeros, s), "q4_tile launch");
    if (a.ksplit > 1) check_hip(lm::launch_q4_join(a, s), "q4_join launch");
    static const char* const names[] = {"32x128", "64x128", "48x128"};
    set_plan("%sq4_tile %s tile=%s teams=%d ksplit=%d%s", own_sums ? "" : copy ? "q4_prep_copy+" : "q4_prep+", type_name(a.x_type), names[plan.config],
             plan.teams, a.ksplit, a.ksplit > 1 ? " +join" : "");
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

int64_t edsl_hip_q4_packed_bytes(int64_t K, int64_t N, int group, int scale_type, int has_zeros) {
  int64_t bytes = -1;
  rt::guarded([&] { bytes = rt::q4_checked_layout(K, N, group, scale_type, has_zeros != 0).bytes; });
  return bytes;
}

int edsl_hip_q4_pack_launch(const uint8_t* q, int64_t ldq, const void* scales, int64_t lds, int scale_type,
                            const uint8_t* zeros, int64_t ldz, int64_t K, int64_t N, int group, void* packed,
                            size_t packed_bytes, void* stream) {
  return rt::guarded([&] {
    lm::Q4PackArgs a{};
    a.q = q, a.scales = scales, a.zeros = zeros, a.packed = static_cast<char*>(packed);
    a.ldq = ldq, a.lds = lds, a.ldz = ldz, a.K = K, a.N = N, a.group = group, a.scale_type = scale_type;
    rt::q4_pack(a, packed_bytes, stream);
  });
}

int edsl_hip_q4_dense_launch(const void* X, int64_t ldx, int x_type, const float* x_scales, const void* packed,
                             const void* bias, int bias_type, void* Y, int64_t ldy, int y_type, int64_t M, int64_t N,
                             int64_t K, int group, int scale_type, int has_zeros, int epilogue, float alpha,
                             void* stream) {
  return rt::guarded([&] {
    lm::Q4Args a{};
    a.x = X, a.x_scales = x_scales, a.w = static_cast<const char*>(packed), a.bias = bias, a.y = Y;
    a.ldx = ldx, a.ldy = ldy, a.x_type = x_type, a.y_type = y_type;
    a.bias_type = bias_type, a.epi = epilogue, a.alpha = alpha;
    rt::q4_dense(a, M, N, K, group, scale_type, has_zeros != 0, stream);
  });
}

}  // extern "C"

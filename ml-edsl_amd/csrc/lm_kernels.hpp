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

// ------------------------------------------------------------- sampling
struct SampleArgs {
  const void* x;
  const float* uniforms;
  void* tokens;
  float* logprobs;           // or nullptr
  const float* temperature;  // [M] each, or nullptr: `_all` for all rows
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int64_t ldx, M, V;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int shift;  // masses are in units of 2^-shift
  int type;
  bool ids64;
};
hipError_t launch_sample_tokens(const SampleArgs& a, hipStream_t stream);

// --------------------------------------------------- layers on groups of rows
// How tiles fill the CUs (lm_tile.hpp).
struct TileRounds {
  int cus, quarters, halves;
};
struct GroupedArgs {
  const void* x;
  const void* w;        // expert e at w + e * stride_w
  const void* bias;     // [E][N], rows of ldbias, or nullptr
  const void* offsets;  // [E + 1]
  void* y;
  int64_t ldx, ldw, stride_w, ldbias, ldy, T, K, N;
  int E, skip;  // experts of up to `skip` rows are left to the streaming kernel
  int epi, type;
  float alpha;
  bool ids64;
  bool turned;  // w's k are contiguous, not its columns
  int cus;
  TileRounds rounds;
};
constexpr int kGroupedSkinnyRows = 32;  // experts with up to this many rows may stream their weights
// direct: all rows start on 16 bytes, and K (of the product over rows) is whole pieces of 16 bytes.
template <int TYPE>
hipError_t launch_grouped_rows(const GroupedArgs& a, bool direct, hipStream_t stream);
template <int TYPE>
hipError_t launch_grouped_skinny(const GroupedArgs& a, hipStream_t stream);

struct GroupedWeightArgs {
  const void* a;  // dw[e] = a[e's rows]^T b[e's rows], plus `scale` times that of `more`, in b's place
  const void* b;
  const void* more;  // or nullptr
  const void* offsets;
  void* dw;
  float scale;
  bool more_is_a;  // in a's place
  int64_t lda, ldb, lddw, stride_dw, T, M, N;
  int E, type, dw_type;
  bool ids64;
};
template <int TYPE>
hipError_t launch_grouped_weights(const GroupedWeightArgs& a, bool direct, bool big, hipStream_t stream);

// dz = dy * act'(y), and the sums of dz over each expert's rows.
struct GroupedActArgs {
  const void* dy;
  const void* y;   // or nullptr: no activation
  void* dz;        // or nullptr
  void* up;        // dy where y > 0, else 0, or nullptr
  void* down;      // with it: dy elsewhere
  float* partials; // [tiles][N], where the sums are wanted
  void* db;        // [E][N], rows of lddb, or nullptr
  const void* offsets;
  int64_t lddy, ldy, lddz, lddb, T, N;
  float slope;  // where y <= 0
  int E, type, db_type;
  bool ids64;
};
constexpr int kGroupedActRows = 32;  // rows whose sums are taken together
// The most such tiles that T rows in E groups can have.
constexpr int64_t grouped_act_tiles(int64_t T, int64_t E) { return T / kGroupedActRows + (E < T ? E : T); }
hipError_t launch_grouped_act(const GroupedActArgs& a, hipStream_t stream);

// ----------------------------------------------------------- 8-bit layer
struct I8PackArgs {
  const int8_t* q;
  const void* scales;
  char* packed;
  int64_t ldq, K, N;
  int scale_type;
};
constexpr int64_t i8_blocks(int64_t K) { return (K + 127) / 128 * 2; }  // of 64 k
constexpr int64_t i8_tiles(int64_t N) { return (N + 15) / 16; }
constexpr int64_t i8_scales_at(int64_t K, int64_t N) { return i8_tiles(N) * i8_blocks(K) * 1024; }
hipError_t launch_i8_pack(const I8PackArgs& a, hipStream_t stream);

struct I8Args {
  const int8_t* x;
  const float* x_scales;  // or nullptr
  const char* w;          // as packed
  const float* w_scales;
  const void* bias;  // or nullptr
  void* y;
  int64_t ldx, ldy;
  int M, N, K, epi, y_type, bias_type;
  float alpha;
  int cus;
  TileRounds rounds;
};
hipError_t launch_i8_tile(const I8Args& a, bool direct, hipStream_t stream);
hipError_t launch_i8_skinny(const I8Args& a, int rows16, int cols16, hipStream_t stream);

}  // namespace lm
}  // namespace edsl

// The dense layer on groups of rows: each expert's weights on its own run of rows,
// offsets[e] .. offsets[e+1], known on the device only.
//
//   y_r = epi(x_r W_e + b_e);  dx_r = dz_r W_e^T;  dW_e = sum_r x_r^T dz_r
//
// Row tiles are numbered over all experts by a prefix sum that every wave takes of
// the offsets; the grid is the most tiles there can be, and workgroups past the
// real number end at once. Offsets are cut to 0 .. T, so that none leads outside.
//
// Three kernels. Groups of a few rows stream their weights (lm_skinny.hpp), bound by memory: 2 rows at 8 bf16
// experts of 4096 x 4096 in 12.4 us (4.5 TB/s of the weights in use), 96 at 64 of 2048 x 1024 in 50 to 53 (4.1 TB/s). Others take tiles (lm_tile.hpp),
// bound by the matrix cores: 8192 rows at 8 of 4096 x 4096 in 276 to 284 us (0.97 to 1.0 PFLOP/s; one group of 4096 rows there in
// 124 to 142, the vendor's product in 128); f32 4096 x 4096 x 4096 at 134 to 141 TFLOP/s of 157. dW has the rows as its
// depth: 345 us from the same 8192 rows, 104 of them the 537 MB of f32 results at the copy's rate.
#pragma once

#include "lm_kernels.hpp"
#include "lm_skinny.hpp"
#include "lm_tile.hpp"

namespace edsl {
namespace lm {

struct GroupOffsets {
  const void* p;
  int64_t rows;  // T
  int experts;
  bool wide;  // 64 bits
  __device__ __forceinline__ int64_t at(int e) const {
    const int64_t v = wide ? static_cast<const int64_t*>(p)[e] : (int64_t)static_cast<const int32_t*>(p)[e];
    return v < 0 ? 0 : v > rows ? rows : v;
  }
};

struct RowTile {
  int expert;
  int64_t first, end;  // rows of the tile, and the end of its expert's
};

// The tiles of `bm` rows of experts of more than `skip` rows, over all experts, by a
// wave: a lane holds one expert of each 64. Whole tiles are numbered apart from the
// last ones of experts, which have fewer rows.
struct RowTiles {
  const GroupOffsets& g;
  int bm, skip;

  // Whole tiles of an expert, and whether it has another one.
  __device__ __forceinline__ int of(int e, int64_t* first, int64_t* end, int* part) const {
    *part = 0;
    if (e >= g.experts) return 0;
    *first = g.at(e);
    *end = g.at(e + 1);
    const int64_t n = *end - *first;
    if (n <= skip || n <= 0) return 0;
    *part = n % bm != 0;
    return (int)(n / bm);
  }
  __device__ __forceinline__ void total(int64_t* whole, int64_t* parts) const {
    *whole = *parts = 0;
    for (int e = 0; e < g.experts; e += 64) {
      int64_t first, end;
      int part, sum = of(e + (int)threadIdx.x % 64, &first, &end, &part);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
      *whole += __builtin_amdgcn_readfirstlane(sum);
      *parts += __popcll(__ballot(part));
    }
  }
  // Whole tile `t`, or part `t`; false where there are fewer.
  __device__ __forceinline__ bool find(bool parts, int64_t t, RowTile* tile) const {
    const int lane = threadIdx.x % 64;
    int64_t before = 0;
    for (int e = 0; e < g.experts; e += 64) {
      int64_t first = 0, end = 0;
      int part;
      const int whole = of(e + lane, &first, &end, &part), mine = parts ? part : whole;
      int upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(upto, d);
        if (lane >= d) upto += v;
      }
      const uint64_t past = __ballot(before + upto > t);
      if (past) {
        const int l = __builtin_ctzll(past);
        const int64_t at = parts ? __shfl(whole, l) : t - before - (__shfl(upto, l) - __shfl(mine, l));
        *tile = {__builtin_amdgcn_readfirstlane(e + l), uniform(__shfl(first, l) + at * bm), uniform(__shfl(end, l))};
        return true;
      }
      before += __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
    }
    return false;
  }
  static __device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                     (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
  }
};

__device__ __forceinline__ GroupOffsets offsets_of(const GroupedArgs& a) {
  return {a.offsets, a.T, a.E, a.ids64};
}

// One tile: rows `first` to `end` at most, columns from n0 to `stop` at most.
template <typename Tl, int BKIND>
__device__ __forceinline__ void grouped_rows_tile(const GroupedArgs& a, const RowTile& t, int n0, u32x4* lds) {
  using T = typename Tl::T;
  const TileOperand oa{static_cast<const char*>(a.x) + t.first * a.ldx * (int64_t)sizeof(T), a.ldx,
                       (int)min(t.end - t.first, (int64_t)Tl::BM), a.T};
  const TileOperand ob{static_cast<const char*>(a.w) +
                           (t.expert * a.stride_w + (BKIND == kRows ? n0 * a.ldw : (int64_t)n0)) * (int64_t)sizeof(T),
                       a.ldw, (int)(a.N - n0), a.N};
  typename Tl::Acc acc[Tl::MI][Tl::NI];
  Tl::product(oa, ob, (int)a.K, lds, acc);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const auto finish = [&](float (&v)[4], typename Tl::Acc sum, const float (&bias)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a.bias ? __fadd_rn(sum[e], bias[e]) : sum[e];
    activate(v, a.epi, a.alpha);
  };
#pragma unroll
  for (int j = 0; j < Tl::NI; j += 2) {
    const int first = n0 + 16 * (wave % Tl::WN * Tl::NI + j), n = first + 4 * (lane / 16);
    float bias[2][4] = {};
    if (a.bias)
#pragma unroll
      for (int b = 0; b < 2 && j + b < Tl::NI; ++b)
        if (n + 16 * b < a.N) get4_typed(a.bias, t.expert * a.ldbias + n + 16 * b, a.type, bias[b], (int)a.N - n - 16 * b);
#pragma unroll
    for (int i = 0; i < Tl::MI; ++i) {
      const int64_t row = t.first + 16 * (wave / Tl::WN * Tl::MI + i);
      T* const to = static_cast<T*>(a.y) + row * a.ldy;
      float v0[4], v1[4];
      finish(v0, acc[i][j], bias[0]);
      if constexpr (Tl::NI > 1) {
        finish(v1, acc[i][j + 1], bias[1]);
        put_blocks(to, a.ldy, t.end - row, first, a.N, v0, v1);
      } else {
        put4(to + lane % 16 * a.ldy, n, a.N, v0, row + lane % 16 < t.end);
      }
    }
  }
}

// Big tiles, and Half (half as many columns) and Quarter ones for what is left of a round; the
// same type where there are none.
template <typename Big, typename Half, typename Quarter, int BKIND>
__global__ void __launch_bounds__(Big::kThreads, Big::kWavesPerSimd) grouped_rows_kernel(GroupedArgs a) {
  static_assert(Big::kThreads == Half::kThreads && Big::kThreads == Quarter::kThreads, "one launch");
  constexpr int kLds = Big::kLds > Half::kLds ? (Big::kLds > Quarter::kLds ? Big::kLds : Quarter::kLds)
                                              : (Half::kLds > Quarter::kLds ? Half::kLds : Quarter::kLds);
  __shared__ u32x4 lds[kLds];
  const int tiles_n = (int)((a.N + Big::BN - 1) / Big::BN);
  const GroupOffsets g = offsets_of(a);
  const RowTiles tiles{g, Big::BM, a.skip};
  int64_t whole, parts;
  tiles.total(&whole, &parts);
  // Offsets that do not rise could make more tiles than the grid is made for.
  const int most = 0x3fffffff / tiles_n;
  whole = min(whole, (int64_t)most), parts = min(parts, most - whole);
  TileTurn turn;
  if (!tile_turn((int)block_of(), (int)(whole + parts) * tiles_n, (int)whole * tiles_n, a.rounds, &turn)) return;
  // Whole tiles first, then the experts' last ones.
  const bool part = turn.tile >= whole * tiles_n;
  int tn;
  const int row = row_of_tile(turn.tile - (part ? (int)whole * tiles_n : 0), (int)(part ? parts : whole), tiles_n, &tn);
  RowTile t;
  if (!tiles.find(part, row, &t)) return;
  t.end = min(t.end, t.first + Big::BM);
  int n0 = tn * Big::BN;
  if (turn.pieces == 1) return grouped_rows_tile<Big, BKIND>(a, t, n0, lds);
  n0 += turn.sub % 2 * (Big::BN / 2);
  t.first += turn.sub / 2 * (Big::BM / 2);
  if (n0 >= a.N || t.first >= t.end) return;
  if constexpr (!std::is_same<Half, Quarter>::value)
    if (turn.pieces == 2) return grouped_rows_tile<Half, BKIND>(a, t, n0, lds);
  if constexpr (!std::is_same<Big, Quarter>::value) {
    t.end = min(t.end, t.first + Quarter::BM);
    grouped_rows_tile<Quarter, BKIND>(a, t, n0, lds);
  }
}

// Experts of up to kGroupedSkinnyRows rows: a workgroup an expert and column block.
template <typename T, int BKIND, int NJ, int WAVES, int U, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) grouped_skinny_kernel(GroupedArgs a) {
  using S1 = Skinny<T, BKIND, 1, NJ, WAVES, U, AHEAD>;
  using S2 = Skinny<T, BKIND, 2, NJ, WAVES, U, AHEAD>;
  __shared__ typename S1::Acc lds[S1::kSlots];
  const GroupOffsets g = offsets_of(a);
  const int e = blockIdx.y;
  const int64_t first = g.at(e), count = g.at(e + 1) - first;
  if (count <= 0 || count > kGroupedSkinnyRows) return;
  const int rows = (int)count, n0 = (int)blockIdx.x * S1::kCols16;
  const char* const x = static_cast<const char*>(a.x) + first * a.ldx * (int64_t)sizeof(T);
  const char* const w = static_cast<const char*>(a.w) + e * a.stride_w * (int64_t)sizeof(T);
  const auto store = [&](int m, int n, float sum) {
    float v[1] = {sum};
    if (a.bias) v[0] = __fadd_rn(sum, (float)static_cast<const T*>(a.bias)[e * a.ldbias + n]);
    activate(v, a.epi, a.alpha);
    static_cast<T*>(a.y)[(first + m) * a.ldy + n] = (T)v[0];
  };
  if (rows <= 16)
    S1::run(x, a.ldx, rows, w, a.ldw, (int)a.K, (int)a.N, n0, lds, store);
  else
    S2::run(x, a.ldx, rows, w, a.ldw, (int)a.K, (int)a.N, n0, lds, store);
}

// dW of two products at (m, n) as one sum over the expert's `rows`, in their order: a term is one product or the
// other, never 0 times an infinity that the other one has.
template <typename T>
__device__ float grouped_weights_term_by_term(const GroupedWeightArgs& a, int64_t first, int64_t rows, int m, int n) {
  const T* const up = static_cast<const T*>(a.more_is_a ? a.a : a.b) + (a.more_is_a ? first * a.lda + m : first * a.ldb + n);
  const T* const down = static_cast<const T*>(a.more) + (a.more_is_a ? first * a.lda + m : first * a.ldb + n);
  const T* const other = static_cast<const T*>(a.more_is_a ? a.b : a.a) + (a.more_is_a ? first * a.ldb + n : first * a.lda + m);
  const int64_t ld = a.more_is_a ? a.lda : a.ldb, ld_other = a.more_is_a ? a.ldb : a.lda;
  float sum = 0.0f;
#pragma unroll 1
  for (int64_t r = 0; r < rows && sum == sum; r += 8) {  // NaN is the end
    float u[8], d[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t at = min(r + i, rows - 1);
      u[i] = (float)up[at * ld], d[i] = (float)down[at * ld], o[i] = (float)other[at * ld_other];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (r + i < rows) sum = fmaf(d[i] == 0.0f ? u[i] : a.scale * d[i], o[i], sum);
  }
  return sum;
}

// The workgroup's results at (m0, n0) of which a lane's `lost` are NaN: those are summed again, but where a column holds NaN,
// which is what they are then. 8192 rows at 8 of 4096 x 4096 in 0.83 to 0.9 ms without any; with an infinity in one row of x in
// 1.8, with a row of NaN in each group in 3.6, and in 88 where a row of each is infinite, so that all results are summed again.
template <typename Tl>
__device__ __forceinline__ void grouped_weights_again(const GroupedWeightArgs& a, int expert, int m0, int n0,
                                                                int64_t first, int64_t rows, uint32_t lost,
                                                                bool* nan_at) {
  using T = typename Tl::T;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  // A thread looks one column through.
  static_assert(Tl::BM + Tl::BN <= Tl::kThreads, "a thread a column");
  if (tid < Tl::BM + Tl::BN) {
    const bool of_a = tid < Tl::BM;
    const int col = of_a ? m0 + tid : n0 + tid - Tl::BM;
    const int64_t ld = of_a ? a.lda : a.ldb;
    const auto has = [&](const void* p) {
      const T* const from = static_cast<const T*>(p) + first * ld + col;
      bool found = false;
#pragma unroll 8
      for (int64_t r = 0; r < rows; ++r) found |= from[r * ld] != from[r * ld];
      return found;
    };
    bool found = false;
    if (col < (of_a ? a.M : a.N)) found = has(of_a ? a.a : a.b) || (of_a == a.more_is_a && has(a.more));
    nan_at[tid] = found;
  }
  __syncthreads();
#pragma unroll 1
  for (; lost; lost &= lost - 1) {
    const int bit = __builtin_ctz(lost), i = bit / (4 * Tl::NI), j = bit / 4 % Tl::NI;
    const int m = m0 + 16 * (wave / Tl::WN * Tl::MI + i) + lane % 16;
    const int n = n0 + 16 * (wave % Tl::WN * Tl::NI + j) + 4 * (lane / 16) + bit % 4;
    if (m >= a.M || n >= a.N || nan_at[m - m0] || nan_at[Tl::BM + n - n0]) continue;
    const float sum = grouped_weights_term_by_term<T>(a, first, rows, m, n);
    const int64_t at = expert * a.stride_dw + m * a.lddw + n;
    if (a.dw_type == kF32)
      static_cast<float*>(a.dw)[at] = sum;
    else
      static_cast<T*>(a.dw)[at] = (T)sum;
  }
}

// dW: an expert's tile of [M][N], its rows the depth. Experts without rows get zeros. MORE: of two products, each
// with zeros where the other has its terms. Results of NaN, as those zeros make of infinities in the rows, are summed again.
template <typename Tl, bool MORE>
__global__ void __launch_bounds__(Tl::kThreads, Tl::kWavesPerSimd) grouped_weights_kernel(GroupedWeightArgs a) {
  using T = typename Tl::T;
  __shared__ u32x4 lds[Tl::kLds];
  const int tiles_m = (int)((a.M + Tl::BM - 1) / Tl::BM), tiles_n = (int)((a.N + Tl::BN - 1) / Tl::BN);
  const int64_t total = (int64_t)tiles_m * tiles_n * a.E;
  if (block_of() >= total) return;
  // Each XCD has a part of every expert: their depths differ.
  const int expert = (int)(block_of() / (uint32_t)(tiles_m * tiles_n));
  int tn;
  const int tm = row_of_tile(xcd_order((int)(block_of() % (uint32_t)(tiles_m * tiles_n)), tiles_m * tiles_n), tiles_m,
                             tiles_n, &tn);
  const int m0 = tm * Tl::BM, n0 = tn * Tl::BN;
  const GroupOffsets g{a.offsets, a.T, a.E, a.ids64};
  const int64_t first = g.at(expert), rows = max(g.at(expert + 1) - first, (int64_t)0);
  typename Tl::Acc acc[Tl::MI][Tl::NI];
#pragma unroll
  for (int i = 0; i < Tl::MI; ++i)
#pragma unroll
    for (int j = 0; j < Tl::NI; ++j) acc[i][j] = typename Tl::Acc{};
  const auto operand = [&](const void* p, int64_t ld, int at, int64_t all) {
    return TileOperand{static_cast<const char*>(p) + (first * ld + at) * (int64_t)sizeof(T), ld, (int)(all - at), all};
  };
  if constexpr (MORE) {
    Tl::add_product(operand(a.more_is_a ? a.more : a.a, a.lda, m0, a.M), operand(a.more_is_a ? a.b : a.more, a.ldb, n0, a.N),
                    (int)rows, lds, acc);
#pragma unroll
    for (int i = 0; i < Tl::MI; ++i)
#pragma unroll
      for (int j = 0; j < Tl::NI; ++j) acc[i][j] *= a.scale;
  }
  Tl::add_product(operand(a.a, a.lda, m0, a.M), operand(a.b, a.ldb, n0, a.N), (int)rows, lds, acc);
  const int wave = threadIdx.x / 64;
#pragma unroll
  for (int i = 0; i < Tl::MI; ++i) {
    const int m = m0 + 16 * (wave / Tl::WN * Tl::MI + i);
    const int64_t at = expert * a.stride_dw + m * a.lddw;
#pragma unroll
    for (int j = 0; j < Tl::NI; j += 2) {
      const int first = n0 + 16 * (wave % Tl::WN * Tl::NI + j);
      const float v0[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      const float v1[4] = {acc[i][j + 1][0], acc[i][j + 1][1], acc[i][j + 1][2], acc[i][j + 1][3]};
      if (a.dw_type == kF32)
        put_blocks(static_cast<float*>(a.dw) + at, a.lddw, a.M - m, first, a.N, v0, v1);
      else
        put_blocks(static_cast<T*>(a.dw) + at, a.lddw, a.M - m, first, a.N, v0, v1);
    }
  }
  if constexpr (MORE) {
    static_assert(Tl::MI * Tl::NI * 4 <= 32, "a bit for each of a lane's results");
    uint32_t lost = 0;
#pragma unroll
    for (int i = 0; i < Tl::MI; ++i)
#pragma unroll
      for (int j = 0; j < Tl::NI; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) lost |= (uint32_t)(acc[i][j][e] != acc[i][j][e]) << ((i * Tl::NI + j) * 4 + e);
    uint32_t* const any = reinterpret_cast<uint32_t*>(lds);
    if (threadIdx.x == 0) *any = 0;
    __syncthreads();
    if (lost) *any = 1;
    __syncthreads();
    if (*any == 0) return;
    __threadfence();  // other lanes of the wave have stored them
    __syncthreads();
    grouped_weights_again<Tl>(a, expert, m0, n0, first, rows, lost, reinterpret_cast<bool*>(lds));
  }
}

}  // namespace lm
}  // namespace edsl

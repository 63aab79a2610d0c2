// The dense layer on groups of rows: each expert's weights on its own run of rows,
// offsets[e] .. offsets[e+1], known on the device only.
//
//   y_r = epi(x_r W_e + b_e);  dx_r = dz_r W_e^T;  dW_e = sum_r x_r^T dz_r
//
// Row tiles are numbered over all experts by a prefix sum that every wave takes of
// the offsets; the grid is the most tiles there can be, and workgroups past the
// real number end at once. Offsets are cut to 0 .. T, so that none leads outside.
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
// wave: a lane holds one expert of each 64.
struct RowTiles {
  const GroupOffsets& g;
  int bm, skip;

  __device__ __forceinline__ int of(int e, int64_t* first, int64_t* end) const {
    if (e >= g.experts) return 0;
    *first = g.at(e);
    *end = g.at(e + 1);
    const int64_t n = *end - *first;
    return n > skip ? (int)((n + bm - 1) / bm) : 0;
  }
  __device__ __forceinline__ int64_t total() const {
    int64_t total = 0;
    for (int e = 0; e < g.experts; e += 64) {
      int64_t first, end;
      int sum = of(e + (int)threadIdx.x % 64, &first, &end);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
      total += __builtin_amdgcn_readfirstlane(sum);
    }
    return total;
  }
  // Tile `t`; false where there are fewer.
  __device__ __forceinline__ bool find(int64_t t, RowTile* tile) const {
    const int lane = threadIdx.x % 64;
    int64_t before = 0;
    for (int e = 0; e < g.experts; e += 64) {
      int64_t first = 0, end = 0;
      const int mine = of(e + lane, &first, &end);
      int upto = mine;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(upto, d);
        if (lane >= d) upto += v;
      }
      const uint64_t past = __ballot(before + upto > t);
      if (past) {
        const int l = __builtin_ctzll(past);
        const int64_t row = __shfl(first, l) + (t - before - (__shfl(upto, l) - __shfl(mine, l))) * bm;
        *tile = {__builtin_amdgcn_readfirstlane(e + l), uniform(row), uniform(__shfl(end, l))};
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

// Workgroup w's tile and column strip: eight row tiles go along the columns together,
// one XCD's workgroups among them.
__device__ __forceinline__ bool find_tile(const RowTiles& tiles, int tiles_n, int64_t w, RowTile* tile, int* tn) {
  // Offsets that do not rise could make more than the grid is made for.
  const int64_t total = min(tiles.total(), (int64_t)(0x7fffffff / tiles_n));
  if (w >= total * tiles_n) return false;
  const int at = xcd_order((int)w, (int)(total * tiles_n));
  constexpr int kGroup = 8;
  const int group = at / (kGroup * tiles_n), first = group * kGroup;
  const int rows = min((int)total - first, kGroup), in = at - group * kGroup * tiles_n;
  *tn = in / rows;
  return tiles.find(first + in % rows, tile);
}

__device__ __forceinline__ GroupOffsets offsets_of(const GroupedArgs& a) {
  return {a.offsets, a.T, a.E, a.ids64};
}

template <typename Tl, int BKIND>
__global__ void __launch_bounds__(Tl::kThreads, 1) grouped_rows_kernel(GroupedArgs a) {
  using T = typename Tl::T;
  __shared__ u32x4 lds[2 * Tl::kStage];
  const int tiles_n = (int)((a.N + Tl::BN - 1) / Tl::BN);
  RowTile t;
  int tn;
  const GroupOffsets g = offsets_of(a);
  if (!find_tile(RowTiles{g, Tl::BM, a.skip}, tiles_n, block_of(), &t, &tn)) return;
  const int n0 = tn * Tl::BN;
  const TileOperand oa{static_cast<const char*>(a.x) + t.first * a.ldx * (int64_t)sizeof(T), a.ldx,
                       (int)min(t.end - t.first, (int64_t)Tl::BM)};
  const TileOperand ob{static_cast<const char*>(a.w) +
                           (t.expert * a.stride_w + (BKIND == kRows ? n0 * a.ldw : (int64_t)n0)) * (int64_t)sizeof(T),
                       a.ldw, (int)(a.N - n0)};
  typename Tl::Acc acc[Tl::MI][Tl::NI];
  Tl::product(oa, ob, (int)a.K, lds, acc);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int j = 0; j < Tl::NI; ++j) {
    const int n = n0 + 16 * (wave % Tl::WN * Tl::NI + j) + 4 * (lane / 16), left = (int)a.N - n;
    if (left <= 0) break;
    float bias[4] = {};
    if (a.bias) get4_typed(a.bias, t.expert * a.ldbias + n, a.type, bias, left);
#pragma unroll
    for (int i = 0; i < Tl::MI; ++i) {
      const int64_t row = t.first + 16 * (wave / Tl::WN * Tl::MI + i) + lane % 16;
      if (row >= t.end) break;
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a.bias ? __fadd_rn(acc[i][j][e], bias[e]) : acc[i][j][e];
      activate(v, a.epi, a.alpha);
      put4(static_cast<T*>(a.y) + row * a.ldy + n, v, left);
    }
  }
}

// Experts of up to kGroupedSkinnyRows rows: a workgroup an expert and column block.
template <typename T, int BKIND, int NJ, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) grouped_skinny_kernel(GroupedArgs a) {
  using S1 = Skinny<T, BKIND, 1, NJ, WAVES>;
  using S2 = Skinny<T, BKIND, 2, NJ, WAVES>;
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

// dW: an expert's tile of [M][N], its rows the depth. Experts without rows get zeros.
template <typename Tl>
__global__ void __launch_bounds__(Tl::kThreads, 1) grouped_weights_kernel(GroupedWeightArgs a) {
  using T = typename Tl::T;
  __shared__ u32x4 lds[2 * Tl::kStage];
  const int tiles_m = (int)((a.M + Tl::BM - 1) / Tl::BM), tiles_n = (int)((a.N + Tl::BN - 1) / Tl::BN);
  const int64_t total = (int64_t)tiles_m * tiles_n * a.E;
  if (block_of() >= total) return;
  const int at = xcd_order((int)block_of(), (int)total);
  const int expert = at / (tiles_m * tiles_n);
  int in = at - expert * tiles_m * tiles_n;
  constexpr int kGroup = 8;
  const int group = in / (kGroup * tiles_n), first_m = group * kGroup, rows_m = min(tiles_m - first_m, kGroup);
  in -= group * kGroup * tiles_n;
  const int m0 = (first_m + in % rows_m) * Tl::BM, n0 = in / rows_m * Tl::BN;
  const GroupOffsets g{a.offsets, a.T, a.E, a.ids64};
  const int64_t first = g.at(expert), rows = max(g.at(expert + 1) - first, (int64_t)0);
  const TileOperand oa{static_cast<const char*>(a.a) + (first * a.lda + m0) * (int64_t)sizeof(T), a.lda, (int)(a.M - m0)};
  const TileOperand ob{static_cast<const char*>(a.b) + (first * a.ldb + n0) * (int64_t)sizeof(T), a.ldb, (int)(a.N - n0)};
  typename Tl::Acc acc[Tl::MI][Tl::NI];
  Tl::product(oa, ob, (int)rows, lds, acc);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
#pragma unroll
  for (int i = 0; i < Tl::MI; ++i) {
    const int m = m0 + 16 * (wave / Tl::WN * Tl::MI + i) + lane % 16;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < Tl::NI; ++j) {
      const int n = n0 + 16 * (wave % Tl::WN * Tl::NI + j) + 4 * (lane / 16);
      const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (n < a.N) put4_typed(a.dw, expert * a.stride_dw + m * a.lddw + n, a.dw_type, v, (int)a.N - n);
    }
  }
}

}  // namespace lm
}  // namespace edsl

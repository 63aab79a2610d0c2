// Launches of the layers on groups of rows of one type.
#pragma once

#include <algorithm>

#include "lm_grouped.hpp"

namespace edsl {
namespace lm {

template <typename T>
struct GroupedLaunch {
  template <typename Tl, int BKIND>
  static hipError_t rows_tile(const GroupedArgs& a, hipStream_t stream) {
    // The most tiles that T rows in E groups can have.
    const int64_t groups = std::min<int64_t>(a.E, a.T / (a.skip + 1));
    const int64_t tiles = (a.T / Tl::BM + groups) * ((a.N + Tl::BN - 1) / Tl::BN);
    if (tiles == 0) return hipSuccess;
    hipLaunchKernelGGL((grouped_rows_kernel<Tl, BKIND>), grid_of(tiles), dim3(Tl::kThreads), 0, stream, a);
    return launched();
  }
  template <int BKIND>
  static hipError_t rows_kind(const GroupedArgs& a, int tile, hipStream_t stream) {
    if (tile == kGroupedTileAny) return rows_tile<Tile<T, kRows, BKIND, 128, 128, 2, 2, false>, BKIND>(a, stream);
    if constexpr (sizeof(T) == 2)
      if (tile == kGroupedTile256) return rows_tile<Tile<T, kRows, BKIND, 256, 256, 2, 4, true>, BKIND>(a, stream);
    return rows_tile<Tile<T, kRows, BKIND, 128, 128, 2, 2, true>, BKIND>(a, stream);
  }
  static hipError_t rows(const GroupedArgs& a, int tile, hipStream_t stream) {
    return a.turned ? rows_kind<kRows>(a, tile, stream) : rows_kind<kCols>(a, tile, stream);
  }

  template <int BKIND, int NJ>
  static hipError_t skinny_cols(const GroupedArgs& a, hipStream_t stream) {
    constexpr int kWaves = 8;
    const unsigned blocks = (unsigned)((a.N + 16 * NJ - 1) / (16 * NJ));
    hipLaunchKernelGGL((grouped_skinny_kernel<T, BKIND, NJ, kWaves>), dim3(blocks, (unsigned)a.E), dim3(64 * kWaves), 0,
                       stream, a);
    return launched();
  }
  static hipError_t skinny(const GroupedArgs& a, hipStream_t stream) {
    if (a.turned) return skinny_cols<kRows, 1>(a, stream);
    return skinny_cols<kCols, 4>(a, stream);
  }

  template <typename Tl>
  static hipError_t weights_tile(const GroupedWeightArgs& a, hipStream_t stream) {
    const int64_t tiles = ((a.M + Tl::BM - 1) / Tl::BM) * ((a.N + Tl::BN - 1) / Tl::BN) * a.E;
    hipLaunchKernelGGL((grouped_weights_kernel<Tl>), grid_of(tiles), dim3(Tl::kThreads), 0, stream, a);
    return launched();
  }
  static hipError_t weights(const GroupedWeightArgs& a, int tile, hipStream_t stream) {
    if (tile == kGroupedTileAny) return weights_tile<Tile<T, kCols, kCols, 128, 128, 2, 2, false>>(a, stream);
    if constexpr (sizeof(T) == 2)
      if (tile == kGroupedTile256) return weights_tile<Tile<T, kCols, kCols, 256, 256, 2, 4, true>>(a, stream);
    return weights_tile<Tile<T, kCols, kCols, 128, 128, 2, 2, true>>(a, stream);
  }
};

}  // namespace lm
}  // namespace edsl

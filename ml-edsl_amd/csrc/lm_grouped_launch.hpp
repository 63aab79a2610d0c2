// Launches of the layers on groups of rows of one type.
#pragma once

#include <algorithm>

#include "lm_grouped.hpp"

namespace edsl {
namespace lm {

template <typename T>
struct GroupedLaunch {
  template <int BKIND, typename Big, typename Half = Big, typename Quarter = Half>
  static hipError_t rows_tiles(GroupedArgs a, int quarters, int halves, hipStream_t stream) {
    // The most tiles that T rows in E groups can have.
    const int64_t groups = std::min<int64_t>(a.E, a.T / (a.skip + 1));
    const int64_t tiles = (a.T / Big::BM + groups) * ((a.N + Big::BN - 1) / Big::BN);
    if (tiles == 0) return hipSuccess;
    a.rounds = {a.cus, quarters, halves};
    hipLaunchKernelGGL((grouped_rows_kernel<Big, Half, Quarter, BKIND>), grid_of(tile_turns(tiles, a.rounds)),
                       dim3(Big::kThreads), 0, stream, a);
    return launched();
  }
  template <int BKIND, bool DIRECT>
  static hipError_t rows_kind(const GroupedArgs& a, hipStream_t stream) {
    if constexpr (sizeof(T) == 4) {
      // Bound by the matrix cores, which f32 keeps eight times as long, so that small tiles are nearly as good. Up to
      // a round of 128 x 128: of 64 x 64 and 32 x 64 the one whose rounds of the CUs take less, one of 32 x 64 0.6 of
      // the other's (300 x 512 x 1024 in 11.8 and 15.9 us on 32 x 64 and 64 x 64, 700 x 900 x 1500 of three experts in 34 and 40,
      // 1000 x 1024 x 1024 in 27.6 and 27.0, 2000 x 1008 x 1008 of five in 61 and 57). Beyond it 128 x 128, with 64 x 64 for
      // what rounds leave (2049^3 in 190 us, 288 on 128 x 128 alone; 2000 x 1008 x 1008 so in 62 against 50 on 64 x 64).
      constexpr int kStages = DIRECT ? 3 : 2;
      using Small = Tile<T, kRows, BKIND, 64, 64, 2, 4, DIRECT, kStages>;
      const auto tiles = [&](int64_t rows, int64_t cols) {
        return (a.T / rows + std::min<int64_t>(a.E, a.T)) * ((a.N + cols - 1) / cols);
      };
      if (tiles(128, 128) > a.cus)
        return rows_tiles<BKIND, Tile<T, kRows, BKIND, 128, 128, 2, 4, DIRECT>, Small>(a, a.cus, 0, stream);
      const auto rounds = [&](int64_t rows) { return (tiles(rows, 64) + a.cus - 1) / a.cus; };
      if (5 * rounds(64) <= 3 * rounds(32)) return rows_tiles<BKIND, Small>(a, 0, 0, stream);
      return rows_tiles<BKIND, Tile<T, kRows, BKIND, 32, 64, 1, 4, DIRECT, kStages>>(a, 0, 0, stream);
    } else if constexpr (!DIRECT) {
      // Registers hold two stages on their way for no larger tile.
      return rows_tiles<BKIND, Tile<T, kRows, BKIND, 128, 128, 2, 4, false>>(a, 0, 0, stream);
    } else {
      // Rounds of 256 x 256 (bf16 4096^3 in 115 to 136 us, on 128 x 128 in 136 to 175), up to a quarter of a round left in 128 x 128
      // and up to half in 256 x 128: 1000 x 4096 x 4096 in 51 us, 2048 in 78, 4500 in 153; on whole tiles 95, 105 and 194.
      return rows_tiles<BKIND, Tile<T, kRows, BKIND, 256, 256, 2, 4, true>, Tile<T, kRows, BKIND, 256, 128, 4, 2, true, 3>,
                        Tile<T, kRows, BKIND, 128, 128, 2, 4, true, 3>>(a, a.cus / 4, a.cus / 2, stream);
    }
  }
  static hipError_t rows(const GroupedArgs& a, bool direct, hipStream_t stream) {
    if (a.turned) return direct ? rows_kind<kRows, true>(a, stream) : rows_kind<kRows, false>(a, stream);
    return direct ? rows_kind<kCols, true>(a, stream) : rows_kind<kCols, false>(a, stream);
  }

  template <int BKIND, int NJ, int U, int AHEAD>
  static hipError_t skinny_cols(const GroupedArgs& a, hipStream_t stream) {
    constexpr int kWaves = 8;
    const unsigned blocks = (unsigned)((a.N + 16 * NJ - 1) / (16 * NJ));
    hipLaunchKernelGGL((grouped_skinny_kernel<T, BKIND, NJ, kWaves, U, AHEAD>), dim3(blocks, (unsigned)a.E), dim3(64 * kWaves), 0,
                       stream, a);
    return launched();
  }
  static hipError_t skinny(const GroupedArgs& a, hipStream_t stream) {
    // Workgroups of 16 columns of the experts that may have rows, and of more columns where these are many:
    // 2 rows of 8 experts of 4096 x 4096 bf16 in 8.3 us on 16 columns, on 32 in 13.8; 96 rows at 64 of 2048 x 1024 in 57.7 on
    // 16, 52 on 32 and 54 on 64; 200 there in 64 on 32 and 57 on 64, 16 at 8 of 4096 x 4096 in 57 and 50.
    const int64_t groups = (a.N + 15) / 16 * std::min<int64_t>(a.E, a.T);
    const bool many = groups > 2 * (int64_t)a.cus;
    if (a.turned) {
      if (!many) return skinny_cols<kRows, 1, 2, 2>(a, stream);
      return 2 * a.T > 3 * (int64_t)a.E ? skinny_cols<kRows, 4, 2, 1>(a, stream) : skinny_cols<kRows, 2, 2, 2>(a, stream);
    }
    // Columns contiguous: 64, with 8 bytes a lane and row; 128 of 16 bits where these are many (96 rows of 64 experts in
    // 46.5 us against 49; 2 rows of 8 in 15.7 against 12.1).
    if constexpr (sizeof(T) == 2)
      if (groups > 8 * (int64_t)a.cus && a.N >= 8) return skinny_cols<kCols, 8, 1, 1>(a, stream);
    return skinny_cols<kCols, 4, 1, 1>(a, stream);
  }

  template <typename Tl>
  static hipError_t weights_tile(const GroupedWeightArgs& a, hipStream_t stream) {
    const int64_t tiles = ((a.M + Tl::BM - 1) / Tl::BM) * ((a.N + Tl::BN - 1) / Tl::BN) * a.E;
    if constexpr (sizeof(T) == 2 && Tl::BM == 128)
      if (a.more) {
        hipLaunchKernelGGL((grouped_weights_kernel<Tl, true>), grid_of(tiles), dim3(Tl::kThreads), 0, stream, a);
        return launched();
      }
    if (a.more) return hipErrorInvalidValue;  // half of dW would be left out
    hipLaunchKernelGGL((grouped_weights_kernel<Tl, false>), grid_of(tiles), dim3(Tl::kThreads), 0, stream, a);
    return launched();
  }
  static hipError_t weights(const GroupedWeightArgs& a, bool direct, bool big, hipStream_t stream) {
    if (!direct) return weights_tile<Tile<T, kCols, kCols, 128, 128, 2, 4, false>>(a, stream);
    if constexpr (sizeof(T) == 2)
      if (big) return weights_tile<Tile<T, kCols, kCols, 256, 256, 2, 4, true>>(a, stream);
    return weights_tile<Tile<T, kCols, kCols, 128, 128, 2, 4, true>>(a, stream);
  }
};

}  // namespace lm
}  // namespace edsl

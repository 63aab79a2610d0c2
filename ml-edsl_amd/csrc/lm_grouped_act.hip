// The way back through the activation of a layer on groups of rows, and its
// bias's gradient: dz = dy (y > 0), or dy times the slope elsewhere, and
//   db_e = sum over e's rows of dz.
// Bound by memory: 8192 x 4096 bf16 with both in 42 us (201 MB at 4.8 TB/s), sums alone in 21.
// dz is rounded to its type, the matrix instructions' operand, for dX and bf16 dW (a 16-bit dy times a slope of 0.01 is 2^-9 or
// 2^-12 of it off, f16 below 2^-14 half of 2^-24); db sums it before that, and dW in f32 and of f16 through a slope
// takes dy's two parts as they are, the lower one's product scaled. Rows are
// summed in tiles of 32 whose sums a second launch adds in their order, in 64 bits (6 of those 42 us), so that the same call
// gives the same bits. A thread has its own 8 or 4 columns and eight rows on their way; with a wave's threads
// along the rows, joined through LDS, the same took 92 us.
#include <algorithm>

#include "lm_grouped.hpp"

namespace edsl {
namespace lm {

namespace {

constexpr int kActRows = kGroupedActRows, kActThreads = 256, kAhead = 8;

// A workgroup takes rows of one expert and a strip of columns, a thread its own columns of them.
template <typename T>
__global__ void __launch_bounds__(kActThreads) grouped_act_kernel(GroupedActArgs a) {
  constexpr int VEC = kVec<T>, COLS = kActThreads * VEC;
  const int tiles_n = (int)((a.N + COLS - 1) / COLS);
  const GroupOffsets g{a.offsets, a.T, a.E, a.ids64};
  // The tile's number is its place among the partial sums: whole tiles of rows first, then the experts'
  // last ones.
  const int w = (int)block_of(), tile = w / tiles_n;
  const int64_t col = (int64_t)(w % tiles_n) * COLS + (int)threadIdx.x * VEC;
  const RowTiles tiles{g, kActRows, 0};
  int64_t whole, parts;
  tiles.total(&whole, &parts);
  const bool part = tile >= whole;
  RowTile t;
  // Past what the partial sums have room for: the grid's last workgroups, where offsets do not rise.
  if (tile >= grouped_act_tiles(a.T, a.E)) return;
  if (!tiles.find(part, part ? tile - whole : tile, &t)) return;
  if (col >= a.N) return;
  const int64_t end = min(t.first + kActRows, t.end);
  float sum[VEC] = {};
  const auto rows = [&](auto inside) {
    const auto get = [&](const void* p, int64_t ld, int64_t row) {
      const T* const from = static_cast<const T*>(p) + row * ld;
      if constexpr (decltype(inside)::value) return load_packed<T, VEC>(from + col);
      return load_guarded<T, VEC>(from, col, a.N);
    };
    for (int64_t row = t.first; row < end; row += kAhead) {
      // Rows past the last one are read as it is, and do not count.
      Packed<T, VEC> dy[kAhead], y[kAhead];
#pragma unroll
      for (int r = 0; r < kAhead; ++r) dy[r] = get(a.dy, a.lddy, min(row + r, end - 1));
      if (a.y)
#pragma unroll
        for (int r = 0; r < kAhead; ++r) y[r] = get(a.y, a.ldy, min(row + r, end - 1));
#pragma unroll
      for (int r = 0; r < kAhead; ++r) {
        if (row + r >= end) break;
        Packed<T, VEC> dz, up, down;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float d = (float)dy[r].v[e];
          const bool is_up = !a.y || (float)y[r].v[e] > 0.0f;
          const float v = is_up ? d : a.slope == 0.0f ? 0.0f : d * a.slope;
          dz.v[e] = (T)v;
          up.v[e] = is_up ? dy[r].v[e] : (T)0.0f;
          down.v[e] = is_up ? (T)0.0f : dy[r].v[e];
          sum[e] += v;
        }
        const auto put = [&](void* to, const Packed<T, VEC>& v) {
          store_guarded<T, VEC>(static_cast<T*>(to) + (row + r) * a.lddz, col, a.N, v);
        };
        if (a.dz) put(a.dz, dz);
        if (a.up) put(a.up, up), put(a.down, down);
      }
    }
  };
  // Loads in flight wait at a branch of their own: whole vectors have none.
  if (col + VEC <= a.N)
    rows(std::true_type{});
  else
    rows(std::false_type{});
  if (!a.db) return;
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (col + e < a.N) a.partials[(int64_t)tile * a.N + col + e] = sum[e];
}

// A wave has a quarter of an expert's tiles, successive ones, and a lane one column: sums of 2^20 bf16 rows of one expert
// and 64 columns, 32768 tiles, in 632 us, with one thread for all of a column's tiles in 1386; 8192 rows at 8 of 4096 columns
// in 20.8 and 21.3.
constexpr int kBiasWaves = 4;
__global__ void __launch_bounds__(64 * kBiasWaves) grouped_bias_kernel(GroupedActArgs a) {
  const GroupOffsets g{a.offsets, a.T, a.E, a.ids64};
  const int expert = blockIdx.y, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t n = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 64 + lane;
  const auto rows_of = [&](int e) { return max(g.at(e + 1) - g.at(e), (int64_t)0); };
  // The expert's whole tiles, and the place of its last one behind all whole tiles.
  int64_t before = 0, all = 0, parts = 0;
  for (int e = lane; e < a.E; e += 64) {
    const int64_t rows = rows_of(e);
    all += rows / kActRows;
    if (e < expert) before += rows / kActRows, parts += rows % kActRows != 0;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) before += __shfl_xor(before, d), all += __shfl_xor(all, d), parts += __shfl_xor(parts, d);
  const int64_t most = grouped_act_tiles(a.T, a.E);  // what the partial sums have room for
  const int64_t rows = rows_of(expert), tiles = min(rows / kActRows, max(most - before, (int64_t)0));
  // In 64 bits: their number does not add to the error of a tile's own sum, 31 roundings.
  double sum = 0.0;
  if (n < a.N) {
    const int64_t share = (tiles + kBiasWaves - 1) / kBiasWaves, end = min((wave + 1) * share, tiles);
    int64_t t = wave * share;
    for (; t + 8 <= end; t += 8) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = a.partials[(before + t + i) * a.N + n];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += (double)v[i];
    }
    for (; t < end; ++t) sum += (double)a.partials[(before + t) * a.N + n];
    if (wave == kBiasWaves - 1 && rows % kActRows != 0 && all + parts < most)
      sum += (double)a.partials[(all + parts) * a.N + n];
  }
  __shared__ double sums[kBiasWaves][64];
  sums[wave][lane] = sum;
  __syncthreads();
  if (wave != 0 || n >= a.N) return;
#pragma unroll
  for (int w = 1; w < kBiasWaves; ++w) sum += sums[w][lane];
  const float s = (float)sum;
  const int64_t at = expert * a.lddb + n;
  if (a.db_type == kF32)
    static_cast<float*>(a.db)[at] = s;
  else if (a.db_type == kBf16)
    static_cast<bf16*>(a.db)[at] = (bf16)s;
  else
    static_cast<f16*>(a.db)[at] = (f16)s;
}

template <typename T>
hipError_t launch_act_type(const GroupedActArgs& a, hipStream_t stream) {
  constexpr int COLS = kActThreads * kVec<T>;
  const int64_t tiles = grouped_act_tiles(a.T, a.E) * ((a.N + COLS - 1) / COLS);
  hipLaunchKernelGGL((grouped_act_kernel<T>), grid_of(tiles), dim3(kActThreads), 0, stream, a);
  return launched();
}

}  // namespace

hipError_t launch_grouped_act(const GroupedActArgs& a, hipStream_t stream) {
  if (a.T > 0) {
    const hipError_t e = a.type == kF32    ? launch_act_type<float>(a, stream)
                         : a.type == kBf16 ? launch_act_type<bf16>(a, stream)
                                           : launch_act_type<f16>(a, stream);
    if (e != hipSuccess) return e;
  }
  if (a.db) {
    const int64_t blocks = (a.N + 63) / 64, along = std::min<int64_t>(blocks, 1 << 20);  // under 2^32 threads an axis
    hipLaunchKernelGGL(grouped_bias_kernel, dim3((unsigned)along, (unsigned)a.E, (unsigned)((blocks + along - 1) / along)),
                       dim3(64 * kBiasWaves), 0, stream, a);
    return launched();
  }
  return hipSuccess;
}

}  // namespace lm
}  // namespace edsl

// The dense layer in 8-bit integers with a scale for each row of x and each column
// of W:
//   y[m][n] = epi(xs[m] ws[n] sum_k x[m][k] w[k][n] + b[n])
// Sums are 32-bit integers: exact for K < 2^17.
//
// Weights are laid out once in blocks of 16 columns x 64 k, the 1024 bytes that a
// wave's matrix instruction takes, successive k together: any load of them is one run.
//
// A few rows stream the weights (lm_skinny.hpp), bound by memory: 1 x 8192 x 8192 in 11.4 us, 5.9 TB/s (three sets
// of weights in turn stay in the Infinity Cache; the copy's rate is 5.2); at 33 x 4096 x 4097, 12.4 us, the way of
// eight blocks a wave one after the other is the time. More rows take tiles (lm_tile.hpp), bound by the matrix cores and their
// power: 4096 x 4096 x 4096 in 57.5 to 67 us by box, 2.0 to 2.4 POP/s (the vendor's product 69 to 86), 8192 x 8192 x 8192 in 480 (2.3). Rows of x
// off 16 bytes go through registers: 4097 x 4097 x 4097 in 137 to 142, since a turn's wait for its packed weights is also one
// for the two stages of x on their way.
#include "lm_kernels.hpp"
#include "lm_skinny.hpp"
#include "lm_tile.hpp"

namespace edsl {
namespace lm {
namespace {

// 64 k x 64 columns a workgroup; zeros past K and N.
__global__ void __launch_bounds__(256) i8_pack_kernel(I8PackArgs a) {
  __shared__ uint8_t t[64][64 + 4];
  const int64_t kblocks = i8_blocks(a.K), tiles = i8_tiles(a.N), groups = (tiles + 3) / 4;
  const int64_t w = block_of();
  if (w >= groups * kblocks) return;
  const int64_t kb = w % kblocks, n0 = w / kblocks * 64;
  const int tid = threadIdx.x;
  {
    const int64_t k = kb * 64 + tid / 4, n = n0 + tid % 4 * 16;
    Packed<int8_t, 16> v{};
    if (k < a.K && n < a.N) v = load_guarded<int8_t, 16>(a.q + k * a.ldq, n, a.N);
#pragma unroll
    for (int e = 0; e < 16; ++e) t[tid / 4][tid % 4 * 16 + e] = (uint8_t)v.v[e];
  }
  __syncthreads();
  const int64_t tile = n0 / 16 + tid / 64;
  const int lane = tid % 64;
  if (tile < tiles) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        r[i] |= (uint32_t)t[lane / 16 * 16 + 4 * i + e][tid / 64 * 16 + lane % 16] << (8 * e);
    }
    *reinterpret_cast<u32x4*>(a.packed + (tile * kblocks + kb) * 1024 + lane * 16) = r;
    if (kb == 0 && lane < 16) {
      const int64_t n = tile * 16 + lane;
      reinterpret_cast<float*>(a.packed + i8_scales_at(a.K, a.N))[n] =
          n < a.N ? get_typed(a.scales, n, a.scale_type) : 0.0f;
    }
  }
}

template <typename Tl>
__device__ __forceinline__ void i8_tile(const I8Args& a, int m0, int n0, u32x4* lds) {
  const int64_t tile_bytes = i8_blocks(a.K) * 1024;
  const TileOperand oa{reinterpret_cast<const char*>(a.x) + m0 * a.ldx, a.ldx, min(a.M - m0, Tl::BM), a.M};
  const TileOperand ob{a.w + n0 / 16 * tile_bytes, tile_bytes, min(a.N - n0, Tl::BN), a.N};
  typename Tl::Acc acc[Tl::MI][Tl::NI];
  Tl::product(oa, ob, a.K, lds, acc);
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  float xs[Tl::MI];
#pragma unroll
  for (int i = 0; i < Tl::MI; ++i) {
    const int m = m0 + 16 * (wave / Tl::WN * Tl::MI + i) + lane % 16;
    xs[i] = a.x_scales && m < a.M ? a.x_scales[m] : 1.0f;
  }
  const auto finish = [&](float (&v)[4], i32x4 sum, f32x4 ws, float scale, const float (&bias)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = (float)sum[e] * ws[e] * scale;
      if (a.bias) v[e] = __fadd_rn(v[e], bias[e]);
    }
    activate(v, a.epi, a.alpha);
  };
#pragma unroll
  for (int j = 0; j < Tl::NI; j += 2) {
    const int first = n0 + 16 * (wave % Tl::WN * Tl::NI + j), n = first + 4 * (lane / 16);
    float bias[2][4] = {};
    f32x4 ws[2] = {};
#pragma unroll
    for (int b = 0; b < 2; ++b)
      if (n + 16 * b < a.N) {
        if (a.bias) get4_typed(a.bias, n + 16 * b, a.bias_type, bias[b], a.N - n - 16 * b);
        ws[b] = *reinterpret_cast<const f32x4*>(a.w_scales + n + 16 * b);  // kept for whole blocks of 16
      }
#pragma unroll
    for (int i = 0; i < Tl::MI; ++i) {
      const int m = m0 + 16 * (wave / Tl::WN * Tl::MI + i);
      float v0[4], v1[4];
      finish(v0, acc[i][j], ws[0], xs[i], bias[0]);
      finish(v1, acc[i][j + 1], ws[1], xs[i], bias[1]);
      if (a.y_type == kF32)
        put_blocks(static_cast<float*>(a.y) + m * a.ldy, a.ldy, a.M - m, first, a.N, v0, v1);
      else if (a.y_type == kBf16)
        put_blocks(static_cast<bf16*>(a.y) + m * a.ldy, a.ldy, a.M - m, first, a.N, v0, v1);
      else
        put_blocks(static_cast<f16*>(a.y) + m * a.ldy, a.ldy, a.M - m, first, a.N, v0, v1);
    }
  }
}

// Big tiles, and Half and Quarter ones for what is left of a round of the CUs.
template <typename Big, typename Half, typename Quarter>
__global__ void __launch_bounds__(Big::kThreads, Big::kWavesPerSimd) i8_tile_kernel(I8Args a) {
  constexpr int kLds = Big::kLds > Half::kLds ? (Big::kLds > Quarter::kLds ? Big::kLds : Quarter::kLds)
                                              : (Half::kLds > Quarter::kLds ? Half::kLds : Quarter::kLds);
  __shared__ u32x4 lds[kLds];
  const int tiles_m = (a.M + Big::BM - 1) / Big::BM, tiles_n = (a.N + Big::BN - 1) / Big::BN;
  TileTurn turn;
  if (!tile_turn((int)block_of(), tiles_m * tiles_n, tiles_m * tiles_n, a.rounds, &turn)) return;
  int tn;
  int m0 = row_of_tile(turn.tile, tiles_m, tiles_n, &tn) * Big::BM, n0 = tn * Big::BN;
  if (turn.pieces == 1) return i8_tile<Big>(a, m0, n0, lds);
  n0 += turn.sub % 2 * (Big::BN / 2);
  m0 += turn.sub / 2 * (Big::BM / 2);
  if (n0 >= a.N || m0 >= a.M) return;
  if constexpr (!std::is_same<Big, Quarter>::value) {
    if (turn.pieces == 2) return i8_tile<Half>(a, m0, n0, lds);
    i8_tile<Quarter>(a, m0, n0, lds);
  }
}

template <int MT, int NJ, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) i8_skinny_kernel(I8Args a) {
  // Few operands a block are read further ahead: 33 x 4096 x 4097 in 12.4 us with two blocks of weights on
  // their way, with one in 14.0; 1 x 8192 x 8192 in 11.3 with one of four steps, in 11.9 with two.
  constexpr int U = MT * NJ == 1 ? 4 : MT * NJ <= 8 && MT < 4 ? 2 : 1;
  constexpr int AHEAD = MT * NJ == 1 || NJ == 4 || (NJ == 1 && MT > 2) ? 1 : 2;
  using S = Skinny<int8_t, kBlocks, MT, NJ, WAVES, U, AHEAD>;
  __shared__ typename S::Acc lds[S::kSlots];
  const int m0 = (int)blockIdx.y * 16 * MT;
  S::run(a.x + m0 * a.ldx, a.ldx, min(a.M - m0, 16 * MT), a.w, i8_blocks(a.K) * 1024, a.K, a.N,
         (int)blockIdx.x * S::kCols16, lds, [&](int m, int n, int sum) {
           m += m0;
           float v[1] = {(float)sum * a.w_scales[n] * (a.x_scales ? a.x_scales[m] : 1.0f)};
           if (a.bias) v[0] = __fadd_rn(v[0], get_typed(a.bias, n, a.bias_type));
           activate(v, a.epi, a.alpha);
           const int64_t at = m * a.ldy + n;
           if (a.y_type == kF32)
             static_cast<float*>(a.y)[at] = v[0];
           else if (a.y_type == kBf16)
             static_cast<bf16*>(a.y)[at] = (bf16)v[0];
           else
             static_cast<f16*>(a.y)[at] = (f16)v[0];
         });
}

template <typename Big, typename Half = Big, typename Quarter = Half>
hipError_t launch_tiles(I8Args a, int quarters, int halves, hipStream_t stream) {
  const int64_t tiles = (int64_t)((a.M + Big::BM - 1) / Big::BM) * ((a.N + Big::BN - 1) / Big::BN);
  a.rounds = {a.cus, quarters, halves};
  hipLaunchKernelGGL((i8_tile_kernel<Big, Half, Quarter>), grid_of(tile_turns(tiles, a.rounds)), dim3(Big::kThreads), 0,
                     stream, a);
  return launched();
}

// 64 columns: of up to 32 rows. What no kernel is made for is an error: Y would keep what it held.
template <int MT>
hipError_t launch_skinny(const I8Args& a, int cols16, hipStream_t stream) {
  constexpr int kWaves = 8;
  if (cols16 != 1 && cols16 != 2 && (cols16 != 4 || MT > 2)) return hipErrorInvalidValue;
  const dim3 grid((unsigned)((a.N + 16 * cols16 - 1) / (16 * cols16)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
  if (cols16 == 1)
    hipLaunchKernelGGL((i8_skinny_kernel<MT, 1, kWaves>), grid, dim3(64 * kWaves), 0, stream, a);
  else if (cols16 == 2)
    hipLaunchKernelGGL((i8_skinny_kernel<MT, 2, kWaves>), grid, dim3(64 * kWaves), 0, stream, a);
  else if constexpr (MT <= 2)
    hipLaunchKernelGGL((i8_skinny_kernel<MT, 4, kWaves>), grid, dim3(64 * kWaves), 0, stream, a);
  return launched();
}

}  // namespace

hipError_t launch_i8_pack(const I8PackArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(i8_pack_kernel, grid_of((i8_tiles(a.N) + 3) / 4 * i8_blocks(a.K)), dim3(256), 0, stream, a);
  return launched();
}

hipError_t launch_i8_tile(const I8Args& a, bool direct, hipStream_t stream) {
  if (!direct) return launch_tiles<Tile<int8_t, kRows, kBlocks, 128, 128, 2, 4, false>>(a, 0, 0, stream);
  return launch_tiles<Tile<int8_t, kRows, kBlocks, 256, 256, 2, 4, true>, Tile<int8_t, kRows, kBlocks, 256, 128, 4, 2, true, 3>,
                      Tile<int8_t, kRows, kBlocks, 128, 128, 2, 4, true, 3>>(a, a.cus / 4, a.cus / 2, stream);
}

hipError_t launch_i8_skinny(const I8Args& a, int rows16, int cols16, hipStream_t stream) {
  if (rows16 == 1) return launch_skinny<1>(a, cols16, stream);
  if (rows16 == 2) return launch_skinny<2>(a, cols16, stream);
  if (rows16 == 3) return launch_skinny<3>(a, cols16, stream);
  if (rows16 == 4) return launch_skinny<4>(a, cols16, stream);
  return hipErrorInvalidValue;
}

}  // namespace lm
}  // namespace edsl

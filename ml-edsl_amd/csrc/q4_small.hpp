// The 4-bit layer on up to 16 rows: the weights' bytes are the time.
//
// A workgroup of 8 waves takes NT tiles of 16 columns; its waves split K by
// blocks of 128 in turn, so that together they read 8 KB runs of a tile. A
// wave's 16-byte load of a lane is its operand for four matrix instructions.
// Rows of x come straight from the caches, in operand order; rows past M repeat
// the last one. The sums of x that the zero points multiply are a matrix
// instruction with a constant operand. The waves' sums meet in LDS.
#pragma once

#include "q4.hpp"

namespace edsl {
namespace lm {

constexpr int kSmallWaves = 8;

template <int XT>
struct SmallX;  // planes; the raw vector of 8 elements; its operands

template <>
struct SmallX<kBf16> {
  using T = bf16;
  using E = Q4Elem<false>;
  static constexpr int kPlanes = 1;
  static __device__ __forceinline__ void operands(const Packed<T, 8>& r, bf16x8 (&o)[1]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[0][j] = r.v[j];
  }
};
template <>
struct SmallX<kF16> {
  using T = f16;
  using E = Q4Elem<true>;
  static constexpr int kPlanes = 1;
  static __device__ __forceinline__ void operands(const Packed<T, 8>& r, f16x8 (&o)[1]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[0][j] = r.v[j];
  }
};
template <>
struct SmallX<kF32> {
  using T = float;
  using E = Q4Elem<false>;
  static constexpr int kPlanes = 3;
  static __device__ __forceinline__ void operands(const Packed<T, 8>& r, bf16x8 (&o)[3]) {
    u32x4 p[3];
    split3_operands(r.v, p);
#pragma unroll
    for (int i = 0; i < 3; ++i) o[i] = __builtin_bit_cast(bf16x8, p[i]);
  }
};
template <>
struct SmallX<kI8> {
  using T = int8_t;
  using E = Q4Elem<false>;
  static constexpr int kPlanes = 1;
  static __device__ __forceinline__ void operands(const Packed<T, 8>& r, bf16x8 (&o)[1]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[0][j] = (bf16)(float)r.v[j];
  }
};
template <>
struct SmallX<kE4m3> {
  using T = uint8_t;
  using E = Q4Elem<false>;
  static constexpr int kPlanes = 1;
  static __device__ __forceinline__ void operands(const Packed<T, 8>& r, bf16x8 (&o)[1]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) w |= (uint32_t)r.v[4 * h + j] << (8 * j);
      const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
      const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
      o[0][4 * h] = a[0], o[0][4 * h + 1] = a[1], o[0][4 * h + 2] = b[0], o[0][4 * h + 3] = b[1];
    }
  }
};

// What a wave reads of one block.
template <int XT, int NT, int SPB, bool ZEROS>
struct SmallBlock {
  Packed<typename SmallX<XT>::T, 8> x[4];
  u32x4 w[NT];
  uint32_t scale[NT][SPB], zero[ZEROS ? NT : 1][SPB];  // as read
};

template <int XT, int NT, int SPB, bool ZEROS>
__device__ __forceinline__ void small_load(const Q4Args& a, const typename SmallX<XT>::T* x, int64_t tile, int block,
                                           int lane, SmallBlock<XT, NT, SPB, ZEROS>& r) {
  const int k0 = 128 * block + 8 * (lane / 16);
#pragma unroll
  for (int s = 0; s < 4; ++s) r.x[s] = load_guarded<typename SmallX<XT>::T, 8>(x, k0 + 32 * s, a.K);
  const int sb = block / a.blocks_per_scale;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    r.w[t] = *reinterpret_cast<const u32x4*>(a.w + ((tile + t) * a.blocks + block) * 1024 + 16 * lane);
    const int64_t at = (((tile + t) * a.scale_blocks + sb) * 16 + lane % 16) * SPB;
#pragma unroll
    for (int g = 0; g < SPB; ++g) {
      r.scale[t][g] = q4_scale_bits(a.w + a.scales_at, a.scale_bytes, at + g);
      if constexpr (ZEROS) r.zero[t][g] = reinterpret_cast<const uint8_t*>(a.w + a.zeros_at)[at + g];
    }
  }
}

template <int XT, int NT, int SPB, bool ZEROS>
__device__ __forceinline__ void small_block(const Q4Args& a, const SmallBlock<XT, NT, SPB, ZEROS>& r,
                                            f32x4 (&sum)[NT]) {
  using X = SmallX<XT>;
  using V = typename X::E::V;
  constexpr int STEPS = 4 / SPB;
  V minus;  // the constant operand of the sums of x
#pragma unroll
  for (int j = 0; j < 8; ++j) minus[j] = ZEROS ? -1.0f : -8.0f - q4_offset(XT);
#pragma unroll
  for (int g = 0; g < SPB; ++g) {
    V o[STEPS][X::kPlanes];
    f32x4 xs = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      X::operands(r.x[g * STEPS + s], o[s]);
#pragma unroll
      for (int p = X::kPlanes - 1; p >= 0; --p) xs = X::E::mfma(o[s][p], minus, xs);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f32x4 acc = xs;
      if constexpr (ZEROS) {
        const float zero = q4_offset(XT) + (float)r.zero[t][g];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= zero;
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        V w;
        if constexpr (XT == kF32)
          w = q4_weights_f32(r.w[t][g * STEPS + s]);
        else
          w = q4_weights<XT == kF16>(r.w[t][g * STEPS + s]);
#pragma unroll
        for (int p = X::kPlanes - 1; p >= 0; --p) acc = X::E::mfma(o[s][p], w, acc);
      }
      const float scale = q4_scale(r.scale[t][g], a.scale_type);
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[t][i] = fmaf(acc[i], scale, sum[t][i]);
    }
  }
}

template <int XT, int NT, int SPB, bool ZEROS>
__global__ void __launch_bounds__(64 * kSmallWaves) q4_small_kernel(Q4Args a) {
  using T = typename SmallX<XT>::T;
  __shared__ float part[kSmallWaves][16][16 * NT];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int64_t tiles = (a.N + 15) / 16;
  const int64_t first = (int64_t)(blockIdx.x / a.ksplit) * NT;
  const int slice = blockIdx.x % a.ksplit;
  // The last workgroup's tiles may reach past the end: it repeats the last ones
  // and stores each column once.
  const int64_t tile = first + NT <= tiles ? first : (tiles > NT ? tiles - NT : 0);
  const int b0 = (int)((int64_t)a.blocks * slice / a.ksplit), b1 = (int)((int64_t)a.blocks * (slice + 1) / a.ksplit);
  const int row = lane % 16 < a.M ? lane % 16 : a.M - 1;
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
  f32x4 sum[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) sum[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  SmallBlock<XT, NT, SPB, ZEROS> now, next;
  int b = b0 + wave;
  if (b < b1) small_load<XT, NT, SPB, ZEROS>(a, x, tile, b, lane, now);
  while (b < b1) {
    const int after = b + kSmallWaves;
    if (after < b1) small_load<XT, NT, SPB, ZEROS>(a, x, tile, after, lane, next);
    small_block<XT, NT, SPB, ZEROS>(a, now, sum);
    now = next;
    b = after;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = 4 * (lane / 16) + i;
      if (m < a.M) part[wave][m][16 * t + lane % 16] = sum[t][i];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < a.M * 16 * NT; i += 64 * kSmallWaves) {
    const int m = i / (16 * NT), c = i % (16 * NT);
    const int64_t n = 16 * tile + c;
    if (n >= a.N || n < 16 * first) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kSmallWaves; ++w) v += part[w][m][c];
    if (a.ksplit > 1) {
      a.partials[((int64_t)slice * a.M + m) * a.N + n] = v;
    } else {
      float out[1] = {v};
      q4_store<1>(a, {m}, {(int)n}, {true}, out);
    }
  }
}

template <int XT, int NT, int SPB>
hipError_t launch_small_zeros(const Q4Args& a, bool zeros, hipStream_t stream) {
  const int64_t tiles = (a.N + 15) / 16;
  const dim3 grid((unsigned)((tiles + NT - 1) / NT * a.ksplit)), block(64 * kSmallWaves);
  if (zeros)
    hipLaunchKernelGGL((q4_small_kernel<XT, NT, SPB, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((q4_small_kernel<XT, NT, SPB, false>), grid, block, 0, stream, a);
  return launched();
}

template <int XT, int NT>
hipError_t launch_small_spb(const Q4Args& a, int spb, bool zeros, hipStream_t stream) {
  if (spb == 4) return launch_small_zeros<XT, NT, 4>(a, zeros, stream);
  if (spb == 2) return launch_small_zeros<XT, NT, 2>(a, zeros, stream);
  return launch_small_zeros<XT, NT, 1>(a, zeros, stream);
}

template <int XT>
hipError_t launch_q4_small(const Q4Args& a, int nt, int spb, bool zeros, hipStream_t stream) {
  if (nt == 4) return launch_small_spb<XT, 4>(a, spb, zeros, stream);
  if (nt == 2) return launch_small_spb<XT, 2>(a, spb, zeros, stream);
  return launch_small_spb<XT, 1>(a, spb, zeros, stream);
}

}  // namespace lm
}  // namespace edsl

// Device helpers of the language-model operators: element types of 16 and 8
// bits, vectors of any alignment, sums over a wave and a workgroup.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace edsl {
namespace lm {

typedef __bf16 bf16;
typedef _Float16 f16;

// The elements of one 16-byte vector, the unit of every load and store below.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// A vector at an address aligned to its element only: rows start anywhere. The
// hardware takes 16-byte accesses at any address.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Packed {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Packed<T, N> load_packed(const T* p) {
  return *reinterpret_cast<const Packed<T, N>*>(p);
}

// Elements i0 .. i0+VEC-1 of a row of n, `fill` past its end.
template <typename T, int VEC>
__device__ __forceinline__ Packed<T, VEC> load_guarded(const T* row, int64_t i0, int64_t n, T fill = T(0)) {
  if (i0 + VEC <= n) return load_packed<T, VEC>(row + i0);
  Packed<T, VEC> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = i0 + e < n ? row[i0 + e] : fill;
  return r;
}

// A vector that this kernel does not read again, past the caches' order of use: the
// norm of 4096 x 8192 bf16 to 8 bits in 44 us, with plain stores in 51, its backward
// pass of 4096 x 4096 in 33.4 against 35.8; what reads the result next is no slower.
template <typename T, int N>
__device__ __forceinline__ void store_streamed(T* p, const Packed<T, N>& r) {
  static_assert(sizeof(r) % 4 == 0, "whole words");
  typedef uint32_t Words __attribute__((ext_vector_type(sizeof(r) / 4)));
  typedef Words Aligned __attribute__((aligned(sizeof(T))));
  __builtin_nontemporal_store(__builtin_bit_cast(Words, r), reinterpret_cast<Aligned*>(p));
}
template <typename T, int VEC>
__device__ __forceinline__ void store_guarded(T* row, int64_t i0, int64_t n, const Packed<T, VEC>& r) {
  if (i0 + VEC <= n) {
    store_streamed<T, VEC>(row + i0, r);
    return;
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    if (i0 + e < n) row[i0 + e] = r.v[e];
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

struct Sum {
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
// NaN loses.
struct Max {
  static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};
// NaN wins (v_maximum3_f32).
struct MaxNan {
  static __device__ __forceinline__ float of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
};

// The combination over runs of LANES lanes (16, 32, 64): lanes 1 and 2 apart,
// mirrored in 8 and in 16 by DPP, then 16 and 32 apart. Every lane of a run has the
// same bits: both sides of each step add the same two values, which holds as long
// as the compiler does not fuse the caller's product into its side of the first.
template <typename Op, int LANES>
__device__ __forceinline__ float lanes_all(float v) {
  asm("" : "+v"(v));
  v = Op::of(v, dpp<0xB1>(v));
  v = Op::of(v, dpp<0x4E>(v));
  v = Op::of(v, dpp<0x141>(v));
  v = Op::of(v, dpp<0x140>(v));
  if constexpr (LANES > 16) v = Op::of(v, __shfl_xor(v, 16));
  if constexpr (LANES > 32) v = Op::of(v, __shfl_xor(v, 32));
  return v;
}
// Over the wave, in a scalar register.
template <typename Op>
__device__ __forceinline__ float wave_all(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, lanes_all<Op, 64>(v))));
}

// A grid of n workgroups along x and y: a launch takes less than 2^32 threads along
// each. block_of() numbers them; the last ones may be past n, which is less than 2^31.
inline dim3 grid_of(int64_t n) {
  constexpr int64_t kRow = int64_t(1) << 20;
  return n <= kRow ? dim3((unsigned)n) : dim3((unsigned)kRow, (unsigned)((n + kRow - 1) / kRow));
}
__device__ __forceinline__ uint32_t block_of() { return blockIdx.y * gridDim.x + blockIdx.x; }

// hipSuccess or the first error of a launch.
inline hipError_t launched() { return hipGetLastError(); }

}  // namespace lm
}  // namespace edsl

// The dense layer on 4-bit weights: the layout of packed weights, and what the
// kernels of it share.
//
//   y = epi(xs[m] * sum_k x[m][k] s[g][n] (q[k][n] - z[g][n]) + b[n]),  g = k / group
//
// Products are exact: q in 0..15 and the integers of an 8-bit x are exact in
// bf16 (q in f16 too), bf16 and f16 x are what the matrix cores take, and an
// f32 x is the exact sum of three bf16 terms. Sums are 32-bit. Inside a group
//   sum x (q - z) = sum x q - z sum x,
// with the second term the starting value of the accumulator, so that a weight
// is never rounded: its scale multiplies the group's sum.
#pragma once

#include "common.hpp"
#include "lm_common.hpp"
#include "lm_kernels.hpp"

namespace edsl {
namespace lm {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Packed weights: blocks of 16 columns x 128 k, [N/16][K/128] rounded up, 1024
// bytes each: lane l of a wave has 16 bytes, column l % 16, and word s of them
// holds k = 32 s + 8 (l / 16) + j, j = 0..3 in the low and j = 4..7 in the high
// nibbles of its bytes. That is the operand of the 16x16x32 matrix instruction,
// lane for lane, four in a row: a wave's load is one 1024-byte line of memory.
// Behind them the scales [N/16][SB][16][spb] and zero points likewise in bytes:
// spb = 128 / group scales of a column in a block and SB = K/128 where the group
// is less than 128, else spb = 1 and SB = K/group. All padding is zero.
struct Q4Layout {
  int64_t tiles_n, blocks, scale_blocks;
  int spb, blocks_per_scale, scale_bytes;
  bool zeros;
  int64_t scales_at, zeros_at, bytes;
};

inline Q4Layout q4_layout(int64_t K, int64_t N, int group, int scale_type, bool zeros) {
  Q4Layout l{};
  l.tiles_n = (N + 15) / 16;
  l.blocks = (K + 127) / 128;
  l.spb = group < 128 ? 128 / group : 1;
  l.blocks_per_scale = group < 128 ? 1 : group / 128;
  l.scale_blocks = (l.blocks + l.blocks_per_scale - 1) / l.blocks_per_scale;
  l.scale_bytes = type_bytes(scale_type);
  l.zeros = zeros;
  const int64_t scales = l.tiles_n * l.scale_blocks * 16 * l.spb;
  l.scales_at = l.tiles_n * l.blocks * 1024;
  l.zeros_at = l.scales_at + (scales * l.scale_bytes + 255) / 256 * 256;
  l.bytes = l.zeros_at + (zeros ? (scales + 255) / 256 * 256 : 0);
  return l;
}

struct Q4Args {
  const void* x;
  const float* x_scales;  // or nullptr
  const char* w;          // packed
  const void* bias;       // or nullptr
  void* y;
  float* partials;  // [ksplit][M][N] sums where ksplit > 1
  int64_t ldx, ldy, scales_at, zeros_at;
  int M, N, K;
  int blocks, scale_blocks, blocks_per_scale;
  int ksplit;  // workgroups that split K
  int x_type, scale_type, y_type, bias_type, epi;
  float alpha;
  // Tiles of many rows: x prepared (q4_prep_kernel), or x itself where its rows
  // are whole 16-byte aligned blocks.
  const void* xp;       // [planes][M][ldp]
  int64_t ldp, plane;   // elements
  const float* xs;      // [blocks * spb][xs_ld]: minus (8 times, without zero points) the sums of x in each group
  int64_t xs_ld;
};

template <bool F16>
struct Q4Elem;
template <>
struct Q4Elem<false> {
  using V = bf16x8;
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // Eight weights of a word. As an 8-bit float of 4 exponent bits the byte n in
  // 0..15 is n / 512 (0..7 subnormal), so that the conversion with a factor of
  // 512 gives n: 7 instructions for 8 weights, no table.
  static __device__ __forceinline__ V weights(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
    return V{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};
template <>
struct Q4Elem<true> {
  using V = f16x8;
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ V weights(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false);
    const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true);
    const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false);
    const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true);
    return V{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
};

// Scale i of an array of this type, as f32.
__device__ __forceinline__ float q4_scale(const char* p, int type, int64_t i) {
  if (type == kF32) return reinterpret_cast<const float*>(p)[i];
  const uint32_t h = reinterpret_cast<const uint16_t*>(p)[i];
  if (type == kBf16) return __builtin_bit_cast(float, h << 16);
  return (float)__builtin_bit_cast(f16, (uint16_t)h);
}

// Three bf16 terms whose sum is v, to the last bit of it while they are normal:
// each takes the leading 8 bits of what is left, cut off.
struct Split3 {
  uint32_t hi, mid, lo;  // in the upper halves
};
__device__ __forceinline__ Split3 split3(float v) {
  Split3 r;
  r.hi = __builtin_bit_cast(uint32_t, v) & 0xffff0000u;
  const float a = v - __builtin_bit_cast(float, r.hi);
  r.mid = __builtin_bit_cast(uint32_t, a) & 0xffff0000u;
  const float b = a - __builtin_bit_cast(float, r.mid);
  r.lo = __builtin_bit_cast(uint32_t, b) & 0xffff0000u;
  return r;
}

__device__ __forceinline__ float q4_load_as_float(const void* p, int type, int64_t i) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  if (type == kBf16) return (float)static_cast<const bf16*>(p)[i];
  return (float)static_cast<const f16*>(p)[i];
}

// y[m][n] from the sum over k.
__device__ __forceinline__ void q4_store(const Q4Args& a, int m, int n, float v) {
  if (a.x_scales) v *= a.x_scales[m];
  const float b = a.bias ? q4_load_as_float(a.bias, a.bias_type, n) : 0.0f;
  v = epilogue_rt(v, b, a.alpha, a.epi);
  const int64_t at = (int64_t)m * a.ldy + n;
  if (a.y_type == kF32)
    static_cast<float*>(a.y)[at] = v;
  else if (a.y_type == kBf16)
    static_cast<bf16*>(a.y)[at] = (bf16)v;
  else
    static_cast<f16*>(a.y)[at] = (f16)v;
}

// q4_small.hpp, one source file for each type of x.
template <int XT>
hipError_t launch_q4_small(const Q4Args& a, int nt, int spb, bool zeros, hipStream_t stream);
// q4_tile.hip; f32 has the first two only.
enum : int { kQ4Tile32x128 = 0, kQ4Tile64x128 = 1, kQ4Tile128x128 = 2 };
hipError_t launch_q4_tile(const Q4Args& a, int config, int spb, bool zeros, hipStream_t stream);
struct Q4PrepArgs {
  const void* x;
  void* xp;  // or nullptr: sums only
  float* xs;
  int64_t ldx, ldp, plane, xs_ld;
  int M, K, blocks, spb, x_type;
  float factor;  // of the sums: -1, or -8 without zero points
};
hipError_t launch_q4_prep(const Q4PrepArgs& a, hipStream_t stream);
hipError_t launch_q4_join(const Q4Args& a, hipStream_t stream);
struct Q4PackArgs {
  const uint8_t* q;      // [K][N], row stride ldq
  const void* scales;    // [G][N], row stride lds
  const uint8_t* zeros;  // [G][N], row stride ldz, or nullptr
  char* packed;
  int64_t ldq, lds, ldz;
  int64_t K, N;
  int group, scale_type;
  Q4Layout layout;
};
hipError_t launch_q4_pack(const Q4PackArgs& a, hipStream_t stream);

}  // namespace lm
}  // namespace edsl

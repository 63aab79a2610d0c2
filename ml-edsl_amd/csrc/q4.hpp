// The dense layer on 4-bit weights: the layout of packed weights, and what the
// kernels of it share.
//
//   y = epi(xs[m] * sum_k x[m][k] s[g][n] (q[k][n] - z[g][n]) + b[n]),  g = k / group
//
// Products are exact: q in 0..15 and the integers of an 8-bit x are exact in
// bf16 and f16, bf16 and f16 x are what the matrix cores take, and an
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
// holds k = 32 s + 8 (l / 16) + j, even j in nibble j / 2 of its lower half, odd
// ones in the upper half's. That is the operand of the 16x16x32 matrix
// instruction, lane for lane, four in a row: a wave's load is one 1024-byte run.
// Behind them the scales [N/16][SB][16][spb] and the zero points in bytes likewise:
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
  // At the end room for what a 32-bit load of the last scale reads past it, and,
  // without zero points, an 8 that stands for all of them.
  l.bytes = l.zeros_at + (zeros ? (scales + 255) / 256 * 256 : 0);
  if (l.bytes > 0) l.bytes += 256;
  return l;
}

// Which reading of a scale's bits is kept (q4_scale).
struct Q4ScaleMask {
  uint32_t f32, bf16, f16;
};
inline Q4ScaleMask q4_scale_mask(int type) {
  return {type == kF32 ? ~0u : 0u, type == kBf16 ? ~0u : 0u, type == kF16 ? ~0u : 0u};
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
  int blocks, scale_blocks;
  uint32_t scale_magic;  // block / blocks_per_scale = block * magic >> 32, blocks up to 2^16
  int ksplit;  // workgroups that split K
  int slice_blocks;  // blocks of a slice of K (the last may have fewer)
  int scale_bytes;
  int64_t zero_step;  // of a group's zero point: 1, or 0 where all are the one at zeros_at
  int x_type, y_type, bias_type, epi;
  Q4ScaleMask scale_mask;
  float alpha;
  // Tiles of many rows: x prepared (q4_prep_kernel), or x itself where its rows
  // are whole 16-byte aligned blocks of 16 bits.
  const void* xp;       // [planes][M][ldp]
  int64_t ldp, plane;   // elements
  const float* xs;      // [blocks][xs_ld / 16][spb][16]: minus the sums of x in each group, times offset + 8 without zero points
  int64_t xs_ld;
};

__device__ __forceinline__ int q4_scale_block(const Q4Args& a, int block) {
  return a.scale_magic ? (int)__umulhi((uint32_t)block, a.scale_magic) : block;
}

template <bool F16>
struct Q4Elem;
template <>
struct Q4Elem<false> {
  using V = bf16x8;
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static constexpr int kShift = 3;            // of a weight in the mantissa of 16 .. 31
  static constexpr uint32_t kBase = 0x41804180u;  // 16, twice
};
template <>
struct Q4Elem<true> {
  using V = f16x8;
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static constexpr int kShift = 6;
  static constexpr uint32_t kBase = 0x4c004c00u;
};

// Eight weights of a word, in the order of k, as kQ4Offset + q: in the mantissa
// of 16 .. 31 an integer 0 .. 15 is its own bits, so two weights cost one shift
// and one and-or, and the 16 goes with the zero point. The sums then hold
// 16 sum x more than they need, which costs up to two of their bits.
constexpr float kQ4Offset = 16.0f;
template <bool F16>
__device__ __forceinline__ typename Q4Elem<F16>::V q4_weights(uint32_t w) {
  using E = Q4Elem<F16>;
  // One of the two constants in a vector register: an instruction takes one scalar.
  const uint32_t mask = (15u << E::kShift) * 0x10001u;
  uint32_t base = E::kBase;
  asm("" : "+v"(base));
  u32x4 r;
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int s = 4 * p - E::kShift;
    r[p] = ((s >= 0 ? w >> s : w << -s) & mask) | base;
  }
  return __builtin_bit_cast(typename E::V, r);
}
// For f32 x, as q itself: as an 8-bit float of 4 exponent bits the byte n in
// 0 .. 15 is n / 512 (0 .. 7 subnormal), so the conversion with a factor of 512
// gives n. They come in the order k = 0 4 1 5 2 6 3 7, in which x is split too.
__device__ __forceinline__ bf16x8 q4_weights_f32(uint32_t w) {
  const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// What a weight is held above q for x of this type.
constexpr float q4_offset(int x_type) { return x_type == kF32 ? 0.0f : kQ4Offset; }

// A scale as it lies in memory: 32 bits from its address on (the packed weights'
// end leaves room). Read one way for all types and decoded where it is used, so
// that no load waits at a branch. `row`: uniform, of a tile's column 0 and first
// group; the lane's part of the address is 32 bits.
__device__ __forceinline__ uint32_t q4_scale_bits(const char* row, uint32_t offset) {
  const auto v = load_packed<uint16_t, 2>(reinterpret_cast<const uint16_t*>(row + offset));
  return v.v[0] | (uint32_t)v.v[1] << 16;
}
// All three readings, one kept: a branch would wait for the load.
__device__ __forceinline__ float q4_scale(uint32_t bits, const Q4ScaleMask& k) {
  const uint32_t half = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(f16, (uint16_t)bits));
  return __builtin_bit_cast(float, (bits & k.f32) | ((bits << 16) & k.bf16) | (half & k.f16));
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

// Eight elements of an f32 x as operands of three products, in the order of
// q4_weights_f32.
__device__ __forceinline__ void split3_operands(const float (&v)[8], u32x4 (&p)[3]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const Split3 a = split3(v[j]), b = split3(v[j + 4]);
    p[0][j] = (a.hi >> 16) | b.hi;
    p[1][j] = (a.mid >> 16) | b.mid;
    p[2][j] = (a.lo >> 16) | b.lo;
  }
}

__device__ __forceinline__ float q4_load_as_float(const void* p, int type, int64_t i) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  if (type == kBf16) return (float)static_cast<const bf16*>(p)[i];
  return (float)static_cast<const f16*>(p)[i];
}

// Writes C outputs of a lane, y[m[i]][n[i]], from their sums over k; `in`: those
// that exist. The branches are taken once for all of them.
template <int C>
__device__ __forceinline__ void q4_store(const Q4Args& a, const int (&m)[C], const int (&n)[C], const bool (&in)[C],
                                         float (&v)[C]) {
  if (a.x_scales)
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (in[i]) v[i] *= a.x_scales[m[i]];
  if (a.bias)
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (in[i]) v[i] = __fadd_rn(v[i], q4_load_as_float(a.bias, a.bias_type, n[i]));
  switch (epi_act(a.epi)) {
    case ACT_RELU:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = apply_epilogue_f32<epi_code(false, ACT_RELU)>(v[i], 0.0f, 0.0f);
      break;
    case ACT_LEAKY:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = apply_epilogue_f32<epi_code(false, ACT_LEAKY)>(v[i], 0.0f, a.alpha);
      break;
    case ACT_IF_RELU:
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] = apply_epilogue_f32<epi_code(false, ACT_IF_RELU)>(v[i], 0.0f, 0.0f);
      break;
    default:
      break;
  }
  if (a.y_type == kF32) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (in[i]) static_cast<float*>(a.y)[(int64_t)m[i] * a.ldy + n[i]] = v[i];
  } else if (a.y_type == kBf16) {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (in[i]) static_cast<bf16*>(a.y)[(int64_t)m[i] * a.ldy + n[i]] = (bf16)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (in[i]) static_cast<f16*>(a.y)[(int64_t)m[i] * a.ldy + n[i]] = (f16)v[i];
  }
}

// q4_small.hpp, one source file for each type of x.
template <int XT>
hipError_t launch_q4_small(const Q4Args& a, int nt, int waves, int spb, hipStream_t stream);
// q4_tile.hip.
enum : int { kQ4Tile32x128 = 0, kQ4Tile64x128 = 1, kQ4Tile48x128 = 2 };
hipError_t launch_q4_tile(const Q4Args& a, int config, int spb, int teams, bool zeros, hipStream_t stream);
struct Q4PrepArgs {
  const void* x;
  void* xp;   // or nullptr: sums only
  float* xs;  // or nullptr: a copy only
  int64_t ldx, ldp, plane, xs_ld;
  int M, K, blocks, spb, x_type;
  float factor;  // of the sums
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

// The 4-bit layer on up to 32 rows: the weights' bytes are the time.
//
// A workgroup of 8 waves (4 or 2 of wide layers) takes NT tiles of 16 columns; its
// waves split K by blocks of 128 in turn, so that together they read 8 KB runs of a
// tile, and their sums meet in LDS. A wave's 16-byte load of a lane is its operand for four
// matrix instructions. x comes from the caches in whole lines, 16 bytes of a row
// to a lane, and takes operand order through a few KB of LDS that are the wave's
// own (no barrier): loaded in operand order, where neighbouring lanes are rows,
// a wave's loads of 16 rows took four times as long as its weights'. Rows past M
// repeat the last one. The sums of x that the zero points multiply are a matrix
// instruction with a constant operand.
//
// Bound by memory where the layer is large: 1 x 8192 x 8192 in 8.5 to 9.0 us, 4.1
// TB/s with the weights in the Infinity Cache, 11.0 from HBM (a launch and the join
// of the waves' sums are some 4 of them); else by latency: 16 x 4096 x 4097 int8 in
// 7.2, four blocks a wave.
#pragma once

#include <type_traits>

#include "q4.hpp"

namespace edsl {
namespace lm {

// How x of a type is read: bytes of an element, operands that it makes.
template <int XT>
struct SmallX {
  static constexpr int kBytes = type_bytes(XT);
  static constexpr int kPlanes = XT == kF32 ? 3 : 1;
  static constexpr bool kF16Math = XT == kF16;
  using E = Q4Elem<kF16Math>;
  using V = typename E::V;
  using U = std::conditional_t<kBytes == 1, uint8_t, std::conditional_t<kBytes == 2, uint16_t, uint32_t>>;
  static constexpr int kChunks = 8 * kBytes;           // 16-byte chunks of a row's block
  static constexpr int kLoads = 16 * kChunks / 64;     // of a wave for 16 rows
};

// What a wave reads of one block.
template <int XT, int NT, int MT, int SPB>
struct SmallBlock {
  using X = SmallX<XT>;
  u32x4 x[MT][X::kLoads];
  u32x4 w[NT];
  uint32_t scale[NT][SPB], zero[NT][SPB];  // as read
};

// Where a lane's loads of x start: its row of each load, its chunk.
template <int XT, int MT>
struct SmallRows {
  const char* at[MT][SmallX<XT>::kLoads];
};

// Reads a block. Past `last`, the last block read this way, weights are not
// fetched and x and the scales are the last one's: every turn then has the same
// loads, and a turn's wait leaves the later ones' in flight. GUARD: the block
// that K ends in.
template <bool GUARD, int XT, int NT, int MT, int SPB>
__device__ __forceinline__ void small_load(const Q4Args& a, const SmallRows<XT, MT>& rows, int tile, int block,
                                           int last, int lane, const i32x4 (&rsrc)[NT],
                                           SmallBlock<XT, NT, MT, SPB>& r) {
  using X = SmallX<XT>;
  const int in = block < last ? block : last;
  using U = typename X::U;
  constexpr int PER = 16 / X::kBytes;  // elements of a chunk
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int l = 0; l < X::kLoads; ++l) {
      const U* const at = reinterpret_cast<const U*>(rows.at[i][l]) + 128 * in;
      if constexpr (GUARD) {
        const int k = 128 * in + PER * (lane % X::kChunks);  // of the chunk; zeros past K
        r.x[i][l] = __builtin_bit_cast(u32x4, load_guarded<U, PER>(at - k, k, a.K));
      } else {
        r.x[i][l] = __builtin_bit_cast(u32x4, load_packed<U, PER>(at));
      }
    }
  const int sb = q4_scale_block(a, in);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    r.w[t] = __builtin_bit_cast(u32x4, raw_buffer_load_i32x4(rsrc[t], 1024 * block + 16 * lane, 0, 0));
    // Uniform bases, 32 bits a lane.
    const int64_t at = ((tile + t) * (int64_t)a.scale_blocks + sb) * (16 * SPB);
    const char* const scales = a.w + a.scales_at + at * a.scale_bytes;
    const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(a.w + a.zeros_at) + at * a.zero_step;
#pragma unroll
    for (int g = 0; g < SPB; ++g) {
      r.scale[t][g] = q4_scale_bits(scales + g * a.scale_bytes, (uint32_t)(lane % 16 * SPB * a.scale_bytes));
      r.zero[t][g] = zeros[(uint32_t)((lane % 16 * SPB + g) * (int)a.zero_step)];
    }
  }
}

// A wave's own piece of LDS: 16 rows of a block, chunk c of row r at c ^ r (so
// that 16 rows' reads of one chunk meet all banks; rows of 8 chunks share a line).
template <int XT>
__device__ __forceinline__ int small_chunk(int row, int c) {
  constexpr int C = SmallX<XT>::kChunks;
  return row * C + (c ^ (C >= 16 ? row : row / 2));
}

// The operands of step s of a block for 16 rows.
template <int XT>
__device__ __forceinline__ void small_operands(const u32x4* lds, int s, int lane,
                                               typename SmallX<XT>::V (&out)[SmallX<XT>::kPlanes]) {
  using X = SmallX<XT>;
  using V = typename X::V;
  const int row = lane % 16, q = lane / 16;
  if constexpr (X::kBytes == 4) {
    const f32x4 lo = __builtin_bit_cast(f32x4, lds[small_chunk<XT>(row, 8 * s + 2 * q)]);
    const f32x4 hi = __builtin_bit_cast(f32x4, lds[small_chunk<XT>(row, 8 * s + 2 * q + 1)]);
    const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    u32x4 p[3];
    split3_operands(v, p);
#pragma unroll
    for (int i = 0; i < 3; ++i) out[i] = __builtin_bit_cast(V, p[i]);
  } else if constexpr (X::kBytes == 2) {
    out[0] = __builtin_bit_cast(V, lds[small_chunk<XT>(row, 4 * s + q)]);
  } else {
    const uint64_t v = reinterpret_cast<const uint64_t*>(&lds[small_chunk<XT>(row, 2 * s + q / 2)])[q % 2];
    V o;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = (uint32_t)(v >> (32 * h));
      if constexpr (XT == kE4m3) {
        const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
        const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
        o[4 * h] = a[0], o[4 * h + 1] = a[1], o[4 * h + 2] = b[0], o[4 * h + 3] = b[1];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[4 * h + j] = (bf16)(float)(int8_t)(w >> (8 * j));
      }
    }
    out[0] = o;
  }
}

template <int XT, int NT, int MT, int SPB>
__device__ __forceinline__ void small_block(const Q4ScaleMask& mask, const SmallBlock<XT, NT, MT, SPB>& r, u32x4* lds,
                                            int lane, f32x4 (&sum)[MT][NT]) {
  using X = SmallX<XT>;
  using V = typename X::V;
  constexpr int STEPS = 4 / SPB;
  V minus;  // the constant operand of the sums of x
#pragma unroll
  for (int j = 0; j < 8; ++j) minus[j] = -1.0f;
  // x takes operand order through the wave's LDS, whose operations are in order.
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int l = 0; l < X::kLoads; ++l)
      lds[i * 16 * X::kChunks + small_chunk<XT>((64 / X::kChunks) * l + lane / X::kChunks, lane % X::kChunks)] =
          r.x[i][l];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int g = 0; g < SPB; ++g) {
    f32x4 xs[MT], acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      xs[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int s = g * STEPS; s < (g + 1) * STEPS; ++s) {
      V w[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (XT == kF32)
          w[t] = q4_weights_f32(r.w[t][s]);
        else
          w[t] = q4_weights<X::kF16Math>(r.w[t][s]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        V o[X::kPlanes];
        small_operands<XT>(lds + i * 16 * X::kChunks, s, lane, o);
#pragma unroll
        for (int p = X::kPlanes - 1; p >= 0; --p) {
          xs[i] = X::E::mfma(o[p], minus, xs[i]);
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[i][t] = X::E::mfma(o[p], w[t], acc[i][t]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float zero = q4_offset(XT) + (float)r.zero[t][g], scale = q4_scale(r.scale[t][g], mask);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[i][t][e] = fmaf(fmaf(xs[i][e], zero, acc[i][t][e]), scale, sum[i][t][e]);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Waves of a SIMD: two workgroups on a CU where what the two blocks, the operands,
// the sums and a second row tile's part of each group take fits half of its registers
// (24 x 4096 x 4096 int8 in groups of 32 in 9.6 us on one, with 35 registers spilled for
// two in 18.4). 16-bit x in two row and column tiles and groups of 32 spills 4 of 256.
template <int XT, int NT, int MT, int SPB>
constexpr int kSmallOccupancy = 2 * (4 * MT * SmallX<XT>::kLoads + 4 * NT + 2 * NT * SPB) +
                                            4 * SmallX<XT>::kPlanes + 8 * MT * NT + 2 * (MT - 1) * SPB + 4 * NT + 44 <=
                                        128
                                    ? 4
                                    : 2;

template <int XT, int NT, int MT, int SPB, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, (kSmallOccupancy<XT, NT, MT, SPB>)) q4_small_kernel(Q4Args a) {
  using X = SmallX<XT>;
  constexpr int PIECE = 16 * MT * X::kChunks;  // of a wave, in chunks
  constexpr int ROWS = 16 * MT, COLS = 16 * NT;
  constexpr int BYTES = WAVES * (PIECE * 16 > ROWS * COLS * 4 ? PIECE * 16 : ROWS * COLS * 4);
  __shared__ u32x4 lds[BYTES / 16];  // the waves' pieces, then their sums
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int tiles = (a.N + 15) / 16;
  const int first = (int)(blockIdx.z * gridDim.x + blockIdx.x) * NT, slice = blockIdx.y;
  if (first >= tiles) return;  // whole workgroups
  // The last workgroup's tiles may reach past the end: it repeats the last ones
  // and stores each column once.
  const int tile = first + NT <= tiles ? first : tiles - NT;
  const int b0 = slice * a.slice_blocks, b1 = min(a.blocks, b0 + a.slice_blocks);
  SmallRows<XT, MT> rows;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int l = 0; l < X::kLoads; ++l) {
      const int row = min(16 * i + (64 / X::kChunks) * l + lane / X::kChunks, a.M - 1);
      rows.at[i][l] = static_cast<const char*>(a.x) + X::kBytes * (row * a.ldx) + 16 * (lane % X::kChunks);
    }
  i32x4 rsrc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) rsrc[t] = buffer_rsrc(a.w + (int64_t)(tile + t) * a.blocks * 1024, (int64_t)a.blocks * 1024);
  f32x4 sum[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) sum[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  u32x4* const piece = lds + wave * PIECE;
  // Two blocks in turn: one is on its way while the other is multiplied. Turns
  // past the end have scales of zero. (Four in turn, in the registers of one
  // workgroup a CU, were slower: 11.3 against 10.4 us at 1 x 8192 x 8192.)
  const int full = min(a.K / 128, b1);
  SmallBlock<XT, NT, MT, SPB> buf[2];
  int b = b0 + wave;
  if (b < full) {
    small_load<false>(a, rows, tile, b, full - 1, lane, rsrc, buf[0]);
    // Loads stay where they are written: the scheduler would put them off to their use.
    __builtin_amdgcn_sched_barrier(0);
    do {
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        small_load<false>(a, rows, tile, b + WAVES, full - 1, lane, rsrc, buf[d ^ 1]);
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t on = b < full ? ~0u : 0u;
        small_block({a.scale_mask.f32 & on, a.scale_mask.bf16 & on, a.scale_mask.f16 & on}, buf[d], piece, lane, sum);
        b += WAVES;
        __builtin_amdgcn_sched_barrier(0);
      }
    } while (b < full);
  }
  if (full < b1 && wave == (full - b0) % WAVES) {
    small_load<true>(a, rows, tile, full, full, lane, rsrc, buf[0]);
    small_block(a.scale_mask, buf[0], piece, lane, sum);
  }
  __syncthreads();
  float* const part = reinterpret_cast<float*>(lds);  // [wave][row][column]
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        part[(wave * ROWS + 16 * i + 4 * (lane / 16) + e) * COLS + 16 * t + lane % 16] = sum[i][t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < a.M * COLS; i += 64 * WAVES) {
    const int m = i / COLS, c = i % COLS;
    const int n = 16 * tile + c;
    if (n >= a.N || n < 16 * first) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += part[(w * ROWS + m) * COLS + c];
    if (a.ksplit > 1) {
      a.partials[((int64_t)slice * a.M + m) * a.N + n] = v;
    } else {
      float out[1] = {v};
      q4_store<1>(a, {m}, {n}, {true}, out);
    }
  }
}

template <int XT, int NT, int MT, int WAVES>
hipError_t launch_small_spb(const Q4Args& a, int spb, hipStream_t stream) {
  const int tiles = (a.N + 15) / 16;
  const dim3 columns = grid_of((tiles + NT - 1) / NT), block(64 * WAVES);
  const dim3 grid(columns.x, (unsigned)a.ksplit, columns.y);
  if (spb == 4)
    hipLaunchKernelGGL((q4_small_kernel<XT, NT, MT, 4, WAVES>), grid, block, 0, stream, a);
  else if (spb == 2)
    hipLaunchKernelGGL((q4_small_kernel<XT, NT, MT, 2, WAVES>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((q4_small_kernel<XT, NT, MT, 1, WAVES>), grid, block, 0, stream, a);
  return launched();
}

template <int XT>
hipError_t launch_q4_small(const Q4Args& a, int nt, int waves, int spb, hipStream_t stream) {
  if constexpr (XT != kF32) {  // three operands of 32 rows do not fit the registers
    if (a.M > 16)
      return nt == 2 ? launch_small_spb<XT, 2, 2, 8>(a, spb, stream) : launch_small_spb<XT, 1, 2, 8>(a, spb, stream);
  }
  if (nt == 1) return launch_small_spb<XT, 1, 1, 8>(a, spb, stream);
  if (waves == 2) return launch_small_spb<XT, 2, 1, 2>(a, spb, stream);
  if (waves == 4) return launch_small_spb<XT, 2, 1, 4>(a, spb, stream);
  return launch_small_spb<XT, 2, 1, 8>(a, spb, stream);
}

}  // namespace lm
}  // namespace edsl

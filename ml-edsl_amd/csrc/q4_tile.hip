// The 4-bit layer on more than 16 rows: tiles on the matrix cores.
//
// A workgroup of 4 waves takes 16 MT WM rows x 16 NT WN columns. A wave loads and
// unpacks the weights of its own columns in registers; x goes through LDS, one
// block of 128 k ahead, in operand order with 16-byte chunks exchanged by row so
// that reads hit all banks. Each group's accumulators start at the prepared
// -zero * sum x and are scaled into the 32-bit totals at its end.
#include "q4.hpp"

namespace edsl {
namespace lm {
namespace {

template <bool F16, int PLANES, int MT, int NT, int WM, int WN, int SPB, bool ZEROS>
__global__ void __launch_bounds__(256) q4_tile_kernel(Q4Args a) {
  using E = Q4Elem<F16>;
  using V = typename E::V;
  constexpr int BM = 16 * MT * WM, STEPS = 4 / SPB;
  static_assert(WM * WN == 4, "four waves");
  constexpr int CHUNKS = PLANES * BM * 16 / 256;  // 16-byte chunks of a block of x, a thread's
  __shared__ u32x4 lds[2][PLANES * BM * 16];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int wm = wave % WM, wn = wave / WM;
  const int64_t tiles = (a.N + 15) / 16;
  const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (int)((tiles + NT * WN - 1) / (NT * WN));
  const int slice = blockIdx.x / (tiles_m * tiles_n);
  int tm, tn;
  tile_coords(blockIdx.x % (tiles_m * tiles_n), tiles_m, tiles_n, tm, tn);
  const int64_t first = ((int64_t)tn * WN + wn) * NT;
  const int m0 = tm * BM;
  const int b0 = (int)((int64_t)a.blocks * slice / a.ksplit), b1 = (int)((int64_t)a.blocks * (slice + 1) / a.ksplit);

  // Chunk i of a block: row i / 16 of the planes, its k chunk (i % 16) ^ (row % 16).
  const char* src[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = c * 256 + tid, r = i / 16, plane = r / BM, row = m0 + r % BM;
    const int64_t at = plane * a.plane + (int64_t)(row < a.M ? row : a.M - 1) * a.ldp + 8 * ((i % 16) ^ (r % 16));
    src[c] = static_cast<const char*>(a.xp) + 2 * at;
  }
  u32x4 xr[CHUNKS];
  const auto load_x = [&](int b) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) xr[c] = *reinterpret_cast<const u32x4*>(src[c] + (int64_t)b * 256);
  };
  const auto store_x = [&](int buf) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) lds[buf][c * 256 + tid] = xr[c];
  };
  u32x4 w[2][NT];
  const auto load_w = [&](int b, u32x4 (&r)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t tile = first + t < tiles ? first + t : tiles - 1;
      r[t] = *reinterpret_cast<const u32x4*>(a.w + (tile * a.blocks + b) * 1024 + 16 * lane);
    }
  };
  f32x4 sum[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) sum[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  if (b0 < b1) {
    load_x(b0);
    load_w(b0, w[0]);
    store_x(0);
  }
  for (int b = b0; b < b1; ++b) {
    const int buf = (b - b0) & 1;
    __syncthreads();
    const bool more = b + 1 < b1;
    if (more) {
      load_x(b + 1);
      load_w(b + 1, w[1]);
    }
    const int sb = b / a.blocks_per_scale;
#pragma unroll
    for (int g = 0; g < SPB; ++g) {
      float scale[NT], zero[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t tile = first + t < tiles ? first + t : tiles - 1;
        const int64_t at = ((tile * a.scale_blocks + sb) * 16 + lane % 16) * SPB + g;
        scale[t] = q4_scale(a.w + a.scales_at, a.scale_type, at);
        if constexpr (ZEROS) zero[t] = (float)reinterpret_cast<const uint8_t*>(a.w + a.zeros_at)[at];
      }
      f32x4 acc[MT][NT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int m = m0 + 16 * (wm * MT + i) + 4 * (lane / 16);
        const f32x4 xs = *reinterpret_cast<const f32x4*>(a.xs + ((int64_t)b * SPB + g) * a.xs_ld + m);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[i][t] = xs;
          if constexpr (ZEROS)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][t][e] *= zero[t];
        }
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int step = g * STEPS + s;
        V q[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) q[t] = E::weights(w[0][t][step]);
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p)
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int r = p * BM + 16 * (wm * MT + i) + lane % 16;
            const V x = __builtin_bit_cast(V, lds[buf][r * 16 + ((4 * step + lane / 16) ^ (r % 16))]);
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][t] = E::mfma(x, q[t], acc[i][t]);
          }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[i][t][e] = fmaf(acc[i][t][e], scale[t], sum[i][t][e]);
    }
    if (more) {
      store_x(buf ^ 1);
#pragma unroll
      for (int t = 0; t < NT; ++t) w[0][t] = w[1][t];
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t n = 16 * (first + t) + lane % 16;
    if (n >= a.N) continue;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = m0 + 16 * (wm * MT + i) + 4 * (lane / 16) + e;
        if (m >= a.M) continue;
        if (a.ksplit > 1)
          a.partials[((int64_t)slice * a.M + m) * a.N + n] = sum[i][t][e];
        else
          q4_store(a, m, (int)n, sum[i][t][e]);
      }
  }
}

template <bool F16, int PLANES, int MT, int NT, int WM, int WN, int SPB>
hipError_t launch_tile_zeros(const Q4Args& a, bool zeros, hipStream_t stream) {
  const int64_t tiles = (a.N + 15) / 16;
  const int64_t tm = (a.M + 16 * MT * WM - 1) / (16 * MT * WM), tn = (tiles + NT * WN - 1) / (NT * WN);
  const dim3 grid((unsigned)(tm * tn * a.ksplit)), block(256);
  if (zeros)
    hipLaunchKernelGGL((q4_tile_kernel<F16, PLANES, MT, NT, WM, WN, SPB, true>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((q4_tile_kernel<F16, PLANES, MT, NT, WM, WN, SPB, false>), grid, block, 0, stream, a);
  return launched();
}

template <bool F16, int PLANES, int MT, int NT, int WM, int WN>
hipError_t launch_tile_spb(const Q4Args& a, int spb, bool zeros, hipStream_t stream) {
  if (spb == 4) return launch_tile_zeros<F16, PLANES, MT, NT, WM, WN, 4>(a, zeros, stream);
  if (spb == 2) return launch_tile_zeros<F16, PLANES, MT, NT, WM, WN, 2>(a, zeros, stream);
  return launch_tile_zeros<F16, PLANES, MT, NT, WM, WN, 1>(a, zeros, stream);
}

template <bool F16, int PLANES>
hipError_t launch_tile_config(const Q4Args& a, int config, int spb, bool zeros, hipStream_t stream) {
  if (config == kQ4Tile32x128) return launch_tile_spb<F16, PLANES, 2, 2, 1, 4>(a, spb, zeros, stream);
  if (config == kQ4Tile64x128) return launch_tile_spb<F16, PLANES, 4, 2, 1, 4>(a, spb, zeros, stream);
  if constexpr (PLANES == 1) return launch_tile_spb<F16, 1, 4, 4, 2, 2>(a, spb, zeros, stream);
  return hipErrorInvalidValue;
}

// ------------------------------------------------------------------- x
// A wave takes a row of x, 8 elements a lane: converts them where a copy is
// wanted (bf16 terms of f32, bf16 of 8 bits; zeros past K) and adds up each
// group's.
template <int XT>
__global__ void __launch_bounds__(256) q4_prep_kernel(Q4PrepArgs a) {
  const int lane = threadIdx.x % 64;
  const int row = blockIdx.x * 4 + threadIdx.x / 64;
  if (row >= a.M) return;
  const int lanes = 16 / a.spb;  // of a group
  for (int k0 = 8 * lane; k0 < 128 * a.blocks; k0 += 512) {
    float v[8];
    u32x4 out[3];
    if constexpr (XT == kE4m3) {
      const auto r = load_guarded<uint8_t, 8>(static_cast<const uint8_t*>(a.x) + row * a.ldx, k0, a.K);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w |= (uint32_t)r.v[4 * h + j] << (8 * j);
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
        v[4 * h] = (float)lo[0], v[4 * h + 1] = (float)lo[1], v[4 * h + 2] = (float)hi[0], v[4 * h + 3] = (float)hi[1];
      }
    } else if constexpr (XT == kI8) {
      const auto r = load_guarded<int8_t, 8>(static_cast<const int8_t*>(a.x) + row * a.ldx, k0, a.K);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)r.v[j];
    } else if constexpr (XT == kF32) {
      const auto r = load_guarded<float, 8>(static_cast<const float*>(a.x) + row * a.ldx, k0, a.K);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r.v[j];
    } else if constexpr (XT == kF16) {
      const auto r = load_guarded<f16, 8>(static_cast<const f16*>(a.x) + row * a.ldx, k0, a.K);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)r.v[j];
      out[0] = __builtin_bit_cast(u32x4, r);
    } else {
      const auto r = load_guarded<bf16, 8>(static_cast<const bf16*>(a.x) + row * a.ldx, k0, a.K);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = (float)r.v[j];
    }
    if (a.xp) {
      if constexpr (XT != kF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const Split3 p = split3(v[2 * j]), q = split3(v[2 * j + 1]);
          out[0][j] = (p.hi >> 16) | q.hi;
          if constexpr (XT == kF32) {
            out[1][j] = (p.mid >> 16) | q.mid;
            out[2][j] = (p.lo >> 16) | q.lo;
          }
        }
      }
#pragma unroll
      for (int p = 0; p < (XT == kF32 ? 3 : 1); ++p)
        *reinterpret_cast<u32x4*>(static_cast<char*>(a.xp) + 2 * (p * a.plane + row * a.ldp + k0)) = out[p];
    }
    float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    s += dpp<0xB1>(s);
    s += dpp<0x4E>(s);
    if (lanes > 4) s += dpp<0x141>(s);
    if (lanes > 8) s += dpp<0x140>(s);
    if (lane % lanes == 0) a.xs[(int64_t)(k0 / (8 * lanes)) * a.xs_ld + row] = a.factor * s;
  }
}

// y from the slices' sums, in their order.
__global__ void __launch_bounds__(256) q4_join_kernel(Q4Args a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)a.M * a.N;
  if (i >= all) return;
  float v = 0.0f;
  for (int s = 0; s < a.ksplit; ++s) v += a.partials[s * all + i];
  q4_store(a, (int)(i / a.N), (int)(i % a.N), v);
}

// ------------------------------------------------------------------ packing
// A workgroup of 256 threads packs a block of 16 columns x 128 k, a word each.
__global__ void __launch_bounds__(256) q4_pack_kernel(Q4PackArgs a) {
  const int64_t tile = blockIdx.x / a.layout.blocks, block = blockIdx.x % a.layout.blocks;
  // Threads of a wave take 16 columns by 4 runs of 8 k of one step.
  const int lane = threadIdx.x % 64, step = threadIdx.x / 64;
  const int64_t n = 16 * tile + lane % 16, k0 = 128 * block + 32 * step + 8 * (lane / 16);
  uint32_t w = 0;
  if (n < a.N)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + j < a.K) w |= (uint32_t)(a.q[(k0 + j) * a.ldq + n] & 15) << (j < 4 ? 8 * j : 8 * (j - 4) + 4);
  reinterpret_cast<uint32_t*>(a.packed + (tile * a.layout.blocks + block) * 1024)[4 * lane + step] = w;
  // Its scales and zero points, by the first block of each group.
  const int spb = a.layout.spb, bps = a.layout.blocks_per_scale;
  if (block % bps != 0 || threadIdx.x >= 16 * spb) return;
  const int c = threadIdx.x / spb, g = threadIdx.x % spb;
  const int64_t col = 16 * tile + c, sb = block / bps, group = sb * spb + g, groups = (a.K + a.group - 1) / a.group;
  const bool in = col < a.N && group < groups;
  const int64_t at = ((tile * a.layout.scale_blocks + sb) * 16 + c) * spb + g;
  if (a.scale_type == kF32)
    reinterpret_cast<float*>(a.packed + a.layout.scales_at)[at] =
        in ? static_cast<const float*>(a.scales)[group * a.lds + col] : 0.0f;
  else
    reinterpret_cast<uint16_t*>(a.packed + a.layout.scales_at)[at] =
        in ? static_cast<const uint16_t*>(a.scales)[group * a.lds + col] : (uint16_t)0;
  if (a.zeros)
    reinterpret_cast<uint8_t*>(a.packed + a.layout.zeros_at)[at] = in ? a.zeros[group * a.ldz + col] & 15 : 0;
}

}  // namespace

hipError_t launch_q4_tile(const Q4Args& a, int config, int spb, bool zeros, hipStream_t stream) {
  if (a.x_type == kF16) return launch_tile_config<true, 1>(a, config, spb, zeros, stream);
  if (a.x_type == kF32) return launch_tile_config<false, 3>(a, config, spb, zeros, stream);
  return launch_tile_config<false, 1>(a, config, spb, zeros, stream);
}

hipError_t launch_q4_prep(const Q4PrepArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.M + 3) / 4)), block(256);
  switch (a.x_type) {
    case kF32: hipLaunchKernelGGL((q4_prep_kernel<kF32>), grid, block, 0, stream, a); break;
    case kBf16: hipLaunchKernelGGL((q4_prep_kernel<kBf16>), grid, block, 0, stream, a); break;
    case kF16: hipLaunchKernelGGL((q4_prep_kernel<kF16>), grid, block, 0, stream, a); break;
    case kI8: hipLaunchKernelGGL((q4_prep_kernel<kI8>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((q4_prep_kernel<kE4m3>), grid, block, 0, stream, a); break;
  }
  return launched();
}

hipError_t launch_q4_join(const Q4Args& a, hipStream_t stream) {
  const int64_t all = (int64_t)a.M * a.N;
  hipLaunchKernelGGL(q4_join_kernel, dim3((unsigned)((all + 255) / 256)), dim3(256), 0, stream, a);
  return launched();
}

hipError_t launch_q4_pack(const Q4PackArgs& a, hipStream_t stream) {
  if (a.layout.blocks == 0 || a.layout.tiles_n == 0) return hipSuccess;
  hipLaunchKernelGGL(q4_pack_kernel, dim3((unsigned)(a.layout.tiles_n * a.layout.blocks)), dim3(256), 0, stream, a);
  return launched();
}

}  // namespace lm
}  // namespace edsl

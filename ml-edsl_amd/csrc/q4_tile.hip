// The 4-bit layer on more than 16 rows: tiles on the matrix cores.
//
// A workgroup takes 16 MT rows x 64 NT columns by teams of 4 waves; the blocks of 128
// k go to the teams in turn, whose sums meet in LDS at the end. A wave loads and
// unpacks the weights of its own columns in registers, a block ahead; x and its
// groups' sums go from memory straight to LDS, a stage ahead, with 16-byte chunks
// exchanged by row so that reads hit all banks. Each group's accumulators start at
// the prepared -zero * sum x and are scaled into the 32-bit totals at its end; with
// OWN_SUMS a matrix instruction with a constant operand sums x instead.
//
// Bound by power and by the matrix cores and vector ALUs together where M is
// large: 4096^3 in 153 us without zero points and 163 with them, the sums of
// x included (898 and 843 TFLOP/s, 80 and 75 % of what the vendor's bf16 product
// reaches there), 8192^3 with them in 1098 us (1.0 PFLOP/s, 80 %). Tiles of 128x128
// and 128x256 (half and a third of the traffic) are no faster, 164 to 172 us, nor
// are fragments read ahead or a forced order of products and unpacking. With few
// rows a block's loads and the launches bound it: 33 x 8192 x 8192 in 17.4 us, 7 of
// them the weights' bytes, some 4 the join's launch. 8-bit x is copied to bf16 first and
// multiplied at that rate: 128 x 4096 x 4096 int8 in 20.4 us, bf16 in 17.4; 4096^3 in 159.
#include "q4.hpp"

namespace edsl {
namespace lm {
namespace {

// 16 bytes a lane from memory, `base` (uniform) + `offset`, to LDS, `to` (the
// wave's own) + 16 lane. As the instruction itself: for its intrinsic the
// compiler lets every later read of LDS wait for it, whichever buffer it reads,
// which left nothing on the way while a stage was multiplied. It has no result
// register; wait_loads() is what waits for it. m0 is declared as written.
__device__ __forceinline__ void to_lds(const void* base, uint32_t offset, void* to) {
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)at)), "v"(offset), "s"(base)
               : "memory", "m0");
}

// Waits for the wave's loads, those to LDS among them (vmcnt 0).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

template <bool F16, int PLANES, int MT, int NT, int SPB, bool ZEROS, int TEAMS, bool OWN_SUMS>
__global__ void __launch_bounds__(256 * TEAMS, 2) q4_tile_kernel(Q4Args a) {
  using E = Q4Elem<F16>;
  using V = typename E::V;
  constexpr int BM = 16 * MT, STEPS = 4 / SPB;
  // A stage of x in LDS: SS steps of 32 k, CPR 16-byte chunks a row.
  constexpr int SS = PLANES == 3 ? 2 : 4, CPR = 4 * SS, STAGES = 4 / SS;
  constexpr int ALL = PLANES * BM * CPR, CHUNKS = (ALL + 255) / 256;  // a thread's
  __shared__ u32x4 lds_all[TEAMS][2][ALL];
  __shared__ f32x4 sums_all[TEAMS][2][SPB * BM / 4];  // a block's sums of x: [BM / 16][SPB][16]
  const int tid = threadIdx.x % 256, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const int team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 256) : 0;
  auto& lds = lds_all[team];
  auto& sums = sums_all[team];
  const int64_t tiles = (a.N + 15) / 16;
  const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (int)((tiles + 4 * NT - 1) / (4 * NT));
  const int block = (int)block_of();
  const int slice = block / (tiles_m * tiles_n);
  if (slice >= a.ksplit) return;  // whole workgroups
  int tm, tn;
  tile_coords(block % (tiles_m * tiles_n), tiles_m, tiles_n, tm, tn);
  const int64_t first = ((int64_t)tn * 4 + wave) * NT;
  const int m0 = tm * BM;
  const int b0 = slice * a.slice_blocks, b1 = min(a.blocks, b0 + a.slice_blocks);

  // Row r's chunk c lies at c ^ swizzle(r): 16 rows' reads of one chunk meet all banks.
  const auto swizzle = [](int r) { return CPR == 16 ? r % 16 : (r / 2) % 8; };
  // Addresses are a uniform base and 32 bits a lane, so that they stay out of the
  // vector registers (the runtime bounds K for it); rows past M repeat the last.
  static_assert(BM * CPR % 64 == 0, "a wave's chunk is of one plane");
  uint32_t src[CHUNKS];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = c * 256 + tid, r = i / CPR, row = m0 + r % BM;
    src[c] = (uint32_t)(((int64_t)(row < a.M ? row : a.M - 1) - m0) * a.ldp + 8 * ((i % CPR) ^ swizzle(r))) * 2u;
  }
  const char* const xp = static_cast<const char*>(a.xp) + 2 * m0 * a.ldp;
  const auto load_x = [&](int stage, u32x4* to) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int i = c * 256 + wave * 64;
      if (ALL % 256 == 0 || i < ALL)
        to_lds(xp + 2 * (BM * CPR % 256 == 0 ? c * 256 / (BM * CPR) : i / (BM * CPR)) * a.plane +
                   (int64_t)stage * (16 * CPR),
               src[c], to + i);
    }
  };
  const auto load_sums = [&](int b, f32x4* to) {
    // The groups' sums of 16 rows lie together (Q4Args::xs), so that a block's sums of
    // the tile's rows are one run and a lane's offset is small, however many rows there are.
    if (!OWN_SUMS && tid < SPB * BM / 4)
      to_lds(a.xs + ((int64_t)b * a.xs_ld + m0) * SPB, 16u * (uint32_t)tid, to + wave * 64);
  };
  const uint32_t scale_offset = lane % 16 * SPB * a.scale_bytes;
  struct Weights {
    u32x4 w[NT];
    uint32_t scale[NT][SPB], zero[ZEROS ? NT : 1][SPB];  // as read
  };
  const auto load_w = [&](int b, Weights& r) {
    const int sb = q4_scale_block(a, b);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // Uniform bases, 32 bits a lane: no vector instruction goes into addresses.
      const int64_t tile = first + t < tiles ? first + t : tiles - 1;
      r.w[t] = *reinterpret_cast<const u32x4*>(a.w + (tile * a.blocks + b) * 1024 + (uint32_t)(16 * lane));
      const int64_t at = (tile * a.scale_blocks + sb) * (16 * SPB);
      const char* const scales = a.w + a.scales_at + at * a.scale_bytes;
      const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(a.w + a.zeros_at) + at;
#pragma unroll
      for (int g = 0; g < SPB; ++g) {
        r.scale[t][g] = q4_scale_bits(scales + g * a.scale_bytes, scale_offset);
        if constexpr (ZEROS) r.zero[t][g] = zeros[(uint32_t)(lane % 16 * SPB + g)];
      }
    }
  };
  f32x4 sum[MT][NT], acc[MT][NT], own[OWN_SUMS ? MT : 1];
  V minus;  // the constant operand of the sums of x
#pragma unroll
  for (int j = 0; j < 8; ++j) minus[j] = -1.0f;
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < NT; ++t) sum[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  Weights now, next;
  // One stage: starts the next one's loads, and multiplies this one.
  const auto turn = [&](int b, int stage, const u32x4* x_now, u32x4* x_next, const f32x4* sums_now,
                        f32x4* sums_next) {
    wait_loads();
    __syncthreads();
    if (TEAMS > 1 && b >= b1) return;  // the last turn of a team without a block
    if (stage < STAGES - 1)
      load_x(b * STAGES + stage + 1, x_next);
    else if (b + TEAMS < b1)
      load_x((b + TEAMS) * STAGES, x_next);
    if (stage == 0 && b + TEAMS < b1) {
      load_sums(b + TEAMS, sums_next);
      load_w(b + TEAMS, next);
    }
#pragma unroll
    for (int s = 0; s < SS; ++s) {
      const int step = stage * SS + s, g = step / STEPS;
      if (step % STEPS == 0) {
        float zero[NT];
        if constexpr (ZEROS)
#pragma unroll
          for (int t = 0; t < NT; ++t) zero[t] = (PLANES == 3 ? 0.0f : kQ4Offset) + (float)now.zero[t][g];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if constexpr (OWN_SUMS) {
            own[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[i][t] = own[i];
            continue;
          }
          const f32x4 xs = sums_now[4 * (i * SPB + g) + lane / 16];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[i][t] = xs;
            if constexpr (ZEROS)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][t][e] *= zero[t];
          }
        }
      }
      V q[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (PLANES == 3)
          q[t] = q4_weights_f32(now.w[t][step]);
        else
          q[t] = q4_weights<F16>(now.w[t][step]);
      }
#pragma unroll
      for (int p = PLANES - 1; p >= 0; --p)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int r = p * BM + 16 * i + lane % 16;
          const V x = __builtin_bit_cast(V, x_now[r * CPR + ((4 * s + lane / 16) ^ swizzle(r))]);
          if constexpr (OWN_SUMS) own[i] = E::mfma(x, minus, own[i]);
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[i][t] = E::mfma(x, q[t], acc[i][t]);
        }
      if (step % STEPS == STEPS - 1) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float scale = q4_scale(now.scale[t][g], a.scale_mask);
          const float zero = kQ4Offset + (ZEROS ? (float)now.zero[ZEROS ? t : 0][g] : 8.0f);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (OWN_SUMS) acc[i][t][e] = fmaf(own[i][e], zero, acc[i][t][e]);
              sum[i][t][e] = fmaf(acc[i][t][e], scale, sum[i][t][e]);
            }
        }
      }
    }
  };
  if (b0 + team < b1) {
    load_x((b0 + team) * STAGES, lds[0]);
    load_sums(b0 + team, sums[0]);
    load_w(b0 + team, now);
  }
  int odd = 0;
  for (int first_b = b0; first_b < b1; first_b += TEAMS, odd ^= 1) {
    const int b = first_b + team;
    if constexpr (STAGES == 1) {
      turn(b, 0, lds[odd], lds[odd ^ 1], sums[odd], sums[odd ^ 1]);
    } else {
      turn(b, 0, lds[0], lds[1], sums[odd], sums[odd ^ 1]);
      turn(b, 1, lds[1], lds[0], sums[odd], sums[odd ^ 1]);
    }
    now = next;
  }
  if constexpr (TEAMS > 1) {
    // The first team adds the others' sums to its own, in their order.
    static_assert(MT * NT * 256 <= 2 * ALL, "a team's sums fit its stages of x");
    __syncthreads();
    if (team > 0)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t) lds[0][(i * NT + t) * 256 + tid] = __builtin_bit_cast(u32x4, sum[i][t]);
    __syncthreads();
    if (team > 0) return;
#pragma unroll
    for (int other = 1; other < TEAMS; ++other)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          sum[i][t] += __builtin_bit_cast(f32x4, lds_all[other][0][(i * NT + t) * 256 + tid]);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    int m[4 * NT], n[4 * NT];
    bool in[4 * NT];
    float v[4 * NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 4 * t + e;
        m[j] = m0 + 16 * i + 4 * (lane / 16) + e;
        n[j] = (int)(16 * (first + t)) + lane % 16;
        in[j] = m[j] < a.M && n[j] < a.N;
        v[j] = sum[i][t][e];
      }
    if (a.ksplit > 1) {
#pragma unroll
      for (int j = 0; j < 4 * NT; ++j)
        if (in[j]) a.partials[((int64_t)slice * a.M + m[j]) * a.N + n[j]] = v[j];
    } else {
      q4_store<4 * NT>(a, m, n, in, v);
    }
  }
}

template <bool F16, int PLANES, int MT, int NT, int SPB, bool ZEROS>
hipError_t launch_tile_teams(const Q4Args& a, int teams, hipStream_t stream) {
  const int64_t tiles = (a.N + 15) / 16;
  const int64_t tm = (a.M + 16 * MT - 1) / (16 * MT), tn = (tiles + 4 * NT - 1) / (4 * NT);
  const dim3 grid = grid_of(tm * tn * a.ksplit);
  if constexpr (PLANES == 1) {
    if (teams == 2 && !a.xs) {
      hipLaunchKernelGGL((q4_tile_kernel<F16, 1, MT, NT, SPB, ZEROS, 2, true>), grid, dim3(512), 0, stream, a);
      return launched();
    }
  }
  if (teams == 2)
    hipLaunchKernelGGL((q4_tile_kernel<F16, PLANES, MT, NT, SPB, ZEROS, 2, false>), grid, dim3(512), 0, stream, a);
  else
    hipLaunchKernelGGL((q4_tile_kernel<F16, PLANES, MT, NT, SPB, ZEROS, 1, false>), grid, dim3(256), 0, stream, a);
  return launched();
}

template <bool F16, int PLANES, int MT, int NT, int SPB>
hipError_t launch_tile_zeros(const Q4Args& a, int teams, bool zeros, hipStream_t stream) {
  return zeros ? launch_tile_teams<F16, PLANES, MT, NT, SPB, true>(a, teams, stream)
               : launch_tile_teams<F16, PLANES, MT, NT, SPB, false>(a, teams, stream);
}

template <bool F16, int PLANES, int MT, int NT>
hipError_t launch_tile_spb(const Q4Args& a, int spb, int teams, bool zeros, hipStream_t stream) {
  if (spb == 4) return launch_tile_zeros<F16, PLANES, MT, NT, 4>(a, teams, zeros, stream);
  if (spb == 2) return launch_tile_zeros<F16, PLANES, MT, NT, 2>(a, teams, zeros, stream);
  return launch_tile_zeros<F16, PLANES, MT, NT, 1>(a, teams, zeros, stream);
}

template <bool F16, int PLANES>
hipError_t launch_tile_config(const Q4Args& a, int config, int spb, int teams, bool zeros, hipStream_t stream) {
  if (config == kQ4Tile32x128) return launch_tile_spb<F16, PLANES, 2, 2>(a, spb, teams, zeros, stream);
  if (config == kQ4Tile64x128) return launch_tile_spb<F16, PLANES, 4, 2>(a, spb, teams, zeros, stream);
  return launch_tile_spb<F16, PLANES, 3, 2>(a, spb, teams, zeros, stream);
}

// ------------------------------------------------------------------- x
// A wave takes 512 k of a row of x, 8 elements a lane: converts them where a copy is
// wanted (bf16 terms of f32, bf16 of 8 bits; zeros past K) and adds up each
// group's.
template <int XT>
__global__ void __launch_bounds__(256) q4_prep_kernel(Q4PrepArgs a) {
  const int lane = threadIdx.x % 64;
  // Rows along x and z (a launch takes less than 2^32 threads along each).
  const int64_t row = ((int64_t)blockIdx.z * gridDim.x + blockIdx.x) * 4 + threadIdx.x / 64;
  if (row >= a.M) return;
  const int lanes = 16 / a.spb;  // of a group
  if (const int k0 = 512 * blockIdx.y + 8 * lane; k0 < 128 * a.blocks) {
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
      if constexpr (XT == kF32) {
        split3_operands(v, out);
      } else if constexpr (XT != kF16) {
        // Exact in bf16: its upper half.
#pragma unroll
        for (int j = 0; j < 4; ++j)
          out[0][j] = (__builtin_bit_cast(uint32_t, v[2 * j]) >> 16) |
                      (__builtin_bit_cast(uint32_t, v[2 * j + 1]) & 0xffff0000u);
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
    if (a.xs && lane % lanes == 0) {
      const int block = k0 / 128, group = k0 % 128 / (8 * lanes);
      a.xs[((block * a.xs_ld + row / 16 * 16) * a.spb + 16 * group) + row % 16] = a.factor * s;
    }
  }
}

// y from the slices' sums, in their order.
__global__ void __launch_bounds__(256) q4_join_kernel(Q4Args a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)a.M * a.N;
  if (i >= all) return;
  float v = 0.0f;
  for (int s = 0; s < a.ksplit; ++s) v += a.partials[s * all + i];
  float out[1] = {v};
  q4_store<1>(a, {(int)(i / a.N)}, {(int)(i % a.N)}, {true}, out);
}

// ------------------------------------------------------------------ packing
// A workgroup of 256 threads packs a block of 128 k of four tiles: reads rows of 64
// columns, 4 bytes a thread, into LDS, and each wave puts its tile's words together.
__global__ void __launch_bounds__(256) q4_pack_kernel(Q4PackArgs a) {
  constexpr int PITCH = 68;  // bytes of a row in LDS
  __shared__ uint8_t q[128 * PITCH];
  const int64_t first = 4 * (block_of() / a.layout.blocks), block = block_of() % a.layout.blocks;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  {
    const int c = threadIdx.x % 16 * 4;
    const int64_t n = 16 * first + c;
#pragma unroll 8
    for (int r = threadIdx.x / 16; r < 128; r += 16) {
      const int64_t k = 128 * block + r;
      Packed<uint8_t, 4> v{};
      if (k < a.K && n < a.N) v = load_guarded<uint8_t, 4>(a.q + k * a.ldq, n, a.N);
      *reinterpret_cast<uint32_t*>(&q[r * PITCH + c]) = __builtin_bit_cast(uint32_t, v);
    }
  }
  __syncthreads();
  const int64_t tile = first + wave;
  if (tile >= a.layout.tiles_n) return;
  u32x4 words;
#pragma unroll
  for (int step = 0; step < 4; ++step) {
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w |= (uint32_t)(q[(32 * step + 8 * (lane / 16) + j) * PITCH + 16 * wave + lane % 16] & 15)
           << (4 * (j / 2) + 16 * (j % 2));
    words[step] = w;
  }
  reinterpret_cast<u32x4*>(a.packed + (tile * a.layout.blocks + block) * 1024)[lane] = words;
  // Its scales and zero points, by the first block of each group.
  const int spb = a.layout.spb, bps = a.layout.blocks_per_scale;
  if (!a.zeros && block_of() == 0 && threadIdx.x < 16) a.packed[a.layout.zeros_at + threadIdx.x] = 8;
  if (block % bps != 0 || lane >= 16 * spb) return;
  const int c = lane / spb, g = lane % spb;
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

hipError_t launch_q4_tile(const Q4Args& a, int config, int spb, int teams, bool zeros, hipStream_t stream) {
  if (a.x_type == kF16) return launch_tile_config<true, 1>(a, config, spb, teams, zeros, stream);
  if (a.x_type == kF32) return launch_tile_config<false, 3>(a, config, spb, teams, zeros, stream);
  return launch_tile_config<false, 1>(a, config, spb, teams, zeros, stream);
}

hipError_t launch_q4_prep(const Q4PrepArgs& a, hipStream_t stream) {
  const dim3 rows = grid_of(((int64_t)a.M + 3) / 4), grid(rows.x, (unsigned)((a.blocks + 3) / 4), rows.y), block(256);
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
  hipLaunchKernelGGL(q4_pack_kernel, grid_of((a.layout.tiles_n + 3) / 4 * a.layout.blocks), dim3(256), 0, stream, a);
  return launched();
}

}  // namespace lm
}  // namespace edsl

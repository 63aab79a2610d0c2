// A few rows against a layer's weights: what is read once is the weights, and the
// time is theirs. The waves of a workgroup take blocks of K in turn, each with the next ones'
// loads on their way while it multiplies this one, and meet in LDS once.
// No operand goes through LDS before: rows of x come in the instruction's order, and
// so do weights whose k are contiguous (kRows) or that are laid out so (kBlocks).
// Where columns are contiguous (kCols), a lane reads kChunk successive k of NJ
// successive columns and turns them in registers, so that NJ instructions take one
// of its columns each; the order of the columns is put right where they are stored.
//
// Bound by memory where workgroups fill the CUs: 4 to 5.9 TB/s of weights (8-bit 1 x 8192 x 8192 in 11.4 us; 16
// bf16 rows at 8 experts of 4096 x 4096 in 50, 4.7 TB/s); by the loads' way where they do not (16 x 4096 x 4096 bf16 in 10.6 us
// with k contiguous, in 14.6 of 64 workgroups with columns contiguous: lines of 128 bytes take 64 columns).
#pragma once

#include "lm_tile.hpp"

namespace edsl {
namespace lm {

template <typename T, int KIND, int MT, int NJ, int WAVES, int U, int AHEAD>
struct Skinny {
  using E = TileElem<T>;
  using Acc = typename E::Acc;
  static constexpr int kChunk = E::kChunk, kStep = 4 * kChunk;
  static constexpr int kDepth = U * kStep;        // k of a block: U steps
  static constexpr int kCols16 = 16 * NJ;         // columns of a workgroup
  static constexpr int kSlots = WAVES * NJ * 64;  // Acc of LDS

  struct Rows {
    u32x4 v[U][MT];
  };
  struct Weights {
    u32x4 b[KIND == kCols ? 1 : U][KIND == kCols ? 1 : NJ];
    Packed<T, NJ> raw[KIND == kCols ? U : 1][KIND == kCols ? kChunk : 1];
  };

  const char* xrow[MT];  // the lane's rows, at its first k
  const char* wcol[NJ];  // its columns (kCols: the first one)
  int64_t ld;            // of the weights
  int lane, chunk_at;

  // `rows` of x and `n` columns of weights; columns from n0 on.
  __device__ __forceinline__ void init(const void* x, int64_t ldx, int rows, const void* w, int64_t ldw, int N,
                                       int n0) {
    lane = threadIdx.x % 64;
    chunk_at = lane / 16 * kChunk;
    ld = ldw;
#pragma unroll
    for (int i = 0; i < MT; ++i)
      xrow[i] = static_cast<const char*>(x) +
                (min(16 * i + lane % 16, rows - 1) * ldx + chunk_at) * (int64_t)sizeof(T);
    if constexpr (KIND == kCols) {
      wcol[0] = static_cast<const char*>(w) + (chunk_at * ldw + column(0, lane % 16, N, n0)) * (int64_t)sizeof(T);
    } else if constexpr (KIND == kRows) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        wcol[j] = static_cast<const char*>(w) +
                  (min(column(j, lane % 16, N, n0), N - 1) * ldw + chunk_at) * (int64_t)sizeof(T);
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        wcol[j] = static_cast<const char*>(w) + min(n0 / 16 + j, (N - 1) / 16) * ldw + lane * 16;
    }
  }

  // The layer's column that instruction j gives in its column c. Past the last one
  // kCols repeats columns before it (N is at least NJ), the others have no column.
  static __device__ __forceinline__ int column(int j, int c, int N, int n0) {
    return KIND == kCols ? min(n0 + NJ * c, N - NJ) + j : n0 + 16 * j + c;
  }

  __device__ __forceinline__ void load(Rows& r, int k0) const {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        r.v[u][i] = __builtin_bit_cast(
            u32x4, load_packed<T, kChunk>(reinterpret_cast<const T*>(xrow[i]) + k0 + u * kStep));
  }
  __device__ __forceinline__ void load(Weights& r, int k0) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (KIND == kCols)
#pragma unroll
        for (int q = 0; q < kChunk; ++q)
          r.raw[u][q] = load_packed<T, NJ>(reinterpret_cast<const T*>(wcol[0]) + (int64_t)(k0 + u * kStep + q) * ld);
      else
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if constexpr (KIND == kRows)
            r.b[u][j] = __builtin_bit_cast(
                u32x4, load_packed<T, kChunk>(reinterpret_cast<const T*>(wcol[j]) + k0 + u * kStep));
          else
            r.b[u][j] = *reinterpret_cast<const u32x4*>(wcol[j] + (int64_t)(k0 / kStep + u) * 1024);
        }
    }
  }

  // The same where the block goes past K: zeros there.
  __device__ __forceinline__ void load_tail(Rows& r, Weights& w, int k0, int K) const {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * kStep, left = K - (k + chunk_at);
#pragma unroll
      for (int i = 0; i < MT; ++i)
        r.v[u][i] = __builtin_bit_cast(
            u32x4, load_guarded<T, kChunk>(reinterpret_cast<const T*>(xrow[i]) + k, 0, left));
      if constexpr (KIND == kRows)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          w.b[u][j] =
              __builtin_bit_cast(u32x4, load_guarded<T, kChunk>(reinterpret_cast<const T*>(wcol[j]) + k, 0, left));
      if constexpr (KIND == kBlocks)  // they hold zeros up to whole pairs of steps
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          w.b[u][j] = k < K ? *reinterpret_cast<const u32x4*>(wcol[j] + (int64_t)(k / kStep) * 1024) : u32x4{0, 0, 0, 0};
      if constexpr (KIND == kCols)
#pragma unroll
        for (int q = 0; q < kChunk; ++q) {
          w.raw[u][q] = Packed<T, NJ>{};
          if (q < left)
            w.raw[u][q] = load_packed<T, NJ>(reinterpret_cast<const T*>(wcol[0]) + (int64_t)(k + q) * ld);
        }
    }
  }

  // Column j of kChunk rows of NJ, as an operand.
  template <int Q>
  static __device__ __forceinline__ u32x4 turned(const Packed<T, NJ> (&raw)[Q], int j) {
    u32x4 v;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = __builtin_bit_cast(uint32_t, raw[q].v[j]);
    } else {
      typedef uint32_t Words __attribute__((ext_vector_type(NJ / 2)));
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t x = __builtin_bit_cast(Words, raw[2 * q])[j / 2], y = __builtin_bit_cast(Words, raw[2 * q + 1])[j / 2];
        v[q] = __builtin_amdgcn_perm(y, x, j % 2 ? 0x07060302u : 0x05040100u);
      }
    }
    return v;
  }

  static __device__ __forceinline__ void multiply(const Rows& r, const Weights& w, Acc (&acc)[MT][NJ]) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        u32x4 b;
        if constexpr (KIND == kCols)
          b = turned(w.raw[u], j);
        else
          b = w.b[u][j];
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][j] = E::mul(r.v[u][i], b, acc[i][j]);
      }
  }

  // store(row, column, sum) of every output of the workgroup's columns.
  template <typename Store>
  static __device__ __forceinline__ void run(const void* x, int64_t ldx, int rows, const void* w, int64_t ldw, int K,
                                             int N, int n0, Acc* lds, Store&& store) {
    Skinny s;
    s.init(x, ldx, rows, w, ldw, N, n0);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = s.lane;
    Acc acc[MT][NJ];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = Acc{};
    const int blocks = K / kDepth;
    // The wave's blocks: AHEAD of weights on their way, from memory, and one of x, from the caches. Past the
    // last one it reads that again.
    const int last = blocks - 1 - (blocks - 1 - wave) % WAVES;
    Rows x_now, x_next;
    Weights ring[AHEAD];
    if (wave < blocks) {
#pragma unroll
      for (int a = 0; a < AHEAD; ++a) s.load(ring[a], min(wave + a * WAVES, last) * kDepth);
      s.load(x_now, wave * kDepth);
#pragma unroll 1
      for (int b = wave; b < blocks; b += AHEAD * WAVES) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
          const int at = b + a * WAVES;
          if (a > 0 && at >= blocks) break;  // uniform
          s.load(x_next, min(at + WAVES, last) * kDepth);
          multiply(x_now, ring[a], acc);
          s.load(ring[a], min(at + AHEAD * WAVES, last) * kDepth);
          x_now = x_next;
        }
      }
    }
    if (blocks * kDepth < K && wave == blocks % WAVES) {
      s.load_tail(x_now, ring[0], blocks * kDepth, K);
      multiply(x_now, ring[0], acc);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if (16 * i >= rows) break;  // uniform
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NJ; ++j) lds[(wave * NJ + j) * 64 + lane] = acc[i][j];
      __syncthreads();
      for (int at = threadIdx.x; at < NJ * 64; at += 64 * WAVES) {
        Acc sum = lds[at];
#pragma unroll
        for (int v = 1; v < WAVES; ++v) sum += lds[v * NJ * 64 + at];
        const int l = at % 64, n = column(at / 64, l % 16, N, n0);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = 16 * i + 4 * (l / 16) + e;
          if (m < rows && n < N) store(m, n, sum[e]);
        }
      }
    }
  }
};

}  // namespace lm
}  // namespace edsl

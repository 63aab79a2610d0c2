// Tiles of a matrix product on the matrix cores, C[m][n] = sum_k A[m][k] B[k][n]:
// what the layers on groups of rows and on 8-bit weights share.
//
// A workgroup of WM x WN waves takes BM x BN outputs; a stage of 128 bytes of k a row
// goes from memory straight to LDS while the one before it is multiplied, two
// stages in turn, one barrier a stage. An operand lies in memory, and in LDS, with
// k contiguous (kRows), with its own index contiguous (kCols: read through the
// transposing LDS load, or element by element in f32) or laid out as the
// instruction takes it (kBlocks, 8-bit weights). 16-byte chunks change places by row
// so that a fragment's reads meet all banks. Where a row starts off 16 bytes, or a
// chunk would cross its end, the chunks go through registers instead, cut
// element by element (ASYNC false).
//
// The two operands are given to the instruction in exchanged places, so that a lane
// ends with four successive n of one row: wide stores.
#pragma once

#include "common.hpp"
#include "lm_common.hpp"

namespace edsl {
namespace lm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

enum OperandKind : int { kRows = 0, kCols = 1, kBlocks = 2 };

// A lane's 16 bytes of one operand against the other's: kStep k for a wave.
template <typename T>
struct TileElem;
template <>
struct TileElem<bf16> {
  typedef bf16 V __attribute__((ext_vector_type(8)));
  using Acc = f32x4;
  static constexpr int kChunk = 8;
  static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
  }
};
template <>
struct TileElem<f16> {
  typedef f16 V __attribute__((ext_vector_type(8)));
  using Acc = f32x4;
  static constexpr int kChunk = 8;
  static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, a), __builtin_bit_cast(V, b), c, 0, 0, 0);
  }
};
template <>
struct TileElem<int8_t> {
  using Acc = i32x4;
  static constexpr int kChunk = 16;
  static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0,
                                                 0);
  }
};
template <>
struct TileElem<float> {
  using Acc = f32x4;
  static constexpr int kChunk = 4;
  static __device__ __forceinline__ Acc mul(u32x4 a, u32x4 b, Acc c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], y[i], c, 0, 0, 0);
    return c;
  }
};

// 16 bytes a lane from memory, descriptor `from` + `offset`, to LDS, `to` (the wave's
// own) + 16 lane; zeros at offsets past the descriptor's end. As the instruction
// itself: for its intrinsic the compiler lets every later read of LDS wait for it,
// whichever buffer it reads. It has no result register; wait_tile_loads() is what waits
// for it.
__device__ __forceinline__ void tile_to_lds(i32x4 from, int offset, const void* to) {
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)at)), "v"(offset), "s"(from)
               : "memory", "m0");
}
// vmcnt 0.
__device__ __forceinline__ void wait_tile_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// One operand of a tile: `n` of its own index's elements are there from `base` on.
struct TileOperand {
  const char* base;  // its first element at k = 0
  int64_t ld;        // elements from one row of memory to the next
  int n;
};

// MN of an operand's own index in LDS and its loads by THREADS threads.
template <typename T, int KIND, int MN, int THREADS, bool ASYNC>
struct TileSide {
  static constexpr int kChunk = TileElem<T>::kChunk;
  static constexpr int kDepth = 8 * kChunk;  // k of a stage
  static constexpr int kAll = MN * 8;        // chunks of a stage
  static constexpr int kMine = kAll / THREADS;
  static_assert(kAll % THREADS == 0 && (MN % 128 == 0 || KIND == kRows), "whole chunks, whole banks");
  static constexpr int kPerRow = KIND == kCols ? MN / kChunk : 8;
  static constexpr int kOutside = (int)0x80000000;  // an offset past every descriptor

  // Chunk `at` of LDS: its row of memory and its first element there.
  static __device__ __forceinline__ void place(int at, int& row, int& col) {
    row = at / kPerRow;
    int c = at % kPerRow;
    if constexpr (KIND == kRows)
      c ^= (row / 2) % 8;  // rows of 128 bytes: two meet all banks
    else if constexpr (sizeof(T) == 4)
      c ^= ((row / 4) % 4) * 4;  // 16 columns, 64 bytes: four rows' meet all banks
    else
      c ^= ((row % 4) | ((row / 8 % 2) << 2)) << 1;  // 16 columns, 32 bytes: eight rows'
    col = c * kChunk;
  }

  int offset[ASYNC ? kMine : 1];
  u32x4 held[ASYNC ? 1 : kMine];

  __device__ __forceinline__ void init(const TileOperand& o, int tid) {
    if constexpr (ASYNC) {
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        const int at = c * THREADS + tid;
        if constexpr (KIND == kBlocks) {
          // Blocks of 16 columns x 64 k, `ld` bytes from 16 columns to the next.
          offset[c] = (int)((at / 128) * o.ld) + (at % 128) * 16;
        } else {
          int row, col;
          place(at, row, col);
          offset[c] = (int)(((int64_t)row * o.ld + col) * (int64_t)sizeof(T));
        }
      }
    }
  }

  // Starts the loads of the stage at k0 of K.
  __device__ __forceinline__ void load(const TileOperand& o, int K, int k0, u32x4* lds, int tid, int wave) {
    if constexpr (ASYNC) {
      i32x4 from;
      if constexpr (KIND == kRows) {
        from = buffer_rsrc(o.base + (int64_t)k0 * sizeof(T), ((o.n - 1) * o.ld + K - k0) * (int64_t)sizeof(T));
      } else if constexpr (KIND == kCols) {
        from = buffer_rsrc(o.base + k0 * o.ld * (int64_t)sizeof(T), ((K - k0 - 1) * o.ld + o.n) * (int64_t)sizeof(T));
      } else {
        from = buffer_rsrc(o.base + (int64_t)k0 * 16, (int64_t)((o.n + 15) / 16) * o.ld - (int64_t)k0 * 16);
      }
      const bool tail = KIND == kRows && k0 + kDepth > K;  // rows go on past K
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        int at = offset[c];
        if (tail) {
          int row, col;
          place(c * THREADS + tid, row, col);
          if (k0 + col >= K) at = kOutside;
        }
        tile_to_lds(from, at, lds + c * THREADS + wave * 64);
      }
    } else {
      static_assert(KIND != kBlocks, "blocks are always aligned");
#pragma unroll
      for (int c = 0; c < kMine; ++c) {
        int row, col;
        place(c * THREADS + tid, row, col);
        const int rows = KIND == kRows ? o.n : K - k0, left = KIND == kRows ? K - k0 : o.n;
        held[c] = u32x4{0, 0, 0, 0};
        if (row < rows && col < left) {
          const T* const p = reinterpret_cast<const T*>(o.base) +
                             (KIND == kRows ? (int64_t)row * o.ld + k0 : (int64_t)(row + k0) * o.ld);
          held[c] = __builtin_bit_cast(u32x4, load_guarded<T, kChunk>(p, col, left));
        }
      }
    }
  }
  __device__ __forceinline__ void put(u32x4* lds, int tid) {
    if constexpr (!ASYNC)
#pragma unroll
      for (int c = 0; c < kMine; ++c) lds[c * THREADS + tid] = held[c];
  }

  // The fragment of block `b` (16 of the operand's index) at step s (half a stage).
  static __device__ __forceinline__ u32x4 fragment(const u32x4* lds, int b, int s, int lane) {
    const int i = lane % 16, g = lane / 16;
    if constexpr (KIND == kRows) {
      const int row = b * 16 + i;
      return lds[row * 8 + ((4 * s + g) ^ ((row / 2) % 8))];
    } else if constexpr (KIND == kBlocks) {
      return lds[(b * 2 + s) * 64 + lane];
    } else if constexpr (sizeof(T) == 4) {
      const float* const p = reinterpret_cast<const float*>(lds) + (16 * s + 4 * g) * MN + ((b ^ g) * 16) + i;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = p[e * MN];
      return __builtin_bit_cast(u32x4, v);
    } else {
      // Lanes 4 q + j of 16 give columns 4 j .. 4 j + 3 of row q and receive column
      // i of rows 0 .. 3.
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4* Lds;
      const char* const p = reinterpret_cast<const char*>(lds) + (32 * s + 8 * g + i / 4) * (2 * MN) +
                            ((b ^ ((i / 4) | ((g % 2) << 2))) * 32) + 8 * (i % 4);
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * 2 * MN)));
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    }
  }
};

template <typename T_, int AKIND, int BKIND, int BM_, int BN_, int WM_, int WN_, bool ASYNC>
struct Tile {
  using T = T_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  using E = TileElem<T>;
  using Acc = typename E::Acc;
  using A = TileSide<T, AKIND, BM, kThreads, ASYNC>;
  using B = TileSide<T, BKIND, BN, kThreads, ASYNC || BKIND == kBlocks>;
  static constexpr int kStage = A::kAll + B::kAll;  // chunks

  // acc[i][j][e]: row 16 (wave's MI + i) + lane % 16, column 16 (wave's NI + j) + 4 (lane / 16) + e.
  static __device__ __forceinline__ void product(const TileOperand& oa, const TileOperand& ob, int K, u32x4* lds,
                                                 Acc (&acc)[MI][NI]) {
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = Acc{};
    A a;
    B b;
    a.init(oa, tid);
    b.init(ob, tid);
    const int stages = (K + A::kDepth - 1) / A::kDepth;
    if (stages > 0) {
      a.load(oa, K, 0, lds, tid, wave);
      b.load(ob, K, 0, lds + A::kAll, tid, wave);
      a.put(lds, tid);
      b.put(lds + A::kAll, tid);
    }
    for (int st = 0; st < stages; ++st) {
      u32x4* const now = lds + (st % 2) * kStage;
      u32x4* const next = lds + ((st + 1) % 2) * kStage;
      if constexpr (ASYNC || BKIND == kBlocks) wait_tile_loads();
      __syncthreads();
      if (st + 1 < stages) {
        a.load(oa, K, (st + 1) * A::kDepth, next, tid, wave);
        b.load(ob, K, (st + 1) * A::kDepth, next + A::kAll, tid, wave);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u32x4 fa[MI], fb[NI];
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[j] = B::fragment(now + A::kAll, wn * NI + j, s, lane);
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[i] = A::fragment(now, wm * MI + i, s, lane);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j) acc[i][j] = E::mul(fb[j], fa[i], acc[i][j]);
      }
      if (!ASYNC && st + 1 < stages) {
        a.put(next, tid);
        b.put(next + A::kAll, tid);
      }
    }
  }
};

template <typename To>
__device__ __forceinline__ Packed<To, 4> get4(const To* p, int n) {
  if (n >= 4) return load_packed<To, 4>(p);
  Packed<To, 4> r{};
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) r.v[e] = p[e];
  return r;
}
__device__ __forceinline__ void get4_typed(const void* p, int64_t at, int type, float (&v)[4], int n) {
  if (type == 0) {
    const auto r = get4(static_cast<const float*>(p) + at, n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = r.v[e];
  } else if (type == 1) {
    const auto r = get4(static_cast<const bf16*>(p) + at, n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)r.v[e];
  } else {
    const auto r = get4(static_cast<const f16*>(p) + at, n);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)r.v[e];
  }
}

// Four values to successive elements of a row of `type`, of which `n` are there.
template <typename To>
__device__ __forceinline__ void put4(To* p, const float (&v)[4], int n) {
  Packed<To, 4> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.v[e] = (To)v[e];
  if (n >= 4)
    *reinterpret_cast<Packed<To, 4>*>(p) = r;
  else
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) p[e] = r.v[e];
}
__device__ __forceinline__ void put4_typed(void* p, int64_t at, int type, const float (&v)[4], int n) {
  if (type == 0)
    put4(static_cast<float*>(p) + at, v, n);
  else if (type == 1)
    put4(static_cast<bf16*>(p) + at, v, n);
  else
    put4(static_cast<f16*>(p) + at, v, n);
}
__device__ __forceinline__ float get_typed(const void* p, int64_t at, int type) {
  if (type == 0) return static_cast<const float*>(p)[at];
  if (type == 1) return (float)static_cast<const bf16*>(p)[at];
  return (float)static_cast<const f16*>(p)[at];
}

// The activation of an epilogue code (uniform), as apply_epilogue_f32 has it.
template <int N>
__device__ __forceinline__ void activate(float (&v)[N], int epi, float alpha) {
  const int act = epi_act(epi);
  if (act == ACT_NONE) return;
#pragma unroll
  for (int e = 0; e < N; ++e)
    v[e] = act == ACT_RELU      ? apply_epilogue_f32<epi_code(false, ACT_RELU)>(v[e], 0.0f, alpha)
           : act == ACT_IF_RELU ? apply_epilogue_f32<epi_code(false, ACT_IF_RELU)>(v[e], 0.0f, alpha)
                                : apply_epilogue_f32<epi_code(false, ACT_LEAKY)>(v[e], 0.0f, alpha);
}

// Tile `w` of total, those of one XCD successive (workgroup w runs on XCD w % 8).
__device__ __forceinline__ int xcd_order(int w, int total) {
  const int x = w % 8, per = total / 8, more = total % 8;
  return x * per + min(x, more) + w / 8;
}

}  // namespace lm
}  // namespace edsl

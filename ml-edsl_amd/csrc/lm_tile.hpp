// Tiles of a matrix product on the matrix cores, C[m][n] = sum_k A[m][k] B[k][n]:
// what the layers on groups of rows and on 8-bit weights share.
//
// A workgroup of WM x WN waves takes BM x BN outputs. Stages of 128 bytes of k a row
// go from memory straight to LDS, two or three of them in turn. Half a stage's fragments
// are read into registers while the half before it is multiplied. In the middle of a stage
// all of it is in registers and the next one has arrived: there is its only barrier, and
// there the loads into its place start, one after every few products, since a wave
// waits for each of them to be taken.
//
// An operand lies in memory, and in LDS, with k contiguous (kRows), with its own index
// contiguous (kCols: read through the transposing LDS load, or element by element in f32)
// or laid out as the instruction takes it (kBlocks, 8-bit weights). 16-byte chunks change
// places by row so that a fragment's reads meet all banks. Where a row starts off 16 bytes, or a
// chunk would cross its end (DIRECT false), they go through registers instead, loaded from any address.
//
// The two operands are given to the instruction in exchanged places, so that a lane
// ends with four successive n of one row: wide stores.
//
// Measured, bf16 4096^3, random values: 256x256 tiles in 123 us (1.12 PFLOP/s; the vendor's product
// takes 128), of which 12 are launch, first loads and stores. Without its loads a product
// takes 112, without its reads of LDS 126, with neither 98: the matrix cores at the clock that power
// leaves them come first, then the loads' way from L2 (48 bytes a clock and CU at most). Matrix
// instructions of one wave a SIMD start every 32 cycles, of two every 16: tiles have eight waves (32 x 64 ones four, of
// several workgroups a CU). Stages of 64 bytes a row, four in LDS, took 137 us (half lines twice); 16 waves with
// a barrier between loads and products 128. Through registers 4096 x 4097 x 4097 takes 233 to 241 us.
// A stage of a lone workgroup takes 0.42 us, through registers 0.5: the loads' way, with two stages of them under way.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "lm_common.hpp"
#include "lm_kernels.hpp"

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
// whichever buffer it reads. It has no result register; tile_arrived() is what waits
// for it.
__device__ __forceinline__ void tile_to_lds(i32x4 from, int offset, const void* to) {
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)to;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane((int)at)), "v"(offset), "s"(from)
               : "memory", "m0");
}
// All waves' loads but their last N have arrived, and their reads of LDS.
template <int N>
__device__ __forceinline__ void tile_arrived() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// All waves' reads and writes of LDS have ended; loads to registers go on.
__device__ __forceinline__ void tile_met() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One operand of a tile: `n` of its own index's elements are there from `base` on.
struct TileOperand {
  const char* base;  // its first element at k = 0
  int64_t ld;        // elements from one row of memory to the next
  int n;
  int64_t all;  // of its own index's elements, those before `base` too
};

// MN of an operand's own index in LDS and its loads by THREADS threads.
template <typename T, int KIND, int MN, int THREADS, bool DIRECT>
struct TileSide {
  static constexpr int kChunk = TileElem<T>::kChunk;
  static constexpr int kDepth = 8 * kChunk;  // k of a stage
  static constexpr int kAll = MN * 8;        // chunks of a stage
  static constexpr int kMine = kAll / THREADS;
  static_assert(kAll % THREADS == 0 && (MN % (sizeof(T) == 4 ? 64 : 128) == 0 || KIND != kCols), "whole chunks, whole banks");
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

  int offset[DIRECT ? kMine : 1];
  const T* from[DIRECT ? 1 : kMine];  // of the first stage
  int by[!DIRECT && KIND == kCols ? kMine : 1];  // columns that a chunk starts before its place
  u32x4 held[2][DIRECT ? 1 : kMine];  // two stages

  __device__ __forceinline__ void init(const TileOperand& o, int tid) {
#pragma unroll
    for (int c = 0; c < kMine; ++c) {
      const int at = c * THREADS + tid;
      if constexpr (KIND == kBlocks) {
        // Blocks of 16 columns x 64 k, `ld` bytes from 16 columns to the next.
        offset[c] = (int)((at / 128) * o.ld) + (at % 128) * 16;
      } else {
        int row, col;
        place(at, row, col);
        if constexpr (DIRECT) {
          offset[c] = (int)(((int64_t)row * o.ld + col) * (int64_t)sizeof(T));
        } else {
          // Rows past the last one repeat it: nobody stores their sums. Chunks past the last column are its row's
          // last elements.
          if constexpr (KIND == kRows) {
            row = min(row, o.n - 1);
          } else {
            by[c] = o.all >= kChunk ? max(col - (o.n - kChunk), 0) : 0;
            col -= by[c];
          }
          from[c] = reinterpret_cast<const T*>(o.base) + row * o.ld + col;
        }
      }
    }
  }

  // A stage at k0 of K, `left` of K from there.
  struct Source {
    i32x4 from;
    int k0, left;
  };
  static __device__ __forceinline__ Source source(const TileOperand& o, int K, int k0) {
    if constexpr (!DIRECT) return {i32x4{}, k0, K - k0};
    if constexpr (KIND == kRows)
      return {buffer_rsrc(o.base + (int64_t)k0 * sizeof(T), ((o.n - 1) * o.ld + K - k0) * (int64_t)sizeof(T)), k0,
              K - k0};
    // Of a word that is not all inside nothing is read: the last row's end is its last word's.
    if constexpr (KIND == kCols)
      return {buffer_rsrc(o.base + k0 * o.ld * (int64_t)sizeof(T),
                          (((K - k0 - 1) * o.ld + o.n) * (int64_t)sizeof(T) + 3) & ~(int64_t)3),
              k0, K - k0};
    return {buffer_rsrc(o.base + (int64_t)k0 * 16, (int64_t)((o.n + 15) / 16) * o.ld - (int64_t)k0 * 16), k0, K - k0};
  }
  // Starts load c of kMine of a stage, which has all its rows and columns where WHOLE.
  template <bool WHOLE = false>
  __device__ __forceinline__ void load(int c, const Source& s, const TileOperand& o, u32x4* lds, int tid, int wave,
                                       int hold = 0) {
    int row, col;
    if constexpr (DIRECT) {
      int at = offset[c];
      if constexpr (KIND == kRows) {  // rows go on past K
        place(c * THREADS + tid, row, col);
        at = col < s.left ? at : kOutside;
      }
      tile_to_lds(s.from, at, lds + c * THREADS + wave * 64);
    } else {
      static_assert(KIND != kBlocks, "blocks are always aligned");
      if constexpr (KIND == kRows) {
        if (WHOLE || s.left >= kDepth) {  // uniform
          held[hold][c] = __builtin_bit_cast(u32x4, load_packed<T, kChunk>(from[c] + s.k0));
        } else {
          place(c * THREADS + tid, row, col);
          held[hold][c] = __builtin_bit_cast(u32x4, load_guarded<T, kChunk>(from[c] + s.k0, 0, s.left - col));
        }
      } else {
        // What depends on a loaded value waits for it: chunks are moved to their places as they are put.
        const T* const p = from[c] + s.k0 * o.ld;
        place(c * THREADS + tid, row, col);
        if (WHOLE || (s.left >= kDepth && o.all >= kChunk)) {  // uniform
          held[hold][c] = __builtin_bit_cast(u32x4, load_packed<T, kChunk>(p));
        } else {
          held[hold][c] = u32x4{0, 0, 0, 0};
          if (row < s.left)
            held[hold][c] = o.all >= kChunk
                                ? __builtin_bit_cast(u32x4, load_packed<T, kChunk>(p))
                                : __builtin_bit_cast(u32x4, load_guarded<T, kChunk>(p, col, o.n));
        }
      }
    }
  }
  // The elements from `by` on, from the first place on.
  static __device__ __forceinline__ u32x4 moved(u32x4 v, int by) {
    const unsigned bits = (unsigned)by * 8 * sizeof(T);
    const uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
    const uint64_t up = bits < 64 ? hi >> bits : 0;
    const uint64_t low = bits == 0 ? lo : bits < 64 ? lo >> bits | hi << (64 - bits) : bits < 128 ? hi >> (bits - 64) : 0;
    return u32x4{(uint32_t)low, (uint32_t)(low >> 32), (uint32_t)up, (uint32_t)(up >> 32)};
  }
  __device__ __forceinline__ void put(const TileOperand& o, u32x4* lds, int tid, int hold) {
    if constexpr (!DIRECT) {
      if (KIND == kCols && o.n < MN && o.all >= kChunk)  // uniform
#pragma unroll
        for (int c = 0; c < kMine; ++c) held[hold][c] = moved(held[hold][c], by[KIND == kCols ? c : 0]);
#pragma unroll
      for (int c = 0; c < kMine; ++c) lds[c * THREADS + tid] = held[hold][c];
    }
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

// NS stages in LDS.
template <typename T_, int AKIND, int BKIND, int BM_, int BN_, int WM_, int WN_, bool DIRECT, int NS = 2>
struct Tile {
  using T = T_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  using E = TileElem<T>;
  using Acc = typename E::Acc;
  using A = TileSide<T, AKIND, BM, kThreads, DIRECT>;
  using B = TileSide<T, BKIND, BN, kThreads, DIRECT || BKIND == kBlocks>;
  static constexpr int kStage = A::kAll + B::kAll;  // chunks
  static constexpr int kLds = NS * kStage;
  // Waves a SIMD that LDS leaves room for: two workgroups of eight waves a CU, or one.
  static constexpr int kWavesPerSimd = kLds * 16 <= 80 * 1024 ? 4 : 2;

  // acc[i][j][e]: row 16 (wave's MI + i) + lane % 16, column 16 (wave's NI + j) + 4 (lane / 16) + e.
  static __device__ __forceinline__ void product(const TileOperand& oa, const TileOperand& ob, int K, u32x4* lds,
                                                 Acc (&acc)[MI][NI]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = Acc{};
    add_product(oa, ob, K, lds, acc);
  }
  static __device__ __forceinline__ void add_product(const TileOperand& oa, const TileOperand& ob, int K, u32x4* lds,
                                                     Acc (&acc)[MI][NI]) {
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wm = wave / WN, wn = wave % WN;
    const int stages = (K + A::kDepth - 1) / A::kDepth;
    if (stages == 0) return;
    A a;
    B b;
    a.init(oa, tid);
    b.init(ob, tid);
    constexpr int kLoads = A::kMine + B::kMine;  // of a stage, a thread
    constexpr int kAll = A::kMine + B::kMine;
    struct Fragments {
      u32x4 a[MI], b[NI];
    };
    const auto read = [&](const u32x4* from, int s, Fragments& f) {
#pragma unroll
      for (int j = 0; j < NI; ++j) f.b[j] = B::fragment(from + A::kAll, wn * NI + j, s, lane);
#pragma unroll
      for (int i = 0; i < MI; ++i) f.a[i] = A::fragment(from, wm * MI + i, s, lane);
    };
    struct Sources {
      typename A::Source a;
      typename B::Source b;
    };
    // Stages past the last one read nothing: their descriptors, or their elements, are none.
    const auto sources = [&](int st) {
      return Sources{A::source(oa, K, st * A::kDepth), B::source(ob, K, st * A::kDepth)};
    };
    const auto load = [&](int c, const Sources& s, u32x4* to, int hold, auto whole) {
      constexpr bool kWhole = decltype(whole)::value;
      if (c < A::kMine)
        a.template load<kWhole>(c, s.a, oa, to, tid, wave, hold);
      else
        b.template load<kWhole>(c - A::kMine, s.b, ob, to + A::kAll, tid, wave, hold);
    };
    const auto load_all = [&](int st, u32x4* to, int hold, auto whole) {
      const Sources s = sources(st);
#pragma unroll
      for (int c = 0; c < kAll; ++c) load(c, s, to, hold, whole);
    };
    const auto put_all = [&](u32x4* to, int hold) {
      a.put(oa, to, tid, hold);
      b.put(ob, to + A::kAll, tid, hold);
    };
    const auto run = [&](auto working) {
      constexpr bool kWorks = decltype(working)::value;
      Fragments f0, f1;
      if constexpr (DIRECT) {
#pragma unroll
        for (int st = 0; st < NS; ++st) load_all(st, lds + st * kStage, 0, std::false_type{});
        tile_arrived<(NS - 1) * kLoads>();
        if constexpr (kWorks) read(lds, 0, f0);
        int at = 0;
        for (int st = 0; st < stages; ++st) {
          u32x4* const now = lds + at * kStage;
          at = at + 1 == NS ? 0 : at + 1;
          u32x4* const next = lds + at * kStage;
          if constexpr (kWorks) {
            __builtin_amdgcn_sched_barrier(0);
            read(now, 1, f1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
              for (int j = 0; j < NI; ++j) acc[i][j] = E::mul(f0.b[j], f0.a[i], acc[i][j]);
          }
          const Sources s = sources(st + NS);
          __builtin_amdgcn_sched_barrier(0);
          tile_arrived<(NS - 2) * kLoads>();
          if constexpr (kWorks) read(next, 0, f0);
          // The loads between the products: a wave waits for each to be taken.
#pragma unroll
          for (int c = 0; c < kAll; ++c) {
            __builtin_amdgcn_sched_barrier(0);
            load(c, s, now, 0, std::false_type{});
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (kWorks)
#pragma unroll
              for (int m = c * MI * NI / kAll; m < (c + 1) * MI * NI / kAll; ++m)
                acc[m / NI][m % NI] = E::mul(f1.b[m % NI], f1.a[m / NI], acc[m / NI][m % NI]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        tile_arrived<0>();  // nothing is on its way to LDS when the workgroup ends
      } else {
        static_assert(DIRECT || NS == 2, "a stage at a time goes through registers");
        constexpr int kHeld = BKIND == kBlocks ? A::kMine : kAll;
        // One stage in LDS, two on their way in registers. Blocks of weights go straight to LDS, a stage ahead.
        const auto turn = [&](int st, int hold, auto whole) {
          u32x4* const now = lds + st % 2 * kStage;
          u32x4* const next = lds + (st + 1) % 2 * kStage;
          if constexpr (BKIND == kBlocks)
            tile_arrived<0>();
          else
            tile_met();
          if constexpr (BKIND == kBlocks) {
            const Sources s = sources(st + 1);
#pragma unroll
            for (int c = 0; c < B::kMine; ++c) b.load(c, s.b, ob, next + A::kAll, tid, wave);
          }
          if constexpr (kWorks)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              read(now, s, f0);
#pragma unroll
              for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = E::mul(f0.b[j], f0.a[i], acc[i][j]);
            }
          put_all(next, hold);
          const Sources s = sources(st + 3);
#pragma unroll
          for (int c = 0; c < kHeld; ++c) load(c, s, next, hold, whole);
        };
        const auto start = [&](auto whole) {
          load_all(0, lds, 0, whole);
          put_all(lds, 0);
          const Sources one = sources(1), two = sources(2);
#pragma unroll
          for (int c = 0; c < kHeld; ++c) load(c, one, lds, 0, whole);
#pragma unroll
          for (int c = 0; c < kHeld; ++c) load(c, two, lds, 1, whole);
        };
        // Turns that start loads of whole stages have no branch between their loads: where paths of more and of
        // fewer loads meet, the compiler waits for all.
        const int even = ((AKIND == kRows || oa.all >= A::kChunk) && (BKIND != kCols || ob.all >= A::kChunk)
                              ? K / A::kDepth - 3 : 0) / 2 * 2;
        int st = 0;
        if (even > 0) {
          start(std::true_type{});
          for (; st < even; st += 2) {
            turn(st, 0, std::true_type{});
            turn(st + 1, 1, std::true_type{});
          }
        } else {
          start(std::false_type{});
        }
#pragma unroll 1
        for (; st + 2 <= stages; st += 2) {
          turn(st, 0, std::false_type{});
          turn(st + 1, 1, std::false_type{});
        }
        if (st < stages) turn(st, 0, std::false_type{});
        tile_arrived<0>();
      }
    };
    // A wave whose rows are all past the operand's leaves the matrix cores to the others.
    if (wm * MI * 16 < oa.n)
      run(std::true_type{});
    else
      run(std::false_type{});
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

// What a wave has of 16 rows and of two neighbouring blocks of 16 columns, a lane four of each of its row
// (Tile::product), to the rows from `first` on, `ld` apart, of which `rows` are there, and from column n0 on of `cols`. 16 bytes a
// lane: of 16-bit outputs, lanes 16 apart exchange halves, so that the even ones have eight of the first block and the
// odd ones of the second; of 32-bit ones, lanes eight rows apart exchange a block, so that a store has 128 bytes of each of
// eight rows (gradients of 8 x 4096 x 4096 in f32 from 8192 rows in 354 us, in pieces of 64 bytes in 374). Past the
// caches: these in 326 us and with plain stores in 388, from 512 rows in 130 and 189.
template <typename To>
__device__ __forceinline__ void put_blocks(To* first, int64_t ld, int64_t rows, int n0, int64_t cols, const float (&v0)[4],
                                           const float (&v1)[4]) {
  const int lane = threadIdx.x % 64, g = lane / 16;
  if constexpr (sizeof(To) == 4) {
    const bool upper = lane & 8;
    Packed<float, 4> low, high;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float got = dpp<0x128>(upper ? v0[e] : v1[e]);  // the other's, of a row's 16 lanes eight on
      low.v[e] = upper ? got : v0[e];
      high.v[e] = upper ? v1[e] : got;
    }
    const int row = lane % 8, n = n0 + (upper ? 16 : 0) + 4 * g;
    if (row < rows) store_guarded<float, 4>(first + row * ld, n, cols, low);
    if (row + 8 < rows) store_guarded<float, 4>(first + (row + 8) * ld, n, cols, high);
  } else {
    typedef uint32_t Two __attribute__((ext_vector_type(2)));
    Packed<To, 4> r0, r1;
#pragma unroll
    for (int e = 0; e < 4; ++e) r0.v[e] = (To)v0[e], r1.v[e] = (To)v1[e];
    const Two a = __builtin_bit_cast(Two, r0), b = __builtin_bit_cast(Two, r1);
    const auto low = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto high = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    const u32x4 all{low[0], high[0], low[1], high[1]};
    const int row = lane % 16;
    if (row < rows)
      store_guarded<To, 8>(first + row * ld, n0 + 16 * (g % 2) + 8 * (g / 2), cols, __builtin_bit_cast(Packed<To, 8>, all));
  }
}
// A row's outputs of one block, four a lane.
template <typename To>
__device__ __forceinline__ void put4(To* row, int n, int64_t cols, const float (&v)[4], bool there) {
  Packed<To, 4> r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r.v[e] = (To)v[e];
  if (there) store_guarded<To, 4>(row, n, cols, r);
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

// Eight row tiles go along the columns together.
constexpr int kTogether = 8;
// Tile `at` of rows x tiles_n: its row tile and column strip.
__device__ __forceinline__ int row_of_tile(int at, int rows, int tiles_n, int* tn) {
  const int group = at / (kTogether * tiles_n), first = group * kTogether, high = min(rows - first, kTogether);
  at -= group * kTogether * tiles_n;
  *tn = at / high;
  return first + at % high;
}

// Which tile a workgroup takes of `total` tiles of the largest shape: those come in whole rounds of the
// CUs, and what is left is cut in four where there are up to `quarters` tiles, or else in two up to `halves`.
struct TileTurn {
  int tile, sub, pieces;  // piece `sub` of 1, 2 or 4
};
// The most workgroups, whatever `total` up to `most` is.
inline int64_t tile_turns(int64_t most, const TileRounds& r) { return most + 3 * r.quarters + r.halves; }
__device__ __forceinline__ bool tile_turn(int w, int total, int first_part, const TileRounds& r, TileTurn* turn) {
  int whole = total / r.cus * r.cus, left = total - whole;
  const int pieces = left <= r.quarters ? 4 : left <= r.halves ? 2 : 1;
  if (pieces == 1) whole = total, left = 0;
  if (w < whole) {
    // Tiles from first_part on have fewer rows: each XCD has its share of both.
    const int even = min(whole, first_part);
    *turn = {w < even ? xcd_order(w, even) : even + xcd_order(w - even, whole - even), 0, 1};
    return true;
  }
  w -= whole;
  if (w >= left * pieces) return false;
  w = xcd_order(w, left * pieces);
  *turn = {whole + w / pieces, w % pieces, pieces};
  return true;
}

}  // namespace lm
}  // namespace edsl

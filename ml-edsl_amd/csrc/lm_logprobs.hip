// Log probabilities of given tokens under softmax(scale * logits), with
// log-sum-exp, entropy and the largest alternatives; and the gradient of the
// logits.
//
// With m = max x and c = scale * log2(e), in units of log 2:
//   u_j = (x_j - m) c;  e_j = 2^u_j;  s = sum e_j;  t = sum e_j u_j
//   lse = scale m + ln2 log2 s;  logprob = scale (x_token - m) - ln2 log2 s;
//   entropy = ln2 (log2 s - t / s)
// The difference is taken before the product, so that logits of the type's
// lowest value do not overflow.
//
// Bound by memory: a logit is read once, into registers, where its workgroup
// finds the maximum, the sums and the alternatives. Second come the vector ALUs,
// some seven operations and an exponential an element: 2048 x 50256 in bf16 46 us
// (4.5 TB/s), with five alternatives 47, in f32 70 (5.9 TB/s). The gradient of 2048
// x 50256 bf16 logits takes 71 us (5.8 TB/s). One row of 50256 takes 6.1 us, with
// eight alternatives 8.2: one workgroup's latency.
//
// Alternatives: the threads' maxima fall into 64 classes by lane. At least k
// elements reach the k-th largest class maximum T, and few more do where large
// logits are spread over the lanes; these go to a list and are ranked by
// counting, by (value, lower index). Lists that do not fit (rows of equal
// values) are found one by one instead.
#include "kernels.hpp"
#include "lm_common.hpp"
#include "lm_kernels.hpp"

namespace edsl {
namespace lm {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kVectors = 256;  // vectors that hold candidates, of one workgroup
constexpr int kList = 512;     // its candidates
constexpr int kMaxChunks = 64; // parts of a row: one lane each in the join
constexpr int kNoIndex = 0x7fffffff;

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// Part of a row: its maximum m (0 where all of it is -inf), s and t.
struct Part {
  float m, s, t;
};

// Adds up parts over the 64 lanes: every lane returns the sum. `any`: the lane's
// part is not all -inf.
__device__ __forceinline__ Part wave_join(Part p, bool any, float c) {
  float m = wave_all<Max>(any ? p.m : neg_inf());
  if (m == neg_inf()) m = 0.0f;
  // A part of -inf alone has s = t = 0, or NaN where it holds one.
  const float d = any ? fmaxf((p.m - m) * c, -1000.0f) : 0.0f;
  // m = +inf: the difference is NaN, and fmaxf dropped it, but s is NaN already.
  const float f = __builtin_amdgcn_exp2f(d);
  return {m, wave_all<Sum>(p.s * f), wave_all<Sum>((p.t + p.s * d) * f)};
}

template <int CTRL>
__device__ __forceinline__ int dpp_int(int v) {
  return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true);
}

__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

// The largest T, to 20 leading bits, that at least k of the 64 lanes' values reach.
__device__ __forceinline__ float kth_of_lanes(float v, int k) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, v);
  const uint32_t key = bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 12; --b) {
    const uint32_t c = t | (1u << b);
    if (__popcll(__ballot(key >= c)) >= k) t = c;
  }
  // Keys below -inf's stand for NaN: no value is under -inf.
  const uint32_t low = 0x007fffffu;  // the key of -inf
  if (t <= low) return neg_inf();
  return __builtin_bit_cast(float, (t >> 31) ? t ^ 0x80000000u : ~t);
}

__device__ __forceinline__ int64_t id_at(const void* ids, bool ids64, int64_t i) {
  return ids64 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}
__device__ __forceinline__ void put_id(void* ids, bool ids64, int64_t i, int v) {
  if (ids64)
    static_cast<int64_t*>(ids)[i] = v;
  else
    static_cast<int32_t*>(ids)[i] = v;
}

// The given token's logit, read early by the thread that writes the results.
struct Given {
  bool in;  // inside the vocabulary
  float x;
};
template <typename T>
__device__ __forceinline__ Given read_given(const LogprobsArgs& a, int64_t row) {
  Given g{false, 0.0f};
  if (a.logprobs) {
    const int64_t id = id_at(a.tokens, a.ids64, row);
    g.in = id >= 0 && id < a.V;
    if (g.in) g.x = (float)static_cast<const T*>(a.x)[row * a.ldx + id];
  }
  return g;
}

// The results of a row, by one thread, from its whole sums.
__device__ __forceinline__ void finish_row(const LogprobsArgs& a, int64_t row, Given g, Part p, bool none, float log_s) {
  if (a.lse) a.lse[row] = none ? neg_inf() : fmaf(kLn2, log_s, a.scale * p.m);
  if (a.entropy) a.entropy[row] = none ? 0.0f : kLn2 * (log_s - p.t / p.s);
  if (a.logprobs) a.logprobs[row] = !g.in ? 0.0f : none ? neg_inf() : fmaf(-kLn2, log_s, (g.x - p.m) * a.scale);
}

// The workspace: the parts of all rows, then k (value, index) pairs of each.
struct Pair {
  float v;
  int i;
};
__device__ __forceinline__ Part* parts_of(const LogprobsArgs& a, int64_t row) {
  return reinterpret_cast<Part*>(a.partials) + row * a.chunks;
}
__device__ __forceinline__ Pair* pairs_of(const LogprobsArgs& a, int64_t row) {
  return reinterpret_cast<Pair*>(a.partials + (a.M * a.chunks * (int64_t)sizeof(Part) + 15) / 16 * 16) +
         row * a.chunks * a.k;
}

// An alternative of a row, to its results.
__device__ __forceinline__ void put_top(const LogprobsArgs& a, int64_t row, int r, float value, int index, Part p,
                                        bool bad, bool none, float log_s) {
  a.top[row * a.k + r] = bad ? __builtin_nanf("") : none ? neg_inf() : fmaf(-kLn2, log_s, (value - p.m) * a.scale);
  put_id(a.top_ids, a.ids64, row * a.k + r, bad ? -1 : index);
}

template <typename T, int THREADS, int NV, bool TOP>
__global__ void __launch_bounds__(THREADS, NV <= 8 ? 8 : 4) logprobs_kernel(LogprobsArgs a, int64_t part_len) {
  constexpr int VEC = kVec<T>, WAVES = THREADS / 64;
  using Vals = Packed<T, VEC>;
  __shared__ float maxima[TOP ? WAVES : 1][64];
  __shared__ Part parts[WAVES];
  __shared__ float list_v[TOP ? kList : 1];
  __shared__ int list_i[TOP ? kList : 1];
  __shared__ u32x4 vector_v[TOP ? kVectors : 1];
  __shared__ int vector_i[TOP ? kVectors : 1];
  __shared__ int vectors, count;
  __shared__ float best_v[WAVES];
  __shared__ int best_i[WAVES];
  const int64_t row = block_of() / (uint32_t)a.chunks;
  if (row >= a.M) return;
  const int chunk = (int)(block_of() - row * a.chunks);
  const int64_t first = chunk * part_len;
  const int n = (int)(first + part_len < a.V ? part_len : a.V - first);  // > 0
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx + first;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const float c = a.scale * kLog2e;
  Given given{};
  if (tid == 0) {
    vectors = count = 0;
    if (a.chunks == 1) given = read_given<T>(a, row);
  }

  // The part stays in registers in its own type: 16-byte vectors, whole ones
  // without a check, -inf past the end.
  u32x4 v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = (j * THREADS + tid) * VEC;
    if ((j + 1) * THREADS * VEC <= n)
      v[j] = __builtin_bit_cast(u32x4, load_packed<T, VEC>(x + at));
    else
      v[j] = __builtin_bit_cast(u32x4, load_guarded<T, VEC>(x, at, n, (T)neg_inf()));
  }
  float top = neg_inf();
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const auto r = __builtin_bit_cast(Vals, v[j]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) top = fmaxf(top, (float)r.v[e]);
    // Else the compiler keeps all elements in 32 bits, twice the registers.
    asm("" : "+v"(v[j]));
  }
  if constexpr (TOP) maxima[wave][lane] = top;
  const bool any = top > neg_inf();
  Part p{any ? top : 0.0f, 0.0f, 0.0f};
  const auto add_up = [&](auto u_of) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (j * THREADS * VEC >= n) break;
      const auto r = __builtin_bit_cast(Vals, v[j]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float u = u_of((float)r.v[e]);
        const float w = __builtin_amdgcn_exp2f(u);
        p.s += w;
        p.t = fmaf(w, fmaxf(u, -200.0f), p.t);  // 0 for -inf: w is 0 there
      }
    }
  };
  // One fma an element, where the rounding of m c is 8 at most, so that no power of two
  // of it overflows. (m is the thread's own maximum: one whose elements all have a mask
  // of -1e10, say, is enough for the other way, which has no such limit.)
  const float mc = p.m * c;
  if (__all(fabsf(mc) < 0x1p28f)) {
    add_up([&](float x) { return fmaf(x, c, -mc); });
    // What was subtracted is m c rounded: back to m itself.
    const float d = fmaf(p.m, c, -mc), f = __builtin_amdgcn_exp2f(-d);
    p.t = (p.t - d * p.s) * f;
    p.s *= f;
  } else {
    add_up([&](float x) { return (x - p.m) * c; });
  }
  if constexpr (TOP)
#pragma unroll
    for (int j = 0; j < NV; ++j) asm("" : "+v"(v[j]));
  p = wave_join(p, any, c);
  if (lane == 0) parts[wave] = p;
  __syncthreads();
  // Every wave adds the waves' parts up for itself.
  Part all = lane < WAVES ? parts[lane] : Part{0.0f, 0.0f, 0.0f};
  all = wave_join(all, all.s > 0.0f || all.s != all.s, c);
  const bool bad = all.s != all.s;      // a NaN, or +inf less itself
  const bool none = !bad && all.s == 0.0f;
  const float log_s = log2f(all.s);

  const bool whole = a.chunks == 1;
  if (tid == 0) {
    if (whole)
      finish_row(a, row, given, all, none, log_s);
    else
      parts_of(a, row)[chunk] = all;
  }
  if constexpr (TOP) {
    const int k = a.k;
    // The r-th alternative: to the row's results, or to the join.
    const auto put = [&](int r, float value, int index) {
      if (whole)
        put_top(a, row, r, value, index, all, bad, none, log_s);
      else
        pairs_of(a, row)[chunk * k + r] = {value, index == kNoIndex ? index : (int)first + index};
    };
    if (bad) {
      if (tid < k) put(tid, neg_inf(), kNoIndex);
      return;
    }
    // By the first wave: the others leave the CU to its other workgroups.
    if (wave == 0) {
      float classes = maxima[0][lane];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) classes = fmaxf(classes, maxima[w][lane]);
      const float t = kth_of_lanes(classes, k);
      if (lane == 0) best_v[0] = t;
    }
    __syncthreads();
    const float least = best_v[0];
    // Vectors with an element that reaches it, then those elements.
    if (__any(any && top >= least)) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j * THREADS * VEC >= n) break;
        const auto r = __builtin_bit_cast(Vals, v[j]);
        float most = neg_inf();
#pragma unroll
        for (int e = 0; e < VEC; ++e) most = fmaxf(most, (float)r.v[e]);
        if (most >= least && most > neg_inf()) {
          const int at = atomicAdd(&vectors, 1);
          if (at < kVectors) {
            vector_v[at] = v[j];
            vector_i[at] = (j * THREADS + tid) * VEC;
          }
        }
        asm("" : "+v"(v[j]));
      }
    }
    __syncthreads();
    const int held = vectors;
    for (int i = tid; i < (held < kVectors ? held : kVectors) * VEC; i += THREADS) {
      const float value = (float)reinterpret_cast<const T*>(vector_v)[i];
      if (value >= least && value > neg_inf()) {
        const int at = atomicAdd(&count, 1);
        if (at < kList) {
          list_v[at] = value;
          list_i[at] = vector_i[i / VEC] + i % VEC;
        }
      }
    }
    __syncthreads();
    const int found = count;
    if (held <= kVectors && found <= kList) {
      // Eight threads a candidate (65 x 32001 with 20 alternatives in 8.2 us, one
      // thread each in 9.9).
      for (int i = tid / 8; i < found; i += THREADS / 8) {
        const float value = list_v[i];
        const int index = list_i[i];
        int rank = 0;
#pragma unroll 4
        for (int j = tid % 8; j < found; j += 8) rank += better(list_v[j], list_i[j], value, index);
        rank += dpp_int<0xB1>(rank);
        rank += dpp_int<0x4E>(rank);
        rank += dpp_int<0x141>(rank);
        if (tid % 8 == 0 && rank < k) put(rank, value, index);
      }
      if (found < k && wave == 0) {
        // Fewer than k are not -inf: the others are the first of those that are.
        bool masked = lane < n;
        for (int j = 0; j < found; ++j) masked = masked && list_i[j] != lane;
        const uint64_t set = __ballot(masked);
        const int r = found + __popcll(set & ((1ull << lane) - 1));
        if (masked && r < k) put(r, neg_inf(), lane);
        const int filled = found + __popcll(set);  // a part shorter than k
        if (lane < k && lane >= filled) put(lane, neg_inf(), kNoIndex);
      }
      return;
    }
    // One alternative after the other: the best that follows the last one. From
    // memory again, which leaves the registers to the other workgroups' rows.
    // (best_v is free: its readers are past a barrier.)
    float last_v = __builtin_inff();
    int last_i = -1;
    for (int r = 0; r < k; ++r) {
      float bv = neg_inf();
      int bi = kNoIndex;
      for (int at = tid * VEC; at < n; at += THREADS * VEC) {
        const auto vals = load_guarded<T, VEC>(x, at, n, (T)neg_inf());
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float value = (float)vals.v[e];
          if (at + e < n && better(last_v, last_i, value, at + e) && better(value, at + e, bv, bi)) {
            bv = value;
            bi = at + e;
          }
        }
      }
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const float ov = __shfl_xor(bv, d);
        const int oi = __shfl_xor(bi, d);
        if (better(ov, oi, bv, bi)) {
          bv = ov;
          bi = oi;
        }
      }
      if (lane == 0) {
        best_v[wave] = bv;
        best_i[wave] = bi;
      }
      __syncthreads();
      bv = best_v[0];
      bi = best_i[0];
      for (int w = 1; w < WAVES; ++w)
        if (better(best_v[w], best_i[w], bv, bi)) {
          bv = best_v[w];
          bi = best_i[w];
        }
      __syncthreads();
      if (tid == 0) put(r, bv, bi);
      last_v = bv;
      last_i = bi;
    }
  }
}

// Joins the parts of a row, one a lane, in one wave; its alternatives come from
// the parts' by the same way as theirs from the logits.
template <typename T>
__global__ void __launch_bounds__(64) logprobs_join_kernel(LogprobsArgs a) {
  constexpr int kFew = 128;
  __shared__ Pair pairs[kMaxChunks * kMaxTop];
  __shared__ Pair list[kFew];
  __shared__ int count;
  const int64_t row = block_of();
  if (row >= a.M) return;
  const int lane = threadIdx.x, k = a.k, n = a.chunks * k;
  const Given given = read_given<T>(a, row);
  Part p = lane < a.chunks ? parts_of(a, row)[lane] : Part{0.0f, 0.0f, 0.0f};
  const Pair* const from = pairs_of(a, row);
  float top = neg_inf();
#pragma unroll 4
  for (int i = lane; i < n; i += 64) {
    const Pair q = from[i];
    pairs[i] = q;
    top = fmaxf(top, q.v);
  }
  if (lane == 0) count = 0;
  const float c = a.scale * kLog2e;
  p = wave_join(p, p.s > 0.0f || p.s != p.s, c);
  const bool bad = p.s != p.s, none = !bad && p.s == 0.0f;
  const float log_s = log2f(p.s);
  if (lane == 0) finish_row(a, row, given, p, none, log_s);
  if (k == 0) return;
  if (bad) {
    if (lane < k) put_top(a, row, lane, 0.0f, 0, p, bad, none, log_s);
    return;
  }
  const float least = kth_of_lanes(top, k);
  __syncthreads();
  for (int i = lane; i < n; i += 64)
    if (pairs[i].v >= least && pairs[i].i != kNoIndex) {
      const int at = atomicAdd(&count, 1);
      if (at < kFew) list[at] = pairs[i];
    }
  __syncthreads();
  const int found = count;
  if (found <= kFew && found >= k) {
    for (int i = lane; i < found; i += 64) {
      const Pair q = list[i];
      int rank = 0;
      for (int j = 0; j < found; ++j) rank += better(list[j].v, list[j].i, q.v, q.i);
      if (rank < k) put_top(a, row, rank, q.v, q.i, p, bad, none, log_s);
    }
    return;
  }
  // Many equal ones: each part's are in order, so the row's are taken from the
  // heads of the parts' lists.
  int at = 0;
  for (int r = 0; r < k; ++r) {
    const bool has = lane < a.chunks && at < k;
    const Pair q = has ? pairs[lane * k + at] : Pair{neg_inf(), kNoIndex};
    float bv = q.v;
    int bi = q.i;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const float ov = __shfl_xor(bv, d);
      const int oi = __shfl_xor(bi, d);
      if (better(ov, oi, bv, bi)) {
        bv = ov;
        bi = oi;
      }
    }
    if (has && q.i == bi && q.i != kNoIndex) ++at;
    if (lane == 0) put_top(a, row, r, bv, bi, p, bad, none, log_s);
  }
}

template <typename T, int THREADS, int NV>
hipError_t launch_parts(const LogprobsArgs& a, int64_t part_len, hipStream_t stream) {
  const dim3 grid = grid_of(a.M * a.chunks);
  if (a.k > 0)
    hipLaunchKernelGGL((logprobs_kernel<T, THREADS, NV, true>), grid, dim3(THREADS), 0, stream, a, part_len);
  else
    hipLaunchKernelGGL((logprobs_kernel<T, THREADS, NV, false>), grid, dim3(THREADS), 0, stream, a, part_len);
  return launched();
}

// Elements of a part, a multiple of the vector.
int64_t part_length(int64_t V, int chunks, int vec) {
  const int64_t len = (V + chunks - 1) / chunks;
  return (len + vec - 1) / vec * vec;
}

template <typename T>
hipError_t launch_logprobs(const LogprobsArgs& a, hipStream_t stream) {
  const int64_t len = part_length(a.V, a.chunks, kVec<T>), vecs = len / kVec<T>;
  hipError_t e;
  if (vecs <= 256)
    e = launch_parts<T, 256, 1>(a, len, stream);
  else if (a.many && vecs <= 512)
    e = launch_parts<T, 256, 2>(a, len, stream);
  else if (a.many && vecs <= 1024)
    e = launch_parts<T, 256, 4>(a, len, stream);
  else if (vecs <= 1024)
    e = launch_parts<T, 1024, 1>(a, len, stream);
  else if (vecs <= 2048)
    e = launch_parts<T, 1024, 2>(a, len, stream);
  else if (vecs <= 4096)
    e = launch_parts<T, 1024, 4>(a, len, stream);
  else if (vecs <= 8192)
    e = launch_parts<T, 1024, 8>(a, len, stream);
  else
    e = launch_parts<T, 1024, 16>(a, len, stream);
  if (e != hipSuccess || a.chunks == 1) return e;
  hipLaunchKernelGGL((logprobs_join_kernel<T>), grid_of(a.M), dim3(64), 0, stream, a);
  return launched();
}

// ---------------------------------------------------------------- backward
// p_j = exp(d_j), d_j = scale x_j - lse (one rounding, exact where p is near 1);
// dx_j = scale (dlp ([j == token] - p_j) - dent p_j (d_j + entropy)).
// The bracket is one fma of d and g + dent entropy. The token's own element is
// put right by the thread that has it.
constexpr int kBackThreads = 256, kBackVecs = 4;

template <typename T, bool ENT>
__global__ void __launch_bounds__(kBackThreads) logprobs_backward_kernel(LogprobsBackwardArgs a, int chunks) {
  constexpr int VEC = kVec<T>;
  using Vals = Packed<T, VEC>;
  const int64_t row = block_of() / (uint32_t)chunks;
  if (row >= a.M) return;
  const int first = (int)(block_of() - row * chunks) * (kBackThreads * kBackVecs * VEC);
  const int n = (int)a.V - first;
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx + first;
  T* const dx = static_cast<T*>(a.dx) + row * a.lddx + first;
  Vals v[kBackVecs];
  const bool full = n >= kBackThreads * kBackVecs * VEC;
  if (full) {
#pragma unroll
    for (int j = 0; j < kBackVecs; ++j) v[j] = load_packed<T, VEC>(x + (j * kBackThreads + threadIdx.x) * VEC);
  } else {
#pragma unroll
    for (int j = 0; j < kBackVecs; ++j)
      v[j] = load_guarded<T, VEC>(x, (j * kBackThreads + threadIdx.x) * VEC, n, (T)neg_inf());
  }
  const float lse = a.lse[row];
  int id = -1;  // the token's place here
  float g = 0.0f;
  if (a.dlogprobs) {
    const int64_t t = id_at(a.tokens, a.ids64, row);
    if (t >= 0 && t < a.V) {
      g = a.scale * a.dlogprobs[row];
      id = (int)t - first;
    }
  }
  float gh = ENT ? a.scale * a.dentropy[row] : 0.0f;
  float base = ENT ? fmaf(gh, a.entropy[row], g) : g;
  const bool none = lse == neg_inf();
  if (none) g = gh = base = 0.0f;
  const float offset = none ? 0.0f : lse;  // p is 0 there: every logit is -inf, or its gradient counts as 0
#pragma unroll
  for (int j = 0; j < kBackVecs; ++j) {
    const int i0 = (j * kBackThreads + threadIdx.x) * VEC;
    Vals r;
    float out[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = fmaf((float)v[j].v[e], a.scale, -offset);
      const float p = none ? 0.0f : __builtin_amdgcn_exp2f(d * kLog2e);
      float q = base;
      if constexpr (ENT) q = fmaf(gh, fmaxf(d, -200.0f), base);  // p is 0 below
      out[e] = -p * q;
    }
    if ((unsigned)(id - i0) < (unsigned)VEC)
#pragma unroll
      for (int e = 0; e < VEC; ++e) out[e] += i0 + e == id ? g : 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = (T)out[e];
    if (full)
      store_streamed<T, VEC>(dx + i0, r);
    else if (i0 < n)
      store_guarded<T, VEC>(dx, i0, n, r);
  }
}

template <typename T>
hipError_t launch_backward(const LogprobsBackwardArgs& a, hipStream_t stream) {
  const int64_t per = kBackThreads * kBackVecs * kVec<T>;
  const int chunks = (int)((a.V + per - 1) / per);
  const dim3 grid = grid_of(a.M * chunks), block(kBackThreads);
  if (a.dentropy)
    hipLaunchKernelGGL((logprobs_backward_kernel<T, true>), grid, block, 0, stream, a, chunks);
  else
    hipLaunchKernelGGL((logprobs_backward_kernel<T, false>), grid, block, 0, stream, a, chunks);
  return launched();
}

}  // namespace

// As few parts of a row as fit a workgroup's registers: with one there is no join (1 x
// 50256 with 8 alternatives in 8.2 us, in 24 parts 10.1; 65 x 32001 with 20 in 8.2, in 3
// parts 12.4).
// Twice the registers where there is no second row for the CU.
int logprobs_chunks(int64_t M, int64_t V, int type, int cus) {
  const int vec = 16 / type_bytes(type);
  const int64_t most = 1024 * (M <= cus ? 16 : 8) * vec;
  const int64_t want = (V + most - 1) / most;
  // Rounding the length up to vectors may leave the last parts empty: fewer, then.
  const int64_t len = part_length(V, (int)want, vec);
  return (int)((V + len - 1) / len);
}

size_t logprobs_partial_bytes(int64_t M, int chunks, int k) {
  return chunks > 1 ? ((size_t)M * chunks * sizeof(Part) + 15) / 16 * 16 + (size_t)M * chunks * k * sizeof(Pair) : 0;
}

hipError_t launch_token_logprobs(const LogprobsArgs& a, hipStream_t stream) {
  if (a.type == kF32) return launch_logprobs<float>(a, stream);
  if (a.type == kBf16) return launch_logprobs<bf16>(a, stream);
  return launch_logprobs<f16>(a, stream);
}

hipError_t launch_token_logprobs_backward(const LogprobsBackwardArgs& a, hipStream_t stream) {
  if (a.type == kF32) return launch_backward<float>(a, stream);
  if (a.type == kBf16) return launch_backward<bf16>(a, stream);
  return launch_backward<f16>(a, stream);
}

}  // namespace lm
}  // namespace edsl

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
// finds the maximum, the sums and the alternatives. Second comes the exponential
// unit, one operation an element.
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

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kList = 512;   // candidates of one workgroup
constexpr int kMaxChunks = 64;  // parts of a row: one lane each in the join
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

// The results of a row, by one thread, from its whole sums.
template <typename T>
__device__ __forceinline__ void finish_row(const LogprobsArgs& a, int64_t row, Part p, bool none, float log_s) {
  if (a.lse) a.lse[row] = none ? neg_inf() : fmaf(kLn2, log_s, a.scale * p.m);
  if (a.entropy) a.entropy[row] = none ? 0.0f : kLn2 * (log_s - p.t / p.s);
  if (a.logprobs) {
    const int64_t id = id_at(a.tokens, a.ids64, row);
    float lp = 0.0f;
    if (id >= 0 && id < a.V) {
      const float x = (float)static_cast<const T*>(a.x)[row * a.ldx + id];
      lp = none ? neg_inf() : fmaf(-kLn2, log_s, (x - p.m) * a.scale);
    }
    a.logprobs[row] = lp;
  }
}

// One part's place in the workspace: Part, then k (value, index) pairs.
__device__ __forceinline__ char* part_at(char* base, int64_t row, int chunk, int chunks, int k) {
  return base + (row * chunks + chunk) * (int64_t)(16 + 8 * k);
}

template <typename T, int THREADS, int NV, bool TOP>
__global__ void __launch_bounds__(THREADS) logprobs_kernel(LogprobsArgs a, int64_t part_len) {
  constexpr int VEC = kVec<T>, WAVES = THREADS / 64;
  __shared__ float maxima[TOP ? WAVES : 1][64];
  __shared__ Part parts[WAVES];
  __shared__ float list_v[TOP ? kList : 1];
  __shared__ int list_i[TOP ? kList : 1];
  __shared__ int count;
  __shared__ float best_v[WAVES];
  __shared__ int best_i[WAVES];
  const int64_t row = (int64_t)blockIdx.x / a.chunks;
  const int chunk = (int)((int64_t)blockIdx.x - row * a.chunks);
  const int64_t first = chunk * part_len;
  const int n = (int)(first + part_len < a.V ? part_len : a.V - first);  // > 0
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx + first;
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const float c = a.scale * kLog2e;
  if (tid == 0) count = 0;

  Packed<T, VEC> v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = load_guarded<T, VEC>(x, (j * THREADS + tid) * VEC, n, (T)neg_inf());
  float top = neg_inf();
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) top = fmaxf(top, (float)v[j].v[e]);
  if constexpr (TOP) maxima[wave][lane] = top;
  const bool any = top > neg_inf();
  Part p{any ? top : 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (j * THREADS * VEC >= n) break;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float u = ((float)v[j].v[e] - p.m) * c;
      const float w = __builtin_amdgcn_exp2f(u);
      p.s += w;
      p.t = fmaf(w, fmaxf(u, -200.0f), p.t);  // 0 for -inf: e is 0 there
    }
  }
  p = wave_join(p, any, c);
  if (lane == 0) parts[wave] = p;
  __syncthreads();
  // Every wave adds the waves' parts up for itself.
  Part all = lane < WAVES ? parts[lane] : Part{0.0f, 0.0f, 0.0f};
  all = wave_join(all, all.s > 0.0f || all.s != all.s, c);
  const bool bad = all.s != all.s;      // a NaN, or +inf less itself
  const bool none = !bad && all.s == 0.0f;
  const float log_s = log2f(all.s);

  char* const out = a.chunks > 1 ? part_at(a.partials, row, chunk, a.chunks, a.k) : nullptr;
  if (tid == 0) {
    if (out)
      *reinterpret_cast<Part*>(out) = all;
    else
      finish_row<T>(a, row, all, none, log_s);
  }
  if constexpr (TOP) {
    const int k = a.k;
    // The r-th alternative: to the row's results, or to the join.
    const auto put = [&](int r, float value, int index) {
      if (out) {
        float* const q = reinterpret_cast<float*>(out + 16) + 2 * r;
        q[0] = value;
        reinterpret_cast<int*>(q)[1] = index == kNoIndex ? index : (int)first + index;
      } else {
        a.top[row * k + r] = none ? neg_inf() : fmaf(-kLn2, log_s, (value - all.m) * a.scale);
        put_id(a.top_ids, a.ids64, row * k + r, index);
      }
    };
    if (bad) {
      if (tid < k) put(tid, __builtin_nanf(""), out ? kNoIndex : -1);
      return;
    }
    float classes = maxima[0][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) classes = fmaxf(classes, maxima[w][lane]);
    const float least = kth_of_lanes(classes, k);
    if (any && top >= least) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float value = (float)v[j].v[e];
          if (value >= least && value > neg_inf()) {
            const int at = atomicAdd(&count, 1);
            if (at < kList) {
              list_v[at] = value;
              list_i[at] = (j * THREADS + tid) * VEC + e;
            }
          }
        }
    }
    __syncthreads();
    const int found = count;
    if (found <= kList) {
      for (int i = tid; i < found; i += THREADS) {
        const float value = list_v[i];
        const int index = list_i[i];
        int rank = 0;
        for (int j = 0; j < found; ++j) rank += better(list_v[j], list_i[j], value, index);
        if (rank < k) put(rank, value, index);
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
    // One alternative after the other: the best that follows the last one.
    float last_v = __builtin_inff();
    int last_i = -1;
    for (int r = 0; r < k; ++r) {
      float bv = neg_inf();
      int bi = kNoIndex;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float value = (float)v[j].v[e];
          const int index = (j * THREADS + tid) * VEC + e;
          if (index < n && better(last_v, last_i, value, index) && better(value, index, bv, bi)) {
            bv = value;
            bi = index;
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

// Joins the parts of a row, one a lane. Each part's alternatives are in order: the
// row's are taken from the heads of the lists.
template <typename T>
__global__ void __launch_bounds__(64) logprobs_join_kernel(LogprobsArgs a) {
  __shared__ float heads_v[kMaxChunks * kMaxTop];
  __shared__ int heads_i[kMaxChunks * kMaxTop];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x, k = a.k;
  const char* const mine = part_at(a.partials, row, lane < a.chunks ? lane : 0, a.chunks, k);
  Part p = lane < a.chunks ? *reinterpret_cast<const Part*>(mine) : Part{0.0f, 0.0f, 0.0f};
  if (lane < a.chunks)
    for (int r = 0; r < k; ++r) {
      heads_v[lane * kMaxTop + r] = reinterpret_cast<const float*>(mine + 16)[2 * r];
      heads_i[lane * kMaxTop + r] = reinterpret_cast<const int*>(mine + 16)[2 * r + 1];
    }
  const float c = a.scale * kLog2e;
  p = wave_join(p, p.s > 0.0f || p.s != p.s, c);
  const bool bad = p.s != p.s, none = !bad && p.s == 0.0f;
  const float log_s = log2f(p.s);
  if (lane == 0) finish_row<T>(a, row, p, none, log_s);
  int at = 0;  // a lane reads its own entries only
  for (int r = 0; r < k; ++r) {
    const bool has = lane < a.chunks && at < k && !bad;
    const float v = has ? heads_v[lane * kMaxTop + at] : neg_inf();
    const int i = has ? heads_i[lane * kMaxTop + at] : kNoIndex;
    float bv = v;
    int bi = i;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const float ov = __shfl_xor(bv, d);
      const int oi = __shfl_xor(bi, d);
      if (better(ov, oi, bv, bi)) {
        bv = ov;
        bi = oi;
      }
    }
    if (has && i == bi && i != kNoIndex) ++at;
    if (lane == 0) {
      a.top[row * k + r] = bad ? __builtin_nanf("") : none ? neg_inf() : fmaf(-kLn2, log_s, (bv - p.m) * a.scale);
      put_id(a.top_ids, a.ids64, row * k + r, bad ? -1 : bi);
    }
  }
}

template <typename T, int THREADS, int NV>
hipError_t launch_parts(const LogprobsArgs& a, int64_t part_len, hipStream_t stream) {
  const dim3 grid((unsigned)(a.M * a.chunks));
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
  else if (vecs <= 512)
    e = launch_parts<T, 256, 2>(a, len, stream);
  else if (vecs <= 1024)
    e = launch_parts<T, 256, 4>(a, len, stream);
  else if (vecs <= 2048)
    e = launch_parts<T, 1024, 2>(a, len, stream);
  else if (vecs <= 4096)
    e = launch_parts<T, 1024, 4>(a, len, stream);
  else
    e = launch_parts<T, 1024, 8>(a, len, stream);
  if (e != hipSuccess || a.chunks == 1) return e;
  hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3((unsigned)a.M), dim3(64), 0, stream, a);
  return launched();
}

// ---------------------------------------------------------------- backward
// p_j = exp(d_j), d_j = scale x_j - lse (one rounding, exact where p is near 1);
// dx_j = scale (dlp ([j == token] - p_j) - dent p_j (d_j + entropy)).
constexpr int kBackThreads = 256, kBackVecs = 4;

template <typename T, bool ENT>
__global__ void __launch_bounds__(kBackThreads) logprobs_backward_kernel(LogprobsBackwardArgs a, int chunks) {
  constexpr int VEC = kVec<T>;
  const int64_t row = (int64_t)blockIdx.x / chunks;
  const int64_t first = ((int64_t)blockIdx.x - row * chunks) * (kBackThreads * kBackVecs * VEC);
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
  T* const dx = static_cast<T*>(a.dx) + row * a.lddx;
  const float lse = a.lse[row];
  const bool none = lse == neg_inf();
  int64_t id = -1;
  float g = 0.0f;
  if (a.dlogprobs) {
    id = id_at(a.tokens, a.ids64, row);
    if (id >= 0 && id < a.V) g = a.scale * a.dlogprobs[row];
    else id = -1;
  }
  const float h = ENT ? a.entropy[row] : 0.0f, gh = ENT ? a.scale * a.dentropy[row] : 0.0f;
  Packed<T, VEC> v[kBackVecs];
#pragma unroll
  for (int j = 0; j < kBackVecs; ++j)
    v[j] = load_guarded<T, VEC>(x, first + (j * kBackThreads + threadIdx.x) * VEC, a.V, (T)neg_inf());
#pragma unroll
  for (int j = 0; j < kBackVecs; ++j) {
    const int64_t i0 = first + (j * kBackThreads + threadIdx.x) * VEC;
    if (i0 >= a.V) break;
    Packed<T, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = fmaf((float)v[j].v[e], a.scale, -lse);
      const float p = __builtin_amdgcn_exp2f(d * kLog2e);
      float q = g;
      if constexpr (ENT) q = fmaf(gh, fmaxf(d, -200.0f) + h, g);  // p is 0 below
      float out = -p * q;
      if (i0 + e == id) out += g;
      r.v[e] = (T)(none ? 0.0f : out);
    }
    store_guarded<T, VEC>(dx, i0, a.V, r);
  }
}

template <typename T>
hipError_t launch_backward(const LogprobsBackwardArgs& a, hipStream_t stream) {
  const int64_t per = kBackThreads * kBackVecs * kVec<T>;
  const int chunks = (int)((a.V + per - 1) / per);
  const dim3 grid((unsigned)(a.M * chunks)), block(kBackThreads);
  if (a.dentropy)
    hipLaunchKernelGGL((logprobs_backward_kernel<T, true>), grid, block, 0, stream, a, chunks);
  else
    hipLaunchKernelGGL((logprobs_backward_kernel<T, false>), grid, block, 0, stream, a, chunks);
  return launched();
}

}  // namespace

// One workgroup a row where there are rows enough for the chip or the row is
// short; else as many parts as there are CUs for, of 2048 elements at least.
int logprobs_chunks(int64_t M, int64_t V, int type, int cus) {
  const int64_t most = 1024 * 8 * (16 / type_bytes(type));  // what a workgroup holds
  const int64_t least = (V + most - 1) / most;
  int64_t want = M > 0 ? cus / M : 1;
  if (want > V / 2048) want = V / 2048;
  if (want > kMaxChunks) want = kMaxChunks;
  if (want < least) want = least;
  const int vec = 16 / type_bytes(type);
  // Rounding the length up to vectors may leave the last parts empty: fewer, then.
  const int64_t len = part_length(V, (int)want, vec);
  return (int)((V + len - 1) / len);
}

size_t logprobs_partial_bytes(int64_t M, int chunks, int k) {
  return chunks > 1 ? (size_t)M * chunks * (16 + 8 * (size_t)k) : 0;
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

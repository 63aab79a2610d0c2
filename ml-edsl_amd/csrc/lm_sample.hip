// Tokens drawn from logits with given uniform numbers: temperature, top-k, top-p and
// min-p for each row.
//
// With m = max x, T the temperature and w_i = e^((x_i - m) / T), kept are
//   the k largest logits (equal ones by their index);
//   of these, in falling order, those with less than p of their mass before them;
//   and of these the ones with w_i >= min_p;
// drawn is the first index i, in the vocabulary's order, at which the running mass
// of the kept ones exceeds u times the whole of it.
//
// A token next to a border changes with the last bits of a sum, so masses are
// integers: w_i 2^s to nearest, s = 46 for up to 2^16 logits and one less for each
// doubling, from a 64-bit exponential. Their sums are exact in 64 bits, whatever the order,
// so that atomics give the same bits each time. A weight below 2^-47 of the largest is 0.
//
// One workgroup takes a row, a wave a run of it. Top-k and top-p: the logits fall into
// 2048 bins by their distance from m, with counts and masses; the bin that holds a border is
// found by a prefix sum, and the border in it by ranking the bin's few logits (by their
// keys' digits, from the row again, where they are many). Every pass but the first reads the row from
// the caches.
#include <algorithm>

#include "lm_common.hpp"
#include "lm_kernels.hpp"

namespace edsl {
namespace lm {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr float kRange = 48.0f;  // octaves below the maximum that the bins cover: past 47 a weight is 0
constexpr int kList = 1024;      // logits of a border's bin that are ranked
// log 2 in two parts: its first 36 bits and the rest.
constexpr double kLn2High = 0x1.62e42fefap-1, kLn2Low = 0x1.cf79abc9e3b3ap-40;

// e^t for t <= 0, times 2^s, to the nearest integer: Taylor's sum to the twelfth power on half an octave about 0,
// 2e-16 off. Under 2^-47 of 2^s it is 0.
__device__ __forceinline__ u64 weight_of(double t, int s) {
  if (!(t > -35.0)) return 0;  // 50 octaves; -inf
  const double n = __builtin_rint(t * 1.4426950408889634074);
  double r = fma(n, -kLn2High, t);
  r = fma(n, -kLn2Low, r);
  double p = 1.0 / 479001600.0;
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  // Added to 2^52, the sum's low bits are the rounded integer.
  const double v = __builtin_ldexp(p, (int)n + s) + 4503599627370496.0;
  return __builtin_bit_cast(u64, v) - 0x4330000000000000ull;
}

// Logits in their order as unsigned integers; -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __builtin_bit_cast(float, (key >> 31) ? key ^ 0x80000000u : ~key);
}

__device__ __forceinline__ u64 wave_sum(u64 v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}
// The sum over lanes up to this one.
__device__ __forceinline__ u64 wave_prefix(u64 v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 u = __shfl_up(v, d);
    if ((int)(threadIdx.x % 64) >= d) v += u;
  }
  return v;
}

// A border in falling order: logits above `key` are kept, and the first `ties` of the `equal` ones at it.
struct Border {
  uint32_t key;
  uint32_t ties, equal;
};

struct Shared {
  uint32_t count[kBins];
  u64 mass[kBins];
  uint32_t list_key[kList];
  u64 list_q[kList];
  u64 wave[kWaves];
  float wave_max[kWaves];
  u64 before;  // found by find()
  int found;
  uint32_t listed;
  Border border;
  int first;
};

template <typename T>
struct Row {
  static constexpr int VEC = kVec<T>, kLine = 64 * VEC, kAhead = 4;
  const T* x;
  int V;
  Shared& sh;
  float m, to_bins;
  double inv_t;
  int s;

  __device__ __forceinline__ int begin() const { return (int)(threadIdx.x / 64) * run(); }
  // Elements of a wave's run.
  __device__ __forceinline__ int run() const { return (V + kWaves * kLine - 1) / (kWaves * kLine) * kLine; }

  // f(x, index) of every element of the wave's run, its lines in order.
  template <typename F>
  __device__ __forceinline__ void scan(F&& f) const {
    const int lane = threadIdx.x % 64, from = begin(), to = min(V, from + run());
    int i = from;
    for (; i + kAhead * kLine <= to; i += kAhead * kLine) {
      Packed<T, VEC> r[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) r[a] = load_packed<T, VEC>(x + i + a * kLine + lane * VEC);
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
#pragma unroll
        for (int e = 0; e < VEC; ++e) f((float)r[a].v[e], i + a * kLine + lane * VEC + e);
    }
    for (; i < to; i += kLine) {
      const int at = i + lane * VEC;
      if (at >= to) break;
      const Packed<T, VEC> r = load_guarded<T, VEC>(x, at, to, T(-__builtin_inff()));
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (at + e < to) f((float)r.v[e], at + e);
    }
  }

  __device__ __forceinline__ int bin_of(float v) const { return (int)fminf((m - v) * to_bins, (float)(kBins - 1)); }
  __device__ __forceinline__ double exponent(float v) const { return ((double)v - (double)m) * inv_t; }
  __device__ __forceinline__ u64 weight(float v) const { return weight_of(exponent(v), s); }

  // The first of n (up to two a thread) values whose running sum reaches `target`: sh.found, and sh.before the sum before it;
  // -1 where none does.
  template <typename Value>
  __device__ __forceinline__ void find(int n, u64 target, Value&& value) const {
    const int tid = threadIdx.x;
    const u64 a = 2 * tid < n ? value(2 * tid) : 0, b = 2 * tid + 1 < n ? value(2 * tid + 1) : 0;
    const u64 upto = wave_prefix(a + b);
    __syncthreads();
    if (tid % 64 == 63) sh.wave[tid / 64] = upto;
    if (tid == 0) sh.found = -1;
    __syncthreads();
    u64 before = upto - (a + b);
    for (int w = 0; w < tid / 64; ++w) before += sh.wave[w];
    if (before < target && target <= before + a + b) {
      const bool second = target > before + a;
      sh.found = 2 * tid + second;
      sh.before = before + (second ? a : 0);
    }
    __syncthreads();
  }

  // The border in bin `b`, `n` elements, at which the running sum of q, in falling
  // order, reaches `target` >= 1; 1 a logit, or its weight where MASS.
  template <bool MASS>
  __device__ __forceinline__ Border border_in(int b, uint32_t n, u64 target) const {
    const int tid = threadIdx.x;
    if (n <= kList) {
      if (tid == 0) sh.listed = 0;
      __syncthreads();
      scan([&](float v, int) {
        if (bin_of(v) == b) {
          const uint32_t at = atomicAdd(&sh.listed, 1u);
          if (at < (uint32_t)kList) sh.list_key[at] = key_of(v);
        }
      });
      __syncthreads();
      const uint32_t mine = tid < (int)n ? sh.list_key[tid] : 0;
      u64 q = 0;
      if (tid < (int)n) sh.list_q[tid] = q = MASS ? weight(value_of(mine)) : 1;
      __syncthreads();
      if (tid < (int)n) {
        u64 above = 0;
        uint32_t equal = 0;
        for (uint32_t i = 0; i < n; ++i) {
          const uint32_t other = sh.list_key[i];
          if (other > mine) above += sh.list_q[i];
          equal += other == mine;
        }
        // The same for all of equal key.
        if (above < target && target <= above + equal * q)
          sh.border = {mine, (uint32_t)((target - above + q - 1) / q), equal};
      }
      __syncthreads();
      return sh.border;
    }
    // Digit by digit of the keys, from the row.
    uint32_t prefix = 0;
    u64 q = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) sh.list_q[tid] = 0;
      __syncthreads();
      scan([&](float v, int) {
        const uint32_t key = key_of(v);
        if (bin_of(v) == b && (shift == 24 || key >> (shift + 8) == prefix))
          atomicAdd(&sh.list_q[255 - ((key >> shift) & 255)], MASS ? weight(v) : 1);
      });
      __syncthreads();
      find(256, target, [&](int i) { return sh.list_q[i]; });
      const int digit = sh.found;
      target -= sh.before;
      q = sh.list_q[digit];
      prefix = prefix << 8 | (uint32_t)(255 - digit);
    }
    const u64 one = MASS ? weight(value_of(prefix)) : 1;
    return {prefix, (uint32_t)((target + one - 1) / one), (uint32_t)(q / one)};
  }

  // The index of the `nth` (from 1) element, in their order, that `is` holds for, by running sums of q(x, index): the first at which
  // they reach nth. sh.first; every thread returns it.
  template <typename Q>
  __device__ __forceinline__ int locate(u64 mine, u64 nth, Q&& q) const {
    // `mine`: the sum of the wave's run, in all lanes.
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid % 64 == 0) sh.wave[tid / 64] = mine;
    __syncthreads();
    u64 before = 0;
    int w = 0;
    while (w < kWaves - 1 && before + sh.wave[w] < nth) before += sh.wave[w++];
    const int from = w * run(), to = min(V, from + run());
    const int per = (to - from + kThreads - 1) / kThreads;
    const int first = min(from + tid * per, to), last = min(first + per, to);
    u64 sum = 0;
    for (int i = first; i < last; ++i) sum += q((float)x[i], i);
    const u64 upto = wave_prefix(sum);
    __syncthreads();
    if (tid % 64 == 63) sh.wave[tid / 64] = upto;
    if (tid == 0) sh.first = -1;
    __syncthreads();
    before += upto - sum;
    for (int v = 0; v < tid / 64; ++v) before += sh.wave[v];
    if (before < nth && nth <= before + sum) {
      int i = first;
      for (; i < last - 1; ++i) {
        before += q((float)x[i], i);
        if (before >= nth) break;
      }
      sh.first = i;
    }
    __syncthreads();
    return sh.first;
  }
};

template <typename V>
__device__ __forceinline__ V setting(const V* each, V all, int64_t row) {
  return each ? each[row] : all;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  __shared__ Shared sh;
  const int64_t row = block_of();
  if (row >= a.M) return;
  const int tid = threadIdx.x, V = (int)a.V;
  Row<T> r{static_cast<const T*>(a.x) + row * a.ldx, V, sh, 0.0f, 0.0f, 0.0, a.shift};

  const float temperature = setting(a.temperature, a.temperature_all, row);
  const float top_p = setting(a.top_p, a.top_p_all, row), min_p = setting(a.min_p, a.min_p_all, row);
  const int top_k = setting(a.top_k, a.top_k_all, row);
  const float uniform = a.uniforms[row];
  const auto done = [&](int64_t token, float logprob) {
    if (tid == 0) {
      if (a.ids64)
        static_cast<int64_t*>(a.tokens)[row] = token;
      else
        static_cast<int32_t*>(a.tokens)[row] = (int32_t)token;
      if (a.logprobs) a.logprobs[row] = logprob;
    }
  };

  float most = -__builtin_inff();
  r.scan([&](float v, int) { most = MaxNan::of(most, v); });
  most = lanes_all<MaxNan, 64>(most);
  if (tid % 64 == 0) sh.wave_max[tid / 64] = most;
  __syncthreads();
  most = sh.wave_max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) most = MaxNan::of(most, sh.wave_max[w]);
  // All uniform over the workgroup from here.
  const bool fine = temperature >= 0.0f && temperature < __builtin_inff() && top_p == top_p && min_p == min_p &&
                    uniform == uniform;
  if (!(most < __builtin_inff()) || !fine) return done(-1, __builtin_nanf(""));
  if (most == -__builtin_inff()) return done(-1, most);
  r.m = most;
  if (temperature == 0.0f) {
    int first = V;
    r.scan([&](float v, int i) { first = v == most && i < first ? i : first; });
#pragma unroll
    for (int d = 1; d < 64; d *= 2) first = min(first, __shfl_xor(first, d));
    if (tid % 64 == 0) sh.wave[tid / 64] = (u64)first;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) first = min(first, (int)sh.wave[w]);
    return done(first, 0.0f);
  }
  r.inv_t = 1.0 / (double)temperature;
  // Finite, so that the maximum is in the first bin.
  r.to_bins = fminf((float)(kBins / kRange * 1.4426950408889634 * r.inv_t), 1e30f);

  const bool use_k = top_k > 0 && top_k < V, use_p = top_p < 1.0f;
  Border border{0, 0, 0};
  bool bounded = false;
  if (use_k || use_p) {
    for (int i = tid; i < kBins; i += kThreads) sh.count[i] = 0, sh.mass[i] = 0;
    __syncthreads();
    // The last bin's weights are 0: whether they are kept changes nothing.
    r.scan([&](float v, int) {
      const int b = r.bin_of(v);
      if (b < kBins - 1) {
        atomicAdd(&sh.count[b], 1u);
        if (use_p) atomicAdd(&sh.mass[b], r.weight(v));
      }
    });
    __syncthreads();
    u64 total = 0;
    int last_bin = kBins;
    if (use_k) {
      r.find(kBins, (u64)top_k, [&](int i) { return (u64)sh.count[i]; });
      last_bin = sh.found;
      if (last_bin >= 0) {
        border = r.template border_in<false>(last_bin, sh.count[last_bin], (u64)top_k - sh.before);
        bounded = true;
      } else {
        last_bin = kBins;
      }
    }
    if (use_p) {
      // The mass of the k largest: whole bins, and of the border's bin what is above it and its ties.
      u64 mine = 0;
      for (int i = tid; i < min(last_bin, kBins); i += kThreads) mine += sh.mass[i];
      if (bounded) {
        r.scan([&](float v, int) {
          if (r.bin_of(v) == last_bin && key_of(v) > border.key) mine += r.weight(v);
        });
        if (tid == 0) mine += border.ties * r.weight(value_of(border.key));
      }
      mine = wave_sum(mine);
      __syncthreads();
      if (tid % 64 == 0) sh.wave[tid / 64] = mine;
      __syncthreads();
      for (int w = 0; w < kWaves; ++w) total += sh.wave[w];
      const double part = __builtin_ceil((double)fmaxf(top_p, 0.0f) * (double)total);
      const u64 target = max((u64)1, min(total, (u64)part));
      r.find(kBins, target, [&](int i) { return sh.mass[i]; });
      const int b = sh.found;
      border = r.template border_in<true>(b, sh.count[b], target - sh.before);
      bounded = true;
    }
  }

  // Ties: the index of the last one that is kept.
  int last_tie = V;
  if (bounded && border.ties < border.equal) {
    const auto is_tie = [&](float v, int) { return (u64)(key_of(v) == border.key); };
    u64 ties = 0;
    r.scan([&](float v, int i) { ties += is_tie(v, i); });
    last_tie = r.locate(wave_sum(ties), border.ties, is_tie);
  }
  // Logits under `low` have no weight or are under min_p of the largest for sure: most
  // need no exponential.
  const double least = min_p > 0.0f ? log(fmin((double)min_p, 1.0)) : -__builtin_inf();
  const float low = (float)(fmax(least, -33.5) * (double)temperature * 1.000001 + (double)most) -
                    1e-6f * fabsf(most) - 1e-37f;
  const auto mass_of = [&](float v, int i) -> u64 {
    if (!(v >= low)) return 0;
    if (bounded) {
      const uint32_t key = key_of(v);
      if (key < border.key || (key == border.key && i > last_tie)) return 0;
    }
    const double t = r.exponent(v);
    return t >= least ? weight_of(t, r.s) : 0;
  };
  u64 mine = 0;
  r.scan([&](float v, int i) { mine += mass_of(v, i); });
  mine = wave_sum(mine);
  __syncthreads();
  if (tid % 64 == 0) sh.wave[tid / 64] = mine;
  __syncthreads();
  u64 total = 0;
  for (int w = 0; w < kWaves; ++w) total += sh.wave[w];
  const double u = fmin(fmax((double)uniform, 0.0), 1.0);
  const u64 target = min((u64)(u * (double)total), total - 1);
  const int token = r.locate(mine, target + 1, mass_of);
  if (tid == 0) {
    const u64 w = r.weight((float)r.x[token]);
    done(token, (float)-log1p((double)(total - w) / (double)w));
  }
}

}  // namespace

hipError_t launch_sample_tokens(const SampleArgs& a, hipStream_t stream) {
  const auto kernel = a.type == kF32 ? sample_kernel<float> : a.type == kBf16 ? sample_kernel<bf16> : sample_kernel<f16>;
  hipLaunchKernelGGL(kernel, grid_of(a.M), dim3(kThreads), 0, stream, a);
  return launched();
}

}  // namespace lm
}  // namespace edsl

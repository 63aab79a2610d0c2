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
// so that atomics give the same bits each time. A weight below half a unit, 2^-(s+1) of the largest, is 0.
//
// One workgroup takes a row, a wave a run of it. Top-k and top-p: the logits fall into
// 2048 bins by their distance from m, with counts and masses; the bin that holds a border is
// found by a prefix sum, and the border in it by ranking the bin's few logits (by their
// keys' digits where they are many). As soon as a bound of the kept logits is known, those above
// it are candidates in LDS and the row is read no more: for top-k that is the k-th largest of the
// threads' maxima, for min-p alone its weight, for top-p its border's bin. More than
// 12288 candidates are read from the row, in the caches, each time: 0.9 of the mass of 50256 normal logits of
// deviation 2.5, some 6000 of them, in 52.6 us for 256 rows, with room for 4096 in 63.5.
//
// Bound by one workgroup's way through its row: 50256 logits in 7 us for the largest (greedy), 17 with top-k 50, 21 with
// all settings, 23 drawn from the whole row (13 of them its exponentials, 64-bit vector time), 42 to 53 with top-p 0.9 (its masses
// and again those of the kept, a prefix sum, ranks); 256 rows take what one takes.
#include <algorithm>

#include "lm_common.hpp"
#include "lm_kernels.hpp"

namespace edsl {
namespace lm {
namespace {

typedef unsigned long long u64;

// Lambdas that are not inlined take what they capture through memory.
#define INLINE __attribute__((always_inline))

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kMostRow = 1 << 21;
constexpr float kRange = 48.0f;  // octaves below the maximum that the bins cover: past s + 1, 47 at most, a weight is 0
constexpr int kList = 1024;      // logits of a border's bin that are ranked
// Candidates that are kept apart from the row; the registers leave room for one workgroup a CU in any case.
constexpr int kKept = 12288;
constexpr int kFew = 256;        // of those, so many are ranked against each other

// v or 0, without a branch: the compiler would put all that v takes into it, one element after the other.
__device__ __forceinline__ double only(bool keep, double v) {
  uint32_t mask = keep ? ~0u : 0u;
  asm("" : "+v"(mask));
  const u64 bits = __builtin_bit_cast(u64, v);
  return __builtin_bit_cast(double, (u64)((uint32_t)(bits >> 32) & mask) << 32 | ((uint32_t)bits & mask));
}

// 2^y for y <= 0, plus `grid` = 2^(52-s): a double whose low 52 bits are 2^(y+s) to the nearest integer. 2^f is Taylor's
// sum to the eleventh power on half an octave about 0, 7e-15 off (the coefficients are (log 2)^k / k!), powers of two
// come by the exponent's bits, and adding 1.5 2^52 leaves the nearest integer in the low ones: conversions and v_ldexp_f64 run
// at a quarter of an fma's rate. Masked logits, y = -inf, come out as 2^-60: 0.
__device__ __forceinline__ double weight_on(double y, double grid) {
  y = fmax(y, -60.0);
  const double shifted = y + 0x1.8p52;
  const double f = y - (shifted - 0x1.8p52);
  double p = 0x1.e8cac7351bb25p-32;
  p = fma(p, f, 0x1.e4cf5158b8ecap-28);
  p = fma(p, f, 0x1.b5253d395e7c4p-24);
  p = fma(p, f, 0x1.62c0223a5c824p-20);
  p = fma(p, f, 0x1.ffcbfc588b0c7p-17);
  p = fma(p, f, 0x1.430912f86c787p-13);
  p = fma(p, f, 0x1.5d87fe78a6731p-10);
  p = fma(p, f, 0x1.3b2ab6fba4e77p-7);
  p = fma(p, f, 0x1.c6b08d704a0c0p-5);
  p = fma(p, f, 0x1.ebfbdff82c58fp-3);
  p = fma(p, f, 0x1.62e42fefa39efp-1);
  p = fma(p, f, 1.0);
  const u64 bits = __builtin_bit_cast(u64, p);
  const uint32_t high = (uint32_t)(bits >> 32) + ((uint32_t)__builtin_bit_cast(u64, shifted) << 20);
  return __builtin_bit_cast(double, (u64)high << 32 | (uint32_t)bits) + grid;
}
__device__ __forceinline__ u64 units_of(double w) { return __builtin_bit_cast(u64, w) & 0xfffffffffffffull; }

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
  float kept_x[kKept];  // candidates, in no order
  int kept_i[kKept];
  uint32_t list_key[kList + 8];
  u64 list_q[kList + 8];
  u64 wave[kWaves];
  float wave_max[kWaves];
  u64 before;  // found by find()
  int found;
  uint32_t listed;
  Border border;
  int first;
};

// One block of LDS, whoever asks: by its name, so that accesses are to LDS for the compiler too.
__device__ __forceinline__ Shared& shared() {
  __shared__ Shared s;
  return s;
}

// Successive elements.
template <int N>
struct Some {
  static constexpr int kN = N;
  float v[N];
  int first;
};

template <typename T>
struct Row {
  static constexpr int kLine = 64 * kVec<T>;
  const T* x;
  int V;
  float m, half_m, to_bins;  // to_bins: of half a difference
  double octaves;  // log2(e) / T
  double grid, units;  // weight_on's; 2^s
  int kept;  // candidates, or -1: all of the row

  __device__ __forceinline__ int begin() const { return (int)(threadIdx.x / 64) * run(); }
  // Elements of a wave's run.
  __device__ __forceinline__ int run() const { return (V + kWaves * kLine - 1) / (kWaves * kLine) * kLine; }

  // f(some elements) of every candidate; of a row, a wave's run in the order of its lines. kAhead: lines on their
  // way. The code of f stands kAhead times for each element of a vector, and a workgroup that runs it a few times has
  // to fetch it: short vectors where it is long (kHeavy).
  template <int kAhead, bool kHeavy = false, typename F>
  __device__ __forceinline__ void scan(F&& f) const {
    if (kept >= 0) {
#pragma unroll 1
      for (int i = threadIdx.x; i < kept; i += kThreads) f(Some<1>{{shared().kept_x[i]}, shared().kept_i[i]});
      return;
    }
    lines<kHeavy ? 4 : kVec<T>, kAhead>(f);
  }
  // Lines of 64 vectors of VEC elements.
  template <int VEC, int kAhead, typename F>
  __device__ __forceinline__ void lines(F&& f) const {
    constexpr int kLine = 64 * VEC;
    const int lane = threadIdx.x % 64, from = begin(), to = min(V, from + run());
    const int whole = max(to - from, 0) / kLine;
#pragma unroll 1
    for (int i = 0; i < whole; i += kAhead) {
      Packed<T, VEC> r[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        r[a] = load_packed<T, VEC>(x + from + min(i + a, whole - 1) * kLine + lane * VEC);
#pragma unroll
      for (int a = 0; a < kAhead; ++a)
        if (i + a < whole) {
          Some<VEC> some;
          some.first = from + (i + a) * kLine + lane * VEC;
#pragma unroll
          for (int e = 0; e < VEC; ++e) some.v[e] = (float)r[a].v[e];
          f(some);
        }
    }
#pragma unroll 1
    for (int i = from + whole * kLine + lane; i < to; i += 64) f(Some<1>{{(float)x[i]}, i});
  }

  // From here on only the elements that `is` holds for, where they are few enough.
  template <typename Is>
  __device__ __forceinline__ void keep(Is&& is) {
    __syncthreads();
    if (threadIdx.x == 0) shared().listed = 0;
    __syncthreads();
    scan<6>([&](const auto& some) INLINE {
#pragma unroll
      for (int e = 0; e < some.kN; ++e)
        if (is(some.v[e])) {
          const uint32_t at = atomicAdd(&shared().listed, 1u);
          if (at < (uint32_t)kKept) shared().kept_x[at] = some.v[e], shared().kept_i[at] = some.first + e;
        }
    });
    __syncthreads();
    if (shared().listed <= (uint32_t)kKept) kept = (int)shared().listed;
    __syncthreads();
  }

  // Of half the difference: that of two finite logits may be past the largest f32, and only -inf is infinitely far.
  __device__ __forceinline__ int bin_of(float v) const {
    return (int)fminf(fmaf(-0.5f, v, half_m) * to_bins, (float)(kBins - 1));
  }
  // log2 of an element's weight.
  __device__ __forceinline__ double exponent(float v) const { return ((double)v - (double)m) * octaves; }
  __device__ __forceinline__ u64 weight(float v) const { return units_of(weight_on(exponent(v), grid)); }
  // The same as a multiple of the unit. A thread's sum of these is exact: V 2^-10 2^s is under 2^53.
  __device__ __forceinline__ double weight_real(float v) const { return weight_on(exponent(v), grid) - grid; }

  // The sum of shared().wave of the waves before this one.
  static __device__ __forceinline__ u64 waves_before() {
    u64 sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += w < (int)(threadIdx.x / 64) ? shared().wave[w] : 0;
    return sum;
  }

  // The first of n (up to two a thread) values whose running sum reaches `target`: shared().found, and shared().before the sum before it;
  // -1 where none does.
  template <typename Value>
  __device__ __forceinline__ void find(int n, u64 target, Value&& value) const {
    const int tid = threadIdx.x;
    const u64 a = 2 * tid < n ? value(2 * tid) : 0, b = 2 * tid + 1 < n ? value(2 * tid + 1) : 0;
    const u64 upto = wave_prefix(a + b);
    __syncthreads();
    if (tid % 64 == 63) shared().wave[tid / 64] = upto;
    if (tid == 0) shared().found = -1;
    __syncthreads();
    u64 before = upto - (a + b) + waves_before();
    if (before < target && target <= before + a + b) {
      const bool second = target > before + a;
      shared().found = 2 * tid + second;
      shared().before = before + (second ? a : 0);
    }
    __syncthreads();
  }

  // The border in bin `b` at which the running sum of q, in falling order, reaches
  // `target` >= 1; q is 1 a logit, or its weight where MASS.
  template <bool MASS>
  __device__ __forceinline__ Border border_in(int b, u64 target) const {
    const int tid = threadIdx.x;
    if (tid == 0) shared().listed = 0;
    __syncthreads();
    scan<6>([&](const auto& some) INLINE {
#pragma unroll
      for (int e = 0; e < some.kN; ++e)
        if (bin_of(some.v[e]) == b) {
          const uint32_t at = atomicAdd(&shared().listed, 1u);
          if (at < (uint32_t)kList) shared().list_key[at] = key_of(some.v[e]);
        }
    });
    __syncthreads();
    const int n = (int)shared().listed;
    if (n <= kList) {
      const uint32_t mine = tid < n ? shared().list_key[tid] : 0;
      u64 q = 0;
      if (tid < n) shared().list_q[tid] = q = MASS ? weight(value_of(mine)) : 1;
      if (tid < 8) shared().list_key[n + tid] = 0;  // no logit's key
      __syncthreads();
      if (tid < n) {
        u64 above = 0;
        uint32_t equal = 0;
#pragma unroll 1
        for (int i = 0; i < n; i += 8)
#pragma unroll
          for (int e = 0; e < 8; ++e) {  // read together: a read takes as long as all of them
            const uint32_t other = shared().list_key[i + e];
            const u64 theirs = shared().list_q[i + e];
            above += other > mine ? theirs : 0;
            equal += other == mine;
          }
        // The same for all of equal key.
        if (above < target && target <= above + equal * q)
          shared().border = {mine, (uint32_t)((target - above + q - 1) / q), equal};
      }
      __syncthreads();
      return shared().border;
    }
    // Digit by digit of the keys, from the row.
    uint32_t prefix = 0;
    u64 q = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      if (tid < 256) shared().list_q[tid] = 0;
      __syncthreads();
      scan<2, true>([&](const auto& some) INLINE {
#pragma unroll
        for (int e = 0; e < some.kN; ++e) {
          const uint32_t key = key_of(some.v[e]);
          if (bin_of(some.v[e]) == b && (shift == 24 || key >> (shift + 8) == prefix))
            atomicAdd(&shared().list_q[255 - ((key >> shift) & 255)], MASS ? weight(some.v[e]) : 1);
        }
      });
      __syncthreads();
      find(256, target, [&](int i) INLINE { return shared().list_q[i]; });
      const int digit = shared().found;
      target -= shared().before;
      q = shared().list_q[digit];
      prefix = prefix << 8 | (uint32_t)(255 - digit);
    }
    const u64 one = MASS ? weight(value_of(prefix)) : 1;
    return {prefix, (uint32_t)((target + one - 1) / one), (uint32_t)(q / one)};
  }

  // The first index at which the running sum of q(x, index), in the order of the indexes, reaches
  // nth; every thread returns it. `mine`: the sum of the wave's run, in all lanes.
  template <typename Q>
  __device__ __forceinline__ int locate(u64 mine, u64 nth, Q&& q) const {
    const int tid = threadIdx.x;
    if (kept >= 0) {
      u64 rest = nth;
      int shift = 31, b = 0;  // all
      if (kept > kFew) {
        // Candidates by bins of their index.
        shift = 0;
        while ((V - 1) >> shift >= kBins) ++shift;
        static_assert(kMostRow / kBins <= kList, "a bin's candidates fit the list");
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads) shared().mass[i] = 0;
        __syncthreads();
        for (int i = tid; i < kept; i += kThreads) {
          const u64 w = q(shared().kept_x[i], shared().kept_i[i]);
          if (w) atomicAdd(&shared().mass[shared().kept_i[i] >> shift], w);
        }
        __syncthreads();
        find(kBins, nth, [&](int i) INLINE { return shared().mass[i]; });
        b = shared().found, rest = nth - shared().before;
      }
      __syncthreads();
      if (tid == 0) shared().listed = 0;
      __syncthreads();
      for (int i = tid; i < kept; i += kThreads) {
        const u64 w = shared().kept_i[i] >> shift == b ? q(shared().kept_x[i], shared().kept_i[i]) : 0;
        if (w) {
          const uint32_t at = atomicAdd(&shared().listed, 1u);
          shared().list_key[at] = (uint32_t)shared().kept_i[i], shared().list_q[at] = w;
        }
      }
      __syncthreads();
      const int n = (int)shared().listed;
      if (tid < 8) shared().list_key[n + tid] = 0xffffffffu;
      __syncthreads();
      if (tid < n) {
        u64 upto = 0;
        const uint32_t own = shared().list_key[tid];
#pragma unroll 1
        for (int i = 0; i < n; i += 8)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const u64 theirs = shared().list_q[i + e];
            upto += shared().list_key[i + e] <= own ? theirs : 0;
          }
        if (upto - shared().list_q[tid] < rest && rest <= upto) shared().first = (int)own;
      }
      __syncthreads();
      return shared().first;
    }
    __syncthreads();
    if (tid % 64 == 0) shared().wave[tid / 64] = mine;
    __syncthreads();
    u64 before = 0;
    int w = 0;
    while (w < kWaves - 1 && before + shared().wave[w] < nth) before += shared().wave[w++];
    const int from = w * run(), to = min(V, from + run());
    const int per = (to - from + kThreads - 1) / kThreads;
    const int first = min(from + tid * per, to), last = min(first + per, to);
    // Four at a time, so that their loads are under way together.
    u64 sum = 0, four[4] = {};
    for (int i = first; i < last; i += 4) {
      float v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)x[min(i + e, last - 1)];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += four[e] = i + e < last ? q(v[e], i + e) : 0;
    }
    const u64 upto = wave_prefix(sum);
    __syncthreads();
    if (tid % 64 == 63) shared().wave[tid / 64] = upto;
    if (tid == 0) shared().first = -1;
    __syncthreads();
    before += upto - sum + waves_before();
    if (before < nth && nth <= before + sum) {
      int i = first;
      if (per > 4) {
        for (; i < last - 1; ++i) {
          before += q((float)x[i], i);
          if (before >= nth) break;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e) {
          before += four[e];
          i += before < nth && first + e < last - 1;
        }
      }
      shared().first = i;
    }
    __syncthreads();
    return shared().first;
  }
};

template <typename V>
__device__ __forceinline__ V setting(const V* each, V all, int64_t row) {
  return each ? each[row] : all;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  const int64_t row = block_of();
  if (row >= a.M) return;
  const int tid = threadIdx.x, V = (int)a.V;
  Row<T> r{static_cast<const T*>(a.x) + row * a.ldx, V, 0.0f, 0.0f, 0.0f, 0.0, ldexp(1.0, 52 - a.shift), ldexp(1.0, a.shift), -1};

  const float temperature = setting(a.temperature, a.temperature_all, row);
  const float top_p = setting(a.top_p, a.top_p_all, row), min_p = setting(a.min_p, a.min_p_all, row);
  const int top_k = setting(a.top_k, a.top_k_all, row);
  const float uniform = a.uniforms[row];
  const auto done = [&](int64_t token, float logprob) INLINE {
    if (tid == 0) {
      if (a.ids64)
        static_cast<int64_t*>(a.tokens)[row] = token;
      else
        static_cast<int32_t*>(a.tokens)[row] = (int32_t)token;
      if (a.logprobs) a.logprobs[row] = logprob;
    }
  };

  float own_most = -__builtin_inff();
  r.template lines<kVec<T>, 8>([&](const auto& some) INLINE {
#pragma unroll
    for (int e = 0; e < some.kN; ++e) own_most = MaxNan::of(own_most, some.v[e]);
  });
  float most = lanes_all<MaxNan, 64>(own_most);
  if (tid % 64 == 0) shared().wave_max[tid / 64] = most;
  __syncthreads();
  most = shared().wave_max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) most = MaxNan::of(most, shared().wave_max[w]);
  // All uniform over the workgroup from here.
  const bool fine = temperature >= 0.0f && temperature < __builtin_inff() && top_p == top_p && min_p == min_p &&
                    uniform == uniform;
  if (!(most < __builtin_inff()) || !fine) return done(-1, __builtin_nanf(""));
  if (most == -__builtin_inff()) return done(-1, most);
  r.m = most, r.half_m = 0.5f * most;
  if (temperature == 0.0f) {
    int first = V;
    r.template scan<6>([&](const auto& some) INLINE {
#pragma unroll
      for (int e = some.kN - 1; e >= 0; --e) first = some.v[e] == most && some.first + e < first ? some.first + e : first;
    });
#pragma unroll
    for (int d = 1; d < 64; d *= 2) first = min(first, __shfl_xor(first, d));
    if (tid % 64 == 0) shared().wave[tid / 64] = (u64)first;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) first = min(first, (int)shared().wave[w]);
    return done(first, 0.0f);
  }
  r.octaves = 1.4426950408889634074 / (double)temperature;
  // Finite, so that the maximum is in the first bin.
  r.to_bins = fminf((float)(2 * (kBins / kRange) * r.octaves), 1e30f);

  const bool use_k = top_k > 0 && top_k < V, use_p = top_p < 1.0f;
  // The least logit of a weight of min_p of the largest, by halving the keys between two that are and are
  // not: a few steps about where it has to be, or all of them where rounding has moved it further.
  float low = -__builtin_inff();
  if (min_p > 0.0f) {
    const double least = log2(fmin((double)min_p, 1.0));
    const auto reaches = [&](uint32_t key) INLINE { return r.exponent(value_of(key)) >= least; };
    uint32_t out = key_of(low), in = key_of(most);
    const uint32_t about = max(out + 8, min(in, key_of((float)(least / r.octaves + (double)most))));
    if (reaches(min(in, about + 8)) && !reaches(about - 8)) in = min(in, about + 8), out = about - 8;
    while (out + 1 < in) {
      const uint32_t mid = out + (in - out) / 2;
      (reaches(mid) ? in : out) = mid;
    }
    low = value_of(in);
  }
  const auto clear = [&]() INLINE {
    __syncthreads();
    for (int i = tid; i < kBins; i += kThreads) shared().count[i] = 0, shared().mass[i] = 0;
    __syncthreads();
  };
  if (use_k && top_k <= kThreads) {
    // At least k logits are as large as the k-th largest of the threads' maxima, and few more.
    clear();
    const int b = r.bin_of(own_most);
    if (b < kBins - 1) atomicAdd(&shared().count[b], 1u);
    __syncthreads();
    r.find(kBins, (u64)top_k, [&](int i) INLINE { return (u64)shared().count[i]; });
    const int upto = shared().found;
    if (upto >= 0) r.keep([&](float v) INLINE { return r.bin_of(v) <= upto; });
  } else if (!use_k && !use_p && min_p > 0.0f) {
    r.keep([&](float v) INLINE { return v >= low; });
  }
  Border border{0, 0, 0};
  bool bounded = false;
  if (use_k || use_p) {
    clear();
    // The last bin's weights are 0: whether they are kept changes nothing.
    r.template scan<4, true>([&](const auto& some) INLINE {
      int b[some.kN];
      bool any = false;
#pragma unroll
      for (int e = 0; e < some.kN; ++e) b[e] = r.bin_of(some.v[e]), any |= b[e] < kBins - 1;
      if (!any) return;
      u64 w[some.kN];
      if (use_p)
#pragma unroll
        for (int e = 0; e < some.kN; ++e) w[e] = r.weight(some.v[e]);
#pragma unroll
      for (int e = 0; e < some.kN; ++e)
        if (b[e] < kBins - 1) {
          atomicAdd(&shared().count[b[e]], 1u);
          if (use_p) atomicAdd(&shared().mass[b[e]], w[e]);
        }
    });
    __syncthreads();
    // Candidates of all bins up to a border's, where the row was searched.
    const auto narrow = [&](int b) INLINE {
      if (r.kept >= 0) return;
      u64 n = 0;
      for (int i = tid; i <= b; i += kThreads) n += shared().count[i];
      n = wave_sum(n);
      __syncthreads();
      if (tid % 64 == 0) shared().wave[tid / 64] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) n += shared().wave[w];
      if (n <= kKept) r.keep([&](float v) INLINE { return r.bin_of(v) <= b; });
    };
    u64 total = 0;
    int last_bin = kBins;
    if (use_k) {
      r.find(kBins, (u64)top_k, [&](int i) INLINE { return (u64)shared().count[i]; });
      const u64 rest = (u64)top_k - shared().before;
      last_bin = shared().found;
      if (last_bin >= 0) {
        narrow(last_bin);
        border = r.template border_in<false>(last_bin, rest);
        bounded = true;
      } else {
        last_bin = kBins;
      }
    }
    if (use_p) {
      // The mass of the k largest: whole bins, and of the border's bin what is above it and its ties.
      u64 mine = 0;
      for (int i = tid; i < min(last_bin, kBins); i += kThreads) mine += shared().mass[i];
      if (bounded) {
        r.template scan<2, true>([&](const auto& some) INLINE {
#pragma unroll
          for (int e = 0; e < some.kN; ++e)
            if (r.bin_of(some.v[e]) == last_bin && key_of(some.v[e]) > border.key) mine += r.weight(some.v[e]);
        });
        if (tid == 0) mine += border.ties * r.weight(value_of(border.key));
      }
      mine = wave_sum(mine);
      __syncthreads();
      if (tid % 64 == 0) shared().wave[tid / 64] = mine;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) total += shared().wave[w];
      const double part = __builtin_ceil((double)fmaxf(top_p, 0.0f) * (double)total);
      const u64 target = max((u64)1, min(total, (u64)part));
      r.find(kBins, target, [&](int i) INLINE { return shared().mass[i]; });
      const int b = shared().found;
      const u64 rest = target - shared().before;
      narrow(b);
      border = r.template border_in<true>(b, rest);
      bounded = true;
    }
  }

  // Ties: the index of the last one that is kept.
  int last_tie = V;
  if (bounded && border.ties < border.equal) {
    const auto is_tie = [&](float v, int) INLINE { return (u64)(key_of(v) == border.key); };
    u64 ties = 0;
    r.template scan<6>([&](const auto& some) INLINE {
#pragma unroll
      for (int e = 0; e < some.kN; ++e) ties += is_tie(some.v[e], some.first + e);
    });
    last_tie = r.locate(wave_sum(ties), border.ties, is_tie);
  }
  // Kept are logits above `edge` and, up to index last_tie, those at it.
  float edge = bounded ? value_of(border.key) : -__builtin_inff();
  if (low > edge) edge = low, last_tie = V;
  const auto counts = [&](float v, int i) INLINE { return v > edge || (v == edge && i <= last_tie); };
  const auto mass_of = [&](float v, int i) INLINE -> u64 { return counts(v, i) ? r.weight(v) : 0; };
  double real = 0.0;
  r.template scan<4, true>([&](const auto& some) INLINE {
    bool any = false;
#pragma unroll
    for (int e = 0; e < some.kN; ++e) any |= counts(some.v[e], some.first + e);
    if (any)  // most logits need no exponential
#pragma unroll
      for (int e = 0; e < some.kN; ++e)
        real += only(counts(some.v[e], some.first + e), r.weight_real(some.v[e]));
  });
  const u64 mine = wave_sum((u64)(real * r.units));
  __syncthreads();
  if (tid % 64 == 0) shared().wave[tid / 64] = mine;
  __syncthreads();
  u64 total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) total += shared().wave[w];
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

// Root-mean-square norm with the residual's addition, and its backward pass.
//
//   h = x + r;  rstd = (mean h^2 + eps)^(-1/2);  y = h rstd w
//   8-bit y:    s = max |y| / Q (Q = 127 or 448),  q = y / s to nearest even, as
//               h w Q / max |h w|: rstd, the same above and below, is left out
//   backward:   t = dy w;  xh = h rstd;  dx = rstd (t - xh mean(t xh)) + dh;
//               dw = sum over rows of dy xh
//
// Bound by memory: about one operation a byte. A row is read once and held in
// registers between the sum and the output. 4096 x 8192 bf16 with a residual to 8
// bits: 43 us, 5.5 TB/s; a copy of 1 GiB reaches 5.0. The backward pass reads dy, h
// and dh once and leaves one row of partials a CU: 4096 x 4096 bf16 in 29 us, 4.6
// TB/s, the join of the partials (4 us) included. One row takes 4 us, a launch's time.
#include <type_traits>

#include "kernels.hpp"
#include "lm_common.hpp"
#include "lm_kernels.hpp"

namespace edsl {
namespace lm {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// What y holds.
enum : int { kOutSame = 0, kOutI8 = 1, kOutE4m3 = 2 };

// (sum a, max b) over the TPR threads that share a row, in all of them. `lds`
// holds two floats a wave; a barrier precedes its next use.
template <int TPR>
__device__ __forceinline__ void row_reduce(float& a, float& b, float* lds, bool want_b) {
  if constexpr (TPR < 64) {
    a = lanes_all<Sum, TPR>(a);
    if (want_b) b = lanes_all<MaxNan, TPR>(b);
  } else {
    a = wave_all<Sum>(a);
    if (want_b) b = wave_all<MaxNan>(b);
  }
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) {
      lds[2 * wave] = a;
      lds[2 * wave + 1] = b;
    }
    __syncthreads();
    a = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) a += lds[2 * w];
    if (want_b) {
      b = lds[1];
#pragma unroll
      for (int w = 1; w < W; ++w) b = MaxNan::of(b, lds[2 * w + 1]);
    }
  }
}

template <typename T>
__device__ __forceinline__ float weight_at(const void* w, bool f32, int64_t i) {
  return f32 ? static_cast<const float*>(w)[i] : (float)static_cast<const T*>(w)[i];
}

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int64_t i0, int64_t n, float (&v)[VEC]) {
  if (f32) {
    const auto r = load_guarded<float, VEC>(static_cast<const float*>(w), i0, n);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = r.v[e];
  } else {
    const auto r = load_guarded<T, VEC>(static_cast<const T*>(w), i0, n);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)r.v[e];
  }
}

// An 8-bit row's quotients h w Q / max |h w|. Q over the power of two above it has 7
// bits at most, so that its product with h w is exact where h w has 17 bits, and the
// quotient is a correctly rounded one: values halfway between two codes are common
// among products of few bits, and go to the even code. (The product of y and a
// rounded 1 / s put 3 codes in 100000 of bf16 rows on the wrong side. It took 42.6 us
// at 4096 x 8192 bf16 to int8, this takes 42.9; 2048 x 4096 to e4m3 10.7 and 11.0.)
template <int OUT>
struct RowCodes {
  static constexpr float kTop = OUT == kOutI8 ? 127.0f : 448.0f, kAbove = OUT == kOutI8 ? 128.0f : 512.0f;
  float by, most, inv;  // of h w; max |h w| by the same power of two; its reciprocal, or 0: codes of 0

  // From max |h w|; returns the row's scale.
  __device__ __forceinline__ float set(float amax, float rstd) {
    const float scale = amax * rstd / kTop;
    const float up = amax < 0x1p-60f ? 0x1p64f : 1.0f;  // away from subnormal numbers
    by = up * (kTop / kAbove);
    most = amax * up;
    inv = scale >= 0x1p-126f ? 1.0f / most : 0.0f;
    return scale;
  }
  __device__ __forceinline__ float of(float hw) const {
    const float t = hw * by, q = t * inv;
    return fmaf(fmaf(-q, most, t), inv, q) * kAbove;
  }
};
template <>
struct RowCodes<kOutSame> {
  __device__ __forceinline__ float set(float, float) { return 0.0f; }
};

// Writes elements i0 .. i0+VEC-1 of a row's y.
template <typename T, int OUT, int VEC>
__device__ __forceinline__ void store_y(void* y, int64_t row_at, int64_t i0, int64_t n, const float (&h)[VEC],
                                        const float (&w)[VEC], float rstd, const RowCodes<OUT>& codes) {
  if constexpr (OUT == kOutSame) {
    Packed<T, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = (T)(h[e] * rstd * w[e]);
    store_guarded<T, VEC>(static_cast<T*>(y) + row_at, i0, n, r);
  } else {
    Packed<uint8_t, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      uint32_t code = 0;
      if constexpr (OUT == kOutI8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float q = __builtin_amdgcn_fmed3f(rintf(codes.of(h[e + j] * w[e + j])), -127.0f, 127.0f);
          code |= ((uint32_t)(int)q & 0xffu) << (8 * j);
        }
      } else {
        float q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = __builtin_amdgcn_fmed3f(codes.of(h[e + j] * w[e + j]), -448.0f, 448.0f);
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        code = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], c, true);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) r.v[e + j] = (uint8_t)(code >> (8 * j));
    }
    store_guarded<uint8_t, VEC>(static_cast<uint8_t*>(y) + row_at, i0, n, r);
  }
}

// A thread's vectors of a row: no check where the threads' vectors are the row,
// one a vector where it is whole vectors (then no load waits for another), one an
// element else.
template <typename T, int TPR, int NV>
__device__ __forceinline__ void load_row(const T* row, int t, int64_t n, Packed<T, kVec<T>> (&v)[NV]) {
  constexpr int VEC = kVec<T>;
  if (n == (int64_t)TPR * NV * VEC) {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = load_packed<T, VEC>(row + (j * TPR + t) * VEC);
  } else if (n % VEC == 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      v[j] = Packed<T, VEC>{};
      if ((j * TPR + t) * VEC < n) v[j] = load_packed<T, VEC>(row + (j * TPR + t) * VEC);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = load_guarded<T, VEC>(row, (j * TPR + t) * VEC, n);
  }
}

template <typename T, int TPR, int NV>
__device__ __forceinline__ void load_weights(const void* w, bool f32, int t, int64_t n, float (&v)[NV][kVec<T>]) {
  constexpr int VEC = kVec<T>;
  if (f32 && sizeof(T) != 4) {
#pragma unroll
    for (int j = 0; j < NV; ++j) load_weight<T, VEC>(w, true, (j * TPR + t) * VEC, n, v[j]);
    return;
  }
  Packed<T, VEC> p[NV];
  load_row<T, TPR, NV>(static_cast<const T*>(w), t, n, p);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[j][e] = (float)p[j].v[e];
}

// TPR threads hold one row of up to TPR * NV vectors in registers; workgroups of
// 256 threads (or TPR) take 256 / TPR rows.
template <typename T, int OUT, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) rms_norm_kernel(NormArgs a) {
  constexpr int VEC = kVec<T>, BLOCK = TPR < 256 ? 256 : TPR, ROWS = BLOCK / TPR;
  __shared__ float lds[2 * BLOCK / 64];
  const int64_t row = (int64_t)block_of() * ROWS + threadIdx.x / TPR;
  if (row >= a.M) return;  // by lanes or waves where they hold a row, without barriers, else by workgroups
  const int t = threadIdx.x % TPR;
  const bool wf32 = a.weight_type == kF32;
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
  float h[NV][VEC], w[NV][VEC];
  Packed<T, VEC> px[NV], pr[NV];
  load_row<T, TPR, NV>(x, t, a.N, px);
  if (a.residual) load_row<T, TPR, NV>(static_cast<const T*>(a.residual) + row * a.ldr, t, a.N, pr);
  load_weights<T, TPR, NV>(a.weight, wf32, t, a.N, w);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[j][e] = (float)px[j].v[e];
  if (a.residual)
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[j][e] += (float)pr[j].v[e];
  float sum = 0.0f, amax = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum = fmaf(h[j][e], h[j][e], sum);
      if constexpr (OUT != kOutSame) amax = MaxNan::of(amax, fabsf(h[j][e] * w[j][e]));
    }
  row_reduce<TPR>(sum, amax, lds, OUT != kOutSame);
  const float rstd = 1.0f / sqrtf(sum / (float)a.N + a.eps);
  RowCodes<OUT> codes;
  if (const float scale = codes.set(amax, rstd); OUT != kOutSame && t == 0) a.scales[row] = scale;
  if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t i0 = ((int64_t)j * TPR + t) * VEC;
    if (i0 >= a.N) break;
    if (a.total) {
      Packed<T, VEC> r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = (T)h[j][e];
      store_guarded<T, VEC>(static_cast<T*>(a.total) + row * a.ldt, i0, a.N, r);
    }
    store_y<T, OUT, VEC>(a.y, row * a.ldy, i0, a.N, h[j], w[j], rstd, codes);
  }
}

// Rows of any length: one workgroup of 1024 threads reads the row twice, and
// writes in the second pass only, so that the outputs may be the inputs.
template <typename T, int OUT>
__global__ void __launch_bounds__(1024) rms_norm_long_kernel(NormArgs a) {
  constexpr int VEC = kVec<T>;
  __shared__ float lds[32];
  const int64_t row = block_of();
  if (row >= a.M) return;
  const bool wf32 = a.weight_type == kF32;
  const T* const x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* const res = a.residual ? static_cast<const T*>(a.residual) + row * a.ldr : nullptr;
  float h[VEC], w[VEC], sum = 0.0f, amax = 0.0f;
  const auto load = [&](int64_t i0) {
    const auto v = load_guarded<T, VEC>(x, i0, a.N);
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] = (float)v.v[e];
    if (res) {
      const auto r = load_guarded<T, VEC>(res, i0, a.N);
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[e] += (float)r.v[e];
    }
    load_weight<T, VEC>(a.weight, wf32, i0, a.N, w);
  };
  for (int64_t i0 = (int64_t)threadIdx.x * VEC; i0 < a.N; i0 += 1024 * VEC) {
    load(i0);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      sum = fmaf(h[e], h[e], sum);
      if constexpr (OUT != kOutSame) amax = MaxNan::of(amax, fabsf(h[e] * w[e]));
    }
  }
  row_reduce<1024>(sum, amax, lds, OUT != kOutSame);
  const float rstd = 1.0f / sqrtf(sum / (float)a.N + a.eps);
  RowCodes<OUT> codes;
  if (const float scale = codes.set(amax, rstd); OUT != kOutSame && threadIdx.x == 0) a.scales[row] = scale;
  if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
  for (int64_t i0 = (int64_t)threadIdx.x * VEC; i0 < a.N; i0 += 1024 * VEC) {
    load(i0);
    if (a.total) {
      Packed<T, VEC> r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = (T)h[e];
      store_guarded<T, VEC>(static_cast<T*>(a.total) + row * a.ldt, i0, a.N, r);
    }
    store_y<T, OUT, VEC>(a.y, row * a.ldy, i0, a.N, h, w, rstd, codes);
  }
}

template <typename T, int OUT, int TPR, int NV>
hipError_t launch_row(const NormArgs& a, hipStream_t stream) {
  constexpr int BLOCK = TPR < 256 ? 256 : TPR, ROWS = BLOCK / TPR;
  hipLaunchKernelGGL((rms_norm_kernel<T, OUT, TPR, NV>), grid_of((a.M + ROWS - 1) / ROWS), dim3(BLOCK), 0, stream, a);
  return launched();
}

// Threads of a row x vectors of a thread. Short rows share a wave (262144 x 128 bf16
// in 22 us on 16 threads each against 59 on 64) or take one without a barrier (65536
// x 1024 in 46 on 64x2 against 76 on 256x1). More threads rather than vectors from 513
// vectors on (4096 x 8192 bf16 to 8 bits 42.8 us on 512x2 against 44.1 on 256x4; 2048 x
// 16384 49 on 1024x2 against 54 on 1024x4), and below where a CU has one row at most
// (`few`; 256 x 4096 bf16 3.7 against 4.1), but not for many (2001 x 2001 f32 7.7 on
// 256x2 against 8.2; 2048 x 4096 bf16 to 8 bits 11.0 against 12.3). Rows beyond 4096
// vectors are read twice: 2048 x 40960 bf16 with a residual in 236 us, 201 of them its bytes.
template <typename T, int OUT>
hipError_t launch_norm(const NormArgs& a, bool few, hipStream_t stream, const char** plan) {
  const int64_t vecs = (a.N + kVec<T> - 1) / kVec<T>;
  if (vecs <= 16) return *plan = "row=16x1", launch_row<T, OUT, 16, 1>(a, stream);
  if (vecs <= 32) return *plan = "row=32x1", launch_row<T, OUT, 32, 1>(a, stream);
  if (vecs <= 64) return *plan = "row=64x1", launch_row<T, OUT, 64, 1>(a, stream);
  if (vecs <= 128) return *plan = "row=64x2", launch_row<T, OUT, 64, 2>(a, stream);
  if (vecs <= 256) return *plan = "row=256x1", launch_row<T, OUT, 256, 1>(a, stream);
  if (vecs <= 512 && few) return *plan = "row=512x1", launch_row<T, OUT, 512, 1>(a, stream);
  if (vecs <= 512) return *plan = "row=256x2", launch_row<T, OUT, 256, 2>(a, stream);
  if (vecs <= 1024) return *plan = "row=512x2", launch_row<T, OUT, 512, 2>(a, stream);
  if (vecs <= 2048) return *plan = "row=1024x2", launch_row<T, OUT, 1024, 2>(a, stream);
  if (vecs <= 4096) return *plan = "row=1024x4", launch_row<T, OUT, 1024, 4>(a, stream);
  *plan = "row=long";
  hipLaunchKernelGGL((rms_norm_long_kernel<T, OUT>), grid_of(a.M), dim3(1024), 0, stream, a);
  return launched();
}

template <typename T>
hipError_t launch_norm_out(const NormArgs& a, bool few, hipStream_t stream, const char** plan) {
  if (a.y_type == kI8) return launch_norm<T, kOutI8>(a, few, stream, plan);
  if (a.y_type == kE4m3) return launch_norm<T, kOutE4m3>(a, few, stream, plan);
  return launch_norm<T, kOutSame>(a, few, stream, plan);
}

// ---------------------------------------------------------------- backward
// The backward pass. A workgroup of 1024 threads is 1024 / TPR teams with a row
// each; a thread keeps the same NV vectors of columns in every row, its part of
// dweight in registers, and the teams join theirs through LDS at the end, so that
// there is one row of partials a CU. Where the registers hold it, the next row is on
// its way while one is summed, in registers of its own and by the same loads every
// turn, whatever the row: a load under a branch, or a copied register, would wait
// for all of them (4096 x 4096 bf16 30 us against 33, 4096 x 8192 53 against 59).
// WF32: the weight is f32 and x is not. DH: dh is there. WHOLE: rows are whole
// vectors.
template <typename T, int TPR, int NV, bool WF32, bool DH, bool WHOLE>
__global__ void __launch_bounds__(1024, 4) rms_norm_backward_kernel(NormBackwardArgs a) {
  constexpr int VEC = kVec<T>, TEAMS = 1024 / TPR, WAVES = TPR / 64;
  constexpr int DEPTH = NV * VEC > 8 ? 1 : 2;  // rows in registers; three were no faster
  using Vals = Packed<T, VEC>;
  using W = std::conditional_t<WF32, float, T>;
  __shared__ float lds[2][16];
  __shared__ float joined[TEAMS > 1 ? TPR * NV * VEC : 1];
  const int team = threadIdx.x / TPR, t = threadIdx.x % TPR;
  Packed<W, VEC> w[NV];  // zeros past the row's end
  if constexpr (WF32) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      w[j] = load_guarded<W, VEC>(static_cast<const W*>(a.weight), (j * TPR + t) * VEC, a.N);
  } else {
    load_row<T, TPR, NV>(static_cast<const T*>(a.weight), t, a.N, w);
  }
  float dw[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[j][e] = 0.0f;
  struct Row {
    Vals dy[NV], h[NV], dh[DH ? NV : 1];
    float rstd;
  };
  // Rows stay packed: opened for the sum and again for the gradient, they take
  // half of the registers.
  const auto keep_packed = [](Vals (&v)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      u32x4 raw = __builtin_bit_cast(u32x4, v[j]);
      asm("" : "+v"(raw));
      v[j] = __builtin_bit_cast(Vals, raw);
    }
  };
  // Vectors past a whole row's end repeat its last one: their weights are zero.
  const auto load_vectors = [&](const void* p, int64_t at, auto& v) {
    const T* const row = static_cast<const T*>(p) + at;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i0 = (j * TPR + t) * VEC;
      if constexpr (WHOLE)
        v[j] = load_packed<T, VEC>(row + (i0 < (int)a.N ? i0 : (int)a.N - VEC));
      else
        v[j] = load_guarded<T, VEC>(row, i0, a.N);
    }
  };
  const auto load = [&](int64_t row, Row& r) {
    if (row >= a.M) row = a.M - 1;  // not used
    load_vectors(a.dy, row * a.lddy, r.dy);
    load_vectors(a.h, row * a.ldh, r.h);
    if constexpr (DH) load_vectors(a.dh, row * a.lddh, r.dh);
    r.rstd = a.rstd[row];
  };
  const int64_t step = (int64_t)a.groups * TEAMS;
  int64_t first = (int64_t)blockIdx.x * TEAMS;  // the first team's row; every team turns as often
  int turn = 0;
  const auto one = [&](Row& now) {
    const int64_t row = first + team;
    const float rstd = now.rstd;
    const bool in = row < a.M;
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float g = in ? (float)now.dy[j].v[e] : 0.0f, xh = in ? (float)now.h[j].v[e] * rstd : 0.0f;
        dot = fmaf(g * (float)w[j].v[e], xh, dot);
        dw[j][e] = fmaf(g, xh, dw[j][e]);
      }
    keep_packed(now.dy);
    keep_packed(now.h);
    // Two buffers in turn: the barrier of the next row stands between the reads
    // of one and its next writes.
    if constexpr (TPR < 64)
      dot = lanes_all<Sum, TPR>(dot);
    else
      dot = wave_all<Sum>(dot);
    if constexpr (WAVES > 1) {
      if (t % 64 == 0) lds[turn][threadIdx.x / 64] = dot;
      __syncthreads();
      dot = 0.0f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) dot += lds[turn][team * WAVES + i];
      turn ^= 1;
    }
    const float mean = dot / (float)a.N;
    T* const pdx = static_cast<T*>(a.dx) + row * a.lddx;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int64_t i0 = ((int64_t)j * TPR + t) * VEC;
      if (!in || i0 >= a.N) break;
      Vals r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = (float)now.h[j].v[e] * rstd;
        float d = rstd * fmaf(-xh, mean, (float)now.dy[j].v[e] * (float)w[j].v[e]);
        if constexpr (DH) d += (float)now.dh[j].v[e];
        r.v[e] = (T)d;
      }
      store_guarded<T, VEC>(pdx, i0, a.N, r);
    }
  };
  Row rows[DEPTH];
  if (first < a.M) {
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) load(first + d * step + team, rows[d]);
    bool more = true;
    while (more) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        if (more) {
          load(first + (DEPTH - 1) * step + team, rows[(d + DEPTH - 1) % DEPTH]);
          __builtin_amdgcn_sched_barrier(0);
          one(rows[d]);
          first += step;
          more = first < a.M;
        }
      }
    }
  }
  if (!a.dweight) return;
  if constexpr (TEAMS > 1) {
    for (int i = 0; i < TEAMS; ++i) {
      if (team == i)
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float& s = joined[(j * TPR + t) * VEC + e];
            s = i == 0 ? dw[j][e] : s + dw[j][e];
          }
      __syncthreads();
    }
  }
  if (team != 0) return;
  float* const part = a.partials + (int64_t)blockIdx.x * a.N;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t i0 = ((int64_t)j * TPR + t) * VEC;
    if (i0 >= a.N) break;
    Packed<float, VEC> r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = TEAMS > 1 ? joined[i0 + e] : dw[j][e];
    store_guarded<float, VEC>(part, i0, a.N, r);
  }
}

// Rows of any length, one workgroup a row at a time, each read twice; dweight is
// added up in the workgroup's row of partials.
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_backward_long_kernel(NormBackwardArgs a) {
  constexpr int VEC = kVec<T>;
  __shared__ float lds[2][32];
  const bool wf32 = a.weight_type == kF32;
  float* const part = a.dweight ? a.partials + (int64_t)blockIdx.x * a.N : nullptr;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.M; row += a.groups, turn ^= 1) {
    const T* const pdy = static_cast<const T*>(a.dy) + row * a.lddy;
    const T* const ph = static_cast<const T*>(a.h) + row * a.ldh;
    const float rstd = a.rstd[row];
    float dot = 0.0f, none = 0.0f, w[VEC];
    for (int64_t i0 = (int64_t)threadIdx.x * VEC; i0 < a.N; i0 += 1024 * VEC) {
      const auto dy = load_guarded<T, VEC>(pdy, i0, a.N);
      const auto h = load_guarded<T, VEC>(ph, i0, a.N);
      load_weight<T, VEC>(a.weight, wf32, i0, a.N, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) dot = fmaf((float)dy.v[e] * w[e], (float)h.v[e] * rstd, dot);
    }
    row_reduce<1024>(dot, none, lds[turn], false);
    const float mean = dot / (float)a.N;
    for (int64_t i0 = (int64_t)threadIdx.x * VEC; i0 < a.N; i0 += 1024 * VEC) {
      const auto dy = load_guarded<T, VEC>(pdy, i0, a.N);
      const auto h = load_guarded<T, VEC>(ph, i0, a.N);
      load_weight<T, VEC>(a.weight, wf32, i0, a.N, w);
      Packed<T, VEC> dh, r;
      if (a.dh) dh = load_guarded<T, VEC>(static_cast<const T*>(a.dh) + row * a.lddh, i0, a.N);
      Packed<float, VEC> dw;
      if (part && row != blockIdx.x)
        dw = load_guarded<float, VEC>(part, i0, a.N);
      else
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw.v[e] = 0.0f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = (float)h.v[e] * rstd;
        float d = rstd * fmaf(-xh, mean, (float)dy.v[e] * w[e]);
        if (a.dh) d += (float)dh.v[e];
        r.v[e] = (T)d;
        dw.v[e] = fmaf((float)dy.v[e], xh, dw.v[e]);
      }
      store_guarded<T, VEC>(static_cast<T*>(a.dx) + row * a.lddx, i0, a.N, r);
      if (part) store_guarded<float, VEC>(part, i0, a.N, dw);
    }
  }
}

// dweight[n] = the sum of the groups' partials, in a fixed order: 16 columns a
// workgroup, so that there is one for most CUs, the groups in 64 interleaved
// parts that are then joined in order.
__global__ void __launch_bounds__(1024) dweight_kernel(const float* partials, int groups, int64_t N, float* dweight) {
  __shared__ float lds[64][17];
  const int c = threadIdx.x % 16, part = threadIdx.x / 16;
  const int64_t first_n = (int64_t)block_of() * 16, n = first_n + c;
  float s = 0.0f;
  if (n < N)
#pragma unroll 4
    for (int g = part; g < groups; g += 64) s += partials[(int64_t)g * N + n];
  lds[part][c] = s;
  __syncthreads();
  if (threadIdx.x < 256) {  // sixteen threads a column
    const int col = threadIdx.x / 16, first = threadIdx.x % 16 * 4;
    float v = 0.0f;
#pragma unroll
    for (int p = 0; p < 4; ++p) v += lds[first + p][col];
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    const int64_t at = first_n + col;
    if (first == 0 && at < N) dweight[at] = v;
  }
}

// Threads of a row, 0 for rows of any length: a vector each, two of f32 (4096 x
// 4096 f32 in 52 us, with one in 59); twice that of the longest rows, though four of
// f32 spill 7 registers (2048 x 16384 in 89 us, read twice in 156), 69 where rows are
// not whole vectors, and with dh 141 or 171 (139 us, read twice 173). 65536 x 128 bf16
// in 22 us, 42 on 64 threads. Rows read twice also add to their partials in memory:
// 2048 x 20480 bf16 in 164 us, with dh 195.
int backward_threads(int64_t N, int type) {
  int64_t vecs = (N * type_bytes(type) + 15) / 16;
  if (vecs > (type == kF32 ? 4096 : 2048)) return 0;
  if (type == kF32) vecs = (vecs + 1) / 2;
  return vecs <= 16 ? 16 : vecs <= 32 ? 32 : vecs <= 64 ? 64 : vecs <= 128 ? 128 : vecs <= 256 ? 256 : vecs <= 512 ? 512 : 1024;
}

template <typename T, int TPR, int NV, bool WF32, bool DH>
void launch_backward_whole(const NormBackwardArgs& a, hipStream_t stream) {
  if (a.N % kVec<T> == 0)
    hipLaunchKernelGGL((rms_norm_backward_kernel<T, TPR, NV, WF32, DH, true>), dim3(a.groups), dim3(1024), 0, stream, a);
  else
    hipLaunchKernelGGL((rms_norm_backward_kernel<T, TPR, NV, WF32, DH, false>), dim3(a.groups), dim3(1024), 0, stream, a);
}

template <typename T, int TPR, int NV>
void launch_backward_rows(const NormBackwardArgs& a, hipStream_t stream) {
  if (sizeof(T) != 4 && a.weight_type == kF32)
    a.dh ? launch_backward_whole<T, TPR, NV, sizeof(T) != 4, true>(a, stream)
         : launch_backward_whole<T, TPR, NV, sizeof(T) != 4, false>(a, stream);
  else
    a.dh ? launch_backward_whole<T, TPR, NV, false, true>(a, stream)
         : launch_backward_whole<T, TPR, NV, false, false>(a, stream);
}

template <typename T>
hipError_t launch_backward(const NormBackwardArgs& a, hipStream_t stream) {
  constexpr int NV = sizeof(T) == 4 ? 2 : 1;
  const int64_t vecs = (a.N + kVec<T> - 1) / kVec<T>;
  if (a.M > 0) {
    switch (backward_threads(a.N, a.type)) {
      case 16: launch_backward_rows<T, 16, NV>(a, stream); break;
      case 32: launch_backward_rows<T, 32, NV>(a, stream); break;
      case 64: launch_backward_rows<T, 64, NV>(a, stream); break;
      case 128: launch_backward_rows<T, 128, NV>(a, stream); break;
      case 256: launch_backward_rows<T, 256, NV>(a, stream); break;
      case 512: launch_backward_rows<T, 512, NV>(a, stream); break;
      case 1024:
        if (vecs <= 1024 * NV)
          launch_backward_rows<T, 1024, NV>(a, stream);
        else
          launch_backward_rows<T, 1024, 2 * NV>(a, stream);
        break;
      default:
        hipLaunchKernelGGL((rms_norm_backward_long_kernel<T>), dim3(a.groups), dim3(1024), 0, stream, a);
    }
    if (const hipError_t e = launched(); e != hipSuccess) return e;
  }
  if (!a.dweight) return hipSuccess;
  hipLaunchKernelGGL(dweight_kernel, grid_of((a.N + 15) / 16), dim3(1024), 0, stream, a.partials,
                     a.M > 0 ? a.groups : 0, a.N, a.dweight);
  return launched();
}

}  // namespace

hipError_t launch_rms_norm(const NormArgs& a, int cus, hipStream_t stream, const char** plan) {
  const bool few = a.M <= cus;
  if (a.type == kF32) return launch_norm_out<float>(a, few, stream, plan);
  if (a.type == kBf16) return launch_norm_out<bf16>(a, few, stream, plan);
  return launch_norm_out<f16>(a, few, stream, plan);
}

int rms_norm_backward_groups(int64_t M, int64_t N, int type, int cus) {
  const int tpr = backward_threads(N, type);
  const int64_t teams = tpr > 0 ? 1024 / tpr : 1;
  const int64_t wgs = (M + teams - 1) / teams;
  return (int)(wgs < 1 ? 1 : wgs < cus ? wgs : cus);
}

hipError_t launch_rms_norm_backward(const NormBackwardArgs& a, hipStream_t stream) {
  if (a.type == kF32) return launch_backward<float>(a, stream);
  if (a.type == kBf16) return launch_backward<bf16>(a, stream);
  return launch_backward<f16>(a, stream);
}

}  // namespace lm
}  // namespace edsl

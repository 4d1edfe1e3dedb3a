// libflyb200: the row operators next to the quantised products (include/flyb200.h): residual addition, root-mean-square
// norm and quantisation in one kernel; gated activation and quantisation in one kernel.
//
//   norm     h = round(x + r), n = h * w * rsqrt(mean(h^2) + eps)           (h is what is stored as the new residual)
//   gated    v = g / (1 + exp(-g)) * u
//
// and of n or v, held in fp32: codes per row (scale s = max|v| * (1 / qmax), 0 -> 1; code = nearest(v / s), ties to even),
// MXFP8 codes and E8M0 scales per 32 values as per_1x32_f8_quant, or values rounded to the type of x.
//
// Bound: memory.  Each input is read once and each output written once; between its reductions and its conversion a row stays in
// registers as the fp32 values that are converted.
#include "../../include/flyb200.h"
#include "host_common.h"
#include "quant_kernel.cuh"
#include "gemm_kernels.cuh"
#include "mx_quant_kernel.cuh"

#include <atomic>
#include <cstring>

using namespace flyb200;

namespace {

enum : int { Q_NONE = FLYB200_ROWQ_NONE, Q_FP8 = FLYB200_ROWQ_FP8, Q_INT8 = FLYB200_ROWQ_INT8, Q_MXFP8 = FLYB200_ROWQ_MXFP8 };

struct RowParams {
  void* y;          // codes or values, rows of `width` without gaps
  void* scale;      // fp32 per row, or E8M0 bytes [rows, width / 32]
  void* h;          // norm: x + residual (may be x or residual itself), or null
  const void* x;    // norm [rows, width]; gated [rows, 2 width]
  const void* r;    // norm: residual or null
  const void* w;    // norm: weight
  long long x_stride, r_stride, h_stride;  // in elements
  int rows, width;
  int warps_per_row;
  int w_f32;        // the weight is fp32, whatever x is
  float eps;
};

template <typename T>
constexpr int VEC_OF = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (std::is_same<T, float>::value) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// N = 1: one element; else a 16-byte vector.  Plain loads: the norm may write its sum over what it read.
template <typename T, int N>
struct Raw {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> load_raw(const T* p) {
  Raw<T, N> o;
  if constexpr (N == 1) {
    o.v[0] = *p;
  } else {
    *reinterpret_cast<uint4*>(&o) = *reinterpret_cast<const uint4*>(p);
  }
  return o;
}
template <typename T, int N>
__device__ __forceinline__ void store_raw(T* p, const Raw<T, N>& o) {
  if constexpr (N == 1) {
    *p = o.v[0];
  } else {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&o);
  }
}
template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& o, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_f32(o.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> pack(const float (&v)[N]) {
  Raw<T, N> o;
#pragma unroll
  for (int i = 0; i < N; ++i) o.v[i] = from_f32<T>(v[i]);
  return o;
}
// a + b, rounded once.  The sum of two 16-bit numbers in fp32 and then to 16 bits is the same: either fp32 holds it
// exactly, or the smaller number is less than half a step of the larger one.
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> add_raw(const Raw<T, N>& a, const Raw<T, N>& b) {
  Raw<T, N> o;
  if constexpr (N == 8 && std::is_same<T, __half>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<__half2*>(&o)[i] = __hadd2(reinterpret_cast<const __half2*>(&a)[i], reinterpret_cast<const __half2*>(&b)[i]);
  } else if constexpr (N == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<__nv_bfloat162*>(&o)[i] = __hadd2(reinterpret_cast<const __nv_bfloat162*>(&a)[i], reinterpret_cast<const __nv_bfloat162*>(&b)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = from_f32<T>(to_f32(a.v[i]) + to_f32(b.v[i]));
  }
  return o;
}
// The weights of N channels, of T or fp32.
template <typename T, int N>
__device__ __forceinline__ void load_weight(const RowParams& p, int k, float (&w)[N]) {
  if (!std::is_same<T, float>::value && p.w_f32) {
    const float* q = static_cast<const float*>(p.w) + k;
    if constexpr (N == 1) {
      w[0] = __ldg(q);
    } else {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const float4 t = __ldg(reinterpret_cast<const float4*>(q + i));
        w[i] = t.x, w[i + 1] = t.y, w[i + 2] = t.z, w[i + 3] = t.w;
      }
    }
  } else {
    const T* q = static_cast<const T*>(p.w) + k;
    Raw<T, N> o;
    if constexpr (N == 1) {
      o.v[0] = *q;
    } else {
      *reinterpret_cast<uint4*>(&o) = __ldg(reinterpret_cast<const uint4*>(q));
    }
    unpack(o, w);
  }
}

// Larger magnitude; NaN if one is NaN.
__device__ __forceinline__ float max_abs(float m, float v) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(m), "f"(fabsf(v)));
  return d;
}

// Sum and maximum over the `wpr` warps of a row, the same in all of their threads.  `red`: 2 x 32 words of the block,
// `first`: the row's first warp in the block, `bar`: a named barrier of the row's own.  Fixed order.
template <bool SUM, bool MAX>
__device__ __forceinline__ void row_reduce(float& sum, float& mx, int wpr, int first, int bar, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if constexpr (SUM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if constexpr (MAX) mx = max_abs(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  }
  if (wpr > 1) {
    if (lane == 0) red[warp] = sum, red[32 + warp] = mx;
    named_bar_sync(bar, 32 * wpr);
    if constexpr (SUM) sum = lane < wpr ? red[first + lane] : 0.0f;
    if constexpr (MAX) mx = lane < wpr ? red[32 + first + lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if constexpr (SUM) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if constexpr (MAX) mx = max_abs(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
  }
}

template <int Q>
constexpr float QMAX_OF = Q == Q_INT8 ? 127.0f : 448.0f;

// What turns the values of a row into codes: code = nearest(v * inv), or, where inv would leave the range of fp32, nearest(v / s).
struct RowScale {
  float s;    // what is stored
  float mul;  // qmax / max, of the values as they are passed to encode(), and what its rounding left of it
  float low;
  bool divide;
};
// Values in code units.  int8, where a step is as small against the largest values as against the smallest ones, has them rounded
// once.
template <int Q>
__device__ __forceinline__ float in_units(float v, const RowScale& s) {
  return Q == Q_INT8 ? fmaf(v, s.mul, v * s.low) : v * s.mul;
}
// Scale of a row whose values are `u * f` (f > 0) with max |u| = m: the code of u needs neither f nor s, u * (qmax / m) is the
// same number, rounded once or twice.
template <int Q>
__device__ __forceinline__ RowScale row_scale(float m, float f) {
  RowScale o;
  o.s = __fmul_rn(__fmul_rn(m, f), 1.0f / QMAX_OF<Q>);
  if (o.s == 0.0f) o.s = 1.0f;
  o.divide = false;
  o.mul = m > 0.0f ? __fdiv_rn(QMAX_OF<Q>, m) : 0.0f;
  o.low = fmaf(-o.mul, m, m > 0.0f ? QMAX_OF<Q> : 0.0f) * (o.mul * (1.0f / QMAX_OF<Q>));
  return o;
}
// Whether the short form above holds: finite, and neither the maximum nor the scale near the lower end of fp32.  A row of zeros with an
// infinite f (no eps) is 0 times infinity.
template <int Q>
__device__ __forceinline__ bool row_is_plain(float m, float f) {
  return m == 0.0f ? f < INFINITY : m >= 1e-30f && m < INFINITY && f > 0.0f && m * f >= 1e-30f && m * f < INFINITY;
}

// N codes of values already multiplied into code units; int8: the nearest integer by adding 1.5 * 2^23, whose last bits are
// then the integer in two's complement (|q| <= 127.5).
template <int Q>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  if constexpr (Q == Q_INT8) {
    constexpr float MAGIC = 12582912.0f;
    const uint32_t lo = __byte_perm(__float_as_uint(a + MAGIC), __float_as_uint(b + MAGIC), 0x0040);
    const uint32_t hi = __byte_perm(__float_as_uint(c + MAGIC), __float_as_uint(d + MAGIC), 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
}
template <int Q, int N>
__device__ __forceinline__ void store_codes(uint8_t* y, const float (&q)[N]) {
  if constexpr (N == 1) {
    *y = static_cast<uint8_t>(codes4<Q>(q[0], 0.0f, 0.0f, 0.0f));
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint32_t*>(y) = codes4<Q>(q[0], q[1], q[2], q[3]);
  } else {
    *reinterpret_cast<uint2*>(y) = make_uint2(codes4<Q>(q[0], q[1], q[2], q[3]), codes4<Q>(q[4], q[5], q[6], q[7]));
  }
}
// Codes of a row that row_is_plain refuses: values v in fp32, scrubbed as the per-token quantiser does, divided.
template <int Q, int N>
__device__ __forceinline__ void store_codes_divided(uint8_t* y, const float (&v)[N], float s) {
  float q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = __fdiv_rn(scrub(v[i], QMAX_OF<Q>), s);
    q[i] = fminf(fmaxf(q[i], -QMAX_OF<Q>), QMAX_OF<Q>);
  }
  store_codes<Q, N>(y, q);
}

// MXFP8 block of 32 values held by 32 / N neighbouring lanes: codes and the scale byte, as per_1x32_f8_quant.  All lanes of
// the warp call it.
template <int N>
__device__ __forceinline__ void store_mx(uint8_t* y, uint8_t* scale, int k, bool in, const float (&v)[N]) {
  uint32_t mb = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) mb = max(mb, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = 1; o < 32 / N; o <<= 1) mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, o));
  if (!in) return;
  const float m = mb > 0x7F800000u ? __uint_as_float(mb) : fmaxf(__uint_as_float(mb), 1e-30f);
  const uint32_t e = e8m0_of(__fmul_rn(m, 1.0f / 448.0f));
  if (k % 32 == 0) scale[k / 32] = static_cast<uint8_t>(e);
  float q[N];
  if (e == 0xFFu) {  // the scale is NaN, and so is every code
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = __uint_as_float(0x7FFFFFFFu);
  } else {
    // 2^(127 - e); the least scale byte is that of 1e-30 / 448, so it is a normal number
    const float inv = __uint_as_float(e == 254u ? 0x00400000u : (254u - e) << 23);
    const float s = __uint_as_float(e << 23);
#pragma unroll
    for (int i = 0; i < N; ++i) q[i] = s < 1e-30f ? __fdiv_rn(v[i], 1e-30f) : __fmul_rn(v[i], inv);
  }
  store_codes<Q_MXFP8, N>(y + k, q);
}

// ---- norm ---------------------------------------------------------------------------------------------------------------

// h w f, multiplied in the order that stays in range: h w may be infinite where h f w is not, and a very large f (no eps, small rows)
// may bring back what h w has lost below 2^-126.  Up to this f that is at most 2^-126 of the value.
constexpr float LARGE_F = 16777216.0f;
__device__ __forceinline__ float normed(float h, float w, float f) {
  const float v = h * w;
  return fabsf(v) < INFINITY && f <= LARGE_F ? v * f : h * f * w;
}
// N values from what the thread has read or written before.
template <typename T, int N>
__device__ __forceinline__ void normed_at(const RowParams& p, const T* row, int k, float f, float (&v)[N]) {
  float h[N], w[N];
  unpack(load_raw<T, N>(row + k), h);
  load_weight<T, N>(p, k, w);
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = normed(h[j], w[j], f);
}

// Sum of squares and maximum of |h w| of N elements.
template <bool MAX, int N>
__device__ __forceinline__ void norm_stats(const float (&h)[N], const float (&w)[N], float& sum, float& mx) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sum = fmaf(h[i], h[i], sum);
    if constexpr (MAX) mx = max_abs(mx, h[i] * w[i]);
  }
}

// Single pass: the row's NV vectors per thread stay in registers, all loads of a thread are in flight together.  16384 x 8192 bf16 with
// residual to fp8: 212 us with the sums as they were read and read twice, 185 with h w in fp32 between the passes and packed additions, 170 with
// two vectors a thread in place of four (64 registers and spills); floor 144.
template <typename T, int Q, int NV>
__global__ void __launch_bounds__(1024) rmsnorm_row_kernel(RowParams p) {
  constexpr int N = VEC_OF<T>;
  constexpr bool ROWQ = Q == Q_FP8 || Q == Q_INT8;
  __shared__ float red[64];
  pdl_wait(p.x, p.r, p.w, p.y, p.h, p.scale);
  pdl_trigger();
  const int wpr = p.warps_per_row, tpr = 32 * wpr;
  const int group = threadIdx.x / tpr, tid = threadIdx.x % tpr;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + group;
  if (row >= p.rows) return;
  const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
  const T* rr = static_cast<const T*>(p.r) + row * p.r_stride;
  T* hr = static_cast<T*>(p.h) + row * p.h_stride;
  Raw<T, N> raw[NV], res[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (i * tpr + tid) * N;
    if (k < p.width) {
      raw[i] = load_raw<T, N>(xr + k);
      if (p.r) res[i] = load_raw<T, N>(rr + k);
    }
  }
  float v[NV][N], sum = 0.0f, mx = 0.0f;  // v: h w
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (i * tpr + tid) * N;
    if (k >= p.width) {
#pragma unroll
      for (int j = 0; j < N; ++j) v[i][j] = 0.0f;
      continue;
    }
    if (p.r) {
      raw[i] = add_raw<T, N>(raw[i], res[i]);
      store_raw<T, N>(hr + k, raw[i]);
    }
    float w[N];
    unpack(raw[i], v[i]);
    load_weight<T, N>(p, k, w);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      sum = fmaf(v[i][j], v[i][j], sum);
      v[i][j] *= w[j];
      mx = max_abs(mx, v[i][j]);  // without codes per row, the thread's own
    }
  }
  row_reduce<true, ROWQ>(sum, mx, wpr, group * wpr, 1 + group, red);
  const float f = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(p.width)), p.eps));

  if constexpr (ROWQ) {
    uint8_t* yr = static_cast<uint8_t*>(p.y) + row * p.width;
    float* scale = static_cast<float*>(p.scale) + row;
    if (row_is_plain<Q>(mx, f)) {
      const RowScale s = row_scale<Q>(mx, f);
      if (tid == 0) *scale = s.s;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (i * tpr + tid) * N;
        if (k >= p.width) break;
#pragma unroll
        for (int j = 0; j < N; ++j) v[i][j] = in_units<Q>(v[i][j], s);
        store_codes<Q, N>(yr + k, v[i]);
      }
    } else {  // the same branch in all threads of the row
      const T* again = p.r ? hr : xr;
      float far[N], amax = 0.0f, none = 0.0f;
#pragma unroll 1
      for (int k = tid * N; k < p.width; k += tpr * N) {
        normed_at(p, again, k, f, far);
#pragma unroll
        for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(scrub(far[j], QMAX_OF<Q>)));
      }
      if (wpr > 1) named_bar_sync(1 + group, tpr);  // `red` is read above
      row_reduce<false, true>(none, amax, wpr, group * wpr, 1 + group, red);
      float s = __fmul_rn(amax, 1.0f / QMAX_OF<Q>);
      if (s == 0.0f) s = 1.0f;
      if (tid == 0) *scale = s;
#pragma unroll 1
      for (int k = tid * N; k < p.width; k += tpr * N) {
        normed_at(p, again, k, f, far);
        store_codes_divided<Q, N>(yr + k, far, s);
      }
    }
  } else {
    auto store = [&](int k, const float (&u)[N]) {
      const bool in = k < p.width;
      if constexpr (Q == Q_MXFP8) {
        store_mx<N>(static_cast<uint8_t*>(p.y) + row * p.width, static_cast<uint8_t*>(p.scale) + row * (p.width / 32), k, in, u);
      } else if (in) {
        store_raw<T, N>(static_cast<T*>(p.y) + row * p.width + k, pack<T, N>(u));
      }
    };
    if (__all_sync(0xffffffffu, mx < INFINITY && f <= LARGE_F)) {  // a warp's lanes meet in store_mx
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[i][j] *= f;
        store((i * tpr + tid) * N, v[i]);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < NV; ++i) {
        const int k = (i * tpr + tid) * N;
        float u[N] = {};
        if (k < p.width) normed_at(p, p.r ? hr : xr, k, f, u);
        store(k, u);
      }
    }
  }
}

// Any row: a block per row in two or three passes, the later ones over what the same thread has read or written before.
// N = 1 where a size, a stride or an address is not a multiple of 16 bytes.
template <typename T, int Q, int N>
__global__ void __launch_bounds__(512) rmsnorm_any_kernel(RowParams p) {
  constexpr bool ROWQ = Q == Q_FP8 || Q == Q_INT8;
  __shared__ float red[64];
  pdl_wait(p.x, p.r, p.w, p.y, p.h, p.scale);
  pdl_trigger();
  const int wpr = blockDim.x / 32, step = blockDim.x * N;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
    if (p.r) {
      const T* rr = static_cast<const T*>(p.r) + row * p.r_stride;
      T* hr = static_cast<T*>(p.h) + row * p.h_stride;
      for (int k = threadIdx.x * N; k < p.width; k += step) {
        float a[N], b[N];
        unpack(load_raw<T, N>(xr + k), a);
        unpack(load_raw<T, N>(rr + k), b);
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] += b[j];
        store_raw<T, N>(hr + k, pack<T, N>(a));
      }
      xr = hr;  // every thread reads back what it wrote itself
    }
    float sum = 0.0f, mx = 0.0f;
    for (int k = threadIdx.x * N; k < p.width; k += step) {
      float h[N], w[N];
      unpack(load_raw<T, N>(xr + k), h);
      if constexpr (ROWQ) load_weight<T, N>(p, k, w);
      norm_stats<ROWQ, N>(h, w, sum, mx);
    }
    row_reduce<true, ROWQ>(sum, mx, wpr, 0, 1, red);
    __syncthreads();  // `red` is used again
    const float f = __frsqrt_rn(__fadd_rn(__fdiv_rn(sum, static_cast<float>(p.width)), p.eps));
    RowScale s = {1.0f, 0.0f, 0.0f, false};
    if constexpr (ROWQ) {
      if (row_is_plain<Q>(mx, f)) {
        s = row_scale<Q>(mx, f);
      } else {
        float amax = 0.0f, none = 0.0f;
        for (int k = threadIdx.x * N; k < p.width; k += step) {
          float v[N];
          normed_at(p, xr, k, f, v);
#pragma unroll
          for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(scrub(v[j], QMAX_OF<Q>)));
        }
        row_reduce<false, true>(none, amax, wpr, 0, 1, red);
        __syncthreads();
        s.s = __fmul_rn(amax, 1.0f / QMAX_OF<Q>);
        if (s.s == 0.0f) s.s = 1.0f;
        s.divide = true;
      }
      if (threadIdx.x == 0) static_cast<float*>(p.scale)[row] = s.s;
    }
    for (int k0 = 0; k0 < p.width; k0 += step) {  // all lanes stay for the shuffles of store_mx
      const int k = k0 + threadIdx.x * N;
      const bool in = k < p.width;
      float h[N] = {}, w[N];
      if (in) {
        unpack(load_raw<T, N>(xr + k), h);
        load_weight<T, N>(p, k, w);
#pragma unroll
        for (int j = 0; j < N; ++j) h[j] = ROWQ && !s.divide ? in_units<Q>(h[j] * w[j], s) : normed(h[j], w[j], f);
      }
      if constexpr (ROWQ) {
        uint8_t* y = static_cast<uint8_t*>(p.y) + row * p.width + k;
        if (in) s.divide ? store_codes_divided<Q, N>(y, h, s.s) : store_codes<Q, N>(y, h);
      } else if constexpr (Q == Q_MXFP8) {
        store_mx<N>(static_cast<uint8_t*>(p.y) + row * p.width, static_cast<uint8_t*>(p.scale) + row * (p.width / 32), k, in, h);
      } else if (in) {
        store_raw<T, N>(static_cast<T*>(p.y) + row * p.width + k, pack<T, N>(h));
      }
    }
  }
}

// ---- gated activation ---------------------------------------------------------------------------------------------------

// g / (1 + exp(-g)) * u.  exp(-x) = 2^t (1 + lo) with t = -x log2(e) rounded and lo = -x - t ln 2, what the roundings of the product and of
// both constants left; a reciprocal with one step of Newton's method, which makes it good to its last place.
__device__ __forceinline__ float exp_lo(float x, float t) {
  constexpr double LN2 = 0.69314718055994530942;
  constexpr float HIGH = static_cast<float>(LN2), LOW = static_cast<float>(LN2 - static_cast<double>(HIGH));
  return fmaf(t, -LOW, fmaf(t, -HIGH, -x));
}
__device__ __forceinline__ float reciprocal(float d) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return fmaf(fmaf(-d, r, 1.0f), r, r);
}
constexpr float GATE_NEAR = 87.0f;
// Up to |g| = 87, where neither 1 + exp(-g) nor its reciprocal leaves the range of normal numbers; NaN.
__device__ __forceinline__ float gated_near(float g, float u) {
  const float t = g * -1.44269504f;
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return g * reciprocal(1.0f + fmaf(e, exp_lo(g, t), e)) * u;
}
// Any g, for g < 0 as g exp(g) / (1 + exp(g)) * u: e = exp(-|g|) keeps the places that fp32 has below 2^-126 and is 0 beyond 104, while
// u may be large.  -Inf times 0 is NaN.
__device__ __noinline__ float gated_far(float g, float u) {
  const float x = fminf(fabsf(g), 105.0f), t = x * -1.44269504f;
  float e;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = fmaf(e, exp_lo(x, t), e);
  return g * (g < 0.0f ? e : 1.0f) * reciprocal(1.0f + e) * u;
}

// All take the form for near gates throughout, and the other one again where one of a thread's gates is far.  That one throughout costs
// more: 8192 x 28672 bf16 to fp8 268 us in place of 231.
template <typename T, int N>
__device__ __forceinline__ void gated_at(const T* xr, int width, int k, float (&v)[N]) {
  float g[N], u[N], top = 0.0f;
  unpack(load_raw<T, N>(xr + k), g);
  unpack(load_raw<T, N>(xr + width + k), u);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    top = fmaxf(top, fabsf(g[j]));
    v[j] = gated_near(g[j], u[j]);
  }
  if (top > GATE_NEAR) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (fabsf(g[j]) > GATE_NEAR) v[j] = gated_far(g[j], u[j]);
  }
}

// Of a row in registers, read once more: the values and their maximum.
template <typename T, int N, int NV>
__device__ __forceinline__ void far_gates(const T* xr, int width, int first, int step, float (&v)[NV][N], float& mx) {
  mx = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = first + i * step;
    if (k >= width) break;
    float g[N], u[N];
    unpack(load_raw<T, N>(xr + k), g);
    unpack(load_raw<T, N>(xr + width + k), u);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (fabsf(g[j]) > GATE_NEAR) v[i][j] = gated_far(g[j], u[j]);
      mx = max_abs(mx, v[i][j]);
    }
  }
}

// Per-row scale: the row's fp32 values stay in registers between the maximum and the conversion.
template <typename T, int Q, int NV>
__global__ void __launch_bounds__(1024) silu_row_kernel(RowParams p) {
  constexpr int N = VEC_OF<T>;
  __shared__ float red[64];
  pdl_wait(p.x, p.y, p.scale);
  pdl_trigger();
  const int wpr = p.warps_per_row, tpr = 32 * wpr;
  const int group = threadIdx.x / tpr, tid = threadIdx.x % tpr;
  const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x / tpr) + group;
  if (row >= p.rows) return;
  const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
  Raw<T, N> g[NV], u[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (i * tpr + tid) * N;
    if (k < p.width) {
      g[i] = load_raw<T, N>(xr + k);
      u[i] = load_raw<T, N>(xr + p.width + k);
    }
  }
  float v[NV][N], mx = 0.0f, top = 0.0f, none = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * tpr + tid) * N >= p.width) break;
    float b[N];
    unpack(g[i], v[i]);
    unpack(u[i], b);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      top = fmaxf(top, fabsf(v[i][j]));
      v[i][j] = gated_near(v[i][j], b[j]);
      mx = max_abs(mx, v[i][j]);
    }
  }
  if (top > GATE_NEAR) far_gates<T, N, NV>(xr, p.width, tid * N, tpr * N, v, mx);
  row_reduce<false, true>(none, mx, wpr, group * wpr, 1 + group, red);
  uint8_t* yr = static_cast<uint8_t*>(p.y) + row * p.width;
  float* scale = static_cast<float*>(p.scale) + row;
  if (row_is_plain<Q>(mx, 1.0f)) {
    const RowScale s = row_scale<Q>(mx, 1.0f);
    if (tid == 0) *scale = s.s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * tpr + tid) * N;
      if (k >= p.width) break;
#pragma unroll
      for (int j = 0; j < N; ++j) v[i][j] = in_units<Q>(v[i][j], s);
      store_codes<Q, N>(yr + k, v[i]);
    }
  } else {
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * tpr + tid) * N >= p.width) break;
#pragma unroll
      for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(scrub(v[i][j], QMAX_OF<Q>)));
    }
    if (wpr > 1) named_bar_sync(1 + group, tpr);  // `red` is read above
    row_reduce<false, true>(none, amax, wpr, group * wpr, 1 + group, red);
    float s = __fmul_rn(amax, 1.0f / QMAX_OF<Q>);
    if (s == 0.0f) s = 1.0f;
    if (tid == 0) *scale = s;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int k = (i * tpr + tid) * N;
      if (k >= p.width) break;
      store_codes_divided<Q, N>(yr + k, v[i], s);
    }
  }
}

// Per-row scale of wide rows, many of them: a row in registers is more than half of an SM's, so there is no second block whose loads
// could go on while this one reduces, converts and stores.  Here the loads run ahead of all that, over the ends of rows: every thread copies its own
// vectors into a ring in shared memory and reads them back itself, so that nothing but its own wait stands between the two - no
// barrier, no flag, no other thread.  us, 8192 x 28672 bf16 to fp8: 296 with the kernel above, 231 to 236 here; 250 to 262 with a warp of its own that
// filled the ring by bulk copies (floor 180).
constexpr int RING_THREADS = 512, RING_WARPS = RING_THREADS / 32;
constexpr int RING_CHUNK = 16 * RING_THREADS;  // bytes of gate values, and as many of up values: a vector of each per thread
constexpr int RING_SLOTS = 13;
constexpr int RING_BYTES = RING_SLOTS * 2 * RING_CHUNK;

__device__ __forceinline__ void copy16_once(uint32_t dst, const void* src, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}

template <typename T, int Q, int NV>
__global__ void __launch_bounds__(RING_THREADS, 1) silu_ring_kernel(RowParams p) {
  constexpr int N = VEC_OF<T>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float reds[3][64];  // of even rows, of odd rows, of the second maximum
  const int tid = threadIdx.x;
  const uint8_t* mine = smem + tid * 16;
  const uint32_t base = smem_u32(mine);
  pdl_wait(p.x, p.y, p.scale);
  pdl_trigger();
  const uint64_t once = l2_policy_evict_first();

  long long ahead_row = blockIdx.x;
  int ahead_k = tid * N, ahead_slot = 0;
  auto copy_next = [&]() {  // one group, empty behind the last row and for threads behind a row's end
    if (ahead_row < p.rows) {
      if (ahead_k < p.width) {
        const T* from = static_cast<const T*>(p.x) + ahead_row * p.x_stride + ahead_k;
        const uint32_t at = base + ahead_slot * 2 * RING_CHUNK;
        copy16_once(at, from, once);
        copy16_once(at + RING_CHUNK, from + p.width, once);
      }
      ahead_k += RING_THREADS * N;
      if (ahead_k >= NV * RING_THREADS * N) {
        ahead_k = tid * N;
        ahead_row += gridDim.x;
      }
    }
    if (++ahead_slot == RING_SLOTS) ahead_slot = 0;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < RING_SLOTS - 1; ++i) copy_next();

  int slot = 0, odd = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    float v[NV][N], mx = 0.0f, top = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(RING_SLOTS - 2) : "memory");  // the oldest one is here
      if ((i * RING_THREADS + tid) * N < p.width) {
        float u[N];
        const uint8_t* at = mine + slot * 2 * RING_CHUNK;
        unpack(load_raw<T, N>(reinterpret_cast<const T*>(at)), v[i]);
        unpack(load_raw<T, N>(reinterpret_cast<const T*>(at + RING_CHUNK)), u);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          top = fmaxf(top, fabsf(v[i][j]));
          v[i][j] = gated_near(v[i][j], u[j]);
          mx = max_abs(mx, v[i][j]);
        }
      }
      if (++slot == RING_SLOTS) slot = 0;
      copy_next();  // over the slot that was read one time earlier
    }
    if (top > GATE_NEAR) far_gates<T, N, NV>(static_cast<const T*>(p.x) + row * p.x_stride, p.width, tid * N, RING_THREADS * N, v, mx);
    row_reduce<false, true>(none, mx, RING_WARPS, 0, 1, reds[odd]);  // nobody writes over it before all are at the next row's barrier
    odd ^= 1;
    uint8_t* yr = static_cast<uint8_t*>(p.y) + row * p.width;
    float* scale = static_cast<float*>(p.scale) + row;
    if (row_is_plain<Q>(mx, 1.0f)) {
      const RowScale s = row_scale<Q>(mx, 1.0f);
      if (tid == 0) *scale = s.s;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (i * RING_THREADS + tid) * N;
        if (k >= p.width) break;
#pragma unroll
        for (int j = 0; j < N; ++j) v[i][j] = in_units<Q>(v[i][j], s);
        store_codes<Q, N>(yr + k, v[i]);
      }
    } else {
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if ((i * RING_THREADS + tid) * N >= p.width) break;
#pragma unroll
        for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(scrub(v[i][j], QMAX_OF<Q>)));
      }
      row_reduce<false, true>(none, amax, RING_WARPS, 0, 1, reds[2]);
      float s = __fmul_rn(amax, 1.0f / QMAX_OF<Q>);
      if (s == 0.0f) s = 1.0f;
      if (tid == 0) *scale = s;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int k = (i * RING_THREADS + tid) * N;
        if (k >= p.width) break;
        store_codes_divided<Q, N>(yr + k, v[i], s);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Per-row scale of any row: two or three passes that compute the values again.
template <typename T, int Q, int N>
__global__ void __launch_bounds__(512) silu_any_kernel(RowParams p) {
  __shared__ float red[64];
  pdl_wait(p.x, p.y, p.scale);
  pdl_trigger();
  const int wpr = blockDim.x / 32, step = blockDim.x * N;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* xr = static_cast<const T*>(p.x) + row * p.x_stride;
    float v[N], mx = 0.0f, none = 0.0f;
    for (int k = threadIdx.x * N; k < p.width; k += step) {
      gated_at<T, N>(xr, p.width, k, v);
#pragma unroll
      for (int j = 0; j < N; ++j) mx = max_abs(mx, v[j]);
    }
    row_reduce<false, true>(none, mx, wpr, 0, 1, red);
    __syncthreads();
    RowScale s = {1.0f, 0.0f, 0.0f, false};
    if (row_is_plain<Q>(mx, 1.0f)) {
      s = row_scale<Q>(mx, 1.0f);
    } else {
      float amax = 0.0f;
      for (int k = threadIdx.x * N; k < p.width; k += step) {
        gated_at<T, N>(xr, p.width, k, v);
#pragma unroll
        for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(scrub(v[j], QMAX_OF<Q>)));
      }
      row_reduce<false, true>(none, amax, wpr, 0, 1, red);
      __syncthreads();
      s.s = __fmul_rn(amax, 1.0f / QMAX_OF<Q>);
      if (s.s == 0.0f) s.s = 1.0f;
      s.divide = true;
    }
    if (threadIdx.x == 0) static_cast<float*>(p.scale)[row] = s.s;
    uint8_t* yr = static_cast<uint8_t*>(p.y) + row * p.width;
    for (int k = threadIdx.x * N; k < p.width; k += step) {
      gated_at<T, N>(xr, p.width, k, v);
      if (s.divide) {
        store_codes_divided<Q, N>(yr + k, v, s.s);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = in_units<Q>(v[j], s);
        store_codes<Q, N>(yr + k, v);
      }
    }
  }
}

// No row statistics (MXFP8 blocks, or values of x's type): a thread takes N values wherever they are.  Eight blocks an SM: 8192 x 28672 bf16 216 us
// (six blocks 230), to MXFP8 300 (320).
template <typename T, int Q, int N>
__global__ void __launch_bounds__(256, 8) silu_flat_kernel(RowParams p) {
  pdl_wait(p.x, p.y, p.scale);
  pdl_trigger();
  const int per_row = p.width / N;
  const int parts = (per_row + 255) / 256;  // blocks of a row
  const long long row = blockIdx.x / static_cast<unsigned>(parts);
  const int k = ((blockIdx.x % static_cast<unsigned>(parts)) * 256 + threadIdx.x) * N;
  const bool in = k < p.width;
  float v[N] = {};
  if (in) gated_at<T, N>(static_cast<const T*>(p.x) + row * p.x_stride, p.width, k, v);
  if constexpr (Q == Q_MXFP8) {
    store_mx<N>(static_cast<uint8_t*>(p.y) + row * p.width, static_cast<uint8_t*>(p.scale) + row * (p.width / 32), k, in, v);
  } else if (in) {
    store_raw<T, N>(static_cast<T*>(p.y) + row * p.width + k, pack<T, N>(v));
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------

#define CUDA_TRY(expr)                                                  \
  do {                                                                  \
    cudaError_t _e = (expr);                                            \
    if (_e != cudaSuccess) return host::record_cuda_error(_e, #expr);   \
  } while (0)

constexpr int SMS = 148;  // that the shapes of launches are meant for

bool multiple(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Warps that share a row of `vecs` vectors, at most `most_vecs` per thread: as few as that allows, more while the rows
// alone would leave the SMs with less than two blocks of eight warps each.  0: the row does not fit.
int warps_per_row(int rows, int vecs, int most_vecs, int most_warps) {
  int wpr = 1;
  while (wpr < most_warps && vecs > 32 * wpr * most_vecs) wpr *= 2;
  if (vecs > 32 * wpr * most_vecs) return 0;
  while (wpr < most_warps && vecs > 32 * wpr && static_cast<long long>(rows) * wpr < 2LL * SMS * 8) wpr *= 2;
  return wpr;
}
int threads_of(int wpr) { return 32 * (wpr < 8 ? 8 : wpr); }
unsigned blocks_of(int rows, int wpr) {
  const int per = wpr < 8 ? 8 / wpr : 1;
  return static_cast<unsigned>((static_cast<long long>(rows) + per - 1) / per);
}
constexpr int ANY_BLOCKS = SMS * 4;

template <typename T, int Q>
cudaError_t launch_norm(RowParams p, bool vectors, cudaStream_t s) {
  constexpr int N = VEC_OF<T>;
  const int vecs = p.width / N;
  int wpr = vectors ? warps_per_row(p.rows, vecs, N == 8 ? 2 : 4, 32) : 0;
  if (vectors && !wpr) wpr = warps_per_row(p.rows, vecs, 4, 32);
  if (!wpr) {
    const dim3 grid(p.rows < ANY_BLOCKS ? p.rows : ANY_BLOCKS);
    return vectors ? host::launch_dependent(rmsnorm_any_kernel<T, Q, N>, grid, 512, 0, s, p)
                   : host::launch_dependent(rmsnorm_any_kernel<T, Q, 1>, grid, 512, 0, s, p);
  }
  const int nv = (vecs + 32 * wpr - 1) / (32 * wpr);
  p.warps_per_row = wpr;
  const dim3 grid(blocks_of(p.rows, wpr));
  const int t = threads_of(wpr);
  return nv == 1   ? host::launch_dependent(rmsnorm_row_kernel<T, Q, 1>, grid, t, 0, s, p)
         : nv == 2 ? host::launch_dependent(rmsnorm_row_kernel<T, Q, 2>, grid, t, 0, s, p)
                   : host::launch_dependent(rmsnorm_row_kernel<T, Q, 4>, grid, t, 0, s, p);
}

// Vectors of a row from which on the ring is taken.
constexpr int RING_FROM = 2 * RING_THREADS;

template <typename T, int Q, int NV>
cudaError_t launch_silu_ring(RowParams p, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load(std::memory_order_acquire) & bit)) {
    if (cudaError_t e = cudaFuncSetAttribute(silu_ring_kernel<T, Q, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES)) return e;
    done.fetch_or(bit, std::memory_order_release);
  }
  int sms = 0;
  if (host::sm_count(&sms)) return cudaErrorInvalidDevice;
  return host::launch_dependent(silu_ring_kernel<T, Q, NV>, dim3(p.rows < sms ? p.rows : sms), RING_THREADS, RING_BYTES, s, p);
}

template <typename T, int Q>
cudaError_t launch_silu(RowParams p, bool vectors, cudaStream_t s) {
  constexpr int N = VEC_OF<T>;
  if constexpr (Q == Q_NONE || Q == Q_MXFP8) {
    const int per_row = vectors ? p.width / N : p.width;
    const long long blocks = static_cast<long long>((per_row + 255) / 256) * p.rows;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
    return vectors ? host::launch_dependent(silu_flat_kernel<T, Q, N>, dim3(static_cast<unsigned>(blocks)), 256, 0, s, p)
                   : host::launch_dependent(silu_flat_kernel<T, Q, 1>, dim3(static_cast<unsigned>(blocks)), 256, 0, s, p);
  } else {
    const int vecs = p.width / N;
    if (vectors && vecs > RING_FROM && vecs <= 8 * RING_THREADS && p.rows > SMS) {
      const int nv = (vecs + RING_THREADS - 1) / RING_THREADS;
      return nv <= 3   ? launch_silu_ring<T, Q, 3>(p, s)
             : nv == 4 ? launch_silu_ring<T, Q, 4>(p, s)
             : nv == 5 ? launch_silu_ring<T, Q, 5>(p, s)
             : nv == 6 ? launch_silu_ring<T, Q, 6>(p, s)
             : nv == 7 ? launch_silu_ring<T, Q, 7>(p, s)
                       : launch_silu_ring<T, Q, 8>(p, s);
    }
    const int wpr = vectors ? warps_per_row(p.rows, vecs, 4, 32) : 0;
    if (!wpr) {
      const dim3 grid(p.rows < ANY_BLOCKS ? p.rows : ANY_BLOCKS);
      return vectors ? host::launch_dependent(silu_any_kernel<T, Q, N>, grid, 512, 0, s, p)
                     : host::launch_dependent(silu_any_kernel<T, Q, 1>, grid, 512, 0, s, p);
    }
    const int nv = (vecs + 32 * wpr - 1) / (32 * wpr);
    p.warps_per_row = wpr;
    const dim3 grid(blocks_of(p.rows, wpr));
    const int t = threads_of(wpr);
    return nv == 1   ? host::launch_dependent(silu_row_kernel<T, Q, 1>, grid, t, 0, s, p)
           : nv == 2 ? host::launch_dependent(silu_row_kernel<T, Q, 2>, grid, t, 0, s, p)
                     : host::launch_dependent(silu_row_kernel<T, Q, 4>, grid, t, 0, s, p);
  }
}

template <typename T, bool NORM>
cudaError_t launch_quant(const RowParams& p, int quant, bool vectors, cudaStream_t s) {
  switch (quant) {
    case Q_NONE: return NORM ? launch_norm<T, Q_NONE>(p, vectors, s) : launch_silu<T, Q_NONE>(p, vectors, s);
    case Q_FP8: return NORM ? launch_norm<T, Q_FP8>(p, vectors, s) : launch_silu<T, Q_FP8>(p, vectors, s);
    case Q_INT8: return NORM ? launch_norm<T, Q_INT8>(p, vectors, s) : launch_silu<T, Q_INT8>(p, vectors, s);
    default: return NORM ? launch_norm<T, Q_MXFP8>(p, vectors, s) : launch_silu<T, Q_MXFP8>(p, vectors, s);
  }
}
template <bool NORM>
cudaError_t launch_rows(const RowParams& p, int x_dtype, int quant, bool vectors, cudaStream_t s) {
  return x_dtype == QX_F32   ? launch_quant<float, NORM>(p, quant, vectors, s)
         : x_dtype == QX_F16 ? launch_quant<__half, NORM>(p, quant, vectors, s)
                             : launch_quant<__nv_bfloat16, NORM>(p, quant, vectors, s);
}

}  // namespace

extern "C" {

int flyb200_rmsnorm_quant(void* y, void* scale, void* residual_out, const void* x, const void* residual, const void* weight,
                          int rows, int K, long long x_stride, long long residual_stride, long long residual_out_stride,
                          float eps, int x_dtype, int weight_f32, int quant, void* stream) {
  if (!y || !x || !weight || rows < 0 || K <= 0 || K > 0x3fffffff || x_dtype < QX_F32 || x_dtype > QX_BF16) return FLYB200_E_BAD_ARG;
  if (quant < Q_NONE || quant > Q_MXFP8 || (quant != Q_NONE) != (scale != nullptr)) return FLYB200_E_BAD_ARG;
  if ((residual != nullptr) != (residual_out != nullptr) || !(eps >= 0.0f)) return FLYB200_E_BAD_ARG;
  if (x_stride < K || (residual && (residual_stride < K || residual_out_stride < K))) return FLYB200_E_BAD_ARG;
  if (quant == Q_MXFP8 && K % 32 != 0) return FLYB200_E_UNSUPPORTED;
  const int e = x_dtype == QX_F32 ? 4 : 2, n = 16 / e;
  if (!multiple(x, e) || !multiple(residual, e) || !multiple(residual_out, e) || !multiple(weight, weight_f32 ? 4 : e) ||
      !multiple(y, quant == Q_NONE ? e : 1) || (quant != Q_MXFP8 && !multiple(scale, 4)))
    return FLYB200_E_BAD_ALIGN;
  if (rows == 0) return FLYB200_OK;
  bool vectors = K % n == 0 && x_stride % n == 0 && multiple(x, 16) && multiple(weight, 16) && multiple(y, quant == Q_NONE ? 16 : n);
  if (residual)
    vectors = vectors && residual_stride % n == 0 && residual_out_stride % n == 0 && multiple(residual, 16) && multiple(residual_out, 16);
  const RowParams p = {y, scale, residual_out, x, residual, weight, x_stride, residual_stride, residual_out_stride, rows, K, 0, weight_f32 ? 1 : 0, eps};
  CUDA_TRY(launch_rows<true>(p, x_dtype, quant, vectors, static_cast<cudaStream_t>(stream)));
  return FLYB200_OK;
}

int flyb200_silu_mul_quant(void* y, void* scale, const void* x, int rows, int inter, long long x_stride, int x_dtype, int quant,
                           void* stream) {
  if (!y || !x || rows < 0 || inter <= 0 || inter > 0x3fffffff || x_dtype < QX_F32 || x_dtype > QX_BF16) return FLYB200_E_BAD_ARG;
  if (quant < Q_NONE || quant > Q_MXFP8 || (quant != Q_NONE) != (scale != nullptr) || x_stride < 2ll * inter) return FLYB200_E_BAD_ARG;
  if (quant == Q_MXFP8 && inter % 32 != 0) return FLYB200_E_UNSUPPORTED;
  const int e = x_dtype == QX_F32 ? 4 : 2, n = 16 / e;
  if (!multiple(x, e) || !multiple(y, quant == Q_NONE ? e : 1) || (quant != Q_MXFP8 && !multiple(scale, 4))) return FLYB200_E_BAD_ALIGN;
  if (rows == 0) return FLYB200_OK;
  const bool vectors = inter % n == 0 && x_stride % n == 0 && multiple(x, 16) && multiple(y, quant == Q_NONE ? 16 : n);
  const RowParams p = {y, scale, nullptr, x, nullptr, nullptr, x_stride, 0, 0, rows, inter, 0, 0, 0.0f};
  if (quant == Q_NONE || quant == Q_MXFP8) {
    const long long blocks = ((vectors ? inter / n : inter) + 255ll) / 256 * rows;
    if (blocks > 0x7fffffffll) return FLYB200_E_UNSUPPORTED;
  }
  CUDA_TRY(launch_rows<false>(p, x_dtype, quant, vectors, static_cast<cudaStream_t>(stream)));
  return FLYB200_OK;
}

}  // extern "C"

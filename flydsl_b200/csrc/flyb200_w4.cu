// libflyb200: products of few tokens on 4-bit weights with a scale (and zero point) per group of inputs
// (flyb200_gemv_w4a16 in include/flyb200.h).
//
//   c[m, n] = epilogue(sum_g scale[n, g] * sum_{k in g} (q[n, k] - z[n, g]) * a[m, k])
//
// Bound: the weight stream, N K / 2 bytes.  The multiply is the warp-level tensor instruction (16 weight rows x 8 tokens x 16
// inputs, fp32 sums) on codes that stay in registers from the load to the multiply: a product of up to 64 tokens on
// 4-bit codes has no operand that a shared-memory or tensor-memory instruction could take as it is.
// A code becomes a 16-bit number by putting it into the mantissa of 128 (bf16) or 1024 (fp16) and subtracting that
// plus the zero point: two instructions for two codes, and exact.  The scale multiplies the fp32 sum of its group, so no
// weight is rounded.
#include "../../include/flyb200.h"
#include "host_common.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

using namespace flyb200;

namespace {

constexpr int WARPS = 8;
constexpr int CHUNK = 128;  // inputs that a warp takes at a time: 64 bytes of a row of codes

struct W4Params {
  void* c;
  const void* a;
  const uint8_t* q;
  const void* scale;
  const uint8_t* zero;
  const void* bias;
  int M, N, K, epilogue;
};

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  static constexpr uint32_t MAGIC = 0x43004300u;  // 128, 128: the last place of the mantissa is 1
  __device__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static float value(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Pair<__half> {
  static constexpr uint32_t MAGIC = 0x64006400u;  // 1024, 1024
  __device__ static uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ static float value(__half v) { return __half2float(v); }
  __device__ static __half round(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ float activation(float v, int epi) {
  if (epi == FLYB200_EPI_BIAS_RELU) return fmaxf(v, 0.0f);
  if (epi == FLYB200_EPI_BIAS_SILU) return v / (1.0f + expf(-v));
  if (epi == FLYB200_EPI_BIAS_GELU) {  // the tanh form, as the other products'
    const float y = 0.7978845608f * (v + 0.044715f * (v * v * v));
    const float e = expf(-2.0f * fabsf(y));
    return 0.5f * v * ((y > 0.0f ? 2.0f : 2.0f * e) / (1.0f + e));
  }
  return v;
}

// A block takes 16 MT rows of weights and 8 NT tokens; its warps take chunks of the inputs in turn, so that neighbouring warps
// read neighbouring bytes of a row, and their sums are added up in a fixed order at the end.
//
// Inputs in an instruction: lane (g, c) holds rows g and g + 8 of the weights and token g, and of every group the inputs
// [c G / 4, (c + 1) G / 4), that is one contiguous piece of a row of codes.  Word i of it (8 codes) feeds two instructions;
// which of the 16 input slots a code takes does not matter as long as the activations take the same one: codes k and k + 4 of
// a word share a register, so the activations k and k + 4 do.
template <typename T, int G, int MT, int NT>
__global__ void __launch_bounds__(32 * WARPS) gemv_w4_kernel(W4Params p) {
  constexpr int GROUPS = CHUNK / G;  // of a chunk
  constexpr int WORDS = G / 32;      // words of a lane per row and group
  constexpr int R = 16 * MT, TOK = 8 * NT, PITCH = R + 4;
  __shared__ float red[WARPS * TOK * PITCH];
  pdl_wait(p.c, p.a, p.q, p.scale, p.zero, p.bias);
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * R, m0 = blockIdx.y * TOK;
  const size_t row_bytes = p.K / 2;
  const int n_groups = p.K / G;
  const T* scales = static_cast<const T*>(p.scale);

  float acc[MT][NT][4] = {};
  for (int k0 = warp * CHUNK; k0 < p.K; k0 += WARPS * CHUNK) {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      const int kg = k0 + j * G;
      if (kg >= p.K) break;
      uint32_t x[NT][WORDS][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int m = m0 + 8 * t + g;
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.a) + static_cast<size_t>(m) * p.K + kg + c * (G / 4));
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          const uint4 v = m < p.M ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
          x[t][i][0] = __byte_perm(v.x, v.z, 0x5410), x[t][i][1] = __byte_perm(v.x, v.z, 0x7632);
          x[t][i][2] = __byte_perm(v.y, v.w, 0x5410), x[t][i][3] = __byte_perm(v.y, v.w, 0x7632);
        }
      }
#pragma unroll
      for (int r = 0; r < MT; ++r) {
        uint32_t w[2][WORDS], offset[2];
        float s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int n = n0 + 16 * r + 8 * h + g;
          const bool in = n < p.N;
          const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + static_cast<size_t>(n) * row_bytes + kg / 2 + c * (G / 8));
#pragma unroll
          for (int i = 0; i < WORDS; ++i) w[h][i] = 0u;
          s[h] = 0.0f;
          offset[h] = Pair<T>::MAGIC;
          if (in) {
            if constexpr (WORDS == 4) {
              const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
              w[h][0] = v.x, w[h][1] = v.y, w[h][2] = v.z, w[h][3] = v.w;
            } else if constexpr (WORDS == 2) {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
              w[h][0] = v.x, w[h][1] = v.y;
            } else {
              w[h][0] = __ldg(src);
            }
            const size_t at = static_cast<size_t>(n) * n_groups + kg / G;
            s[h] = Pair<T>::value(scales[at]);
            offset[h] += 0x10001u * (p.zero ? static_cast<uint32_t>(p.zero[at]) & 15u : 8u);
          }
        }
        float sum[NT][4] = {};
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
          uint32_t d[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int b = 0; b < 4; ++b) d[h][b] = Pair<T>::sub(((w[h][i] >> (4 * b)) & 0x000F000Fu) | Pair<T>::MAGIC, offset[h]);
#pragma unroll
          for (int b = 0; b < 4; b += 2) {
            const uint32_t frag[4] = {d[0][b], d[1][b], d[0][b + 1], d[1][b + 1]};
#pragma unroll
            for (int t = 0; t < NT; ++t) Pair<T>::mma(sum[t], frag, x[t][i][b], x[t][i][b + 1]);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][t][e] = fmaf(s[e >> 1], sum[t][e], acc[r][t][e]);
      }
    }
  }

  float* mine = red + warp * TOK * PITCH;
#pragma unroll
  for (int r = 0; r < MT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(8 * t + 2 * c + (e & 1)) * PITCH + 16 * r + 8 * (e >> 1) + g] = acc[r][t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < R * TOK; i += 32 * WARPS) {
    const int m = i / R, n = i % R;
    if (m0 + m >= p.M || n0 + n >= p.N) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += red[w * TOK * PITCH + m * PITCH + n];
    if (p.epilogue != FLYB200_EPI_NONE) v = activation(v + Pair<T>::value(static_cast<const T*>(p.bias)[n0 + n]), p.epilogue);
    static_cast<T*>(p.c)[static_cast<size_t>(m0 + m) * p.N + n0 + n] = Pair<T>::round(v);
  }
}

#define CUDA_TRY(expr)                                                  \
  do {                                                                  \
    cudaError_t _e = (expr);                                            \
    if (_e != cudaSuccess) return host::record_cuda_error(_e, #expr);   \
  } while (0)

template <typename T, int G, int MT, int NT>
cudaError_t launch(const W4Params& p, cudaStream_t s) {
  const dim3 grid((p.N + 16 * MT - 1) / (16 * MT), (p.M + 8 * NT - 1) / (8 * NT));
  return host::launch_dependent(gemv_w4_kernel<T, G, MT, NT>, grid, 32 * WARPS, 0, s, p);
}
template <typename T, int G>
cudaError_t launch_tokens(const W4Params& p, cudaStream_t s) {
  if (p.M <= 8) return launch<T, G, 4, 1>(p, s);
  if (p.M <= 16) return launch<T, G, 2, 2>(p, s);
  return launch<T, G, 2, 4>(p, s);
}
template <typename T>
cudaError_t launch_group(const W4Params& p, int group, cudaStream_t s) {
  return group == 32 ? launch_tokens<T, 32>(p, s) : group == 64 ? launch_tokens<T, 64>(p, s) : launch_tokens<T, 128>(p, s);
}

}  // namespace

extern "C" int flyb200_gemv_w4a16(void* c, const void* a, const void* q, const void* scale, const void* zero, const void* bias, int M,
                                  int N, int K, int group, int dtype, int epilogue, void* stream) {
  if (!c || !a || !q || !scale || M < 0 || N <= 0 || K <= 0) return FLYB200_E_BAD_ARG;
  if (dtype != FLYB200_DT_FP16 && dtype != FLYB200_DT_BF16) return FLYB200_E_BAD_ARG;
  if (epilogue < FLYB200_EPI_NONE || epilogue > FLYB200_EPI_BIAS_GELU || (epilogue != FLYB200_EPI_NONE && !bias)) return FLYB200_E_BAD_ARG;
  if (group != 32 && group != 64 && group != 128) return FLYB200_E_BAD_ARG;
  if (K % group != 0 || N > 0x7fffff00 || M > 32 * 65535) return FLYB200_E_UNSUPPORTED;
  auto multiple = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (!multiple(a, 16) || !multiple(q, 16) || !multiple(c, 2) || !multiple(scale, 2) || !multiple(bias, 2)) return FLYB200_E_BAD_ALIGN;
  if (M == 0) return FLYB200_OK;
  const W4Params p = {c, a, static_cast<const uint8_t*>(q), scale, static_cast<const uint8_t*>(zero), bias, M, N, K, epilogue};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  CUDA_TRY(dtype == FLYB200_DT_FP16 ? launch_group<__half>(p, group, s) : launch_group<__nv_bfloat16>(p, group, s));
  return FLYB200_OK;
}

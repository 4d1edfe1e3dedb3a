// What the kernels of the 4-bit products share: 16-bit types, decoding of codes, activations.
#pragma once
#include "gemm_kernels.cuh"

namespace flyb200 {

// The usual way to decode small integers without a conversion: a code becomes the 16-bit number MAGIC + code by putting it into the last
// places of MAGIC's mantissa; less() then takes the zero
// point off, given as the bits ZERO + zero point, exactly.  bf16: the result is q - z times 2^-12, so that the sum of a
// group stays in the range of fp32 whatever the activations are; UNIT takes it back from the result, where a scale times UNIT need not be
// in range.
template <typename T>
struct W4;
template <>
struct W4<__nv_bfloat16> {
  static constexpr uint32_t MAGIC = 0x4300u, ZERO = 0xBD00u, FORMAT = 1;  // 128, -128 * 2^-12: the last place of the mantissa is 1
  static constexpr float UNIT = 4096.0f;
  __device__ static uint32_t less(uint32_t a, uint32_t b) {
    const uint32_t small = 0x39803980u;  // 2^-12
    const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&small),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static float value(unsigned short v) { return __uint_as_float(static_cast<uint32_t>(v) << 16); }
  __device__ static __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct W4<__half> {
  static constexpr uint32_t MAGIC = 0x6400u, ZERO = MAGIC, FORMAT = 0;  // 1024
  static constexpr float UNIT = 1.0f;
  __device__ static uint32_t less(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static float value(unsigned short v) { return __half2float(__ushort_as_half(v)); }
  __device__ static __half round(float v) { return __float2half_rn(v); }
};

// 8 codes of a word as four pairs of neighbours, less the zero point; `offset`: ZERO + zero point, twice.
template <typename T>
__device__ __forceinline__ void decode_pairs(uint32_t w, uint32_t offset, uint32_t* d) {
  const uint32_t odd = w >> 4;
  constexpr uint32_t BITS = W4<T>::MAGIC * 0x10001u;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint32_t v = __byte_perm(w, odd, static_cast<uint32_t>(b) | static_cast<uint32_t>(4 + b) << 8), m;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(v), "r"(0x000F000Fu), "r"(BITS));  // (v & mask) | BITS
    d[b] = W4<T>::less(m, offset);
  }
}

__device__ __forceinline__ float w4_activation(float v, int epi) {
  if (epi == EPI_BIAS_RELU) return fmaxf(v, 0.0f);
  if (epi == EPI_BIAS_SILU) return v / (1.0f + expf(-v));
  if (epi == EPI_BIAS_GELU) {
    const float y = 0.7978845608f * (v + 0.044715f * (v * v * v));
    const float e = expf(-2.0f * fabsf(y));
    return 0.5f * v * ((y > 0.0f ? 2.0f : 2.0f * e) / (1.0f + e));
  }
  return v;
}

}  // namespace flyb200

// Helpers shared by the dense operators (linear.cu, norm.cu, act8.cu): element access in fp32 or bf16
// storage, 16-byte vectors, the activations with their derivatives chosen at run time, and the 8-bit codes
// of activation checkpoints.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace gl {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V consecutive elements as fp32; V * sizeof(T) = 16 bytes (aligned) or V = 1.
template <typename T>
constexpr int kVec16 = 16 / (int)sizeof(T);

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32<T>(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(r[i] << 16);
      v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
    }
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
}

// act(z) and act'(z) of the dense operators: the framework's identity / ReLU / GELU (erf form) and
// SiLU z / (1 + e^-z).  Unlike the pooled layers' fmaxf, ReLU hands a NaN on.
__device__ __forceinline__ float dense_act(int act, float z) {
  if (act == GL_ACT_IDENTITY) return z;
  if (act == GL_ACT_RELU) return z < 0.f ? 0.f : z;
  if (act == GL_ACT_GELU) return act_f<GL_ACT_GELU>(z);
  return z / (1.f + expf(-z));
}

__device__ __forceinline__ float dense_slope(int act, float z) {
  if (act == GL_ACT_IDENTITY) return 1.f;
  if (act == GL_ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if (act == GL_ACT_GELU) return dact_f<GL_ACT_GELU>(z);
  const float s = 1.f / (1.f + expf(-z));
  return s * (1.f + z * (1.f - s));
}

// ---- 8-bit codes ----
// An activation checkpoint holds x [rows, C] as int8 codes with one exponent byte per 32 consecutive
// channels: x ~ code * 2^(byte - 127), 2^(byte - 127) the smallest power of two (from 2^-126 on) with
// max |x| <= 127 * 2^(byte - 127).  A power-of-two scale makes the division exact, so the codes do not
// depend on how they are computed, and a 7-bit multiple of a power of two is a bf16 number: the tensor
// cores take the values as they stand.  Byte 255 marks a block that held a NaN or an infinity; it
// reads back as NaN.
constexpr int kActBlock = 32;

__device__ __forceinline__ int act8_exponent(float amax) {
  const int bits = __float_as_int(amax);                 // amax >= 0, or NaN
  if (bits >= 0x7F800000) return 255;
  const int e = (bits >> 23) - (((bits & 0x7FFFFF) <= 0x7E0000) ? 6 : 5);   // 1.984375 = 127 / 64
  return e < 1 ? 1 : e;
}

// 2^(127 - byte), exact for byte 1 .. 249 (an exponent of a finite maximum is at most 249).
__device__ __forceinline__ float act8_inverse(int byte) { return __int_as_float((254 - byte) << 23); }

__device__ __forceinline__ float act8_scale(int byte) {
  return byte == 255 ? __int_as_float(0x7FC00000) : __int_as_float(byte << 23);
}

// act'(z) as one byte: rint(192 d) + 32, d in [-1/6, 1.161]; 0 and 1 are exact.
__device__ __forceinline__ uint32_t slope_code(float d) {
  return (uint32_t)(min(max(__float2int_rn(d * 192.f), -32), 223) + 32);
}

__device__ __forceinline__ float slope_value(uint32_t code) { return (float)((int)code - 32) * (1.f / 192.f); }

}  // namespace gl

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

// Host: any of the given pointers (NULL: absent) is no multiple of `bytes`.
template <typename... P>
inline bool off_type(int bytes, P... p) {
  return ((reinterpret_cast<uintptr_t>(p) | ...) & (uintptr_t)(bytes - 1)) != 0;
}

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

// V elements held as loaded (16 bytes, or one element) until they are used.
template <typename T, int V>
struct Vec16 {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&f)[V]) const { load_vec<T, V>(reinterpret_cast<const T*>(&v), f); }
};
template <typename T>
struct Vec16<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f32<T>(v); }
};

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
//
// FAST is for results that are stored in bf16: exponentials and quotients by the hardware's approximations, and
// the normal distribution's tail as s (b0 + .. + b5 s^5) e^(-z^2 / 2) with s = 1 / (1 + 0.3 |z|), the form of Hastings'
// approximations of erfc, whose exponential is also the density that act' needs.  The b are our own, fitted for
// the least relative error, since GELU multiplies the tail by z and nothing else: 1.7e-6 for |z| up to 5, 5.3e-5 from there
// to 13, where the density leaves fp32 (half a bf16 step is at least 2e-3 relative).  With erff and expf the backward
// kernels were bound by arithmetic, not memory.
__device__ __forceinline__ float ex2_approx(float x) {   // 2^x; denormals are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <bool FAST>
__device__ __forceinline__ void normal_cdf_pdf(float z, float& cdf, float& pdf) {
  if constexpr (FAST) {
    const float e = ex2_approx(z * z * (-0.5f * 1.4426950408889634f));       // e^(-z^2 / 2)
    const float s = rcp_approx(fmaf(fabsf(z), 0.3f, 1.f));
    float q = fmaf(s, -0.0817056596f, 0.229728952f);
    q = fmaf(s, fmaf(s, q, -0.0323179811f), 0.152237385f);
    q = s * fmaf(s, fmaf(s, q, 0.111820899f), 0.120235749f);
    const float tail = q * e;
    cdf = z < 0.f ? tail : 1.f - tail;
    pdf = 0.3989422804014327f * e;
  } else {
    cdf = 0.5f * (1.f + erff(z * 0.7071067811865476f));
    pdf = 0.3989422804014327f * expf(-0.5f * z * z);
  }
}

template <bool FAST>
__device__ __forceinline__ float logistic(float z) {
  if constexpr (FAST) return rcp_approx(1.f + ex2_approx(z * -1.4426950408889634f));
  else return 1.f / (1.f + expf(-z));
}

template <int ACT, bool FAST>
__device__ __forceinline__ float dense_act(float z) {
  if constexpr (ACT == GL_ACT_IDENTITY) return z;
  if constexpr (ACT == GL_ACT_RELU) return z < 0.f ? 0.f : z;
  if constexpr (ACT == GL_ACT_GELU) {
    if constexpr (!FAST) return act_f<GL_ACT_GELU>(z);
    float cdf, pdf;
    normal_cdf_pdf<FAST>(z, cdf, pdf);
    return z * cdf;
  }
  return z * logistic<FAST>(z);
}

// act'(z), and act(z) in `a`.
template <int ACT, bool FAST>
__device__ __forceinline__ float dense_slope(float z, float& a) {
  if constexpr (ACT == GL_ACT_IDENTITY) {
    a = z;
    return 1.f;
  } else if constexpr (ACT == GL_ACT_RELU) {
    a = z < 0.f ? 0.f : z;
    return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  } else if constexpr (ACT == GL_ACT_GELU) {
    float cdf, pdf;
    normal_cdf_pdf<FAST>(z, cdf, pdf);
    a = z * cdf;
    return fmaf(z, pdf, cdf);
  } else {
    const float s = logistic<FAST>(z);
    a = z * s;
    return s * fmaf(z, 1.f - s, 1.f);
  }
}

template <int ACT, bool FAST>
__device__ __forceinline__ float dense_slope(float z) {
  float a;
  return dense_slope<ACT, FAST>(z, a);
}

// f(constant<activation>) for the activation chosen at run time: the branch stays outside f's loops.
template <int ACT>
struct ActTag {
  static constexpr int value = ACT;
};
#pragma nv_exec_check_disable
template <typename F>
__host__ __device__ __forceinline__ void with_act(int act, F f) {
  if (act == GL_ACT_IDENTITY) f(ActTag<GL_ACT_IDENTITY>());
  else if (act == GL_ACT_RELU) f(ActTag<GL_ACT_RELU>());
  else if (act == GL_ACT_GELU) f(ActTag<GL_ACT_GELU>());
  else f(ActTag<GL_ACT_SILU>());
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

// act'(z) as one byte: rint(192 d) + 32, d in [-1/6, 1.156]; 0 and 1 are exact.  Code 255, past every act' (the largest,
// GELU's, is 1.129), is a NaN.
__device__ __forceinline__ uint32_t slope_code(float d) {
  return d != d ? 255u : (uint32_t)(min(max(__float2int_rn(d * 192.f), -32), 222) + 32);
}

__device__ __forceinline__ float slope_value(uint32_t code) {
  return code == 255u ? __int_as_float(0x7FC00000) : (float)((int)code - 32) * (1.f / 192.f);
}

// act'(z) in 16 bits (bf16 layers): steps of 2^-14, exact at 0 and 1.  A NaN becomes the code that reads as -2, which
// no act' has; it reads back as NaN.
__device__ __forceinline__ uint32_t slope_code16(float d) {
  return d != d ? 0x8000u : (uint32_t)(__float2int_rn(d * 16384.f) & 0xFFFF);
}
__device__ __forceinline__ float slope_value16(uint32_t code) {
  return code == 0x8000u ? __int_as_float(0x7FC00000) : (float)(int16_t)code * (1.f / 16384.f);
}

}  // namespace gl

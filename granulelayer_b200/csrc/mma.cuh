// Dense bf16 matrix products on tcgen05 for the linear operator (linear.cu): the kernel's parameters and the
// launch entry of mma.cu.
//   out[m, n] = sum over term pairs (i, j) and k of A_i[m, k] B_j[n, k], then LinEpilogue
// A and B are bf16 "planes": one where the operand is a bf16 tensor, three (v = v1 + v2 + v3) where it is fp32.
// Each operand is stored with k contiguous (K-major) or with its row index contiguous (MN-major), so the three
// products of a linear layer read x, w and dz as they lie in memory.
#pragma once

#include "dense.cuh"

namespace gl {

// What follows the sum over k for an element (m, n): z = sum + bias, slope = act'(z), out = act(z) + residual, all in
// storage type `dtype`.  (Adding to an fp32 gradient is a residual that is the output itself.)
struct LinEpilogue {
  const void* bias;
  const void* residual;
  void* out;
  void* slope;
  int64_t ldr, ldo, lds;
  int dtype, act, slope_kind;
};

// db[n] (=, or += with accumulate) the sum of `rows` partial rows part[r N + n] in row order: work that a product's
// epilogue warps do while they wait for their first tile.
struct SumRows {
  const float* part;
  void* out;
  int64_t rows, N;
  int dtype, accumulate;
};

// One warp, 32 columns from n0 on.
__device__ __forceinline__ void sum_rows(const SumRows& j, int64_t n0) {
  const int64_t n = n0 + (threadIdx.x & 31);
  if (n >= j.N) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  int64_t r = 0;
  for (; r + 16 <= j.rows; r += 16) {
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = j.part[(r + k) * j.N + n];
#pragma unroll
    for (int k = 0; k < 16; ++k) s[k & 3] += v[k];
  }
  for (; r < j.rows; ++r) s[0] += j.part[r * j.N + n];
  const float t = (s[0] + s[1]) + (s[2] + s[3]);
  if (j.accumulate) reinterpret_cast<float*>(j.out)[n] += t;
  else if (j.dtype == GL_DTYPE_F32) reinterpret_cast<float*>(j.out)[n] = t;
  else reinterpret_cast<__nv_bfloat16*>(j.out)[n] = __float2bfloat16_rn(t);
}

// A bf16 operand of `planes` planes `plane` elements apart: element (r, k) at ptr[r ld + k], or ptr[k ld + r] when
// `mn`.  ptr 16-byte aligned, ld and plane multiples of 8.
struct MmaOperand {
  const void* ptr;
  int64_t ld, plane;
  int planes, mn;
};

// One product, and up to two in one launch (the gradients of a layer's input and weight: their tiles share the
// machine's waves, and a launch is saved).
struct MmaJob {
  MmaOperand a, b;
  int64_t M, N, K;
  LinEpilogue e;
};
struct MmaSize {
  int64_t M, N, K;
  int npa, npb, b_mn;   // planes of A and B, B MN-major
};

int64_t mma_work_bytes(const MmaSize* sizes, int n, int sms);   // scratch for split sums
// side.part NULL: none; *status (NULL: not wanted) is set to 1 by a wait that ran out.
int mma_run(const MmaJob* jobs, int n, const SumRows& side, void* work, int32_t* status, cudaStream_t st);

// N elements of type T from p on: as 16-byte vectors where `vec`.
template <typename T, int N>
__device__ __forceinline__ void ld_span(const T* p, bool vec, float (&v)[N]) {
  constexpr int V = kVec16<T>;
  if constexpr (N % V == 0) {
    if (vec) {
#pragma unroll
      for (int k = 0; k < N; k += V) {
        float t[V];
        load_vec<T, V>(p + k, t);
#pragma unroll
        for (int j = 0; j < V; ++j) v[k + j] = t[j];
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = to_f32<T>(p[k]);
}

template <typename T, int N>
__device__ __forceinline__ void st_span(T* p, bool vec, const float (&v)[N]) {
  constexpr int V = kVec16<T>;
  if constexpr (N % V == 0) {
    if (vec) {
#pragma unroll
      for (int k = 0; k < N; k += V) {
        float t[V];
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = v[k + j];
        store_vec<T, V>(p + k, t);
      }
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) p[k] = from_f32<T>(v[k]);
}

template <int N>
__device__ __forceinline__ void st_slope(const LinEpilogue& e, int64_t m, int64_t n, bool vec, const float (&d)[N]) {
  const int64_t i = m * e.lds + n;
  if (e.slope_kind == GL_SLOPE_F32) {
    st_span<float, N>(reinterpret_cast<float*>(e.slope) + i, vec, d);
  } else if (e.slope_kind == GL_SLOPE_I16) {
    uint16_t* q = reinterpret_cast<uint16_t*>(e.slope) + i;
    if constexpr (N == 8) {
      if (vec) {
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = slope_code16(d[2 * k]) | (slope_code16(d[2 * k + 1]) << 16);
        *reinterpret_cast<uint4*>(q) = make_uint4(u[0], u[1], u[2], u[3]);
        return;
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) q[k] = (uint16_t)slope_code16(d[k]);
  } else {
    uint8_t* q = reinterpret_cast<uint8_t*>(e.slope) + i;
    if constexpr (N == 8) {
      if (vec) {
        uint32_t u[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k / 4] |= slope_code(d[k]) << (8 * (k % 4));
        *reinterpret_cast<uint2*>(q) = make_uint2(u[0], u[1]);
        return;
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) q[k] = (uint8_t)slope_code(d[k]);
  }
}

// N consecutive elements of row m from column n on (inside the row); `vec`: every given tensor's base and row
// stride is a multiple of 16 bytes (of 8 for a byte slope) and n of N.
template <typename T, int N>
__device__ __forceinline__ void lin_finish_as(const LinEpilogue& e, int64_t m, int64_t n, bool vec, float (&z)[N]) {
  if (e.bias) {
    float t[N];
    ld_span<T, N>(reinterpret_cast<const T*>(e.bias) + n, vec, t);
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] += t[k];
  }
  float r[N];
  if (e.residual) ld_span<T, N>(reinterpret_cast<const T*>(e.residual) + m * e.ldr + n, vec, r);
  with_act(e.act, [&](auto tag) {
    constexpr int ACT = decltype(tag)::value;
    if (e.slope_kind) {
      float d[N];
#pragma unroll
      for (int k = 0; k < N; ++k) d[k] = dense_slope<ACT, sizeof(T) == 2>(z[k], z[k]);
      st_slope<N>(e, m, n, vec, d);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = dense_act<ACT, sizeof(T) == 2>(z[k]);
    }
  });
  if (e.residual) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] += r[k];
  }
  st_span<T, N>(reinterpret_cast<T*>(e.out) + m * e.ldo + n, vec, z);
}

template <int N>
__device__ __forceinline__ void lin_finish(const LinEpilogue& e, int64_t m, int64_t n, bool vec, float (&z)[N]) {
  if (e.dtype == GL_DTYPE_F32) lin_finish_as<float, N>(e, m, n, vec, z);
  else lin_finish_as<__nv_bfloat16, N>(e, m, n, vec, z);
}

}  // namespace gl

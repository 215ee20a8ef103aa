// Dense bf16 matrix products on tcgen05 for the linear operator (linear.cu): the kernel's parameters and the
// launch entry of mma.cu.
//   out[m, n] = sum over term pairs (i, j) and k of A_i[m, k] B_j[n, k], then LinEpilogue
// A and B are bf16 "planes": one where the operand is a bf16 tensor, three (v = v1 + v2 + v3) where it is fp32.
// Each operand is stored with k contiguous (K-major) or with its row index contiguous (MN-major), so the three
// products of a linear layer read x, w and dz as they lie in memory.
#pragma once

#include "dense.cuh"

namespace gl {

// What follows the sum over k for an element (m, n).
struct LinEpilogue {
  const void* bias;
  const void* residual;
  void* out;
  void* z;
  uint8_t* slope;
  int64_t ldr, ldo, ldz, lds;
  int dtype, act, accumulate;
};

// A bf16 operand of `planes` planes `plane` elements apart: element (r, k) at ptr[r ld + k], or ptr[k ld + r] when
// `mn`.  ptr 16-byte aligned, ld and plane multiples of 8.
struct MmaOperand {
  const void* ptr;
  int64_t ld, plane;
  int planes, mn;
};

// Scratch that mma_product needs (split sums), and the product itself.
int64_t mma_work_bytes(int64_t M, int64_t N, int64_t K, int a_planes, int b_planes, int sms);
int mma_product(const MmaOperand& a, const MmaOperand& b, int64_t M, int64_t N, int64_t K, const LinEpilogue& e,
                void* work, cudaStream_t st);

__device__ __forceinline__ float ld_dense(const void* p, int64_t i, int dtype) {
  return dtype == GL_DTYPE_F32 ? reinterpret_cast<const float*>(p)[i]
                               : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void st_dense(void* p, int64_t i, int dtype, float v) {
  if (dtype == GL_DTYPE_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ void lin_finish(const LinEpilogue& e, int64_t m, int64_t n, float z) {
  if (e.accumulate) {
    reinterpret_cast<float*>(e.out)[m * e.ldo + n] += z;
    return;
  }
  if (e.bias) z += ld_dense(e.bias, n, e.dtype);
  if (e.z) st_dense(e.z, m * e.ldz + n, e.dtype, z);
  if (e.slope) e.slope[m * e.lds + n] = (uint8_t)slope_code(dense_slope(e.act, z));
  float y = dense_act(e.act, z);
  if (e.residual) y += ld_dense(e.residual, m * e.ldr + n, e.dtype);
  st_dense(e.out, m * e.ldo + n, e.dtype, y);
}

// N consecutive elements of row m from n on, all inside the row and 16-byte aligned where they are accessed as
// vectors (`vec`: every given tensor's base and row stride are).
template <int N>
__device__ __forceinline__ void ld_span(const void* p, int64_t i, int dtype, bool vec, float (&v)[N]) {
  if (!vec) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = ld_dense(p, i + k, dtype);
  } else if (dtype == GL_DTYPE_F32) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      float t[4];
      load_vec<float, 4>(reinterpret_cast<const float*>(p) + i + k, t);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[k + j] = t[j];
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 8) {
      float t[8];
      load_vec<__nv_bfloat16, 8>(reinterpret_cast<const __nv_bfloat16*>(p) + i + k, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k + j] = t[j];
    }
  }
}

template <int N>
__device__ __forceinline__ void st_span(void* p, int64_t i, int dtype, bool vec, const float (&v)[N]) {
  if (!vec) {
#pragma unroll
    for (int k = 0; k < N; ++k) st_dense(p, i + k, dtype, v[k]);
  } else if (dtype == GL_DTYPE_F32) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const float t[4] = {v[k], v[k + 1], v[k + 2], v[k + 3]};
      store_vec<float, 4>(reinterpret_cast<float*>(p) + i + k, t);
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; k += 8) {
      const float t[8] = {v[k], v[k + 1], v[k + 2], v[k + 3], v[k + 4], v[k + 5], v[k + 6], v[k + 7]};
      store_vec<__nv_bfloat16, 8>(reinterpret_cast<__nv_bfloat16*>(p) + i + k, t);
    }
  }
}

// act(z) in place; the branch on the activation is outside the loops.
template <int N>
__device__ __forceinline__ void dense_act_all(int act, float (&z)[N]) {
  if (act == GL_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = dense_act(GL_ACT_RELU, z[k]);
  } else if (act == GL_ACT_GELU) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = dense_act(GL_ACT_GELU, z[k]);
  } else if (act == GL_ACT_SILU) {
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = dense_act(GL_ACT_SILU, z[k]);
  }
}

// lin_finish for N consecutive columns.
template <int N>
__device__ __forceinline__ void lin_finish_span(const LinEpilogue& e, int64_t m, int64_t n, bool vec, float (&z)[N]) {
  float t[N];
  if (e.accumulate) {
    ld_span<N>(e.out, m * e.ldo + n, GL_DTYPE_F32, vec, t);
#pragma unroll
    for (int k = 0; k < N; ++k) t[k] += z[k];
    st_span<N>(e.out, m * e.ldo + n, GL_DTYPE_F32, vec, t);
    return;
  }
  if (e.bias) {
    ld_span<N>(e.bias, n, e.dtype, vec, t);
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] += t[k];
  }
  if (e.z) st_span<N>(e.z, m * e.ldz + n, e.dtype, vec, z);
  if (e.slope) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      uint32_t u = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) u |= slope_code(dense_slope(e.act, z[k + j])) << (8 * j);
      uint8_t* q = e.slope + m * e.lds + n + k;
      if (vec) {
        *reinterpret_cast<uint32_t*>(q) = u;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = (uint8_t)(u >> (8 * j));
      }
    }
  }
  dense_act_all<N>(e.act, z);
  if (e.residual) {
    ld_span<N>(e.residual, m * e.ldr + n, e.dtype, vec, t);
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] += t[k];
  }
  st_span<N>(e.out, m * e.ldo + n, e.dtype, vec, z);
}

}  // namespace gl

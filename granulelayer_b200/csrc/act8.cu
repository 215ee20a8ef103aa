// Activation checkpoints in 8 bits: write x [rows, C] (fp32 or bf16) as int8 codes and one exponent byte per
// 32 channels, and read it back (dense.cuh states the code).  No counterpart in the reference, whose layers
// save their inputs as they are (sparse_pooling/autograd.py:380-396).
//
// Both directions are bound by HBM: per element sizeof(T) + 1 + 1/32 bytes.  Encoding, a lane
// holds 8 channels, so four neighbouring lanes share a block and find its maximum with two shuffles.  8192 x 4096 fp32:
// encode 32 us (5.2 TB/s), decode 28 us (6.0 TB/s); bf16 30 us (3.3 TB/s: as many instructions
// an element as fp32 for half the bytes) and 17 us (6.1 TB/s).
#include "dense.cuh"

namespace gl {

struct Act8Params {
  const void* x;
  void* out;
  int8_t* codes;
  uint8_t* exps;
  int64_t rows, C, ldx, ldc, nblk;
};

// A warp takes U consecutive segments of 32 lanes at a time (N channels per lane, L lanes per block), so that four
// 16-byte loads are in flight and one division serves them.  Codes are rounded by adding 1.5 * 2^23, whose sum
// holds the integer in its low byte: no conversion instructions.  ALIGNED: rows' 16-byte vectors are, else elements are
// accessed one by one.
template <typename T>
__device__ __forceinline__ void load_aligned8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    load_vec<T, 8>(p, v);
  } else {
    float a[4], b[4];
    load_vec<T, 4>(p, a);
    load_vec<T, 4>(p + 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  }
}
// Channels per lane.  Writing fp32 back, 16 bytes a lane (8 channels, 32 bytes apart: 38 instead of 28 us at 8192 x 4096);
// encoding fp32, 8 channels (two shuffles instead of three for half as many maxima: 32 instead of 40 us).
template <typename T, bool ENCODE>
__host__ __device__ constexpr int act8_lane() { return ENCODE ? 8 : 16 / (int)sizeof(T); }

struct Act8At {
  int64_t row, c;
};

template <typename T, bool ENCODE, bool ALIGNED>
__global__ void __launch_bounds__(256) act8_kernel(Act8Params p) {
  constexpr int N = act8_lane<T, ENCODE>(), L = kActBlock / N, U = ENCODE && sizeof(T) == 4 ? 2 : 4;
  const int lane = threadIdx.x & 31;
  const int64_t segs = (p.nblk * L + 31) / 32, total = p.rows * segs, C32 = p.nblk * kActBlock;
  const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5) * U;
  for (int64_t w = ((int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * U; w < total; w += step) {
    Act8At at[U];
    bool live[U];                               // the lane's block exists
    int64_t row = total < (1ll << 31) ? (int64_t)((unsigned)w / (unsigned)segs) : w / segs;
    int64_t seg = w - row * segs;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      at[u] = Act8At{row, (seg * 32 + lane) * N};
      live[u] = row < p.rows && at[u].c < C32;
      if (++seg == segs) {
        seg = 0;
        ++row;
      }
    }
    if constexpr (ENCODE) {
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const T* src = reinterpret_cast<const T*>(p.x) + at[u].row * p.ldx + at[u].c;
        if (ALIGNED && live[u] && at[u].c + N <= p.C) {
          load_aligned8<T>(src, v[u]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) v[u][i] = live[u] && at[u].c + i < p.C ? to_f32<T>(src[i]) : 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        int m = 0;                              // |v| ordered by its bits: a NaN is above every number
#pragma unroll
        for (int i = 0; i < N; ++i) m = max(m, __float_as_int(v[u][i]) & 0x7FFFFFFF);
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, o));
        if (!live[u]) continue;
        const int byte = act8_exponent(__int_as_float(m));
        const float inv = byte == 255 ? 0.f : act8_inverse(byte);
        uint32_t q[N / 4];
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          uint32_t b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float t = v[u][i + j] * inv;
            if (byte == 249) t = fminf(fmaxf(t, -63.f), 63.f);   // 64 * 2^122 would read back as an infinity
            b[j] = __float_as_uint(t + 12582912.f);
          }
          q[i / 4] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        }
        int8_t* dst = p.codes + at[u].row * p.ldc + at[u].c;
        *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
        if (lane % L == 0) p.exps[at[u].row * p.nblk + at[u].c / kActBlock] = (uint8_t)byte;
      }
    } else {
      uint32_t q[U][N / 4];
      uint8_t e[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!live[u]) continue;
        e[u] = p.exps[at[u].row * p.nblk + at[u].c / kActBlock];
        const int8_t* src = p.codes + at[u].row * p.ldc + at[u].c;
        if constexpr (N == 4) {
          q[u][0] = *reinterpret_cast<const uint32_t*>(src);
        } else {
          const uint2 t = *reinterpret_cast<const uint2*>(src);
          q[u][0] = t.x;
          q[u][N / 4 - 1] = t.y;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!live[u] || at[u].c >= p.C) continue;
        const float s = act8_scale(e[u]);
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)(int8_t)(q[u][i / 4] >> (8 * (i % 4))) * s;
        T* dst = reinterpret_cast<T*>(p.out) + at[u].row * p.ldx + at[u].c;
        if (ALIGNED && at[u].c + N <= p.C) {
          store_vec<T, N>(dst, v);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (at[u].c + i < p.C) dst[i] = from_f32<T>(v[i]);
        }
      }
    }
  }
}

template <typename T, bool ENCODE>
static int launch_act8(const GlAct8Args& a, cudaStream_t st) {
  Act8Params p{a.x, a.out, a.codes, a.exps, a.rows, a.C, a.ldx, a.ldc, (a.C + kActBlock - 1) / kActBlock};
  const void* t = ENCODE ? a.x : a.out;
  const bool aligned = ((uintptr_t)t & 15) == 0 && (a.ldx * (int64_t)sizeof(T)) % 16 == 0;
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const int64_t segs = (p.nblk * (kActBlock / act8_lane<T, ENCODE>()) + 31) / 32;
  const int64_t need = (a.rows * segs + 31) / 32, cap = (int64_t)sms * 16;
  const unsigned blocks = (unsigned)(need < cap ? need : cap);
  if (aligned) act8_kernel<T, ENCODE, true><<<blocks, 256, 0, st>>>(p);
  else act8_kernel<T, ENCODE, false><<<blocks, 256, 0, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e);
  count_launches(1);
  return GL_OK;
}

static int check_act8(const GlAct8Args* a, bool encode) {
  if (!a) return GL_ERR_NULL;
  if (a->rows < 0 || a->C < 1 || a->ldx < a->C || a->ldc < (a->C + kActBlock - 1) / kActBlock * kActBlock ||
      a->ldc % kActBlock)
    return GL_ERR_SHAPE;
  if (a->dtype != GL_DTYPE_F32 && a->dtype != GL_DTYPE_BF16) return GL_ERR_UNSUPPORTED;
  if (a->rows == 0) return GL_OK;
  if (!(encode ? a->x : (const void*)a->out) || !a->codes || !a->exps) return GL_ERR_NULL;
  if (off_type(a->dtype == GL_DTYPE_F32 ? 4 : 2, encode ? a->x : (const void*)a->out) || off_type(16, a->codes))
    return GL_ERR_ALIGN;
  return GL_OK;
}

}  // namespace gl

using namespace gl;

extern "C" int gl_act8_encode(const GlAct8Args* args, void* stream) {
  const int rc = check_act8(args, true);
  if (rc || args->rows == 0) return rc;
  return args->dtype == GL_DTYPE_F32 ? launch_act8<float, true>(*args, (cudaStream_t)stream)
                                     : launch_act8<__nv_bfloat16, true>(*args, (cudaStream_t)stream);
}

extern "C" int gl_act8_decode(const GlAct8Args* args, void* stream) {
  const int rc = check_act8(args, false);
  if (rc || args->rows == 0) return rc;
  return args->dtype == GL_DTYPE_F32 ? launch_act8<float, false>(*args, (cudaStream_t)stream)
                                     : launch_act8<__nv_bfloat16, false>(*args, (cudaStream_t)stream);
}

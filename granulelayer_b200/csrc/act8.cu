// Activation checkpoints in 8 bits: write x [rows, C] (fp32 or bf16) as int8 codes and one exponent byte per
// 32 channels, and read it back (dense.cuh states the code).  No counterpart in the reference, whose layers
// save their inputs as they are (sparse_pooling/autograd.py:380-396).
//
// Both directions are bound by HBM: per element sizeof(T) + 1 + 1/32 bytes.  A lane holds 16 bytes of x (4
// fp32 or 8 bf16 channels), so 8 or 4 neighbouring lanes share a block and find its maximum with 3 or 2
// shuffles; a warp's iteration covers 128 or 256 channels of one row, and its loads and code stores are
// contiguous.
#include "dense.cuh"

namespace gl {

struct Act8Params {
  const void* x;
  void* out;
  int8_t* codes;
  uint8_t* exps;
  int64_t rows, C, ldx, ldc, nblk;
};

// A warp takes U = 4 segments of 32 lanes at a time, so that four loads are in flight; N channels per lane, L = 32 / N
// lanes per block.  ALIGNED: rows' 16-byte vectors are, else elements are accessed one by one.
template <typename T, bool ENCODE, bool ALIGNED>
__global__ void __launch_bounds__(256) act8_kernel(Act8Params p) {
  constexpr int N = kVec16<T>, L = kActBlock / N, U = 4;
  const int lane = threadIdx.x & 31;
  const int64_t segs = (p.nblk * L + 31) / 32, total = p.rows * segs;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < total; w += warps * U) {
    int64_t row[U], c[U];
    bool live[U];                               // the lane's block exists
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = w + u * warps;
      row[u] = total < (1ll << 31) ? (int64_t)((unsigned)k / (unsigned)segs) : k / segs;
      c[u] = ((k - row[u] * segs) * 32 + lane) * N;
      live[u] = k < total && c[u] < p.nblk * kActBlock;
    }
    if constexpr (ENCODE) {
      float v[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const T* src = reinterpret_cast<const T*>(p.x) + row[u] * p.ldx + c[u];
        if (ALIGNED && live[u] && c[u] + N <= p.C) {
          load_vec<T, N>(src, v[u]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) v[u][i] = live[u] && c[u] + i < p.C ? to_f32<T>(src[i]) : 0.f;
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
        const int most = byte == 249 ? 63 : 127;   // 64 * 2^122 would read back as an infinity
        uint32_t q[N / 4];
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          uint32_t b = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            b |= (uint32_t)(max(min(__float2int_rn(v[u][i + j] * inv), most), -most) & 0xFF) << (8 * j);
          q[i / 4] = b;
        }
        int8_t* dst = p.codes + row[u] * p.ldc + c[u];
        if constexpr (N == 4) *reinterpret_cast<uint32_t*>(dst) = q[0];
        else *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
        if (lane % L == 0) p.exps[row[u] * p.nblk + c[u] / kActBlock] = (uint8_t)byte;
      }
    } else {
      uint32_t q[U][N / 4];
      uint8_t e[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!live[u]) continue;
        e[u] = p.exps[row[u] * p.nblk + c[u] / kActBlock];
        const int8_t* src = p.codes + row[u] * p.ldc + c[u];
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
        if (!live[u] || c[u] >= p.C) continue;
        const float s = act8_scale(e[u]);
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)(int8_t)(q[u][i / 4] >> (8 * (i % 4))) * s;
        T* dst = reinterpret_cast<T*>(p.out) + row[u] * p.ldx + c[u];
        if (ALIGNED && c[u] + N <= p.C) {
          store_vec<T, N>(dst, v);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (c[u] + i < p.C) dst[i] = from_f32<T>(v[i]);
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
  const int64_t segs = (p.nblk * (kActBlock / kVec16<T>) + 31) / 32;
  const int64_t need = (a.rows * segs + 7) / 8, cap = (int64_t)sms * 8;
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
  if ((uintptr_t)a->codes & 15) return GL_ERR_ALIGN;
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

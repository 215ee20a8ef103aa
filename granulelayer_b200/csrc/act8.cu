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

// One warp per (row, segment of 32 lanes); LANE_CH channels per lane, 32 / LANE_CH lanes per block.  VEC is
// LANE_CH where a row's 16-byte vectors are aligned, else 1 (element accesses).
template <typename T, bool ENCODE, bool ALIGNED>
__global__ void __launch_bounds__(256) act8_kernel(Act8Params p) {
  constexpr int N = kVec16<T>;
  constexpr int L = kActBlock / N;          // lanes per block
  const int lane = threadIdx.x & 31;
  const int64_t segs = (p.nblk * L + 31) / 32;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w < p.rows * segs; w += warps) {
    const int64_t row = w / segs, c = ((w - row * segs) * 32 + lane) * N;
    const int64_t blk = c / kActBlock;
    const bool whole = c + N <= p.C;
    float v[N];
    if constexpr (ENCODE) {
      const T* src = reinterpret_cast<const T*>(p.x) + row * p.ldx + c;
      if (ALIGNED && whole) {
        load_vec<T, N>(src, v);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = c + i < p.C ? to_f32<T>(src[i]) : 0.f;
      }
      int m = 0;                            // |v| ordered by its bits: a NaN is above every number
#pragma unroll
      for (int i = 0; i < N; ++i) m = max(m, __float_as_int(v[i]) & 0x7FFFFFFF);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, o));
      if (blk < p.nblk) {
        const int byte = act8_exponent(__int_as_float(m));
        const float inv = byte == 255 ? 0.f : act8_inverse(byte);
        const int most = byte == 249 ? 63 : 127;   // 64 * 2^122 would read back as an infinity
        uint32_t q[N / 4];
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          uint32_t u = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) u |= (uint32_t)(max(min(__float2int_rn(v[i + j] * inv), most), -most) & 0xFF) << (8 * j);
          q[i / 4] = u;
        }
        int8_t* dst = p.codes + row * p.ldc + c;
        if constexpr (N == 4) *reinterpret_cast<uint32_t*>(dst) = q[0];
        else *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
        if (lane % L == 0) p.exps[row * p.nblk + blk] = (uint8_t)byte;
      }
    } else if (c < p.C) {
      const float s = act8_scale(p.exps[row * p.nblk + blk]);
      const int8_t* src = p.codes + row * p.ldc + c;
      uint32_t q[N / 4];
      if constexpr (N == 4) {
        q[0] = *reinterpret_cast<const uint32_t*>(src);
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(src);
        q[0] = u.x;
        q[N / 4 - 1] = u.y;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)(int8_t)(q[i / 4] >> (8 * (i % 4))) * s;
      T* dst = reinterpret_cast<T*>(p.out) + row * p.ldx + c;
      if (ALIGNED && whole) {
        store_vec<T, N>(dst, v);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (c + i < p.C) dst[i] = from_f32<T>(v[i]);
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
  const int64_t need = (a.rows * segs + 7) / 8, cap = (int64_t)sms * 32;
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

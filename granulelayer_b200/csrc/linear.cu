// Matrix product with bias, activation and residual, forward and backward (no counterpart in the reference).
//   z = x w^T + bias, y = act(z) + residual
//   dz = dy act'(z), dx = dz w, dw = dz^T x, db = sum over rows of dz
//
// The products run on the tensor cores (mma.cu).  bf16 operands whose rows are 16-byte aligned are read where they
// lie; others are first copied to aligned rows, and fp32 operands are split into three bf16 planes
// (v = v1 + v2 + v3, 24 significand bits for 2^-110 <= |v|; an infinity gives NaN, since it meets all of the other
// operand's terms, of either sign or zero).
// An 8-bit checkpoint of x is one plane even for fp32 layers: its values are bf16 numbers.  A few rows (serving
// single tokens) run row kernels instead, which read w once and are bound by HBM.
//
// dz is written once, rounded to bf16 in bf16 layers and split in fp32 ones, with the column sums of its fp32
// values; where dy itself is dz (identity, bf16, aligned) only the sums are taken.  The rounding is what a bf16 operand of
// the tensor cores costs: dx and dw of 1024 x 4096 x 4096 are 2.3e-3 off in the 2-norm, 1.7e-3 of which is their own
// rounding; a second term of dz would double both products (355 of 654 us of kernels at 8192 x 4096 x 4096).
#include "mma.cuh"

namespace gl {

// ---- operands for the tensor cores ----

__device__ __forceinline__ float bf16_range(float v) {
  constexpr float kMost = 3.38953138925153547590e38f;                 // 0x7F7F
  return fabsf(v) < INFINITY ? fminf(fmaxf(v, -kMost), kMost) : v;    // a NaN or an infinity as it is
}

// v as NP bf16 terms.  A NaN or an infinity stays in the first term (and its remainder is NaN); of several terms the first
// is at most bf16's largest value, so that finite values above it (to fp32's largest, 2^-9 more) stay finite.
template <int NP>
__device__ __forceinline__ void bf16_terms(const float (&v)[8], uint4 (&out)[NP]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (NP > 1) {
        u[i] = j == 0 ? pack_bf16(bf16_range(r[2 * i]), bf16_range(r[2 * i + 1])) : pack_bf16(r[2 * i], r[2 * i + 1]);
      } else {
        u[i] = pack_bf16(r[2 * i], r[2 * i + 1]);
      }
      r[2 * i] -= __uint_as_float(u[i] << 16);
      r[2 * i + 1] -= __uint_as_float(u[i] & 0xFFFF0000u);
    }
    out[j] = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

// 8 elements from p on, `left` of them inside the row (others 0).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int64_t left, bool aligned, float (&v)[8]) {
  if (aligned && left >= 8) {
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
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32<T>(p[i]) : 0.f;
  }
}

// Up to two matrices rows x K (row stride ld) -> planes [NP][rows][K rounded up to 8], in one launch.
struct PackJob {
  const void* src;
  uint16_t* dst;
  int64_t rows, nk, K, ld;   // nk = ceil(K / 8)
  int aligned;
};

template <typename T, int NP>
__device__ __forceinline__ void lin_pack(const PackJob& j0, const PackJob& j1, unsigned block, unsigned blocks) {
  const int64_t n0 = j0.rows * j0.nk, total = n0 + j1.rows * j1.nk;
  for (int64_t t = block * 256ll + threadIdx.x; t < total; t += blocks * 256ll) {
    const bool second = t >= n0;
    const PackJob& j = second ? j1 : j0;
    const int64_t i = second ? t - n0 : t, r = i / j.nk, k = (i - r * j.nk) * 8, plane = j.rows * j.nk * 8;
    float v[8];
    load8<T>(reinterpret_cast<const T*>(j.src) + r * j.ld + k, j.K - k, j.aligned, v);
    uint4 u[NP];
    bf16_terms<NP>(v, u);
#pragma unroll
    for (int q = 0; q < NP; ++q) *reinterpret_cast<uint4*>(j.dst + q * plane + i * 8) = u[q];
  }
}

template <typename T, int NP>
__global__ void __launch_bounds__(256) lin_pack_kernel(PackJob j0, PackJob j1) {
  lin_pack<T, NP>(j0, j1, blockIdx.x, gridDim.x);
}

constexpr int kDzRows = 32;   // rows of one block of the dz kernel, and of one partial column sum

template <int KIND>
__device__ __forceinline__ float slope_at(const void* slope, int64_t i) {
  if constexpr (KIND == GL_SLOPE_F32) return reinterpret_cast<const float*>(slope)[i];
  else if constexpr (KIND == GL_SLOPE_I16) return slope_value16(reinterpret_cast<const uint16_t*>(slope)[i]);
  else return slope_value(reinterpret_cast<const uint8_t*>(slope)[i]);
}

// Eight saved derivatives from element i on, as one aligned load (two for fp32).
template <int KIND>
__device__ __forceinline__ void slope8(const void* slope, int64_t i, float (&d)[8]) {
  if constexpr (KIND == GL_SLOPE_F32) {
    ld_span<float, 8>(reinterpret_cast<const float*>(slope) + i, true, d);
  } else if constexpr (KIND == GL_SLOPE_I16) {
    const uint4 t = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(slope) + i);
    const uint32_t u[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) d[k] = slope_value16((u[k / 2] >> (16 * (k & 1))) & 0xFFFF);
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(slope) + i);
#pragma unroll
    for (int k = 0; k < 8; ++k) d[k] = slope_value(((k < 4 ? u.x : u.y) >> (8 * (k % 4))) & 0xFF);
  }
}

// dz planes [NP][M][Np] (where `dz` is given) and the column sums of each block of kDzRows rows.  A warp spans 256
// columns of a row, and the block's eight warps take every eighth row.  VEC: a lane holds eight consecutive
// columns, in 16-byte accesses; else (rows that are not aligned, or cut) lane + 32 i, in coalesced single ones.
template <typename T, int NP, int KIND, bool VEC>
__device__ __forceinline__ void lin_dz_rows(const T* dy, const void* slope, uint16_t* dz, float (&sum)[8], int64_t m0,
                                            int64_t m1, int64_t n0, int64_t N, int64_t plane, int64_t Np,
                                            int64_t lddy, int64_t lds) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int h = 0; h < kDzRows / 8; ++h) {
    const int64_t m = m0 + warp + 8 * h;
    if (m >= m1) break;
    float d[8];
    if constexpr (VEC) {
      const int64_t n = n0 + lane * 8;
      ld_span<T, 8>(dy + m * lddy + n, true, d);
      if constexpr (KIND != GL_SLOPE_NONE) {
        float s[8];
        slope8<KIND>(slope, m * lds + n, s);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] *= s[i];
      }
      if (dz) {
        uint4 u[NP];
        bf16_terms<NP>(d, u);
#pragma unroll
        for (int j = 0; j < NP; ++j) *reinterpret_cast<uint4*>(dz + j * plane + m * Np + n) = u[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t n = n0 + lane + 32 * i;
        d[i] = n < N ? to_f32<T>(dy[m * lddy + n]) : 0.f;
        if constexpr (KIND != GL_SLOPE_NONE) d[i] *= n < N ? slope_at<KIND>(slope, m * lds + n) : 0.f;
      }
      if (dz) {
        uint4 u[NP];
        bf16_terms<NP>(d, u);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          const uint32_t q[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int64_t n = n0 + lane + 32 * i;
            if (n < Np) dz[j * plane + m * Np + n] = (uint16_t)(q[i / 2] >> (16 * (i & 1)));
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += d[i];
  }
}

// Blocks past dz_blocks pack the products' other operands (a launch less).
template <typename T, int NP, int KIND>
__global__ void __launch_bounds__(256) lin_dz_kernel(const T* dy, const void* slope, uint16_t* dz, float* part,
                                                     int64_t M, int64_t N, int64_t lddy, int64_t lds, int aligned,
                                                     unsigned dz_blocks, PackJob j0, PackJob j1) {
  __shared__ float red[8][256 + 8];
  if (blockIdx.x >= dz_blocks) {
    lin_pack<T, NP>(j0, j1, blockIdx.x - dz_blocks, gridDim.x - dz_blocks);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t segs = (N + 255) / 256, Np = (N + 7) / 8 * 8, plane = M * Np;
  const int64_t rc = blockIdx.x / segs, n0 = (blockIdx.x - rc * segs) * 256;
  const int64_t m0 = rc * kDzRows, m1 = min(M, m0 + kDzRows);
  const bool vec = aligned && n0 + 256 <= N;
  float sum[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) sum[i] = 0.f;
  if (vec) lin_dz_rows<T, NP, KIND, true>(dy, slope, dz, sum, m0, m1, n0, N, plane, Np, lddy, lds);
  else lin_dz_rows<T, NP, KIND, false>(dy, slope, dz, sum, m0, m1, n0, N, plane, Np, lddy, lds);
  if (part == nullptr) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) red[warp][lane + 33 * i] = sum[i];
  __syncthreads();
  const int c = threadIdx.x;                                 // column of the block's 256
  const int src = vec ? c / 8 + 33 * (c % 8) : c % 32 + 33 * (c / 32);
  if (n0 + c < N) {
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) s += red[r][src];
    part[rc * N + n0 + c] = s;
  }
}

// db by itself, for calls that want no product.
__global__ void __launch_bounds__(128) lin_db_kernel(SumRows j) {
  sum_rows(j, ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 5)) * 32);
}

// ---- a few rows ----

// W warps per output column n: each streams its part of w's row n, four 16-byte loads in flight, against MT rows of x
// (from L1), fp32 sums, shuffles and one shared-memory step between the W warps.  Bound by reading w; W grows with the
// row, so that the machine has enough of it in flight (4096 -> 2048 fp32, one token: W = 1 10.2 us, W = 2 7.2 us,
// 4.7 TB/s; 4096 -> 4096 bf16 W = 1 8.1 us, W = 2 8.8 us, eight loads 10.3 us).  What is left of a row after its last
// 4 W 32 16-byte loads is read element by element, so that widths which are no multiple of that run below this rate (one
// token to 4096 outputs, right after a write of 256 MB; K = 768, 1536, 4096, 5120, 11008, 14336: bf16 6.1, 7.0, 10.9,
// 16.1, 29.0, 33.4 us, fp32 6.5, 8.7, 19.7, 23.3, 42.2, 50.0 us).
template <typename T, int MT, int W, bool ALIGNED>
__global__ void __launch_bounds__(128) lin_rows_kernel(const T* x, const T* w, int M, int64_t N, int64_t K,
                                                       int64_t ldx, int64_t ldw, LinEpilogue e) {
  constexpr int V = ALIGNED ? kVec16<T> : 1, U = 4;
  __shared__ float red[4][MT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % W;
  const int64_t n = (int64_t)blockIdx.x * (4 / W) + warp / W;
  if (part == 0 && n < N && lane < M && e.residual)          // lane t finishes row t
    asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const T*>(e.residual) + lane * e.ldr + n));
  float acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = 0.f;
  if (n < N) {
    const T* row = w + n * ldw;
    constexpr int64_t kStep = (int64_t)W * 32 * V;            // k between a lane's loads
    int64_t k = (int64_t)(part * 32 + lane) * V;
    for (; k + (U - 1) * kStep + V <= K; k += U * kStep) {
      Vec16<T, V> wv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) wv[u].load(row + k + u * kStep);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float wf[V];
        wv[u].get(wf);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (t < M) {
            float xf[V];
            load_vec<T, V>(x + t * ldx + k + u * kStep, xf);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[t] = fmaf(xf[i], wf[i], acc[t]);
          }
        }
      }
    }
    for (; k < K; k += kStep) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (k + i < K) {
          const float wf = to_f32<T>(row[k + i]);
#pragma unroll
          for (int t = 0; t < MT; ++t)
            if (t < M) acc[t] = fmaf(to_f32<T>(x[t * ldx + k + i]), wf, acc[t]);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[t] += __shfl_xor_sync(kFullMask, acc[t], o);
  }
  float z[1] = {acc[0]};
#pragma unroll
  for (int t = 1; t < MT; ++t)
    if (lane == t) z[0] = acc[t];
  if constexpr (W > 1) {
    if (lane < MT) red[warp][lane] = z[0];
    __syncthreads();
    if (part != 0) return;
    if (lane < MT) {
      z[0] = red[warp][lane];
#pragma unroll
      for (int q = 1; q < W; ++q) z[0] += red[warp + q][lane];
    }
  }
  if (n < N && lane < M) lin_finish<1>(e, lane, n, false, z);
}

// Rows up to which the row kernels run.  4096 -> 4096 right after a write of 256 MB: bf16 4 rows 15.6 us here; 5 rows 36.3 us
// here and 16.5 us on the tensor cores, whose time the rows hardly change.  fp32 8 rows 37.5 us here; on the tensor cores 9
// and 16 rows 79.6 us (29.6 in splitting w), where this kernel takes 41.3 and 54.8 us: fp32's limit is below where they meet.
template <typename T>
constexpr int kRows = sizeof(T) == 4 ? 8 : 4;

template <typename T, int MT, int W>
static void launch_rows_w(const GlLinearArgs& a, const LinEpilogue& e, bool aligned, cudaStream_t st) {
  const unsigned blocks = (unsigned)((a.N + 4 / W - 1) / (4 / W));
  if (aligned)
    lin_rows_kernel<T, MT, W, true><<<blocks, 128, 0, st>>>((const T*)a.x, (const T*)a.w, (int)a.M, a.N, a.K, a.ldx,
                                                            a.ldw, e);
  else
    lin_rows_kernel<T, MT, W, false><<<blocks, 128, 0, st>>>((const T*)a.x, (const T*)a.w, (int)a.M, a.N, a.K, a.ldx,
                                                             a.ldw, e);
}

template <typename T, int MT>
static void launch_rows(const GlLinearArgs& a, const LinEpilogue& e, bool aligned, cudaStream_t st) {
  const int64_t loads = a.K * (int64_t)sizeof(T) / 512;       // 16-byte loads of a row, per lane of one warp
  if (loads <= 16) launch_rows_w<T, MT, 1>(a, e, aligned, st);
  else if (loads <= 32) launch_rows_w<T, MT, 2>(a, e, aligned, st);
  else launch_rows_w<T, MT, 4>(a, e, aligned, st);
}

template <typename T>
static int run_rows(const GlLinearArgs& a, const LinEpilogue& e, bool aligned, cudaStream_t st) {
  if (a.M == 1) launch_rows<T, 1>(a, e, aligned, st);
  else if (a.M == 2) launch_rows<T, 2>(a, e, aligned, st);
  else if (kRows<T> == 4 || a.M <= 4) launch_rows<T, 4>(a, e, aligned, st);
  else launch_rows<T, kRows<T>>(a, e, aligned, st);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_cuda_error(err);
  count_launches(1);
  return GL_OK;
}

// ---- host ----

static bool rows16(const void* p, int64_t ld, int esize) {
  return ((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0;
}
static int slope_bytes(int kind) { return kind == GL_SLOPE_F32 ? 4 : kind == GL_SLOPE_I16 ? 2 : 1; }
static int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

static int lin_checks(int64_t M, int64_t N, int64_t K, int dtype, int act) {
  if (M < 0 || N < 1 || K < 1) return GL_ERR_SHAPE;
  if ((dtype != GL_DTYPE_F32 && dtype != GL_DTYPE_BF16) || act < GL_ACT_IDENTITY || act > GL_ACT_SILU)
    return GL_ERR_UNSUPPORTED;
  return GL_OK;
}

// Byte offsets of the workspace's parts (each 256-byte aligned) and its size.
struct LinWork {
  int64_t part = 0, dz = 0, x = 0, w = 0, split = 0, total = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = total;
    total += up(bytes, 256);
    return at;
  }
};

static bool few_rows(int64_t M, int dtype) {
  return M <= (dtype == GL_DTYPE_F32 ? kRows<float> : kRows<__nv_bfloat16>);
}

static LinWork lin_fwd_work(int64_t M, int64_t N, int64_t K, int dtype, bool unaligned, int sms) {
  LinWork w;
  if (M == 0 || few_rows(M, dtype)) return w;
  const int np = dtype == GL_DTYPE_F32 ? 3 : 1;
  if (np == 3 || unaligned) {
    w.x = w.take(np * M * up(K, 8) * 2);
    w.w = w.take(np * N * up(K, 8) * 2);
  }
  const MmaSize size{M, N, K, np, np, 0};
  w.split = w.take(mma_work_bytes(&size, 1, sms));
  return w;
}

// `want`: GL_LINEAR_DX / GL_LINEAR_DW, the products of the call.
static LinWork lin_bwd_work(int64_t M, int64_t N, int64_t K, int dtype, bool codes, bool unaligned, int want, int sms) {
  LinWork w;
  if (M == 0) return w;
  const int np = dtype == GL_DTYPE_F32 ? 3 : 1, npx = codes ? 1 : np;
  w.part = w.take(up(M, kDzRows) / kDzRows * N * 4);
  w.dz = w.take(np * M * up(N, 8) * 2);
  if (np == 3 || unaligned) w.w = w.take(np * N * up(K, 8) * 2);
  if (np == 3 || unaligned || codes) w.x = w.take(npx * M * up(K, 8) * 2);
  MmaSize size[2];
  int n = 0;
  if (want & GL_LINEAR_DX) size[n++] = MmaSize{M, K, N, np, np, 1};
  if (want & GL_LINEAR_DW) size[n++] = MmaSize{N, K, M, np, npx, 1};
  w.split = w.take(n ? mma_work_bytes(size, n, sms) : 0);
  return w;
}

// Operands for the tensor cores: a matrix [rows, K] itself where it is aligned bf16, else packed into `dst` by one
// launch for all of a call's matrices.
template <typename T>
struct Packer {
  static constexpr int NP = sizeof(T) == 4 ? 3 : 1;
  PackJob job[2] = {};
  int n = 0;
  MmaOperand add(const void* src, int64_t rows, int64_t K, int64_t ld, int mn, void* dst) {
    const bool aligned = rows16(src, ld, sizeof(T));
    if (NP == 1 && aligned) return MmaOperand{src, ld, 0, 1, mn};
    job[n++] = PackJob{src, (uint16_t*)dst, rows, (K + 7) / 8, K, ld, aligned};
    return MmaOperand{dst, up(K, 8), rows * up(K, 8), NP, mn};
  }
  unsigned blocks(int sms) const {
    const int64_t total = job[0].rows * job[0].nk + job[1].rows * job[1].nk, need = (total + 255) / 256;
    const int64_t cap = 16ll * sms;
    return (unsigned)(need < cap ? need : cap);
  }
  int run(int sms, cudaStream_t st) {
    if (n == 0) return GL_OK;
    lin_pack_kernel<T, NP><<<blocks(sms), 256, 0, st>>>(job[0], job[1]);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return set_cuda_error(err);
    count_launches(1);
    return GL_OK;
  }
};

template <typename T>
static int run_linear_fwd(const GlLinearArgs& a, const LinEpilogue& e, const LinWork& w, int sms, cudaStream_t st) {
  char* work = (char*)a.work;
  Packer<T> pack;
  const MmaOperand x = pack.add(a.x, a.M, a.K, a.ldx, 0, work + w.x);
  const MmaOperand wt = pack.add(a.w, a.N, a.K, a.ldw, 0, work + w.w);
  if (int rc = pack.run(sms, st)) return rc;
  const MmaJob job{x, wt, a.M, a.N, a.K, e};
  return mma_run(&job, 1, SumRows{}, work + w.split, a.status, st);
}

template <typename T, int KIND>
static int launch_dz(const GlLinearBwdArgs& a, uint16_t* dz, float* part, bool aligned, const Packer<T>& pack, int sms,
                     cudaStream_t st) {
  const int64_t blocks = up(a.M, kDzRows) / kDzRows * ((a.N + 255) / 256);
  const unsigned more = pack.n ? pack.blocks(sms) : 0;
  if (blocks + more > 0x7FFFFFFF) return GL_ERR_SHAPE;
  lin_dz_kernel<T, sizeof(T) == 4 ? 3 : 1, KIND><<<(unsigned)blocks + more, 256, 0, st>>>(
      (const T*)a.dy, a.slope, dz, part, a.M, a.N, a.lddy, a.lds, aligned, (unsigned)blocks, pack.job[0], pack.job[1]);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_cuda_error(err);
  count_launches(1);
  return GL_OK;
}

template <typename T>
static int run_linear_bwd(const GlLinearBwdArgs& a, const LinWork& w, int sms, cudaStream_t st) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1;
  char* work = (char*)a.work;
  const int ss = slope_bytes(a.slope_kind);
  const bool aligned = rows16(a.dy, a.lddy, sizeof(T)) &&
                       (a.slope_kind == GL_SLOPE_NONE ||
                        (a.slope_kind == GL_SLOPE_U8 ? (((uintptr_t)a.slope | a.lds) & 7) == 0 : rows16(a.slope, a.lds, ss)));
  const bool dy_is_dz = NP == 1 && aligned && a.slope_kind == GL_SLOPE_NONE;
  const bool write = !dy_is_dz && (a.dx || a.dw);
  MmaOperand dz{a.dy, a.lddy, 0, 1, 0};
  if (!dy_is_dz) dz = MmaOperand{work + w.dz, up(a.N, 8), a.M * up(a.N, 8), NP, 0};
  Packer<T> pack;
  MmaOperand wt{}, x{};
  if (a.dx) wt = pack.add(a.w, a.N, a.K, a.ldw, 1, work + w.w);   // w with its K columns as rows
  if (a.dw && a.codes) {
    GlAct8Args d{};
    d.out = work + w.x;
    d.codes = const_cast<int8_t*>(a.codes);
    d.exps = const_cast<uint8_t*>(a.exps);
    d.rows = a.M; d.C = a.K; d.ldx = up(a.K, 8); d.ldc = a.ldc; d.dtype = GL_DTYPE_BF16;
    if (int rc = gl_act8_decode(&d, st)) return rc;
    x = MmaOperand{work + w.x, up(a.K, 8), 0, 1, 1};
  } else if (a.dw) {
    x = pack.add(a.x, a.M, a.K, a.ldx, 1, work + w.x);
  }
  if (write || a.db) {
    uint16_t* out = write ? (uint16_t*)(work + w.dz) : nullptr;
    float* part = a.db ? (float*)(work + w.part) : nullptr;
    const int rc = a.slope_kind == GL_SLOPE_NONE  ? launch_dz<T, GL_SLOPE_NONE>(a, out, part, aligned, pack, sms, st)
                   : a.slope_kind == GL_SLOPE_F32 ? launch_dz<T, GL_SLOPE_F32>(a, out, part, aligned, pack, sms, st)
                   : a.slope_kind == GL_SLOPE_I16 ? launch_dz<T, GL_SLOPE_I16>(a, out, part, aligned, pack, sms, st)
                                                  : launch_dz<T, GL_SLOPE_U8>(a, out, part, aligned, pack, sms, st);
    if (rc) return rc;
  } else if (int rc = pack.run(sms, st)) {
    return rc;
  }
  SumRows db{};     // done beside the products
  if (a.db) db = SumRows{(const float*)(work + w.part), a.db, up(a.M, kDzRows) / kDzRows, a.N, a.dtype, a.accumulate};
  if (a.db && !a.dx && !a.dw) {
    lin_db_kernel<<<(unsigned)((a.N + 127) / 128), 128, 0, st>>>(db);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return set_cuda_error(err);
    count_launches(1);
    return GL_OK;
  }
  MmaJob jobs[2];
  int n = 0;
  if (a.dx) {   // [M, K] = dz [M, N] w [N, K]
    LinEpilogue e{};
    e.dtype = a.dtype;
    e.out = a.dx;
    e.ldo = a.lddx;
    jobs[n++] = MmaJob{dz, wt, a.M, a.K, a.N, e};
  }
  if (a.dw) {   // [N, K] = dz^T [N, M] x [M, K]
    LinEpilogue e{};
    e.dtype = a.dtype;
    e.out = a.dw;
    e.ldo = a.K;
    if (a.accumulate) {
      e.residual = a.dw;
      e.ldr = a.K;
      e.dtype = GL_DTYPE_F32;
    }
    dz.mn = 1;
    jobs[n++] = MmaJob{dz, x, a.N, a.K, a.M, e};
  }
  return mma_run(jobs, n, db, work + w.split, a.status, st);
}

}  // namespace gl

using namespace gl;

extern "C" int64_t gl_linear_work_bytes(int64_t M, int64_t N, int64_t K, int32_t dtype, int32_t flags) {
  if (int rc = lin_checks(M, N, K, dtype, 0)) return rc;
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const bool unaligned = (flags & GL_LINEAR_UNALIGNED) != 0;
  if (flags & GL_LINEAR_BACKWARD)
    return lin_bwd_work(M, N, K, dtype, (flags & GL_LINEAR_CODES) != 0, unaligned, flags, sms).total;
  return lin_fwd_work(M, N, K, dtype, unaligned, sms).total;
}

extern "C" int gl_linear_fwd(const GlLinearArgs* args, void* stream) {
  if (!args) return GL_ERR_NULL;
  const GlLinearArgs& a = *args;
  if (int rc = lin_checks(a.M, a.N, a.K, a.dtype, a.act)) return rc;
  if (a.slope_kind < GL_SLOPE_NONE || a.slope_kind > GL_SLOPE_U8) return GL_ERR_UNSUPPORTED;
  if (a.ldx < a.K || a.ldw < a.K || a.ldy < a.N || (a.residual && a.ldr < a.N) || (a.slope_kind && a.lds < a.N))
    return GL_ERR_SHAPE;
  if (a.M == 0) return GL_OK;
  if (!a.x || !a.w || !a.y || (a.slope_kind && !a.slope)) return GL_ERR_NULL;
  const int es = a.dtype == GL_DTYPE_F32 ? 4 : 2;
  if (off_type(es, a.x, a.w, a.bias, a.residual, a.y) || off_type(slope_bytes(a.slope_kind), a.slope) ||
      off_type(4, a.status))
    return GL_ERR_ALIGN;
  const LinEpilogue e{a.bias, a.residual, a.y, a.slope, a.ldr, a.ldy, a.lds, a.dtype, a.act, a.slope_kind};
  const bool aligned = rows16(a.x, a.ldx, es) && rows16(a.w, a.ldw, es);
  cudaStream_t st = (cudaStream_t)stream;
  if (few_rows(a.M, a.dtype))
    return a.dtype == GL_DTYPE_F32 ? run_rows<float>(a, e, aligned, st) : run_rows<__nv_bfloat16>(a, e, aligned, st);
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const LinWork w = lin_fwd_work(a.M, a.N, a.K, a.dtype, !aligned, sms);
  if (w.total > 0 && (!a.work || a.work_bytes < w.total)) return GL_ERR_WORKSPACE;
  if ((uintptr_t)a.work & 255) return GL_ERR_ALIGN;
  return a.dtype == GL_DTYPE_F32 ? run_linear_fwd<float>(a, e, w, sms, st)
                                 : run_linear_fwd<__nv_bfloat16>(a, e, w, sms, st);
}

extern "C" int gl_linear_bwd(const GlLinearBwdArgs* args, void* stream) {
  if (!args) return GL_ERR_NULL;
  const GlLinearBwdArgs& a = *args;
  if (int rc = lin_checks(a.M, a.N, a.K, a.dtype, GL_ACT_IDENTITY)) return rc;
  if (a.slope_kind < GL_SLOPE_NONE || a.slope_kind > GL_SLOPE_U8) return GL_ERR_UNSUPPORTED;
  const bool codes = a.codes != nullptr;
  if (a.lddy < a.N || (a.slope_kind && a.lds < a.N) || (a.dw && !codes && a.ldx < a.K) ||
      (codes && (a.ldc < up(a.K, kActBlock) || a.ldc % kActBlock)) || (a.dx && (a.ldw < a.K || a.lddx < a.K)))
    return GL_ERR_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.M == 0) {   // an empty batch: zero gradients (nothing is added to accumulated ones)
    if (a.accumulate) return GL_OK;
    const size_t es = a.dtype == GL_DTYPE_F32 ? 4 : 2;
    cudaError_t e = cudaSuccess;
    if (a.dw) e = cudaMemsetAsync(a.dw, 0, (size_t)(a.N * a.K) * es, st);
    if (e == cudaSuccess && a.db) e = cudaMemsetAsync(a.db, 0, (size_t)a.N * es, st);
    return e == cudaSuccess ? GL_OK : set_cuda_error(e);
  }
  if (!a.dx && !a.dw && !a.db) return GL_OK;
  if (!a.dy || (a.slope_kind && !a.slope) || (a.dx && !a.w) ||
      (a.dw && !codes && !a.x) || (codes && !a.exps))
    return GL_ERR_NULL;
  const int es = a.dtype == GL_DTYPE_F32 ? 4 : 2;
  if (off_type(es, a.dy, codes ? nullptr : a.x, a.w, a.dx) || off_type(a.accumulate ? 4 : es, a.dw, a.db) ||
      off_type(slope_bytes(a.slope_kind), a.slope) || off_type(16, a.codes) || off_type(4, a.status))
    return GL_ERR_ALIGN;
  const bool aligned = (!a.dx || rows16(a.w, a.ldw, es)) && (!a.dw || codes || rows16(a.x, a.ldx, es));
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const int want = (a.dx ? GL_LINEAR_DX : 0) | (a.dw ? GL_LINEAR_DW : 0);
  const LinWork w = lin_bwd_work(a.M, a.N, a.K, a.dtype, codes, !aligned, want, sms);
  if (w.total > 0 && (!a.work || a.work_bytes < w.total)) return GL_ERR_WORKSPACE;
  if ((uintptr_t)a.work & 255) return GL_ERR_ALIGN;
  return a.dtype == GL_DTYPE_F32 ? run_linear_bwd<float>(a, w, sms, st) : run_linear_bwd<__nv_bfloat16>(a, w, sms, st);
}

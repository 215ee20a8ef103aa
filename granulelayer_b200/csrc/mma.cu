// The matrix product of the linear operator on the 5th-generation tensor cores (mma.cuh states it).
//
// A persistent CTA takes output tiles of 128 x BN (and, with split sums, ranges of k).  Ten warps:
//   producer (one lane)  TMA loads of 64 k of every plane of A and B into a ring of 128-byte-swizzled stages
//   issuer (one lane)    tcgen05.mma 128 x BN x 16 per 16 k and term pair, accumulators in TMEM (two buffers)
//   eight epilogue warps TMEM -> registers -> bias, activation, residual -> memory, while the next tile runs
// handing over through mbarriers: full / empty per stage, done / free per accumulator.
//
// fp32 operands come as three bf16 planes; the six products of term pairs i + j <= 2 run smallest first.  The
// tensor core's fp32 accumulation does not round to nearest, so with several planes a sum over k is cut into
// chunks: each chunk's accumulator is added to registers in fp32 while the next one runs.
//
// K-major tiles are one TMA box (64 k wide, 128 or BN rows).  MN-major tiles are boxes of 64 rows-by-64 k; the
// matrix descriptor walks them with 2048 bytes per 16 k and 8192 bytes per 64 rows.  Edges in every
// dimension are the tensor map's zero fill.  Every wait has an iteration limit; a CTA whose wait runs out writes
// NaN to what it has not computed, waits (again bounded) for its own copies and leaves.
#include <cuda.h>

#include "mma.cuh"
#include "tc5.cuh"

namespace gl {

constexpr int kMmBM = 128, kMmBK = 64, kMmThreads = 320, kMmEpiWarps = 8;
constexpr uint32_t kMmWaitLimit = 1u << 20;
constexpr uint32_t kMmPlaneA = kMmBM * kMmBK * 2;

struct MmaParams {
  int64_t M, N;
  int tiles_m, tiles_n, kblocks, chunk, splits, split_blocks;
  int a_mn, b_mn, vec;
  float* part;
  LinEpilogue e;
};

__host__ __device__ constexpr uint32_t mm_stage_bytes(int BN, int NPA, int NPB) {
  return NPA * kMmPlaneA + NPB * (uint32_t)BN * kMmBK * 2;
}
__host__ __device__ constexpr int mm_stages(int BN, int NPA, int NPB) {
  const int n = (int)((227 * 1024 - 2048) / mm_stage_bytes(BN, NPA, NPB));
  return n > 8 ? 8 : n;
}

struct MmaShared {
  uint64_t full[8], empty[8], done[2], free_[2];
  uint32_t tmem;
  int dead;
};

__device__ __forceinline__ void mm_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mm_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mm_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Bounded wait; after the first one that ran out anywhere in the CTA all give up at once.
__device__ __forceinline__ bool mm_wait(MmaShared& sh, uint64_t& bar, uint32_t parity) {
  volatile int* dead = &sh.dead;
  if (*dead) return false;
  const uint32_t a = t5_smem_u32(&bar);
  for (int i = 0; i < 16; ++i) {
    if (t5_mbar_wait(a, parity, kMmWaitLimit / 16)) return true;
    if (*dead) return false;
  }
  *dead = 1;
  return false;
}

struct MmaTile {
  int64_t m0, n0;
  int k0, k1, split;
};

// Work item -> tile and k range.  Tiles run in bands of 8 rows of tiles so that concurrent CTAs share operands in L2.
__device__ __forceinline__ MmaTile mm_tile(const MmaParams& p, int64_t item, int BN) {
  MmaTile t;
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  t.split = (int)(item / tiles);
  const int64_t i = item - t.split * tiles, band = i / (8ll * p.tiles_n), first = band * 8;
  const int64_t rows = min((int64_t)8, p.tiles_m - first), j = i - band * 8 * p.tiles_n;
  t.m0 = (first + j % rows) * kMmBM;
  t.n0 = (j / rows) * BN;
  t.k0 = t.split * p.split_blocks;
  t.k1 = min(p.kblocks, t.k0 + p.split_blocks);
  return t;
}

template <int BN, int NPA, int NPB>
__global__ void __launch_bounds__(kMmThreads, 1)
    mma_kernel(const __grid_constant__ CUtensorMap ta, const __grid_constant__ CUtensorMap tb, const MmaParams p) {
  constexpr int ST = mm_stages(BN, NPA, NPB);
  constexpr uint32_t kStage = mm_stage_bytes(BN, NPA, NPB), kPlaneB = BN * kMmBK * 2;
  constexpr uint32_t kCols = 2 * BN;                 // TMEM columns: two accumulators
  constexpr bool MULTI = NPA > 1;
  constexpr int HALF = BN >= 64 ? BN / 2 : BN;        // columns per epilogue warp
  extern __shared__ unsigned char mm_raw[];
  __shared__ MmaShared sh;
  const uint32_t smem = (t5_smem_u32(mm_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (warp == 9) t5_tmem_alloc(t5_smem_u32(&sh.tmem), kCols);
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      t5_mbar_init(t5_smem_u32(&sh.full[i]), 1);
      t5_mbar_init(t5_smem_u32(&sh.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      t5_mbar_init(t5_smem_u32(&sh.done[i]), 1);
      t5_mbar_init(t5_smem_u32(&sh.free_[i]), BN >= 64 ? kMmEpiWarps : 4);
    }
    sh.dead = 0;
  }
  t5_fence_before_sync();
  __syncthreads();
  t5_fence_after_sync();
  const uint32_t tmem = sh.tmem;
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits;

  if (warp == 8) {
    if (lane == 0) {
      uint32_t it = 0;
      bool live = true;
      for (int64_t item = blockIdx.x; item < items && live; item += gridDim.x) {
        const MmaTile t = mm_tile(p, item, BN);
        for (int kb = t.k0; kb < t.k1; ++kb, ++it) {
          const int s = it % ST;
          if (it >= ST && !mm_wait(sh, sh.empty[s], ((it / ST) - 1) & 1)) {
            live = false;
            break;
          }
          const uint32_t bar = t5_smem_u32(&sh.full[s]), a = smem + s * kStage, b = a + NPA * kMmPlaneA;
          mm_expect(bar, kStage);
#pragma unroll
          for (int i = 0; i < NPA; ++i) {
            if (p.a_mn) {
              for (int h = 0; h < 2; ++h)
                mm_load(a + i * kMmPlaneA + h * 8192, &ta, (int)t.m0 + 64 * h, kb * kMmBK, i, bar);
            } else {
              mm_load(a + i * kMmPlaneA, &ta, kb * kMmBK, (int)t.m0, i, bar);
            }
          }
#pragma unroll
          for (int i = 0; i < NPB; ++i) {
            if (BN >= 64 && p.b_mn) {
              for (int h = 0; h < BN / 64; ++h)
                mm_load(b + i * kPlaneB + h * 8192, &tb, (int)t.n0 + 64 * h, kb * kMmBK, i, bar);
            } else {
              mm_load(b + i * kPlaneB, &tb, kb * kMmBK, (int)t.n0, i, bar);
            }
          }
        }
      }
      if (!live) {   // the copies in flight must land before the CTA's shared memory goes away
        for (uint32_t j = it > ST ? it - ST : 0; j < it; ++j)
          t5_mbar_wait(t5_smem_u32(&sh.full[j % ST]), (j / ST) & 1, kMmWaitLimit);
      }
    }
  } else if (warp == 9) {
    if (lane == 0) {
      const uint32_t idesc = t5_idesc_bf16(kMmBM, BN, p.a_mn, p.b_mn);
      const uint32_t ka = p.a_mn ? 2048u : 32u, kb_ = p.b_mn ? 2048u : 32u;   // bytes per 16 k
      uint32_t it = 0, ch = 0;
      bool live = true;
      for (int64_t item = blockIdx.x; item < items && live; item += gridDim.x) {
        const MmaTile t = mm_tile(p, item, BN);
        for (int c0 = t.k0; c0 < t.k1 && live; c0 += p.chunk, ++ch) {
          const int c1 = min(t.k1, c0 + p.chunk), buf = ch & 1;
          if (ch >= 2 && !mm_wait(sh, sh.free_[buf], ((ch >> 1) - 1) & 1)) {
            live = false;
            break;
          }
          t5_fence_after_sync();
          const uint32_t d = tmem + buf * BN;
          uint32_t acc = 0;
          for (int kb = c0; kb < c1; ++kb, ++it) {
            const int s = it % ST;
            if (!mm_wait(sh, sh.full[s], (it / ST) & 1)) {
              live = false;
              break;
            }
            t5_fence_after_sync();
            const uint32_t a = smem + s * kStage, b = a + NPA * kMmPlaneA;
#pragma unroll
            for (int sum = (NPA > 1 ? 2 : 0); sum >= 0; --sum) {
#pragma unroll
              for (int i = 0; i < NPA; ++i) {
                const int j = sum - i;
                if (j < 0 || j >= NPB) continue;
#pragma unroll
                for (int k = 0; k < kMmBK / 16; ++k) {
                  t5_mma_bf16(d, t5_desc_sw128(a + i * kMmPlaneA + k * ka, 8192, 1024),
                              t5_desc_sw128(b + j * kPlaneB + k * kb_, 8192, 1024), idesc, acc);
                  acc = 1;
                }
              }
            }
            t5_commit(t5_smem_u32(&sh.empty[s]));
          }
          if (live) t5_commit(t5_smem_u32(&sh.done[buf]));
        }
      }
    }
  } else if (BN >= 64 || warp < 4) {
    const int row = 32 * (warp & 3) + lane, half = BN >= 64 ? warp >> 2 : 0;
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    uint32_t ch = 0;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
      const MmaTile t = mm_tile(p, item, BN);
      const int64_t m = t.m0 + row, n0 = t.n0 + half * HALF;
      float sum[MULTI ? HALF : 1];
      for (int c0 = t.k0; c0 < t.k1; c0 += p.chunk, ++ch) {
        const int buf = ch & 1;
        const bool ok = __all_sync(kFullMask, mm_wait(sh, sh.done[buf], (ch >> 1) & 1));
        t5_fence_after_sync();
        const bool last = c0 + p.chunk >= t.k1;
#pragma unroll
        for (int q = 0; q < HALF / 32; ++q) {
          float v[32];
          t5_ld32(tmem + lane_base + (uint32_t)(buf * BN + half * HALF + 32 * q), v);
          if (!ok) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7FC00000);
          }
          if constexpr (MULTI) {
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[32 * q + i] = c0 == t.k0 ? v[i] : sum[32 * q + i] + v[i];
          } else {
            if (q == HALF / 32 - 1) {                   // the accumulator is read: free it before the stores
              t5_fence_before_sync();
              __syncwarp();
              if (lane == 0) mm_arrive(t5_smem_u32(&sh.free_[buf]));
            }
          }
          if constexpr (!MULTI) {
            const int64_t n = n0 + 32 * q;
            if (m < p.M && n < p.N) {
              if (p.part) {
                float* out = p.part + (t.split * p.M + m) * p.N;
                if (n + 32 <= p.N) {
                  st_span<32>(out, n, GL_DTYPE_F32, (p.N & 3) == 0, v);
                } else {
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (n + i < p.N) out[n + i] = v[i];
                }
              } else if (n + 32 <= p.N) {
                lin_finish_span<32>(p.e, m, n, p.vec, v);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (n + i < p.N) lin_finish(p.e, m, n + i, v[i]);
              }
            }
          }
        }
        if constexpr (MULTI) {
          t5_fence_before_sync();
          __syncwarp();
          if (lane == 0) mm_arrive(t5_smem_u32(&sh.free_[buf]));
          if (last) {
#pragma unroll
            for (int q = 0; q < HALF / 32; ++q) {
              const int64_t n = n0 + 32 * q;
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = sum[32 * q + i];
              if (m >= p.M || n >= p.N) continue;
              if (p.part) {
                float* out = p.part + (t.split * p.M + m) * p.N;
                if (n + 32 <= p.N) {
                  st_span<32>(out, n, GL_DTYPE_F32, (p.N & 3) == 0, v);
                } else {
#pragma unroll
                  for (int i = 0; i < 32; ++i)
                    if (n + i < p.N) out[n + i] = v[i];
                }
              } else if (n + 32 <= p.N) {
                lin_finish_span<32>(p.e, m, n, p.vec, v);
              } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (n + i < p.N) lin_finish(p.e, m, n + i, v[i]);
              }
            }
          }
        }
      }
    }
  }
  __syncthreads();
  t5_fence_after_sync();
  if (warp == 9) t5_tmem_dealloc(tmem, kCols);
}

// Sums the splits of a product in split order and finishes the elements, four columns per thread.
__global__ void __launch_bounds__(256) mma_join_kernel(const float* part, int64_t M, int64_t N, int splits,
                                                       LinEpilogue e, int vec) {
  const int64_t nq = (N + 3) / 4, total = M * nq;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t m = i / nq, n = (i - m * nq) * 4;
    const float* src = part + m * N + n;
    if ((N & 3) == 0) {
      float4 s = *reinterpret_cast<const float4*>(src);
      for (int k = 1; k < splits; ++k) {
        const float4 t = *reinterpret_cast<const float4*>(src + k * M * N);
        s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
      }
      const float z[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) lin_finish(e, m, n + j, z[j]);
    } else {
      for (int j = 0; j < 4 && n + j < N; ++j) {
        float s = src[j];
        for (int k = 1; k < splits; ++k) s += src[k * M * N + j];
        lin_finish(e, m, n + j, s);
      }
    }
  }
}

// ---- host ----
struct MmaPlan {
  int BN, splits, split_blocks, chunk;
  int64_t tiles_m, tiles_n;
};

// Tile width and number of splits of k: the least estimated time, in clocks of one SM.  A 64-wide k block costs the
// larger of its MMAs (BN / 2 clocks a term) and its loads (about 56 bytes a clock for one SM of many); split
// sums add their partial tiles' traffic and a second launch.
static MmaPlan mma_plan(int64_t M, int64_t N, int64_t K, int npa, int npb, bool b_mn, int sms) {
  MmaPlan best{};
  double best_t = 1e300;
  const int64_t kb = (K + kMmBK - 1) / kMmBK;
  const int terms = npa == 1 ? 1 : (npb == 1 ? 3 : 6);
  for (int BN : {256, 128, 64, 32}) {
    if (BN == 256 && npa > 1) continue;
    if (BN == 32 && (b_mn || npa > 1)) continue;
    const int64_t tm = (M + kMmBM - 1) / kMmBM, tn = (N + BN - 1) / BN, tiles = tm * tn;
    const double load = mm_stage_bytes(BN, npa, npb) / 56.0, mma = terms * 2.0 * BN;
    const double block = (load > mma ? load : mma) + 20;
    for (int s = 1; s <= 32 && s <= kb; ++s) {
      const int64_t sb = (kb + s - 1) / s;
      if ((kb + sb - 1) / sb != s) continue;
      const int64_t waves = (tiles * s + sms - 1) / sms;
      double t = (double)waves * sb * block + 2500.0 + (double)BN * 6 * waves;
      if (s > 1) t += 3000.0 + (double)M * N * (s + 1) * 4 / 2500.0;
      if (t < best_t) {
        best_t = t;
        best = MmaPlan{BN, s, (int)sb, npa > 1 ? 2 : 1 << 30, tm, tn};
      }
    }
  }
  return best;
}

int64_t mma_work_bytes(int64_t M, int64_t N, int64_t K, int npa, int npb, int sms) {
  int64_t most = 0;
  for (int b_mn = 0; b_mn < 2; ++b_mn) {
    const MmaPlan pl = mma_plan(M, N, K, npa, npb, b_mn, sms);
    const int64_t n = pl.splits > 1 ? 4 * pl.splits * M * N : 0;
    if (n > most) most = n;
  }
  return most;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* q = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &q, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      q = nullptr;
    return (EncodeTiled)q;
  }();
  return fn;
}

// Tensor map of an operand with `rows` rows and K of k: boxes of 64 k x `box` rows, or 64 rows x 64 k (mn).
static int operand_map(CUtensorMap* map, const MmaOperand& o, int64_t rows, int64_t K, int box) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return GL_ERR_DEVICE;
  const cuuint64_t dims[3] = {(cuuint64_t)(o.mn ? rows : K), (cuuint64_t)(o.mn ? K : rows), (cuuint64_t)o.planes};
  const int64_t plane = o.planes > 1 ? o.plane : o.ld * (int64_t)dims[1];
  const cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)plane * 2};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)(o.mn ? 64 : box), 1}, ones[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.ptr), dims, strides, boxes, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? GL_OK : GL_ERR_SHAPE;
}

template <int BN, int NPA, int NPB>
static int launch_mma(const CUtensorMap& ta, const CUtensorMap& tb, const MmaParams& p, int sms, cudaStream_t st) {
  const size_t smem = mm_stages(BN, NPA, NPB) * mm_stage_bytes(BN, NPA, NPB) + 1024;
  if (int rc = ensure_dynamic_smem((const void*)mma_kernel<BN, NPA, NPB>, smem)) return rc;
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.splits;
  mma_kernel<BN, NPA, NPB><<<(unsigned)(items < sms ? items : sms), kMmThreads, smem, st>>>(ta, tb, p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e);
  count_launches(1);
  return GL_OK;
}

static bool aligned16(const void* p, int64_t ld, int esize) {
  return p == nullptr || (((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0);
}

int mma_product(const MmaOperand& a, const MmaOperand& b, int64_t M, int64_t N, int64_t K, const LinEpilogue& e,
                void* work, cudaStream_t st) {
  if (M > 0x7FFFFF00 || N > 0x7FFFFF00 || K > 0x7FFFFF00) return GL_ERR_SHAPE;
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  const MmaPlan pl = mma_plan(M, N, K, a.planes, b.planes, b.mn, sms);
  CUtensorMap ta, tb;
  if (int rc = operand_map(&ta, a, M, K, kMmBM)) return rc;
  if (int rc = operand_map(&tb, b, N, K, pl.BN)) return rc;
  MmaParams p{};
  p.M = M; p.N = N; p.tiles_m = (int)pl.tiles_m; p.tiles_n = (int)pl.tiles_n;
  p.kblocks = (int)((K + kMmBK - 1) / kMmBK); p.chunk = pl.chunk < p.kblocks ? pl.chunk : p.kblocks;
  p.splits = pl.splits; p.split_blocks = pl.split_blocks; p.a_mn = a.mn; p.b_mn = b.mn; p.e = e;
  const int es = e.dtype == GL_DTYPE_F32 || e.accumulate ? 4 : 2;
  p.vec = aligned16(e.out, e.ldo, es) && aligned16(e.z, e.ldz, es) && aligned16(e.residual, e.ldr, es) &&
          aligned16(e.bias, 0, es) && aligned16(e.slope, e.lds, 1);
  p.part = pl.splits > 1 ? (float*)work : nullptr;
  if (pl.splits > 1 && !work) return GL_ERR_WORKSPACE;
  int rc = GL_ERR_UNSUPPORTED;
  if (a.planes == 1 && b.planes == 1) {
    rc = pl.BN == 256   ? launch_mma<256, 1, 1>(ta, tb, p, sms, st)
         : pl.BN == 128 ? launch_mma<128, 1, 1>(ta, tb, p, sms, st)
         : pl.BN == 64  ? launch_mma<64, 1, 1>(ta, tb, p, sms, st)
                        : launch_mma<32, 1, 1>(ta, tb, p, sms, st);
  } else if (a.planes == 3 && b.planes == 3) {
    rc = pl.BN == 128 ? launch_mma<128, 3, 3>(ta, tb, p, sms, st) : launch_mma<64, 3, 3>(ta, tb, p, sms, st);
  } else if (a.planes == 3 && b.planes == 1) {
    rc = pl.BN == 128 ? launch_mma<128, 3, 1>(ta, tb, p, sms, st) : launch_mma<64, 3, 1>(ta, tb, p, sms, st);
  }
  if (rc || pl.splits == 1) return rc;
  const int64_t quads = M * ((N + 3) / 4), need = (quads + 255) / 256;
  mma_join_kernel<<<(unsigned)(need < 8 * sms ? need : 8 * sms), 256, 0, st>>>(p.part, M, N, pl.splits, e, p.vec);
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return set_cuda_error(err);
  count_launches(1);
  return GL_OK;
}

}  // namespace gl

// The matrix product of the linear operator on the 5th-generation tensor cores (mma.cuh states it).
//
// A persistent CTA, or a pair of CTAs, takes output tiles of 128 (256) x BN and, with split sums, ranges of k.  Ten
// warps per CTA:
//   producer  TMA loads of 64 k of a plane of A and of B into a ring of 128-byte-swizzled slots
//   issuer (of a pair, the even CTA's)  tcgen05.mma per 16 k and term pair, two accumulators in TMEM
//   eight epilogue warps TMEM -> registers -> shared memory -> bias, activation, residual -> memory, row by row in
//                        whole sectors, while the next tile runs
// handing over through mbarriers: full / empty per slot, done / free per accumulator.
//
// Pairs (cta_group::2, 256 x 256 tiles): each CTA loads its 128 rows of A and half of B, so a CTA moves 32 KB through
// its shared memory per 64 k instead of 48 KB, both from L2 and to the tensor core; that traffic, not the MMA
// rate, bounds the 128 x 256 tile of one CTA.
//
// fp32 operands come as three bf16 planes; a slot holds plane i of both, and the products of term pairs (i, j),
// i + j <= 2, run as their slots arrive.  The tensor core's fp32 accumulation truncates, so the pair (0, 0) has an
// accumulator of its own that the five small pairs (2^-8 of its size and less) do not disturb, and a sum over k is
// cut into chunks of 512: each chunk's accumulators are added to registers in fp32 (rounding to nearest) while the
// next one runs.  (One accumulator for all pairs needed chunks of 128 for 0.8e-6 in the 2-norm at K = 4096, where plain
// fp32 products are 1.0e-6 off, and reading it that often cost a fifth of the time.)
//
// bf16 operands: a sum over k of terms of one sign that stays in one accumulator comes out small by up to k / 16 2^-23 of
// itself (measured 2.2e-6 at k = 1024, 1.4e-5 at 4096, 1.8e-4 at 32768).  Where the result is kept in fp32 (added to an
// fp32 gradient, or a split's partial tile) a sum over k is therefore cut into chunks of kMmLongChunk blocks too, and each
// chunk is added to memory, by the thread that stored the one before, while the next one runs (dx and an fp32 dw of
// 8192 x 4096 x 4096: 404 -> 424 us; 40000 rows, 4096 x 1024, one sign: 2.3e-4 -> below 1e-5 off).  A bf16 result takes one
// accumulator; splits see to it that it sums at most kMmLongest blocks (7e-4 for one sign; half a bf16 step is 2^-9 to
// 2^-8).
//
// K-major tiles are one TMA box (64 k wide, all rows of the tile); MN-major tiles are boxes of 64 rows by 64 k, which
// the matrix descriptor walks with 2048 bytes per 16 k and 8192 bytes per 64 rows.  Edges in every dimension are
// the tensor map's zero fill.  Every wait has a limit in time and in iterations; a CTA whose wait runs out sets the call's
// status word, writes NaN to what it has not computed, waits (again bounded) for its own copies and products and leaves.
// Otherwise it leaves when every slot has been given back: by then its copies have landed, the tensor core has read them,
// and no arrival is on its way to a barrier of a CTA that is gone.
#include <cuda.h>

#include "mma.cuh"
#include "tc5.cuh"

namespace gl {

constexpr int kMmBM = 128, kMmBK = 64, kMmThreads = 320, kMmEpiWarps = 8, kMmMaxSlots = 20;
// A wait gives up after 4 s by the GPU's clock and 2^17 polls, or after 2^28 polls.  The longest that a sound launch waits is
// an epilogue for its tile's sum: at most 2^25 blocks of k in 32 splits, 0.4 s.
constexpr uint64_t kMmWaitNs = 4000000000ull;
constexpr uint32_t kMmWaitPolls = 1024, kMmWaitLeast = 128, kMmWaitMost = 1u << 18;
constexpr uint32_t kMmDrainPolls = 1u << 16;                   // for what is on its way already
constexpr int kMmLongChunk = 32, kMmLongest = 2048;            // in blocks of 64 k
constexpr int kMmPitch = 36;                                   // floats per row of a warp's 32 x 32 epilogue tile
constexpr uint32_t kMmEpiBytes = kMmEpiWarps * 32 * kMmPitch * 4;

struct MmaOne {
  int64_t M, N;
  int tiles_m, tiles_n, kblocks, splits, split_blocks;
  int a_mn, b_mn, vec, npb, chunk;   // chunk: blocks of k in one accumulator
  uint32_t a_bytes;            // of a plane of A as loaded
  float* part;
  LinEpilogue e;
};
struct MmaParams {
  MmaOne job[2];
  int64_t items0, items;       // work items of job 0, of all
  int slots;
  uint32_t a_slot, b_bytes;    // bytes of a slot for A, for B
  SumRows side;
  int32_t* status;             // optional: set to 1 by a wait that ran out
};

// A slot: a plane of A (128 rows, or as many as there are) and of B (this CTA's share of BN rows), 64 k each; the ring
// takes what the epilogue's tiles leave of the shared memory.  (The tensor core reads 128 rows of A whatever a slot
// holds: the rows past a short A are whatever follows in shared memory, and give accumulator rows nobody reads.)
constexpr uint32_t kMmRing = 227 * 1024 - 2048 - kMmEpiBytes;

struct MmaShared {
  uint64_t full[kMmMaxSlots], empty[kMmMaxSlots], done[4], free_[4], last;
  uint32_t tmem;
  int dead;
  int32_t* status;
};

__device__ __forceinline__ void mm_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Arrive on an mbarrier of the even CTA of the pair (or of this CTA).
template <int CTAS>
__device__ __forceinline__ void mm_arrive(uint32_t bar) {
  if constexpr (CTAS == 1) {
    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
  } else {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(remote) : "r"(bar));
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
  }
}

// TMA load into this CTA's shared memory; its bytes count on `bar` (of a pair: a shared::cluster address in the even
// CTA).
template <int CTAS>
__device__ __forceinline__ void mm_load(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CTAS == 1) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  }
}

__device__ __forceinline__ uint64_t mm_now() {
  uint64_t ns;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(ns));
  return ns;
}

// Bounded wait; after the first one that ran out anywhere in the CTA all give up at once.
__device__ __forceinline__ bool mm_wait(MmaShared& sh, uint64_t& bar, uint32_t parity) {
  const uint32_t a = t5_smem_u32(&bar);
  if (t5_mbar_wait(a, parity, 1)) return true;
  volatile int* dead = &sh.dead;
  uint64_t from = 0;
  for (uint32_t i = 0; i < kMmWaitMost; ++i) {
    if (*dead) return false;
    if (t5_mbar_wait(a, parity, kMmWaitPolls)) return true;
    const uint64_t now = mm_now();
    if (i == 0) from = now;
    if (i >= kMmWaitLeast && now - from > kMmWaitNs) break;
  }
  *dead = 1;
  if (sh.status) {
    *(volatile int32_t*)sh.status = 1;     // may lie in host memory
    __threadfence_system();
  }
  return false;
}

// For a whole warp: the same answer in every lane.
__device__ __forceinline__ bool mm_wait_warp(MmaShared& sh, uint64_t& bar, uint32_t parity) {
  return __all_sync(kFullMask, mm_wait(sh, bar, parity));
}

// One lane of a converged warp.  elect.sync rather than lane == 0: the compiler then knows that one thread issues the
// tensor instructions and need not loop over the active ones (8192 x 4096 x 4096: 254 -> 210 us).  The whole warp runs
// the loops around them, so that addresses and descriptors stay in uniform registers.
__device__ __forceinline__ bool mm_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// Position in the ring of slots: index and the parity of its current round.
struct MmaRing {
  int slots, s = 0;
  uint32_t round = 0;
  __device__ __forceinline__ explicit MmaRing(int n) : slots(n) {}
  __device__ __forceinline__ void next() {
    if (++s == slots) {
      s = 0;
      ++round;
    }
  }
  __device__ __forceinline__ uint32_t uses(int slot) const { return round + (slot < s); }   // of a slot, so far
};

struct MmaTile {
  int64_t m0, n0;
  int k0, k1, split, job;
};

// Work item -> job, tile and k range.  Tiles run in bands of 8 rows of tiles so that concurrent CTAs share operands in L2.
template <int JOBS>
__device__ __forceinline__ MmaTile mm_tile(const MmaParams& p, int64_t item, int BM, int BN) {
  MmaTile t;
  t.job = JOBS == 1 ? 0 : item >= p.items0;   // one job: its parameters are constants of the launch
  const MmaOne& o = p.job[JOBS == 1 ? 0 : t.job];
  const int64_t tiles = (int64_t)o.tiles_m * o.tiles_n, it = t.job ? item - p.items0 : item;
  t.split = (int)(it / tiles);
  const int64_t i = it - t.split * tiles, band = i / (8ll * o.tiles_n), first = band * 8;
  const int64_t rows = min((int64_t)8, o.tiles_m - first), j = i - band * 8 * o.tiles_n;
  t.m0 = (first + j % rows) * BM;
  t.n0 = (j / rows) * BN;
  t.k0 = t.split * o.split_blocks;
  t.k1 = min(o.kblocks, t.k0 + o.split_blocks);
  return t;
}

// ---- epilogue of a warp's 32 x 32 block at (m0, n0) ----
// The accumulator gives lane r row r.  Through shared memory a lane gets, eight values at a time, what lies well in
// memory: where rows are aligned and the block is whole in n (VEC), columns 8 (lane % 4) .. + 7 of row lane / 4 + 8 h,
// in 16-byte accesses that fill sectors; else column `lane` of rows 8 h .. 8 h + 7, whose accesses coalesce across
// lanes.  Eight at a time and not 32: a launch fetches its code from L2, and unrolled epilogues cost small products
// 2 us.  FULL false (gradients): no bias, activation or slope.
template <typename T, bool FULL, bool VEC>
__device__ __forceinline__ void mm_finish8(const LinEpilogue& e, float (&z)[8], int64_t m, int64_t n, int rows) {
  T* out = reinterpret_cast<T*>(e.out) + m * e.ldo + n;
  float r[8];
  if (e.residual) {
    const T* p = reinterpret_cast<const T*>(e.residual) + m * e.ldr + n;
    if constexpr (VEC) {
      ld_span<T, 8>(p, true, r);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = i < rows ? to_f32<T>(p[i * e.ldr]) : 0.f;
    }
  }
  if constexpr (FULL) {
    if (e.bias) {
      const T* p = reinterpret_cast<const T*>(e.bias) + n;
      float b[VEC ? 8 : 1];
      ld_span<T, VEC ? 8 : 1>(p, VEC, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] += b[VEC ? i : 0];
    }
    with_act(e.act, [&](auto tag) {
      constexpr int ACT = decltype(tag)::value;
      if (e.slope_kind) {
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = dense_slope<ACT, sizeof(T) == 2>(z[i], z[i]);
        if constexpr (VEC) {
          st_slope<8>(e, m, n, true, d);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float t[1] = {d[i]};
            if (i < rows) st_slope<1>(e, m + i, n, false, t);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = dense_act<ACT, sizeof(T) == 2>(z[i]);
      }
    });
  }
  if (e.residual) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] += r[i];
  }
  if constexpr (VEC) {
    st_span<T, 8>(out, true, z);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < rows) out[i * e.ldo] = from_f32<T>(z[i]);
  }
}

// `more`: not the sum's first chunk (only where the sums are kept in fp32; of a gradient that is added to, the residual is
// what the chunk before left).
template <bool FULL, bool VEC>
__device__ __forceinline__ void mm_store_rows(const MmaOne& p, const float* tile, int64_t m0, int64_t n0, int split,
                                              bool more) {
  const int lane = threadIdx.x & 31, rows = (int)min((int64_t)32, p.M - m0);
  const int c = VEC ? (lane & 3) * 8 : lane;
  const int64_t n = n0 + c;
  if (!VEC && n >= p.N) return;
#pragma unroll 2
  for (int h = 0; h < 4; ++h) {
    const int r = 8 * h + (VEC ? lane >> 2 : 0);
    if (r >= rows) break;
    float z[8];
    if constexpr (VEC) {
      const float4 a = *reinterpret_cast<const float4*>(tile + r * kMmPitch + c);
      const float4 b = *reinterpret_cast<const float4*>(tile + r * kMmPitch + c + 4);
      z[0] = a.x; z[1] = a.y; z[2] = a.z; z[3] = a.w; z[4] = b.x; z[5] = b.y; z[6] = b.z; z[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) z[i] = tile[(r + i) * kMmPitch + c];
    }
    if (p.part) {
      float* out = p.part + (split * p.M + m0 + r) * p.N + n;
      if constexpr (VEC) {
        if (more) {
          float t[8];
          ld_span<float, 8>(out, true, t);
#pragma unroll
          for (int i = 0; i < 8; ++i) z[i] += t[i];
        }
        st_span<float, 8>(out, true, z);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (r + i < rows) out[i * p.N] = more ? out[i * p.N] + z[i] : z[i];
      }
    } else if (p.e.dtype == GL_DTYPE_F32) {
      mm_finish8<float, FULL, VEC>(p.e, z, m0 + r, n, rows - r);
    } else {
      mm_finish8<__nv_bfloat16, FULL, VEC>(p.e, z, m0 + r, n, rows - r);
    }
  }
}

template <bool FULL>
__device__ __forceinline__ void mm_store_block(const MmaOne& p, float* tile, const float* v, int64_t m0, int64_t n0,
                                               int split, bool more) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 32; j += 4)
    *reinterpret_cast<float4*>(tile + lane * kMmPitch + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
  __syncwarp();
  if (p.vec && n0 + 32 <= p.N) mm_store_rows<FULL, true>(p, tile, m0, n0, split, more);
  else mm_store_rows<FULL, false>(p, tile, m0, n0, split, more);
  __syncwarp();
}

// Asks L2 for the residual of a warp's rows m0 .. + 31, columns n0 .. + cols - 1, while its accumulator is being made.
__device__ __forceinline__ void mm_prefetch(const MmaOne& p, int64_t m0, int64_t n0, int cols) {
  const int lane = threadIdx.x & 31;
  if (p.part || !p.e.residual || m0 + lane >= p.M) return;
  const int es = p.e.dtype == GL_DTYPE_F32 ? 4 : 2;
  const char* row = reinterpret_cast<const char*>(p.e.residual) + (m0 + lane) * p.e.ldr * es;
  const int64_t end = min(p.N, n0 + cols) * es;
  for (int64_t b = n0 * es; b < end; b += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + b));
}

template <int CTAS, int BN, int NPA, bool FULL, int JOBS>
__global__ void __launch_bounds__(kMmThreads, 1)
    mma_kernel(const __grid_constant__ CUtensorMap ta0, const __grid_constant__ CUtensorMap tb0,
               const __grid_constant__ CUtensorMap ta1, const __grid_constant__ CUtensorMap tb1,
               const __grid_constant__ MmaParams p) {
  constexpr int BNC = BN / CTAS, BM = kMmBM * CTAS;
  constexpr bool MULTI = NPA > 1;
  constexpr int NB = 2;                              // accumulator buffers, of one or (MULTI) two accumulators
  constexpr uint32_t kCols = NB * (MULTI ? 2 : 1) * BN;   // TMEM columns
  constexpr int HALF = BN >= 64 ? BN / 2 : BN;        // columns per epilogue warp
  constexpr int kEpi = BN >= 64 ? kMmEpiWarps : 4;    // epilogue warps at work
  extern __shared__ unsigned char mm_raw[];
  __shared__ MmaShared sh;
  const uint32_t pad = ((t5_smem_u32(mm_raw) + 1023u) & ~1023u) - t5_smem_u32(mm_raw);
  const uint32_t smem = t5_smem_u32(mm_raw) + pad;
  float* epi = reinterpret_cast<float*>(mm_raw + pad + kMmRing / 1024 * 1024);
  const uint32_t slot_bytes = p.a_slot + p.b_bytes;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = CTAS == 1 ? 0 : (int)(blockIdx.x & 1);
  if (warp == 9) {
    if constexpr (CTAS == 1) t5_tmem_alloc(t5_smem_u32(&sh.tmem), kCols);
    else t5_tmem_alloc2(t5_smem_u32(&sh.tmem), kCols);
  }
  if (tid == 0) {
    for (int i = 0; i < p.slots; ++i) {
      t5_mbar_init(t5_smem_u32(&sh.full[i]), 1);
      t5_mbar_init(t5_smem_u32(&sh.empty[i]), 1);
    }
    for (int i = 0; i < NB; ++i) {
      t5_mbar_init(t5_smem_u32(&sh.done[i]), 1);
      t5_mbar_init(t5_smem_u32(&sh.free_[i]), kEpi * CTAS);
    }
    t5_mbar_init(t5_smem_u32(&sh.last), 1);
    sh.dead = 0;
    sh.status = p.status;
  }
  __syncwarp();
  t5_fence_before_sync();
  if constexpr (CTAS == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  t5_fence_after_sync();
  const uint32_t tmem = sh.tmem;
  const int64_t items = p.items;
  const int64_t first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (warp == 8) {
    const bool lead = mm_elect();
    MmaRing r(p.slots);
    bool live = true;
    for (int64_t item = first; item < items && live; item += step) {
      const MmaTile t = mm_tile<JOBS>(p, item, BM, BN);
      const MmaOne& o = p.job[JOBS == 1 ? 0 : t.job];
      const CUtensorMap* ta = JOBS == 1 || !t.job ? &ta0 : &ta1;
      const CUtensorMap* tb = JOBS == 1 || !t.job ? &tb0 : &tb1;
      const int a_mn = o.a_mn, b_mn = o.b_mn, npb = o.npb;
      const uint32_t a_bytes = o.a_bytes;
      const int m0 = (int)t.m0 + kMmBM * rank, n0 = (int)t.n0 + BNC * rank;
      for (int kb = t.k0; kb < t.k1 && live; ++kb) {
#pragma unroll
        for (int i = 0; i < NPA; ++i, r.next()) {
          if (r.round && !mm_wait_warp(sh, sh.empty[r.s], (r.round - 1) & 1)) {
            live = false;
            break;
          }
          const uint32_t bar = t5_smem_u32(&sh.full[r.s]);
          uint32_t rbar = bar;                           // the even CTA's barrier of this slot
          const uint32_t a = smem + r.s * slot_bytes, b = a + p.a_slot;
          if constexpr (CTAS == 2) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(rbar) : "r"(bar));
          if (lead) {
            if (rank == 0) mm_expect(bar, CTAS * (a_bytes + (i < npb ? p.b_bytes : 0u)));
            if (a_mn) {
              mm_load<CTAS>(a, ta, m0, kb * kMmBK, i, rbar);
              mm_load<CTAS>(a + 8192, ta, m0 + 64, kb * kMmBK, i, rbar);
            } else {
              mm_load<CTAS>(a, ta, kb * kMmBK, m0, i, rbar);
            }
            if (i < npb) {
              if (BNC >= 64 && b_mn) {
#pragma unroll
                for (int h = 0; h < BNC / 64; ++h)
                  mm_load<CTAS>(b + h * 8192, tb, n0 + 64 * h, kb * kMmBK, i, rbar);
              } else {
                mm_load<CTAS>(b, tb, kb * kMmBK, n0, i, rbar);
              }
            }
          }
          __syncwarp();
        }
      }
    }
    for (int i = 0; i < p.slots && live; ++i)      // every slot given back
      if (r.uses(i)) live = mm_wait_warp(sh, sh.empty[i], (r.uses(i) - 1) & 1);
    if (!live) {   // the copies in flight must land before the shared memory goes away
      if (rank == 0) {
        for (int i = 0; i < p.slots; ++i)
          if (r.uses(i)) t5_mbar_wait(t5_smem_u32(&sh.full[i]), (r.uses(i) - 1) & 1, kMmDrainPolls);
      } else {     // theirs count on the other CTA's barriers: time enough for any copy
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
      }
    }
  } else if (warp == 9) {
    if (rank == 0) {
      const bool lead = mm_elect();
      const uint64_t desc = t5_desc_sw128(smem, 8192, 1024);   // of A in slot 0; the address field counts 16 bytes
      MmaRing r(p.slots);
      uint32_t ch = 0;
      bool live = true;
      auto commit = [&](uint64_t& bar) {
        const uint32_t a = t5_smem_u32(&bar);
        if (lead) {
          if constexpr (CTAS == 1) t5_commit(a);
          else t5_commit_pair(a);
        }
        __syncwarp();
      };
      for (int64_t item = first; item < items && live; item += step) {
        const MmaTile t = mm_tile<JOBS>(p, item, BM, BN);
        const MmaOne& o = p.job[JOBS == 1 ? 0 : t.job];
        const uint32_t idesc = t5_idesc_bf16(BM, BN, 0, 0) | ((uint32_t)o.a_mn << 15) | ((uint32_t)o.b_mn << 16);
        const int npb = o.npb, chunk = o.chunk;
        const uint32_t ka = (o.a_mn ? 2048u : 32u) >> 4, kb_ = (o.b_mn ? 2048u : 32u) >> 4;   // 16-byte units per 16 k
        for (int c0 = t.k0; c0 < t.k1 && live; c0 += chunk, ++ch) {
          const int c1 = min(t.k1, c0 + chunk), buf = ch % NB;
          if (ch >= NB && !mm_wait_warp(sh, sh.free_[buf], (ch / NB - 1) & 1)) {
            live = false;
            break;
          }
          t5_fence_after_sync();
          // one plane: accumulator buf; several: the leading products into one, all others into another
          const uint32_t d = tmem + buf * (MULTI ? 2 : 1) * BN;
          uint32_t acc[2] = {0, 0};
          auto product = [&](int which, int sa, int sb) {   // the plane of A in slot sa by the plane of B in slot sb
            const uint64_t ad = desc + sa * (slot_bytes >> 4);
            const uint64_t bd = desc + (sb * slot_bytes + p.a_slot >> 4);
            if (lead) {
#pragma unroll
              for (int k = 0; k < kMmBK / 16; ++k) {
                if constexpr (CTAS == 1) t5_mma_bf16(d + which * BN, ad + k * ka, bd + k * kb_, idesc, acc[which] | k);
                else t5_mma_bf16_pair(d + which * BN, ad + k * ka, bd + k * kb_, idesc, acc[which] | k);
              }
            }
            acc[which] = 1;
          };
          for (int kb = c0; kb < c1 && live; ++kb) {
            int slot[NPA];
#pragma unroll
            for (int i = 0; i < NPA; ++i, r.next()) {
              slot[i] = r.s;
              if (live && !mm_wait_warp(sh, sh.full[r.s], r.round & 1)) live = false;
              if (!live) continue;
              t5_fence_after_sync();
              if constexpr (NPA == 1) {
                product(0, slot[0], slot[0]);
              } else if (i == 0) {
                product(0, slot[0], slot[0]);
              } else if (i == 1) {
                product(1, slot[1], slot[0]);
                if (npb > 1) {
                  product(1, slot[0], slot[1]);
                  product(1, slot[1], slot[1]);
                }
                commit(sh.empty[slot[1]]);
              } else {
                product(1, slot[2], slot[0]);
                if (npb > 1) product(1, slot[0], slot[2]);
                commit(sh.empty[slot[2]]);
              }
            }
            if (live) commit(sh.empty[slot[0]]);
          }
          if (live) commit(sh.done[buf]);
        }
      }
      if (!live) {   // what has been issued must end before the tensor memory is freed
        commit(sh.last);
        t5_mbar_wait(t5_smem_u32(&sh.last), 0, kMmDrainPolls);
      }
    }
  } else if (warp < kEpi) {
    const int half = warp >> 2;
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    float* tile = epi + warp * 32 * kMmPitch;
    if (p.side.part) {
      for (int64_t n = ((int64_t)blockIdx.x * kEpi + warp) * 32; n < p.side.N; n += (int64_t)gridDim.x * kEpi * 32)
        sum_rows(p.side, n);
    }
    uint32_t ch = 0;
    for (int64_t item = first; item < items; item += step) {
      const MmaTile t = mm_tile<JOBS>(p, item, BM, BN);
      const MmaOne& o = p.job[JOBS == 1 ? 0 : t.job];
      const int64_t m0 = t.m0 + kMmBM * rank + 32 * (warp & 3), n0 = t.n0 + half * HALF;
      float sum[MULTI ? HALF : 1];
      mm_prefetch(o, m0, n0, HALF);
      for (int c0 = t.k0; c0 < t.k1; c0 += o.chunk, ++ch) {
        const int buf = ch % NB;
        const bool ok = mm_wait_warp(sh, sh.done[buf], (ch / NB) & 1);
        t5_fence_after_sync();
        const uint32_t cols = tmem + lane_base + (uint32_t)(buf * (MULTI ? 2 : 1) * BN + half * HALF);
        if constexpr (MULTI) {   // one load for all of the warp's columns: each waits for the MMAs in flight
          static_assert(HALF == 32 || HALF == 64, "columns per warp");
#pragma unroll
          for (int which = 1; which >= 0; --which) {
            float v[HALF];
            if constexpr (HALF == 64) t5_ld64(cols + which * BN, v);
            else t5_ld32(cols + which * BN, v);
            if (which == 0) {
              t5_fence_before_sync();
              __syncwarp();
              if (lane == 0) mm_arrive<CTAS>(t5_smem_u32(&sh.free_[buf]));
            }
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
              if (!ok) v[i] = __int_as_float(0x7FC00000);
              sum[i] = which == 1 && c0 == t.k0 ? v[i] : sum[i] + v[i];
            }
          }
        } else {
#pragma unroll
          for (int q = 0; q < HALF / 32; ++q) {
            float v[32];
            t5_ld32(cols + 32 * q, v);
            if (!ok) {
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __int_as_float(0x7FC00000);
            }
            if (q == HALF / 32 - 1) {                    // the accumulator is read: free it before the stores
              t5_fence_before_sync();
              __syncwarp();
              if (lane == 0) mm_arrive<CTAS>(t5_smem_u32(&sh.free_[buf]));
            }
            if (m0 < o.M && n0 + 32 * q < o.N) mm_store_block<FULL>(o, tile, v, m0, n0 + 32 * q, t.split, c0 > t.k0);
          }
        }
      }
      if constexpr (MULTI) {
#pragma unroll
        for (int q = 0; q < HALF / 32; ++q) {
          if (m0 < o.M && n0 + 32 * q < o.N) mm_store_block<FULL>(o, tile, sum + 32 * q, m0, n0 + 32 * q, t.split, false);
        }
      }
    }
  }
  __syncwarp();
  t5_fence_before_sync();
  if constexpr (CTAS == 1) {
    __syncthreads();
  } else {   // no CTA of a pair leaves while the other may still signal it or use its memory
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  t5_fence_after_sync();
  if (warp == 9) {
    if constexpr (CTAS == 1) t5_tmem_dealloc(tmem, kCols);
    else t5_tmem_dealloc2(tmem, kCols);
  }
}

// Sums the splits of a product in split order and finishes the elements, eight columns per thread (one where rows are
// not aligned).
template <int W>
__global__ void __launch_bounds__(256) mma_join_kernel(const float* part, int64_t M, int64_t N, int splits,
                                                       LinEpilogue e) {
  const int64_t nq = N / W, total = M * nq;
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int64_t m = i / nq, n = (i - m * nq) * W;
    float z[W], t[W];
    ld_span<float, W>(part + m * N + n, true, z);
#pragma unroll 4
    for (int k = 1; k < splits; ++k) {
      ld_span<float, W>(part + (k * M + m) * N + n, true, t);
#pragma unroll
      for (int j = 0; j < W; ++j) z[j] += t[j];
    }
    lin_finish<W>(e, m, n, true, z);
  }
}

// ---- host ----
struct MmaPlan {
  int ctas, BN;
  int splits[2], split_blocks[2];
};

// Tile shape and splits of k: the least estimated time, in clocks of one SM, fitted to measured products (256 x 256
// pairs 610 clocks per 64 k, 128 x 32 tiles 400 however few bytes, epilogues 37 clocks a column).  64 k cost the
// larger of the MMAs (2 BN clocks a term) and the loads (60 bytes a clock into one SM of many), a fifth of the smaller
// and a hand-over; an epilogue runs beside the next item's sum; split sums add their partial tiles' traffic and a
// launch.
static MmaPlan mma_search(const MmaSize* z, int n, int sms) {
  MmaPlan best{};
  double best_t = 1e300;
  struct Shape { int ctas, BN; };
  static const int kSplits[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32};
  for (Shape sh : {Shape{2, 256}, Shape{2, 128}, Shape{1, 128}, Shape{1, 64}, Shape{1, 32}}) {
    bool fits = true;
    for (int j = 0; j < n; ++j) {
      if (sh.BN == 32 && (z[j].b_mn || z[j].npa > 1)) fits = false;
      if (sh.BN == 256 && z[j].npa > 1) fits = false;          // four accumulators fill the tensor memory
    }
    if (!fits) continue;
    const double wide = sms / sh.ctas, epilogue = 800 + sh.BN * 37.0;
    double tiles[2] = {0, 0}, block[2] = {0, 0}, out[2] = {0, 0};
    int64_t kb[2] = {1, 1};
    for (int j = 0; j < n; ++j) {
      const int64_t bm = kMmBM * sh.ctas;
      const int terms = z[j].npa == 1 ? 1 : (z[j].npb == 1 ? 3 : 6);
      const double bytes = z[j].npa * (double)(z[j].M < kMmBM ? z[j].M : kMmBM) * kMmBK * 2 +
                           z[j].npb * (double)(sh.BN / sh.ctas) * kMmBK * 2;
      const double load = bytes / 60.0, mma = terms * 2.0 * sh.BN;
      tiles[j] = (double)((z[j].M + bm - 1) / bm) * (double)((z[j].N + sh.BN - 1) / sh.BN);
      block[j] = (load > mma ? load + 0.2 * mma : mma + 0.2 * load) + 50;
      if (block[j] < 400) block[j] = 400;
      kb[j] = (z[j].K + kMmBK - 1) / kMmBK;
      out[j] = (double)z[j].M * z[j].N;
    }
    for (int s0 : kSplits) {
      if (s0 > kb[0]) break;
      for (int s1 : kSplits) {
        if (s1 > 1 && (n < 2 || s1 > kb[1])) break;
        const int s[2] = {s0, s1};
        bool long_k = false;                                     // one accumulator over too much of it
        for (int j = 0; j < n; ++j)
          if (z[j].npa == 1 && (kb[j] + s[j] - 1) / s[j] > kMmLongest && s[j] < 32) long_k = true;
        if (long_k) continue;
        double sum = 0, longest = 0, extra = 0, items = 0;
        for (int j = 0; j < n; ++j) {
          double t = (double)((kb[j] + s[j] - 1) / s[j]) * block[j];
          if (t < epilogue) t = epilogue;
          sum += tiles[j] * s[j] * t;
          items += tiles[j] * s[j];
          if (t > longest) longest = t;
          if (s[j] > 1) extra += 5000.0 + out[j] * (s[j] + 1) * 4 / 2500.0;
        }
        const double waves = (double)(int64_t)((items + wide - 1) / wide);
        const double even = sum / items * waves;                 // every CTA the same number of items
        const double t = (even > longest ? even : longest) + epilogue + extra + 500.0 * (sh.ctas - 1);
        if (t < best_t) {
          best_t = t;
          best = MmaPlan{sh.ctas, sh.BN, {s0, s1}, {1, 1}};
          for (int j = 0; j < n; ++j) best.split_blocks[j] = (int)((kb[j] + s[j] - 1) / s[j]);
        }
      }
    }
  }
  for (int j = 0; j < n; ++j) {   // no empty splits
    const int64_t kb = (z[j].K + kMmBK - 1) / kMmBK;
    best.splits[j] = (int)((kb + best.split_blocks[j] - 1) / best.split_blocks[j]);
  }
  return best;
}

// mma_search with the last plans of this thread at hand: a search costs more host time than a launch.
static MmaPlan mma_plan(const MmaSize* z, int n, int sms) {
  struct Entry {
    MmaSize z[2];
    int n, sms;
    MmaPlan plan;
  };
  static thread_local Entry cache[64];
  int64_t h = n;
  for (int j = 0; j < n; ++j) h = h * 31 + z[j].M * 17 + z[j].N * 7 + z[j].K * 3 + z[j].npa + 2 * z[j].npb + z[j].b_mn;
  Entry& e = cache[h & 63];
  bool hit = e.n == n && e.sms == sms;
  for (int j = 0; j < n && hit; ++j)
    hit = e.z[j].M == z[j].M && e.z[j].N == z[j].N && e.z[j].K == z[j].K && e.z[j].npa == z[j].npa &&
          e.z[j].npb == z[j].npb && e.z[j].b_mn == z[j].b_mn;
  if (!hit) {
    e.n = n;
    e.sms = sms;
    for (int j = 0; j < n; ++j) e.z[j] = z[j];
    e.plan = mma_search(z, n, sms);
  }
  return e.plan;
}

static int64_t split_bytes(const MmaSize& z, int splits) {
  return splits > 1 ? (4 * splits * z.M * z.N + 255) / 256 * 256 : 0;
}

int64_t mma_work_bytes(const MmaSize* z, int n, int sms) {
  const MmaPlan pl = mma_plan(z, n, sms);
  int64_t bytes = 0;
  for (int j = 0; j < n; ++j) bytes += split_bytes(z[j], pl.splits[j]);
  return bytes;
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
  const auto encode = [&] {
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.ptr), dims, strides, boxes, ones,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {   // a thread whose first CUDA call this is: bind its device's context
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e != cudaSuccess) return set_cuda_error(e);
    r = encode();
  }
  return r == CUDA_SUCCESS ? GL_OK : r == CUDA_ERROR_INVALID_VALUE ? GL_ERR_SHAPE : GL_ERR_DEVICE;
}

template <int CTAS, int BN, int NPA, bool FULL, int JOBS>
static int launch_mma(const CUtensorMap (&map)[4], const MmaParams& p, int sms, cudaStream_t st) {
  const auto kernel = mma_kernel<CTAS, BN, NPA, FULL, JOBS>;
  const size_t smem = kMmRing + kMmEpiBytes + 1024;
  if (int rc = ensure_dynamic_smem((const void*)kernel, smem)) return rc;
  const int64_t most = sms / CTAS;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((p.items < most ? p.items : most) * CTAS));
  cfg.blockDim = dim3(kMmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = CTAS;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = CTAS > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, map[0], map[1], map[2], map[3], p);
  if (e != cudaSuccess) return set_cuda_error(e);
  count_launches(1);
  return GL_OK;
}

template <int NPA, bool FULL, int JOBS>
static int launch_shape(const MmaPlan& pl, const CUtensorMap (&map)[4], const MmaParams& p, int sms, cudaStream_t st) {
  if constexpr (NPA == 1) {
    if (pl.BN == 256) return launch_mma<2, 256, 1, FULL, JOBS>(map, p, sms, st);
    if constexpr (JOBS == 1)                                       // an MN-major B has no 32-wide tiles
      if (pl.BN == 32) return launch_mma<1, 32, 1, FULL, JOBS>(map, p, sms, st);
  }
  if (pl.ctas == 2) return launch_mma<2, 128, NPA, FULL, JOBS>(map, p, sms, st);
  if (pl.BN == 128) return launch_mma<1, 128, NPA, FULL, JOBS>(map, p, sms, st);
  return launch_mma<1, 64, NPA, FULL, JOBS>(map, p, sms, st);
}

template <int NPA>
static int launch_jobs(const MmaPlan& pl, const CUtensorMap (&map)[4], const MmaParams& p, int n, bool full, int sms,
                       cudaStream_t st) {
  if (n == 2) return launch_shape<NPA, false, 2>(pl, map, p, sms, st);   // gradients: no activation
  return full ? launch_shape<NPA, true, 1>(pl, map, p, sms, st) : launch_shape<NPA, false, 1>(pl, map, p, sms, st);
}

static bool aligned16(const void* p, int64_t ld, int esize) {
  return p == nullptr || (((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0);
}

// Every tensor of an epilogue can be accessed in 16-byte pieces.
static bool epilogue_vec(const LinEpilogue& e) {
  const int es = e.dtype == GL_DTYPE_F32 ? 4 : 2;
  const int ss = e.slope_kind == GL_SLOPE_F32 ? 4 : e.slope_kind == GL_SLOPE_I16 ? 2 : 1;
  return aligned16(e.out, e.ldo, es) && aligned16(e.residual, e.ldr, es) && aligned16(e.bias, 0, es) &&
         (ss == 1 ? e.slope == nullptr || (((uintptr_t)e.slope | e.lds) & 7) == 0 : aligned16(e.slope, e.lds, ss));
}

int mma_run(const MmaJob* jobs, int n, const SumRows& side, void* work, int32_t* status, cudaStream_t st) {
  int sms = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  MmaSize z[2];
  for (int j = 0; j < n; ++j) {
    const MmaJob& q = jobs[j];
    if (q.M > 0x7FFFFF00 || q.N > 0x7FFFFF00 || q.K > 0x7FFFFF00) return GL_ERR_SHAPE;
    z[j] = MmaSize{q.M, q.N, q.K, q.a.planes, q.b.planes, q.b.mn};
  }
  const MmaPlan pl = mma_plan(z, n, sms);
  CUtensorMap map[4];
  MmaParams p{};
  bool full = false;
  char* scratch = (char*)work;
  for (int j = 0; j < n; ++j) {
    const MmaJob& q = jobs[j];
    MmaOne& o = p.job[j];
    // a tile of fewer rows than 128 loads those; the rest of the slot stays as it is, for rows of the accumulator that
    // nobody reads
    const int a_rows = q.M < kMmBM && !q.a.mn ? (int)(q.M + 7) / 8 * 8 : kMmBM;
    if (int rc = operand_map(&map[2 * j], q.a, q.M, q.K, a_rows)) return rc;
    if (int rc = operand_map(&map[2 * j + 1], q.b, q.N, q.K, pl.BN / pl.ctas)) return rc;
    o.M = q.M;
    o.N = q.N;
    o.tiles_m = (int)((q.M + kMmBM * pl.ctas - 1) / (kMmBM * pl.ctas));
    o.tiles_n = (int)((q.N + pl.BN - 1) / pl.BN);
    o.kblocks = (int)((q.K + kMmBK - 1) / kMmBK);
    o.splits = pl.splits[j];
    o.split_blocks = pl.split_blocks[j];
    o.a_mn = q.a.mn;
    o.b_mn = q.b.mn;
    o.npb = q.b.planes;
    o.a_bytes = (uint32_t)a_rows * kMmBK * 2;
    o.e = q.e;
    o.vec = epilogue_vec(q.e);
    if (o.splits > 1) {
      if (!work) return GL_ERR_WORKSPACE;
      o.part = (float*)scratch;
      scratch += split_bytes(z[j], o.splits);
      o.vec = q.N % 4 == 0;
    } else if (q.e.bias || q.e.act != GL_ACT_IDENTITY || q.e.slope_kind) {
      full = true;
    }
    // bf16 operands: chunks only where each can be added to fp32 memory, else one (k block numbers stay below 2^25)
    const bool added = o.part != nullptr || (q.e.dtype == GL_DTYPE_F32 && q.e.residual == q.e.out);
    o.chunk = q.a.planes > 1 ? 8 : added ? kMmLongChunk : 1 << 30;
    p.items += (int64_t)o.tiles_m * o.tiles_n * o.splits;
    if (j == 0) p.items0 = p.items;
    if (o.a_bytes > p.a_slot) p.a_slot = o.a_bytes;
  }
  if (n == 1) map[2] = map[3] = map[0];
  p.b_bytes = (uint32_t)(pl.BN / pl.ctas) * kMmBK * 2;
  p.slots = (int)(kMmRing / 1024 * 1024 / (p.a_slot + p.b_bytes));
  if (p.slots > kMmMaxSlots) p.slots = kMmMaxSlots;
  p.side = side;
  p.status = status;
  const int rc = z[0].npa == 1 ? launch_jobs<1>(pl, map, p, n, full, sms, st) : launch_jobs<3>(pl, map, p, n, full, sms, st);
  if (rc) return rc;
  for (int j = 0; j < n; ++j) {
    if (pl.splits[j] == 1) continue;
    const MmaJob& q = jobs[j];
    const bool wide = epilogue_vec(q.e) && q.N % 8 == 0;
    const int64_t units = wide ? q.M * (q.N / 8) : q.M * q.N, need = (units + 255) / 256, cap = 16ll * sms;
    const unsigned blocks = (unsigned)(need < cap ? need : cap);
    if (wide) mma_join_kernel<8><<<blocks, 256, 0, st>>>(p.job[j].part, q.M, q.N, pl.splits[j], q.e);
    else mma_join_kernel<1><<<blocks, 256, 0, st>>>(p.job[j].part, q.M, q.N, pl.splits[j], q.e);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess) return set_cuda_error(err);
    count_launches(1);
  }
  return GL_OK;
}

}  // namespace gl

// Group norm with an affine map and an activation over channels-last tensors x [S, P, C] (S samples, P
// positions, C channels in G groups of cpg = C / G), forward and backward.  No counterpart in the reference.
//
//   mu, var   mean and biased variance of x over a (sample, group)'s m = P cpg elements, rstd = 1 / sqrt(var + eps)
//   y = act(u), u = h gamma + beta, h = (x - mu) rstd
//   backward: du = dy act'(u), q = du gamma,
//   dx = rstd (q - mean(q) - h mean(q h)), dgamma = sum du h, dbeta = sum du
//
// Bound by HBM: forward 2, backward 3 elements of traffic per element, when every input is read once.
// Two families:
//  * resident kernels: a cluster of R <= 8 CTAs owns one (sample, segment of whole groups); each CTA keeps its
//    positions of the segment in shared memory, so the data comes from HBM once, and the group sums cross the
//    cluster through distributed shared memory.  The variance is a second pass over the resident data
//    (sum (x - mu)^2), not a difference of squares.
//  * streaming kernels, for samples that do not fit a cluster's shared memory: per-channel partial statistics of
//    chunks of positions (shifted by the chunk's first value, merged with Chan's formula), a join, and an
//    elementwise pass; x is read twice.
// A thread owns whole 16-byte vectors of channels and walks over positions, so all sums are first per channel:
// group boundaries need no alignment, and with A_c = sum du h, B_c = sum du the backward's group means are
// sum gamma_c A_c / m and sum gamma_c B_c / m.  No atomics: every sum has one order.
#include <cooperative_groups.h>

#include "dense.cuh"

namespace cg = cooperative_groups;

namespace gl {

constexpr int kNormThreads = 256;
constexpr int kNormMaxCluster = 8;

struct NormParams {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  const int8_t* codes;
  const uint8_t* exps;
  void* out;            // y or dx (contiguous)
  float* mean;          // [S, G]
  float* rstd;
  float* part;          // workspace
  int64_t S, P, C, G, cpg, sx, px, sdy, pdy, ldc, nblk;
  int64_t nseg, npart;  // resident: segments per sample; backward: rows of partial dgamma / dbeta
  int64_t PR;           // positions per CTA (resident) or chunk (streaming)
  int64_t chunks;
  int ng, cs, R, pdtype, act;   // act: chosen by the launch (a template argument of the kernels)
  float eps;
};

__device__ __forceinline__ float ld_param(const void* p, int64_t i, int dtype, float none) {
  if (p == nullptr) return none;
  return dtype == GL_DTYPE_F32 ? reinterpret_cast<const float*>(p)[i]
                               : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

// N raw elements (16 bytes, or one element).
template <typename T, int N>
struct Raw {
  uint4 v;
};
template <typename T>
struct Raw<T, 1> {
  T v;
};

template <typename T, int N>
__device__ __forceinline__ void unpack(const Raw<T, N>& r, float (&f)[N]) {
  load_vec<T, N>(reinterpret_cast<const T*>(&r.v), f);
}

// N channels from c on of a row's checkpoint, as the storage type (exact: 7-bit multiples of a power of two).
template <typename T, int N>
__device__ __forceinline__ Raw<T, N> read_codes(const NormParams& p, int64_t row, int64_t c) {
  const float s = act8_scale(p.exps[row * p.nblk + c / kActBlock]);
  const int8_t* q = p.codes + row * p.ldc + c;
  float f[N];
  if constexpr (N == 1) {
    f[0] = (float)*q * s;
  } else {
    uint32_t u[N / 4];
    if constexpr (N == 4) {
      u[0] = *reinterpret_cast<const uint32_t*>(q);
    } else {
      const uint2 t = *reinterpret_cast<const uint2*>(q);
      u[0] = t.x;
      u[N / 4 - 1] = t.y;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)(int8_t)(u[i / 4] >> (8 * (i % 4))) * s;
  }
  Raw<T, N> r;
  store_vec<T, N>(reinterpret_cast<T*>(&r.v), f);
  return r;
}

// x of sample s, position q, channel c on.
template <typename T, int N, bool CKPT>
__device__ __forceinline__ Raw<T, N> read_x(const NormParams& p, int64_t s, int64_t q, int64_t c) {
  if constexpr (CKPT) return read_codes<T, N>(p, s * p.P + q, c);
  else return *reinterpret_cast<const Raw<T, N>*>(reinterpret_cast<const T*>(p.x) + s * p.sx + q * p.px + c);
}

template <typename T, int N>
__device__ __forceinline__ Raw<T, N> read_dy(const NormParams& p, int64_t s, int64_t q, int64_t c) {
  return *reinterpret_cast<const Raw<T, N>*>(reinterpret_cast<const T*>(p.dy) + s * p.sdy + q * p.pdy + c);
}

// gs[g] = sum over the group's channels and the TY rows of red[row * cs + c], for the CTA's ngl groups: a warp
// per group where there is enough to add, else a thread.
__device__ __forceinline__ void group_sums(const float* red, int cs, int rows, int ngl, int cpg, float* gs) {
  const int tid = threadIdx.x, lane = tid & 31;
  if (cpg * rows >= 64) {
    for (int g = tid >> 5; g < ngl; g += kNormThreads / 32) {
      float s = 0.f;
      for (int r = 0; r < rows; ++r)
        for (int c = lane; c < cpg; c += 32) s += red[r * cs + g * cpg + c];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
      if (lane == 0) gs[g] = s;
    }
  } else {
    for (int g = tid; g < ngl; g += kNormThreads) {
      float s = 0.f;
      for (int r = 0; r < rows; ++r)
        for (int c = 0; c < cpg; ++c) s += red[r * cs + g * cpg + c];
      gs[g] = s;
    }
  }
}

// Sum of gs[g] over the cluster's CTAs, in rank order (every CTA computes the same value).
__device__ __forceinline__ float cluster_total(float* gs, int g, int R) {
  if (R == 1) return gs[g];
  cg::cluster_group cl = cg::this_cluster();
  float s = 0.f;
  for (int r = 0; r < R; ++r) s += cl.map_shared_rank(gs, r)[g];
  return s;
}

__device__ __forceinline__ void norm_barrier(int R) {
  if (R == 1) __syncthreads();
  else cg::this_cluster().sync();
}


// ---- resident forward ----
template <typename T, int N, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_fwd_resident(NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  Raw<T, N>* tile = reinterpret_cast<Raw<T, N>*>(smem);
  const int tid = threadIdx.x, R = p.R, rank = blockIdx.x % R, cpg = (int)p.cpg;
  const int64_t item = blockIdx.x / R, s = item / p.nseg;
  const int g0 = (int)(item - s * p.nseg) * p.ng;
  const int ngl = min(p.ng, (int)p.G - g0), csl = ngl * cpg, nv = csl / N;
  const int64_t c0 = (int64_t)g0 * cpg;
  float* red = reinterpret_cast<float*>(smem + (((size_t)p.PR * p.cs * sizeof(T) + 15) & ~(size_t)15));
  float* gs = red + max(p.cs, kNormThreads * N);       // [2][ng]
  float* stat = gs + 2 * p.ng;                         // [2][ng]: mean, rstd
  const int TX = min(nv, kNormThreads), TY = kNormThreads / TX;
  const int tx = tid % TX, ty = tid / TX;
  const int64_t q0 = rank * p.PR;
  const int np = (int)max((int64_t)0, min(p.PR, p.P - q0));
  const float inv_m = 1.f / ((float)p.P * (float)cpg);

  if (ty < TY) {
    for (int col = tx; col < nv; col += TX) {
      float acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      const int64_t c = c0 + (int64_t)col * N;
      int q = ty;
      for (; q + 3 * TY < np; q += 4 * TY) {           // four loads in flight
        Raw<T, N> r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = read_x<T, N, false>(p, s, q0 + q + k * TY, c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          tile[(q + k * TY) * nv + col] = r[k];
          float f[N];
          unpack<T, N>(r[k], f);
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] += f[i];
        }
      }
      for (; q < np; q += TY) {
        const Raw<T, N> r = read_x<T, N, false>(p, s, q0 + q, c);
        tile[q * nv + col] = r;
        float f[N];
        unpack<T, N>(r, f);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += f[i];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) red[ty * csl + col * N + i] = acc[i];
    }
  }
  __syncthreads();
  group_sums(red, csl, TY, ngl, cpg, gs);
  norm_barrier(R);
  for (int g = tid; g < ngl; g += kNormThreads) stat[g] = cluster_total(gs, g, R) * inv_m;
  __syncthreads();

  if (ty < TY) {
    for (int col = tx; col < nv; col += TX) {
      float acc[N], mu[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        acc[i] = 0.f;
        mu[i] = stat[(col * N + i) / cpg];
      }
#pragma unroll 4
      for (int q = ty; q < np; q += TY) {
        float f[N];
        unpack<T, N>(tile[q * nv + col], f);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += (f[i] - mu[i]) * (f[i] - mu[i]);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) red[ty * csl + col * N + i] = acc[i];
    }
  }
  __syncthreads();
  group_sums(red, csl, TY, ngl, cpg, gs + p.ng);
  norm_barrier(R);
  for (int g = tid; g < ngl; g += kNormThreads) {
    const float rs = 1.f / sqrtf(cluster_total(gs + p.ng, g, R) * inv_m + p.eps);
    stat[p.ng + g] = rs;
    if (rank == 0) {
      p.mean[s * p.G + g0 + g] = stat[g];
      p.rstd[s * p.G + g0 + g] = rs;
    }
  }
  norm_barrier(R);                                     // peers are done with this CTA's gs; stat is visible

  if (ty < TY) {
    T* out = reinterpret_cast<T*>(p.out);
    for (int col = tx; col < nv; col += TX) {
      float mul[N], sub[N], bet[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int cl = col * N + i, g = cl / cpg;
        mul[i] = stat[p.ng + g] * ld_param(p.w, c0 + cl, p.pdtype, 1.f);
        sub[i] = stat[g];
        bet[i] = ld_param(p.b, c0 + cl, p.pdtype, 0.f);
      }
#pragma unroll 2
      for (int q = ty; q < np; q += TY) {
        float f[N];
        unpack<T, N>(tile[q * nv + col], f);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = dense_act<ACT, sizeof(T) == 2>(fmaf(f[i] - sub[i], mul[i], bet[i]));
        store_vec<T, N>(out + (s * p.P + q0 + q) * p.C + c0 + (int64_t)col * N, f);
      }
    }
  }
}

// ---- backward, resident ----
// A cluster keeps one segment and walks over samples, adding its dgamma / dbeta in shared memory; one partial
// row per CTA goes to the join.
template <typename T, int N, int ACT, bool CKPT>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_resident(NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const size_t tbytes = ((size_t)p.PR * p.cs * sizeof(T) + 15) & ~(size_t)15;
  Raw<T, N>* xt = reinterpret_cast<Raw<T, N>*>(smem);
  Raw<T, N>* dt = reinterpret_cast<Raw<T, N>*>(smem + tbytes);
  const int tid = threadIdx.x, R = p.R, rank = blockIdx.x % R, cpg = (int)p.cpg;
  const int64_t cluster = blockIdx.x / R, walkers = (gridDim.x / R) / p.nseg, walker = cluster / p.nseg;
  const int g0 = (int)(cluster - walker * p.nseg) * p.ng;
  const int ngl = min(p.ng, (int)p.G - g0), csl = ngl * cpg, nv = csl / N;
  const int64_t c0 = (int64_t)g0 * cpg;
  const int rf = max(p.cs, kNormThreads * N);
  float* ra = reinterpret_cast<float*>(smem + 2 * tbytes);   // sum du h per channel
  float* rb = ra + rf;                                       // sum du per channel
  float* da = rb + rf;                                       // dgamma, dbeta of this CTA
  float* db = da + p.cs;
  float* gs = db + p.cs;                                     // [2 parities][2][ng]
  float* stat = gs + 4 * p.ng;                               // [2][ng]: mean(q), mean(q h)
  const int TX = min(nv, kNormThreads), TY = kNormThreads / TX;
  const int tx = tid % TX, ty = tid / TX;
  const int64_t q0 = rank * p.PR;
  const int np = (int)max((int64_t)0, min(p.PR, p.P - q0));
  const float inv_m = 1.f / ((float)p.P * (float)cpg);
  for (int c = tid; c < csl; c += kNormThreads) da[c] = db[c] = 0.f;
  int par = 0;
  for (int64_t s = walker; s < p.S; s += walkers, par ^= 1) {
    float* gsp = gs + par * 2 * p.ng;
    if (ty < TY) {
      for (int col = tx; col < nv; col += TX) {
        float aa[N], ab[N], mul[N], sub[N], gam[N], bet[N];
        const int64_t c = c0 + (int64_t)col * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int64_t g = s * p.G + g0 + (col * N + i) / cpg;
          aa[i] = ab[i] = 0.f;
          mul[i] = p.rstd[g];
          sub[i] = p.mean[g];
          gam[i] = ld_param(p.w, c + i, p.pdtype, 1.f);
          bet[i] = ld_param(p.b, c + i, p.pdtype, 0.f);
        }
        for (int q = ty; q < np; q += 2 * TY) {
          Raw<T, N> rx[2], rd[2];
          const bool two = q + TY < np;
          rx[0] = read_x<T, N, CKPT>(p, s, q0 + q, c);
          rd[0] = read_dy<T, N>(p, s, q0 + q, c);
          if (two) {
            rx[1] = read_x<T, N, CKPT>(p, s, q0 + q + TY, c);
            rd[1] = read_dy<T, N>(p, s, q0 + q + TY, c);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (k == 1 && !two) break;
            xt[(q + k * TY) * nv + col] = rx[k];
            dt[(q + k * TY) * nv + col] = rd[k];
            float f[N], d[N];
            unpack<T, N>(rx[k], f);
            unpack<T, N>(rd[k], d);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float h = (f[i] - sub[i]) * mul[i];
              const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(h, gam[i], bet[i]));
              aa[i] = fmaf(du, h, aa[i]);
              ab[i] += du;
            }
          }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          ra[ty * csl + col * N + i] = aa[i];
          rb[ty * csl + col * N + i] = ab[i];
        }
      }
    }
    __syncthreads();
    for (int c = tid; c < csl; c += kNormThreads) {
      float a = 0.f, b = 0.f;
      for (int r = 0; r < TY; ++r) {
        a += ra[r * csl + c];
        b += rb[r * csl + c];
      }
      da[c] += a;
      db[c] += b;
      const float gam = ld_param(p.w, c0 + c, p.pdtype, 1.f);
      ra[c] = a * gam;
      rb[c] = b * gam;
    }
    __syncthreads();
    group_sums(rb, csl, 1, ngl, cpg, gsp);
    group_sums(ra, csl, 1, ngl, cpg, gsp + p.ng);
    norm_barrier(R);
    for (int g = tid; g < 2 * ngl; g += kNormThreads) {
      const int k = g / ngl, gg = g - k * ngl;
      stat[k * p.ng + gg] = cluster_total(gsp + k * p.ng, gg, R) * inv_m;
    }
    __syncthreads();
    if (ty < TY) {
      T* out = reinterpret_cast<T*>(p.out);
      for (int col = tx; col < nv; col += TX) {
        float mul[N], sub[N], gam[N], bet[N], m1[N], m2[N];
        const int64_t c = c0 + (int64_t)col * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int gl_ = (col * N + i) / cpg;
          const int64_t g = s * p.G + g0 + gl_;
          mul[i] = p.rstd[g];
          sub[i] = p.mean[g];
          gam[i] = ld_param(p.w, c + i, p.pdtype, 1.f);
          bet[i] = ld_param(p.b, c + i, p.pdtype, 0.f);
          m1[i] = stat[gl_];
          m2[i] = stat[p.ng + gl_];
        }
        for (int q = ty; q < np; q += TY) {
          float f[N], d[N];
          unpack<T, N>(xt[q * nv + col], f);
          unpack<T, N>(dt[q * nv + col], d);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float h = (f[i] - sub[i]) * mul[i];
            const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(h, gam[i], bet[i]));
            f[i] = mul[i] * (fmaf(du, gam[i], -m1[i]) - h * m2[i]);
          }
          store_vec<T, N>(out + (s * p.P + q0 + q) * p.C + c, f);
        }
      }
    }
    __syncthreads();                                   // ra / rb / stat / tiles free; gs alternates by parity
  }
  float* row = p.part + ((walker * R + rank) * 2) * p.C + c0;
  for (int c = tid; c < csl; c += kNormThreads) {
    row[c] = da[c];
    row[p.C + c] = db[c];
  }
  norm_barrier(R);                                     // no CTA leaves while a peer may still read its gs
}

// ---- streaming kernels ----
// Thread mapping of a chunk: blockDim 256 = TX vectors x TY positions; channel segments of 256 vectors.
struct ChunkAt {
  int64_t s, q0, c;
  int np, TY, ty, tx, TX;
  bool live;
};

template <int N>
__device__ __forceinline__ ChunkAt chunk_at(const NormParams& p) {
  ChunkAt a;
  const int64_t nv = p.C / N, segs = (nv + kNormThreads - 1) / kNormThreads;
  const int64_t seg = blockIdx.x % segs, sc = blockIdx.x / segs;
  a.s = sc / p.chunks;
  a.q0 = (sc - a.s * p.chunks) * p.PR;
  a.np = (int)min(p.PR, p.P - a.q0);
  const int64_t left = nv - seg * kNormThreads;
  a.TX = (int)min((int64_t)kNormThreads, left);
  a.TY = kNormThreads / a.TX;
  a.tx = threadIdx.x % a.TX;
  a.ty = threadIdx.x / a.TX;
  a.c = (seg * kNormThreads + a.tx) * N;
  a.live = a.ty < a.TY;
  return a;
}

// part[(s chunks + chunk) C + c] = (mean, sum of squared deviations) of the chunk's values of channel c.
template <typename T, int N>
__global__ void __launch_bounds__(kNormThreads) norm_stats_kernel(NormParams p) {
  __shared__ float r1[kNormThreads * N], r2[kNormThreads * N];
  const ChunkAt a = chunk_at<N>(p);
  float k0[N], s1[N], s2[N];
  if (a.live) {
    unpack<T, N>(read_x<T, N, false>(p, a.s, a.q0, a.c), k0);
#pragma unroll
    for (int i = 0; i < N; ++i) s1[i] = s2[i] = 0.f;
#pragma unroll 4
    for (int q = a.ty; q < a.np; q += a.TY) {
      float f[N];
      unpack<T, N>(read_x<T, N, false>(p, a.s, a.q0 + q, a.c), f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = f[i] - k0[i];
        s1[i] += d;
        s2[i] = fmaf(d, d, s2[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      r1[(a.ty * a.TX + a.tx) * N + i] = s1[i];
      r2[(a.ty * a.TX + a.tx) * N + i] = s2[i];
    }
  }
  __syncthreads();
  if (a.live && a.ty == 0) {
    float2* out = reinterpret_cast<float2*>(p.part) + (a.s * p.chunks + a.q0 / p.PR) * p.C + a.c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t1 = 0.f, t2 = 0.f;
      for (int r = 0; r < a.TY; ++r) {
        t1 += r1[(r * a.TX + a.tx) * N + i];
        t2 += r2[(r * a.TX + a.tx) * N + i];
      }
      const float dm = t1 / (float)a.np;
      out[i] = make_float2(k0[i] + dm, fmaxf(t2 - dm * t1, 0.f));
    }
  }
}

// mean and rstd of each (sample, group) from the chunks' channel statistics (one block each).
__global__ void __launch_bounds__(kNormThreads) norm_stats_join_kernel(NormParams p) {
  __shared__ float red[kNormThreads / 32 + 1];
  const int64_t s = blockIdx.x / p.G, g = blockIdx.x % p.G, n = p.chunks * p.cpg;
  const float2* part = reinterpret_cast<const float2*>(p.part) + s * p.chunks * p.C + g * p.cpg;
  const float m = (float)p.P * (float)p.cpg;
  auto total = [&](float v) {
    __syncthreads();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float t = 0.f;
    for (int i = 0; i < kNormThreads / 32; ++i) t += red[i];
    return t;
  };
  float v = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += kNormThreads) {
    const int64_t ch = i / p.cpg;
    v += part[ch * p.C + (i - ch * p.cpg)].x * (float)min(p.PR, p.P - ch * p.PR);
  }
  const float mu = total(v) / m;
  v = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += kNormThreads) {
    const int64_t ch = i / p.cpg;
    const float2 t = part[ch * p.C + (i - ch * p.cpg)];
    v += t.y + (t.x - mu) * (t.x - mu) * (float)min(p.PR, p.P - ch * p.PR);
  }
  const float var = total(v) / m;
  if (threadIdx.x == 0) {
    p.mean[blockIdx.x] = mu;
    p.rstd[blockIdx.x] = 1.f / sqrtf(var + p.eps);
  }
}

template <typename T, int N, int ACT>
__global__ void __launch_bounds__(kNormThreads) norm_apply_kernel(NormParams p) {
  const ChunkAt a = chunk_at<N>(p);
  if (!a.live) return;
  float mul[N], sub[N], bet[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t g = a.s * p.G + (a.c + i) / p.cpg;
    mul[i] = p.rstd[g] * ld_param(p.w, a.c + i, p.pdtype, 1.f);
    sub[i] = p.mean[g];
    bet[i] = ld_param(p.b, a.c + i, p.pdtype, 0.f);
  }
  T* out = reinterpret_cast<T*>(p.out);
#pragma unroll 4
  for (int q = a.ty; q < a.np; q += a.TY) {
    float f[N];
    unpack<T, N>(read_x<T, N, false>(p, a.s, a.q0 + q, a.c), f);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = dense_act<ACT, sizeof(T) == 2>(fmaf(f[i] - sub[i], mul[i], bet[i]));
    store_vec<T, N>(out + (a.s * p.P + a.q0 + q) * p.C + a.c, f);
  }
}

// Per chunk and channel: dgamma and dbeta partials, part[((s chunks + chunk) 2 + {0, 1}) C + c].
template <typename T, int N, int ACT, bool CKPT>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_stats_kernel(NormParams p) {
  __shared__ float r1[kNormThreads * N], r2[kNormThreads * N];
  const ChunkAt a = chunk_at<N>(p);
  if (a.live) {
    float s1[N], s2[N], mul[N], sub[N], gam[N], bet[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int64_t g = a.s * p.G + (a.c + i) / p.cpg;
      s1[i] = s2[i] = 0.f;
      mul[i] = p.rstd[g];
      sub[i] = p.mean[g];
      gam[i] = ld_param(p.w, a.c + i, p.pdtype, 1.f);
      bet[i] = ld_param(p.b, a.c + i, p.pdtype, 0.f);
    }
#pragma unroll 2
    for (int q = a.ty; q < a.np; q += a.TY) {
      float f[N], d[N];
      unpack<T, N>(read_x<T, N, CKPT>(p, a.s, a.q0 + q, a.c), f);
      unpack<T, N>(read_dy<T, N>(p, a.s, a.q0 + q, a.c), d);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float h = (f[i] - sub[i]) * mul[i];
        const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(h, gam[i], bet[i]));
        s1[i] = fmaf(du, h, s1[i]);
        s2[i] += du;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      r1[(a.ty * a.TX + a.tx) * N + i] = s1[i];
      r2[(a.ty * a.TX + a.tx) * N + i] = s2[i];
    }
  }
  __syncthreads();
  if (a.live && a.ty == 0) {
    float* out = p.part + (a.s * p.chunks + a.q0 / p.PR) * 2 * p.C + a.c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t1 = 0.f, t2 = 0.f;
      for (int r = 0; r < a.TY; ++r) {
        t1 += r1[(r * a.TX + a.tx) * N + i];
        t2 += r2[(r * a.TX + a.tx) * N + i];
      }
      out[i] = t1;
      out[p.C + i] = t2;
    }
  }
}

// coef[(s G + g) 2] = mean(q), mean(q h) of each (sample, group); coef follows the partials.
__global__ void __launch_bounds__(kNormThreads) norm_bwd_join_kernel(NormParams p, float* coef) {
  __shared__ float red[2 * (kNormThreads / 32)];
  const int64_t s = blockIdx.x / p.G, g = blockIdx.x % p.G, n = p.chunks * p.cpg;
  const float m = (float)p.P * (float)p.cpg;
  float va = 0.f, vb = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += kNormThreads) {
    const int64_t ch = i / p.cpg, c = g * p.cpg + (i - ch * p.cpg);
    const float* row = p.part + (s * p.chunks + ch) * 2 * p.C + c;
    const float gam = ld_param(p.w, c, p.pdtype, 1.f);
    va = fmaf(row[0], gam, va);
    vb = fmaf(row[p.C], gam, vb);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    va += __shfl_xor_sync(kFullMask, va, o);
    vb += __shfl_xor_sync(kFullMask, vb, o);
  }
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = va;
    red[kNormThreads / 32 + (threadIdx.x >> 5)] = vb;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    va = vb = 0.f;
    for (int i = 0; i < kNormThreads / 32; ++i) {
      va += red[i];
      vb += red[kNormThreads / 32 + i];
    }
    coef[blockIdx.x * 2] = vb / m;
    coef[blockIdx.x * 2 + 1] = va / m;
  }
}

template <typename T, int N, int ACT, bool CKPT>
__global__ void __launch_bounds__(kNormThreads) norm_bwd_apply_kernel(NormParams p, const float* coef) {
  const ChunkAt a = chunk_at<N>(p);
  if (!a.live) return;
  float mul[N], sub[N], gam[N], bet[N], m1[N], m2[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int64_t g = a.s * p.G + (a.c + i) / p.cpg;
    mul[i] = p.rstd[g];
    sub[i] = p.mean[g];
    m1[i] = coef[2 * g];
    m2[i] = coef[2 * g + 1];
    gam[i] = ld_param(p.w, a.c + i, p.pdtype, 1.f);
    bet[i] = ld_param(p.b, a.c + i, p.pdtype, 0.f);
  }
  T* out = reinterpret_cast<T*>(p.out);
#pragma unroll 2
  for (int q = a.ty; q < a.np; q += a.TY) {
    float f[N], d[N];
    unpack<T, N>(read_x<T, N, CKPT>(p, a.s, a.q0 + q, a.c), f);
    unpack<T, N>(read_dy<T, N>(p, a.s, a.q0 + q, a.c), d);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float h = (f[i] - sub[i]) * mul[i];
      const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(h, gam[i], bet[i]));
      f[i] = mul[i] * (fmaf(du, gam[i], -m1[i]) - h * m2[i]);
    }
    store_vec<T, N>(out + (a.s * p.P + a.q0 + q) * p.C + a.c, f);
  }
}

// dgamma / dbeta = the partial rows' sums in row order; 32 channels per block, 8 row lanes.
__global__ void __launch_bounds__(256) norm_param_join_kernel(const float* part, int64_t rows, int64_t C, void* dw,
                                                              void* db, int pdtype, int accumulate) {
  __shared__ float red[8][2][33];
  const int lane = threadIdx.x & 31, r0 = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float a = 0.f, b = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int64_t r = r0; r < rows; r += 8) {
      a += part[r * 2 * C + c];
      b += part[r * 2 * C + C + c];
    }
  }
  red[r0][0][lane] = a;
  red[r0][1][lane] = b;
  __syncthreads();
  if (r0 < 2 && c < C) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) t += red[r][r0][lane];
    void* out = r0 == 0 ? dw : db;
    if (out != nullptr) {
      if (accumulate) reinterpret_cast<float*>(out)[c] += t;
      else if (pdtype == GL_DTYPE_F32) reinterpret_cast<float*>(out)[c] = t;
      else reinterpret_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(t);
    }
  }
}

// ---- host ----
struct NormPlan {
  bool resident;
  int N, ng, cs, R;
  int64_t nseg, PR, chunks, walkers, npart;
  size_t smem;
};

// Segments of whole groups, cluster size and positions per CTA; falls back to streaming where a segment does
// not fit kNormMaxCluster CTAs.  A segment is at least 128 bytes of channels (a full line per position), wider
// while there are more than four segments for each SM, and its vectors must not straddle segments.
static NormPlan norm_plan(int64_t S, int64_t P, int64_t C, int64_t G, int esize, bool vec, bool bwd, int sms,
                          int smem_max) {
  NormPlan pl{};
  const int64_t cpg = C / G;
  pl.N = vec ? 16 / esize : 1;
  const int tiles = bwd ? 2 : 1;
  auto fixed = [&](int64_t cs, int64_t ng) -> int64_t {      // floats beside the tiles
    const int64_t red = cs > kNormThreads * pl.N ? cs : (int64_t)kNormThreads * pl.N;
    return 4 * (bwd ? 2 * red + 2 * cs + 6 * ng : red + 4 * ng) + 32;
  };
  int64_t ng = 1;
  while (ng < G && (ng * cpg) % pl.N) ++ng;
  const int64_t unit = ng;
  while (ng + unit <= G && ng * cpg * esize < 128) ng += unit;
  if (ng > G || (ng * cpg) % pl.N) ng = G;
  while (ng * 2 <= G && S * ((G + 2 * ng - 1) / (2 * ng)) >= 4 * sms && P * ng * 2 * cpg * esize * tiles <= 32768) ng *= 2;
  for (int64_t cap : {(int64_t)(smem_max / 2 - 1024), (int64_t)smem_max}) {
    for (int R = 1; R <= kNormMaxCluster; R *= 2) {
      const int64_t PR = (P + R - 1) / R, cs = ng * cpg;
      if (cs > (1 << 20) || PR > (1 << 20)) continue;
      const int64_t bytes = tiles * ((PR * cs * esize + 15) / 16 * 16) + fixed(cs, ng);
      if (bytes > cap) continue;
      pl.resident = true;
      pl.ng = (int)ng;
      pl.cs = (int)cs;
      pl.R = R;
      pl.PR = PR;
      pl.nseg = (G + ng - 1) / ng;
      pl.smem = (size_t)bytes;
      const int64_t per_sm = cap == smem_max ? 1 : (smem_max + 1024) / (bytes + 1024) > 8 ? 8 : (smem_max + 1024) / (bytes + 1024);
      const int64_t want = (sms * per_sm + R * pl.nseg - 1) / (R * pl.nseg);
      pl.walkers = S < want ? S : want;
      pl.npart = pl.walkers * R;
      return pl;
    }
  }
  // streaming: about 8 blocks per SM, at least 32 positions each
  const int64_t segs = (C / pl.N + kNormThreads - 1) / kNormThreads;
  int64_t chunks = (8 * (int64_t)sms + S * segs - 1) / (S * segs);
  const int64_t most = (P + 31) / 32;
  if (chunks > most) chunks = most;
  pl.PR = (P + chunks - 1) / chunks;
  pl.chunks = (P + pl.PR - 1) / pl.PR;
  pl.npart = S * pl.chunks;
  return pl;
}

static int norm_checks(int64_t S, int64_t P, int64_t C, int64_t G, int dtype, int pdtype, int act) {
  if (S < 0 || P < 0 || C < 1 || G < 1 || C % G) return GL_ERR_SHAPE;
  if ((dtype != GL_DTYPE_F32 && dtype != GL_DTYPE_BF16) || (pdtype != GL_DTYPE_F32 && pdtype != GL_DTYPE_BF16) ||
      act < GL_ACT_IDENTITY || act > GL_ACT_SILU)
    return GL_ERR_UNSUPPORTED;
  return GL_OK;
}

static bool vec_rows(const void* p, int64_t a, int64_t b, int64_t C, int esize) {
  return ((uintptr_t)p & 15) == 0 && (a * esize) % 16 == 0 && (b * esize) % 16 == 0 && (C * esize) % 16 == 0;
}

template <typename K>
static int launch_cluster(K kernel, const NormParams& p, int64_t blocks, int R, size_t smem, cudaStream_t st) {
  if (blocks > 0x7FFFFFFF) return GL_ERR_SHAPE;
  if (int rc = ensure_dynamic_smem((const void*)kernel, smem)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kNormThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)R;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return set_cuda_error(e);
  count_launches(1);
  return GL_OK;
}

static int launched(int n) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e);
  count_launches(n);
  return GL_OK;
}

template <typename T, int N, int ACT>
static int run_norm_fwd_act(NormParams& p, const NormPlan& pl, cudaStream_t st) {
  if (pl.resident) return launch_cluster(norm_fwd_resident<T, N, ACT>, p, p.S * pl.nseg * pl.R, pl.R, pl.smem, st);
  const int64_t segs = (p.C / N + kNormThreads - 1) / kNormThreads, blocks = p.S * pl.chunks * segs;
  if (blocks > 0x7FFFFFFF || p.S * p.G > 0x7FFFFFFF) return GL_ERR_SHAPE;
  norm_stats_kernel<T, N><<<(unsigned)blocks, kNormThreads, 0, st>>>(p);
  norm_stats_join_kernel<<<(unsigned)(p.S * p.G), kNormThreads, 0, st>>>(p);
  norm_apply_kernel<T, N, ACT><<<(unsigned)blocks, kNormThreads, 0, st>>>(p);
  return launched(3);
}

template <typename T, int N>
static int run_norm_fwd(NormParams& p, const NormPlan& pl, cudaStream_t st) {
  int rc = GL_ERR_UNSUPPORTED;
  with_act(p.act, [&](auto tag) { rc = run_norm_fwd_act<T, N, decltype(tag)::value>(p, pl, st); });
  return rc;
}

template <typename T, int N, int ACT, bool CKPT>
static int run_norm_bwd_act(NormParams& p, const NormPlan& pl, const GlNormBwdArgs& a, cudaStream_t st) {
  if (pl.resident) {
    if (int rc = launch_cluster(norm_bwd_resident<T, N, ACT, CKPT>, p, pl.walkers * pl.nseg * pl.R, pl.R, pl.smem, st))
      return rc;
  } else {
    const int64_t segs = (p.C / N + kNormThreads - 1) / kNormThreads, blocks = p.S * pl.chunks * segs;
    if (blocks > 0x7FFFFFFF || p.S * p.G > 0x7FFFFFFF) return GL_ERR_SHAPE;
    float* coef = p.part + pl.npart * 2 * p.C;
    norm_bwd_stats_kernel<T, N, ACT, CKPT><<<(unsigned)blocks, kNormThreads, 0, st>>>(p);
    norm_bwd_join_kernel<<<(unsigned)(p.S * p.G), kNormThreads, 0, st>>>(p, coef);
    norm_bwd_apply_kernel<T, N, ACT, CKPT><<<(unsigned)blocks, kNormThreads, 0, st>>>(p, coef);
    if (int rc = launched(3)) return rc;
  }
  if (!a.dw && !a.db) return GL_OK;
  norm_param_join_kernel<<<(unsigned)((p.C + 31) / 32), 256, 0, st>>>(p.part, pl.npart, p.C, a.dw, a.db, a.pdtype,
                                                                     a.accumulate);
  return launched(1);
}

template <typename T, int N, bool CKPT>
static int run_norm_bwd(NormParams& p, const NormPlan& pl, const GlNormBwdArgs& a, cudaStream_t st) {
  int rc = GL_ERR_UNSUPPORTED;
  with_act(p.act, [&](auto tag) { rc = run_norm_bwd_act<T, N, decltype(tag)::value, CKPT>(p, pl, a, st); });
  return rc;
}

// Zero parameter gradients of an empty batch (nothing is added to accumulated ones).
static int zero_params(const GlNormBwdArgs& a, cudaStream_t st) {
  if (a.accumulate) return GL_OK;
  const size_t n = (size_t)a.C * (a.pdtype == GL_DTYPE_F32 ? 4 : 2);
  for (void* q : {a.dw, a.db}) {
    if (!q) continue;
    const cudaError_t e = cudaMemsetAsync(q, 0, n, st);
    if (e != cudaSuccess) return set_cuda_error(e);
  }
  return GL_OK;
}

}  // namespace gl

using namespace gl;

extern "C" int64_t gl_norm_work_bytes(int64_t S, int64_t P, int64_t C, int64_t G, int32_t dtype, int32_t backward) {
  if (S < 0 || P < 0 || C < 1 || G < 1 || C % G || (dtype != GL_DTYPE_F32 && dtype != GL_DTYPE_BF16))
    return GL_ERR_SHAPE;
  if (S == 0 || P == 0) return 0;
  int sms = 0, smem = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (int rc = device_smem_optin(&smem)) return rc;
  const int esize = dtype == GL_DTYPE_F32 ? 4 : 2;
  int64_t most = 0;
  for (int vec = 0; vec < 2; ++vec) {     // the call's alignment decides which of the two plans runs
    if (vec && (C * esize) % 16) continue;
    const NormPlan pl = norm_plan(S, P, C, G, esize, vec, backward != 0, sms, smem);
    const int64_t n = backward ? 4 * (pl.npart * 2 * C + (pl.resident ? 0 : 2 * S * G))
                               : (pl.resident ? 0 : 8 * S * pl.chunks * C);
    if (n > most) most = n;
  }
  return most;
}

extern "C" int gl_norm_fwd(const GlNormArgs* args, void* stream) {
  if (!args) return GL_ERR_NULL;
  const GlNormArgs& a = *args;
  if (int rc = norm_checks(a.S, a.P, a.C, a.G, a.dtype, a.pdtype, a.act)) return rc;
  if (a.px < a.C || a.sx < 0) return GL_ERR_SHAPE;
  if (a.S == 0 || a.P == 0) return GL_OK;
  if (!a.x || !a.y || !a.mean || !a.rstd) return GL_ERR_NULL;
  int sms = 0, smem = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (int rc = device_smem_optin(&smem)) return rc;
  const int esize = a.dtype == GL_DTYPE_F32 ? 4 : 2;
  const bool vec = vec_rows(a.x, a.sx, a.px, a.C, esize) && vec_rows(a.y, 0, 0, a.C, esize);
  const NormPlan pl = norm_plan(a.S, a.P, a.C, a.G, esize, vec, false, sms, smem);
  if (!pl.resident && (!a.work || a.work_bytes < 8 * a.S * pl.chunks * a.C)) return GL_ERR_WORKSPACE;
  NormParams p{};
  p.x = a.x; p.w = a.w; p.b = a.b; p.out = a.y; p.mean = a.mean; p.rstd = a.rstd; p.part = (float*)a.work;
  p.S = a.S; p.P = a.P; p.C = a.C; p.G = a.G; p.cpg = a.C / a.G; p.sx = a.sx; p.px = a.px;
  p.nseg = pl.nseg; p.PR = pl.PR; p.chunks = pl.chunks; p.ng = pl.ng; p.cs = pl.cs; p.R = pl.R;
  p.pdtype = a.pdtype; p.act = a.act; p.eps = a.eps;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.dtype == GL_DTYPE_F32) return vec ? run_norm_fwd<float, 4>(p, pl, st) : run_norm_fwd<float, 1>(p, pl, st);
  return vec ? run_norm_fwd<__nv_bfloat16, 8>(p, pl, st) : run_norm_fwd<__nv_bfloat16, 1>(p, pl, st);
}

extern "C" int gl_norm_bwd(const GlNormBwdArgs* args, void* stream) {
  if (!args) return GL_ERR_NULL;
  const GlNormBwdArgs& a = *args;
  if (int rc = norm_checks(a.S, a.P, a.C, a.G, a.dtype, a.pdtype, a.act)) return rc;
  const bool ckpt = a.codes != nullptr;
  if ((!ckpt && (a.px < a.C || a.sx < 0)) || a.pdy < a.C || a.sdy < 0) return GL_ERR_SHAPE;
  const int64_t nblk = (a.C + kActBlock - 1) / kActBlock;
  if (ckpt && (a.ldc < nblk * kActBlock || a.ldc % kActBlock)) return GL_ERR_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.S == 0 || a.P == 0) return zero_params(a, st);
  if (!a.dy || !a.dx || !a.mean || !a.rstd || (!ckpt && !a.x) || (ckpt && !a.exps) || !a.work) return GL_ERR_NULL;
  if (ckpt && ((uintptr_t)a.codes & 15)) return GL_ERR_ALIGN;
  int sms = 0, smem = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (int rc = device_smem_optin(&smem)) return rc;
  const int esize = a.dtype == GL_DTYPE_F32 ? 4 : 2;
  const bool vec = (ckpt || vec_rows(a.x, a.sx, a.px, a.C, esize)) && vec_rows(a.dy, a.sdy, a.pdy, a.C, esize) &&
                   vec_rows(a.dx, 0, 0, a.C, esize);
  const NormPlan pl = norm_plan(a.S, a.P, a.C, a.G, esize, vec, true, sms, smem);
  if (a.work_bytes < 4 * (pl.npart * 2 * a.C + (pl.resident ? 0 : 2 * a.S * a.G))) return GL_ERR_WORKSPACE;
  NormParams p{};
  p.x = a.x; p.dy = a.dy; p.w = a.w; p.b = a.b; p.codes = a.codes; p.exps = a.exps; p.out = a.dx;
  p.mean = const_cast<float*>(a.mean); p.rstd = const_cast<float*>(a.rstd); p.part = (float*)a.work;
  p.S = a.S; p.P = a.P; p.C = a.C; p.G = a.G; p.cpg = a.C / a.G; p.sx = a.sx; p.px = a.px; p.sdy = a.sdy;
  p.pdy = a.pdy; p.ldc = a.ldc; p.nblk = nblk; p.nseg = pl.nseg; p.npart = pl.npart; p.PR = pl.PR;
  p.chunks = pl.chunks; p.ng = pl.ng; p.cs = pl.cs; p.R = pl.R; p.pdtype = a.pdtype; p.act = a.act;
  if (a.dtype == GL_DTYPE_F32) {
    if (ckpt) return vec ? run_norm_bwd<float, 4, true>(p, pl, a, st) : run_norm_bwd<float, 1, true>(p, pl, a, st);
    return vec ? run_norm_bwd<float, 4, false>(p, pl, a, st) : run_norm_bwd<float, 1, false>(p, pl, a, st);
  }
  using B = __nv_bfloat16;
  if (ckpt) return vec ? run_norm_bwd<B, 8, true>(p, pl, a, st) : run_norm_bwd<B, 1, true>(p, pl, a, st);
  return vec ? run_norm_bwd<B, 8, false>(p, pl, a, st) : run_norm_bwd<B, 1, false>(p, pl, a, st);
}

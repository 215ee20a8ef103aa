// Group norm with an affine map and an activation over channels-last tensors x [S, P, C] (S samples, P
// positions, C channels in G groups of cpg = C / G), forward and backward.  No counterpart in the reference.
//
//   mu, var   mean and biased variance of x over a (sample, group)'s m = P cpg elements, rstd = 1 / sqrt(var + eps)
//   y = act(u), u = h gamma + beta, h = (x - mu) rstd
//   backward: du = dy act'(u), q = du gamma,
//   dx = rstd (q - mean(q) - h mean(q h)), dgamma = sum du h, dbeta = sum du
// With an 8-bit checkpoint the backward pass forms h from the read-back x and the saved mean and rstd of the original one.
//
// Bound by HBM where the data comes from there: forward 2, backward 3 elements of traffic per element if every input
// is read once; arithmetic (about 16 and 40 instructions an element with an activation) is not far behind.
// Three families:
//  * row kernels (P = 1: tokens, each with its own statistics; groups that a warp can hold): L lanes keep a
//    group in registers, reductions are shuffles, no barrier at all; several samples per warp are in flight.
//  * resident kernels, for small samples: a block owns one (sample, segment of whole groups) in shared memory, one
//    launch, x read once.
//  * streaming kernels: chunks of positions give partial statistics, and an elementwise pass, in the opposite block
//    order, merges those of its groups;
//    x is read twice, the second time from L2 as far as it fits, and no block waits for another.  (Clusters of 8 blocks
//    that kept 64-channel segments of such samples in distributed shared memory read them once, but in 128-byte
//    pieces between cluster barriers: 69 + 160 us forward and backward at 16 x 4096 x 512 bf16.)
// Variances are sums of squared deviations, never differences of squares: the row and resident kernels take the mean
// first; the streaming ones take both of four positions at a time and merge such pairs (RunningStats), so that no value,
// wherever it stands, is a shift for the others.  Outside the row kernels a thread owns whole
// 16-byte vectors of channels and walks over positions, so all sums are first per channel: group boundaries need no
// alignment, and with A_c = sum du h, B_c = sum du the backward's group means are sum gamma_c A_c / m and
// sum gamma_c B_c / m.  No atomics: every sum has one order.
#include "dense.cuh"

namespace gl {

struct NormParams {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  const int8_t* codes;
  const uint8_t* exps;
  void* out;            // y or dx (contiguous)
  void* dw;             // streaming backward: joined beside the elementwise pass
  void* db;
  float* mean;          // [S, G]
  float* rstd;
  float* part;          // workspace: partial dgamma / dbeta rows [npart][2][C] (backward)
  float* gpart;         // streaming: per (sample, chunk, group) statistics or sums [S][chunks][G][2]
  int64_t S, P, C, G, cpg, sx, px, sdy, pdy, ldc, nblk;
  int64_t nseg, npart;  // segments per sample; rows of part
  int64_t PR;           // positions per chunk (resident: all)
  int64_t chunks, blocks;
  int ng, cs, pdtype, accumulate;
  int nsub, subc;       // streaming, groups too wide for a block: parts of a group, channels of a part (ng = 1)
  float eps;
};

__device__ __forceinline__ float ld_param(const void* p, int64_t i, int dtype, float none) {
  if (p == nullptr) return none;
  return dtype == GL_DTYPE_F32 ? reinterpret_cast<const float*>(p)[i]
                               : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

// N parameters from channel c on; whole vectors where they are 16-byte aligned.
template <int N>
__device__ __forceinline__ void ld_params(const void* p, int64_t c, int dtype, float none, float (&v)[N]) {
  if (N > 1 && p != nullptr && (((uintptr_t)p | c * (dtype == GL_DTYPE_F32 ? 4 : 2)) & 15) == 0 && N * (dtype == GL_DTYPE_F32 ? 4 : 2) % 16 == 0) {
    if (dtype == GL_DTYPE_F32) {
#pragma unroll
      for (int k = 0; k + 4 <= N; k += 4) {
        const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + c + k);
        v[k] = a.x; v[k + 1] = a.y; v[k + 2] = a.z; v[k + 3] = a.w;
      }
    } else if constexpr (N == 8) {
      load_vec<__nv_bfloat16, 8>(reinterpret_cast<const __nv_bfloat16*>(p) + c, v);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = ld_param(p, c + i, dtype, none);
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

// ---- what a CTA of the resident and streaming kernels works on ----
// A segment of ngl whole groups, or a part of one (csl channels from c0 on, cpg to a group, nv vectors) of sample s,
// positions q0 .. q0 + np - 1; thread (tx, ty) owns vector columns tx, tx + TX, .. and every TY-th position.
template <int N, int NT>
struct Slab {
  int64_t s, c0, q0, at;   // at: position range (rank or chunk)
  int g0, ngl, csl, cpg, nv, np, TX, TY, tx, ty, rows;
  __device__ __forceinline__ Slab(const NormParams& p, int64_t s_, int64_t seg, int64_t part) {
    s = s_;
    if (p.nsub == 1) {
      g0 = (int)seg * p.ng;
      ngl = min(p.ng, (int)p.G - g0);
      cpg = (int)p.cpg;
      csl = ngl * cpg;
      c0 = (int64_t)g0 * p.cpg;
    } else {
      g0 = (int)(seg / p.nsub);
      const int64_t off = (seg - (int64_t)g0 * p.nsub) * p.subc;
      ngl = 1;
      cpg = csl = (int)min((int64_t)p.subc, p.cpg - off);
      c0 = (int64_t)g0 * p.cpg + off;
    }
    nv = csl / N;
    at = part;
    q0 = part * p.PR;
    np = (int)max((int64_t)0, min(p.PR, p.P - q0));
    TX = min(nv, NT);
    TY = NT / TX;
    tx = (int)threadIdx.x % TX;
    ty = (int)threadIdx.x / TX;
    rows = 32 % TX == 0 ? NT / 32 : TY;
  }
  __device__ __forceinline__ bool live() const { return ty < TY; }
  // A column's sums to red[row csl + channel], one row per warp where a warp's lanes share columns, else per ty.
  __device__ __forceinline__ void put(float (&acc)[N], float* red, int col) const {
    if (32 % TX == 0) {
      for (int o = TX; o < 32; o *= 2)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += __shfl_xor_sync(kFullMask, acc[i], o);
      if ((int)(threadIdx.x & 31) < TX) {
#pragma unroll
        for (int i = 0; i < N; ++i) red[(threadIdx.x >> 5) * csl + col * N + i] = acc[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) red[ty * csl + col * N + i] = acc[i];
    }
  }
};

// Floats of one `red` array: rows * csl is at most NT * N, or cs where a segment is wider than a row of threads.
__host__ __device__ inline int64_t norm_red(int64_t cs, int N, int NT) { return cs > (int64_t)NT * N ? cs : (int64_t)NT * N; }

// gs[g] = sum over the group's channels and the rows of red[row * cs + c]: a warp per group where there is enough to
// add, else a thread.
template <int NT>
__device__ __forceinline__ void group_sums(const float* red, int cs, int rows, int ngl, int cpg, float* gs) {
  const int tid = threadIdx.x, lane = tid & 31;
  if (cpg * rows >= 64) {
    for (int g = tid >> 5; g < ngl; g += NT / 32) {
      float s = 0.f;
      if (cpg >= 32) {
        for (int r = 0; r < rows; ++r)
          for (int c = lane; c < cpg; c += 32) s += red[r * cs + g * cpg + c];
      } else {
        const int per = 32 / cpg, c = lane % cpg;            // rows at a time
        if (lane < per * cpg)
          for (int r = lane / cpg; r < rows; r += per) s += red[r * cs + g * cpg + c];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
      if (lane == 0) gs[g] = s;
    }
  } else {
    for (int g = tid; g < ngl; g += NT) {
      float s = 0.f;
      for (int r = 0; r < rows; ++r)
        for (int c = 0; c < cpg; ++c) s += red[r * cs + g * cpg + c];
      gs[g] = s;
    }
  }
}

// s / m for a sum of m values, inv = 1 / m: rounded once, so that the mean of values that are all alike is that value (s inv
// is off by up to an ulp of it, which rstd = 1 / sqrt(eps) of such a group magnifies).
__device__ __forceinline__ float mean_of(float s, float m, float inv) {
  const float q = s * inv;
  return fmaf(fmaf(-q, m, s), inv, q);
}

// A vector of channels' constants: h = (x - sub) mul, and gamma, beta.  (For bf16 x, x mul + (-mean mul) would be an
// operation less, 30.4 instead of 31.6 us in the elementwise pass of 16 x 4096 x 512 with SiLU, but leaves |mean| mul 2^-24 of
// a value that is the mean.)
template <int N>
struct ChanConst {
  float mul[N], sub[N], gam[N], bet[N];
  __device__ __forceinline__ float h(float x, int i) const { return (x - sub[i]) * mul[i]; }
  template <typename F>
  __device__ __forceinline__ void load(const NormParams& p, int64_t c, F stat) {   // stat(i, mean, rstd)
    ld_params<N>(p.w, c, p.pdtype, 1.f, gam);
    ld_params<N>(p.b, c, p.pdtype, 0.f, bet);
#pragma unroll
    for (int i = 0; i < N; ++i) stat(i, sub[i], mul[i]);
  }
};

// ---- resident forward ----
template <typename T, int N, int NT, int ACT>
__global__ void __launch_bounds__(NT) norm_fwd_resident(NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  Raw<T, N>* tile = reinterpret_cast<Raw<T, N>*>(smem);
  const int tid = threadIdx.x, cpg = (int)p.cpg;
  const int64_t s = blockIdx.x / (unsigned)p.nseg;
  const Slab<N, NT> a(p, s, blockIdx.x % (unsigned)p.nseg, 0);
  float* red = reinterpret_cast<float*>(smem + (((size_t)p.PR * p.cs * sizeof(T) + 15) & ~(size_t)15));
  float* gs = red + norm_red(p.cs, N, NT);             // [2][ng]
  float* stat = gs + 2 * p.ng;                         // [2][ng]: mean, rstd
  const float m = (float)p.P * (float)cpg, inv_m = 1.f / m;

  if (a.live()) {
    for (int col = a.tx; col < a.nv; col += a.TX) {
      float acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      const int64_t c = a.c0 + (int64_t)col * N;
      int q = a.ty;
      for (; q + 3 * a.TY < a.np; q += 4 * a.TY) {     // four loads in flight
        Raw<T, N> r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = read_x<T, N, false>(p, s, a.q0 + q + k * a.TY, c);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          tile[(q + k * a.TY) * a.nv + col] = r[k];
          float f[N];
          unpack<T, N>(r[k], f);
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] += f[i];
        }
      }
      for (; q < a.np; q += a.TY) {
        const Raw<T, N> r = read_x<T, N, false>(p, s, a.q0 + q, c);
        tile[q * a.nv + col] = r;
        float f[N];
        unpack<T, N>(r, f);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += f[i];
      }
      a.put(acc, red, col);
    }
  }
  __syncthreads();
  group_sums<NT>(red, a.csl, a.rows, a.ngl, cpg, gs);
  __syncthreads();
  for (int g = tid; g < a.ngl; g += NT) stat[g] = mean_of(gs[g], m, inv_m);
  __syncthreads();

  if (a.live()) {
    for (int col = a.tx; col < a.nv; col += a.TX) {
      float acc[N], mu[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        acc[i] = 0.f;
        mu[i] = stat[(col * N + i) / cpg];
      }
#pragma unroll 4
      for (int q = a.ty; q < a.np; q += a.TY) {
        float f[N];
        unpack<T, N>(tile[q * a.nv + col], f);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(f[i] - mu[i], f[i] - mu[i], acc[i]);
      }
      a.put(acc, red, col);
    }
  }
  __syncthreads();
  group_sums<NT>(red, a.csl, a.rows, a.ngl, cpg, gs + p.ng);
  __syncthreads();
  for (int g = tid; g < a.ngl; g += NT) {
    const float rs = 1.f / sqrtf(gs[p.ng + g] * inv_m + p.eps);
    stat[p.ng + g] = rs;
    p.mean[s * p.G + a.g0 + g] = stat[g];
    p.rstd[s * p.G + a.g0 + g] = rs;
  }
  __syncthreads();

  if (a.live()) {
    T* out = reinterpret_cast<T*>(p.out);
    for (int col = a.tx; col < a.nv; col += a.TX) {
      ChanConst<N> k;
      const int64_t c = a.c0 + (int64_t)col * N;
      k.load(p, c, [&](int i, float& mean, float& rstd) {
        const int g = (col * N + i) / cpg;
        mean = stat[g];
        rstd = stat[p.ng + g];
      });
#pragma unroll 2
      for (int q = a.ty; q < a.np; q += a.TY) {
        float f[N];
        unpack<T, N>(tile[q * a.nv + col], f);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = dense_act<ACT, sizeof(T) == 2>(fmaf(k.h(f[i], i), k.gam[i], k.bet[i]));
        store_vec<T, N>(out + (s * p.P + a.q0 + q) * p.C + c, f);
      }
    }
  }
}

// ---- resident backward ----
// A block keeps one segment and walks over samples, adding its dgamma / dbeta in shared memory; one partial row per
// block goes to the join.
template <typename T, int N, int NT, int ACT, bool CKPT>
__global__ void __launch_bounds__(NT) norm_bwd_resident(NormParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const size_t tbytes = ((size_t)p.PR * p.cs * sizeof(T) + 15) & ~(size_t)15;
  Raw<T, N>* xt = reinterpret_cast<Raw<T, N>*>(smem);
  Raw<T, N>* dt = reinterpret_cast<Raw<T, N>*>(smem + tbytes);
  const int tid = threadIdx.x, cpg = (int)p.cpg;
  const int64_t walkers = gridDim.x / (unsigned)p.nseg, walker = blockIdx.x / (unsigned)p.nseg;
  const int64_t rf = norm_red(p.cs, N, NT);
  float* ra = reinterpret_cast<float*>(smem + 2 * tbytes);   // sum du h per channel
  float* rb = ra + rf;                                       // sum du per channel
  float* da = rb + rf;                                       // dgamma, dbeta of this CTA
  float* db = da + p.cs;
  float* gs = db + p.cs;                                     // [2][ng]
  float* stat = gs + 2 * p.ng;                               // [2][ng]: mean(q), mean(q h)
  const float inv_m = 1.f / ((float)p.P * (float)cpg);
  const Slab<N, NT> a(p, walker, blockIdx.x % (unsigned)p.nseg, 0);
  for (int c = tid; c < a.csl; c += NT) da[c] = db[c] = 0.f;
  for (int64_t s = walker; s < p.S; s += walkers) {
    if (a.live()) {
      for (int col = a.tx; col < a.nv; col += a.TX) {
        float aa[N], ab[N];
        ChanConst<N> k;
        const int64_t c = a.c0 + (int64_t)col * N;
        k.load(p, c, [&](int i, float& mean, float& rstd) {
          const int64_t g = s * p.G + a.g0 + (col * N + i) / cpg;
          mean = p.mean[g];
          rstd = p.rstd[g];
        });
#pragma unroll
        for (int i = 0; i < N; ++i) aa[i] = ab[i] = 0.f;
        for (int q = a.ty; q < a.np; q += 2 * a.TY) {
          Raw<T, N> rx[2], rd[2];
          const bool two = q + a.TY < a.np;
          rx[0] = read_x<T, N, CKPT>(p, s, a.q0 + q, c);
          rd[0] = read_dy<T, N>(p, s, a.q0 + q, c);
          if (two) {
            rx[1] = read_x<T, N, CKPT>(p, s, a.q0 + q + a.TY, c);
            rd[1] = read_dy<T, N>(p, s, a.q0 + q + a.TY, c);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (j == 1 && !two) break;
            xt[(q + j * a.TY) * a.nv + col] = rx[j];
            dt[(q + j * a.TY) * a.nv + col] = rd[j];
            float f[N], d[N];
            unpack<T, N>(rx[j], f);
            unpack<T, N>(rd[j], d);
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float h = k.h(f[i], i);
              const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(h, k.gam[i], k.bet[i]));
              aa[i] = fmaf(du, h, aa[i]);
              ab[i] += du;
            }
          }
        }
        a.put(aa, ra, col);
        a.put(ab, rb, col);
      }
    }
    __syncthreads();
    for (int c = tid; c < a.csl; c += NT) {
      float va = 0.f, vb = 0.f;
      for (int r = 0; r < a.rows; ++r) {
        va += ra[r * a.csl + c];
        vb += rb[r * a.csl + c];
      }
      da[c] += va;
      db[c] += vb;
      const float gam = ld_param(p.w, a.c0 + c, p.pdtype, 1.f);
      ra[c] = va * gam;
      rb[c] = vb * gam;
    }
    __syncthreads();
    group_sums<NT>(rb, a.csl, 1, a.ngl, cpg, gs);
    group_sums<NT>(ra, a.csl, 1, a.ngl, cpg, gs + p.ng);
    __syncthreads();
    for (int g = tid; g < a.ngl; g += NT) {
      stat[g] = gs[g] * inv_m;
      stat[p.ng + g] = gs[p.ng + g] * inv_m;
    }
    __syncthreads();
    if (a.live()) {
      T* out = reinterpret_cast<T*>(p.out);
      for (int col = a.tx; col < a.nv; col += a.TX) {
        float m1[N], m2[N];
        ChanConst<N> k;
        const int64_t c = a.c0 + (int64_t)col * N;
        k.load(p, c, [&](int i, float& mean, float& rstd) {
          const int g = (col * N + i) / cpg;
          mean = p.mean[s * p.G + a.g0 + g];
          rstd = p.rstd[s * p.G + a.g0 + g];
          m1[i] = stat[g];
          m2[i] = stat[p.ng + g];
        });
#pragma unroll 2
        for (int q = a.ty; q < a.np; q += a.TY) {
          float f[N], d[N];
          unpack<T, N>(xt[q * a.nv + col], f);
          unpack<T, N>(dt[q * a.nv + col], d);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float h = k.h(f[i], i);
            const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(h, k.gam[i], k.bet[i]));
            f[i] = k.mul[i] * (fmaf(du, k.gam[i], -m1[i]) - h * m2[i]);
          }
          store_vec<T, N>(out + (s * p.P + a.q0 + q) * p.C + c, f);
        }
      }
    }
    __syncthreads();                                   // shared memory is free for the next sample
  }
  float* row = p.part + walker * 2 * p.C + a.c0;
  for (int c = tid; c < a.csl; c += NT) {
    row[c] = da[c];
    row[p.C + c] = db[c];
  }
}

// ---- streaming kernels: a block per (sample, chunk of positions, segment) ----
// Blocks of 256 threads, kFwdBlocks / kBwdBlocks to an SM (the registers of U loads in flight and the channels'
// constants), and one whole wave of them: a block's statistics and merges cost as much as several positions.
constexpr int kFwdBlocks = 4, kBwdBlocks = 3;

// A thread's column of a [positions][channels] operand: element vectors `step` positions apart.
template <typename T, int N>
struct Column {
  const T* p;
  int64_t step;
  __device__ __forceinline__ Column(const void* base, int64_t s, int64_t q, int64_t c, int64_t ss, int64_t ps, int TY)
      : p(reinterpret_cast<const T*>(base) + s * ss + q * ps + c), step(ps * TY) {}
  __device__ __forceinline__ Raw<T, N> at(int k) const { return *reinterpret_cast<const Raw<T, N>*>(p + k * step); }
  __device__ __forceinline__ void next(int u) { p += u * step; }
};
// x, or its checkpoint.
template <typename T, int N, bool CKPT>
struct XColumn : Column<T, N> {
  __device__ __forceinline__ XColumn(const NormParams& p, int64_t s, int64_t q, int64_t c, int TY)
      : Column<T, N>(p.x, s, q, c, p.sx, p.px, TY) {}
};
template <typename T, int N>
struct XColumn<T, N, true> {
  const NormParams& p;
  int64_t row, c;
  int TY;
  __device__ __forceinline__ XColumn(const NormParams& p_, int64_t s, int64_t q, int64_t c_, int TY_)
      : p(p_), row(s * p_.P + q), c(c_), TY(TY_) {}
  __device__ __forceinline__ Raw<T, N> at(int k) const { return read_codes<T, N>(p, row + k * TY, c); }
  __device__ __forceinline__ void next(int u) { row += u * TY; }
};

// f(x values[, dy values], index of the position in the block) for every position of the thread's column, U positions'
// loads in flight.
template <int U, typename T, int N, typename X, typename F>
__device__ __forceinline__ void walk(const Slab<N, 256>& a, X x, F f) {
  for (int q = a.ty; q < a.np; q += U * a.TY, x.next(U)) {
    Raw<T, N> r[U];
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (q + k * a.TY < a.np) r[k] = x.at(k);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (q + k * a.TY < a.np) {
        float v[N];
        unpack<T, N>(r[k], v);
        f(v, q + k * a.TY);
      }
    }
  }
}
template <int U, typename T, int N, typename X, typename D, typename F>
__device__ __forceinline__ void walk(const Slab<N, 256>& a, X x, D d, F f) {
  for (int q = a.ty; q < a.np; q += U * a.TY, x.next(U), d.next(U)) {
    Raw<T, N> r[U], e[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (q + k * a.TY < a.np) {
        r[k] = x.at(k);
        e[k] = d.at(k);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (q + k * a.TY < a.np) {
        float v[N], w[N];
        unpack<T, N>(r[k], v);
        unpack<T, N>(e[k], w);
        f(v, w, q + k * a.TY);
      }
    }
  }
}

template <int N, int NT>
__device__ __forceinline__ Slab<N, NT> chunk_slab(const NormParams& p, unsigned block) {
  const unsigned nseg = (unsigned)p.nseg, chunks = (unsigned)p.chunks;   // 32-bit divisions: block numbers are
  const unsigned sc = block / nseg, s = sc / chunks;
  return Slab<N, NT>(p, s, block - sc * nseg, sc - s * chunks);
}

// Lanes (a power of two, at most a warp) that merge one group's chunks in the elementwise kernels: all groups of a block
// at once where they fit, since every merge is a chain of loads.
template <int NT>
__device__ __forceinline__ int group_lanes(int ngl) {
  int l = 32;
  while (l > 1 && NT / l < ngl) l >>= 1;
  return l;
}

// This block's first entry in a chunk's row of gpart, and the number of elements behind entry (chunk, part).
__device__ __forceinline__ int64_t entry0(const NormParams& p, int g0) {   // of the statistics kernels
  return p.nsub == 1 ? g0 : (int64_t)(blockIdx.x % (unsigned)p.nseg);
}
__device__ __forceinline__ float entry_count(const NormParams& p, int64_t ch, int64_t part) {
  const int64_t c = p.nsub == 1 ? p.cpg : min((int64_t)p.subc, p.cpg - part * p.subc);
  return (float)min(p.PR, p.P - ch * p.PR) * (float)c;
}

// Mean and sum of squared deviations of the values seen so far, N channels.  Two sets a and b make one by
//   mean = mean_a + d n_b / n, m2 = m2_a + m2_b + d^2 n_a n_b / n, d = mean_b - mean_a, n = n_a + n_b
// (Chan, Golub and LeVeque), all of m2's terms positive.  lo holds what the mean's rounding left of the last steps: over a
// thread's column the mean would otherwise drift by the square root of its length in roundings.  Differences from the
// chunk's first value, their sum and sum of squares, took 20.1 instead of 22.4 us at 16 x 4096 x 512 bf16, but where that
// value stands far off they cancel: a channel 1000 deviations off at position 0 of 600 x 4096 x 64 fp32 put the variance off
// by up to 1.5e-2.
template <typename T, int N>
struct RunningStats {
  float mean[N], lo[N], m2[N], n;
  __device__ __forceinline__ RunningStats() : n(0.f) {
#pragma unroll
    for (int i = 0; i < N; ++i) mean[i] = lo[i] = m2[i] = 0.f;
  }
  static __device__ __forceinline__ float element(const Raw<T, N>& r, int i) {   // one, so that 32 need no registers at once
    if constexpr (N == 1) {
      return to_f32<T>(r.v);
    } else {
      const uint32_t u[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
      if constexpr (sizeof(T) == 4) return __uint_as_float(u[i]);
      else return __uint_as_float(i & 1 ? u[i / 2] & 0xFFFF0000u : u[i / 2] << 16);
    }
  }
  // A channel's mean mb and squared deviations q of more values, w = n_b / n and cw = n_a n_b / n.
  __device__ __forceinline__ void merge(int i, float mb, float q, float w, float cw) {
    const float d = (mb - mean[i]) - lo[i], t = fmaf(d, w, lo[i]), to = mean[i] + t;
    m2[i] = fmaf(d * d, cw, m2[i] + q);
    lo[i] = t - (to - mean[i]);
    mean[i] = to;
  }
  __device__ __forceinline__ void add4(const Raw<T, N> (&r)[4]) {
    const float w = 4.f / (n + 4.f), cw = n * w;
    n += 4.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float a = element(r[0], i), b = element(r[1], i), c = element(r[2], i), d = element(r[3], i);
      const float mb = 0.25f * ((a + b) + (c + d));
      a -= mb;
      b -= mb;
      c -= mb;
      d -= mb;
      merge(i, mb, fmaf(a, a, fmaf(b, b, fmaf(c, c, d * d))), w, cw);
    }
  }
  __device__ __forceinline__ void add(const Raw<T, N>& r) {
    const float w = 1.f / (n + 1.f), cw = n * w;
    n += 1.f;
#pragma unroll
    for (int i = 0; i < N; ++i) merge(i, element(r, i), 0.f, w, cw);
  }
  // The sets of the lanes TX, 2 TX, .. apart, in all of them.
  __device__ __forceinline__ void merge_lanes(int TX) {
    for (int o = TX; o < 32; o *= 2) {
      const float nb = __shfl_xor_sync(kFullMask, n, o), w = nb > 0.f ? nb / (n + nb) : 0.f, cw = n * w;
      n += nb;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = __shfl_xor_sync(kFullMask, mean[i], o) - mean[i];
        m2[i] = fmaf(d * d, cw, m2[i] + __shfl_xor_sync(kFullMask, m2[i], o));
        mean[i] = fmaf(d, w, mean[i]);
      }
    }
  }
};

// gpart[((s chunks + chunk) G + g) nsub + part] = (mean, sum of squared deviations) of the chunk's values of the group,
// or of its part.
template <typename T, int N, int NT>
__global__ void __launch_bounds__(NT, kFwdBlocks) norm_stats_kernel(NormParams p) {
  extern __shared__ float sf[];
  const Slab<N, NT> a = chunk_slab<N, NT>(p, blockIdx.x);
  const int64_t rf = norm_red(p.cs, N, NT);
  float* r1 = sf;                                       // [rows][csl] means
  float* r2 = sf + rf;                                  // and squared deviations
  float* gm = r2 + rf;                                  // [ng]
  float* gv = gm + p.ng;
  const int cpg = a.cpg;
  const float n = (float)a.np;
  const bool lanes = 32 % a.TX == 0;                    // a warp's lanes share columns (all of them are live)
  if (a.live()) {
    for (int col = a.tx; col < a.nv; col += a.TX) {
      const int64_t c = a.c0 + (int64_t)col * N;
      RunningStats<T, N> st;
      XColumn<T, N, false> x(p, a.s, a.q0 + a.ty, c, a.TY);
      int q = a.ty;
      for (; q + 3 * a.TY < a.np; q += 4 * a.TY, x.next(4)) {
        const Raw<T, N> r[4] = {x.at(0), x.at(1), x.at(2), x.at(3)};
        st.add4(r);
      }
      Raw<T, N> r[3];
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (q + k * a.TY < a.np) r[k] = x.at(k);
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (q + k * a.TY < a.np) st.add(r[k]);
      if (lanes) st.merge_lanes(a.TX);
      if (!lanes || (int)(threadIdx.x & 31) < a.TX) {
        const int row = (lanes ? (int)threadIdx.x >> 5 : a.ty) * a.csl + col * N;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          r1[row + i] = st.mean[i];
          r2[row + i] = st.m2[i];
        }
      }
    }
  }
  __syncthreads();
  // Positions behind row r: of the `per` threads of its column, those from r per on.
  const int per = lanes ? 32 / a.TX : 1, whole = a.np / a.TY, rest = a.np - whole * a.TY;
  const auto behind = [&](int r) { return (float)(whole * per + min(max(rest - r * per, 0), per)); };
  for (int c = threadIdx.x; c < a.csl; c += NT) {       // channel c: mean and squared deviations (row 0 has values)
    const float m0 = r1[c];
    float t = 0.f, v = 0.f;
    for (int r = 1; r < a.rows; ++r) t = fmaf(behind(r), r1[r * a.csl + c] - m0, t);
    const float mean = m0 + t / n;
    for (int r = 0; r < a.rows; ++r) {
      const float k = behind(r), d = r1[r * a.csl + c] - mean;
      if (k > 0.f) v += fmaf(k * d, d, r2[r * a.csl + c]);
    }
    r1[c] = mean;
    r2[c] = v;
  }
  __syncthreads();
  group_sums<NT>(r1, a.csl, 1, a.ngl, cpg, gm);
  __syncthreads();
  for (int c = threadIdx.x; c < a.csl; c += NT) {       // Chan: n (mean_c - mean_g)^2 joins the deviations
    const float d = r1[c] - gm[c / cpg] / (float)cpg;
    r2[c] = fmaf(n * d, d, r2[c]);
  }
  __syncthreads();
  group_sums<NT>(r2, a.csl, 1, a.ngl, cpg, gv);
  __syncthreads();
  float2* out = reinterpret_cast<float2*>(p.gpart) + (a.s * p.chunks + a.at) * p.G * p.nsub + entry0(p, a.g0);
  for (int g = threadIdx.x; g < a.ngl; g += NT) out[g] = make_float2(gm[g] / (float)cpg, gv[g]);
}

// The groups' statistics from the chunks' (every block the same sums), then act(h gamma + beta).
template <typename T, int N, int NT, int ACT>
__global__ void __launch_bounds__(NT, kFwdBlocks) norm_apply_kernel(NormParams p) {
  extern __shared__ float sf[];
  const Slab<N, NT> a = chunk_slab<N, NT>(p, gridDim.x - 1 - blockIdx.x);
  const int cpg = a.cpg, lane = threadIdx.x & 31;
  float* mean = sf;                                     // [ng]
  float* rstd = sf + p.ng;
  const float2* part = reinterpret_cast<const float2*>(p.gpart) + (a.s * p.chunks * p.G + a.g0) * p.nsub;
  const float m = (float)p.P * (float)p.cpg;
  const int entries = (int)(p.chunks * p.nsub), gl = group_lanes<NT>(a.ngl), l = lane % gl;
  for (int g = threadIdx.x / gl; g < (a.ngl + 31) / 32 * 32; g += NT / gl) {   // whole warps: shuffles below
    const bool in = g < a.ngl;
    const float first = in ? part[(int64_t)g * p.nsub].x : 0.f;   // exact where the entries agree
    float v = 0.f;
#pragma unroll 4
    for (int j = l; j < entries; j += gl) {
      const int ch = p.nsub == 1 ? j : j / p.nsub;
      if (in)
        v = fmaf(part[((int64_t)ch * p.G + g) * p.nsub + (j - ch * p.nsub)].x - first,
                 entry_count(p, ch, j - ch * p.nsub), v);
    }
    for (int o = gl / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    const float mu = first + v / m;
    v = 0.f;
#pragma unroll 4
    for (int j = l; j < entries; j += gl) {
      const int ch = p.nsub == 1 ? j : j / p.nsub;
      if (!in) continue;
      const float2 t = part[((int64_t)ch * p.G + g) * p.nsub + (j - ch * p.nsub)];
      v += fmaf((t.x - mu) * (t.x - mu), entry_count(p, ch, j - ch * p.nsub), t.y);
    }
    for (int o = gl / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    if (in && l == 0) {
      const float rs = 1.f / sqrtf(v / m + p.eps);
      mean[g] = mu;
      rstd[g] = rs;
      if (a.q0 == 0 && a.c0 == a.g0 * p.cpg) {       // the group's first block
        p.mean[a.s * p.G + a.g0 + g] = mu;
        p.rstd[a.s * p.G + a.g0 + g] = rs;
      }
    }
  }
  __syncthreads();
  if (!a.live()) return;
  T* out = reinterpret_cast<T*>(p.out);
  for (int col = a.tx; col < a.nv; col += a.TX) {
    // u = (x - sub) mul + add
    float mul[N], sub[N], add[N], gam[N];
    const int64_t c = a.c0 + (int64_t)col * N;
    ld_params<N>(p.w, c, p.pdtype, 1.f, gam);
    ld_params<N>(p.b, c, p.pdtype, 0.f, add);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = (col * N + i) / cpg;
      mul[i] = rstd[g] * gam[i];
      sub[i] = mean[g];
    }
    T* to = out + (a.s * p.P + a.q0) * p.C + c;
    walk<4, T, N>(a, XColumn<T, N, false>(p, a.s, a.q0 + a.ty, c, a.TY), [&](float (&f)[N], int q) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        f[i] = dense_act<ACT, sizeof(T) == 2>(fmaf(f[i] - sub[i], mul[i], add[i]));
      store_vec<T, N>(to + q * p.C, f);
    });
  }
}

// Per chunk: dgamma and dbeta partial rows, and each group's sums of q and q h in gpart.
template <typename T, int N, int NT, int ACT, bool CKPT>
__global__ void __launch_bounds__(NT, kBwdBlocks) norm_bwd_stats_kernel(NormParams p) {
  extern __shared__ float sf[];
  const Slab<N, NT> a = chunk_slab<N, NT>(p, blockIdx.x);
  const int64_t rf = norm_red(p.cs, N, NT);
  float* ra = sf;
  float* rb = sf + rf;
  float* gq = rb + rf;                                  // [ng] sums of q h, of q
  float* gs = gq + p.ng;
  const int cpg = a.cpg;
  if (a.live()) {
    for (int col = a.tx; col < a.nv; col += a.TX) {
      // xc = x - mean, u = xc mul gamma + beta; sum du xc is scaled by rstd at the end
      float aa[N], ab[N], sub[N], ga[N], bet[N], mul[N];
      const int64_t c = a.c0 + (int64_t)col * N;
      ld_params<N>(p.w, c, p.pdtype, 1.f, ga);
      ld_params<N>(p.b, c, p.pdtype, 0.f, bet);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t g = a.s * p.G + a.g0 + (col * N + i) / cpg;
        sub[i] = p.mean[g];
        mul[i] = p.rstd[g];
        ga[i] *= mul[i];
        aa[i] = ab[i] = 0.f;
      }
      walk<2, T, N>(a, XColumn<T, N, CKPT>(p, a.s, a.q0 + a.ty, c, a.TY),
                    Column<T, N>(p.dy, a.s, a.q0 + a.ty, c, p.sdy, p.pdy, a.TY),
                    [&](const float (&f)[N], const float (&d)[N], int) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float xc = f[i] - sub[i];
          const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(xc, ga[i], bet[i]));
          aa[i] = fmaf(du, xc, aa[i]);
          ab[i] += du;
        }
      });
#pragma unroll
      for (int i = 0; i < N; ++i) aa[i] *= mul[i];
      a.put(aa, ra, col);
      a.put(ab, rb, col);
    }
  }
  __syncthreads();
  const int64_t chunk = a.s * p.chunks + a.at;
  float* row = p.part + chunk * 2 * p.C + a.c0;
  for (int c = threadIdx.x; c < a.csl; c += NT) {
    float va = 0.f, vb = 0.f;
    for (int r = 0; r < a.rows; ++r) {
      va += ra[r * a.csl + c];
      vb += rb[r * a.csl + c];
    }
    row[c] = va;
    row[p.C + c] = vb;
    const float gam = ld_param(p.w, a.c0 + c, p.pdtype, 1.f);
    ra[c] = va * gam;
    rb[c] = vb * gam;
  }
  __syncthreads();
  group_sums<NT>(ra, a.csl, 1, a.ngl, cpg, gq);
  group_sums<NT>(rb, a.csl, 1, a.ngl, cpg, gs);
  __syncthreads();
  float2* out = reinterpret_cast<float2*>(p.gpart) + chunk * p.G * p.nsub + entry0(p, a.g0);
  for (int g = threadIdx.x; g < a.ngl; g += NT) out[g] = make_float2(gs[g], gq[g]);
}

// dgamma / dbeta of 32 channels = the partial rows' sums in a fixed order: by `warps` row lanes.
__device__ __forceinline__ void param_join(const float* part, int64_t rows, int64_t C, int64_t c0, void* dw, void* db,
                                           int pdtype, int accumulate, float* red, int warps) {
  const int lane = threadIdx.x & 31, r0 = threadIdx.x >> 5;
  const int64_t c = c0 + lane;
  float a = 0.f, b = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int64_t r = r0; r < rows; r += warps) {
      a += part[r * 2 * C + c];
      b += part[r * 2 * C + C + c];
    }
  }
  red[(r0 * 2) * 33 + lane] = a;
  red[(r0 * 2 + 1) * 33 + lane] = b;
  __syncthreads();
  if (r0 < 2 && c < C) {
    float t = 0.f;
    for (int r = 0; r < warps; ++r) t += red[(r * 2 + r0) * 33 + lane];
    void* out = r0 == 0 ? dw : db;
    if (out != nullptr) {
      if (accumulate) reinterpret_cast<float*>(out)[c] += t;
      else if (pdtype == GL_DTYPE_F32) reinterpret_cast<float*>(out)[c] = t;
      else reinterpret_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(t);
    }
  }
}

__global__ void __launch_bounds__(512) norm_param_join_kernel(const float* part, int64_t rows, int64_t C, void* dw,
                                                              void* db, int pdtype, int accumulate) {
  __shared__ float red[16 * 2 * 33];
  param_join(part, rows, C, (int64_t)blockIdx.x * 32, dw, db, pdtype, accumulate, red, 16);
}

// The groups' means of q and q h from the chunks', then dx; blocks past p.blocks join dgamma / dbeta.
template <typename T, int N, int NT, int ACT, bool CKPT>
__global__ void __launch_bounds__(NT, kBwdBlocks) norm_bwd_apply_kernel(NormParams p) {
  extern __shared__ float sf[];
  if ((int64_t)blockIdx.x >= p.blocks) {
    param_join(p.part, p.npart, p.C, ((int64_t)blockIdx.x - p.blocks) * 32, p.dw, p.db, p.pdtype, p.accumulate, sf,
               NT / 32);
    return;
  }
  const Slab<N, NT> a = chunk_slab<N, NT>(p, (unsigned)p.blocks - 1 - blockIdx.x);
  const int cpg = a.cpg, lane = threadIdx.x & 31;
  float* s1 = sf;                                       // [ng] mean(q), mean(q h)
  float* s2 = sf + p.ng;
  const float2* part = reinterpret_cast<const float2*>(p.gpart) + (a.s * p.chunks * p.G + a.g0) * p.nsub;
  const int entries = (int)(p.chunks * p.nsub), gl = group_lanes<NT>(a.ngl), l = lane % gl;
  for (int g = threadIdx.x / gl; g < (a.ngl + 31) / 32 * 32; g += NT / gl) {
    const bool in = g < a.ngl;
    float v1 = 0.f, v2 = 0.f;
#pragma unroll 4
    for (int j = l; j < entries; j += gl) {
      const int ch = p.nsub == 1 ? j : j / p.nsub;
      if (!in) continue;
      const float2 t = part[((int64_t)ch * p.G + g) * p.nsub + (j - ch * p.nsub)];
      v1 += t.x;
      v2 += t.y;
    }
    for (int o = gl / 2; o > 0; o >>= 1) {
      v1 += __shfl_xor_sync(kFullMask, v1, o);
      v2 += __shfl_xor_sync(kFullMask, v2, o);
    }
    if (in && l == 0) {
      const float m = (float)p.P * (float)p.cpg;
      s1[g] = v1 / m;
      s2[g] = v2 / m;
    }
  }
  __syncthreads();
  if (!a.live()) return;
  T* out = reinterpret_cast<T*>(p.out);
  for (int col = a.tx; col < a.nv; col += a.TX) {
    // xc = x - mean, u = xc ga + beta with ga = rstd gamma, dx = du ga - xc rstd^2 mean(q h) - rstd mean(q)
    float sub[N], ga[N], bet[N], bx[N], cc[N];
    const int64_t c = a.c0 + (int64_t)col * N;
    ld_params<N>(p.w, c, p.pdtype, 1.f, ga);
    ld_params<N>(p.b, c, p.pdtype, 0.f, bet);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int g = (col * N + i) / cpg;
      const float rs = p.rstd[a.s * p.G + a.g0 + g];
      sub[i] = p.mean[a.s * p.G + a.g0 + g];
      ga[i] *= rs;
      bx[i] = -rs * rs * s2[g];
      cc[i] = -rs * s1[g];
    }
    T* to = out + (a.s * p.P + a.q0) * p.C + c;
    walk<2, T, N>(a, XColumn<T, N, CKPT>(p, a.s, a.q0 + a.ty, c, a.TY),
                  Column<T, N>(p.dy, a.s, a.q0 + a.ty, c, p.sdy, p.pdy, a.TY),
                  [&](float (&f)[N], const float (&d)[N], int q) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float xc = f[i] - sub[i];
        const float du = d[i] * dense_slope<ACT, sizeof(T) == 2>(fmaf(xc, ga[i], bet[i]));
        f[i] = fmaf(du, ga[i], fmaf(xc, bx[i], cc[i]));
      }
      store_vec<T, N>(to + q * p.C, f);
    });
  }
}

// ---- row kernels (P = 1) ----
// L lanes (a power of two) hold a group of cpg = nvg N channels, V vectors each (lane l: vectors l, l + L, ..); a warp
// holds 32 / L neighbouring groups.  Eight warps of a block share the groups and take different samples.
constexpr int kRowWarps = 8;

struct RowAt {
  int g, l;        // group, lane within it
  bool live;
};
template <int L>
__device__ __forceinline__ RowAt row_at(const NormParams& p) {
  const int lane = threadIdx.x & 31;
  RowAt a;
  a.g = (int)blockIdx.x % (int)p.nseg * (32 / L) + lane / L;
  a.l = lane % L;
  a.live = a.g < (int)p.G;
  if (!a.live) a.g = (int)p.G - 1;
  return a;
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
  return v;
}

// U samples of a warp at a time, so that U V loads are in flight.
template <typename T, int N, int L, int V, int ACT>
__global__ void __launch_bounds__(32 * kRowWarps) norm_fwd_rows(NormParams p) {
  constexpr int U = V >= 4 ? 1 : 4 / V;
  const RowAt a = row_at<L>(p);
  const int nvg = (int)p.cpg / N, warp = threadIdx.x >> 5;
  const int64_t c0 = (int64_t)a.g * p.cpg;
  const float inv = 1.f / (float)p.cpg;
  const int64_t step = (int64_t)(gridDim.x / p.nseg) * kRowWarps * U;
  for (int64_t s0 = ((int64_t)(blockIdx.x / p.nseg) * kRowWarps + warp) * U; s0 < p.S; s0 += step) {
    Raw<T, N> r[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (s0 + u < p.S && a.l + v * L < nvg) r[u][v] = read_x<T, N, false>(p, s0 + u, 0, c0 + (a.l + v * L) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= p.S) break;                            // the same for the whole warp
      float t = 0.f, f[N];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (a.l + v * L < nvg) {
          unpack<T, N>(r[u][v], f);
#pragma unroll
          for (int i = 0; i < N; ++i) t += f[i];
        }
      }
      const float mu = mean_of(lanes_sum<L>(t), (float)p.cpg, inv);
      t = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (a.l + v * L < nvg) {
          unpack<T, N>(r[u][v], f);
#pragma unroll
          for (int i = 0; i < N; ++i) t = fmaf(f[i] - mu, f[i] - mu, t);
        }
      }
      const float rs = 1.f / sqrtf(lanes_sum<L>(t) * inv + p.eps);
      if (a.live && a.l == 0) {
        p.mean[(s0 + u) * p.G + a.g] = mu;
        p.rstd[(s0 + u) * p.G + a.g] = rs;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (a.live && a.l + v * L < nvg) {
          const int64_t c = c0 + (a.l + v * L) * N;
          unpack<T, N>(r[u][v], f);
#pragma unroll
          for (int i = 0; i < N; ++i)
            f[i] = dense_act<ACT, sizeof(T) == 2>(fmaf(f[i] - mu, rs * ld_param(p.w, c + i, p.pdtype, 1.f),
                                                       ld_param(p.b, c + i, p.pdtype, 0.f)));
          store_vec<T, N>(reinterpret_cast<T*>(p.out) + (s0 + u) * p.C + c, f);
        }
      }
    }
  }
}

// A lane adds its channels' dgamma / dbeta over the samples of its warp; the block's warps are summed at the end into
// one partial row per block of samples.
template <typename T, int N, int L, int V, int ACT, bool CKPT>
__global__ void __launch_bounds__(32 * kRowWarps) norm_bwd_rows(NormParams p) {
  extern __shared__ float sf[];                            // [warps][2][32 V N]
  const RowAt a = row_at<L>(p);
  const int nvg = (int)p.cpg / N, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c0 = (int64_t)a.g * p.cpg, walker = blockIdx.x / p.nseg, walkers = gridDim.x / p.nseg;
  const float inv = 1.f / (float)p.cpg;
  float gam[V][N], bet[V][N], da[V][N], db[V][N];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = a.l + v * L < nvg;
      gam[v][i] = in ? ld_param(p.w, c0 + (a.l + v * L) * N + i, p.pdtype, 1.f) : 0.f;
      bet[v][i] = in ? ld_param(p.b, c0 + (a.l + v * L) * N + i, p.pdtype, 0.f) : 0.f;
      da[v][i] = db[v][i] = 0.f;
    }
  Raw<T, N> rx[V], rd[V];
  float mu = 0.f, rs = 0.f;
  const auto load = [&](int64_t s) {
    mu = p.mean[s * p.G + a.g];
    rs = p.rstd[s * p.G + a.g];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (a.l + v * L < nvg) {
        rx[v] = read_x<T, N, CKPT>(p, s, 0, c0 + (a.l + v * L) * N);
        rd[v] = read_dy<T, N>(p, s, 0, c0 + (a.l + v * L) * N);
      }
    }
  };
  int64_t s = walker * kRowWarps + warp;
  if (s < p.S) load(s);
  while (s < p.S) {
    float h[V][N], du[V][N], t1 = 0.f, t2 = 0.f;
    const float r = rs;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (a.l + v * L < nvg) {
        unpack<T, N>(rx[v], h[v]);
        unpack<T, N>(rd[v], du[v]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          h[v][i] = (h[v][i] - mu) * r;
          du[v][i] *= dense_slope<ACT, sizeof(T) == 2>(fmaf(h[v][i], gam[v][i], bet[v][i]));
          da[v][i] = fmaf(du[v][i], h[v][i], da[v][i]);
          db[v][i] += du[v][i];
          t1 = fmaf(du[v][i], gam[v][i], t1);
          t2 = fmaf(du[v][i] * gam[v][i], h[v][i], t2);
        }
      }
    }
    const int64_t cur = s;
    s += walkers * kRowWarps;
    if (s < p.S) load(s);                                  // the next sample's loads run under this one's reduction
    t1 = lanes_sum<L>(t1) * inv;
    t2 = lanes_sum<L>(t2) * inv;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (a.live && a.l + v * L < nvg) {
        float f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = r * (fmaf(du[v][i], gam[v][i], -t1) - h[v][i] * t2);
        store_vec<T, N>(reinterpret_cast<T*>(p.out) + cur * p.C + c0 + (a.l + v * L) * N, f);
      }
    }
  }
  constexpr int W = 32 * V * N;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      sf[(warp * 2) * W + (v * N + i) * 32 + lane] = da[v][i];
      sf[(warp * 2 + 1) * W + (v * N + i) * 32 + lane] = db[v][i];
    }
  __syncthreads();
  // thread -> (which, vector element, lane): sums over the warps, written by the lane's owner pattern
  for (int j = threadIdx.x; j < 2 * W; j += 32 * kRowWarps) {
    const int which = j / W, e = j - which * W, ln = e % 32, vi = e / 32, v = vi / N, i = vi - v * N;
    const int g = (int)blockIdx.x % (int)p.nseg * (32 / L) + ln / L, vec = ln % L + v * L;
    if (g >= (int)p.G || vec >= nvg) continue;
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) t += sf[(w * 2 + which) * W + e];
    p.part[(walker * 2 + which) * p.C + (int64_t)g * p.cpg + vec * N + i] = t;
  }
}

// ---- host ----
enum { kNormRows, kNormResident, kNormStream };
struct NormPlan {
  int kind, N, NT, ng, cs, L, V, nsub, subc;
  int64_t nseg, PR, chunks, walkers, npart, gparts;   // gparts: floats of gpart
  size_t smem;
};

// Which family, and its sizes.
//  rows       P = 1, aligned, a group of at most 8 vectors a lane (measured at 1024 x 4096 fp32 in 64 groups: forward
//             and backward 36 + 79 us resident, without it)
//  resident   a segment's positions fit a block's shared memory.  A segment is at least 128 bytes of channels (a full
//             line per position), wider while there are more than four segments for each SM; vectors do not straddle
//             segments.
//  streaming  otherwise
static NormPlan norm_plan(int64_t S, int64_t P, int64_t C, int64_t G, int esize, bool vec, bool bwd, int sms,
                          int smem_max) {
  NormPlan pl{};
  const int64_t cpg = C / G;
  pl.N = vec ? 16 / esize : 1;
  pl.nsub = 1;
  if (P == 1 && vec && cpg % pl.N == 0 && G < (1 << 30)) {
    const int64_t nvg = cpg / pl.N;
    int L = 1;
    while (L < 32 && L < nvg) L *= 2;
    int V = 1;
    while (V * L < nvg) V *= 2;
    if (V <= (bwd ? 4 : 8)) {
      pl.kind = kNormRows;
      pl.L = L;
      pl.V = V;
      pl.nseg = (G + 32 / L - 1) / (32 / L);
      const int64_t per = kRowWarps * (bwd ? 1 : (V >= 4 ? 1 : 4 / V));   // samples of a block at a time
      const int64_t most = (S + per - 1) / per, want = (sms * (bwd ? 4 : 8) + pl.nseg - 1) / pl.nseg;
      pl.walkers = most < want ? most : want;
      pl.npart = pl.walkers;
      pl.smem = bwd ? (size_t)kRowWarps * 2 * 32 * V * pl.N * 4 : 0;
      return pl;
    }
  }
  const int tiles = bwd ? 2 : 1;
  int64_t ng = 1;
  while (ng < G && (ng * cpg) % pl.N) ++ng;
  const int64_t unit = ng;
  while (ng + unit <= G && ng * cpg * esize < 128) ng += unit;
  if (ng > G || (ng * cpg) % pl.N) ng = G;
  while (ng * 2 <= G && S * ((G + 2 * ng - 1) / (2 * ng)) >= 4 * sms && P * ng * 2 * cpg * esize * tiles <= 32768) ng *= 2;
  pl.ng = (int)ng;
  const int64_t cs = ng * cpg;
  pl.nseg = (G + ng - 1) / ng;
  if (cs <= (1 << 20) && P <= (1 << 20)) {
    pl.cs = (int)cs;
    const int64_t tile = tiles * ((P * cs * esize + 15) / 16 * 16);
    const int NT = vec && tile > 32768 ? 512 : 256;
    const int64_t red = norm_red(cs, pl.N, NT);
    const int64_t bytes = tile + 4 * (bwd ? 2 * red + 2 * cs + 4 * ng : red + 4 * ng) + 32;
    if (tile <= smem_max && bytes <= smem_max) {
      pl.kind = kNormResident;
      pl.PR = P;
      pl.NT = NT;
      pl.smem = (size_t)bytes;
      int64_t per_sm = (smem_max + 1024) / (bytes + 1024);
      if (per_sm > 2048 / NT) per_sm = 2048 / NT;
      const int64_t want = (sms * per_sm + pl.nseg - 1) / pl.nseg;
      pl.walkers = S < want ? S : want;
      pl.npart = pl.walkers;
      return pl;
    }
  }
  // streaming: one wave of blocks, at least 16 positions each where there are that many; groups too wide for a block's
  // sums in parts of 4096 channels
  pl.kind = kNormStream;
  pl.NT = 256;
  while (ng + unit <= G && (ng + unit) * cpg <= 256 * pl.N) ng += unit;   // whole rows where they fit a row of threads
  pl.ng = (int)ng;
  pl.cs = (int)(ng * cpg);
  pl.nseg = (G + ng - 1) / ng;
  if (ng * cpg > 16384) {
    if (cpg % pl.N) pl.N = 1;      // parts start where groups do
    ng = 1;
    pl.subc = 4096;
    pl.nsub = (int)((cpg + pl.subc - 1) / pl.subc);
    pl.cs = pl.nsub > 1 ? pl.subc : (int)cpg;
    pl.ng = 1;
    pl.nseg = G * pl.nsub;
  }
  int64_t chunks = (int64_t)sms * (bwd ? kBwdBlocks : kFwdBlocks) / (S * pl.nseg);
  if (chunks < 1) chunks = 1;
  const int64_t most = (P + 15) / 16;
  if (chunks > most) chunks = most;
  pl.PR = (P + chunks - 1) / chunks;
  pl.chunks = (P + pl.PR - 1) / pl.PR;
  pl.npart = S * pl.chunks;
  pl.gparts = S * pl.chunks * G * pl.nsub * 2;
  pl.smem = (size_t)(4 * (2 * norm_red(pl.cs, pl.N, 256) + 2 * ng));
  return pl;
}

// Floats of workspace.
static int64_t norm_floats(const NormPlan& pl, int64_t C, bool bwd) {
  return (bwd ? pl.npart * 2 * C : 0) + pl.gparts;
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
static int launch_norm(K kernel, const NormParams& p, int64_t blocks, int threads, size_t smem, cudaStream_t st) {
  if (blocks > 0x7FFFFFFF) return GL_ERR_SHAPE;
  if (int rc = ensure_dynamic_smem((const void*)kernel, smem)) return rc;
  kernel<<<(unsigned)blocks, (unsigned)threads, smem, st>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e);
  count_launches(1);
  return GL_OK;
}

// f(ActTag L, ActTag V) for a row plan (the tags carry plain integers).
template <int MAXV, typename F>
static void with_row_shape(int L, int V, F f) {
  const auto pick_v = [&](auto l) {
    if (V == 1) f(l, ActTag<1>());
    if constexpr (decltype(l)::value == 32) {      // more than one vector a lane only with all 32 lanes
      if (V == 2) f(l, ActTag<2>());
      if (V == 4) f(l, ActTag<4>());
      if constexpr (MAXV >= 8)
        if (V == 8) f(l, ActTag<8>());
    }
  };
  switch (L) {
    case 1: pick_v(ActTag<1>()); break;
    case 2: pick_v(ActTag<2>()); break;
    case 4: pick_v(ActTag<4>()); break;
    case 8: pick_v(ActTag<8>()); break;
    case 16: pick_v(ActTag<16>()); break;
    default: pick_v(ActTag<32>()); break;
  }
}

template <typename T, int N, int ACT>
static int run_norm_fwd_act(NormParams& p, const NormPlan& pl, cudaStream_t st) {
  if constexpr (N > 1) {
    if (pl.kind == kNormRows) {
      int rc = GL_ERR_UNSUPPORTED;
      with_row_shape<8>(pl.L, pl.V, [&](auto l, auto v) {
        rc = launch_norm(norm_fwd_rows<T, N, decltype(l)::value, decltype(v)::value, ACT>, p, pl.nseg * pl.walkers,
                         32 * kRowWarps, 0, st);
      });
      return rc;
    }
    if (pl.kind == kNormResident && pl.NT == 512)
      return launch_norm(norm_fwd_resident<T, N, 512, ACT>, p, p.S * pl.nseg, 512, pl.smem, st);
  }
  if (pl.kind == kNormResident)
    return launch_norm(norm_fwd_resident<T, N, 256, ACT>, p, p.S * pl.nseg, 256, pl.smem, st);
  const int64_t blocks = p.S * pl.chunks * pl.nseg;
  if (int rc = launch_norm(norm_stats_kernel<T, N, 256>, p, blocks, 256, pl.smem, st)) return rc;
  return launch_norm(norm_apply_kernel<T, N, 256, ACT>, p, blocks, 256, pl.smem, st);
}

template <typename T, int N>
static int run_norm_fwd(NormParams& p, int act, const NormPlan& pl, cudaStream_t st) {
  int rc = GL_ERR_UNSUPPORTED;
  with_act(act, [&](auto tag) { rc = run_norm_fwd_act<T, N, decltype(tag)::value>(p, pl, st); });
  return rc;
}

template <typename T, int N, int ACT, bool CKPT>
static int run_norm_bwd_act(NormParams& p, const NormPlan& pl, cudaStream_t st) {
  const int64_t joins = p.dw || p.db ? (p.C + 31) / 32 : 0;
  int rc = GL_ERR_UNSUPPORTED;
  if (pl.kind == kNormStream) {
    p.blocks = p.S * pl.chunks * pl.nseg;
    const size_t smem = pl.smem < 8 * 2 * 33 * 4 ? 8 * 2 * 33 * 4 : pl.smem;
    rc = launch_norm(norm_bwd_stats_kernel<T, N, 256, ACT, CKPT>, p, p.blocks, 256, pl.smem, st);
    if (rc) return rc;
    return launch_norm(norm_bwd_apply_kernel<T, N, 256, ACT, CKPT>, p, p.blocks + joins, 256, smem, st);
  }
  if constexpr (N > 1) {
    if (pl.kind == kNormRows) {
      with_row_shape<4>(pl.L, pl.V, [&](auto l, auto v) {
        rc = launch_norm(norm_bwd_rows<T, N, decltype(l)::value, decltype(v)::value, ACT, CKPT>, p,
                            pl.nseg * pl.walkers, 32 * kRowWarps, pl.smem, st);
      });
    } else if (pl.NT == 512) {
      rc = launch_norm(norm_bwd_resident<T, N, 512, ACT, CKPT>, p, pl.walkers * pl.nseg, 512, pl.smem, st);
    }
  }
  if (pl.kind == kNormResident && pl.NT == 256)
    rc = launch_norm(norm_bwd_resident<T, N, 256, ACT, CKPT>, p, pl.walkers * pl.nseg, 256, pl.smem, st);
  if (rc || !joins) return rc;
  norm_param_join_kernel<<<(unsigned)joins, 512, 0, st>>>(p.part, pl.npart, p.C, p.dw, p.db, p.pdtype, p.accumulate);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e);
  count_launches(1);
  return GL_OK;
}

template <typename T, int N, bool CKPT>
static int run_norm_bwd(NormParams& p, int act, const NormPlan& pl, cudaStream_t st) {
  int rc = GL_ERR_UNSUPPORTED;
  with_act(act, [&](auto tag) { rc = run_norm_bwd_act<T, N, decltype(tag)::value, CKPT>(p, pl, st); });
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
    const int64_t n = 4 * norm_floats(pl, C, backward != 0);
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
  if (off_type(a.dtype == GL_DTYPE_F32 ? 4 : 2, a.x, a.y) || off_type(a.pdtype == GL_DTYPE_F32 ? 4 : 2, a.w, a.b) ||
      off_type(4, a.mean, a.rstd) || off_type(16, a.work))
    return GL_ERR_ALIGN;
  int sms = 0, smem = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (int rc = device_smem_optin(&smem)) return rc;
  const int esize = a.dtype == GL_DTYPE_F32 ? 4 : 2;
  const bool vec = vec_rows(a.x, a.sx, a.px, a.C, esize) && vec_rows(a.y, 0, 0, a.C, esize);
  const NormPlan pl = norm_plan(a.S, a.P, a.C, a.G, esize, vec, false, sms, smem);
  if (pl.gparts > 0 && (!a.work || a.work_bytes < 4 * pl.gparts)) return GL_ERR_WORKSPACE;
  NormParams p{};
  p.x = a.x; p.w = a.w; p.b = a.b; p.out = a.y; p.mean = a.mean; p.rstd = a.rstd; p.gpart = (float*)a.work;
  p.S = a.S; p.P = a.P; p.C = a.C; p.G = a.G; p.cpg = a.C / a.G; p.sx = a.sx; p.px = a.px;
  p.nseg = pl.nseg; p.PR = pl.PR; p.chunks = pl.chunks; p.ng = pl.ng; p.cs = pl.cs;
  p.nsub = pl.nsub; p.subc = pl.subc;
  p.pdtype = a.pdtype; p.eps = a.eps;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.dtype == GL_DTYPE_F32) return pl.N > 1 ? run_norm_fwd<float, 4>(p, a.act, pl, st) : run_norm_fwd<float, 1>(p, a.act, pl, st);
  return pl.N > 1 ? run_norm_fwd<__nv_bfloat16, 8>(p, a.act, pl, st) : run_norm_fwd<__nv_bfloat16, 1>(p, a.act, pl, st);
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
  if (off_type(a.dtype == GL_DTYPE_F32 ? 4 : 2, ckpt ? nullptr : a.x, a.dy, a.dx) ||
      off_type(a.pdtype == GL_DTYPE_F32 ? 4 : 2, a.w, a.b) ||
      off_type(a.accumulate || a.pdtype == GL_DTYPE_F32 ? 4 : 2, a.dw, a.db) || off_type(4, a.mean, a.rstd) ||
      off_type(16, a.work, a.codes))
    return GL_ERR_ALIGN;
  int sms = 0, smem = 0;
  if (int rc = device_sm_count(&sms)) return rc;
  if (int rc = device_smem_optin(&smem)) return rc;
  const int esize = a.dtype == GL_DTYPE_F32 ? 4 : 2;
  const bool vec = (ckpt || vec_rows(a.x, a.sx, a.px, a.C, esize)) && vec_rows(a.dy, a.sdy, a.pdy, a.C, esize) &&
                   vec_rows(a.dx, 0, 0, a.C, esize);
  const NormPlan pl = norm_plan(a.S, a.P, a.C, a.G, esize, vec, true, sms, smem);
  if (a.work_bytes < 4 * norm_floats(pl, a.C, true)) return GL_ERR_WORKSPACE;
  NormParams p{};
  p.x = a.x; p.dy = a.dy; p.w = a.w; p.b = a.b; p.codes = a.codes; p.exps = a.exps; p.out = a.dx;
  p.mean = const_cast<float*>(a.mean); p.rstd = const_cast<float*>(a.rstd); p.part = (float*)a.work;
  p.gpart = p.part + pl.npart * 2 * a.C; p.dw = a.dw; p.db = a.db; p.accumulate = a.accumulate;
  p.S = a.S; p.P = a.P; p.C = a.C; p.G = a.G; p.cpg = a.C / a.G; p.sx = a.sx; p.px = a.px; p.sdy = a.sdy;
  p.pdy = a.pdy; p.ldc = a.ldc; p.nblk = nblk; p.nseg = pl.nseg; p.npart = pl.npart; p.PR = pl.PR;
  p.chunks = pl.chunks; p.ng = pl.ng; p.cs = pl.cs;
  p.nsub = pl.nsub; p.subc = pl.subc; p.pdtype = a.pdtype;
  if (a.dtype == GL_DTYPE_F32) {
    if (ckpt) return pl.N > 1 ? run_norm_bwd<float, 4, true>(p, a.act, pl, st) : run_norm_bwd<float, 1, true>(p, a.act, pl, st);
    return pl.N > 1 ? run_norm_bwd<float, 4, false>(p, a.act, pl, st) : run_norm_bwd<float, 1, false>(p, a.act, pl, st);
  }
  using B = __nv_bfloat16;
  if (ckpt) return pl.N > 1 ? run_norm_bwd<B, 8, true>(p, a.act, pl, st) : run_norm_bwd<B, 1, true>(p, a.act, pl, st);
  return pl.N > 1 ? run_norm_bwd<B, 8, false>(p, a.act, pl, st) : run_norm_bwd<B, 1, false>(p, a.act, pl, st);
}

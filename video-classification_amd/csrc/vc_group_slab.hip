// Group normalisation in one pass over the data: a workgroup takes a slab of W channels -- whole groups, 16 to 128 bytes of a
// row -- of one sample, holds all S positions of it in registers, and reads and writes every element once (the two-pass
// form of vc_group.hip reads the input twice forward, input and gradient twice backward).
//
// Covered: groups of 1, 2, 4, 8, .. 64 channels whose slab fits the register file, up to 512 threads x 28 (bf16) or 16
// (fp32) vectors of eight values forward and 8 backward, which holds the input and the gradient.  (512 threads with 256
// registers each hold as much as 1024 with 128 and spend half as many on what every thread needs besides the data.)  The slabs
// of a sample lie next to each other on one XCD, so the parts of a 128-byte line that different slabs read meet in its L2.
//
// Bound by memory: 128 x 56 x 56 x 256 bf16 forward 105 us (3.9 TB/s; two passes take 45 us more), 64 x 28 x
// 28 x 512 with a shortcut 28 us (5.4 TB/s, partly from the last-level cache), 2 x 7 x 7 x 512 in one launch of 5 us.
#include "vc_group.h"

namespace {

// Eight values as they lie in memory.  again() hides where the registers came from, so that a later pass unpacks bf16 once
// more instead of the compiler keeping the fp32 form, twice the size, alive in between.
template <typename T>
struct Vec8;
template <>
struct Vec8<bf16> {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  u32x4 v;
  __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const u32x4*>(p); }
  __device__ __forceinline__ void zero() { v = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ float operator[](int i) const {
    return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
  }
  __device__ __forceinline__ void again() { asm volatile("" : "+v"(v)); }
};
template <>
struct Vec8<float> {
  f32x4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = *reinterpret_cast<const f32x4*>(p);
    b = *reinterpret_cast<const f32x4*>(p + 4);
  }
  __device__ __forceinline__ void zero() { a = b = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ float operator[](int i) const { return i < 4 ? a[i & 3] : b[i & 3]; }
  __device__ __forceinline__ void again() {}
};

struct Slab {
  int S, C, G, cpg;
  int lg;      // log2 of the vector columns of a slab
  int slabs;   // slabs of a sample
  int gspan;   // vector columns of a group (1 where a vector holds several groups)
};

__device__ __forceinline__ int slab_run(int id, int total) {  // workgroups of one XCD take a contiguous run
  const int q = total >> 3, r = total & 7, xcd = id & 7, idx = id >> 3;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

// Sums of NV values per thread over the thread rows of its column (and over the columns of its group), the same for every
// thread of them.  red: one buffer per call.
template <int NT, int NV>
__device__ __forceinline__ void slab_sum(float (&s)[NV], float (&red)[NT / 64][8][NV], int lg, int gspan) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cvb = 1 << lg;
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    for (int o = cvb; o < 64; o <<= 1) s[g] += __shfl_xor(s[g], o, 64);
    for (int o = 1; o < gspan; o <<= 1) s[g] += __shfl_xor(s[g], o, 64);
  }
  if (lane < cvb)
#pragma unroll
    for (int g = 0; g < NV; ++g) red[wave][lane][g] = s[g];
  __syncthreads();
  const int tx = threadIdx.x & (cvb - 1);
#pragma unroll
  for (int g = 0; g < NV; ++g) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) t += red[w][tx][g];
    s[g] = t;
  }
}

template <int ACT, int NGV, typename T, int K>
__device__ __forceinline__ void slab_write(const Vec8<T> (&v)[K], const T* res, T* y, size_t at, size_t step, int ty, int ry,
                                           int S, const float (&mu)[NGV], const float (&a)[8], const float (&be)[8]) {
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (ty + j * ry >= S) continue;
    F8 o;
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = fmaf(v[j][i] - mu[i * NGV / 8], a[i], be[i]);
    if (res) {
      const F8 e = load8(res + at + j * step);
#pragma unroll
      for (int i = 0; i < 8; ++i) o.v[i] += e.v[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) o.v[i] = act_fwd<ACT>(o.v[i]);
    store8(y + at + j * step, o);
  }
}

// NGV: groups of one vector (8 / cpg, at least 1)
template <typename T, int NT, int K, int NGV>
__global__ __launch_bounds__(NT) void gn_slab_fwd_kernel(Slab k, const T* __restrict__ x, const T* __restrict__ res,
                                                         const float* __restrict__ gamma, const float* __restrict__ beta,
                                                         T* __restrict__ y, float* __restrict__ mean,
                                                         float* __restrict__ rstd, float eps, int act) {
  __shared__ float r1[NT / 64][8][NGV], r2[NT / 64][8][NGV];
  const int v0 = slab_run(blockIdx.x, gridDim.x), n = v0 / k.slabs;
  const int tx = threadIdx.x & ((1 << k.lg) - 1), ty = threadIdx.x >> k.lg, ry = NT >> k.lg;
  const int c = (((v0 - n * k.slabs) << k.lg) + tx) * 8;
  const size_t at = ((size_t)n * k.S + ty) * k.C + c, step = (size_t)ry * k.C;
  Vec8<T> v[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (ty + j * ry < k.S) v[j].load(x + at + j * step);
    else v[j].zero();
  }
  float s[NGV];
#pragma unroll
  for (int g = 0; g < NGV; ++g) s[g] = 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i * NGV / 8] += v[j][i];
  slab_sum<NT, NGV>(s, r1, k.lg, k.gspan);
  const float m = (float)k.S * (float)k.cpg;
  float mu[NGV], q[NGV];
#pragma unroll
  for (int g = 0; g < NGV; ++g) {
    mu[g] = s[g] / m;
    q[g] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < K; ++j) v[j].again();
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (ty + j * ry < k.S)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = v[j][i] - mu[i * NGV / 8];
        q[i * NGV / 8] = fmaf(d, d, q[i * NGV / 8]);
      }
  slab_sum<NT, NGV>(q, r2, k.lg, k.gspan);
#pragma unroll
  for (int g = 0; g < NGV; ++g) {
    q[g] = 1.f / sqrtf(q[g] / m + eps);
    if (ty == 0 && (tx & (k.gspan - 1)) == 0) {
      const size_t o = (size_t)n * k.G + c / k.cpg + g;
      mean[o] = mu[g];
      rstd[o] = q[g];
    }
  }
#pragma unroll
  for (int j = 0; j < K; ++j) v[j].again();
  float ga[8], be[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ga[i] = (gamma ? gamma[c + i] : 1.f) * q[i * NGV / 8];
    be[i] = beta ? beta[c + i] : 0.f;
  }
  if (act == ACT_RELU) slab_write<ACT_RELU, NGV, T, K>(v, res, y, at, step, ty, ry, k.S, mu, ga, be);
  else if (act == ACT_SILU) slab_write<ACT_SILU, NGV, T, K>(v, res, y, at, step, ty, ry, k.S, mu, ga, be);
  else if (act == ACT_GELU) slab_write<ACT_GELU, NGV, T, K>(v, res, y, at, step, ty, ry, k.S, mu, ga, be);
  else slab_write<ACT_NONE, NGV, T, K>(v, res, y, at, step, ty, ry, k.S, mu, ga, be);
}

template <typename T, int NT, int K, int NGV>
struct SlabBwd {
  float (&red)[NT / 64][8][16];
  float (&tot)[64][2];
  const Slab& k;
  const T* res;
  const float* gamma;
  float* ab;
  T *dx, *dres;

  template <int ACT>
  __device__ __forceinline__ void go(Vec8<T> (&v)[K], Vec8<T> (&g)[K], int n, int tx, int ty, int ry, int c, size_t at,
                                     size_t step, const float (&mu)[NGV], const float (&rs)[NGV], const float (&ga)[8],
                                     const float (&be)[8]) {
    float s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (ty + j * ry >= k.S) continue;
      F8 e;
      if (ACT != ACT_NONE && res) e = load8(res + at + j * step);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xh = (v[j][i] - mu[i * NGV / 8]) * rs[i * NGV / 8];
        float z = fmaf(xh, ga[i], be[i]);
        if (ACT != ACT_NONE && res) z += e.v[i];
        const float dz = g[j][i] * act_slope<ACT>(z);
        s[2 * i] += dz;
        s[2 * i + 1] = fmaf(dz, xh, s[2 * i + 1]);
      }
    }
    slab_sum<NT, 16>(s, red, k.lg, 1);
    if (ty == 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        tot[tx * 8 + i][0] = s[2 * i];
        tot[tx * 8 + i][1] = s[2 * i + 1];
        ab[(size_t)n * 2 * k.C + c + i] = s[2 * i];
        ab[(size_t)n * 2 * k.C + k.C + c + i] = s[2 * i + 1];
      }
    if (!dx && !dres) return;
    __syncthreads();
    const float m = (float)k.S * (float)k.cpg;
    float c1[NGV], c2[NGV];
#pragma unroll
    for (int q = 0; q < NGV; ++q) {
      const int first = (tx * 8 + q * (8 / NGV)) / k.cpg * k.cpg;  // of the group, within the slab
      const float* gp = gamma ? gamma + c - tx * 8 + first : nullptr;
      c1[q] = c2[q] = 0.f;
      for (int i = 0; i < k.cpg; ++i) {
        const float w = gp ? gp[i] : 1.f;
        c1[q] = fmaf(w, tot[first + i][0], c1[q]);
        c2[q] = fmaf(w, tot[first + i][1], c2[q]);
      }
      c1[q] /= m;
      c2[q] /= m;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      v[j].again();
      g[j].again();
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (ty + j * ry >= k.S) continue;
      F8 e, d, o;
      if (ACT != ACT_NONE && res) e = load8(res + at + j * step);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float xh = (v[j][i] - mu[i * NGV / 8]) * rs[i * NGV / 8];
        float z = fmaf(xh, ga[i], be[i]);
        if (ACT != ACT_NONE && res) z += e.v[i];
        d.v[i] = g[j][i] * act_slope<ACT>(z);
        o.v[i] = rs[i * NGV / 8] * (fmaf(ga[i], d.v[i], -c1[i * NGV / 8]) - xh * c2[i * NGV / 8]);
      }
      if (dx) store8(dx + at + j * step, o);
      if (dres) store8(dres + at + j * step, d);
    }
  }
};

template <typename T, int NT, int K, int NGV>
__global__ __launch_bounds__(NT) void gn_slab_bwd_kernel(Slab k, const T* __restrict__ x, const T* __restrict__ dy,
                                                         const T* __restrict__ res, const float* __restrict__ gamma,
                                                         const float* __restrict__ beta, const float* __restrict__ mean,
                                                         const float* __restrict__ rstd, T* __restrict__ dx,
                                                         T* __restrict__ dres, float* __restrict__ ab, int act) {
  __shared__ float red[NT / 64][8][16];
  __shared__ float tot[64][2];
  const int v0 = slab_run(blockIdx.x, gridDim.x), n = v0 / k.slabs;
  const int tx = threadIdx.x & ((1 << k.lg) - 1), ty = threadIdx.x >> k.lg, ry = NT >> k.lg;
  const int c = (((v0 - n * k.slabs) << k.lg) + tx) * 8;
  const size_t at = ((size_t)n * k.S + ty) * k.C + c, step = (size_t)ry * k.C;
  Vec8<T> v[K], g[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (ty + j * ry < k.S) {
      v[j].load(x + at + j * step);
      g[j].load(dy + at + j * step);
    } else {
      v[j].zero();
      g[j].zero();
    }
  }
  float mu[NGV], rs[NGV], ga[8], be[8];
#pragma unroll
  for (int q = 0; q < NGV; ++q) {
    const size_t o = (size_t)n * k.G + c / k.cpg + q;
    mu[q] = mean[o];
    rs[q] = rstd[o];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    ga[i] = gamma ? gamma[c + i] : 1.f;
    be[i] = beta ? beta[c + i] : 0.f;
  }
  SlabBwd<T, NT, K, NGV> b{red, tot, k, res, gamma, ab, dx, dres};
  if (act == ACT_RELU) b.template go<ACT_RELU>(v, g, n, tx, ty, ry, c, at, step, mu, rs, ga, be);
  else if (act == ACT_SILU) b.template go<ACT_SILU>(v, g, n, tx, ty, ry, c, at, step, mu, rs, ga, be);
  else if (act == ACT_GELU) b.template go<ACT_GELU>(v, g, n, tx, ty, ry, c, at, step, mu, rs, ga, be);
  else b.template go<ACT_NONE>(v, g, n, tx, ty, ry, c, at, step, mu, rs, ga, be);
}

// The slab of a call, or false: vector columns 2^lg so that S positions of it fit `most` vectors per workgroup.  The widest
// slab that fits, up to 128 bytes of a row, narrowed while that leaves CUs without a workgroup.
bool pick(Slab& k, int esize, int N, int S, int C, int G, int64_t most) {
  const int cpg = C / G;
  if (C % 8 || cpg > 64 || (cpg & (cpg - 1))) return false;
  const int span = cpg > 8 ? cpg / 8 : 1, cv = C / 8;
  int lg = 0;
  while ((1 << lg) < span) ++lg;
  const int least = lg;
  if (((int64_t)S << lg) > most || cv % (1 << lg)) return false;
  while (lg < 3 && (16 << lg) * (esize / 2) < 128 && cv % (2 << lg) == 0 && ((int64_t)S << (lg + 1)) <= most) ++lg;
  // 16-byte pieces of rows waste most of every line unless the tensor fits the L2s (56 x 56 x 256 bf16 backward: 450 us
  // against 230 in two passes)
  if ((8 << lg) * esize < 32 && cv > (1 << lg) && (int64_t)N * S * C * esize > (16 << 20)) return false;
  while (lg > least && (int64_t)N * (cv >> lg) < 256) --lg;
  k.S = S;
  k.C = C;
  k.G = G;
  k.cpg = cpg;
  k.lg = lg;
  k.slabs = cv >> lg;
  k.gspan = span;
  return (int64_t)N * k.slabs < (1ll << 23);  // a launch holds fewer than 2^32 threads, 512 to a slab
}

#define BY_GROUPS(cpg, ...)                                          \
  do {                                                               \
    if (cpg >= 8) { constexpr int NGV = 1; __VA_ARGS__; }            \
    else if (cpg == 4) { constexpr int NGV = 2; __VA_ARGS__; }       \
    else if (cpg == 2) { constexpr int NGV = 4; __VA_ARGS__; }       \
    else { constexpr int NGV = 8; __VA_ARGS__; }                     \
  } while (0)

template <typename T, int NT, int K>
void fwd_go(const Slab& k, int N, const void* x, const void* res, const float* gamma, const float* beta, void* y, float* mean,
            float* rstd, float eps, int act, hipStream_t st) {
  BY_GROUPS(k.cpg, hipLaunchKernelGGL((gn_slab_fwd_kernel<T, NT, K, NGV>), dim3(N * k.slabs), dim3(NT), 0, st, k, (const T*)x,
                                      (const T*)res, gamma, beta, (T*)y, mean, rstd, eps, act));
}
template <typename T, int NT, int K>
void bwd_go(const Slab& k, int N, const void* x, const void* dy, const void* res, const float* gamma, const float* beta,
            const float* mean, const float* rstd, void* dx, void* dres, float* ab, int act, hipStream_t st) {
  BY_GROUPS(k.cpg, hipLaunchKernelGGL((gn_slab_bwd_kernel<T, NT, K, NGV>), dim3(N * k.slabs), dim3(NT), 0, st, k, (const T*)x,
                                      (const T*)dy, (const T*)res, gamma, beta, mean, rstd, (T*)dx, (T*)dres, ab, act));
}

template <typename T>
bool fwd_by_size(const void* x, const void* res, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                 int N, int S, int C, int G, float eps, int act, hipStream_t st) {
  constexpr bool two = sizeof(T) == 2;
  Slab k;
  if (!pick(k, sizeof(T), N, S, C, G, 512 * (two ? 28 : 16))) return false;
  const int64_t v = (int64_t)S << k.lg;
  if (v <= 256 * 4) fwd_go<T, 256, 4>(k, N, x, res, gamma, beta, y, mean, rstd, eps, act, st);
  else if (v <= 512 * 8) fwd_go<T, 512, 8>(k, N, x, res, gamma, beta, y, mean, rstd, eps, act, st);
  else if (v <= 512 * 16) fwd_go<T, 512, 16>(k, N, x, res, gamma, beta, y, mean, rstd, eps, act, st);
  else if constexpr (two) fwd_go<T, 512, 28>(k, N, x, res, gamma, beta, y, mean, rstd, eps, act, st);
  return true;
}
template <typename T>
bool bwd_by_size(const void* x, const void* dy, const void* res, const float* gamma, const float* beta, const float* mean,
                 const float* rstd, void* dx, void* dres, float* ab, int N, int S, int C, int G, int act, hipStream_t st) {
  Slab k;
  if (!pick(k, sizeof(T), N, S, C, G, 512 * 8)) return false;
  const int64_t v = (int64_t)S << k.lg;
  if (v <= 256 * 4) bwd_go<T, 256, 4>(k, N, x, dy, res, gamma, beta, mean, rstd, dx, dres, ab, act, st);
  else bwd_go<T, 512, 8>(k, N, x, dy, res, gamma, beta, mean, rstd, dx, dres, ab, act, st);
  return true;
}

}  // namespace

bool vc_gn_slab_fwd(int dtype, const void* x, const void* res, const float* gamma, const float* beta, void* y, float* mean,
                    float* rstd, int N, int S, int C, int G, float eps, int act, hipStream_t st) {
  return dtype == VC_BF16 ? fwd_by_size<bf16>(x, res, gamma, beta, y, mean, rstd, N, S, C, G, eps, act, st)
                          : fwd_by_size<float>(x, res, gamma, beta, y, mean, rstd, N, S, C, G, eps, act, st);
}
bool vc_gn_slab_bwd(int dtype, const void* x, const void* dy, const void* res, const float* gamma, const float* beta,
                    const float* mean, const float* rstd, void* dx, void* dres, float* ab, int N, int S, int C, int G,
                    int act, hipStream_t st) {
  return dtype == VC_BF16 ? bwd_by_size<bf16>(x, dy, res, gamma, beta, mean, rstd, dx, dres, ab, N, S, C, G, act, st)
                          : bwd_by_size<float>(x, dy, res, gamma, beta, mean, rstd, dx, dres, ab, N, S, C, G, act, st);
}

// Group normalisation with its activation on channels-last maps x[n][s][c] (n samples of S positions and C channels),
// forward and backward, fp32 / bf16 storage, fp32 arithmetic.
//
//   group g of sample n: m = S * C / G values, mean and (biased) variance over them, rstd = 1 / sqrt(var + eps)
//   z = (x - mean) * rstd * gamma_c + beta_c (+ residual),   y = act(z)
//   dz = dy * act'(z);  A_c = sum_s dz, B_c = sum_s dz * xhat;  dgamma_c += sum_n B_c, dbeta_c += sum_n A_c
//   dx = rstd * (gamma_c * dz - c1 - xhat * c2),  c1 = sum_{c in g} gamma_c A_c / m,  c2 = sum_{c in g} gamma_c B_c / m
//
// All of it is bound by memory.  128 x 56 x 56 x 256 in bf16 (206 MB a map): backward 110 us for the sums (3.7 TB/s), 121 us
// for the gradients (5.1 TB/s), 11 us of joins; a large copy runs at 4.8 TB/s.  Sums never use atomics: every block writes
// the partial sums of its own rows and a small kernel joins them in a fixed order, so results repeat bit for bit.
//
// Variance without cancellation: a thread sums (x - p) and (x - p)^2 around p, the first value it meets of that channel,
// which costs one subtraction more than raw sums and keeps the error of a thread's second moment at (its row count) units
// in the last place of that moment itself, however far the mean lies from zero.  Threads, blocks and channels are then
// joined by the exact identity for the union of two samples (means and second moments about the means).
#include <initializer_list>

#include "vc_group.h"

namespace {

constexpr int GT = 256;  // threads per block

template <typename T, int V>
__device__ __forceinline__ void loadv(const T* p, float (&v)[V]) {
  if constexpr (V == 8) {
    const F8 r = load8(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = r.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(p[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void storev(T* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    F8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = v[i];
    store8(p, r);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = from_f32<T>(v[i]);
  }
}

// How a launch covers [N][S][C]: a block owns `rows` consecutive positions of one sample and up to 256 vector columns;
// its threads are `ry` rows of `cvb` columns (the rest idle when cvb does not divide 256).
struct Cover {
  int S, C, G, cpg;
  int cv;      // vector columns of a row, C / V
  int cvb;     // vector columns of a block, min(cv, 256)
  int ry;      // thread rows
  int rows;    // positions per block
  int chunks;  // blocks along S
};

// grid (chunks, N, column slabs)
template <int V>
struct Slot {
  int tx, ty, n, r0, r1, c;
  bool on;
  __device__ __forceinline__ Slot(const Cover& k) {
    ty = threadIdx.x / k.cvb;
    tx = threadIdx.x - ty * k.cvb;
    n = blockIdx.y;
    r0 = blockIdx.x * k.rows;
    r1 = min(k.S, r0 + k.rows);
    const int col = blockIdx.z * k.cvb + tx;
    c = col * V;
    on = ty < k.ry && col < k.cv;
  }
};

// part[(n * chunks + chunk) * 2 * C + c] = mean of the block's rows of channel c, [... + C + c] = their second moment
template <typename T, int V>
__global__ __launch_bounds__(GT) void gn_stats_kernel(Cover k, const T* __restrict__ x, float* __restrict__ part) {
  __shared__ float sm[GT * V], sq[GT * V];
  __shared__ float sn[GT];
  const Slot<V> t(k);
  float p[V], s[V], q[V];
  int cnt = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] = s[i] = q[i] = 0.f;
  if (t.on && t.r0 + t.ty < t.r1) {
    const T* xp = x + ((size_t)t.n * k.S + t.r0 + t.ty) * k.C + t.c;
    const size_t step = (size_t)k.ry * k.C;
    loadv<T, V>(xp, p);
    cnt = 1;
    int r = t.r0 + t.ty + k.ry;
    xp += step;
    for (; r + 3 * k.ry < t.r1; r += 4 * k.ry, xp += 4 * step, cnt += 4) {
      float v[4][V];
#pragma unroll
      for (int u = 0; u < 4; ++u) loadv<T, V>(xp + u * step, v[u]);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = v[u][i] - p[i];
          s[i] += d;
          q[i] = fmaf(d, d, q[i]);
        }
    }
    for (; r < t.r1; r += k.ry, xp += step, ++cnt) {
      float v[V];
      loadv<T, V>(xp, v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = v[i] - p[i];
        s[i] += d;
        q[i] = fmaf(d, d, q[i]);
      }
    }
  }
  const float inv = cnt ? 1.f / (float)cnt : 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sm[threadIdx.x * V + i] = p[i] + s[i] * inv;
    sq[threadIdx.x * V + i] = fmaxf(0.f, q[i] - s[i] * s[i] * inv);
    if (q[i] != q[i]) sq[threadIdx.x * V + i] = q[i];
  }
  sn[threadIdx.x] = (float)cnt;
  // join thread rows pairwise: rows [0, w) take rows [w, 2w); counts are those of whole thread rows, never of columns
  int w = 1;
  while (w < k.ry) w <<= 1;
  for (w >>= 1; w > 0; w >>= 1) {
    __syncthreads();
    const int a = threadIdx.x, b = a + w * k.cvb;
    if (t.on && t.ty < w && t.ty + w < k.ry && sn[b] > 0.f) {  // thread rows fill from the front: sn[a] >= sn[b]
      const float na = sn[a], nb = sn[b], wb = nb / (na + nb);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = sm[b * V + i] - sm[a * V + i];
        sm[a * V + i] += d * wb;
        sq[a * V + i] += sq[b * V + i] + d * d * (na * wb);
      }
      sn[a] = na + nb;
    }
  }
  if (t.on && t.ty == 0) {  // a column's sums end in its own thread of row 0
    float* o = part + ((size_t)t.n * k.chunks + blockIdx.x) * 2 * k.C + t.c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o[i] = sm[threadIdx.x * V + i];
      o[k.C + i] = sq[threadIdx.x * V + i];
    }
  }
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// One wave per (group, sample): mean and rstd of the group from its chunks x channels partial statistics.
__global__ __launch_bounds__(64) void gn_join_kernel(Cover k, const float* __restrict__ part, float* __restrict__ mean,
                                                     float* __restrict__ rstd, float eps) {
  const int g = blockIdx.x, n = blockIdx.y;
  const float* p = part + (size_t)n * k.chunks * 2 * k.C + (size_t)g * k.cpg;
  const int items = k.chunks * k.cpg;
  const double total = (double)k.S * k.cpg;
  double a = 0.0;
  for (int i = threadIdx.x; i < items; i += 64) {
    const int ch = i / k.cpg, c = i - ch * k.cpg;
    a += (double)min(k.rows, k.S - ch * k.rows) * (double)p[(size_t)ch * 2 * k.C + c];
  }
  const double mu = wave_sum_d(a) / total;
  double m2 = 0.0;
  for (int i = threadIdx.x; i < items; i += 64) {
    const int ch = i / k.cpg, c = i - ch * k.cpg;
    const float* e = p + (size_t)ch * 2 * k.C + c;
    const double d = (double)e[0] - mu;
    m2 += (double)e[k.C] + (double)min(k.rows, k.S - ch * k.rows) * d * d;
  }
  m2 = wave_sum_d(m2);
  if (threadIdx.x == 0) {
    mean[(size_t)n * k.G + g] = (float)mu;
    rstd[(size_t)n * k.G + g] = (float)(1.0 / sqrt(m2 / total + (double)eps));
  }
}

// per-channel constants of a thread: mean, rstd, gamma, beta
template <int V>
struct Chan {
  float mu[V], rs[V], ga[V], be[V];
  __device__ __forceinline__ Chan(const Cover& k, int n, int c, const float* mean, const float* rstd, const float* gamma,
                                  const float* beta) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int g = (c + i) / k.cpg;
      mu[i] = mean[(size_t)n * k.G + g];
      rs[i] = rstd[(size_t)n * k.G + g];
      ga[i] = gamma ? gamma[c + i] : 1.f;
      be[i] = beta ? beta[c + i] : 0.f;
    }
  }
};

// y = act((x - mean) * rstd * gamma + beta (+ res))
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(GT) void gn_apply_kernel(Cover k, const T* __restrict__ x, const T* __restrict__ res,
                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                      const float* __restrict__ gamma, const float* __restrict__ beta,
                                                      T* __restrict__ y) {
  const Slot<V> t(k);
  if (!t.on) return;
  const Chan<V> h(k, t.n, t.c, mean, rstd, gamma, beta);
  float a[V];
#pragma unroll
  for (int i = 0; i < V; ++i) a[i] = h.rs[i] * h.ga[i];
  size_t o = ((size_t)t.n * k.S + t.r0 + t.ty) * k.C + t.c;
  const size_t step = (size_t)k.ry * k.C;
#pragma unroll 4
  for (int r = t.r0 + t.ty; r < t.r1; r += k.ry, o += step) {
    float v[V], e[V];
    loadv<T, V>(x + o, v);
    if (RES) loadv<T, V>(res + o, e);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float z = fmaf(v[i] - h.mu[i], a[i], h.be[i]);
      if (RES) z += e[i];
      v[i] = act_fwd<ACT>(z);
    }
    storev<T, V>(y + o, v);
  }
}

// part[(n * chunks + chunk) * 2 * C + c] = sum of dz over the block's rows, [... + C + c] = sum of dz * xhat
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(GT) void gn_bwd_reduce_kernel(Cover k, const T* __restrict__ x, const T* __restrict__ dy,
                                                           const T* __restrict__ res, const float* __restrict__ mean,
                                                           const float* __restrict__ rstd,
                                                           const float* __restrict__ gamma,
                                                           const float* __restrict__ beta, float* __restrict__ part) {
  __shared__ float sa[GT * V], sb[GT * V];
  const Slot<V> t(k);
  float A[V], B[V];
#pragma unroll
  for (int i = 0; i < V; ++i) A[i] = B[i] = 0.f;
  if (t.on) {
    const Chan<V> h(k, t.n, t.c, mean, rstd, gamma, beta);
    size_t o = ((size_t)t.n * k.S + t.r0 + t.ty) * k.C + t.c;
    const size_t step = (size_t)k.ry * k.C;
#pragma unroll 2
    for (int r = t.r0 + t.ty; r < t.r1; r += k.ry, o += step) {
      float v[V], d[V], e[V];
      loadv<T, V>(x + o, v);
      loadv<T, V>(dy + o, d);
      if (RES) loadv<T, V>(res + o, e);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xh = (v[i] - h.mu[i]) * h.rs[i];
        float z = fmaf(xh, h.ga[i], h.be[i]);
        if (RES) z += e[i];
        const float dz = d[i] * act_slope<ACT>(z);
        A[i] += dz;
        B[i] = fmaf(dz, xh, B[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    sa[threadIdx.x * V + i] = A[i];
    sb[threadIdx.x * V + i] = B[i];
  }
  int w = 1;
  while (w < k.ry) w <<= 1;
  for (w >>= 1; w > 0; w >>= 1) {
    __syncthreads();
    if (t.on && t.ty < w && t.ty + w < k.ry) {
      const int a = threadIdx.x, b = a + w * k.cvb;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sa[a * V + i] += sa[b * V + i];
        sb[a * V + i] += sb[b * V + i];
      }
    }
  }
  if (t.on && t.ty == 0) {
    float* o = part + ((size_t)t.n * k.chunks + blockIdx.x) * 2 * k.C + t.c;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o[i] = sa[threadIdx.x * V + i];
      o[k.C + i] = sb[threadIdx.x * V + i];
    }
  }
}

// One wave per (group, sample): ab[n][0 / 1][c] = A_c, B_c over all chunks, coef[n][g] = (c1, c2)
__global__ __launch_bounds__(64) void gn_bwd_join_kernel(Cover k, const float* __restrict__ part,
                                                         const float* __restrict__ gamma, float* __restrict__ ab,
                                                         float2* __restrict__ coef) {
  const int g = blockIdx.x, n = blockIdx.y;
  const float* p = part + (size_t)n * k.chunks * 2 * k.C;
  // a channel is summed by `fan` lanes, each taking every fan-th chunk
  int fan = 1;
  while (fan < 64 && fan * 2 * k.cpg <= 64) fan <<= 1;
  const int per = 64 / fan, f = threadIdx.x % fan;
  double t1 = 0.0, t2 = 0.0;
  for (int c0 = 0; c0 < k.cpg; c0 += per) {
    const int ci = c0 + (int)threadIdx.x / fan;
    double a = 0.0, b = 0.0;
    const int c = g * k.cpg + ci;
    if (ci < k.cpg)
      for (int ch = f; ch < k.chunks; ch += fan) {
        a += (double)p[(size_t)ch * 2 * k.C + c];
        b += (double)p[(size_t)ch * 2 * k.C + k.C + c];
      }
    for (int o = fan >> 1; o > 0; o >>= 1) {
      a += __shfl_xor(a, o, 64);
      b += __shfl_xor(b, o, 64);
    }
    if (ci < k.cpg && f == 0) {
      ab[(size_t)n * 2 * k.C + c] = (float)a;
      ab[(size_t)n * 2 * k.C + k.C + c] = (float)b;
      const double w = gamma ? (double)gamma[c] : 1.0;
      t1 += w * a;
      t2 += w * b;
    }
  }
  t1 = wave_sum_d(t1);
  t2 = wave_sum_d(t2);
  if (threadIdx.x == 0) {
    const double m = (double)k.S * k.cpg;
    coef[(size_t)n * k.G + g] = make_float2((float)(t1 / m), (float)(t2 / m));
  }
}

// dgamma[c] (+)= sum_n B_c, dbeta[c] (+)= sum_n A_c (added to where bit 0 / bit 1 of `add` is set): 64 channels x 4 runs of
// samples per block, runs joined in order, in doubles: a run is up to 16384 samples long
__global__ __launch_bounds__(GT) void gn_bwd_params_kernel(const float* __restrict__ ab, float* __restrict__ dgamma,
                                                           float* __restrict__ dbeta, int N, int C, int add) {
  __shared__ double sa[4][64], sb[4][64];
  const int e = threadIdx.x & 63, run = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + e;
  double a = 0.0, b = 0.0;
  if (c < C)
#pragma unroll 4
    for (int n = run; n < N; n += 4) {
      a += (double)ab[(size_t)n * 2 * C + c];
      b += (double)ab[(size_t)n * 2 * C + C + c];
    }
  sa[run][e] = a;
  sb[run][e] = b;
  __syncthreads();
  if (run == 0 && c < C) {
    if (dbeta) dbeta[c] = (add & 2 ? dbeta[c] : 0.f) + (float)((sa[0][e] + sa[1][e]) + (sa[2][e] + sa[3][e]));
    if (dgamma) dgamma[c] = (add & 1 ? dgamma[c] : 0.f) + (float)((sb[0][e] + sb[1][e]) + (sb[2][e] + sb[3][e]));
  }
}

// dx = rstd * (gamma * dz - c1 - xhat * c2), dres = dz.  With few samples (fold) the first workgroups of sample 0 also
// write the parameters' gradients, which saves the launch of gn_bwd_params_kernel.
struct Fold {
  const float* ab;
  float *dgamma, *dbeta;
  int N, add;
};
template <typename T, int V, int ACT, bool RES>
__global__ __launch_bounds__(GT) void gn_bwd_apply_kernel(Cover k, const T* __restrict__ x, const T* __restrict__ dy,
                                                          const T* __restrict__ res, const float* __restrict__ mean,
                                                          const float* __restrict__ rstd,
                                                          const float* __restrict__ gamma,
                                                          const float* __restrict__ beta,
                                                          const float2* __restrict__ coef, T* __restrict__ dx,
                                                          T* __restrict__ dres, Fold f) {
  const Slot<V> t(k);
  if (!t.on) return;
  if (f.N && t.n == 0 && blockIdx.x == 0 && t.ty == 0)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float a = 0.f, b = 0.f;
      for (int n = 0; n < f.N; ++n) {
        a += f.ab[(size_t)n * 2 * k.C + t.c + i];
        b += f.ab[(size_t)n * 2 * k.C + k.C + t.c + i];
      }
      if (f.dbeta) f.dbeta[t.c + i] = (f.add & 2 ? f.dbeta[t.c + i] : 0.f) + a;
      if (f.dgamma) f.dgamma[t.c + i] = (f.add & 1 ? f.dgamma[t.c + i] : 0.f) + b;
    }
  const Chan<V> h(k, t.n, t.c, mean, rstd, gamma, beta);
  float c1[V], c2[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 e = coef[(size_t)t.n * k.G + (t.c + i) / k.cpg];
    c1[i] = e.x;
    c2[i] = e.y;
  }
  size_t o = ((size_t)t.n * k.S + t.r0 + t.ty) * k.C + t.c;
  const size_t step = (size_t)k.ry * k.C;
#pragma unroll 2
  for (int r = t.r0 + t.ty; r < t.r1; r += k.ry, o += step) {
    float v[V], d[V], e[V];
    loadv<T, V>(x + o, v);
    loadv<T, V>(dy + o, d);
    if (RES) loadv<T, V>(res + o, e);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float xh = (v[i] - h.mu[i]) * h.rs[i];
      float z = fmaf(xh, h.ga[i], h.be[i]);
      if (RES) z += e[i];
      d[i] *= act_slope<ACT>(z);
      v[i] = h.rs[i] * (fmaf(h.ga[i], d[i], -c1[i]) - xh * c2[i]);
    }
    if (dx) storev<T, V>(dx + o, v);
    if (dres) storev<T, V>(dres + o, d);
  }
}

// `rows` is chosen so that a launch has the five blocks per CU that are resident at once where the data allows it, and so
// that a thread still sums a few rows: the partial statistics of a block are 8 bytes per channel
Cover make_cover(int N, int S, int C, int G, int V) {
  Cover k;
  k.S = S;
  k.C = C;
  k.G = G;
  k.cpg = C / G;
  k.cv = C / V;
  k.cvb = k.cv < GT ? k.cv : GT;
  k.ry = GT / k.cvb;
  const int64_t slabs = ceil_div(k.cv, k.cvb);
  const int64_t want = ceil_div64(5 * 256, (int64_t)N * slabs);  // chunks per sample
  int64_t rows = ceil_div64(S, want);
  const int64_t least = (int64_t)k.ry * 8;
  if (rows < least) rows = least;
  rows = ceil_div64(rows, k.ry) * k.ry;
  if (rows > S) rows = S;
  k.rows = (int)rows;
  k.chunks = (int)ceil_div64(S, rows);
  return k;
}

int vec_of(int C, std::initializer_list<const void*> ps) {
  if (C % 8) return 1;
  for (const void* p : ps)
    if (p && ((uintptr_t)p & 15)) return 1;
  return 8;
}

int check_gn(const char* who, int dtype, int64_t N, int64_t S, int64_t C, int64_t G, int act) {
  if (dtype != VC_F32 && dtype != VC_BF16) {
    vc_set_error("%s: unsupported dtype %d", who, dtype);
    return VC_ERR_DTYPE;
  }
  VC_CHECK_SHAPE(N > 0 && S > 0 && C > 0 && G > 0, "%s: empty shape N=%lld S=%lld C=%lld G=%lld", who, (long long)N,
                 (long long)S, (long long)C, (long long)G);
  VC_CHECK_SHAPE(C % G == 0, "%s: %lld channels do not split into %lld groups", who, (long long)C, (long long)G);
  // N is a grid's second extent, G its first; positions are 32-bit with room for a block's rows
  VC_CHECK_SHAPE(N <= 65535 && S <= (1 << 30) && C <= (1 << 20), "%s: N, S or C too large (at most 65535, 2^30, 2^20)", who);
  VC_CHECK_ARG(act >= ACT_NONE && act <= ACT_GELU, "%s: unknown activation %d", who, act);
  return VC_OK;
}

#define GN_ACT(act, ...)                                                 \
  do {                                                                   \
    if (act == ACT_RELU) { constexpr int ACT = ACT_RELU; __VA_ARGS__; }  \
    else if (act == ACT_SILU) { constexpr int ACT = ACT_SILU; __VA_ARGS__; } \
    else if (act == ACT_GELU) { constexpr int ACT = ACT_GELU; __VA_ARGS__; } \
    else { constexpr int ACT = ACT_NONE; __VA_ARGS__; }                  \
  } while (0)
#define GN_ACT_RES(act, res, ...)              \
  do {                                         \
    if (res) {                                 \
      constexpr bool RES = true;               \
      GN_ACT(act, __VA_ARGS__);                \
    } else {                                   \
      constexpr bool RES = false;              \
      GN_ACT(act, __VA_ARGS__);                \
    }                                          \
  } while (0)

template <typename T, int V>
int fwd_go(const Cover& k, int N, const void* x, const void* res, const float* gamma, const float* beta, void* y,
           float* mean, float* rstd, float* ws, float eps, int act, hipStream_t st) {
  const dim3 grid(k.chunks, N, ceil_div(k.cv, k.cvb));
  hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(GT), 0, st, k, (const T*)x, ws);
  hipLaunchKernelGGL(gn_join_kernel, dim3(k.G, N), dim3(64), 0, st, k, ws, mean, rstd, eps);
  GN_ACT_RES(act, res,
             hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, RES>), grid, dim3(GT), 0, st, k, (const T*)x, (const T*)res,
                                mean, rstd, gamma, beta, (T*)y));
  VC_LAUNCH_CHECK("vc_group_norm_fwd");
  return VC_OK;
}

template <typename T, int V>
int bwd_go(const Cover& k, int N, const void* x, const void* dy, const void* res, const float* gamma, const float* beta,
           const float* mean, const float* rstd, void* dx, void* dres, float* dgamma, float* dbeta, float* ws, int act,
           int add, hipStream_t st) {
  const dim3 grid(k.chunks, N, ceil_div(k.cv, k.cvb));
  float* ab = ws + (size_t)N * k.chunks * 2 * k.C;
  float2* coef = (float2*)(ab + (size_t)N * 2 * k.C);
  GN_ACT_RES(act, res,
             hipLaunchKernelGGL((gn_bwd_reduce_kernel<T, V, ACT, RES>), grid, dim3(GT), 0, st, k, (const T*)x,
                                (const T*)dy, (const T*)res, mean, rstd, gamma, beta, ws));
  hipLaunchKernelGGL(gn_bwd_join_kernel, dim3(k.G, N), dim3(64), 0, st, k, ws, gamma, ab, coef);
  const bool params = dgamma || dbeta, fold = params && (dx || dres) && N <= 8;
  if (params && !fold)
    hipLaunchKernelGGL(gn_bwd_params_kernel, dim3(ceil_div(k.C, 64)), dim3(GT), 0, st, ab, dgamma, dbeta, N, k.C, add);
  const Fold f{ab, dgamma, dbeta, fold ? N : 0, add};
  if (dx || dres)
    GN_ACT_RES(act, res,
               hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, ACT, RES>), grid, dim3(GT), 0, st, k, (const T*)x,
                                  (const T*)dy, (const T*)res, mean, rstd, gamma, beta, coef, (T*)dx, (T*)dres, f));
  VC_LAUNCH_CHECK("vc_group_norm_bwd");
  return VC_OK;
}

}  // namespace

extern "C" {

// floats of workspace of a forward or backward call, enough for either vector width
int64_t vc_group_norm_workspace_floats(int N, int S, int C, int G) {
  if (N <= 0 || S <= 0 || C <= 0 || G <= 0) return 0;
  int64_t most = 0;
  for (int v = 1; v <= 8; v += 7) {
    if (C % v) continue;
    const Cover k = make_cover(N, S, C, G, v);
    const int64_t f = (int64_t)N * ((int64_t)k.chunks * 2 * C + 2 * C + 2 * G);
    if (f > most) most = f;
  }
  return most;
}

int vc_group_norm_fwd(int dtype, const void* x, const void* residual, const float* gamma, const float* beta, void* y,
                      float* mean, float* rstd, float* workspace, int N, int S, int C, int G, float eps, int act,
                      hipStream_t stream) {
  const int rc = check_gn("vc_group_norm_fwd", dtype, N, S, C, G, act);
  if (rc != VC_OK) return rc;
  VC_CHECK_ARG(x && y && mean && rstd && workspace, "vc_group_norm_fwd: null pointer");
  const int V = vec_of(C, {x, residual, y});
  if (V == 8 && vc_gn_slab_fwd(dtype, x, residual, gamma, beta, y, mean, rstd, N, S, C, G, eps, act, stream)) {
    VC_LAUNCH_CHECK("vc_group_norm_fwd");
    return VC_OK;
  }
  const Cover k = make_cover(N, S, C, G, V);
  if (dtype == VC_BF16)
    return V == 8 ? fwd_go<bf16, 8>(k, N, x, residual, gamma, beta, y, mean, rstd, workspace, eps, act, stream)
                  : fwd_go<bf16, 1>(k, N, x, residual, gamma, beta, y, mean, rstd, workspace, eps, act, stream);
  return V == 8 ? fwd_go<float, 8>(k, N, x, residual, gamma, beta, y, mean, rstd, workspace, eps, act, stream)
                : fwd_go<float, 1>(k, N, x, residual, gamma, beta, y, mean, rstd, workspace, eps, act, stream);
}

int vc_group_norm_bwd(int dtype, const void* x, const void* dy, const void* residual, const float* gamma,
                      const float* beta, const float* mean, const float* rstd, void* dx, void* dresidual, float* dgamma,
                      float* dbeta, float* workspace, int N, int S, int C, int G, int act, int accumulate,
                      hipStream_t stream) {
  const int rc = check_gn("vc_group_norm_bwd", dtype, N, S, C, G, act);
  if (rc != VC_OK) return rc;
  VC_CHECK_ARG(x && dy && mean && rstd && workspace, "vc_group_norm_bwd: null pointer");
  VC_CHECK_ARG(((uintptr_t)workspace & 7) == 0, "vc_group_norm_bwd: workspace must be 8-byte aligned");
  const int V = vec_of(C, {x, dy, residual, dx, dresidual});
  if (V == 8 && vc_gn_slab_bwd(dtype, x, dy, residual, gamma, beta, mean, rstd, dx, dresidual, workspace, N, S, C, G, act,
                               stream)) {
    if (dgamma || dbeta)
      hipLaunchKernelGGL(gn_bwd_params_kernel, dim3(ceil_div(C, 64)), dim3(GT), 0, stream, workspace, dgamma, dbeta, N, C,
                         accumulate);
    VC_LAUNCH_CHECK("vc_group_norm_bwd");
    return VC_OK;
  }
  const Cover k = make_cover(N, S, C, G, V);
  if (dtype == VC_BF16)
    return V == 8 ? bwd_go<bf16, 8>(k, N, x, dy, residual, gamma, beta, mean, rstd, dx, dresidual, dgamma, dbeta, workspace, act, accumulate, stream)
                  : bwd_go<bf16, 1>(k, N, x, dy, residual, gamma, beta, mean, rstd, dx, dresidual, dgamma, dbeta, workspace, act, accumulate, stream);
  return V == 8 ? bwd_go<float, 8>(k, N, x, dy, residual, gamma, beta, mean, rstd, dx, dresidual, dgamma, dbeta, workspace, act, accumulate, stream)
                : bwd_go<float, 1>(k, N, x, dy, residual, gamma, beta, mean, rstd, dx, dresidual, dgamma, dbeta, workspace, act, accumulate, stream);
}

}  // extern "C"

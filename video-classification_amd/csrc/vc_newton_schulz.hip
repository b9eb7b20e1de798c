// Orthogonalisation of weight updates by Newton-Schulz products, many matrices per launch.
//
//   X_0 = G / (|G|_F + e);   S = X X^T,  X <- a X + (b S + c S S) X,  `steps` times;   with X the wide orientation of G
// (m <= n; a tall matrix is transposed on the way in and out).  The polynomial drives every singular value towards 1.
//
// 2 m^2 n + 2 m^3 + 2 m^2 n operations a step (S and S S are symmetric: only tiles on and below the diagonal are computed
// and stored twice), bound by the matrix pipes for large matrices and by launches for small ones, so all matrices of a
// call share three launches a step.
//
// Precision: a gradient's small singular values are amplified by a^steps (485 for the usual coefficients) and with them the
// rounding of X, so bf16 products leave errors of 1 % of the largest entry for random matrices and 50 % for matrices of
// low rank with a little noise (2e-3 and 6e-2 in single fp16 terms).  Everything is therefore held in two fp16 terms
// (vc_gemm16.h: 22 bits), which is as accurate as fp32 products at three MFMA each.
//
// Scales.  rho = |G| / (|G| + e), Y = X / rho: Y_0 = G / |G| has unit norm however small G is, and the products with rho^2 S
// follow X exactly.  With `cap` the largest value any iterate takes on [0, 1] and `gain` the largest ratio of an iterate
// to its start, |Y| <= min(cap / rho, gain), which fixes the power of two that scales Y into fp16; S and the polynomial
// of S are scaled by powers of two from cap alone.
#include "vc_gemm16.h"

namespace {

constexpr int NS_MAX = 64;        // matrices per launch
constexpr int NORM_CHUNK = 1 << 14;

// One matrix of a launch, in its wide orientation (m <= n).
struct NsMat {
  const void* g;
  void* out;
  int64_t at;  // its buffers in the workspace, in fp16 elements
  int m, n;
  int tall;    // G is [n][m]
  int t0;      // first workgroup of this matrix in the launch
};
struct NsArgs {
  NsMat mat[NS_MAX];
  int count;
};

// m <- mu m + f g;  u = f g + mu m (nesterov) or m
__global__ __launch_bounds__(256) void muon_momentum_kernel(const float* __restrict__ g, float* __restrict__ m,
                                                            float* __restrict__ u, int64_t n, float mu, int nesterov,
                                                            float f) {
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    const f32x4 gv = *reinterpret_cast<const f32x4*>(g + i);
    f32x4 mv = *reinterpret_cast<const f32x4*>(m + i), uv;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float e = gv[k] * f;
      mv[k] = fmaf(mu, mv[k], e);
      uv[k] = nesterov ? fmaf(mu, mv[k], e) : mv[k];
    }
    *reinterpret_cast<f32x4*>(m + i) = mv;
    *reinterpret_cast<f32x4*>(u + i) = uv;
  }
}

// p <- (1 - lr wd) p - lr scale u, one scale per 64 elements (parameters start on 64-element boundaries)
__global__ __launch_bounds__(256) void muon_apply_kernel(float* __restrict__ p, const float* __restrict__ u,
                                                         const float* __restrict__ scale, int64_t n,
                                                         const float* __restrict__ lr_dev, float wd) {
  const float lr = *lr_dev, keep = 1.f - lr * wd;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    f32x4 pv = *reinterpret_cast<const f32x4*>(p + i);
    const f32x4 uv = *reinterpret_cast<const f32x4*>(u + i);
    const float s = lr * scale[i >> 6];
#pragma unroll
    for (int k = 0; k < 4; ++k) pv[k] = fmaf(keep, pv[k], -s * uv[k]);
    *reinterpret_cast<f32x4*>(p + i) = pv;
  }
}

__host__ __device__ inline int up64(int v) { return (v + 63) / 64 * 64; }
__host__ __device__ inline int64_t up128(int64_t v) { return (v + 127) / 128 * 128; }

// Buffers of one matrix, two planes each: X [m][ldn] and X^T [n][ldm] twice (read and written in turn), S and P [m][ldm].
struct NsView {
  int ldm, ldn;
  int64_t x, xt, xo, xto, s, p, end;
  __host__ __device__ NsView(const NsMat& t, int parity) {
    ldm = up64(t.m);
    ldn = up64(t.n);
    const int64_t ex = up128(2ll * t.m * ldn), et = up128(2ll * t.n * ldm), es = up128(2ll * t.m * ldm);
    const int64_t half = ex + et;
    x = t.at + (parity ? half : 0);
    xo = t.at + (parity ? 0 : half);
    xt = x + ex;
    xto = xo + ex;
    s = t.at + 2 * half;
    p = s + es;
    end = p + es;
  }
};

// what the kernels read per matrix, written by ns_scale_kernel
struct NsScale {
  double inv;  // 2^ey / |G| (0 for a zero matrix)
  float rho, rho2;
  int ey, pad;
};

__device__ __forceinline__ int find_mat(const NsArgs& a, int block) {
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.mat[mid].t0 <= block) lo = mid;
    else hi = mid - 1;
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// sum of squares of NORM_CHUNK elements, in double: no overflow, no underflow
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs a, double* __restrict__ part) {
  __shared__ double sm[4];
  const int i = find_mat(a, blockIdx.x);
  const NsMat& t = a.mat[i];
  const int64_t total = (int64_t)t.m * t.n, e0 = (int64_t)(blockIdx.x - t.t0) * NORM_CHUNK;
  const int64_t e1 = e0 + NORM_CHUNK < total ? e0 + NORM_CHUNK : total;
  const T* g = (const T*)t.g;
  double s = 0.0;
  if (((uintptr_t)g & 15) == 0) {
    for (int64_t e = e0 + threadIdx.x * 8; e < e1; e += 2048) {
      if (e + 8 <= e1) {
        const F8 v = load8(g + e);
#pragma unroll
        for (int k = 0; k < 8; ++k) s += (double)v.v[k] * (double)v.v[k];
      } else
        for (int64_t k = e; k < e1; ++k) s += (double)to_f32(g[k]) * (double)to_f32(g[k]);
    }
  } else
    for (int64_t e = e0 + threadIdx.x; e < e1; e += 256) s += (double)to_f32(g[e]) * (double)to_f32(g[e]);
  s = wave_sum_f64(s);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// one wave per matrix
__global__ __launch_bounds__(64) void ns_scale_kernel(NsArgs a, int blocks, const double* __restrict__ part, double eps,
                                                      float cap, float gain, NsScale* __restrict__ sc) {
  const int i = blockIdx.x;
  const int b0 = a.mat[i].t0, b1 = i + 1 < a.count ? a.mat[i + 1].t0 : blocks;
  double s = 0.0;
  for (int b = b0 + threadIdx.x; b < b1; b += 64) s += part[b];
  s = wave_sum_f64(s);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s), rho = norm / (norm + eps);
    const double bound = rho > 0.0 && (double)cap / rho < (double)gain ? (double)cap / rho : (double)gain;
    NsScale o;
    o.ey = (int)floor(log2(60000.0 / bound));
    o.inv = norm > 0.0 ? ldexp(1.0 / norm, o.ey) : (norm == 0.0 ? 0.0 : norm);  // NaN stays NaN
    o.rho = norm > 0.0 ? (float)rho : (norm == 0.0 ? 0.f : (float)norm);
    o.rho2 = o.rho * o.rho;
    o.pad = 0;
    sc[i] = o;
  }
}

// Y_0 in both orders: 64 x 64 tiles of the wide orientation through LDS, zeros in the padding
template <typename T>
__global__ __launch_bounds__(256) void ns_init_kernel(NsArgs a, f16* __restrict__ ws, const NsScale* __restrict__ sc) {
  __shared__ float sm[64][65];
  const int i = find_mat(a, blockIdx.x);
  const NsMat& t = a.mat[i];
  const NsView w(t, 0);
  const int id = blockIdx.x - t.t0, tn = w.ldn / 64;
  const int r0 = id / tn * 64, c0 = id % tn * 64;  // rows < m, columns < n of X
  const double inv = sc[i].inv;
  const T* g = (const T*)t.g;
  for (int e = threadIdx.x; e < 4096; e += 256) {
    const int hi = e >> 6, lo = e & 63;  // lo runs along G's rows
    const int r = t.tall ? r0 + lo : r0 + hi, c = t.tall ? c0 + hi : c0 + lo;
    float v = 0.f;
    if (r < t.m && c < t.n) v = (float)((double)to_f32(t.tall ? g[(int64_t)c * t.m + r] : g[(int64_t)r * t.n + c]) * inv);
    sm[r - r0][c - c0] = v;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 512; e += 256) {
    const int hi = e >> 3, lo = (e & 7) * 8;
    f16x8 h, l;
    if (r0 + hi < t.m) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f16 u, v;
        f16_split(sm[hi][lo + k], u, v);
        h[k] = u;
        l[k] = v;
      }
      f16* d = ws + w.x + (int64_t)(r0 + hi) * w.ldn + c0 + lo;
      *reinterpret_cast<f16x8*>(d) = h;
      *reinterpret_cast<f16x8*>(d + (int64_t)t.m * w.ldn) = l;
    }
    if (c0 + hi < t.n) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f16 u, v;
        f16_split(sm[lo + k][hi], u, v);
        h[k] = u;
        l[k] = v;
      }
      f16* d = ws + w.xt + (int64_t)(c0 + hi) * w.ldm + r0 + lo;
      *reinterpret_cast<f16x8*>(d) = h;
      *reinterpret_cast<f16x8*>(d + (int64_t)t.n * w.ldm) = l;
    }
  }
}

struct NsStep {
  float a, b, c;
  int es, ep;  // scale exponents of S and of P = b S + c S^2
  int last;
};

// The symmetric products.  SQUARE false: S = rho^2 Y Y^T; true: P = b S + c S S.  Tiles on and below the diagonal; the mirror
// of an off-diagonal tile is stored with it.
template <bool SQUARE>
__global__ __launch_bounds__(G_THREADS, 2) void ns_sym_kernel(NsArgs a, f16* __restrict__ ws,
                                                              const NsScale* __restrict__ sc, NsStep st, int parity) {
  typedef G16<2, 2> G;
  __shared__ __attribute__((aligned(1024))) f16 smem[G::LDS];
  const int i = find_mat(a, blockIdx.x);
  const NsMat& t = a.mat[i];
  const NsView w(t, parity);
  const int id = blockIdx.x - t.t0;
  int tm = (int)((sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);  // id = tm (tm + 1) / 2 + tn, tn <= tm
  while ((tm + 1) * (tm + 2) / 2 <= id) ++tm;
  while (tm * (tm + 1) / 2 > id) --tm;
  tm = __builtin_amdgcn_readfirstlane(tm);
  const int tn = id - tm * (tm + 1) / 2;
  const int m0 = tm * GM, n0 = tn * GM;
  const f16* src = ws + (SQUARE ? w.s : w.x);
  const int ld = SQUARE ? w.ldm : w.ldn;
  const int64_t plane = (int64_t)t.m * ld;
  f32x4 acc[4][4];
  G::zero(acc);
  G::run(acc, src + (int64_t)m0 * ld, plane, ld, t.m - m0, src + (int64_t)n0 * ld, plane, ld, t.m - n0, 0, ld, smem);
  const int lane = threadIdx.x & 63, q = lane >> 4, l15 = lane & 15;
  const int wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  const f16* s = ws + w.s;
  f16* dst = ws + (SQUARE ? w.p : w.s);
  const int64_t pl = (int64_t)t.m * w.ldm;
  const float rho2 = sc[i].rho2;
  const int e = SQUARE ? st.ep - 2 * st.es : st.es - 2 * sc[i].ey;
  const float sb = ldexpf(st.b, st.ep - st.es);
#pragma unroll
  for (int ii = 0; ii < 4; ++ii)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = m0 + wm * 64 + ii * 16 + q * 4, c = n0 + wn * 64 + j * 16 + l15;
      f16x4 hi, lo;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v;
        if (SQUARE) {
          v = st.c * ldexpf(acc[ii][j][k], e);
          if (r + k < t.m && c < t.m) {
            const int64_t o = (int64_t)(r + k) * w.ldm + c;
            v = fmaf(sb, (float)s[o] + (float)s[o + pl], v);
          }
        } else
          v = rho2 * ldexpf(acc[ii][j][k], e);
        f16 h, l;
        f16_split(v, h, l);
        hi[k] = h;
        lo[k] = l;
        if (r + k < t.m && c < w.ldm) {
          const int64_t o = (int64_t)(r + k) * w.ldm + c;
          dst[o] = h;
          dst[o + pl] = l;
        }
      }
      if (tm != tn && c < t.m && r < w.ldm) {
        const int64_t o = (int64_t)c * w.ldm + r;
        *reinterpret_cast<f16x4*>(dst + o) = hi;
        *reinterpret_cast<f16x4*>(dst + o + pl) = lo;
      }
    }
}

// X <- a X + P X, into the other pair of buffers, or the result in G's orientation after the last step
template <typename T>
__global__ __launch_bounds__(G_THREADS, 2) void ns_update_kernel(NsArgs a, f16* __restrict__ ws,
                                                                 const NsScale* __restrict__ sc, NsStep st, int parity) {
  typedef G16<2, 2> G;
  __shared__ __attribute__((aligned(1024))) f16 smem[G::LDS];
  const int i = find_mat(a, blockIdx.x);
  const NsMat& t = a.mat[i];
  const NsView w(t, parity);
  const int tiles_m = (t.m + GM - 1) / GM;
  const int id = blockIdx.x - t.t0;
  const int tn = id / tiles_m, tm = id - tn * tiles_m;
  const int m0 = tm * GM, n0 = tn * GM;
  const int64_t pp = (int64_t)t.m * w.ldm, px = (int64_t)t.m * w.ldn, pt = (int64_t)t.n * w.ldm;
  const f16 *x = ws + w.x, *xt = ws + w.xt;
  f32x4 acc[4][4];
  G::zero(acc);
  G::run(acc, ws + w.p + (int64_t)m0 * w.ldm, pp, w.ldm, t.m - m0, xt + (int64_t)n0 * w.ldm, pt, w.ldm, t.n - n0, 0, w.ldm,
         smem);
  const int lane = threadIdx.x & 63, q = lane >> 4, l15 = lane & 15;
  const int wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  f16 *xo = ws + w.xo, *xto = ws + w.xto;
  const float rho = sc[i].rho;
  const int ey = sc[i].ey;
#pragma unroll
  for (int ii = 0; ii < 4; ++ii)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = m0 + wm * 64 + ii * 16 + q * 4, c = n0 + wn * 64 + j * 16 + l15;
      f16x4 hi, lo;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float v = ldexpf(acc[ii][j][k], -st.ep);
        const int64_t o = (int64_t)(r + k) * w.ldn + c;
        if (r + k < t.m && c < t.n) v = fmaf(st.a, (float)x[o] + (float)x[o + px], v);
        if (st.last) {
          if (r + k < t.m && c < t.n)
            ((T*)t.out)[t.tall ? (int64_t)c * t.m + r + k : (int64_t)(r + k) * t.n + c] = from_f32<T>(rho * ldexpf(v, -ey));
          continue;
        }
        f16 h, l;
        f16_split(v, h, l);
        hi[k] = h;
        lo[k] = l;
        if (r + k < t.m && c < w.ldn) {
          xo[o] = h;
          xo[o + px] = l;
        }
      }
      if (!st.last && c < t.n && r < w.ldm) {
        const int64_t o = (int64_t)c * w.ldm + r;
        *reinterpret_cast<f16x4*>(xto + o) = hi;
        *reinterpret_cast<f16x4*>(xto + o + pt) = lo;
      }
    }
}

// steps = 0: the normalised matrix itself
template <typename T>
__global__ __launch_bounds__(256) void ns_copy_kernel(NsArgs a, const NsScale* __restrict__ sc) {
  const int i = find_mat(a, blockIdx.x);
  const NsMat& t = a.mat[i];
  const int64_t total = (int64_t)t.m * t.n, e0 = (int64_t)(blockIdx.x - t.t0) * NORM_CHUNK;
  const int64_t e1 = e0 + NORM_CHUNK < total ? e0 + NORM_CHUNK : total;
  const double f = ldexp(sc[i].inv, -sc[i].ey) * (double)sc[i].rho;
  for (int64_t e = e0 + threadIdx.x; e < e1; e += 256)
    ((T*)t.out)[e] = from_f32<T>((float)((double)to_f32(((const T*)t.g)[e]) * f));
}

int64_t norm_blocks(int64_t m, int64_t n) { return ceil_div64(m * n, NORM_CHUNK); }

int check_ns(const char* who, int dtype, int count, const int* rows, const int* cols) {
  if (dtype != VC_F32 && dtype != VC_BF16) {
    vc_set_error("%s: unsupported dtype %d", who, dtype);
    return VC_ERR_DTYPE;
  }
  VC_CHECK_ARG(count > 0 && rows && cols, "%s: no matrices", who);
  for (int i = 0; i < count; ++i)
    // 128 rows have to fit a 32-bit buffer descriptor
    VC_CHECK_SHAPE(rows[i] > 0 && cols[i] > 0 && rows[i] <= (1 << 20) && cols[i] <= (1 << 20) &&
                       (int64_t)rows[i] * cols[i] <= (1ll << 31),
                   "%s: matrix %d of %d x %d (sides from 1 to 2^20, at most 2^31 elements)", who, i, rows[i], cols[i]);
  return VC_OK;
}

}  // namespace

extern "C" {

int64_t vc_newton_schulz_bytes(int count, const int* rows, const int* cols) {
  if (check_ns("vc_newton_schulz_bytes", VC_F32, count, rows, cols) != VC_OK) return -1;
  int64_t most = 0;
  for (int b = 0; b < count; b += NS_MAX) {
    int64_t elems = 0, blocks = 0;
    for (int i = b; i < count && i < b + NS_MAX; ++i) {
      const int m = rows[i] < cols[i] ? rows[i] : cols[i], n = rows[i] < cols[i] ? cols[i] : rows[i];
      NsMat t{};
      t.m = m;
      t.n = n;
      elems += NsView(t, 0).end;
      blocks += norm_blocks(m, n);
    }
    const int64_t bytes = NS_MAX * (int64_t)sizeof(NsScale) + up128(blocks * 8) + elems * 2;
    if (bytes > most) most = bytes;
  }
  return most;
}

int vc_newton_schulz(int dtype, int count, const void* const* g, void* const* out, const int* rows, const int* cols,
                     int steps, const float* coeffs, double eps, float cap, float gain, float pmax, void* workspace,
                     hipStream_t stream) {
  const int rc = check_ns("vc_newton_schulz", dtype, count, rows, cols);
  if (rc != VC_OK) return rc;
  VC_CHECK_ARG(g && out && workspace && (coeffs || !steps), "vc_newton_schulz: null pointer");
  VC_CHECK_ARG(((uintptr_t)workspace & 255) == 0, "vc_newton_schulz: workspace must be 256-byte aligned");
  VC_CHECK_ARG(steps >= 0 && steps <= 64 && eps >= 0.0, "vc_newton_schulz: steps %d outside [0, 64] or eps %g negative", steps, eps);
  VC_CHECK_ARG(cap >= 1.f && cap <= 16.f && gain >= 1.f && gain <= 8192.f && pmax > 0.f && pmax <= 8192.f,
               "vc_newton_schulz: bounds cap %g, gain %g, pmax %g outside [1, 16], [1, 8192], (0, 8192]", (double)cap,
               (double)gain, (double)pmax);
  for (int i = 0; i < count; ++i) VC_CHECK_ARG(g[i] && out[i], "vc_newton_schulz: null matrix %d", i);
  NsScale* sc = (NsScale*)workspace;
  double* part = (double*)((char*)workspace + NS_MAX * sizeof(NsScale));
  NsStep st;
  st.es = (int)floorf(log2f(60000.f / (cap * cap)));
  st.ep = (int)floorf(log2f(60000.f / pmax));
  for (int b = 0; b < count; b += NS_MAX) {
    NsArgs a;
    a.count = count - b < NS_MAX ? count - b : NS_MAX;
    int64_t blocks = 0, t_init = 0, t_sym = 0, t_upd = 0;
    for (int i = 0; i < a.count; ++i) blocks += norm_blocks(rows[b + i], cols[b + i]);
    int64_t at = 0;
    int tn[NS_MAX], ti[NS_MAX], ts[NS_MAX], tu[NS_MAX];
    f16* ws = (f16*)((char*)part + up128(blocks * 8));
    blocks = 0;
    for (int i = 0; i < a.count; ++i) {
      NsMat& t = a.mat[i];
      const int r = rows[b + i], c = cols[b + i];
      t.g = g[b + i];
      t.out = out[b + i];
      t.tall = r > c;
      t.m = t.tall ? c : r;
      t.n = t.tall ? r : c;
      t.at = at;
      at = NsView(t, 0).end;
      tn[i] = (int)blocks;
      ti[i] = (int)t_init;
      ts[i] = (int)t_sym;
      tu[i] = (int)t_upd;
      blocks += norm_blocks(t.m, t.n);
      t_init += (int64_t)(up64(t.m) / 64) * (up64(t.n) / 64);
      const int64_t tm = ceil_div(t.m, GM), tnn = ceil_div(t.n, GM);
      t_sym += tm * (tm + 1) / 2;
      t_upd += tm * tnn;
    }
    VC_CHECK_SHAPE(blocks < (1ll << 31) && t_init < (1ll << 31) && t_sym < (1ll << 31) && t_upd < (1ll << 31),
                   "vc_newton_schulz: too many tiles");
    auto with = [&](const int* first) {
      for (int i = 0; i < a.count; ++i) a.mat[i].t0 = first[i];
    };
    const bool bf = dtype == VC_BF16;
    with(tn);
    if (bf) hipLaunchKernelGGL((ns_norm_kernel<bf16>), dim3((unsigned)blocks), dim3(256), 0, stream, a, part);
    else hipLaunchKernelGGL((ns_norm_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, stream, a, part);
    hipLaunchKernelGGL(ns_scale_kernel, dim3(a.count), dim3(64), 0, stream, a, (int)blocks, part, eps, cap, gain, sc);
    if (steps == 0) {
      if (bf) hipLaunchKernelGGL((ns_copy_kernel<bf16>), dim3((unsigned)blocks), dim3(256), 0, stream, a, sc);
      else hipLaunchKernelGGL((ns_copy_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, stream, a, sc);
    }
    with(ti);
    if (steps) {
      if (bf) hipLaunchKernelGGL((ns_init_kernel<bf16>), dim3((unsigned)t_init), dim3(256), 0, stream, a, ws, sc);
      else hipLaunchKernelGGL((ns_init_kernel<float>), dim3((unsigned)t_init), dim3(256), 0, stream, a, ws, sc);
    }
    for (int k = 0; k < steps; ++k) {
      st.a = coeffs[3 * k];
      st.b = coeffs[3 * k + 1];
      st.c = coeffs[3 * k + 2];
      st.last = k == steps - 1;
      with(ts);
      hipLaunchKernelGGL((ns_sym_kernel<false>), dim3((unsigned)t_sym), dim3(G_THREADS), 0, stream, a, ws, sc, st, k & 1);
      hipLaunchKernelGGL((ns_sym_kernel<true>), dim3((unsigned)t_sym), dim3(G_THREADS), 0, stream, a, ws, sc, st, k & 1);
      with(tu);
      if (bf)
        hipLaunchKernelGGL((ns_update_kernel<bf16>), dim3((unsigned)t_upd), dim3(G_THREADS), 0, stream, a, ws, sc, st, k & 1);
      else
        hipLaunchKernelGGL((ns_update_kernel<float>), dim3((unsigned)t_upd), dim3(G_THREADS), 0, stream, a, ws, sc, st, k & 1);
    }
    VC_LAUNCH_CHECK("vc_newton_schulz");
  }
  return VC_OK;
}

int vc_muon_momentum(const float* g, float* m, float* u, int64_t n, float mu, int nesterov, float grad_scale,
                     hipStream_t stream) {
  VC_CHECK_ARG(g && m && u, "vc_muon_momentum: null pointer");
  VC_CHECK_SHAPE(n > 0 && n % 64 == 0, "vc_muon_momentum: n = %lld is not a positive multiple of 64", (long long)n);
  VC_CHECK_ARG((((uintptr_t)g | (uintptr_t)m | (uintptr_t)u) & 15) == 0, "vc_muon_momentum: buffers must be 16-byte aligned");
  const int64_t b = ceil_div64(n, 1024);
  hipLaunchKernelGGL(muon_momentum_kernel, dim3((unsigned)(b < 4096 ? b : 4096)), dim3(256), 0, stream, g, m, u, n, mu,
                     nesterov, grad_scale);
  VC_LAUNCH_CHECK("vc_muon_momentum");
  return VC_OK;
}

int vc_muon_apply(float* p, const float* u, const float* scale, int64_t n, const float* lr_dev, float wd,
                  hipStream_t stream) {
  VC_CHECK_ARG(p && u && scale && lr_dev, "vc_muon_apply: null pointer");
  VC_CHECK_SHAPE(n > 0 && n % 64 == 0, "vc_muon_apply: n = %lld is not a positive multiple of 64", (long long)n);
  VC_CHECK_ARG((((uintptr_t)p | (uintptr_t)u) & 15) == 0, "vc_muon_apply: buffers must be 16-byte aligned");
  const int64_t b = ceil_div64(n, 1024);
  hipLaunchKernelGGL(muon_apply_kernel, dim3((unsigned)(b < 4096 ? b : 4096)), dim3(256), 0, stream, p, u, scale, n, lr_dev,
                     wd);
  VC_LAUNCH_CHECK("vc_muon_apply");
  return VC_OK;
}

}  // extern "C"

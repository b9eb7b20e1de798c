// Orthogonalisation of weight updates by Newton-Schulz products, many matrices per launch.
//
//   X_0 = G / (|G|_F + e);   S = X X^T,  X <- a X + (b S + c S S) X,  `steps` times;   with X the wide orientation of G
// (m <= n; a tall matrix is transposed on the way in and out).  The polynomial drives every singular value towards 1.
//
// m^2 n + m^3 + 2 m^2 n operations a step (S and S S are symmetric: only tiles on and below the diagonal are computed
// and stored twice), bound by the matrix pipes for large matrices and by the chain of launches for small ones, so all
// matrices of a call share each launch, three a step and a join where a reduction is cut.
//   4096 x 4096: S 210 + 9 us, P 212 + 10, update 389 (1.06 PFLOP/s of fp16 products); 5 steps 3.9 ms
//   52 matrices of a ResNet-50 (64 to 2048 rows): 190 us a step, 0.97 ms in all
//   4 matrices of up to 256 x 1152, on 64 x 64 tiles: 23 us a step -- six microseconds a launch, most of them latency
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
#include <type_traits>

#include "vc_gemm16.h"

namespace {

constexpr int NS_MAX = 64;        // matrices per launch
constexpr int NORM_CHUNK = 1 << 14;
// Launches with up to this many products (m^2 n for S, m^3 for P, 2 m^2 n for the update) work on 64 x 64 tiles, which are four
// times as many and a quarter as long, the others on 128 x 128, which load half as much per product.  64 against 128, us,
// joins included: S of 1024^2 (1.1 G) 13 / 17, 512 x 4608 (1.2 G) 17 / 23, 1536^2 (3.6 G) 30 / 26, 1024 x 4096 (4.3 G) 36 /
// 29; P of 1024 rows (1.1 G) 14 / 19, the ResNet-50 set (2.8 G) 25 / 31, 1536^2 30 / 27; updates of 1024^2 (2.1 G) 15 / 30,
// 512 x 4608 (2.4 G) 20 / 20, 1536^2 (7.2 G) 46 / 44, 1024 x 4096 (8.6 G) 44 / 37.
constexpr double NS_SMALL_SYM = 3e9, NS_SMALL_UPDATE = 5e9;

// What a launch numbers its workgroups by, matrix after matrix.
enum { BY_NORM, BY_INIT, BY_UPDATE, BY_S, BY_P, BY_JOIN_S, BY_JOIN_P, KINDS };

// One matrix of a call, in its wide orientation (m <= n).  The table of them lies in the workspace: read from the kernel
// arguments, which live in host memory, its lookups cost every workgroup microseconds.
struct NsMat {
  const void* g;
  void* out;
  int64_t at;        // its buffers in the workspace, in fp16 elements
  int m, n;
  int tall;          // G is [n][m]
  int first[KINDS];  // first workgroup of this matrix
  // symmetric products S and P: tiles [0, direct) are worked by one workgroup each, the others in `slices` runs of the
  // reduction whose partial tiles start at p0 and are joined by a second launch
  struct Cut {
    int direct, slices, p0;
  } cut[2];
};
constexpr int NS_CHUNK = 32;  // table entries that fit a launch's arguments
struct NsChunk {
  NsMat mat[NS_CHUNK];
};
__global__ __launch_bounds__(64) void ns_table_kernel(NsChunk c, NsMat* __restrict__ table, int count) {
  if ((int)threadIdx.x < count) table[threadIdx.x] = c.mat[threadIdx.x];
}

// the matrix a workgroup belongs to: every lane looks at one entry
__device__ __forceinline__ int find_mat(const NsMat* __restrict__ table, int count, int kind, int block) {
  const int lane = threadIdx.x & 63;
  const int f = lane < count ? table[lane].first[kind] : 0x7fffffff;
  return __builtin_amdgcn_readfirstlane(63 - __builtin_clzll(__ballot(f <= block)));
}

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

// Buffers of one matrix, two planes each: X [m][ldn] twice (read and written in turn), S and P [m][ldm].
struct NsView {
  int ldm, ldn;
  int64_t x, xo, s, p, end;
  __host__ __device__ NsView(const NsMat& t, int parity) {
    ldm = up64(t.m);
    ldn = up64(t.n);
    const int64_t ex = up128(2ll * t.m * ldn), es = up128(2ll * t.m * ldm);
    x = t.at + (parity ? ex : 0);
    xo = t.at + (parity ? 0 : ex);
    s = t.at + 2 * ex;
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

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// sum of squares of NORM_CHUNK elements, in double: no overflow, no underflow
template <typename T>
__global__ __launch_bounds__(256) void ns_norm_kernel(const NsMat* __restrict__ table, int count,
                                                    double* __restrict__ part) {
  __shared__ double sm[4];
  const int i = find_mat(table, count, BY_NORM, blockIdx.x);
  const NsMat t = table[i];
  const int64_t total = (int64_t)t.m * t.n, e0 = (int64_t)(blockIdx.x - t.first[BY_NORM]) * NORM_CHUNK;
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
__global__ __launch_bounds__(64) void ns_scale_kernel(const NsMat* __restrict__ table, int count, int blocks,
                                                     const double* __restrict__ part, double eps, float cap, float gain,
                                                     NsScale* __restrict__ sc) {
  const int i = blockIdx.x;
  const int b0 = table[i].first[BY_NORM], b1 = i + 1 < count ? table[i + 1].first[BY_NORM] : blocks;
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

// Y_0: 64 x 64 tiles of the wide orientation, through LDS where G is tall; zeros in the padding
template <typename T>
__global__ __launch_bounds__(256) void ns_init_kernel(const NsMat* __restrict__ table, int count, f16* __restrict__ ws,
                                                    const NsScale* __restrict__ sc) {
  __shared__ float sm[64][65];
  const int i = find_mat(table, count, BY_INIT, blockIdx.x);
  const NsMat t = table[i];
  const NsView w(t, 0);
  const int id = blockIdx.x - t.first[BY_INIT], tn = w.ldn / 64;
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
    if (r0 + hi >= t.m) continue;
    f16x8 h, l;
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
}

struct NsStep {
  float a, b, c;
  int es, ep;  // scale exponents of S and of P = b S + c S^2
  int last;
};

// Tile `id` of the lower triangle of tm x tm tiles, in bands of eight tile rows walked column by column.
__device__ __forceinline__ void tri_tile(int id, int tiles, int& m, int& n) {
  int b = 0;
  while (32 * (b + 1) * (b + 1) + 4 * (b + 1) <= id) ++b;  // 64 b + 36 tiles in a whole band b
  int w = id - (32 * b * b + 4 * b);
  const int rows = tiles - 8 * b < 8 ? tiles - 8 * b : 8;
  if (w < rows * 8 * b) {
    n = w / rows;
    m = 8 * b + w % rows;
  } else {
    w -= rows * 8 * b;
    int j = 0;
    while (w >= rows - j) {
      w -= rows - j;
      ++j;
    }
    n = 8 * b + j;
    m = n + w;
  }
  m = __builtin_amdgcn_readfirstlane(m);
  n = __builtin_amdgcn_readfirstlane(n);
}
// workgroups of one XCD (every eighth) take a contiguous run of [0, total)
__device__ __forceinline__ int xcd_run(int id, int total) {
  const int q = total >> 3, r = total & 7, xcd = id & 7, idx = id >> 3;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
}

// What becomes of an accumulated tile (rows m0 + .. in registers, columns n0 + .. across lanes) of a symmetric product:
// S = rho^2 Y Y^T, or P = b S + c S S (SQUARE).  It is stored at (column, row) and, off the diagonal, at (row, column), both
// in whole 16-byte pieces.
template <bool SQUARE, int TB>
__device__ __forceinline__ void sym_store(const f32x4 (&acc)[TB][TB], const NsMat& t, const NsView& w, f16* ws,
                                          const NsScale& sc, const NsStep& st, int m0, int n0, float* tile) {
  const f16* s = ws + w.s;
  f16* dst = ws + (SQUARE ? w.p : w.s);
  const int64_t pl = (int64_t)t.m * w.ldm;
  const float f = SQUARE ? ldexpf(st.c, st.ep - 2 * st.es) : ldexpf(sc.rho2, st.es - 2 * sc.ey);
  const float sb = ldexpf(st.b, st.ep - st.es);
  const bool mirror = m0 != n0;
  typedef Tile16<TB> L;
#pragma unroll
  for (int half = 0; half < L::HALVES; ++half) {
    const int c0 = n0 + half * 64;
    f16x8 sh[L::UNITS], sl[L::UNITS];  // S where it is needed, on its way while the tile passes through LDS
    if (SQUARE)
#pragma unroll
      for (int u = 0; u < L::UNITS; ++u) {
        const int e = threadIdx.x + u * G_THREADS;
        const int64_t o = (int64_t)min(c0 + e / L::VPR, t.m - 1) * w.ldm + min(m0 + e % L::VPR * 8, w.ldm - 8);
        sh[u] = *reinterpret_cast<const f16x8*>(s + o);
        sl[u] = *reinterpret_cast<const f16x8*>(s + o + pl);
      }
    L::put(acc, half, tile);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < L::UNITS; ++u) {
      const int e = threadIdx.x + u * G_THREADS, cl = e / L::VPR, rl = e % L::VPR * 8;
      F8 v = L::get(tile, cl, rl);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v.v[k] *= f;
        if (SQUARE) v.v[k] = fmaf(sb, (float)sh[u][k] + (float)sl[u][k], v.v[k]);
      }
      if (mirror) L::set(tile, cl, rl, v);
      if (c0 + cl < t.m && m0 + rl < w.ldm) {
        f16x8 h, l;
        f16_split8(v, h, l);
        f16* d = dst + (int64_t)(c0 + cl) * w.ldm + m0 + rl;
        *reinterpret_cast<f16x8*>(d) = h;
        *reinterpret_cast<f16x8*>(d + pl) = l;
      }
    }
    __syncthreads();
    if (mirror) {
#pragma unroll
      for (int u = 0; u < L::UNITS; ++u) {
        const int e = threadIdx.x + u * G_THREADS, rl = e >> 3, cl = (e & 7) * 8;
        F8 v;
#pragma unroll
        for (int k = 0; k < 8; ++k) v.v[k] = tile[L::at(cl + k, rl)];
        if (m0 + rl < t.m) {  // below the diagonal every column of the tile is inside
          f16x8 h, l;
          f16_split8(v, h, l);
          f16* d = dst + (int64_t)(m0 + rl) * w.ldm + c0 + cl;
          *reinterpret_cast<f16x8*>(d) = h;
          *reinterpret_cast<f16x8*>(d + pl) = l;
        }
      }
      __syncthreads();
    }
  }
}

// A tile, or a slice of the reduction of one, of a symmetric product; tiles on and below the diagonal only.
template <bool SQUARE, int TB>
__global__ __launch_bounds__(G_THREADS, 2) void ns_sym_kernel(const NsMat* __restrict__ table, int count, f16* __restrict__ ws,
                                                              const NsScale* __restrict__ sc, NsStep st, int parity,
                                                              float* __restrict__ part) {
  typedef G16<2, 2, ROW, ROW, TB> G;
  __shared__ __attribute__((aligned(1024))) f16 smem[G::LDS];
  const int i = find_mat(table, count, SQUARE ? BY_P : BY_S, blockIdx.x);
  const NsMat t = table[i];
  const NsMat::Cut cut = t.cut[SQUARE];
  const NsView w(t, parity);
  const int tiles = (t.m + G::T - 1) / G::T, all = tiles * (tiles + 1) / 2;
  int id = blockIdx.x - t.first[SQUARE ? BY_P : BY_S];  // whole tiles first, then slices; each kind spread over the XCDs by itself
  id = id < cut.direct ? xcd_run(id, cut.direct) : cut.direct + xcd_run(id - cut.direct, (all - cut.direct) * cut.slices);
  const int ld = SQUARE ? w.ldm : w.ldn;
  int tile = id, k0 = 0, k1 = ld, slot = -1;
  if (id >= cut.direct) {
    slot = id - cut.direct;
    tile = cut.direct + slot / cut.slices;
    const int per = (ld / G::BK + cut.slices - 1) / cut.slices * G::BK, s = slot % cut.slices;
    k0 = s * per;
    k1 = min(ld, k0 + per);
  }
  int tm, tn;
  tri_tile(tile, tiles, tm, tn);
  const int m0 = tm * G::T, n0 = tn * G::T;
  const f16* src = ws + (SQUARE ? w.s : w.x);
  const int64_t plane = (int64_t)t.m * ld;
  f32x4 acc[TB][TB];
  G::zero(acc);
  G::run(acc, Op16{src + (int64_t)m0 * ld, plane, ld, t.m - m0, 0}, Op16{src + (int64_t)n0 * ld, plane, ld, t.m - n0, 0}, k0,
         k1, smem);
  if (slot >= 0) {
    f32x4* o = reinterpret_cast<f32x4*>(part + ((int64_t)cut.p0 + slot) * G::T * G::T) + threadIdx.x;
#pragma unroll
    for (int e = 0; e < TB * TB; ++e) o[e * G_THREADS] = acc[e / TB][e % TB];
    return;
  }
  sym_store<SQUARE, TB>(acc, t, w, ws, sc[i], st, m0, n0, reinterpret_cast<float*>(smem));
}

// Joins the slices of a tile in order.  A workgroup takes 64 x 64 of it, of a 128 x 128 tile the part of one wave: reading
// its slices is what a join spends its time on (eight of 128 x 128 are 512 KiB: 13 us in one workgroup, 5 in four).
template <bool SQUARE, int TB>
__global__ __launch_bounds__(G_THREADS, 2) void ns_sym_join_kernel(const NsMat* __restrict__ table, int count, f16* __restrict__ ws,
                                                                   const NsScale* __restrict__ sc, NsStep st, int parity,
                                                                   const float* __restrict__ part) {
  constexpr int T = 32 * TB, PARTS = TB * TB / 4;
  __shared__ __attribute__((aligned(1024))) float smem[Tile16<2>::FLOATS];
  const int i = find_mat(table, count, SQUARE ? BY_JOIN_P : BY_JOIN_S, blockIdx.x);
  const NsMat t = table[i];
  const NsMat::Cut cut = t.cut[SQUARE];
  const NsView w(t, parity);
  const int id = blockIdx.x - t.first[SQUARE ? BY_JOIN_P : BY_JOIN_S], e0 = id / PARTS, wave = id % PARTS;
  int tm, tn;
  tri_tile(cut.direct + e0, (t.m + T - 1) / T, tm, tn);
  const int m0 = tm * T + (wave >> 1) * 64, n0 = tn * T + (wave & 1) * 64;
  if (m0 < n0 || m0 >= t.m) return;  // the mirror image of another part, or nothing
  const int lane = threadIdx.x & 63, wm = threadIdx.x >> 7, wn = (threadIdx.x >> 6) & 1;
  // where this thread's blocks (2 wm + i, 2 wn + j) of the part lie in a slice
  const int at = TB == 4 ? wave * 64 + lane + (wm * 8 + wn * 2) * G_THREADS : threadIdx.x;
  f32x4 acc[2][2];
  G16<2, 2, ROW, ROW, 2>::zero(acc);
  const f32x4* p = reinterpret_cast<const f32x4*>(part + ((int64_t)cut.p0 + (int64_t)e0 * cut.slices) * T * T) + at;
#pragma unroll 4
  for (int s = 0; s < cut.slices; ++s, p += T * T / 4)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e >> 1][e & 1] += p[((e >> 1) * TB + (e & 1)) * G_THREADS];
  sym_store<SQUARE, 2>(acc, t, w, ws, sc[i], st, m0, n0, smem);
}

// X <- a X + P X, into the other buffer, or the result in G's orientation after the last step.  The columns of X run along
// the registers, so X is read and written in groups of four.
template <typename T, int TB>
__global__ __launch_bounds__(G_THREADS, 2) void ns_update_kernel(const NsMat* __restrict__ table, int count, f16* __restrict__ ws,
                                                                 const NsScale* __restrict__ sc, NsStep st, int parity) {
  typedef G16<2, 2, COL, ROW, TB> G;
  typedef Tile16<TB> L;
  __shared__ __attribute__((aligned(1024))) f16 smem[G::LDS];
  const int i = find_mat(table, count, BY_UPDATE, blockIdx.x);
  const NsMat t = table[i];
  const NsView w(t, parity);
  const int tiles_m = (t.m + G::T - 1) / G::T, tiles_n = (t.n + G::T - 1) / G::T;
  int tm, tn, slice;
  g16_tile(blockIdx.x - t.first[BY_UPDATE], 1, tiles_m, tiles_n, slice, tm, tn);
  const int m0 = tm * G::T, n0 = tn * G::T;
  const int64_t pp = (int64_t)t.m * w.ldm, px = (int64_t)t.m * w.ldn;
  const f16* x = ws + w.x;
  f32x4 acc[TB][TB];
  G::zero(acc);
  G::run(acc, Op16{x, px, w.ldn, t.m, n0}, Op16{ws + w.p + (int64_t)m0 * w.ldm, pp, w.ldm, t.m - m0, 0}, 0, w.ldm, smem);
  f16* xo = ws + w.xo;
  const float f = ldexpf(1.f, -st.ep), fo = sc[i].rho;
  const int ey = sc[i].ey;
  T* out = (T*)t.out;
  const bool vec = !t.tall && t.n % 8 == 0 && ((uintptr_t)out & 15) == 0;
  float* tile = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int half = 0; half < L::HALVES; ++half) {
    const int r0 = m0 + half * 64;
    f16x8 xh[L::UNITS], xl[L::UNITS];  // X's tile, on its way while P X passes through LDS
#pragma unroll
    for (int u = 0; u < L::UNITS; ++u) {
      const int e = threadIdx.x + u * G_THREADS;
      const int64_t o = (int64_t)min(r0 + e / L::VPR, t.m - 1) * w.ldn + min(n0 + e % L::VPR * 8, w.ldn - 8);
      xh[u] = *reinterpret_cast<const f16x8*>(x + o);
      xl[u] = *reinterpret_cast<const f16x8*>(x + o + px);
    }
    L::put(acc, half, tile);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < L::UNITS; ++u) {
      const int e = threadIdx.x + u * G_THREADS, rl = e / L::VPR, cl = e % L::VPR * 8, r = r0 + rl, c = n0 + cl;
      F8 v = L::get(tile, rl, cl);
#pragma unroll
      for (int k = 0; k < 8; ++k) v.v[k] = fmaf(st.a, (float)xh[u][k] + (float)xl[u][k], v.v[k] * f);
      if (st.last) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v.v[k] = fo * ldexpf(v.v[k], -ey);
      }
      if (st.last && t.tall) {  // the result is transposed: through LDS once more
        L::set(tile, rl, cl, v);
      } else if (st.last) {
        if (r < t.m && c < t.n) {
          T* d = out + (int64_t)r * t.n + c;
          if (vec) store8(d, v);
          else
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (c + k < t.n) d[k] = from_f32<T>(v.v[k]);
        }
      } else if (r < t.m && c < w.ldn) {
        f16x8 h, l;
        f16_split8(v, h, l);
        const int64_t o = (int64_t)r * w.ldn + c;
        *reinterpret_cast<f16x8*>(xo + o) = h;
        *reinterpret_cast<f16x8*>(xo + o + px) = l;
      }
    }
    __syncthreads();
    if (st.last && t.tall) {
      for (int e = threadIdx.x; e < G::T * 64; e += G_THREADS) {
        const int cl = e >> 6, rl = e & 63;
        if (n0 + cl < t.n && r0 + rl < t.m) out[(int64_t)(n0 + cl) * t.m + r0 + rl] = from_f32<T>(tile[L::at(rl, cl)]);
      }
      __syncthreads();
    }
  }
}

// steps = 0: the normalised matrix itself
template <typename T>
__global__ __launch_bounds__(256) void ns_copy_kernel(const NsMat* __restrict__ table, int count,
                                                    const NsScale* __restrict__ sc) {
  const int i = find_mat(table, count, BY_NORM, blockIdx.x);
  const NsMat t = table[i];
  const int64_t total = (int64_t)t.m * t.n, e0 = (int64_t)(blockIdx.x - t.first[BY_NORM]) * NORM_CHUNK;
  const int64_t e1 = e0 + NORM_CHUNK < total ? e0 + NORM_CHUNK : total;
  const double f = ldexp(sc[i].inv, -sc[i].ey) * (double)sc[i].rho;
  for (int64_t e = e0 + threadIdx.x; e < e1; e += 256)
    ((T*)t.out)[e] = from_f32<T>((float)((double)to_f32(((const T*)t.g)[e]) * f));
}

// Matrices of at most 16 rows (columns, if tall): all steps in one workgroup, X in LDS, in fp64 where it fits twice and
// fp32 otherwise.  A 128 x 128 product tile would be nine tenths padding, and a matrix this small has nothing to average
// the two-term rounding over: its result was off by up to five times fp32's error.  One workgroup's time grows with
// m^2 n (12 x 199 in 49 us; 16 x 2200 in 230 against 173 for the launches of the tiled form), hence the third bound.
constexpr int SMALL_ROWS = 16, SMALL_ELEMS = 36000, SMALL_THREADS = 512, SMALL_MAX = 96;
struct NsSmall {
  const void* g;
  void* out;
  int m, n, tall;
};
struct NsSmallArgs {
  NsSmall mat[SMALL_MAX];
};
bool is_small(int rows, int cols) {
  const int64_t m = rows < cols ? rows : cols, total = (int64_t)rows * cols;
  return m <= SMALL_ROWS && total <= SMALL_ELEMS && m * total <= 200000;
}

template <typename F>
__device__ __forceinline__ F wave_sum_of(F v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

struct NsCoeffs {
  float v[3 * 64];
};

template <typename T, typename F>
__device__ __forceinline__ void small_steps(const NsSmall& t, const NsCoeffs& c, int steps, double eps, F* x,
                                            F (&s)[SMALL_ROWS][SMALL_ROWS + 1], F (&p)[SMALL_ROWS][SMALL_ROWS],
                                            double (&sums)[SMALL_THREADS / 64]) {
  constexpr int R = SMALL_ROWS;
  const int m = t.m, n = t.n, total = m * n;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T* g = (const T*)t.g;
  double sq = 0.0;
  for (int e = threadIdx.x; e < total; e += SMALL_THREADS) {
    const float v = to_f32(g[e]);
    x[t.tall ? e % m * n + e / m : e] = v;
    sq += (double)v * (double)v;
  }
  sq = wave_sum_f64(sq);
  if (lane == 0) sums[wave] = sq;
  for (int e = threadIdx.x; e < R * R; e += SMALL_THREADS) p[e / R][e % R] = 0;
  __syncthreads();
  double norm = 0.0;
#pragma unroll
  for (int w = 0; w < SMALL_THREADS / 64; ++w) norm += sums[w];
  norm = sqrt(norm) + eps;
  const double inv = norm == 0.0 ? 0.0 : 1.0 / norm;
  for (int e = threadIdx.x; e < total; e += SMALL_THREADS) x[e] = (F)((double)x[e] * inv);
  for (int k = 0; k < steps; ++k) {
    __syncthreads();
    // S: a wave per pair of rows
    for (int pr = wave; pr < m * (m + 1) / 2; pr += SMALL_THREADS / 64) {
      int i = (int)((sqrtf(8.f * pr + 1.f) - 1.f) * 0.5f);
      while ((i + 1) * (i + 2) / 2 <= pr) ++i;
      while (i * (i + 1) / 2 > pr) --i;
      const int j = pr - i * (i + 1) / 2;
      F d = 0;
      for (int e = lane; e < n; e += 64) d = fma(x[i * n + e], x[j * n + e], d);
      d = wave_sum_of(d);
      if (lane == 0) s[i][j] = s[j][i] = d;
    }
    __syncthreads();
    // P = b S + c S S
    const F ca = c.v[3 * k], cb = c.v[3 * k + 1], cc = c.v[3 * k + 2];
    for (int e = threadIdx.x; e < m * m; e += SMALL_THREADS) {
      const int i = e / m, j = e - i * m;
      F d = 0;
      for (int q = 0; q < m; ++q) d = fma(s[i][q], s[q][j], d);
      p[i][j] = fma(cb, s[i][j], cc * d);
    }
    __syncthreads();
    // X <- a X + P X: a thread owns whole columns
    for (int e = threadIdx.x; e < n; e += SMALL_THREADS) {
      F v[R];
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] = i < m ? x[i * n + e] : (F)0;
      for (int i = 0; i < m; ++i) {
        F d = 0;
#pragma unroll
        for (int q = 0; q < R; ++q) d = fma(p[i][q], v[q], d);
        x[i * n + e] = fma(ca, x[i * n + e], d);
      }
    }
  }
  __syncthreads();
  T* o = (T*)t.out;
  for (int e = threadIdx.x; e < total; e += SMALL_THREADS) o[e] = from_f32<T>((float)x[t.tall ? e % m * n + e / m : e]);
}

template <typename T>
__global__ __launch_bounds__(SMALL_THREADS) void ns_small_kernel(NsSmallArgs a, NsCoeffs c, int steps, double eps) {
  constexpr int R = SMALL_ROWS;
  __shared__ __attribute__((aligned(16))) float x[SMALL_ELEMS];  // [m][n]
  __shared__ double s[R][R + 1], p[R][R], sums[SMALL_THREADS / 64];
  const NsSmall t = a.mat[blockIdx.x];
  if (t.m * t.n <= SMALL_ELEMS / 2) small_steps<T, double>(t, c, steps, eps, (double*)x, s, p, sums);
  else
    small_steps<T, float>(t, c, steps, eps, x, reinterpret_cast<float(&)[R][R + 1]>(s), reinterpret_cast<float(&)[R][R]>(p),
                          sums);
}

int sym_tiles(const NsMat& t, int tile) {
  const int n = ceil_div(t.m, tile);
  return n * (n + 1) / 2;
}

// How the symmetric products of a launch are cut.  `slots` workgroups (two per CU, or one) run at once.
//  - Fewer tiles than slots: every reduction is cut into runs of about equal length so that the runs fill the slots.
//  - One matrix with a little more than whole rounds of tiles: the tiles of the last round are cut instead of leaving
//    most of the chip idle for it (4096 x 4096: 528 tiles on 512 slots).
// Fills cut[square] of every matrix and returns the partial tiles; the reduction is in k-steps of 32.
int64_t cut_sym(NsMat* mats, int n, int square, int tile) {
  int64_t slots = 512, tiles = 0, work = 0, parts = 0;
  auto len = [&](const NsMat& t) { return up64(square ? t.m : t.n) / 32; };
  for (int i = 0; i < n; ++i) {
    tiles += sym_tiles(mats[i], tile);
    work += (int64_t)sym_tiles(mats[i], tile) * len(mats[i]);
  }
  if (work < 512 * 16) slots = 256;  // short runs: one workgroup per CU
  for (int i = 0; i < n; ++i) {
    const NsMat& t = mats[i];
    NsMat::Cut& c = mats[i].cut[square];
    const int all = sym_tiles(t, tile);
    c.direct = all;
    c.slices = 1;
    if (tiles < slots) {
      const int64_t run = ceil_div64(work, slots) > 8 ? ceil_div64(work, slots) : 8;
      const int64_t s = len(t) / run;
      if (s > 1) {
        c.slices = (int)(s < 8 ? s : 8);
        c.direct = 0;
      }
    } else if (n == 1 && tiles % slots && tiles % slots <= slots / 2) {
      const int tail = (int)(tiles % slots), room = (int)(slots / tail);
      const int s = room < len(t) / 4 ? room : len(t) / 4;
      if (s > 1) {
        c.slices = s < 8 ? s : 8;
        c.direct = all - tail;
      }
    }
    c.p0 = (int)parts;
    parts += (int64_t)(all - c.direct) * c.slices;
  }
  return parts;
}

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

// The table of a launch's matrices, the workgroups of every kind of launch, and where everything lies in the workspace:
// [table | NsScale per matrix | partial norms | partial tiles | fp16 buffers]
struct NsLayout {
  NsMat mat[NS_MAX];
  int64_t blocks[KINDS];
  int64_t norms, part, bufs, bytes;
  int tile_s, tile_p, tile_u;  // 128 or 64
  NsLayout(const int* rows, const int* cols, int count) {
    int64_t at = 0;
    double ws = 0, wp = 0;
    for (int i = 0; i < count; ++i) {
      NsMat& t = mat[i];
      t = NsMat{};
      t.tall = rows[i] > cols[i];
      t.m = t.tall ? cols[i] : rows[i];
      t.n = t.tall ? rows[i] : cols[i];
      t.at = at;
      at = NsView(t, 0).end;
      ws += (double)t.m * t.m * t.n;
      wp += (double)t.m * t.m * t.m;
    }
    tile_s = ws <= NS_SMALL_SYM ? 64 : 128;
    tile_p = wp <= NS_SMALL_SYM ? 64 : 128;
    tile_u = 2 * ws <= NS_SMALL_UPDATE ? 64 : 128;
    const int64_t ps = cut_sym(mat, count, 0, tile_s) * tile_s * tile_s, pp = cut_sym(mat, count, 1, tile_p) * tile_p * tile_p;
    for (int k = 0; k < KINDS; ++k) {
      blocks[k] = 0;
      for (int i = 0; i < count; ++i) {
        NsMat& t = mat[i];
        t.first[k] = (int)blocks[k];
        const bool sq = k == BY_P || k == BY_JOIN_P;
        const NsMat::Cut& c = t.cut[sq];
        const int tile = k == BY_UPDATE ? tile_u : sq ? tile_p : tile_s;
        blocks[k] += k == BY_NORM     ? ceil_div64((int64_t)t.m * t.n, NORM_CHUNK)
                     : k == BY_INIT   ? (int64_t)(up64(t.m) / 64) * (up64(t.n) / 64)
                     : k == BY_UPDATE ? (int64_t)ceil_div(t.m, tile) * ceil_div(t.n, tile)
                     : k <= BY_P      ? c.direct + (int64_t)(sym_tiles(t, tile) - c.direct) * c.slices
                                      : (int64_t)(sym_tiles(t, tile) - c.direct) * (tile * tile / 4096);
      }
    }
    norms = NS_MAX * (int64_t)(sizeof(NsMat) + sizeof(NsScale));
    part = norms + up128(blocks[BY_NORM] * 8);
    bufs = part + (ps > pp ? ps : pp) * 4;
    bytes = bufs + at * 2;
  }
};

}  // namespace

extern "C" {

int64_t vc_newton_schulz_bytes(int count, const int* rows, const int* cols) {
  if (check_ns("vc_newton_schulz_bytes", VC_F32, count, rows, cols) != VC_OK) return -1;
  int64_t most = 256;
  for (int b = 0; b < count;) {
    int r[NS_MAX], c[NS_MAX], n = 0;
    for (; b < count && n < NS_MAX; ++b)
      if (!is_small(rows[b], cols[b])) {
        r[n] = rows[b];
        c[n++] = cols[b];
      }
    const int64_t bytes = n ? NsLayout(r, c, n).bytes : 0;
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
  NsStep st;
  st.es = (int)floorf(log2f(60000.f / (cap * cap)));
  st.ep = (int)floorf(log2f(60000.f / pmax));
  const bool bf = dtype == VC_BF16;
  NsMat* table = (NsMat*)workspace;
  NsScale* sc = (NsScale*)(table + NS_MAX);
  NsSmallArgs small;
  int ns = 0;
  auto flush = [&]() {
    NsCoeffs c{};
    for (int k = 0; k < 3 * steps; ++k) c.v[k] = coeffs[k];
    if (ns) hipLaunchKernelGGL((bf ? ns_small_kernel<bf16> : ns_small_kernel<float>), dim3(ns), dim3(SMALL_THREADS), 0, stream, small, c, steps, eps);
    ns = 0;
  };
  for (int b = 0; b < count;) {
    int r[NS_MAX], c[NS_MAX], src[NS_MAX], n = 0;
    for (; b < count && n < NS_MAX; ++b) {
      if (is_small(rows[b], cols[b])) {
        const bool tall = rows[b] > cols[b];
        small.mat[ns++] = NsSmall{g[b], out[b], tall ? cols[b] : rows[b], tall ? rows[b] : cols[b], tall};
        if (ns == SMALL_MAX) flush();
      } else {
        r[n] = rows[b];
        c[n] = cols[b];
        src[n++] = b;
      }
    }
    if (!n) break;  // the rest was small
    NsLayout l(r, c, n);
    for (int k = 0; k < KINDS; ++k)  // a launch holds fewer than 2^32 threads
      VC_CHECK_SHAPE(l.blocks[k] < (1 << 24), "vc_newton_schulz: the matrices of a launch are more than 2^24 tiles");
    double* norms = (double*)((char*)workspace + l.norms);
    float* part = (float*)((char*)workspace + l.part);
    f16* ws = (f16*)((char*)workspace + l.bufs);
    for (int i = 0; i < n; ++i) {
      l.mat[i].g = g[src[i]];
      l.mat[i].out = out[src[i]];
    }
    for (int i = 0; i < n; i += NS_CHUNK) {
      NsChunk e;
      const int k = n - i < NS_CHUNK ? n - i : NS_CHUNK;
      memcpy(e.mat, l.mat + i, k * sizeof(NsMat));
      hipLaunchKernelGGL(ns_table_kernel, dim3(1), dim3(64), 0, stream, e, table + i, k);
    }
    auto launch = [&](int kind, auto kernel, int threads, auto... args) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)l.blocks[kind]), dim3(threads), 0, stream, table, n, args...);
    };
    launch(BY_NORM, bf ? ns_norm_kernel<bf16> : ns_norm_kernel<float>, 256, norms);
    hipLaunchKernelGGL(ns_scale_kernel, dim3(n), dim3(64), 0, stream, table, n, (int)l.blocks[BY_NORM], norms, eps, cap, gain, sc);
    if (steps == 0) launch(BY_NORM, bf ? ns_copy_kernel<bf16> : ns_copy_kernel<float>, 256, sc);
    else launch(BY_INIT, bf ? ns_init_kernel<bf16> : ns_init_kernel<float>, 256, ws, sc);
    for (int k = 0; k < steps; ++k) {
      st.a = coeffs[3 * k];
      st.b = coeffs[3 * k + 1];
      st.c = coeffs[3 * k + 2];
      st.last = k == steps - 1;
      auto sym = [&](auto square, auto tb) {
        constexpr bool SQ = decltype(square)::value;
        constexpr int TB = decltype(tb)::value;
        launch(SQ ? BY_P : BY_S, ns_sym_kernel<SQ, TB>, G_THREADS, ws, sc, st, k & 1, part);
        const int join = SQ ? BY_JOIN_P : BY_JOIN_S;
        if (l.blocks[join]) launch(join, ns_sym_join_kernel<SQ, TB>, G_THREADS, ws, sc, st, k & 1, part);
      };
      const std::integral_constant<int, 2> t64;
      const std::integral_constant<int, 4> t128;
      if (l.tile_s == 64) sym(std::false_type(), t64);
      else sym(std::false_type(), t128);
      if (l.tile_p == 64) sym(std::true_type(), t64);
      else sym(std::true_type(), t128);
      if (l.tile_u == 64) launch(BY_UPDATE, bf ? ns_update_kernel<bf16, 2> : ns_update_kernel<float, 2>, G_THREADS, ws, sc, st, k & 1);
      else launch(BY_UPDATE, bf ? ns_update_kernel<bf16, 4> : ns_update_kernel<float, 4>, G_THREADS, ws, sc, st, k & 1);
    }
  }
  flush();
  VC_LAUNCH_CHECK("vc_newton_schulz");
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

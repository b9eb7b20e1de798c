// Softmax cross entropy of a linear classifier, z = x W^T + b over V classes, without the logit matrix: forward keeps a
// running maximum and sum per row and tile of classes, backward recomputes the logits of a piece of the classes at a time.
//
//   lse_n = log sum_v exp(z_nv),  loss_n = lse_n - (1 - eps) z_{n,t_n} - eps / V sum_v z_nv
//   d_nv = (exp(z_nv - lse_n) - (1 - eps) [v = t_n] - eps / V) r_n          (r_n the row's weight in the loss)
//   dx = d W,  dW += d^T x,  db += sum_n d
// Rows whose target is ignore_index have r_n = 0 and are never read: the rows that count are packed one behind the other, and
// every kernel behind the packing works on those alone, their number read from the device.  (Masked-token losses and padded
// batches leave out most of their rows; a quarter of them ignored takes a quarter off every product.)
//
// 2 N V K operations forward, 6 N V K backward (the logits once more, dx, dW): bound by the matrix pipes for the sizes where
// time matters, which is why the logits are recomputed rather than kept: N x V fp32 logits written and read cost as much
// as the product at K = 1024 and gigabytes of memory.  8192 x 1024 x 65536 in bf16: 4.4 - 4.7 ms forward and backward by
// card, 1.0 PFLOP/s over its four products; 2048 x 512 x 20011 forward: 65 us, 54 of them the statistics (0.8 PFLOP/s).
//
// All products run on fp16 terms (vc_gemm16.h).  x and W are scaled by one power of two each (from their largest finite
// magnitude), but for rows whose own largest value lies more than 16 binades below it, which are scaled by themselves: no row
// takes precision from another one.  bf16 values are exact in one term over 29 binades and within 2^-23 of their row's largest
// magnitude below that, fp32 values take two terms (22 bits).  An fp32 master weight next to bf16 activations takes one
// term (11 bits, against the 8 of a bf16 copy).  d is at most 1 in magnitude and is scaled by 2^15: one term (2^-11 of
// the value) where the gradient it makes is bf16, two where it is fp32.
#include "vc_gemm16.h"

namespace {

constexpr int AMAX_MOST = 1024;  // partial maxima per operand, at most

// ---- scales ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ float finite_mag(float v) {
  const float a = fabsf(v);
  return a <= 3.4028235e38f ? a : 0.f;  // NaN and infinities do not set the scale
}

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Row8 {  // eight values in one wide load whatever their alignment
  T v[8];
};

// rowmax[r] = largest finite magnitude of row r (not of rows that do not count); returns that of all rows this lane met.  As
// many lanes per row as it has groups of eight values, up to a wave, and four rows at once, so that their loads overlap
// (65536 + 8192 rows of 1024 in bf16: 40 us, 45 one by one).
template <typename T>
__device__ __forceinline__ float amax_rows(const T* p, int64_t rows, int K, const int64_t* target, int64_t ignore,
                                           float* rowmax, int block, int nblocks) {
  constexpr int U = 4;
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < K) lanes <<= 1;
  const int lane = threadIdx.x & 63, k0 = (lane & (lanes - 1)) * 8, per = 64 / lanes;
  const int64_t step = (int64_t)nblocks * 4 * per;  // rows between those of a lane
  float most = 0.f;
  for (int64_t first = ((int64_t)block * 4 + (threadIdx.x >> 6)) * per; first < rows; first += U * step) {
    bool on[U];
    const T* row[U];
    float m[U];
    const T* some = nullptr;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = first + lane / lanes + u * step;
      on[u] = r < rows && !(target && target[r] == ignore);
      row[u] = p + r * K;
      if (on[u]) some = row[u];
      m[u] = 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (!on[u]) row[u] = some;  // another row in place of one that does not count, whose values are dropped
    int k = some ? k0 : K;
    for (; k + 8 <= K; k += lanes * 8) {
      Row8<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const Row8<T>*>(row[u] + k);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) m[u] = fmaxf(m[u], finite_mag(to_f32(v[u].v[e])));
    }
    for (; k < K; ++k)  // the lane with the rows' last, partial group
#pragma unroll
      for (int u = 0; u < U; ++u) m[u] = fmaxf(m[u], finite_mag(to_f32(row[u][k])));
    for (int o = 1; o < lanes; o <<= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) m[u] = fmaxf(m[u], __shfl_xor(m[u], o, 64));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!on[u]) continue;
      if (k0 == 0) rowmax[first + lane / lanes + u * step] = m[u];
      most = fmaxf(most, m[u]);
    }
  }
  return most;
}

// The rows of a call in the order they are packed: order[0 .. count) = the rows that count, in order, then the others;
// target[k] = class of the k-th of them, -1 if there is no such class.
struct RowList {
  int *order, *target, *count;  // count[1], count[2]: cleared here, set where a row of x / of W has a scale of its own
};

// One workgroup, 4096 rows at a time.  Rows that do not count get their loss (0) and prediction (0) here.
__device__ __forceinline__ void list_rows(const int64_t* __restrict__ target, int64_t ignore, int N, int V, const RowList& l,
                                          float* __restrict__ rowloss, int64_t* __restrict__ pred) {
  constexpr int U = 16;
  __shared__ int counts[2][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int base = 0;
  for (int n0 = 0, par = 0; n0 < N; n0 += U * 256, par ^= 1) {
    int64_t t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) t[u] = target[min(n0 + u * 256 + (int)threadIdx.x, N - 1)];
    uint64_t keep[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      keep[u] = __ballot(n0 + u * 256 + (int)threadIdx.x < N && t[u] != ignore);
      if (lane == 0) counts[par][u * 4 + wave] = __popcll(keep[u]);
    }
    __syncthreads();
    const int mine = counts[par][lane];
    int upto = mine;  // inclusive sum over the 64 runs of 64 rows
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o, 64);
      if (lane >= o) upto += v;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = n0 + u * 256 + threadIdx.x;
      const int before = base + __shfl(upto - mine, u * 4 + wave, 64) + __popcll(keep[u] & ((1ull << lane) - 1));
      if (n >= N) continue;
      if (keep[u] >> lane & 1) {
        l.order[before] = n;
        l.target[before] = t[u] >= 0 && t[u] < V ? (int)t[u] : -1;
      } else {
        l.order[N - 1 - (n - before)] = n;
        rowloss[n] = 0.f;
        if (pred) pred[n] = 0;
      }
    }
    base += __shfl(upto, 63, 64);
  }
  if (threadIdx.x == 0) {
    l.count[0] = base;
    l.count[1] = l.count[2] = 0;
  }
}

// amax[0 .. xb) / [AMAX_MOST ..] = largest finite magnitudes met by the xb blocks of x / the next ones' of W; the last block
// lists the rows
template <typename TX, typename TW>
__global__ __launch_bounds__(256) void ce_amax_kernel(const TX* __restrict__ x, const TW* __restrict__ w, int N, int V,
                                                      int K, const int64_t* __restrict__ target, int64_t ignore,
                                                      float* __restrict__ amax, int xb, RowList rows,
                                                      float* __restrict__ rowloss, int64_t* __restrict__ pred,
                                                      float* __restrict__ xmax, float* __restrict__ wmax) {
  __shared__ float sm[4];
  const int b = blockIdx.x, wb = (int)gridDim.x - 1 - xb;
  if (b == xb + wb) {
    list_rows(target, ignore, N, V, rows, rowloss, pred);
    return;
  }
  float m = b < xb ? amax_rows(x, N, K, target, ignore, xmax, b, xb)
                   : amax_rows(w, V, K, (const int64_t*)nullptr, 0, wmax, b - xb, wb);
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) amax[b < xb ? b : AMAX_MOST + b - xb] = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
}

// exponent e with 2^14 <= amax 2^e < 2^15 (0 for an operand without a finite value other than zero)
__device__ __forceinline__ int scale_exp(const float* amax, int parts, float* sm) {
  float m = 0.f;
  for (int i = threadIdx.x; i < parts; i += 256) m = fmaxf(m, amax[i]);
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  return m > 0.f ? 14 - ilogbf(m) : 0;
}

// ---- packing -----------------------------------------------------------------------------------------------------
// Amax and packing pass over x and W once each: 40 + 70 us for (8192 + 65536) x 1024 in bf16 (3.8 and 4.3 TB/s), 2 % of the
// call.
//
// A row whose largest value lies more than this many binades below the operand's is scaled by itself.  Up to there the
// operand's scale keeps 2^-23 of the row's own largest value: half of fp16's last step, 2^-25, next to at least 2^(14 - 16).
constexpr int OWN_SCALE = 16;

// dst[plane][row][ld] = terms of src[order[row]][k] 2^e (order null: row), zeros behind K; exps[row] = e, e0 or the row's own
// scale, and then *own = 1.  A wave per row and 512 columns.
template <typename T>
__device__ __forceinline__ void pack_rows(const T* __restrict__ src, f16* __restrict__ dst, int64_t plane, int rows, int K,
                                          int ld, int planes, int e0, const int* order, int64_t unit,
                                          const float* __restrict__ rowmax, int* __restrict__ exps, int* __restrict__ own) {
  const int per = (ld + 511) / 512;
  const int64_t row = unit / per;
  if (row >= rows) return;
  const int c0 = (int)(unit - row * per) * 512 + (threadIdx.x & 63) * 8;
  if (c0 >= ld) return;
  const int64_t from = order ? order[row] : row;
  const T* s = src + from * K;
  const float most = rowmax[from];
  int e = most > 0.f ? 14 - ilogbf(most) : e0;
  if (e - e0 <= OWN_SCALE) e = e0;
  if (c0 == 0) {
    exps[row] = e;
    if (e != e0) *own = 1;
  }
  float v[8];
  if (c0 + 8 <= K) {
    const Row8<T> t = *reinterpret_cast<const Row8<T>*>(s + c0);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(t.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < K ? to_f32(s[c0 + i]) : 0.f;
  }
  f16x8 hi, lo;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f16 h, l;
    f16_split(ldexpf(v[i], e), h, l);
    hi[i] = h;
    lo[i] = l;
  }
  *reinterpret_cast<f16x8*>(dst + row * ld + c0) = hi;
  if (planes == 2) *reinterpret_cast<f16x8*>(dst + plane + row * ld + c0) = lo;
}

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// bias log2(e); a finite one stays finite (a mask of the type's lowest value is no -inf: a row that it leaves nothing else
// spreads its probability evenly)
template <typename T>
__device__ __forceinline__ float bias_log2(T b) {
  const float v = to_f32(b) * LOG2E, most = 3.4028235e38f;
  return fabsf(to_f32(b)) <= most ? fminf(fmaxf(v, -most), most) : v;
}

// exps[0] / [1] = scale exponents of x / W, [2] = rows that count, [3] / [4] = whether rows of x / W have their own; the first
// `xblocks` workgroups pack x, the others W and the bias: bl = bias log2(e) over whole tiles of classes, -inf behind the last
// one, which leaves the epilogues of the products four plain vector loads (clamped and converted there, these cost a fifth of
// a tile's time).
template <typename TX, typename TW>
__global__ __launch_bounds__(256) void ce_pack_kernel(const TX* __restrict__ x, const TW* __restrict__ w, int N, int V,
                                                      int K, int ld, int px, int pw, const int* __restrict__ order,
                                                      const float* __restrict__ amax, f16* __restrict__ xp,
                                                      f16* __restrict__ wp, int* __restrict__ exps, int xblocks, int xb,
                                                      int wb, const TW* __restrict__ bias, float* __restrict__ bl,
                                                      const float* __restrict__ xmax, const float* __restrict__ wmax,
                                                      int* __restrict__ ex, int* __restrict__ ew) {
  __shared__ float sm[4];
  const bool isx = (int)blockIdx.x < xblocks;
  const int e = scale_exp(isx ? amax : amax + AMAX_MOST, isx ? xb : wb, sm);
  if (threadIdx.x == 0 && ((int)blockIdx.x == 0 || (int)blockIdx.x == xblocks)) exps[isx ? 0 : 1] = e;
  const int64_t unit = (int64_t)(isx ? blockIdx.x : blockIdx.x - xblocks) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (isx) pack_rows(x, xp, (int64_t)N * ld, exps[2], K, ld, px, e, order, unit, xmax, ex, exps + 3);
  else {
    pack_rows(w, wp, (int64_t)V * ld, V, K, ld, pw, e, (const int*)nullptr, unit, wmax, ew, exps + 4);
    const int64_t v = (int64_t)(blockIdx.x - xblocks) * 256 + threadIdx.x;  // four rows or more per workgroup: all classes
    if (v < (V + GM - 1) / GM * GM) bl[v] = v >= V ? -INFINITY : bias ? bias_log2(bias[v]) : 0.f;
  }
}

// A forward call whose operands are bf16 with K a multiple of 64 and that keeps nothing for a backward pass multiplies them as
// they are: no scales, no copy of W (2048 x 512 x 20011: 75 -> 64 us), the rows that count copied one behind the other.
__global__ __launch_bounds__(256) void ce_list_kernel(const int64_t* __restrict__ target, int64_t ignore, int N, int V, RowList rows,
                                                      float* __restrict__ rowloss, int64_t* __restrict__ pred) {
  list_rows(target, ignore, N, V, rows, rowloss, pred);
}
__global__ __launch_bounds__(256) void ce_copy_kernel(const bf16* __restrict__ x, int V, int K, const int* __restrict__ order,
                                                      bf16* __restrict__ xp, int* __restrict__ exps,
                                                      const bf16* __restrict__ bias, float* __restrict__ bl) {
  if (blockIdx.x == 0 && threadIdx.x < 2) exps[threadIdx.x] = 0;
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  for (int64_t v = first; v < (V + GM - 1) / GM * GM; v += step) bl[v] = v >= V ? -INFINITY : bias ? bias_log2(bias[v]) : 0.f;
  const int per = K / 8;
  const int64_t total = (int64_t)exps[2] * per;
  const bool vec = ((uintptr_t)x & 15) == 0;
  for (int64_t u = first; u < total; u += step) {
    const int64_t row = u / per;
    const int c = (int)(u - row * per) * 8;
    const bf16* s = x + (int64_t)order[row] * K + c;
    bf16x8 v;
    if (vec) v = *reinterpret_cast<const bf16x8*>(s);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = s[e];
    *reinterpret_cast<bf16x8*>(xp + row * K + c) = v;
  }
}

// ---- logits of a 128-class x 128-row tile ---------------------------------------------------------------------------
// Everything behind the products works on z log2(e): the exponentials are then one subtraction and one v_exp_f32.
struct CeArgs {
  const f16* w;      // [pw][V][ld]
  const f16* x;      // [px][N][ld]
  const float* bl;   // bias log2(e), -inf behind the last class
  const int* target; // of the packed rows
  const int* exps;
  const int *ex, *ew;  // scale exponents of the packed rows and of the classes
  int N, V, K, ld, db_bf16;
  int tiles_v;

  __device__ __forceinline__ int rows() const { return exps[2]; }
  // this workgroup's tile; false behind the rows that count (one row tile is worked even if there are none)
  __device__ __forceinline__ bool tile(int& tv, int& tn) const {
    const int tiles_n = max(1, (rows() + GM - 1) / GM), total = tiles_v * tiles_n;
    if ((int)blockIdx.x >= total) return false;
    int slice;
    g16_tile(blockIdx.x, 1, tiles_v, tiles_n, slice, tv, tn);
    return true;
  }
};

// acc = z log2(e) without the bias, which follows in `bias` (-inf behind the last class): rows v0 + .., columns n0 + ..
template <int PW, int PX, bool BF = false>
__device__ __forceinline__ void logit_tile(const CeArgs& a, int v0, int n0, f16* smem, f32x4 (&acc)[4][4],
                                           f32x4 (&bias)[4], float& scale) {
  typedef G16<PW, PX, ROW, ROW, 4, BF> G;
  G::zero(acc);
  if (a.rows() > n0)  // not where no row counts: G16 reads operands of one row at least
    G::run(acc, Op16{a.w + (int64_t)v0 * a.ld, (int64_t)a.V * a.ld, a.ld, a.V - v0, 0},
           Op16{a.x + (int64_t)n0 * a.ld, (int64_t)a.N * a.ld, a.ld, a.rows() - n0, 0}, 0, (a.K + G::BK - 1) / G::BK * G::BK, smem);
  const float* bl = a.bl + v0 + (threadIdx.x >> 7) * 64 + ((threadIdx.x & 63) >> 4) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = *reinterpret_cast<const f32x4*>(bl + i * 16);
  const int es = -(a.exps[0] + a.exps[1]);
  if (!BF && (a.exps[3] | a.exps[4] || es < -120 || es > 120)) {  // scales by rows and classes, or beyond one factor's range
    const int lane = threadIdx.x & 63, n = n0 + (threadIdx.x >> 6 & 1) * 64 + (lane & 15);
    const int v = v0 + (threadIdx.x >> 7) * 64 + (lane >> 4) * 4;
    int er[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) er[j] = a.ex[max(min(n + j * 16, a.rows() - 1), 0)];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int ec = a.ew[min(v + i * 16 + r, a.V - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j][r] = ldexpf(acc[i][j][r], -(er[j] + ec));
      }
    scale = LOG2E;
  } else
    scale = ldexpf(LOG2E, es);
}

// position of class t among this lane's 16 of a tile column (i * 4 + r), or -1
__device__ __forceinline__ int lane_class(int t, int v0) {
  const int lane = threadIdx.x & 63, d = t - (v0 + (threadIdx.x >> 7) * 64 + (lane >> 4) * 4);
  return (unsigned)d < 64u && (d & 12) == 0 ? (d >> 4) * 4 + (d & 3) : -1;
}
__device__ __forceinline__ int row_target(const CeArgs& a, int n) {
  const int t = a.target[max(min(n, a.rows() - 1), 0)];
  return n < a.rows() ? t : -1;
}

// ---- forward: statistics of a tile -----------------------------------------------------------------------------------
struct Stat {
  float m, s, z;  // running maximum, sum of 2^(z - m), sum of z (all in units of log2)
  int arg;        // lowest class that attains m
};
__device__ __forceinline__ void stat_join(Stat& a, const Stat& b) {
  if (b.m > a.m || (b.m == a.m && b.arg < a.arg)) a.arg = b.arg;
  const float m = fmaxf(a.m, b.m);
  const float ref = m == -INFINITY ? 0.f : m;  // nothing but -inf so far: 2^(-inf - 0) = 0
  a.s = a.s * __builtin_amdgcn_exp2f(a.m - ref) + b.s * __builtin_amdgcn_exp2f(b.m - ref);
  a.m = m;
  a.z += b.z;
}
// 1.0 PFLOP/s at K = 1024 (1.08 - 1.16 ms for 8192 x 65536), 0.8 at K = 512, where eight k-steps carry the same epilogue: 64
// exponentials a thread and the joins, the maximum first, so that they cost no exponentials of their own.
//
// part[vt][n] = (max, sum, sum z, arg) of the tile, zt[n] = the target's logit.  MORE: also sum z and arg (label smoothing,
// predictions), which cost four operations more per logit.
template <int PW, int PX, bool MORE, bool BF>
__global__ __launch_bounds__(G_THREADS, 2) void ce_stats_kernel(CeArgs a, float4* __restrict__ part,
                                                                float* __restrict__ zt) {
  __shared__ __attribute__((aligned(1024))) f16 smem[G16<PW, PX>::LDS];
  int tv, tn;
  if (!a.tile(tv, tn)) return;
  const int v0 = tv * GM, n0 = tn * GM;
  f32x4 acc[4][4];
  f32x4 bias[4];
  float scale;
  logit_tile<PW, PX, BF>(a, v0, n0, smem, acc, bias, scale);
  const int lane = threadIdx.x & 63, q = lane >> 4, l15 = lane & 15;
  const int wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  float4* xch = reinterpret_cast<float4*>(smem);
  Stat st[4];
  int target[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) target[j] = row_target(a, n0 + wn * 64 + j * 16 + l15);
  // the maximum over the wave's 64 classes first, so that no lane's sum needs rescaling when they are joined
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    st[j] = Stat{-INFINITY, 0.f, 0.f, a.V};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        acc[i][j][r] = fmaf(acc[i][j][r], scale, bias[i][r]);
        st[j].m = fmaxf(st[j].m, acc[i][j][r]);
      }
  }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) st[j].m = fmaxf(st[j].m, __shfl_xor(st[j].m, o, 64));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + wn * 64 + j * 16 + l15;
    if (MORE) {
#pragma unroll
      for (int e = 15; e >= 0; --e) {
        const int v = v0 + wm * 64 + (e >> 2) * 16 + q * 4 + (e & 3);
        const float z = acc[e >> 2][j][e & 3];
        if (z == st[j].m) st[j].arg = v;
        if (v < a.V) st[j].z += z;
      }
    }
    const int hit = lane_class(target[j], v0);
    if (hit >= 0) {
      float z = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e == hit) z = acc[e >> 2][j][e & 3];
      zt[n] = z;  // a target lies in [0, V), its row counts
    }
    const float ref = st[j].m == -INFINITY ? 0.f : st[j].m;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[j].s += __builtin_amdgcn_exp2f(acc[i][j][r] - ref);
  }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      st[j].s += __shfl_xor(st[j].s, o, 64);
      if (MORE) {
        st[j].z += __shfl_xor(st[j].z, o, 64);
        st[j].arg = min(st[j].arg, __shfl_xor(st[j].arg, o, 64));
      }
    }
  if (wm == 1 && q == 0)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      xch[wn * 64 + j * 16 + l15] = make_float4(st[j].m, st[j].s, st[j].z, __int_as_float(st[j].arg));
  __syncthreads();
  if (wm == 0 && q == 0)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = wn * 64 + j * 16 + l15;
      const float4 o = xch[c];
      stat_join(st[j], Stat{o.x, o.y, o.z, __float_as_int(o.w)});
      if (n0 + c < a.rows())
        part[(int64_t)tv * a.N + n0 + c] = make_float4(st[j].m, st[j].s, st[j].z, __int_as_float(st[j].arg));
    }
}

// Per packed row, from its joined statistics: the maximum and the log2 of the sum, apart (next to a maximum of 2^24 and more
// the other one would vanish in their sum, and the probabilities with it); at its place in the call: loss (NaN for a target
// outside [0, V)) and arg-max.
struct CeRows {
  const float* zt;
  const int *target, *order, *exps;
  int N, V, tiles_v;
  float smooth;
  float2* lse;
  float* rowloss;
  int64_t* pred;
};
__device__ __forceinline__ float row_out(const CeRows& k, int n, const Stat& s) {
  const float m = s.m == -INFINITY ? 0.f : s.m, l = log2f(s.s);
  k.lse[n] = make_float2(m, l);
  float loss = NAN;
  if (k.target[n] >= 0) {
    const float d = m - k.zt[n];
    loss = LN2 * (l + (k.smooth > 0.f ? (1.f - k.smooth) * d + k.smooth * (m - s.z / (float)k.V) : d));
  }
  const int at = k.order[n];
  k.rowloss[at] = loss;
  if (k.pred) k.pred[at] = s.arg < k.V ? s.arg : 0;
  return loss;
}
__device__ __forceinline__ Stat row_join(const CeRows& k, const float4* part, int n, int t0, int t1) {
  Stat s{-INFINITY, 0.f, 0.f, k.V};
#pragma unroll 4
  for (int t = t0; t < t1; ++t) {
    const float4 o = part[(int64_t)t * k.N + n];
    stat_join(s, Stat{o.x, o.y, o.z, __float_as_int(o.w)});
  }
  return s;
}

// 8 rows x 32 runs of tiles per block
__global__ __launch_bounds__(256) void ce_join_kernel(CeRows k, const float4* __restrict__ part) {
  __shared__ Stat sm[32][8];
  const int e = threadIdx.x & 7, run = threadIdx.x >> 3;
  const int n = blockIdx.x * 8 + e, per = (k.tiles_v + 31) / 32, rows = k.exps[2];
  if (blockIdx.x * 8 >= rows) return;
  Stat s{-INFINITY, 0.f, 0.f, k.V};
  if (n < rows) s = row_join(k, part, n, run * per, min(k.tiles_v, (run + 1) * per));
  sm[run][e] = s;
  __syncthreads();
#pragma unroll
  for (int w = 16; w > 1; w >>= 1) {
    if (run < w) {
      stat_join(s, sm[run + w][e]);
      sm[run][e] = s;
    }
    __syncthreads();
  }
  if (run == 0 && n < rows) {
    stat_join(s, sm[1][e]);
    row_out(k, n, s);
  }
}

// loss (nullable) = sum of the row losses (mean: divided by the counted rows, or by 1 if there are none), total[0] = that
// count; correct (nullable) = counted rows whose arg-max is the target.  One block.
// JOIN: the rows' statistics have not been joined yet (few rows and tiles: one launch instead of two).
template <bool JOIN>
__global__ __launch_bounds__(1024) void ce_total_kernel(CeRows k, const float4* __restrict__ part, int mean,
                                                        float* __restrict__ loss, float* __restrict__ total,
                                                        int* __restrict__ correct) {
  __shared__ double sd[16];
  __shared__ int sk[16];
  double a = 0.0;
  int hits = 0;
  const int rows = k.exps[2];
  for (int n = threadIdx.x; n < rows; n += 1024) {
    const int at = k.order[n];
    a += (double)(JOIN ? row_out(k, n, row_join(k, part, n, 0, k.tiles_v)) : k.rowloss[at]);
    if (k.pred && k.pred[at] == k.target[n]) ++hits;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    hits += __shfl_xor(hits, o, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    sd[threadIdx.x >> 6] = a;
    sk[threadIdx.x >> 6] = hits;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) {
      a += sd[i];
      hits += sk[i];
    }
    if (loss) *loss = (float)(mean ? a / (double)max(rows, 1) : a);
    total[0] = (float)rows;
    if (correct) *correct = hits;
  }
}

// ---- backward ------------------------------------------------------------------------------------------------------
// Per-row upstream gradients: rs[k] = weight of packed row k relative to the largest one, fac[0] = that largest weight, fac[1] =
// 0.  If a weight other than 0 lies more than 2^16 below the largest, rs[k] = the weight itself, fac[0] = fac[1] = 1: d is kept
// without the weights, which dx takes on as it is written, and dW in its product.
__global__ __launch_bounds__(1024) void ce_weights_kernel(const float* __restrict__ g, const int* __restrict__ order,
                                                          const int* __restrict__ exps, float* __restrict__ rs,
                                                          float* __restrict__ fac) {
  __shared__ float sm[16];
  const int rows = exps[2];
  float big = 0.f;
  for (int k = threadIdx.x; k < rows; k += 1024) big = fmaxf(big, finite_mag(g[order[k]]));
  big = wave_max(big);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = big;
  __syncthreads();
  big = sm[0];
  for (int i = 1; i < 16; ++i) big = fmaxf(big, sm[i]);
  if (!(big > 0.f)) big = 1.f;
  int own = 0;
  for (int k = threadIdx.x; k < rows; k += 1024) {
    const float w = fabsf(g[order[k]]);
    own |= w > 0.f && w < ldexpf(big, -OWN_SCALE);
  }
  own = __syncthreads_or(own);
  for (int k = threadIdx.x; k < rows; k += 1024) rs[k] = own ? g[order[k]] : g[order[k]] / big;
  if (threadIdx.x == 0) {
    fac[0] = own ? 1.f : big;
    fac[1] = own ? 1.f : 0.f;
  }
}

constexpr float D_SCALE = 32768.f;  // of d's fp16 terms, and of dbpart

// The largest row weight: what ce_weights_kernel found, or for a mean or sum the upstream gradient itself.
struct CeFac {
  const float* fac;    // per-row weights
  const float* g;      // else the one gradient,
  const float* total;  // of a mean (the counted rows) or, null, of a sum
  // whether d is kept without the rows' weights
  __device__ __forceinline__ bool own() const { return fac && fac[1] != 0.f; }
  __device__ __forceinline__ float get() const { return fac ? fac[0] : total ? g[0] / fmaxf(total[0], 1.f) : g[0]; }
};

__device__ __forceinline__ float row16_sum(float v) {  // over the 16 lanes of a DPP row
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, true));
  return v;
}

// fac 2^e as a factor of [1/2, 1) and an exponent: applied one after the other, neither underflows where their product, a
// gradient of tiny operands, does not.
struct Factor {
  float f;
  int e;
  __device__ __forceinline__ Factor(float fac, int exp) : f(__builtin_amdgcn_frexp_mantf(fac)), e(exp + __builtin_amdgcn_frexp_expf(fac)) {}
  __device__ __forceinline__ float operator()(float v) const { return ldexpf(v * f, e); }
};

template <typename T>
__device__ __forceinline__ void bias_out(T* db, float s, const CeFac& fac, int add) {
  *db = from_f32<T>((add ? to_f32(*db) : 0.f) + Factor(fac.get(), -15)(s));  // of D_SCALE
}

// 8192 x 1024 against a piece of 8192 classes: 154 - 166 us, 0.83 - 0.89 PFLOP/s; the tile leaves through LDS in rows of 256 bytes.
//
// One 128 x 128 tile of d for the classes [vbeg, vbeg + vcols), as dn[n][vcols] in PD terms scaled by 2^15, and its column
// sums dbpart[tile n][v] (db itself where there is one row tile).
template <int PW, int PX, int PD>
__global__ __launch_bounds__(G_THREADS, 2) void ce_grad_kernel(CeArgs a, const float2* __restrict__ lse,
                                                               const float* __restrict__ rs, float smooth, int vbeg,
                                                               int vcols, f16* __restrict__ dn,
                                                               float* __restrict__ dbpart, CeFac fac, void* db, int add) {
  __shared__ __attribute__((aligned(1024))) f16 smem[G16<PW, PX>::LDS];
  __shared__ float sb[2][GM];
  int tv, tn;
  if (!a.tile(tv, tn)) return;
  const int v0 = vbeg + tv * GM, n0 = tn * GM;
  f32x4 acc[4][4];
  f32x4 bias[4];
  float scale;
  logit_tile<PW, PX>(a, v0, n0, smem, acc, bias, scale);
  const int lane = threadIdx.x & 63, q = lane >> 4, l15 = lane & 15;
  const int wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
  const float each = smooth / (float)a.V * D_SCALE;
  float col[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) col[i][r] = 0.f;
  const int64_t plane = (int64_t)a.N * vcols;
  const int rows = a.rows();
  int target[4];
  float weight[4], top[4], low[4];  // 2^((z - top) + low) is the scaled probability
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + wn * 64 + j * 16 + l15;
    target[j] = row_target(a, n);
    const float2 s = lse[max(min(n, rows - 1), 0)];
    top[j] = s.x;
    low[j] = 15.f - s.y;
    weight[j] = n < rows ? 1.f : 0.f;
    if (target[j] < 0) low[j] = NAN;
  }
  if (rs)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + wn * 64 + j * 16 + l15;
      if (n < rows) weight[j] = rs[n];
    }
  const bool own = fac.own();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float m = top[j], l = low[j];
    const bool live = weight[j] != 0.f;  // a row without weight vanishes whatever it holds
    const float w = own ? 1.f : weight[j], wb = own ? weight[j] : 1.f;  // of d and, beyond that, of the bias's gradient
    const int hit = lane_class(target[j], v0);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        acc[i][j][r] = __builtin_amdgcn_exp2f((fmaf(acc[i][j][r], scale, bias[i][r]) - m) + l);
    if (smooth > 0.f)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (v0 + wm * 64 + i * 16 + q * 4 + r < a.V) acc[i][j][r] -= each;
    if (hit >= 0)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e == hit) acc[e >> 2][j][e & 3] -= (1.f - smooth) * D_SCALE;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        acc[i][j][r] = live ? acc[i][j][r] * w : 0.f;
        col[i][r] = fmaf(acc[i][j][r], wb, col[i][r]);
      }
  }
  float* tile = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    Tile16<4>::put(acc, half, tile);
    __syncthreads();
    F8 d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) d[u] = Tile16<4>::get(tile, (threadIdx.x >> 4) + u * 16, (threadIdx.x & 15) * 8);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = threadIdx.x + u * G_THREADS, n = n0 + half * 64 + (e >> 4);
      f16x8 hi, lo;
      f16_split8(d[u], hi, lo);
      if (n < rows) {
        f16* o = dn + (int64_t)n * vcols + (v0 - vbeg + (e & 15) * 8);
        *reinterpret_cast<f16x8*>(o) = hi;
        if (PD == 2) *reinterpret_cast<f16x8*>(o + plane) = lo;
      }
    }
    __syncthreads();
  }
  if (dbpart) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float s = row16_sum(col[i][r]);
        if (l15 == 0) sb[wn][wm * 64 + i * 16 + q * 4 + r] = s;
      }
    __syncthreads();
    const int v = v0 + threadIdx.x;
    if (threadIdx.x < GM && v < a.V) {
      const float s = sb[0][threadIdx.x] + sb[1][threadIdx.x];
      if (a.N > GM) dbpart[(int64_t)tn * a.V + v] = s;
      else if (a.db_bf16) bias_out((bf16*)db + v, s, fac, add);  // the only row tile
      else bias_out((float*)db + v, s, fac, add);
    }
  }
}

// db[v] (+)= fac sum over the row tiles of dbpart[tile][v], up to 32768 of them and therefore in doubles
template <typename T>
__global__ __launch_bounds__(256) void ce_bias_kernel(const float* __restrict__ dbpart, const int* __restrict__ exps, int V,
                                                      CeFac fac, int add, T* __restrict__ db) {
  const int tiles = max(1, (exps[2] + GM - 1) / GM);
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= V) return;
  double s = 0.0;
#pragma unroll 4
  for (int t = 0; t < tiles; ++t) s += (double)dbpart[(int64_t)t * V + v];
  bias_out(db + v, (float)s, fac, add);
}

// slices of a reduction of length k (a multiple of 64) over `tiles` output tiles: two workgroups per CU where the slices
// are at least 1024 long, else one, down to 256 elements; at most 16
__host__ __device__ inline void slices(int tiles, int k, int& s, int& per) {
  if (tiles < 1) tiles = 1;
  int want = 512 / tiles;
  if (want > 1 && k / want < 1024) want = 256 / tiles;
  const int most = k / 256 < 16 ? k / 256 : 16;
  if (want > most) want = most;
  if (want < 1) want = 1;
  per = ((k + want - 1) / want + 63) / 64 * 64;
  s = (k + per - 1) / per;
}

// out[m][c] = factor * sum over the reduction of (row side)[m] (column side)[c]: dx = d W and dW = d^T x.  Operands that lie
// along the reduction the wrong way are read from LDS with transposing reads, so nothing is stored twice.  137 - 147 and
// 132 - 140 us by card for a piece of 8192 classes of 8192 x 1024 (1.0 PFLOP/s); fp32 dW of bf16 rows, d in two terms: 88 - 100 us
// per piece of 8192 classes at K = 768 and three quarters of 4096 rows.
struct MmArgs {
  Op16 c, m;                   // column side (W or x, COL) and row side (d: ROW for dx, COL for dW), at their corners
  int M, Nn, k;                // rows and columns of the result, reduction length of dx (a multiple of 64)
  int tiles_m, tiles_n, splits;
  int piece;                   // dx: classes of a whole piece, whose slices every piece takes
  const int* order;            // dx: where its packed rows go
  float* part;                 // [splits][M, of dx: rows that count][pitch], or null: write out
  int pitch;                   // of part (dx: a multiple of 8) or out
  int add;                     // add to what part / out hold
  void* out;                   // [M][Nn]
  CeFac fac;
  const int* exps;             // exps[2] = rows that count: rows of dx that are worked, reduction length of dW
  int which;                   // whose scale exponent the column side carries
  const int* own;              // the column side's scale exponents along the reduction, for exps[3 + which]
  const float* rs;             // the rows' weights, for fac.own()
};

// whether the product goes by own_product: the column side has scales of its own along the reduction, or is to take the
// rows' weights (dW)
__device__ __forceinline__ bool mm_own(const CeFac& fac, const int* exps, int which) {
  return exps[3 + which] || (which == 0 && fac.own());
}
__device__ __forceinline__ Factor mm_factor(const CeFac& fac, const int* exps, int which) {
  return Factor(fac.get(), mm_own(fac, exps, which) ? 0 : -15 - exps[which]);
}

// The product where the column side's scales, or for dW the rows' weights, differ along the reduction (some rows of x or of W, or
// some upstream gradients, lie more than 2^16 below the largest): its values as they are, on the fp32 matrix instructions,
// whose range holds all of them.  Operands come straight from memory: a step of 4096 x 768 x 16384 in bf16 takes 3.2 ms
// (rows) or 4.1 (classes) instead of 0.58; data with such rows is not what training usually meets.
template <int PC, int PM, int KM>
__device__ __forceinline__ void own_product(f32x4 (&acc)[4][4], const Op16& c, const Op16& m, const int* own, const float* rs,
                                            int k0, int k1) {
  const int lane = threadIdx.x & 63, q = lane >> 4, l15 = lane & 15;
  const int wave = threadIdx.x >> 6, wc = wave >> 1, wr = wave & 1;
  for (int k = k0; k < k1; k += 4) {
    const int kk = k + q;
    const bool on = kk < c.n;  // the reduction's true length
    const int e = on ? -own[kk] : 0;
    const float w = on && rs ? rs[kk] : 1.f;
    float fc[4], fm[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = c.side + (wc * 4 + i) * 16 + l15;
      fc[i] = 0.f;
      if (on && col < c.ld) {
        const f16* p = c.p + (int64_t)kk * c.ld + col;
        fc[i] = ldexpf(PC == 2 ? (float)p[0] + (float)p[c.plane] : (float)p[0], e);
      }
      const int row = (wr * 4 + i) * 16 + l15;
      fm[i] = 0.f;
      if (on && (KM == ROW ? row < m.n : m.side + row < m.ld)) {
        const f16* p = KM == ROW ? m.p + (int64_t)row * m.ld + kk : m.p + (int64_t)kk * m.ld + m.side + row;
        fm[i] = (PM == 2 ? (float)p[0] + (float)p[m.plane] : (float)p[0]) * (1.f / D_SCALE) * w;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fc[i], fm[j], acc[i][j], 0, 0, 0);
  }
}

template <int PC, int PM, int KM, typename T>
__global__ __launch_bounds__(G_THREADS, 2) void ce_mm_kernel(MmArgs g) {
  typedef G16<PC, PM, COL, KM> G;
  __shared__ __attribute__((aligned(1024))) f16 smem[G::LDS];
  const int rows = g.exps[2];
  const int tiles_m = KM == ROW ? max(1, (rows + GM - 1) / GM) : g.tiles_m, tiles = tiles_m * g.tiles_n;
  int splits = g.splits, per = 0;
  if (KM == ROW && g.part) slices(tiles, g.piece, splits, per);  // by the rows that count
  int split = blockIdx.x / tiles, tm, tn;
  const bool idle = split >= splits;  // dx: behind the rows that count
  if (idle) {
    if (g.part) return;  // ce_dx_kernel writes their zeros
    const int id = blockIdx.x - tiles;
    tm = tiles_m + id / g.tiles_n;
    tn = id % g.tiles_n;
    split = 0;
  } else
    g16_tile(blockIdx.x, splits, tiles_m, g.tiles_n, split, tm, tn);
  const int m0 = tm * GM, n0 = tn * GM;
  f32x4 acc[4][4];
  G::zero(acc);
  const int klen = KM == ROW ? g.k : (rows + 63) / 64 * 64;
  if (KM == COL) per = ((klen + splits - 1) / splits + 63) / 64 * 64;
  else if (!g.part) per = klen;
  const int k0 = split * per, k1 = min(klen, k0 + per);
  Op16 c = g.c, m = g.m;
  c.side = n0;
  if (KM == ROW) {
    m.p += (int64_t)m0 * m.ld;
    m.n = rows - m0;
  } else {
    m.side = m0;
    m.n = c.n = rows;
  }
  if (!idle && rows > (KM == ROW ? m0 : 0)) {  // not where no row counts
    if (mm_own(g.fac, g.exps, g.which))
      own_product<PC, PM, KM>(acc, c, m, g.own, KM == COL && g.fac.own() ? g.rs : nullptr, k0, k1);
    else G::run(acc, c, m, k0, k1, smem);
  }
  const int lane = threadIdx.x & 63, q = lane >> 4, l15 = lane & 15;
  const int wave = threadIdx.x >> 6, wc = wave >> 1, wr = wave & 1;
  float* part = g.part ? g.part + (int64_t)split * (KM == ROW ? rows : g.M) * g.pitch : nullptr;
  if (!part) {
    const Factor f = mm_factor(g.fac, g.exps, g.which);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = f(acc[i][j][e]);
    if (KM == ROW && g.fac.own())
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = g.rs[max(min(m0 + wr * 64 + j * 16 + l15, rows - 1), 0)];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i][j] *= w;
      }
  }
  // dx: packed rows go to their places, those that do not count as zeros
  const int live = KM == ROW ? rows : g.M, end = KM == ROW && part ? rows : g.M;
  int64_t at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = m0 + wr * 64 + j * 16 + l15, r = min(row, g.M - 1);
    at[j] = (int64_t)(KM == ROW && !part ? g.order[r] : r) * g.pitch;
    if (row >= live)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Rows of any length: four results are one access of the result's own alignment, the last few of a row one by one.
  typedef f32x4 u32x4 __attribute__((aligned(4)));
  typedef bf16x4 u16x4 __attribute__((aligned(2)));
  // what is added to comes first: the stores could alias these loads and would hold them back
  if (g.add) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = n0 + wc * 64 + i * 16 + q * 4;
        if (col > g.pitch - 4) continue;
        const int64_t o = at[j] + col;
        if (part) acc[i][j] += *reinterpret_cast<const u32x4*>(part + o);
        else if constexpr (sizeof(T) == 4) acc[i][j] += *reinterpret_cast<const u32x4*>((const float*)g.out + o);
        else {
          const bf16x4 r = *reinterpret_cast<const u16x4*>((const bf16*)g.out + o);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] += (float)r[e];
        }
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (m0 + wr * 64 + j * 16 + l15 >= end) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = n0 + wc * 64 + i * 16 + q * 4;  // four results of one row
      const int64_t o = at[j] + col;
      const f32x4 v = acc[i][j];
      if (col <= g.pitch - 4) {
        if (part) *reinterpret_cast<u32x4*>(part + o) = v;
        else if constexpr (sizeof(T) == 4) *reinterpret_cast<u32x4*>((float*)g.out + o) = v;
        else *reinterpret_cast<u16x4*>((bf16*)g.out + o) = bf16x4{(bf16)v[0], (bf16)v[1], (bf16)v[2], (bf16)v[3]};
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e) {
          if (col + e >= g.pitch) break;
          if (part) part[o + e] = g.add ? part[o + e] + v[e] : v[e];
          else {
            T* out = (T*)g.out + o + e;
            *out = from_f32<T>(g.add ? to_f32(*out) + v[e] : v[e]);
          }
        }
      }
    }
  }
}

// dx[order[r]] = factor * sum over the slices, in order, of packed row r; zeros for rows that do not count.  A wave per row and
// 512 columns.
template <typename T>
__global__ __launch_bounds__(256) void ce_dx_kernel(const float* __restrict__ part, int piece, int N, int K, CeFac fac,
                                                    const int* __restrict__ exps, const int* __restrict__ order,
                                                    const float* __restrict__ rs, int vec, T* __restrict__ out) {
  const int per = (K + 511) / 512;
  const int rows = exps[2];
  int splits, len;
  slices(max(1, (rows + GM - 1) / GM) * ((K + GM - 1) / GM), piece, splits, len);
  const int pitch = (K + 7) / 8 * 8;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), n = (int64_t)rows * pitch;
  const int r = (int)(unit / per), c0 = (int)(unit - (int64_t)r * per) * 512 + (threadIdx.x & 63) * (vec ? 8 : 1);
  if (r >= N) return;
  const bool live = r < rows;
  const Factor f = mm_factor(fac, exps, 1);
  const float w = live && fac.own() ? rs[r] : 1.f;
  const float* p = part + (int64_t)r * pitch;
  T* o = out + (int64_t)order[r] * K;
  if (vec) {
    if (c0 >= K) return;
    F8 s;
#pragma unroll
    for (int e = 0; e < 8; ++e) s.v[e] = 0.f;
    if (live)
#pragma unroll 4
      for (int k = 0; k < splits; ++k) {
        const F8 v = load8(p + k * n + c0);
#pragma unroll
        for (int e = 0; e < 8; ++e) s.v[e] += v.v[e];
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) s.v[e] = f(s.v[e]) * w;
    if (!live)
#pragma unroll
      for (int e = 0; e < 8; ++e) s.v[e] = 0.f;
    store8(o + c0, s);
  } else {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.f;
    if (live)
      for (int k = 0; k < splits; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += p[k * n + min(c0 + e * 64, K - 1)];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e * 64 < K) o[c0 + e * 64] = from_f32<T>(live ? f(s[e]) * w : 0.f);
  }
}

// out (+)= factor * sum over the slices, in order
template <typename T>
__global__ __launch_bounds__(256) void ce_reduce_kernel(const float* __restrict__ part, int slices, int64_t n,
                                                        CeFac fac, const int* __restrict__ exps, int which, int add, T* __restrict__ out) {
  const Factor f = mm_factor(fac, exps, which);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
#pragma unroll 4
    for (int k = 0; k < slices; ++k) s += part[k * n + i];
    s = f(s);
    out[i] = from_f32<T>(add ? to_f32(out[i]) + s : s);
  }
}

// ---- host side: shapes and workspaces ---------------------------------------------------------------------------------
int pad64(int v) { return (v + 63) / 64 * 64; }
int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

struct Plan {
  int ld, px, pw;              // row length and terms of the packed operands
  int pdx, pdw, pd;            // terms of d for dx and dW, and the larger of the two
  int piece, pieces;           // classes of a piece
  int sx, sw;                  // slices of the reductions of dx (per piece, if all rows count) and dW
  // forward workspace (saved for backward): packed x, packed W, exponents and count, bias, row list, lse, total, scales
  int64_t o_xp, o_wp, o_exps, o_bl, o_order, o_target, o_lse, o_total, o_ex, o_ew, saved;
  // forward scratch
  int64_t f_amax, f_part, f_zt, f_xmax, f_wmax, fwd;
  // backward scratch
  int64_t b_rs, b_fac, b_dn, b_db, b_px, b_pw, bwd;
};

Plan make_plan(int xf32, int wf32, int N, int V, int K) {
  Plan p;
  p.ld = pad64(K);
  p.px = xf32 ? 2 : 1;
  p.pw = xf32 ? 2 : 1;
  p.pdx = xf32 ? 2 : 1;
  p.pdw = wf32 ? 2 : 1;
  p.pd = p.pdx > p.pdw ? p.pdx : p.pdw;
  // a piece of d stays below 128 MiB, half of the last-level cache
  int64_t cols = (128ll << 20) / ((int64_t)N * 2 * p.pd) / GM * GM;
  if (cols < GM) cols = GM;
  const int all = (V + GM - 1) / GM * GM;
  p.pieces = (int)((all + cols - 1) / cols);
  p.piece = (int)(((all / GM + p.pieces - 1) / p.pieces) * GM);
  p.pieces = (all + p.piece - 1) / p.piece;
  const int tn = ceil_div(N, GM), tk = ceil_div(K, GM);
  int per;
  slices(tn * tk, p.piece, p.sx, per);
  slices((p.piece / GM) * tk, pad64(N), p.sw, per);
  int64_t o = 0;
  auto take = [&](int64_t bytes) {
    const int64_t at = o;
    o += up256(bytes);
    return at;
  };
  p.o_xp = take((int64_t)p.px * N * p.ld * 2);
  p.o_wp = take((int64_t)p.pw * V * p.ld * 2);
  p.o_exps = take(32);
  p.o_bl = take((int64_t)all * 4);
  p.o_order = take((int64_t)N * 4);
  p.o_target = take((int64_t)N * 4);
  p.o_lse = take((int64_t)N * 8);
  p.o_total = take(16);
  p.o_ex = take((int64_t)N * 4);
  p.o_ew = take((int64_t)V * 4);
  p.saved = o;
  o = 0;
  p.f_amax = take(2 * AMAX_MOST * 4);
  p.f_part = take((int64_t)ceil_div(V, GM) * N * 16);
  p.f_zt = take((int64_t)N * 4);
  p.f_xmax = take((int64_t)N * 4);
  p.f_wmax = take((int64_t)V * 4);
  p.fwd = o;
  o = 0;
  p.b_rs = take((int64_t)N * 4);
  p.b_fac = take(16);
  p.b_dn = take((int64_t)p.pd * N * p.piece * 2);
  p.b_db = take((int64_t)tn * V * 4);
  // dx in slices: fewer rows that count take more of them, s <= 512 / (row tiles x tk), so s x rows stays below this
  const int64_t most = 512 * GM / tk > N ? 512 * GM / tk : N;
  p.b_px = (p.pieces > 1 || p.sx > 1) ? take((most < 16ll * N ? most : 16ll * N) * ((K + 7) / 8 * 8) * 4) : -1;
  p.b_pw = p.sw > 1 ? take((int64_t)p.sw * p.piece * K * 4) : -1;
  p.bwd = o;
  return p;
}

int check_ce(const char* who, int xdtype, int wdtype, int N, int V, int K, float smooth) {
  for (int d : {xdtype, wdtype})
    if (d != VC_F32 && d != VC_BF16) {
      vc_set_error("%s: unsupported dtype %d", who, d);
      return VC_ERR_DTYPE;
    }
  VC_CHECK_ARG(xdtype == VC_BF16 || wdtype == VC_F32, "%s: fp32 rows need fp32 weights", who);
  VC_CHECK_SHAPE(N > 0 && V > 0 && K > 0, "%s: empty shape N=%d V=%d K=%d", who, N, V, K);
  // 128 rows of an operand have to fit a 32-bit buffer descriptor, tiles a grid
  VC_CHECK_SHAPE(K <= (1 << 20) && N <= (1 << 22) && V <= (1 << 22), "%s: N, V or K too large (at most 2^22, 2^22, 2^20)",
                 who);
  // a launch holds fewer than 2^32 threads
  VC_CHECK_SHAPE((int64_t)ceil_div(N, GM) * ceil_div(V, GM) < (1 << 24),
                 "%s: %d rows against %d classes are more than 2^24 tiles of logits", who, N, V);
  VC_CHECK_SHAPE(((int64_t)N + V) * ceil_div(K, 512) < (1 << 26) - 8,
                 "%s: %d rows and %d classes of %d are more than 2^26 pieces of 512 to pack", who, N, V, K);
  VC_CHECK_ARG(smooth >= 0.f && smooth <= 1.f, "%s: label smoothing %g outside [0, 1]", who, (double)smooth);
  return VC_OK;
}

template <typename TX, typename TW>
void pack_go(const Plan& p, const void* x, const void* w, const void* bias, int N, int V, int K, const int64_t* target, int64_t ignore,
             float* rowloss, int64_t* pred, char* saved, char* ws, hipStream_t st) {
  float *amax = (float*)(ws + p.f_amax), *xmax = (float*)(ws + p.f_xmax), *wmax = (float*)(ws + p.f_wmax);
  const int per = ceil_div(p.ld, 512);
  const int xb = (int)ceil_div64((int64_t)N * per, 4), wb = (int)ceil_div64((int64_t)V * per, 4);
  auto blocks = [](int64_t elems) {  // of one vector per thread where that is enough blocks
    const int64_t b = ceil_div64(elems, 2048);
    return (int)(b < AMAX_MOST ? b : AMAX_MOST);
  };
  const int xa = blocks((int64_t)N * K), wa = blocks((int64_t)V * K);
  hipLaunchKernelGGL((ce_amax_kernel<TX, TW>), dim3(xa + wa + 1), dim3(256), 0, st, (const TX*)x, (const TW*)w, N, V, K,
                     target, ignore, amax, xa, RowList{(int*)(saved + p.o_order), (int*)(saved + p.o_target), (int*)(saved + p.o_exps) + 2},
                     rowloss, pred, xmax, wmax);
  hipLaunchKernelGGL((ce_pack_kernel<TX, TW>), dim3(xb + wb), dim3(256), 0, st, (const TX*)x, (const TW*)w, N, V, K, p.ld,
                     p.px, p.pw, (const int*)(saved + p.o_order), amax, (f16*)(saved + p.o_xp), (f16*)(saved + p.o_wp),
                     (int*)(saved + p.o_exps), xb, xa, wa, (const TW*)bias, (float*)(saved + p.o_bl), xmax, wmax,
                     (int*)(saved + p.o_ex), (int*)(saved + p.o_ew));
}

template <int PC, int PM, int KM>
void mm_go(const MmArgs& g, int out_bf16, hipStream_t st) {
  int blocks = g.tiles_m * g.tiles_n * g.splits;
  if (KM == ROW && g.part) blocks = max(g.tiles_m * g.tiles_n, 512);  // more than one slice only up to 512 workgroups
  const dim3 grid(blocks), blk(G_THREADS);
  if (out_bf16) hipLaunchKernelGGL((ce_mm_kernel<PC, PM, KM, bf16>), grid, blk, 0, st, g);
  else hipLaunchKernelGGL((ce_mm_kernel<PC, PM, KM, float>), grid, blk, 0, st, g);
}
template <int PW, int PX, bool BF = false>
void stats_go(const CeArgs& a, bool more, float4* part, float* zt, hipStream_t st) {
  const dim3 grid(a.tiles_v * ceil_div(a.N, GM)), blk(G_THREADS);
  if (more) hipLaunchKernelGGL((ce_stats_kernel<PW, PX, true, BF>), grid, blk, 0, st, a, part, zt);
  else hipLaunchKernelGGL((ce_stats_kernel<PW, PX, false, BF>), grid, blk, 0, st, a, part, zt);
}
template <int PW, int PX, int PD>
void grad_go(const CeArgs& a, const float2* lse, const float* rs, float smooth, int vbeg, int vcols, f16* dn, float* dbp,
             const CeFac& fac, void* db, int add, hipStream_t st) {
  hipLaunchKernelGGL((ce_grad_kernel<PW, PX, PD>), dim3(a.tiles_v * ceil_div(a.N, GM)), dim3(G_THREADS), 0, st, a, lse, rs, smooth,
                     vbeg, vcols, dn, dbp, fac, db, add);
}
template <int KM>
void mm_terms(int pc, int pm, const MmArgs& g, int out_bf16, hipStream_t st) {
  if (pm == 1) mm_go<1, 1, KM>(g, out_bf16, st);
  else if (pc == 1) mm_go<1, 2, KM>(g, out_bf16, st);
  else mm_go<2, 2, KM>(g, out_bf16, st);
}
void dx_go(const float* part, int piece, int N, int K, const CeFac& fac, const int* exps, const int* order, const float* rs,
           void* dx, int out_bf16, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div64((int64_t)N * ceil_div(K, 512), 4));
  const int vec = K % 8 == 0 && ((uintptr_t)dx & 15) == 0;
  if (out_bf16) hipLaunchKernelGGL((ce_dx_kernel<bf16>), grid, dim3(256), 0, st, part, piece, N, K, fac, exps, order, rs, vec, (bf16*)dx);
  else hipLaunchKernelGGL((ce_dx_kernel<float>), grid, dim3(256), 0, st, part, piece, N, K, fac, exps, order, rs, vec, (float*)dx);
}
void reduce_go(const float* part, int slices, int64_t n, const CeFac& fac, const int* exps, int which, int add, void* out,
               int out_bf16, hipStream_t st) {
  const int grid = (int)(ceil_div64(n, 256) < 4096 ? ceil_div64(n, 256) : 4096);
  if (out_bf16)
    hipLaunchKernelGGL((ce_reduce_kernel<bf16>), dim3(grid), dim3(256), 0, st, part, slices, n, fac, exps, which, add, (bf16*)out);
  else
    hipLaunchKernelGGL((ce_reduce_kernel<float>), dim3(grid), dim3(256), 0, st, part, slices, n, fac, exps, which, add, (float*)out);
}

}  // namespace

extern "C" {

int64_t vc_linear_ce_bytes(int what, int xdtype, int wdtype, int N, int V, int K) {
  if (check_ce("vc_linear_ce_bytes", xdtype, wdtype, N, V, K, 0.f) != VC_OK) return -1;
  const Plan p = make_plan(xdtype == VC_F32, wdtype == VC_F32, N, V, K);
  return what == 0 ? p.saved : what == 1 ? p.fwd : what == 2 ? p.bwd : what == 4 ? p.fwd + p.saved : -1;
}

int vc_linear_ce_fwd(int xdtype, int wdtype, const void* x, const void* w, const void* bias, const int64_t* target,
                     int64_t ignore_index, float smoothing, int mean, float* row_loss, float* loss, int64_t* pred,
                     int* correct, void* saved, void* workspace, int N, int V, int K, hipStream_t stream) {
  const int rc = check_ce("vc_linear_ce_fwd", xdtype, wdtype, N, V, K, smoothing);
  if (rc != VC_OK) return rc;
  VC_CHECK_ARG(x && w && target && row_loss && workspace, "vc_linear_ce_fwd: null pointer");
  VC_CHECK_ARG(loss || !mean, "vc_linear_ce_fwd: a mean without its place");
  VC_CHECK_ARG(!correct || pred, "vc_linear_ce_fwd: the count of correct rows needs pred");
  VC_CHECK_ARG((((uintptr_t)saved | (uintptr_t)workspace) & 255) == 0, "vc_linear_ce_fwd: buffers must be 256-byte aligned");
  const Plan p = make_plan(xdtype == VC_F32, wdtype == VC_F32, N, V, K);
  char *ws = (char*)workspace, *sv = saved ? (char*)saved : ws + p.fwd;
  const bool raw = !saved && xdtype == VC_BF16 && wdtype == VC_BF16 && K % 64 == 0 && ((uintptr_t)w & 15) == 0;
  const RowList list{(int*)(sv + p.o_order), (int*)(sv + p.o_target), (int*)(sv + p.o_exps) + 2};
  if (raw) {
    hipLaunchKernelGGL(ce_list_kernel, dim3(1), dim3(256), 0, stream, target, ignore_index, N, V, list, row_loss, pred);
    const int64_t units = (int64_t)N * (K / 8), most = units > V ? units : V;
    hipLaunchKernelGGL(ce_copy_kernel, dim3((unsigned)(ceil_div64(most, 256) < 2048 ? ceil_div64(most, 256) : 2048)), dim3(256), 0,
                       stream, (const bf16*)x, V, K, list.order, (bf16*)(sv + p.o_xp), (int*)(sv + p.o_exps), (const bf16*)bias,
                       (float*)(sv + p.o_bl));
  } else if (xdtype == VC_F32) pack_go<float, float>(p, x, w, bias, N, V, K, target, ignore_index, row_loss, pred, sv, ws, stream);
  else if (wdtype == VC_F32) pack_go<bf16, float>(p, x, w, bias, N, V, K, target, ignore_index, row_loss, pred, sv, ws, stream);
  else pack_go<bf16, bf16>(p, x, w, bias, N, V, K, target, ignore_index, row_loss, pred, sv, ws, stream);
  CeArgs a{raw ? (const f16*)w : (const f16*)(sv + p.o_wp), (const f16*)(sv + p.o_xp), (const float*)(sv + p.o_bl),
           list.target, (const int*)(sv + p.o_exps), (const int*)(sv + p.o_ex), (const int*)(sv + p.o_ew), N, V, K, p.ld,
           wdtype == VC_BF16, ceil_div(V, GM)};
  float4* part = (float4*)(ws + p.f_part);
  float* zt = (float*)(ws + p.f_zt);
  const bool more = smoothing > 0.f || pred;
  if (raw) stats_go<1, 1, true>(a, more, part, zt, stream);
  else if (p.pw == 2) stats_go<2, 2>(a, more, part, zt, stream);
  else stats_go<1, 1>(a, more, part, zt, stream);
  const CeRows rows{zt, a.target, (const int*)(sv + p.o_order), a.exps, N, V, a.tiles_v, smoothing, (float2*)(sv + p.o_lse), row_loss, pred};
  float* total = (float*)(sv + p.o_total);
  const bool sums = loss || correct;
  if (sums && N <= 1024 && a.tiles_v <= 16) {
    hipLaunchKernelGGL(ce_total_kernel<true>, dim3(1), dim3(1024), 0, stream, rows, part, mean, loss, total, correct);
  } else {
    hipLaunchKernelGGL(ce_join_kernel, dim3(ceil_div(N, 8)), dim3(256), 0, stream, rows, part);
    if (sums)
      hipLaunchKernelGGL(ce_total_kernel<false>, dim3(1), dim3(1024), 0, stream, rows, part, mean, loss, total, correct);
  }
  VC_LAUNCH_CHECK("vc_linear_ce_fwd");
  return VC_OK;
}

int vc_linear_ce_bwd(int xdtype, int wdtype, float smoothing, int mean,
                     int per_row, const float* dloss, const void* saved, void* dx, void* dw, void* db,
                     void* workspace, int accumulate, int N, int V, int K, hipStream_t stream) {
  const int rc = check_ce("vc_linear_ce_bwd", xdtype, wdtype, N, V, K, smoothing);
  if (rc != VC_OK) return rc;
  VC_CHECK_ARG(dloss && saved && workspace, "vc_linear_ce_bwd: null pointer");
  VC_CHECK_ARG(!(mean && per_row), "vc_linear_ce_bwd: a mean has one upstream gradient");
  VC_CHECK_ARG((((uintptr_t)saved | (uintptr_t)workspace) & 255) == 0, "vc_linear_ce_bwd: buffers must be 256-byte aligned");
  if (!dx && !dw && !db) return VC_OK;
  const Plan p = make_plan(xdtype == VC_F32, wdtype == VC_F32, N, V, K);
  const char* sv = (const char*)saved;
  char* ws = (char*)workspace;
  const f16 *xp = (const f16*)(sv + p.o_xp), *wp = (const f16*)(sv + p.o_wp);
  f16* dn = (f16*)(ws + p.b_dn);
  const int* exps = (const int*)(sv + p.o_exps);
  const int* order = (const int*)(sv + p.o_order);
  const int *ex = (const int*)(sv + p.o_ex), *ew = (const int*)(sv + p.o_ew);
  const float2* lse = (const float2*)(sv + p.o_lse);
  float *rs = (float*)(ws + p.b_rs), *big = (float*)(ws + p.b_fac), *dbp = (float*)(ws + p.b_db);
  const CeFac fac{per_row ? big : nullptr, dloss, mean ? (const float*)(sv + p.o_total) : nullptr};
  const int tn = ceil_div(N, GM), tk = ceil_div(K, GM);
  if (per_row) hipLaunchKernelGGL(ce_weights_kernel, dim3(1), dim3(1024), 0, stream, dloss, order, exps, rs, big);
  else rs = nullptr;
  for (int c = 0; c < p.pieces; ++c) {
    const int vbeg = c * p.piece;
    const int vcols = p.piece < ceil_div(V - vbeg, GM) * GM ? p.piece : ceil_div(V - vbeg, GM) * GM;
    CeArgs a{wp, xp, (const float*)(sv + p.o_bl), (const int*)(sv + p.o_target), exps, ex, ew, N, V, K, p.ld, wdtype == VC_BF16, vcols / GM};
    float* dbq = db ? dbp : nullptr;
    if (p.pw == 2) grad_go<2, 2, 2>(a, lse, rs, smoothing, vbeg, vcols, dn, dbq, fac, db, accumulate & 2, stream);
    else if (p.pd == 2) grad_go<1, 1, 2>(a, lse, rs, smoothing, vbeg, vcols, dn, dbq, fac, db, accumulate & 2, stream);
    else grad_go<1, 1, 1>(a, lse, rs, smoothing, vbeg, vcols, dn, dbq, fac, db, accumulate & 2, stream);
    const int rows = vcols < V - vbeg ? vcols : V - vbeg;
    MmArgs g{};
    g.Nn = g.pitch = K;
    g.tiles_n = tk;
    g.fac = fac;
    g.exps = exps;
    g.rs = rs;
    if (dx) {
      g.c = Op16{wp + (int64_t)vbeg * p.ld, (int64_t)V * p.ld, p.ld, rows, 0};
      g.m = Op16{dn, (int64_t)N * vcols, vcols, N, 0};
      g.M = N;
      g.order = order;
      g.k = pad64(rows);
      g.tiles_m = tn;
      g.splits = p.sx;
      g.piece = p.piece;
      g.part = p.b_px >= 0 ? (float*)(ws + p.b_px) : nullptr;
      g.add = c > 0;
      g.out = dx;
      g.which = 1;
      g.own = ew + vbeg;
      if (g.part) g.pitch = (K + 7) / 8 * 8;
      mm_terms<ROW>(p.pw, p.pdx, g, xdtype == VC_BF16, stream);
    }
    if (dw) {
      char* out = (char*)dw + (int64_t)vbeg * K * (wdtype == VC_BF16 ? 2 : 4);
      g.c = Op16{xp, (int64_t)N * p.ld, p.ld, N, 0};
      g.m = Op16{dn, (int64_t)N * vcols, vcols, N, 0};
      g.M = rows;
      g.k = pad64(N);
      g.tiles_m = ceil_div(rows, GM);
      g.splits = p.sw;
      g.pitch = K;
      g.part = p.b_pw >= 0 ? (float*)(ws + p.b_pw) : nullptr;
      g.add = g.part ? 0 : accumulate & 1;
      g.out = out;
      g.which = 0;
      g.own = ex;
      mm_terms<COL>(p.px, p.pdw, g, wdtype == VC_BF16, stream);
      if (g.part) reduce_go(g.part, p.sw, (int64_t)rows * K, fac, exps, 0, accumulate & 1, out, wdtype == VC_BF16, stream);
    }
  }
  if (dx && p.b_px >= 0)
    dx_go((const float*)(ws + p.b_px), p.piece, N, K, fac, exps, order, rs, dx, xdtype == VC_BF16, stream);
  if (db && tn > 1) {
    if (wdtype == VC_BF16)
      hipLaunchKernelGGL((ce_bias_kernel<bf16>), dim3(ceil_div(V, 256)), dim3(256), 0, stream, dbp, exps, V, fac,
                         accumulate & 2, (bf16*)db);
    else
      hipLaunchKernelGGL((ce_bias_kernel<float>), dim3(ceil_div(V, 256)), dim3(256), 0, stream, dbp, exps, V, fac,
                         accumulate & 2, (float*)db);
  }
  VC_LAUNCH_CHECK("vc_linear_ce_bwd");
  return VC_OK;
}

}  // extern "C"

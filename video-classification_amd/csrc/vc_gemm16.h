// 128 x 128 tiles of C[m][n] = sum_k A[m][k] B[n][k] on 16-bit floats with fp32 accumulation (v_mfma_f32_16x16x32_f16),
// either operand in one or two terms.
//
// Two terms: a value x, scaled by a power of two into fp16's range, is held as hi = fp16(x) and lo = fp16(x - hi), 22
// bits in all (an absolute floor of 2^-25 of the scaled unit), and the product is hi*hi + hi*lo + lo*hi: three MFMA of
// the 2.5 PFLOP/s kind per product against the 157 TFLOP/s of the fp32 matrix instructions, at fp32's accuracy.
//
// Layout: rows of `ld` elements, ld a multiple of 64 with zeros behind the last column, the second term one `plane`
// behind the first.  Four waves in a 2 x 2 grid own 64 x 64 each.  Two LDS stages of (PA + PB) x 128 rows x BK elements
// (BK = 64 for single terms, 32 otherwise, so at most 32 KiB a stage and two workgroups per CU); a stage's rows hold
// their 16-byte chunks permuted so that the 16 rows of a fragment read fall into 16 different 16-byte slots of the 256-byte
// bank row.  Stages are filled by LDS-DMA requests in opaque assembly (with the builtin the compiler waits for every
// outstanding request before each LDS read); rows beyond the matrix lie outside the buffer descriptor and read as zero.
#pragma once
#include "vc_common.h"

namespace {

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int GM = 128;       // rows of A and of B per tile
constexpr int G_THREADS = 256;

__device__ __forceinline__ void g16_dma(const i32x4_t& rs, unsigned lds_byte, unsigned voff, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(lds_byte), "v"(voff), "s"(rs), "s"(soff)
               : "memory");
}
__device__ __forceinline__ unsigned g16_lds(const void* p) {
  return (unsigned)(size_t)(__attribute__((address_space(3))) const void*)p;
}
// buffer descriptor of `rows` rows of ld elements at p (wave-uniform); the range check yields zeros behind them
__device__ __forceinline__ i32x4_t g16_desc(const f16* p, int rows, int ld) {
  const uint64_t u = (uint64_t)p;
  i32x4_t d;
  d[0] = __builtin_amdgcn_readfirstlane((int)u);
  d[1] = __builtin_amdgcn_readfirstlane((int)(u >> 32));
  d[2] = __builtin_amdgcn_readfirstlane((int)((unsigned)(rows < GM ? rows : GM) * (unsigned)ld * 2u));
  d[3] = 0x00020000;
  return d;
}

// A value of 22 bits in two fp16 terms.
__device__ __forceinline__ void f16_split(float v, f16& hi, f16& lo) {
  hi = (f16)v;
  lo = (f16)(v - (float)hi);
}

template <int PA, int PB>
struct G16 {
  static constexpr int BK = PA + PB == 2 ? 64 : 32;
  static constexpr int PLANE = GM * BK;              // elements of one plane of a stage
  static constexpr int STAGE = (PA + PB) * PLANE;
  static constexpr int LDS = 2 * STAGE;              // elements of shared memory
  static constexpr int CH = BK / 8;                  // 16-byte chunks of a row
  static constexpr int RPI = 64 / CH;                // rows one wave request fills
  static constexpr int REQ = GM / RPI / 4;           // requests per wave, plane and stage

  __device__ static __forceinline__ int swz(int row) { return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }

  // acc[i][j][r] += sum over k in [k0, k1) for A row wm*64 + i*16 + (lane>>4)*4 + r and B row wn*64 + j*16 + (lane&15)
  // of the tile whose first rows a and b point at, `ar` / `br` rows of them present.  k0, k1 multiples of BK.  The LDS is
  // free again for the caller when the function returns.
  __device__ static __forceinline__ void run(f32x4 (&acc)[4][4], const f16* a, int64_t aplane, int lda, int ar,
                                             const f16* b, int64_t bplane, int ldb, int br, int k0, int k1, f16* smem) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1, l15 = lane & 15, q = lane >> 4;
    i32x4_t da[PA], db[PB];
#pragma unroll
    for (int p = 0; p < PA; ++p) da[p] = g16_desc(a + p * aplane, ar, lda);
#pragma unroll
    for (int p = 0; p < PB; ++p) db[p] = g16_desc(b + p * bplane, br, ldb);
    unsigned va[REQ], vb[REQ];
#pragma unroll
    for (int t = 0; t < REQ; ++t) {
      const int row = (t * 4 + wave) * RPI + lane / CH, c = (lane % CH) ^ swz(row);
      va[t] = (unsigned)row * (unsigned)lda * 2u + c * 16u;
      vb[t] = (unsigned)row * (unsigned)ldb * 2u + c * 16u;
    }
    auto stage = [&](int s, int k) {
      f16* base = smem + s * STAGE + wave * RPI * BK;
#pragma unroll
      for (int p = 0; p < PA; ++p)
#pragma unroll
        for (int t = 0; t < REQ; ++t) g16_dma(da[p], g16_lds(base + p * PLANE + t * 4 * RPI * BK), va[t], k * 2);
#pragma unroll
      for (int p = 0; p < PB; ++p)
#pragma unroll
        for (int t = 0; t < REQ; ++t) g16_dma(db[p], g16_lds(base + (PA + p) * PLANE + t * 4 * RPI * BK), vb[t], k * 2);
    };
    const int arow = wm * 64 + l15, brow = wn * 64 + l15;
    k0 = __builtin_amdgcn_readfirstlane(k0);
    k1 = __builtin_amdgcn_readfirstlane(k1);
    int s = 0;
    if (k0 < k1) stage(0, k0);
    for (int k = k0; k < k1; k += BK, s ^= 1) {
      // this wave's requests have landed and its reads are done; behind the barrier so are the others', and nobody reads
      // the other stage any more
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (k + BK < k1) stage(s ^ 1, k + BK);
      const f16* st = smem + s * STAGE;
#pragma unroll
      for (int kk = 0; kk < BK / 32; ++kk) {
        f16x8 fa[PA][4], fb[PB][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ra = arow + i * 16, rb = brow + i * 16;
#pragma unroll
          for (int p = 0; p < PA; ++p)
            fa[p][i] = *reinterpret_cast<const f16x8*>(st + p * PLANE + ra * BK + (((kk * 4 + q) ^ swz(ra)) << 3));
#pragma unroll
          for (int p = 0; p < PB; ++p)
            fb[p][i] = *reinterpret_cast<const f16x8*>(st + (PA + p) * PLANE + rb * BK + (((kk * 4 + q) ^ swz(rb)) << 3));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[0][i], fb[0][j], acc[i][j], 0, 0, 0);
            if constexpr (PB == 2)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[0][i], fb[1][j], acc[i][j], 0, 0, 0);
            if constexpr (PA == 2)
              acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[1][i], fb[0][j], acc[i][j], 0, 0, 0);
          }
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }

  __device__ static __forceinline__ void zero(f32x4 (&acc)[4][4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
};

// Workgroup -> tile: consecutive workgroups of one XCD (every eighth) walk bands of eight tile rows, so that the rows of A
// and B they share stay in that XCD's L2.
__device__ __forceinline__ void g16_tile(int id, int total, int tm, int tn, int& m, int& n) {
  const int q = total >> 3, r = total & 7, xcd = id & 7, idx = id >> 3;
  const int v = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  const int band = v / (8 * tn), first = band * 8, rows = tm - first < 8 ? tm - first : 8;
  const int w = v - band * 8 * tn;
  m = first + w % rows;
  n = w / rows;
}

}  // namespace

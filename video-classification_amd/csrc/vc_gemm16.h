// Tiles of C[m][n] = sum_k A[m][k] B[n][k] on 16-bit floats with fp32 accumulation (v_mfma_f32_16x16x32_f16),
// either operand in one or two terms.
//
// Two terms: a value x, scaled by a power of two into fp16's range, is held as hi = fp16(x) and lo = fp16(x - hi), 22
// bits in all (an absolute floor of 2^-25 of the scaled unit), and the product is hi*hi + hi*lo + lo*hi: three MFMA of
// the 2.5 PFLOP/s kind per product against the 157 TFLOP/s of the fp32 matrix instructions, at fp32's accuracy.
//
// An operand is stored with the reduction along its rows (ROW: [tile side][k], rows of `ld` elements, ld a multiple of
// 64 with zeros behind the last column) or across them (COL: [k][tile side], ld a multiple of 8; it is then read from LDS
// with the transposing ds_read_b64_tr_b16, so no operand is ever copied into the other order).  The second term lies one
// `plane` behind the first.
//
// Tiles of 64 x 64 (TB = 2) serve launches that would leave most of the chip idle: a quarter of the work per k-step and in the
// epilogue, four stages in flight instead of two.
//
// Four waves in a 2 x 2 grid own 64 x 64 (32 x 32) each.  Two LDS stages of (PA + PB) x 128 x BK elements (BK = 64 for single
// terms, 32 otherwise: at most 32 KiB a stage), so that two workgroups share a CU.  ROW stages permute the 16-byte chunks of a
// row so that the 16 rows of a fragment read fall into 16 different slots of the 256-byte bank row; COL stages permute
// the 32-byte blocks of a row so that the eight rows of a transposing read fall on different groups of banks.  Stages
// are filled by LDS-DMA requests in opaque assembly (with the builtin the compiler waits for every outstanding request
// before each LDS read); what lies behind the operand's last row falls outside its buffer descriptor and reads as zero.
//
// Measured: 1.0 PFLOP/s of products in one term (8192 x 1024 x 8192: 132 us) and 1.06 of the three products in two terms
// (4096^3: 389 us, 353 TFLOP/s of fp32 accuracy), where the library's fp16 product of 8192^3 reaches 1.38 and its fp32
// product 0.153.  Bound by the matrix pipes at the clock they leave (62 % of the busy CUs' cycles, 1.84 - 1.98 GHz) and by
// what surrounds a tile: prologue and epilogue of 8 to 16 k-steps.  Tried on the large tile and slower: 256 x 128, four stages,
// three workgroups per CU, tiles chained in one workgroup.
#pragma once
#include "vc_common.h"

namespace {

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int GM = 128;       // rows of A and of B per large tile
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
// buffer descriptor of `bytes` bytes at p (wave-uniform); reads behind them yield zero
__device__ __forceinline__ i32x4_t g16_desc(const f16* p, unsigned bytes) {
  const uint64_t u = (uint64_t)p;
  i32x4_t d;
  d[0] = __builtin_amdgcn_readfirstlane((int)u);
  d[1] = __builtin_amdgcn_readfirstlane((int)(u >> 32));
  d[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  d[3] = 0x00020000;
  return d;
}

enum { ROW = 0, COL = 1 };

// One operand of a tile, of one row at least: an empty descriptor and the scalar offset of a k-step are not to meet, for the
// range check may subtract one from the other.  ROW: p = the tile's first row, n = rows from there on.  COL: p = row 0 of the
// matrix, side = the tile's first column, n = rows (the true length of the reduction).
struct Op16 {
  const f16* p;
  int64_t plane;
  int ld, n, side;
};

// A value of 22 bits in two fp16 terms.
__device__ __forceinline__ void f16_split(float v, f16& hi, f16& lo) {
  hi = (f16)v;
  lo = (f16)(v - (float)hi);
}

// TB: blocks of 16 on either side of a wave's part of the tile, 4 (tiles of 128 x 128) or 2 (64 x 64).  BF: the operands are
// bf16 as they came (one term each).
template <int PA, int PB, int KA = ROW, int KB = ROW, int TB = 4, bool BF = false>
struct G16 {
  __device__ static __forceinline__ f32x4 mma(const f16x8& a, const f16x8& b, const f32x4& c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }

  static constexpr int T = 32 * TB;                  // rows of A and of B per tile
  static constexpr int BK = PA + PB == 2 ? 64 : 32;
  static constexpr int PLANE = T * BK;               // elements of one plane of a stage
  static constexpr int STAGE = (PA + PB) * PLANE;
  static constexpr int NS = TB == 4 ? 2 : 4;         // stages
  static constexpr int LDS = NS * STAGE;             // elements of shared memory
  static constexpr int CH = BK / 8;                  // 16-byte chunks of a ROW stage's row
  static constexpr int RPI = 64 / CH;                // rows of it that one wave request fills
  static constexpr int REQ = T * BK / 2048;          // requests per wave, plane and stage (1 KiB each)
  static constexpr int LPR = T / 8;                  // 16-byte chunks of a COL stage's row
  static constexpr int PER = (PA + PB) * REQ;        // requests per wave and stage

  // A 16-byte read is served 16 lanes at a time, lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31 of each half of the wave: with
  // 64-byte rows (BK = 32) the four groups of four rows need 0, 2, 3, 1 for both sets to meet 16 different slots (0, 1, 2, 3
  // left a third to a half of the LDS cycles to conflicts).
  __device__ static __forceinline__ int rswz(int row) {
    return BK == 64 ? (row >> 1) & 7 : (((row >> 2) & 1) << 1) ^ (((row >> 3) & 1) * 3);
  }
  __device__ static __forceinline__ int cswz(int row) {
    return TB == 4 ? (row & 3) | ((row >> 1) & 4) : ((row >> 1) & 1) | ((row >> 2) & 2);
  }

  // byte offset of this lane's 16 bytes of request t, relative to the tile's corner of the k-step
  template <int KIND>
  __device__ static __forceinline__ unsigned src_off(int t, int wave, int lane, int ld) {
    if (KIND == ROW) {
      const int row = (t * 4 + wave) * RPI + lane / CH;
      return (unsigned)row * (unsigned)ld * 2u + (unsigned)((lane % CH) ^ rswz(row)) * 16u;
    }
    const int row = (t * 4 + wave) * (64 / LPR) + lane / LPR, pos = lane % LPR;
    return (unsigned)row * (unsigned)ld * 2u + (unsigned)((((pos >> 1) ^ cswz(row)) << 1) | (pos & 1)) * 16u;
  }

  // A staged operand plane: its descriptor, moved along the reduction by a scalar offset (ROW) or by its base (COL).
  template <int KIND>
  struct Stream {
    i32x4_t d;
    uint64_t at;     // COL: address of the k-step's corner
    uint64_t step;   // COL: bytes of a k-step
    int left, ld2, side2;
    __device__ __forceinline__ void open(const Op16& o, int plane, int k0) {
      if (KIND == ROW) {
        d = g16_desc(o.p + plane * o.plane, (unsigned)(o.n < T ? o.n : T) * (unsigned)o.ld * 2u);
        return;
      }
      const uint64_t u = (uint64_t)(o.p + plane * o.plane + (int64_t)k0 * o.ld + o.side);
      at = (uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)u) |
           ((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32);
      ld2 = __builtin_amdgcn_readfirstlane(o.ld * 2);
      side2 = __builtin_amdgcn_readfirstlane(o.side * 2);
      left = __builtin_amdgcn_readfirstlane(o.n - k0);
      step = (uint64_t)BK * (unsigned)ld2;
      d[3] = 0x00020000;
    }
    __device__ __forceinline__ void stage(unsigned lds, const unsigned (&v)[REQ], int k) {
      if (KIND == ROW) {
#pragma unroll
        for (int t = 0; t < REQ; ++t) g16_dma(d, lds + t * 4096, v[t], k * 2);
        return;
      }
      const int rows = left < BK ? left : BK;
      d[0] = (int)at;
      d[1] = (int)(at >> 32);
      d[2] = rows > 0 ? rows * ld2 - side2 : 0;
#pragma unroll
      for (int t = 0; t < REQ; ++t) g16_dma(d, lds + t * 4096, v[t], 0);
      at += step;
      left -= BK;
    }
  };

  // Fragment of the 16 tile rows (ROW) or columns (COL) of block `blk` (0 .. 2 TB - 1), 32 reduction elements from kk * 32.  The swizzles
  // are those of the row within its block: adding a block does not change them.
  template <int KIND>
  __device__ static __forceinline__ f16x8 frag(const f16* st, int blk, int kk, int lane) {
    const int l15 = lane & 15, q = lane >> 4;
    if (KIND == ROW)
      return *reinterpret_cast<const f16x8*>(st + (blk * 16 + l15) * BK + (((kk * 4 + q) ^ rswz(l15)) << 3));
    typedef short s16x4_t __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4_t lds4;
    const int r0 = 8 * q + ((lane >> 2) & 3);  // this lane supplies row r0, columns 4 (lane & 3) .. + 3, then row r0 + 4
    const f16* p = st + (kk * 32 + r0) * T + ((blk ^ cswz(r0)) << 4) + (lane & 3) * 4;
    union {
      s16x4_t h[2];
      f16x8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 4 * T));
    return u.v;
  }

  // acc[i][j][r] += sum over k in [k0, k1) of A's tile row (wm*TB + i)*16 + (lane>>4)*4 + r and B's tile row (wn*TB + j)*16 +
  // (lane&15).  k0, k1 multiples of BK.  The LDS is free again for the caller when the function returns.
  //
  // A k-step is two phases: single terms its two 32-deep halves, two terms the product of the first terms and then the mixed
  // ones.  While a phase multiplies out of registers the next phase's fragments are read, one read behind every second
  // product, so no product waits for LDS.  The barrier lies between the phases: by then every wave has read all of the
  // stage, which takes the k-step NS further on, and has waited for its own requests of the next one.
  __device__ static __forceinline__ void run(f32x4 (&acc)[TB][TB], const Op16& a, const Op16& b, int k0, int k1, f16* smem) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    unsigned va[REQ], vb[REQ];
#pragma unroll
    for (int t = 0; t < REQ; ++t) {
      va[t] = src_off<KA>(t, wave, lane, a.ld);
      vb[t] = src_off<KB>(t, wave, lane, b.ld);
    }
    k0 = __builtin_amdgcn_readfirstlane(k0);
    k1 = __builtin_amdgcn_readfirstlane(k1);
    if (k0 >= k1) return;
    Stream<KA> sa[PA];
    Stream<KB> sb[PB];
#pragma unroll
    for (int p = 0; p < PA; ++p) sa[p].open(a, p, k0);
#pragma unroll
    for (int p = 0; p < PB; ++p) sb[p].open(b, p, k0);
    auto stage = [&](int s, int k) {
      const unsigned base = g16_lds(smem + s * STAGE) + wave * 1024;
#pragma unroll
      for (int p = 0; p < PA; ++p) sa[p].stage(base + p * PLANE * 2, va, k);
#pragma unroll
      for (int p = 0; p < PB; ++p) sb[p].stage(base + (PA + p) * PLANE * 2, vb, k);
    };
    constexpr bool ONE = PA + PB == 2;  // phase 2: the second half, or the second terms
    constexpr int SP = TB / 2;          // products per read
    f16x8 a1[TB], b1[TB], a2[TB], b2[TB];
    // fragment r of a phase: the first TB are A's (where the phase has its own), then B's
    auto read1 = [&](const f16* st, int r, f16x8(&fa)[TB], f16x8(&fb)[TB]) __attribute__((always_inline)) {
      if (r < TB) fa[r] = frag<KA>(st, wm * TB + r, 0, lane);
      else fb[r - TB] = frag<KB>(st + PA * PLANE, wn * TB + r - TB, 0, lane);
    };
    auto read2 = [&](const f16* st, int r) __attribute__((always_inline)) {
      if (r < TB) {
        if (ONE) a2[r] = frag<KA>(st, wm * TB + r, 1, lane);
        else if (PA == 2) a2[r] = frag<KA>(st + PLANE, wm * TB + r, 0, lane);
      } else if (ONE) b2[r - TB] = frag<KB>(st + PA * PLANE, wn * TB + r - TB, 1, lane);
      else if (PB == 2) b2[r - TB] = frag<KB>(st + (PA + 1) * PLANE, wn * TB + r - TB, 0, lane);
    };
#pragma unroll
    for (int d = 0; d < NS; ++d)
      if (k0 + d * BK < k1) stage(d, k0 + d * BK);
    if (k0 + (NS - 1) * BK < k1)
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((NS - 1) * PER) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int r = 0; r < 2 * TB; ++r) read1(smem, r, a1, b1);
    int s = 0;
    for (int k = k0; k < k1; k += BK) {
      const int next = NS == 2 ? s ^ 1 : s + 1 == NS ? 0 : s + 1;
      const f16 *st = smem + s * STAGE, *sn = smem + next * STAGE;
#pragma unroll
      for (int n = 0; n < TB * TB; ++n) {
        const int i = n / TB, j = n % TB;
        acc[i][j] = mma(a1[i], b1[j], acc[i][j]);
        if (n % SP == 0) read2(st, n / SP);
        __builtin_amdgcn_sched_barrier(0);
      }
      // the next step's requests have landed; the NS - 2 behind it may be on their way
      if (NS > 2 && k + (NS - 1) * BK < k1)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * PER) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (k + NS * BK < k1) stage(s, k + NS * BK);
      // behind the last k-step the reads below meet stale LDS, which is never multiplied
      f16x8 an[TB], bn[TB];
#pragma unroll
      for (int n = 0; n < TB * TB; ++n) {
        const int i = n / TB, j = n % TB;
        if (ONE) acc[i][j] = mma(a2[i], b2[j], acc[i][j]);
        else if (PB == 2) acc[i][j] = mma(a1[i], b2[j], acc[i][j]);
        if (n % SP == 0) read1(sn, n / SP, an, bn);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (!ONE && PA == 2)
#pragma unroll
        for (int n = 0; n < TB * TB; ++n)
          acc[n / TB][n % TB] = mma(a2[n / TB], b1[n % TB], acc[n / TB][n % TB]);
#pragma unroll
      for (int r = 0; r < TB; ++r) {
        a1[r] = an[r];
        b1[r] = bn[r];
      }
      s = next;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  }

  __device__ static __forceinline__ void zero(f32x4 (&acc)[TB][TB]) {
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
};

// An accumulated tile through LDS, so that global memory sees whole rows: fp32, [B row][A row], 64 B rows at a time (of a
// 128 x 128 tile those of the waves with wn == half).  Rows are padded by four floats and their groups of four permuted by
// the row, so that reading along them, in 16-byte pieces, or across them meets few bank conflicts.
template <int TB>
struct Tile16 {
  static constexpr int T = 32 * TB, PITCH = T + 4, FLOATS = 64 * PITCH, HALVES = T / 64;
  static constexpr int VPR = T / 8, UNITS = 64 * VPR / G_THREADS;  // pieces of eight values: of a row, per thread

  __device__ static __forceinline__ int at(int row, int col) {
    return row * PITCH + ((((col >> 2) ^ (row >> 3)) << 2) | (col & 3));
  }
  __device__ static __forceinline__ void put(const f32x4 (&acc)[TB][TB], int half, float* t) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, l15 = lane & 15;
    if (HALVES == 2 && (wave & 1) != half) return;
    const int row0 = HALVES == 2 ? 0 : (wave & 1) * 32;
#pragma unroll
    for (int i = 0; i < TB; ++i)
#pragma unroll
      for (int j = 0; j < TB; ++j)
        *reinterpret_cast<f32x4*>(t + at(row0 + j * 16 + l15, ((wave >> 1) * TB + i) * 16 + q * 4)) = acc[i][j];
  }
  // eight consecutive values of a row (col a multiple of 8)
  __device__ static __forceinline__ F8 get(const float* t, int row, int col) {
    F8 r;
    const f32x4 a = *reinterpret_cast<const f32x4*>(t + at(row, col)), b = *reinterpret_cast<const f32x4*>(t + at(row, col + 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r.v[e] = a[e];
      r.v[4 + e] = b[e];
    }
    return r;
  }
  __device__ static __forceinline__ void set(float* t, int row, int col, const F8& v) {
    *reinterpret_cast<f32x4*>(t + at(row, col)) = f32x4{v.v[0], v.v[1], v.v[2], v.v[3]};
    *reinterpret_cast<f32x4*>(t + at(row, col + 4)) = f32x4{v.v[4], v.v[5], v.v[6], v.v[7]};
  }
};
__device__ __forceinline__ void f16_split8(const F8& v, f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f16 h, l;
    f16_split(v.v[e], h, l);
    hi[e] = h;
    lo[e] = l;
  }
}

// Workgroup -> tile (of a slice of the reduction): consecutive workgroups of one XCD (every eighth) walk bands of eight tile
// rows, slice after slice, so that the rows of A and B they share stay in that XCD's L2.
__device__ __forceinline__ void g16_tile(int id, int slices, int tm, int tn, int& slice, int& m, int& n) {
  const int tiles = tm * tn, total = tiles * slices;
  const int q = total >> 3, r = total & 7, xcd = id & 7, idx = id >> 3;
  int v = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
  slice = 0;
  if (slices > 1) {
    slice = v / tiles;
    v -= slice * tiles;
  }
  const int band = v / (8 * tn), first = band * 8, rows = tm - first < 8 ? tm - first : 8;
  const int w = v - band * 8 * tn;
  m = first + w % rows;
  n = w / rows;
}

}  // namespace

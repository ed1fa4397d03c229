// Matrix product of 16-bit operands for shapes that the matrix pipe bounds, fp32 accumulation:
//   R[r, c] = sum over the segments q and over k of A_q[r, k] B_q[c, k]
// (segments: pairs of planes of operands that are sums of 16-bit terms; one segment for plain operands).
//
// A workgroup owns a BM x BN tile and walks the contraction in steps of 64.  Both operands' parts of a step go from memory straight
// to the LDS (buffer_load ... lds, 1 KiB per wave instruction) into the stage that the previous step has left, while this step's
// fragments are multiplied: one barrier a step.  The stages keep the operands as they lie in memory:
//   contraction along the rows ("rows"): [tile rows][64], a row = 8 chunks of 16 bytes, chunk c of row r in slot c ^ (r >> 1 & 7);
//     a fragment is one ds_read_b128 per lane, and the 16 rows it touches at one c lie on 16 different 16-byte slots of the banks;
//   contraction down the columns ("columns"): [64][tile rows], chunk c of line k in slot c ^ 2 (k & 3 | (k >> 3 & 1) << 2);
//     a fragment is two transposing reads (ds_read_b64_tr_b16: lane j of 16 hands in the address of row j / 4, columns 4 (j % 4) ..,
//     and receives column j of the four rows); the eight lines of a half wave lie on different 32-byte slots.
// The DMA writes 16 bytes per lane in lane order, so the swizzle is applied by choosing which chunk a lane fetches.
// Reads past the end (rows, or the tail of the contraction) are given an offset beyond the descriptor, which returns zeros.
//
// 256 x 256 by eight waves of 128 x 64: a step is 64 MFMAs per wave (2048 cycles a SIMD pair) against 64 KiB from memory and 192 KiB
// of fragments from the LDS; 128 x 128 by four waves of 64 x 64 for results with too few large tiles (two workgroups per CU).
#pragma once
#include "pp_rows.h"
#include "pp_spconv.h"  // pp_xcd_remap

typedef unsigned gm_u32x4 __attribute__((ext_vector_type(4)));
typedef short gm_s16x4 __attribute__((ext_vector_type(4)));
typedef float gm_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 gm_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gm_f16x8 __attribute__((ext_vector_type(8)));

#define GM_SEGMENTS 6
#define GM_BK 64

struct GemmArgs {
  const void *a[GM_SEGMENTS], *b[GM_SEGMENTS];
  int segments;
  int64_t m, n, k;
  int64_t lda, ldb;            // elements between rows of A / B (columns form: between lines of the contraction); multiples of 8
  int64_t a_batch, b_batch;    // elements between batch elements
  int splits;                  // parts of the contraction (blockIdx.y)
  int64_t k_per_split;         // multiple of GM_BK
  int lower;                   // square results: only tiles on and below the diagonal
};

__device__ __forceinline__ gm_f32x4 gm_mma(gm_u32x4 x, gm_u32x4 y, gm_f32x4 c, pp_bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gm_bf16x8, x), __builtin_bit_cast(gm_bf16x8, y), c, 0, 0, 0);
}
__device__ __forceinline__ gm_f32x4 gm_mma(gm_u32x4 x, gm_u32x4 y, gm_f32x4 c, pp_f16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gm_f16x8, x), __builtin_bit_cast(gm_f16x8, y), c, 0, 0, 0);
}

// One operand's stage of ROWS x 64 elements, filled by WAVES waves.  COLUMNS: the contraction runs down the columns
template <bool COLUMNS, int ROWS, int WAVES>
struct GemmStage {
  static constexpr int INSTR = ROWS * GM_BK * 2 / 1024, PER = INSTR / WAVES;  // wave instructions of 1 KiB
  static constexpr int CHUNKS = COLUMNS ? ROWS / 8 : 8;                        // 16-byte chunks of a stage line
  static constexpr int LINES = 64 / CHUNKS;                                    // lines of an instruction
  static_assert(INSTR % WAVES == 0 && 64 % CHUNKS == 0, "the stage is whole instructions of every wave");
  unsigned off[PER];  // byte offset of the lane's chunk from the tile's corner at this step; all ones: past the operand's end

  static __device__ __forceinline__ int swizzle(int line) { return COLUMNS ? 2 * ((line & 3) | ((line >> 3) & 1) << 2) : (line >> 1) & 7; }
  static __device__ __forceinline__ int line(int i) {
    return ((threadIdx.x >> 6) * PER + i) * LINES + (threadIdx.x & 63) / CHUNKS;
  }
  static __device__ __forceinline__ int chunk(int i) { return (threadIdx.x & 63) % CHUNKS ^ swizzle(line(i)); }

  __device__ __forceinline__ void init(int64_t row0, int64_t rows, int64_t ld) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool in = COLUMNS ? row0 + chunk(i) * 8 < rows : row0 + line(i) < rows;
      off[i] = in ? (unsigned)(line(i) * ld * 2 + chunk(i) * 16) : 0xFFFFFFFFu;
    }
  }
  // corner: first element of the tile at this step; left: what is left of the contraction; lds: the stage's byte address
  __device__ __forceinline__ void fetch(const void* corner, int64_t left, unsigned lds) const {
    const uint64_t base = (uint64_t)(uintptr_t)corner;
    const gm_u32x4 d = {(unsigned)__builtin_amdgcn_readfirstlane((unsigned)base),
                        (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(base >> 32) & 0xFFFFu), 0x80000000u, 0x00020000u};
    const unsigned at = __builtin_amdgcn_readfirstlane(lds + (threadIdx.x >> 6) * PER * 1024u);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      unsigned o = off[i];
      if (left < GM_BK && (COLUMNS ? line(i) : chunk(i) * 8) >= left) o = 0xFFFFFFFFu;
      asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds" ::"v"(o), "s"(at + i * 1024u), "s"(d)
                   : "memory", "m0");
    }
  }
  // the 16 x 32 fragment at rows r0 .., contraction kk .. of the stage at `lds`
  static __device__ __forceinline__ gm_u32x4 fragment(const char* lds, int r0, int kk) {
    const int lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15;
    if constexpr (!COLUMNS) {
      const int r = r0 + j;
      return *(const gm_u32x4*)(lds + r * 128 + (((kk >> 3) + q) ^ swizzle(r)) * 16);
    } else {
      union {
        gm_s16x4 h[2];
        gm_u32x4 v;
      } u;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kk + 8 * q + 4 * h + (j >> 2), c = (r0 >> 3) + ((j & 3) >> 1);
        const char* p = lds + k * (ROWS * 2) + (c ^ swizzle(k)) * 16 + (j & 1) * 8;
        u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gm_s16x4*)p);
      }
      return u.v;
    }
  }
};

// Epi: init(...) is the caller's; block(ti, tj, split, batch) is called once, put(row, column, v) for every lane's four neighbouring
// columns of a row (row < m; columns may pass n), done(lds) at the end by all threads
template <typename T, bool AC, bool BC, int BM, int BN, int WM, int WN, typename Epi>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64, BM * BN > 128 * 128 ? 1 : 2) void k_gemm(GemmArgs g, Epi epi) {
  constexpr int WAVES = BM / WM * (BN / WN), FM = WM / 16, FN = WN / 16;
  constexpr int A_BYTES = BM * GM_BK * 2, STAGE = (BM + BN) * GM_BK * 2;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t tm = (g.m + BM - 1) / BM, tn = (g.n + BN - 1) / BN;
  // neighbouring tiles on one XCD's cache: every XCD gets a contiguous range of tiles, walked in bands of eight tile rows
  const unsigned t = pp_xcd_remap(blockIdx.x, gridDim.x);
  int64_t ti, tj;
  if (g.lower) {
    ti = (int64_t)((sqrt(8.0 * (double)t + 1.0) - 1.0) * 0.5);
    while ((ti + 1) * (ti + 2) / 2 <= (int64_t)t) ++ti;
    while (ti * (ti + 1) / 2 > (int64_t)t) --ti;
    tj = (int64_t)t - ti * (ti + 1) / 2;
  } else {
    const int64_t band = (int64_t)t / (8 * tn), first = band * 8, high = tm - first < 8 ? tm - first : 8, in = (int64_t)t - band * 8 * tn;
    ti = first + in % high;
    tj = in / high;
  }
  const int split = blockIdx.y;
  const int64_t batch = blockIdx.z, m0 = ti * BM, n0 = tj * BN;
  const int64_t k0 = split * g.k_per_split, k1 = k0 + g.k_per_split < g.k ? k0 + g.k_per_split : g.k;
  const int64_t steps = k1 > k0 ? (k1 - k0 + GM_BK - 1) / GM_BK : 0, total = steps * g.segments;
  GemmStage<AC, BM, WAVES> sa;
  GemmStage<BC, BN, WAVES> sb;
  sa.init(m0, g.m, g.lda);
  sb.init(n0, g.n, g.ldb);
  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const int64_t oa = batch * g.a_batch + (AC ? m0 : m0 * g.lda), ob = batch * g.b_batch + (BC ? n0 : n0 * g.ldb);
  auto fetch = [&](int64_t s) {
    const int q = (int)(s / steps);
    const int64_t k = k0 + (s - q * steps) * GM_BK;
    const unsigned at = base + (unsigned)(s & 1) * STAGE;
    sa.fetch((const T*)g.a[q] + oa + (AC ? k * g.lda : k), k1 - k, at);
    sb.fetch((const T*)g.b[q] + ob + (BC ? k * g.ldb : k), k1 - k, at + A_BYTES);
  };
  const int wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
  gm_f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = (gm_f32x4){0.f, 0.f, 0.f, 0.f};
  if (total > 0) fetch(0);
  for (int64_t s = 0; s < total; ++s) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this step's stage is in the LDS ...
    __syncthreads();                                  // ... for every wave, and the other one has been read by all
    if (s + 1 < total) fetch(s + 1);
    const char* const at = lds + (s & 1) * STAGE;
#pragma unroll
    for (int kk = 0; kk < GM_BK; kk += 32) {
      gm_u32x4 fb[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = GemmStage<BC, BN, WAVES>::fragment(at + A_BYTES, wn + 16 * j, kk);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const gm_u32x4 fa = GemmStage<AC, BM, WAVES>::fragment(at, wm + 16 * i, kk);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = gm_mma(fb[j], fa, acc[i][j], T());  // B first: a lane gets neighbours of one row
      }
    }
  }
  epi.block(m0, n0, split, batch);
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t r = m0 + wm + 16 * i + (lane & 15);
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
      if (r < g.m) epi.put(r, n0 + wn + 16 * j + 4 * (lane >> 4), j, v);
    }
  }
  if constexpr (Epi::COLUMN_SUMS) {
    __syncthreads();
    epi.template done<BM, BN, WM, WN>((float*)lds, wm, wn, n0, (int64_t)ti);
  }
}

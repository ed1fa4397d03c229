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

// A wave's WM x 64 results to memory.  A lane holds row l & 15 and columns 4 (l >> 4) .. + 3 of every 16 x 16 fragment; through ROWS
// rows of the wave's own LDS (256 bytes a row, 16-byte chunk c of row r in slot c ^ (r & 15): no bank conflicts either way) it gets
// eight neighbouring columns instead, eight lanes a row: whole lines to memory, and one short loop of epilogue code.  (Working on
// the fragments where they lie, the unrolled epilogue was 100 KB of code that ran once a tile, and took as long as the products:
// 8192 x 1024 -> 4096 with silu 104 us, of which 83 us without the loads of the loop.)
// Epi: block(first of the lane's columns, split, batch) once; load(row, Row&) asks for what a row's epilogue reads, put(row, Row, v)
// finishes it (rows may pass the end: both check)
template <int FM, int FN, int ROWS, typename Epi>
__device__ __forceinline__ void gm_epilogue(Epi& epi, const gm_f32x4 (&acc)[FM][FN], float* __restrict__ lds, int64_t row0, int64_t col0, int split,
                                            int64_t batch) {
  static_assert(FN == 4 && ROWS % 16 == 0 && FM * 16 % ROWS == 0, "a wave's columns are 64");
  const int lane = threadIdx.x & 63;
  epi.block(col0 + 8 * (lane & 7), split, batch);
#pragma unroll
  for (int p = 0; p < FM * 16 / ROWS; ++p) {
#pragma unroll
    for (int i = 0; i < ROWS / 16; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        *(gm_f32x4*)(lds + (16 * i + (lane & 15)) * 64 + ((4 * j + (lane >> 4)) ^ (lane & 15)) * 4) = acc[p * (ROWS / 16) + i][j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 2
    for (int t = 0; t < ROWS / 8; ++t) {
      const int lr = 8 * t + (lane >> 3);
      const int64_t r = row0 + p * ROWS + lr;
      typename Epi::Row row;
      epi.load(r, row);
      const gm_f32x4 lo = *(const gm_f32x4*)(lds + lr * 64 + ((2 * (lane & 7)) ^ (lr & 15)) * 4);
      const gm_f32x4 hi = *(const gm_f32x4*)(lds + lr * 64 + ((2 * (lane & 7) + 1) ^ (lr & 15)) * 4);
      float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      epi.put(r, row, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <typename T, bool AC, bool BC, int BM, int BN, int WM, int WN, typename Epi>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64, BM * BN > 128 * 128 ? 1 : 2) void k_gemm(GemmArgs g, Epi epi) {
  constexpr int WAVES = BM / WM * (BN / WN), FM = WM / 16, FN = WN / 16;
  constexpr int A_BYTES = BM * GM_BK * 2, STAGE = (BM + BN) * GM_BK * 2;
  static_assert((STAGE & (STAGE - 1)) == 0, "the stages alternate by a bit of the address");
  __shared__ __attribute__((aligned(2 * STAGE))) char lds[2 * STAGE];
  const int wave = threadIdx.x >> 6;
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
  // the corner of the next step to be fetched, what is left of its segment, and the stage it goes to
  const int64_t oa = batch * g.a_batch + (AC ? m0 + k0 * g.lda : m0 * g.lda + k0), ob = batch * g.b_batch + (BC ? n0 + k0 * g.ldb : n0 * g.ldb + k0);
  const int64_t da = AC ? GM_BK * g.lda : GM_BK, db = BC ? GM_BK * g.ldb : GM_BK;
  const T *pa = (const T*)g.a[0] + oa, *pb = (const T*)g.b[0] + ob;
  int64_t left = k1 - k0;
  int segment = 0;
  unsigned to = base;
  auto fetch = [&]() {
    sa.fetch(pa, left, to);
    sb.fetch(pb, left, to + A_BYTES);
    pa += da;
    pb += db;
    left -= GM_BK;
    to ^= STAGE;
    if (left <= 0 && ++segment < g.segments) {
      pa = (const T*)g.a[segment] + oa;
      pb = (const T*)g.b[segment] + ob;
      left = k1 - k0;
    }
  };
  const int wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
  gm_f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = (gm_f32x4){0.f, 0.f, 0.f, 0.f};
  // fragments are read one half step ahead of the MFMAs that take them, the stage behind them one step ahead of that: the wait and
  // the barrier stand between the halves, when this stage has been read to its end and the next one has had a step's time to arrive
  gm_u32x4 fa[2][FM], fb[2][FN];
  const char* at = lds;
  auto read = [&](int half) {
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[half][j] = GemmStage<BC, BN, WAVES>::fragment(at + A_BYTES, wn + 16 * j, 32 * half);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[half][i] = GemmStage<AC, BM, WAVES>::fragment(at, wm + 16 * i, 32 * half);
  };
  auto multiply = [&](int half) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = gm_mma(fb[half][j], fa[half][i], acc[i][j], T());  // B first: a lane gets neighbours of one row
  };
  if (total > 0) {
    fetch();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (total > 1) fetch();
    read(0);
    for (int64_t s = 1; s < total; ++s) {
      read(1);
      __builtin_amdgcn_sched_barrier(0);  // (left alone, the scheduler moves the reads behind the products, in front of the wait)
      multiply(0);
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the next stage has arrived, this one has been read ...
      __syncthreads();                                            // ... by every wave
      if (s + 1 < total) fetch();
      at = lds + ((s & 1) ? STAGE : 0);
      read(0);
      __builtin_amdgcn_sched_barrier(0);
      multiply(1);
    }
    read(1);
    multiply(0);
    multiply(1);
  }
  __syncthreads();  // the stages are free
  constexpr int ROWS = 2 * STAGE / WAVES >= 64 * 64 * 4 ? 64 : 32;
  gm_epilogue<FM, FN, ROWS>(epi, acc, (float*)lds + wave * ROWS * 64, m0 + wm, n0 + wn, split, batch);
  if constexpr (Epi::COLUMN_SUMS) {
    __syncthreads();
    epi.template done<BM, BN, WM, WN>((float*)lds, wm, wn, n0, (int64_t)ti);
  }
}

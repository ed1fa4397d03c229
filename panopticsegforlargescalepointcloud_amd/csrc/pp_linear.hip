// Linear layer with bias, activation and residual in the epilogue, and its gradients, on [rows, channels] features:
//   z = x W^T + b,  y = act(z) + r;   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz,  dr = dy
// Three kernels: the tile kernel described here takes any width, type and alignment; aligned 16-bit operands that the matrix pipe bounds go
// through pp_gemm.h, narrow 16-bit layers through the streaming kernel further down (lin_wide, lin_stream_lds).  A workgroup of four waves owns a BM x BN tile of the result and walks the contraction
// in steps of BK: every operand is brought to the LDS as rows of consecutive contraction elements (an operand whose contraction runs
// down its columns is transposed on the way, in registers), 16 bytes at a time, XOR-swizzled so that the fragment reads of 16 rows
// spread over all banks; the next step's loads are in flight while this step's fragments are multiplied.
// fp32 operands are split exactly into three bf16 terms (8 + 8 + 8 bits) when they are staged, and a product is the six largest of its
// nine bf16 products (the others are at most 2^-23 of it), accumulated in fp32: an fp32-accurate evaluation at 2.7 times the rate of the fp32 matrix instructions.
// Infinities and NaN do what they do in a plain sum (lin_exact).  bf16 and fp16 operands are multiplied as they are, accumulated in fp32.
// Nothing is kept for the backward pass but x: z is recomputed from it (the layers are bound by memory, a stored z would cost a write
// and a read of its own, and its rounding would enter the gradients).  dz is rounded to the element type once, as the matrix
// instructions take it: half a step of each of its values, 2.3e-3 instead of 1.7e-3 over dx and dW in bf16.  A second plane of what is
// left would give it back for twice the products (8192 x 1024 -> 4096: 145 of 320 us), which a 16-bit layer is not chosen for.  The weight gradient's rows are cut into parts, whose sums are added in a fixed order: results repeat.
#include "pp_gemm.h"


enum { LIN_FWD = 0, LIN_DZ = 1, LIN_STORE = 2, LIN_PART = 3 };

struct LinArgs {
  const void *a, *b;     // A: m rows of the contraction k (or [k, m] where it runs down the columns), B: n of it (or [k, n])
  int64_t m, k, lda, ldb, ldo;
  int n;
  int va, vb;            // A / B may be read in 16-byte (columns: 8-byte) vectors
  const void *bias, *extra;  // extra: the residual (LIN_FWD) or dy (LIN_DZ), [m, n] of row length n
  int act;
  float slope;
  void* out;
  int n_out;             // columns written (LIN_DZ pads its rows with zeros up to here)
  float *part, *part_bias;   // LIN_PART: part[splits][m][n]; LIN_DZ: part_bias[row tile][n] (nullable)
  int64_t k_per_split;
};

template <typename T> struct LinType {
  static constexpr int PLANES = 1, BK = 64, BUFS = 2;
};
template <> struct LinType<float> {
  static constexpr int PLANES = 3, BK = 32, BUFS = 1;
};

// eight elements of the contraction, in the form they have in the LDS: PLANES x 16 bytes
template <typename T> struct LinChunk { gm_u32x4 p[LinType<T>::PLANES]; };

// hi, mid and lo, each the nearest bf16 to what is left: hi + mid + lo is v exactly (24 bits in 8 and two signs), |mid| <= 2^-8 |v| and
// |lo| <= 2^-16 |v| of either sign, so that the products left out, mid lo + lo mid + lo lo, are at most 2^-23 of v w and cancel in long
// sums (cut off instead of rounded the terms all have v's sign: up to 2^-21, always towards 0).  The same number of instructions: the
// conversion makes two values at once.  hi overflows above the largest bf16: see lin_exact.  A bf16 ends at 2^-133: what of a term lies
// below is lost, so operands below 2^-109 are kept to 2^-134, not to 24 bits
typedef float lin_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 lin_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void lin_pack(const float (&v)[8], LinChunk<float>& c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    lin_f32x2 r = {v[2 * i], v[2 * i + 1]};
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const unsigned q = __builtin_bit_cast(unsigned, __builtin_convertvector(r, lin_bf16x2));
      c.p[p][i] = q;
      if (p < 2) r = (lin_f32x2){r[0] - __uint_as_float(q << 16), r[1] - __uint_as_float(q & 0xFFFF0000u)};
    }
  }
}
__device__ __forceinline__ void lin_pack(const pp_bf16 (&v)[8], LinChunk<pp_bf16>& c) { __builtin_memcpy(&c.p[0], v, 16); }
__device__ __forceinline__ void lin_pack(const pp_f16 (&v)[8], LinChunk<pp_f16>& c) { __builtin_memcpy(&c.p[0], v, 16); }

__device__ __forceinline__ gm_f32x4 lin_mma(const LinChunk<pp_bf16>& x, const LinChunk<pp_bf16>& y, gm_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gm_bf16x8, x.p[0]), __builtin_bit_cast(gm_bf16x8, y.p[0]), c, 0, 0, 0);
}
__device__ __forceinline__ gm_f32x4 lin_mma(const LinChunk<pp_f16>& x, const LinChunk<pp_f16>& y, gm_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gm_f16x8, x.p[0]), __builtin_bit_cast(gm_f16x8, y.p[0]), c, 0, 0, 0);
}
__device__ __forceinline__ gm_f32x4 lin_mma(const LinChunk<float>& x, const LinChunk<float>& y, gm_f32x4 c) {
#pragma unroll
  for (int s = 2; s >= 0; --s)  // smallest products first
#pragma unroll
    for (int i = 0; i <= s; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gm_bf16x8, x.p[i]), __builtin_bit_cast(gm_bf16x8, y.p[s - i]), c, 0, 0, 0);
  return c;
}

// LDS position (in 16-byte chunks) of chunk c of row r: rows of CH chunks; 16 neighbouring rows at one c fall on 16 different slots
template <int CH>
__device__ __forceinline__ int lin_at(int r, int c) {
  return r * CH + (c ^ (CH == 8 ? (r >> 1) & 7 : (r >> 2) & 3));
}

// One operand's part of a step, ROWS rows of BK contraction elements, on its way from memory to the LDS through registers
template <typename T, bool STRIDED, int ROWS>
struct LinStage {
  static constexpr int BK = LinType<T>::BK, CH = BK / 8, PLANES = LinType<T>::PLANES;
  static constexpr int COLS = sizeof(T) == 2 ? 4 : 2;                      // strided: columns of a unit
  static constexpr int UNITS = STRIDED ? ROWS / COLS * CH : ROWS * CH;
  static constexpr int PER = (UNITS + 255) / 256;
  static constexpr int E = STRIDED ? 8 * COLS : 8;
  T v[PER][E];

  // row0, k0: the tile's corner; rows, k1: where the operand ends
  __device__ __forceinline__ void load(const T* __restrict__ src, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int64_t k1, bool vec) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int unit = threadIdx.x + 256 * i;
      if (UNITS % 256 != 0 && unit >= UNITS) continue;
      if constexpr (!STRIDED) {
        const int64_t r = row0 + unit / CH, k = k0 + (unit % CH) * 8;
        const T* p = src + r * ld + k;
        if (vec) {
          constexpr int W = 16 / (int)sizeof(T);
#pragma unroll
          for (int h = 0; h < 8 / W; ++h) {
            gm_u32x4 q = {0u, 0u, 0u, 0u};
            if (r < rows && k + h * W < k1) q = *(const gm_u32x4*)(p + h * W);
            __builtin_memcpy(&v[i][h * W], &q, 16);
          }
        } else {
          // eight elements from any address, later rows' among them at the end (taken out below, when all loads are on their way)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = (T)0.f;
          if (r < rows && (rows - r) * ld - k >= 8) {
            __builtin_memcpy(&v[i][0], p, 8 * sizeof(T));
          } else if (r < rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (k + e < k1) v[i][e] = p[e];
          }
        }
      } else {
        const int64_t c = row0 + (unit % (ROWS / COLS)) * COLS, k = k0 + unit / (ROWS / COLS) * 8;
        const T* p = src + k * ld + c;
        if (vec) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            unsigned long long q = 0ull;
            if (k + e < k1 && c < rows) q = *(const unsigned long long*)(p + e * ld);
            __builtin_memcpy(&v[i][e * COLS], &q, 8);
          }
        } else {
          // (columns behind `rows`: results that nobody stores.)  One branch around the eight loads: a branch to each, and they wait for
          // one another (weight gradient of 50 k rows, 75 and 133 wide, fp16: 36 us, 19.6 us now)
#pragma unroll
          for (int e = 0; e < 8 * COLS; ++e) v[i][e] = (T)0.f;
          if (c < rows && (k1 - k - 7) * ld - c >= COLS) {
#pragma unroll
            for (int e = 0; e < 8; ++e) __builtin_memcpy(&v[i][e * COLS], p + e * ld, COLS * sizeof(T));
          } else if (c < rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
              for (int j = 0; j < COLS; ++j)
                if (k + e < k1 && c + j < rows) v[i][e * COLS + j] = p[e * ld + j];
          }
        }
      }
    }
    if (!STRIDED && !vec) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int unit = threadIdx.x + 256 * i;
        const int64_t k = k0 + (unit % CH) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = k + e < k1 ? v[i][e] : (T)0.f;
      }
    }
  }
  __device__ __forceinline__ void put(gm_u32x4* __restrict__ lds) const {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int unit = threadIdx.x + 256 * i;
      if (UNITS % 256 != 0 && unit >= UNITS) continue;
#pragma unroll
      for (int j = 0; j < (STRIDED ? COLS : 1); ++j) {
        T w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = v[i][STRIDED ? e * COLS + j : e];
        LinChunk<T> c;
        lin_pack(w, c);
        const int r = STRIDED ? (unit % (ROWS / COLS)) * COLS + j : unit / CH, ch = STRIDED ? unit / (ROWS / COLS) : unit % CH;
#pragma unroll
        for (int p = 0; p < PLANES; ++p) lds[p * ROWS * CH + lin_at<CH>(r, ch)] = c.p[p];
      }
    }
  }
};

template <typename T, int ROWS>
__device__ __forceinline__ LinChunk<T> lin_fragment(const gm_u32x4* __restrict__ lds, int row, int ch) {
  constexpr int CH = LinType<T>::BK / 8;
  LinChunk<T> c;
#pragma unroll
  for (int p = 0; p < LinType<T>::PLANES; ++p) c.p[p] = lds[p * ROWS * CH + lin_at<CH>(row, ch)];
  return c;
}

// What becomes of eight neighbouring columns of a row of a product (gm_epilogue)
template <typename T, int MODE>
struct LinEpilogue {
  static constexpr bool COLUMN_SUMS = MODE == LIN_DZ, FUSED = MODE == LIN_FWD || MODE == LIN_DZ;
  struct Row {
    float x[FUSED ? 8 : 1];
  };
  LinArgs a;
  int split, valid;
  int64_t c;
  float b[FUSED ? 8 : 1];
  float zs[COLUMN_SUMS ? 8 : 1];  // sums of dz over the lane's rows, before its rounding: the bias gradient's

  __device__ __forceinline__ void block(int64_t first_column, int split_, int64_t) {
    split = split_;
    c = first_column;
    valid = a.n - c < 8 ? (int)(a.n - c) : 8;
#pragma unroll
    for (int e = 0; e < (FUSED ? 8 : 1); ++e) b[e] = FUSED && a.bias && e < valid ? (float)((const T*)a.bias)[c + e] : 0.f;
#pragma unroll
    for (int e = 0; e < (COLUMN_SUMS ? 8 : 1); ++e) zs[e] = 0.f;
  }
  __device__ __forceinline__ void load(int64_t r, Row& w) const {
    if constexpr (FUSED) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w.x[e] = 0.f;
      if (!a.extra || r >= a.m) return;
      const T* p = (const T*)a.extra + r * a.n + c;
      if (a.n % 8 == 0) {  // (uniform)
        if (valid > 0) pp_load_any<T, 8>(p, w.x);
      } else if (valid == 8) {
        pp_load_any<T, 8>(p, w.x);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < valid) w.x[e] = (float)p[e];
      }
    }
  }
  __device__ __forceinline__ void put(int64_t r, Row& w, float (&v)[8]) {
    if (r >= a.m) return;
    if constexpr (FUSED) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += b[e];
      if (MODE == LIN_FWD) {
        pp_act(v, a.act, a.slope);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += w.x[e];
      } else {
        pp_dact(w.x, v, a.act, a.slope);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = e < valid ? w.x[e] : 0.f;  // (padding is 0, whatever the row holds)
          zs[e] += v[e];
        }
      }
    }
    if constexpr (MODE == LIN_PART) {
      store<float>(a.part + ((int64_t)split * a.m + r) * a.n + c, v, valid);
    } else {
      store<T>((T*)a.out + r * a.ldo + c, v, (int)(a.n_out - c < 8 ? a.n_out - c : 8));
    }
  }
  template <typename O>
  __device__ __forceinline__ void store(O* __restrict__ o, const float (&v)[8], int count) const {
    if ((MODE == LIN_PART ? a.n : a.n_out) % 8 == 0) {  // (uniform)
      if (count > 0) pp_store_any<O, 8>(o, v);
    } else if (count == 8) {
      pp_store_any<O, 8>(o, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) o[e] = (O)v[e];
    }
  }
  // column sums of a BM x BN tile: the lanes of a column, then the waves above each other.  red: LDS that nobody reads any more
  template <int BM, int BN, int WM, int WN>
  __device__ __forceinline__ void done(float* red, int wm, int wn, int64_t n0, int64_t row_tile) {
    if (!a.part_bias) return;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = zs[e];
#pragma unroll
      for (int d = 8; d < 64; d <<= 1) v += __shfl_xor(v, d);
      if (lane < 8) red[wm / WM * BN + wn + 8 * lane + e] = v;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < BN; t += blockDim.x)
      if (n0 + t < a.n) {
        float v = 0.f;
        for (int q = 0; q < BM / WM; ++q) v += red[q * BN + t];
        a.part_bias[row_tile * a.n + n0 + t] = v;
      }
  }
};

// fp32: where a term is infinite, NaN or so large that its first plane overflows, its planes make the products NaN.  Such results of a wave are
// made again from the operands as they are, one multiplication and addition at a time (in fp64: a sum that fp32 holds is not lost half
// way).  In front of the epilogue: inside its loop it made 325 k x 96 -> 96 training 2 % longer
// (8192 x 1024 -> 1024 forward 0.12 ms, 0.15 with a NaN in every row, where a sum ends at it, 8.3 with an infinity in every row)
template <bool AS, bool BS, int FM, int FN>
__device__ __forceinline__ void lin_exact(const LinArgs& a, gm_f32x4 (&acc)[FM][FN], int64_t row0, int64_t col0, int64_t k0, int64_t k1) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) sum += (acc[i][j][0] + acc[i][j][1]) + (acc[i][j][2] + acc[i][j][3]);
  if (!__any(sum != sum)) return;
  const int lane = threadIdx.x & 63;
  const float *A = (const float*)a.a, *B = (const float*)a.b;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int64_t r = row0 + 16 * i + (lane & 15), c = col0 + 16 * j + 4 * (lane >> 4);
      float any = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) any += acc[i][j][e];
      if (any == any || r >= a.m) continue;
      double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 1
      for (int64_t k = k0; k < k1; k += 4) {  // (four terms of four results on their way at once: an operand may hold infinities in every row)
        float x[4], y[4][4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          x[h] = k + h < k1 ? A[AS ? (k + h) * a.lda + r : r * a.lda + k + h] : 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) y[h][e] = k + h < k1 && c + e < a.n ? B[BS ? (k + h) * a.ldb + c + e : (c + e) * a.ldb + k + h] : 0.f;
        }
        bool done = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int h = 0; h < 4; ++h) s[e] = fma((double)x[h], (double)y[h][e], s[e]);
          done &= s[e] != s[e];
        }
        if (done) break;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = acc[i][j][e] == acc[i][j][e] ? acc[i][j][e] : (float)s[e];
    }
}

// BM x BN tile, four waves of WM x WN each.  AS / BS: the contraction runs down the columns of A / B
template <typename T, bool AS, bool BS, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(256, 2) void k_linear_tile(LinArgs a) {
  constexpr int BK = LinType<T>::BK, CH = BK / 8, PLANES = LinType<T>::PLANES, BUFS = LinType<T>::BUFS;
  constexpr int FM = WM / 16, FN = WN / 16, STEP = PLANES * (BM + BN) * CH;
  __shared__ gm_u32x4 lds[BUFS * STEP];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
  const int64_t m0 = (int64_t)blockIdx.x * BM;
  const int n0 = blockIdx.y * BN;
  int64_t k = 0, k1 = a.k;
  if (MODE == LIN_PART) {
    k = (int64_t)blockIdx.z * a.k_per_split;
    k1 = k + a.k_per_split < a.k ? k + a.k_per_split : a.k;
  }
  const int64_t k0 = k;
  const T *pa = (const T*)a.a, *pb = (const T*)a.b;
  gm_f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = (gm_f32x4){0.f, 0.f, 0.f, 0.f};
  LinStage<T, AS, BM> sa;
  LinStage<T, BS, BN> sb;
  if (k < k1) {
    sa.load(pa, a.lda, m0, a.m, k, k1, a.va);
    sb.load(pb, a.ldb, n0, a.n, k, k1, a.vb);
  }
  for (int step = 0; k < k1; k += BK, ++step) {
    gm_u32x4* const at = lds + (BUFS == 2 ? (step & 1) * STEP : 0);
    if (BUFS == 1) __syncthreads();  // the last step's fragments have been read
    sa.put(at);
    sb.put(at + PLANES * BM * CH);
    __syncthreads();
    if (k + BK < k1) {
      sa.load(pa, a.lda, m0, a.m, k + BK, k1, a.va);
      sb.load(pb, a.ldb, n0, a.n, k + BK, k1, a.vb);
    }
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      const int ch = kk * 4 + (lane >> 4);
      LinChunk<T> fb[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[j] = lin_fragment<T, BN>(at + PLANES * BM * CH, wn + 16 * j + (lane & 15), ch);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const LinChunk<T> fa = lin_fragment<T, BM>(at, wm + 16 * i + (lane & 15), ch);
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = lin_mma(fb[j], fa, acc[i][j]);  // B first: a lane gets four neighbours of one row
      }
    }
  }
  if constexpr (sizeof(T) == 4) lin_exact<AS, BS, FM, FN>(a, acc, m0 + wm, n0 + wn, k0, k1);
  LinEpilogue<T, MODE> epi;
  epi.a = a;
  __syncthreads();
  gm_epilogue<FM, FN, 32>(epi, acc, (float*)lds + wave * 32 * 64, m0 + wm, n0 + wn, blockIdx.z, 0);
  if constexpr (MODE == LIN_DZ) {
    __syncthreads();
    epi.template done<BM, BN, WM, WN>((float*)lds, wm, wn, n0, blockIdx.x);
  }
}

// ---- narrow layers over many rows, 16 bits --------------------------------------------------------------------------------------------------------
// Up to 160 channels either side the weights fit the LDS, in the order of their fragments, and a wave needs nothing but 16 rows at a time:
// they go from memory into the registers of the MFMA operand (lane (l & 15, l >> 4): row l & 15, eight neighbouring channels), the next 16
// are asked for before these are multiplied, no barrier, no LDS traffic but the weights'.  The result has row l & 15 in a lane and four
// neighbouring columns of every 16, and goes to memory from there.
// Backward the two layers of the chain meet in the registers: dz is made where z comes out, and the columns 32 t + 4 q + (0 .. 3) and 16 + that
// of a lane are, as they lie, its eight elements of the operand of dx = dz W over a contraction step of 32 -- in an order of their own, which
// the fragments of W^T are laid out in.  dz is written for the weight gradient only.
// Bound: memory where the activation leaves it (64 -> 64: 16 rows are 4 KB, 580 cycles of a compute unit's share of the bandwidth, against 16
// MFMAs of 16 cycles and 400 cycles of GELU on one of four SIMDs): no load of the loop is masked but the row's last eight elements, no store
// but the last columns', and only the tensor's very end is read one by one -- masks of every load took 1.38 times as long at 160 -> 160.
// KB, NB: at least the 32-channel steps of cin and cout; kb, nb: these.
#define LIN_STREAM_WAVES 8
struct LinStreamArgs {
  const void *x, *w, *bias, *extra;  // extra: the residual forward, dy backward; [n, cout]
  int64_t n, ldz;
  int cin, cout, kb, nb, act;
  float slope;
  void *y, *dx, *dz;                 // y forward; backward dx and dz (nullable both; [n, ldz])
  float* part_bias;                  // backward [grid][cout], nullable
};

// N elements of a tensor of `total` from any place in it, in one access but at its very end (zeros behind it)
template <typename T, int N>
__device__ __forceinline__ typename PPVec<T, N>::type lin_take(const T* __restrict__ base, int64_t at, int64_t total) {
  typename PPVec<T, N>::type q;
  if (at + N <= total) {
    __builtin_memcpy(&q, base + at, sizeof(q));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = at + e < total ? base[at + e] : (T)0.f;
  }
  return q;
}
// four of a row's 16 columns from `at` on, of which `count` (the same in every lane) exist
template <typename T>
__device__ __forceinline__ void lin_put4(T* __restrict__ p, const float (&v)[4], int count, int at) {
  if (count >= 16 || at + 4 <= count) {
    pp_store_any<T, 4>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (at + e < count) p[e] = (T)v[e];
  }
}
template <typename T>
__device__ __forceinline__ LinChunk<T> lin_chunk(typename PPVec<T, 8>::type q) {
  T v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = q[e];
  LinChunk<T> c;
  lin_pack(v, c);
  return c;
}

template <typename T, int KB, int NB, bool BACKWARD>
__global__ __launch_bounds__(64 * LIN_STREAM_WAVES, 2) void k_linear_stream(LinStreamArgs a) {
  static_assert(sizeof(T) == 2, "one plane");
  extern __shared__ gm_u32x4 frag[];  // W: [kb][2 nb][64]; backward W^T: [nb][2 kb][64]; bias fp32 [32 nb]
  typedef typename PPVec<T, 8>::type Vec8;
  typedef typename PPVec<T, 4>::type Vec4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, q = lane >> 4;
  const int NT = 2 * a.nb, KT = 2 * a.kb;
  gm_u32x4* const back = frag + (size_t)a.kb * NT * 64;
  float* const bias = (float*)(back + (BACKWARD ? (size_t)a.nb * KT * 64 : 0));
  const T* const w = (const T*)a.w;
  const int64_t tiles = (a.n + 15) / 16, stride = (int64_t)gridDim.x * LIN_STREAM_WAVES;
  const bool want_z = !BACKWARD || a.act != PP_ACT_NONE;
  Vec8 xn[KB];
  Vec4 en[2 * NB];
  float zs[BACKWARD ? 2 * NB : 1][4] = {};
  const int64_t x_end = a.n * a.cin, e_end = a.n * a.cout;
  gm_u32x4 tail;  // what of the last step's eight elements lies in the row
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int left = a.cin - 32 * (a.kb - 1) - 8 * q - 2 * e;
    tail[e] = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
  }
  // (a row behind the last reads the last one and stores nothing; columns behind the last are dropped)
  auto ask = [&](int64_t tile) {
    const int64_t r = tile * 16 + j < a.n ? tile * 16 + j : a.n - 1;
    if (want_z) {
#pragma unroll
      for (int s = 0; s < KB; ++s)
        if (s < a.kb) xn[s] = lin_take<T, 8>((const T*)a.x, r * a.cin + 32 * s + 8 * q, x_end);
    }
    if (a.extra) {
#pragma unroll
      for (int t = 0; t < 2 * NB; ++t)
        if (t < NT) en[t] = lin_take<T, 4>((const T*)a.extra, r * a.cout + 16 * t + 4 * q, e_end);
    }
  };
  int64_t tile = (int64_t)blockIdx.x * LIN_STREAM_WAVES + wave;
  if (!BACKWARD && tile < tiles) ask(tile);
  for (int i = threadIdx.x; i < a.kb * NT * 64; i += blockDim.x) {
    const int l = i & 63, t = i >> 6, r = t % NT * 16 + (l & 15), k = t / NT * 32 + 8 * (l >> 4);
    Vec8 v = lin_take<T, 8>(w, r < a.cout ? r * a.cin + k : a.cout * a.cin, a.cout * a.cin);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < a.cin ? v[e] : (T)0.f;
    frag[i] = lin_chunk<T>(v).p[0];
  }
  if (BACKWARD && a.dx)
    for (int i = threadIdx.x; i < a.nb * KT * 64; i += blockDim.x) {
      const int l = i & 63, t = i >> 6, m = t % KT * 16 + (l & 15), k = t / KT * 32 + 4 * (l >> 4);
      Vec8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int o = k + (e < 4 ? e : 12 + e);
        v[e] = o < a.cout && m < a.cin ? w[(int64_t)o * a.cin + m] : (T)0.f;
      }
      back[i] = lin_chunk<T>(v).p[0];
    }
  for (int i = threadIdx.x; i < 32 * a.nb; i += blockDim.x) bias[i] = a.bias && i < a.cout ? (float)((const T*)a.bias)[i] : 0.f;
  __syncthreads();
  if (BACKWARD && tile < tiles) ask(tile);
  for (; tile < tiles; tile += stride) {
    const int64_t r = tile * 16 + j;
    gm_f32x4 acc[2 * NB];
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) acc[t] = (gm_f32x4){0.f, 0.f, 0.f, 0.f};
    Vec4 ex[2 * NB];
#pragma unroll
    for (int t = 0; t < 2 * NB; ++t) ex[t] = en[t];
    LinChunk<T> xc[KB];
    if (want_z) {
#pragma unroll
      for (int s = 0; s < KB; ++s)
        if (s < a.kb) {
          xc[s] = lin_chunk<T>(xn[s]);
          if (s == a.kb - 1) xc[s].p[0] &= tail;
        }
    }
    if (tile + stride < tiles) ask(tile + stride);
    if (want_z) {
#pragma unroll
      for (int s = 0; s < KB; ++s)
        if (s < a.kb) {
#pragma unroll
          for (int t = 0; t < 2 * NB; ++t)
            if (t < NT) {
              LinChunk<T> f;
              f.p[0] = frag[(s * NT + t) * 64 + lane];
              acc[t] = lin_mma(f, xc[s], acc[t]);
            }
        }
    }
    if constexpr (!BACKWARD) {
#pragma unroll
      for (int t = 0; t < 2 * NB; ++t)
        if (t < NT) {
          const int c = 16 * t + 4 * q;
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = acc[t][e] + bias[c + e];
          pp_act(v, a.act, a.slope);
          if (a.extra) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += (float)ex[t][e];
          }
          if (r < a.n) lin_put4<T>((T*)a.y + r * a.cout + c, v, a.cout - 16 * t, 4 * q);
        }
    } else {
      LinChunk<T> dc[NB];
#pragma unroll
      for (int u = 0; u < NB; ++u)
        if (u < a.nb) {
          Vec8 d;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int t = 2 * u + h, c = 16 * t + 4 * q;
            float z[4], g[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              z[e] = acc[t][e] + bias[c + e];
              g[e] = (float)ex[t][e];  // (0 behind the last row and column, whatever z is)
            }
            pp_dact(g, z, a.act, a.slope);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              g[e] = r < a.n && c + e < a.cout ? g[e] : 0.f;
              zs[t][e] += g[e];
              d[4 * h + e] = (T)g[e];
            }
            if (a.dz && r < a.n) lin_put4<T>((T*)a.dz + r * a.ldz + c, g, (int)a.ldz - 16 * t, 4 * q);
          }
          dc[u] = lin_chunk<T>(d);
        }
      if (a.dx) {
#pragma unroll
        for (int t = 0; t < 2 * KB; ++t)
          if (t < KT) {
            gm_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < NB; ++u)
              if (u < a.nb) {
                LinChunk<T> f;
                f.p[0] = back[(u * KT + t) * 64 + lane];
                s = lin_mma(f, dc[u], s);
              }
            const int c = 16 * t + 4 * q;
            const float v[4] = {s[0], s[1], s[2], s[3]};
            if (r < a.n) lin_put4<T>((T*)a.dx + r * a.cin + c, v, a.cin - 16 * t, 4 * q);
          }
      }
    }
  }
  if constexpr (BACKWARD) {
    if (a.part_bias) {  // a column's rows in a wave, then the waves, in order
      float* const red = (float*)frag;
      __syncthreads();
#pragma unroll
      for (int t = 0; t < 2 * NB; ++t)
        if (t < NT) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = zs[t][e];
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d);
            if (j == 0) red[wave * NT * 16 + 16 * t + 4 * q + e] = v;
          }
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.cout; c += blockDim.x) {
        float v = 0.f;
        for (int k = 0; k < LIN_STREAM_WAVES; ++k) v += red[k * NT * 16 + c];
        a.part_bias[(int64_t)blockIdx.x * a.cout + c] = v;
      }
    }
  }
}

// out[i] = sum of part[q][i] over the q of this group (blockIdx.y of gridDim.y), S slices of a block's threads over q, added in order
template <typename T>
__global__ __launch_bounds__(256) void k_linear_sum(const float* __restrict__ part, int64_t parts, int64_t n, int S, T* __restrict__ out) {
  __shared__ double red[256];
  const int cols = 256 / S, cl = threadIdx.x % cols, sl = threadIdx.x / cols;
  const int64_t i = (int64_t)blockIdx.x * cols + cl;
  const int64_t per = (parts + gridDim.y - 1) / gridDim.y, q0 = blockIdx.y * per, q1 = q0 + per < parts ? q0 + per : parts;
  double s = 0.0;
  if (i < n) {
#pragma unroll 4
    for (int64_t q = q0 + sl; q < q1; q += S) s += (double)part[q * n + i];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (sl == 0 && i < n) {
    for (int k = 1; k < S; ++k) s += red[k * cols + cl];
    out[(int64_t)blockIdx.y * n + i] = (T)(float)s;
  }
}

// the same for few parts of a large matrix: four neighbouring values a thread
template <typename T>
__global__ __launch_bounds__(256) void k_linear_sum4(const float* __restrict__ part, int parts, int64_t n, T* __restrict__ out) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 4
  for (int q = 0; q < parts; ++q) {
    const float4 v = *(const float4*)(part + q * n + i);
    s[0] += (double)v.x;
    s[1] += (double)v.y;
    s[2] += (double)v.z;
    s[3] += (double)v.w;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) out[i + e] = (T)(float)s[e];
}

// column sums of a part of the rows of [n, c]: part[blockIdx.y][c]; 64 columns a block, four rows side by side.  In fp64: a thread's rows grow
// with n, and sums of one sign in fp32 would lose n 2^-25 / 1024 of them (dy of 0.1, 10 M rows: 3.7e-4)
template <typename T>
__global__ __launch_bounds__(256) void k_linear_columns(const T* __restrict__ x, int64_t n, int c, int64_t rows_per_part, float* __restrict__ part) {
  __shared__ double red[256];
  const int col = blockIdx.x * 64 + (threadIdx.x & 63), rl = threadIdx.x >> 6;
  const int64_t r0 = blockIdx.y * rows_per_part, r1 = r0 + rows_per_part < n ? r0 + rows_per_part : n;
  double s = 0.0;
  if (col < c) {
#pragma unroll 8
    for (int64_t r = r0 + rl; r < r1; r += 4) s += (double)(float)x[r * c + col];
  }
  red[threadIdx.x] = s;
  __syncthreads();
  if (rl == 0 && col < c) part[(int64_t)blockIdx.y * c + col] = (float)(red[threadIdx.x] + red[threadIdx.x + 64] + red[threadIdx.x + 128] + red[threadIdx.x + 192]);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------
template <typename T, bool AS, bool BS, int MODE, int BM, int BN, int WM, int WN>
static int lin_go(const LinArgs& a, int splits, hipStream_t s) {
  const int64_t mt = (a.m + BM - 1) / BM;
  const int nt = ((MODE == LIN_DZ ? a.n_out : a.n) + BN - 1) / BN;
  PP_REQUIRE(mt <= 0x7FFFFFFF && nt <= 65535 && splits <= 65535, "pp_linear_act: too many tiles");
  hipLaunchKernelGGL((k_linear_tile<T, AS, BS, MODE, BM, BN, WM, WN>), dim3((unsigned)mt, nt, splits), dim3(256), 0, s, a);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
static bool lin_aligned(const void* p, int64_t ld, int bytes, size_t size) { return (uintptr_t)p % bytes == 0 && (ld * size) % bytes == 0; }

// The wide kernel (pp_gemm.h) serves 16-bit operands whose rows start on 16 bytes, where the matrix pipe bounds: from 192 columns and
// 128 of the contraction on (narrower results spend their time on reading A once, which the tile kernel above does as well)
#define LIN_WIDE_COLUMNS 192
template <typename T, bool AS, bool BS, int MODE>
static bool lin_wide(const LinArgs& a) {
  if (sizeof(T) != 2) return false;
  return a.n >= LIN_WIDE_COLUMNS && a.k >= 128 && a.m >= 128 && lin_aligned(a.a, a.lda, 16, 2) && lin_aligned(a.b, a.ldb, 16, 2) && a.n_out == a.n;
}
static int64_t lin_tiles(int64_t m, int64_t n, int t) { return ((m + t - 1) / t) * ((n + t - 1) / t); }

template <typename T, bool AS, bool BS, int MODE, int BM, int BN, int WM, int WN>
static int lin_go_wide(const LinArgs& a, int splits, hipStream_t s) {
  LinEpilogue<T, MODE> e{};
  e.a = a;
  GemmArgs g{};
  g.a[0] = a.a; g.b[0] = a.b; g.segments = 1; g.m = a.m; g.n = a.n; g.k = a.k; g.lda = a.lda; g.ldb = a.ldb;
  g.splits = splits; g.k_per_split = splits > 1 ? a.k_per_split : (a.k + GM_BK - 1) / GM_BK * GM_BK;
  const int64_t tiles = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
  PP_REQUIRE(tiles <= 0x7FFFFFFF && splits <= 65535, "pp_linear_act: too many tiles");
  hipLaunchKernelGGL((k_gemm<T, AS, BS, BM, BN, WM, WN, LinEpilogue<T, MODE>>), dim3((unsigned)tiles, splits, 1),
                     dim3(BM / WM * (BN / WN) * 64), 0, s, g, e);
  PP_LAUNCH_CHECK();
  return PP_OK;
}

// rows of a workgroup's tile.  Two 128 x 128 workgroups on a compute unit run the loop faster than one of 256 x 256 (contraction 4096,
// 8192 x 1024 results: 66 against 117 us), but a tile costs its start and its epilogue: with contractions below 2048 and enough tiles for
// the chip the large ones win (1024, 8192 x 4096: 86 against 115 us)
template <typename T, bool AS, bool BS, int MODE>
static int lin_tile_rows(const LinArgs& a) {
  return lin_wide<T, AS, BS, MODE>(a) && MODE != LIN_PART && a.k < 2048 && lin_tiles(a.m, a.n, 256) >= 192 ? 256 : 128;
}
template <typename T, bool AS, bool BS, int MODE>
static int lin_tile(const LinArgs& a, int splits, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (lin_wide<T, AS, BS, MODE>(a)) {
      if constexpr (MODE != LIN_PART)
        if (lin_tile_rows<T, AS, BS, MODE>(a) == 256) return lin_go_wide<T, AS, BS, MODE, 256, 256, 128, 64>(a, splits, s);
      return lin_go_wide<T, AS, BS, MODE, 128, 128, 64, 64>(a, splits, s);
    }
  }
  if (a.n > 64) return lin_go<T, AS, BS, MODE, 128, 128, 64, 64>(a, splits, s);
  return lin_go<T, AS, BS, MODE, 128, 64, 32, 64>(a, splits, s);
}


// parts of the weight gradient's contraction: about two workgroups per compute unit, at least 256 rows (wide kernel: 512) each, and at most
// as many as a chain of fp32 additions stands: 2048 in fp32 (64 steps of six: terms of one sign lose 384 2^-24 of their sum at most; they
// lost 9e-5 of 10 M rows in 512 parts), 65536 in 16 bits (2048 steps: 2048 2^-24, a quarter of fp16's half step); longer ones where a matrix
// is so wide that its parts would take more room than the rows themselves
static int lin_splits(int64_t n, int cin, int cout, bool wide, size_t bytes) {
  const int64_t tiles = (int64_t)((cout + 127) / 128) * ((cin + (cin > 64 ? 127 : 63)) / (cin > 64 ? 128 : 64));
  const int64_t rows = wide ? 512 : 256, chain = bytes == 4 ? 2048 : 65536, room = (int64_t)cin * cout / ((int64_t)cin + cout);
  const int64_t most = chain > room ? chain : room;
  int64_t s = 512 / tiles;
  if (s > (n + rows - 1) / rows) s = (n + rows - 1) / rows;
  if (s < (n + most - 1) / most) s = (n + most - 1) / most;
  return s < 1 ? 1 : s > 65535 ? 65535 : (int)s;  // (the launch's third dimension)
}
#define LIN_SUM_GROUPS 32
#define LIN_COLUMN_PARTS 512  // at most; a part has at least LIN_COLUMN_ROWS rows
#define LIN_COLUMN_ROWS 1024
#define LIN_STREAM_GRID_MAX 256
// more parts than this are added in LIN_SUM_GROUPS groups first, whose sums lie behind them
#define LIN_SUM_DIRECT 512
static size_t lin_sum_rows(int64_t parts) { return (size_t)(parts > LIN_SUM_DIRECT ? parts + LIN_SUM_GROUPS : parts); }
static int64_t lin_ldz(int cout) { return (cout + 7) / 8 * 8; }

// workgroups of the narrow kernel: what finds room on the chip at once (two of a compute unit forward, up to 96 channels; the registers leave
// one backward).  Backward a lane adds its column's gradients over its tiles in fp32: at most LIN_STREAM_CHAIN of them, so that the sum is off
// by 2^-15 of its terms' at most whatever n is
#define LIN_STREAM_CHAIN 1024
static int64_t lin_stream_grid(int64_t n, bool backward) {
  const int64_t tiles = (n + 16 * LIN_STREAM_WAVES - 1) / (16 * LIN_STREAM_WAVES), long_n = (tiles + LIN_STREAM_CHAIN - 1) / LIN_STREAM_CHAIN;
  const int64_t most = !backward ? 2 * LIN_STREAM_GRID_MAX : long_n > LIN_STREAM_GRID_MAX ? long_n : LIN_STREAM_GRID_MAX;
  return tiles < most ? tiles : most;
}

// rows of the bias gradient's parts: row tiles (or column parts without an activation), or the narrow kernel's workgroups; room to add them
static size_t lin_bias_rows(int64_t n, int act) {
  const size_t tiles = act == PP_ACT_NONE ? LIN_COLUMN_PARTS : (size_t)((n + 127) / 128), stream = (size_t)lin_stream_grid(n, true);
  return (tiles > stream ? tiles : stream) + LIN_SUM_GROUPS;
}

extern "C" size_t pp_linear_act_bwd_workspace(int32_t dtype, int64_t n, int32_t cin, int32_t cout, int32_t act) {
  if (n < 0 || cin < 1 || cout < 1) return 0;
  const int p0 = lin_splits(n, cin, cout, false, pp_dtype_bytes(dtype)), p1 = lin_splits(n, cin, cout, true, pp_dtype_bytes(dtype));
  const size_t parts = lin_sum_rows(p0 > p1 ? p0 : p1);
  const size_t bias = lin_bias_rows(n, act);
  return pp_align(parts * cout * cin * 4) + pp_align(bias * cout * 4) +
         (act == PP_ACT_NONE ? 0 : pp_align((size_t)n * lin_ldz(cout) * pp_dtype_bytes(dtype))) + 256;
}

// sums of `parts` rows of n values (room: lin_sum_rows)
template <typename T>
static int lin_sum(float* part, int64_t parts, int64_t n, T* out, hipStream_t s) {
  if (parts <= 16 && n % 4 == 0 && n >= 65536) {
    hipLaunchKernelGGL((k_linear_sum4<T>), dim3((unsigned)((n / 4 + 255) / 256)), dim3(256), 0, s, part, (int)parts, n, out);
    PP_LAUNCH_CHECK();
    return PP_OK;
  }
  if (parts > LIN_SUM_DIRECT) {
    float* const mid = part + parts * n;
    hipLaunchKernelGGL((k_linear_sum<float>), dim3((unsigned)((n + 15) / 16), LIN_SUM_GROUPS), dim3(256), 0, s, part, parts, n, 16, mid);
    part = mid;
    parts = LIN_SUM_GROUPS;
  }
  int S = 1;
  while (S < 16 && S < parts) S *= 2;
  const int64_t cols = 256 / S;
  hipLaunchKernelGGL((k_linear_sum<T>), dim3((unsigned)((n + cols - 1) / cols), 1), dim3(256), 0, s, part, parts, n, S, out);
  PP_LAUNCH_CHECK();
  return PP_OK;
}

// LDS of the narrow kernel, 0 where the tiles serve: fp32 (its three planes leave room for one workgroup of a compute unit: 300 k x 64 -> 64
// forward 57 us against 45), fewer than 64 rows (16 x 160 -> 160 forward 12.3 : 9.3), and aligned widths that fill the tiles' columns --
// forward, where the rows are wide against the results (fp16 300 k x 128 -> 64 48 us against 38; 96 -> 64 31 : 38, 96 -> 128 56 : 67), or
// where the tiles fill the chip and the waves here have no second 16 rows to read ahead (65536 x 128 -> 128 25 : 17; 8192 rows 11.4 : 11.3,
// 300 k 65 : 68); backward with few rows, where more workgroups share the tiles, and no z is needed (8192 x 64 -> 128 36 : 30, 65536 57 : 59) or
// the weights are large (8192 x 160 -> 160 48 : 42, 65536 82 : 92).  Else this one: 300 k x 160 -> 160 87 : 128 forward, 246 : 345 backward with
// the activation; 75 -> 133 74 : 155 and 183 : 300; 1024 x 96 -> 96 forward 7.1 : 10.1, backward 29 : 32 (160 -> 160 forward 11.9 : 11.0).
#define LIN_STREAM_ROWS 64
template <typename T>
static size_t lin_stream_lds(int64_t n, int cin, int cout, int act, bool backward) {
  if (sizeof(T) != 2 || cin > 160 || cout > 160 || n < LIN_STREAM_ROWS) return 0;
  if (!backward && cin % 8 == 0 && cout % 64 == 0) {
    if (cin > 96 && cout <= 64) return 0;
    if ((cin > 64 || cout > 64) && n >= 32768 && n < 131072) return 0;
  }
  if (backward && n < 65536 && (act == PP_ACT_NONE || (cin > 128 && cout > 128))) return 0;
  const size_t kb = (cin + 31) / 32, nb = (cout + 31) / 32;
  return kb * nb * 2048 * (backward ? 2 : 1) + nb * 128;  // (103 KB at most)
}
template <typename T, int KB, int NB, bool BACKWARD>
static int lin_stream_go(const LinStreamArgs& a, size_t lds, hipStream_t s) {
  PP_HIP(hipFuncSetAttribute((const void*)k_linear_stream<T, KB, NB, BACKWARD>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL((k_linear_stream<T, KB, NB, BACKWARD>), dim3((unsigned)lin_stream_grid(a.n, BACKWARD)), dim3(64 * LIN_STREAM_WAVES), lds, s, a);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
template <typename T, bool BACKWARD>
static int lin_stream(LinStreamArgs& a, size_t lds, hipStream_t s) {
  a.kb = (a.cin + 31) / 32;
  a.nb = (a.cout + 31) / 32;
#define LIN_BY_NB(KB)                                                    \
  return a.nb <= 2   ? lin_stream_go<T, KB, 2, BACKWARD>(a, lds, s)      \
         : a.nb == 3 ? lin_stream_go<T, KB, 3, BACKWARD>(a, lds, s)      \
                     : lin_stream_go<T, KB, 5, BACKWARD>(a, lds, s);
  if (a.kb <= 2) LIN_BY_NB(2)
  if (a.kb == 3) LIN_BY_NB(3)
  LIN_BY_NB(5)
#undef LIN_BY_NB
}

static int lin_check(int32_t dtype, int64_t n, int32_t cin, int32_t cout, int32_t act) {
  PP_REQUIRE(pp_rows_dtype_ok(dtype), "pp_linear_act: unknown element type");
  PP_REQUIRE(pp_rows_act_ok(act), "pp_linear_act: unknown activation");
  PP_REQUIRE(cin >= 1 && cin <= (1 << 20) && cout >= 1 && cout <= (1 << 20), "pp_linear_act: channels out of range");
  PP_REQUIRE(n >= 0 && n < ((int64_t)1 << 31), "pp_linear_act: rows out of range");  // (a launch has less than 2^32 threads)
  return PP_OK;
}

template <typename T>
static LinArgs lin_base(const void* x, int64_t n, int cin, const void* w, int cout, const void* bias, int act, float slope) {
  LinArgs a{};
  a.a = x; a.b = w; a.m = n; a.n = cout; a.k = cin; a.lda = cin; a.ldb = cin;
  a.va = lin_aligned(x, cin, 16, sizeof(T)); a.vb = lin_aligned(w, cin, 16, sizeof(T));
  a.bias = bias; a.act = act; a.slope = slope;
  return a;
}

template <typename T>
static int lin_forward(const void* x, int64_t n, int cin, const void* w, int cout, const void* bias, int act, float slope,
                       const void* residual, void* y, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (const size_t lds = lin_stream_lds<T>(n, cin, cout, act, false)) {
      LinStreamArgs a{};
      a.x = x; a.w = w; a.bias = bias; a.extra = residual; a.n = n; a.cin = cin; a.cout = cout; a.act = act; a.slope = slope; a.y = y;
      return lin_stream<T, false>(a, lds, s);
    }
  LinArgs a = lin_base<T>(x, n, cin, w, cout, bias, act, slope);
  a.extra = residual; a.out = y; a.ldo = cout; a.n_out = cout;
  return lin_tile<T, false, false, LIN_FWD>(a, 1, s);
}

template <typename T>
static int lin_backward(const void* x, const void* dy, int64_t n, int cin, const void* w, int cout, const void* bias, int act, float slope,
                        void* dx, void* dw, void* db, PPArena& ws, hipStream_t s) {
  const int p0 = lin_splits(n, cin, cout, false, sizeof(T)), p1 = lin_splits(n, cin, cout, true, sizeof(T));
  float* part = ws.take<float>(lin_sum_rows(p0 > p1 ? p0 : p1) * cout * cin);
  float* part_bias = ws.take<float>(lin_bias_rows(n, act) * cout);
  PP_REQUIRE(part && part_bias, "pp_linear_act_bwd: workspace layout");
  const T* dz = (const T*)dy;
  int64_t ldz = cout, bias_parts = 0;
  int rc;
  const size_t stream = lin_stream_lds<T>(n, cin, cout, act, true);
  if (stream) {
    LinStreamArgs a{};
    a.x = x; a.w = w; a.bias = bias; a.extra = dy; a.n = n; a.cin = cin; a.cout = cout; a.act = act; a.slope = slope; a.dx = dx;
    if (act != PP_ACT_NONE && dw) {
      ldz = a.ldz = lin_ldz(cout);
      a.dz = ws.take<T>((size_t)n * ldz);
      PP_REQUIRE(a.dz, "pp_linear_act_bwd: workspace layout");
      dz = (const T*)a.dz;
    }
    a.part_bias = db ? part_bias : nullptr;
    bias_parts = lin_stream_grid(n, true);
    if constexpr (sizeof(T) == 2)
      if (dx || db || a.dz)
        if ((rc = lin_stream<T, true>(a, stream, s)) != PP_OK) return rc;
  } else if (act != PP_ACT_NONE) {
    ldz = lin_ldz(cout);
    T* z = ws.take<T>((size_t)n * ldz);
    PP_REQUIRE(z || n == 0, "pp_linear_act_bwd: workspace layout");
    dz = z;
    if (n) {
      LinArgs a = lin_base<T>(x, n, cin, w, cout, bias, act, slope);
      a.extra = dy; a.out = z; a.ldo = ldz; a.n_out = (int)ldz;
      a.part_bias = db ? part_bias : nullptr;
      const int rows = lin_tile_rows<T, false, false, LIN_DZ>(a);
      bias_parts = (n + rows - 1) / rows;
      if ((rc = lin_tile<T, false, false, LIN_DZ>(a, 1, s)) != PP_OK) return rc;
    }
  } else if (db && n) {
    bias_parts = (n + LIN_COLUMN_ROWS - 1) / LIN_COLUMN_ROWS;
    if (bias_parts > LIN_COLUMN_PARTS) bias_parts = LIN_COLUMN_PARTS;
    hipLaunchKernelGGL((k_linear_columns<T>), dim3((unsigned)((cout + 63) / 64), (unsigned)bias_parts), dim3(256), 0, s, (const T*)dy, n, cout,
                       (n + bias_parts - 1) / bias_parts, part_bias);
    PP_LAUNCH_CHECK();
  }
  if (dx && n && !stream) {
    LinArgs a{};
    a.a = dz; a.lda = ldz; a.b = w; a.ldb = cin; a.m = n; a.n = cin; a.k = cout; a.out = dx; a.ldo = cin; a.n_out = cin;
    a.va = lin_aligned(dz, ldz, 16, sizeof(T)); a.vb = lin_aligned(w, cin, 8, sizeof(T));
    if ((rc = lin_tile<T, false, true, LIN_STORE>(a, 1, s)) != PP_OK) return rc;
  }
  if (dw) {
    LinArgs a{};
    a.a = dz; a.lda = ldz; a.b = x; a.ldb = cin; a.m = cout; a.n = cin; a.k = n;
    a.va = lin_aligned(dz, ldz, 8, sizeof(T)); a.vb = lin_aligned(x, cin, 8, sizeof(T));
    a.part = part; a.n_out = cin;
    const int splits = lin_wide<T, true, true, LIN_PART>(a) ? p1 : p0;
    a.k_per_split = ((n + splits - 1) / splits + 63) / 64 * 64;
    if ((rc = lin_tile<T, true, true, LIN_PART>(a, splits, s)) != PP_OK) return rc;
    if ((rc = lin_sum<T>(part, splits, (int64_t)cout * cin, (T*)dw, s)) != PP_OK) return rc;
  }
  return db ? lin_sum<T>(part_bias, bias_parts, cout, (T*)db, s) : PP_OK;
}

extern "C" int pp_linear_act_fwd(const void* x, int32_t dtype, int64_t n, int32_t cin, const void* weight, int32_t cout, const void* bias,
                                 int32_t act, float slope, const void* residual, void* y, pp_stream_t stream) {
  int rc = lin_check(dtype, n, cin, cout, act);
  if (rc != PP_OK) return rc;
  PP_REQUIRE(weight && (n == 0 || (x && y)), "pp_linear_act_fwd: null pointer");
  if (n == 0) return PP_OK;
  hipStream_t s = pp_s(stream);
  if (dtype == PP_F32) return lin_forward<float>(x, n, cin, weight, cout, bias, act, slope, residual, y, s);
  if (dtype == PP_BF16) return lin_forward<pp_bf16>(x, n, cin, weight, cout, bias, act, slope, residual, y, s);
  return lin_forward<pp_f16>(x, n, cin, weight, cout, bias, act, slope, residual, y, s);
}

extern "C" int pp_linear_act_bwd(const void* x, const void* dy, int32_t dtype, int64_t n, int32_t cin, const void* weight, int32_t cout,
                                 const void* bias, int32_t act, float slope, void* dx, void* dweight, void* dbias, void* ws,
                                 size_t ws_bytes, pp_stream_t stream) {
  int rc = lin_check(dtype, n, cin, cout, act);
  if (rc != PP_OK) return rc;
  PP_REQUIRE(weight && ws && (n == 0 || (x && dy)), "pp_linear_act_bwd: null pointer");
  PP_REQUIRE((uintptr_t)ws % 16 == 0, "pp_linear_act_bwd: the workspace must be 16-byte aligned");
  if (ws_bytes < pp_linear_act_bwd_workspace(dtype, n, cin, cout, act)) {
    pp_set_error("pp_linear_act_bwd: workspace too small");
    return PP_ERR_WORKSPACE;
  }
  PPArena arena(ws, ws_bytes);
  hipStream_t s = pp_s(stream);
  if (dtype == PP_F32) return lin_backward<float>(x, dy, n, cin, weight, cout, bias, act, slope, dx, dweight, dbias, arena, s);
  if (dtype == PP_BF16) return lin_backward<pp_bf16>(x, dy, n, cin, weight, cout, bias, act, slope, dx, dweight, dbias, arena, s);
  return lin_backward<pp_f16>(x, dy, n, cin, weight, cout, bias, act, slope, dx, dweight, dbias, arena, s);
}

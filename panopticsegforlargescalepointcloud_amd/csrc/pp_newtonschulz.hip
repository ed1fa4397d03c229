// Orthogonalisation of a batch of matrices by Newton-Schulz products: X = G / (|G| + eps), then `steps` times
//   X <- X (a I + b S + c S^2),  S = X^T X                  (on the shorter side: S = X X^T, X from the left, where G is wide)
// Two forms.  Up to a short side of NS_PANEL_MAX: all of it is a polynomial of the first S.  With P = a I + b S + c S^2 the next S is P S P, and the result is X Q with Q the product
// of all P: the long matrix is read twice (for S, and to be multiplied by Q) instead of three times a step, and the steps work on
// matrices of the short side only.  S, P and Q are symmetric and commute, so half of each product's tiles is computed and mirrored.
// S is held and multiplied in fp64: in the directions of small singular values P is a I, so rounding errors of S grow by a^2 = 11.9 a
// step there; fp64 leaves 1e-12 of them after five steps, fp32 would leave 1e-2.  |G|^2 is the trace of S.  Behind some fifteen steps even
// fp64's errors have grown to the size of S (the Q of directions that G does not have grows by a each step without end), so longer calls
// go in rounds: at most NS_ROUND steps are one, more are rounds of NS_ROUND_LONG, between which X is written in fp32 and S formed anew.
// Above it: the iteration as it is written, on the bf16 matrix pipe with operands in two or three planes (further down).
#include "pp_gemm.h"

typedef double ns_f64x4 __attribute__((ext_vector_type(4)));

// ---- one step in one launch, for a short side of at most NS_PANEL_MAX ------------------------------------------------------------
// All factors are polynomials of S, so a workgroup that holds the whole of S in its LDS can take 16 rows of everything through a step on
// its own: with s, q its rows of S and Q,
//   t = s S, p = a e + b s + c t (rows of P);  u = p S, v = u S, w = v S: the next S's rows  a u + b v + c w  (= P S P, as P = a I + b S + c S^2
//   applied to u from the right);  y = q S, z = y S: the next Q's rows  a q + b y + c z.
// Six small products instead of three whole ones between which every workgroup would have to wait for all others; the rows of S and of Q
// are taken by different workgroups.  SB = 16-column blocks of the padded short side; wave w of eight computes column block w of a panel
// product (waves behind the last block repeat it: no branches around the MFMAs).  A product is N / 4 MFMAs of 64 cycles a wave, two
// waves a SIMD: at N = 96 1.3 us of it, four in a row.
#define NS_PANEL_MAX 128
#define NS_ROUND 8
#define NS_ROUND_LONG 5

template <int SB>
struct NsPanel {
  static constexpr int N = SB * 16, LD = N + 2;  // 16 rows of a panel at one k fall on 16 different pairs of banks
  // out = panel x S, column block cb.  panel: [16][LD], S: [N][N], both in the LDS
  static __device__ __forceinline__ ns_f64x4 multiply(const double* __restrict__ panel, const double* __restrict__ S, int cb) {
    const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
    ns_f64x4 out = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 8
    for (int k = 0; k < N; k += 4) out = __builtin_amdgcn_mfma_f64_16x16x4f64(panel[j * LD + k + q], S[at(k + q, cb * 16 + j)], out, 0, 0, 0);
    return out;
  }
  // four rows k .. k + 3 are read at the same 16 columns (128 bytes): where a row is whole 256 bytes, odd rows' halves are exchanged
  static __device__ __forceinline__ int at(int r, int c) { return r * N + (SB % 2 == 0 ? c ^ ((r & 1) << 4) : c); }
};

struct NsStepArgs {
  const double *S, *Q;  // [batch][s][s]; Q null: the identity times alpha (first step of a round)
  double *S2, *Q2;      // S2 null: not wanted (last step)
  int64_t s;
  double a, b, c;
  double eps;           // first step: S is the unscaled one, alpha = 1 / (sqrt(trace S) + eps)
  int scaled;           // later rounds: S is that of an X of this iteration, alpha = 1
};

// a symmetric [s][s] matrix into the LDS, zeros around it; 512 threads
template <int SB>
__device__ __forceinline__ void ns_square(double* __restrict__ S, const double* __restrict__ gS, int64_t s) {
  typedef NsPanel<SB> P;
  constexpr int N = P::N;
  constexpr int PART = (N * N + 511) / 512 < 16 ? (N * N + 511) / 512 : 16;  // loads in flight
  for (int i0 = threadIdx.x; i0 < N * N; i0 += 512 * PART) {
    double v[PART];
#pragma unroll
    for (int e = 0; e < PART; ++e) {
      const int i = i0 + 512 * e, r = i / N, c = i % N;
      const bool in = i < N * N && r < s && c < s;
      v[e] = gS[in ? r * s + c : 0];
      v[e] = in ? v[e] : 0.0;
    }
#pragma unroll
    for (int e = 0; e < PART; ++e)
      if (i0 + 512 * e < N * N) S[P::at((i0 + 512 * e) / N, (i0 + 512 * e) % N)] = v[e];
  }
}

template <int SB>
__global__ __launch_bounds__(512) void k_ns_step(NsStepArgs g) {
  typedef NsPanel<SB> P;
  constexpr int N = P::N, LD = P::LD;
  extern __shared__ double mem[];
  double *S = mem, *panel = mem + N * N, *red = panel + 16 * LD;  // red: 8
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, q = lane >> 4;
  const int cb = wave < SB ? wave : SB - 1;
  const bool rows_of_q = blockIdx.x < SB;
  const int64_t batch = blockIdx.y, s = g.s, r0 = (rows_of_q ? blockIdx.x : blockIdx.x - SB) * 16;
  const double* gS = g.S + batch * s * s;
  const bool first = g.Q == nullptr;
  ns_square<SB>(S, gS, s);
  double alpha = 1.0;
  __syncthreads();
  if (first && !g.scaled) {
    double v = 0.0;
    for (int i = threadIdx.x; i < N; i += 512) v += S[P::at(i, i)];
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if (lane == 0) red[wave] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < 8; ++w) v += red[w];
    alpha = 1.0 / (sqrt(v) + g.eps);
    for (int i = threadIdx.x; i < N * N; i += 512) S[i] *= alpha * alpha;
    __syncthreads();
  }
#pragma unroll
  for (int i = threadIdx.x; i < 16 * N; i += 512) {
    const int r = i / N, c = i % N;
    double v;
    if (!rows_of_q) {
      v = S[P::at(r0 + r, c)];
    } else if (first) {
      v = r0 + r == c && c < s ? alpha : 0.0;
    } else {
      const bool in = r0 + r < s && c < s;
      v = g.Q[batch * s * s + (in ? (r0 + r) * s + c : 0)];
      v = in ? v : 0.0;
    }
    panel[r * LD + c] = v;
  }
  __syncthreads();
  // a lane's values of a panel: rows q + 4 e of its wave's column
  const int col = cb * 16 + j;
  auto put = [&](const ns_f64x4& v) {
    __syncthreads();  // the panel has been read
    if (wave < SB)
#pragma unroll
      for (int e = 0; e < 4; ++e) panel[(q + 4 * e) * LD + col] = v[e];
    __syncthreads();
  };
  ns_f64x4 keep, t, u;
#pragma unroll
  for (int e = 0; e < 4; ++e) keep[e] = panel[(q + 4 * e) * LD + col];
  t = P::multiply(panel, S, cb);
  double* to = g.S2;
  if (rows_of_q) {
    put(t);
    u = P::multiply(panel, S, cb);
    keep = g.a * keep + g.b * t + g.c * u;
    to = g.Q2;
  } else {
    keep = g.b * keep + g.c * t;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r0 + q + 4 * e == col) keep[e] += g.a;
    put(keep);  // p
    u = P::multiply(panel, S, cb);
    put(u);
    t = P::multiply(panel, S, cb);  // v
    put(t);
    keep = P::multiply(panel, S, cb);  // w
    keep = g.a * u + g.b * t + g.c * keep;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t r = r0 + q + 4 * e;
    if (wave < SB && r < s && col < s) to[(batch * s + r) * s + col] = keep[e];
  }
}

// The long side's two passes for the same short sides.  A part is NS_LONG of the long side by the whole short side, in the LDS as fp32, a
// tall matrix as rows of N, a wide one as rows of NS_LONG.  A fragment is 16 x 4 values: the Gram matrix takes 16 of the short side and 4
// of the long one, the product with Q 16 of the long and 4 of the short side.  Rows are padded so that its values lie on 64 different
// banks (16 along a row: rows 16 apart modulo 64; 4 along a row: 4 apart); at N = 128, where Q leaves no room for it, Q's pass exchanges
// columns instead.
#define NS_LONG 64
template <int SB, bool APPLY>
struct NsPart {
  static constexpr int N = SB * 16;
  static constexpr bool SWAP = APPLY && SB == 8;
  static constexpr int LD_TALL = SWAP ? N : APPLY ? N + 4 : N + (SB % 2 == 0 ? 16 : 0), LD_WIDE = SWAP ? NS_LONG : NS_LONG + (APPLY ? 16 : 4);
  static constexpr int FLOATS = NS_LONG * LD_TALL > N * LD_WIDE ? NS_LONG * LD_TALL : N * LD_WIDE;
  static __device__ __forceinline__ int tall_at(int r, int c) { return r * LD_TALL + (SWAP ? c ^ ((r & 15) << 2) : c); }
  static __device__ __forceinline__ int wide_at(int r, int c) { return r * LD_WIDE + (SWAP ? c ^ ((r & 3) << 4) : c); }
  // element (short i, long k) of the part
  static __device__ __forceinline__ int at(bool tall, int i, int k) { return tall ? tall_at(k, i) : wide_at(i, k); }
  // g: the part's corner, `len` of the long side left; vec: rows may be read four elements at a time
  template <typename T>
  static __device__ __forceinline__ void load(float* __restrict__ x, const T* __restrict__ g, bool tall, int64_t ld, int s, int len, bool vec) {
    const int rows = tall ? NS_LONG : N, cols = tall ? N : NS_LONG, have_rows = tall ? len : s, have_cols = tall ? s : len;
    if (vec) {
      constexpr int PER = (NS_LONG * N / 4 + 511) / 512;
      float v[PER][4];
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int i = threadIdx.x + 512 * e, r = i / (cols / 4), c = i % (cols / 4) * 4;
        const bool in = r < have_rows && c < have_cols;
        pp_load<T, 4>(g + (in ? r * ld + c : 0), v[e]);
#pragma unroll
        for (int u = 0; u < 4; ++u) v[e][u] = in ? v[e][u] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int i = threadIdx.x + 512 * e, r = i / (cols / 4), c = i % (cols / 4) * 4;
        if (r < rows) *(float4*)(x + (tall ? tall_at(r, c) : wide_at(r, c))) = make_float4(v[e][0], v[e][1], v[e][2], v[e][3]);
      }
    } else {
      constexpr int PER = NS_LONG * N / 512;
      float v[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int i = threadIdx.x + 512 * e, r = i / cols, c = i % cols;
        const bool in = r < have_rows && c < have_cols;
        v[e] = (float)g[in ? r * ld + c : 0];
        v[e] = in ? v[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) {
        const int i = threadIdx.x + 512 * e;
        x[tall ? tall_at(i / cols, i % cols) : wide_at(i / cols, i % cols)] = v[e];
      }
    }
  }
};

// S of every splits-th part: its tiles on and below the diagonal, the eight waves in turn.  A workgroup per part as long as all of them find
// room on the chip at once (NS_GRAM_BLOCKS: four of a compute unit), a whole number of parts each behind that: what they leave behind
// for k_ns_sum is s^2 fp64 a workgroup, which a workgroup per part made six times the matrix itself ([4 M, 96] x 6: 27 GB)
#define NS_GRAM_BLOCKS 1024
template <typename T, int SB>
__global__ __launch_bounds__(512) void k_ns_part_gram(const T* __restrict__ g, int64_t m, int64_t n, int splits, int vec, double* __restrict__ part) {
  constexpr int TILES = SB * (SB + 1) / 2, PER = (TILES + 7) / 8;
  typedef NsPart<SB, false> X;
  __shared__ float x[X::FLOATS];
  const bool tall = m >= n;
  const int64_t s = tall ? n : m, l = tall ? m : n, batch = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, q = lane >> 4;
  int ta[PER], tb[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    int t = wave + 8 * i < TILES ? wave + 8 * i : TILES - 1, r = 0;
    while (t > r) t -= ++r;
    ta[i] = r;
    tb[i] = t;
  }
  ns_f64x4 acc[PER] = {};
  for (int64_t l0 = (int64_t)blockIdx.x * NS_LONG; l0 < l; l0 += (int64_t)splits * NS_LONG) {
    X::load(x, g + batch * m * n + (tall ? l0 * n : l0), tall, n, (int)s, (int)(l - l0 < NS_LONG ? l - l0 : NS_LONG), vec);
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < NS_LONG; k += 4)
#pragma unroll
      for (int i = 0; i < PER; ++i)
        acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)x[X::at(tall, ta[i] * 16 + j, k + q)], (double)x[X::at(tall, tb[i] * 16 + j, k + q)],
                                                      acc[i], 0, 0, 0);
    __syncthreads();  // the part has been read
  }
  double* o = part + (batch * splits + blockIdx.x) * s * s;
#pragma unroll
  for (int i = 0; i < PER; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t r = ta[i] * 16 + q + 4 * e, c = tb[i] * 16 + j;
      if (wave + 8 * i < TILES && r < s && c < s) o[r * s + c] = acc[i][e];
    }
}

// out = X Q (tall) or Q X of a part; alpha is in Q
template <typename T, typename O, int SB>
__global__ __launch_bounds__(512) void k_ns_part_apply(const T* __restrict__ g, int64_t m, int64_t n, int vec, const double* __restrict__ Q,
                                                       O* __restrict__ out) {
  typedef NsPanel<SB> P;
  typedef NsPart<SB, true> X;
  constexpr int N = SB * 16, TILES = SB * (NS_LONG / 16), PER = TILES / 8 + (TILES % 8 != 0);
  extern __shared__ double mem[];
  double* const S = mem;
  float* const x = (float*)(mem + N * N);
  const bool tall = m >= n;
  const int64_t s = tall ? n : m, l = tall ? m : n, l0 = (int64_t)blockIdx.x * NS_LONG, batch = blockIdx.y;
  const int64_t corner = batch * m * n + (tall ? l0 * n : l0);
  const int len = (int)(l - l0 < NS_LONG ? l - l0 : NS_LONG);
  ns_square<SB>(S, Q + batch * s * s, s);
  X::load(x, g + corner, tall, n, (int)s, len, vec);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, q = lane >> 4;
  ns_f64x4 acc[PER] = {};
  __syncthreads();
#pragma unroll 4
  for (int k = 0; k < N; k += 4)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int t = wave + 8 * i < TILES ? wave + 8 * i : TILES - 1, tl = t % (NS_LONG / 16), ts = t / (NS_LONG / 16);
      const double xv = (double)x[X::at(tall, k + q, tl * 16 + j)], sv = S[P::at(k + q, ts * 16 + j)];
      acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64(tall ? xv : sv, tall ? sv : xv, acc[i], 0, 0, 0);
    }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int t = wave + 8 * i, tl = t % (NS_LONG / 16), ts = t / (NS_LONG / 16);
    if (t >= TILES) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = (tall ? tl : ts) * 16 + q + 4 * e, c = (tall ? ts : tl) * 16 + j;
      if (r < (tall ? len : (int)s) && c < (tall ? (int)s : len)) out[corner + r * n + c] = (O)(float)acc[i][e];
    }
  }
}

// adds the parts of S in their order (eight slices of a workgroup's threads over the parts), both triangles from the lower one
__global__ __launch_bounds__(256) void k_ns_sum(const double* __restrict__ part, int splits, int64_t s, double* __restrict__ out) {
  __shared__ double red[256];
  const int64_t i = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31), batch = blockIdx.y;
  const int sl = threadIdx.x >> 5;
  const int64_t r = i / s, c = i - r * s;
  const bool in = i < s * s && c <= r;
  double v = 0.0;
  if (in) {
#pragma unroll 4
    for (int q = sl; q < splits; q += 8) v += part[(batch * splits + q) * s * s + i];
  }
  red[threadIdx.x] = v;
  __syncthreads();
  if (sl == 0 && in) {
    for (int k = 1; k < 8; ++k) v += red[k * 32 + threadIdx.x];
    out[batch * s * s + i] = v;
    out[batch * s * s + c * s + r] = v;
  }
}
// ---- short sides above NS_PANEL_MAX -------------------------------------------------------------------------------------------------
// Here the products are large enough for the matrix pipe, and fp64 is 32 times slower than bf16 on it: the iteration runs as it is
// defined, X <- X P with S = X^T X, T = S S, P = a I + b S + c T anew in every step (an error of S is not carried on, so no growth of it
// beyond what the definition has in fp32).  Matrices are sums of bf16 planes, hi + lo (16 bits) for 16-bit results, hi + mid + lo (24
// bits) for fp32 ones; a product takes the plane pairs above the last plane's rounding (3, or 6), on k_gemm.  X starts as G 2^e with 2^e
// the power of two at 1 / (|G| + eps), which needs no rounding (bf16: one plane); the rest of the scale, f in [1, 2), enters the first P.
// Two planes carry 2^-17 of a value (P and X are rounded to them, each step), three 2^-25: below the half step of the results' type.
// S and T: lower tiles, the contraction in parts to fill the chip, added in order where S's and P's planes are made.  All products take
// 128 x 128 tiles (X P at 2 x [1024, 4096]: 57 us, 84 us with 256 x 256 ones, which leave half of the chip without work).

struct NsScale {  // per batch element
  float f, pad;
};

// partial sums of squares of a batch element: part[batch][NS_NORM_PARTS]
#define NS_NORM_PARTS 64
template <typename T>
__global__ __launch_bounds__(256) void k_ns_norm(const T* __restrict__ g, int64_t count, double* __restrict__ part) {
  __shared__ double red[4];
  const T* p = g + (int64_t)blockIdx.y * count;
  double v = 0.0;
  constexpr int W = 16 / (int)sizeof(T);
  const bool vec = count % W == 0 && (uintptr_t)g % 16 == 0;
  const int64_t vecs = vec ? count / W : 0;
#pragma unroll 4
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < vecs; i += NS_NORM_PARTS * 256) {
    float x[W];
    pp_load<T, W>(p + i * W, x);
#pragma unroll
    for (int e = 0; e < W; ++e) v = fma((double)x[e], (double)x[e], v);
  }
#pragma unroll 4
  for (int64_t i = vecs * W + (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += NS_NORM_PARTS * 256) {
    const double x = (double)(float)p[i];
    v = fma(x, x, v);
  }
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) part[(int64_t)blockIdx.y * NS_NORM_PARTS + blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

// v as NP bf16 terms
template <int NP>
__device__ __forceinline__ void ns_planes(float v, pp_bf16 (&p)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    p[i] = (pp_bf16)v;
    v -= (float)p[i];
  }
}

// X = G 2^e in NP planes [m][ld], zeros behind the columns; f of the batch element
template <typename T, int NP>
__global__ __launch_bounds__(256) void k_ns_scale(const T* __restrict__ g, int64_t m, int64_t n, int64_t ld, const double* __restrict__ part,
                                                  double eps, pp_bf16* __restrict__ planes, int64_t plane, NsScale* __restrict__ scale) {
  const int64_t batch = blockIdx.y;
  double v = part[batch * NS_NORM_PARTS + (threadIdx.x & 63)];
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  const double alpha = 1.0 / (sqrt(v) + eps);
  double two = 1.0;
  float f;
  if (alpha > 0.0 && alpha < 1e300) {
    int e;
    f = 2.f * (float)frexp(alpha, &e);
    two = ldexp(1.0, e - 1);
  } else {
    f = (float)alpha;  // 0, infinity or NaN: the result is NaN, as the definition's
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) scale[batch].f = f;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8, r = i / ld, c = i - r * ld;
  if (r >= m) return;
  gm_u32x4 out[NP];
  pp_bf16* const o = (pp_bf16*)out;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    pp_bf16 p[NP];
    ns_planes<NP>(c + k < n ? (float)((double)(float)g[batch * m * n + r * n + c + k] * two) : 0.f, p);
#pragma unroll
    for (int q = 0; q < NP; ++q) o[q * 8 + k] = p[q];
  }
#pragma unroll
  for (int q = 0; q < NP; ++q) *(gm_u32x4*)(planes + q * plane + batch * m * ld + i) = out[q];
}

// epilogue of S and T: the part's fp32 sums
struct NsPartEpilogue {
  static constexpr bool COLUMN_SUMS = false;
  struct Row {};
  float* part;
  int64_t s, ld;
  int splits;
  int64_t c;
  float* o;
  __device__ __forceinline__ void block(int64_t first_column, int split, int64_t batch) {
    c = first_column;
    o = part + (batch * splits + split) * s * ld + c;
  }
  __device__ __forceinline__ void load(int64_t, Row&) const {}
  __device__ __forceinline__ void put(int64_t r, Row&, float (&v)[8]) {
    if (r < s && c < ld) pp_store<float, 8>(o + r * ld, v);
  }
};
// epilogue of X P: the next X's planes, zeros behind the columns, or after the last step the result
template <typename T, int NP>
struct NsXEpilogue {
  static constexpr bool COLUMN_SUMS = false;
  struct Row {};
  pp_bf16* planes;
  int64_t plane, m, n, ld;
  T* out;  // nullable
  int vec;
  int64_t c, at;
  __device__ __forceinline__ void block(int64_t first_column, int, int64_t batch) {
    c = first_column;
    at = batch;
  }
  __device__ __forceinline__ void load(int64_t, Row&) const {}
  __device__ __forceinline__ void put(int64_t r, Row&, float (&v)[8]) {
    if (r >= m || c >= n) return;
    if (out) {
      T* const o = out + (at * m + r) * n + c;
      if (vec) {
        pp_store<T, 8>(o, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < n) o[e] = (T)v[e];
      }
      return;
    }
    gm_u32x4 w[NP];
    pp_bf16* const o = (pp_bf16*)w;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pp_bf16 p[NP];
      ns_planes<NP>(c + e < n ? v[e] : 0.f, p);
#pragma unroll
      for (int q = 0; q < NP; ++q) o[q * 8 + e] = p[q];
    }
#pragma unroll
    for (int q = 0; q < NP; ++q) *(gm_u32x4*)(planes + q * plane + (at * m + r) * ld + c) = w[q];
  }
};

// A 32 x 32 tile on or below the diagonal and its mirror image: adds the parts, then
//   S32 null: S -> planes, S kept in fp32 (to `keep`);   else: P = f (c0 I + c1 f^2 S + c2 f^4 T) -> planes, T the parts' sum
template <int NP>
__global__ __launch_bounds__(256) void k_ns_square(const float* __restrict__ part, int splits, int64_t s, int64_t ld, float* __restrict__ keep,
                                                   const float* __restrict__ S32, const NsScale* __restrict__ scale, double c0, double c1,
                                                   double c2, pp_bf16* __restrict__ planes, int64_t plane) {
  __shared__ float tile[32][33];
  int ti = (int)((sqrtf(8.f * (float)blockIdx.x + 1.f) - 1.f) * 0.5f);
  while ((ti + 1) * (ti + 2) / 2 <= (int)blockIdx.x) ++ti;
  while (ti * (ti + 1) / 2 > (int)blockIdx.x) --ti;
  const int tj = (int)blockIdx.x - ti * (ti + 1) / 2;
  const int64_t batch = blockIdx.y, size = s * ld;
  const int x = threadIdx.x & 31;
  const double f = scale ? (double)scale[batch].f : 1.0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int y = (threadIdx.x >> 5) + 8 * k;
    const int64_t r = ti * 32 + y, c = tj * 32 + x;
    float v = 0.f;
    if (r < s && c < s) {
      float sum = 0.f;
#pragma unroll 4
      for (int q = 0; q < splits; ++q) sum += part[(batch * splits + q) * size + r * ld + c];
      if (S32) {
        const double t = c2 * (f * f) * (f * f) * (double)sum + c1 * (f * f) * (double)S32[batch * size + r * ld + c] + (r == c ? c0 : 0.0);
        v = (float)(f * t);
      } else {
        v = sum;
        keep[batch * size + r * ld + c] = v;
      }
    }
    tile[y][x] = v;
  }
  __syncthreads();
#pragma unroll
  for (int mirror = 0; mirror < 2; ++mirror) {
    if (mirror && ti == tj) break;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int y = (threadIdx.x >> 5) + 8 * k;
      const int64_t r = (mirror ? tj : ti) * 32 + y, c = (mirror ? ti : tj) * 32 + x;
      if (r >= s || c >= ld) continue;  // (columns s .. ld - 1 get the zeros of the tile)
      pp_bf16 p[NP];
      ns_planes<NP>(mirror || (ti == tj && x > y) ? tile[x][y] : tile[y][x], p);
#pragma unroll
      for (int q = 0; q < NP; ++q) planes[q * plane + batch * size + r * ld + c] = p[q];
    }
  }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------
// workgroups of a matrix's Gram matrix
static int ns_gram_splits(int64_t batch, int64_t l) {
  const int64_t parts = (l + NS_LONG - 1) / NS_LONG, room = batch > 0 && batch < NS_GRAM_BLOCKS ? NS_GRAM_BLOCKS / batch : 1;
  if (parts <= room) return (int)parts;
  const int64_t each = (parts + room - 1) / room;
  return (int)((parts + each - 1) / each);
}
static int64_t ns_lower(int64_t s, int64_t t) {
  const int64_t k = (s + t - 1) / t;
  return k * (k + 1) / 2;
}
// parts of a contraction of length k behind the lower 128 x 128 tiles of an s x s result: two workgroups per compute unit, a part is at
// least 256 long
static int ns_splits(int64_t batch, int64_t s, int64_t k) {
  int64_t q = 512 / (ns_lower(s, 128) * batch);
  if (q > (k + 255) / 256) q = (k + 255) / 256;
  return q < 1 ? 1 : (int)q;
}
static int64_t ns_round8(int64_t v) { return (v + 7) / 8 * 8; }

struct NsLargeWs {
  double* norm;
  NsScale* scale;
  float *part, *S32;
  pp_bf16 *X[2], *S, *P;
};
static size_t ns_large_ws(PPArena* ws, int planes, int64_t batch, int64_t m, int64_t n, NsLargeWs* w) {
  const int64_t s = m < n ? m : n, l = m < n ? n : m, ld = ns_round8(s), xs = batch * m * ns_round8(n), ss = batch * s * ld;
  const int s0 = ns_splits(batch, s, l), s1 = ns_splits(batch, s, s);
  const size_t sizes[8] = {(size_t)batch * NS_NORM_PARTS * 8, (size_t)batch * sizeof(NsScale), (size_t)(s0 > s1 ? s0 : s1) * ss * 4, (size_t)ss * 4,
                           (size_t)xs * planes * 2, (size_t)xs * planes * 2, (size_t)ss * planes * 2, (size_t)ss * planes * 2};
  size_t total = 0;
  void* at[8];
  for (int i = 0; i < 8; ++i) {
    total += pp_align(sizes[i]);
    if (ws) at[i] = ws->take<char>(sizes[i]);
  }
  if (ws) *w = NsLargeWs{(double*)at[0], (NsScale*)at[1], (float*)at[2], (float*)at[3], {(pp_bf16*)at[4], (pp_bf16*)at[5]}, (pp_bf16*)at[6], (pp_bf16*)at[7]};
  return total;
}

extern "C" size_t pp_newton_schulz_workspace_for(int32_t dtype, int64_t batch, int64_t m, int64_t n, int32_t steps) {
  if (batch < 0 || m < 1 || n < 1 || m > 65536 * 64 || n > 65536 * 64) return 0;
  const int64_t s = m < n ? m : n, l = m < n ? n : m;
  if (s > NS_PANEL_MAX) return ns_large_ws(nullptr, dtype == PP_F32 ? 3 : 2, batch > 0 ? batch : 1, m, n, nullptr) + 256;
  return pp_align((size_t)ns_gram_splits(batch, l) * batch * s * s * sizeof(double)) + 4 * pp_align((size_t)batch * s * s * sizeof(double)) +
         (steps > NS_ROUND ? 2 * pp_align((size_t)batch * m * n * sizeof(float)) : 0) + 256;
}
extern "C" size_t pp_newton_schulz_workspace(int64_t batch, int64_t m, int64_t n) {
  return pp_newton_schulz_workspace_for(PP_F32, batch, m, n, NS_ROUND + 1);  // (what needs most)
}

template <int SB>
static int ns_step_launch(const NsStepArgs& p, unsigned batch, hipStream_t st) {
  typedef NsPanel<SB> P;
  const size_t lds = ((size_t)P::N * P::N + 16 * P::LD + 8) * sizeof(double);
  PP_HIP(hipFuncSetAttribute((const void*)k_ns_step<SB>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  hipLaunchKernelGGL((k_ns_step<SB>), dim3(p.S2 ? 2 * SB : SB, batch), dim3(512), lds, st, p);  // (rows of Q first)
  PP_LAUNCH_CHECK();
  return PP_OK;
}
template <typename T, int SB>
static int ns_part_gram_launch(const T* g, int64_t m, int64_t n, int splits, int vec, double* part, unsigned batch, hipStream_t st) {
  hipLaunchKernelGGL((k_ns_part_gram<T, SB>), dim3((unsigned)splits, batch), dim3(512), 0, st, g, m, n, splits, vec, part);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
template <typename T, typename O, int SB>
static int ns_part_apply_launch(const T* g, int64_t m, int64_t n, int vec, const double* Q, O* out, unsigned batch, hipStream_t st) {
  const size_t lds = (size_t)SB * 16 * SB * 16 * sizeof(double) + NsPart<SB, true>::FLOATS * sizeof(float);
  PP_HIP(hipFuncSetAttribute((const void*)k_ns_part_apply<T, O, SB>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const int64_t l = m >= n ? m : n;
  hipLaunchKernelGGL((k_ns_part_apply<T, O, SB>), dim3((unsigned)((l + NS_LONG - 1) / NS_LONG), batch), dim3(512), lds, st, g, m, n, vec, Q, out);
  PP_LAUNCH_CHECK();
  return PP_OK;
}
#define NS_BY_BLOCKS(CALL) \
  switch ((s + 15) / 16) { \
    case 1: return CALL(1); \
    case 2: return CALL(2); \
    case 3: return CALL(3); \
    case 4: return CALL(4); \
    case 5: return CALL(5); \
    case 6: return CALL(6); \
    case 7: return CALL(7); \
    default: return CALL(8); \
  }
static int ns_step(const NsStepArgs& p, unsigned batch, hipStream_t st) {
  const int64_t s = p.s;
#define NS_CALL(SB) ns_step_launch<SB>(p, batch, st)
  NS_BY_BLOCKS(NS_CALL)
#undef NS_CALL
}
template <typename T>
static int ns_part_gram(const T* g, int64_t m, int64_t n, int64_t s, int splits, int vec, double* part, unsigned batch, hipStream_t st) {
#define NS_CALL(SB) ns_part_gram_launch<T, SB>(g, m, n, splits, vec, part, batch, st)
  NS_BY_BLOCKS(NS_CALL)
#undef NS_CALL
}
template <typename T, typename O>
static int ns_part_apply(const T* g, int64_t m, int64_t n, int64_t s, int vec, const double* Q, O* out, unsigned batch, hipStream_t st) {
#define NS_CALL(SB) ns_part_apply_launch<T, O, SB>(g, m, n, vec, Q, out, batch, st)
  NS_BY_BLOCKS(NS_CALL)
#undef NS_CALL
}

// plane pairs of a product of operands of pa and pb planes, the smallest first: pairs whose product is below the last plane are left out
static void ns_segments(GemmArgs& g, const pp_bf16* a, int64_t a_plane, int pa, const pp_bf16* b, int64_t b_plane, int pb, int planes) {
  g.segments = 0;
  for (int sum = planes - 1; sum >= 0; --sum)
    for (int i = 0; i <= sum; ++i)
      if (i < pa && sum - i < pb) {
        g.a[g.segments] = a + i * a_plane;
        g.b[g.segments++] = b + (sum - i) * b_plane;
      }
}
template <bool AC, bool BC, int BM, int BN, int WM, int WN, typename Epi>
static int ns_gemm(GemmArgs& g, const Epi& e, int64_t batch, hipStream_t st) {
  const int64_t tiles = g.lower ? ns_lower(g.m, BM) : ((g.m + BM - 1) / BM) * ((g.n + BN - 1) / BN);
  PP_REQUIRE(tiles <= 0x7FFFFFFF, "pp_newton_schulz: too many tiles");
  if (g.splits < 1) g.splits = 1;
  g.k_per_split = ((g.k + g.splits - 1) / g.splits + GM_BK - 1) / GM_BK * GM_BK;
  hipLaunchKernelGGL((k_gemm<pp_bf16, AC, BC, BM, BN, WM, WN, Epi>), dim3((unsigned)tiles, g.splits, (unsigned)batch),
                     dim3(BM / WM * (BN / WN) * 64), 0, st, g, e);
  PP_LAUNCH_CHECK();
  return PP_OK;
}

template <typename T, int NP>
static int ns_large(const T* g, int64_t batch, int64_t m, int64_t n, int steps, double ca, double cb, double cc, double eps, T* out, PPArena& ws,
                    hipStream_t st) {
  const bool tall = m >= n;
  const int64_t s = tall ? n : m, l = tall ? m : n, ld = ns_round8(s), ldx = ns_round8(n), xplane = batch * m * ldx, splane = batch * s * ld;
  NsLargeWs w;
  ns_large_ws(&ws, NP, batch, m, n, &w);
  PP_REQUIRE(w.norm && w.scale && w.part && w.S32 && w.X[0] && w.X[1] && w.S && w.P, "pp_newton_schulz: workspace layout");
  const unsigned nb = (unsigned)batch;
  hipLaunchKernelGGL((k_ns_norm<T>), dim3(NS_NORM_PARTS, nb), dim3(256), 0, st, g, m * n, w.norm);
  hipLaunchKernelGGL((k_ns_scale<T, NP>), dim3((unsigned)((m * ldx / 8 + 255) / 256), nb), dim3(256), 0, st, g, m, n, ldx, w.norm, eps, w.X[0], xplane,
                     w.scale);
  PP_LAUNCH_CHECK();
  int rc;
  for (int k = 0; k < steps; ++k) {
    const pp_bf16* X = w.X[k & 1];
    const int px = k == 0 && sizeof(T) == 2 && NP == 2 && __is_same(T, pp_bf16) ? 1 : NP;  // (bf16: G 2^e is one plane)
    GemmArgs a{};
    a.m = a.n = s; a.k = l; a.lda = a.ldb = ldx; a.a_batch = a.b_batch = m * ldx; a.lower = 1; a.splits = ns_splits(batch, s, l);
    ns_segments(a, X, xplane, px, X, xplane, px, NP);
    NsPartEpilogue pe{};
    pe.part = w.part; pe.s = s; pe.ld = ld; pe.splits = a.splits;
    rc = tall ? ns_gemm<true, true, 128, 128, 64, 64>(a, pe, batch, st) : ns_gemm<false, false, 128, 128, 64, 64>(a, pe, batch, st);
    if (rc != PP_OK) return rc;
    const unsigned sq = (unsigned)ns_lower(s, 32);
    hipLaunchKernelGGL((k_ns_square<NP>), dim3(sq, nb), dim3(256), 0, st, w.part, a.splits, s, ld, w.S32, (const float*)nullptr,
                       (const NsScale*)nullptr, 0.0, 0.0, 0.0, w.S, splane);
    a = GemmArgs{};
    a.m = a.n = a.k = s; a.lda = a.ldb = ld; a.a_batch = a.b_batch = s * ld; a.lower = 1; a.splits = ns_splits(batch, s, s);
    ns_segments(a, w.S, splane, NP, w.S, splane, NP, NP);
    pe.splits = a.splits;
    if ((rc = ns_gemm<false, false, 128, 128, 64, 64>(a, pe, batch, st)) != PP_OK) return rc;
    hipLaunchKernelGGL((k_ns_square<NP>), dim3(sq, nb), dim3(256), 0, st, w.part, a.splits, s, ld, (float*)nullptr, w.S32,
                       k == 0 ? w.scale : (const NsScale*)nullptr, ca, cb, cc, w.P, splane);
    PP_LAUNCH_CHECK();
    NsXEpilogue<T, NP> xe{};
    xe.planes = w.X[~k & 1]; xe.plane = xplane; xe.m = m; xe.n = n; xe.ld = ldx; xe.out = k == steps - 1 ? out : nullptr;
    xe.vec = n % 8 == 0 && (uintptr_t)out % 16 == 0;
    a = GemmArgs{};
    a.m = m; a.n = n; a.k = s;
    if (tall) {
      a.lda = ldx; a.a_batch = m * ldx; a.ldb = ld; a.b_batch = s * ld;
      ns_segments(a, X, xplane, px, w.P, splane, NP, NP);
      rc = ns_gemm<false, false, 128, 128, 64, 64>(a, xe, batch, st);
    } else {
      a.lda = ld; a.a_batch = s * ld; a.ldb = ldx; a.b_batch = m * ldx;
      ns_segments(a, w.P, splane, NP, X, xplane, px, NP);
      rc = ns_gemm<false, true, 128, 128, 64, 64>(a, xe, batch, st);
    }
    if (rc != PP_OK) return rc;
  }
  return PP_OK;
}

// one round for short sides up to NS_PANEL_MAX: out = X times the polynomials of its S, `steps` of them
template <typename T, typename O>
static int ns_round(const T* x, int64_t batch, int64_t m, int64_t n, NsStepArgs p, int steps, O* out, double* part, double* const (&mats)[4], hipStream_t st) {
  const int64_t s = p.s;
  const int splits = ns_gram_splits(batch, m < n ? n : m);
  const unsigned nb = (unsigned)batch;
  const int vec = n % 4 == 0 && (uintptr_t)x % (4 * sizeof(T)) == 0;
  int rc = ns_part_gram<T>(x, m, n, s, splits, vec, part, nb, st);
  if (rc != PP_OK) return rc;
  hipLaunchKernelGGL(k_ns_sum, dim3((unsigned)((s * s + 31) / 32), nb), dim3(256), 0, st, part, splits, s, mats[0]);
  PP_LAUNCH_CHECK();
  for (int k = 0; k < steps; ++k) {  // S in mats[0], mats[1] in turn, Q in mats[2], mats[3]
    p.S = mats[k & 1]; p.S2 = k == steps - 1 ? nullptr : mats[~k & 1];
    p.Q = k == 0 ? nullptr : mats[2 + (~k & 1)]; p.Q2 = mats[2 + (k & 1)];
    if ((rc = ns_step(p, nb, st)) != PP_OK) return rc;
  }
  return ns_part_apply<T, O>(x, m, n, s, vec, mats[2 + (~steps & 1)], out, nb, st);
}

template <typename T>
static int ns_run(const void* g, int64_t batch, int64_t m, int64_t n, int steps, double ca, double cb, double cc, double eps, void* out,
                  PPArena& ws, hipStream_t st) {
  const int64_t s = m < n ? m : n;
  if (s > NS_PANEL_MAX) return ns_large<T, sizeof(T) == 2 ? 2 : 3>((const T*)g, batch, m, n, steps, ca, cb, cc, eps, (T*)out, ws, st);
  double* part = ws.take<double>((size_t)ns_gram_splits(batch, m < n ? n : m) * batch * s * s);
  double* mats[4];
  for (double*& p : mats) p = ws.take<double>((size_t)batch * s * s);
  PP_REQUIRE(part && mats[3], "pp_newton_schulz: workspace layout");
  NsStepArgs p{};
  p.s = s; p.a = ca; p.b = cb; p.c = cc; p.eps = eps;
  if (steps <= NS_ROUND) return ns_round<T, T>((const T*)g, batch, m, n, p, steps, (T*)out, part, mats, st);
  float* X[2];
  for (float*& x : X) x = ws.take<float>((size_t)batch * m * n);
  PP_REQUIRE(X[1], "pp_newton_schulz: workspace layout");
  int rc = ns_round<T, float>((const T*)g, batch, m, n, p, NS_ROUND_LONG, X[0], part, mats, st);
  p.scaled = 1;
  int at = 0;
  for (steps -= NS_ROUND_LONG; rc == PP_OK && steps > NS_ROUND_LONG; steps -= NS_ROUND_LONG, at ^= 1)
    rc = ns_round<float, float>(X[at], batch, m, n, p, NS_ROUND_LONG, X[at ^ 1], part, mats, st);
  return rc == PP_OK ? ns_round<float, T>(X[at], batch, m, n, p, steps, (T*)out, part, mats, st) : rc;
}

extern "C" int pp_newton_schulz(const void* g, int32_t dtype, int64_t batch, int64_t m, int64_t n, int32_t steps, double ca, double cb,
                                double cc, double eps, void* out, void* ws, size_t ws_bytes, pp_stream_t stream) {
  PP_REQUIRE(pp_rows_dtype_ok(dtype), "pp_newton_schulz: unknown element type");
  PP_REQUIRE(batch >= 0 && batch <= 65535 && m >= 1 && n >= 1 && m <= 65536 * 64 && n <= 65536 * 64, "pp_newton_schulz: sizes out of range");
  PP_REQUIRE((m < n ? m : n) <= 8192, "pp_newton_schulz: the shorter side is at most 8192");
  PP_REQUIRE(steps >= 1 && steps <= 100, "pp_newton_schulz: steps must be in [1,100]");
  PP_REQUIRE(eps >= 0.0, "pp_newton_schulz: eps must not be negative");
  if (batch == 0) return PP_OK;
  PP_REQUIRE(g && out && ws && (uintptr_t)ws % 16 == 0, "pp_newton_schulz: null or unaligned pointer");
  if (ws_bytes < pp_newton_schulz_workspace_for(dtype, batch, m, n, steps)) {
    pp_set_error("pp_newton_schulz: workspace too small");
    return PP_ERR_WORKSPACE;
  }
  PPArena arena(ws, ws_bytes);
  hipStream_t s = pp_s(stream);
  if (dtype == PP_F32) return ns_run<float>(g, batch, m, n, steps, ca, cb, cc, eps, out, arena, s);
  if (dtype == PP_BF16) return ns_run<pp_bf16>(g, batch, m, n, steps, ca, cb, cc, eps, out, arena, s);
  return ns_run<pp_f16>(g, batch, m, n, steps, ca, cb, cc, eps, out, arena, s);
}

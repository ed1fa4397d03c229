// Orthogonalisation of a batch of matrices by Newton-Schulz products: X = G / (|G| + eps), then `steps` times
//   X <- X (a I + b S + c S^2),  S = X^T X                  (on the shorter side: S = X X^T, X from the left, where G is wide)
// All of it is a polynomial of the first S.  With P = a I + b S + c S^2 the next S is P S P, and the result is X Q with Q the product
// of all P: the long matrix is read twice (for S, and to be multiplied by Q) instead of three times a step, and the steps work on
// matrices of the short side only.  S, P and Q are symmetric and commute, so half of each product's tiles is computed and mirrored.
// S is held and multiplied in fp64: in the directions of small singular values P is a I, so rounding errors of S grow by a^2 = 11.9 a
// step there; fp64 leaves 1e-12 of them after five steps, fp32 would leave 1e-2.  |G|^2 is the trace of S.
#include "pp_rows.h"

typedef double ns_f64x4 __attribute__((ext_vector_type(4)));

#define NS_TILE 64
#define NS_BK 16

enum { NS_GRAM = 0, NS_CHAIN = 1, NS_APPLY = 2 };

// one product R = A B of a launch; element (row, k) of A at a[row * ars + k * aks], (k, col) of B at b[col * brs + k * bks]
struct NsJob {
  const void *a, *b;
  void* out;
  const double* add;  // NS_CHAIN: out = c0 I + c1 add + c2 R (nullable: c2 R)
  double c0, c1, c2;
  int pow1, pow2;     // powers of the batch element's alpha that multiply c1 and c2 (the first step works on the unscaled S)
};
struct NsArgs {
  NsJob job[2];
  int jobs;
  int64_t rows, cols, k;       // of R
  int64_t ars, aks, brs, bks, ors;
  int64_t a_batch, b_batch, out_batch;
  const double* alpha;         // [batch]
  int splits;
  int64_t k_per_split;
  int symmetric;               // only tiles on and below the diagonal are computed; NS_CHAIN mirrors them
};

// four values a thread brings of a NS_TILE x NS_BK part: rows run along the threads where they are neighbours in memory, else k does
template <typename T>
__device__ __forceinline__ void ns_load(const T* __restrict__ p, int64_t rs, int64_t ks, int64_t row0, int64_t rows, int64_t k0, int64_t k1,
                                        double (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = rs == 1 ? threadIdx.x & 63 : (threadIdx.x >> 4) + 16 * i, k = rs == 1 ? (threadIdx.x >> 6) + 4 * i : threadIdx.x & 15;
    v[i] = row0 + r < rows && k0 + k < k1 ? (double)p[(row0 + r) * rs + (k0 + k) * ks] : 0.0;
  }
}
__device__ __forceinline__ void ns_put(double* __restrict__ lds, int64_t rs, const double (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = rs == 1 ? threadIdx.x & 63 : (threadIdx.x >> 4) + 16 * i, k = rs == 1 ? (threadIdx.x >> 6) + 4 * i : threadIdx.x & 15;
    lds[k * (NS_TILE + 16) + r] = v[i];  // rows of 80 doubles: four k of a fragment fall on both halves of the banks
  }
}

template <typename TA, typename TB, typename TO, int MODE>
__global__ __launch_bounds__(256) void k_ns_tile(NsArgs g) {
  __shared__ double sa[2][NS_BK * (NS_TILE + 16)], sb[2][NS_BK * (NS_TILE + 16)];
  int64_t ti, tj;
  if (g.symmetric) {  // blockIdx.x counts the tiles on and below the diagonal, row by row
    ti = (int64_t)((sqrt(8.0 * (double)blockIdx.x + 1.0) - 1.0) * 0.5);
    while ((ti + 1) * (ti + 2) / 2 <= (int64_t)blockIdx.x) ++ti;
    while (ti * (ti + 1) / 2 > (int64_t)blockIdx.x) --ti;
    tj = (int64_t)blockIdx.x - ti * (ti + 1) / 2;
  } else {
    const int64_t tc = (g.cols + NS_TILE - 1) / NS_TILE;
    ti = blockIdx.x / tc;
    tj = blockIdx.x - ti * tc;
  }
  const int which = MODE == NS_CHAIN ? blockIdx.y : 0;
  const int split = MODE == NS_GRAM ? blockIdx.y : 0;
  const int64_t batch = blockIdx.z;
  const NsJob& job = g.job[which];
  const TA* a = (const TA*)job.a + batch * g.a_batch;
  const TB* b = (const TB*)job.b + batch * g.b_batch;
  const int64_t r0 = ti * NS_TILE, c0 = tj * NS_TILE;
  int64_t k = 0, k1 = g.k;
  if (MODE == NS_GRAM) {
    k = split * g.k_per_split;
    k1 = k + g.k_per_split < g.k ? k + g.k_per_split : g.k;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = (wave & 1) * 32, wc = (wave >> 1) * 32;
  ns_f64x4 acc[2][2] = {};
  double va[4], vb[4];
  if (k < k1) {
    ns_load(a, g.ars, g.aks, r0, g.rows, k, k1, va);
    ns_load(b, g.brs, g.bks, c0, g.cols, k, k1, vb);
  }
  for (int step = 0; k < k1; k += NS_BK, ++step) {
    double *la = sa[step & 1], *lb = sb[step & 1];
    ns_put(la, g.ars, va);
    ns_put(lb, g.brs, vb);
    __syncthreads();
    if (k + NS_BK < k1) {
      ns_load(a, g.ars, g.aks, r0, g.rows, k + NS_BK, k1, va);
      ns_load(b, g.brs, g.bks, c0, g.cols, k + NS_BK, k1, vb);
    }
#pragma unroll
    for (int kk = 0; kk < NS_BK; kk += 4) {
      const int at = (kk + (lane >> 4)) * (NS_TILE + 16) + (lane & 15);
      double fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = la[at + wr + 16 * i];
        fb[i] = lb[at + wc + 16 * i];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f64_16x16x4f64(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
  }
  // lane (l & 15, l >> 4), value e: row (l >> 4) + 4 e, column l & 15 of the fragment
  double c1 = job.c1, c2 = job.c2;
  if (g.alpha) {
    const double al = g.alpha[batch];
    for (int p = 0; p < job.pow1; ++p) c1 *= al;
    for (int p = 0; p < job.pow2; ++p) c2 *= al;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t r = r0 + wr + 16 * i + (lane >> 4) + 4 * e, c = c0 + wc + 16 * j + (lane & 15);
        if (r >= g.rows || c >= g.cols) continue;
        const double v = acc[i][j][e];
        if (MODE == NS_GRAM) {
          ((double*)job.out)[(batch * g.splits + split) * g.rows * g.cols + r * g.cols + c] = v;
        } else if (MODE == NS_APPLY) {
          ((TO*)job.out)[batch * g.out_batch + r * g.ors + c] = (TO)(float)(c2 * v);
        } else if (!g.symmetric || c <= r) {
          double* o = (double*)job.out + batch * g.out_batch;
          double w = c2 * v;
          if (job.add) w += c1 * job.add[batch * g.out_batch + r * g.cols + c];
          if (r == c) w += job.c0;
          o[r * g.cols + c] = w;
          if (g.symmetric) o[c * g.cols + r] = w;
        }
      }
}

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
  const double *S, *Q;  // [batch][s][s]; Q null: the identity times alpha (first step)
  double *S2, *Q2;      // S2 null: not wanted (last step)
  int64_t s;
  double a, b, c;
  double eps;           // first step: S is the unscaled one, alpha = 1 / (sqrt(trace S) + eps)
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
  if (first) {
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

// S of a part: its tiles on and below the diagonal, the eight waves in turn
template <typename T, int SB>
__global__ __launch_bounds__(512) void k_ns_part_gram(const T* __restrict__ g, int64_t m, int64_t n, int splits, int vec, double* __restrict__ part) {
  constexpr int TILES = SB * (SB + 1) / 2, PER = (TILES + 7) / 8;
  typedef NsPart<SB, false> X;
  __shared__ float x[X::FLOATS];
  const bool tall = m >= n;
  const int64_t s = tall ? n : m, l = tall ? m : n, l0 = (int64_t)blockIdx.x * NS_LONG, batch = blockIdx.y;
  X::load(x, g + batch * m * n + (tall ? l0 * n : l0), tall, n, (int)s, (int)(l - l0 < NS_LONG ? l - l0 : NS_LONG), vec);
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
  __syncthreads();
#pragma unroll 4
  for (int k = 0; k < NS_LONG; k += 4)
#pragma unroll
    for (int i = 0; i < PER; ++i)
      acc[i] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)x[X::at(tall, ta[i] * 16 + j, k + q)], (double)x[X::at(tall, tb[i] * 16 + j, k + q)], acc[i],
                                                    0, 0, 0);
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
template <typename T, int SB>
__global__ __launch_bounds__(512) void k_ns_part_apply(const T* __restrict__ g, int64_t m, int64_t n, int vec, const double* __restrict__ Q,
                                                       T* __restrict__ out) {
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
      if (r < (tall ? len : (int)s) && c < (tall ? (int)s : len)) out[corner + r * n + c] = (T)(float)acc[i][e];
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
// alpha = 1 / (|G| + eps)
__global__ __launch_bounds__(64) void k_ns_alpha(const double* __restrict__ S, int64_t s, double eps, double* __restrict__ alpha) {
  const double* p = S + (int64_t)blockIdx.x * s * s;
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < s; i += 64) v += p[i * s + i];
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  if (threadIdx.x == 0) alpha[blockIdx.x] = 1.0 / (sqrt(v) + eps);
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------
static int64_t ns_lower_tiles(int64_t s) {
  const int64_t t = (s + NS_TILE - 1) / NS_TILE;
  return t * (t + 1) / 2;
}
// parts of the long side: about two workgroups per compute unit, at least 128 of it each
static int ns_splits(int64_t batch, int64_t s, int64_t l) {
  if (s <= NS_PANEL_MAX) return (int)((l + NS_LONG - 1) / NS_LONG);
  int64_t q = 512 / (ns_lower_tiles(s) * batch);
  if (q > (l + 127) / 128) q = (l + 127) / 128;
  return q < 1 ? 1 : (int)q;
}

extern "C" size_t pp_newton_schulz_workspace(int64_t batch, int64_t m, int64_t n) {
  if (batch < 0 || m < 1 || n < 1 || m > 65536 * 64 || n > 65536 * 64) return 0;
  const int64_t s = m < n ? m : n, l = m < n ? n : m;
  const size_t one = pp_align((size_t)batch * s * s * sizeof(double));
  return pp_align((size_t)ns_splits(batch > 0 ? batch : 1, s, l) * batch * s * s * sizeof(double)) + 6 * one +
         pp_align((size_t)batch * sizeof(double)) + 256;
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
template <typename T, int SB>
static int ns_part_apply_launch(const T* g, int64_t m, int64_t n, int vec, const double* Q, T* out, unsigned batch, hipStream_t st) {
  const size_t lds = (size_t)SB * 16 * SB * 16 * sizeof(double) + NsPart<SB, true>::FLOATS * sizeof(float);
  PP_HIP(hipFuncSetAttribute((const void*)k_ns_part_apply<T, SB>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  const int64_t l = m >= n ? m : n;
  hipLaunchKernelGGL((k_ns_part_apply<T, SB>), dim3((unsigned)((l + NS_LONG - 1) / NS_LONG), batch), dim3(512), lds, st, g, m, n, vec, Q, out);
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
template <typename T>
static int ns_part_apply(const T* g, int64_t m, int64_t n, int64_t s, int vec, const double* Q, T* out, unsigned batch, hipStream_t st) {
#define NS_CALL(SB) ns_part_apply_launch<T, SB>(g, m, n, vec, Q, out, batch, st)
  NS_BY_BLOCKS(NS_CALL)
#undef NS_CALL
}

template <typename T>
static int ns_run(const void* g, int64_t batch, int64_t m, int64_t n, int steps, double ca, double cb, double cc, double eps, void* out,
                  PPArena& ws, hipStream_t st) {
  const bool tall = m >= n;
  const int64_t s = tall ? n : m, l = tall ? m : n;
  const int splits = ns_splits(batch, s, l);
  double* part = ws.take<double>((size_t)splits * batch * s * s);
  double* mats[6];
  for (double*& p : mats) p = ws.take<double>((size_t)batch * s * s);
  double* alpha = ws.take<double>((size_t)batch);
  PP_REQUIRE(part && mats[5] && alpha, "pp_newton_schulz: workspace layout");
  const unsigned low = (unsigned)ns_lower_tiles(s), nb = (unsigned)batch;
  const bool panels = s <= NS_PANEL_MAX;
  const int vec = n % 4 == 0 && (uintptr_t)g % (4 * sizeof(T)) == 0;
  if (panels) {
    int rc = ns_part_gram<T>((const T*)g, m, n, s, splits, vec, part, nb, st);
    if (rc != PP_OK) return rc;
    hipLaunchKernelGGL(k_ns_sum, dim3((unsigned)((s * s + 31) / 32), nb), dim3(256), 0, st, part, splits, s, mats[0]);
    PP_LAUNCH_CHECK();
  } else {  // S of the matrix as it is
    NsArgs a{};
    a.job[0].a = a.job[0].b = g; a.job[0].out = part;
    a.rows = a.cols = s; a.k = l;
    a.ars = a.brs = tall ? 1 : n; a.aks = a.bks = tall ? n : 1;
    a.a_batch = a.b_batch = m * n;
    a.splits = splits; a.k_per_split = ((l + splits - 1) / splits + NS_BK - 1) / NS_BK * NS_BK; a.symmetric = 1;
    hipLaunchKernelGGL((k_ns_tile<T, T, double, NS_GRAM>), dim3(low, splits, nb), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_ns_sum, dim3((unsigned)((s * s + 31) / 32), nb), dim3(256), 0, st, part, splits, s, mats[0]);
    hipLaunchKernelGGL(k_ns_alpha, dim3(nb), dim3(64), 0, st, mats[0], s, eps, alpha);
    PP_LAUNCH_CHECK();
  }
  double *S = mats[0], *P = mats[1], *U = mats[2], *N = mats[3], *Q = mats[4], *R = mats[5];
  if (panels) {
    NsStepArgs p{};
    p.s = s; p.a = ca; p.b = cb; p.c = cc; p.eps = eps;
    for (int k = 0; k < steps; ++k) {
      p.S = k & 1 ? N : S; p.S2 = k == steps - 1 ? nullptr : (k & 1 ? S : N);
      p.Q = k == 0 ? nullptr : (k & 1 ? Q : R); p.Q2 = k & 1 ? R : Q;
      int rc = ns_step(p, nb, st);
      if (rc != PP_OK) return rc;
    }
    return ns_part_apply<T>((const T*)g, m, n, s, vec, steps & 1 ? Q : R, (T*)out, nb, st);
  }
  NsArgs a{};
  a.rows = a.cols = a.k = s; a.ars = a.brs = 1; a.aks = a.bks = s; a.ors = s;
  a.a_batch = a.b_batch = a.out_batch = s * s; a.alpha = alpha; a.symmetric = 1;
  auto chain = [&](int jobs) -> int {
    hipLaunchKernelGGL((k_ns_tile<double, double, double, NS_CHAIN>), dim3(low, jobs, nb), dim3(256), 0, st, a);
    PP_LAUNCH_CHECK();
    return PP_OK;
  };
  int rc;
  for (int k = 0; k < steps; ++k) {
    const int p = k == 0 ? 2 : 0;  // S is scaled by alpha^2 from the second step on
    a.job[0] = NsJob{S, S, P, S, ca, cb, cc, p, 2 * p};
    if ((rc = chain(1)) != PP_OK) return rc;
    const bool last = k == steps - 1;
    int jobs = 0;
    if (k > 0) {  // Q <- Q P
      a.job[jobs++] = NsJob{Q, P, R, nullptr, 0.0, 0.0, 1.0, 0, 0};
    }
    if (!last) a.job[jobs++] = NsJob{S, P, U, nullptr, 0.0, 0.0, 1.0, 0, p};
    if (jobs && (rc = chain(jobs)) != PP_OK) return rc;
    if (k > 0) {
      double* t = Q; Q = R; R = t;
    } else {  // Q = P: the next step's P goes elsewhere
      double* t = Q; Q = P; P = t;
    }
    if (!last) {  // S <- U P with this step's P (in Q after the first step)
      a.job[0] = NsJob{U, k == 0 ? Q : P, N, nullptr, 0.0, 0.0, 1.0, 0, 0};
      if ((rc = chain(1)) != PP_OK) return rc;
      double* t = S; S = N; N = t;
    }
  }
  NsArgs e{};
  e.alpha = alpha; e.k = s; e.rows = m; e.cols = n; e.ors = n; e.out_batch = m * n;
  e.job[0].c2 = 1.0; e.job[0].pow2 = 1; e.job[0].out = out;
  const int64_t tiles = ((m + NS_TILE - 1) / NS_TILE) * ((n + NS_TILE - 1) / NS_TILE);
  PP_REQUIRE(tiles <= 0x7FFFFFFF, "pp_newton_schulz: too many tiles");
  if (tall) {
    e.job[0].a = g; e.ars = n; e.aks = 1; e.a_batch = m * n;
    e.job[0].b = Q; e.brs = 1; e.bks = s; e.b_batch = s * s;
    hipLaunchKernelGGL((k_ns_tile<T, double, T, NS_APPLY>), dim3((unsigned)tiles, 1, nb), dim3(256), 0, st, e);
  } else {
    e.job[0].a = Q; e.ars = 1; e.aks = s; e.a_batch = s * s;
    e.job[0].b = g; e.brs = 1; e.bks = n; e.b_batch = m * n;
    hipLaunchKernelGGL((k_ns_tile<double, T, T, NS_APPLY>), dim3((unsigned)tiles, 1, nb), dim3(256), 0, st, e);
  }
  PP_LAUNCH_CHECK();
  return PP_OK;
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
  if (ws_bytes < pp_newton_schulz_workspace(batch, m, n)) {
    pp_set_error("pp_newton_schulz: workspace too small");
    return PP_ERR_WORKSPACE;
  }
  PPArena arena(ws, ws_bytes);
  hipStream_t s = pp_s(stream);
  if (dtype == PP_F32) return ns_run<float>(g, batch, m, n, steps, ca, cb, cc, eps, out, arena, s);
  if (dtype == PP_BF16) return ns_run<pp_bf16>(g, batch, m, n, steps, ca, cb, cc, eps, out, arena, s);
  return ns_run<pp_f16>(g, batch, m, n, steps, ca, cb, cc, eps, out, arena, s);
}

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

// adds the parts of S in their order, both triangles from the lower one
__global__ __launch_bounds__(256) void k_ns_sum(const double* __restrict__ part, int splits, int64_t s, double* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, batch = blockIdx.y;
  if (i >= s * s) return;
  const int64_t r = i / s, c = i - r * s;
  if (c > r) return;
  double v = 0.0;
  for (int q = 0; q < splits; ++q) v += part[(batch * splits + q) * s * s + i];
  out[batch * s * s + i] = v;
  out[batch * s * s + c * s + r] = v;
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
  {  // S of the matrix as it is
    NsArgs a{};
    a.job[0].a = a.job[0].b = g; a.job[0].out = part;
    a.rows = a.cols = s; a.k = l;
    a.ars = a.brs = tall ? 1 : n; a.aks = a.bks = tall ? n : 1;
    a.a_batch = a.b_batch = m * n;
    a.splits = splits; a.k_per_split = ((l + splits - 1) / splits + NS_BK - 1) / NS_BK * NS_BK; a.symmetric = 1;
    hipLaunchKernelGGL((k_ns_tile<T, T, double, NS_GRAM>), dim3(low, splits, nb), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k_ns_sum, dim3((unsigned)((s * s + 255) / 256), nb), dim3(256), 0, st, part, splits, s, mats[0]);
    hipLaunchKernelGGL(k_ns_alpha, dim3(nb), dim3(64), 0, st, mats[0], s, eps, alpha);
    PP_LAUNCH_CHECK();
  }
  double *S = mats[0], *P = mats[1], *U = mats[2], *N = mats[3], *Q = mats[4], *R = mats[5];
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

// Group normalisation over the rows of a batch element, with an activation, on [rows, channels] features (channels last).
//
// Batch element s owns the positions [off[s], off[s+1]) of the row sequence (position p = row order[p], or row p); group g its
// C / G neighbouring channels.  With m = rows of s times C / G:
//   mean = sum x / m,  var = sum x^2 / m - mean^2,  xh = (x - mean) / sqrt(var + eps),  z = xh w_c + b_c,  y = act(z)
//   dz = dy act'(z);  db_c = sum dz, dw_c = sum dz xh over ALL rows;  h = dz w_c;  dx = rstd (h - mean_g(h) - xh mean_g(h xh))
// All sums are fp64: the difference sum x^2 / m - mean^2 loses (mean / std)^2 of the accumulator's precision, which fp32 does not
// have to spare where a feature sits far from 0; the fp64 rate is far above what the loads deliver.  No atomics: a chunk of positions
// writes its sums to slots of its own, and they are added in a fixed order, so results repeat bit for bit.
//
// The row sequence is cut into chunks, whatever the batch elements' lengths are.  The pairs (chunk j, element s) that meet form a
// staircase, along which j + s grows by one at every step: slot j + s is its pair's alone, and an element's slots are neighbours.
// Offsets and row orders are read on the device and not trusted: positions are clamped to [0, rows], rows outside are passed over.
#include "pp_rows.h"

#define GN_MAX_CHUNKS 1024
#define GN_MAX_C 1024

struct GnArgs {
  const void *x, *dy;
  void* out;  // y forward, dx backward
  int64_t n;
  int c, g;
  const int64_t* off;
  int64_t b;
  const int64_t* order;
  const float *weight, *bias;
  double eps;
  int act;
  float slope;
  float *mean, *rstd;   // [b, g]; written forward, read backward
  double* slots;        // forward [slot][g][2], backward [slot][2][c]
  double* totals;       // backward [chunk][2][c]
  float* coef;          // backward [b, g][2]: mean(h), mean(h xh)
  float *dweight, *dbias;
  int64_t rows_per_chunk;
  int chunks;
};

// first i in [0, count] with off[i] > p (count if there is none)
__device__ __forceinline__ int64_t gn_upper(const int64_t* __restrict__ off, int64_t count, int64_t p) {
  int64_t lo = 0, hi = count;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (off[mid] > p) hi = mid; else lo = mid + 1;
  }
  return lo;
}
__device__ __forceinline__ int64_t gn_clamp(int64_t v, int64_t n) { return v < 0 ? 0 : (v > n ? n : v); }

// the row at position p, -1 if the order holds no row there
__device__ __forceinline__ int64_t gn_row(const GnArgs& a, int64_t p) {
  if (!a.order) return p;
  const int64_t r = a.order[p];
  return r >= 0 && r < a.n ? r : -1;
}

// A block's threads over a chunk: `lpr` threads side by side on a row (VEC channels each, NC times 256 threads apart where a row is
// wider than the block), `rps` rows at a time
template <int VEC, int NC>
struct GnLane {
  int lpr, rps, rin, cc;
  bool on;
  __device__ GnLane(int c) {
    const int cv = c / VEC;
    lpr = cv < 256 ? cv : 256;
    rps = 256 / lpr;
    rin = threadIdx.x / lpr;
    cc = threadIdx.x - rin * lpr;
    on = rin < rps;
  }
  __device__ int channel(int k) const { return (cc + 256 * k) * VEC; }
  __device__ bool has(int k, int c) const { return NC == 1 || channel(k) < c; }
};

// mean, 1/std, weight and bias of a thread's channels
template <int VEC, int NC>
struct GnAffine {
  float w[NC][VEC], b[NC][VEC];
  __device__ GnAffine(const GnArgs& a, const GnLane<VEC, NC>& ln) {
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int u = 0; u < VEC; ++u) {
        const bool in = ln.on && ln.has(k, a.c);
        w[k][u] = a.weight && in ? a.weight[ln.channel(k) + u] : 1.f;
        b[k][u] = a.bias && in ? a.bias[ln.channel(k) + u] : 0.f;
      }
  }
};

// sums of a thread's rows [p, e) -> LDS red[2][rps][c]; FORWARD: x, x^2; else dz, dz xh
template <typename T, int VEC, int NC, bool FORWARD>
__device__ __forceinline__ void gn_rows_sum(const GnArgs& a, const GnLane<VEC, NC>& ln, const GnAffine<VEC, NC>& af, int64_t p, int64_t e,
                                            const float (&mu)[NC][VEC], const float (&rs)[NC][VEC], double* __restrict__ red) {
  double s0[NC][VEC], s1[NC][VEC];
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int u = 0; u < VEC; ++u) s0[k][u] = s1[k][u] = 0.0;
  if (ln.on) {
    constexpr int U = NC == 1 ? 4 : 1;  // rows in flight
    for (int64_t q = p + ln.rin; q < e; q += (int64_t)U * ln.rps) {
      float xv[U][NC][VEC], dv[U][NC][VEC];
      bool ok[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t pos = q + (int64_t)i * ln.rps;
        const int64_t r = pos < e ? gn_row(a, pos) : -1;
        ok[i] = r >= 0;
#pragma unroll
        for (int k = 0; k < NC; ++k)
          if (ok[i] && ln.has(k, a.c)) {
            pp_load<T, VEC>((const T*)a.x + r * a.c + ln.channel(k), xv[i][k]);
            if (!FORWARD) pp_load<T, VEC>((const T*)a.dy + r * a.c + ln.channel(k), dv[i][k]);
          }
      }
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int k = 0; k < NC; ++k)
          if (ok[i] && ln.has(k, a.c)) {
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
              if (FORWARD) {
                const double v = (double)xv[i][k][u];
                s0[k][u] += v;
                s1[k][u] = fma(v, v, s1[k][u]);
              } else {
                const float xh = (xv[i][k][u] - mu[k][u]) * rs[k][u];
                const double dz = (double)(dv[i][k][u] * pp_dact1(fmaf(xh, af.w[k][u], af.b[k][u]), a.act, a.slope));
                s0[k][u] += dz;
                s1[k][u] = fma(dz, (double)xh, s1[k][u]);
              }
            }
          }
    }
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (ln.has(k, a.c)) {
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          red[ln.rin * a.c + ln.channel(k) + u] = s0[k][u];
          red[(ln.rps + ln.rin) * a.c + ln.channel(k) + u] = s1[k][u];
        }
      }
  }
}

// group sums of red[2][rps][c]: calls put(g, sum0, sum1) on one thread per group.  FORWARD: plain sums; else weighted by w_c.
// `tpg` neighbouring threads (a power of two, at most a wave) share a group
template <bool WEIGHTED, typename Put>
__device__ __forceinline__ void gn_group_sums(const GnArgs& a, int rps, const double* __restrict__ red, Put put) {
  int tpg = 64;
  while (tpg > 1 && tpg * a.g > 256) tpg >>= 1;
  const int cg = a.c / a.g, j = threadIdx.x & (tpg - 1), step = 256 / tpg;
  for (int g0 = 0; g0 < a.g; g0 += step) {  // uniform bounds: the shuffles below need the whole wave
    const int g = g0 + (int)threadIdx.x / tpg;
    double v0 = 0.0, v1 = 0.0;
    if (g < a.g) {
      const int entries = rps * cg;
      for (int e = j; e < entries; e += tpg) {
        const int r = e / cg, ch = g * cg + (e - r * cg);
        const double wt = WEIGHTED && a.weight ? (double)a.weight[ch] : 1.0;
        v0 += wt * red[r * a.c + ch];
        v1 += wt * red[(rps + r) * a.c + ch];
      }
    }
    for (int d = tpg >> 1; d > 0; d >>= 1) {
      v0 += __shfl_xor(v0, d);
      v1 += __shfl_xor(v1, d);
    }
    if (j == 0 && g < a.g) put(g, v0, v1);
  }
}

// mean and 1/std from the sums over m values
__device__ __forceinline__ void gn_moments(double s0, double s1, double m, double eps, float* mean, float* rstd) {
  const double mu = s0 / m, var = s1 / m - mu * mu;
  *mean = (float)mu;
  *rstd = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps));  // (a NaN stays one)
}

// y or dx of the rows [p, e) of one batch element
template <typename T, int VEC, int NC, bool FORWARD>
__device__ __forceinline__ void gn_rows_apply(const GnArgs& a, const GnLane<VEC, NC>& ln, const GnAffine<VEC, NC>& af, int64_t p, int64_t e,
                                              const float (&mu)[NC][VEC], const float (&rs)[NC][VEC], const float (&ka)[NC][VEC],
                                              const float (&kb)[NC][VEC]) {
  if (!ln.on) return;
  constexpr int U = NC == 1 ? 2 : 1;
  for (int64_t q = p + ln.rin; q < e; q += (int64_t)U * ln.rps) {
    float xv[U][NC][VEC], dv[U][NC][VEC];
    int64_t row[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t pos = q + (int64_t)i * ln.rps;
      row[i] = pos < e ? gn_row(a, pos) : -1;
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (row[i] >= 0 && ln.has(k, a.c)) {
          pp_load<T, VEC>((const T*)a.x + row[i] * a.c + ln.channel(k), xv[i][k]);
          if (!FORWARD) pp_load<T, VEC>((const T*)a.dy + row[i] * a.c + ln.channel(k), dv[i][k]);
        }
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (row[i] >= 0 && ln.has(k, a.c)) {
          float o[VEC];
#pragma unroll
          for (int u = 0; u < VEC; ++u) {
            const float xh = (xv[i][k][u] - mu[k][u]) * rs[k][u];
            const float z = fmaf(xh, af.w[k][u], af.b[k][u]);
            if (FORWARD) {
              o[u] = pp_act1(z, a.act, a.slope);
            } else {
              const float h = dv[i][k][u] * pp_dact1(z, a.act, a.slope) * af.w[k][u];
              o[u] = rs[k][u] * (h - ka[k][u] - xh * kb[k][u]);
            }
          }
          pp_store<T, VEC>((T*)a.out + row[i] * a.c + ln.channel(k), o);
        }
  }
}

// rows at positions [p, e) that belong to no batch element: zeros
template <typename T, int VEC, int NC>
__device__ __forceinline__ void gn_rows_zero(const GnArgs& a, const GnLane<VEC, NC>& ln, int64_t p, int64_t e) {
  if (!ln.on) return;
  const float o[VEC] = {};
  for (int64_t q = p + ln.rin; q < e; q += ln.rps) {
    const int64_t r = gn_row(a, q);
    if (r < 0) continue;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (ln.has(k, a.c)) pp_store<T, VEC>((T*)a.out + r * a.c + ln.channel(k), o);
  }
}

// per-(element, group) values of a thread's channels: v[k][u] = table[(s * g + group) * stride]
template <int VEC, int NC>
__device__ __forceinline__ void gn_per_channel(const GnArgs& a, const GnLane<VEC, NC>& ln, const float* __restrict__ table, int stride,
                                               int64_t s, float (&v)[NC][VEC]) {
  const int cg = a.c / a.g;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int u = 0; u < VEC; ++u)
      v[k][u] = ln.on && ln.has(k, a.c) ? table[(s * a.g + (ln.channel(k) + u) / cg) * stride] : 0.f;
}

// ---- long batch elements: sums of chunks, their sums per element, then the rows --------------------------------------------------
template <typename T, int VEC, int NC, bool FORWARD>
__global__ __launch_bounds__(256) void k_gn_chunk_sums(GnArgs a) {
  extern __shared__ double red[];
  const GnLane<VEC, NC> ln(a.c);
  const GnAffine<VEC, NC> af(a, ln);
  const int64_t start = (int64_t)blockIdx.x * a.rows_per_chunk;
  const int64_t end = start + a.rows_per_chunk < a.n ? start + a.rows_per_chunk : a.n;
  double t0[GN_MAX_C / 256] = {}, t1[GN_MAX_C / 256] = {};
  int64_t p = start;
  while (p < end) {
    const int64_t hi = gn_upper(a.off, a.b + 1, p);
    if (hi == a.b + 1) break;
    const int64_t e = a.off[hi] < end ? a.off[hi] : end;  // > p by the search
    if (hi > 0) {
      const int64_t s = hi - 1, slot = (int64_t)blockIdx.x + s;
      float mu[NC][VEC] = {}, rs[NC][VEC] = {};
      if (!FORWARD) {
        gn_per_channel<VEC, NC>(a, ln, a.mean, 1, s, mu);
        gn_per_channel<VEC, NC>(a, ln, a.rstd, 1, s, rs);
      }
      gn_rows_sum<T, VEC, NC, FORWARD>(a, ln, af, p, e, mu, rs, red);
      __syncthreads();
      if (FORWARD) {
        gn_group_sums<false>(a, ln.rps, red, [&](int g, double v0, double v1) {
          a.slots[(slot * a.g + g) * 2] = v0;
          a.slots[(slot * a.g + g) * 2 + 1] = v1;
        });
      } else {
#pragma unroll
        for (int k = 0; k < GN_MAX_C / 256; ++k) {
          const int ch = threadIdx.x + 256 * k;
          if (ch < a.c) {
            double v0 = 0.0, v1 = 0.0;
            for (int r = 0; r < ln.rps; ++r) {
              v0 += red[r * a.c + ch];
              v1 += red[(ln.rps + r) * a.c + ch];
            }
            a.slots[slot * 2 * a.c + ch] = v0;
            a.slots[(slot * 2 + 1) * a.c + ch] = v1;
            t0[k] += v0;
            t1[k] += v1;
          }
        }
      }
      __syncthreads();
    }
    p = e;
  }
  if (!FORWARD) {
#pragma unroll
    for (int k = 0; k < GN_MAX_C / 256; ++k) {
      const int ch = threadIdx.x + 256 * k;
      if (ch < a.c) {
        a.totals[(int64_t)blockIdx.x * 2 * a.c + ch] = t0[k];
        a.totals[((int64_t)blockIdx.x * 2 + 1) * a.c + ch] = t1[k];
      }
    }
  }
}

// one wave per (element, group) adds the slots of the element; backward: a weighted sum over the group's channels too.  The blocks
// behind them (backward) add the chunks' totals to dweight and dbias, eight channels a block
template <bool FORWARD>
__global__ __launch_bounds__(256) void k_gn_finish(GnArgs a, int64_t group_blocks) {
  if (!FORWARD && (int64_t)blockIdx.x >= group_blocks) {
    __shared__ double sm[2][32][8];
    const int cl = threadIdx.x & 7, j = threadIdx.x >> 3, ch = (int)(blockIdx.x - group_blocks) * 8 + cl;
    double v0 = 0.0, v1 = 0.0;
    if (ch < a.c)
      for (int q = j; q < a.chunks; q += 32) {
        v0 += a.totals[(int64_t)q * 2 * a.c + ch];
        v1 += a.totals[((int64_t)q * 2 + 1) * a.c + ch];
      }
    sm[0][j][cl] = v0;
    sm[1][j][cl] = v1;
    __syncthreads();
    if (j != 0 || ch >= a.c) return;
    v0 = v1 = 0.0;
    for (int q = 0; q < 32; ++q) {
      v0 += sm[0][q][cl];
      v1 += sm[1][q][cl];
    }
    if (a.dbias) a.dbias[ch] = (float)v0;
    if (a.dweight) a.dweight[ch] = (float)v1;
    return;
  }
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= a.b * a.g) return;
  const int64_t s = w / a.g;
  const int g = (int)(w - s * a.g), cg = a.c / a.g;
  const int64_t o0 = gn_clamp(a.off[s], a.n), o1 = gn_clamp(a.off[s + 1], a.n);
  double v0 = 0.0, v1 = 0.0;
  if (o1 > o0) {
    const int64_t j0 = o0 / a.rows_per_chunk, j1 = (o1 - 1) / a.rows_per_chunk;
    if (FORWARD) {
      for (int64_t j = j0 + lane; j <= j1; j += 64) {
        v0 += a.slots[((j + s) * a.g + g) * 2];
        v1 += a.slots[((j + s) * a.g + g) * 2 + 1];
      }
    } else {
      const int64_t entries = (j1 - j0 + 1) * cg;
      for (int64_t e = lane; e < entries; e += 64) {
        const int64_t j = j0 + e / cg;
        const int ch = g * cg + (int)(e % cg);
        const double wt = a.weight ? (double)a.weight[ch] : 1.0;
        v0 += wt * a.slots[(j + s) * 2 * a.c + ch];
        v1 += wt * a.slots[((j + s) * 2 + 1) * a.c + ch];
      }
    }
  }
  for (int d = 32; d > 0; d >>= 1) {
    v0 += __shfl_xor(v0, d);
    v1 += __shfl_xor(v1, d);
  }
  if (lane != 0) return;
  const double m = (double)(o1 - o0) * cg;
  if (FORWARD) {
    float mu = 0.f, rs = 0.f;
    if (o1 > o0) gn_moments(v0, v1, m, a.eps, &mu, &rs);
    a.mean[w] = mu;
    a.rstd[w] = rs;
  } else {
    a.coef[2 * w] = o1 > o0 ? (float)(v0 / m) : 0.f;
    a.coef[2 * w + 1] = o1 > o0 ? (float)(v1 / m) : 0.f;
  }
}

template <typename T, int VEC, int NC, bool FORWARD>
__global__ __launch_bounds__(256) void k_gn_chunk_apply(GnArgs a) {
  const GnLane<VEC, NC> ln(a.c);
  const GnAffine<VEC, NC> af(a, ln);
  int64_t p = (int64_t)blockIdx.x * a.rows_per_chunk;
  const int64_t end = p + a.rows_per_chunk < a.n ? p + a.rows_per_chunk : a.n;
  while (p < end) {
    const int64_t hi = gn_upper(a.off, a.b + 1, p);
    const int64_t e = hi <= a.b && a.off[hi] < end ? a.off[hi] : end;
    if (hi == 0 || hi > a.b) {
      gn_rows_zero<T, VEC, NC>(a, ln, p, e);
    } else {
      const int64_t s = hi - 1;
      float mu[NC][VEC], rs[NC][VEC], ka[NC][VEC] = {}, kb[NC][VEC] = {};
      gn_per_channel<VEC, NC>(a, ln, a.mean, 1, s, mu);
      gn_per_channel<VEC, NC>(a, ln, a.rstd, 1, s, rs);
      if (!FORWARD) {
        gn_per_channel<VEC, NC>(a, ln, a.coef, 2, s, ka);
        gn_per_channel<VEC, NC>(a, ln, a.coef + 1, 2, s, kb);
      }
      gn_rows_apply<T, VEC, NC, FORWARD>(a, ln, af, p, e, mu, rs, ka, kb);
    }
    p = e;
  }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------
static int64_t gn_rows_per_chunk(int64_t n) {
  const int64_t r = (n + GN_MAX_CHUNKS - 1) / GN_MAX_CHUNKS;
  return r < 64 ? 64 : r;
}
static int gn_chunks(int64_t n) { return (int)((n + gn_rows_per_chunk(n) - 1) / gn_rows_per_chunk(n)); }

extern "C" size_t pp_group_norm_workspace(int64_t n, int64_t b, int32_t c, int32_t groups, int32_t backward) {
  if (n < 0 || b < 0 || c < 1 || groups < 1) return 0;
  const size_t slots = (size_t)gn_chunks(n) + (size_t)b + 1;
  if (!backward) return pp_align(slots * groups * 2 * sizeof(double));
  return pp_align(slots * 2 * c * sizeof(double)) + pp_align((size_t)(gn_chunks(n) + 1) * 2 * c * sizeof(double)) +
         pp_align((size_t)b * groups * 2 * sizeof(float) + 1);
}

template <typename T, int VEC, int NC, bool FORWARD>
static int gn_launch(GnArgs& a, hipStream_t s) {
  const int cv = a.c / VEC, rps = 256 / (cv < 256 ? cv : 256);
  const size_t lds = (size_t)rps * a.c * 2 * sizeof(double);
  a.rows_per_chunk = gn_rows_per_chunk(a.n);
  a.chunks = gn_chunks(a.n);
  if (a.chunks) {
    hipLaunchKernelGGL((k_gn_chunk_sums<T, VEC, NC, FORWARD>), dim3(a.chunks), dim3(256), lds, s, a);
    PP_LAUNCH_CHECK();
  }
  const int64_t gb = (a.b * a.g + 3) / 4, cb = FORWARD ? 0 : (a.c + 7) / 8;
  if (gb + cb) {
    hipLaunchKernelGGL((k_gn_finish<FORWARD>), dim3((unsigned)(gb + cb)), dim3(256), 0, s, a, gb);
    PP_LAUNCH_CHECK();
  }
  if (a.chunks) {
    hipLaunchKernelGGL((k_gn_chunk_apply<T, VEC, NC, FORWARD>), dim3(a.chunks), dim3(256), 0, s, a);
    PP_LAUNCH_CHECK();
  }
  return PP_OK;
}

// 16-byte vectors where every row starts on one (the row's bytes are a multiple of 16 and so are the pointers); single elements else
template <typename T, bool FORWARD>
static int gn_type(GnArgs& a, hipStream_t s) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.out;
  if (a.c % VEC == 0 && at % 16 == 0) return gn_launch<T, VEC, 1, FORWARD>(a, s);
  return a.c <= 256 ? gn_launch<T, 1, 1, FORWARD>(a, s) : gn_launch<T, 1, GN_MAX_C / 256, FORWARD>(a, s);
}
template <bool FORWARD>
static int gn_dispatch(GnArgs& a, int dtype, hipStream_t s) {
  if (dtype == PP_F32) return gn_type<float, FORWARD>(a, s);
  return dtype == PP_BF16 ? gn_type<pp_bf16, FORWARD>(a, s) : gn_type<pp_f16, FORWARD>(a, s);
}

static int gn_check(int32_t dtype, int64_t n, int32_t c, int32_t groups, const int64_t* offsets, int64_t b, int32_t act) {
  PP_REQUIRE(pp_rows_dtype_ok(dtype), "pp_group_norm: unknown element type");
  PP_REQUIRE(pp_rows_act_ok(act), "pp_group_norm: unknown activation");
  PP_REQUIRE(c >= 1 && c <= GN_MAX_C, "pp_group_norm: channels must be in [1,1024]");
  PP_REQUIRE(groups >= 1 && c % groups == 0, "pp_group_norm: the groups must divide the channels");
  PP_REQUIRE(n >= 0 && n <= ((int64_t)1 << 40) && b >= 0 && b <= ((int64_t)1 << 31) / groups, "pp_group_norm: rows or batch out of range");
  PP_REQUIRE(offsets, "pp_group_norm: null offsets");
  return PP_OK;
}

extern "C" int pp_group_norm_fwd(const void* x, int32_t dtype, int64_t n, int32_t c, int32_t groups, const int64_t* offsets, int64_t b,
                                 const int64_t* order, const float* weight, const float* bias, double eps, int32_t act, float slope,
                                 void* y, float* mean, float* rstd, void* ws, size_t ws_bytes, pp_stream_t stream) {
  int rc = gn_check(dtype, n, c, groups, offsets, b, act);
  if (rc != PP_OK) return rc;
  PP_REQUIRE((n == 0 || (x && y)) && (b == 0 || (mean && rstd)) && ws, "pp_group_norm_fwd: null pointer");
  PP_REQUIRE((uintptr_t)ws % 16 == 0, "pp_group_norm_fwd: the workspace must be 16-byte aligned");
  if (ws_bytes < pp_group_norm_workspace(n, b, c, groups, 0)) {
    pp_set_error("pp_group_norm_fwd: workspace too small");
    return PP_ERR_WORKSPACE;
  }
  GnArgs a{};
  a.x = x; a.out = y; a.n = n; a.c = c; a.g = groups; a.off = offsets; a.b = b; a.order = order;
  a.weight = weight; a.bias = bias; a.eps = eps; a.act = act; a.slope = slope; a.mean = mean; a.rstd = rstd;
  a.slots = (double*)ws;
  return gn_dispatch<true>(a, dtype, pp_s(stream));
}

extern "C" int pp_group_norm_bwd(const void* x, const void* dy, int32_t dtype, int64_t n, int32_t c, int32_t groups,
                                 const int64_t* offsets, int64_t b, const int64_t* order, const float* weight, const float* bias,
                                 const float* mean, const float* rstd, int32_t act, float slope, void* dx, float* dweight, float* dbias,
                                 void* ws, size_t ws_bytes, pp_stream_t stream) {
  int rc = gn_check(dtype, n, c, groups, offsets, b, act);
  if (rc != PP_OK) return rc;
  PP_REQUIRE((n == 0 || (x && dy && dx)) && (b == 0 || (mean && rstd)) && ws, "pp_group_norm_bwd: null pointer");
  PP_REQUIRE((uintptr_t)ws % 16 == 0, "pp_group_norm_bwd: the workspace must be 16-byte aligned");
  if (ws_bytes < pp_group_norm_workspace(n, b, c, groups, 1)) {
    pp_set_error("pp_group_norm_bwd: workspace too small");
    return PP_ERR_WORKSPACE;
  }
  GnArgs a{};
  a.x = x; a.dy = dy; a.out = dx; a.n = n; a.c = c; a.g = groups; a.off = offsets; a.b = b; a.order = order;
  a.weight = weight; a.bias = bias; a.act = act; a.slope = slope;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dweight = dweight; a.dbias = dbias;
  PPArena arena(ws, ws_bytes);
  a.slots = arena.take<double>(((size_t)gn_chunks(n) + b + 1) * 2 * c);
  a.totals = arena.take<double>((size_t)(gn_chunks(n) + 1) * 2 * c);
  a.coef = arena.take<float>((size_t)b * groups * 2);
  PP_REQUIRE(a.slots && a.totals && a.coef, "pp_group_norm_bwd: workspace layout");
  return gn_dispatch<false>(a, dtype, pp_s(stream));
}

// Group normalisation over the rows of a batch element, with an activation, on [rows, channels] features (channels last).
//
// Batch element s owns the positions [off[s], off[s+1]) of the row sequence (position p = row order[p], or row p); group g its
// C / G neighbouring channels.  With m = rows of s times C / G:
//   d = x - pivot,  mean = pivot + sum d / m,  var = sum d^2 / m - (sum d / m)^2,  xh = (x - mean) / sqrt(var + eps),  z = xh w_c + b_c,  y = act(z)
//   dz = dy act'(z);  db_c = sum dz, dw_c = sum dz xh over ALL rows;  h = dz w_c;  dx = rstd (h - mean_g(h) - xh mean_g(h xh))
// All sums are fp64, of the distances d to a pivot, the first value that a group has in its batch element: a difference of mean squares
// loses (distance / std)^2 of the accumulator's precision, and a mean lies within sqrt(m) std of any of its values, however far from 0 it
// is (squares of x itself: 70 k equal values of 30000 had a spread of 5e-4, 1 / std 1.2 % off).  No atomics: a chunk of positions
// writes its sums to slots of its own, and they are added in a fixed order, so results repeat bit for bit.
//
// The row sequence is cut into chunks, whatever the batch elements' lengths are.  The pairs (chunk j, element s) that meet form a
// staircase, along which j + s grows by one at every step: slot j + s is its pair's alone, and an element's slots are neighbours.
// Two launches: the chunks' sums, and the rows, whose workgroups first add the slots of their elements.
// Offsets and row orders are read on the device and not trusted: positions are clamped to [0, rows], rows outside are passed over.
#include "pp_rows.h"

#define GN_MAX_CHUNKS 1024
#define GN_MAX_C 1024
#define GN_FINISH_BLOCKS (1 << 22)

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
  double* slots;        // [slot][g][2]: sums of d, d^2 forward, of h, h xh backward
  float* pivot;         // forward [b, g]
  double* totals;       // backward [chunk][2][c]: sums of dz, dz xh; null: nobody wants the parameters' gradients
  float* coef;          // backward [b, g][2]: mean(h), mean(h xh), where k_gn_finish makes them
  float *dweight, *dbias;
  int64_t rows_per_chunk, rows_per_block;  // positions of a workgroup of the first, and of the second pass
  int chunks, blocks;
};

// first i in [from, count] with off[i] > p (count if there is none); the whole wave searches, 64 offsets a turn
__device__ __forceinline__ int64_t gn_upper(const int64_t* __restrict__ off, int64_t from, int64_t count, int64_t p) {
  const int lane = threadIdx.x & 63;
  int64_t lo = from, hi = count < from + 64 ? count : from + 64;
  for (bool near = from > 0;; near = false) {  // behind an element that has been found, the next one is mostly its neighbour
    if (!near) hi = count;
    while (hi - lo > 64) {
      const int64_t step = (hi - lo + 63) / 64, i = lo + (lane + 1) * step - 1;
      const unsigned long long over = __ballot(i >= hi || off[i] > p);
      const int first = over ? __builtin_ctzll(over) : 63;
      lo += first * step;
      hi = lo + step < hi ? lo + step : hi;
    }
    const unsigned long long over = __ballot(lo + lane < hi && off[lo + lane] > p);
    if (over) return lo + __builtin_ctzll(over);
    if (!near) return count;
    lo = hi;
  }
}
__device__ __forceinline__ int64_t gn_clamp(int64_t v, int64_t n) { return v < 0 ? 0 : (v > n ? n : v); }

// A chunk: its first position, and where its rows lie in x, dy and out (without an order, from here on)
template <typename T, bool ORDER>
struct GnChunk {
  int64_t start;
  int len;
  const T *x, *dy;
  T* out;
  const int64_t* order;
  __device__ GnChunk(const GnArgs& a, int64_t rows) {
    start = (int64_t)blockIdx.x * rows;
    len = (int)(a.n - start < rows ? a.n - start : rows);
    const int64_t at = ORDER ? 0 : start * a.c;
    x = (const T*)a.x + at;
    dy = (const T*)a.dy + at;
    out = (T*)a.out + at;
    order = ORDER ? a.order + start : nullptr;
  }
  // the element at position p of the chunk (uniform): false if there is none; *e: where it or the rows of none end
  __device__ __forceinline__ bool element(const GnArgs& a, int p, int64_t* hi, int64_t* s, int* e) const {
    *hi = gn_upper(a.off, *hi, a.b + 1, start + p);
    int64_t end = len;
    if (*hi <= a.b) {
      const int64_t o = a.off[*hi] - start;
      end = o < end ? o : end;
    }
    // (an end behind p in any case, whatever is written over the offsets meanwhile)
    *e = __builtin_amdgcn_readfirstlane(end > p ? (int)end : p + 1);
    *s = *hi - 1;
    return *hi > 0 && *hi <= a.b;
  }
};

// Where a thread's rows p, p + step, .. < e of a chunk lie: element offsets of U rows at a time, negative behind the end.  ORDER: the
// rows' numbers are read from the order, a turn ahead of the rows
template <bool B> struct GnOffset { typedef int type; };
template <> struct GnOffset<true> { typedef int64_t type; };
template <bool ORDER, int U>
struct GnRows {
  typedef typename GnOffset<ORDER>::type Offset;
  int q, e, step;
  Offset next[ORDER ? U : 1];
  template <typename Chunk>
  __device__ __forceinline__ GnRows(const GnArgs& a, const Chunk& ch, int p, int end, int step_) : q(p), e(end), step(step_) {
    if (ORDER) ask(a, ch);
  }
  template <typename Chunk>
  __device__ __forceinline__ void ask(const GnArgs& a, const Chunk& ch) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int pos = q + i * step;
      const int64_t r = pos < e ? ch.order[pos] : -1;
      next[ORDER ? i : 0] = r >= 0 && r < a.n ? (Offset)(r * a.c) : -1;  // (an order that holds no row there: passed over)
    }
  }
  __device__ __forceinline__ bool more() const { return q < e; }
  template <typename Chunk>
  __device__ __forceinline__ void turn(const GnArgs& a, const Chunk& ch, Offset (&at)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i) at[i] = ORDER ? next[ORDER ? i : 0] : (q + i * step < e ? (Offset)((q + i * step) * a.c) : -1);
    q += U * step;
    if (ORDER) ask(a, ch);
  }
};

// A block's threads over a chunk: `lpr` threads side by side on a row (VEC channels each, NC times 256 threads apart where a row is
// wider than the block), `rps` rows at a time
template <int VEC, int NC>
struct GnLane {
  int lpr, rps, rin, cc;
  bool on;
  int group[NC][VEC];  // of the thread's channels
  __device__ GnLane(const GnArgs& a) {
    const int cv = a.c / VEC, cg = a.c / a.g;
    lpr = cv < 256 ? cv : 256;
    rps = 256 / lpr;
    rin = threadIdx.x / lpr;
    cc = threadIdx.x - rin * lpr;
    on = rin < rps;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int u = 0; u < VEC; ++u) group[k][u] = on && has(k, a.c) ? (channel(k) + u) / cg : 0;
  }
  __device__ int channel(int k) const { return (cc + 256 * k) * VEC; }
  __device__ bool has(int k, int c) const { return NC == 1 || channel(k) < c; }
};

// weight and bias of a thread's channels
template <int VEC, int NC>
struct GnAffine {
  float w[NC][VEC], b[NC][VEC];
  template <typename Lane>
  __device__ GnAffine(const GnArgs& a, const Lane& ln) {
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

// a vector on its way: kept as it lies in memory
template <typename T, int VEC>
struct GnRaw {
  typename PPVec<T, VEC>::type v;
  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (VEC == 1) v[0] = *p; else v = *(const typename PPVec<T, VEC>::type*)p;
  }
  __device__ __forceinline__ float operator[](int u) const { return (float)v[u]; }
};

// the pivots of a thread's channels in element s: the first channel of the group in the element's first row r, at position o (0 where there is none,
// r < 0).  The chunk that begins the element at o leaves them for the second pass
template <bool ORDER>
__device__ __forceinline__ int64_t gn_first_row(const GnArgs& a, int64_t s, int64_t* o) {
  *o = gn_clamp(a.off[s], a.n);
  int64_t r = *o < a.n ? *o : -1;
  if (ORDER && r >= 0) r = a.order[*o];
  return r < a.n ? r : -1;
}
template <typename T, int VEC, int NC, typename Lane>
__device__ __forceinline__ void gn_pivots(const GnArgs& a, const Lane& ln, int64_t s, int64_t r, bool begins, float (&pv)[NC][VEC]) {
  const int cg = a.c / a.g;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int u = 0; u < VEC; ++u) pv[k][u] = r >= 0 ? (float)((const T*)a.x)[r * a.c + ln.group[k][u] * cg] : 0.f;
  if (!begins || ln.rin != 0) return;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int u = 0; u < VEC; ++u)
      if (ln.has(k, a.c) && ln.channel(k) + u == ln.group[k][u] * cg) a.pivot[s * a.g + ln.group[k][u]] = pv[k][u];
}

// A thread's sums over the rows [p, e) of an element -> LDS red[2][rps][c], times the channel's weight backward.
// FORWARD: d, d^2, the pivots read behind the first rows; else dz, dz xh, which are added to the thread's totals as they are
template <typename T, int VEC, int NC, bool FORWARD, bool ORDER, typename Lane>
__device__ __forceinline__ void gn_rows_sum(const GnArgs& a, const GnChunk<T, ORDER>& chunk, const Lane& ln, const GnAffine<VEC, NC>& af, int p, int e,
                                            int64_t s, float (&mu)[NC][VEC], const float (&rs)[NC][VEC], double* __restrict__ red,
                                            double (&t0)[FORWARD ? 1 : NC][VEC], double (&t1)[FORWARD ? 1 : NC][VEC]) {
  if (!ln.on) return;
  double s0[NC][VEC], s1[NC][VEC];
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int u = 0; u < VEC; ++u) s0[k][u] = s1[k][u] = 0.0;
  constexpr int U = NC > 1 ? 1 : FORWARD || sizeof(T) == 2 ? 4 : 2;  // rows in flight
  int64_t o = 0, first = 0;
  if (FORWARD) first = gn_first_row<ORDER>(a, s, &o);
  bool pivots = false;
  GnRows<ORDER, U> rows(a, chunk, p + ln.rin, e, ln.rps);
  while (rows.more()) {
    GnRaw<T, VEC> xr[U][NC], dr[U][NC];
    typename GnOffset<ORDER>::type at[U];
    rows.turn(a, chunk, at);
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (at[i] >= 0 && ln.has(k, a.c)) {
          xr[i][k].load(chunk.x + (at[i] + ln.channel(k)));
          if (!FORWARD) dr[i][k].load(chunk.dy + (at[i] + ln.channel(k)));
        }
    if (FORWARD && !pivots) {
      gn_pivots<T, VEC, NC>(a, ln, s, first, chunk.start + p == o, mu);
      pivots = true;
    }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (at[i] >= 0 && ln.has(k, a.c)) {
#pragma unroll
          for (int u = 0; u < VEC; ++u) {
            if (FORWARD) {
              const double v = (double)xr[i][k][u] - (double)mu[k][u];
              s0[k][u] += v;
              s1[k][u] = fma(v, v, s1[k][u]);
            } else {
              const float d = xr[i][k][u] - mu[k][u], xh = d * rs[k][u];
              const double dz = (double)(dr[i][k][u] * pp_dact1(fmaf(d, rs[k][u] * af.w[k][u], af.b[k][u]), a.act, a.slope));
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
        const double w = FORWARD ? 1.0 : (double)af.w[k][u];
        red[ln.rin * a.c + ln.channel(k) + u] = w * s0[k][u];
        red[(ln.rps + ln.rin) * a.c + ln.channel(k) + u] = w * s1[k][u];
        if constexpr (!FORWARD) {
          t0[k][u] += s0[k][u];
          t1[k][u] += s1[k][u];
        }
      }
    }
}

// group sums of red[2][rps][c]: calls put(g, sum0, sum1) on one thread per group.  `tpg` neighbouring threads (a power of two, at most
// a wave) share a group
template <typename Put>
__device__ __forceinline__ void gn_group_sums(const GnArgs& a, int rps, const double* __restrict__ red, Put put) {
  int tpg = 64;
  while (tpg > 1 && tpg * a.g > 256) tpg >>= 1;
  const int cg = a.c / a.g, j = threadIdx.x & (tpg - 1), step = 256 / tpg;
  const int dr = tpg / cg, dc = tpg - dr * cg, r0 = j / cg, c0 = j - r0 * cg;
  for (int g0 = 0; g0 < a.g; g0 += step) {  // uniform bounds: the shuffles below need the whole wave
    const int g = g0 + (int)threadIdx.x / tpg;
    double v0 = 0.0, v1 = 0.0;
    if (g < a.g) {
      int ch = c0;
      for (int r = r0; r < rps;) {
        v0 += red[r * a.c + g * cg + ch];
        v1 += red[(rps + r) * a.c + g * cg + ch];
        r += dr;
        ch += dc;
        if (ch >= cg) {
          ch -= cg;
          ++r;
        }
      }
    }
    for (int d = tpg >> 1; d > 0; d >>= 1) {
      v0 += __shfl_xor(v0, d);
      v1 += __shfl_xor(v1, d);
    }
    if (j == 0 && g < a.g) put(g, v0, v1);
  }
}

// mean and 1/std from the sums over m values' distances to the pivot
__device__ __forceinline__ void gn_moments(double s0, double s1, double m, double eps, float pivot, float* mean, float* rstd) {
  const double mu = s0 / m, var = s1 / m - mu * mu;
  *mean = (float)((double)pivot + mu);
  *rstd = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + eps));  // (a NaN stays one)
}

// y or dx of the rows [p, e) of one batch element.  z = (x - mean) (rstd w) + b both ways, the same three operations, so that the two agree
// about the side of a kink.  x - mean comes first: it is exact where x is near the mean (one-row elements, constant channels: z = b), where
// x (rstd w) + (b - mean rstd w) would leave |x| rstd 2^-24, with rstd up to 1 / sqrt(eps).  Backward ka, kb = mean(h), mean(h xh)
template <typename T, int VEC, int NC, bool FORWARD, bool ORDER, typename Lane>
__device__ __forceinline__ void gn_rows_apply(const GnArgs& a, const GnChunk<T, ORDER>& chunk, const Lane& ln, const GnAffine<VEC, NC>& af, int p, int e,
                                              const float (&mu)[NC][VEC], const float (&rs)[NC][VEC], const float (&ka)[NC][VEC],
                                              const float (&kb)[NC][VEC]) {
  if (!ln.on) return;
  // rows in flight: forward three, what 64 registers hold with mean, rstd w and b (2.5 M x 96 bf16, gelu: 375 us a pass, 392 with four)
  constexpr int U = NC > 1 ? 1 : FORWARD ? 3 : 4;
  GnRows<ORDER, U> rows(a, chunk, p + ln.rin, e, ln.rps);
  while (rows.more()) {
    GnRaw<T, VEC> xr[U][NC], dr[U][NC];
    typename GnOffset<ORDER>::type at[U];
    rows.turn(a, chunk, at);
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (at[i] >= 0 && ln.has(k, a.c)) {
          xr[i][k].load(chunk.x + (at[i] + ln.channel(k)));
          if (!FORWARD) dr[i][k].load(chunk.dy + (at[i] + ln.channel(k)));
        }
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (at[i] >= 0 && ln.has(k, a.c)) {
          float o[VEC];
          if (FORWARD) {
#pragma unroll
            for (int u = 0; u < VEC; ++u) o[u] = fmaf(xr[i][k][u] - mu[k][u], ka[k][u], af.b[k][u]);
            pp_act(o, a.act, a.slope);
          } else {
            float xh[VEC], z[VEC];
#pragma unroll
            for (int u = 0; u < VEC; ++u) {
              const float d = xr[i][k][u] - mu[k][u];
              xh[u] = d * rs[k][u];
              z[u] = fmaf(d, rs[k][u] * af.w[k][u], af.b[k][u]);
              o[u] = dr[i][k][u] * af.w[k][u];
            }
            pp_dact(o, z, a.act, a.slope);
#pragma unroll
            for (int u = 0; u < VEC; ++u) o[u] = rs[k][u] * (o[u] - ka[k][u] - xh[u] * kb[k][u]);
          }
          pp_store<T, VEC>(chunk.out + (at[i] + ln.channel(k)), o);
        }
  }
}

// rows at positions [p, e) that belong to no batch element: zeros
template <typename T, int VEC, int NC, bool ORDER, typename Lane>
__device__ __forceinline__ void gn_rows_zero(const GnArgs& a, const GnChunk<T, ORDER>& chunk, const Lane& ln, int p, int e) {
  if (!ln.on) return;
  const float o[VEC] = {};
  GnRows<ORDER, 1> rows(a, chunk, p + ln.rin, e, ln.rps);
  while (rows.more()) {
    typename GnOffset<ORDER>::type at[1];
    rows.turn(a, chunk, at);
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (at[0] >= 0 && ln.has(k, a.c)) pp_store<T, VEC>(chunk.out + (at[0] + ln.channel(k)), o);
  }
}

// per-(element, group) values of a thread's channels: v[k][u] = table[(s * g + group) * stride]
template <int VEC, int NC, typename Lane>
__device__ __forceinline__ void gn_per_channel(const GnArgs& a, const Lane& ln, const float* __restrict__ table, int stride,
                                               int64_t s, float (&v)[NC][VEC]) {
  const float* const row = table + s * a.g * stride;
#pragma unroll
  for (int k = 0; k < NC; ++k)
#pragma unroll
    for (int u = 0; u < VEC; ++u) v[k][u] = row[ln.group[k][u] * stride];
}

// ---- first pass: the sums of a chunk's elements ---------------------------------------------------------------------------------------
template <typename T, int VEC, int NC, bool FORWARD, bool ORDER>
__global__ __launch_bounds__(256, NC == 1 ? 4 : 1) void k_gn_chunk_sums(GnArgs a) {
  extern __shared__ double red[];
  const GnLane<VEC, NC> ln(a);
  const GnAffine<VEC, NC> af(a, ln);
  const GnChunk<T, ORDER> chunk(a, a.rows_per_chunk);
  double t0[FORWARD ? 1 : NC][VEC] = {}, t1[FORWARD ? 1 : NC][VEC] = {};
  int64_t hi = 0, s;
  for (int p = 0, e; p < chunk.len; p = e) {
    if (!chunk.element(a, p, &hi, &s, &e)) continue;
    const int64_t slot = (int64_t)blockIdx.x + s;
    float mu[NC][VEC] = {}, rs[NC][VEC] = {};
    if (!FORWARD) {
      gn_per_channel<VEC, NC>(a, ln, a.mean, 1, s, mu);
      gn_per_channel<VEC, NC>(a, ln, a.rstd, 1, s, rs);
    }
    gn_rows_sum<T, VEC, NC, FORWARD, ORDER>(a, chunk, ln, af, p, e, s, mu, rs, red, t0, t1);
    __syncthreads();
    gn_group_sums(a, ln.rps, red, [&](int g, double v0, double v1) {
      a.slots[(slot * a.g + g) * 2] = v0;
      a.slots[(slot * a.g + g) * 2 + 1] = v1;
    });
    __syncthreads();
  }
  if constexpr (!FORWARD) {
    if (!a.totals) return;
    if (ln.on)
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (ln.has(k, a.c)) {
#pragma unroll
          for (int u = 0; u < VEC; ++u) {
            red[ln.rin * a.c + ln.channel(k) + u] = t0[k][u];
            red[(ln.rps + ln.rin) * a.c + ln.channel(k) + u] = t1[k][u];
          }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.c; i += 256) {
      const int part = i >= a.c, ch = i - part * a.c;
      double v = 0.0;
#pragma unroll 4
      for (int r = 0; r < ln.rps; ++r) v += red[(part * ln.rps + r) * a.c + ch];
      a.totals[(int64_t)blockIdx.x * 2 * a.c + i] = v;
    }
  }
}

// what the second pass takes from the sums of a group: mean and 1/std forward, the two means backward
template <bool FORWARD>
__device__ __forceinline__ void gn_stat(const GnArgs& a, int64_t s, int g, double v0, double v1, double m, float* first, float* second) {
  if (FORWARD) {
    gn_moments(v0, v1, m, a.eps, a.pivot[s * a.g + g], first, second);
  } else {
    *first = (float)(v0 / m);
    *second = (float)(v1 / m);
  }
}
// floor(v / d) of numbers below 2^53: the quotient of their doubles is off by less than one
__device__ __forceinline__ int64_t gn_quotient(int64_t v, int64_t d) {
  int64_t q = (int64_t)((double)v / (double)d);
  if (q * d > v) --q;
  return q;
}
// the slots of element s are those of the chunks j0 .. j1 it lies in, at j + s
__device__ __forceinline__ bool gn_slots(const GnArgs& a, int64_t s, int64_t* j0, int64_t* j1, double* m) {
  const int64_t o0 = gn_clamp(a.off[s], a.n), o1 = gn_clamp(a.off[s + 1], a.n);
  if (o1 <= o0) return false;
  *j0 = gn_quotient(o0, a.rows_per_chunk);
  *j1 = gn_quotient(o1 - 1, a.rows_per_chunk);
  *m = (double)(o1 - o0) * (a.c / a.g);
  return true;
}

// dweight and dbias of four channels from the chunks' totals.  red: 512 doubles
__device__ __forceinline__ void gn_parameters(const GnArgs& a, int block, double* __restrict__ red) {
  const int cl = threadIdx.x & 3, j = threadIdx.x >> 2, ch = block * 4 + cl;
  double v0 = 0.0, v1 = 0.0;
  if (ch < a.c) {
#pragma unroll 4
    for (int q = j; q < a.chunks; q += 64) {
      v0 += a.totals[(int64_t)q * 2 * a.c + ch];
      v1 += a.totals[((int64_t)q * 2 + 1) * a.c + ch];
    }
  }
  red[threadIdx.x] = v0;
  red[256 + threadIdx.x] = v1;
  __syncthreads();
  if (j >= 2 || ch >= a.c) return;
  v0 = 0.0;
#pragma unroll 8
  for (int q = 0; q < 64; ++q) v0 += red[256 * j + q * 4 + cl];
  if (j == 0 && a.dbias) a.dbias[ch] = (float)v0;
  if (j == 1 && a.dweight) a.dweight[ch] = (float)v0;
}

// Between the passes: one wave per (element, group) adds its slots, in turns where there are more than GN_FINISH_BLOCKS workgroups' worth (a
// launch has less than 2^32 threads); backward, the workgroups behind them make the parameters' gradients
template <bool FORWARD>
__global__ __launch_bounds__(256) void k_gn_finish(GnArgs a, int64_t group_blocks) {
  if (!FORWARD && (int64_t)blockIdx.x >= group_blocks) {
    __shared__ double red[512];
    gn_parameters(a, (int)(blockIdx.x - group_blocks), red);
    return;
  }
  const int lane = threadIdx.x & 63;
  for (int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); w < a.b * a.g; w += group_blocks * 4) {
    const int64_t s = w / a.g;
    const int g = (int)(w - s * a.g);
    int64_t j0, j1;
    double m, v0 = 0.0, v1 = 0.0;
    const bool any = gn_slots(a, s, &j0, &j1, &m);
    if (any)
      for (int64_t j = j0 + lane; j <= j1; j += 64) {
        v0 += a.slots[((j + s) * a.g + g) * 2];
        v1 += a.slots[((j + s) * a.g + g) * 2 + 1];
      }
    for (int d = 32; d > 0; d >>= 1) {
      v0 += __shfl_xor(v0, d);
      v1 += __shfl_xor(v1, d);
    }
    if (lane != 0) continue;
    float first = 0.f, second = 0.f;
    if (any) gn_stat<FORWARD>(a, s, g, v0, v1, m, &first, &second);
    (FORWARD ? a.mean : a.coef)[FORWARD ? w : 2 * w] = first;
    (FORWARD ? a.rstd : a.coef)[FORWARD ? w : 2 * w + 1] = second;
  }
}

// The same inside the second pass: the workgroup's threads over slots and groups, -> stat[g][2] in the LDS, and to mean and rstd by the
// workgroup that has the element's first row.  red: 512 doubles
template <bool FORWARD>
__device__ __forceinline__ void gn_inline_stats(const GnArgs& a, int64_t s, bool first_rows, double* __restrict__ red, float* __restrict__ stat) {
  int64_t j0 = 0, j1 = -1;
  double m = 1.0;
  gn_slots(a, s, &j0, &j1, &m);
  const int gw = a.g < 256 ? a.g : 256, S = 256 / gw, sl = threadIdx.x / gw, gi = threadIdx.x - sl * gw;
  for (int g0 = 0; g0 < a.g; g0 += gw) {
    const int g = g0 + gi;
    double v0 = 0.0, v1 = 0.0;
    if (sl < S && g < a.g) {
#pragma unroll 4
      for (int64_t j = j0 + sl; j <= j1; j += S) {
        v0 += a.slots[((j + s) * a.g + g) * 2];
        v1 += a.slots[((j + s) * a.g + g) * 2 + 1];
      }
    }
    __syncthreads();  // (the last element's rows have read stat, the last turn's sums have been read)
    red[threadIdx.x] = v0;
    red[256 + threadIdx.x] = v1;
    __syncthreads();
    if (sl == 0 && g < a.g) {
      for (int k = 1; k < S; ++k) {
        v0 += red[k * gw + gi];
        v1 += red[256 + k * gw + gi];
      }
      gn_stat<FORWARD>(a, s, g, v0, v1, m, &stat[2 * g], &stat[2 * g + 1]);
      if (FORWARD && first_rows) {
        a.mean[s * a.g + g] = stat[2 * g];
        a.rstd[s * a.g + g] = stat[2 * g + 1];
      }
    }
  }
  __syncthreads();
}

// ---- second pass: the rows ----------------------------------------------------------------------------------------------------------
// INLINE: the element's slots are added here, and workgroups behind those of the rows write what no row does: backward the parameters'
// gradients, forward zeros as the statistics of batch elements without rows, 256 of them each
template <typename T, int VEC, int NC, bool FORWARD, bool ORDER, bool INLINE>
__global__ __launch_bounds__(256, NC > 1 ? 1 : INLINE ? 4 : FORWARD ? 8 : 5) void k_gn_chunk_apply(GnArgs a) {
  extern __shared__ double red[];                            // INLINE: 512 doubles
  float* const stat = (float*)(red + (INLINE ? 512 : 0));    // [g][2]
  if (INLINE && (int)blockIdx.x >= a.blocks) {
    const int block = (int)blockIdx.x - a.blocks;
    if (!FORWARD) return gn_parameters(a, block, red);
    const int64_t s = (int64_t)block * 256 + threadIdx.x;
    if (s < a.b && gn_clamp(a.off[s + 1], a.n) <= gn_clamp(a.off[s], a.n))
      for (int g = 0; g < a.g; ++g) a.mean[s * a.g + g] = a.rstd[s * a.g + g] = 0.f;
    return;
  }
  const GnLane<VEC, NC> ln(a);
  const GnAffine<VEC, NC> af(a, ln);
  const GnChunk<T, ORDER> chunk(a, a.rows_per_block);
  int64_t hi = 0, s;
  for (int p = 0, e; p < chunk.len; p = e) {
    if (!chunk.element(a, p, &hi, &s, &e)) {
      gn_rows_zero<T, VEC, NC, ORDER>(a, chunk, ln, p, e);
      continue;
    }
    float mu[NC][VEC], rs[NC][VEC], ka[NC][VEC] = {}, kb[NC][VEC] = {};
    if (!FORWARD || !INLINE) {
      gn_per_channel<VEC, NC>(a, ln, a.mean, 1, s, mu);
      gn_per_channel<VEC, NC>(a, ln, a.rstd, 1, s, rs);
    }
    if (INLINE) {
      gn_inline_stats<FORWARD>(a, s, chunk.start + p == gn_clamp(a.off[s], a.n), red, stat);
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int u = 0; u < VEC; ++u) {
          const int g = ln.group[k][u];
          (FORWARD ? mu : ka)[k][u] = stat[2 * g];
          (FORWARD ? rs : kb)[k][u] = stat[2 * g + 1];
        }
    } else if (!FORWARD) {
      gn_per_channel<VEC, NC>(a, ln, a.coef, 2, s, ka);
      gn_per_channel<VEC, NC>(a, ln, a.coef + 1, 2, s, kb);
    }
    if (FORWARD) {
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int u = 0; u < VEC; ++u) ka[k][u] = rs[k][u] * af.w[k][u];
    }
    gn_rows_apply<T, VEC, NC, FORWARD, ORDER>(a, chunk, ln, af, p, e, mu, rs, ka, kb);
  }
}

// ---- launches ---------------------------------------------------------------------------------------------------------------------
// First pass: at most GN_MAX_CHUNKS chunks, which all find room on the chip at once.  Second pass: the same while a workgroup has less than
// 64 KiB to do, then as many as it takes (a few rounds of workgroups leave no compute unit idle at the end for long)
static int64_t gn_rows_per_chunk(int64_t n) {
  const int64_t r = (n + GN_MAX_CHUNKS - 1) / GN_MAX_CHUNKS;
  return r < 32 ? 32 : r;
}
static int64_t gn_rows_per_block(int64_t n, int64_t row_bytes) {
  const int64_t r = gn_rows_per_chunk(n), most = 65536 / row_bytes < 32 ? 32 : 65536 / row_bytes, least = n / (1 << 30) + 1;
  return (r < most ? r : most) > least ? (r < most ? r : most) : least;
}
static int gn_chunks(int64_t n) { return (int)((n + gn_rows_per_chunk(n) - 1) / gn_rows_per_chunk(n)); }

extern "C" size_t pp_group_norm_workspace(int64_t n, int64_t b, int32_t c, int32_t groups, int32_t backward) {
  if (n < 0 || b < 0 || c < 1 || groups < 1) return 0;
  const size_t slots = pp_align(((size_t)gn_chunks(n) + (size_t)b + 1) * groups * 2 * sizeof(double));
  if (!backward) return slots + pp_align((size_t)b * groups * sizeof(float) + 1);
  return slots + pp_align((size_t)(gn_chunks(n) + 1) * 2 * c * sizeof(double)) +
         pp_align((size_t)b * groups * 2 * sizeof(float) + 1);
}

// The second pass adds an element's slots itself where that is at most GN_INLINE bytes for an element of average length, and all of its
// workgroups fit on the chip at once (a launch less); a longer one is better off with the registers that takes, so that more waves hide
// its loads (2.5 M x 96 bf16, 64 elements, gelu: rows 407 us inline, 279 us at half as many registers)
#define GN_INLINE (64 * 1024)
template <typename T, int VEC, int NC, bool FORWARD, bool ORDER>
static void gn_sums(const GnArgs& a, hipStream_t s) {
  const int cv = a.c / VEC, rps = 256 / (cv < 256 ? cv : 256);
  hipLaunchKernelGGL((k_gn_chunk_sums<T, VEC, NC, FORWARD, ORDER>), dim3(a.chunks), dim3(256), (size_t)rps * a.c * 2 * sizeof(double), s, a);
}
template <typename T, int VEC, int NC, bool FORWARD, bool ORDER>
static int gn_launch(GnArgs& a, hipStream_t s) {
  a.rows_per_chunk = gn_rows_per_chunk(a.n);
  a.chunks = gn_chunks(a.n);
  a.rows_per_block = gn_rows_per_block(a.n, (int64_t)a.c * sizeof(T));
  a.blocks = a.out ? (int)((a.n + a.rows_per_block - 1) / a.rows_per_block) : 0;  // (backward without dx: no second pass)
  const bool in = a.b > 0 && a.blocks <= GN_MAX_CHUNKS && (a.chunks / a.b + 2) * a.g * (int64_t)(2 * sizeof(double)) <= GN_INLINE;
  if (a.chunks) {
    // eight channels of 16 bits at a time where the loads bound, as in long forward sums (2.5 M x 96: 126 us, 170 us with four); elsewhere
    // the registers they take cost more waves than they are worth (see gn_order)
    constexpr int WIDE = FORWARD && sizeof(T) == 2 && VEC == 4 ? 8 : VEC;
    if (WIDE != VEC && !in && a.c % WIDE == 0 && (uintptr_t)a.x % 16 == 0)
      gn_sums<T, WIDE, NC, FORWARD, ORDER>(a, s);
    else
      gn_sums<T, VEC, NC, FORWARD, ORDER>(a, s);
    PP_LAUNCH_CHECK();
  }
  const int64_t gw = (a.b * a.g + 3) / 4, gb = gw < GN_FINISH_BLOCKS ? gw : GN_FINISH_BLOCKS, pb = FORWARD || !a.totals ? 0 : (a.c + 3) / 4;
  if (in) {
    const int64_t more = FORWARD ? (a.b + 255) / 256 : pb;
    if (a.blocks + more == 0) return PP_OK;
    hipLaunchKernelGGL((k_gn_chunk_apply<T, VEC, NC, FORWARD, ORDER, true>), dim3((unsigned)(a.blocks + more)), dim3(256),
                       512 * sizeof(double) + (size_t)a.g * 2 * sizeof(float), s, a);
    PP_LAUNCH_CHECK();
    return PP_OK;
  }
  if (gb + pb) {
    hipLaunchKernelGGL((k_gn_finish<FORWARD>), dim3((unsigned)(gb + pb)), dim3(256), 0, s, a, gb);
    PP_LAUNCH_CHECK();
  }
  if (a.blocks) {
    hipLaunchKernelGGL((k_gn_chunk_apply<T, VEC, NC, FORWARD, ORDER, false>), dim3((unsigned)a.blocks), dim3(256), 0, s, a);
    PP_LAUNCH_CHECK();
  }
  return PP_OK;
}

// Vectors of four channels where every row starts on one; single elements else.  (Eight channels of 16 bits are the wider load, but the
// registers they take leave half the waves: 1500 elements, 180 k x 64 bf16, backward sums 140 us with eight, 38 us with four.)
template <typename T, int VEC, int NC, bool FORWARD>
static int gn_order(GnArgs& a, hipStream_t s) {
  return a.order ? gn_launch<T, VEC, NC, FORWARD, true>(a, s) : gn_launch<T, VEC, NC, FORWARD, false>(a, s);
}
template <typename T, bool FORWARD>
static int gn_type(GnArgs& a, hipStream_t s) {
  constexpr int VEC = 4;
  const uintptr_t at = (uintptr_t)a.x | (uintptr_t)a.dy | (uintptr_t)a.out;
  if (a.c % VEC == 0 && at % (VEC * sizeof(T)) == 0) return gn_order<T, VEC, 1, FORWARD>(a, s);
  return a.c <= 256 ? gn_order<T, 1, 1, FORWARD>(a, s) : gn_order<T, 1, GN_MAX_C / 256, FORWARD>(a, s);
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
  PP_REQUIRE(n >= 0 && n <= ((int64_t)1 << 39) / c && b >= 0 && b <= ((int64_t)1 << 31) / groups, "pp_group_norm: rows or batch out of range");
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
  PPArena arena(ws, ws_bytes);
  a.slots = arena.take<double>(((size_t)gn_chunks(n) + b + 1) * 2 * groups);
  a.pivot = arena.take<float>((size_t)b * groups);
  PP_REQUIRE(a.slots && a.pivot, "pp_group_norm_fwd: workspace layout");
  return gn_dispatch<true>(a, dtype, pp_s(stream));
}

extern "C" int pp_group_norm_bwd(const void* x, const void* dy, int32_t dtype, int64_t n, int32_t c, int32_t groups,
                                 const int64_t* offsets, int64_t b, const int64_t* order, const float* weight, const float* bias,
                                 const float* mean, const float* rstd, int32_t act, float slope, void* dx, float* dweight, float* dbias,
                                 void* ws, size_t ws_bytes, pp_stream_t stream) {
  int rc = gn_check(dtype, n, c, groups, offsets, b, act);
  if (rc != PP_OK) return rc;
  PP_REQUIRE((n == 0 || (x && dy)) && (b == 0 || (mean && rstd)) && ws, "pp_group_norm_bwd: null pointer");
  PP_REQUIRE((uintptr_t)ws % 16 == 0, "pp_group_norm_bwd: the workspace must be 16-byte aligned");
  if (!dx && !dweight && !dbias) return PP_OK;
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
  a.slots = arena.take<double>(((size_t)gn_chunks(n) + b + 1) * 2 * groups);
  a.totals = arena.take<double>((size_t)(gn_chunks(n) + 1) * 2 * c);
  a.coef = arena.take<float>((size_t)b * groups * 2);
  PP_REQUIRE(a.slots && a.totals && a.coef, "pp_group_norm_bwd: workspace layout");
  if (!dweight && !dbias) a.totals = nullptr;
  return gn_dispatch<false>(a, dtype, pp_s(stream));
}

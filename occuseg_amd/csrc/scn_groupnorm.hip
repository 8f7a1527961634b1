// Group norm over ragged samples with its activation, channels last (gfx950); the sample offsets it runs over.
//
//   y = act((x - mean_sg) rstd_sg w_c + b_c),   statistics over the n_s sites of sample s x the C / G planes of group g
//   dz = dy act'(z), xh = (x - mean) rstd, dn = dz w:
//   dx = rstd (dn - <dn> - xh <dn xh>),  db_c = sum dz,  dw_c = sum dz xh      (<> over the same n_s C / G values)
//
// HBM bound: forward reads x twice and writes y, backward reads x and dy twice and writes dx; a sample's values are needed before
// its statistics are known, and 154 MB (600k sites x 64 planes) do not stay on the chip.
//
// Three launches a direction: sums per CHUNK of rows, a join of the chunks in fp64 in a fixed order, the apply pass.  A chunk is
// 2^shift rows of one sample: chunk b belongs to the last sample s with (offsets[s] >> shift) + s <= b, which needs no table, no
// read-back of the lengths, and at most (N >> shift) + samples workgroups.  The rows of a chunk are one contiguous span, walked in
// 16-byte vectors whatever C is: the vectors step through the span by a multiple of lcm(C, vector), so every thread keeps the same
// planes, and their constants, for the whole chunk.
#include "scn_pointwise.h"

namespace scn {

struct GnArgs {
  const int64_t *offsets;
  int64_t N;
  int S, C, G, cpg;
  int shift;   // rows per chunk = 1 << shift
  int period;  // vectors per lcm(C, V) elements; a thread steps by a multiple of it
  int step;    // ... this many vectors (a multiple of `period`; of at most 256 vectors if that is possible)
  float leak;
};

// the sample and the rows of chunk b; false: an empty chunk.  Every wave finds it by itself, 64 samples a look: one look for up to 64
// samples, three for 65535.
__device__ __forceinline__ bool gn_chunk(const GnArgs &a, int64_t b, int &s, int64_t &r0, int64_t &r1) {
  s = 0;
  for (int hi = a.S;;) {  // the sample looked for is in s .. hi - 1
    const int step = (hi - s + 63) >> 6, i = s + lane_id() * step;
    const int n = __popcll(__ballot(i < hi && (a.offsets[min(i, a.S - 1)] >> a.shift) + i <= b));
    if (n == 0) return false;
    s += (n - 1) * step;
    if (step == 1) break;
    hi = min(hi, s + step);
  }
  const int64_t start = max(a.offsets[s], (int64_t)0), end = min(a.offsets[s + 1], a.N);
  r0 = start + ((b - ((start >> a.shift) + s)) << a.shift);
  r1 = min(r0 + ((int64_t)1 << a.shift), end);
  return start <= r0 && r0 < r1;  // (the first: offsets that do not ascend are never followed outside of the tensor)
}

// The apply passes take the chunks from the last to the first, eight at a time: what the sums pass read last is still in the XCD's L2
// (workgroup ids go round the 8 of them, chunk b stays on b % 8) and in the memory-side cache: 600k x 64 in fp32, a train pass, 226 us;
// 234 from the first to the last.
__device__ __forceinline__ int64_t gn_backwards(int chunk_blocks) {
  const int b = blockIdx.x;
  return (int64_t)(((chunk_blocks + 7) / 8 - 1 - b / 8) * 8 + b % 8);
}

// f(i, vector) for the thread's vectors of the span [0, span) of p: vector q, q + step, ...; the span's last vector may be partial,
// its missing elements are zeros.
template <int UNROLL, class T, int V, class F>
__device__ __forceinline__ void gn_walk(const T *p, int span, int q, int step, F &&f) {
  int i = q * V;
  const int d = step * V;
  for (; i + (UNROLL - 1) * d + V <= span; i += UNROLL * d) {
    Pack<T, V> v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) v[u] = load_pack<T, V>(p + i + u * d);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) f(i + u * d, V, v[u]);
  }
  for (; i < span; i += d) {
    Pack<T, V> v;
    const int n = min(V, span - i);
    if (n == V) v = load_pack<T, V>(p + i);
    else
#pragma unroll
      for (int j = 0; j < V; ++j) v.v[j] = j < n ? p[i + j] : (T)0.f;
    f(i, n, v);
  }
}
// ... of two tensors: f(i, n, vector of p, vector of g), all of a round requested before any is used
template <int UNROLL, class T, int V, class F>
__device__ __forceinline__ void gn_walk2(const T *p, const T *g, int span, int q, int step, F &&f) {
  int i = q * V;
  const int d = step * V;
  for (; i + (UNROLL - 1) * d + V <= span; i += UNROLL * d) {
    Pack<T, V> v[UNROLL], w[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      v[u] = load_pack<T, V>(p + i + u * d);
      w[u] = load_pack<T, V>(g + i + u * d);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) f(i + u * d, V, v[u], w[u]);
  }
  for (; i < span; i += d) {
    Pack<T, V> v, w;
    const int n = min(V, span - i);
    if (n == V) {
      v = load_pack<T, V>(p + i);
      w = load_pack<T, V>(g + i);
    } else
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v.v[j] = j < n ? p[i + j] : (T)0.f;
        w.v[j] = j < n ? g[i + j] : (T)0.f;
      }
    f(i, n, v, w);
  }
}
template <class T, int V>
__device__ __forceinline__ void gn_store(T *p, int n, const Pack<T, V> &v) {
  if (n == V) store_pack<T, V>(p, v);
  else
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) p[j] = v.v[j];
}

// f(j, plane's group, (mean, rstd), weight, bias) for the V planes of vector q in sample s.  Planes that lie side by side come by 16
// bytes, and one pair of statistics serves them all if they are of one group: 8 planes take 5 loads instead of 24.
template <int V, class F>
__device__ __forceinline__ void gn_planes(const GnArgs &a, int q, const float2 *stats, const float *weight, const float *bias, F &&f) {
  int c = q * V % a.C, g = c / a.cpg, r = c % a.cpg;
  if (a.C % V == 0) {
    Pack<float, V> w, b;
#pragma unroll
    for (int j = 0; j < V; ++j) w.v[j] = 1.f, b.v[j] = 0.f;
    if (weight) w = load_pack<float, V>(weight + c);
    if (bias) b = load_pack<float, V>(bias + c);
    float2 st = stats[g];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f(j, g, st, w.v[j], b.v[j]);
      if (j < V - 1 && ++r == a.cpg) r = 0, st = stats[++g];
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    f(j, g, stats[g], weight ? weight[c] : 1.f, bias ? bias[c] : 0.f);
    ++c;
    if (++r == a.cpg) r = 0, ++g;
    if (c == a.C) c = g = 0;
  }
}

// ------------------------------------------------------------------ forward ---
// partial[chunk][group] = (mean, sum of squared deviations).  Every thread sums its planes' deviations from the plane's first value
// in the chunk: sums of squares of values far from zero would cancel.  The entries are joined by the deviations of their means.
template <class T, int V>
__global__ void __launch_bounds__(256) k_gn_stats(const T *x, GnArgs a, float2 *partial) {
  extern __shared__ float2 ent[];  // [step * V] (mean, squared deviations) per element of a step
  int s;
  int64_t r0, r1;
  if (!gn_chunk(a, blockIdx.x, s, r0, r1)) return;
  const int span = (int)(r1 - r0) * a.C, E = a.step * V;
  const int full = span / E, rest = span % E;  // element e of a step is in full + (e < rest) of them
  const T *p = x + r0 * a.C;
  for (int q = threadIdx.x; q < a.step; q += 256) {
    float pivot[V], s1[V], s2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) pivot[j] = s1[j] = s2[j] = 0.f;
    gn_walk<8, T, V>(p, span, q, a.step, [&](int i, int n, const Pack<T, V> &v) {
      if (i == q * V)
#pragma unroll
        for (int j = 0; j < V; ++j) pivot[j] = (float)v.v[j];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = j < n ? (float)v.v[j] - pivot[j] : 0.f;
        s1[j] += d;
        s2[j] = fmaf(d, d, s2[j]);
      }
    });
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = q * V + j;
      const float m = e < span ? s1[j] / (float)(full + (e < rest)) : 0.f;
      ent[e] = make_float2(pivot[j] + m, e < span ? fmaxf(s2[j] - s1[j] * m, 0.f) : 0.f);
    }
  }
  __syncthreads();
  // tpg threads (a power of two, within a wave) per group
  int tpg = 64;
  while (tpg > 1 && tpg * a.G > 256) tpg >>= 1;
  const int sub = threadIdx.x & (tpg - 1), dk = tpg / a.cpg * a.C, dj = tpg % a.cpg, k0 = sub / a.cpg * a.C, j0 = sub % a.cpg;
  // f(entry, how many values it stands for) for this thread's entries of group g: planes g cpg .. of every row of a step
  auto entries = [&](int g, auto &&f) __attribute__((always_inline)) {
    for (int k = k0, j = j0; k < E;) {
      const int e = k + g * a.cpg + j;
      if (e < span) f(ent[e], (float)(full + (e < rest)));
      k += dk;
      j += dj;
      if (j >= a.cpg) j -= a.cpg, k += a.C;
    }
  };
  for (int g0 = 0; g0 < a.G; g0 += 256 / tpg) {
    const int g = g0 + threadIdx.x / tpg;
    const bool on = g < a.G;
    float pv = 0.f, sum = 0.f, sq = 0.f, mean = 0.f;
    if (on) {
      pv = ent[g * a.cpg].x;  // (row 0 is there)
      entries(g, [&](float2 v, float n) { sum = fmaf(n, v.x - pv, sum); });
    }
    for (int o = 1; o < tpg; o <<= 1) sum += __shfl_xor(sum, o);
    if (on) {
      mean = pv + sum / (float)((int)(r1 - r0) * a.cpg);
      entries(g, [&](float2 v, float n) { sq += fmaf(n * (v.x - mean), v.x - mean, v.y); });
    }
    for (int o = 1; o < tpg; o <<= 1) sq += __shfl_xor(sq, o);
    if (on && sub == 0) partial[(int64_t)blockIdx.x * a.G + g] = make_float2(mean, sq);
  }
}

// stats[s][g] = (mean, rstd): the chunks' means and deviations joined in fp64, in a fixed order.  Workgroup (s, y): JOIN groups of one
// sample, each by 1024 / JOIN threads.
constexpr int JOIN = 4;
__global__ void __launch_bounds__(1024) k_gn_join(const float2 *partial, GnArgs a, double eps, float2 *stats) {
  __shared__ double red[2][16][JOIN];
  const int s = blockIdx.x, g = blockIdx.y * JOIN + threadIdx.x % JOIN, slot = threadIdx.x / JOIN, wave = threadIdx.x >> 6;
  const int64_t start = max(a.offsets[s], (int64_t)0), end = min(a.offsets[s + 1], a.N), rows = end - start;
  const int64_t b0 = (start >> a.shift) + s;
  const int chunks = rows > 0 ? (int)((rows + ((int64_t)1 << a.shift) - 1) >> a.shift) : 0;
  double s1 = 0, s2 = 0;
  if (g < a.G)
#pragma unroll 4
    for (int c = slot; c < chunks; c += 1024 / JOIN) {
      const float2 v = partial[(b0 + c) * a.G + g];
      const double n = (double)min(rows - ((int64_t)c << a.shift), (int64_t)1 << a.shift) * a.cpg, m = v.x;
      s1 += n * m;
      s2 += (double)v.y + n * m * m;
    }
#pragma unroll
  for (int o = JOIN; o < 64; o <<= 1) {
    s1 += __shfl_xor(s1, o);
    s2 += __shfl_xor(s2, o);
  }
  if (lane_id() < JOIN) {
    red[0][wave][lane_id()] = s1;
    red[1][wave][lane_id()] = s2;
  }
  __syncthreads();
  if (threadIdx.x >= JOIN || g >= a.G) return;
  s1 = s2 = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    s1 += red[0][k][threadIdx.x];
    s2 += red[1][k][threadIdx.x];
  }
  float2 out = make_float2(0.f, 0.f);
  if (chunks > 0) {  // (NaN in the sample: fmax drops it; the mean has it)
    const double n = (double)rows * a.cpg, m = s1 / n, var = fmax(s2 / n - m * m, 0.0);
    out = make_float2((float)m, (float)(1.0 / sqrt(var + eps)));
  }
  stats[(int64_t)s * a.G + g] = out;
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(256)
    k_gn_apply(const T *x, T *y, GnArgs a, const float2 *stats, const float *weight, const float *bias, int chunk_blocks) {
  int s;
  int64_t r0, r1;
  if (!gn_chunk(a, gn_backwards(chunk_blocks), s, r0, r1)) return;
  const int span = (int)(r1 - r0) * a.C;
  const T *p = x + r0 * a.C;
  T *o = y + r0 * a.C;
  for (int q = threadIdx.x; q < a.step; q += 256) {
    float mean[V], w[V], b[V];
    gn_planes<V>(a, q, stats + (int64_t)s * a.G, weight, bias, [&](int j, int, float2 st, float wj, float bj) {
      mean[j] = st.x;
      w[j] = st.y * wj;
      b[j] = bj;
    });
    gn_walk<4, T, V>(p, span, q, a.step, [&](int i, int n, const Pack<T, V> &v) {
      Pack<T, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[j] = (T)act_value<ACT, T>(fmaf((float)v.v[j] - mean[j], w[j], b[j]), a.leak);
      gn_store<T, V>(o + i, n, r);
    });
  }
}

// Few sites: one launch, a workgroup per sample and group that keeps its values in registers (402 sites x 448 planes, 32 groups, fp32:
// 7.6 us on the device, 18 with the call; 25 in three launches).  1024 threads x GN_SMALL_PER values, in
// row order: a thread's next value is 1024 values on.
constexpr int GN_SMALL_PER = 32;
template <class T, int ACT>
__global__ void __launch_bounds__(1024)
    k_gn_small(const T *x, T *y, GnArgs a, double eps, float2 *stats, const float *weight, const float *bias) {
  __shared__ float red[16];
  const int s = blockIdx.x, g = blockIdx.y;
  const int64_t start = max(a.offsets[s], (int64_t)0), end = min(a.offsets[s + 1], a.N);
  const int n = (int)max(end - start, (int64_t)0) * a.cpg;
  float2 *st = stats + (int64_t)s * a.G + g;
  if (n == 0) {
    if (threadIdx.x == 0) *st = make_float2(0.f, 0.f);
    return;
  }
  auto block_sum = [&](float v) __attribute__((always_inline)) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if (lane_id() == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) v += red[w];
    return v;
  };
  const int dr = 1024 / a.cpg, dj = 1024 % a.cpg, r0 = (int)threadIdx.x / a.cpg, j0 = (int)threadIdx.x % a.cpg;
  const int64_t base = start * a.C + g * a.cpg;
  const T *p = x + base;
  const float pivot = (float)p[0];
  float v[GN_SMALL_PER], sum = 0.f, sq = 0.f;
  int r = r0, j = j0;
#pragma unroll
  for (int i = 0; i < GN_SMALL_PER; ++i) {
    v[i] = 0.f;
    if (1024 * i < n) {  // (uniform)
      if (1024 * i + (int)threadIdx.x < n) v[i] = (float)p[(int64_t)r * a.C + j] - pivot;
      r += dr;
      j += dj;
      if (j >= a.cpg) j -= a.cpg, ++r;
    }
  }
#pragma unroll
  for (int i = 0; i < GN_SMALL_PER; ++i) sum += v[i];
  const float mean = block_sum(sum) / (float)n;  // (of the deviations from the pivot)
#pragma unroll
  for (int i = 0; i < GN_SMALL_PER; ++i) {
    v[i] -= mean;
    if (1024 * i + (int)threadIdx.x < n) sq = fmaf(v[i], v[i], sq);
  }
  const float rstd = (float)(1.0 / sqrt((double)block_sum(sq) / n + eps));
  if (threadIdx.x == 0) *st = make_float2(pivot + mean, rstd);
  r = r0, j = j0;
#pragma unroll
  for (int i = 0; i < GN_SMALL_PER; ++i) {
    if (1024 * i >= n) break;
    if (1024 * i + (int)threadIdx.x < n) {
      const int c = g * a.cpg + j;
      y[base + (int64_t)r * a.C + j] =
          (T)act_value<ACT, T>(fmaf(v[i], rstd * (weight ? weight[c] : 1.f), bias ? bias[c] : 0.f), a.leak);
    }
    r += dr;
    j += dj;
    if (j >= a.cpg) j -= a.cpg, ++r;
  }
}

// ----------------------------------------------------------------- backward ---
// partial[chunk][plane] = (sum dz, sum dz xh).  Slopes as exact as fp32 features': d_weight and d_bias are fp32, and the errors of
// 16-bit features' slopes, below their rounding, would be the largest there.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(256)
    k_gn_bwd_sums(const T *x, const T *dy, GnArgs a, const float2 *stats, const float *weight, const float *bias, float2 *partial) {
  extern __shared__ float2 ent[];
  int s;
  int64_t r0, r1;
  if (!gn_chunk(a, blockIdx.x, s, r0, r1)) return;
  const int span = (int)(r1 - r0) * a.C, E = a.step * V;
  const T *p = x + r0 * a.C, *g = dy + r0 * a.C;
  for (int q = threadIdx.x; q < a.step; q += 256) {
    float mean[V], rstd[V], w[V], b[V], s1[V], s2[V];
    gn_planes<V>(a, q, stats + (int64_t)s * a.G, weight, bias, [&](int j, int, float2 st, float wj, float bj) {
      mean[j] = st.x;
      rstd[j] = st.y;
      w[j] = st.y * wj;
      b[j] = bj;
      s1[j] = s2[j] = 0.f;
    });
    gn_walk2<4, T, V>(p, g, span, q, a.step, [&](int i, int n, const Pack<T, V> &v, const Pack<T, V> &d) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float c = (float)v.v[j] - mean[j];
        const float dz = j < n ? (float)d.v[j] * act_slope<ACT, float>(fmaf(c, w[j], b[j]), a.leak) : 0.f;
        s1[j] += dz;
        s2[j] = fmaf(dz, c * rstd[j], s2[j]);
      }
    });
#pragma unroll
    for (int j = 0; j < V; ++j) ent[q * V + j] = make_float2(s1[j], s2[j]);
  }
  __syncthreads();
  // a plane's entries: the rows of a step, by `slots` threads if there are several a plane
  const int slots = a.C <= 128 ? 256 / a.C : 1;
  float2 *out = partial + (int64_t)blockIdx.x * a.C;
  for (int t0 = threadIdx.x; t0 < a.C * slots; t0 += 256) {
    float2 t = make_float2(0.f, 0.f);
    for (int e = t0; e < E; e += a.C * slots) {
      t.x += ent[e].x;
      t.y += ent[e].y;
    }
    if (slots == 1) out[t0] = t;
    else ent[t0] = t;  // (nobody else reads this entry)
  }
  if (slots == 1) return;
  __syncthreads();
  if ((int)threadIdx.x < a.C) {
    float2 t = ent[threadIdx.x];
    for (int k = 1; k < slots; ++k) {
      t.x += ent[threadIdx.x + k * a.C].x;
      t.y += ent[threadIdx.x + k * a.C].y;
    }
    out[threadIdx.x] = t;
  }
}

// sums[s][plane]: the chunks of one sample, fp64, in a fixed order; 8 planes x 128 slots a workgroup
constexpr int BJOIN = 8;
__global__ void __launch_bounds__(1024) k_gn_bwd_join(const float2 *partial, GnArgs a, float2 *sums) {
  __shared__ double red[2][16][BJOIN];
  const int s = blockIdx.x, c = blockIdx.y * BJOIN + threadIdx.x % BJOIN, slot = threadIdx.x / BJOIN, wave = threadIdx.x >> 6;
  const int64_t start = max(a.offsets[s], (int64_t)0), end = min(a.offsets[s + 1], a.N), rows = end - start;
  const int64_t b0 = (start >> a.shift) + s;
  const int chunks = rows > 0 ? (int)((rows + ((int64_t)1 << a.shift) - 1) >> a.shift) : 0;
  double s1 = 0, s2 = 0;
  if (c < a.C)
#pragma unroll 4
    for (int k = slot; k < chunks; k += 1024 / BJOIN) {
      const float2 v = partial[(b0 + k) * a.C + c];
      s1 += v.x;
      s2 += v.y;
    }
#pragma unroll
  for (int o = BJOIN; o < 64; o <<= 1) {
    s1 += __shfl_xor(s1, o);
    s2 += __shfl_xor(s2, o);
  }
  if (lane_id() < BJOIN) {
    red[0][wave][lane_id()] = s1;
    red[1][wave][lane_id()] = s2;
  }
  __syncthreads();
  if (threadIdx.x >= BJOIN || c >= a.C) return;
  s1 = s2 = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    s1 += red[0][k][threadIdx.x];
    s2 += red[1][k][threadIdx.x];
  }
  sums[(int64_t)s * a.C + c] = make_float2((float)s1, (float)s2);
}

// dx; the workgroups behind the chunks add the planes' sums over the samples (d_weight, d_bias), fp64, in a fixed order: PLANES planes x
// 256 / PLANES slots each.  (One thread a plane takes 0.27 us a sample: 5000 samples of 26 sites x 64, fp32, a backward pass of 1372 us, 170
// so; 512 of 254 sites 165 and 47.)
constexpr int PLANES = 4;
template <class T, int V, int ACT>
__global__ void __launch_bounds__(256)
    k_gn_bwd_apply(const T *x, const T *dy, T *dx, GnArgs a, const float2 *stats, const float *weight, const float *bias,
                   const float2 *sums, float *d_weight, float *d_bias, int chunk_blocks) {
  extern __shared__ float2 grp[];  // [G] (<dn>, <dn xh>)
  __shared__ double red[2][4][PLANES];
  const int padded = (chunk_blocks + 7) / 8 * 8;
  if ((int)blockIdx.x >= padded) {
    const int c = ((int)blockIdx.x - padded) * PLANES + threadIdx.x % PLANES, wave = threadIdx.x >> 6;
    double s1 = 0, s2 = 0;
    if (c < a.C)
#pragma unroll 4
      for (int s = threadIdx.x / PLANES; s < a.S; s += 256 / PLANES) {
        const float2 v = sums[(int64_t)s * a.C + c];
        s1 += v.x;
        s2 += v.y;
      }
#pragma unroll
    for (int o = PLANES; o < 64; o <<= 1) {
      s1 += __shfl_xor(s1, o);
      s2 += __shfl_xor(s2, o);
    }
    if (lane_id() < PLANES) {
      red[0][wave][lane_id()] = s1;
      red[1][wave][lane_id()] = s2;
    }
    __syncthreads();
    if (threadIdx.x >= PLANES || c >= a.C) return;
    s1 = s2 = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s1 += red[0][k][threadIdx.x];
      s2 += red[1][k][threadIdx.x];
    }
    if (d_bias) d_bias[c] = (float)s1;
    if (d_weight) d_weight[c] = (float)s2;
    return;
  }
  int s;
  int64_t r0, r1;
  if (!gn_chunk(a, gn_backwards(chunk_blocks), s, r0, r1)) return;
  const int64_t rows = min(a.offsets[s + 1], a.N) - max(a.offsets[s], (int64_t)0);
  for (int g = threadIdx.x; g < a.G; g += 256) {
    float m1 = 0.f, m2 = 0.f;
    for (int c = g * a.cpg; c < (g + 1) * a.cpg; ++c) {
      const float2 v = sums[(int64_t)s * a.C + c];
      const float w = weight ? weight[c] : 1.f;
      m1 = fmaf(w, v.x, m1);
      m2 = fmaf(w, v.y, m2);
    }
    const float n = (float)rows * (float)a.cpg;
    grp[g] = make_float2(m1 / n, m2 / n);
  }
  __syncthreads();
  const int span = (int)(r1 - r0) * a.C;
  const T *p = x + r0 * a.C, *g = dy + r0 * a.C;
  T *o = dx + r0 * a.C;
  for (int q = threadIdx.x; q < a.step; q += 256) {
    float mean[V], w[V], b[V], m1[V], m2[V];
    gn_planes<V>(a, q, stats + (int64_t)s * a.G, weight, bias, [&](int j, int gi, float2 st, float wj, float bj) {
      mean[j] = st.x;
      w[j] = st.y * wj;
      b[j] = bj;
      m1[j] = grp[gi].x * st.y;
      m2[j] = grp[gi].y * st.y * st.y;
    });
    gn_walk2<4, T, V>(p, g, span, q, a.step, [&](int i, int n, const Pack<T, V> &v, const Pack<T, V> &d) {
      Pack<T, V> r;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float c = (float)v.v[j] - mean[j];
        const float dz = (float)d.v[j] * act_slope<ACT, T>(fmaf(c, w[j], b[j]), a.leak);
        r.v[j] = (T)(fmaf(dz, w[j], -m1[j]) - c * m2[j]);
      }
      gn_store<T, V>(o + i, n, r);
    });
  }
}

// ------------------------------------------------------------ sample offsets ---
// offsets[s] = first site whose key is at or behind sample s's first key: the keys ascend
__global__ void k_sample_offsets(const uint64_t *keys, int64_t N, int64_t S, int64_t *offsets) {
  for (int64_t s = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; s <= S; s += (int64_t)gridDim.x * blockDim.x) {
    int64_t lo = 0, hi = N;
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if ((int64_t)(keys[mid] >> 31) < s) lo = mid + 1; else hi = mid;
    }
    offsets[s] = s == S ? N : lo;
  }
}

// ---------------------------------------------------------------------- host ---
static int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// 16-byte vectors if their period fits a workgroup, single elements else (an odd plane count above 256)
static bool gn_wide(int C, int V) { return C / gcd(C, V) <= 256 || C % V == 0; }

static GnArgs gn_args(const int64_t *offsets, int64_t N, int C, int G, int64_t S, int dtype, int V, double leak) {
  GnArgs a;
  a.offsets = offsets;
  a.N = N;
  a.S = (int)S;
  a.C = C;
  a.G = G;
  a.cpg = C / G;
  a.leak = (float)leak;
  a.period = C / gcd(C, V);
  a.step = a.period <= 256 ? 256 / a.period * a.period : a.period;
  // Chunks of 32 KB of a large tensor: 154 MB in fp32 take 91 us forwards, 100 with 16 KB; 45 MB in bf16 36, 38 with 64 KB.  Of a small one
  // 512 chunks, none below 16 KB.
  const int64_t row = (int64_t)C * (dtype == SCN_F32 ? 4 : 2), most = 32768;
  int64_t bytes = N * row / 512;
  bytes = bytes < 16384 ? 16384 : bytes > most ? most : bytes;
  a.shift = 0;
  while (a.shift < 20 && (row << (a.shift + 1)) <= bytes) ++a.shift;
  return a;
}
static int64_t gn_chunks(const GnArgs &a) { return (a.N >> a.shift) + a.S; }

// The one-launch path, by what was measured on the device (fp32; one launch / three, which cost the host some 5 us more):
//   at most 512 workgroups, two a CU: 1024 sites x 512 planes in groups of one, 4 samples: 34 / 12 us; x 128: 9.6 / 10.3
//   values a workgroup, on average: groups of one, 4 groups, 1 sample: 8192 sites 8.3 / 10.3 us, 16,384 11.7 / 10.3
//   elements in all, a group of fewer than four planes as four (a row of a group costs its cache line however little of it is wanted):
//   groups of one, 4 samples: 4096 sites x 32 6.2 / 10.4 us, 32,768 x 32 16.7 / 11.3, 32,768 x 1024 417 / 98
// and, as one sample may have all N sites, a group's values fit the registers whatever the lengths are.
static bool gn_small(int64_t N, int C, int G, int64_t S) {
  const int64_t cpg = C / G, values = N * cpg;
  return values <= 1024 * GN_SMALL_PER && S * G <= 512 && values <= S * 8192 && N * G * (cpg < 4 ? 4 : cpg) <= 1 << 20;
}

template <class T, int V>
static int gn_forward(const void *x, void *y, float *stats, GnArgs a, const float *weight, const float *bias, double eps, int act,
                      void *temp, hipStream_t st) {
  const unsigned chunks = (unsigned)gn_chunks(a);
  float2 *partial = (float2 *)temp;
  if (gn_small(a.N, a.C, a.G, a.S)) {
    auto small = act == SCN_ACT_SILU ? k_gn_small<T, SCN_ACT_SILU> : act == SCN_ACT_GELU ? k_gn_small<T, SCN_ACT_GELU> : k_gn_small<T, SCN_ACT_LEAKY>;
    small<<<dim3(a.S, a.G), 1024, 0, st>>>((const T *)x, (T *)y, a, eps, (float2 *)stats, weight, bias);
    SCN_CHECK_LAUNCH();
    return 0;
  }
  k_gn_stats<T, V><<<chunks, 256, sizeof(float2) * a.step * V, st>>>((const T *)x, a, partial);
  SCN_CHECK_LAUNCH();
  k_gn_join<<<dim3(a.S, (a.G + JOIN - 1) / JOIN), 1024, 0, st>>>(partial, a, eps, (float2 *)stats);
  SCN_CHECK_LAUNCH();
  auto apply = act == SCN_ACT_SILU ? k_gn_apply<T, V, SCN_ACT_SILU>
               : act == SCN_ACT_GELU ? k_gn_apply<T, V, SCN_ACT_GELU> : k_gn_apply<T, V, SCN_ACT_LEAKY>;
  apply<<<(chunks + 7) / 8 * 8, 256, 0, st>>>((const T *)x, (T *)y, a, (const float2 *)stats, weight, bias, (int)chunks);
  SCN_CHECK_LAUNCH();
  return 0;
}

template <class T, int V>
static int gn_backward(const void *x, const void *dy, void *dx, const float *stats, GnArgs a, const float *weight, const float *bias,
                       float *d_weight, float *d_bias, int act, void *temp, hipStream_t st) {
  const unsigned chunks = (unsigned)gn_chunks(a);
  float2 *partial = (float2 *)temp, *sums = partial + (int64_t)chunks * a.C;
  auto k1 = act == SCN_ACT_SILU ? k_gn_bwd_sums<T, V, SCN_ACT_SILU>
            : act == SCN_ACT_GELU ? k_gn_bwd_sums<T, V, SCN_ACT_GELU> : k_gn_bwd_sums<T, V, SCN_ACT_LEAKY>;
  k1<<<chunks, 256, sizeof(float2) * a.step * V, st>>>((const T *)x, (const T *)dy, a, (const float2 *)stats, weight, bias, partial);
  SCN_CHECK_LAUNCH();
  k_gn_bwd_join<<<dim3(a.S, (a.C + BJOIN - 1) / BJOIN), 1024, 0, st>>>(partial, a, sums);
  SCN_CHECK_LAUNCH();
  auto k2 = act == SCN_ACT_SILU ? k_gn_bwd_apply<T, V, SCN_ACT_SILU>
            : act == SCN_ACT_GELU ? k_gn_bwd_apply<T, V, SCN_ACT_GELU> : k_gn_bwd_apply<T, V, SCN_ACT_LEAKY>;
  k2<<<(chunks + 7) / 8 * 8 + (a.C + PLANES - 1) / PLANES, 256, sizeof(float2) * a.G, st>>>((const T *)x, (const T *)dy, (T *)dx, a, (const float2 *)stats,
                                                                  weight, bias, sums, d_weight, d_bias, (int)chunks);
  SCN_CHECK_LAUNCH();
  return 0;
}

static int gn_check(int64_t N, int C, int G, int64_t S, int dtype, int act) {
  SCN_REQUIRE(dtype == SCN_F32 || dtype == SCN_BF16 || dtype == SCN_F16, "group norm: dtype");
  SCN_REQUIRE(act == SCN_ACT_LEAKY || act == SCN_ACT_SILU || act == SCN_ACT_GELU, "group norm: activation");
  SCN_REQUIRE(C >= 1 && C <= SCN_GROUP_NORM_MAX_PLANES, "group norm: 1 to 4096 planes");
  SCN_REQUIRE(G >= 1 && C % G == 0, "group norm: the planes must divide into the groups");
  SCN_REQUIRE(S >= 1 && S <= 65535 && N >= 0 && N < ((int64_t)1 << 31), "group norm: 1 to 65535 samples, fewer than 2^31 sites");
  return 0;
}

template <class F>
static int gn_dispatch(int dtype, int C, F &&f) {
  const bool wide = gn_wide(C, dtype == SCN_F32 ? 4 : 8);
  if (dtype == SCN_F32) return wide ? f((float)0, std::integral_constant<int, 4>()) : f((float)0, std::integral_constant<int, 1>());
  if (dtype == SCN_BF16) return wide ? f((__bf16)0, std::integral_constant<int, 8>()) : f((__bf16)0, std::integral_constant<int, 1>());
  return wide ? f((_Float16)0, std::integral_constant<int, 8>()) : f((_Float16)0, std::integral_constant<int, 1>());
}

}  // namespace scn

using namespace scn;

extern "C" {

int scn_sample_offsets(const uint64_t *site_keys, int64_t N, int64_t samples, int64_t *offsets, void *stream) {
  SCN_REQUIRE(N >= 0 && samples >= 1 && samples < ((int64_t)1 << 31) && offsets, "sample offsets: arguments");
  k_sample_offsets<<<(unsigned)((samples + 256) / 256), 256, 0, as_stream(stream)>>>(site_keys, N, samples, offsets);
  SCN_CHECK_LAUNCH();
  return 0;
}

size_t scn_group_norm_temp_bytes(int64_t N, int planes, int groups, int64_t samples, int dtype, int backward) {
  if (gn_check(N, planes, groups, samples, dtype, 0) || (!backward && gn_small(N, planes, groups, samples))) return 0;
  const GnArgs a = gn_args(nullptr, N, planes, groups, samples, dtype, 1, 0);
  return sizeof(float2) * (size_t)(backward ? (gn_chunks(a) + samples) * planes : gn_chunks(a) * groups);
}

int scn_group_norm_forward(const void *x, void *y, float *stats, const int64_t *offsets, const float *weight, const float *bias,
                           double eps, int act, double leakiness, int64_t N, int planes, int groups, int64_t samples, int dtype,
                           void *temp, size_t temp_bytes, void *stream) {
  if (int e = gn_check(N, planes, groups, samples, dtype, act)) return e;
  SCN_REQUIRE(stats && offsets && (N == 0 || (x && y)), "group norm: pointers");
  const size_t need = scn_group_norm_temp_bytes(N, planes, groups, samples, dtype, 0);
  SCN_REQUIRE(need == 0 || (temp && temp_bytes >= need), "group norm: workspace");
  return gn_dispatch(dtype, planes, [&](auto t, auto v) {
    constexpr int V = decltype(v)::value;
    return gn_forward<decltype(t), V>(x, y, stats, gn_args(offsets, N, planes, groups, samples, dtype, V, leakiness), weight, bias,
                                      eps, act, temp, as_stream(stream));
  });
}

int scn_group_norm_backward(const void *x, const void *d_y, void *d_x, const float *stats, const int64_t *offsets,
                            const float *weight, const float *bias, float *d_weight, float *d_bias, int act, double leakiness,
                            int64_t N, int planes, int groups, int64_t samples, int dtype, void *temp, size_t temp_bytes,
                            void *stream) {
  if (int e = gn_check(N, planes, groups, samples, dtype, act)) return e;
  SCN_REQUIRE(stats && offsets && (N == 0 || (x && d_y && d_x)), "group norm: pointers");
  SCN_REQUIRE(temp && temp_bytes >= scn_group_norm_temp_bytes(N, planes, groups, samples, dtype, 1), "group norm: workspace");
  return gn_dispatch(dtype, planes, [&](auto t, auto v) {
    constexpr int V = decltype(v)::value;
    return gn_backward<decltype(t), V>(x, d_y, d_x, stats, gn_args(offsets, N, planes, groups, samples, dtype, V, leakiness), weight,
                                       bias, d_weight, d_bias, act, temp, as_stream(stream));
  });
}

}  // extern "C"

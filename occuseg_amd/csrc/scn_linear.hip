// 1x1 convolution with its epilogue, y = residual + drop(act(x W + b)), its gradients, and dropout alone (gfx950).
//
//   backward:  f = drop'(.) act'(x W + b), left by the forward pass;  dz = dy f;  dx = dz W^T;  dW = x^T dz;  db = column sums of dz
//
// Sites are many (up to 600k) and planes few (16 to 512), so the products are HBM bound but for the widest: 2 n_in n_out flops for
// n_in + n_out values, 16 to 128 flops a byte where fp32 MFMA balances at 20 and bf16 at 300.  Everything that belongs to a row is
// done while it is in registers.
//
// Products: v_mfma 16x16, the WEIGHT as the A operand and the sites as B: the four results of a lane are then four consecutive
// planes of one site -- one random-number counter, one wide store -- and 16 sites x 64 bytes a store instruction.  The order of the
// reduction is free as long as both operands agree: a lane's 16 bytes of a row, loaded straight from global memory, ARE its B
// operands (one 16x16x32 of 16-bit types, four 16x16x4 of fp32).  The weights are laid out in LDS in the order of the A operands.
#include "scn_pointwise.h"

#include <type_traits>

namespace scn {

// ------------------------------------------------------------------- dropout ---
// One launch, every element read and written once; the mask is made of the counter (20 32x32 products per 4 elements, behind the
// loads of a kernel that is HBM bound).  A thread's item: Q quads of planes of one site; `items` a row.  It keeps (row, item) by
// steps of (drow, ditem): no division.
template <class T, int Q, bool WHOLE>
__global__ void __launch_bounds__(256)
    k_dropout(const T *x, int64_t ldx, T *y, int64_t N, int C, int items, int64_t drow, int ditem, uint32_t threshold, float scale,
              const int64_t *rng) {
  const int64_t first = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row = first / items;
  int item = (int)(first - row * items);
  const RngKey key = rng_key(rng);
  for (; row < N; row += drow, item += ditem) {
    if (item >= items) {
      item -= items;
      if (++row >= N) break;
    }
    const int c = item * 4 * Q, n = WHOLE ? 4 * Q : min(4 * Q, C - c);
    const T *p = x + row * ldx + c;
    Pack<T, 4 * Q> v;
    if (n == 4 * Q) v = load_pack<T, 4 * Q>(p);
    else
#pragma unroll
      for (int j = 0; j < 4 * Q; ++j) v.v[j] = j < n ? p[j] : (T)0.f;
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      const Words w = philox(key, (uint32_t)(item * Q + u), (uint32_t)row);
#pragma unroll
      for (int j = 0; j < 4; ++j) v.v[4 * u + j] = w.w[j] >= threshold ? (T)((float)v.v[4 * u + j] * scale) : (T)0.f;
    }
    T *o = y + row * C + c;
    if (n == 4 * Q) store_pack<T, 4 * Q>(o, v);
    else
#pragma unroll
      for (int j = 0; j < 4 * Q; ++j)
        if (j < n) o[j] = v.v[j];
  }
}

__global__ void k_rng_take(int64_t *state, int64_t *used) {
  const int64_t seed = state[0], offset = state[1];
  used[0] = seed;
  used[1] = offset;
  state[1] = offset + 1;
}

// ------------------------------------------------------------------ products ---
// one k-group = four lane quarters x 16 bytes of a row: 16 fp32 or 32 16-bit values
template <class T> struct Frag;
template <> struct Frag<float> { using type = floatx4; };
template <> struct Frag<__bf16> { using type = bf16x8; };
template <> struct Frag<_Float16> { using type = halfx8; };

__device__ __forceinline__ floatx4 mma(const floatx4 &a, const floatx4 &b, floatx4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ floatx4 mma(const bf16x8 &a, const bf16x8 &b, const floatx4 &c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ floatx4 mma(const halfx8 &a, const halfx8 &b, const floatx4 &c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// n of the V elements at p, zeros behind them
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_some(const T *p, int n) {
  if (n >= V) return load_pack<T, V>(p);
  Pack<T, V> r;
#pragma unroll
  for (int j = 0; j < V; ++j) r.v[j] = j < n ? p[j] : (T)0.f;
  return r;
}
template <class T, int V>
__device__ __forceinline__ void store_some(T *p, const Pack<T, V> &v, int n) {
  if (n >= V) store_pack<T, V>(p, v);
  else
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) p[j] = v.v[j];
}

struct LinearArgs {
  const void *in, *scale;  // rows [N, K] at ld_in elements; MODE 1: times scale [N, K] (may be NULL)
  int64_t ld_in;
  const void *weight;  // MODE 0: [K, M], MODE 1: [M, K]
  const void *bias, *residual;
  int64_t ld_res;
  void *out, *factor;
  const int64_t *rng;
  int64_t N;
  int K, M;
  int groups, chunk_groups;  // k-groups in all, and per pass through LDS
  int col_blocks, row_blocks;
  uint32_t threshold;
  float leak, keep_scale;
};

constexpr int LIN_ROWS = 128;  // rows of a workgroup's tile: 4 waves x 2 x 16

// the plane of A row i of column tile t: 16 bytes of consecutive planes per lane (16-bit types: of two tiles together)
template <class T>
__device__ __forceinline__ int tile_col(int t, int i) {
  return sizeof(T) == 4 ? 16 * t + i : 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
}

// MODE 0: forward with the epilogue.  MODE 1: dx.
// A workgroup holds the weights of NT x 16 output planes in LDS -- all of K, once, if they fit (then its waves walk their rows
// without a barrier), else `chunk_groups` at a time -- and walks the row tiles row_block, row_block + row_blocks, ...
template <class T, int NT, int MODE, int ACT>
__global__ void __launch_bounds__(256) k_linear(LinearArgs a) {
  constexpr int V = Elem<T>::V, KG = 4 * V;
  constexpr bool EXACT = sizeof(T) == 4;
  using F = typename Frag<T>::type;
  extern __shared__ char smem[];
  F *wl = (F *)smem;  // [tile][k-group of the chunk][lane]
  float *bl = (float *)(wl + (size_t)NT * a.chunk_groups * 64);
  const int lane = lane_id(), wave = threadIdx.x >> 6, li = lane & 15, lq = lane >> 4;
  // the column blocks of one row block run on one XCD (workgroup ids go round the 8 of them): its rows come from that L2 once
  const int per = a.row_blocks * a.col_blocks, id = blockIdx.x;
  int cb, rb;
  if (per % (8 * a.col_blocks) == 0) {
    const int xcd = id & 7, j = id >> 3;
    cb = j % a.col_blocks;
    rb = j / a.col_blocks * 8 + xcd;
  } else {
    cb = id % a.col_blocks;
    rb = id / a.col_blocks;
  }
  const int m0 = cb * NT * 16;
  const T *in = (const T *)a.in, *sc = (const T *)a.scale, *wt = (const T *)a.weight;
  if (MODE == 0 && threadIdx.x < NT * 16) {
    const int m = m0 + threadIdx.x;
    bl[threadIdx.x] = a.bias && m < a.M ? (float)((const T *)a.bias)[m] : 0.f;
  }
  RngKey key = {};
  if (MODE == 0 && a.threshold) key = rng_key(a.rng);
  bool staged = false;
  const int64_t tiles = (a.N + LIN_ROWS - 1) / LIN_ROWS;
  for (int64_t tile = rb; tile < tiles; tile += a.row_blocks) {
    floatx4 acc[2][NT];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[u][t] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int64_t row0 = tile * LIN_ROWS + wave * 32 + li;
    // (rows behind the last are read as the last and not written)
    const T *p[2] = {in + min(row0, a.N - 1) * a.ld_in + lq * V, in + min(row0 + 16, a.N - 1) * a.ld_in + lq * V};
    const T *ps[2] = {nullptr, nullptr};
    if (MODE == 1 && sc) {
      ps[0] = sc + min(row0, a.N - 1) * a.K + lq * V;
      ps[1] = sc + min(row0 + 16, a.N - 1) * a.K + lq * V;
    }
    for (int g0 = 0; g0 < a.groups; g0 += a.chunk_groups) {
      const int ng = min(a.chunk_groups, a.groups - g0);
      if (!staged || a.groups > a.chunk_groups) {
        __syncthreads();
        for (int e = threadIdx.x; e < NT * ng * 64; e += 256) {
          const int l = e & 63, g = (e >> 6) % ng, t = (e >> 6) / ng;
          const int m = m0 + tile_col<T>(t, l & 15), k = (g0 + g) * KG + (l >> 4) * V;
          Pack<T, V> v;
          if (MODE == 1) {
            if (m < a.M) v = load_some<T, V>(wt + (int64_t)m * a.K + k, a.K - k);
            else
#pragma unroll
              for (int j = 0; j < V; ++j) v.v[j] = (T)0.f;
          } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v.v[j] = m < a.M && k + j < a.K ? wt[(int64_t)(k + j) * a.M + m] : (T)0.f;
          }
          __builtin_memcpy(&wl[((size_t)t * a.chunk_groups + g) * 64 + l], &v, 16);
        }
        __syncthreads();
        staged = true;
      }
      auto load_row = [&](int u, int g) __attribute__((always_inline)) {
        const int k = (g0 + g) * KG, left = a.K - k - lq * V;
        Pack<T, V> v = left >= V ? load_pack<T, V>(p[u] + k) : load_some<T, V>(p[u] + k, left);
        if (MODE == 1 && sc) {
          const Pack<T, V> f = left >= V ? load_pack<T, V>(ps[u] + k) : load_some<T, V>(ps[u] + k, left);
#pragma unroll
          for (int j = 0; j < V; ++j) v.v[j] = (T)((float)v.v[j] * (float)f.v[j]);
        }
        F r;
        __builtin_memcpy(&r, &v, 16);
        return r;
      };
#pragma unroll 4
      for (int g = 0; g < ng; ++g) {
        const F b0 = load_row(0, g), b1 = load_row(1, g);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const F w = wl[((size_t)t * a.chunk_groups + g) * 64 + lane];
          acc[0][t] = mma(w, b0, acc[0][t]);
          acc[1][t] = mma(w, b1, acc[1][t]);
        }
      }
    }
    constexpr int TP = V / 4;  // tiles per 16-byte store
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t row = row0 + 16 * u;
      if (row >= a.N) continue;
#pragma unroll
      for (int t = 0; t < NT; t += TP) {
        const int cl = tile_col<T>(t, 4 * lq), m = m0 + cl;
        if (m >= a.M) continue;
        Pack<T, V> y;
        if (MODE == 1) {
#pragma unroll
          for (int j = 0; j < V; ++j) y.v[j] = (T)acc[u][t + j / 4][j & 3];
        } else {
          Pack<T, V> f, res;
          if (a.residual) res = load_some<T, V>((const T *)a.residual + row * a.ld_res + m, a.M - m);
#pragma unroll
          for (int q = 0; q < TP; ++q) {
            Words w;
            if (a.threshold) w = philox(key, (uint32_t)((m >> 2) + q), (uint32_t)row);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float value, slope;
              act_value_slope<ACT, EXACT>(acc[u][t + q][j] + bl[cl + 4 * q + j], a.leak, value, slope);
              if (a.threshold) {
                const bool keep = w.w[j] >= a.threshold;
                value = keep ? value * a.keep_scale : 0.f;
                slope = keep ? slope * a.keep_scale : 0.f;
              }
              if (a.residual) value += (float)res.v[4 * q + j];
              y.v[4 * q + j] = (T)value;
              f.v[4 * q + j] = (T)slope;
            }
          }
          if (a.factor) store_some<T, V>((T *)a.factor + row * a.M + m, f, a.M - m);
        }
        store_some<T, V>((T *)a.out + row * a.M + m, y, a.M - m);
      }
    }
  }
}

// ------------------------------------------------------------------- dweight ---
// dW = x^T dz: the reduction runs over the rows, both operands are walked along their planes.  A wave's tile is 64 x 64: a lane
// loads 4 consecutive planes of a row, which are its elements of four A (B) tiles with the planes interleaved by four -- fp32
// needs nothing else; of 16-bit types eight rows are loaded and transposed in registers.  No LDS in the loop.
// Workgroup (slice, tile): four waves take the slice's row steps in turn, join through LDS and write one slab; slabs are added by
// k_linear_dw_join in slice order.
struct DwArgs {
  const void *x, *dy, *scale;
  int64_t ldx, ld_dy, N;
  int Ci, Co, tiles_i, tiles_o, slices;
  int64_t slice_rows;
  float *slab;      // [slices][Ci][Co], then [slices][Co]
  int want_bias;
};

template <class T>
__global__ void __launch_bounds__(256) k_linear_dw(DwArgs a) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int ROWS = F32 ? 4 : 32;  // rows of one step
  constexpr int RE = F32 ? 1 : 8;     // ... of one lane
  using F = typename Frag<T>::type;
  __shared__ float red[2][64 * 64 + 64];
  const int lane = lane_id(), wave = threadIdx.x >> 6, li = lane & 15, lq = lane >> 4;
  const int tiles = a.tiles_i * a.tiles_o;
  // (all tiles of a slice run on one XCD while its rows are in that L2)
  int slice, tile;
  if (a.slices % 8 == 0) {
    slice = (blockIdx.x >> 3) / tiles * 8 + (blockIdx.x & 7);
    tile = (blockIdx.x >> 3) % tiles;
  } else {
    slice = blockIdx.x / tiles;
    tile = blockIdx.x % tiles;
  }
  const int ci0 = tile / a.tiles_o * 64, co0 = tile % a.tiles_o * 64;
  const bool bias = a.want_bias && ci0 == 0;
  const int64_t r0 = slice * a.slice_rows, r1 = min(r0 + a.slice_rows, a.N);
  const int ci = ci0 + 4 * li, co = co0 + 4 * li, ni = a.Ci - ci, no = a.Co - co;
  const T *px = (const T *)a.x + ci, *pd = (const T *)a.dy + co, *ps = a.scale ? (const T *)a.scale + co : nullptr;
  floatx4 acc[4][4], sums[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sums[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  for (int64_t r = r0 + wave * ROWS; r < r1; r += 4 * ROWS) {
    Pack<T, 4> vx[RE], vd[RE];
#pragma unroll
    for (int e = 0; e < RE; ++e) {
      const int64_t row = r + lq * RE + e;
      const bool in = row < r1;
      vx[e] = load_some<T, 4>(px + row * a.ldx, in ? ni : 0);
      vd[e] = load_some<T, 4>(pd + row * a.ld_dy, in ? no : 0);
      if (ps) {
        const Pack<T, 4> f = load_some<T, 4>(ps + row * a.Co, in ? no : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) vd[e].v[j] = (T)((float)vd[e].v[j] * (float)f.v[j]);
      }
    }
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[0].v[i], vd[0].v[j], acc[i][j], 0, 0, 0);
      if (bias)
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[0][j] += vd[0].v[j];
    } else {
      F fx[4], fd[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          fx[j][e] = vx[e].v[j];
          fd[j][e] = vd[e].v[j];
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mma(fx[i], fd[j], acc[i][j]);
      if (bias) {  // column sums: a product with ones, every row of the result the same
        F one;
#pragma unroll
        for (int e = 0; e < 8; ++e) one[e] = (T)1.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[j] = mma(one, fd[j], sums[j]);
      }
    }
  }
  // column 4 li + j: fp32 has it in sums[0][j] of the four lane quarters, 16-bit types in sums[j][0] of each of them
  float bsum[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bsum[j] = F32 ? sums[0][j] : sums[j][0];
    if (F32) {
      bsum[j] += __shfl_xor(bsum[j], 16);
      bsum[j] += __shfl_xor(bsum[j], 32);
    }
  }
  // waves 2, 3 hand over to 0, 1; then 1 to 0
#pragma unroll
  for (int half = 2; half >= 1; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
      float *d = red[wave - half];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) *(floatx4 *)(d + ((i * 4 + j) * 64 + lane) * 4) = acc[i][j];
      if (lq == 0)
#pragma unroll
        for (int j = 0; j < 4; ++j) d[4096 + 4 * li + j] = bsum[j];
    }
    __syncthreads();
    if (wave < half) {
      const float *d = red[wave];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += *(const floatx4 *)(d + ((i * 4 + j) * 64 + lane) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) bsum[j] += d[4096 + 4 * li + j];
    }
    __syncthreads();
  }
  if (wave != 0) return;
  float *slab = a.slab + (int64_t)slice * a.Ci * a.Co;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = ci0 + 16 * lq + 4 * r + i;  // A row 4 lq + r of tile i
      if (row < a.Ci && no > 0) {
        Pack<float, 4> v = {{acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]}};
        store_some<float, 4>(slab + (int64_t)row * a.Co + co, v, no);
      }
    }
  if (bias && lq == 0 && no > 0) {
    Pack<float, 4> v = {{bsum[0], bsum[1], bsum[2], bsum[3]}};
    store_some<float, 4>(a.slab + (int64_t)a.slices * a.Ci * a.Co + (int64_t)slice * a.Co + co, v, no);
  }
}

// the slabs added in slice order; element e of [Ci * Co] then [Co]
template <class T>
__global__ void __launch_bounds__(256) k_linear_dw_join(const float *slab, int slices, int64_t nw, int nb, T *d_weight, T *d_bias) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= nw + nb) return;
  const bool w = e < nw;
  const float *p = w ? slab + e : slab + slices * nw + (e - nw);
  const int64_t step = w ? nw : nb;
  float s = 0.f;
#pragma unroll 8
  for (int i = 0; i < slices; ++i) s += p[i * step];
  if (w) d_weight[e] = (T)s;
  else d_bias[e - nw] = (T)s;
}

// ---------------------------------------------------------------------- host ---
static int lin_check(int64_t N, int n_in, int n_out, int dtype) {
  SCN_REQUIRE(dtype == SCN_F32 || dtype == SCN_BF16 || dtype == SCN_F16, "linear: dtype");
  SCN_REQUIRE(n_in >= 1 && n_out >= 1 && n_in <= 65536 && n_out <= 65536, "linear: 1 to 65536 planes");
  SCN_REQUIRE(N >= 0 && N < ((int64_t)1 << 31), "linear: fewer than 2^31 sites");
  return 0;
}

template <class F>
static int by_type(int dtype, F &&f) {
  if (dtype == SCN_F32) return f((float)0);
  if (dtype == SCN_BF16) return f((__bf16)0);
  return f((_Float16)0);
}

template <class T, int NT, int MODE, int ACT>
static int linear_launch(LinearArgs a, hipStream_t st) {
  constexpr int KG = 4 * Elem<T>::V, group_bytes = NT * 64 * 16;
  a.groups = (a.K + KG - 1) / KG;
  a.chunk_groups = a.groups;
  if (a.groups * group_bytes > 49152) a.chunk_groups = 32768 / group_bytes;
  a.col_blocks = (a.M + NT * 16 - 1) / (NT * 16);
  const int64_t tiles = (a.N + LIN_ROWS - 1) / LIN_ROWS;
  int64_t rows = 1024 / a.col_blocks;
  if (rows < 1) rows = 1;
  if (a.groups > a.chunk_groups || rows > tiles) rows = tiles;  // (weights that do not stay: one tile a workgroup)
  a.row_blocks = (int)rows;
  const size_t lds = (size_t)a.chunk_groups * group_bytes + NT * 16 * 4;
  k_linear<T, NT, MODE, ACT><<<(unsigned)(rows * a.col_blocks), 256, lds, st>>>(a);
  SCN_CHECK_LAUNCH();
  return 0;
}
template <class T, int MODE, int ACT>
static int linear_by_width(const LinearArgs &a, hipStream_t st) {
  if (a.M <= 32) return linear_launch<T, 2, MODE, ACT>(a, st);
  if (a.M <= 64) return linear_launch<T, 4, MODE, ACT>(a, st);
  return linear_launch<T, 8, MODE, ACT>(a, st);
}

// rows a slice of dW holds: enough slices to fill the chip with its tiles, no slice below 256 rows
static int dw_slices(int64_t N, int n_in, int n_out) {
  const int64_t tiles = (int64_t)((n_in + 63) / 64) * ((n_out + 63) / 64);
  int64_t s = (1024 + tiles - 1) / tiles, most = (N + 255) / 256;
  if (s > most) s = most;
  if (s >= 8) s &= ~(int64_t)7;
  return (int)(s < 1 ? 1 : s);
}

}  // namespace scn

using namespace scn;

extern "C" {

int scn_dropout(const void *x, int64_t ldx, void *y, int64_t N, int planes, int dtype, double p, const int64_t *rng, void *stream) {
  if (int e = lin_check(N, planes, 1, dtype)) return e;
  SCN_REQUIRE(p >= 0 && p < 1, "dropout: 0 <= p < 1");
  if (N == 0) return 0;
  SCN_REQUIRE(x && y && rng && ldx >= planes, "dropout: pointers");
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int Q = Elem<T>::V / 4;
    const bool whole = planes % (4 * Q) == 0;
    const int items = (planes + 4 * Q - 1) / (4 * Q);
    int64_t blocks = (N * items + 255) / 256;
    if (blocks > 4096) blocks = 4096;
    const int64_t step = blocks * 256;
    auto k = whole ? k_dropout<T, Q, true> : k_dropout<T, Q, false>;
    k<<<(unsigned)blocks, 256, 0, as_stream(stream)>>>((const T *)x, ldx, (T *)y, N, planes, items, step / items,
                                                       (int)(step % items), drop_threshold(p), (float)(1.0 / (1.0 - p)), rng);
    SCN_CHECK_LAUNCH();
    return 0;
  });
}

int scn_rng_take(int64_t *state, int64_t *used, void *stream) {
  SCN_REQUIRE(state && used, "rng: pointers");
  k_rng_take<<<1, 1, 0, as_stream(stream)>>>(state, used);
  SCN_CHECK_LAUNCH();
  return 0;
}

int scn_linear_forward(const void *x, int64_t ldx, const void *weight, const void *bias, const void *residual, int64_t ld_res,
                       void *y, void *factor, int64_t N, int n_in, int n_out, int act, double leakiness, double p,
                       const int64_t *rng, int dtype, void *stream) {
  if (int e = lin_check(N, n_in, n_out, dtype)) return e;
  SCN_REQUIRE(act == SCN_ACT_LEAKY || act == SCN_ACT_SILU || act == SCN_ACT_GELU, "linear: activation");
  SCN_REQUIRE(p >= 0 && p < 1 && (p == 0 || rng), "linear: 0 <= p < 1, with random words if it is not 0");
  if (N == 0) return 0;
  SCN_REQUIRE(x && weight && y && ldx >= n_in && (!residual || ld_res >= n_out), "linear: pointers");
  LinearArgs a = {};
  a.in = x;
  a.ld_in = ldx;
  a.weight = weight;
  a.bias = bias;
  a.residual = residual;
  a.ld_res = ld_res;
  a.out = y;
  a.factor = factor;
  a.rng = rng;
  a.N = N;
  a.K = n_in;
  a.M = n_out;
  a.threshold = drop_threshold(p);
  a.leak = (float)leakiness;
  a.keep_scale = (float)(1.0 / (1.0 - p));
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (act == SCN_ACT_SILU) return linear_by_width<T, 0, SCN_ACT_SILU>(a, as_stream(stream));
    if (act == SCN_ACT_GELU) return linear_by_width<T, 0, SCN_ACT_GELU>(a, as_stream(stream));
    return linear_by_width<T, 0, SCN_ACT_LEAKY>(a, as_stream(stream));
  });
}

int scn_linear_dinput(const void *d_y, int64_t ld_dy, const void *factor, const void *weight, void *d_x, int64_t N, int n_in,
                      int n_out, int dtype, void *stream) {
  if (int e = lin_check(N, n_in, n_out, dtype)) return e;
  if (N == 0) return 0;
  SCN_REQUIRE(d_y && weight && d_x && ld_dy >= n_out, "linear: pointers");
  LinearArgs a = {};
  a.in = d_y;
  a.ld_in = ld_dy;
  a.scale = factor;
  a.weight = weight;
  a.out = d_x;
  a.N = N;
  a.K = n_out;
  a.M = n_in;
  return by_type(dtype, [&](auto t) { return linear_by_width<decltype(t), 1, SCN_ACT_LEAKY>(a, as_stream(stream)); });
}

size_t scn_linear_dweight_temp_bytes(int64_t N, int n_in, int n_out) {
  return sizeof(float) * (size_t)dw_slices(N, n_in, n_out) * ((size_t)n_in * n_out + n_out);
}

int scn_linear_dweight(const void *x, int64_t ldx, const void *d_y, int64_t ld_dy, const void *factor, void *d_weight, void *d_bias,
                       int64_t N, int n_in, int n_out, int dtype, void *temp, size_t temp_bytes, void *stream) {
  if (int e = lin_check(N, n_in, n_out, dtype)) return e;
  SCN_REQUIRE(d_weight && (N == 0 || (x && d_y)) && ldx >= n_in && ld_dy >= n_out, "linear: pointers");
  SCN_REQUIRE(temp && temp_bytes >= scn_linear_dweight_temp_bytes(N, n_in, n_out), "linear: workspace");
  DwArgs a = {};
  a.x = x;
  a.dy = d_y;
  a.scale = factor;
  a.ldx = ldx;
  a.ld_dy = ld_dy;
  a.N = N;
  a.Ci = n_in;
  a.Co = n_out;
  a.tiles_i = (n_in + 63) / 64;
  a.tiles_o = (n_out + 63) / 64;
  a.slices = dw_slices(N, n_in, n_out);
  a.slice_rows = ((N + a.slices - 1) / a.slices + 127) / 128 * 128;
  a.slab = (float *)temp;
  a.want_bias = d_bias != nullptr;
  const int64_t nw = (int64_t)n_in * n_out;
  const int nb = d_bias ? n_out : 0;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    k_linear_dw<T><<<(unsigned)(a.slices * a.tiles_i * a.tiles_o), 256, 0, as_stream(stream)>>>(a);
    SCN_CHECK_LAUNCH();
    k_linear_dw_join<T><<<(unsigned)((nw + nb + 255) / 256), 256, 0, as_stream(stream)>>>(a.slab, a.slices, nw, nb, (T *)d_weight,
                                                                                         (T *)d_bias);
    SCN_CHECK_LAUNCH();
    return 0;
  });
}

}  // extern "C"

// 1x1 convolution with its epilogue, y = residual + drop(act(x W + b)), its gradients, and dropout alone (gfx950).
//
//   backward:  f = act'(x W + b), 0 where dropped, left by the forward pass;  dz = dy f / (1 - p), 0 where f is 0;
//              dx = dz W^T;  dW = x^T dz;  db = column sums of dz
//
// Sites are many (up to 600k) and planes few (16 to 512), so the products are HBM bound but for the widest: 2 n_in n_out flops for
// n_in + n_out values, 16 to 128 flops a byte where fp32 MFMA balances at 28 and bf16 at 200.  Everything that belongs to a row is
// done while it is in registers.
//
// Products: v_mfma 16x16, the WEIGHT as the A operand and the sites as B: the four results of a lane are then four consecutive
// planes of one site.  The order of the reduction is free as long as both operands agree: a lane's 16 bytes of a row, loaded straight
// from global memory, ARE its B operands (one 16x16x32 of 16-bit types, four 16x16x4 of fp32).  The weights are laid out in LDS in the
// order of the A operands.
#include "scn_pointwise.h"

namespace scn {

// n of the V elements at p, zeros behind them (16-bit ones packed as they come, or each would keep a register of its own)
template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_some(const T *p, int n) {
  if (n >= V) return load_pack<T, V>(p);
  Pack<T, V> r;
  if constexpr (sizeof(T) == 2) {
    const uint16_t *q = (const uint16_t *)p;
    uint32_t w[V / 2];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      w[j] = 2 * j < n ? q[2 * j] : 0u;
      if (2 * j + 1 < n) w[j] |= (uint32_t)q[2 * j + 1] << 16;
      asm("" : "+v"(w[j]));
    }
    __builtin_memcpy(&r, w, sizeof(r));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = j < n ? p[j] : (T)0.f;
  }
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

// ------------------------------------------------------------------- dropout ---
// Every element read and written once; the mask is made of the counter.  A thread keeps its planes -- Q quads -- and walks the
// sites, `rows` of a step at a time: the products of the counter that belong to the planes are made once.  Four rows are requested
// before the first is used.  HBM bound: 601,674 x 128 bf16 take 65 us = 4.7 TB/s, a copy of as many bytes 58.
template <class T, int Q, bool WHOLE>
__global__ void __launch_bounds__(256)
    k_dropout(const T *x, int64_t ldx, T *y, int64_t N, int C, int items, int rows, uint32_t threshold, float scale, const int64_t *rng) {
  const int item = rows > 1 ? (int)threadIdx.x % items : (int)(blockIdx.y * 256 + threadIdx.x);
  const int sub = rows > 1 ? (int)threadIdx.x / items : 0;
  if (item >= items || sub >= rows) return;
  const RngKey key = rng_key(rng);
  const int c = item * 4 * Q, n = WHOLE ? 4 * Q : min(4 * Q, C - c);
  PhiloxPlane plane[Q];
#pragma unroll
  for (int u = 0; u < Q; ++u) plane[u] = philox_plane(key, (uint32_t)(item * Q + u));
  const int64_t step = (int64_t)gridDim.x * rows;
  auto masked = [&](Pack<T, 4 * Q> &v, int64_t row) __attribute__((always_inline)) {
    const PhiloxSite site = philox_site(key, (uint32_t)row);
#pragma unroll
    for (int u = 0; u < Q; ++u) {
      const Words w = philox(key, plane[u], site);
#pragma unroll
      for (int j = 0; j < 4; ++j) v.v[4 * u + j] = w.w[j] >= threshold ? (T)((float)v.v[4 * u + j] * scale) : (T)0.f;
    }
  };
  int64_t row = (int64_t)blockIdx.x * rows + sub;
  if (n == 4 * Q)
    for (; row + 3 * step < N; row += 4 * step) {
      Pack<T, 4 * Q> v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = load_pack<T, 4 * Q>(x + (row + i * step) * ldx + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        masked(v[i], row + i * step);
        store_pack<T, 4 * Q>(y + (row + i * step) * C + c, v[i]);
      }
    }
  for (; row < N; row += step) {
    Pack<T, 4 * Q> v = load_some<T, 4 * Q>(x + row * ldx + c, n);
    masked(v, row);
    store_some<T, 4 * Q>(y + row * C + c, v, n);
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

// What the backward pass needs of activation and mask, one value per output: the slope, 0 for a dropped element.  (dy slope is what is
// multiplied with; 1 / (1 - p) is applied to the sums.)  dz = dy slope is the matrix units' operand, 16-bit features' in two parts (split,
// below); a slope's own rounding is all that it loses, so slopes are kept finer than the features:
//   FACTOR_FLOAT  fp32 features: fp32
//   FACTOR_WIDE   bf16 features: sign, 6 bits of exponent, 9 of mantissa: 2^-10 of a slope down to 2^-60 (slopes of saturated units are
//                 small, and bf16 holds what they make of dy), 2^-60 below
//   FACTOR_SHORT  fp16 features: the smooth activations' slopes are below 1.13, and above -0.13, where those of saturated units are:
//                 positive ones 3 bits of exponent and 12 of mantissa (2^-13 of a slope down to 2^-6, 2^-19 below: next to the slope's
//                 zero), negative ones 5 and 10 (2^-11 down to 2^-33, 2^-44 below); 0x7fff: NaN
//   FACTOR_SIGN   leaky ReLU of 16-bit features, whose slope may be any number: 2: 1, 1: leak, 0: dropped
enum { FACTOR_NONE, FACTOR_FLOAT, FACTOR_WIDE, FACTOR_SHORT, FACTOR_SIGN };
template <class T> struct FactorOf { using type = int16_t; };
template <> struct FactorOf<float> { using type = float; };

// (the low bits of the exponent of a fp32 2^126 times larger, which are 192 more -- the largest are NaN's -- and the upper of its mantissa)
__device__ __forceinline__ int16_t wide_float(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, fabsf(v) * 0x1p126f), sign = __builtin_bit_cast(uint32_t, v) >> 16 & 0x8000u;
  return (int16_t)(__builtin_elementwise_sub_sat(b, (192u << 23) - 0x2000u) >> 14 | sign);
}
__device__ __forceinline__ float wide_float_value(int16_t q) {
  return __builtin_bit_cast(float, ((uint32_t)(int)q << 14 & 0x9fffc000u) | 0x60000000u) * 0x1p-126f;
}
// (the low bits of the exponent of a fp32 2^120 or 2^93 times smaller -- its subnormal numbers are the format's -- and the upper of its
// mantissa)
__device__ __forceinline__ int16_t short_float(float v) {
  const bool negative = v < 0;
  const uint32_t b = __builtin_bit_cast(uint32_t, fabsf(v) * (negative ? 0x1p-93f : 0x1p-120f));
  const int shift = negative ? 13 : 11;
  return (int16_t)(min((b + (1u << shift >> 1)) >> shift, 0x7fffu) | (negative ? 0x8000u : 0u));  // (only NaN, not below 0, reaches 0x7fff)
}
__device__ __forceinline__ float short_float_value(int16_t q) {
  const bool negative = q < 0;
  const float v = __builtin_bit_cast(float, ((uint32_t)q & 0x7fffu) << (negative ? 13 : 11)) * (negative ? -0x1p93f : 0x1p120f);
  return q == 0x7fff ? __builtin_nanf("") : v;
}

// dy times the slope; 0 where that is 0, whatever dy is there: infinity and NaN in dropped places stay there
template <int FACTOR, class Q>
__device__ __forceinline__ float times_factor(float dy, Q q, float leak) {
  if constexpr (FACTOR == FACTOR_FLOAT) return q == 0 ? 0.f : dy * (float)q;
  if constexpr (FACTOR == FACTOR_WIDE) return q == 0 ? 0.f : dy * wide_float_value((int16_t)q);
  float slope = q == 2 ? 1.f : q == 1 ? leak : 0.f;
  if constexpr (FACTOR == FACTOR_SHORT) slope = short_float_value((int16_t)q);
  return slope == 0 ? 0.f : dy * slope;
}

// z of 16-bit features as two operands, z rounded and what that lost, whose products are added one behind the other: what is lost is the
// square of a rounding (fp16: and what lies below its subnormal numbers).  One operand alone doubles the variance of the gradients' own
// rounding (bf16 dx and dW off by 2.4e-3 instead of 1.7e-3, relative), and the matrix pipe waits for memory either way: 177,001 x 128 to
// 512, bf16, GELU, one call behind the other, dx 94 us with one and with two, dW 108 and 109.  (Where rounding would give infinity: the
// largest number, and the rest beside it; infinity and NaN are in the rest.)
template <class T>
__device__ __forceinline__ void split(float z, T &rounded, T &rest) {
  constexpr float most = std::is_same<T, __bf16>::value ? 0x1.fep127f : 65504.f;
  rounded = (T)__builtin_amdgcn_fmed3f(z, -most, most);
  rest = (T)(z - (float)rounded);
}

struct LinearArgs {
  const void *in, *factor_in;  // rows [N, K] at ld_in elements; MODE 1: times the factors [N, K]
  int64_t ld_in;
  const void *weight;  // MODE 0: [K, M], MODE 1 and `transposed`: [M, K]
  int transposed;
  const void *bias, *residual;
  int64_t ld_res;
  void *out, *factor;
  const int64_t *rng;
  int64_t N;
  int K, M;
  int groups, chunk_groups;  // k-groups in all, and per pass through LDS
  int col_blocks, row_blocks;
  uint32_t threshold;
  float leak, up;
};

constexpr int ACT_NONE = 3;  // SCN_ACT_LEAKY with slope 1

// one output's activation and mask, and its factor
template <class T, int ACT, bool DROP>
__device__ __forceinline__ float activated(float z, bool keep, const LinearArgs &a, typename FactorOf<T>::type &factor) {
  float value = z, slope = 1.f;
  if constexpr (ACT != ACT_NONE) act_value_slope<ACT, T>(z, a.leak, value, slope);
  if constexpr (DROP) value = keep ? value * a.up : 0.f;
  if constexpr (sizeof(T) == 4) factor = slope;
  else if constexpr (ACT == ACT_NONE) factor = 2;
  else if constexpr (ACT == SCN_ACT_LEAKY) factor = z > 0 ? 2 : 1;
  else if constexpr (std::is_same<T, __bf16>::value) factor = wide_float(slope);
  else factor = short_float(slope);
  if (DROP && !keep) factor = 0;
  return value;
}

// waves of a workgroup: all that the registers of a CU hold if the weights stay in LDS
constexpr int lin_waves(int nt, bool stay) { return !stay ? 4 : nt == 8 ? 12 : 16; }

constexpr int lin_piece(int nt) { return nt < 4 ? 16 * nt : 64; }  // planes of a tile that go through LDS together
// ... as the sums they are, or, where nothing but a factor is missing, as the 16-bit values that will be stored: half the room, so the
// weights of 512 planes stay (dx of 177,001 x 128 to 512, bf16: 103 to 92 us)
constexpr bool lin_packed(int mode, int size) { return mode == 1 && size == 2; }
constexpr int lin_piece_bytes(int nt, bool packed) { return packed ? 16 * (lin_piece(nt) + 8) * 2 : 16 * (lin_piece(nt) + 4) * 4; }

// MODE 0: forward with the epilogue, X its activation.  MODE 1: dx, X how the factors are stored.
// A workgroup holds the weights of NT x 16 output planes in LDS -- all of K, once, if they fit (STAY): then it has a CU to itself and
// its waves take 32-row tiles without a barrier -- else `chunk_groups` at a time, and its waves keep together.  Tiles are taken from a
// counter in LDS: the older of the waves on a SIMD come first at its matrix pipe and take 15 us a tile where the youngest take 37
// (200,000 x 128 to 128, fp32), so that equal shares would end at 50 to 85 us.
// Beside fp32 MFMAs a vector instruction costs 8 or more of the matrix pipe's cycles, and the epilogue alone fills half the time of
// a 16-bit layer: addresses are a scalar base and one 32-bit offset a lane for all tiles, the bias is what the accumulators start
// from, and the epilogue is compiled for each activation, with and without dropout and factors.
// Measured, medians with inputs that are not cached: 601,674 x 64 to 20, fp32, 45 us = 4.5 TB/s; 177,001 x 64 to 128, fp32, GELU, dropout,
// residual and factors, 68 us = 4.7 TB/s (forward), 45 us = 5.1 TB/s (dx); 177,001 x 128 to 512, GELU, dropout and factors, bf16 140 us =
// 2.9 TB/s (forward: some 31 vector instructions an output), 109 us = 3.7 TB/s (dx), fp16 148 and 111 us; without activation and dropout,
// bf16, 59 us = 3.8 TB/s and 62 us = 3.6 TB/s; fp32 that is not bound by memory: 200,000 x 128 to 128 96 us = 68 TFLOP/s, 100,000 x 512 to
// 512 538 us = 97 TFLOP/s.
template <class T, int NT, int MODE, int X, bool STAY>
__global__ void __launch_bounds__(64 * lin_waves(NT, STAY), NT == 8 || !STAY ? 3 : 4) k_linear(LinearArgs a) {
  constexpr int WAVES = lin_waves(NT, STAY), THREADS = 64 * WAVES;
  constexpr int V = Elem<T>::V, KG = 4 * V;
  constexpr bool PACKED = lin_packed(MODE, sizeof(T));
  constexpr int PC = lin_piece(NT), PITCH = PACKED ? PC + 8 : PC + 4, LPR = PC / V, RPI = 64 / LPR;  // planes, lanes a row, rows an instruction of a piece
  constexpr bool FACTORS = MODE == 1 && X != FACTOR_NONE, SPLIT = FACTORS && sizeof(T) == 2;
  using F = typename Frag<T>::type;
  using Q = typename FactorOf<T>::type;
  extern __shared__ char smem[];
  F *wl = (F *)smem;  // [k-group of the chunk][tile][lane]
  float *bl = (float *)(wl + (size_t)NT * a.chunk_groups * 64);
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lq = lane >> 4;
  float *sw = bl + NT * 16 + wave * (lin_piece_bytes(NT, PACKED) / 4);
  int *next = (int *)(bl + NT * 16 + WAVES * (lin_piece_bytes(NT, PACKED) / 4));  // the next tile of this workgroup
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
  const T *in = (const T *)a.in, *wt = (const T *)a.weight;
  const Q *fi = (const Q *)a.factor_in;
  if (threadIdx.x < NT * 16) {
    const int m = m0 + threadIdx.x;
    bl[threadIdx.x] = MODE == 0 && a.bias && m < a.M ? (float)((const T *)a.bias)[m] : 0.f;
  }
  RngKey key = {};
  if (MODE == 0 && a.threshold) key = rng_key(a.rng);
  const int full = a.K / KG;  // k-groups that lie inside the rows
  const int tiles = (int)(STAY ? (a.N + 31) / 32 : (a.N + 127) / 128 * 4);
  if (threadIdx.x == 0) *next = WAVES;

  // weights of k-groups g0 .. g0 + ng in the order of the A operands, several loads a thread in flight
  auto stage = [&](int g0, int ng) __attribute__((always_inline)) {
    constexpr int B = 4;
    if (MODE == 1 || NT == 8 || !STAY || a.transposed) {  // [M, K]: a lane's V elements lie together
      for (int e0 = threadIdx.x; e0 < NT * ng * 64; e0 += THREADS * B) {
        Pack<T, V> v[B];
#pragma unroll
        for (int i = 0; i < B; ++i) {
          const int e = e0 + THREADS * i, l = e & 63, t = (e >> 6) % NT, g = (e >> 6) / NT;
          const int m = m0 + 16 * t + (l & 15), k = (g0 + g) * KG + (l >> 4) * V;
          v[i] = load_some<T, V>(wt + (int64_t)m * a.K + k, e < NT * ng * 64 && m < a.M ? a.K - k : 0);
        }
#pragma unroll
        for (int i = 0; i < B; ++i)
          if (e0 + THREADS * i < NT * ng * 64) __builtin_memcpy(&wl[e0 + THREADS * i], &v[i], 16);
      }
    } else {  // [K, M]: V planes of one k, spread over V lanes' places
      constexpr int MV = NT * 16 / V;  // vectors a row
      const int n = MV * ng * KG;
      T *lds = (T *)wl;
      for (int e = threadIdx.x; e < n; e += THREADS) {
        const int m = e % MV * V, k = e / MV;
        const Pack<T, V> v = load_some<T, V>(wt + (int64_t)(g0 * KG + k) * a.M + m0 + m, g0 * KG + k < a.K ? a.M - m0 - m : 0);
#pragma unroll
        for (int j = 0; j < V; ++j) lds[(((k / KG * NT + (m + j) / 16) * 64 + k % KG / V * 16 + (m + j) % 16) * V) + k % V] = v.v[j];
      }
    }
  };
  if (STAY) stage(0, a.groups);
  __syncthreads();

  // a piece of results: 16 sites x PC planes from LDS, this lane's V planes of every RPI-th of them.  WHOLE: all of them are there, and
  // everything is requested before any of it is used
  auto finish = [&](auto whole, auto drop, auto fac, int64_t row0, int pc) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole)::value, DROP = decltype(drop)::value, FAC = decltype(fac)::value;
    constexpr int IT = 16 / RPI;
    const int r0 = lane / LPR, c = lane % LPR * V, m = m0 + pc + c, left = WHOLE ? V : a.M - m;
    const int rows = WHOLE ? 16 : (int)min((int64_t)16, a.N - row0);
    if (left <= 0) return;
    // (scalar bases, 32-bit offsets)
    T *out = (T *)a.out + row0 * a.M + m0 + pc;
    Q *fo = (Q *)a.factor + row0 * a.M + m0 + pc;
    const T *res = (const T *)a.residual + row0 * a.ld_res + m0 + pc;
    const unsigned o0 = (unsigned)(r0 * a.M + c), res0 = (unsigned)(r0 * (int)a.ld_res + c);
    Pack<T, V> rv[IT];
    if (MODE == 0 && a.residual)
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const T *p = res + (int64_t)(i * RPI) * a.ld_res + res0;
        rv[i] = WHOLE ? load_pack<T, V>(p) : load_some<T, V>(p, i * RPI + r0 < rows ? left : 0);
      }
    if constexpr (PACKED) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const Pack<T, V> y = load_pack<T, V>((const T *)sw + (i * RPI + r0) * PITCH + c);
        T *o = out + (int64_t)(i * RPI) * a.M + o0;
        if constexpr (WHOLE) store_pack<T, V>(o, y);
        else if (i * RPI + r0 < rows) store_some<T, V>(o, y, left);
      }
      return;
    }
    float z[IT][V];
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const floatx4 v = *(const floatx4 *)(sw + (i * RPI + r0) * PITCH + c + j);
        z[i][j] = v[0], z[i][j + 1] = v[1], z[i][j + 2] = v[2], z[i][j + 3] = v[3];
      }
    PhiloxPlane plane[V / 4];
    if constexpr (DROP)
#pragma unroll
      for (int q = 0; q < V / 4; ++q) plane[q] = philox_plane(key, (uint32_t)((m >> 2) + q));
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      Pack<T, V> y;
      Pack<Q, V> f;
      if constexpr (MODE == 0) {
        PhiloxSite site;
        if constexpr (DROP) site = philox_site(key, (uint32_t)(row0 + i * RPI) + r0);
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
          Words w;
          if constexpr (DROP) w = philox(key, plane[q], site);
#pragma unroll
          for (int j = 4 * q; j < 4 * q + 4; ++j) z[i][j] = activated<T, X, DROP>(z[i][j], !DROP || w.w[j & 3] >= a.threshold, a, f.v[j]);
        }
        if (a.residual)
#pragma unroll
          for (int j = 0; j < V; ++j) z[i][j] += (float)rv[i].v[j];
      }
#pragma unroll
      for (int j = 0; j < V; ++j) y.v[j] = (T)(MODE == 1 ? z[i][j] * a.up : z[i][j]);
      T *o = out + (int64_t)(i * RPI) * a.M + o0;
      Q *fp = fo + (int64_t)(i * RPI) * a.M + o0;
      if constexpr (WHOLE) {
        if constexpr (FAC) store_pack<Q, V>(fp, f);
        store_pack<T, V>(o, y);
      } else if (i * RPI + r0 < rows) {
        if constexpr (FAC) store_some<Q, V>(fp, f, left);
        store_some<T, V>(o, y, left);
      }
      __builtin_amdgcn_sched_barrier(0);  // (one row's epilogue at a time)
    }
  };
  auto finish_as = [&](auto whole, int64_t row0, int pc) __attribute__((always_inline)) {
    if constexpr (MODE == 1) finish(whole, std::false_type(), std::false_type(), row0, pc);
    else if (a.threshold)
      a.factor ? finish(whole, std::true_type(), std::true_type(), row0, pc) : finish(whole, std::true_type(), std::false_type(), row0, pc);
    else
      a.factor ? finish(whole, std::false_type(), std::true_type(), row0, pc) : finish(whole, std::false_type(), std::false_type(), row0, pc);
  };

  for (int i = wave;;) {
    const int tile = STAY ? i * a.row_blocks + rb : rb * 4 + i;
    if (tile >= tiles) break;
    const int64_t row0 = (int64_t)tile * 32;
    // (rows behind the last are read as the last and not written; of tiles behind the last, too)
    const int64_t base = min(row0, a.N - 1);
    const int last = (int)min((int64_t)31, a.N - 1 - base);
    const T *p = in + base * a.ld_in;
    const Q *pf = fi + base * a.K;
    unsigned op[2], of[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = min(li + 16 * u, last);
      op[u] = (unsigned)(r * (int)a.ld_in + lq * V);
      of[u] = (unsigned)(r * a.K + lq * V);
    }
    floatx4 acc[2][NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[0][t] = acc[1][t] = *(const floatx4 *)(bl + 16 * t + 4 * lq);

    // k-groups: the rows of G of them are requested together (a row's two halves of a cache line one behind the other), then multiplied
    auto request = [&](auto whole, auto &v, auto &f, int g) __attribute__((always_inline)) {
      constexpr bool WHOLE = decltype(whole)::value;
      constexpr int G = sizeof(v) / sizeof(v[0]);
      const T *pk = p + g * KG;
      const Q *pfk = pf + g * KG;
      const int left = a.K - g * KG - lq * V;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < G; ++i) {
          v[i][u] = WHOLE ? load_pack<T, V>(pk + i * KG + op[u]) : load_some<T, V>(pk + i * KG + op[u], left - i * KG);
          if constexpr (FACTORS) f[i][u] = WHOLE ? load_pack<Q, V>(pfk + i * KG + of[u]) : load_some<Q, V>(pfk + i * KG + of[u], left - i * KG);
        }
    };
    auto multiply = [&](auto &v, auto &f, const F *wg) __attribute__((always_inline)) {
      constexpr int G = sizeof(v) / sizeof(v[0]);
#pragma unroll
      for (int i = 0; i < G; ++i) {
        F b[2], rest[2], w[NT];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if constexpr (FACTORS) {
            Pack<T, V> r;
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float z = times_factor<X>((float)v[i][u].v[j], f[i][u].v[j], a.leak);
              if constexpr (SPLIT) split(z, v[i][u].v[j], r.v[j]);
              else v[i][u].v[j] = (T)z;
            }
            if constexpr (SPLIT) __builtin_memcpy(&rest[u], &r, 16);
          }
          __builtin_memcpy(&b[u], &v[i][u], 16);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) w[t] = wg[(i * NT + t) * 64];
        if constexpr (sizeof(T) == 4) {  // (no product waits for the one in front of it)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int u = 0; u < 2; ++u) acc[u][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[t][j], b[u][j], acc[u][t], 0, 0, 0);
        } else {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              acc[u][t] = mma(w[t], b[u], acc[u][t]);
              if constexpr (SPLIT) acc[u][t] = mma(w[t], rest[u], acc[u][t]);
            }
        }
        if (NT == 8 || SPLIT) __builtin_amdgcn_sched_barrier(0);  // (one k-group's operands in registers at a time)
      }
    };
    auto batch = [&](auto count, auto whole, int g, const F *wg) __attribute__((always_inline)) {
      Pack<T, V> v[decltype(count)::value][2];
      Pack<Q, V> f[decltype(count)::value][2];
      request(whole, v, f, g);
      multiply(v, f, wg);
    };
    for (int g0 = 0; g0 < a.groups; g0 += a.chunk_groups) {
      const int ng = min(a.chunk_groups, a.groups - g0), nf = min(ng, full - g0);
      const F *wg = wl + lane;
      int g = 0;
      if constexpr (!STAY) {
        __syncthreads();
        stage(g0, ng);
        __syncthreads();
      }
      if (STAY && NT < 8 && !FACTORS)
        for (; g + 4 <= nf; g += 4, wg += 4 * NT * 64) batch(std::integral_constant<int, 4>(), std::true_type(), g0 + g, wg);
      for (; g + 2 <= nf; g += 2, wg += 2 * NT * 64) batch(std::integral_constant<int, 2>(), std::true_type(), g0 + g, wg);
      for (; g < nf; ++g, wg += NT * 64) batch(std::integral_constant<int, 1>(), std::true_type(), g0 + g, wg);
      if (g < ng) batch(std::integral_constant<int, 1>(), std::false_type(), g0 + g, wg);
    }
    // Results go through LDS, 16 sites x PC planes of a wave at a time: a lane then has 16 bytes of a row and its neighbours the bytes
    // beside them, 4 rows x 256 bytes (fp32) or 8 rows x 128 an instruction.  Stored from where the product leaves them they are
    // 16 pieces of 64 bytes, half a cache line each: 226 MB of the wide layer took 149 us that way, of 43 at the copy rate.
#pragma unroll 1
    for (int piece = 0; piece < 2 * NT * 16 / PC; ++piece) {
      constexpr int PPU = NT * 16 / PC;  // pieces of 16 rows
#pragma unroll
      for (int k = 0; k < 2 * PPU; ++k)
        if (k == piece) {
#pragma unroll
          for (int t = 0; t < PC / 16; ++t) {
            const floatx4 v = acc[k / PPU][k % PPU * (PC / 16) + t];
            if constexpr (PACKED)
              store_pack<T, 4>((T *)sw + li * PITCH + 16 * t + 4 * lq, {{(T)(v[0] * a.up), (T)(v[1] * a.up), (T)(v[2] * a.up), (T)(v[3] * a.up)}});
            else *(floatx4 *)(sw + li * PITCH + 16 * t + 4 * lq) = v;
          }
        }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const int64_t r = row0 + piece / PPU * 16;
      const int pc = piece % PPU * PC;
      if (r + 16 <= a.N && m0 + pc + PC <= a.M) finish_as(std::true_type(), r, pc);
      else finish_as(std::false_type(), r, pc);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    if constexpr (!STAY) break;
    if (lane == 0) i = atomicAdd(next, 1);
    i = __builtin_amdgcn_readfirstlane(i);
  }
}

// weight [K, M] -> [M, K], 32 x 32 at a time
template <class T>
__global__ void __launch_bounds__(256) k_linear_transpose(const T *w, T *out, int K, int M) {
  __shared__ T tile[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, k0 = blockIdx.y * 32, m0 = blockIdx.x * 32;
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    if (k0 + y + i < K && m0 + x < M) tile[y + i][x] = w[(int64_t)(k0 + y + i) * M + m0 + x];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    if (m0 + y + i < M && k0 + x < K) out[(int64_t)(m0 + y + i) * K + k0 + x] = tile[x][y + i];
}

// Up to R rows (a serving loop's single sites): bound by one trip to memory for the weights, which the tiles above would make with a
// few workgroups in many steps.  A workgroup has 16 output planes; its threads share out the reduction, 16 bytes of a weight row
// each, and join in the wave, then through LDS: another order of additions than that of the tiles, so a row's last bits may differ.
template <class T, int R, int ACT>
__global__ void __launch_bounds__(1024) k_linear_few(LinearArgs a) {
  constexpr int V = Elem<T>::V, LC = 16 / V, PHASES = 1024 / LC;
  __shared__ float red[16][R][16];
  const int m0 = blockIdx.x * 16, cl = threadIdx.x % LC * V, m = m0 + cl;
  const T *x = (const T *)a.in, *wt = (const T *)a.weight;
  float acc[R][V];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) acc[r][j] = 0.f;
  for (int k = threadIdx.x / LC; k < a.K; k += PHASES) {
    const Pack<T, V> w = load_some<T, V>(wt + (int64_t)k * a.M + m, a.M - m);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float xv = (float)x[min((int64_t)r, a.N - 1) * a.ld_in + k];
#pragma unroll
      for (int j = 0; j < V; ++j) acc[r][j] = fmaf(xv, (float)w.v[j], acc[r][j]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < V; ++j) {
#pragma unroll
      for (int o = LC; o < 64; o <<= 1) acc[r][j] += __shfl_xor(acc[r][j], o);
    }
  if (lane_id() < LC)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < V; ++j) red[threadIdx.x >> 6][r][cl + j] = acc[r][j];
  __syncthreads();
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15, mo = m0 + c;
  if (row >= R || row >= a.N || mo >= a.M) return;
  float z = 0.f;
#pragma unroll
  for (int w = 0; w < 16; ++w) z += red[w][row][c];
  z += a.bias ? (float)((const T *)a.bias)[mo] : 0.f;
  bool keep = true;
  if (a.threshold) {
    const RngKey key = rng_key(a.rng);
    const Words w = philox(key, philox_plane(key, (uint32_t)mo >> 2), philox_site(key, (uint32_t)row));
    keep = ((mo & 2) ? (mo & 1) ? w.w[3] : w.w[2] : (mo & 1) ? w.w[1] : w.w[0]) >= a.threshold;
  }
  typename FactorOf<T>::type f;
  float y = activated<T, ACT, true>(z, keep, a, f);
  if (a.residual) y += (float)((const T *)a.residual)[row * a.ld_res + mo];
  ((T *)a.out)[(int64_t)row * a.M + mo] = (T)y;
  if (a.factor) ((typename FactorOf<T>::type *)a.factor)[(int64_t)row * a.M + mo] = f;
}

// ------------------------------------------------------------------- dweight ---
// dW = x^T dz: the reduction runs over the rows, both operands are walked along their planes.  A wave's tile is 64 TI x 64: a lane
// loads 4 consecutive planes of a row, which are its elements of four A (B) tiles with the planes interleaved by four -- fp32
// needs nothing else; of 16-bit types eight rows are loaded and transposed in registers.  No LDS in the loop.  Planes behind the last
// are read as what follows in memory: they reach only results that are not stored.  Steps whose reads would leave a tensor are
// loaded element by element (the last rows of the last slice).
// Workgroup (slice, tile): four waves take the slice's row steps in turn, join through LDS and write one slab; slabs are added by
// k_linear_dw_join in slice order.
// HBM bound; medians with inputs that are not cached, without the join's 4 to 8 us: 177,001 x 64 to 128, fp32, with factors 50 us = 4.5
// TB/s; 128 to 512, bf16, 105 us = 3.9 TB/s (without factors 62 us = 3.6 TB/s).  Few sites: a step's latency three times over and the
// waves' join, 16 us for 50,001 x 35 to 77, fp16, and 4 for the slabs.
struct DwArgs {
  const void *x, *dy, *factor;
  int64_t ldx, ld_dy, N;
  int Ci, Co, tiles_i, tiles_o, slices;
  int64_t slice_rows;
  float *slab;      // [slices][Ci][Co], then [slices][Co]
  int want_bias;
  float leak, up;
};

// rows r for which the 64 planes from c0 of rows up to r lie in the memory of a [N, C] tensor with rows at ld
__device__ __forceinline__ int64_t rows_inside(int64_t N, int64_t ld, int C, int c_end) {
  const int64_t room = (N - 1) * ld + C - c_end;
  return room < 0 ? 0 : min(N, room / ld + 1);
}

template <class T, int TI, int FACTOR>
__global__ void __launch_bounds__(256, 2) k_linear_dw(DwArgs a) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int RE = F32 ? 4 : 8;  // rows of a lane in one step
  constexpr int ROWS = 4 * RE;
  using F = typename Frag<T>::type;
  using Q = typename FactorOf<T>::type;
  __shared__ float red[TI * 64 * 64 + 64];
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lq = lane >> 4;
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
  const int ci0 = tile / a.tiles_o * 64 * TI, co0 = tile % a.tiles_o * 64;
  const bool bias = a.want_bias && ci0 == 0;
  const int64_t r0 = slice * a.slice_rows, r1 = min(r0 + a.slice_rows, a.N);
  // a step's rows from scalar addresses, a lane's part of them from 32-bit offsets
  const T *px = (const T *)a.x + ci0, *pd = (const T *)a.dy + co0;
  const Q *pf = (const Q *)a.factor + co0;
  int64_t inside = min(rows_inside(a.N, a.ldx, a.Ci, ci0 + 64 * TI), rows_inside(a.N, a.ld_dy, a.Co, co0 + 64));
  if (FACTOR != FACTOR_NONE) inside = min(inside, rows_inside(a.N, a.Co, a.Co, co0 + 64));
  inside = min(inside, r1);
  floatx4 acc[4 * TI][4], sums = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4 * TI; ++i) acc[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
  auto step = [&](auto whole, int64_t r) __attribute__((always_inline)) {
    constexpr bool WHOLE = decltype(whole)::value;
    constexpr int ES = F32 ? 4 : 1;  // rows from one of a lane's to its next
    Pack<T, 4> vx[TI][RE], vd[RE];
    Pack<Q, 4> vf[RE];
    const T *p = px + r * a.ldx, *d = pd + r * a.ld_dy;
    const Q *q = pf + r * a.Co;
    int l = lane;
    if (!WHOLE) asm volatile("" : "+v"(l));  // (nothing of these steps is kept in registers through the loop of the whole ones)
    const int lr = F32 ? l >> 4 : (l >> 4) * RE;  // a lane's first row (fp32: a load of four whole rows; 16-bit: a lane's eight rows)
    const int lc = 4 * (l & 15), ci = ci0 + lc, no = a.Co - co0 - lc;
    const unsigned ox = (unsigned)(lr * (int)a.ldx + lc), od = (unsigned)(lr * (int)a.ld_dy + lc), of = (unsigned)(lr * a.Co + lc);
#pragma unroll
    for (int e = 0; e < RE; ++e) {
      const bool in = r + ES * e + lr < r1;
#pragma unroll
      for (int t = 0; t < TI; ++t)
        vx[t][e] = WHOLE ? load_pack<T, 4>(p + 64 * t + ox) : load_some<T, 4>(p + 64 * t + ox, in ? a.Ci - ci - 64 * t : 0);
      vd[e] = WHOLE ? load_pack<T, 4>(d + od) : load_some<T, 4>(d + od, in ? no : 0);
      if constexpr (FACTOR != FACTOR_NONE) vf[e] = WHOLE ? load_pack<Q, 4>(q + of) : load_some<Q, 4>(q + of, in ? no : 0);
      p += ES * a.ldx;
      d += ES * a.ld_dy;
      q += ES * a.Co;
      if (!WHOLE) __builtin_amdgcn_sched_barrier(0);  // (a row at a time: nothing to gain, and fewer registers)
    }
    auto dz = [&](int e, int j) __attribute__((always_inline)) {
      if constexpr (FACTOR != FACTOR_NONE) return times_factor<FACTOR>((float)vd[e].v[j], vf[e].v[j], a.leak);
      return (float)vd[e].v[j];
    };
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < RE; ++e) {
        floatx4 z;
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = dz(e, j);
        sums += z;
#pragma unroll
        for (int i = 0; i < 4 * TI; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vx[i / 4][e].v[i & 3], z[j], acc[i][j], 0, 0, 0);
      }
    } else {
      F fx[4 * TI];
#pragma unroll
      for (int i = 0; i < 4 * TI; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) fx[i][e] = vx[i / 4][e].v[i & 3];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        F fd, rest;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = dz(e, j);
          sums[j] += z;
          T value = (T)z, low = (T)0.f;
          if constexpr (FACTOR != FACTOR_NONE) split(z, value, low);
          fd[e] = value;
          rest[e] = low;
        }
#pragma unroll
        for (int i = 0; i < 4 * TI; ++i) acc[i][j] = mma(fx[i], fd, acc[i][j]);
        if constexpr (FACTOR != FACTOR_NONE)
#pragma unroll
          for (int i = 0; i < 4 * TI; ++i) acc[i][j] = mma(fx[i], rest, acc[i][j]);
        if (TI == 2) __builtin_amdgcn_sched_barrier(0);  // (one column tile's operands in registers at a time)
      }
    }
  };
  int64_t r = r0 + wave * ROWS;
  for (; r + ROWS <= inside; r += 4 * ROWS) step(std::true_type(), r);
  for (; r < r1; r += 4 * ROWS) step(std::false_type(), r);
  // sums[j] of column 4 li + j: the four lane quarters' rows
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sums[j] += __shfl_xor(sums[j], 16);
    sums[j] += __shfl_xor(sums[j], 32);
  }
  // waves 1, 2, 3 hand over to wave 0, one after the other
#pragma unroll 1
  for (int w = 1; w < 4; ++w) {
    if (wave == w) {
#pragma unroll
      for (int i = 0; i < 4 * TI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) *(floatx4 *)(red + ((i * 4 + j) * 64 + lane) * 4) = acc[i][j];
      if (lq == 0)
#pragma unroll
        for (int j = 0; j < 4; ++j) red[TI * 4096 + 4 * li + j] = sums[j];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < 4 * TI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += *(const floatx4 *)(red + ((i * 4 + j) * 64 + lane) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[j] += red[TI * 4096 + 4 * li + j];
    }
    __syncthreads();
  }
  if (wave != 0) return;
  float *slab = a.slab + (int64_t)slice * a.Ci * a.Co;
  const int co = co0 + 4 * li, no = a.Co - co;
#pragma unroll
  for (int i = 0; i < 4 * TI; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int row = ci0 + 64 * (i / 4) + 16 * lq + 4 * q + (i & 3);  // A row 4 lq + q of tile i
      if (row < a.Ci && no > 0) {
        Pack<float, 4> v = {{acc[i][0][q] * a.up, acc[i][1][q] * a.up, acc[i][2][q] * a.up, acc[i][3][q] * a.up}};
        store_some<float, 4>(slab + (int64_t)row * a.Co + co, v, no);
      }
    }
  if (bias && lq == 0 && no > 0) {
    Pack<float, 4> v = {{sums[0] * a.up, sums[1] * a.up, sums[2] * a.up, sums[3] * a.up}};
    store_some<float, 4>(a.slab + (int64_t)a.slices * a.Ci * a.Co + (int64_t)slice * a.Co + co, v, no);
  }
}

// the slabs added: wave w of 16 takes slabs w, w + 16, ..., then the waves in order; element e of [Ci * Co] then [Co]
template <class T>
__global__ void __launch_bounds__(1024) k_linear_dw_join(const float *slab, int slices, int64_t nw, int nb, T *d_weight, T *d_bias) {
  __shared__ float red[16][64];
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int64_t e = (int64_t)blockIdx.x * 64 + lane;
  const bool in = e < nw + nb, w = e < nw;
  const float *p = w ? slab + e : slab + slices * nw + (e - nw);
  const int64_t step = w ? nw : nb;
  float s = 0.f;
  if (in)
#pragma unroll 8
    for (int i = wave; i < slices; i += 16) s += p[i * step];
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || !in) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += red[i][lane];
  if (w) d_weight[e] = (T)s;
  else d_bias[e - nw] = (T)s;
}

// ---------------------------------------------------------------------- host ---
constexpr int64_t LIN_MAX_LD = (int64_t)1 << 26;  // (31 rows of it in 32 bits)
static int lin_check(int64_t N, int n_in, int n_out, int dtype) {
  SCN_REQUIRE(dtype == SCN_F32 || dtype == SCN_BF16 || dtype == SCN_F16, "linear: dtype");
  SCN_REQUIRE(n_in >= 1 && n_out >= 1 && n_in <= 65536 && n_out <= 65536, "linear: 1 to 65536 planes");
  SCN_REQUIRE((int64_t)n_in * n_out <= ((int64_t)1 << 27), "linear: at most 2^27 weights");  // (16 threads each, of 2^32 a launch)
  SCN_REQUIRE(N >= 0 && N < ((int64_t)1 << 31), "linear: fewer than 2^31 sites");
  return 0;
}

template <class F>
static int by_type(int dtype, F &&f) {
  if (dtype == SCN_F32) return f((float)0);
  if (dtype == SCN_BF16) return f((__bf16)0);
  return f((_Float16)0);
}

// The forward pass's weights come as [n_in, n_out].  Workgroups whose weights stay in LDS scatter them there themselves: 5,000 to 200,000
// sites x 64..128 to 20..256 planes take 1.5 to 5 us less than with a launch (2.5 us where they are cached, 5 where not) that lays them out
// as [n_out, n_in] first.  That launch is needed where the weights do not stay and every workgroup fetches all of them (four column tiles
// of 22 k-groups do), and for the eight column tiles that many outputs of 16-bit types are worth (200,000 x 128 to 256, bf16: 40.7 us,
// 47.6 without; to 128 30.2 and 29.4; 600,000 x 448 to 256, where eight do not stay and four do, 308 and 338).
constexpr int64_t LIN_WIDE = (int64_t)1 << 25;  // sites x n_out
constexpr int LIN_LDS = 163840;  // of a CU
constexpr int LIN_FEW = 4;  // up to this many sites: k_linear_few
// eight column tiles fill the chip and pad no more than four
static bool lin_wide(int64_t N, int M) {
  return M > 64 && (N + 127) / 128 * ((M + 127) / 128) >= 256 && (M + 63) / 64 == 2 * ((M + 127) / 128);
}
static bool lin_transposes(int64_t N, int n_in, int n_out, int dtype) {
  const int row = n_in * (dtype == SCN_F32 ? 4 : 2);
  return N > LIN_FEW && (row > 22 * 64 || (dtype != SCN_F32 && N * n_out >= LIN_WIDE && lin_wide(N, n_out)));
}

template <class T, int NT, int MODE, int X>
static int linear_launch(LinearArgs a, hipStream_t st) {
  constexpr int KG = 4 * Elem<T>::V, group_bytes = NT * 64 * 16;
  // bias, results, next tile
  auto rest = [](int waves) { return NT * 16 * 4 + waves * lin_piece_bytes(NT, lin_packed(MODE, sizeof(T))) + 16; };
  a.groups = (a.K + KG - 1) / KG;
  a.chunk_groups = a.groups;
  a.col_blocks = (a.M + NT * 16 - 1) / (NT * 16);
  const bool stay = a.groups * group_bytes + rest(lin_waves(NT, true)) <= LIN_LDS;
  int64_t rows, lds;
  if (stay) {  // one workgroup a CU, the column blocks of a row block on one XCD
    rows = a.col_blocks <= 32 ? 32 / a.col_blocks * 8 : 256 / a.col_blocks;
    const int64_t tiles = (a.N + 31) / 32;
    if (rows > tiles) rows = tiles;
    if (rows < 1) rows = 1;
    lds = a.groups * group_bytes + rest(lin_waves(NT, true));
  } else {
    a.chunk_groups = 32768 / group_bytes;
    rows = (a.N + 127) / 128;
    lds = a.chunk_groups * group_bytes + rest(lin_waves(NT, false));
  }
  SCN_REQUIRE(rows * a.col_blocks < ((int64_t)1 << 22), "linear: sites x planes beyond a launch of 2^32 threads");
  a.row_blocks = (int)rows;
  auto k = stay ? k_linear<T, NT, MODE, X, true> : k_linear<T, NT, MODE, X, false>;
  k<<<(unsigned)(rows * a.col_blocks), 64 * lin_waves(NT, stay), lds, st>>>(a);
  SCN_CHECK_LAUNCH();
  return 0;
}
// wide column blocks read the rows least often; narrower ones while the chip is not full, if they pad fewer planes, or for fp32, whose
// matrix instructions are what counts (200,000 x 128 to 256: 148 us, 160 with eight column tiles)
template <class T, int MODE, int X>
static int linear_by_width(const LinearArgs &a, hipStream_t st) {
  if (a.M <= 32 || (a.N + 127) / 128 * ((a.M + 63) / 64) < 256) return linear_launch<T, 2, MODE, X>(a, st);
  if constexpr (sizeof(T) == 2)
    if (lin_wide(a.N, a.M) && (MODE == 1 || a.transposed)) return linear_launch<T, 8, MODE, X>(a, st);
  return linear_launch<T, 4, MODE, X>(a, st);
}
template <class T, int ACT>
static int linear_forward(const LinearArgs &a, hipStream_t st) {
  if (a.N > LIN_FEW) return linear_by_width<T, 0, ACT>(a, st);
  const unsigned blocks = (unsigned)((a.M + 15) / 16);
  if (a.N == 1) k_linear_few<T, 1, ACT><<<blocks, 1024, 0, st>>>(a);
  else k_linear_few<T, 4, ACT><<<blocks, 1024, 0, st>>>(a);
  SCN_CHECK_LAUNCH();
  return 0;
}

// 1 / (1 - p); without factors the pass had no dropout
static float keep_scale(const void *factor, double p) { return factor ? (float)(1.0 / (1.0 - p)) : 1.f; }
// f(how the factors are stored)
template <class T, class F>
static int by_factor(const void *factor, int act, F &&f) {
  if (!factor) return f(std::integral_constant<int, FACTOR_NONE>());
  if constexpr (sizeof(T) == 4) return f(std::integral_constant<int, FACTOR_FLOAT>());
  else if (act == SCN_ACT_LEAKY) return f(std::integral_constant<int, FACTOR_SIGN>());
  else return f(std::integral_constant<int, std::is_same<T, __bf16>::value ? FACTOR_WIDE : FACTOR_SHORT>());
}

// row slices of dW: with its 64 x 64 tiles four workgroups a CU (two of the wide ones), no slice below 256 rows
static int dw_slices(int64_t N, int n_in, int n_out) {
  const int64_t tiles = (int64_t)((n_in + 63) / 64) * ((n_out + 63) / 64);
  int64_t s = (1024 + tiles - 1) / tiles, most = (N + 255) / 256;
  if (s > most) s = most;
  if (s >= 8) s &= ~(int64_t)7;
  return (int)(s < 1 ? 1 : s);
}
template <class T, int TI, int FACTOR>
static void dw_launch(DwArgs a, hipStream_t st) {
  a.tiles_i = (a.Ci + 64 * TI - 1) / (64 * TI);
  a.tiles_o = (a.Co + 63) / 64;
  k_linear_dw<T, TI, FACTOR><<<(unsigned)(a.slices * a.tiles_i * a.tiles_o), 256, 0, st>>>(a);
}

}  // namespace scn

using namespace scn;

extern "C" {

int scn_dropout(const void *x, int64_t ldx, void *y, int64_t N, int planes, int dtype, double p, const int64_t *rng, void *stream) {
  if (int e = lin_check(N, planes, 1, dtype)) return e;
  SCN_REQUIRE(p >= 0 && p < 1, "dropout: 0 <= p < 1");
  if (N == 0) return 0;
  SCN_REQUIRE(x && y && rng && ldx >= planes, "dropout: pointers and strides");
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int Q = Elem<T>::V / 4;
    const bool whole = planes % (4 * Q) == 0;
    const int items = (planes + 4 * Q - 1) / (4 * Q), rows = items <= 128 ? 256 / items : 1, slabs = items <= 128 ? 1 : (items + 255) / 256;
    int64_t blocks = (N + rows - 1) / rows, most = 4096 / slabs;
    if (blocks > most) blocks = most < 1 ? 1 : most;
    auto k = whole ? k_dropout<T, Q, true> : k_dropout<T, Q, false>;
    k<<<dim3((unsigned)blocks, slabs), 256, 0, as_stream(stream)>>>((const T *)x, ldx, (T *)y, N, planes, items, rows, drop_threshold(p),
                                                                  (float)(1.0 / (1.0 - p)), rng);
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

size_t scn_linear_forward_temp_bytes(int64_t N, int n_in, int n_out, int dtype) {
  return lin_transposes(N, n_in, n_out, dtype) ? (size_t)n_in * n_out * (dtype == SCN_F32 ? 4 : 2) : 0;
}

int scn_linear_forward(const void *x, int64_t ldx, const void *weight, const void *bias, const void *residual, int64_t ld_res,
                       void *y, void *factor, int64_t N, int n_in, int n_out, int act, double leakiness, double p,
                       const int64_t *rng, int dtype, void *temp, size_t temp_bytes, void *stream) {
  if (int e = lin_check(N, n_in, n_out, dtype)) return e;
  SCN_REQUIRE(act == SCN_ACT_LEAKY || act == SCN_ACT_SILU || act == SCN_ACT_GELU, "linear: activation");
  SCN_REQUIRE(p >= 0 && p < 1 && (p == 0 || rng), "linear: 0 <= p < 1, with random words if it is not 0");
  if (N == 0) return 0;
  SCN_REQUIRE(x && weight && y && ldx >= n_in && ldx <= LIN_MAX_LD && (!residual || (ld_res >= n_out && ld_res <= LIN_MAX_LD)),
              "linear: pointers and strides");
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
  a.up = (float)(1.0 / (1.0 - p));
  const bool transpose = lin_transposes(N, n_in, n_out, dtype);
  SCN_REQUIRE(!transpose || (temp && temp_bytes >= scn_linear_forward_temp_bytes(N, n_in, n_out, dtype)), "linear: workspace");
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (transpose) {
      k_linear_transpose<T><<<dim3((n_out + 31) / 32, (n_in + 31) / 32), 256, 0, as_stream(stream)>>>((const T *)weight, (T *)temp, n_in,
                                                                                                    n_out);
      SCN_CHECK_LAUNCH();
      a.weight = temp;
      a.transposed = 1;
    }
    if (act == SCN_ACT_SILU) return linear_forward<T, SCN_ACT_SILU>(a, as_stream(stream));
    if (act == SCN_ACT_GELU) return linear_forward<T, SCN_ACT_GELU>(a, as_stream(stream));
    if (a.leak == 1.f) return linear_forward<T, ACT_NONE>(a, as_stream(stream));
    return linear_forward<T, SCN_ACT_LEAKY>(a, as_stream(stream));
  });
}

int scn_linear_dinput(const void *d_y, int64_t ld_dy, const void *factor, const void *weight, void *d_x, int64_t N, int n_in,
                      int n_out, int act, double leakiness, double p, int dtype, void *stream) {
  if (int e = lin_check(N, n_in, n_out, dtype)) return e;
  SCN_REQUIRE(p >= 0 && p < 1, "linear: 0 <= p < 1");
  if (N == 0) return 0;
  SCN_REQUIRE(d_y && weight && d_x && ld_dy >= n_out && ld_dy <= LIN_MAX_LD, "linear: pointers and strides");
  LinearArgs a = {};
  a.in = d_y;
  a.ld_in = ld_dy;
  a.factor_in = factor;
  a.leak = (float)leakiness;
  a.up = keep_scale(factor, p);
  a.weight = weight;
  a.out = d_x;
  a.N = N;
  a.K = n_out;
  a.M = n_in;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_factor<T>(factor, act, [&](auto f) { return linear_by_width<T, 1, decltype(f)::value>(a, as_stream(stream)); });
  });
}

size_t scn_linear_dweight_temp_bytes(int64_t N, int n_in, int n_out) {
  return sizeof(float) * (size_t)dw_slices(N, n_in, n_out) * ((size_t)n_in * n_out + n_out);
}

int scn_linear_dweight(const void *x, int64_t ldx, const void *d_y, int64_t ld_dy, const void *factor, void *d_weight, void *d_bias,
                       int64_t N, int n_in, int n_out, int act, double leakiness, double p, int dtype, void *temp,
                       size_t temp_bytes, void *stream) {
  if (int e = lin_check(N, n_in, n_out, dtype)) return e;
  SCN_REQUIRE(p >= 0 && p < 1, "linear: 0 <= p < 1");
  SCN_REQUIRE(d_weight && (N == 0 || (x && d_y)) && ldx >= n_in && ld_dy >= n_out && ldx <= LIN_MAX_LD && ld_dy <= LIN_MAX_LD,
              "linear: pointers and strides");
  SCN_REQUIRE(temp && temp_bytes >= scn_linear_dweight_temp_bytes(N, n_in, n_out), "linear: workspace");
  DwArgs a = {};
  a.x = x;
  a.dy = d_y;
  a.factor = factor;
  a.leak = (float)leakiness;
  a.up = keep_scale(factor, p);
  a.ldx = ldx;
  a.ld_dy = ld_dy;
  a.N = N;
  a.Ci = n_in;
  a.Co = n_out;
  a.slices = dw_slices(N, n_in, n_out);
  a.slice_rows = ((N + a.slices - 1) / a.slices + 127) / 128 * 128;
  a.slab = (float *)temp;
  a.want_bias = d_bias != nullptr;
  const int64_t nw = (int64_t)n_in * n_out;
  const int nb = d_bias ? n_out : 0;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_factor<T>(factor, act, [&](auto f) {
      constexpr int FACTOR = decltype(f)::value;
      // (128 planes of x a tile: d_y and the factors are read half as often)
      if (n_in > 64) dw_launch<T, 2, FACTOR>(a, as_stream(stream));
      else dw_launch<T, 1, FACTOR>(a, as_stream(stream));
      return 0;
    });
    SCN_CHECK_LAUNCH();
    k_linear_dw_join<T><<<(unsigned)((nw + nb + 63) / 64), 1024, 0, as_stream(stream)>>>(a.slab, a.slices, nw, nb, (T *)d_weight,
                                                                                         (T *)d_bias);
    SCN_CHECK_LAUNCH();
    return 0;
  });
}

}  // extern "C"

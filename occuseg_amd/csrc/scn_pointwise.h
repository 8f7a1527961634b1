// What the pointwise operators share (group norm, dropout, 1x1 convolution): element types, activations with their slopes,
// the counter-based random words.  gfx950 only.
#pragma once
#include "scn_common.h"

namespace scn {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// V elements = 16 bytes
template <class T> struct Elem;
template <> struct Elem<float> { static constexpr int V = 4; };
template <> struct Elem<__bf16> { static constexpr int V = 8; };
template <> struct Elem<_Float16> { static constexpr int V = 8; };

// n consecutive elements whose address is a multiple of the ELEMENT size only (odd plane counts, column slices): one wide global
// access all the same, gfx950 takes them at any address
template <class T, int N>
struct Pack {
  T v[N];
};
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
  Pack<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

// ---------------------------------------------------------------- activations ---
// ACT: SCN_ACT_LEAKY  z > 0 ? z : leak * z      (leak 0 = ReLU, 1 = none)
//      SCN_ACT_SILU   z / (1 + e^-z)
//      SCN_ACT_GELU   z Phi(z), Phi the normal distribution function
// EXACT (float features): expf / erff.  Otherwise the result is rounded to 8 or 11 bits behind this: the hardware's exp2, and
// Phi from Abramowitz & Stegun, Handbook of Mathematical Functions, 7.1.26 (|error of erf| <= 1.5e-7), which shares its
// exponential with the slope.
template <int ACT, bool EXACT>
__device__ __forceinline__ void act_value_slope(float z, float leak, float &value, float &slope) {
  if (ACT == SCN_ACT_LEAKY) {
    slope = z > 0 ? 1.f : leak;
    value = z > 0 ? z : z * leak;
  } else if (ACT == SCN_ACT_SILU) {
    const float e = EXACT ? expf(-z) : __expf(-z);
    const float s = EXACT ? 1.f / (1.f + e) : __builtin_amdgcn_rcpf(1.f + e);
    value = z * s;
    slope = s * fmaf(z, 1.f - s, 1.f);
  } else {
    float cdf, dens;  // Phi(z), its derivative
    if (EXACT) {
      cdf = fmaf(0.5f, erff(z * 0.70710678f), 0.5f);
      dens = 0.39894228f * expf(-0.5f * z * z);
    } else {
      const float e = __expf(-0.5f * z * z);
      const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
      const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
      const float tail = 0.5f * poly * e;  // 1 - Phi(|z|)
      cdf = z > 0 ? 1.f - tail : tail;
      dens = 0.39894228f * e;
    }
    value = z * cdf;
    slope = fmaf(z, dens, cdf);
  }
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_value(float z, float leak) {
  float v, s;
  act_value_slope<ACT, EXACT>(z, leak, v, s);
  return v;
}
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_slope(float z, float leak) {
  float v, s;
  act_value_slope<ACT, EXACT>(z, leak, v, s);
  return s;
}

// --------------------------------------------------------------- random words ---
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel Random Numbers: As Easy as 1, 2, 3; SC 2011): four 32-bit words per
// (site, four planes), a function of the counter (plane / 4, site, offset) and the key = seed alone, so the backward pass -- and
// any other kernel that needs the mask -- makes them again instead of reading them.  20 products of 32 x 32 bits per 4 elements.
struct Words {
  uint32_t w[4];
};
struct RngKey {
  uint32_t k0, k1, c2, c3;
};
__device__ __forceinline__ RngKey rng_key(const int64_t *rng) {
  const uint64_t seed = (uint64_t)rng[0], offset = (uint64_t)rng[1];
  return RngKey{(uint32_t)seed, (uint32_t)(seed >> 32), (uint32_t)offset, (uint32_t)(offset >> 32)};
}
__device__ __forceinline__ Words philox(RngKey key, uint32_t quad, uint32_t site) {
  uint32_t c0 = quad, c1 = site, c2 = key.c2, c3 = key.c3, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}
// an element is kept iff its word >= p 2^32
inline uint32_t drop_threshold(double p) { return (uint32_t)(p * 4294967296.0); }

}  // namespace scn

// What the pointwise operators share (group norm, dropout, 1x1 convolution): element types, activations with their slopes,
// the counter-based random words.  gfx950 only.
#pragma once
#include "scn_common.h"

#include <type_traits>

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
// One reciprocal and one exponential of the hardware each (1 ulp; an exponent x is off by |x| 2^-24, where e^x is as small).  The tail
// 1 - Phi(t), t >= 0, is the density phi(t) -- which the slope needs too -- times a smooth function of t, here a polynomial in
// s = 1 / (1 + c t) without a constant term, fitted to (1 - Phi) / phi over t <= 40 by iteratively reweighted least squares.  Largest
// relative error of z Phi(z) as these steps compute it in fp32, |z| <= 3 and |z| <= 9 (where the exponent's rounding counts: up to 58):
// nine terms (float features) 6.5e-7 and 3.8e-6, seven (fp16, whose half step is 4.9e-4) 3.2e-6 and 4.4e-6, five (bf16: 3.9e-3) 6.0e-5
// and 6.1e-5; z / (1 + e^-z), |z| <= 16: 5.5e-7.
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
template <class T> constexpr int act_terms() { return sizeof(T) == 4 ? 9 : std::is_same<T, __bf16>::value ? 5 : 7; }

template <int ACT, class T>
__device__ __forceinline__ void act_value_slope(float z, float leak, float &value, float &slope) {
  if (ACT == SCN_ACT_LEAKY) {
    slope = z > 0 ? 1.f : leak;
    value = z * slope;
  } else if (ACT == SCN_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + exp2_hw(z * -1.44269504f));
    value = z * s;
    slope = fmaf(value, 1.f - s, s);
  } else {
    const float dens = exp2_hw(fmaf(z * z, -0.72134752f, -1.32574806f)), t = fabsf(z);
    float p;
    if (act_terms<T>() == 9) {
      const float s = __builtin_amdgcn_rcpf(fmaf(0.36f, t, 1.f));
      p = fmaf(s, -0.075829186f, 0.349820765f);
      p = fmaf(s, p, -0.560674736f);
      p = fmaf(s, p, 0.269293545f);
      p = fmaf(s, p, -0.001043101f);
      p = fmaf(s, p, 0.240750164f);
      p = fmaf(s, p, 0.310843324f);
      p = fmaf(s, p, 0.360157293f);
      p = fmaf(s, p, 0.359996093f) * s;
    } else if (act_terms<T>() == 7) {
      const float s = __builtin_amdgcn_rcpf(fmaf(0.38f, t, 1.f));
      p = fmaf(s, 0.122704407f, -0.401142778f);
      p = fmaf(s, p, 0.286758777f);
      p = fmaf(s, p, 0.150356744f);
      p = fmaf(s, p, 0.335371260f);
      p = fmaf(s, p, 0.379249847f);
      p = fmaf(s, p, 0.380019100f) * s;
    } else {
      const float s = __builtin_amdgcn_rcpf(fmaf(0.39f, t, 1.f));
      p = fmaf(s, -0.218651797f, 0.413951101f);
      p = fmaf(s, p, 0.270861309f);
      p = fmaf(s, p, 0.397368879f);
      p = fmaf(s, p, 0.389709251f) * s;
    }
    const float tail = p * dens, cdf = z > 0 ? 1.f - tail : tail;
    value = z * cdf;
    slope = fmaf(z, dens, cdf);
  }
}
template <int ACT, class T>
__device__ __forceinline__ float act_value(float z, float leak) {
  float v, s;
  act_value_slope<ACT, T>(z, leak, v, s);
  return v;
}
template <int ACT, class T>
__device__ __forceinline__ float act_slope(float z, float leak) {
  float v, s;
  act_value_slope<ACT, T>(z, leak, v, s);
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
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }
// Products of rounds 1 to 3 depend on the plane (P) or on the site (S) alone: c = (quad, site, c2, c3) gives
//   round 1: quad M0 (P), c2 M1 (uniform)    round 2: f(site) M0 (S), f(quad) M1 (P)    round 3: f(quad) M0 (P), both M1
// so a thread that keeps its planes makes 16 of the 20 per site, one that keeps both halves 15.
struct PhiloxPlane {
  uint32_t c1, c2x, r3lo, r3hi;  // see philox_plane
};
struct PhiloxSite {
  uint32_t hi, lo;
};
constexpr uint32_t PH_M0 = 0xD2511F53u, PH_M1 = 0xCD9E8D57u, PH_W0 = 0x9E3779B9u, PH_W1 = 0xBB67AE85u;
__device__ __forceinline__ PhiloxPlane philox_plane(RngKey k, uint32_t quad) {
  const uint64_t a1 = (uint64_t)quad * PH_M0, b1 = (uint64_t)k.c2 * PH_M1;
  // after round 1: (hi(b1) ^ site ^ k0, lo(b1), hi(a1) ^ c3 ^ k1, lo(a1))
  const uint64_t b2 = (uint64_t)xor3((uint32_t)(a1 >> 32), k.c3, k.k1) * PH_M1;
  // after round 2: (hi(b2) ^ lo(b1) ^ k0', lo(b2), hi(a2) ^ lo(a1) ^ k1', lo(a2)),  a2 = (hi(b1) ^ site ^ k0) M0
  const uint64_t a3 = (uint64_t)xor3((uint32_t)(b2 >> 32), (uint32_t)b1, k.k0 + PH_W0) * PH_M0;
  // round 3 takes c1 = lo(b2) ^ k0'', c2 ^ .. = lo(a1) ^ k1', and a3
  return PhiloxPlane{(uint32_t)b2 ^ (k.k0 + 2 * PH_W0), (uint32_t)a1 ^ (k.k1 + PH_W1), (uint32_t)a3, (uint32_t)(a3 >> 32) ^ (k.k1 + 2 * PH_W1)};
}
__device__ __forceinline__ PhiloxSite philox_site(RngKey k, uint32_t site) {
  const uint64_t b1 = (uint64_t)k.c2 * PH_M1;
  const uint64_t a2 = (uint64_t)xor3((uint32_t)(b1 >> 32), site, k.k0) * PH_M0;
  return PhiloxSite{(uint32_t)(a2 >> 32), (uint32_t)a2};
}
__device__ __forceinline__ Words philox(RngKey k, const PhiloxPlane &p, const PhiloxSite &s) {
  // round 3
  const uint64_t b3 = (uint64_t)(s.hi ^ p.c2x) * PH_M1;
  uint32_t c0 = (uint32_t)(b3 >> 32) ^ p.c1, c1 = (uint32_t)b3, c2 = p.r3hi ^ s.lo, c3 = p.r3lo;
  uint32_t k0 = k.k0 + 3 * PH_W0, k1 = k.k1 + 3 * PH_W1;
#pragma unroll
  for (int r = 3; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * PH_M0, b = (uint64_t)c2 * PH_M1;
    c0 = xor3((uint32_t)(b >> 32), c1, k0);
    c1 = (uint32_t)b;
    c2 = xor3((uint32_t)(a >> 32), c3, k1);
    c3 = (uint32_t)a;
    k0 += PH_W0;
    k1 += PH_W1;
  }
  return Words{{c0, c1, c2, c3}};
}
// an element is kept iff its word >= p 2^32
inline uint32_t drop_threshold(double p) { return (uint32_t)(p * 4294967296.0); }

}  // namespace scn

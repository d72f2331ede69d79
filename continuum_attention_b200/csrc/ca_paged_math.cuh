// ca_paged_math.cuh -- the scalar work per score that the two tensor-core kernels over a paged
// cache share: from a run of scores to weights in two 16-bit parts.
#pragma once

#include "ca_paged.cuh"

namespace ca {
namespace paged {

constexpr float kRescaleNats = 8.f;   // the reference maximum moves when it grows by more

// The reference that exponentials are taken from, in log2 units, for the reference maximum m.  In f16 weights stand
// 2^4 above it: the largest is then e^8 2^4 = 47700 (a weight is at most its segments' larger exponential), and
// small ones are whole down to 2^-18 of that of m itself instead of 2^-14.
template <typename T>
__device__ __forceinline__ float reference2(float m) {
  return m == -INFINITY ? 0.f : std::is_same<T, __half>::value ? fmaf(m, kLog2e, -4.f) : m * kLog2e;
}

// a weight pair as two 16-bit parts: hi + lo keeps 16 bits (bf16) or 21 (f16)
template <typename T>
__device__ __forceinline__ void split2(float2 w, uint32_t& hi, uint32_t& lo);
template <>
__device__ __forceinline__ void split2<__nv_bfloat16>(float2 w, uint32_t& hi, uint32_t& lo) {
  const uint32_t u0 = __float_as_uint(w.x), u1 = __float_as_uint(w.y);
  hi = __byte_perm(u0, u1, 0x7632);   // bf16 by truncation; the remainder is exact
  const float2 r = sub2(w, make_float2(__uint_as_float(u0 & 0xffff0000u), __uint_as_float(u1 & 0xffff0000u)));
  const __nv_bfloat162 l = __floats2bfloat162_rn(r.x, r.y);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
template <>
__device__ __forceinline__ void split2<__half>(float2 w, uint32_t& hi, uint32_t& lo) {
  // 10 bits of mantissa by truncation, exact in f16 above its subnormals (below 2^-14 hi rounds by 2^-25 at
  // most); the remainder is exact
  const float2 t = make_float2(__uint_as_float(__float_as_uint(w.x) & 0xffffe000u),
                               __uint_as_float(__float_as_uint(w.y) & 0xffffe000u));
  const __half2 h = __floats2half2_rn(t.x, t.y);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  const float2 r = sub2(w, t);
  const __half2 l = __floats2half2_rn(r.x, r.y);
  lo = *reinterpret_cast<const uint32_t*>(&l);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
// A segment's M0 and M1 from their closed forms; near d = 0 from M1's series, el ps, and M0 = e - d M1.  (The latter
// everywhere would cost a select less, and far from 0 all but e 2^-22 of M0's precision.)
__device__ __forceinline__ void near_zero(float& m0, float& m1, float nd, float el, float ps, float e, float thr) {
  asm("{\n\t.reg .pred p;\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tsetp.lt.f32 p, t, %6;\n\t"
      "@p mul.f32 %1, %3, %4;\n\t@p fma.rn.f32 %0, %2, %1, %5;\n\t}"
      : "+f"(m0), "+f"(m1) : "f"(nd), "f"(el), "f"(ps), "f"(e), "f"(thr));
}
// Weights of one lane's run of one row, as two 16-bit parts.  sv[j] = scaled scores of keys (kc + j, kc + NJ + j),
// sL that of key kc - 1, m2 the reference maximum in log2 units.  Parts j weigh keys (kc - 1 + j, kc + NJ - 1 + j);
// first is the pair of place 0, unsplit, but for the mass that ends at key kc - 1, which is the lane's to
// the left; last is the mass that ends at the run's last key.  Pair by pair, each needing the one before:
// a score's registers take its weight's parts.
// edge (of the whole warp) adds the half caps of keys 0 and i where this run weighs them.  Key i's belongs to
// this piece when i >= lowest: the piece before it has weighed its own last key to the end.  (One body with
// a jump around the caps: a second body for edges cost 30 moves a tile where the two meet.)
template <typename T, int NJ>
__device__ __forceinline__ void weigh(const float2 (&sv)[NJ], float m2, float sL, bool edge, int kc, int i, int lowest,
                                      uint32_t (&hi)[NJ], uint32_t (&lo)[NJ], float2& first, float& last, float2& z2) {
  const float2 l2e = splat2(kLog2e), nm2 = splat2(-m2);
  auto exps = [&](float2 v) {
    const float2 arg = fma2(v, l2e, nm2);
    return make_float2(ex2_approx(arg.x), ex2_approx(arg.y));
  };
  const float2 e_end = exps(sv[NJ - 1]);
  float2 sl0 = make_float2(sL, sv[NJ - 1].x);
  float2 el0 = make_float2(ex2_approx(fmaf(sL, kLog2e, -m2)), e_end.x);
  float2 m1_before = splat2(0.f);
  // four pairs side by side, step by step: their chains hide each other's latencies
#pragma unroll
  for (int j0 = 0; j0 < NJ; j0 += 4) {
    float2 e[4], nd[4], rn[4], ps[4], m1[4], w[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) e[t] = j0 + t == NJ - 1 ? e_end : exps(sv[j0 + t]);
#pragma unroll
    for (int t = 0; t < 4; ++t) nd[t] = sub2(t ? sv[j0 + t - 1] : sl0, sv[j0 + t]);                  // -d
#pragma unroll
    for (int t = 0; t < 4; ++t) rn[t] = make_float2(rcp_approx(nd[t].x), rcp_approx(nd[t].y));     // -1/d
#pragma unroll
    for (int t = 0; t < 4; ++t) ps[t] = fma2(splat2(-1.f / 30.f), nd[t], splat2(1.f / 8.f));      // J1's series in -nd
#pragma unroll
    for (int t = 0; t < 4; ++t) ps[t] = fma2(ps[t], nd[t], splat2(-1.f / 3.f));
#pragma unroll
    for (int t = 0; t < 4; ++t) ps[t] = fma2(ps[t], nd[t], splat2(1.f / 2.f));
#pragma unroll
    for (int t = 0; t < 4; ++t) w[t] = mul2(sub2(t ? e[t - 1] : el0, e[t]), rn[t]);                 // M0
#pragma unroll
    for (int t = 0; t < 4; ++t) m1[t] = mul2(sub2(w[t], e[t]), rn[t]);                              // M1, closed
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const float2 el = t ? e[t - 1] : el0;
      near_zero(w[t].x, m1[t].x, nd[t].x, el.x, ps[t].x, e[t].x, kSeriesMaxFwd);
      near_zero(w[t].y, m1[t].y, nd[t].y, el.y, ps[t].y, e[t].y, kSeriesMaxFwd);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      z2 = add2(z2, w[t]);
      w[t] = sub2(w[t], m1[t]);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (j0 + t > 0) w[t] = add2(w[t], t ? m1[t - 1] : m1_before);
    if (edge) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float2 el = t ? e[t - 1] : el0;
        const int kx = kc + j0 + t - 1, ky = kx + NJ;      // the keys these weights belong to
        const float nx = (kx == 0 && i >= 0 ? 0.5f : 0.f) + (kx == i && i >= lowest ? 0.5f : 0.f);
        const float2 cap = make_float2(nx > 0.f ? nx * el.x : 0.f, ky == i ? 0.5f * el.y : 0.f);
        w[t] = add2(w[t], cap);
        z2 = add2(z2, cap);
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (j0 + t > 0) split2<T>(w[t], hi[j0 + t], lo[j0 + t]);
      else first = w[t];
    }
    m1_before = m1[3];
    sl0 = sv[j0 + 3];
    el0 = e[3];
  }
  first.y += m1_before.x;
  last = m1_before.y;
}

}  // namespace paged
}  // namespace ca

// Eight consecutive elements of a row at a time, in any of the library's float types or in int8, and the
// division that turns a flat item index into a row: shared by the kernels of the eight-bit operators.
#pragma once

#include "../../include/da_b200.h"
#include "common.cuh"

namespace da {

// n / d for n < 2^31 as a multiplication: with l = ceil(log2 d) and m = floor(2^(31 + l) / d) + 1 the
// quotient is mulhi(n, m) >> (l - 1) (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994, for 31-bit dividends).
struct Div31 {
  static constexpr int64_t kMax = 0x7fffffffLL;
  uint32_t d, m, s;
  explicit Div31(uint32_t divisor) : d(divisor), m(0), s(0) {
    uint32_t l = 0;
    while ((uint64_t(1) << l) < d) ++l;
    if (l > 0) {
      m = (uint32_t)((uint64_t(1) << (31 + l)) / d + 1);
      s = l - 1;
    }
  }
  DA_DEV uint32_t div(uint32_t n) const { return m ? __umulhi(n, m) >> s : n; }
};

inline bool vec8_ok(const void* p, int dtype, int64_t ld) {  // 16-byte accesses of 8 elements
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * (dtype == DA_F32 ? 4 : 2) % 16 == 0;
}

DA_DEV void load8(const void* p, int dtype, int64_t off, float* v) {
  if (dtype == DA_F32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + off);
    const float4 a = s[0], b = s[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + off);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = dtype == DA_BF16 ? unpack2<__nv_bfloat16>(u[e]) : unpack2<__half>(u[e]);
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
  }
}

DA_DEV void store8(void* p, int dtype, int64_t off, const float* v) {
  if (dtype == DA_F32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + off);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      u[e] = dtype == DA_BF16 ? pack2<__nv_bfloat16>(v[2 * e], v[2 * e + 1]) : pack2<__half>(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + off) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}

DA_DEV float load1(const void* p, int dtype, int64_t off) {
  if (dtype == DA_F32) return static_cast<const float*>(p)[off];
  if (dtype == DA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[off]);
  return __half2float(static_cast<const __half*>(p)[off]);
}

DA_DEV void store1(void* p, int dtype, int64_t off, float v) {
  if (dtype == DA_F32) static_cast<float*>(p)[off] = v;
  else if (dtype == DA_BF16) static_cast<__nv_bfloat16*>(p)[off] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[off] = __float2half_rn(v);
}

// v as a tensor of this dtype holds it.
DA_DEV float round_to(float v, int dtype) {
  if (dtype == DA_BF16) return __bfloat162float(__float2bfloat16_rn(v));
  if (dtype == DA_F16) return __half2float(__float2half_rn(v));
  return v;
}

// Eight integers in [-128, 127] as bytes, lowest column first.
DA_DEV uint2 pack_s8x8(const int* o) {
  auto four = [](const int* i) {
    const uint32_t lo = __byte_perm(i[0], i[1], 0x0040), hi = __byte_perm(i[2], i[3], 0x0040);
    return __byte_perm(lo, hi, 0x5410);
  };
  return make_uint2(four(o), four(o + 4));
}

// Eight bytes as signed integers in fp32: a byte xor 0x80 in the low mantissa bits of 2^23 is 2^23 + 128 + value.
DA_DEV void unpack_s8x8(uint2 w, float* v) {
  const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    v[e] = __uint_as_float(__byte_perm(u[e >> 2], 0x4b000000u, 0x7540 | (e & 3))) - 8388736.f;
}

// GELU in its exact form, z times the normal distribution function, and its derivative.  The distribution
// function comes from Hastings' approximation of erfc (Abramowitz and Stegun 7.1.26, absolute error at
// most 1.5e-7): with x = |z| / sqrt(2) and t = 1 / (1 + 0.3275911 x), erfc(x) = t (a1 + ... + a5 t^4) exp(-x^2),
// whose exponential is the density that the derivative needs too.
struct NormalCdf {
  float cdf, density;  // Phi(z), and exp(-z^2 / 2) without its factor 1 / sqrt(2 pi)
};
DA_DEV NormalCdf normal_cdf(float z) {
  const float x = fabsf(z) * 0.70710678118654752f;
  const float t = __fdividef(1.f, fmaf(0.3275911f, x, 1.f));
  float poly = fmaf(1.061405429f, t, -1.453152027f);
  poly = fmaf(poly, t, 1.421413741f);
  poly = fmaf(poly, t, -0.284496736f);
  poly = fmaf(poly, t, 0.254829592f);
  const float density = ex2(z * z * -0.72134752044448170f);  // exp(-z^2 / 2)
  const float tail = 0.5f * poly * t * density;              // Phi(-|z|)
  return {z >= 0.f ? 1.f - tail : tail, density};
}
DA_DEV float gelu8(float z) { return z * normal_cdf(z).cdf; }

}  // namespace da

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

// Two fp32 values in one register pair; multiplications and additions of pairs take one issue slot.
struct F2 {
  unsigned long long v;
};
DA_DEV F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
DA_DEV void split(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
DA_DEV F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
DA_DEV F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
DA_DEV F2 dup(float a) { return f2(a, a); }

// The lower tail of the normal distribution, Phi(-|z|), and its density without the factor 1 / sqrt(2 pi), for
// two values: Hastings' approximation of erfc (Abramowitz and Stegun 7.1.26, absolute error at most 1.5e-7).
// With x = |z| / sqrt(2) and t = 1 / (1 + 0.3275911 x), erfc(x) = t (a1 + ... + a5 t^4) exp(-x^2), and Phi(-|z|) is
// half of it; the exponential is the density that GELU's derivative needs too.  The two reciprocals come from
// one, of their product (|z| is cut at 1e4, where the density is 0): the special-function unit, 16 lanes a clock
// against 128 for additions, is what bounds an epilogue with GELU.
constexpr float kCut = 1e4f;
DA_DEV void normal_tail2(float z0, float z1, F2& tail, F2& density) {
  const F2 z = f2(z0, z1);
  const F2 arg = mul2(mul2(z, dup(-0.72134752044448170f)), z);  // -z^2 / 2 in base 2
  const F2 a = fma2(f2(fminf(fabsf(z0), kCut), fminf(fabsf(z1), kCut)), dup(0.23164188f), dup(1.f));
  float a0, a1, g0, g1;
  split(a, a0, a1);
  split(arg, g0, g1);
  const F2 t = mul2(dup(__fdividef(1.f, a0 * a1)), f2(a1, a0));
  density = f2(ex2(g0), ex2(g1));
  F2 poly = fma2(t, dup(0.5f * 1.061405429f), dup(0.5f * -1.453152027f));
  poly = fma2(poly, t, dup(0.5f * 1.421413741f));
  poly = fma2(poly, t, dup(0.5f * -0.284496736f));
  poly = fma2(poly, t, dup(0.5f * 0.254829592f));
  tail = mul2(mul2(poly, t), density);
}

// GELU in its exact form: z Phi(z) = max(z, 0) - |z| Phi(-|z|); an infinity keeps its limit, inf or 0.
DA_DEV float gelu_of(float z, float tail) {
  return fmaf(-fminf(fabsf(z), kCut), tail, fmaxf(z, 0.f));  // (NaN: max is 0, but the tail is NaN)
}
DA_DEV void gelu2(float& z0, float& z1) {
  F2 tail, density;
  normal_tail2(z0, z1, tail, density);
  float t0, t1;
  split(tail, t0, t1);
  z0 = gelu_of(z0, t0);
  z1 = gelu_of(z1, t1);
}

// GELU'(z) = Phi(z) + z density / sqrt(2 pi), and z becomes GELU(z).
DA_DEV void gelu_grad2(float& z0, float& z1, float& s0, float& s1) {
  F2 tail, density;
  normal_tail2(z0, z1, tail, density);
  float t0, t1, d0, d1;
  split(tail, t0, t1);
  split(mul2(mul2(density, dup(0.39894228040143268f)), f2(z0, z1)), d0, d1);
  s0 = d0 + (z0 > 0.f ? 1.f - t0 : t0);
  s1 = d1 + (z1 > 0.f ? 1.f - t1 : t1);
  z0 = gelu_of(z0, t0);
  z1 = gelu_of(z1, t1);
}

}  // namespace da

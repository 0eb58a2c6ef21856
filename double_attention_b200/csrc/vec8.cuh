// Pieces that the kernels of the eight-bit operators share: the division that turns a flat item index into a row,
// single values of any float type, packed fp32 pairs, bytes to and from fp32, and GELU.
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

// Two fp32 values in one register pair; additions and multiplications of pairs take one issue slot.
struct F2 {
  unsigned long long v;
};
DA_DEV F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
DA_DEV F2 dup(float a) { return f2(a, a); }
DA_DEV void split(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
DA_DEV F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
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
// A pair of 16-bit values in fp32, and two fp32 values rounded to a pair.
template <typename T>
DA_DEV F2 widen(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  const float2 f = unpack2<T>(w);
  return f2(f.x, f.y);
}
template <typename T>
DA_DEV uint32_t narrow(F2 x) {
  float a, b;
  split(x, a, b);
  return pack2<T>(a, b);
}

// Eight 16-bit values from the m-th on (m in [0, 8]) of the sixteen in a, b.
DA_DEV uint4 shift16(uint4 a, uint4 b, int m) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t u[6], v[5];
#pragma unroll
  for (int i = 0; i < 6; ++i) u[i] = m & 4 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) v[i] = m & 2 ? u[i + 1] : u[i];
  if (m == 8) return b;
  return m & 1 ? make_uint4(__funnelshift_r(v[0], v[1], 16), __funnelshift_r(v[1], v[2], 16),
                            __funnelshift_r(v[2], v[3], 16), __funnelshift_r(v[3], v[4], 16))
               : make_uint4(v[0], v[1], v[2], v[3]);
}

// Integers by addition: for |v| < 2^22, v + kRoundAt rounds v to the nearest integer (ties to even), which the
// low byte of the sum's bits holds in two's complement when it lies in [-128, 127].
constexpr float kRoundAt = 12582912.f;  // 1.5 * 2^23
// The low bytes of four such sums.
DA_DEV uint32_t low_bytes(F2 lo, F2 hi) {
  float a, b, c, d;
  split(lo, a, b);
  split(hi, c, d);
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                     __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
}
// Four bytes as signed integers in fp32: a byte xor 0x80 in the low mantissa bits of 2^23 is 2^23 + 128 + value.
DA_DEV void signed_bytes(uint32_t w, F2& lo, F2& hi) {
  w ^= 0x80808080u;
  auto one = [&](uint32_t sel) { return __uint_as_float(__byte_perm(w, 0x4b000000u, sel)); };
  lo = add2(f2(one(0x7540), one(0x7541)), dup(-8388736.f));
  hi = add2(f2(one(0x7542), one(0x7543)), dup(-8388736.f));
}

// The lower tail of the normal distribution, Phi(-|z|), for two values, and -|z|.  log2 Phi(-u) is smooth and nearly a
// parabola, so a polynomial of degree 9 on [0, 10] and one power of two give the tail: fitted by iteratively
// reweighted least squares towards the smallest largest error of Phi, within 1.4e-7 of it, and to 8e-4 of its own
// size down to Phi(-10) = 8e-24, where |z| is cut.  One special-function instruction a value (16 lanes a clock
// against 128 for additions) and no division: the issue slots are what a kernel with GELU runs out of.
DA_DEV F2 normal_tail2(F2 z, F2& minus_abs) {
  float z0, z1, g0, g1;
  split(z, z0, z1);
  minus_abs = f2(fmaxf(-fabsf(z0), -10.f), fmaxf(-fabsf(z1), -10.f));  // (a NaN becomes -10)
  F2 p = fma2(minus_abs, dup(-2.2549588862830205e-08f), dup(-7.857490800233791e-07f));
  p = fma2(p, minus_abs, dup(-9.545614375383593e-06f));
  p = fma2(p, minus_abs, dup(-2.497381683497224e-05f));
  p = fma2(p, minus_abs, dup(0.000564999645575881f));
  p = fma2(p, minus_abs, dup(0.007658606860786676f));
  p = fma2(p, minus_abs, dup(0.05292050912976265f));
  p = fma2(p, minus_abs, dup(-0.45906803011894226f));
  p = fma2(p, minus_abs, dup(1.1511218547821045f));
  p = fma2(p, minus_abs, dup(-0.9999997019767761f));
  split(p, g0, g1);
  return f2(ex2(g0), ex2(g1));
}
DA_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// max(z, 0) - |z| Phi(-|z|) = z Phi(z): GELU in its exact form.  An infinity keeps its limit, inf or 0.
DA_DEV F2 gelu_of(F2 z, F2 tail, F2 minus_abs) {
  float z0, z1;
  split(z, z0, z1);
  return fma2(minus_abs, tail, f2(max_nan(z0, 0.f), max_nan(z1, 0.f)));
}
DA_DEV F2 gelu2(F2 z) {
  F2 minus_abs;
  const F2 tail = normal_tail2(z, minus_abs);
  return gelu_of(z, tail, minus_abs);
}
// GELU'(z) = Phi(z) + z exp(-z^2 / 2) / sqrt(2 pi), Phi(z) = 1/2 + sign(z) (1/2 - Phi(-|z|)); z becomes GELU(z).
DA_DEV F2 gelu_grad2(F2& z) {
  F2 minus_abs;
  const F2 tail = normal_tail2(z, minus_abs);
  float z0, z1, h0, h1, g0, g1;
  split(z, z0, z1);
  split(mul2(mul2(z, dup(-0.72134752044448170f)), z), g0, g1);  // -z^2 / 2 in base 2
  split(fma2(tail, dup(-1.f), dup(0.5f)), h0, h1);
  const F2 odd = f2(copysignf(h0, z0), copysignf(h1, z1));
  const F2 density = mul2(f2(ex2(g0), ex2(g1)), dup(0.39894228040143268f));
  const F2 slope = add2(fma2(density, z, odd), dup(0.5f));
  z = gelu_of(z, tail, minus_abs);
  return slope;
}

}  // namespace da

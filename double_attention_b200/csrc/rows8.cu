// Rows in 8 bits: residual add + norm whose rows leave in int8, the row quantiser and its inverse.
//
//   r = x + branch             rounded to the residual's dtype; the norm reads the rounded value
//   RMS norm:    v = r w,      rstd = 1 / sqrt(mean(r^2) + eps),  y = v rstd
//   LayerNorm:   y = (r - mean) rstd w + b
//   quantiser:   y = x
//   a = max |y|,  scale = a / 127,  q = rint(y 127 / a)
// For the RMS norm rstd cancels out of q: q = rint(v * (127 / max|v|)) and scale = max|v| rstd / 127, so q
// does not depend on the order in which the squares are added; maxima do not either.
//
// A row whose largest |v| is at most 1e-36 (127 / a would overflow) becomes q = 0 with scale 0.  A row that
// holds a NaN or an infinity gets a scale of NaN, so that it never decodes to plausible numbers.
//
// Bound: HBM.  One pass; a row stays in registers between its reductions (a warp up to 1024 columns, a block of up to
// 512 threads up to 16384; wider rows are read again, mostly from L2).  Measured: 262144 x 512 from an fp32 residual and a
// bf16 branch in 215 us (11 bytes an element, 6.9 TB/s), 8192 x 4096 quantised from bf16 in 16 us (6.3 TB/s), one row of
// 512 in 2.1 us; odd widths: 100003 x 501 in 94 us (5.8 TB/s).  LayerNorm: the same 214 us at 262144 x 512 and 2.4 us for
// one row; rows over several warps wait at two barriers for each of its three reductions, where the RMS norm has one
// barrier: 16384 x 4096 with a branch in 76 us (bf16) and 123 us (fp32 residual) against 72 and 112, and without one, with
// less to read under the waits, 64 against 39 (bf16), 16384 x 8192 from fp16 129 against 80.
#include "common.cuh"
#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace {

enum : int { kQuantize = 0, kRms = 1, kLayer = 2 };
constexpr float kTiny = 1e-36f;

struct NormArgs {
  const void* x;
  const void* branch;
  const void* weight;
  const void* bias;
  void* x_out;
  int8_t* q;
  float* scale;
  int64_t ldx, ldb, ldo, ldq, rows;
  int x_dtype, branch_dtype, weight_dtype, bias_dtype, kind, D;
  float eps;
  int aligned;  // weight and bias start on 16 bytes
};

// Sum and largest bit pattern over the threads of a row: a warp (kT = 32), a block of kT threads, or the block whatever
// its size (kT = 0; at most 32 warps).  `red`: a slot a warp.  Every thread adds in the same order (a butterfly adds
// the same pairs in every lane).
DA_DEV float warp_sum(float v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int kT>
DA_DEV float add_warps(const float* red) {
  if constexpr (kT == 0) {
    const int lane = threadIdx.x & 31;
    return warp_sum(lane < (int)blockDim.x / 32 ? red[lane] : 0.f);
  }
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < kT / 32; ++i) v += red[i];
  return v;
}
template <int kT>
DA_DEV uint32_t max_warps(const float* red) {
  if constexpr (kT == 0) {
    const int lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < (int)blockDim.x / 32 ? __float_as_uint(red[lane]) : 0);
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kT / 32; ++i) m = max(m, __float_as_uint(red[i]));
  return m;
}
template <int kT>
DA_DEV float row_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (kT != 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = add_warps<kT>(red);
  }
  return v;
}
template <int kT>
DA_DEV uint32_t row_max(uint32_t m, float* red) {
  m = __reduce_max_sync(0xffffffffu, m);
  if constexpr (kT != 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(m);
    __syncthreads();
    m = max_warps<kT>(red);
  }
  return m;
}
// Both at once for a row over several warps, behind one barrier (`red`, 64 slots, not in use).
template <int kT>
DA_DEV void row_sum_max(float& v, uint32_t& m, float* red) {
  v = warp_sum(v);
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = v;
    red[32 + (threadIdx.x >> 5)] = __uint_as_float(m);
  }
  __syncthreads();
  v = add_warps<kT>(red);
  m = max_warps<kT>(red + 32);
}

DA_DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest magnitude of three; a NaN wins.
DA_DEV float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The row's factor on v and its scale from the largest |v| and rstd (1 for the quantiser and the LayerNorm).
DA_DEV void row_scale(uint32_t amax_bits, float rstd, float& inv, float& scale) {
  const float amax = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) {
    inv = 0.f;
    scale = __uint_as_float(0x7fffffffu);
  } else if (amax <= kTiny && rstd == rstd) {  // (false for a NaN)
    inv = 0.f;
    scale = 0.f;
  } else {
    inv = __fdiv_rn(127.f, amax);
    scale = __fdiv_rn(amax * rstd, 127.f);
  }
}

DA_DEV int quant(float v, float inv) {  // NaN converts to 0
  return max(-127, min(127, __float2int_rn(__fmul_rn(v, inv))));
}

// Eight values as four pairs.
template <typename T>
struct Eight {  // as loaded
  uint4 w;
  DA_DEV void load(const void* p, int64_t off) { w = *reinterpret_cast<const uint4*>(static_cast<const T*>(p) + off); }
  DA_DEV void pairs(F2* v) const {
    v[0] = widen<T>(w.x);
    v[1] = widen<T>(w.y);
    v[2] = widen<T>(w.z);
    v[3] = widen<T>(w.w);
  }
  DA_DEV void from(const F2* v) { w = make_uint4(narrow<T>(v[0]), narrow<T>(v[1]), narrow<T>(v[2]), narrow<T>(v[3])); }
  DA_DEV void store(void* p, int64_t off) const { *reinterpret_cast<uint4*>(static_cast<T*>(p) + off) = w; }
};
template <>
struct Eight<float> {
  float4 a, b;
  DA_DEV void load(const void* p, int64_t off) {
    a = reinterpret_cast<const float4*>(static_cast<const float*>(p) + off)[0];
    b = reinterpret_cast<const float4*>(static_cast<const float*>(p) + off)[1];
  }
  DA_DEV void pairs(F2* v) const {
    v[0] = f2(a.x, a.y);
    v[1] = f2(a.z, a.w);
    v[2] = f2(b.x, b.y);
    v[3] = f2(b.z, b.w);
  }
  DA_DEV void from(const F2* v) {
    split(v[0], a.x, a.y);
    split(v[1], a.z, a.w);
    split(v[2], b.x, b.y);
    split(v[3], b.z, b.w);
  }
  DA_DEV void store(void* p, int64_t off) const {
    reinterpret_cast<float4*>(static_cast<float*>(p) + off)[0] = a;
    reinterpret_cast<float4*>(static_cast<float*>(p) + off)[1] = b;
  }
};
template <typename T>
constexpr int code_of() {
  return std::is_same<T, float>::value ? DA_F32 : std::is_same<T, __nv_bfloat16>::value ? DA_BF16 : DA_F16;
}
struct None {};

// Eight weights (or biases) from column `col` on, columns outside [0, D) as 0.  `aligned`: p is on 16 bytes; then
// fp32 comes in as the two or three aligned groups of 4 that hold the columns (eight single loads a thread, each
// warp-wide over 8 lines, set the time of shifted rows: 30001 x 1501 in 61 us, so in 45).
template <bool kShift>
DA_DEV void load_columns(const void* p, int dtype, bool aligned, int col, int D, F2* v) {
  const int skip = col & 3;  // the same for the whole row
  if (!kShift && dtype == DA_F32) {
    Eight<float> e;
    e.load(p, col);
    e.pairs(v);
  } else if (kShift && dtype == DA_F32 && aligned && col >= skip && col - skip + 12 <= D) {
    const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p) + col - skip);
    const float4 a = __ldg(src), b = __ldg(src + 1), c = __ldg(src + 2);
    const float f[12] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w};
    auto from = [&](int k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = f2(f[k + 2 * i], f[k + 2 * i + 1]);
    };
    if (skip == 0) from(0);
    else if (skip == 1) from(1);
    else if (skip == 2) from(2);
    else from(3);
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = col + i >= 0 && col + i < D ? load1(p, dtype, col + i) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
  }
}

// A warp (kT = 32) or a block (of kT threads, or any) per row, 8 * kNV elements per thread, 16 bytes an access.  kShift: dense tensors of any width D.  Their
// row r starts r D mod 8 elements after a multiple of 8, so a thread takes the groups of 8 that are aligned in
// memory; the row's first and last groups mask what belongs to its neighbours, and q, whose rows do start on 16
// bytes, goes through shared memory to be moved by the row's offset.
template <typename TX, typename TB, int kKind, int kT, int kNV, bool kShift>
__global__ void __launch_bounds__(kT == 32 ? 256 : kT ? kT : 512) norm_int8_kernel(const NormArgs p) {
  constexpr bool kBranch = !std::is_same<TB, None>::value;
  const int threads = kT ? kT : blockDim.x;  // of a row; 8 rows, a warp each, or one
  const int slots_of_row = kNV * threads + 1;      // groups of a row's window, and one more that a shifted read touches
  __shared__ float red[kT == 32 ? 1 : 64];
  extern __shared__ uint2 moved[];  // kShift
  grid_dependency_wait();
  grid_launch_dependents();
  const int in_block = kT == 32 ? threadIdx.x / 32 : 0, t = kT == 32 ? threadIdx.x % 32 : threadIdx.x;
  const int64_t row = kT == 32 ? (int64_t)blockIdx.x * 8 + in_block : blockIdx.x;
  if (row >= p.rows) return;  // a whole warp (kT = 32) or never (one row per block)
  const int off = kShift ? (int)(row * p.D % 8) : 0;  // the row's start within its first group
  const int64_t bx = kShift ? row * p.D - off : row * p.ldx, bb = kShift ? bx : row * p.ldb, bo = kShift ? bx : row * p.ldo;
  const int end = off + p.D;  // the row is [off, end) of the window
  Eight<TX> x[kNV];
  Eight<typename std::conditional<kBranch, TB, float>::type> br[kBranch ? kNV : 1];
#pragma unroll
  for (int c = 0; c < kNV; ++c) {
    const int at = (c * threads + t) * 8;
    if (at < end) {
      // (only the tensor's very last group can reach past its end)
      if (!kShift || bx + at + 8 <= p.rows * p.D) {
        x[c].load(p.x, bx + at);
        if constexpr (kBranch) br[c].load(p.branch, bb + at);
      } else {
        float f[8];
        F2 v[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = at + i < end ? load1(p.x, code_of<TX>(), bx + at + i) : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
        x[c].from(v);
        if constexpr (kBranch) {
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = at + i < end ? load1(p.branch, code_of<TB>(), bb + at + i) : 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
          br[c].from(v);
        }
      }
    }
  }
  F2 v[kNV][4];
  const F2 zero = dup(0.f);
  auto inside = [&](int at, F2* w) {  // zeroes what lies outside the row
    if (at >= off && at + 8 <= end) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      split(w[i], a, b);
      const int k = at + 2 * i;
      w[i] = f2(k >= off && k < end ? a : 0.f, k + 1 >= off && k + 1 < end ? b : 0.f);
    }
  };
#pragma unroll
  for (int c = 0; c < kNV; ++c) {
    const int at = (c * threads + t) * 8;
    if (at < end) {
      x[c].pairs(v[c]);
      if constexpr (kBranch) {
        F2 b[4];
        br[c].pairs(b);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = add2(v[c][i], b[i]);
        x[c].from(v[c]);
        if (!kShift || (at >= off && at + 8 <= end)) {
          x[c].store(p.x_out, bo + at);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float f[2];
            split(v[c][i / 2], f[0], f[1]);
            if (at + i >= off && at + i < end) store1(p.x_out, code_of<TX>(), bo + at + i, f[i % 2]);
          }
        }
        x[c].pairs(v[c]);  // as rounded to the residual's dtype
      }
      if constexpr (kShift) inside(at, v[c]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[c][i] = zero;
    }
  }
  float rstd = 1.f, squares = 0.f;
  if constexpr (kKind == kRms) {
    // v = r w needs no sum: rows over several warps are reduced once, to sum and largest value (16384 x 8192 from fp16 in
    // 79 us, with a barrier for each 99).  A warp's own sum waits for none: taken first, with its root under the weights'
    // loads, 100000 x 512 takes 31 us, else 34.
    F2 s = zero;
#pragma unroll
    for (int c = 0; c < kNV; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = fma2(v[c][i], v[c][i], s);
    float lo, hi;
    split(s, lo, hi);
    squares = lo + hi;
    if constexpr (kT == 32) rstd = 1.f / sqrtf(row_sum<kT>(squares, red) / (float)p.D + p.eps);
#pragma unroll
    for (int c = 0; c < kNV; ++c) {
      const int at = (c * threads + t) * 8;
      if (!p.weight || at >= end) continue;
      F2 w[4];
      load_columns<kShift>(p.weight, p.weight_dtype, p.aligned, at - off, p.D, w);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[c][i] = mul2(v[c][i], w[i]);
    }
  }
  if constexpr (kKind == kLayer) {
    auto total = [&](F2 s) {
      float a, b;
      split(s, a, b);
      return row_sum<kT>(a + b, red) / (float)p.D;
    };
    F2 s = zero;
#pragma unroll
    for (int c = 0; c < kNV; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) s = add2(s, v[c][i]);
    const F2 mean = dup(-total(s));
    s = zero;
#pragma unroll
    for (int c = 0; c < kNV; ++c) {
      const int at = (c * threads + t) * 8;
      if (at < end) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = add2(v[c][i], mean);
        if constexpr (kShift) inside(at, v[c]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s = fma2(v[c][i], v[c][i], s);
    }
    rstd = 1.f / sqrtf(total(s) + p.eps);
#pragma unroll
    for (int c = 0; c < kNV; ++c) {
      const int at = (c * threads + t) * 8;
      if (at >= end) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[c][i] = mul2(v[c][i], dup(rstd));
      if (p.weight) {
        F2 w[4], b[4] = {zero, zero, zero, zero};
        load_columns<kShift>(p.weight, p.weight_dtype, p.aligned, at - off, p.D, w);
        if (p.bias) load_columns<kShift>(p.bias, p.bias_dtype, p.aligned, at - off, p.D, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = fma2(v[c][i], w[i], b[i]);
      }
    }
  }
  float a = 0.f;
#pragma unroll
  for (int c = 0; c < kNV; ++c)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      split(v[c][i], lo, hi);
      a = max_abs(a, lo, hi);
    }
  float inv, scale;
  uint32_t largest = abs_bits(a);
  if constexpr (kKind == kRms && kT != 32) {
    row_sum_max<kT>(squares, largest, red);
    rstd = 1.f / sqrtf(squares / (float)p.D + p.eps);
  } else {
    largest = row_max<kT>(largest, red);
  }
  row_scale(largest, kKind == kRms ? rstd : 1.f, inv, scale);
  // |v inv| exceeds 127 by a rounding at most.  The product is rounded before the sum (a fused pair would round once,
  // and an element in 1e5 would differ from the other variants' rint(v inv)).
  auto whole = [&](F2 x) {
    float lo, hi;
    split(x, lo, hi);
    return f2(__fadd_rn(__fmul_rn(lo, inv), kRoundAt), __fadd_rn(__fmul_rn(hi, inv), kRoundAt));
  };
  auto bytes = [&](F2 lo, F2 hi) { return low_bytes(whole(lo), whole(hi)); };
  uint2* slots = moved + in_block * slots_of_row;
#pragma unroll
  for (int c = 0; c < kNV; ++c) {
    const int at = (c * threads + t) * 8;
    if (at >= end) continue;
    const uint2 o = make_uint2(bytes(v[c][0], v[c][1]), bytes(v[c][2], v[c][3]));
    if constexpr (kShift) slots[c * threads + t] = o;
    else *reinterpret_cast<uint2*>(p.q + row * p.ldq + at) = o;
  }
  if constexpr (kShift) {
    if constexpr (kT == 32) __syncwarp();
    else __syncthreads();
#pragma unroll
    for (int c = 0; c < kNV; ++c) {
      const int col = (c * threads + t) * 8;  // bytes col .. + 8 of the row are off further on in the window
      if (col >= p.D) continue;
      const uint2 lo = slots[c * threads + t], hi = slots[c * threads + t + 1];
      const uint32_t w[4] = {lo.x, lo.y, hi.x, hi.y};
      const bool second = off >= 4;
      const uint32_t w0 = second ? w[1] : w[0], w1 = second ? w[2] : w[1], w2 = second ? w[3] : w[2];
      // (past the row's end these are bytes of no meaning, in the padding of q's row)
      *reinterpret_cast<uint2*>(p.q + row * p.ldq + col) =
          make_uint2(__funnelshift_r(w0, w1, off % 4 * 8), __funnelshift_r(w1, w2, off % 4 * 8));
    }
  }
  if (t == 0) p.scale[row] = scale;
}

// Any strides, alignments and mixtures of dtypes: one block per row, an element a load (each thread reads back only
// what it wrote itself); rows wider than the register variants hold come here too, and 16-bit residuals with a branch of
// another type.  Three passes of single elements: 16384 x 4096, bf16 residual and fp16 branch, in 357 us (both bf16: 72),
// 4096 x 20000 from bf16 in 223 us (16384 columns, in registers: 53).
template <int kT>
__global__ void __launch_bounds__(kT) norm_int8_any_kernel(const NormArgs p) {
  __shared__ float red[32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t row = blockIdx.x;
  const void* src = p.branch ? p.x_out : p.x;
  const int64_t base = row * (p.branch ? p.ldo : p.ldx);
  float s = 0.f;
  for (int col = threadIdx.x; col < p.D; col += kT) {
    float r = load1(p.x, p.x_dtype, row * p.ldx + col);
    if (p.branch) {
      r = round_to(r + load1(p.branch, p.branch_dtype, row * p.ldb + col), p.x_dtype);
      store1(p.x_out, p.x_dtype, base + col, r);
    }
    s += p.kind == kLayer ? r : r * r;
  }
  float mean = 0.f, rstd = 1.f;
  if (p.kind != kQuantize) {
    s = row_sum<0>(s, red) / (float)p.D;
    if (p.kind == kLayer) {
      mean = s;
      s = 0.f;
      for (int col = threadIdx.x; col < p.D; col += kT) {
        const float d = load1(src, p.x_dtype, base + col) - mean;
        s = fmaf(d, d, s);
      }
      s = row_sum<0>(s, red) / (float)p.D;
    }
    rstd = 1.f / sqrtf(s + p.eps);
  }
  auto value = [&](int col) {
    float r = load1(src, p.x_dtype, base + col);
    const float w = p.weight ? load1(p.weight, p.weight_dtype, col) : 1.f;
    if (p.kind == kRms) return p.weight ? r * w : r;
    if (p.kind == kLayer) {
      r = (r - mean) * rstd;
      if (p.weight) r = fmaf(r, w, p.bias ? load1(p.bias, p.bias_dtype, col) : 0.f);
    }
    return r;
  };
  uint32_t a = 0;
  for (int col = threadIdx.x; col < p.D; col += kT) a = max(a, abs_bits(value(col)));
  a = row_max<0>(a, red);
  float inv, scale;
  row_scale(a, p.kind == kRms ? rstd : 1.f, inv, scale);
  for (int col = threadIdx.x; col < p.D; col += kT) p.q[row * p.ldq + col] = (int8_t)quant(value(col), inv);
  if (threadIdx.x == 0) p.scale[row] = scale;
}

// out = q * scale, one rounding to the output dtype.  A thread takes 8 outputs: of a row that starts on 16 bytes, or
// (kShift) 8 aligned ones of a dense tensor of any width, whose bytes of q are then two loads and a shift; else
// (kVec false) one by one.  Bound: HBM; 262144 x 512 to bf16 in 67 us (3 bytes an element, 6.0 TB/s).
template <typename T, bool kVec, bool kShift>
__global__ void __launch_bounds__(256) dequant_int8_kernel(const int8_t* q, int64_t ldq, const float* scale,
                                                           int64_t row0, int64_t items, Div31 per_row, int D,
                                                           void* out, int64_t ldo) {
  constexpr int kItems = 4;  // a thread's, all loaded before the first is used
  grid_dependency_wait();
  grid_launch_dependents();
  uint2 w[kItems];
  float s[kItems];
  int64_t row[kItems];
  int col[kItems];  // of the first output; negative in a shifted row's first group
  auto live = [&](int k) { return col[k] < D; };
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = ((int64_t)blockIdx.x * kItems + k) * 256 + threadIdx.x;
    const uint32_t r = per_row.div((uint32_t)i);
    row[k] = row0 + r;
    const int at = (int)((uint32_t)i - r * per_row.d) * 8;
    const int off = kShift ? (int)(row[k] * D % 8) : 0;
    col[k] = i < items ? at - off : D;
    if (!live(k)) continue;
    s[k] = scale[row[k]];
    const int8_t* src = q + row[k] * ldq + at;
    if constexpr (!kVec) {
      uint32_t b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = at + e < D ? (uint8_t)src[e] : 0;
      w[k] = make_uint2(b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24, b[4] | b[5] << 8 | b[6] << 16 | b[7] << 24);
    } else if constexpr (!kShift) {
      w[k] = *reinterpret_cast<const uint2*>(src);
    } else {  // bytes at - off .. + 8: of the aligned eight before, and of those from `at` on
      const uint2 zero = make_uint2(0, 0);
      const uint2 lo = off && at > 0 ? *reinterpret_cast<const uint2*>(src - 8) : zero;
      const uint2 hi = at < D ? *reinterpret_cast<const uint2*>(src) : zero;
      const uint32_t v[4] = {lo.x, lo.y, hi.x, hi.y};
      const int skip = 8 - off;  // 1 to 8 bytes of the sixteen
      const uint32_t w0 = skip >= 4 ? v[1] : v[0], w1 = skip >= 4 ? v[2] : v[1], w2 = skip >= 4 ? v[3] : v[2];
      w[k] = skip == 8 ? hi : make_uint2(__funnelshift_r(w0, w1, skip % 4 * 8), __funnelshift_r(w1, w2, skip % 4 * 8));
    }
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    if (!live(k)) continue;
    F2 v[4];
    signed_bytes(w[k].x, v[0], v[1]);
    signed_bytes(w[k].y, v[2], v[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = mul2(v[e], dup(s[k]));
    const int64_t base = row[k] * ldo + col[k];
    if (kVec && col[k] >= 0 && col[k] + 8 <= D) {
      Eight<T> o;
      o.from(v);
      o.store(out, base);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float f[2];
        split(v[e / 2], f[0], f[1]);
        if (col[k] + e >= 0 && col[k] + e < D) store1(out, code_of<T>(), base + e, f[e % 2]);
      }
    }
  }
}

template <typename T>
int launch_dequant(const int8_t* q, int64_t ldq, const float* scale, int64_t rows, int64_t D, void* out, int64_t ldo,
                   cudaStream_t st) {
  const bool q8 = ldq % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const bool rows16 = q8 && D % 8 == 0 && vec8_ok(out, code_of<T>(), ldo);
  const bool shift = !rows16 && q8 && ldo == D && vec8_ok(out, code_of<T>(), 8) && ldq >= (D + 7) / 8 * 8;
  const Div31 per_row((uint32_t)((D + (shift ? 7 : 0) + 7) / 8));
  const int64_t slab = Div31::kMax / per_row.d;  // rows whose items stay below 2^31
  auto kern = rows16 ? dequant_int8_kernel<T, true, false>
                     : shift ? dequant_int8_kernel<T, true, true> : dequant_int8_kernel<T, false, false>;
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t n = (rows - r0 < slab ? rows - r0 : slab) * per_row.d;
    if (int rc = launch_kernel(kern, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, st, false, q, ldq, scale, r0, n, per_row,
                               (int)D, out, ldo))
      return rc;
  }
  return DA_OK;
}

template <typename TX, typename TB, int kKind, bool kShift, int kT, int kNV>
int launch_t(const NormArgs& p, int threads, cudaStream_t st) {
  const int64_t blocks = kT == 32 ? (p.rows + 7) / 8 : p.rows;
  if (blocks > 0x7fffffffLL) return DA_ERR_SHAPE;
  const int smem = !kShift ? 0 : kT == 32 ? 8 * (kNV * 32 + 1) * 8 : (kNV * threads + 1) * 8;
  return launch_kernel(norm_int8_kernel<TX, TB, kKind, kT, kNV, kShift>, dim3((unsigned)blocks), dim3(threads), smem, st,
                       false, p);
}
// As few threads a row as hold it with 32 values each: more loads in flight a thread and fewer warps at a barrier
// (a block of 256 for every row above 1024 columns: 30001 x 1501 in 82 us, against 61 us so), and none that idle
// (in powers of two, 16384 x 8191 with an fp32 residual took 403 us, so 255).  A size that the compiler does not know
// costs 5 to 10 % (16384 x 8192 from fp16 in 80 us, else 88), so the common ones are known.
template <typename TX, typename TB, int kKind, bool kShift>
int launch_shift(const NormArgs& p, cudaStream_t st) {
  const int window = p.D + (kShift ? 7 : 0);
  if (window <= 256) return launch_t<TX, TB, kKind, kShift, 32, 1>(p, 256, st);
  if (window <= 512) return launch_t<TX, TB, kKind, kShift, 32, 2>(p, 256, st);
  if (window <= 768) return launch_t<TX, TB, kKind, kShift, 32, 3>(p, 256, st);
  if (window <= 1024) return launch_t<TX, TB, kKind, kShift, 32, 4>(p, 256, st);
  const int threads = (window + 1023) / 1024 * 32;
  if (threads == 64) return launch_t<TX, TB, kKind, kShift, 64, 4>(p, threads, st);
  if (threads == 128) return launch_t<TX, TB, kKind, kShift, 128, 4>(p, threads, st);
  if (threads == 256) return launch_t<TX, TB, kKind, kShift, 256, 4>(p, threads, st);
  return launch_t<TX, TB, kKind, kShift, 0, 4>(p, threads, st);
}
template <typename TX, typename TB>
int launch_types(const NormArgs& p, bool shift, cudaStream_t st) {
  if constexpr (std::is_same<TB, None>::value)
    if (p.kind == kQuantize)
      return shift ? launch_shift<TX, TB, kQuantize, true>(p, st) : launch_shift<TX, TB, kQuantize, false>(p, st);
  if (p.kind == kRms) return shift ? launch_shift<TX, TB, kRms, true>(p, st) : launch_shift<TX, TB, kRms, false>(p, st);
  return shift ? launch_shift<TX, TB, kLayer, true>(p, st) : launch_shift<TX, TB, kLayer, false>(p, st);
}
int launch_any(const NormArgs& p, cudaStream_t st) {
  if (p.rows > 0x7fffffffLL) return DA_ERR_SHAPE;
  const dim3 grid((unsigned)p.rows);
  if (p.D <= 512) return launch_kernel(norm_int8_any_kernel<64>, grid, dim3(64), 0, st, false, p);
  if (p.D <= 8192) return launch_kernel(norm_int8_any_kernel<256>, grid, dim3(256), 0, st, false, p);
  return launch_kernel(norm_int8_any_kernel<1024>, grid, dim3(1024), 0, st, false, p);
}

bool float_dtype(int d) { return d == DA_F16 || d == DA_BF16 || d == DA_F32; }

}  // namespace
}  // namespace da

extern "C" int da_norm_int8(const void* x, int x_dtype, int64_t ldx, const void* branch, int branch_dtype, int64_t ldb,
                            const void* weight, int weight_dtype, const void* bias, int bias_dtype, int kind,
                            int64_t rows, int64_t D, float eps, void* x_out, int64_t ldo, int8_t* q, int64_t ldq,
                            float* scale, void* stream) {
  using namespace da;
  if (!x || !q || !scale || (branch && !x_out)) return DA_ERR_NULL;
  if (kind < kQuantize || kind > kLayer) return DA_ERR_UNSUPPORTED;
  if (kind == kQuantize && (branch || weight || bias)) return DA_ERR_UNSUPPORTED;
  if (bias && (kind != kLayer || !weight)) return DA_ERR_UNSUPPORTED;
  if (rows <= 0 || D <= 0 || D > 0x7ffffff0LL || ldq < D || ldx < 0 || ldb < 0 || (branch && ldo < D))
    return DA_ERR_SHAPE;
  if (!float_dtype(x_dtype) || (branch && !float_dtype(branch_dtype)) || (weight && !float_dtype(weight_dtype)) ||
      (bias && !float_dtype(bias_dtype)))
    return DA_ERR_DTYPE;
  if (int rc = bind_device(x)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const NormArgs p{x,    branch, weight,  bias,         x_out,        q,          scale, ldx,    ldb, ldo,
                   ldq,  rows,   x_dtype, branch_dtype, weight_dtype, bias_dtype, kind,  (int)D, eps,
                   (reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(bias)) % 16 == 0};
  // 16-byte groups of 8 elements: rows that all start on one, or dense tensors of any width
  const bool based = vec8_ok(x, x_dtype, 8) && (!branch || (vec8_ok(branch, branch_dtype, 8) && vec8_ok(x_out, x_dtype, 8))) &&
                     ldq % 8 == 0 && ldq >= (D + 7) / 8 * 8 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const bool rows16 = D % 8 == 0 && vec8_ok(x, x_dtype, ldx) &&
                      (!branch || (vec8_ok(branch, branch_dtype, ldb) && vec8_ok(x_out, x_dtype, ldo))) &&
                      (!weight || vec8_ok(weight, weight_dtype, 8)) && (!bias || vec8_ok(bias, bias_dtype, 8));
  const bool dense = ldx == D && (!branch || (ldb == D && ldo == D));
  const bool shift = !rows16;
  if (!based || !(rows16 || dense) || D + (shift ? 7 : 0) > 16384) return launch_any(p, st);
  if (x_dtype == DA_F32) {
    if (!branch) return launch_types<float, None>(p, shift, st);
    if (branch_dtype == DA_F32) return launch_types<float, float>(p, shift, st);
    if (branch_dtype == DA_BF16) return launch_types<float, __nv_bfloat16>(p, shift, st);
    return launch_types<float, __half>(p, shift, st);
  }
  if (branch && branch_dtype != x_dtype) return launch_any(p, st);
  if (x_dtype == DA_BF16)
    return branch ? launch_types<__nv_bfloat16, __nv_bfloat16>(p, shift, st) : launch_types<__nv_bfloat16, None>(p, shift, st);
  return branch ? launch_types<__half, __half>(p, shift, st) : launch_types<__half, None>(p, shift, st);
}

extern "C" int da_dequant_int8(const int8_t* q, int64_t ldq, const float* scale, int64_t rows, int64_t D, void* out,
                               int out_dtype, int64_t ldo, void* stream) {
  using namespace da;
  if (!q || !scale || !out) return DA_ERR_NULL;
  if (rows <= 0 || D <= 0 || D > 0x7ffffff0LL || ldq < 0 || ldo < D) return DA_ERR_SHAPE;
  if (!float_dtype(out_dtype)) return DA_ERR_DTYPE;
  if (int rc = bind_device(q)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == DA_F32) return launch_dequant<float>(q, ldq, scale, rows, D, out, ldo, st);
  if (out_dtype == DA_BF16) return launch_dequant<__nv_bfloat16>(q, ldq, scale, rows, D, out, ldo, st);
  return launch_dequant<__half>(q, ldq, scale, rows, D, out, ldo, st);
}

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
// holds a NaN or an infinity gets a scale of NaN or infinity, so that it never decodes to plausible
// numbers: |v| is compared as an unsigned integer, which orders NaN above infinity above every number.
//
// Bound: HBM.  One pass; a row stays in registers between its reductions (one warp per row up to 1024
// columns, one block per row up to 32768; wider rows are read again, mostly from L2).
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
};

// Sum and largest bit pattern over the kT threads of a row (kT a multiple of 32; a block-wide row uses
// `red`, one slot per warp).
template <int kT>
DA_DEV float row_sum(float v, float* red) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (kT > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < kT / 32; ++i) v += red[i];  // same order in every thread
  }
  return v;
}
template <int kT>
DA_DEV uint32_t row_max(uint32_t v, float* red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if constexpr (kT > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = __uint_as_float(v);
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < kT / 32; ++i) v = max(v, __float_as_uint(red[i]));
  }
  return v;
}

DA_DEV uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The row's factor on v and its scale from the largest |v| and rstd (1 for the quantiser and the LayerNorm).
DA_DEV void row_scale(uint32_t amax_bits, float rstd, float& inv, float& scale) {
  const float amax = __uint_as_float(amax_bits);
  if (amax <= kTiny && rstd == rstd) {  // (false for NaN)
    inv = 0.f;
    scale = 0.f;
  } else {
    inv = __fdiv_rn(127.f, amax);
    scale = __fdiv_rn(amax * rstd, 127.f);
  }
}

DA_DEV int quant(float v, float inv) {  // NaN converts to 0
  return max(-127, min(127, __float2int_rn(v * inv)));
}

// kT threads per row, 8 * kNV elements per thread; kVec: 8 consecutive columns per access (16-byte aligned
// rows, D a multiple of 8), else single elements kT columns apart.
template <int kT, int kNV, bool kVec>
__global__ void __launch_bounds__(kT > 256 ? kT : 256) norm_int8_kernel(const NormArgs p) {
  constexpr int kBlock = kT > 256 ? kT : 256;
  __shared__ float red[kBlock / 32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int t = threadIdx.x % kT;
  const int64_t row = (int64_t)blockIdx.x * (kBlock / kT) + threadIdx.x / kT;
  if (row >= p.rows) return;  // a whole warp (kT = 32) or never (one row per block)
  float v[kNV][8];
#pragma unroll
  for (int c = 0; c < kNV; ++c) {
    if constexpr (kVec) {
      const int col = (c * kT + t) * 8;
      if (col < p.D) {
        load8(p.x, p.x_dtype, row * p.ldx + col, v[c]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = (c * 8 + e) * kT + t;
        v[c][e] = col < p.D ? load1(p.x, p.x_dtype, row * p.ldx + col) : 0.f;
      }
    }
  }
  if (p.branch) {
#pragma unroll
    for (int c = 0; c < kNV; ++c) {
      if constexpr (kVec) {
        const int col = (c * kT + t) * 8;
        if (col < p.D) {
          float b[8];
          load8(p.branch, p.branch_dtype, row * p.ldb + col, b);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[c][e] = round_to(v[c][e] + b[e], p.x_dtype);
          store8(p.x_out, p.x_dtype, row * p.ldo + col, v[c]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int col = (c * 8 + e) * kT + t;
          if (col < p.D) {
            v[c][e] = round_to(v[c][e] + load1(p.branch, p.branch_dtype, row * p.ldb + col), p.x_dtype);
            store1(p.x_out, p.x_dtype, row * p.ldo + col, v[c][e]);
          }
        }
      }
    }
  }
  float rstd = 1.f;
  if (p.kind != kQuantize) {
    float s = 0.f, mean = 0.f;
    if (p.kind == kLayer) {
#pragma unroll
      for (int c = 0; c < kNV; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[c][e];
      mean = row_sum<kT>(s, red) / (float)p.D;
      s = 0.f;
    }
#pragma unroll
    for (int c = 0; c < kNV; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = kVec ? (c * kT + t) * 8 + e : (c * 8 + e) * kT + t;
        const float d = col < p.D ? v[c][e] - mean : 0.f;
        s = fmaf(d, d, s);
      }
    rstd = 1.f / sqrtf(row_sum<kT>(s, red) / (float)p.D + p.eps);
#pragma unroll
    for (int c = 0; c < kNV; ++c) {
      float w[8], b[8];
      if constexpr (kVec) {
        const int col = (c * kT + t) * 8;
        if (col < p.D) {
          if (p.weight) load8(p.weight, p.weight_dtype, col, w);
          if (p.bias) load8(p.bias, p.bias_dtype, col, b);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int col = (c * 8 + e) * kT + t;
          if (col < p.D) {
            if (p.weight) w[e] = load1(p.weight, p.weight_dtype, col);
            if (p.bias) b[e] = load1(p.bias, p.bias_dtype, col);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = kVec ? (c * kT + t) * 8 + e : (c * 8 + e) * kT + t;
        if (col < p.D) {
          if (p.kind == kRms) {
            if (p.weight) v[c][e] *= w[e];
          } else {
            v[c][e] = (v[c][e] - mean) * rstd;
            if (p.weight) v[c][e] = fmaf(v[c][e], w[e], p.bias ? b[e] : 0.f);
          }
        }
      }
    }
  }
  uint32_t a = 0;
#pragma unroll
  for (int c = 0; c < kNV; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, abs_bits(v[c][e]));  // columns past D hold 0
  a = row_max<kT>(a, red);
  float inv, scale;
  row_scale(a, p.kind == kRms ? rstd : 1.f, inv, scale);
#pragma unroll
  for (int c = 0; c < kNV; ++c) {
    if constexpr (kVec) {
      const int col = (c * kT + t) * 8;
      if (col < p.D) {
        int o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = quant(v[c][e], inv);
        *reinterpret_cast<uint2*>(p.q + row * p.ldq + col) = pack_s8x8(o);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = (c * 8 + e) * kT + t;
        if (col < p.D) p.q[row * p.ldq + col] = (int8_t)quant(v[c][e], inv);
      }
    }
  }
  if (t == 0) p.scale[row] = scale;
}

// Rows wider than the register variants hold: one block per row, the row read again for every reduction
// (each thread reads back only what it wrote itself).
__global__ void __launch_bounds__(1024) norm_int8_wide_kernel(const NormArgs p) {
  constexpr int kT = 1024;
  __shared__ float red[kT / 32];
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
    s = row_sum<kT>(s, red) / (float)p.D;
    if (p.kind == kLayer) {
      mean = s;
      s = 0.f;
      for (int col = threadIdx.x; col < p.D; col += kT) {
        const float d = load1(src, p.x_dtype, base + col) - mean;
        s = fmaf(d, d, s);
      }
      s = row_sum<kT>(s, red) / (float)p.D;
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
  a = row_max<kT>(a, red);
  float inv, scale;
  row_scale(a, p.kind == kRms ? rstd : 1.f, inv, scale);
  for (int col = threadIdx.x; col < p.D; col += kT) p.q[row * p.ldq + col] = (int8_t)quant(value(col), inv);
  if (threadIdx.x == 0) p.scale[row] = scale;
}

// out = q * scale, one rounding to the output dtype; a thread takes 8 columns of one row.
template <bool kVec>
__global__ void __launch_bounds__(256) dequant_int8_kernel(const int8_t* q, int64_t ldq, const float* scale,
                                                           int64_t row0, int64_t items, Div31 per_row, int D,
                                                           void* out, int out_dtype, int64_t ldo) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= items) return;
  const uint32_t r = per_row.div((uint32_t)i);
  const int64_t row = row0 + r;
  const int col = (int)((uint32_t)i - r * per_row.d) * 8;
  const float s = scale[row];
  if constexpr (kVec) {
    float v[8];
    unpack_s8x8(*reinterpret_cast<const uint2*>(q + row * ldq + col), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= s;
    store8(out, out_dtype, row * ldo + col, v);
  } else {
    for (int e = 0; e < 8 && col + e < D; ++e)
      store1(out, out_dtype, row * ldo + col + e, (float)q[row * ldq + col + e] * s);
  }
}

template <int kT, bool kVec>
int launch_norm(const NormArgs& p, cudaStream_t st) {
  constexpr int kBlock = kT > 256 ? kT : 256;
  const int64_t blocks = (p.rows + kBlock / kT - 1) / (kBlock / kT);
  if (blocks > 0x7fffffffLL) return DA_ERR_SHAPE;
  const dim3 grid((unsigned)blocks), block(kBlock);
  const int nv = (p.D + kT * 8 - 1) / (kT * 8);
  if (kT == 1024 || nv > 3) return launch_kernel(norm_int8_kernel<kT, 4, kVec>, grid, block, 0, st, false, p);
  if (nv == 3) return launch_kernel(norm_int8_kernel<kT, 3, kVec>, grid, block, 0, st, false, p);
  if (nv == 2) return launch_kernel(norm_int8_kernel<kT, 2, kVec>, grid, block, 0, st, false, p);
  return launch_kernel(norm_int8_kernel<kT, 1, kVec>, grid, block, 0, st, false, p);
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
                   ldq,  rows,   x_dtype, branch_dtype, weight_dtype, bias_dtype, kind,  (int)D, eps};
  const bool vec = D % 8 == 0 && vec8_ok(x, x_dtype, ldx) && (!branch || vec8_ok(branch, branch_dtype, ldb)) &&
                   (!branch || vec8_ok(x_out, x_dtype, ldo)) && (!weight || vec8_ok(weight, weight_dtype, 8)) &&
                   (!bias || vec8_ok(bias, bias_dtype, 8)) && ldq % 8 == 0 &&
                   reinterpret_cast<uintptr_t>(q) % 8 == 0;
  if (D <= 1024) return vec ? launch_norm<32, true>(p, st) : launch_norm<32, false>(p, st);
  if (D <= 8192) return vec ? launch_norm<256, true>(p, st) : launch_norm<256, false>(p, st);
  if (D <= 32768) return vec ? launch_norm<1024, true>(p, st) : launch_norm<1024, false>(p, st);
  if (rows > 0x7fffffffLL) return DA_ERR_SHAPE;
  return launch_kernel(norm_int8_wide_kernel, dim3((unsigned)rows), dim3(1024), 0, st, false, p);
}

extern "C" int da_dequant_int8(const int8_t* q, int64_t ldq, const float* scale, int64_t rows, int64_t D, void* out,
                               int out_dtype, int64_t ldo, void* stream) {
  using namespace da;
  if (!q || !scale || !out) return DA_ERR_NULL;
  if (rows <= 0 || D <= 0 || D > 0x7ffffff0LL || ldq < 0 || ldo < D) return DA_ERR_SHAPE;
  if (!float_dtype(out_dtype)) return DA_ERR_DTYPE;
  if (int rc = bind_device(q)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool vec = D % 8 == 0 && ldq % 8 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0 && vec8_ok(out, out_dtype, ldo);
  const Div31 per_row((uint32_t)((D + 7) / 8));
  const int64_t slab = Div31::kMax / per_row.d;  // rows whose items stay below 2^31
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t n = (rows - r0 < slab ? rows - r0 : slab) * per_row.d;
    const dim3 grid((unsigned)((n + 255) / 256));
    const int rc = vec ? launch_kernel(dequant_int8_kernel<true>, grid, dim3(256), 0, st, false, q, ldq, scale, r0, n,
                                       per_row, (int)D, out, out_dtype, ldo)
                       : launch_kernel(dequant_int8_kernel<false>, grid, dim3(256), 0, st, false, q, ldq, scale, r0, n,
                                       per_row, (int)D, out, out_dtype, ldo);
    if (rc) return rc;
  }
  return DA_OK;
}

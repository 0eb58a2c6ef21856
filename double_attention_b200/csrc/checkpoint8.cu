// Activation checkpoints in 8 bits: an activation that the backward pass needs again is kept as int8 in
// blocks of 32 columns that share a power-of-two scale.
//
//   a = max |x| over the block,  e = the smallest integer with a <= 127 * 2^e,  q = rint(x 2^-e)
// The scale is a power of two so that the value a checkpoint stands for, q 2^e, is exact in fp16 and bf16:
// the backward's products read exactly what was kept.  e stays in what the activation's dtype holds ([-24, 9]
// for fp16, [-126, 121] otherwise; larger values saturate at 127 * 2^e).  A block that holds a NaN or an
// infinity gets the code -128 for e and decodes to NaN, so that a bad activation still shows in the gradients.
//
//   GELU forward:  h = gelu(z), and z kept.
//   GELU backward from the kept z:  dz = dh gelu'(z),  h = gelu(z) once more, for the next layer's weight gradient.
//
// Layout: q [rows, ceil(D / 32) * 32] int8, columns past D zero; e [rows, ceil(D / 32)] int8.
// Bound: HBM (5 bytes an element forward, 7 backward); a thread takes 8 columns, so the 4 threads of a block
// find its maximum with two shuffles and no row-wide reduction is needed, whatever the width.
#include "common.cuh"
#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace {

constexpr int kNotFinite = -128;
constexpr int kItems = 4;  // groups of 8 columns per thread

struct CkptArgs {
  const void* x;  // z or dh
  void* h;
  void* dz;
  int8_t* q;
  int8_t* e;
  int64_t ldx, ldh, lddz, row0;
  int64_t items;  // groups of 8 columns in this launch (< 2^31)
  Div31 per_row;  // groups of 8 columns in a row of q (a multiple of 4)
  int D, dtype, gelu, e_min, e_max;
};

DA_DEV void load_row8(const void* p, int dtype, int64_t base, int col, int D, bool vec, float* v) {
  if (vec && col + 8 <= D) {
    load8(p, dtype, base + col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < D ? load1(p, dtype, base + col + i) : 0.f;
  }
}
DA_DEV void store_row8(void* p, int dtype, int64_t base, int col, int D, bool vec, const float* v) {
  if (vec && col + 8 <= D) {
    store8(p, dtype, base + col, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < D) store1(p, dtype, base + col + i, v[i]);
  }
}

// 2^e, e in [-126, 127].
DA_DEV float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__global__ void __launch_bounds__(256) checkpoint8_kernel(const CkptArgs p, bool vec_x, bool vec_h) {
  grid_dependency_wait();
  grid_launch_dependents();
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = ((int64_t)blockIdx.x * kItems + k) * 256 + threadIdx.x;
    // the 4 threads of a block of columns stay or leave together (items is a multiple of 4)
    const unsigned mask = __ballot_sync(0xffffffffu, i < p.items);
    if (i >= p.items) continue;
    const uint32_t r = p.per_row.div((uint32_t)i), c = (uint32_t)i - r * p.per_row.d;
    const int64_t row = p.row0 + r;
    const int col = (int)c * 8;
    float v[8];
    load_row8(p.x, p.dtype, row * p.ldx, col, p.D, vec_x, v);
    uint32_t a = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = max(a, __float_as_uint(v[j]) & 0x7fffffffu);
    a = max(a, __shfl_xor_sync(mask, a, 1));
    a = max(a, __shfl_xor_sync(mask, a, 2));
    // a = m 2^E with 1 <= m < 2: 127 * 2^(E - 6) covers it if m <= 1.984375 (mantissa bits 0x7e0000)
    int e = (int)(a >> 23) - 127 - 6 + ((a & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    const bool finite = a < 0x7f800000u;
    e = max(p.e_min, min(p.e_max, e));
    const float inv = pow2i(-e);
    int o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = finite ? max(-127, min(127, __float2int_rn(v[j] * inv))) : 0;
    *reinterpret_cast<uint2*>(p.q + (row * p.per_row.d + c) * 8) = pack_s8x8(o);
    if ((c & 3) == 0) p.e[(row * p.per_row.d + c) >> 2] = (int8_t)(finite ? e : kNotFinite);
    if (p.gelu) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) gelu2(v[j], v[j + 1]);
      store_row8(p.h, p.dtype, row * p.ldh, col, p.D, vec_h, v);
    }
  }
}

// A kept group's 8 values.
DA_DEV void restore8(const CkptArgs& p, int64_t group, float* v) {
  unpack_s8x8(*reinterpret_cast<const uint2*>(p.q + group * 8), v);
  const int e = p.e[group >> 2];
  const float unit = e == kNotFinite ? __uint_as_float(0x7fffffffu) : pow2i(e);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= unit;
}

__global__ void __launch_bounds__(256) checkpoint8_restore_kernel(const CkptArgs p, bool vec_h) {
  grid_dependency_wait();
  grid_launch_dependents();
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = ((int64_t)blockIdx.x * kItems + k) * 256 + threadIdx.x;
    if (i >= p.items) continue;
    const uint32_t r = p.per_row.div((uint32_t)i), c = (uint32_t)i - r * p.per_row.d;
    const int64_t row = p.row0 + r;
    float v[8];
    restore8(p, row * p.per_row.d + c, v);
    store_row8(p.h, p.dtype, row * p.ldh, (int)c * 8, p.D, vec_h, v);
  }
}

__global__ void __launch_bounds__(256) checkpoint8_gelu_bwd_kernel(const CkptArgs p, bool vec_x, bool vec_h,
                                                                   bool vec_dz) {
  grid_dependency_wait();
  grid_launch_dependents();
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = ((int64_t)blockIdx.x * kItems + k) * 256 + threadIdx.x;
    if (i >= p.items) continue;
    const uint32_t r = p.per_row.div((uint32_t)i), c = (uint32_t)i - r * p.per_row.d;
    const int64_t row = p.row0 + r;
    const int col = (int)c * 8;
    if (col >= p.D) continue;
    float z[8], d[8];
    load_row8(p.x, p.dtype, row * p.ldx, col, p.D, vec_x, d);
    restore8(p, row * p.per_row.d + c, z);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float s0, s1;
      gelu_grad2(z[j], z[j + 1], s0, s1);
      d[j] *= s0;
      d[j + 1] *= s1;
    }
    store_row8(p.dz, p.dtype, row * p.lddz, col, p.D, vec_dz, d);
    if (p.h) store_row8(p.h, p.dtype, row * p.ldh, col, p.D, vec_h, z);
  }
}

// Runs `launch(args, grid)` over slabs of rows whose item count stays below 2^31.
template <typename F>
int over_rows(CkptArgs p, int64_t rows, F&& launch) {
  const int64_t slab = Div31::kMax / p.per_row.d;
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    p.row0 = r0;
    p.items = (rows - r0 < slab ? rows - r0 : slab) * (int64_t)p.per_row.d;
    const dim3 grid((unsigned)((p.items + 256 * kItems - 1) / (256 * kItems)));
    if (int rc = launch(p, grid)) return rc;
  }
  return DA_OK;
}

CkptArgs make_args(int64_t D, int dtype) {
  CkptArgs p{nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, Div31((uint32_t)((D + 31) / 32 * 4)),
             (int)D, dtype, 0, -126, 121};
  if (dtype == DA_F16) {
    p.e_min = -24;
    p.e_max = 9;
  }
  return p;
}

bool bad_shape(int64_t rows, int64_t D) { return rows <= 0 || D <= 0 || D > 0x7fffff00LL; }
bool half_dtype(int d) { return d == DA_F16 || d == DA_BF16; }

}  // namespace
}  // namespace da

extern "C" int da_checkpoint8(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t D, int gelu, void* h,
                              int64_t ldh, int8_t* q, int8_t* e, void* stream) {
  using namespace da;
  if (!x || !q || !e || (gelu && !h)) return DA_ERR_NULL;
  if (bad_shape(rows, D) || ldx < 0 || (gelu && ldh < D)) return DA_ERR_SHAPE;
  if (!half_dtype(dtype)) return DA_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(q) % 16) return DA_ERR_ALIGN;
  if (int rc = bind_device(x)) return rc;
  CkptArgs p = make_args(D, dtype);
  p.x = x;
  p.ldx = ldx;
  p.h = h;
  p.ldh = ldh;
  p.q = q;
  p.e = e;
  p.gelu = gelu;
  const bool vx = vec8_ok(x, dtype, ldx), vh = vec8_ok(h, dtype, ldh);
  return over_rows(p, rows, [&](const CkptArgs& a, dim3 grid) {
    return launch_kernel(checkpoint8_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), false, a, vx, vh);
  });
}

extern "C" int da_checkpoint8_restore(const int8_t* q, const int8_t* e, int64_t rows, int64_t D, void* out, int dtype,
                                      int64_t ldo, void* stream) {
  using namespace da;
  if (!q || !e || !out) return DA_ERR_NULL;
  if (bad_shape(rows, D) || ldo < D) return DA_ERR_SHAPE;
  if (!half_dtype(dtype) && dtype != DA_F32) return DA_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(q) % 16) return DA_ERR_ALIGN;
  if (int rc = bind_device(q)) return rc;
  CkptArgs p = make_args(D, dtype);
  p.q = const_cast<int8_t*>(q);
  p.e = const_cast<int8_t*>(e);
  p.h = out;
  p.ldh = ldo;
  const bool vo = vec8_ok(out, dtype, ldo);
  return over_rows(p, rows, [&](const CkptArgs& a, dim3 grid) {
    return launch_kernel(checkpoint8_restore_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), false, a,
                         vo);
  });
}

extern "C" int da_checkpoint8_gelu_bwd(const void* dh, int dtype, int64_t lddh, const int8_t* q, const int8_t* e,
                                       int64_t rows, int64_t D, void* dz, int64_t lddz, void* h, int64_t ldh,
                                       void* stream) {
  using namespace da;
  if (!dh || !q || !e || !dz) return DA_ERR_NULL;
  if (bad_shape(rows, D) || lddh < 0 || lddz < D || (h && ldh < D)) return DA_ERR_SHAPE;
  if (!half_dtype(dtype)) return DA_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(q) % 16) return DA_ERR_ALIGN;
  if (int rc = bind_device(dh)) return rc;
  CkptArgs p = make_args(D, dtype);
  p.x = dh;
  p.ldx = lddh;
  p.q = const_cast<int8_t*>(q);
  p.e = const_cast<int8_t*>(e);
  p.dz = dz;
  p.lddz = lddz;
  p.h = h;
  p.ldh = ldh;
  const bool vx = vec8_ok(dh, dtype, lddh), vh = vec8_ok(h, dtype, ldh), vz = vec8_ok(dz, dtype, lddz);
  return over_rows(p, rows, [&](const CkptArgs& a, dim3 grid) {
    return launch_kernel(checkpoint8_gelu_bwd_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), false, a,
                         vx, vh, vz);
  });
}

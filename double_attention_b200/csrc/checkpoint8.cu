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
// Bound: HBM.  Measured at 262144 x 1536: forward with GELU 299 us (5 bytes an element, 6.7 TB/s), without 181, backward
// 412 us (7 bytes, 6.8 TB/s), restore 179 us (6.7 TB/s).  A thread takes 8 columns,
// so the 4 threads of a block find its maximum with two shuffles and no row-wide reduction is needed, whatever the
// width.  Dense tensors whose width is a multiple of 32 run as one long row; the others find their row by a
// multiplication.  Rows on 16-byte words (kVec): 50000 x 1000 in 48 us forward, 58 backward, 25 restored (1024 wide 41, 55
// and 25).  Dense rows that start anywhere in one go through shared memory (kDense): 50000 x 1001 in 61, 88 and 30 us,
// bound by instructions and shared memory (a value at a time backward took 263, restoring 140).
#include "common.cuh"
#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace {

constexpr int kNotFinite = -128;
constexpr int kItems = 4;  // groups of 8 columns per thread, all loaded before the first is used

struct CkptArgs {
  const void* x;  // z or dh
  void* h;
  void* dz;
  int8_t* q;
  int8_t* e;
  int64_t ldx, ldh, lddz;
  int64_t left;   // values of a dense tensor from this launch's first one on
  int64_t items;  // groups of 8 columns in this launch (below 2^31 unless flat)
  Div31 per_row;  // groups of 8 columns in a row of q (a multiple of 4)
  int D, gelu, e_min, e_max;
  int vec_x, vec_h, vec_dz;  // 16-byte rows
};

// How a tensor's rows lie: one long row; rows on 16-byte words whose width is a multiple of 8; dense rows of any other
// width, whose groups of 8 columns start anywhere in a 16-byte word; or anything.
enum : int { kFlat = 0, kVec = 1, kDense = 2, kAny = 3 };

// Eight 16-bit values of a row, those past D as 0.
template <typename T>
DA_DEV uint4 load_row8(const void* p, int64_t base, int col, int D, bool vec) {
  const T* src = static_cast<const T*>(p) + base + col;
  if (vec && col + 8 <= D) return *reinterpret_cast<const uint4*>(src);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = col + 2 * i < D ? reinterpret_cast<const uint16_t*>(src)[2 * i] : 0;
    const uint32_t hi = col + 2 * i + 1 < D ? reinterpret_cast<const uint16_t*>(src)[2 * i + 1] : 0;
    w[i] = lo | hi << 16;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
DA_DEV void store_row8(void* p, int64_t base, int col, int D, bool vec, uint4 v) {
  T* dst = static_cast<T*>(p) + base + col;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if (vec && col + 8 <= D) {
    *reinterpret_cast<uint4*>(dst) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < D) reinterpret_cast<uint16_t*>(dst)[i] = (uint16_t)(w[i / 2] >> (i % 2 * 16));
  }
}

// 2^e, e in [-126, 127].
DA_DEV float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <int kLies>
using Index = std::conditional_t<kLies == kFlat, int64_t, int>;
template <int kLies>
DA_DEV Index<kLies> index_of(int k) {  // the k-th group of a thread
  return ((Index<kLies>)blockIdx.x * kItems + k) * 256 + threadIdx.x;
}
template <int kLies>
struct Place {  // of a group of 8 columns
  Index<kLies> group;
  int row, col;
};
template <int kLies>
DA_DEV Place<kLies> place_of(const CkptArgs& p, Index<kLies> i) {
  if constexpr (kLies == kFlat) return {i, 0, 0};
  const uint32_t r = p.per_row.div((uint32_t)i), c = (uint32_t)i - r * p.per_row.d;
  return {i, (int)r, (int)c * 8};
}

// kDense: the values of a block's groups are one run of a dense tensor, which goes through shared memory: in 16-byte words
// on the tensor's side and, on the threads', whose groups start at any value, in 32-bit words moved by half a word.
// (Shifted in registers, with the words' other values from neighbouring lanes, storing alone took 15 instructions a
// value: 50000 x 1001 in 90 us forward and 135 backward, now 61 and 88.)
struct Run {
  int64_t base, first, end;  // the values [first, end), base = first rounded down to 16 bytes
};
constexpr int kRunWords = 256 * kItems + 1;  // of 16 bytes
DA_DEV Run run_of(const CkptArgs& p) {
  auto flat = [&](int i) {
    const Place<kDense> at = place_of<kDense>(p, i);
    return (int64_t)at.row * p.D + min(at.col, p.D);
  };
  const int i0 = blockIdx.x * (256 * kItems);
  const int64_t first = flat(i0);
  return {first & ~int64_t(7), first, flat(min((int)p.items, i0 + 256 * kItems))};
}
DA_DEV void load_run(const void* p, const Run& run, int64_t left, uint4* buf) {
  const uint16_t* src = static_cast<const uint16_t*>(p) + run.base;
  const int words = (int)((run.end - run.base + 7) / 8), whole = (int)min((int64_t)words, (left - run.base) / 8);
  uint4 v[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k)
    if (k * 256 + (int)threadIdx.x < whole) v[k] = __ldcs(reinterpret_cast<const uint4*>(src) + k * 256 + threadIdx.x);
#pragma unroll
  for (int k = 0; k < kItems; ++k)
    if (k * 256 + (int)threadIdx.x < whole) buf[k * 256 + threadIdx.x] = v[k];
  // the 1025th word, and the tensor's last values
  if (threadIdx.x == 0 && whole == kRunWords) buf[kRunWords - 1] = reinterpret_cast<const uint4*>(src)[kRunWords - 1];
  if (whole < words && threadIdx.x < 8 && run.base + whole * 8 + threadIdx.x < run.end)
    reinterpret_cast<uint16_t*>(buf)[whole * 8 + threadIdx.x] = src[whole * 8 + threadIdx.x];
}
// A group's 8 values, those past D as 0.
DA_DEV uint4 take_run(const uint4* buf, const Run& run, const Place<kDense>& at, int D) {
  if (at.col >= D) return make_uint4(0, 0, 0, 0);
  const int off = (int)((int64_t)at.row * D + at.col - run.base), s = off % 2 * 16;
  const uint32_t* w = reinterpret_cast<const uint32_t*>(buf) + off / 2;
  uint4 v = make_uint4(__funnelshift_r(w[0], w[1], s), __funnelshift_r(w[1], w[2], s), __funnelshift_r(w[2], w[3], s),
                       __funnelshift_r(w[3], w[4], s));
  if (at.col + 8 > D) {  // the next row's values
    uint32_t* u = &v.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int left = D - at.col - 2 * i;
      u[i] = left >= 2 ? u[i] : left == 1 ? u[i] & 0xffffu : 0;
    }
  }
  return v;
}
DA_DEV void put_run(uint4* buf, const Run& run, const Place<kDense>& at, int D, uint4 v) {
  if (at.col >= D) return;
  const int off = (int)((int64_t)at.row * D + at.col - run.base);
  uint16_t* h = reinterpret_cast<uint16_t*>(buf) + off;
  uint32_t* w = reinterpret_cast<uint32_t*>(buf) + (off + 1) / 2;
  if (at.col + 8 > D) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (at.col + i < D) h[i] = (uint16_t)(u[i / 2] >> (i % 2 * 16));
  } else if (off % 2) {
    h[0] = (uint16_t)v.x;
    w[0] = __funnelshift_r(v.x, v.y, 16);
    w[1] = __funnelshift_r(v.y, v.z, 16);
    w[2] = __funnelshift_r(v.z, v.w, 16);
    h[7] = (uint16_t)(v.w >> 16);
  } else {
    w[0] = v.x;
    w[1] = v.y;
    w[2] = v.z;
    w[3] = v.w;
  }
}
DA_DEV void store_run(void* p, const Run& run, const uint4* buf) {
  uint16_t* dst = static_cast<uint16_t*>(p) + run.base;
  const int from = (int)(run.first - run.base), to = (int)(run.end - run.base);
#pragma unroll
  for (int k = 0; k <= kItems; ++k) {
    const int w = k * 256 + threadIdx.x;
    if (w * 8 >= from && w * 8 + 8 <= to) {
      reinterpret_cast<uint4*>(dst)[w] = buf[w];
    } else if (w * 8 < to && w * 8 + 8 > from) {  // a word shared with another block, or past the tensor
      for (int i = max(from, w * 8); i < min(to, w * 8 + 8); ++i) dst[i] = reinterpret_cast<const uint16_t*>(buf)[i];
    }
  }
}
template <typename T, int kLies>
DA_DEV uint4 load_place(const CkptArgs& p, const Place<kLies>& at) {
  if constexpr (kLies == kFlat) return __ldcs(reinterpret_cast<const uint4*>(p.x) + at.group);
  if constexpr (kLies == kVec) {
    if (at.col >= p.D) return make_uint4(0, 0, 0, 0);
    return __ldcs(reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + at.row * p.ldx + at.col));
  }
  return load_row8<T>(p.x, at.row * p.ldx, at.col, p.D, p.vec_x);
}
// (kDense: to the block's shared memory)
template <typename T, int kLies>
DA_DEV void store_place(const CkptArgs& p, void* out, int64_t ld, int vec, const Place<kLies>& at, const F2* v, uint4* buf,
                        const Run& run) {
  const uint4 w = make_uint4(narrow<T>(v[0]), narrow<T>(v[1]), narrow<T>(v[2]), narrow<T>(v[3]));
  if constexpr (kLies == kFlat) {
    reinterpret_cast<uint4*>(out)[at.group] = w;
  } else if constexpr (kLies == kVec) {
    if (at.col < p.D) *reinterpret_cast<uint4*>(static_cast<T*>(out) + at.row * ld + at.col) = w;
  } else if constexpr (kLies == kDense) {
    put_run(buf, run, at, p.D, w);
  } else {
    store_row8<T>(out, at.row * ld, at.col, p.D, vec, w);
  }
}
// The groups' 8 values each.
template <typename T, int kLies>
DA_DEV void load_places(const CkptArgs& p, const Place<kLies> (&at)[kItems], uint4 (&raw)[kItems], uint4* buf,
                        const Run& run) {
  if constexpr (kLies == kDense) {
    load_run(p.x, run, p.left, buf);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      raw[k] = at[k].group < (int)p.items ? take_run(buf, run, at[k], p.D) : make_uint4(0, 0, 0, 0);
    __syncthreads();  // (a result may take the place)
  } else {
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      raw[k] = at[k].group < (Index<kLies>)p.items ? load_place<T, kLies>(p, at[k]) : make_uint4(0, 0, 0, 0);
  }
}
template <int kLies, int kBuffers>
struct Buffers {
  uint4 words[kLies == kDense ? kBuffers : 1][kLies == kDense ? kRunWords + 1 : 1];  // (a take reads a word further)
};

template <typename T, int kLies>
__global__ void __launch_bounds__(256) checkpoint8_kernel(const CkptArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ Buffers<kLies, 1> buffers;
  uint4* buf = buffers.words[0];
  const Run run = kLies == kDense ? run_of(p) : Run{};
  uint4 raw[kItems];
  Place<kLies> at[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) at[k] = place_of<kLies>(p, index_of<kLies>(k));
  load_places<T, kLies>(p, at, raw, buf, run);
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    // the 16-bit patterns without their signs order as integers, NaN above infinity above every number
    uint32_t m = __vmaxu2(__vmaxu2(raw[k].x & 0x7fff7fffu, raw[k].y & 0x7fff7fffu),
                          __vmaxu2(raw[k].z & 0x7fff7fffu, raw[k].w & 0x7fff7fffu));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    m = max(m & 0xffffu, m >> 16);
    uint32_t a;  // as fp32
    if constexpr (std::is_same<T, __nv_bfloat16>::value) a = m << 16;
    else a = __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    // a = f 2^E with 1 <= f < 2: 127 * 2^(E - 6) covers it if f <= 1.984375 (mantissa bits 0x7e0000)
    const int fit = (int)(a >> 23) - 127 - 6 + ((a & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    const bool finite = a < 0x7f800000u;
    const int e = max(p.e_min, min(p.e_max, fit));
    const F2 inv = dup(pow2i(-e));
    F2 v[4] = {widen<T>(raw[k].x), widen<T>(raw[k].y), widen<T>(raw[k].z), widen<T>(raw[k].w)};
    uint2 q;
    if (fit <= p.e_max) {
      const F2 at_unit = dup(kRoundAt);
      q.x = low_bytes(fma2(v[0], inv, at_unit), fma2(v[1], inv, at_unit));
      q.y = low_bytes(fma2(v[2], inv, at_unit), fma2(v[3], inv, at_unit));
    } else {  // saturating, or not finite
      int o[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo, hi;
        split(mul2(v[j], inv), lo, hi);
        o[2 * j] = finite ? max(-127, min(127, __float2int_rn(lo))) : 0;
        o[2 * j + 1] = finite ? max(-127, min(127, __float2int_rn(hi))) : 0;
      }
      q = pack_s8x8(o);
    }
    const bool live = at[k].group < (Index<kLies>)p.items;
    if (live) {
      *reinterpret_cast<uint2*>(p.q + (int64_t)at[k].group * 8) = q;
      if ((at[k].group & 3) == 0) p.e[at[k].group >> 2] = (int8_t)(finite ? e : kNotFinite);
    }
    if (p.gelu) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = gelu2(v[j]);
      if (live) store_place<T, kLies>(p, p.h, p.ldh, p.vec_h, at[k], v, buf, run);
    }
  }
  if (kLies == kDense && p.gelu) {
    __syncthreads();
    store_run(p.h, run, buf);
  }
}

// A kept group's 8 values.
DA_DEV void restore8(uint2 q, int e, F2* v) {
  const F2 unit = dup(e == kNotFinite ? __uint_as_float(0x7fffffffu) : pow2i(e));
  signed_bytes(q.x, v[0], v[1]);
  signed_bytes(q.y, v[2], v[3]);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = mul2(v[j], unit);
}

template <typename T, int kLies>
__global__ void __launch_bounds__(256) checkpoint8_restore_kernel(const CkptArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ Buffers<kLies, 1> buffers;
  uint4* buf = buffers.words[0];
  const Run run = kLies == kDense ? run_of(p) : Run{};
  uint2 q[kItems] = {};
  int e[kItems] = {};
  Place<kLies> at[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    at[k] = place_of<kLies>(p, index_of<kLies>(k));
    if (at[k].group < (Index<kLies>)p.items) {
      q[k] = *reinterpret_cast<const uint2*>(p.q + (int64_t)at[k].group * 8);
      e[k] = p.e[at[k].group >> 2];
    }
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    if (at[k].group >= (Index<kLies>)p.items) continue;
    F2 v[4];
    restore8(q[k], e[k], v);
    if constexpr (std::is_same<T, float>::value) {
      float* dst = static_cast<float*>(p.h) + (kLies == kFlat ? at[k].group * 8 : at[k].row * p.ldh + at[k].col);
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) split(v[j], f[2 * j], f[2 * j + 1]);
      if constexpr (kLies == kFlat || kLies == kVec) {
        if (kLies == kVec && at[k].col >= p.D) continue;
        reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (at[k].col + j < p.D) dst[j] = f[j];
      }
    } else {
      store_place<T, kLies>(p, p.h, p.ldh, p.vec_h, at[k], v, buf, run);
    }
  }
  if constexpr (kLies == kDense) {
    __syncthreads();
    store_run(p.h, run, buf);
  }
}

template <typename T, int kLies>
__global__ void __launch_bounds__(256) checkpoint8_gelu_bwd_kernel(const CkptArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ Buffers<kLies, 2> buffers;
  uint4 *buf = buffers.words[0], *buf_h = buffers.words[kLies == kDense];
  const Run run = kLies == kDense ? run_of(p) : Run{};
  uint4 raw[kItems];
  uint2 q[kItems] = {};
  int e[kItems] = {};
  Place<kLies> at[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    at[k] = place_of<kLies>(p, index_of<kLies>(k));
    if (at[k].group < (Index<kLies>)p.items) {
      q[k] = *reinterpret_cast<const uint2*>(p.q + (int64_t)at[k].group * 8);
      e[k] = p.e[at[k].group >> 2];
    }
  }
  load_places<T, kLies>(p, at, raw, buf, run);
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    if (at[k].group >= (Index<kLies>)p.items) continue;
    F2 z[4], d[4] = {widen<T>(raw[k].x), widen<T>(raw[k].y), widen<T>(raw[k].z), widen<T>(raw[k].w)};
    restore8(q[k], e[k], z);
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] = mul2(d[j], gelu_grad2(z[j]));
    store_place<T, kLies>(p, p.dz, p.lddz, p.vec_dz, at[k], d, buf, run);
    if (p.h) store_place<T, kLies>(p, p.h, p.ldh, p.vec_h, at[k], z, buf_h, run);
  }
  if constexpr (kLies == kDense) {
    __syncthreads();
    store_run(p.dz, run, buf);
    if (p.h) store_run(p.h, run, buf_h);
  }
}

// Runs the kernel over all groups: at once where the tensors are one long row, else over slabs of rows whose items
// stay below 2^31.
template <typename T, template <typename, int> class Kernel>
int run(CkptArgs p, int64_t rows, int lies, cudaStream_t st) {
  const int64_t per_block = 256 * kItems;
  auto grid = [&] { return dim3((unsigned)((p.items + per_block - 1) / per_block)); };
  if (lies == kFlat && rows * p.per_row.d / per_block < 0x7fffffffLL) {
    p.items = rows * p.per_row.d;
    return launch_kernel(Kernel<T, kFlat>::get(), grid(), dim3(256), 0, st, false, p);
  }
  auto skip = [](auto* ptr, int64_t n) { return ptr ? ptr + n : ptr; };
  const int64_t slab = (Div31::kMax - 2 * per_block) / p.per_row.d / 8 * 8;  // (a slab starts as aligned as its tensor)
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t n = rows - r0 < slab ? rows - r0 : slab;
    CkptArgs s = p;
    s.x = skip(static_cast<const T*>(p.x), r0 * p.ldx);
    s.h = skip(static_cast<T*>(p.h), r0 * p.ldh);
    s.dz = skip(static_cast<T*>(p.dz), r0 * p.lddz);
    s.q += r0 * p.per_row.d * 8;
    s.e += r0 * p.per_row.d / 4;
    s.left = (rows - r0) * p.D;
    s.items = p.items = n * p.per_row.d;
    const int rc = lies == kVec     ? launch_kernel(Kernel<T, kVec>::get(), grid(), dim3(256), 0, st, false, s)
                   : lies == kDense ? launch_kernel(Kernel<T, kDense>::get(), grid(), dim3(256), 0, st, false, s)
                                    : launch_kernel(Kernel<T, kAny>::get(), grid(), dim3(256), 0, st, false, s);
    if (rc) return rc;
  }
  return DA_OK;
}
template <typename T, int kLies>
struct Forward {
  static auto get() { return checkpoint8_kernel<T, kLies>; }
};
template <typename T, int kLies>
struct Restore {
  static auto get() { return checkpoint8_restore_kernel<T, kLies>; }
};
template <typename T, int kLies>
struct GeluBackward {
  static auto get() { return checkpoint8_gelu_bwd_kernel<T, kLies>; }
};

CkptArgs make_args(int64_t D, int dtype, const int8_t* q, const int8_t* e) {
  CkptArgs p{nullptr, nullptr, nullptr, const_cast<int8_t*>(q), const_cast<int8_t*>(e), 0, 0, 0, 0, 0,
             Div31((uint32_t)((D + 31) / 32 * 4)), (int)D, 0, -126, 121, 0, 0, 0};
  if (dtype == DA_F16) {
    p.e_min = -24;
    p.e_max = 9;
  }
  return p;
}
// How a tensor lies, and the common way of two (absent tensors lie flat; kVec and kDense differ in D, so never meet).
int lies_of(const void* p, int64_t ld, int64_t D) {
  if (!p) return kFlat;
  if (reinterpret_cast<uintptr_t>(p) % 16) return kAny;
  if (ld == D && D % 32 == 0) return kFlat;
  if (D % 8 == 0) return ld % 8 == 0 ? kVec : kAny;
  return ld == D ? kDense : kAny;
}
int common(int a, int b) { return a > b ? a : b; }
bool bad_shape(int64_t rows, int64_t D) { return rows <= 0 || D <= 0 || D > 0x7fff0000LL; }  // (8 rows of items stay below 2^31)
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
  CkptArgs p = make_args(D, dtype, q, e);
  p.x = x;
  p.ldx = ldx;
  p.h = h;
  p.ldh = ldh;
  p.gelu = gelu;
  p.vec_x = vec8_ok(x, dtype, ldx);
  p.vec_h = vec8_ok(h, dtype, ldh);
  const int lies = common(lies_of(x, ldx, D), gelu ? lies_of(h, ldh, D) : kFlat);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DA_BF16 ? run<__nv_bfloat16, Forward>(p, rows, lies, st) : run<__half, Forward>(p, rows, lies, st);
}

extern "C" int da_checkpoint8_restore(const int8_t* q, const int8_t* e, int64_t rows, int64_t D, void* out, int dtype,
                                      int64_t ldo, void* stream) {
  using namespace da;
  if (!q || !e || !out) return DA_ERR_NULL;
  if (bad_shape(rows, D) || ldo < D) return DA_ERR_SHAPE;
  if (!half_dtype(dtype) && dtype != DA_F32) return DA_ERR_DTYPE;
  if (reinterpret_cast<uintptr_t>(q) % 16) return DA_ERR_ALIGN;
  if (int rc = bind_device(q)) return rc;
  CkptArgs p = make_args(D, dtype, q, e);
  p.h = out;
  p.ldh = ldo;
  p.vec_h = vec8_ok(out, dtype, ldo);
  const int lies = lies_of(out, ldo, D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == DA_F32) return run<float, Restore>(p, rows, lies == kDense ? kAny : lies, st);
  return dtype == DA_BF16 ? run<__nv_bfloat16, Restore>(p, rows, lies, st) : run<__half, Restore>(p, rows, lies, st);
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
  CkptArgs p = make_args(D, dtype, q, e);
  p.x = dh;
  p.ldx = lddh;
  p.dz = dz;
  p.lddz = lddz;
  p.h = h;
  p.ldh = ldh;
  p.vec_x = vec8_ok(dh, dtype, lddh);
  p.vec_dz = vec8_ok(dz, dtype, lddz);
  p.vec_h = vec8_ok(h, dtype, ldh);
  const int lies = common(lies_of(dh, lddh, D), common(lies_of(dz, lddz, D), lies_of(h, ldh, D)));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DA_BF16 ? run<__nv_bfloat16, GeluBackward>(p, rows, lies, st)
                          : run<__half, GeluBackward>(p, rows, lies, st);
}

// New tokens' routed keys and dense values into the pages of a cache.
//
// Row j of the packed tokens, the i-th new one of its sequence b, goes to position lengths[b] + i: H R key elements from
// [H, tokens, R] and D value elements from [tokens, D], converted to the cache's type with one rounding.  Bytes in and
// out are all there is: a warp takes one token, finds its sequence with a 32-way search of the starts (two dependent
// loads up to 1024 sequences) and copies 16 bytes a lane.  11100 tokens of 512 + 512 columns in bf16, 46 MB in and out: 12.5
// us from memory, 3.7 TB/s (a warp has two to four loads in flight), 7.0 where all of it lies in L2; 64 single tokens 2.9 us, a
// launch's latency.  Sources off 16 bytes go element by element.
#include "host_util.h"
#include "paged.cuh"
#include "vec8.cuh"

namespace da {
namespace paged {

struct AppendParams {
  Cache c;
  const void *keys, *values;
  int64_t k_branch, k_row, v_row;  // strides in elements
  int k_dtype, v_dtype;
  int H, R, D;
  void *key_pages, *value_pages;
  int* status;
};

// Eight elements of a float type as eight 16-bit ones.
template <typename T>
DA_DEV uint4 load8_as(const void* src, int dtype, int64_t off) {
  if (dtype == DA_F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(src) + off);
    const float4 a = p[0], b = p[1];
    return make_uint4(pack2<T>(a.x, a.y), pack2<T>(a.z, a.w), pack2<T>(b.x, b.y), pack2<T>(b.z, b.w));
  }
  uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + off);
  constexpr int own = std::is_same<T, __nv_bfloat16>::value ? DA_BF16 : DA_F16;
  if (dtype != own) {
    using Other = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __half, __nv_bfloat16>;
    uint32_t* u = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<Other>(u[i]);
      u[i] = pack2<T>(f.x, f.y);
    }
  }
  return w;
}

// kVec: rows and branches of the sources start on 16 bytes.
template <typename T, bool kVec>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % 32;
  const int64_t row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (row >= p.c.tokens) return;
  const int b = find_sequence(p.c, row);
  if (b >= p.c.B) return;  // behind the last sequence
  const Sequence s = sequence(p.c, b);
  if (row < s.first) return;  // before the first sequence
  const int64_t at = (int64_t)p.c.lengths[b] + (row - s.first);
  int page = -1;
  if (at >= 0 && at < p.c.capacity) page = p.c.table[b * p.c.table_stride + (at >> p.c.page_shift)];
  if (page < 0 || page >= p.c.pages) {
    if (lane == 0) atomicOr(p.status, DA_DEV_BAD_PAGE);
    return;
  }
  const int64_t slot = ((int64_t)page << p.c.page_shift) + (at & (p.c.page - 1));
  const int wide = p.H * p.R;
  T* k_out = static_cast<T*>(p.key_pages) + slot * wide;
  T* v_out = static_cast<T*>(p.value_pages) + slot * p.D;
  if constexpr (kVec) {
    for (int i = lane * 8; i < wide; i += 256) {
      const int h = i / p.R;
      *reinterpret_cast<uint4*>(k_out + i) = load8_as<T>(p.keys, p.k_dtype, h * p.k_branch + row * p.k_row + (i - h * p.R));
    }
    for (int i = lane * 8; i < p.D; i += 256)
      *reinterpret_cast<uint4*>(v_out + i) = load8_as<T>(p.values, p.v_dtype, row * p.v_row + i);
  } else {
    for (int i = lane; i < wide; i += 32) {
      const int h = i / p.R;
      k_out[i] = from_f32<T>(load1(p.keys, p.k_dtype, h * p.k_branch + row * p.k_row + (i - h * p.R)));
    }
    for (int i = lane; i < p.D; i += 32) v_out[i] = from_f32<T>(load1(p.values, p.v_dtype, row * p.v_row + i));
  }
}

}  // namespace paged
}  // namespace da

extern "C" int da_paged_append(const void* keys, int key_dtype, int64_t key_branch_stride, int64_t key_row_stride,
                               const void* values, int value_dtype, int64_t value_row_stride, int64_t tokens,
                               void* key_pages, void* value_pages, int dtype, int64_t pages, int page, int H, int R, int D,
                               const int* table, int64_t table_stride, int64_t table_cols, const int* lengths,
                               const int* starts, int64_t B, int* status, void* stream) {
  using namespace da;
  if (!keys || !values || !key_pages || !value_pages || !table || !lengths || !starts || !status) return DA_ERR_NULL;
  if (dtype != DA_BF16 && dtype != DA_F16) return DA_ERR_DTYPE;
  for (int t : {key_dtype, value_dtype})
    if (t != DA_BF16 && t != DA_F16 && t != DA_F32) return DA_ERR_DTYPE;
  paged::AppendParams p;
  if (int rc = paged::make_cache(&p.c, table, table_stride, table_cols, lengths, starts, B, tokens, pages, page)) return rc;
  if (H < 1 || R < 8 || R % 8 || D < 8 || D % 8 || (int64_t)H * R > 65536 || D > 65536) return DA_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(key_pages) % 16 || reinterpret_cast<uintptr_t>(value_pages) % 16) return DA_ERR_ALIGN;
  if (tokens == 0 || B == 0) return DA_OK;
  if (int rc = bind_device(key_pages)) return rc;
  p.keys = keys;
  p.values = values;
  p.k_branch = key_branch_stride;
  p.k_row = key_row_stride;
  p.v_row = value_row_stride;
  p.k_dtype = key_dtype;
  p.v_dtype = value_dtype;
  p.H = H;
  p.R = R;
  p.D = D;
  p.key_pages = key_pages;
  p.value_pages = value_pages;
  p.status = status;
  const bool vec = vec8_ok(keys, key_dtype, key_row_stride) && (H == 1 || vec8_ok(keys, key_dtype, key_branch_stride)) &&
                   vec8_ok(values, value_dtype, value_row_stride);
  const bool bf16 = dtype == DA_BF16;
  auto kern = bf16 ? (vec ? paged::append_kernel<__nv_bfloat16, true> : paged::append_kernel<__nv_bfloat16, false>)
                   : (vec ? paged::append_kernel<__half, true> : paged::append_kernel<__half, false>);
  return launch_kernel(kern, dim3((unsigned)((tokens + 7) / 8)), dim3(256), 0, static_cast<cudaStream_t>(stream), false, p);
}

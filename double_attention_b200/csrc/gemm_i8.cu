// int8 matrix product with a scale per row of each operand:
//   C[m, n] = f((sum_k A[m, k] B[n, k]) * sa[m] * sb[n] + bias[n]),  f = identity or GELU
// A [M, K] are int8 activations with a scale per token, B [N, K] int8 weights with a scale per output
// channel.  The sum is exact in int32 (|A|, |B| <= 128 and K <= 131071), so any split of K and any order give
// the same bits; it is converted to fp32, scaled and rounded once to C's dtype.
//
// 64 x 64 tiles, dp4a on operands staged in shared memory, 4 x 4 outputs per thread.
#include "common.cuh"
#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace i8 {

constexpr int64_t kMaxK = 131071;

struct Params {
  const int8_t* a;
  const int8_t* b;
  const float* sa;
  const float* sb;
  const void* bias;
  void* c;
  int64_t lda, ldb, ldc;
  int M, N, K, bias_dtype, c_dtype, gelu;
};

__global__ void __launch_bounds__(256) gemm_kernel(const Params p) {
  __shared__ int sa[16][65], sb[16][65];  // [K group of 4][row]
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t m0 = (int64_t)blockIdx.x * 64;
  const int n0 = blockIdx.y * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 64) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int r = i / 16, g = i % 16, k = k0 + g * 4;
      int va = 0, vb = 0;
      for (int e = 0; e < 4; ++e) {
        if (k + e < p.K && m0 + r < p.M) va |= (int)(uint8_t)p.a[(m0 + r) * p.lda + k + e] << (8 * e);
        if (k + e < p.K && n0 + r < p.N) vb |= (int)(uint8_t)p.b[(int64_t)(n0 + r) * p.ldb + k + e] << (8 * e);
      }
      sa[g][r] = va;
      sb[g][r] = vb;
    }
    __syncthreads();
    for (int g = 0; g < 16; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(sa[g][ty + 16 * i], sb[g][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty + 16 * i;
      const int n = n0 + tx + 16 * j;
      if (m >= p.M || n >= p.N) continue;
      float y = (float)acc[i][j] * p.sa[m] * p.sb[n];
      if (p.bias) y += load1(p.bias, p.bias_dtype, n);
      if (p.gelu) y = gelu8(y);
      store1(p.c, p.c_dtype, m * p.ldc + n, y);
    }
}

}  // namespace i8
}  // namespace da

extern "C" int da_gemm_i8(const int8_t* A, int64_t lda, const float* a_scale, const int8_t* B, int64_t ldb,
                          const float* b_scale, const void* bias, int bias_dtype, int gelu, void* C, int64_t ldc,
                          int c_dtype, int64_t M, int64_t N, int64_t K, int* status, void* stream) {
  using namespace da;
  if (!A || !B || !a_scale || !b_scale || !C || !status) return DA_ERR_NULL;
  if (M <= 0 || N <= 0 || K <= 0 || K > i8::kMaxK || M > 0x7fffffffLL || N > 0x3fffffLL || lda < K || ldb < K || ldc < N)
    return DA_ERR_SHAPE;
  if (c_dtype < DA_F16 || c_dtype > DA_F32 || (bias && (bias_dtype < DA_F16 || bias_dtype > DA_F32)))
    return DA_ERR_DTYPE;
  if (lda % 16 || ldb % 16 || reinterpret_cast<uintptr_t>(A) % 16 || reinterpret_cast<uintptr_t>(B) % 16)
    return DA_ERR_ALIGN;
  if (int rc = bind_device(A)) return rc;
  const i8::Params p{A, B, a_scale, b_scale, bias, C, lda, ldb, ldc, (int)M, (int)N, (int)K, bias_dtype, c_dtype, gelu};
  const dim3 grid((unsigned)((M + 63) / 64), (unsigned)((N + 63) / 64));
  return launch_kernel(i8::gemm_kernel, grid, dim3(256), 0, static_cast<cudaStream_t>(stream), false, p);
}

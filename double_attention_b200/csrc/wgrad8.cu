// Weight gradient of a Linear from the 8-bit checkpoint of its input:
//   dW[n, k] = sum_t dY[t, n] X[t, k],  X[t, k] = q[t, k] 2^e[t, k / 32]
// with fp32 accumulation over the rows.  X is exact in dY's dtype, so nothing is rounded before the sum.
//
// 64 x 64 tiles of dW, both operands staged in shared memory in fp32, 4 x 4 outputs per thread.  The rows are
// split over the grid's third dimension where there are few tiles; partial sums are added in split order.
#include "common.cuh"
#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace wg8 {

struct Params {
  const void* dy;
  const int8_t* q;
  const int8_t* e;
  void* out;
  float* partial;
  int64_t ldy, ldq, lde, ldo, rows, rows_per_split;
  int N, K, dtype, out_dtype;
};

__global__ void __launch_bounds__(256) wgrad_kernel(const Params p) {
  __shared__ float sy[16][64], sx[16][64];  // [row][column]
  grid_dependency_wait();
  grid_launch_dependents();
  const int n0 = blockIdx.x * 64, k0 = blockIdx.y * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int64_t t_end = min(p.rows, (int64_t)(blockIdx.z + 1) * p.rows_per_split);
  float acc[4][4] = {};
  for (int64_t t0 = (int64_t)blockIdx.z * p.rows_per_split; t0 < t_end; t0 += 16) {
    for (int i = threadIdx.x; i < 16 * 64; i += 256) {
      const int64_t t = t0 + i / 64;
      const int c = i % 64;
      float y = 0.f, x = 0.f;
      if (t < t_end && n0 + c < p.N) y = load1(p.dy, p.dtype, t * p.ldy + n0 + c);
      if (t < t_end && k0 + c < p.K) {
        const int e = p.e[t * p.lde + (k0 + c) / 32];
        x = e == -128 ? __uint_as_float(0x7fffffffu)
                      : (float)p.q[t * p.ldq + k0 + c] * __uint_as_float((uint32_t)(e + 127) << 23);
      }
      sy[i / 64][c] = y;
      sx[i / 64][c] = x;
    }
    __syncthreads();
    for (int t = 0; t < 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sy[t][ty + 16 * i], sx[t][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + ty + 16 * i, k = k0 + tx + 16 * j;
      if (n < p.N && k < p.K) p.partial[((int64_t)blockIdx.z * p.N + n) * p.K + k] = acc[i][j];
    }
}

__global__ void __launch_bounds__(256) reduce_kernel(const Params p, int splits) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)p.N * p.K) return;
  float s = 0.f;
  for (int z = 0; z < splits; ++z) s += p.partial[(int64_t)z * p.N * p.K + i];
  store1(p.out, p.out_dtype, i / p.K * p.ldo + i % p.K, s);
}

int splits_for(int64_t N, int64_t K, int64_t rows) {
  const int64_t tiles = ((N + 63) / 64) * ((K + 63) / 64);
  int64_t s = (8LL * sm_count() + tiles - 1) / tiles;
  const int64_t most = (rows + 255) / 256;  // at least 256 rows each
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s > 512 ? 512 : s);
}

}  // namespace wg8
}  // namespace da

extern "C" int64_t da_checkpoint8_wgrad_workspace_elems(int64_t rows, int64_t N, int64_t K) {
  if (rows <= 0 || N <= 0 || K <= 0) return -1;
  return (int64_t)da::wg8::splits_for(N, K, rows) * N * K;
}

extern "C" int da_checkpoint8_wgrad(const void* dy, int dtype, int64_t ldy, const int8_t* q, const int8_t* e,
                                    int64_t rows, int64_t N, int64_t K, void* out, int out_dtype, int64_t ldo,
                                    float* workspace, int64_t workspace_elems, int* status, void* stream) {
  using namespace da;
  if (!dy || !q || !e || !out || !workspace || !status) return DA_ERR_NULL;
  if (rows <= 0 || N <= 0 || K <= 0 || N > 0x3fffffLL || K > 0x3fffffLL || ldy < N || ldo < K) return DA_ERR_SHAPE;
  if ((dtype != DA_F16 && dtype != DA_BF16) || (out_dtype != DA_F32 && out_dtype != dtype)) return DA_ERR_DTYPE;
  if (ldy % 8 || reinterpret_cast<uintptr_t>(dy) % 16 || reinterpret_cast<uintptr_t>(q) % 16) return DA_ERR_ALIGN;
  const int splits = wg8::splits_for(N, K, rows);
  if (workspace_elems < (int64_t)splits * N * K) return DA_ERR_WORKSPACE;
  if (int rc = bind_device(dy)) return rc;
  const int64_t blocks = (K + 31) / 32;
  wg8::Params p{dy, q, e, out, workspace, ldy, blocks * 32, blocks, ldo, rows, ((rows + splits - 1) / splits + 15) / 16 * 16,
                (int)N, (int)K, dtype, out_dtype};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((K + 63) / 64), (unsigned)splits);
  if (int rc = launch_kernel(wg8::wgrad_kernel, grid, dim3(256), 0, st, false, p)) return rc;
  return launch_kernel(wg8::reduce_kernel, dim3((unsigned)((N * K + 255) / 256)), dim3(256), 0, st, false, p, splits);
}

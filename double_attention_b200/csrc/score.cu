// Log probabilities of given tokens, the entropy of their distributions and the top alternatives, and the backward pass.
//
// Row x of V logits, with m = max x, t_i = (x_i - m) log2 e, l = sum 2^t_i and w = sum 2^t_i t_i:
//   log p_i = ln 2 (t_i - log2 l),     H = -sum p log p = ln 2 (log2 l - w / l),
//   dL/dx_i = g ([i = token] - p_i) - h p_i (log p_i + H)   for g = dL/d log p_token, h = dL/dH.
// m, l and w are kept against a running maximum, so the forward reads the logits once (16 bytes a load); the backward
// reads them again and writes the gradient.  Both are bound by those bytes.  Differences from the row's maximum are
// formed first and scaled inside one multiply-add, so that logits far from zero lose nothing; an entry of minus
// infinity counts 0 in l, w and the gradient.  A row with a NaN, with plus infinity or with nothing but minus infinity is
// NaN, as a softmax of it is.
//
// Top alternatives: in order of (value, lowest index), NaN before numbers.  The first pass leaves every warp's (or, where
// a warp has a row, every lane's) largest value; the top-th largest of those is at most the top-th largest value of the
// row, and few values lie above it (about 32 H_32 - 32 H_(32 - top) on independent ones), so a second pass, out of L1 and
// L2, collects what is not below it into a sorted list, one entry a lane.  Ties and hostile orders only make it longer.
#include <math.h>

#include "host_util.h"
#include "vec8.cuh"

namespace da {
namespace score {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int64_t kIgnore = -100;  // a token that is none: log probability 0, no gradient

struct Params {
  const void* logits;
  int64_t ld, rows;
  int V, top;
  const int64_t* tokens;
  float *log_probs, *entropy, *top_log_probs;
  int64_t* top_tokens;
  float* stats;  // [rows][2]: m log2 e and log2 l, or null
};

// 16 bytes of a row as floats.
template <typename T>
struct Vec {
  static constexpr int n = 8;
  static DA_DEV void get(uint4 w, float* x) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2<T>(u[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
  static DA_DEV float one(const T* p) { return unpack2<T>(*reinterpret_cast<const uint16_t*>(p)).x; }
  static DA_DEV uint4 put(const float* x) {
    return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int n = 4;
  static DA_DEV void get(uint4 w, float* x) {
    x[0] = __uint_as_float(w.x);
    x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z);
    x[3] = __uint_as_float(w.w);
  }
  static DA_DEV float one(const float* p) { return *p; }
  static DA_DEV uint4 put(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};

// A row as elements before the first 16-byte boundary, vectors from there on, and elements behind the last vector.
template <typename T>
struct Row {
  const T* p;
  int head, vecs, tail;
  DA_DEV Row(const void* base, int64_t at, int V) {
    p = static_cast<const T*>(base) + at;
    const int off = (int)(reinterpret_cast<uintptr_t>(p) % 16);
    head = off ? (16 - off) / (int)sizeof(T) : 0;
    if (head > V) head = V;
    vecs = (V - head) / Vec<T>::n;
    tail = V - head - vecs * Vec<T>::n;
  }
  DA_DEV int index(int vec) const { return head + vec * Vec<T>::n; }
  DA_DEV uint4 load(int vec) const { return *reinterpret_cast<const uint4*>(p + index(vec)); }
  // The element of the head (threads 0 to 7) or the tail (16 to 23) that thread `tid` takes, or -1.
  DA_DEV int odd(int tid) const {
    if (tid < head) return tid;
    if (tid >= 16 && tid < 16 + tail) return head + vecs * Vec<T>::n + tid - 16;
    return -1;
  }
};

// Running sums against a running maximum (all in log2 units).
struct Sums {
  float m, l, w;  // maximum, sum of 2^t, sum of 2^t t
  DA_DEV void raise(float to) {
    if (to > m) {
      const float d = m - to;
      if (m != -INFINITY) {
        const float c = ex2(d);
        w = c * fmaf(l, d, w);
        l *= c;
      }
      m = to;
    }
  }
  template <int n>
  DA_DEV void add(const float* x) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < n; ++i) top = fmaxf(top, x[i]);
    raise(top * kLog2e);
    const float at = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float t = fmaf(x[i], kLog2e, -at), e = ex2(t);
      l += e;
      w = fmaf(e, fmaxf(t, -1000.f), w);  // (2^t is 0 there: so is the term)
    }
  }
  DA_DEV void merge(const Sums& o) {
    Sums a = o;
    const float to = fmaxf(m, o.m);
    a.raise(to);
    raise(to);
    l += a.l;
    w += a.w;
  }
  DA_DEV Sums shuffled(int o) const {
    return {__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, l, o), __shfl_xor_sync(0xffffffffu, w, o)};
  }
};

// Floats in an order of unsigned integers: NaN above all, the zeros equal.
DA_DEV uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
DA_DEV float value_of(uint32_t k) { return k == 0xffffffffu ? NAN : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
DA_DEV uint64_t entry_of(float x, int index) { return (uint64_t)order_of(x) << 32 | (uint32_t)~index; }

// A warp's largest entries, sorted, the i-th in lane i.
struct List {
  uint64_t mine;  // 0: none
  uint64_t last;  // the top-th, in every lane
  DA_DEV void insert(uint64_t e, int top) {
    const int lane = threadIdx.x % 32;
    const int at = __popc(__ballot_sync(0xffffffffu, mine > e));
    const uint64_t up = __shfl_up_sync(0xffffffffu, mine, 1);
    mine = lane < at ? mine : lane == at ? e : up;
    last = __shfl_sync(0xffffffffu, mine, top - 1);
  }
  // The lanes' values x at `index`, where `in`.
  DA_DEV void offer(float x, int index, bool in, float& floor, int top) {
    uint32_t who = __ballot_sync(0xffffffffu, in && !(x < floor));
    if (!who) return;
    const uint64_t e = entry_of(x, index);
    while (who) {
      const int src = __ffs(who) - 1;
      who &= who - 1;
      const uint64_t c = __shfl_sync(0xffffffffu, e, src);
      if (c > last) insert(c, top);
    }
    if (last) {
      const float f = value_of((uint32_t)(last >> 32));
      if (f > floor) floor = f;
    }
  }
};

// The top-th largest of the lanes' values, in every lane.
DA_DEV float nth_largest(float x, int top) {
  const int lane = threadIdx.x % 32;
  const uint32_t k = order_of(x);
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t o = __shfl_sync(0xffffffffu, k, i);
    rank += o > k || (o == k && i < lane);
  }
  const uint32_t who = __ballot_sync(0xffffffffu, rank == top - 1);
  return __shfl_sync(0xffffffffu, x, __ffs(who) - 1);
}

// kThreads a row: 32 (eight rows a CTA) or 1024.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads == 32 ? 256 : 1024) forward_kernel(const Params p) {
  using V = Vec<T>;
  constexpr int kBatch = 16 / V::n;  // vectors whose largest value is found together
  __shared__ Sums sums[32];
  __shared__ uint64_t found[1024];
  __shared__ int count;
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int tid = kThreads == 32 ? lane : threadIdx.x;
  const int64_t r = kThreads == 32 ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
  if (kThreads == 32 && r >= p.rows) return;
  const Row<T> row(p.logits, r * p.ld, p.V);
  Sums s{-INFINITY, 0.f, 0.f};
  {
    int v = tid;
    for (; v + (2 * kBatch - 1) * kThreads < row.vecs; v += 2 * kBatch * kThreads) {
      uint4 raw[2 * kBatch];
#pragma unroll
      for (int i = 0; i < 2 * kBatch; ++i) raw[i] = row.load(v + i * kThreads);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        float x[16];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) V::get(raw[b * kBatch + i], x + i * V::n);
        s.add<16>(x);
      }
    }
    for (; v < row.vecs; v += kThreads) {
      float x[V::n];
      V::get(row.load(v), x);
      s.add<V::n>(x);
    }
    const int odd = row.odd(tid);
    if (odd >= 0) {
      const float x = V::one(row.p + odd);
      s.add<1>(&x);
    }
  }
  const float own = s.m;  // this thread's largest value times log2 e
#pragma unroll
  for (int o = 16; o; o >>= 1) s.merge(s.shuffled(o));
  float group = own;
  if constexpr (kThreads > 32) {
    group = s.m;  // the warp's
    if (lane == 0) sums[warp] = s;
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    s = sums[lane];
    group = s.m;  // lane i: warp i's
#pragma unroll
    for (int o = 16; o; o >>= 1) s.merge(s.shuffled(o));
  }
  const float at = s.m == -INFINITY ? 0.f : s.m, log_l = log2f(s.l);
  if (tid == 0) {
    const int64_t token = p.tokens[r];
    float lp = token == kIgnore ? 0.f : NAN;
    if (token >= 0 && token < p.V) lp = (fmaf(V::one(row.p + token), kLog2e, -at) - log_l) * kLn2;
    p.log_probs[r] = lp;
    p.entropy[r] = (log_l - s.w / s.l) * kLn2;
    if (p.stats) reinterpret_cast<float2*>(p.stats)[r] = make_float2(at, log_l);
  }
  if (p.top == 0) return;

  // The groups' maxima are products with log2 e: the floor is taken a little lower, so that no rounding lifts it.
  float floor = nth_largest(group, p.top) * kLn2;
  floor -= fabsf(floor) * 1e-6f + 1e-30f;
  List list{0, 0};
  const int all = (row.vecs + kThreads - 1) / kThreads * kThreads;  // every lane takes every turn
  for (int v = tid; v < all; v += kThreads) {
    float x[V::n];
#pragma unroll
    for (int i = 0; i < V::n; ++i) x[i] = -INFINITY;
    const bool in = v < row.vecs;
    if (in) V::get(row.load(v), x);
    bool any = false;
#pragma unroll
    for (int i = 0; i < V::n; ++i) any |= !(x[i] < floor);
    if (!__ballot_sync(0xffffffffu, in && any)) continue;
#pragma unroll
    for (int i = 0; i < V::n; ++i) list.offer(x[i], row.index(v) + i, in, floor, p.top);
  }
  {
    const int odd = row.odd(tid);
    list.offer(odd >= 0 ? V::one(row.p + odd) : 0.f, odd, odd >= 0, floor, p.top);
  }
  auto write = [&](uint64_t e, int rank) {
    p.top_log_probs[r * p.top + rank] = (fmaf(value_of((uint32_t)(e >> 32)), kLog2e, -at) - log_l) * kLn2;
    p.top_tokens[r * p.top + rank] = (uint32_t)~(uint32_t)e;
  };
  if constexpr (kThreads == 32) {
    if (lane < p.top) write(list.mine, lane);
  } else {
    const uint32_t have = __ballot_sync(0xffffffffu, lane < p.top && list.mine != 0);
    int base = 0;
    if (lane == 0 && have) base = atomicAdd(&count, __popc(have));
    base = __shfl_sync(0xffffffffu, base, 0);
    if (have >> lane & 1) found[base + __popc(have & ((1u << lane) - 1))] = list.mine;
    __syncthreads();
    const int n = count;  // at most 32 of each of 32 warps; no two alike, so every one has its rank, in whatever place
    if ((int)threadIdx.x < n) {
      const uint64_t e = found[threadIdx.x];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += found[i] > e;
      if (rank < p.top) write(e, rank);
    }
  }
}

struct BackwardParams {
  const void* logits;
  int64_t ld, rows;
  int V, segments;
  const int64_t* tokens;
  const float *stats, *entropy, *d_log_probs, *d_entropy;
  void* d_logits;
  int64_t ldd;
};

constexpr int kSegment = 2048;  // elements a warp

template <typename T>
__global__ void __launch_bounds__(256) backward_kernel(const BackwardParams p) {
  using V = Vec<T>;
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % 32;
  const int64_t item = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (item >= p.rows * p.segments) return;
  const int64_t r = item / p.segments;
  const int seg = (int)(item - r * p.segments);
  const Row<T> row(p.logits, r * p.ld, p.V);
  T* out = static_cast<T*>(p.d_logits) + r * p.ldd;
  const bool wide = (reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(row.p)) % 16 == 0;
  const float2 st = reinterpret_cast<const float2*>(p.stats)[r];
  const float H = p.entropy[r] * (1.f / kLn2), h = p.d_entropy ? p.d_entropy[r] * kLn2 : 0.f;
  float g = p.d_log_probs ? p.d_log_probs[r] : 0.f;
  const int64_t token = p.tokens[r];
  if (token == kIgnore) g = 0.f;
  else if (token < 0 || token >= p.V) g = p.d_log_probs ? NAN : 0.f;
  const float c = fmaf(h, H, g);
  auto grad = [&](float x, int64_t i) {
    const float t = fmaf(x, kLog2e, -st.x) - st.y;  // log2 p
    const float d = -ex2(t) * fmaf(h, fmaxf(t, -1000.f), c);
    return i == token ? d + g : d;
  };
  constexpr int kVecs = kSegment / V::n;
  const int v0 = seg * kVecs, v1 = min(row.vecs, v0 + kVecs);
#pragma unroll 4
  for (int v = v0 + lane; v < v1; v += 32) {
    float x[V::n];
    V::get(row.load(v), x);
    const int at = row.index(v);
#pragma unroll
    for (int i = 0; i < V::n; ++i) x[i] = grad(x[i], at + i);
    const uint4 w = V::put(x);
    if (wide) {
      *reinterpret_cast<uint4*>(out + at) = w;
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V::n; ++i) out[at + i] = x[i];
    } else {
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<uint16_t*>(out)[at + i] = (uint16_t)(u[i / 2] >> (16 * (i & 1)));
    }
  }
  if (seg == 0) {
    const int odd = row.odd(lane);
    if (odd >= 0) {
      const float d = grad(V::one(row.p + odd), odd);
      if constexpr (sizeof(T) == 4) out[odd] = d;
      else out[odd] = from_f32<T>(d);
    }
  }
}

int check(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t V, const void* tokens) {
  if (dtype != DA_F16 && dtype != DA_BF16 && dtype != DA_F32) return DA_ERR_DTYPE;
  if (rows < 0 || rows > 0x7fffffff || V < 1 || V > 0x7fffff00) return DA_ERR_SHAPE;
  if (rows && (!logits || !tokens)) return DA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DA_F32 ? 4 : 2)) return DA_ERR_ALIGN;
  (void)ld;
  return DA_OK;
}

// A warp a row where rows are short and many, else a CTA of 1024 threads a row.
template <typename T>
int forward(const Params& p, cudaStream_t st) {
  const bool warps = p.V <= 8192 && p.rows >= 4 * sm_count();
  if (warps)
    return launch_kernel(forward_kernel<T, 32>, dim3((unsigned)((p.rows + 7) / 8)), dim3(256), 0, st, false, p);
  return launch_kernel(forward_kernel<T, 1024>, dim3((unsigned)p.rows), dim3(1024), 0, st, false, p);
}

}  // namespace score
}  // namespace da

extern "C" int da_token_log_probs(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t V, const int64_t* tokens,
                                  int top, float* log_probs, float* entropy, float* top_log_probs, int64_t* top_tokens,
                                  float* stats, void* stream) {
  using namespace da;
  if (int rc = score::check(logits, dtype, ld, rows, V, tokens)) return rc;
  if (top < 0 || top > 32 || top > V) return DA_ERR_SHAPE;
  if (rows == 0) return DA_OK;
  if (!log_probs || !entropy || (top && (!top_log_probs || !top_tokens))) return DA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(stats) % 8) return DA_ERR_ALIGN;
  if (int rc = bind_device(logits)) return rc;
  const score::Params p{logits, ld, rows, (int)V, top, tokens, log_probs, entropy, top_log_probs, top_tokens, stats};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == DA_F32    ? score::forward<float>(p, st)
         : dtype == DA_BF16 ? score::forward<__nv_bfloat16>(p, st)
                            : score::forward<__half>(p, st);
}

extern "C" int da_token_log_probs_bwd(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t V,
                                      const int64_t* tokens, const float* stats, const float* entropy,
                                      const float* d_log_probs, const float* d_entropy, void* d_logits, int64_t ldd,
                                      void* stream) {
  using namespace da;
  if (int rc = score::check(logits, dtype, ld, rows, V, tokens)) return rc;
  if (rows == 0) return DA_OK;
  if (!stats || !entropy || !d_logits) return DA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(stats) % 8 || reinterpret_cast<uintptr_t>(d_logits) % (dtype == DA_F32 ? 4 : 2))
    return DA_ERR_ALIGN;
  if (int rc = bind_device(logits)) return rc;
  const int segments = (int)((V + score::kSegment - 1) / score::kSegment);
  const int64_t ctas = (rows * segments + 7) / 8;
  if (ctas > 0x7fffffff) return DA_ERR_SHAPE;
  const score::BackwardParams p{logits, ld, rows, (int)V, segments, tokens, stats, entropy, d_log_probs, d_entropy, d_logits, ldd};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kern = dtype == DA_F32    ? score::backward_kernel<float>
              : dtype == DA_BF16 ? score::backward_kernel<__nv_bfloat16>
                                 : score::backward_kernel<__half>;
  return launch_kernel(kern, dim3((unsigned)ctas), dim3(256), 0, st, false, p);
}

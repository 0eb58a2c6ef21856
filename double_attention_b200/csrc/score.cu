// Log probabilities of given tokens, the entropy of their distributions and the top alternatives, and the backward pass.
//
// Row x of V logits, with m = max x, t_i = (x_i - m) log2 e, l = sum 2^t_i and w = sum 2^t_i t_i:
//   log p_i = x_i - m - ln 2 log2 l,     H = -sum p log p = ln 2 (log2 l - w / l),
//   dL/dx_i = g ([i = token] - p_i) - h p_i (log p_i + H)   for g = dL/d log p_token, h = dL/dH.
// m, l and w are kept against a running maximum, so the forward reads the logits once (16 bytes a load); the backward
// reads them again and writes the gradient.  Differences from the row's maximum are formed first and scaled then, so that
// logits far from zero lose nothing and a row of nothing but the type's lowest value is an even one; an entry of minus
// infinity counts 0 in l, w and the gradient.  A row with a NaN, with plus infinity or with nothing but minus infinity is
// NaN, as a softmax of it is.
//
// Top alternatives: in order of (value, lowest index), NaN before numbers.  The first pass leaves the largest values of 32
// groups (of a lane each where a warp has a row, else of 8 lanes or of a warp); the top-th largest of those is at most the
// top-th largest value of the row, and few values lie above it (about 32 H_32 - 32 H_(32 - top) on independent ones), so a
// second pass, out of L1 and L2, collects what is not below it and ranks it.  Where a warp has a row it looks only at the vectors of lanes that have
// any (16384 rows of 2048 in bf16, top 8: 23.4 us, 28.9 with a second pass over the whole row), takes its floor from
// every lane's two largest where the top are many and halves what is left (top 32: 42.9 us; 65.5 without the second
// values, 104 without either).  Where ties or hostile orders leave more than there is room for, every warp keeps a sorted
// list instead, one entry a lane.
//
// What bounds them, in bf16: the forward at 65536 x 2048 (51 us, 5.2 TB/s) its instructions, with 2^t on a unit of 16 a
// clock taking 30 us alone; the backward there (80 us, 6.7 TB/s read and written) HBM; 16384 x 2048 without alternatives
// 14.4 us; one row of 2048 (2.6 us, with alternatives 4) the latency of a launch, of two dependent reads and of reductions.
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
  float* stats;  // [rows][2]: m and log2 l, or null
};

// 16 bytes of a row: `n` elements.  top() is the largest of them, NaN only where all are; or_nan() NaN where any is.
template <typename T>
struct Vec {
  static constexpr int n = 8;
  using Two = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>;
  static DA_DEV Two two(uint32_t u) { return *reinterpret_cast<Two*>(&u); }
  static DA_DEV uint32_t bits(Two v) { return *reinterpret_cast<uint32_t*>(&v); }
  static DA_DEV uint4 none() {
    constexpr uint32_t w = std::is_same<T, __nv_bfloat16>::value ? 0xff80ff80u : 0xfc00fc00u;
    return make_uint4(w, w, w, w);
  }
  static DA_DEV float top(uint4 w) {
    const float2 f = unpack2<T>(bits(__hmax2(__hmax2(two(w.x), two(w.y)), __hmax2(two(w.z), two(w.w)))));
    return fmaxf(f.x, f.y);
  }
  static DA_DEV float or_nan(uint4 w) {
    const float2 f = unpack2<T>(bits(__hmax2_nan(__hmax2_nan(two(w.x), two(w.y)), __hmax2_nan(two(w.z), two(w.w)))));
    return f.x != f.x ? f.x : f.y != f.y ? f.y : fmaxf(f.x, f.y);
  }
  static DA_DEV F2 pair(uint4 w, int i) { return widen<T>(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w); }
  static DA_DEV float one(const T* p) { return unpack2<T>(*reinterpret_cast<const uint16_t*>(p)).x; }
  static DA_DEV uint4 put(const float* x) {
    return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
};
template <>
struct Vec<float> {
  static constexpr int n = 4;
  static DA_DEV uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static DA_DEV float top(uint4 w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static DA_DEV float or_nan(uint4 w) {
    const float a = __uint_as_float(w.x), b = __uint_as_float(w.y), c = __uint_as_float(w.z), d = __uint_as_float(w.w);
    return a != a || b != b || c != c || d != d ? NAN : top(w);
  }
  static DA_DEV F2 pair(uint4 w, int i) {
    return i == 0 ? f2(__uint_as_float(w.x), __uint_as_float(w.y)) : f2(__uint_as_float(w.z), __uint_as_float(w.w));
  }
  static DA_DEV float one(const float* p) { return *p; }
  static DA_DEV uint4 put(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <typename V>
DA_DEV void values(uint4 w, float* x) {
#pragma unroll
  for (int i = 0; i < V::n / 2; ++i) split(V::pair(w, i), x[2 * i], x[2 * i + 1]);
}

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

// The larger of two, NaN where either is.
DA_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
constexpr float kFar = -10000.f;  // 2^t is 0 there, and 2^t t too, as for t of minus infinity it would not be

// Running sums against a running maximum m of the logits: t = (x - m) log2 e, the difference first.
struct Sums {
  float m, l, w;  // maximum, sum of 2^t, sum of 2^t t
  DA_DEV void raise(float to) {
    if (to > m) {
      if (m != -INFINITY) {
        const float d = fmaxf((m - to) * kLog2e, kFar), c = ex2(d);
        w = c * fmaf(l, d, w);
        l *= c;
      }
      m = to;
    }
  }
  // k vectors at once; their largest value.
  template <typename V, int k>
  DA_DEV float add(const uint4* raw) {
    float top = V::top(raw[0]);
#pragma unroll
    for (int i = 1; i < k; ++i) top = fmaxf(top, V::top(raw[i]));
    raise(top);
    const F2 at = dup(m == -INFINITY ? 0.f : -m), scale = dup(kLog2e);
    F2 ls = f2(l, 0.f), ws = f2(w, 0.f);
#pragma unroll
    for (int i = 0; i < k; ++i) {
#pragma unroll
      for (int j = 0; j < V::n / 2; ++j) {
        float a, b;
        split(mul2(add2(V::pair(raw[i], j), at), scale), a, b);
        a = max_nan(a, kFar);
        b = max_nan(b, kFar);
        const F2 e = f2(ex2(a), ex2(b));
        ls = add2(ls, e);
        ws = fma2(e, f2(a, b), ws);
      }
    }
    float a, b;
    split(ls, a, b);
    l = a + b;
    split(ws, a, b);
    w = a + b;
    return top;
  }
  DA_DEV void add_one(float x) {
    raise(x);
    const float t = max_nan((x - (m == -INFINITY ? 0.f : m)) * kLog2e, kFar), e = ex2(t);
    l += e;
    w = fmaf(e, t, w);
  }
  // Over the warp.
  DA_DEV void reduce() {
    float top = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    raise(top);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, o);
      w += __shfl_xor_sync(0xffffffffu, w, o);
    }
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

// The lanes' values (no NaN) sorted over the warp, the smallest first.
DA_DEV float sorted(float x) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, x, j);
      const bool low = ((lane & j) == 0) == ((lane & k) == 0 || k == 32);
      x = low ? fminf(x, o) : fmaxf(x, o);
    }
  return x;
}
// The top-th largest of them, in every lane.
DA_DEV float nth_largest(float x, int top) { return __shfl_sync(0xffffffffu, sorted(x), 32 - top); }
// The top-th largest of the lanes' firsts and seconds, no second larger than its first: of i firsts and top - i seconds,
// the smallest is at most it, and is it for one i.
DA_DEV float nth_largest(float first, float second, int top) {
  const int lane = threadIdx.x % 32;
  const float a = __shfl_sync(0xffffffffu, sorted(first), 31 - lane);  // the (lane + 1)-th largest
  const float b = __shfl_sync(0xffffffffu, sorted(second), (33 - top + lane) & 31);
  float x = lane >= top ? -INFINITY : lane == top - 1 ? a : fminf(a, b);
#pragma unroll
  for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// kThreads a row: 32 (eight rows a CTA), 256 or 1024.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads == 1024 ? 1024 : 256, kThreads == 1024 ? 1 : 6) forward_kernel(const Params p) {
  using V = Vec<T>;
  constexpr int kBatch = 4;  // loads in flight a thread, their largest value found together
  constexpr int kFound = kThreads == 32 ? 256 : 1024;  // entries that a row has room for
  __shared__ Sums sums[32];
  __shared__ float groups[32];
  __shared__ uint64_t found_all[kThreads == 32 ? 8 : 1][kFound];
  __shared__ int counts[kThreads == 32 ? 8 : 1];
  __shared__ int lanes_all[kThreads == 32 ? 8 : 1][32];
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int tid = kThreads == 32 ? lane : threadIdx.x;
  const int64_t r = kThreads == 32 ? (int64_t)blockIdx.x * 8 + warp : blockIdx.x;
  if (kThreads == 32 && r >= p.rows) return;
  uint64_t* found = found_all[kThreads == 32 ? warp : 0];
  int* count = &counts[kThreads == 32 ? warp : 0];
  auto meet = [] {
    if constexpr (kThreads == 32) __syncwarp();
    else __syncthreads();
  };
  if (tid == 0) *count = 0;
  const Row<T> row(p.logits, r * p.ld, p.V);
  Sums s{-INFINITY, 0.f, 0.f};
  float second = -INFINITY;  // where a warp has a row: the lane's largest value but for the vectors with the largest
  {
    const int odd = row.odd(tid);
    float x = -INFINITY;
    if (odd >= 0) x = V::one(row.p + odd);
    int v = tid;
    if constexpr (kThreads == 32) {
      // (a turn with vectors that are not there costs a warp as much as a full one: the last ones go singly.  A CTA, of
      // which there are few, has them all in flight instead)
      for (; v - lane + (kBatch - 1) * 32 < row.vecs; v += kBatch * 32) {
        uint4 raw[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) raw[i] = v + i * 32 < row.vecs ? row.load(v + i * 32) : V::none();
        const float before = s.m;
        second = fmaxf(second, fminf(before, s.add<V, kBatch>(raw)));
      }
#pragma unroll 1
      for (; v - lane < row.vecs; v += 32) {
        const uint4 raw = v < row.vecs ? row.load(v) : V::none();
        const float before = s.m;
        second = fmaxf(second, fminf(before, s.add<V, 1>(&raw)));
      }
    }
    for (; v < row.vecs; v += kBatch * kThreads) {
      uint4 raw[kBatch];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) raw[i] = v + i * kThreads < row.vecs ? row.load(v + i * kThreads) : V::none();
      s.add<V, kBatch>(raw);
    }
    if (odd >= 0) s.add_one(x);
  }
  float group = s.m;  // lane i: group i's largest value; a group is a lane, or 8 lanes, or a warp
  if constexpr (kThreads == 256) {
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, o));
    if (lane % 8 == 0) groups[threadIdx.x / 8] = group;
  }
  s.reduce();
  if constexpr (kThreads > 32) {
    if (lane == 0) sums[warp] = s;
    __syncthreads();
    s = lane < kThreads / 32 ? sums[lane] : Sums{-INFINITY, 0.f, 0.f};
    group = kThreads == 256 ? groups[lane] : s.m;
    s.reduce();
  }
  const float at = s.m == -INFINITY ? 0.f : s.m, log_l = log2f(s.l);
  if (tid == 0) {
    const int64_t token = p.tokens[r];
    float lp = token == kIgnore ? 0.f : NAN;
    if (token >= 0 && token < p.V) lp = V::one(row.p + token) - at - log_l * kLn2;
    p.log_probs[r] = lp;
    p.entropy[r] = (log_l - s.w / s.l) * kLn2;
    if (p.stats) reinterpret_cast<float2*>(p.stats)[r] = make_float2(at, log_l);
  }
  if (p.top == 0) return;

  // (few more than the top are above the floor of 32 values where the top are few: 9 for 8, but 130 for 32; of 64, 44)
  float floor = kThreads == 32 && p.top > 8 ? nth_largest(group, second, p.top) : nth_largest(group, p.top);
  meet();
  auto write = [&](uint64_t e, int rank) {
    p.top_log_probs[r * p.top + rank] = value_of((uint32_t)(e >> 32)) - at - log_l * kLn2;
    p.top_tokens[r * p.top + rank] = (uint32_t)~(uint32_t)e;
  };
  {
    auto take = [&](float x, int index) {
      const int i = atomicAdd(count, 1);
      if (i < kFound) found[i] = entry_of(x, index);
    };
    auto look = [&](int v) {
      const uint4 raw = row.load(v);
      if (V::or_nan(raw) < floor) return;
      float x[V::n];
      values<V>(raw, x);
      const int index = row.index(v);
      uint32_t in = 0;
#pragma unroll
      for (int i = 0; i < V::n; ++i) in |= (uint32_t)!(x[i] < floor) << i;
      for (; in; in &= in - 1) {
        const int i = index + __ffs(in) - 1;
        take(V::one(row.p + i), i);
      }
    };
    if constexpr (kThreads == 32) {
      // Only lanes whose largest value is not below the floor have any (and, in a row with a NaN, which that value
      // passes over, all may): their vectors, dealt out to the whole warp.
      const bool has = !(group < floor) || s.l != s.l;
      const uint32_t who = __ballot_sync(0xffffffffu, has);
      const int k = __popc(who), bits = 32 - __clz(k - 1);  // (a floor is some lane's value: k > 0)
      int* lanes = lanes_all[warp];
      if (has) lanes[__popc(who & ((1u << lane) - 1))] = lane;
      __syncwarp();
      const int f = lane & ((1 << bits) - 1);
      if (f < k)
        for (int v = lanes[f] + (lane >> bits) * 32; v < row.vecs; v += 1024 >> bits) look(v);
    } else {
#pragma unroll 2
      for (int v = tid; v < row.vecs; v += kThreads) look(v);
    }
    const int odd = row.odd(tid);
    if (odd >= 0) {
      const float x = V::one(row.p + odd);
      if (!(x < floor)) take(x, odd);
    }
  }
  meet();
  int n = *count;
  if constexpr (kThreads == 32) {
    // Ranking takes n^2 / 32 comparisons a lane: where that is many, a higher floor first, halving between this one and
    // the largest until at most `most` of them are left (or no fewer can be, as of equal ones).
    const int most = p.top <= 16 ? 32 : 64;
    if (n > 64 && n <= kFound) {
      uint32_t lo = order_of(floor), hi = 0;
      for (int k = lane; k < n; k += 32) hi = max(hi, (uint32_t)(found[k] >> 32));
      hi = __reduce_max_sync(0xffffffffu, hi);
      while (lo < hi) {  // top or more are not below lo, fewer above hi
        const uint32_t mid = hi - (hi - lo) / 2;
        int c = 0;
        for (int k = lane; k < n; k += 32) c += (uint32_t)(found[k] >> 32) >= mid;
        c = __reduce_add_sync(0xffffffffu, c);
        if (c < p.top) {
          hi = mid - 1;
        } else {
          lo = mid;
          if (c <= most) break;
        }
      }
      int left = 0;
      for (int k = 0; k < n; k += 32) {  // to the front, never past what has been read
        const uint64_t e = k + lane < n ? found[k + lane] : 0;
        const bool in = k + lane < n && (uint32_t)(e >> 32) >= lo;
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (in) found[left + __popc(who & ((1u << lane) - 1))] = e;
        left += __popc(who);
      }
      __syncwarp();
      n = left;
    }
  }
  if (n <= kFound) {
    for (int k = tid; k < n; k += kThreads) {  // no two entries are alike: every one has its rank, in whatever place it lies
      const uint64_t e = found[k];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += found[i] > e;
      if (rank < p.top) write(e, rank);
    }
    return;
  }
  // More than there is room for, as where many are equal: sorted lists of the largest, a warp each, taken in as they come.
  List list{0, 0};
  const int all = (row.vecs + kThreads - 1) / kThreads * kThreads;  // every lane takes every turn
  for (int v = tid; v < all; v += kThreads) {
    const bool in = v < row.vecs;
    const uint4 raw = in ? row.load(v) : V::none();
    if (!__ballot_sync(0xffffffffu, in && !(V::or_nan(raw) < floor))) continue;
    float x[V::n];
    values<V>(raw, x);
#pragma unroll
    for (int i = 0; i < V::n; ++i) list.offer(x[i], row.index(v) + i, in, floor, p.top);
  }
  {
    const int odd = row.odd(tid);
    list.offer(odd >= 0 ? V::one(row.p + odd) : 0.f, odd, odd >= 0, floor, p.top);
  }
  if constexpr (kThreads == 32) {
    if (lane < p.top) write(list.mine, lane);
  } else {
    __syncthreads();
    found[threadIdx.x] = lane < p.top ? list.mine : 0;
    __syncthreads();
    const uint64_t e = found[threadIdx.x];
    if (!e) return;
    int rank = 0;
    for (int i = 0; i < kThreads; ++i) rank += found[i] > e;
    if (rank < p.top) write(e, rank);
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
    const float t = max_nan((x - st.x) * kLog2e - st.y, kFar);  // log2 p
    const float d = -ex2(t) * fmaf(h, t, c);
    return i == token ? d + g : d;
  };
  constexpr int kVecs = kSegment / V::n, kBatch = 4;
  const int v0 = seg * kVecs, v1 = min(row.vecs, v0 + kVecs);
  if (token == kIgnore && h == 0.f) {  // zeros, whatever the row holds
    for (int i = row.index(v0) + lane; i < row.index(v1); i += 32) out[i] = T(0.f);
    if (seg == 0 && row.odd(lane) >= 0) out[row.odd(lane)] = T(0.f);
    return;
  }
  const F2 scale = dup(kLog2e), at_m = dup(-st.x), at_l = dup(-st.y), hs = dup(-h), cs = dup(-c);
  for (int v = v0 + lane; v < v1; v += 32 * kBatch) {
    uint4 raw[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) raw[k] = v + 32 * k < v1 ? row.load(v + 32 * k) : V::none();
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      if (v + 32 * k >= v1) break;
      const int at = row.index(v + 32 * k);
      float x[V::n];
#pragma unroll
      for (int i = 0; i < V::n / 2; ++i) {
        float a, b;
        split(fma2(add2(V::pair(raw[k], i), at_m), scale, at_l), a, b);  // log2 p
        a = max_nan(a, kFar);
        b = max_nan(b, kFar);
        split(mul2(f2(ex2(a), ex2(b)), fma2(hs, f2(a, b), cs)), x[2 * i], x[2 * i + 1]);
      }
      if (token - at >= 0 && token - at < V::n) {
#pragma unroll
        for (int i = 0; i < V::n; ++i)
          if (at + i == token) x[i] += g;
      }
      const uint4 w = V::put(x);
      if (wide) {
        *reinterpret_cast<uint4*>(out + at) = w;
      } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < V::n; ++i) out[at + i] = x[i];
      } else {
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<uint16_t*>(out)[at + i] = (uint16_t)(q[i / 2] >> (16 * (i & 1)));
      }
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

int check(const void* logits, int dtype, int64_t rows, int64_t V, const void* tokens) {
  if (dtype != DA_F16 && dtype != DA_BF16 && dtype != DA_F32) return DA_ERR_DTYPE;
  if (rows < 0 || rows > 0x7fffffff || V < 1 || V > 0x7fffff00) return DA_ERR_SHAPE;
  if (rows && (!logits || !tokens)) return DA_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == DA_F32 ? 4 : 2)) return DA_ERR_ALIGN;
  return DA_OK;
}

// How many threads take a row.  In 16-byte pieces of a row (8 elements of 16 bits): 32 where there are rows enough for that,
// pieces^2 / 312 (16384 x 2048 in bf16: 15 us with 32 threads, 63 with 256, 240 with 1024; 4096 x 8192: 20, 18, 91; 64 x 8192:
// 6.8, 2.7, 4.0), and where 256 threads would not have a piece for each of top groups of 8 (64 x 500, top 20: 4.7, 12.6,
// 11.4).  1024 for rows of more than 2048 pieces, two an SM at most (64 x 50021: 32, 6.3, 5.7; 600 x 50021: 33, 17, 24).
template <typename T>
int forward(const Params& p, cudaStream_t st) {
  const int64_t pieces = p.V / Vec<T>::n;
  const int threads = p.rows * 312 >= pieces * pieces || pieces < 8 * p.top  ? 32
                      : pieces > 2048 && p.rows <= 2 * (int64_t)sm_count() ? 1024
                                                                           : 256;
  if (threads == 32)
    return launch_kernel(forward_kernel<T, 32>, dim3((unsigned)((p.rows + 7) / 8)), dim3(256), 0, st, false, p);
  if (threads == 256) return launch_kernel(forward_kernel<T, 256>, dim3((unsigned)p.rows), dim3(256), 0, st, false, p);
  return launch_kernel(forward_kernel<T, 1024>, dim3((unsigned)p.rows), dim3(1024), 0, st, false, p);
}

}  // namespace score
}  // namespace da

extern "C" int da_token_log_probs(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t V, const int64_t* tokens,
                                  int top, float* log_probs, float* entropy, float* top_log_probs, int64_t* top_tokens,
                                  float* stats, void* stream) {
  using namespace da;
  if (int rc = score::check(logits, dtype, rows, V, tokens)) return rc;
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
  if (int rc = score::check(logits, dtype, rows, V, tokens)) return rc;
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

// Statistics of given tokens under rows of logits, and their gradient.
//
// For a row x [V] with target t, temperature T and k alternatives (m = max x, d_j = (x_j - m) / T, s = sum e^d_j,
// u = sum e^d_j d_j, p = softmax(x / T)):
//   log p(t)  = d_t - log s
//   entropy   = -sum p log p = log s - u / s
//   top i     = the i-th largest x (ties: lowest index first), log p = d - log s
//   T d/dx_j  = g_lp (1[j = t] - p_j) - g_ent p_j (log p_j + H) + sum_i g_i (1[j = id_i] - p_j)
// 1 / T is applied in fp32 to the logits as they are read, as the sampler does: dividing bf16 logits first would round
// them a second time, which at T 0.7 moves a log-prob by 0.009 on average.
// (m, log s) are kept apart for the backward: their sum would round away bits of log s at large m.
//
// Forward: one pass, in the log2 domain about c = fl(m k), k = log2e / T.  One FMA forms y_j = x_j k - c, so
// s' = sum 2^y and u' = sum 2^y y share one offset delta = m k - c (known exactly from another FMA):
// entropy = ln2 (log2 s' - u' / s') does not depend on it, log s = ln2 (log2 s' - delta).  An element
// costs an FMA, an exponential, an add and an FMA; with about 8 cycles a warp the exponential (MUFU) is
// the most of it, 16 elements a cycle and SM, against 11.6 that memory delivers.  A thread keeps (m, s', u')
// of its elements and raises m only when a 16-byte vector holds a larger value.  Values below -1e6 (masked
// tokens) count as -1e6 there; a row with nothing above that, or of a temperature far from 1, is done again exactly.  The alternatives ride along without a second pass over
// the row: the k-th largest of the 32 half-warp maxima bounds the k-th largest element from
// below, so only threads whose own maximum reaches that bound look at their elements again
// (about k of them), and the few candidates are ranked in shared memory.
// Rows whose target is the ignore index are not read at all: zeros, ids -1, zero gradient.
//
// Measured (L2 flushed) at 12288 x 50304 bf16 with a quarter of the rows unscored: forward 242 us (0.93 GB,
// 3.8 TB/s), forward and gradient 570 us (3.09 GB with the second read, 5.4 TB/s).
#include "common/host_utils.h"
#include "common/ptx.cuh"
#include "common/fast_exp2.cuh"

#include <cmath>

namespace tt {
namespace stats {

constexpr int kThreads = 512;
constexpr int kGroups = 32;    // half-warp maxima that bound the k-th largest element
constexpr int kMaxTop = 32;
constexpr int kMaxCand = 512;  // candidates ranked in shared memory; more (mass ties): the slow path
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
static_assert(kThreads / 16 == kGroups && kMaxTop <= kGroups, "one bound per half warp");

template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kVec = 8;
  __device__ static float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static void unpack(const uint4& q, float (&v)[8]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
  __device__ static __nv_bfloat16 round(float x) { return __float2bfloat16_rn(x); }
  // Values of a vector, those below the floor raised to it (a NaN stays), and the largest (NaN left out).
  __device__ static float floored(const uint4& q, float (&v)[8]) {
    constexpr uint32_t kLow = 0xc974c974u;  // bf16 pair of -999424
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t m;
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(kLow));
    uint32_t a, b;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(a) : "r"(w[0]), "r"(w[1]));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(b) : "r"(w[2]), "r"(w[3]));
    asm("max.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    unpack(make_uint4(w[0], w[1], w[2], w[3]), v);
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
};
template <>
struct Elem<float> {
  static constexpr int kVec = 4;
  __device__ static float one(const float* p) { return *p; }
  __device__ static void unpack(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x);
    v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z);
    v[3] = __uint_as_float(q.w);
  }
  __device__ static uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  __device__ static float round(float x) { return x; }
  __device__ static float floored(const uint4& q, float (&v)[4]) {
    unpack(q, v);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(v[i]) : "f"(-1e6f));
      m = fmaxf(m, v[i]);
    }
    return m;
  }
};

// Order of the values as unsigned integers: NaN lowest (0), then -inf .. +inf; -0 equals +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 + 0 = +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// (value, lower index first) as one integer.
__device__ __forceinline__ unsigned long long cand_key(float x, int idx) {
  return (static_cast<unsigned long long>(order_key(x)) << 32) | static_cast<uint32_t>(~idx);
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr float kFloor = -1e6f;  // what lower values count as in the first pass
constexpr float kFar = 9e5f;     // a row whose maximum is further from zero is summed again exactly (c would round too much)
// Temperatures of the one-pass sums.  Up to T = 100 a floored value (1e5 below a maximum above -kFar) is still e^-1000; down
// to T = 0.001 the c of a thread of masked tokens only (1e6 k) is rounded by at most 64, so its 2^y stay finite and the factor
// that drops them is a zero times a number.
constexpr float kMinInvT = 0.01f, kMaxInvT = 1000.0f;

struct Acc {
  float k = kLog2e;  // log2e / T
  float m = -INFINITY, c = 0.0f, s = 0.0f, u = 0.0f;
  __device__ __forceinline__ explicit Acc(float k_) : k(k_) {}
  // Moves the sums from reference `from` to a larger one.
  __device__ __forceinline__ void shift(float from, float to) {
    const float dc = from - to;
    const float f = ex2_mufu(dc);
    u = f == 0.0f ? 0.0f : f * fmaf(dc, s, u);  // dc may be -inf
    s *= f;                                     // a NaN of s stays
  }
  __device__ __forceinline__ void raise(float m2) {  // m2 > m
    const float c2 = m2 * k;
    if (m != -INFINITY) shift(c, c2);
    m = m2;
    c = c2;
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = fmaf(v[i], k, -c);
      const float e = ex2_mufu(y);
      s += e;
      u = fmaf(e, y, u);
    }
  }
  __device__ __forceinline__ void merge(float m2, float s2, float u2) {
    float c2 = m2 == -INFINITY ? 0.0f : m2 * k;
    if (m2 > m) {
      const float a = m, d = c, x = s, y = u;
      m = m2, c = c2, s = s2, u = u2;
      m2 = a, c2 = d, s2 = x, u2 = y;
    }
    if (m2 != -INFINITY) {
      const float dc = c2 - c;
      const float f = ex2_mufu(dc);
      s += f * s2;
      if (f != 0.0f) u += f * fmaf(dc, s2, u2);
    } else {
      s += s2;  // zero, or the NaN of elements that have no maximum
    }
  }
};

// The same sums in natural units about a known maximum, for rows of only masked tokens.
struct AccExact {
  float inv_t = 1.0f, m = -INFINITY, s = 0.0f, u = 0.0f;
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
    const float mm = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = max_nan((v[i] - mm) * inv_t, -1e30f);
      const float e = ex2_mufu(d * kLog2e);
      s += e;
      u = fmaf(e, d, u);
    }
  }
};

__device__ __forceinline__ float block_sum(float v, float* scratch, int lane, int warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < kThreads / 32; ++w) v += scratch[w];
  return v;
}
__device__ __forceinline__ float block_max(float v, float* scratch, int lane, int warp) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = scratch[0];
  for (int w = 1; w < kThreads / 32; ++w) v = fmaxf(v, scratch[w]);
  return v;
}

struct FwdArgs {
  const void* logits;
  long long ld;
  const int64_t* targets;
  int64_t ignore;
  int N, V, k;
  float inv_t;
  float* lp;
  float* ent;
  float* ms;        // [N, 2]: m, log s
  float* top_lp;    // [N, k]
  int64_t* top_id;  // [N, k]
  int* status;
};

// Calls f(first index, elements) for this thread's pieces of the row: 16-byte vectors between
// the first aligned element and the last, single elements around them (rows need not be aligned).
template <typename T>
struct RowSplit {
  int head, nvec;
  const uint4* body;
  const T* x;
  int V;
  __device__ RowSplit(const T* row, int V_) : x(row), V(V_) {
    constexpr int kVec = Elem<T>::kVec;
    const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = min(V, mis ? kVec - mis : 0);
    nvec = (V - head) / kVec;
    body = reinterpret_cast<const uint4*>(row + head);
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) token_stats_fwd_kernel(const FwdArgs a) {
  constexpr int kVec = Elem<T>::kVec;
  __shared__ float red[3][kThreads / 32];
  __shared__ uint32_t gmax[kGroups];
  __shared__ unsigned long long cand[kMaxCand];
  __shared__ unsigned long long best[kThreads / 32];
  __shared__ int n_cand;
  __shared__ uint32_t bound_s;
  __shared__ float total[3];
  const int row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t = a.targets[row];
  if (t < 0 || t >= a.V || t == a.ignore) {  // not scored (uniform over the block)
    if (tid == 0) {
      if (t != a.ignore) atomicCAS(a.status, 0, static_cast<int>(kBadIndex));
      a.lp[row] = 0.0f;
      a.ent[row] = 0.0f;
      a.ms[2 * static_cast<long long>(row)] = 0.0f;
      a.ms[2 * static_cast<long long>(row) + 1] = 0.0f;
    }
    if (tid < a.k) {
      a.top_lp[static_cast<long long>(row) * a.k + tid] = 0.0f;
      a.top_id[static_cast<long long>(row) * a.k + tid] = -1;
    }
    return;
  }
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  const RowSplit<T> rs(x, a.V);
  const int tail = rs.head + rs.nvec * kVec;
  if (tid == 0) n_cand = 0;
  const float kt = kLog2e * a.inv_t;
  Acc acc(kt);
  auto take = [&](const uint4& q) {
    float v[kVec];
    const float vm = Elem<T>::floored(q, v);
    if (vm > acc.m) acc.raise(vm);
    acc.add(v);
  };
  int i = tid;
  for (; i + 3 * kThreads < rs.nvec; i += 4 * kThreads) {  // four loads in flight
    const uint4 q0 = rs.body[i], q1 = rs.body[i + kThreads], q2 = rs.body[i + 2 * kThreads], q3 = rs.body[i + 3 * kThreads];
    take(q0);
    take(q1);
    take(q2);
    take(q3);
  }
  for (; i < rs.nvec; i += kThreads) take(rs.body[i]);
  // the unaligned ends: at most kVec - 1 elements each
  const int edge = tid < rs.head ? tid : (tid - rs.head + tail);
  const bool has_edge = edge < a.V && (tid < rs.head || tid - rs.head < a.V - tail);
  if (has_edge) {
    const float v[1] = {max_nan(Elem<T>::one(x + edge), kFloor)};
    if (v[0] > acc.m) acc.raise(v[0]);
    acc.add(v);
  }
  const uint32_t own_max = acc.m == -INFINITY ? 0u : order_key(acc.m);
  if (a.k > 0) {
    uint32_t g = own_max;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if ((lane & 15) == 0) gmax[tid >> 4] = g;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, acc.m, o);
    const float s2 = __shfl_xor_sync(0xffffffffu, acc.s, o);
    const float u2 = __shfl_xor_sync(0xffffffffu, acc.u, o);
    acc.merge(m2, s2, u2);
  }
  if (lane == 0) {
    red[0][warp] = acc.m;
    red[1][warp] = acc.s;
    red[2][warp] = acc.u;
  }
  __syncthreads();
  if (warp == 0) {  // the warps' sums, in the order of a fixed tree
    Acc w(kt);
    if (lane < kThreads / 32) w.merge(red[0][lane], red[1][lane], red[2][lane]);
#pragma unroll
    for (int o = kThreads / 64; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, w.m, o);
      const float s2 = __shfl_xor_sync(0xffffffffu, w.s, o);
      const float u2 = __shfl_xor_sync(0xffffffffu, w.u, o);
      w.merge(m2, s2, u2);
    }
    if (lane == 0) {
      total[0] = w.m;
      total[1] = w.s;
      total[2] = w.u;
    }
    if (a.k > 0) {  // the k-th largest of the 32 maxima (ties by position)
      const uint32_t mine = gmax[lane];
      int rank = 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const uint32_t other = __shfl_sync(0xffffffffu, mine, j);
        rank += (other > mine || (other == mine && j < lane)) ? 1 : 0;
      }
      // a maximum at the floor says nothing about values below it: all are candidates
      if (rank == a.k - 1) bound_s = mine <= order_key(-kFar) ? 0u : mine;
    }
  }
  __syncthreads();
  Acc all(kt);
  all.m = total[0];
  all.c = all.m == -INFINITY ? 0.0f : all.m * kt;
  all.s = total[1];
  all.u = total[2];
  float row_max = all.m, log_s, entropy;
  if (fabsf(all.m) < kFar && fabsf(all.m) * a.inv_t < kFar && a.inv_t >= kMinInvT && a.inv_t <= kMaxInvT) {
    const float log2_s = log2f(all.s);
    log_s = kLn2 * (log2_s - fmaf(all.m, kt, -all.c));
    entropy = kLn2 * (log2_s - all.u / all.s);
  } else {  // nothing but masked tokens (or NaN), or values near the type's end: the sums about the row's own maximum
    float m = -INFINITY;
    for (int j = tid; j < a.V; j += kThreads) m = fmaxf(m, Elem<T>::one(x + j));
    row_max = block_max(m, red[0], lane, warp);
    AccExact ex;
    ex.inv_t = a.inv_t;
    ex.m = row_max;
    for (int j = tid; j < a.V; j += kThreads) {
      const float v[1] = {Elem<T>::one(x + j)};
      ex.add(v);
    }
    ex.s = block_sum(ex.s, red[1], lane, warp);
    ex.u = block_sum(ex.u, red[2], lane, warp);
    log_s = row_max == -INFINITY ? NAN : logf(ex.s);  // nothing above -inf: 0 / 0
    entropy = log_s - ex.u / ex.s;
  }
  all.m = row_max;
  if (tid == 0) {
    a.lp[row] = fmaf(Elem<T>::one(x + t) - all.m, a.inv_t, -log_s);
    a.ent[row] = entropy;
    a.ms[2 * static_cast<long long>(row)] = all.m;
    a.ms[2 * static_cast<long long>(row) + 1] = log_s;
  }
  if (a.k == 0) return;
  const uint32_t bound = bound_s;
  auto offer = [&](float v, int idx) {
    if (order_key(v) >= bound) {
      const int at = atomicAdd(&n_cand, 1);
      if (at < kMaxCand) cand[at] = cand_key(v, idx);
    }
  };
  if (own_max >= bound) {
    for (int j = tid; j < rs.nvec; j += kThreads) {
      const uint4 q = rs.body[j];
      float v[kVec];
      if (order_key(Elem<T>::floored(q, v)) < bound) continue;  // most vectors
      Elem<T>::unpack(q, v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) offer(v[e], rs.head + j * kVec + e);
    }
    if (has_edge) offer(Elem<T>::one(x + edge), edge);
  }
  __syncthreads();
  const int n = n_cand;
  float* top_lp = a.top_lp + static_cast<long long>(row) * a.k;
  int64_t* top_id = a.top_id + static_cast<long long>(row) * a.k;
  auto emit = [&](int r, unsigned long long key) {
    const int idx = static_cast<int>(~static_cast<uint32_t>(key));
    top_id[r] = idx;
    top_lp[r] = fmaf(Elem<T>::one(x + idx) - all.m, a.inv_t, -log_s);
  };
  if (n <= kMaxCand) {  // rank of each candidate among all (the keys are distinct)
    if (tid < n) {
      const unsigned long long mine = cand[tid];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += cand[j] > mine ? 1 : 0;
      if (rank < a.k) emit(rank, mine);
    }
    return;
  }
  // Mass ties at the bound: k passes, each the largest key below the previous one.
  unsigned long long below = ~0ull;
  for (int r = 0; r < a.k; ++r) {
    unsigned long long b = 0;
    for (int j = tid; j < a.V; j += kThreads) {
      const unsigned long long key = cand_key(Elem<T>::one(x + j), j);
      if (key < below && key > b) b = key;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, b, o);
      b = other > b ? other : b;
    }
    if (lane == 0) best[warp] = b;
    __syncthreads();
    b = best[0];
    for (int w = 1; w < kThreads / 32; ++w) b = best[w] > b ? best[w] : b;
    if (tid == 0) emit(r, b);
    below = b;
    __syncthreads();
  }
}

struct BwdArgs {
  const void* logits;
  long long ld;
  const int64_t* targets;
  int64_t ignore;
  int N, V, k;
  float inv_t;
  const float* ent;
  const float* ms;
  const int64_t* top_id;
  const float* g_lp;   // each may be null
  const float* g_ent;
  const float* g_top;
  void* grad;          // [N, V] contiguous
};

// One block per row: p_j (pull + g_ent log p_j) over the row, then the entries of the target and
// the alternatives once more with their one-hot parts (an index can be both).
template <typename T>
__global__ void __launch_bounds__(kThreads) token_stats_bwd_kernel(const BwdArgs a) {
  constexpr int kVec = Elem<T>::kVec;
  const int row = blockIdx.x, tid = threadIdx.x;
  const int64_t t = a.targets[row];
  const bool scored = t >= 0 && t < a.V && t != a.ignore;
  const T* x = static_cast<const T*>(a.logits) + row * a.ld;
  T* g = static_cast<T*>(a.grad) + static_cast<long long>(row) * a.V;
  const RowSplit<T> out(g, a.V);
  const int tail = out.head + out.nvec * kVec;
  const int edge = tid < out.head ? tid : (tid - out.head + tail);
  const bool has_edge = edge < a.V && (tid < out.head || tid - out.head < a.V - tail);
  uint4* body = reinterpret_cast<uint4*>(g + out.head);
  if (!scored) {
    for (int i = tid; i < out.nvec; i += kThreads) body[i] = make_uint4(0u, 0u, 0u, 0u);
    if (has_edge) g[edge] = Elem<T>::round(0.0f);
    return;
  }
  const float m = a.ms[2 * static_cast<long long>(row)], log_s = a.ms[2 * static_cast<long long>(row) + 1];
  const float g_lp = a.g_lp != nullptr ? a.g_lp[row] : 0.0f;
  const float g_ent = a.g_ent != nullptr ? a.g_ent[row] : 0.0f;
  const float* g_top = a.g_top != nullptr ? a.g_top + static_cast<long long>(row) * a.k : nullptr;
  const int64_t* ids = a.top_id + static_cast<long long>(row) * a.k;
  float pull = fmaf(g_ent, a.ent[row], g_lp);
  if (g_top != nullptr)
    for (int i = 0; i < a.k; ++i) pull += g_top[i];
  // -p (pull + g_ent log p) / T; the floor keeps 0 * -inf out (see Acc::add)
  const float inv_t = a.inv_t, ge = g_ent * inv_t;
  pull *= inv_t;
  auto dense = [&](float v) {
    const float y = max_nan(fmaf(v - m, inv_t, -log_s), -1e30f);
    return -ex2_mufu(y * kLog2e) * fmaf(ge, y, pull);
  };
  // input vectors line up with the output's when both rows start at the same offset
  const bool aligned = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(g)) & 15) == 0;
  const uint4* in = reinterpret_cast<const uint4*>(x + out.head);
  auto one = [&](int i, const uint4& q) {
    float v[kVec];
    Elem<T>::unpack(q, v);
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = dense(v[e]);
    body[i] = Elem<T>::pack(v);
  };
  if (aligned) {
    int i = tid;
    for (; i + 3 * kThreads < out.nvec; i += 4 * kThreads) {
      const uint4 q0 = in[i], q1 = in[i + kThreads], q2 = in[i + 2 * kThreads], q3 = in[i + 3 * kThreads];
      one(i, q0);
      one(i + kThreads, q1);
      one(i + 2 * kThreads, q2);
      one(i + 3 * kThreads, q3);
    }
    for (; i < out.nvec; i += kThreads) one(i, in[i]);
  } else {
    for (int i = tid; i < out.nvec; i += kThreads) {
      float v[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = dense(Elem<T>::one(x + out.head + i * kVec + e));
      body[i] = Elem<T>::pack(v);
    }
  }
  if (has_edge) g[edge] = Elem<T>::round(dense(Elem<T>::one(x + edge)));
  __syncthreads();
  if (tid <= (g_top != nullptr ? a.k : 0)) {
    const int64_t idx = tid == 0 ? t : ids[tid - 1];
    if (idx >= 0 && idx < a.V) {
      float hot = idx == t ? g_lp : 0.0f;
      if (g_top != nullptr)
        for (int i = 0; i < a.k; ++i) hot += ids[i] == idx ? g_top[i] : 0.0f;
      g[idx] = Elem<T>::round(fmaf(hot, inv_t, dense(Elem<T>::one(x + idx))));
    }
  }
}

void check_logits(const torch::Tensor& logits, const torch::Tensor& targets, int64_t k) {
  TT_CHECK(logits.scalar_type() == torch::kBFloat16 || logits.scalar_type() == torch::kFloat32,
           "token_stats: logits must be bfloat16 or float32");
  TT_CHECK(logits.dim() == 2 && logits.stride(1) == 1 && logits.size(1) >= 1, "token_stats: logits must be [N, V], rows contiguous");
  TT_CHECK(logits.size(0) < (1LL << 31) && logits.size(1) < (1LL << 31) - 4 * kThreads * 8, "token_stats: too many rows or columns");
  TT_CHECK(targets.scalar_type() == torch::kInt64 && targets.is_contiguous() && targets.numel() == logits.size(0),
           "token_stats: targets must be contiguous int64 [N]");
  TT_CHECK(k >= 0 && k <= kMaxTop && k <= logits.size(1), "token_stats: top_k must be in [0, min(32, V)]");
}

const float* opt_f32(const c10::optional<torch::Tensor>& t, int64_t numel, const char* name) {
  if (!t.has_value()) return nullptr;
  TT_CHECK(t->scalar_type() == torch::kFloat32 && t->is_contiguous() && t->numel() == numel,
           std::string("token_stats_bwd: ") + name + " must be contiguous fp32");
  return t->data_ptr<float>();
}

float inverse(double temperature) {
  TT_CHECK(temperature > 0 && std::isfinite(temperature) && std::isfinite(static_cast<float>(1.0 / temperature)) &&
               static_cast<float>(1.0 / temperature) > 0,
           "token_stats: temperature must be positive and finite");
  return static_cast<float>(1.0 / temperature);
}

}  // namespace stats

// logits [N, V] (bf16 or fp32, any row stride), targets int64 [N] -> lp, ent fp32 [N], ms fp32 [N, 2],
// top_lp fp32 / top_id int64 [N, k] of softmax(logits / temperature).  Rows whose target is ignore_index are not scored.
void token_stats_fwd(torch::Tensor logits, torch::Tensor targets, int64_t k, int64_t ignore_index, double temperature,
                     torch::Tensor lp, torch::Tensor ent, torch::Tensor ms, torch::Tensor top_lp, torch::Tensor top_id) {
  using namespace stats;
  check_logits(logits, targets, k);
  const int64_t N = logits.size(0), V = logits.size(1);
  TT_CHECK(lp.scalar_type() == torch::kFloat32 && lp.is_contiguous() && lp.numel() == N &&
               ent.scalar_type() == torch::kFloat32 && ent.is_contiguous() && ent.numel() == N &&
               ms.scalar_type() == torch::kFloat32 && ms.is_contiguous() && ms.numel() == 2 * N &&
               top_lp.scalar_type() == torch::kFloat32 && top_lp.is_contiguous() && top_lp.numel() == N * k &&
               top_id.scalar_type() == torch::kInt64 && top_id.is_contiguous() && top_id.numel() == N * k,
           "token_stats: outputs fp32 [N], [N], [N, 2], [N, k] and int64 [N, k]");
  if (N == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  FwdArgs a{logits.data_ptr(), logits.stride(0), targets.data_ptr<int64_t>(), ignore_index, static_cast<int>(N),
            static_cast<int>(V), static_cast<int>(k), inverse(temperature), lp.data_ptr<float>(), ent.data_ptr<float>(), ms.data_ptr<float>(),
            top_lp.data_ptr<float>(), top_id.data_ptr<int64_t>(), device_status_ptr(logits.get_device())};
  if (logits.scalar_type() == torch::kBFloat16)
    token_stats_fwd_kernel<__nv_bfloat16><<<static_cast<unsigned>(N), kThreads, 0, cur_stream()>>>(a);
  else
    token_stats_fwd_kernel<float><<<static_cast<unsigned>(N), kThreads, 0, cur_stream()>>>(a);
  TT_CUDA_CHECK(cudaGetLastError());
}

// grad [N, V] (contiguous, the logits' type) of sum g_lp lp + g_ent ent + g_top top_lp.
void token_stats_bwd(torch::Tensor logits, torch::Tensor targets, int64_t k, int64_t ignore_index, double temperature,
                     torch::Tensor ent, torch::Tensor ms, torch::Tensor top_id, c10::optional<torch::Tensor> g_lp,
                     c10::optional<torch::Tensor> g_ent, c10::optional<torch::Tensor> g_top, torch::Tensor grad) {
  using namespace stats;
  check_logits(logits, targets, k);
  const int64_t N = logits.size(0), V = logits.size(1);
  TT_CHECK(grad.scalar_type() == logits.scalar_type() && grad.is_contiguous() && grad.dim() == 2 && grad.size(0) == N &&
               grad.size(1) == V,
           "token_stats_bwd: grad must be contiguous [N, V] of the logits' type");
  TT_CHECK(ent.scalar_type() == torch::kFloat32 && ent.is_contiguous() && ent.numel() == N &&
               ms.scalar_type() == torch::kFloat32 && ms.is_contiguous() && ms.numel() == 2 * N &&
               top_id.scalar_type() == torch::kInt64 && top_id.is_contiguous() && top_id.numel() == N * k,
           "token_stats_bwd: saved tensors");
  if (N == 0) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  BwdArgs a{logits.data_ptr(), logits.stride(0), targets.data_ptr<int64_t>(), ignore_index, static_cast<int>(N),
            static_cast<int>(V), static_cast<int>(k), inverse(temperature), ent.data_ptr<float>(), ms.data_ptr<float>(),
            top_id.data_ptr<int64_t>(), opt_f32(g_lp, N, "g_lp"), opt_f32(g_ent, N, "g_ent"),
            k > 0 ? opt_f32(g_top, N * k, "g_top") : nullptr, grad.data_ptr()};
  if (logits.scalar_type() == torch::kBFloat16)
    token_stats_bwd_kernel<__nv_bfloat16><<<static_cast<unsigned>(N), kThreads, 0, cur_stream()>>>(a);
  else
    token_stats_bwd_kernel<float><<<static_cast<unsigned>(N), kThreads, 0, cur_stream()>>>(a);
  TT_CUDA_CHECK(cudaGetLastError());
}

}  // namespace tt

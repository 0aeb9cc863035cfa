// Backward of causal attention over packed sequences on sm_100a tensor cores.
//
//   P = 2^(scale log2e S - lse2), dP = dO V^T, dS = P o (dP - delta), delta = rowsum(dO o O)
//   dV = P^T dO, dK = scale dS^T Q (summed over the query heads of a kv head), dQ = scale dS K
//
// Two kernels, one per direction of the sum, instead of one that adds dQ into memory with atomics:
// the scores and dP are formed twice (seven products where five would do), but every sum stays in
// one accumulator in a fixed order, so gradients repeat bit for bit, nothing is staged through an
// fp32 dQ buffer (clear, atomics, conversion), and both kernels keep P and dS in TMEM as the A
// operand of the next product.  The dense backward of this library, which does add dQ with atomics,
// spends more on its dQ path than the two extra products cost here.
//
//   dkv kernel: one CTA per (sequence, 128-key tile, kv head); all query heads of the group and all
//     query tiles that see the keys pass by.  Lanes are keys: S^T and dP^T (128 x 128 each), dV, dK
//     fill the 512 TMEM columns.
//   dq kernel: one CTA per (sequence, 128-query tile, query head); lanes are queries, two score
//     buffers so that the next tile's exponentials run while the tensor core forms dQ.
//
// Rows that a last partial tile took from the next sequence get probability and dS exactly zero, and
// their rows of the operand they are multiplied with are cleared (zero times a neighbour's infinity
// is not zero).
//
// P is rounded to bf16 once for dV, dS once for dQ and dK (the operands of the products); sums, delta and the
// statistics are fp32.
//
// Bound by P and dS passing through TMEM between the products.  14 sequences, 16384 tokens, 16/4 heads, d 128
// (329 GFLOP at five products), each kernel by itself: dkv 257 us, dq 210 us, the row statistics 39 us; 650 TFLOP/s in
// all, 910 counting the seven products that run; with its three schedules (14 us) and the forward the pass takes 795.  One
// long sequence (10365 of 17001 tokens, 8/2 heads, d 64): dkv 490 us, by its longest CTA: the first key tile's column of
// queries, all heads of the group, is 1.4 times the mean load of an SM, and an entry is not split.
#include "attn/packed.cuh"
#include "common/fast_exp2.cuh"

#include <cmath>

namespace tt {
namespace packed {

constexpr int kGroups = 4;               // compute warpgroups, 32 score columns each
constexpr int kCols = kBlock / kGroups;  // 32
constexpr int kBwdThreads = 128 + kGroups * 128;  // warp 0 TMA, warp 1 MMA, warps 4..19 compute
constexpr uint32_t kComputeThreads = kGroups * 128;
// Registers per thread after setmaxnreg: the launch gives 640 threads 96 each, the first warpgroup (TMA and MMA
// issue) hands 32 of its own to the four compute warpgroups, 8 each.
constexpr int kRegIssue = 64, kRegCompute = 104;
static_assert(kRegIssue + kGroups * kRegCompute <= (1 + kGroups) * 96, "register split exceeds the launch");

// Probabilities of 32 scores in pairs: 2^(s scale_log2 + add), add = -lse2 of the column (or row); kPoly of eight
// exponentials on the FMA pipe instead of MUFU.  kAny: a NaN addend (a row that saw a NaN or an infinite score) gives NaN
// in every column; dQ's kernel need not, its dS is NaN by delta.
template <int kPoly, bool kAny, typename Add>
__device__ __forceinline__ void probabilities(const uint32_t (&raw)[kCols], unsigned long long (&pv)[kCols / 2],
                                              float scale_log2, Add add) {
  const unsigned long long s2 = f2_pack(scale_log2, scale_log2);
#pragma unroll
  for (int i = 0; i < kCols / 2; ++i) {
    float a, b;
    f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[2 * i]), __uint_as_float(raw[2 * i + 1])), s2, add(i)), a, b);
    if ((i & 3) == 3) {
      if (kAny) exp2_poly2_any(a, b);
      else exp2_poly2(a, b);
    } else {
      a = ex2_mufu(a);
      b = (kPoly == 3 && (i & 3) == 1) ? (kAny ? exp2_poly_any(b) : exp2_poly(b)) : ex2_mufu(b);
    }
    pv[i] = f2_pack(a, b);
  }
}
__device__ __forceinline__ uint32_t pack_pair(unsigned long long v) {
  float a, b;
  f2_unpack(v, a, b);
  return pack_bf16x2(a, b);
}
// Pairs of columns [lo, hi) kept, the others zero.
__device__ __forceinline__ void keep_columns(unsigned long long (&v)[kCols / 2], int lo, int hi) {
#pragma unroll
  for (int i = 0; i < kCols / 2; ++i) {
    float a, b;
    f2_unpack(v[i], a, b);
    v[i] = f2_pack((2 * i >= lo && 2 * i < hi) ? a : 0.0f, (2 * i + 1 >= lo && 2 * i + 1 < hi) ? b : 0.0f);
  }
}

// ----------------------------------------------------------------- statistics per query row
// Addends of the row's scores and dP: neg_lse2[h][r] = -lse log2e and neg_delta[h][r] = -dO . O in tile-aligned rows
// (packed.cuh: pad_row0); rows past a sequence and rows that see no key get -inf and 0 (probability 0).  kStatsRows
// rows of a 128-row slot per block: the 16-byte loads of a row are few, so the parallelism has to come from the rows.
constexpr int kStatsRows = 16;
__global__ void __launch_bounds__(256) packed_stats_kernel(const Packing p, const int2* __restrict__ list,
                                                           const __nv_bfloat16* __restrict__ o,
                                                           const __nv_bfloat16* __restrict__ o_lo,
                                                           const __nv_bfloat16* __restrict__ dout,
                                                           const float* __restrict__ lse, float* __restrict__ neg_lse2,
                                                           float* __restrict__ neg_delta, long long pad_rows, int Hq, int D) {
  if (list[0].x < 0) return;  // the schedule found the offsets unusable
  const int slot = blockIdx.x / (kBlock / kStatsRows);
  const int r0 = blockIdx.x % (kBlock / kStatsRows) * kStatsRows;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the sequence whose slots include this one: the last b with cu_q[b] / 128 + b <= slot
  int b = 0, n = p.B + 1;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = b + lane * step;
    const bool le = lane * step < n && p.cu_q[at] / kBlock + at <= slot;
    const unsigned mask = __ballot_sync(0xffffffffu, le);
    const int last = mask ? 31 - __clz(mask) : 0;
    b += last * step;
    n = min(step, n - last * step);
  }
  const Seq s = sequence(p, b);
  const int i0 = slot * kBlock - s.pad_row0;  // first query of this slot
  const int vecs = Hq * D / 8, per_head = D / 8;
  for (int r = r0 + warp; r < r0 + kStatsRows; r += 8) {
    const int qi = i0 + r;
    const long long out = static_cast<long long>(slot) * kBlock + r;
    if (qi >= s.qlen || qi + s.off < 0 || b == p.B) {
      for (int h = lane; h < Hq; h += 32) {
        neg_lse2[h * pad_rows + out] = -INFINITY;
        neg_delta[h * pad_rows + out] = 0.0f;
      }
      continue;
    }
    const long long tok = s.q0 + qi;
    const uint4* a = reinterpret_cast<const uint4*>(o + tok * Hq * D);
    const uint4* al = reinterpret_cast<const uint4*>(o_lo + tok * Hq * D);
    const uint4* c = reinterpret_cast<const uint4*>(dout + tok * Hq * D);
    for (int base = 0; base < vecs; base += 32) {
      const int i = base + lane;
      float sum = 0.0f;
      if (i < vecs) {
        const uint4 x = a[i], xl = al[i], y = c[i];
        const uint32_t* lv = reinterpret_cast<const uint32_t*>(&xl);
        const uint32_t* xv = reinterpret_cast<const uint32_t*>(&x);
        const uint32_t* yv = reinterpret_cast<const uint32_t*>(&y);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 xf = unpack_bf16x2(xv[q]), lf = unpack_bf16x2(lv[q]), yf = unpack_bf16x2(yv[q]);
          sum = fmaf(xf.x + lf.x, yf.x, sum);
          sum = fmaf(xf.y + lf.y, yf.y, sum);
        }
      }
      for (int off = per_head / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (i < vecs && (i & (per_head - 1)) == 0) {
        const int h = i / per_head;
        neg_delta[h * pad_rows + out] = -sum;
        neg_lse2[h * pad_rows + out] = lse[static_cast<long long>(h) * p.Nq + tok] * -1.4426950408889634f;
      }
    }
  }
}

struct BwdParams {
  Packing pk;
  const int2* list;
  int Hq, Hkv;
  const float* neg_lse2;   // [Hq, pad_rows]
  const float* neg_delta;  // [Hq, pad_rows]
  long long pad_rows;
  __nv_bfloat16* d0;   // dq, or dk
  __nv_bfloat16* d1;   // dv
  long long d0_n, d0_h, d1_n, d1_h;  // strides of their tokens and heads
  float scale, scale_log2;
  int* status;
};

// W accumulator columns of a row (16 or 32), scaled, as bf16.
template <int W>
__device__ __forceinline__ void store_row(uint32_t taddr, __nv_bfloat16* dst, float scale, bool row_ok) {
  uint32_t rr[W];
  if constexpr (W == 32) tmem_ld32(taddr, rr);
  else tmem_ld16(taddr, rr);
  tmem_ld_wait();
  if (row_ok) {
    uint32_t w[W / 2];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) w[i] = pack_bf16x2(__uint_as_float(rr[2 * i]) * scale, __uint_as_float(rr[2 * i + 1]) * scale);
#pragma unroll
    for (int i = 0; i < W / 8; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
}

// ----------------------------------------------------------------- dK, dV
template <int D>
struct DkvSmem {
  static constexpr int TILE = kBlock * D * 2;
  alignas(1024) uint8_t k[TILE];
  alignas(1024) uint8_t v[TILE];
  alignas(1024) uint8_t q[2][TILE];
  alignas(1024) uint8_t dout[2][TILE];
  alignas(16) float neg_lse2[2][kBlock];
  alignas(16) float neg_delta[2][kBlock];
  uint64_t kv_full, qdo_full[2], qdo_empty[2], s_full, p_ready, dp_full, ds_ready, done;
  uint32_t tmem_slot;
};

// MMA order (one thread), it = (query head of the group, query tile):
//   S^T(0), dP^T(0); per it: [p_ready] dV += P^T dO, S^T(it + 1); [ds_ready] dK += dS^T Q, dP^T(it + 1)
// Compute: P(0); per it: dS(it), P(it + 1).  So dS is formed while the tensor core runs dV and the next
// scores, and the next exponentials while it runs dK and the next dP.
// P^T (dS^T) of a warpgroup's 32 queries is written over the columns that the same warpgroup read
// its scores (dP) from, so the warpgroups need not wait for each other.
template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, const BwdParams p) {
  constexpr uint32_t TILE = DkvSmem<D>::TILE;
  constexpr uint32_t S_COL = 0, DP_COL = kBlock, DV_COL = 2 * kBlock, DK_COL = 2 * kBlock + D;
  constexpr uint32_t TMEM_COLS = 512;
  const int2 entry = p.list[blockIdx.x / p.Hkv];
  if (entry.x < 0) {
    if (entry.x == kRejected) {
      zero_share<D>(p.d0, p.pk.Nk, p.Hkv, p.d0_n, p.d0_h);
      zero_share<D>(p.d1, p.pk.Nk, p.Hkv, p.d1_n, p.d1_h);
    }
    return;
  }
  const int g = static_cast<int>(blockIdx.x) % p.Hkv;
  const int group = p.Hq / p.Hkv;
  const Seq s = sequence(p.pk, entry.x);
  const bool extra = entry.x == p.pk.B;
  const int j0 = entry.y * kBlock;  // first key of the tile
  const int per_head = query_tiles(s, extra, entry.y);
  const int qt0 = first_query_tile(s, entry.y);
  const int n_iter = group * per_head;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (n_iter == 0) {  // keys that no query sees
    const int rows = min(kBlock, s.klen - j0);
    constexpr int NU = D / 8;
    for (int i = threadIdx.x; i < rows * NU; i += kBwdThreads) {
      const long long row = s.k0 + j0 + i / NU;
      reinterpret_cast<uint4*>(p.d0 + row * p.d0_n + g * p.d0_h)[i % NU] = make_uint4(0u, 0u, 0u, 0u);
      reinterpret_cast<uint4*>(p.d1 + row * p.d1_n + g * p.d1_h)[i % NU] = make_uint4(0u, 0u, 0u, 0u);
    }
    return;
  }
  extern __shared__ uint8_t smem_raw[];
  DkvSmem<D>& sm = *reinterpret_cast<DkvSmem<D>*>(align_ptr(smem_raw, 1024));

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDO);
    mbar_init(&sm.kv_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.qdo_full[i], 1);
      mbar_init(&sm.qdo_empty[i], 1);
    }
    mbar_init(&sm.s_full, 1);
    mbar_init(&sm.p_ready, kComputeThreads);
    mbar_init(&sm.dp_full, 1);
    mbar_init(&sm.ds_ready, kComputeThreads);
    mbar_init(&sm.done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_slot;
  const int last_qt = (s.qlen + kBlock - 1) / kBlock - 1;

  if (warp < 4) {
  setmaxnreg_dec<kRegIssue>();
  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ producer (Q, dO, statistics double-buffered)
      mbar_arrive_expect_tx(&sm.kv_full, 2 * TILE);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        tma_load_3d(sm.k + c * kBlock * 128, &tmK, &sm.kv_full, c * 64, g, s.k0 + j0);
        tma_load_3d(sm.v + c * kBlock * 128, &tmV, &sm.kv_full, c * 64, g, s.k0 + j0);
      }
      for (int it = 0; it < n_iter; ++it) {
        const int st = it & 1;
        const int h = g * group + it / per_head;
        const int qt = qt0 + it % per_head;
        if (!mbar_wait(&sm.qdo_empty[st], ((it >> 1) & 1) ^ 1u, p.status, kTimeoutEmpty)) break;
        mbar_arrive_expect_tx(&sm.qdo_full[st], 2 * TILE + 2 * kBlock * 4);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          tma_load_3d(sm.q[st] + c * kBlock * 128, &tmQ, &sm.qdo_full[st], c * 64, h, s.q0 + qt * kBlock);
          tma_load_3d(sm.dout[st] + c * kBlock * 128, &tmDO, &sm.qdo_full[st], c * 64, h, s.q0 + qt * kBlock);
        }
        const long long vo = h * p.pad_rows + s.pad_row0 + static_cast<long long>(qt) * kBlock;
        bulk_load_1d(sm.neg_lse2[st], p.neg_lse2 + vo, kBlock * 4, &sm.qdo_full[st]);
        bulk_load_1d(sm.neg_delta[st], p.neg_delta + vo, kBlock * 4, &sm.qdo_full[st]);
      }
      mbar_wait(&sm.kv_full, 0, p.status, kTimeoutOther);
      for (int it = max(0, n_iter - 2); it < n_iter; ++it)
        mbar_wait(&sm.qdo_full[it & 1], (it >> 1) & 1, p.status, kTimeoutOther);
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer
    const bool lead = elect_one();
    const uint32_t k_lo = desc_k_major(sm.k), v_lo = desc_k_major(sm.v);
    auto score = [&](int it) { product_abt<D>(lead, tmem + S_COL, k_lo, desc_k_major(sm.q[it & 1]), &sm.s_full); };
    auto dprob = [&](int it) { product_abt<D>(lead, tmem + DP_COL, v_lo, desc_k_major(sm.dout[it & 1]), &sm.dp_full); };
    bool ok = mbar_wait_warp(&sm.kv_full, 0, p.status, kTimeoutFull) && mbar_wait_warp(&sm.qdo_full[0], 0, p.status, kTimeoutFull);
    if (ok) {
      tc_fence_after();
      score(0);
      dprob(0);
    }
    for (int it = 0; ok && it < n_iter; ++it) {
      const uint32_t ph = it & 1;
      const bool next = it + 1 < n_iter;
      if (!mbar_wait_warp(&sm.p_ready, ph, p.status, kTimeoutFull)) break;
      tc_fence_after();
      product_ab<D, kCols>(lead, tmem + DV_COL, tmem + S_COL, desc_mn_major(sm.dout[it & 1]), it > 0);
      if (next) {  // in order after dV, which reads P^T from the same columns
        if (!mbar_wait_warp(&sm.qdo_full[(it + 1) & 1], ((it + 1) >> 1) & 1, p.status, kTimeoutFull)) break;
        tc_fence_after();
        score(it + 1);
      }
      if (!mbar_wait_warp(&sm.ds_ready, ph, p.status, kTimeoutFull)) break;
      tc_fence_after();
      product_ab<D, kCols>(lead, tmem + DK_COL, tmem + DP_COL, desc_mn_major(sm.q[it & 1]), it > 0);
      commit(lead, &sm.qdo_empty[it & 1]);
      if (next) dprob(it + 1);
    }
    commit(lead, &sm.done);
    mbar_wait_warp(&sm.done, 0, p.status, kTimeoutOther);
  }
  } else {
    setmaxnreg_inc<kRegCompute>();
    // ------------------------------------------------ compute warpgroups: 32 queries each, one key per thread
    const int wg = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + S_COL + wg * kCols;
    const uint32_t dp_addr = tmem + lane_addr + DP_COL + wg * kCols;
    const int key = j0 + r;
    const int key_row = key - s.off - wg * kCols;  // minus a query tile's first query: first column that sees the key
    const int end_row = s.qlen - wg * kCols;       // likewise: columns that are queries of the sequence
    unsigned long long pv[kCols / 2];
    auto p_phase = [&](int it, int qt) -> bool {
      const int buf = it & 1;
      if (!mbar_wait_warp(&sm.s_full, it & 1, p.status, kTimeoutAccFull)) return false;
      if (!mbar_wait_warp(&sm.qdo_full[buf], (it >> 1) & 1, p.status, kTimeoutFull)) return false;  // the statistics
      tc_fence_after();
      uint32_t raw[kCols];
      tmem_ld32(s_addr, raw);
      const ulonglong2* nl = reinterpret_cast<const ulonglong2*>(sm.neg_lse2[buf] + wg * kCols);
      tmem_ld_wait();
      probabilities<3, true>(raw, pv, p.scale_log2, [&](int i) { return (i & 1) ? nl[i >> 1].y : nl[i >> 1].x; });
      const int lo = key_row - qt * kBlock, hi = end_row - qt * kBlock;
      if (lo > 0 || hi < kCols) keep_columns(pv, lo, hi);
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = pack_pair(pv[i]);
      tmem_st16(s_addr, pk);
      if (qt == last_qt && s.qlen % kBlock != 0) {
        // The tile ends inside: once dP(it), the last product to read these rows as they are, is done, clear
        // dO's and Q's rows of the next sequence.
        if (!mbar_wait_warp(&sm.dp_full, it & 1, p.status, kTimeoutAccFull)) return false;
        clear_rows<D>(sm.dout[buf], s.qlen - qt * kBlock, threadIdx.x - 128, kComputeThreads);
        clear_rows<D>(sm.q[buf], s.qlen - qt * kBlock, threadIdx.x - 128, kComputeThreads);
        fence_proxy_async();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.p_ready);
      return true;
    };
    int qt = qt0;  // query tile of iteration it (its head is it / per_head)
    bool ok = p_phase(0, qt);
    for (int it = 0; ok && it < n_iter; ++it) {
      const int buf = it & 1;
      // ---- dS^T = P^T (dP^T - delta), the scale goes to the end
      if (!mbar_wait_warp(&sm.dp_full, it & 1, p.status, kTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      {
        const ulonglong2* nd = reinterpret_cast<const ulonglong2*>(sm.neg_delta[buf] + wg * kCols);
        uint32_t d[kCols];
        tmem_ld32(dp_addr, d);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < kCols / 2; ++i)
          pv[i] = f2_mul(pv[i], f2_add(f2_pack(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])), (i & 1) ? nd[i >> 1].y : nd[i >> 1].x));
        const int lo = key_row - qt * kBlock, hi = end_row - qt * kBlock;
        if (lo > 0 || hi < kCols) keep_columns(pv, lo, hi);
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack_pair(pv[i]);
        tmem_st16(dp_addr, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.ds_ready);
      if (++qt > last_qt) qt = qt0;
      if (it + 1 < n_iter && !p_phase(it + 1, qt)) ok = false;
    }
    // ---- dK, dV of this thread's key, a quarter of the head dim per warpgroup
    if (ok && mbar_wait_warp(&sm.done, 0, p.status, kTimeoutAccFull)) {
      tc_fence_after();
      const bool key_ok = key < s.klen;
      const long long row = s.k0 + key;
      constexpr int W = D / kGroups;
      store_row<W>(tmem + lane_addr + DK_COL + wg * W, p.d0 + row * p.d0_n + g * p.d0_h + wg * W, p.scale, key_ok);
      store_row<W>(tmem + lane_addr + DV_COL + wg * W, p.d1 + row * p.d1_n + g * p.d1_h + wg * W, 1.0f, key_ok);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

// ----------------------------------------------------------------- dQ
template <int D>
struct DqSmem {
  static constexpr int TILE = kBlock * D * 2;
  alignas(1024) uint8_t q[TILE];
  alignas(1024) uint8_t dout[TILE];
  alignas(1024) uint8_t k[3][TILE];
  alignas(1024) uint8_t v[2][TILE];
  uint64_t q_full, k_full[3], k_empty[3], v_full[2], v_empty[2];
  uint64_t s_full[2], dp_full, dp_taken, ds_ready, done;
  uint32_t tmem_slot;
};
template <int D>
constexpr uint32_t dq_smem_bytes() {
  return static_cast<uint32_t>(offsetof(DqSmem<D>, tmem_slot) + sizeof(uint32_t));
}

// MMA order (one thread), j = key tile:
//   S(0), dP(0), S(1); per j: [dp_taken(j)] dP(j + 1); [ds_ready(j)] dQ += dS(j) K(j), S(j + 2)
// Compute per j: P(j) from score buffer j & 1; [dp_full] dP(j) into registers -> dp_taken; dS(j) over the
// same score buffer -> ds_ready.  The exponentials of tile j + 1 run beside dQ(j) and S(j + 2).
template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, const BwdParams p) {
  constexpr uint32_t TILE = DqSmem<D>::TILE;
  constexpr uint32_t DP_COL = 2 * kBlock, DQ_COL = 3 * kBlock;
  constexpr uint32_t TMEM_COLS = 512;
  const int2 entry = p.list[blockIdx.x / p.Hq];
  if (entry.x < 0) {
    if (entry.x == kRejected) zero_share<D>(p.d0, p.pk.Nq, p.Hq, p.d0_n, p.d0_h);
    return;
  }
  const int h = static_cast<int>(blockIdx.x) % p.Hq;
  const int g = h / (p.Hq / p.Hkv);
  const Seq s = sequence(p.pk, entry.x);
  const bool extra = entry.x == p.pk.B;
  const int i0 = entry.y * kBlock;
  const int n = key_tiles(s, extra, i0, kBlock);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (n == 0) {  // queries that see no key
    const int rows = min(kBlock, s.qlen - i0);
    constexpr int NU = D / 8;
    for (int i = threadIdx.x; i < rows * NU; i += kBwdThreads)
      reinterpret_cast<uint4*>(p.d0 + (s.q0 + i0 + i / NU) * p.d0_n + h * p.d0_h)[i % NU] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  extern __shared__ uint8_t smem_raw[];
  DqSmem<D>& sm = *reinterpret_cast<DqSmem<D>*>(align_ptr(smem_raw, 1024));

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    tma_prefetch_desc(&tmDO);
    mbar_init(&sm.q_full, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
    }
    mbar_init(&sm.dp_full, 1);
    mbar_init(&sm.dp_taken, kComputeThreads);
    mbar_init(&sm.ds_ready, kComputeThreads);
    mbar_init(&sm.done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ producer: K three deep, V two
      mbar_arrive_expect_tx(&sm.q_full, 2 * TILE);
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        tma_load_3d(sm.q + c * kBlock * 128, &tmQ, &sm.q_full, c * 64, h, s.q0 + i0);
        tma_load_3d(sm.dout + c * kBlock * 128, &tmDO, &sm.q_full, c * 64, h, s.q0 + i0);
      }
      for (int j = 0; j < n; ++j) {
        const int ks = j % 3, vs = j & 1;
        if (!mbar_wait(&sm.k_empty[ks], ((j / 3) & 1) ^ 1u, p.status, kTimeoutEmpty)) break;
        mbar_arrive_expect_tx(&sm.k_full[ks], TILE);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.k[ks] + c * kBlock * 128, &tmK, &sm.k_full[ks], c * 64, g, s.k0 + j * kBlock);
        if (!mbar_wait(&sm.v_empty[vs], ((j >> 1) & 1) ^ 1u, p.status, kTimeoutEmpty)) break;
        mbar_arrive_expect_tx(&sm.v_full[vs], TILE);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.v[vs] + c * kBlock * 128, &tmV, &sm.v_full[vs], c * 64, g, s.k0 + j * kBlock);
      }
      mbar_wait(&sm.q_full, 0, p.status, kTimeoutOther);
      for (int j = max(0, n - 3); j < n; ++j) mbar_wait(&sm.k_full[j % 3], (j / 3) & 1, p.status, kTimeoutOther);
      for (int j = max(0, n - 2); j < n; ++j) mbar_wait(&sm.v_full[j & 1], (j >> 1) & 1, p.status, kTimeoutOther);
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer
    const bool lead = elect_one();
    const uint32_t q_lo = desc_k_major(sm.q), do_lo = desc_k_major(sm.dout);
    auto score = [&](int j) { product_abt<D>(lead, tmem + (j & 1) * kBlock, q_lo, desc_k_major(sm.k[j % 3]), &sm.s_full[j & 1]); };
    auto dprob = [&](int j) {
      product_abt<D>(lead, tmem + DP_COL, do_lo, desc_k_major(sm.v[j & 1]), &sm.dp_full);
      commit(lead, &sm.v_empty[j & 1]);
    };
    bool ok = mbar_wait_warp(&sm.q_full, 0, p.status, kTimeoutFull) && mbar_wait_warp(&sm.k_full[0], 0, p.status, kTimeoutFull);
    if (ok) {
      tc_fence_after();
      score(0);
      ok = mbar_wait_warp(&sm.v_full[0], 0, p.status, kTimeoutFull);
    }
    if (ok) {
      tc_fence_after();
      dprob(0);
      if (n > 1) {
        ok = mbar_wait_warp(&sm.k_full[1], 0, p.status, kTimeoutFull);
        if (ok) {
          tc_fence_after();
          score(1);
        }
      }
    }
    for (int j = 0; ok && j < n; ++j) {
      if (j + 1 < n) {
        if (!mbar_wait_warp(&sm.v_full[(j + 1) & 1], ((j + 1) >> 1) & 1, p.status, kTimeoutFull)) break;
        if (!mbar_wait_warp(&sm.dp_taken, j & 1, p.status, kTimeoutFull)) break;
        tc_fence_after();
        dprob(j + 1);
      }
      if (!mbar_wait_warp(&sm.ds_ready, j & 1, p.status, kTimeoutFull)) break;
      tc_fence_after();
      product_ab<D, kCols>(lead, tmem + DQ_COL, tmem + (j & 1) * kBlock, desc_mn_major(sm.k[j % 3]), j > 0);
      commit(lead, &sm.k_empty[j % 3]);
      if (j + 2 < n) {  // in order after dQ(j), which reads dS from the same columns
        if (!mbar_wait_warp(&sm.k_full[(j + 2) % 3], ((j + 2) / 3) & 1, p.status, kTimeoutFull)) break;
        tc_fence_after();
        score(j + 2);
      }
    }
    commit(lead, &sm.done);
    mbar_wait_warp(&sm.done, 0, p.status, kTimeoutOther);
  } else if (warp >= 4) {
    // ------------------------------------------------ compute warpgroups: 32 keys each, one query per thread
    const int wg = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int qi = i0 + r;
    const int seen = min(qi + s.off, s.klen - 1) + 1 - wg * kCols;  // minus a tile's first key: columns below it are seen
    const long long vo = h * p.pad_rows + s.pad_row0 + qi;
    const float neg_lse2 = p.neg_lse2[vo], neg_delta = p.neg_delta[vo];
    const unsigned long long nl2 = f2_pack(neg_lse2, neg_lse2), nd2 = f2_pack(neg_delta, neg_delta);
    const uint32_t dp_addr = tmem + lane_addr + DP_COL + wg * kCols;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const uint32_t s_addr = tmem + lane_addr + (j & 1) * kBlock + wg * kCols;
      if (!mbar_wait_warp(&sm.s_full[j & 1], (j >> 1) & 1, p.status, kTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      unsigned long long pv[kCols / 2];
      {
        uint32_t raw[kCols];
        tmem_ld32(s_addr, raw);
        tmem_ld_wait();
        probabilities<2, false>(raw, pv, p.scale_log2, [&](int) { return nl2; });
      }
      if (!mbar_wait_warp(&sm.dp_full, j & 1, p.status, kTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t d[kCols];
      tmem_ld32(dp_addr, d);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(&sm.dp_taken);
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i)
        pv[i] = f2_mul(pv[i], f2_add(f2_pack(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])), nd2));
      if (seen - j * kBlock < kCols) keep_columns(pv, 0, seen - j * kBlock);
      uint32_t pk[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = pack_pair(pv[i]);
      tmem_st16(s_addr, pk);
      if ((j + 1) * kBlock > s.klen) {  // the last key tile ends inside: K's rows of the next sequence (S(j) has read them)
        clear_rows<D>(sm.k[j % 3], s.klen - j * kBlock, threadIdx.x - 128, kComputeThreads);
        fence_proxy_async();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.ds_ready);
    }
    if (ok && mbar_wait_warp(&sm.done, 0, p.status, kTimeoutAccFull)) {
      tc_fence_after();
      constexpr int W = D / kGroups;
      store_row<W>(tmem + lane_addr + DQ_COL + wg * W, p.d0 + (static_cast<long long>(s.q0) + qi) * p.d0_n + h * p.d0_h + wg * W,
                   p.scale, qi < s.qlen);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace packed

// fp32 elements of the per-row statistics that packed_attn_bwd needs.
int64_t packed_attn_stats_numel(int64_t Nq, int64_t Hq, int64_t B) {
  return 2 * Hq * packed::pad_slots(Nq, B) * packed::kBlock;
}

// Backward of packed_attn_fwd.  o, o_lo, dout contiguous [Nq, Hq, D]; lse [Hq, Nq] from the forward; dq [Nq, Hq, D],
// dk/dv [Nk, Hkv, D] bf16 with any 16-byte-aligned strides (views of one packed buffer, say).  stats: fp32 scratch,
// sched: int32 scratch.
void packed_attn_bwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor o, torch::Tensor o_lo,
                     torch::Tensor dout, torch::Tensor lse, torch::Tensor cu_q, torch::Tensor cu_k, double scale, torch::Tensor dq,
                     torch::Tensor dk, torch::Tensor dv, torch::Tensor stats, torch::Tensor sched) {
  using namespace packed;
  TT_CHECK(q.dim() == 3 && k.dim() == 3, "packed_attn_bwd: q and k must be [tokens, heads, D]");
  const int64_t Nq = q.size(0), Hq = q.size(1), D = q.size(2), Nk = k.size(0), Hkv = k.size(1);
  TT_CHECK(D == 64 || D == 128, "packed_attn_bwd: head_dim must be 64 or 128");
  TT_CHECK(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0, "packed_attn_bwd: Hq must be a multiple of Hkv");
  check_heads(q, Hq, D, "packed_attn_bwd q");
  check_heads(k, Hkv, D, "packed_attn_bwd k");
  check_heads(v, Hkv, D, "packed_attn_bwd v");
  check_heads(o, Hq, D, "packed_attn_bwd o");
  check_heads(o_lo, Hq, D, "packed_attn_bwd o_lo");
  check_heads(dout, Hq, D, "packed_attn_bwd dout");
  check_heads(dq, Hq, D, "packed_attn_bwd dq");
  check_heads(dk, Hkv, D, "packed_attn_bwd dk");
  check_heads(dv, Hkv, D, "packed_attn_bwd dv");
  TT_CHECK(o.is_contiguous() && o_lo.is_contiguous() && dout.is_contiguous() && o.size(0) == Nq && o_lo.size(0) == Nq && dout.size(0) == Nq && dq.size(0) == Nq &&
               v.size(0) == Nk && dk.size(0) == Nk && dv.size(0) == Nk,
           "packed_attn_bwd: token counts; o and dout must be contiguous");
  check_offsets(cu_q, -1, "cu_seqlens");
  check_offsets(cu_k, cu_q.numel(), "cu_seqlens_k");
  const int64_t B = cu_q.numel() - 1;
  TT_CHECK(lse.scalar_type() == torch::kFloat32 && lse.is_contiguous() && lse.numel() == Hq * Nq, "packed_attn_bwd: lse must be fp32 [Hq, Nq]");
  TT_CHECK(scale > 0 && std::isfinite(scale), "packed_attn_bwd: scale must be positive and finite");
  TT_CHECK(stats.scalar_type() == torch::kFloat32 && stats.is_contiguous() && stats.numel() >= packed_attn_stats_numel(Nq, Hq, B) &&
               reinterpret_cast<uintptr_t>(stats.data_ptr()) % 16 == 0,
           "packed_attn_bwd: statistics scratch too small");
  const int64_t q_entries = max_tiles(Nq, B, kBlock), k_entries = max_tiles(Nk, B, kBlock);
  TT_CHECK(sched.scalar_type() == torch::kInt32 && sched.is_contiguous() && sched.numel() >= 2 * std::max(q_entries, k_entries) &&
               reinterpret_cast<uintptr_t>(sched.data_ptr()) % 8 == 0,
           "packed_attn_bwd: schedule scratch too small");
  TT_CHECK(q_entries * Hq < (1LL << 31) && k_entries * Hkv < (1LL << 31), "packed_attn_bwd: too many tiles");
  const c10::cuda::CUDAGuard guard(q.device());
  TT_CUDA_CHECK(cudaSetDevice(q.get_device()));  // binds the context to this thread: the tensor maps need one
  if (Nq == 0 || Nk == 0) {
    dq.zero_();
    dk.zero_();
    dv.zero_();
    return;
  }
  cudaStream_t st = cur_stream();
  int* status = device_status_ptr(q.get_device());
  BwdParams p{};
  p.pk = packing_of(q, k, cu_q, cu_k);
  int2* list = reinterpret_cast<int2*>(sched.data_ptr<int>());
  p.list = list;
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.pad_rows = pad_slots(Nq, B) * kBlock;
  float* neg_lse2 = stats.data_ptr<float>();
  float* neg_delta = neg_lse2 + Hq * p.pad_rows;
  p.neg_lse2 = neg_lse2;
  p.neg_delta = neg_delta;
  p.scale = static_cast<float>(scale);
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  p.status = status;
  const CUtensorMap tq = head_map_3d(q, kBlock, "q"), tk = head_map_3d(k, kBlock, "k"), tv = head_map_3d(v, kBlock, "v"),
                    tdo = head_map_3d(dout, kBlock, "dout");
  // dQ's list first: it checks the offsets, and a bad packing leaves every entry rejected
  schedule(p.pk, kQueryTiles, list, static_cast<int>(q_entries), status, st);
  packed_stats_kernel<<<static_cast<unsigned>(pad_slots(Nq, B) * (kBlock / kStatsRows)), 256, 0, st>>>(
      p.pk, list, reinterpret_cast<const __nv_bfloat16*>(o.data_ptr()), reinterpret_cast<const __nv_bfloat16*>(o_lo.data_ptr()),
      reinterpret_cast<const __nv_bfloat16*>(dout.data_ptr()), lse.data_ptr<float>(), neg_lse2, neg_delta, p.pad_rows, p.Hq, static_cast<int>(D));
  TT_CUDA_CHECK(cudaGetLastError());
  const int device = q.get_device();
  auto launch_dq = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    constexpr size_t smem = dq_smem_bytes<kD>() + 1024;
    allow_smem<&packed_dq_kernel<kD>>(smem, device);
    packed_dq_kernel<kD><<<static_cast<unsigned>(q_entries * Hq), kBwdThreads, smem, st>>>(tq, tk, tv, tdo, p);
    TT_CUDA_CHECK(cudaGetLastError());
  };
  auto launch_dkv = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    constexpr size_t smem = sizeof(DkvSmem<kD>) + 1024;
    allow_smem<&packed_dkv_kernel<kD>>(smem, device);
    packed_dkv_kernel<kD><<<static_cast<unsigned>(k_entries * Hkv), kBwdThreads, smem, st>>>(tq, tk, tv, tdo, p);
    TT_CUDA_CHECK(cudaGetLastError());
  };
  p.d0 = reinterpret_cast<__nv_bfloat16*>(dq.data_ptr());
  p.d0_n = dq.stride(0);
  p.d0_h = dq.stride(1);
  if (D == 128) launch_dq(std::integral_constant<int, 128>{});
  else launch_dq(std::integral_constant<int, 64>{});
  schedule(p.pk, kKeyTiles, list, static_cast<int>(k_entries), status, st);
  p.d0 = reinterpret_cast<__nv_bfloat16*>(dk.data_ptr());
  p.d0_n = dk.stride(0);
  p.d0_h = dk.stride(1);
  p.d1 = reinterpret_cast<__nv_bfloat16*>(dv.data_ptr());
  p.d1_n = dv.stride(0);
  p.d1_h = dv.stride(1);
  if (D == 128) launch_dkv(std::integral_constant<int, 128>{});
  else launch_dkv(std::integral_constant<int, 64>{});
}

}  // namespace tt

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
#include "attn/packed.cuh"
#include "common/fast_exp2.cuh"

#include <cmath>

namespace tt {
namespace packed {

constexpr int kBwdThreads = 384;  // warp 0 TMA, warp 1 MMA, warps 4..11 two compute warpgroups
constexpr int kHalf = kBlock / 2;

// Probabilities of 64 scores: 2^(s scale_log2 - l2), two of eight on the FMA pipe.
template <bool kPerColumn>
__device__ __forceinline__ void probabilities(const uint32_t (&raw)[kHalf], float (&pv)[kHalf], float scale_log2,
                                              const float* l2, float l2_row) {
  const unsigned long long s2 = f2_pack(scale_log2, scale_log2);
#pragma unroll
  for (int i = 0; i < kHalf; i += 2) {
    float a, b;
    const unsigned long long sub = kPerColumn ? f2_pack(-l2[i], -l2[i + 1]) : f2_pack(-l2_row, -l2_row);
    f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[i]), __uint_as_float(raw[i + 1])), s2, sub), a, b);
    if ((i & 7) == 6) {
      exp2_poly2(a, b);
    } else {
      a = ex2_mufu(a);
      b = ex2_mufu(b);
    }
    pv[i] = a;
    pv[i + 1] = b;
  }
}

// ----------------------------------------------------------------- statistics per query row
// lse2[h][r] = lse log2e and delta[h][r] = dO . O in tile-aligned rows (packed.cuh: pad_row0); rows past a
// sequence and rows that see no key get +inf and 0 (probability 0).  One block per 128-row slot.
__global__ void __launch_bounds__(256) packed_stats_kernel(const Packing p, const int2* __restrict__ list,
                                                           const __nv_bfloat16* __restrict__ o,
                                                           const __nv_bfloat16* __restrict__ dout,
                                                           const float* __restrict__ lse, float* __restrict__ lse2,
                                                           float* __restrict__ delta, long long pad_rows, int Hq, int D) {
  if (list[0].x < 0) return;  // the schedule found the offsets unusable
  const int slot = blockIdx.x;
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
  for (int r = warp; r < kBlock; r += 8) {
    const int qi = i0 + r;
    const long long out = static_cast<long long>(slot) * kBlock + r;
    if (qi >= s.qlen || qi + s.off < 0 || b == p.B) {
      for (int h = lane; h < Hq; h += 32) {
        lse2[h * pad_rows + out] = INFINITY;
        delta[h * pad_rows + out] = 0.0f;
      }
      continue;
    }
    const long long tok = s.q0 + qi;
    const uint4* a = reinterpret_cast<const uint4*>(o + tok * Hq * D);
    const uint4* c = reinterpret_cast<const uint4*>(dout + tok * Hq * D);
    for (int base = 0; base < vecs; base += 32) {
      const int i = base + lane;
      float sum = 0.0f;
      if (i < vecs) {
        const uint4 x = a[i], y = c[i];
        const uint32_t* xv = reinterpret_cast<const uint32_t*>(&x);
        const uint32_t* yv = reinterpret_cast<const uint32_t*>(&y);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 xf = unpack_bf16x2(xv[q]), yf = unpack_bf16x2(yv[q]);
          sum = fmaf(xf.x, yf.x, sum);
          sum = fmaf(xf.y, yf.y, sum);
        }
      }
      for (int off = per_head / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (i < vecs && (i & (per_head - 1)) == 0) {
        const int h = i / per_head;
        delta[h * pad_rows + out] = sum;
        lse2[h * pad_rows + out] = lse[static_cast<long long>(h) * p.Nq + tok] * 1.4426950408889634f;
      }
    }
  }
}

struct BwdParams {
  Packing pk;
  const int2* list;
  int Hq, Hkv;
  const float* lse2;   // [Hq, pad_rows]
  const float* delta;  // [Hq, pad_rows]
  long long pad_rows;
  __nv_bfloat16* d0;   // dq, or dk
  __nv_bfloat16* d1;   // dv
  long long d0_n, d0_h, d1_n, d1_h;  // strides of their tokens and heads
  float scale, scale_log2;
  int* status;
};

// 64 accumulator columns-halves of a row, scaled, as bf16.
template <int W>
__device__ __forceinline__ void store_row(uint32_t taddr, __nv_bfloat16* dst, float scale, bool row_ok) {
#pragma unroll
  for (int c = 0; c < W; c += 32) {
    uint32_t rr[32];
    tmem_ld32(taddr + c, rr);
    tmem_ld_wait();
    if (row_ok) {
      float f[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(rr[i]) * scale;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        reinterpret_cast<uint4*>(dst + c)[i] =
            make_uint4(pack_bf16x2(f[8 * i], f[8 * i + 1]), pack_bf16x2(f[8 * i + 2], f[8 * i + 3]),
                       pack_bf16x2(f[8 * i + 4], f[8 * i + 5]), pack_bf16x2(f[8 * i + 6], f[8 * i + 7]));
    }
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
  alignas(16) float lse2[2][kBlock];
  alignas(16) float delta[2][kBlock];
  uint64_t kv_full, qdo_full[2], qdo_empty[2], s_full, p_ready, dp_full, ds_ready, done;
  uint32_t tmem_slot;
};

// MMA order (one thread), it = (query head of the group, query tile):
//   S^T(0), dP^T(0); per it: [p_ready] dV += P^T dO, S^T(it + 1); [ds_ready] dK += dS^T Q, dP^T(it + 1)
// Compute: P(0); per it: dS(it), P(it + 1).  So dS is formed while the tensor core runs dV and the next
// scores, and the next exponentials while it runs dK and the next dP.
// P^T (dS^T) of a warpgroup's 64 queries is written over the columns that the same warpgroup read
// its scores (dP) from, so the two warpgroups need not wait for each other.
template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO, const BwdParams p) {
  constexpr uint32_t TILE = DkvSmem<D>::TILE;
  constexpr uint32_t ID_S = idesc_bf16_f32(kBlock, kBlock, false, false);  // S^T, dP^T
  constexpr uint32_t ID_G = idesc_bf16_f32(kBlock, D, false, true);        // dV, dK (A from TMEM)
  constexpr uint32_t S_COL = 0, DP_COL = kBlock, DV_COL = 2 * kBlock, DK_COL = 2 * kBlock + D;
  constexpr uint32_t TMEM_COLS = 512;
  const int2 entry = p.list[blockIdx.x / p.Hkv];
  if (entry.x < 0) return;
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
    mbar_init(&sm.p_ready, 256);
    mbar_init(&sm.dp_full, 1);
    mbar_init(&sm.ds_ready, 256);
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
        bulk_load_1d(sm.lse2[st], p.lse2 + vo, kBlock * 4, &sm.qdo_full[st]);
        bulk_load_1d(sm.delta[st], p.delta + vo, kBlock * 4, &sm.qdo_full[st]);
      }
      mbar_wait(&sm.kv_full, 0, p.status, kTimeoutOther);
      for (int it = max(0, n_iter - 2); it < n_iter; ++it)
        mbar_wait(&sm.qdo_full[it & 1], (it >> 1) & 1, p.status, kTimeoutOther);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ------------------------------------------------ MMA issuer
      const uint32_t k_b = smem_u32(sm.k), v_b = smem_u32(sm.v);
      auto scores = [&](uint32_t col, uint32_t a_b, uint32_t b_b, uint64_t* bar) {  // [128 keys x 128 queries]
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kBlock * 128) + (kk & 3) * 32;
          umma_f16_ss(tmem + col, sdesc_sw128(a_b + off, 16, 1024), sdesc_sw128(b_b + off, 16, 1024), ID_S, kk > 0 ? 1u : 0u);
        }
        umma_commit(bar);
      };
      auto grads = [&](uint32_t acc, uint32_t a_col, uint32_t b_b, bool first) {  // [128 keys x D] += A [keys x queries] B
#pragma unroll
        for (int kk = 0; kk < kBlock / 16; ++kk)
          umma_f16_ts(tmem + acc, tmem + a_col + (kk >> 2) * kHalf + (kk & 3) * 8,
                      sdesc_sw128(b_b + kk * 2048, kBlock * 128, 1024), ID_G, (!first || kk > 0) ? 1u : 0u);
      };
      bool ok = mbar_wait(&sm.kv_full, 0, p.status, kTimeoutFull) && mbar_wait(&sm.qdo_full[0], 0, p.status, kTimeoutFull);
      if (ok) {
        tc_fence_after();
        scores(S_COL, k_b, smem_u32(sm.q[0]), &sm.s_full);
        scores(DP_COL, v_b, smem_u32(sm.dout[0]), &sm.dp_full);
      }
      for (int it = 0; ok && it < n_iter; ++it) {
        const uint32_t ph = it & 1;
        const bool next = it + 1 < n_iter;
        if (!mbar_wait(&sm.p_ready, ph, p.status, kTimeoutFull)) break;
        tc_fence_after();
        grads(DV_COL, S_COL, smem_u32(sm.dout[it & 1]), it == 0);
        if (next) {  // in order after dV, which reads P^T from the same columns
          if (!mbar_wait(&sm.qdo_full[(it + 1) & 1], ((it + 1) >> 1) & 1, p.status, kTimeoutFull)) break;
          tc_fence_after();
          scores(S_COL, k_b, smem_u32(sm.q[(it + 1) & 1]), &sm.s_full);
        }
        if (!mbar_wait(&sm.ds_ready, ph, p.status, kTimeoutFull)) break;
        tc_fence_after();
        grads(DK_COL, DP_COL, smem_u32(sm.q[it & 1]), it == 0);
        umma_commit(&sm.qdo_empty[it & 1]);
        if (next) scores(DP_COL, v_b, smem_u32(sm.dout[(it + 1) & 1]), &sm.dp_full);
      }
      umma_commit(&sm.done);
      mbar_wait(&sm.done, 0, p.status, kTimeoutOther);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------ compute warpgroups: 64 queries each, one key per thread
    const int half = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + S_COL + half * kHalf;
    const uint32_t dp_addr = tmem + lane_addr + DP_COL + half * kHalf;
    const int key = j0 + r;
    float pv[kHalf];
    // queries [lo, hi) of this warpgroup's 64 see the key
    auto bounds = [&](int it, int& lo, int& hi) {
      const int c0 = (qt0 + it % per_head) * kBlock + half * kHalf;
      lo = key - s.off - c0;
      hi = s.qlen - c0;
    };
    auto p_phase = [&](int it) -> bool {
      const int buf = it & 1;
      if (!mbar_wait_warp(&sm.s_full, it & 1, p.status, kTimeoutAccFull)) return false;
      if (!mbar_wait_warp(&sm.qdo_full[buf], (it >> 1) & 1, p.status, kTimeoutFull)) return false;  // the statistics
      tc_fence_after();
      uint32_t raw[kHalf];
      tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
      tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
      tmem_ld_wait();
      probabilities<true>(raw, pv, p.scale_log2, sm.lse2[buf] + half * kHalf, 0.0f);
      int lo, hi;
      bounds(it, lo, hi);
      if (lo > 0 || hi < kHalf) {
#pragma unroll
        for (int i = 0; i < kHalf; ++i) pv[i] = (i >= lo && i < hi) ? pv[i] : 0.0f;
      }
#pragma unroll
      for (int c = 0; c < kHalf; c += 32) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(pv[c + 2 * i], pv[c + 2 * i + 1]);
        tmem_st16(s_addr + (c >> 1), pk);
      }
      const int qt = qt0 + it % per_head;
      if (qt == last_qt && s.qlen % kBlock != 0) {
        // The tile ends inside: once dP(it), the last product to read these rows as they are, is done, clear
        // dO's and Q's rows of the next sequence.
        if (!mbar_wait_warp(&sm.dp_full, it & 1, p.status, kTimeoutAccFull)) return false;
        clear_rows<D>(sm.dout[buf], s.qlen - qt * kBlock, threadIdx.x - 128, 256);
        clear_rows<D>(sm.q[buf], s.qlen - qt * kBlock, threadIdx.x - 128, 256);
        fence_proxy_async();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.p_ready);
      return true;
    };
    bool ok = p_phase(0);
    for (int it = 0; ok && it < n_iter; ++it) {
      const int buf = it & 1;
      // ---- dS^T = P^T (dP^T - delta), the scale goes to the end
      if (!mbar_wait_warp(&sm.dp_full, it & 1, p.status, kTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      {
        int lo, hi;
        bounds(it, lo, hi);
        const bool masked = lo > 0 || hi < kHalf;
        const float* dl = sm.delta[buf] + half * kHalf;
        uint32_t d0[32], d1[32];
        tmem_ld32(dp_addr, d0);
        tmem_ld32(dp_addr + 32, d1);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t(&cur)[32] = c ? d1 : d0;
          float ds[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) ds[i] = pv[c * 32 + i] * (__uint_as_float(cur[i]) - dl[c * 32 + i]);
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i) ds[i] = (c * 32 + i >= lo && c * 32 + i < hi) ? ds[i] : 0.0f;
          }
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(ds[2 * i], ds[2 * i + 1]);
          tmem_st16(dp_addr + c * 16, pk);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.ds_ready);
      if (it + 1 < n_iter && !p_phase(it + 1)) ok = false;
    }
    // ---- dK, dV of this thread's key, half of the head dim per warpgroup
    if (ok && mbar_wait_warp(&sm.done, 0, p.status, kTimeoutAccFull)) {
      tc_fence_after();
      const bool key_ok = key < s.klen;
      const long long row = s.k0 + key;
      constexpr int DH = D / 2;
      store_row<DH>(tmem + lane_addr + DK_COL + half * DH, p.d0 + row * p.d0_n + g * p.d0_h + half * DH, p.scale, key_ok);
      store_row<DH>(tmem + lane_addr + DV_COL + half * DH, p.d1 + row * p.d1_n + g * p.d1_h + half * DH, 1.0f, key_ok);
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
  constexpr uint32_t ID_S = idesc_bf16_f32(kBlock, kBlock, false, false);
  constexpr uint32_t ID_G = idesc_bf16_f32(kBlock, D, false, true);
  constexpr uint32_t DP_COL = 2 * kBlock, DQ_COL = 3 * kBlock;
  constexpr uint32_t TMEM_COLS = 512;
  const int2 entry = p.list[blockIdx.x / p.Hq];
  if (entry.x < 0) return;
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
    mbar_init(&sm.dp_taken, 256);
    mbar_init(&sm.ds_ready, 256);
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
    if (lane == 0) {
      // ------------------------------------------------ MMA issuer
      const uint32_t q_b = smem_u32(sm.q), do_b = smem_u32(sm.dout);
      auto scores = [&](uint32_t col, uint32_t a_b, uint32_t b_b, uint64_t* bar) {  // [128 queries x 128 keys]
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * (kBlock * 128) + (kk & 3) * 32;
          umma_f16_ss(tmem + col, sdesc_sw128(a_b + off, 16, 1024), sdesc_sw128(b_b + off, 16, 1024), ID_S, kk > 0 ? 1u : 0u);
        }
        umma_commit(bar);
      };
      auto score = [&](int j) { scores((j & 1) * kBlock, q_b, smem_u32(sm.k[j % 3]), &sm.s_full[j & 1]); };
      auto dprob = [&](int j) {
        scores(DP_COL, do_b, smem_u32(sm.v[j & 1]), &sm.dp_full);
        umma_commit(&sm.v_empty[j & 1]);
      };
      bool ok = mbar_wait(&sm.q_full, 0, p.status, kTimeoutFull) && mbar_wait(&sm.k_full[0], 0, p.status, kTimeoutFull);
      if (ok) {
        tc_fence_after();
        score(0);
        ok = mbar_wait(&sm.v_full[0], 0, p.status, kTimeoutFull);
      }
      if (ok) {
        tc_fence_after();
        dprob(0);
        if (n > 1) {
          ok = mbar_wait(&sm.k_full[1], 0, p.status, kTimeoutFull);
          if (ok) {
            tc_fence_after();
            score(1);
          }
        }
      }
      for (int j = 0; ok && j < n; ++j) {
        if (j + 1 < n) {
          if (!mbar_wait(&sm.v_full[(j + 1) & 1], ((j + 1) >> 1) & 1, p.status, kTimeoutFull)) break;
          if (!mbar_wait(&sm.dp_taken, j & 1, p.status, kTimeoutFull)) break;
          tc_fence_after();
          dprob(j + 1);
        }
        if (!mbar_wait(&sm.ds_ready, j & 1, p.status, kTimeoutFull)) break;
        tc_fence_after();
        const uint32_t k_b = smem_u32(sm.k[j % 3]);
#pragma unroll
        for (int kk = 0; kk < kBlock / 16; ++kk)
          umma_f16_ts(tmem + DQ_COL, tmem + (j & 1) * kBlock + (kk >> 2) * kHalf + (kk & 3) * 8,
                      sdesc_sw128(k_b + kk * 2048, kBlock * 128, 1024), ID_G, (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&sm.k_empty[j % 3]);
        if (j + 2 < n) {  // in order after dQ(j), which reads dS from the same columns
          if (!mbar_wait(&sm.k_full[(j + 2) % 3], ((j + 2) / 3) & 1, p.status, kTimeoutFull)) break;
          tc_fence_after();
          score(j + 2);
        }
      }
      umma_commit(&sm.done);
      mbar_wait(&sm.done, 0, p.status, kTimeoutOther);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------ compute warpgroups: 64 keys each, one query per thread
    const int half = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int qi = i0 + r;
    const int lim = min(qi + s.off, s.klen - 1);  // last key this row sees
    const long long vo = h * p.pad_rows + s.pad_row0 + qi;
    const float lse2 = p.lse2[vo], delta = p.delta[vo];
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const uint32_t s_addr = tmem + lane_addr + (j & 1) * kBlock + half * kHalf;
      const uint32_t dp_addr = tmem + lane_addr + DP_COL + half * kHalf;
      if (!mbar_wait_warp(&sm.s_full[j & 1], (j >> 1) & 1, p.status, kTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float pv[kHalf];
      {
        uint32_t raw[kHalf];
        tmem_ld32(s_addr, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
        tmem_ld32(s_addr + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
        tmem_ld_wait();
        probabilities<false>(raw, pv, p.scale_log2, nullptr, lse2);
      }
      if (!mbar_wait_warp(&sm.dp_full, j & 1, p.status, kTimeoutAccFull)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t d0[32], d1[32];
      tmem_ld32(dp_addr, d0);
      tmem_ld32(dp_addr + 32, d1);
      tmem_ld_wait();
      tc_fence_before();
      mbar_arrive(&sm.dp_taken);
      const int hi = lim + 1 - j * kBlock - half * kHalf;  // columns below hi are seen
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t(&cur)[32] = c ? d1 : d0;
        float ds[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) ds[i] = pv[c * 32 + i] * (__uint_as_float(cur[i]) - delta);
        if (hi < kHalf) {
#pragma unroll
          for (int i = 0; i < 32; ++i) ds[i] = c * 32 + i < hi ? ds[i] : 0.0f;
        }
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(ds[2 * i], ds[2 * i + 1]);
        tmem_st16(s_addr + c * 16, pk);
      }
      if ((j + 1) * kBlock > s.klen) {  // the last key tile ends inside: K's rows of the next sequence (S(j) has read them)
        clear_rows<D>(sm.k[j % 3], s.klen - j * kBlock, threadIdx.x - 128, 256);
        fence_proxy_async();
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sm.ds_ready);
    }
    if (ok && mbar_wait_warp(&sm.done, 0, p.status, kTimeoutAccFull)) {
      tc_fence_after();
      constexpr int DH = D / 2;
      store_row<DH>(tmem + lane_addr + DQ_COL + half * DH, p.d0 + (static_cast<long long>(s.q0) + qi) * p.d0_n + h * p.d0_h + half * DH,
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

// Backward of packed_attn_fwd.  o, dout contiguous [Nq, Hq, D]; lse [Hq, Nq] from the forward; dq [Nq, Hq, D],
// dk/dv [Nk, Hkv, D] bf16 with any 16-byte-aligned strides (views of one packed buffer, say).  stats: fp32 scratch,
// sched: int32 scratch.
void packed_attn_bwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor o, torch::Tensor dout,
                     torch::Tensor lse, torch::Tensor cu_q, torch::Tensor cu_k, double scale, torch::Tensor dq,
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
  check_heads(dout, Hq, D, "packed_attn_bwd dout");
  check_heads(dq, Hq, D, "packed_attn_bwd dq");
  check_heads(dk, Hkv, D, "packed_attn_bwd dk");
  check_heads(dv, Hkv, D, "packed_attn_bwd dv");
  TT_CHECK(o.is_contiguous() && dout.is_contiguous() && o.size(0) == Nq && dout.size(0) == Nq && dq.size(0) == Nq &&
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
  float* lse2 = stats.data_ptr<float>();
  float* delta = lse2 + Hq * p.pad_rows;
  p.lse2 = lse2;
  p.delta = delta;
  p.scale = static_cast<float>(scale);
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  p.status = status;
  const CUtensorMap tq = head_map_3d(q, kBlock, "q"), tk = head_map_3d(k, kBlock, "k"), tv = head_map_3d(v, kBlock, "v"),
                    tdo = head_map_3d(dout, kBlock, "dout");
  // dQ's list first: it checks the offsets, and a bad packing leaves every entry empty
  schedule(p.pk, kQueryTiles, list, static_cast<int>(q_entries), status, st);
  packed_stats_kernel<<<static_cast<unsigned>(pad_slots(Nq, B)), 256, 0, st>>>(
      p.pk, list, reinterpret_cast<const __nv_bfloat16*>(o.data_ptr()), reinterpret_cast<const __nv_bfloat16*>(dout.data_ptr()),
      lse.data_ptr<float>(), lse2, delta, p.pad_rows, p.Hq, static_cast<int>(D));
  TT_CUDA_CHECK(cudaGetLastError());
  auto launch = [&](auto kern, size_t smem, int64_t blocks) {
    TT_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
    kern<<<static_cast<unsigned>(blocks), kBwdThreads, smem, st>>>(tq, tk, tv, tdo, p);
    TT_CUDA_CHECK(cudaGetLastError());
  };
  p.d0 = reinterpret_cast<__nv_bfloat16*>(dq.data_ptr());
  p.d0_n = dq.stride(0);
  p.d0_h = dq.stride(1);
  if (D == 128) launch(packed_dq_kernel<128>, dq_smem_bytes<128>() + 1024, q_entries * Hq);
  else launch(packed_dq_kernel<64>, dq_smem_bytes<64>() + 1024, q_entries * Hq);
  schedule(p.pk, kKeyTiles, list, static_cast<int>(k_entries), status, st);
  p.d0 = reinterpret_cast<__nv_bfloat16*>(dk.data_ptr());
  p.d0_n = dk.stride(0);
  p.d0_h = dk.stride(1);
  p.d1 = reinterpret_cast<__nv_bfloat16*>(dv.data_ptr());
  p.d1_n = dv.stride(0);
  p.d1_h = dv.stride(1);
  if (D == 128) launch(packed_dkv_kernel<128>, sizeof(DkvSmem<128>) + 1024, k_entries * Hkv);
  else launch(packed_dkv_kernel<64>, sizeof(DkvSmem<64>) + 1024, k_entries * Hkv);
}

}  // namespace tt

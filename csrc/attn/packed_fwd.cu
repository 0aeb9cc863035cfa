// Causal attention over packed sequences of different lengths on sm_100a tensor cores, forward,
// and the schedule that its backward shares (packed.cuh has the layout of a packing).
//
//   o_i = sum_{j <= i + len_k - len_q} softmax_j(scale q_i . k_j) v_j   within one sequence;
//   query head h reads kv head h / (Hq / Hkv); queries that see no key get zeros.
//
// One CTA per two 128-query tiles that read the same keys: the same tile of two neighbouring query heads of a
// kv head where a group has an even number of them (both tiles see as many keys, and a sequence of one tile
// fills both), else two neighbouring tiles of one head.  Warp 0 loads Q once and streams
// K/V tiles by TMA, warp 1 issues the MMAs for both query tiles in turn, and four warpgroups (warps
// 4-19) are the softmax of whichever tile has its scores: a thread takes 32 scores of one row, the
// four threads of a row share their maxima through shared memory, and P goes back over the scores in
// TMEM as the A operand of O += P V.  While the softmax works on one tile the tensor core runs the
// other's products; all four warpgroups on one tile at a time, rather than two on each, because a
// tile's softmax is on the critical path between its products.  A last, partial key tile takes rows of the next sequence:
// their probabilities are zero, but zero times an infinity or NaN of a neighbour would not be, so
// the softmax warps clear those rows of V before the product.
// Scores that are not finite stay what they are: -inf and masked keys weigh exactly zero, a NaN or +inf makes the rows that
// see it NaN (exp2_poly_any), as the definition does.  A NaN or infinity in V reaches the rows that see it, and may
// reach rows of the same sequence in the same tile that do not (zero times it).
//
// P is rounded to bf16 once, as the A operand; its row sums take the unrounded exponentials.  Three of eight exponentials
// are a polynomial good to 7.5e-5, a twentieth of that rounding.
//
// Bound by the softmax between a tile's two products (TMEM read, maxima, exponentials, P back), which the other
// tile's products hide only in part.  14 sequences, 16384 tokens, 16/4 heads, d 128 (132 GFLOP of visible
// pairs): 192 us, 690 TFLOP/s.  24 sequences of very different lengths (105 GFLOP): 166 us; with
// two warpgroups on each tile 171.
#include "attn/packed.cuh"
#include "common/fast_exp2.cuh"

#include <cmath>

namespace tt {
namespace packed {

// ----------------------------------------------------------------- schedule
constexpr int kSchedThreads = 1024;
constexpr int kBins = 2048;  // work of an entry in tiles, clamped (order only)

// Entries of sequence s, and the work of entry t (which bin: the most work first).
__device__ __forceinline__ int entries_of(const Seq& s, int kind) {
  const int rows = kind == kQueryPairs ? 2 * kBlock : kBlock;
  return ((kind == kKeyTiles ? s.klen : s.qlen) + rows - 1) / rows;
}
__device__ __forceinline__ int bin_of(const Seq& s, bool extra, int kind, int t) {
  const int rows = kind == kQueryPairs ? 2 * kBlock : kBlock;
  const int work = kind == kKeyTiles ? query_tiles(s, extra, t) : key_tiles(s, extra, t * rows, rows);
  return kBins - 1 - min(work, kBins - 1);
}

// One block: check the offsets, count entries per amount of work, and place them by falling work
// (a counting sort; the order within one amount is arbitrary and does not reach the results).
__global__ void __launch_bounds__(kSchedThreads) schedule_kernel(const Packing p, int kind, int2* list, int capacity,
                                                                 int* status) {
  __shared__ int bins[kBins];
  __shared__ int bad, total;
  __shared__ int warp_sum[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad = 0;
  for (int i = tid; i < kBins; i += kSchedThreads) bins[i] = 0;
  __syncthreads();
  bool wrong = tid == 0 && (p.cu_q[0] != 0 || p.cu_k[0] != 0 || p.cu_q[p.B] > p.Nq || p.cu_k[p.B] > p.Nk);
  for (int b = tid; b < p.B; b += kSchedThreads) wrong |= p.cu_q[b + 1] < p.cu_q[b] || p.cu_k[b + 1] < p.cu_k[b];
  if (wrong) bad = 1;
  __syncthreads();
  if (bad) {  // nothing is computed
    if (tid == 0) atomicCAS(status, 0, static_cast<int>(kBadIndex));
    for (int i = tid; i < capacity; i += kSchedThreads) list[i] = make_int2(kRejected, 0);
    return;
  }
  constexpr int kWarps = kSchedThreads / 32;
  for (int b = warp; b <= p.B; b += kWarps) {
    const Seq s = sequence(p, b);
    const int n = entries_of(s, kind);
    for (int t = lane; t < n; t += 32) atomicAdd(&bins[bin_of(s, b == p.B, kind, t)], 1);
  }
  __syncthreads();
  // exclusive prefix over the bins (two per thread)
  const int a0 = bins[2 * tid], a1 = bins[2 * tid + 1];
  int incl = a0 + a1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  int base = 0;
  for (int w = 0; w < warp; ++w) base += warp_sum[w];
  if (tid == kSchedThreads - 1) total = base + incl;
  bins[2 * tid] = base + incl - a0 - a1;
  bins[2 * tid + 1] = base + incl - a1;
  __syncthreads();
  for (int b = warp; b <= p.B; b += kWarps) {
    const Seq s = sequence(p, b);
    const int n = entries_of(s, kind);
    for (int t = lane; t < n; t += 32) {
      const int at = atomicAdd(&bins[bin_of(s, b == p.B, kind, t)], 1);
      if (at < capacity) list[at] = make_int2(b, t);
    }
  }
  for (int i = total + tid; i < capacity; i += kSchedThreads) list[i] = make_int2(kNoEntry, 0);
}
static_assert(kBins == 2 * kSchedThreads, "two bins per thread");

void schedule(const Packing& p, ScheduleKind kind, int2* list, int capacity, int* status, cudaStream_t stream) {
  schedule_kernel<<<1, kSchedThreads, 0, stream>>>(p, static_cast<int>(kind), list, capacity, status);
  TT_CUDA_CHECK(cudaGetLastError());
}

// ----------------------------------------------------------------- forward
constexpr int kThreads = 640;
constexpr int kCols = kBlock / 4;  // score columns of a softmax warpgroup
constexpr int kSoftmaxThreads = 512;
constexpr int kPolyEighths = 3;    // exponentials of eight computed on the FMA pipe (2: 167.2 us, 3: 166.0, 4: 166.6, 0: 178.9
                                   // on 16K packed prompt tokens, 16/4 heads of 128)
// Registers per thread after setmaxnreg: the launch gives 96 each, the first warpgroup hands 32 to the other four.
constexpr int kRegIssue = 64, kRegSoftmax = 104;
static_assert(kRegIssue + 4 * kRegSoftmax <= 5 * 96, "register split exceeds the launch");
constexpr float kRescale = 8.0f;  // log2 units the running maximum may lag behind

struct FwdParams {
  Packing pk;
  const int2* list;
  int Hq, Hkv;
  int head_pairs;    // a CTA's two tiles: 1 one tile of two heads, 0 two tiles of one head
  __nv_bfloat16* o;  // [Nq, Hq, D] contiguous
  __nv_bfloat16* o_lo;  // what rounding o to bf16 left over, same layout (may be null)
  float* lse;        // [Hq, Nq] natural log (may be null)
  float scale_log2;
  int* status;
};

template <int D>
struct FwdSmem {
  static constexpr int TILE = kBlock * D * 2;
  alignas(1024) uint8_t q[2][TILE];
  alignas(1024) uint8_t k[2][TILE];
  alignas(1024) uint8_t v[2][TILE];
  uint64_t q_full;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[2], p_full[2], o_done[2];
  uint64_t done;
  float row_max[2][4][kBlock];  // [query tile][warpgroup][row]; the row sums at the end
  uint32_t tmem_slot;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    packed_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                      const __grid_constant__ CUtensorMap tmV, const FwdParams p) {
  static_assert(D == 64 || D == 128, "head_dim must be 64 or 128");
  constexpr uint32_t TILE = FwdSmem<D>::TILE;
  constexpr uint32_t TMEM_COLS = 512;
  // TMEM: S/P of tile x at columns [128 x, +128) (P: bf16 pairs, each warpgroup's over the first 16 columns of its scores),
  // O of tile x at 256 + x D.
  auto S_COL = [](int x) { return static_cast<uint32_t>(x * kBlock); };
  auto O_COL = [](int x) { return static_cast<uint32_t>(2 * kBlock + x * D); };

  const int units = p.head_pairs ? p.Hq / 2 : p.Hq;
  const int2 entry = p.list[blockIdx.x / units];
  if (entry.x < 0) {  // past the end of the list (uniform over the block, nothing allocated)
    if (entry.x == kRejected) {
      zero_share<D>(p.o, p.pk.Nq, p.Hq, static_cast<long long>(p.Hq) * D, D);
      if (p.o_lo != nullptr) zero_share<D>(p.o_lo, p.pk.Nq, p.Hq, static_cast<long long>(p.Hq) * D, D);
      if (p.lse != nullptr)
        for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < static_cast<long long>(p.Hq) * p.pk.Nq;
             i += static_cast<long long>(gridDim.x) * kThreads)
          p.lse[i] = -INFINITY;
    }
    return;
  }
  const int h0 = static_cast<int>(blockIdx.x) % units * (p.head_pairs ? 2 : 1);
  const int g = h0 / (p.Hq / p.Hkv);
  const Seq s = sequence(p.pk, entry.x);
  const bool extra = entry.x == p.pk.B;
  // tile x: head h0 + x dh, queries from i0 + x di
  const int dh = p.head_pairs ? 1 : 0, di = p.head_pairs ? 0 : kBlock;
  const int i0 = entry.y * (p.head_pairs ? kBlock : 2 * kBlock);
  int n_x[2];
  n_x[0] = key_tiles(s, extra, i0, kBlock);
  n_x[1] = key_tiles(s, extra, i0 + di, kBlock);
  const int n_max = max(n_x[0], n_x[1]);

  extern __shared__ uint8_t smem_raw[];
  FwdSmem<D>& sm = *reinterpret_cast<FwdSmem<D>*>(align_ptr(smem_raw, 1024));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (n_max == 0) {  // no key is seen: zeros
    constexpr int NU = D / 8;
    for (int x = 0; x < 2; ++x) {
      const int first = i0 + x * di, rows = min(kBlock, s.qlen - first);
      for (int i = threadIdx.x; i < rows * NU; i += kThreads) {
        const long long row = s.q0 + first + i / NU;
        reinterpret_cast<uint4*>(p.o + (row * p.Hq + h0 + x * dh) * D)[i % NU] = make_uint4(0u, 0u, 0u, 0u);
        if (p.o_lo != nullptr) reinterpret_cast<uint4*>(p.o_lo + (row * p.Hq + h0 + x * dh) * D)[i % NU] = make_uint4(0u, 0u, 0u, 0u);
      }
      if (p.lse != nullptr)
        for (int i = threadIdx.x; i < rows; i += kThreads)
          p.lse[static_cast<long long>(h0 + x * dh) * p.pk.Nq + s.q0 + first + i] = -INFINITY;
    }
    return;
  }
  // rows past the sequence in its last key tile, where it is one of those seen
  const int n_keys = (s.klen + kBlock - 1) / kBlock;
  const bool clean = n_max == n_keys && s.klen % kBlock != 0;
  const int cleaner = n_x[0] == n_max ? 0 : 1;  // the tile whose P V reads the last V tile first

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    mbar_init(&sm.q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_full[i], 1);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], 1);
      mbar_init(&sm.v_empty[i], 1);
      mbar_init(&sm.s_full[i], 1);
      mbar_init(&sm.p_full[i], kSoftmaxThreads);
      mbar_init(&sm.o_done[i], 1);
    }
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

  if (warp < 4) {
  setmaxnreg_dec<kRegIssue>();
  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer
      mbar_arrive_expect_tx(&sm.q_full, 2 * TILE);
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.q[x] + c * kBlock * 128, &tmQ, &sm.q_full, c * 64, h0 + x * dh, s.q0 + i0 + x * di);
      for (int j = 0; j < n_max; ++j) {
        const int st = j & 1;
        const uint32_t ph = (j >> 1) & 1;
        if (!mbar_wait(&sm.k_empty[st], ph ^ 1u, p.status, kTimeoutEmpty)) break;
        mbar_arrive_expect_tx(&sm.k_full[st], TILE);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.k[st] + c * kBlock * 128, &tmK, &sm.k_full[st], c * 64, g, s.k0 + j * kBlock);
        if (!mbar_wait(&sm.v_empty[st], ph ^ 1u, p.status, kTimeoutEmpty)) break;
        mbar_arrive_expect_tx(&sm.v_full[st], TILE);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(sm.v[st] + c * kBlock * 128, &tmV, &sm.v_full[st], c * 64, g, s.k0 + j * kBlock);
      }
      mbar_wait(&sm.q_full, 0, p.status, kTimeoutOther);
      for (int j = max(0, n_max - 2); j < n_max; ++j) {  // every copy has landed before the block ends
        mbar_wait(&sm.k_full[j & 1], (j >> 1) & 1, p.status, kTimeoutOther);
        mbar_wait(&sm.v_full[j & 1], (j >> 1) & 1, p.status, kTimeoutOther);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer, the two query tiles in turn
    const bool lead = elect_one();
    auto qk = [&](int x, int j) {
      product_abt<D>(lead, tmem + S_COL(x), desc_k_major(sm.q[x]), desc_k_major(sm.k[j & 1]), &sm.s_full[x]);
    };
    auto pv = [&](int x, int j) {
      product_ab<D, kCols>(lead, tmem + O_COL(x), tmem + S_COL(x), desc_mn_major(sm.v[j & 1]), j > 0);
      commit(lead, &sm.o_done[x]);
    };
    bool ok = mbar_wait_warp(&sm.q_full, 0, p.status, kTimeoutFull) && mbar_wait_warp(&sm.k_full[0], 0, p.status, kTimeoutFull);
    if (ok) {
      tc_fence_after();
      for (int x = 0; x < 2; ++x)
        if (n_x[x] > 0) qk(x, 0);
      commit(lead, &sm.k_empty[0]);
    }
    for (int j = 0; ok && j < n_max; ++j) {
      const bool next = j + 1 < n_max;
      if (!mbar_wait_warp(&sm.v_full[j & 1], (j >> 1) & 1, p.status, kTimeoutFull)) break;
      if (next && !mbar_wait_warp(&sm.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, p.status, kTimeoutFull)) break;
      tc_fence_after();
      for (int x = 0; x < 2; ++x) {
        if (j < n_x[x]) {
          if (!mbar_wait_warp(&sm.p_full[x], j & 1, p.status, kTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          pv(x, j);
        }
        if (j + 1 < n_x[x]) qk(x, j + 1);  // in order after PV(x, j), which read P from these columns
      }
      if (!ok) break;
      commit(lead, &sm.v_empty[j & 1]);
      if (next) commit(lead, &sm.k_empty[(j + 1) & 1]);
    }
    commit(lead, &sm.done);
    mbar_wait_warp(&sm.done, 0, p.status, kTimeoutOther);
  }
  } else {
    setmaxnreg_inc<kRegSoftmax>();
    // ------------------------------------------------ softmax: columns [32 wg, +32) of both tiles, one row of each per thread
    const int wg = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const float sl2 = p.scale_log2;
    constexpr int W = D / 4;                         // columns of O that this thread rescales and writes
    float m_ref[2] = {-INFINITY, -INFINITY};         // reference maximum, scaled log2 units (the same in a row's four threads)
    float l[2] = {0.0f, 0.0f};                       // sums over this thread's columns
    // The warpgroups meet once per tile: after a wait that gave up they go on meeting (and compute nothing), so that
    // none is left waiting for another.
    auto meet = [&]() { asm volatile("bar.sync 1, 512;" ::: "memory"); };
    bool ok = true;
    for (int j = 0; j < n_max; ++j) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (j >= n_x[x]) continue;
        if (ok) ok = mbar_wait_warp(&sm.s_full[x], j & 1, p.status, kTimeoutAccFull);
        if (!ok) {
          meet();
          continue;
        }
        tc_fence_after();
        const uint32_t s_addr = tmem + lane_addr + S_COL(x) + wg * kCols;
        uint32_t raw[kCols];
        tmem_ld32(s_addr, raw);
        tmem_ld_wait();
        const int lim = min(i0 + x * di + r + s.off, s.klen - 1);  // last key this row sees (negative: none)
        const int left = lim - j * kBlock - wg * kCols;            // columns up to `left` are seen
        if (left < kCols - 1) {
#pragma unroll
          for (int i = 0; i < kCols; ++i) raw[i] = i > left ? 0xff800000u : raw[i];  // -inf
        }
        float mq[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          mq[q] = fmax3(__uint_as_float(raw[8 * q]), __uint_as_float(raw[8 * q + 1]), __uint_as_float(raw[8 * q + 2]));
          mq[q] = fmax3(mq[q], __uint_as_float(raw[8 * q + 3]), __uint_as_float(raw[8 * q + 4]));
          mq[q] = fmax3(mq[q], __uint_as_float(raw[8 * q + 5]), fmaxf(__uint_as_float(raw[8 * q + 6]), __uint_as_float(raw[8 * q + 7])));
        }
        sm.row_max[x][wg][r] = fmax3(mq[0], mq[1], fmaxf(mq[2], mq[3]));
        // They are overwritten once S(x, j + 1) is there: its product follows P V(x, j), which every thread lets go
        // only after the reads below.
        meet();
        const float m_tile = fmaxf(fmaxf(sm.row_max[x][0][r], sm.row_max[x][1][r]), fmaxf(sm.row_max[x][2][r], sm.row_max[x][3][r])) * sl2;
        // The reference rises only when the tile's maximum exceeds it by more than 2^8: no exponential overflows,
        // and after the first tiles of a row almost none has to be rescaled.
        const bool raise = m_tile > m_ref[x] + kRescale;  // also the first visible tile (m_ref = -inf)
        const float alpha = raise ? ex2_mufu(m_ref[x] - m_tile) : 1.0f;
        if (raise) m_ref[x] = m_tile;
        const float neg_m = (m_ref[x] == -INFINITY) ? 0.0f : -m_ref[x];
        const unsigned long long s2 = f2_pack(sl2, sl2), nm2 = f2_pack(neg_m, neg_m);
        unsigned long long sa = 0ull, sb = 0ull;  // pairs of partial sums
        uint32_t pk[kCols / 2];
#pragma unroll
        for (int i = 0; i < kCols; i += 2) {
          float e0, e1;
          f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[i]), __uint_as_float(raw[i + 1])), s2, nm2), e0, e1);
          // part of the exponentials on the FMA pipe, so that MUFU does not bound the tile
          if ((i & 7) == 6 || (kPolyEighths == 4 && (i & 7) == 2)) {
            exp2_poly2_any(e0, e1);
          } else {
            e0 = ex2_mufu(e0);
            e1 = (kPolyEighths == 3 && (i & 7) == 2) ? exp2_poly_any(e1) : ex2_mufu(e1);
          }
          if (i & 2) sb = f2_add(sb, f2_pack(e0, e1));
          else sa = f2_add(sa, f2_pack(e0, e1));
          pk[i >> 1] = pack_bf16x2(e0, e1);
        }
        tmem_st16(s_addr, pk);
        float s0, s1;
        f2_unpack(f2_add(sa, sb), s0, s1);
        l[x] = l[x] * alpha + (s0 + s1);
        if (__any_sync(0xffffffffu, raise && j > 0)) {  // rare: O under an older reference, this thread's columns
          const uint32_t o_addr = tmem + lane_addr + O_COL(x) + wg * W;
#pragma unroll
          for (int c = 0; c < W; c += 16) {
            uint32_t ov[16];
            tmem_ld16(o_addr + c, ov);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
            tmem_st16(o_addr + c, ov);
          }
        }
        // S(j) is there, so P V(j - 2) is done and this buffer's current or last phase is V(j)'s
        if (clean && x == cleaner && j == n_max - 1) {
          if (!mbar_wait_warp(&sm.v_full[j & 1], (j >> 1) & 1, p.status, kTimeoutFull)) {
            ok = false;
            continue;
          }
          clear_rows<D>(sm.v[j & 1], s.klen - j * kBlock, wg * kBlock + r, kSoftmaxThreads);
          fence_proxy_async();
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&sm.p_full[x]);
      }
    }
    // ------------------------------------------------ O / l and the log-sum-exp
    meet();  // the maxima have been read
#pragma unroll
    for (int x = 0; x < 2; ++x) sm.row_max[x][wg][r] = l[x];
    meet();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int qi = i0 + x * di + r;  // query within the sequence
      const int h = h0 + x * dh;
      const bool row_ok = qi < s.qlen;
      const long long row = s.q0 + qi;
      const long long at = (row * p.Hq + h) * D + wg * W;
      const bool seen = min(qi + s.off, s.klen - 1) >= 0;
      uint32_t w[W / 2], rest[W / 2];
      if (n_x[x] == 0) {
#pragma unroll
        for (int i = 0; i < W / 2; ++i) w[i] = rest[i] = 0u;
      } else {
        if (!ok || !mbar_wait_warp(&sm.o_done[x], (n_x[x] - 1) & 1, p.status, kTimeoutAccFull)) break;
        tc_fence_after();
        const float sum = (sm.row_max[x][0][r] + sm.row_max[x][1][r]) + (sm.row_max[x][2][r] + sm.row_max[x][3][r]);
        const float inv_l = 1.0f / sum;
        uint32_t ov[W];
        const uint32_t o_addr = tmem + lane_addr + O_COL(x) + wg * W;
        if constexpr (W == 32) tmem_ld32(o_addr, ov);
        else tmem_ld16(o_addr, ov);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < W / 2; ++i) {
          const float a = __uint_as_float(ov[2 * i]) * inv_l, c = __uint_as_float(ov[2 * i + 1]) * inv_l;
          w[i] = seen ? pack_bf16x2(a, c) : 0u;
          const float2 f = unpack_bf16x2(w[i]);
          rest[i] = seen ? pack_bf16x2(a - f.x, c - f.y) : 0u;
        }
        if (row_ok && wg == 0 && p.lse != nullptr)
          p.lse[static_cast<long long>(h) * p.pk.Nq + row] = seen ? (m_ref[x] + log2f(sum)) * 0.69314718055994531f : -INFINITY;
      }
      if (row_ok) {
#pragma unroll
        for (int i = 0; i < W / 8; ++i) reinterpret_cast<uint4*>(p.o + at)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        if (p.o_lo != nullptr) {
#pragma unroll
          for (int i = 0; i < W / 8; ++i)
            reinterpret_cast<uint4*>(p.o_lo + at)[i] = make_uint4(rest[4 * i], rest[4 * i + 1], rest[4 * i + 2], rest[4 * i + 3]);
        }
        if (n_x[x] == 0 && wg == 0 && p.lse != nullptr) p.lse[static_cast<long long>(h) * p.pk.Nq + row] = -INFINITY;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace packed

// int32 elements of the schedule that packed_attn_fwd needs.
int64_t packed_attn_schedule_numel(int64_t Nq, int64_t Nk, int64_t B) {
  using namespace packed;
  return 2 * std::max(max_tiles(Nq, B, kBlock), max_tiles(Nk, B, kBlock));
}

// q [Nq, Hq, D], k/v [Nk, Hkv, D] bf16 (any 16-byte-aligned strides), cu_q/cu_k int32 [B + 1] ->
// o [Nq, Hq, D] contiguous; for a backward, lse fp32 [Hq, Nq] and o_lo (o's layout): what the rounding of o left
// over, so that delta = dO . O is not off by it (0.0026 -> 0.0024 relative error of dQ).  sched: int32 scratch.
void packed_attn_fwd(torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor cu_q, torch::Tensor cu_k,
                     double scale, torch::Tensor o, c10::optional<torch::Tensor> lse, c10::optional<torch::Tensor> o_lo,
                     torch::Tensor sched) {
  using namespace packed;
  TT_CHECK(q.dim() == 3 && k.dim() == 3, "packed_attn: q and k must be [tokens, heads, D]");
  const int64_t Nq = q.size(0), Hq = q.size(1), D = q.size(2), Nk = k.size(0), Hkv = k.size(1);
  TT_CHECK(D == 64 || D == 128, "packed_attn: head_dim must be 64 or 128");
  TT_CHECK(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0, "packed_attn: Hq must be a multiple of Hkv");
  check_heads(q, Hq, D, "packed_attn q");
  check_heads(k, Hkv, D, "packed_attn k");
  check_heads(v, Hkv, D, "packed_attn v");
  TT_CHECK(v.size(0) == Nk, "packed_attn: k and v must have as many tokens");
  check_offsets(cu_q, -1, "cu_seqlens");
  check_offsets(cu_k, cu_q.numel(), "cu_seqlens_k");
  const int64_t B = cu_q.numel() - 1;
  check_cuda_bf16(o, "o");
  TT_CHECK(o.is_contiguous() && o.numel() == Nq * Hq * D && reinterpret_cast<uintptr_t>(o.data_ptr()) % 16 == 0,
           "packed_attn: o must be contiguous [Nq, Hq, D]");
  if (lse.has_value())
    TT_CHECK(lse->scalar_type() == torch::kFloat32 && lse->is_contiguous() && lse->numel() == Hq * Nq, "packed_attn: lse must be fp32 [Hq, Nq]");
  if (o_lo.has_value()) {
    check_cuda_bf16(*o_lo, "o_lo");
    TT_CHECK(o_lo->is_contiguous() && o_lo->numel() == o.numel() && reinterpret_cast<uintptr_t>(o_lo->data_ptr()) % 16 == 0,
             "packed_attn: o_lo must be contiguous [Nq, Hq, D]");
  }
  TT_CHECK(scale > 0 && std::isfinite(scale), "packed_attn: scale must be positive and finite");
  TT_CHECK(sched.scalar_type() == torch::kInt32 && sched.is_contiguous() && sched.numel() >= packed_attn_schedule_numel(Nq, Nk, B) &&
               reinterpret_cast<uintptr_t>(sched.data_ptr()) % 8 == 0,
           "packed_attn: schedule scratch too small");
  if (Nq == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  TT_CUDA_CHECK(cudaSetDevice(q.get_device()));  // binds the context to this thread: the tensor maps need one
  if (Nk == 0) {  // no keys at all (a tensor map cannot be empty)
    o.zero_();
    if (lse.has_value()) lse->fill_(-INFINITY);
    if (o_lo.has_value()) o_lo->zero_();
    return;
  }
  FwdParams p{};
  p.pk = packing_of(q, k, cu_q, cu_k);
  p.list = reinterpret_cast<const int2*>(sched.data_ptr<int>());
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.o = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
  p.o_lo = o_lo.has_value() ? reinterpret_cast<__nv_bfloat16*>(o_lo->data_ptr()) : nullptr;
  p.lse = lse.has_value() ? lse->data_ptr<float>() : nullptr;
  p.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  p.status = device_status_ptr(q.get_device());
  const CUtensorMap tq = head_map_3d(q, kBlock, "q"), tk = head_map_3d(k, kBlock, "k"), tv = head_map_3d(v, kBlock, "v");
  p.head_pairs = (Hq / Hkv) % 2 == 0 ? 1 : 0;
  const int64_t entries = max_tiles(Nq, B, p.head_pairs ? kBlock : 2 * kBlock);
  const int64_t blocks = entries * (p.head_pairs ? Hq / 2 : Hq);
  TT_CHECK(blocks < (1LL << 31), "packed_attn: too many tiles");
  schedule(p.pk, p.head_pairs ? kQueryTiles : kQueryPairs, reinterpret_cast<int2*>(sched.data_ptr<int>()), static_cast<int>(entries), p.status, cur_stream());
  const int device = q.get_device();
  auto launch = [&](auto d) {
    constexpr int kD = decltype(d)::value;
    constexpr size_t smem = sizeof(FwdSmem<kD>) + 1024;
    allow_smem<&packed_fwd_kernel<kD>>(smem, device);
    packed_fwd_kernel<kD><<<static_cast<unsigned>(blocks), kThreads, smem, cur_stream()>>>(tq, tk, tv, p);
  };
  if (D == 128) launch(std::integral_constant<int, 128>{});
  else launch(std::integral_constant<int, 64>{});
  TT_CUDA_CHECK(cudaGetLastError());
}

}  // namespace tt

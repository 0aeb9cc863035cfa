// Attention of one new token per sequence over a paged KV cache, every sequence with a length
// of its own.
//
//   o[b, h] = sum_{j < len_b} softmax_j(scale q[b, h] . k[b, j]) v[b, j]
//
// Bound by the K and V bytes (2 * len * Hkv * D * 2 per sequence, read once for all query heads
// of a kv head).  What decides the time besides that is how evenly the work lies over the SMs
// when lengths differ, so it is not split per sequence: all (sequence, kv head, 64-key tile)
// units form one line, and each of the resident CTAs takes an equal stretch of it, whichever
// sequences that crosses.  The lengths stay on the device (a captured step replays with new
// ones): every CTA scans them itself.  A stretch that covers a (sequence, head) whole writes
// its output; otherwise it leaves a partial (max, sum, O in fp32), and the CTA that finishes a
// (sequence, head) last joins its partials in the order of the keys, so the result does not
// depend on which CTA that was.
//
// Inside a CTA: two producer warps stream K and V tiles through a ring of kStages buffers by 16-byte
// asynchronous copies (half a warp per row of a head; pages looked up one tile ahead), so any page
// size and order costs the same; and each of four consumer warps works on 16 keys of a tile by itself:
// S = Q K^T and O += P V as 16x8x16 warp MMAs with the query heads of the kv head as the rows (up to
// 16; tcgen05 needs 64 and would not move one byte faster), P passing from accumulator to operand in
// registers.  The warps' softmax states meet once per stretch, not per tile.
//
// P is rounded to bf16 once, as the MMA operand; maxima, sums, partials and the join are fp32.
//
// Measured (L2 flushed): 140K tokens of 40/8 heads, d 128 (574 MB): 102 us, 5.6 TB/s; 32 sequences of about
// 1.1K tokens, 16/4 heads (74 MB): 28 us, of which about 10 are start-up and the join.
#include "common/host_utils.h"
#include "common/ptx.cuh"
#include "common/fast_exp2.cuh"

#include <mutex>

namespace tt {
namespace paged {

constexpr int kTile = 64;      // keys per unit
constexpr int kWarps = 4;       // consumer warps, 16 keys each
constexpr int kProducers = 64;  // threads of the two producer warps, 32 keys each
constexpr int kThreads = kWarps * 32 + kProducers;
constexpr int kAllWarps = kThreads / 32;
constexpr int kStages = 3;
constexpr int kCtasPerSm = 2;
constexpr int kMaxG = 16;      // query heads per kv head
constexpr float kLog2e = 1.4426950408889634f;
static_assert(kWarps * 16 == kTile, "16 keys per warp");

struct Params {
  const __nv_bfloat16* q;        // [B, Hq, D] with strides
  long long q_ld_b, q_ld_h;
  const __nv_bfloat16* k_pages;  // [pages, page_size, Hkv, D]
  const __nv_bfloat16* v_pages;
  const int* table;              // [B, width]
  const int* lens;               // [B]
  int B, Hq, Hkv, G;
  int width, page_size, num_pages;
  float scale_log2;
  float* part_o;                 // [2 * gridDim.x, G, D]
  float* part_ml;                // [2 * gridDim.x, G, 2]
  int* counters;                 // [B * Hkv], zero between calls
  __nv_bfloat16* out;            // [B, Hq, D] contiguous
  int* status;
};

__device__ __forceinline__ void cp_async16(uint32_t smem, const void* gmem, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(valid ? 16 : 0) : "memory");
}
// Arrive on the barrier when this thread's copies so far have landed (counted in the barrier's expected arrivals).
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void consumers_meet() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
static_assert(kWarps * 32 == 128, "the consumers' barrier");
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int D>
struct Smem {
  alignas(128) uint8_t k[kStages][kTile * D * 2];
  alignas(128) uint8_t v[kStages][kTile * D * 2];
  float m[kWarps][kMaxG], l[kWarps][kMaxG];
  uint64_t full[kStages], empty[kStages];
  int scan[kAllWarps];
  int find[3];
  int last;
};

// Byte offset of 16-byte unit `u` of row `r`: units are permuted by the row within its group of
// 8, so the 8 rows of an ldmatrix fall into distinct banks.
template <int D>
__device__ __forceinline__ uint32_t unit_off(int r, int u) {
  return static_cast<uint32_t>(r * D * 2 + ((u ^ (r & 7)) << 4));
}

// Units of a sequence: its 64-key tiles (0 for an empty one).
__device__ __forceinline__ int seq_len(const Params& p, int b) {
  const int n = p.lens[b];
  const long long most = static_cast<long long>(p.width) * p.page_size;
  return n < 0 ? 0 : static_cast<int>(min(static_cast<long long>(n), most));
}

// Inclusive scan over the block's threads within their warp; base: the sum of the warps before, sum: of all.
__device__ __forceinline__ int block_scan(int n, int lane, int warp, int* scratch, int& base, int& sum) {
  int incl = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  base = 0;
  sum = 0;
#pragma unroll
  for (int w = 0; w < kAllWarps; ++w) {
    if (w < warp) base += scratch[w];
    sum += scratch[w];
  }
  __syncthreads();
  return incl;
}

template <int D>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_decode_kernel(const Params p) {
  static_assert(D == 64 || D == 128, "head_dim 64 or 128");
  constexpr int NU = D / 8;          // 16-byte units per row
  constexpr int KS = D / 16;         // MMA k-steps of Q K^T
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x;

  // ---- the line of units: its length, and where this CTA's stretch begins.  One scan where a step of it holds
  // all sequences, a second one over the steps otherwise.
  int n_first = 0, incl_first = 0;  // of this thread's sequence in the first step
  long long total_tiles = 0;        // tiles per kv head over all sequences
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    const int b = b0 + tid;
    int n = 0;
    if (b < p.B) {
      const int len = seq_len(p, b);
      if (len != p.lens[b] && cta == 0) atomicCAS(p.status, 0, static_cast<int>(kBadIndex));  // negative, or past the table
      n = (len + kTile - 1) / kTile;
      if (len == 0 && b % static_cast<int>(gridDim.x) == cta) {  // no keys: the output is zero
        uint4* o = reinterpret_cast<uint4*>(p.out + static_cast<long long>(b) * p.Hq * D);
        for (int i = 0; i < p.Hq * NU; ++i) o[i] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    int base, sum;
    const int incl = block_scan(n, lane, warp, sm.scan, base, sum) + base;
    if (b0 == 0) {
      n_first = n;
      incl_first = incl;
    }
    total_tiles += sum;
  }
  const long long W = total_tiles * p.Hkv;
  const int ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), W));  // each has a unit at least
  if (cta >= ctas) return;
  const long long u0 = W * cta / ctas, u1 = W * (cta + 1) / ctas;  // this CTA's units
  {
    long long before = 0;  // units of the sequences before b0
    for (int b0 = 0; b0 < p.B; b0 += kThreads) {
      const int b = b0 + tid;
      int n = n_first, incl = incl_first, base, sum = 0;
      if (b0 > 0) {
        n = b < p.B ? (seq_len(p, b) + kTile - 1) / kTile : 0;
        incl = block_scan(n, lane, warp, sm.scan, base, sum) + base;
      } else if (p.B > kThreads) {
        block_scan(n, lane, warp, sm.scan, base, sum);
      }
      const long long first = before + static_cast<long long>(incl - n) * p.Hkv;
      const long long end = first + static_cast<long long>(n) * p.Hkv;
      if (n > 0 && first <= u0 && u0 < end) {
        const int r = static_cast<int>(u0 - first);
        sm.find[0] = b;
        sm.find[1] = r / n;
        sm.find[2] = r % n;
      }
      before += static_cast<long long>(sum) * p.Hkv;
      if (before > u0) break;
    }
  }
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sm.full[i], kProducers);
      mbar_init(&sm.empty[i], kWarps);
    }
    fence_barrier_init();
  }
  __syncthreads();
  int b = sm.find[0], kvh = sm.find[1], tile = sm.find[2];
  int len = seq_len(p, b), n_tiles = (len + kTile - 1) / kTile;

  const int count = static_cast<int>(u1 - u0);
  const uint32_t k_base = smem_u32(sm.k[0]), v_base = smem_u32(sm.v[0]);
  constexpr uint32_t STAGE = kTile * D * 2;

  if (warp >= kWarps) {
    // ---------------------------------------------------------------- producers: keys [32 w, 32 w + 32) of every tile
    const int row0 = (warp - kWarps) * 32;
    int page = -1, off = -1;  // of this lane's key of tile (b, tile); off < 0: no key
    auto look_up = [&]() {
      const int key = tile * kTile + row0 + lane;
      page = -1;
      off = -1;
      if (key < len) {
        const int pi = key / p.page_size;
        off = key - pi * p.page_size;
        page = p.table[static_cast<long long>(b) * p.width + pi];
      }
    };
    look_up();
    for (int i = 0; i < count; ++i) {
      const bool mapped = page >= 0 && page < p.num_pages;
      if (off >= 0 && !mapped) atomicCAS(p.status, 0, static_cast<int>(kBadIndex));
      const int row = off >= 0 && mapped ? page * p.page_size + off : -1;
      const int head = kvh;
      if (++tile * kTile >= len) {  // the tile after this one
        tile = 0;
        if (++kvh == p.Hkv) {
          kvh = 0;
          if (i + 1 < count) {
            do { ++b; len = seq_len(p, b); } while (len == 0);
          }
        }
      }
      if (i + 1 < count) look_up();  // its latency lies beside this tile's copies
      const int st = i % kStages;
      if (!mbar_wait_warp(&sm.empty[st], ((i / kStages) & 1) ^ 1u, p.status, kTimeoutEmpty)) break;
      const int u = lane % NU;
#pragma unroll 4
      for (int j = 0; j < NU; ++j) {  // 32 / NU rows of a head at a time
        const int r = j * (32 / NU) + lane / NU;
        const int from = __shfl_sync(0xffffffffu, row, r);
        const long long at = from >= 0 ? (static_cast<long long>(from) * p.Hkv + head) * D + 8 * u : 0;
        const uint32_t to = st * STAGE + unit_off<D>(row0 + r, u);
        cp_async16(k_base + to, p.k_pages + at, from >= 0);
        cp_async16(v_base + to, p.v_pages + at, from >= 0);
      }
      cp_async_arrive(&sm.full[st]);
    }
    cp_async_wait_all();
    return;
  }
  // ------------------------------------------------------------------ consumers
  const int g = lane >> 2, c2 = 2 * (lane & 3);  // accumulator row (and g + 8), column pair
  const int lr = lane & 7, lm = lane >> 3;       // ldmatrix: row in a matrix, matrix
  int done = 0;
  int seg = 0;  // partial slot of this CTA: 0 for the stretch's first (sequence, head), 1 for its last
  while (done < count) {
    const int seg_tile0 = tile;
    const int seg_tiles = min(n_tiles - tile, count - done);
    // query heads as the A operand of Q K^T (rows past G are zero)
    uint32_t qf[KS][4];
    {
      const __nv_bfloat16* qb = p.q + b * p.q_ld_b + static_cast<long long>(kvh) * p.G * p.q_ld_h;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = g + (i & 1) * 8, c = k * 16 + c2 + (i >> 1) * 8;
          qf[k][i] = r < p.G ? *reinterpret_cast<const uint32_t*>(qb + r * p.q_ld_h + c) : 0u;
        }
      }
    }
    float o[NU][4];
#pragma unroll
    for (int i = 0; i < NU; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;  // rows g, g + 8 of this warp's keys
    for (int it = 0; it < seg_tiles; ++it, ++done, ++tile) {
      const int s = done % kStages;
      if (!mbar_wait_warp(&sm.full[s], (done / kStages) & 1, p.status, kTimeoutFull)) continue;  // and the next, and the end
      const uint32_t kb = k_base + s * STAGE, vb = v_base + s * STAGE;
      const int key0 = tile * kTile + warp * 16;
      if (key0 < len) {  // else none of this warp's keys
      float sc[2][4] = {};
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t bk[4];
        const int r = warp * 16 + (lm >> 1) * 8 + lr;
        ldsm_x4(bk, kb + unit_off<D>(r, 2 * k + (lm & 1)));
        mma_16816(sc[0], qf[k], bk[0], bk[1]);
        mma_16816(sc[1], qf[k], bk[2], bk[3]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + t * 8 + c2 + (j & 1);
          sc[t][j] = key < len ? sc[t][j] * p.scale_log2 : -INFINITY;
        }
      float n0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
      float n1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, x));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, x));
      }
      if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {  // a larger score: rescale (rare after the first tiles)
        const float a0 = n0 > m0 ? ex2_mufu(m0 - n0) : 1.0f, a1 = n1 > m1 ? ex2_mufu(m1 - n1) : 1.0f;
        m0 = fmaxf(m0, n0);
        m1 = fmaxf(m1, n1);
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          o[i][0] *= a0;
          o[i][1] *= a0;
          o[i][2] *= a1;
          o[i][3] *= a1;
        }
      }
      const float r0 = m0 == -INFINITY ? 0.0f : m0, r1 = m1 == -INFINITY ? 0.0f : m1;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sc[t][0] = ex2_mufu(sc[t][0] - r0);
        sc[t][1] = ex2_mufu(sc[t][1] - r0);
        sc[t][2] = ex2_mufu(sc[t][2] - r1);
        sc[t][3] = ex2_mufu(sc[t][3] - r1);
        l0 += sc[t][0] + sc[t][1];
        l1 += sc[t][2] + sc[t][3];
      }
      // accumulator layout of S (16 heads x 16 keys) = operand layout of P
      const uint32_t pa[4] = {pack_bf16x2(sc[0][0], sc[0][1]), pack_bf16x2(sc[0][2], sc[0][3]),
                              pack_bf16x2(sc[1][0], sc[1][1]), pack_bf16x2(sc[1][2], sc[1][3])};
#pragma unroll
      for (int i = 0; i < NU; i += 2) {
        uint32_t bv[4];
        const int r = warp * 16 + (lm & 1) * 8 + lr;
        ldsm_x4_t(bv, vb + unit_off<D>(r, i + (lm >> 1)));
        mma_16816(o[i], pa, bv[0], bv[1]);
        mma_16816(o[i + 1], pa, bv[2], bv[3]);
      }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[s]);
    }
    // ---- the four warps' states of this (sequence, head) into one
#pragma unroll
    for (int x = 1; x < 4; x <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, x);
      l1 += __shfl_xor_sync(0xffffffffu, l1, x);
    }
    if ((lane & 3) == 0) {
      sm.m[warp][g] = m0;
      sm.m[warp][g + 8] = m1;
      sm.l[warp][g] = l0;
      sm.l[warp][g + 8] = l1;
    }
    consumers_meet();
    float M0 = sm.m[0][g], M1 = sm.m[0][g + 8];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      M0 = fmaxf(M0, sm.m[w][g]);
      M1 = fmaxf(M1, sm.m[w][g + 8]);
    }
    const float f0 = m0 == -INFINITY ? 0.0f : ex2_mufu(m0 - M0), f1 = m1 == -INFINITY ? 0.0f : ex2_mufu(m1 - M1);
    // O tiles pass through shared memory in warp order; the K/V ring holds tiles still to come, so a
    // region of its own
    float* acc = reinterpret_cast<float*>(smem_raw + sizeof(Smem<D>));  // [kMaxG][D]
    for (int w = 0; w < kWarps; ++w) {
      if (warp == w) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
          float2* a0 = reinterpret_cast<float2*>(acc + g * D + i * 8 + c2);
          float2* a1 = reinterpret_cast<float2*>(acc + (g + 8) * D + i * 8 + c2);
          const float2 x0 = w ? *a0 : make_float2(0.0f, 0.0f), x1 = w ? *a1 : make_float2(0.0f, 0.0f);
          *a0 = make_float2(x0.x + f0 * o[i][0], x0.y + f0 * o[i][1]);
          *a1 = make_float2(x1.x + f1 * o[i][2], x1.y + f1 * o[i][3]);
        }
      }
      consumers_meet();
    }
    const bool whole = seg_tile0 == 0 && seg_tiles == n_tiles;
    const long long pair = static_cast<long long>(b) * p.Hkv + kvh;
    if (whole) {
      for (int i = tid; i < p.G * D / 2; i += kWarps * 32) {
        const int h = i / (D / 2), d = 2 * (i % (D / 2));
        float M = sm.m[0][h], L = 0.0f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sm.m[w][h]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) L += sm.m[w][h] == -INFINITY ? 0.0f : ex2_mufu(sm.m[w][h] - M) * sm.l[w][h];
        const float inv = 1.0f / L;
        *reinterpret_cast<uint32_t*>(p.out + (pair * p.G + h) * D + d) = pack_bf16x2(acc[h * D + d] * inv, acc[h * D + d + 1] * inv);
      }
    } else {
      const long long slot = 2ll * cta + seg;
      for (int i = tid; i < p.G * D / 4; i += kWarps * 32)
        reinterpret_cast<float4*>(p.part_o + slot * p.G * D)[i] = reinterpret_cast<const float4*>(acc)[i];
      if (tid < p.G) {
        float M = sm.m[0][tid], L = 0.0f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sm.m[w][tid]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) L += sm.m[w][tid] == -INFINITY ? 0.0f : ex2_mufu(sm.m[w][tid] - M) * sm.l[w][tid];
        p.part_ml[(slot * p.G + tid) * 2] = M;
        p.part_ml[(slot * p.G + tid) * 2 + 1] = L;
      }
      // units of this (sequence, head) on the line, and the CTAs that share them
      const long long first = u0 + done - (seg_tile0 + seg_tiles), end = first + n_tiles;
      const int ca = static_cast<int>(((first + 1) * ctas - 1) / W), cb = static_cast<int>((end * ctas - 1) / W);
      __threadfence();
      consumers_meet();
      if (tid == 0) sm.last = atomicAdd(p.counters + pair, 1) == cb - ca ? 1 : 0;
      consumers_meet();
      if (sm.last) {  // all partials are there: join them in key order
        __threadfence();
        if (tid == 0) p.counters[pair] = 0;
        // A CTA's partial of this pair is its first one unless the pair began inside its stretch.
        auto slot_of = [&](int c) { return (2ll * c + ((c == ca && W * c / ctas < first) ? 1 : 0)) * p.G; };
        for (int h = warp; h < p.G; h += kWarps) {  // the heads' maxima and sums, lanes over the partials
          float M = -INFINITY, L = 0.0f;
          for (int c = ca + lane; c <= cb; c += 32) M = fmaxf(M, __ldcg(p.part_ml + (slot_of(c) + h) * 2));
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
          for (int c = ca + lane; c <= cb; c += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + (slot_of(c) + h) * 2));
            if (ml.x != -INFINITY) L = fmaf(ex2_mufu(ml.x - M), ml.y, L);
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
          if (lane == 0) {
            sm.m[0][h] = M;
            sm.l[0][h] = 1.0f / L;
          }
        }
        consumers_meet();
        for (int i = tid; i < p.G * D / 4; i += kWarps * 32) {
          const int h = i / (D / 4), d = 4 * (i % (D / 4));
          const float M = sm.m[0][h];
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          constexpr int kBatch = 8;  // partials loaded at once
          for (int c0 = ca; c0 <= cb; c0 += kBatch) {
            float f[kBatch];
            float4 v[kBatch];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
              const long long sl = slot_of(min(c0 + n, cb)) + h;
              f[n] = __ldcg(p.part_ml + sl * 2);
              v[n] = __ldcg(reinterpret_cast<const float4*>(p.part_o + sl * D + d));
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
              const float w = (c0 + n > cb || f[n] == -INFINITY) ? 0.0f : ex2_mufu(f[n] - M);
              x.x = fmaf(w, v[n].x, x.x);
              x.y = fmaf(w, v[n].y, x.y);
              x.z = fmaf(w, v[n].z, x.z);
              x.w = fmaf(w, v[n].w, x.w);
            }
          }
          const float inv = sm.l[0][h];
          *reinterpret_cast<uint2*>(p.out + (pair * p.G + h) * D + d) =
              make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
        }
      }
    }
    consumers_meet();  // acc, m and l are free again
    seg = 1;
    if (tile == n_tiles) {
      tile = 0;
      if (++kvh == p.Hkv) {
        kvh = 0;
        if (done < count) {
          do { ++b; len = seq_len(p, b); } while (len == 0);
          n_tiles = (len + kTile - 1) / kTile;
        }
      }
    }
  }
}

template <int D>
constexpr size_t smem_bytes() { return sizeof(Smem<D>) + kMaxG * D * sizeof(float); }

// CTAs of a call: all that are resident at once, or fewer where even full tables hold fewer units.
int grid_size(int64_t B, int64_t Hkv, int64_t max_keys, int device) {
  const long long units = static_cast<long long>(B) * Hkv * ((max_keys + kTile - 1) / kTile);
  return static_cast<int>(std::max<long long>(1, std::min<long long>(units, static_cast<long long>(num_sms(device)) * kCtasPerSm)));
}

template <int D>
void launch(const Params& p, int grid, cudaStream_t stream, int device) {
  static std::once_flag once[64];  // a property of the kernel on that device, set once
  std::call_once(once[device & 63], [] {
    TT_CUDA_CHECK(cudaFuncSetAttribute(paged_decode_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem_bytes<D>())));
  });
  paged_decode_kernel<D><<<grid, kThreads, smem_bytes<D>(), stream>>>(p);
}

}  // namespace paged

// fp32 elements of the partials and int32 counters that paged_attention needs for this shape.
std::vector<int64_t> paged_attention_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_keys, int64_t device) {
  TT_CHECK(B >= 0 && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 && D >= 1 && max_keys >= 0, "paged_attention_workspace: sizes");
  const int64_t grid = paged::grid_size(B, Hkv, max_keys, static_cast<int>(device));
  return {2 * grid * (Hq / Hkv) * (D + 2), B * Hkv};
}

// q [B, Hq, D] (any 8-element-aligned strides), pools [pages, page_size, Hkv, D], page_table int32
// [B, width], seq_lens int32 [B] (keys each query attends to, 0: output 0) -> out [B, Hq, D].
// part / counters: workspace of the sizes above; counters are zero before the first call and left zero.
void paged_attention(torch::Tensor q, torch::Tensor k_pages, torch::Tensor v_pages, torch::Tensor page_table,
                     torch::Tensor seq_lens, double scale, torch::Tensor part, torch::Tensor counters, torch::Tensor out) {
  using namespace paged;
  check_cuda_bf16(q, "q");
  check_cuda_bf16(k_pages, "k_pages");
  check_cuda_bf16(v_pages, "v_pages");
  check_cuda_bf16(out, "out");
  TT_CHECK(q.dim() == 3, "paged_attention: q must be [B, Hq, D]");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  TT_CHECK(D == 64 || D == 128, "paged_attention: head_dim must be 64 or 128");
  TT_CHECK(q.stride(2) == 1 && q.stride(0) % 2 == 0 && q.stride(1) % 2 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 4 == 0,
           "paged_attention: q rows must be contiguous and 4-byte aligned");
  TT_CHECK(k_pages.dim() == 4 && k_pages.size(3) == D && v_pages.sizes() == k_pages.sizes() && k_pages.is_contiguous() &&
               v_pages.is_contiguous() && reinterpret_cast<uintptr_t>(k_pages.data_ptr()) % 16 == 0 &&
               reinterpret_cast<uintptr_t>(v_pages.data_ptr()) % 16 == 0,
           "paged_attention: pages must be contiguous 16-byte aligned [pages, page_size, Hkv, D]");
  const int64_t Hkv = k_pages.size(2);
  TT_CHECK(Hkv >= 1 && Hq % Hkv == 0 && Hq / Hkv <= kMaxG && Hq >= Hkv, "paged_attention: Hq / Hkv must be an integer in [1, 16]");
  TT_CHECK(page_table.scalar_type() == torch::kInt32 && page_table.dim() == 2 && page_table.size(0) == B && page_table.is_contiguous(),
           "paged_attention: page_table must be contiguous int32 [B, width]");
  TT_CHECK(seq_lens.scalar_type() == torch::kInt32 && seq_lens.numel() == B && seq_lens.is_contiguous(),
           "paged_attention: seq_lens must be contiguous int32 [B]");
  TT_CHECK(out.is_contiguous() && out.numel() == B * Hq * D && reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
           "paged_attention: out must be a contiguous [B, Hq, D]");
  TT_CHECK(k_pages.size(1) >= 1 && k_pages.size(0) * k_pages.size(1) < (1LL << 31), "paged_attention: at most 2^31 - 1 tokens in a pool");
  TT_CHECK(B * Hkv < (1LL << 31) && page_table.size(1) < (1LL << 31), "paged_attention: sizes");
  if (B == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  const int device = q.get_device();
  Params p{};
  p.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  p.q_ld_b = q.stride(0);
  p.q_ld_h = q.stride(1);
  p.k_pages = reinterpret_cast<const __nv_bfloat16*>(k_pages.data_ptr());
  p.v_pages = reinterpret_cast<const __nv_bfloat16*>(v_pages.data_ptr());
  p.table = page_table.data_ptr<int>();
  p.lens = seq_lens.data_ptr<int>();
  p.B = static_cast<int>(B);
  p.Hq = static_cast<int>(Hq);
  p.Hkv = static_cast<int>(Hkv);
  p.G = static_cast<int>(Hq / Hkv);
  p.width = static_cast<int>(page_table.size(1));
  p.page_size = static_cast<int>(k_pages.size(1));
  p.num_pages = static_cast<int>(k_pages.size(0));
  p.scale_log2 = static_cast<float>(scale) * kLog2e;
  const int grid = grid_size(B, Hkv, static_cast<int64_t>(p.width) * p.page_size, device);
  const int64_t n_o = 2LL * grid * p.G * D;
  TT_CHECK(part.scalar_type() == torch::kFloat32 && part.is_contiguous() && part.numel() >= n_o + 4LL * grid * p.G &&
               reinterpret_cast<uintptr_t>(part.data_ptr()) % 16 == 0,
           "paged_attention: workspace for partials too small");
  TT_CHECK(counters.scalar_type() == torch::kInt32 && counters.is_contiguous() && counters.numel() >= B * Hkv,
           "paged_attention: workspace for counters too small");
  p.part_o = part.data_ptr<float>();
  p.part_ml = p.part_o + n_o;
  p.counters = counters.data_ptr<int>();
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.status = device_status_ptr(device);
  if (D == 128) launch<128>(p, grid, cur_stream(), device);
  else launch<64>(p, grid, cur_stream(), device);
  TT_CUDA_CHECK(cudaGetLastError());
}

}  // namespace tt

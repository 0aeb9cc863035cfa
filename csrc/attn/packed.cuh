// Shared by the kernels of packed (variable-length) attention: how a call's work is listed, and
// the tensor maps of [tokens, heads, D] operands.
//
// Sequences lie one after the other in the token dimension, sequence b at rows
// [cu_q[b], cu_q[b + 1]) of the queries and [cu_k[b], cu_k[b + 1]) of the keys; query i of a
// sequence sees its keys j <= i + (len_k - len_q).  The offsets stay on the device.  A schedule
// kernel turns them into a list of (sequence, tile) entries, the longest first, so that the
// block scheduler hands out the tiles of long sequences before the short ones fill the gaps; the
// host only knows an upper bound of the number of entries: ceil(len / t) summed over B sequences is
// at most floor(N / t) + B.  Rows after the last sequence form one more entry group (sequence B,
// no keys): they get zeros.
#pragma once
#include "common/host_utils.h"
#include "common/ptx.cuh"

namespace tt {
namespace packed {

constexpr int kBlock = 128;  // rows of a query or key tile

// Sequence b of the packing, b == B: the rows after the last one.
struct Seq {
  int q0, qlen, k0, klen;
  int off;       // klen - qlen: query i sees keys up to i + off
  int pad_row0;  // its first row in the tile-aligned per-row arrays (128-row slots)
};

struct Packing {
  const int* cu_q;
  const int* cu_k;
  int B, Nq, Nk;
};

__device__ __forceinline__ Seq sequence(const Packing& p, int b) {
  Seq s;
  s.q0 = p.cu_q[b];
  s.qlen = (b < p.B ? p.cu_q[b + 1] : p.Nq) - s.q0;
  s.k0 = p.cu_k[b];
  s.klen = (b < p.B ? p.cu_k[b + 1] : p.Nk) - s.k0;
  if (b == p.B) {  // rows of no sequence: queries see nothing, keys are seen by nobody
    s.off = -s.qlen;
  } else {
    s.off = s.klen - s.qlen;
  }
  s.pad_row0 = (s.q0 / kBlock + b) * kBlock;
  return s;
}

// Query tiles of `rows` rows / key tiles of 128 rows of a packing, at most.
inline int64_t max_tiles(int64_t n, int64_t B, int64_t rows) { return n / rows + B + 1; }
// 128-row slots of the tile-aligned per-query-row arrays (softmax statistics of the backward).
inline int64_t pad_slots(int64_t Nq, int64_t B) { return Nq / kBlock + B + 1; }

// Number of 128-key tiles that queries [i0, i0 + rows) of the sequence see.
__device__ __forceinline__ int key_tiles(const Seq& s, bool extra, int i0, int rows) {
  if (extra || i0 >= s.qlen) return 0;
  const int last = min(i0 + rows, s.qlen) - 1 + s.off;  // last key the last query sees
  return last < 0 ? 0 : min(last, s.klen - 1) / kBlock + 1;
}
// First 128-query tile that sees key tile j, and the number of tiles from there on.
__device__ __forceinline__ int first_query_tile(const Seq& s, int kt) { return max(0, kt * kBlock - s.off) / kBlock; }
__device__ __forceinline__ int query_tiles(const Seq& s, bool extra, int kt) {
  if (extra) return 0;
  return max(0, (s.qlen + kBlock - 1) / kBlock - first_query_tile(s, kt));
}

// Sequence of a list entry past the end of the list, and of every entry where the offsets are unusable.
constexpr int kNoEntry = -1, kRejected = -2;

// This block's share of zeros for a [tokens, heads, D] tensor with strides (elements): the output of a call whose
// offsets are unusable.
template <int D>
__device__ __forceinline__ void zero_share(__nv_bfloat16* t, long long tokens, int heads, long long ld_n, long long ld_h) {
  constexpr int NU = D / 8;
  const long long all = tokens * heads * NU, step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < all; i += step) {
    const long long row = i / NU;
    reinterpret_cast<uint4*>(t + row / heads * ld_n + row % heads * ld_h)[i % NU] = make_uint4(0u, 0u, 0u, 0u);
  }
}

// Zeroes rows [from, 128) of a swizzled tile of D / 64 chunks (whole 128-byte rows, so the swizzle
// does not matter), by `threads` threads of index t.
template <int D>
__device__ __forceinline__ void clear_rows(uint8_t* tile, int from, int t, int threads) {
  const int per_chunk = (kBlock - from) * 8;
  for (int c = 0; c < D / 64; ++c)
    for (int i = t; i < per_chunk; i += threads)
      *reinterpret_cast<uint4*>(tile + c * kBlock * 128 + from * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
}

// ----------------------------------------------------------------- products
// A product's descriptors live in uniform registers.  Issued by one lane of a diverged warp they are put together
// there anew for every instruction (measured: about 130 cycles an instruction that the tensor core does in 64); so
// the whole warp walks the issue loop, addresses are warp-uniform sums of precomputed low words, and only the
// elected lane runs the instructions themselves.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}
// Descriptor words (see sdesc_sw128): 8-row groups 1024 bytes apart, 128-byte swizzle.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k_major(const void* tile) { return (smem_u32(tile) >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn_major(const void* tile) {  // 64-element chunks 128 rows of 128 bytes apart
  return (smem_u32(tile) >> 4) | (((kBlock * 128u) >> 4) << 16);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(kDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// d [128 x 128] = A B^T over D, both tiles [128 rows x D] K-major; `done` follows it.
template <int D>
__device__ __forceinline__ void product_abt(bool lead, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint64_t* done) {
  constexpr uint32_t kIdesc = idesc_bf16_f32(kBlock, kBlock, false, false);
  if (lead) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const uint32_t off = ((kk >> 2) * (kBlock * 128) + (kk & 3) * 32) >> 4;
      mma_ss(d, a_lo + off, b_lo + off, kIdesc, kk > 0 ? 1u : 0u);
    }
    umma_commit(done);
  }
  __syncwarp();
}
// d [128 x D] (+)= A B: A [128 x 128] as bf16 pairs in TMEM, `kGroup` of its columns in each `kGroup` 32-bit columns (the
// first half of them), B [128 rows x D] in shared memory.
template <int D, int kGroup>
__device__ __forceinline__ void product_ab(bool lead, uint32_t d, uint32_t a_tmem, uint32_t b_lo, bool accumulate) {
  constexpr uint32_t kIdesc = idesc_bf16_f32(kBlock, D, false, true);
  const uint32_t first = accumulate ? 1u : 0u;
  if (lead) {
#pragma unroll
    for (int kk = 0; kk < kBlock / 16; ++kk)
      mma_ts(d, a_tmem + kk * 16 / kGroup * kGroup + (kk * 16 % kGroup) / 2, b_lo + kk * (2048 >> 4), kIdesc, kk > 0 ? 1u : first);
  }
  __syncwarp();
}
__device__ __forceinline__ void commit(bool lead, uint64_t* bar) {
  if (lead) umma_commit(bar);
  __syncwarp();
}

// 3-D tensor map of bf16 [tokens, heads, D] (strides in elements), box {64, 1, rows}, 128-byte swizzle.
inline CUtensorMap head_map_3d(const torch::Tensor& t, int rows, const char* name) {
  const std::string n(name);
  const int64_t N = t.size(0), H = t.size(1), D = t.size(2);
  const int64_t sn = N > 1 ? t.stride(0) : H * D, sh = H > 1 ? t.stride(1) : D;
  TT_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, n + " must be 16-byte aligned");
  CUtensorMap m;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(N)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(sn) * 2};
  cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(rows)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode_tiled_fn()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, t.data_ptr(), dims, strides, box, estr,
                                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                       CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TT_CHECK(r == CUDA_SUCCESS, n + ": cuTensorMapEncodeTiled failed (code " + std::to_string((int)r) + ")");
  return m;
}

// bf16 [N, H, D] with contiguous rows, strides multiples of 8 elements, 16-byte aligned.
inline void check_heads(const torch::Tensor& t, int64_t H, int64_t D, const char* name) {
  const std::string n(name);
  check_cuda_bf16(t, name);
  TT_CHECK(t.dim() == 3 && t.size(2) == D && (H < 0 || t.size(1) == H), n + " must be [tokens, heads, D]");
  TT_CHECK(t.stride(2) == 1 && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) > 0)) &&
               (t.size(1) <= 1 || (t.stride(1) % 8 == 0 && t.stride(1) > 0)) &&
               reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
           n + " must have contiguous head rows, 16-byte aligned positive strides");
  TT_CHECK(t.size(0) < (1LL << 30) && t.size(1) < 65536, n + " is too large");
}

inline void check_offsets(const torch::Tensor& cu, int64_t B1, const char* name) {
  TT_CHECK(cu.scalar_type() == torch::kInt32 && cu.dim() == 1 && cu.is_contiguous() && cu.numel() >= 1 &&
               (B1 < 0 || cu.numel() == B1),
           std::string(name) + " must be contiguous int32 [B + 1]");
}

inline Packing packing_of(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& cu_q, const torch::Tensor& cu_k) {
  Packing p;
  p.cu_q = cu_q.data_ptr<int>();
  p.cu_k = cu_k.data_ptr<int>();
  p.B = static_cast<int>(cu_q.numel() - 1);
  p.Nq = static_cast<int>(q.size(0));
  p.Nk = static_cast<int>(k.size(0));
  return p;
}

// Allows a kernel `smem` bytes of shared memory, once per device (its size is the kernel's own constant).
template <auto kKernel>
inline void allow_smem(size_t smem, int device) {
  static std::once_flag once[64];
  std::call_once(once[device & 63], [&] {
    TT_CUDA_CHECK(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  });
}

enum ScheduleKind { kQueryPairs = 0, kQueryTiles = 1, kKeyTiles = 2 };

// List (int2 {sequence, tile}, longest first, {kNoEntry, 0} past the end) of a packing's query tile pairs, query
// tiles or key tiles; `capacity` entries.  Offsets that do not ascend from 0 within the tokens: kBadIndex in the status
// word, all entries {kRejected, 0}, and the kernels that read the list write zeros.
void schedule(const Packing& p, ScheduleKind kind, int2* list, int capacity, int* status, cudaStream_t stream);

}  // namespace packed
}  // namespace tt

// Pages of a KV cache whose sequences have lengths of their own: writing new tokens into them,
// forking sequences and compacting the pool.
//
// A pool is [layers, pages, page_size, Hkv, D] bf16 (keys and values apart); a page table row
// [width] int32 lists a sequence's pages in order (-1 past its end).  One table serves all
// layers, so fork and move touch it once and the data of every layer in the same launch.
// All three are bound by the bytes they move: 16-byte vectors, several in flight per thread.
//
// Index inputs live on the device and are checked where they are used: an entry out of range is
// skipped and recorded as kBadIndex in the status word; a token at a position past the tables comes back as zeros.
//
// Measured (L2 flushed): appending 16384 tokens of 16/4 heads, d 128 (218 MB): 47 us, 4.6 TB/s; moving 16 KB
// pages of 16 layers (772 MB): 124 us, 6.2 TB/s; forking 8 prompts into 8 answers each over 16 layers
// (537 MB counted, 302 MB of them distinct): 53 us.
#include "common/host_utils.h"
#include "common/ptx.cuh"

namespace tt {
namespace pages {

constexpr int kThreads = 256;

// ----------------------------------------------------------------- rotate and append
struct AppendArgs {
  const __nv_bfloat16* qkv;
  int ld;
  const float* cos_t;
  const float* sin_t;
  int max_pos;
  const int* cu;      // [B + 1]
  const int* start;   // [B] position of each sequence's first token (null: 0)
  int N, B, Hq, Hkv, D;
  float sign;         // -1: inverse rotation
  __nv_bfloat16* q_out;   // [N, Hq, D], row stride ld_q
  __nv_bfloat16* k_out;   // [N, Hkv, D], row stride ld_k (may be null)
  int ld_q, ld_k;
  __nv_bfloat16* k_pages; // [pages, page_size, Hkv, D] (may be null)
  __nv_bfloat16* v_pages;
  const int* table;
  int width, page_size, num_pages;
  int* status;
};

// Largest b with cu[b] <= i, by a warp: 32 probes at a time narrow [lo, hi).
__device__ __forceinline__ int find_sequence(const int* cu, int B, int i, int lane) {
  int lo = 0, n = B;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int b = lo + lane * step;
    const bool le = lane * step < n && cu[b] <= i;
    const unsigned mask = __ballot_sync(0xffffffffu, le);
    const int last = mask ? 31 - __clz(mask) : 0;
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

// One warp per token: its sequence and position once, then 8 pairs (j, j + D/2) of one head per
// lane and step.  x' = x cos - y sin, y' = y cos + x sin, computed in fp32, rounded once.
__global__ void __launch_bounds__(kThreads) rotary_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int tok = static_cast<int>((static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> 5);
  if (tok >= a.N) return;
  const int b = find_sequence(a.cu, a.B, tok, lane);
  const int c0 = a.cu[b];
  const bool inside = tok >= c0 && tok < a.cu[b + 1];
  const int pos = inside ? (a.start != nullptr ? a.start[b] : 0) + tok - c0 : 0;
  const bool bad = pos < 0 || pos >= a.max_pos;
  if (bad && lane == 0) atomicCAS(a.status, 0, static_cast<int>(kBadIndex));
  if (!inside || bad) {  // a token of no sequence, or past the tables: nothing is cached, zeros come back
    for (int i = lane; i < a.Hq * a.D / 8; i += 32)
      reinterpret_cast<uint4*>(a.q_out + static_cast<long long>(tok) * a.ld_q)[i] = make_uint4(0u, 0u, 0u, 0u);
    if (a.k_out != nullptr)
      for (int i = lane; i < a.Hkv * a.D / 8; i += 32)
        reinterpret_cast<uint4*>(a.k_out + static_cast<long long>(tok) * a.ld_k)[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  long long slot = -1;  // the token's row of heads in a page
  if (a.k_pages != nullptr) {
    const int pi = pos / a.page_size;
    const int page = pi < a.width ? a.table[static_cast<long long>(b) * a.width + pi] : -1;
    if (page >= 0 && page < a.num_pages) slot = (static_cast<long long>(page) * a.page_size + pos % a.page_size) * a.Hkv;
    else if (lane == 0) atomicCAS(a.status, 0, static_cast<int>(kBadIndex));
  }
  const int groups = a.D / 16, half = a.D / 2;
  const __nv_bfloat16* src = a.qkv + static_cast<long long>(tok) * a.ld;
  const int rot = (a.Hq + a.Hkv) * groups;
  const float* cr = a.cos_t + static_cast<long long>(pos) * half;
  const float* sr = a.sin_t + static_cast<long long>(pos) * half;
  // A lane keeps its piece of the head where the pieces of a head divide the warp (D = 16 to 256 in powers of two):
  // the angles are then loaded once.
  const bool same_piece = 32 % groups == 0;
  float cs[8], sn[8];
  auto angles = [&](int d0) {
    const float4 ca = *reinterpret_cast<const float4*>(cr + d0), cb = *reinterpret_cast<const float4*>(cr + d0 + 4);
    const float4 sa = *reinterpret_cast<const float4*>(sr + d0), sb = *reinterpret_cast<const float4*>(sr + d0 + 4);
    cs[0] = ca.x, cs[1] = ca.y, cs[2] = ca.z, cs[3] = ca.w, cs[4] = cb.x, cs[5] = cb.y, cs[6] = cb.z, cs[7] = cb.w;
    sn[0] = sa.x, sn[1] = sa.y, sn[2] = sa.z, sn[3] = sa.w, sn[4] = sb.x, sn[5] = sb.y, sn[6] = sb.z, sn[7] = sb.w;
  };
  if (same_piece) angles(8 * (lane % groups));
#pragma unroll 2
  for (int i = lane; i < rot; i += 32) {  // a lane reads both halves of a piece before it writes them (the output may be the input)
    const int h = i / groups, d0 = 8 * (i - h * groups);
    const uint4 lo4 = *reinterpret_cast<const uint4*>(src + h * a.D + d0);
    const uint4 hi4 = *reinterpret_cast<const uint4*>(src + h * a.D + half + d0);
    if (!same_piece) angles(d0);
    const uint32_t* lw = reinterpret_cast<const uint32_t*>(&lo4);
    const uint32_t* hw = reinterpret_cast<const uint32_t*>(&hi4);
    uint4 olo, ohi;
    uint32_t* ol = reinterpret_cast<uint32_t*>(&olo);
    uint32_t* oh = reinterpret_cast<uint32_t*>(&ohi);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = unpack_bf16x2(lw[j]), y = unpack_bf16x2(hw[j]);
      const float s0 = a.sign * sn[2 * j], s1 = a.sign * sn[2 * j + 1];
      ol[j] = pack_bf16x2(x.x * cs[2 * j] - y.x * s0, x.y * cs[2 * j + 1] - y.y * s1);
      oh[j] = pack_bf16x2(y.x * cs[2 * j] + x.x * s0, y.y * cs[2 * j + 1] + x.y * s1);
    }
    if (h < a.Hq) {
      __nv_bfloat16* dst = a.q_out + static_cast<long long>(tok) * a.ld_q + h * a.D + d0;
      *reinterpret_cast<uint4*>(dst) = olo;
      *reinterpret_cast<uint4*>(dst + half) = ohi;
    } else {
      const int kh = h - a.Hq;
      if (a.k_out != nullptr) {
        __nv_bfloat16* dst = a.k_out + static_cast<long long>(tok) * a.ld_k + kh * a.D + d0;
        *reinterpret_cast<uint4*>(dst) = olo;
        *reinterpret_cast<uint4*>(dst + half) = ohi;
      }
      if (slot >= 0) {
        __nv_bfloat16* dst = a.k_pages + (slot + kh) * a.D + d0;
        *reinterpret_cast<uint4*>(dst) = olo;
        *reinterpret_cast<uint4*>(dst + half) = ohi;
      }
    }
  }
  if (slot >= 0) {
    const uint4* v = reinterpret_cast<const uint4*>(src + (a.Hq + a.Hkv) * a.D);
    uint4* dst = reinterpret_cast<uint4*>(a.v_pages + slot * a.D);
    for (int i = lane; i < a.Hkv * a.D / 8; i += 32) dst[i] = v[i];
  }
}

// ----------------------------------------------------------------- fork and move
struct CopyArgs {
  uint4* k;  // [layers, pages, page_vecs]
  uint4* v;
  int layers, num_pages;
  int page_vecs;       // 16-byte vectors of a page
  int chunk;           // vectors a block copies
  int chunks;          // blocks a (page, layer, k or v)
  int n;               // copies
  // fork: parents / children / fresh [n]; move: src / dst [n]
  const int* a0;
  const int* a1;
  const int* a2;
  int* table;          // [rows, width]
  int* lens;           // [rows]
  int rows, width, page_size;
  long long data_blocks;  // blocks that copy data come first, then those of the table
  int* status;
};

constexpr int kInFlight = 8;  // 16-byte loads a thread keeps in flight

// kOnce: the source is read by this copy alone (a fork's source by every child of a parent).
template <bool kOnce>
__device__ __forceinline__ void copy_vecs(uint4* dst, const uint4* src, int n) {
  for (int i = threadIdx.x; i < n; i += kInFlight * kThreads) {
    uint4 r[kInFlight];
#pragma unroll
    for (int j = 0; j < kInFlight; ++j)
      if (i + j * kThreads < n) r[j] = kOnce ? __ldcs(src + i + j * kThreads) : src[i + j * kThreads];
#pragma unroll
    for (int j = 0; j < kInFlight; ++j)
      if (i + j * kThreads < n) {
        if (kOnce) __stcs(dst + i + j * kThreads, r[j]);
        else dst[i + j * kThreads] = r[j];
      }
  }
}

__device__ __forceinline__ void bad_index(int* status) {
  if (threadIdx.x == 0) atomicCAS(status, 0, static_cast<int>(kBadIndex));
}

// Data block `blk`: copy number, layer, k or v, piece of the page.
template <bool kOnce>
__device__ __forceinline__ void copy_page_piece(const CopyArgs& a, long long blk, int src, int dst) {
  const int piece = static_cast<int>(blk % a.chunks);
  const long long rest = blk / a.chunks;
  const int which = static_cast<int>(rest % 2);
  const int layer = static_cast<int>((rest / 2) % a.layers);
  uint4* pool = which ? a.v : a.k;
  const long long base = static_cast<long long>(layer) * a.num_pages;
  const int off = piece * a.chunk;
  copy_vecs<kOnce>(pool + (base + dst) * a.page_vecs + off, pool + (base + src) * a.page_vecs + off, min(a.chunk, a.page_vecs - off));
}

// Child c_i takes the row and length of parent p_i; where fresh f_i >= 0, the parent's page that
// its next token falls into (the partly filled one) is copied to f_i and replaced by it in the child's row.
// The blocks of an entry's data and the one of its row make the same test: an entry is done whole or not at all.
__global__ void __launch_bounds__(kThreads) fork_kernel(const CopyArgs a) {
  const long long blk = blockIdx.x;
  const bool data = blk < a.data_blocks;
  const int i = data ? static_cast<int>(blk / (static_cast<long long>(a.chunks) * 2 * a.layers)) : static_cast<int>(blk - a.data_blocks);
  const int parent = a.a0[i], child = a.a1[i], fresh = a.a2[i];
  if (parent < 0 || parent >= a.rows || child < 0 || child >= a.rows || parent == child || fresh >= a.num_pages) {
    bad_index(a.status);
    return;
  }
  const int len = a.lens[parent];
  const int last = len / a.page_size;
  int src = -1;  // the page that is copied
  if (len >= 0 && fresh >= 0 && last < a.width) src = a.table[static_cast<long long>(parent) * a.width + last];
  if (len < 0 || (fresh >= 0 && (src < 0 || src >= a.num_pages || src == fresh))) {
    bad_index(a.status);
    return;
  }
  if (data) {
    if (fresh >= 0) copy_page_piece<false>(a, blk, src, fresh);
    return;
  }
  const int* from = a.table + static_cast<long long>(parent) * a.width;
  int* to = a.table + static_cast<long long>(child) * a.width;
  for (int j = threadIdx.x; j < a.width; j += kThreads) to[j] = (fresh >= 0 && j == last) ? fresh : from[j];
  if (threadIdx.x == 0) a.lens[child] = len;
}

// Entry i of a move is taken where bisection for src_i over the sources ends at i.  The table's blocks look their pages
// up by that bisection, so data and table agree on every entry, in order or not; and of two neighbours that do not
// ascend one at least fails (the search for the second passes the first).  The probes on the way to a known index need
// no waiting for each other: lane s checks the one of step s.
__device__ __forceinline__ bool found_at(const int* sorted, int n, int i, int key) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
  for (int s = 0; s < lane && lo < hi; ++s) {
    const int mid = (lo + hi) >> 1;
    if (mid < i) lo = mid + 1;
    else hi = mid;
  }
  const int mid = (lo + hi) >> 1;
  return __all_sync(0xffffffffu, lo >= hi || (sorted[mid] < key) == (mid < i));
}
__device__ __forceinline__ bool movable(int src, int dst, int num_pages) {
  return src >= 0 && src < num_pages && dst >= 0 && dst < num_pages && src != dst;
}

// Page src_i becomes dst_i (src ascending, dst a free page): data of every layer, and every
// table entry that named it.  No dst is a src, so the copies are independent of one another.
__global__ void __launch_bounds__(kThreads) move_kernel(const CopyArgs a) {
  const long long blk = blockIdx.x;
  if (blk < a.data_blocks) {
    const int i = static_cast<int>(blk / (static_cast<long long>(a.chunks) * 2 * a.layers));
    const int src = a.a0[i], dst = a.a1[i];
    if (!found_at(a.a0, a.n, i, src) || !movable(src, dst, a.num_pages)) {
      bad_index(a.status);
      return;
    }
    copy_page_piece<true>(a, blk, src, dst);
    return;
  }
  const long long e = (blk - a.data_blocks) * kThreads + threadIdx.x;
  if (e >= static_cast<long long>(a.rows) * a.width) return;
  const int page = a.table[e];
  if (page < 0) return;
  int lo = 0, hi = a.n;  // first source >= page
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.a0[mid] < page) lo = mid + 1;
    else hi = mid;
  }
  if (lo < a.n && a.a0[lo] == page) {
    const int dst = a.a1[lo];
    if (movable(page, dst, a.num_pages)) a.table[e] = dst;
  }
}

void check_i32(const torch::Tensor& t, int64_t numel, const char* what) {
  TT_CHECK(t.scalar_type() == torch::kInt32 && t.is_contiguous() && t.is_cuda() && (numel < 0 || t.numel() == numel),
           std::string(what) + " must be a contiguous CUDA int32 tensor of the right size");
}

// The pools [layers, pages, page_size, Hkv, D] (or one layer's [pages, page_size, Hkv, D]).
CopyArgs pool_args(const torch::Tensor& k_pages, const torch::Tensor& v_pages, const torch::Tensor& table, const char* op) {
  const std::string name(op);
  check_cuda_bf16(k_pages, "k_pages");
  check_cuda_bf16(v_pages, "v_pages");
  TT_CHECK((k_pages.dim() == 4 || k_pages.dim() == 5) && k_pages.is_contiguous() && v_pages.is_contiguous() &&
               v_pages.sizes() == k_pages.sizes(),
           name + ": pools must be contiguous [layers, pages, page_size, Hkv, D] (or without layers)");
  TT_CHECK(reinterpret_cast<uintptr_t>(k_pages.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(v_pages.data_ptr()) % 16 == 0,
           name + ": pools must be 16-byte aligned");
  check_i32(table, -1, "page_table");
  TT_CHECK(table.dim() == 2, name + ": page_table must be [rows, width]");
  const int64_t off = k_pages.dim() - 4;
  const int64_t page_elems = k_pages.size(off + 1) * k_pages.size(off + 2) * k_pages.size(off + 3);
  TT_CHECK(page_elems % 8 == 0, name + ": a page must be a multiple of 16 bytes");
  TT_CHECK(page_elems / 8 < (1LL << 31) && k_pages.size(off) < (1LL << 31) && table.size(0) < (1LL << 31) && table.size(1) < (1LL << 31),
           name + ": sizes");
  CopyArgs a{};
  a.k = reinterpret_cast<uint4*>(k_pages.data_ptr());
  a.v = reinterpret_cast<uint4*>(v_pages.data_ptr());
  a.layers = static_cast<int>(off ? k_pages.size(0) : 1);
  a.num_pages = static_cast<int>(k_pages.size(off));
  a.page_size = static_cast<int>(k_pages.size(off + 1));
  a.page_vecs = static_cast<int>(page_elems / 8);
  // 32 KB a block: enough loads in flight per thread, and enough blocks for a few short pages
  a.chunk = kThreads * kInFlight;
  a.chunks = (a.page_vecs + a.chunk - 1) / a.chunk;
  a.table = table.data_ptr<int>();
  a.rows = static_cast<int>(table.size(0));
  a.width = static_cast<int>(table.size(1));
  a.status = device_status_ptr(k_pages.get_device());
  return a;
}

}  // namespace pages

// Packed tokens qkv [N, >= (Hq + 2 Hkv) D] (q | k | v heads), sequence b at rows [cu[b], cu[b + 1]),
// its first token at position start[b] (0 without start).  q_out [N, Hq, D] (and k_out [N, Hkv, D])
// rotated; with pages, rotated k and v go to (table[b][pos / page_size], pos % page_size).
void rotary_append(torch::Tensor qkv, torch::Tensor cos_t, torch::Tensor sin_t, int64_t Hq, int64_t Hkv, int64_t D,
                   torch::Tensor cu, c10::optional<torch::Tensor> start, bool inverse, torch::Tensor q_out,
                   c10::optional<torch::Tensor> k_out, c10::optional<torch::Tensor> k_pages,
                   c10::optional<torch::Tensor> v_pages, c10::optional<torch::Tensor> page_table) {
  using namespace pages;
  check_cuda_bf16(qkv, "qkv");
  TT_CHECK(Hq >= 1 && Hkv >= 1 && D >= 16 && D % 16 == 0 && D <= 256, "rotary_append: head_dim must be a multiple of 16 up to 256");
  TT_CHECK(qkv.dim() == 2 && qkv.stride(1) == 1 && qkv.size(1) >= (Hq + 2 * Hkv) * D && qkv.stride(0) % 8 == 0 &&
               reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0 && qkv.stride(0) < (1LL << 31) && qkv.size(0) < (1LL << 31),
           "rotary_append: qkv must be [N, >=(Hq+2Hkv)*D] with 16-byte aligned rows");
  TT_CHECK(cos_t.scalar_type() == torch::kFloat32 && cos_t.dim() == 2 && cos_t.size(1) == D / 2 && cos_t.is_contiguous() &&
               sin_t.scalar_type() == torch::kFloat32 && sin_t.sizes() == cos_t.sizes() && sin_t.is_contiguous() &&
               reinterpret_cast<uintptr_t>(cos_t.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(sin_t.data_ptr()) % 16 == 0,
           "rotary_append: cos/sin must be contiguous fp32 [max_pos, D/2]");
  check_i32(cu, -1, "rotary_append: cu_seqlens");
  TT_CHECK(cu.numel() >= 1, "rotary_append: cu_seqlens must be [B + 1]");
  const int64_t N = qkv.size(0), B = cu.numel() - 1;
  auto rows_ok = [&](const torch::Tensor& t, int64_t heads) {
    return t.scalar_type() == torch::kBFloat16 && t.dim() == 3 && t.size(0) == N && t.size(1) == heads && t.size(2) == D &&
           t.stride(2) == 1 && (heads == 1 || t.stride(1) == D) && t.stride(0) % 8 == 0 && t.stride(0) < (1LL << 31) &&
           reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  TT_CHECK(rows_ok(q_out, Hq), "rotary_append: q_out must be bf16 [N, Hq, D], heads adjacent");
  AppendArgs a{};
  a.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  a.ld = static_cast<int>(qkv.stride(0));
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.max_pos = static_cast<int>(cos_t.size(0));
  a.cu = cu.data_ptr<int>();
  if (start.has_value()) {
    check_i32(*start, B, "rotary_append: start");
    a.start = start->data_ptr<int>();
  }
  a.N = static_cast<int>(N);
  a.B = static_cast<int>(B);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.D = static_cast<int>(D);
  a.sign = inverse ? -1.0f : 1.0f;
  a.q_out = reinterpret_cast<__nv_bfloat16*>(q_out.data_ptr());
  a.ld_q = static_cast<int>(q_out.stride(0));
  if (k_out.has_value()) {
    TT_CHECK(rows_ok(*k_out, Hkv), "rotary_append: k_out must be bf16 [N, Hkv, D], heads adjacent");
    a.k_out = reinterpret_cast<__nv_bfloat16*>(k_out->data_ptr());
    a.ld_k = static_cast<int>(k_out->stride(0));
  }
  TT_CHECK(k_pages.has_value() == v_pages.has_value() && k_pages.has_value() == page_table.has_value(),
           "rotary_append: k_pages, v_pages and page_table go together");
  if (k_pages.has_value()) {
    TT_CHECK(k_pages->dim() == 4 && k_pages->size(2) == Hkv && k_pages->size(3) == D, "rotary_append: pages must be [pages, page_size, Hkv, D]");
    const CopyArgs c = pool_args(*k_pages, *v_pages, *page_table, "rotary_append");
    TT_CHECK(page_table->size(0) >= B, "rotary_append: page_table must have a row per sequence");
    a.k_pages = reinterpret_cast<__nv_bfloat16*>(k_pages->data_ptr());
    a.v_pages = reinterpret_cast<__nv_bfloat16*>(v_pages->data_ptr());
    a.table = c.table;
    a.width = c.width;
    a.page_size = c.page_size;
    a.num_pages = c.num_pages;
    TT_CHECK(a.page_size >= 1, "rotary_append: empty pages");
  }
  if (N == 0 || B == 0) {
    if (N > 0) {
      q_out.zero_();
      if (k_out.has_value()) k_out->zero_();
    }
    return;
  }
  const c10::cuda::CUDAGuard guard(qkv.device());
  a.status = device_status_ptr(qkv.get_device());
  const long long blocks = (N * 32 + kThreads - 1) / kThreads;
  rotary_append_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, cur_stream()>>>(a);
  TT_CUDA_CHECK(cudaGetLastError());
}

// For each i: row and length of children[i] become those of parents[i]; fresh[i] >= 0 is a page of the
// child's own that receives the parent's partly filled page.  Children, parents and fresh pages are
// distinct (no child is a parent, no page is given twice): the copies run in no order.
void fork_pages(torch::Tensor k_pages, torch::Tensor v_pages, torch::Tensor page_table, torch::Tensor seq_lens,
                torch::Tensor parents, torch::Tensor children, torch::Tensor fresh) {
  using namespace pages;
  CopyArgs a = pool_args(k_pages, v_pages, page_table, "fork_pages");
  check_i32(seq_lens, a.rows, "fork_pages: seq_lens");
  check_i32(parents, -1, "fork_pages: parents");
  const int64_t n = parents.numel();
  check_i32(children, n, "fork_pages: children");
  check_i32(fresh, n, "fork_pages: fresh");
  TT_CHECK(a.page_size >= 1, "fork_pages: empty pages");
  if (n == 0) return;
  const c10::cuda::CUDAGuard guard(k_pages.device());
  a.n = static_cast<int>(n);
  a.a0 = parents.data_ptr<int>();
  a.a1 = children.data_ptr<int>();
  a.a2 = fresh.data_ptr<int>();
  a.lens = seq_lens.data_ptr<int>();
  a.data_blocks = static_cast<long long>(n) * a.layers * 2 * a.chunks;
  TT_CHECK(a.data_blocks + n < (1LL << 31), "fork_pages: too many pages in one call");
  fork_kernel<<<static_cast<unsigned>(a.data_blocks + n), kThreads, 0, cur_stream()>>>(a);
  TT_CUDA_CHECK(cudaGetLastError());
}

// Moves page src[i] (ascending) to the free page dst[i] in every layer and rewrites the table's entries.
void move_pages(torch::Tensor k_pages, torch::Tensor v_pages, torch::Tensor page_table, torch::Tensor src,
                torch::Tensor dst) {
  using namespace pages;
  CopyArgs a = pool_args(k_pages, v_pages, page_table, "move_pages");
  check_i32(src, -1, "move_pages: src");
  const int64_t n = src.numel();
  check_i32(dst, n, "move_pages: dst");
  if (n == 0) return;
  const c10::cuda::CUDAGuard guard(k_pages.device());
  a.n = static_cast<int>(n);
  a.a0 = src.data_ptr<int>();
  a.a1 = dst.data_ptr<int>();
  a.data_blocks = static_cast<long long>(n) * a.layers * 2 * a.chunks;
  const long long table_blocks = (static_cast<long long>(a.rows) * a.width + kThreads - 1) / kThreads;
  TT_CHECK(a.data_blocks + table_blocks < (1LL << 31), "move_pages: too many pages in one call");
  move_kernel<<<static_cast<unsigned>(a.data_blocks + table_blocks), kThreads, 0, cur_stream()>>>(a);
  TT_CUDA_CHECK(cudaGetLastError());
}

}  // namespace tt

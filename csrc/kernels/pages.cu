// KV pages of sequences that share a prompt: fork, free, compact.
//
// The cache is any contiguous [L, NB, ...] tensor (bf16 pages, int8 pages, the wide-head layout): a page is one
// 16-token block, its bytes of one layer are contiguous, and every kernel here moves bytes.  ref[NB] counts the
// block-table rows that hold a page (0: free).
//
//   fork     row c of the new table takes the parent's pages; ref += 1 on each; a last page that is not full is
//            copied to fresh[c], because parent and child will write different tokens into it.  A child whose ids are
//            out of range or whose fresh page is held gets an empty row
//   free     ref -= 1 on a row's pages, and its length becomes 0 (a second free of the row is a no-op)
//   compact  U = pages held; the i-th held page at or above U moves to the i-th free page below U (the two sets are
//            disjoint and equally large, so all copies may run at once); tables and ref follow
//
// All three are bound by the bytes of the pages they copy (each read once and written once), and at small sizes by
// launches: fork and free are one launch, compact is two (a one-CTA plan over a bitmap of ref, then the copies).
// Copies run in chunks of 16 or 32 KB per CTA that end with the page, all loads of a chunk in flight before its first
// store.  With whole chunks an SM has 96 KB (fork: 6 CTAs, 40 registers a thread) or 128 KB (compact: 4 CTAs, 60
// registers) in flight, against a bandwidth-latency product of 88 KB (44 GB/s per SM x ~2 us).
// Measured: a pool of 18,000 pages compacts at 6.5 TB/s (read + write) after a plan of 8 to 11 us; a fork of 4 children
// over 16 layers and a reset of the counts take 5.1 us in a graph, of 128 children over 8 layers of int8 pages 12.0.
//
// An id outside its range sets kStatusBadArgument and its access is skipped, in every build.
//
// No counterpart in the reference, whose pages live on the host (scheduler/paged_cache.rs:565-748).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

#include "bloom/common.cuh"
#include "bloom/ops_share.h"
#include "bloom/tma_host.h"

namespace bloom {
namespace pages {

constexpr int kPage = 16;
constexpr int kThreads = 256;
// 16-byte loads in flight per thread.  Eight where the copies last (645 MB compacted in 99 us, 106 with four), four in
// a fork, whose CTAs hold them while they ask for their page (34 MB in 12.0 us, 14.5 with eight and four CTAs per SM).
constexpr int kForkVec = 4, kMoveVec = 8;
template <int kVec>
constexpr int kChunk = kThreads * kVec * 16;  // bytes of one copy step of a CTA
constexpr int kPlanThreads = 1024;
constexpr int64_t kMaxPages = 1 << 20;             // the plan's bitmap lives in shared memory (128 KB)

__device__ __forceinline__ void bad(int* status) { atomicOr(status, kStatusBadArgument); }

// One chunk of one page: bytes [off, off + kChunk<kVec>) below `bytes` (a multiple of 16).
template <int kVec>
__device__ __forceinline__ void load_chunk(const uint8_t* src, long off, long bytes, uint4 (&v)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const long o = off + (long)(i * kThreads + threadIdx.x) * 16;
    if (o < bytes) v[i] = __ldg(reinterpret_cast<const uint4*>(src + o));
  }
}
template <int kVec>
__device__ __forceinline__ void store_chunk(uint8_t* dst, long off, long bytes, const uint4 (&v)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const long o = off + (long)(i * kThreads + threadIdx.x) * 16;
    if (o < bytes) *reinterpret_cast<uint4*>(dst + o) = v[i];
  }
}

struct ForkArgs {
  uint8_t* cache;
  long page_bytes, layer_bytes;
  int NB, chunks, items; // chunks of one page of one layer, of all layers
  const int* table;      // [S, W]
  long table_stride;
  const int* lens;       // [S]
  int S, W;
  const int* parents;    // [C], negative: no child (a zero row)
  const int* fresh;      // [C]
  int* ref;              // [NB]
  int* out_table;        // [C, W]
  int* out_lens;         // [C]
  int* status;
};

// A fresh page is claimed before a byte of it is written.  Every CTA of child c asks for the claim: the count of a free
// page goes from 0 to a tag of c, and for the time of the launch it is kClaim | c << kClaimBits | CTAs of c that have
// asked; the last of them makes it 1.  It leaves 0 once and for good, so all CTAs of a child get one answer, and a page
// that somebody holds, or that another child has claimed, is left as it is.  (A first kernel for the claims and a
// dependent one for the copies took 14.6 us where this takes 12.0: 128 children over 8 layers of int8 pages and a reset
// of the counts, in a graph.)
constexpr int kClaimBits = 15, kForkCtas = (1 << kClaimBits) - 1;
constexpr int kForkPerSm = 6;  // CTAs per SM, 40 registers a thread
constexpr int64_t kMaxChildren = 65535;
constexpr uint32_t kClaim = 0x80000000u;
static_assert(kMaxChildren <= 1 << (31 - kClaimBits), "a child's number fits its tag");

// grid (1 + copiers <= kForkCtas, children): CTA 0 of a child writes its row, the others copy its unfinished page.  A child
// is made whole or not at all.
__global__ void __launch_bounds__(kThreads, kForkPerSm) fork_kernel(const ForkArgs a) {
  __shared__ bool claimed;
  uint32_t asked = 0;  // CTAs of the child before this one (thread 0)
  const int c = blockIdx.y;
  const int p = a.parents[c], f = a.fresh[c];
  const bool writer = blockIdx.x == 0;
  int len = p >= 0 && p < a.S ? a.lens[p] : -1;
  bool ok = len >= 0 && len <= a.W * kPage;
  if (!ok) len = 0;
  const int n = (len + kPage - 1) / kPage, full = len / kPage;
  const int* row = a.table + (long)(ok ? p : 0) * a.table_stride;
  const int src = n > full ? row[full] : -1;
  // the fresh page is needed (and looked at) only where the last page is not full
  if (n > full) ok = src >= 0 && src < a.NB && f >= 0 && f < a.NB && src != f;
  int item = blockIdx.x - 1;
  auto place = [&](int page, int it) { return a.cache + (long)(it / a.chunks) * a.layer_bytes + page * a.page_bytes; };
  auto offset = [&](int it) { return (long)(it % a.chunks) * kChunk<kForkVec>; };
  uint4 v[kForkVec];
  if (!writer && ok && n > full) load_chunk<kForkVec>(place(src, item), offset(item), a.page_bytes, v);
  for (int j = threadIdx.x; j < full; j += kThreads) ok = ok && row[j] >= 0 && row[j] < a.NB;
  ok = __syncthreads_and(ok);
  const bool claims = ok && n > full;
  if (claims) {
    if (threadIdx.x == 0) {
      const uint32_t tag = kClaim | static_cast<uint32_t>(c) << kClaimBits;
      const uint32_t was = static_cast<uint32_t>(atomicCAS(a.ref + f, 0, static_cast<int>(tag)));
      const bool mine = was == 0 || (was & ~static_cast<uint32_t>(kForkCtas)) == tag;
      if (mine) asked = static_cast<uint32_t>(atomicAdd(a.ref + f, 1)) & kForkCtas;  // looked at behind the stores
      claimed = mine;
    }
    __syncthreads();
    ok = claimed;
  }
  if (writer) {
    for (int j = threadIdx.x; j < a.W; j += kThreads) {
      int page = 0;
      if (ok && j < full) {
        page = row[j];
        if (atomicAdd(a.ref + page, 1) < 0) bad(a.status);  // shared, and some child's fresh page
      } else if (ok && j < n) {
        page = f;
      }
      a.out_table[(long)c * a.W + j] = page;
    }
    if (threadIdx.x == 0) {
      a.out_lens[c] = ok ? len : 0;
      if (!ok && p >= 0) bad(a.status);
    }
  } else if (claims && ok) {
    store_chunk<kForkVec>(place(f, item), offset(item), a.page_bytes, v);
    for (item += gridDim.x - 1; item < a.items; item += gridDim.x - 1) {
      load_chunk<kForkVec>(place(src, item), offset(item), a.page_bytes, v);
      store_chunk<kForkVec>(place(f, item), offset(item), a.page_bytes, v);
    }
  }
  if (claims && ok && threadIdx.x == 0 && asked + 1 == gridDim.x) atomicExch(a.ref + f, 1);
}

struct FreeArgs {
  const int* table;
  long table_stride;
  int* lens;
  int S, W, NB;
  const int* rows;
  int* ref;
  int* status;
};

// One CTA per entry of rows.  The exchange hands the length to one CTA only, so a row named twice is freed once.
__global__ void __launch_bounds__(128) free_kernel(const FreeArgs a) {
  const int r = a.rows[blockIdx.x];
  if (r < 0) return;
  __shared__ int s_len;
  if (threadIdx.x == 0) {
    int len = 0;
    if (r >= a.S) {
      bad(a.status);
    } else {
      len = atomicExch(a.lens + r, 0);
      if (len < 0 || len > a.W * kPage) {
        bad(a.status);
        len = 0;
      }
    }
    s_len = len;
  }
  __syncthreads();
  const int n = (s_len + kPage - 1) / kPage;
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int page = a.table[(long)r * a.table_stride + j];
    if (page < 0 || page >= a.NB) {
      bad(a.status);
    } else if (atomicSub(a.ref + page, 1) <= 0) {  // nothing held it
      atomicAdd(a.ref + page, 1);
      bad(a.status);
    }
  }
}

struct CompactArgs {
  uint8_t* cache;
  long page_bytes, layer_bytes;
  int NB, L, chunks;
  int* table;
  long table_stride;
  const int* lens;
  int S, W;
  int* ref;
  int* moved;     // [NB] new page id of a held page, -1 of a free one
  int* used;      // [1] U
  int* src;       // [NB / 2 + 1] the moves
  int* dst;
  int* n_moves;   // [1]
  int* status;
};

// Sum over the block of two counters, exclusive prefix returned in place.
__device__ __forceinline__ int2 block_exscan2(int2 v, int2* warp_sums, int2& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int2 x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int ax = __shfl_up_sync(0xffffffffu, x.x, o), ay = __shfl_up_sync(0xffffffffu, x.y, o);
    if (lane >= o) {
      x.x += ax;
      x.y += ay;
    }
  }
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  if (w == 0) {
    int2 y = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int ax = __shfl_up_sync(0xffffffffu, y.x, o), ay = __shfl_up_sync(0xffffffffu, y.y, o);
      if (lane >= o) {
        y.x += ax;
        y.y += ay;
      }
    }
    warp_sums[lane] = y;
  }
  __syncthreads();
  const int2 before = w ? warp_sums[w - 1] : make_int2(0, 0);
  total = warp_sums[31];
  __syncthreads();
  return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// One CTA: ref -> bitmap of held pages in shared memory, U, the list of moves, the map, the new ref.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const CompactArgs a) {
  extern __shared__ uint32_t held[];
  __shared__ int2 sums[32];
  griddep_launch_dependents();
  const int t = threadIdx.x, lane = t & 31;
  const int words = (a.NB + 31) / 32;
  int mine = 0;
  constexpr int kUnroll = 8;
  for (int base = 0; base < words * 32; base += kPlanThreads * kUnroll) {
    int r[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int p = base + u * kPlanThreads + t;
      r[u] = p < a.NB ? a.ref[p] : 0;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int p = base + u * kPlanThreads + t;
      const uint32_t m = __ballot_sync(0xffffffffu, r[u] > 0);
      if (lane == 0 && p < words * 32) {
        held[p >> 5] = m;
        mine += __popc(m);
      }
    }
  }
  int2 tot;
  block_exscan2(make_int2(mine, 0), sums, tot);  // its barriers also publish the bitmap
  const int U = tot.x;
  // holes below U and held pages at or above U, ranked over contiguous runs of words
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  const int w0 = min(t * per, words), w1 = min(w0 + per, words);
  auto split = [&](int w, uint32_t& hole, uint32_t& high) {
    const int left = U - w * 32;  // pages of this word that lie below U
    const uint32_t below = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
    hole = ~held[w] & below;
    high = held[w] & ~below;
  };
  int2 cnt = make_int2(0, 0);
  for (int w = w0; w < w1; ++w) {
    uint32_t hole, high;
    split(w, hole, high);
    cnt.x += __popc(hole);
    cnt.y += __popc(high);
  }
  int2 at = block_exscan2(cnt, sums, tot);
  for (int w = w0; w < w1; ++w) {
    uint32_t hole, high;
    split(w, hole, high);
    for (; hole; hole &= hole - 1) a.dst[at.x++] = w * 32 + __ffs(hole) - 1;
    for (; high; high &= high - 1) a.src[at.y++] = w * 32 + __ffs(high) - 1;
  }
  if (t == 0) {
    *a.used = U;
    *a.n_moves = tot.y;
  }
  for (int p = t; p < a.NB; p += kPlanThreads) {
    const bool h = (held[p >> 5] >> (p & 31)) & 1u;
    if (!h) a.moved[p] = -1;
    else if (p < U) a.moved[p] = p;
  }
  __syncthreads();
  for (int i = t; i < tot.y; i += kPlanThreads) {
    const int s = a.src[i], d = a.dst[i];
    a.moved[s] = d;
    a.ref[d] = a.ref[s];
    a.ref[s] = 0;
  }
}

// CTAs [0, rows) rewrite one table row each, the others copy pages.
__global__ void __launch_bounds__(kThreads) move_kernel(const CompactArgs a) {
  griddep_wait();
  if (blockIdx.x < a.S) {
    const int r = blockIdx.x;
    const int len = a.lens[r];
    if (len < 0 || len > a.W * kPage) {
      if (threadIdx.x == 0) bad(a.status);
      return;
    }
    const int n = (len + kPage - 1) / kPage;
    for (int j = threadIdx.x; j < n; j += kThreads) {
      int* e = a.table + (long)r * a.table_stride + j;
      const int page = *e;
      const int to = page >= 0 && page < a.NB ? a.moved[page] : -1;
      if (to < 0) bad(a.status);  // no such page, or one that nothing holds
      else *e = to;
    }
    return;
  }
  const long items = (long)*a.n_moves * a.L * a.chunks;
  for (long it = blockIdx.x - a.S; it < items; it += gridDim.x - a.S) {
    const int chunk = int(it % a.chunks);
    const long ml = it / a.chunks;
    const int l = int(ml % a.L);
    const int m = int(ml / a.L);
    const long layer = (long)l * a.layer_bytes, off = (long)chunk * kChunk<kMoveVec>;
    // both ids before the loads: the target's would otherwise be fetched after them
    const uint8_t* from = a.cache + layer + a.src[m] * a.page_bytes;
    uint8_t* to = a.cache + layer + a.dst[m] * a.page_bytes;
    uint4 v[kMoveVec];
    load_chunk<kMoveVec>(from, off, a.page_bytes, v);
    store_chunk<kMoveVec>(to, off, a.page_bytes, v);
  }
}

// Shapes and types first, devices last: a wrong call is refused alike with and without a GPU.  The messages are
// single literals: formatting one needs iostreams, which crash where the extension was linked to a libstdc++ of its own.
#define PAGES_INTS(op, t) \
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(), op ": " #t " must be contiguous int32")
#define PAGES_TABLE(op, t, lens)                                                                      \
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1) &&  \
                  (t.size(0) <= 1 || t.stride(0) >= t.size(1)),                                       \
              op ": " #t " must be int32 [S, W] with contiguous rows that do not overlap");           \
  PAGES_INTS(op, lens);                                                                               \
  TORCH_CHECK(lens.size(0) == t.size(0), op ": " #lens " must have one length per table row")
#define PAGES_CACHE(op, c, ref)                                                                                   \
  TORCH_CHECK(c.dim() >= 3 && c.is_contiguous(), op ": " #c " must be contiguous [L, NB, ...]");                  \
  TORCH_CHECK(c.numel() > 0 && c.size(1) <= kMaxPages, op ": " #c " must hold 1 to 2^20 pages");                  \
  TORCH_CHECK(c.stride(1) * c.element_size() % 16 == 0, op ": a page must be a multiple of 16 bytes");            \
  TORCH_CHECK((reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0, op ": " #c " must start on a 16-byte boundary"); \
  PAGES_INTS(op, ref);                                                                                            \
  TORCH_CHECK(ref.size(0) == c.size(1), op ": " #ref " must have one count per page")
#define PAGES_DEVICE(op, a, ...)                                              \
  TORCH_CHECK(a.is_cuda(), op ": tensors must be on a CUDA device");          \
  TORCH_CHECK(on_device(a, __VA_ARGS__), op ": tensors must be on one device")
bool on_device(const torch::Tensor& a, std::initializer_list<const torch::Tensor*> rest) {
  return std::all_of(rest.begin(), rest.end(), [&](const torch::Tensor* t) { return t->device() == a.device(); });
}
template <int kVec>
int page_chunks(const torch::Tensor& c) {
  return int((c.stride(1) * c.element_size() + kChunk<kVec> - 1) / kChunk<kVec>);
}

}  // namespace pages

std::tuple<torch::Tensor, torch::Tensor> kv_fork(torch::Tensor& kv_cache, const torch::Tensor& block_table,
                                                 const torch::Tensor& seq_lens, const torch::Tensor& parents,
                                                 const torch::Tensor& fresh, torch::Tensor& ref) {
  using namespace pages;
  PAGES_CACHE("kv_fork", kv_cache, ref);
  PAGES_TABLE("kv_fork", block_table, seq_lens);
  PAGES_INTS("kv_fork", parents);
  PAGES_INTS("kv_fork", fresh);
  TORCH_CHECK(fresh.size(0) == parents.size(0), "kv_fork: fresh must have one page per child");
  TORCH_CHECK(parents.size(0) <= kMaxChildren, "kv_fork: at most 65535 children");
  PAGES_DEVICE("kv_fork", kv_cache, {&block_table, &seq_lens, &parents, &fresh, &ref});
  const at::cuda::CUDAGuard guard(kv_cache.device());
  const int C = int(parents.size(0)), W = int(block_table.size(1));
  auto table = torch::empty({C, W}, block_table.options());
  auto lens = torch::empty({C}, seq_lens.options());
  if (C == 0) return {table, lens};
  ForkArgs a;
  a.cache = static_cast<uint8_t*>(kv_cache.data_ptr());
  a.page_bytes = kv_cache.stride(1) * kv_cache.element_size();
  a.layer_bytes = a.page_bytes * kv_cache.size(1);
  a.NB = int(kv_cache.size(1));
  a.chunks = page_chunks<kForkVec>(kv_cache);
  TORCH_CHECK(kv_cache.size(0) * a.chunks < (1ll << 30), "kv_fork: pages too large");
  a.items = int(kv_cache.size(0)) * a.chunks;
  a.table = block_table.data_ptr<int>();
  a.table_stride = block_table.stride(0);
  a.lens = seq_lens.data_ptr<int>();
  a.S = int(seq_lens.size(0));
  a.W = W;
  a.parents = parents.data_ptr<int>();
  a.fresh = fresh.data_ptr<int>();
  a.ref = ref.data_ptr<int>();
  a.out_table = table.data_ptr<int>();
  a.out_lens = lens.data_ptr<int>();
  a.status = status_word(kv_cache.get_device());
  // copiers of a child: one per step, and where that is more than one wave of CTAs, as many as are
  const int room = std::min(std::max(kForkPerSm * num_sms(kv_cache.get_device()) / C - 1, 1), kForkCtas - 1);
  const int steps = (a.items + room - 1) / room;
  const dim3 grid(unsigned(1 + (a.items + steps - 1) / steps), unsigned(C));
  fork_kernel<<<grid, kThreads, 0, at::cuda::getCurrentCUDAStream()>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {table, lens};
}

void kv_free(const torch::Tensor& block_table, torch::Tensor& seq_lens, const torch::Tensor& rows,
             torch::Tensor& ref) {
  using namespace pages;
  PAGES_TABLE("kv_free", block_table, seq_lens);
  PAGES_INTS("kv_free", rows);
  PAGES_INTS("kv_free", ref);
  PAGES_DEVICE("kv_free", block_table, {&seq_lens, &rows, &ref});
  if (rows.size(0) == 0) return;
  const at::cuda::CUDAGuard guard(block_table.device());
  FreeArgs a;
  a.table = block_table.data_ptr<int>();
  a.table_stride = block_table.stride(0);
  a.lens = seq_lens.data_ptr<int>();
  a.S = int(seq_lens.size(0));
  a.W = int(block_table.size(1));
  a.NB = int(ref.size(0));
  a.rows = rows.data_ptr<int>();
  a.ref = ref.data_ptr<int>();
  a.status = status_word(block_table.get_device());
  free_kernel<<<unsigned(rows.size(0)), 128, 0, at::cuda::getCurrentCUDAStream()>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

std::tuple<torch::Tensor, torch::Tensor> kv_compact(torch::Tensor& kv_cache, torch::Tensor& block_table,
                                                    const torch::Tensor& seq_lens, torch::Tensor& ref) {
  using namespace pages;
  PAGES_CACHE("kv_compact", kv_cache, ref);
  PAGES_TABLE("kv_compact", block_table, seq_lens);
  PAGES_DEVICE("kv_compact", kv_cache, {&block_table, &seq_lens, &ref});
  const at::cuda::CUDAGuard guard(kv_cache.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int NB = int(kv_cache.size(1));
  auto moved = torch::empty({NB}, ref.options());
  auto used = torch::empty({1}, ref.options());
  const int half = NB / 2 + 1;
  auto ws = torch::empty({2 * half + 1}, ref.options());  // the moves: sources, targets, their number
  CompactArgs a;
  a.cache = static_cast<uint8_t*>(kv_cache.data_ptr());
  a.page_bytes = kv_cache.stride(1) * kv_cache.element_size();
  a.layer_bytes = a.page_bytes * NB;
  a.NB = NB;
  a.L = int(kv_cache.size(0));
  a.chunks = page_chunks<kMoveVec>(kv_cache);
  a.table = block_table.data_ptr<int>();
  a.table_stride = block_table.stride(0);
  a.lens = seq_lens.data_ptr<int>();
  a.S = int(seq_lens.size(0));
  a.W = int(block_table.size(1));
  a.ref = ref.data_ptr<int>();
  a.moved = moved.data_ptr<int>();
  a.used = used.data_ptr<int>();
  a.src = ws.data_ptr<int>();
  a.dst = a.src + half;
  a.n_moves = a.dst + half;
  a.status = status_word(kv_cache.get_device());
  const int smem = (NB + 31) / 32 * 4;
  if (smem > 48 * 1024)  // pools of more than 393,216 pages
    C10_CUDA_CHECK(cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxPages / 8));
  plan_kernel<<<1, kPlanThreads, smem, stream>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  // no more copy CTAs than there can be chunks, and at most 8 per SM (4 at a time; each goes on to further chunks)
  const long most = std::max<long>(1, (long)(NB / 2) * a.L * a.chunks);
  const int copiers = int(std::min<long>(most, 8L * num_sms(kv_cache.get_device())));
  cudaLaunchConfig_t cfg = {};  // a dependent launch: its CTAs are there when the plan is done
  cfg.gridDim = dim3(unsigned(a.S + copiers));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, move_kernel, a));
  return {moved, used};
}

}  // namespace bloom

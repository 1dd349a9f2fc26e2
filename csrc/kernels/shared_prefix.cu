// Decode / verify attention of a batch whose sequences share long prefixes (many completions of one prompt, requests
// behind one system prompt).
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q.k_j
//
// splits exactly at any key: with (o1, m1, l1) over the prefix and (o2, m2, l2) over a row's own pages,
// o = (o1 2^(m1-M) + o2 2^(m2-M)) / (l1 2^(m1-M) + l2 2^(m2-M)).  So the prefix of a group is read once for all of its
// members, as a product with members x q_len x (q heads per KV head) rows, and only the rest is read per sequence.
//
// The prefix kernel (work items: a tile of a group's rows x a range of the prefix) leaves partial sums in fp32, the
// suffix kernel is one CTA (or several over the pages) per sequence, KV head and chunk of rows.  Groups of few rows:
// two launches, the suffix kernel a dependent of the prefix kernel that adds the parts at its end.  Groups of many rows,
// whose prefix is work for the tensor cores: both side by side on two streams, and a third kernel adds the parts.
//
// Bound by: few sequences, a chain of dependent loads (10 us with 4 sequences behind 512 tokens); many, the prefix's
// softmax (50 us for 35 GFLOP) beside the suffixes' pages (63 us for 268 MB of 1 to 511 tokens each): 107 us together
// for 256 sequences behind 8,192 tokens, 93 where each has 256 of its own; the decode kernel that reads every sequence's
// whole table takes 826.  32 sequences behind 4,096 tokens, 128 of their own: 25 us, decode kernel 63.  (32 / 8 heads of
// 128, captured.)
//
// Slots behind a sequence's last token may hold anything (NaN too): scores there are replaced, and V rows there are
// zeroed in shared memory.  A block id outside the cache sets kStatusBadArgument and page 0 is read instead.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <mutex>
#include <vector>

#include "bloom/common.cuh"
#include "bloom/ops_share.h"
#include "bloom/tma_host.h"

namespace cg = cooperative_groups;

namespace bloom {
namespace shared_prefix {

constexpr int PAGE = 16;
constexpr float kNegBig = -1e30f;
constexpr int kStages = 3;   // ring depth of a streaming warp, in pages
constexpr int kMaxWarps = 8; // of a streaming CTA: 8 rings fill an SM's shared memory (and 255 registers its file)

struct Group {  // one row of plan.groups
  int first, members, prefix, chunk;  // first sequence, sequences, shared tokens, prefix tokens per split
};

struct Args {
  const __nv_bfloat16* q;  // [B * ql, nq, D]
  long q_stride;           // elements between token rows
  __nv_bfloat16* out;
  long out_stride;
  const int* table;
  long table_stride;
  int W;
  const int* lens;         // [B]
  const int4* items;       // prefix work: {group, first row, split, -}
  const Group* groups;
  const int2* seqs;        // [B] {shared tokens, splits of them}
  float* part_o;           // [splits, B * ql, nq, D]
  float2* part_ml;         // [splits, B * ql, nq]
  int B, nq, nkv, ql, NB;
  int parts;               // partial sums per prefix split: 2 where the two streams of a CTA leave one each
  uint32_t per_g;          // ceil(2^32 / G), G = nq / nkv: r / G = (r * per_g) >> 32 while r * G < 2^32
  float scale_log2;
  int* status;
};

__device__ __forceinline__ int div_g(const Args& a, int r) {
  return a.per_g ? int(__umulhi(unsigned(r), a.per_g)) : r;  // 0 stands for 2^32: G = 1
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void mma_bf16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Byte address of element (tok, d), d a multiple of 8, of a page that TMA wrote as 2 KB boxes of 64 dims with the
// 128-byte swizzle.
__device__ __forceinline__ uint32_t page_addr(uint32_t base, int tok, int d) {
  return base + ((d >> 6) << 11) + (tok << 7) + (((((d & 63) >> 3) ^ (tok & 7))) << 4);
}

// Length of sequence b, kept inside its table row.
__device__ __forceinline__ int seq_len(const Args& a, int b) {
  const int n = a.lens[b];
  if (n < 0 || n > a.W * PAGE) {
    atomicOr(a.status, kStatusBadArgument);
    return n < 0 ? 0 : a.W * PAGE;
  }
  return n;
}
__device__ __forceinline__ int block_id(const Args& a, const int* row, int page) {
  const int blk = __ldg(row + page);
  if (blk < 0 || blk >= a.NB) {
    atomicOr(a.status, kStatusBadArgument);
    return 0;
  }
  return blk;
}

// The member of a group whose table row the prefix is read through: the first that holds the most of it (members that
// have ended, of length 0, are passed over).  Every lane of the calling warp gets {member, prefix tokens it holds}.
__device__ __forceinline__ int2 prefix_holder(const Args& a, const Group& g) {
  // lengths are taken into the table row; the suffix kernel reports those that are not in it
  unsigned long long best = 0;
#pragma unroll 8
  for (int i = lane_id(); i < g.members; i += 32) {
    const int n = max(0, min(min(__ldg(a.lens + g.first + i), a.W * PAGE), g.prefix));
    const unsigned long long v = (static_cast<unsigned long long>(n) << 32) | (0xffffffffu - unsigned(i));
    best = v > best ? v : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long v = __shfl_xor_sync(0xffffffffu, best, o);
    best = v > best ? v : best;
  }
  return make_int2(g.first + int(0xffffffffu - unsigned(best)), int(best >> 32));
}

template <int D>
constexpr int stage_bytes() { return 2 * PAGE * D * 2; }  // a page's K and V
// Shared memory of a streaming CTA: the warps' rings, after the loop one partial result per warp and row; barriers.
template <int D>
int stream_smem(int warps, int rows) {
  return std::max(warps * kStages * stage_bytes<D>(), warps * rows * (D + 2) * 4) + warps * kStages * 8 + 1024;
}

// Streams keys [k_begin, k_end) of one KV head past up to NT * 8 packed query rows (row r: token q0 + (r0 + r) / G,
// q head kh * G + (r0 + r) % G; limit(r): the last key that it sees) and leaves, in shared memory, row r's O[D], m, l at
// result + r * (D + 2).  A page is read once for all rows.
//
// The products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that keys and dims fill the 16-row side of
// m16n8k16 and 4 to 8 query rows (a GQA group) fill its 8-column side: half the MMAs and half the registers for O of
// the other way round.  P^T moves from accumulator to B fragments by an 8x8 transpose of the warp.  Each warp takes
// every warps-th page through its own TMA ring.  (Loading fragments straight into registers needs no barriers, but
// keeps only a page per warp in flight, and at 128 registers spills: 79 us where the rings take 62 us for 268 MB of
// 2,048 short sequences x heads.)
template <int D, int NT, typename Limit>
__device__ float* stream(const CUtensorMap& tm, const Args& a, uint8_t* smem, int* abort_flag, const int* row, int kh,
                         long q0, int r0, int rows, int k_begin, int k_end, Limit&& limit_of) {
  constexpr int RS = D + 2, kStage = stage_bytes<D>(), kPageB = PAGE * D * 2;
  const int warps = blockDim.x / 32, warp = warp_id(), lane = lane_id(), g = lane >> 2, t4 = lane & 3;
  const int G = a.nq / a.nkv;
  const int p0 = k_begin / PAGE, p1 = k_end > k_begin ? (k_end + PAGE - 1) / PAGE : p0;
  const int first = p0 + warp;
  const int n = p1 > first ? (p1 - first + warps - 1) / warps : 0;
  uint8_t* ring = smem + warp * kStages * kStage;
  uint64_t* bars =
      reinterpret_cast<uint64_t*>(smem + max(warps * kStages * kStage, warps * rows * RS * 4)) + warp * kStages;

  int ids = 0;  // block ids of this warp's next 32 pages, one per lane
  auto fetch_ids = [&](int i) {
    const int p = first + (i + lane) * warps;
    ids = p < p1 ? block_id(a, row, p) : 0;
  };
  auto issue = [&](int i) {
    if ((i & 31) == 0) fetch_ids(i);
    const int blk = __shfl_sync(0xffffffffu, ids, i & 31), s = i % kStages;
    if (lane == 0) {
      const int rowK = (blk * 2 * a.nkv + kh) * PAGE, rowV = rowK + a.nkv * PAGE;
      uint8_t* st = ring + s * kStage;
      mbar_arrive_expect_tx(&bars[s], kStage);
      tma_load_2d(st, &tm, &bars[s], 0, rowK);
      if constexpr (D == 128) tma_load_2d(st + 2048, &tm, &bars[s], 64, rowK);
      tma_load_2d(st + kPageB, &tm, &bars[s], 0, rowV);
      if constexpr (D == 128) tma_load_2d(st + kPageB + 2048, &tm, &bars[s], 64, rowV);
    }
  };
  if (lane == 0) {  // a ring belongs to its warp: no other thread waits on it
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  for (int i = 0; i < kStages && i < n; ++i) issue(i);

  // Q^T fragments: row g of each 8-row tile, dims 16 ks + 2 t4 and the next, + 8
  uint32_t qf[NT][D / 16][2];
  int limit[NT][2], low = 0x7fffffff;  // of rows 8 nt + 2 t4 + e
  float m_run[NT][2], l_run[NT][2], o[NT][D / 16][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int rq = nt * 8 + g, qi = div_g(a, r0 + rq);
    const uint32_t* q =
        reinterpret_cast<const uint32_t*>(a.q + (q0 + qi) * a.q_stride + (kh * G + r0 + rq - qi * G) * D) + t4;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      qf[nt][ks][0] = rq < rows ? __ldg(q + 8 * ks) : 0u;
      qf[nt][ks][1] = rq < rows ? __ldg(q + 8 * ks + 4) : 0u;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * t4 + e;
      limit[nt][e] = r < rows ? min(limit_of(r), k_end - 1) : 0x7fffffff;  // padding rows are not masked, nor used
      low = min(low, limit[nt][e]);
      m_run[nt][e] = kNegBig;
      l_run[nt][e] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
  }
  low = __reduce_min_sync(0xffffffffu, low);
  bool ok = true;
  int i = 0;
  for (; i < n; ++i) {
    const int s = i % kStages;
    ok = __all_sync(0xffffffffu, mbar_wait(&bars[s], (i / kStages) & 1, abort_flag, a.status, kStatusAttnTimeout));
    if (!ok) break;
    const uint32_t sK = smem_u32(ring + s * kStage), sV = sK + kPageB;
    const int tok0 = (first + i * warps) * PAGE;
    if (tok0 + PAGE > k_end) {  // V rows behind the last key: whatever they hold must not meet p = 0
      for (int c = lane; c < PAGE * D / 8; c += 32) {
        const int tok = c & 15, d = (c >> 4) * 8;
        if (tok0 + tok >= k_end)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(page_addr(sV, tok, d)), "r"(0) : "memory");
      }
      __syncwarp();
    }
    float sc[NT][4];  // [key g: rows 2 t4, 2 t4 + 1 | key g + 8: the same]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      uint32_t k[4];
      ldsm_x4(page_addr(sK, lane & 15, 16 * ks + 8 * (lane >> 4)), k[0], k[1], k[2], k[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(sc[nt], k, qf[nt][ks][0], qf[nt][ks][1]);
    }
    const bool whole = tok0 >= k_begin && tok0 + PAGE - 1 <= low;  // every row sees every key of the page
    uint32_t pb[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int idx = tok0 + g + 8 * h;
          float& x = sc[nt][2 * h + e];
          x *= a.scale_log2;
          if (!whole && (idx < k_begin || idx > limit[nt][e])) x = -INFINITY;
        }
        mx[e] = fmaxf(sc[nt][e], sc[nt][2 + e]);
      }
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], w));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], w));
      }
      const bool grows = mx[0] > m_run[nt][0] || mx[1] > m_run[nt][1];
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m_new = fmaxf(m_run[nt][e], mx[e]);
          const float alpha = exp2f(m_run[nt][e] - m_new);
          m_run[nt][e] = m_new;
          l_run[nt][e] *= alpha;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            o[nt][j][e] *= alpha;
            o[nt][j][2 + e] *= alpha;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x0 = exp2f(sc[nt][2 * h] - m_run[nt][0]), x1 = exp2f(sc[nt][2 * h + 1] - m_run[nt][1]);
        l_run[nt][0] += x0;
        l_run[nt][1] += x1;
        // P is rounded to bf16 (2^-8 relative at most) for the tensor cores; l keeps the fp32 sum
        const uint32_t p = pack_bf16x2(x0, x1);
        asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pb[nt][h]) : "r"(p));
      }
    }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {  // dims 16 j + g and + 8
      uint32_t v[4];
      ldsm_x4_t(page_addr(sV, (lane & 7) + 8 * (lane >> 4), 16 * j + (lane & 8)), v[0], v[1], v[2], v[3]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][j], v, pb[nt][0], pb[nt][1]);
    }
    __syncwarp();
    if (i + kStages < n) {
      if (lane == 0) fence_proxy_async();
      issue(i + kStages);
    }
  }
  if (!ok && lane == 0)  // gave up: the loads in flight must land before the shared memory is reused
    for (int k = i; k < n && k < i + kStages; ++k) mbar_drain(&bars[k % kStages], (k / kStages) & 1);
  if (warps > 1) __syncthreads();
  else __syncwarp();
  // the warps' results over their rings, then summed into warp 0's place
  float* cm = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[nt][e];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
      const int r = nt * 8 + 2 * t4 + e;
      if (r < rows) {
        float* w = cm + (warp * rows + r) * RS;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          w[16 * j + g] = o[nt][j][e];
          w[16 * j + 8 + g] = o[nt][j][2 + e];
        }
        if (g == 0) *reinterpret_cast<float2*>(w + D) = make_float2(m_run[nt][e], l);
      }
    }
  if (warps == 1) {
    __syncwarp();
    return cm;
  }
  __syncthreads();
  // one warp per row, the (m, l) of part w in lane w
  for (int r = warp; r < rows; r += warps) {
    const float2 ml = lane < warps ? *reinterpret_cast<const float2*>(cm + (lane * rows + r) * RS + D)
                                   : make_float2(kNegBig, 0.f);
    const float M = warp_max(ml.x), f = exp2f(ml.x - M), L = warp_sum(ml.y * f);
    float O[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) O[c] = 0.f;
    for (int w = 0; w < warps; ++w) {
      const float fw = __shfl_sync(0xffffffffu, f, w);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) O[c] += cm[(w * rows + r) * RS + c * 32 + lane] * fw;
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < D / 32; ++c) cm[r * RS + c * 32 + lane] = O[c];
    if (lane == 0) *reinterpret_cast<float2*>(cm + r * RS + D) = make_float2(M, L);
  }
  __syncthreads();
  return cm;
}

// Prefix work of groups with few rows: the keys stream past at most NT * 8 of them.  grid (items, KV heads).
template <int D, int NT>
__global__ void __launch_bounds__(kMaxWarps * 32) 
    prefix_stream_kernel(const __grid_constant__ CUtensorMap tm, const Args a) {
  griddep_launch_dependents();
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ int abort_flag;
  if (threadIdx.x == 0) abort_flag = 0;
  __syncthreads();
  const int4 it = a.items[blockIdx.x];
  const Group gr = a.groups[it.x];
  const int kh = blockIdx.y, G = a.nq / a.nkv;
  const int2 hold = prefix_holder(a, gr);
  const int k0 = min(it.z * gr.chunk, hold.y), k1 = min(k0 + gr.chunk, hold.y);
  const int rows = min(NT * 8, gr.members * a.ql * G - it.y);
  const long q0 = (long)gr.first * a.ql;
  const float* res = stream<D, NT>(tm, a, smem, &abort_flag, a.table + hold.x * a.table_stride, kh, q0, it.y, rows, k0, k1, [&](int r) {
                                     const int tok = div_g(a, it.y + r);
                                     return seq_len(a, gr.first + tok / a.ql) - a.ql + tok % a.ql;
                                   });
  constexpr int RS = D + 2;
  for (int idx = threadIdx.x; idx < rows * (D / 4); idx += blockDim.x) {
    const int r = idx / (D / 4), d = idx % (D / 4) * 4;
    const long at = ((long)it.z * a.B * a.ql + q0 + div_g(a, it.y + r)) * a.nq + kh * G + (it.y + r - div_g(a, it.y + r) * G);
    const float* p = res + r * RS + d;
    *reinterpret_cast<float4*>(a.part_o + at * D + d) = make_float4(p[0], p[1], p[2], p[3]);
    if (d == 0) a.part_ml[at] = make_float2(res[r * RS + D], res[r * RS + D + 1]);
  }
}

// ---------------------------------------------------------------- prefix on tcgen05
// Groups with more rows than a streaming CTA holds: S = Q K^T and O += P V on the 5th-generation tensor cores, with
// 128 rows per softmax warpgroup, one thread per row (no exchange between threads).  A CTA runs two such streams:
//   pair   (256-row items)  two row tiles over the same K / V tiles, so each K / V tile serves 256 rows
//   single (128-row items)  one row tile, the streams take alternate K / V tiles and leave one partial sum each
// Tiles of 64 keys, so that TMEM holds two S buffers per stream beside the two O (4 x 64 + 2 x 128 columns): S(i + 1)
// is formed while the softmax works on S(i), and the softmax never waits for a product.  P (bf16, two keys per column)
// is written over the first half of its S and read from there as the A operand.  With 128-key tiles and one S buffer
// per stream, S(i + 1) had to wait for P V(i), and each tile's softmax for both: 6,300 cycles per 128 keys of a pair,
// half of them waiting.  The running max is lazy: O is rescaled (and P V(i - 1) waited for) only when a row's max
// grows by more than 2^8.
// Warps 0-7 softmax and epilogue, warp 8 TMA producer and TMEM owner, warps 9 and 10 issue the MMAs of a stream each.
namespace tc {

constexpr int kRows = 128, kKv = 64;
constexpr int kThreads = 256 + 32 + 64;
constexpr int kTmemCols = 512;
constexpr float kLazy = 8.f;  // log2 units

template <int D, bool kPair>
struct Cfg {
  static constexpr int kRegion = kKv * 128;       // 64 dims of a K or V tile: token rows of 128 bytes
  static constexpr int kTile = kKv * D * 2;
  static constexpr int kQ = kRows * D * 2;
  // of the K ring and of the V ring: one row tile waits for memory, two for the tensor cores, and leave room for CTAs
  // of the suffix kernel
  static constexpr int kStages = D == 64 ? 8 : kPair ? 2 : 5;
  static constexpr int kSmem = (kPair ? 2 : 1) * kQ + 2 * kStages * kTile + 512 + 1024;
};

__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Orders the use of loaded registers behind the wait for them: an empty statement that reads and writes them.
__device__ __forceinline__ void pin(float (&v)[16]) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}
// Two fp32 operations in one instruction, and the largest of three.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// D[tmem] (+)= A[tmem] B[smem desc], A: lane = row, two consecutive bf16 k per 32-bit column
__device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}
// V as the B operand, its contiguous dimension being N: 64-element atoms `lbo` bytes apart, 8-key groups 1024 apart.
__device__ __forceinline__ uint64_t desc_mn(uint32_t smem_addr, uint32_t lbo) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>(1024u >> 4) << 32 | static_cast<uint64_t>(1u) << 46 | static_cast<uint64_t>(2u) << 61;
}

// grid (items, KV heads)
template <int D, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tm, const Args a) {
  if constexpr (!kPair) griddep_launch_dependents();
  using C = Cfg<D, kPair>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + (kPair ? 2 : 1) * C::kQ;
  uint8_t* sV = sK + kStages * C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kStages * C::kTile);
  uint64_t *fullK = bars, *emptyK = bars + 8, *fullV = bars + 16, *emptyV = bars + 24;
  // [2 * stream + (tile & 1)]
  uint64_t *s_done = bars + 32, *p_ready = bars + 36, *o_done = bars + 40;
  uint64_t *q_ready = bars + 44, *drain = bars + 45;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 47);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id(), lane = lane_id();
  const int4 it = a.items[blockIdx.x];
  const Group gr = a.groups[it.x];
  const int kh = blockIdx.y, G = a.nq / a.nkv;
  const int2 hold = prefix_holder(a, gr);
  const int* table = a.table + hold.x * a.table_stride;
  const int k0 = min(it.z * gr.chunk, hold.y), k1 = min(k0 + gr.chunk, hold.y);  // k0 is a multiple of kKv
  const int n_kt = (k1 - k0 + kKv - 1) / kKv;
  const int rows = gr.members * a.ql * G;  // of the whole group
  const bool two = kPair && rows - it.y > kRows;  // the second row tile holds rows
  // K / V tiles of stream w, and the i-th of them
  auto count = [&](int w) { return kPair ? (w == 0 || two ? n_kt : 0) : (n_kt - w + 1) / 2; };
  auto tile = [&](int w, int i) { return kPair ? i : 2 * i + w; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&fullK[s], 1);
      mbar_init(&fullV[s], 1);
      mbar_init(&emptyK[s], two ? 2 : 1);
      mbar_init(&emptyV[s], two ? 2 : 1);
    }
    for (int w = 0; w < 4; ++w) {
      mbar_init(&s_done[w], 1);
      mbar_init(&p_ready[w], 4);
      mbar_init(&o_done[w], 1);
    }
    mbar_init(q_ready, kPair ? 8 : 4);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // S(i) of stream w at 128 w + 64 (i & 1), O at 256 + 128 w

  if (warp == 8) {
    // Lane p * (D / 64) + r brings 64 dims of page p of a tile.
    constexpr int kBoxes = kKv / PAGE * (D / 64);
    const int n_pages = (k1 + PAGE - 1) / PAGE, rg = lane % (D / 64);
    auto fetch_id = [&](int t) {  // behind the end: any page, it is masked
      const int page = k0 / PAGE + t * (kKv / PAGE) + lane / (D / 64);
      return lane < kBoxes && t < n_kt ? block_id(a, table, page < n_pages ? page : k0 / PAGE) : 0;
    };
    auto load = [&](int id, uint8_t* dst, uint64_t* bar, int kv) {
      if (lane == 0) mbar_arrive_expect_tx(bar, C::kTile);
      __syncwarp();
      if (lane < kBoxes)
        tma_load_2d(dst + rg * C::kRegion + lane / (D / 64) * 2048, &tm, bar, 64 * rg,
                    ((id * 2 + kv) * a.nkv + kh) * PAGE);
    };
    auto free_slot = [&](uint64_t* bar, int n) {  // one answer for the warp
      return __shfl_sync(0xffffffffu, int(mbar_test(&bar[n % kStages], ((n / kStages) & 1) ^ 1u)), 0) != 0;
    };
    int nK = 0, nV = 0, idK = fetch_id(0), idV = idK;
    bool ok = true;
    uint64_t t_stall = 0;
    uint32_t spins = 0;  // since the last progress
    while (ok && (nK < n_kt || nV < n_kt)) {  // the rings advance on their own; V never runs ahead of K
      bool progressed = false;
      if (nK < n_kt && free_slot(emptyK, nK)) {
        load(idK, sK + nK % kStages * C::kTile, &fullK[nK % kStages], 0);
        idK = fetch_id(++nK);
        progressed = true;
      }
      if (nV < nK && free_slot(emptyV, nV)) {
        load(idV, sV + nV % kStages * C::kTile, &fullV[nV % kStages], 1);
        idV = fetch_id(++nV);
        progressed = true;
      }
      if (progressed) {
        spins = 0;
      } else if ((++spins & 63u) == 0) {
        bool stop = false;
        if (lane == 0) {
          stop = *abort_flag;
          if (spins == 64) t_stall = globaltimer_ns();
          if (!stop && globaltimer_ns() - t_stall > kLocalWaitTimeoutNs) {
            *abort_flag = 1;
            atomicOr(a.status, kStatusAttnTimeout);
            stop = true;
          }
        }
        ok = !__shfl_sync(0xffffffffu, int(stop), 0);
      }
    }
    if (!ok && lane == 0) {  // the loads in flight land before the block leaves (bounded)
      for (int j = max(0, nK - kStages); j < nK; ++j) mbar_drain(&fullK[j % kStages], (j / kStages) & 1);
      for (int j = max(0, nV - kStages); j < nV; ++j) mbar_drain(&fullV[j % kStages], (j / kStages) & 1);
    }
  } else if (warp >= 9) {
    // One warp per stream issues its MMAs.  The whole warp runs the loop and one elected lane issues: operands of
    // tcgen05.mma live in uniform registers, and in a branch on the lane every one of them is moved there for every
    // instruction (90 cycles an MMA for S, 300 for P V: three times the tensor pipe's own work).  One warp for both
    // streams, polling their barriers in turn, spent as long on the polls as on issuing.
    const int w = warp - 9, n = count(w);
    constexpr uint32_t idS = umma_idesc_bf16(kRows, kKv);
    constexpr uint32_t idO = umma_idesc_bf16(kRows, D) | (1u << 16);  // B is MN-major
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.status, kStatusAttnTimeout)) != 0;
    };
    auto issue_s = [&](int i) {
      const int t = tile(w, i), s = t % kStages;
      // the S buffer is free once P V of the tile two back has read P from it
      if (!wait(&fullK[s], (t / kStages) & 1) || (i >= 2 && !wait(&o_done[2 * w + (i & 1)], ((i >> 1) - 1) & 1)))
        return false;
      tc_fence_after();
      const uint64_t dq = umma_desc_sw128(smem_u32(sQ + (kPair ? w * C::kQ : 0)));
      const uint64_t dk = umma_desc_sw128(smem_u32(sK + s * C::kTile));
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)  // descriptors count addresses in 16 bytes
          umma_f16(tmem + 128 * w + 64 * (i & 1), dq + (kk >> 2) * (kRows * 8) + 2 * (kk & 3),
                   dk + (kk >> 2) * (C::kRegion / 16) + 2 * (kk & 3), idS, kk > 0 ? 1u : 0u);
        umma_commit(&s_done[2 * w + (i & 1)]);
        umma_commit(&emptyK[s]);
      }
      __syncwarp();
      return true;
    };
    bool ok = n > 0 && wait(q_ready, 0) && issue_s(0);
    bool issued = ok;
    for (int i = 0; i < n && ok; ++i) {
      if (i + 1 < n && !issue_s(i + 1)) {
        ok = false;
        break;
      }
      const int t = tile(w, i), s = t % kStages;
      if (!wait(&p_ready[2 * w + (i & 1)], (i >> 1) & 1) || !wait(&fullV[s], (t / kStages) & 1)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint64_t dv = desc_mn(smem_u32(sV + s * C::kTile), C::kRegion);
      if (elect_one_sync()) {
#pragma unroll
        for (int kk = 0; kk < kKv / 16; ++kk)
          umma_f16_ts(tmem + 256 + 128 * w, tmem + 128 * w + 64 * (i & 1) + 8 * kk, dv + kk * (16 * 128 / 16), idO,
                      (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&o_done[2 * w + (i & 1)]);
        umma_commit(&emptyV[s]);
      }
      __syncwarp();
    }
    if (!ok && issued) {  // what was issued completes before TMEM is freed
      if (elect_one_sync()) umma_commit(&drain[w]);
      __syncwarp();
      mbar_drain(&drain[w], 0);
    }
  } else {
    const int w = warp >> 2, t = threadIdx.x & (kRows - 1);
    const int r = it.y + (kPair ? w * kRows : 0) + t;
    const bool valid = r < rows;
    const bool any = __any_sync(0xffffffffu, valid);
    const int tok = div_g(a, valid ? r : 0);
    const long token = (long)gr.first * a.ql + tok;
    const int h = kh * G + (valid ? r : 0) - tok * G;
    // scores are scaled by |scale| inside the exponent; its sign goes into q, so that the largest product stays the
    // largest score
    const float scale = fmaxf(fabsf(a.scale_log2), 1e-30f);  // not 0: masked scores are -inf
    const uint32_t sign = a.scale_log2 < 0.f ? 0x80008000u : 0u;
    auto flip = [&](uint4 x) { return make_uint4(x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign); };
    if (kPair || w == 0) {  // this thread's q row, K-major with the 128-byte swizzle
      const uint4* src = reinterpret_cast<const uint4*>(a.q + token * a.q_stride + (long)h * D);
      uint8_t* dst = sQ + (kPair ? w * C::kQ : 0) + t * 128;
      uint4 x[D / 8];  // all of it requested before the first store
#pragma unroll
      for (int c = 0; c < D / 8; ++c) x[c] = __ldg(src + c);
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        *reinterpret_cast<uint4*>(dst + (c >> 3) * (kRows * 128) + (((c & 7) ^ (t & 7)) << 4)) =
            valid ? flip(x[c]) : make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const int limit =
        valid ? min(k1 - 1, seq_len(a, gr.first + tok / a.ql) - a.ql + tok % a.ql) : 0x7fffffff;  // padding: unmasked
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + 256 + 128 * w + lanes;
    float m = kNegBig, l = 0.f;  // m in the scaled log2 domain
    bool failed = false;
    const int n = count(w);
    for (int i = 0; i < n; ++i) {
      const uint32_t tS = tmem + 128 * w + 64 * (i & 1) + lanes;
      if (!mbar_wait(&s_done[2 * w + (i & 1)], (i >> 1) & 1, abort_flag, a.status, kStatusAttnTimeout)) failed = true;
      if (__any_sync(0xffffffffu, failed)) {
        failed = true;
        break;
      }
      tc_fence_after();
      const int kv0 = k0 + tile(w, i) * kKv;
      if (any) {  // a warp of padding rows only signals
        float v[4][16];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x16(tS + 16 * c, v[c]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 4; ++c) pin(v[c]);
        if (!__all_sync(0xffffffffu, kv0 + kKv - 1 <= limit)) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) v[c][e] = kv0 + 16 * c + e <= limit ? v[c][e] : -INFINITY;
        }
        float mc[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mc[c] = fmaxf(v[c][0], v[c][1]);
#pragma unroll
          for (int e = 2; e < 16; e += 2) mc[c] = max3(mc[c], v[c][e], v[c][e + 1]);
        }
        const float mx = fmaxf(max3(mc[0], mc[1], mc[2]), mc[3]);
        const float m_new = fmaxf(m, mx == -INFINITY ? kNegBig : mx * scale);
        const bool grow = m_new > m + kLazy || i == 0;
        const float alpha = grow ? exp2f(m - m_new) : 1.f;
        if (i > 0 && __any_sync(0xffffffffu, grow)) {
          const int j = i - 1;
          if (!mbar_wait(&o_done[2 * w + (j & 1)], (j >> 1) & 1, abort_flag, a.status, kStatusAttnTimeout))
            failed = true;
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            float o[16];
            tmem_ld_32x32b_x16(tO + c, o);
            tmem_wait_ld();
            pin(o);
            uint32_t u[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * alpha);
            tmem_st_x16(tO + c, u);
          }
        }
        if (grow) {
          l *= alpha;
          m = m_new;
        }
        const uint64_t sc2 = pack2(scale, scale), m2 = pack2(-m, -m);
        uint64_t sum[4] = {0, 0, 0, 0};
        // in steps over the whole tile, so that every step has 32 or 64 independent operations
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 16; e += 2) unpack2(fma2(pack2(v[c][e], v[c][e + 1]), sc2, m2), v[c][e], v[c][e + 1]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[c][e] = exp2f(v[c][e]);
          pin(v[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; c += 2) {  // 32 keys -> 16 columns of P
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 16; ++e)  // rounded by 2^-8 at most; l keeps the fp32 sum
            u[e] = pack_bf16x2(v[c + (e >> 3)][2 * (e & 7)], v[c + (e >> 3)][2 * (e & 7) + 1]);
          tmem_st_x16(tS + 8 * c, u);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 16; e += 2) sum[c] = add2(sum[c], pack2(v[c][e], v[c][e + 1]));
        float s0, s1;
        unpack2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), s0, s1);
        l += s0 + s1;
        tmem_wait_st();
      }
      if (kv0 + kKv > k1) {  // V rows behind the last key: whatever they hold must not meet p = 0
        const int tl = tile(w, i), s = tl % kStages;
        if (!mbar_wait(&fullV[s], (tl / kStages) & 1, abort_flag, a.status, kStatusAttnTimeout)) failed = true;
        for (int c = t; c < (kv0 + kKv - k1) * 8; c += kRows)
#pragma unroll
          for (int rg = 0; rg < D / 64; ++rg)
            reinterpret_cast<uint4*>(sV + s * C::kTile + rg * C::kRegion + (k1 - kv0) * 128)[c] = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[2 * w + (i & 1)]);
    }
    if (!failed && n > 0 &&
        !mbar_wait(&o_done[2 * w + ((n - 1) & 1)], ((n - 1) >> 1) & 1, abort_flag, a.status, kStatusAttnTimeout))
      failed = true;
    failed = __any_sync(0xffffffffu, failed);
    if (!failed && any) {
      tc_fence_after();
      const long part = kPair ? it.z : 2 * it.z + w;
      const long at = (part * a.B * a.ql + token) * a.nq + h;
      if (valid) a.part_ml[at] = make_float2(m, l);
#pragma unroll 1
      for (int c = 0; c < D; c += 16) {
        float o[16];
        if (n > 0) {
          tmem_ld_32x32b_x16(tO + c, o);
          tmem_wait_ld();
          pin(o);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = 0.f;
        }
        if (valid)
#pragma unroll
          for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4*>(a.part_o + at * D + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace tc

// Running sum over partial results of one row (a warp; lane `lane` holds dims lane * D / 32 ...).
template <int D>
struct RowSum {
  float M = kNegBig, L = 0.f, O[D / 32] = {};

  __device__ __forceinline__ void scale_to(float m) {
    const float m_new = fmaxf(M, m), f = exp2f(M - m_new);
    M = m_new;
    L *= f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) O[c] *= f;
  }
  // one part: O[D], m, l at p
  __device__ __forceinline__ void add(const float* p) {
    scale_to(p[D]);
    const float w = exp2f(p[D] - M);
    L += p[D + 1] * w;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) O[c] += p[lane_id() * (D / 32) + c] * w;
  }
  // n parts of the workspace, `step` rows apart, part s in lane s & 31
  __device__ __forceinline__ void add_parts(const Args& a, long at, long step, int n) {
    const int lane = lane_id();
    for (int s0 = 0; s0 < n; s0 += 32) {
      const int k = min(32, n - s0);
      const float2 ml = lane < k ? a.part_ml[at + (s0 + lane) * step] : make_float2(kNegBig, 0.f);
      scale_to(warp_max(ml.x));
      const float w = exp2f(ml.x - M);
      L += warp_sum(ml.y * w);
      const float* p = a.part_o + (at + s0 * step) * D + lane * (D / 32);
#pragma unroll 4
      for (int s = 0; s < k; ++s, p += step * D) {
        const float ws = __shfl_sync(0xffffffffu, w, s);
        if constexpr (D == 128) {
          const float4 v = *reinterpret_cast<const float4*>(p);
          O[0] += v.x * ws, O[1] += v.y * ws, O[2] += v.z * ws, O[3] += v.w * ws;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(p);
          O[0] += v.x * ws, O[1] += v.y * ws;
        }
      }
    }
  }
  __device__ __forceinline__ void store(const Args& a, long tok, int h) const {
    const float inv = L > 0.f ? 1.f / L : 0.f;  // a row that sees nothing gives zeros
    __nv_bfloat16* dst = a.out + tok * a.out_stride + h * D + lane_id() * (D / 32);
    if constexpr (D == 128)
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_bf16x2(O[0] * inv, O[1] * inv), pack_bf16x2(O[2] * inv, O[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(O[0] * inv, O[1] * inv);
  }
};

// Each sequence's own keys.  grid (B, KV heads x row chunks, page splits).
// kMerge: a dependent of the prefix kernel, the splits of a row one cluster; adds the prefix's parts and writes the
// result.  Otherwise it runs beside the prefix kernel, and its results are parts `first_part` ... of the workspace.
template <int D, int NT, bool kMerge>
__global__ void __launch_bounds__(kMaxWarps * 32)
    suffix_kernel(const __grid_constant__ CUtensorMap tm, const Args a, int row_chunks, int first_part) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ int abort_flag;
  if (threadIdx.x == 0) abort_flag = 0;
  __syncthreads();
  const int b = blockIdx.x, kh = blockIdx.y / row_chunks, r0 = blockIdx.y % row_chunks * (NT * 8);
  const int G = a.nq / a.nkv, rows = min(NT * 8, a.ql * G - r0);
  const int splits = gridDim.z, me = blockIdx.z, warps = blockDim.x / 32;
  const int2 sh = __ldg(a.seqs + b);
  const int len = seq_len(a, b);
  // this CTA's pages of [prefix, len)
  const int begin = min(sh.x, len), p0 = begin / PAGE, pages = (len + PAGE - 1) / PAGE - p0;
  const int per = (pages + splits - 1) / splits;
  const int k0 = max(begin, (p0 + me * per) * PAGE), k1 = min(len, (p0 + (me + 1) * per) * PAGE);
  float* res = stream<D, NT>(tm, a, smem, &abort_flag, a.table + (long)b * a.table_stride, kh, (long)b * a.ql, r0, rows,
                             min(k0, max(k1, 0)), k1, [&](int r) { return len - a.ql + div_g(a, r0 + r); });
  constexpr int RS = D + 2;
  const long step = (long)a.B * a.ql * a.nq;
  auto row_of = [&](int r, long& tok, int& h) {
    const int qi = div_g(a, r0 + r);
    tok = (long)b * a.ql + qi;
    h = kh * G + (r0 + r - qi * G);
  };
  if constexpr (kMerge) {
    cg::cluster_group cl = cg::this_cluster();
    if (splits > 1) cl.sync();
    griddep_wait();
    // one warp per row, the rows dealt over the CTAs of the cluster
    for (int r = me * warps + warp_id(); r < rows; r += splits * warps) {
      long tok;
      int h;
      row_of(r, tok, h);
      RowSum<D> sum;
      for (int s = 0; s < splits; ++s) sum.add((splits > 1 ? cl.map_shared_rank(res, s) : res) + r * RS);
      sum.add_parts(a, tok * a.nq + h, step, sh.y * a.parts);
      sum.store(a, tok, h);
    }
    if (splits > 1) cl.sync();  // the others may still read this CTA's result
  } else {
    for (int r = warp_id(); r < rows; r += warps) {
      long tok;
      int h;
      row_of(r, tok, h);
      const long at = (first_part + me) * step + tok * a.nq + h;
      const float* p = res + r * RS;
#pragma unroll
      for (int c = lane_id(); c < D; c += 32) a.part_o[at * D + c] = p[c];
      if (lane_id() == 0) a.part_ml[at] = make_float2(p[D], p[D + 1]);
    }
  }
}

// The sum of all parts, one warp per row: the prefix's, and `own` of each sequence from `first_part` on.
template <int D>
__global__ void __launch_bounds__(256) merge_kernel(const Args a, int first_part, int own) {
  const long row = (long)blockIdx.x * 8 + warp_id(), step = (long)a.B * a.ql * a.nq;
  if (row >= step) return;
  const long tok = row / a.nq;
  RowSum<D> sum;
  sum.add_parts(a, row, step, __ldg(a.seqs + tok / a.ql).y * a.parts);
  sum.add_parts(a, row + first_part * step, step, own);
  sum.store(a, tok, int(row - tok * a.nq));
}

// Raises a kernel's limit of dynamic shared memory once per device.
template <typename K>
void allow_smem(K* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (done.load(std::memory_order_acquire) >> dev & 1u) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  // all of an SM's memory as shared memory, also where one CTA of this kernel needs less: CTAs of another come beside it
  C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                      cudaSharedmemCarveoutMaxShared));
  done.fetch_or(uint64_t(1) << dev, std::memory_order_release);
}

template <int D, int NT>
void launch_prefix(const CUtensorMap& tm, const Args& a, int items, cudaStream_t stream) {
  constexpr int kWarps = 4;
  const int smem = stream_smem<D>(kWarps, NT * 8);
  static std::atomic<uint64_t> done{0};
  allow_smem(prefix_stream_kernel<D, NT>, smem, done);
  prefix_stream_kernel<D, NT><<<dim3(items, a.nkv), kWarps * 32, smem, stream>>>(tm, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <int D, bool kPair>
void launch_prefix_tc(const CUtensorMap& tm, const Args& a, int items, cudaStream_t stream) {
  constexpr int smem = tc::Cfg<D, kPair>::kSmem;
  static std::atomic<uint64_t> done{0};
  allow_smem(tc::prefix_tc_kernel<D, kPair>, smem, done);
  tc::prefix_tc_kernel<D, kPair><<<dim3(items, a.nkv), tc::kThreads, smem, stream>>>(tm, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <int D, int NT, bool kMerge>
void launch_suffix(const CUtensorMap& tm, const Args& a, int splits, int first_part, bool dependent, int sms,
                   cudaStream_t stream) {
  const int row_chunks = (a.ql * (a.nq / a.nkv) + NT * 8 - 1) / (NT * 8);
  // Warps per sequence, KV head and row chunk: as many as fill the SMs once.  Each warp costs its start and its share
  // of the merge, and its ring the place of another CTA, so where there are sequences enough one warp takes a whole one:
  // 256 sequences x 8 heads of 64 tokens take 14 us with one warp each, 26 with four; of 256 tokens 47 and 54.
  const long ctas = (long)a.B * a.nkv * row_chunks * splits;
  int warps = 1;
  while (warps * 2 <= kMaxWarps && ctas * warps * 2 <= (long)sms * kMaxWarps) warps *= 2;
  const int smem = stream_smem<D>(warps, std::min(NT * 8, a.ql * (a.nq / a.nkv)));
  static std::atomic<uint64_t> done{0};
  allow_smem(suffix_kernel<D, NT, kMerge>, stream_smem<D>(kMaxWarps, NT * 8), done);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.B, a.nkv * row_chunks, splits);
  cfg.blockDim = dim3(warps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (kMerge && splits > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = at[n].val.clusterDim.y = 1;
    at[n++].val.clusterDim.z = splits;
  }
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, suffix_kernel<D, NT, kMerge>, tm, a, row_chunks, first_part));
}

template <int D, bool kMerge>
void run_suffix(const CUtensorMap& tm, const Args& a, int splits, int first_part, bool dependent, int sms,
                cudaStream_t stream) {
  const int rows = a.ql * (a.nq / a.nkv);
  if (rows <= 8) launch_suffix<D, 1, kMerge>(tm, a, splits, first_part, dependent, sms, stream);
  else if (rows <= 16) launch_suffix<D, 2, kMerge>(tm, a, splits, first_part, dependent, sms, stream);
  else launch_suffix<D, 4, kMerge>(tm, a, splits, first_part, dependent, sms, stream);
}

// Streams of one device for the suffixes of groups of many rows.  They are this file's own: PyTorch hands its pool's
// streams to everybody, and a stream that is joined to a capture belongs to it until the capture ends, with whatever
// its other users launch on it meanwhile.  The mutex is held from the choice of a stream until the caller's stream has
// waited for it, so no other thread brings it into a capture in between.
struct SideStreams {
  static constexpr size_t kMost = 32;  // captures under way may need more
  struct Side {
    cudaStream_t stream, caller;
  };
  std::mutex mutex;
  std::vector<Side> all;
  size_t next = 0;

  // For a capturing caller a stream of its capture (it is there from an earlier call) or a free one, otherwise a free
  // one; each caller's own where it has one, so that callers do not wait for one another.
  c10::cuda::CUDAStream take(const c10::cuda::CUDAStream& caller) {
    auto info = [](cudaStream_t s, unsigned long long& id) {
      cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
      id = 0;
      C10_CUDA_CHECK(cudaStreamGetCaptureInfo(s, &st, &id));
      return st;
    };
    unsigned long long capture = 0, id = 0;
    const bool capturing = info(caller.stream(), capture) == cudaStreamCaptureStatusActive;
    size_t found = all.size();
    for (size_t k = 0; k < all.size(); ++k) {
      const size_t i = (next + k) % all.size();
      const cudaStreamCaptureStatus st = info(all[i].stream, id);
      const bool fits = st == cudaStreamCaptureStatusNone ||
                        (capturing && st == cudaStreamCaptureStatusActive && id == capture);
      if (!fits) continue;
      if (all[i].caller == caller.stream()) return c10::cuda::getStreamFromExternal(all[i].stream, caller.device_index());
      if (found == all.size() && st == cudaStreamCaptureStatusNone) found = i;
    }
    if (all.size() < kMost || found == all.size()) {
      // not an operation of the capture, but one that its mode may forbid
      const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
      cudaStream_t s = nullptr;
      C10_CUDA_CHECK(cudaStreamCreateWithFlags(&s, cudaStreamNonBlocking));
      found = all.size();
      all.push_back({s, nullptr});
    }
    next = (found + 1) % all.size();
    all[found].caller = caller.stream();
    return c10::cuda::getStreamFromExternal(all[found].stream, caller.device_index());
  }
};
// Never destroyed: streams outlive the CUDA context's end at exit.
SideStreams& side_streams(int device) {
  static SideStreams* const per_device = new SideStreams[64];
  return per_device[device];
}

template <int D>
void run(const CUtensorMap& tm, const Args& a, int items, int tile_rows, int prefix_parts, int suffix_splits, int sms,
         c10::cuda::CUDAStream stream) {
  if (tile_rows <= 128 || items == 0) {
    if (items > 0) {
      if (tile_rows == 8) launch_prefix<D, 1>(tm, a, items, stream);
      else if (tile_rows == 16) launch_prefix<D, 2>(tm, a, items, stream);
      else if (tile_rows == 32) launch_prefix<D, 4>(tm, a, items, stream);
      else launch_prefix_tc<D, false>(tm, a, items, stream);
    }
    run_suffix<D, true>(tm, a, suffix_splits, 0, items > 0, sms, stream);
    return;
  }
  // The prefix on the tensor cores and the suffixes from HBM run side by side on two streams.  (As a dependent launch
  // the suffix kernel starts as early, but its wait for the prefix kernel does not end while its CTAs load: 119 us for
  // 256 sequences behind 8,192 tokens, 108 this way; 120 and 103 for 16 groups of 8 that verify four tokens.  With one
  // row tile the prefix is short, and the third launch costs more than it gives: 28 us and 30.)
  SideStreams& streams = side_streams(stream.device_index());
  const std::lock_guard<std::mutex> lock(streams.mutex);
  const c10::cuda::CUDAStream side = streams.take(stream);
  at::cuda::CUDAEvent fork, join;
  fork.record(stream);
  fork.block(side);
  launch_prefix_tc<D, true>(tm, a, items, stream);
  run_suffix<D, false>(tm, a, suffix_splits, prefix_parts, false, sms, side);
  join.record(side);
  join.block(stream);
  const long rows = (long)a.B * a.ql * a.nq;
  merge_kernel<D><<<unsigned((rows + 7) / 8), 256, 0, stream>>>(a, prefix_parts, suffix_splits);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace shared_prefix

// The messages are single literals: formatting one needs iostreams, which crash where the extension was linked to a
// libstdc++ of its own.
#define SP_CHECK(cond, msg) TORCH_CHECK(cond, "shared_prefix_attention: " msg)

void shared_prefix_attention(const torch::Tensor& q, const torch::Tensor& kv_cache, int64_t layer,
                             const torch::Tensor& block_table, const torch::Tensor& seq_lens, torch::Tensor& out,
                             const torch::Tensor& items, const torch::Tensor& groups, const torch::Tensor& seqs,
                             int64_t q_len, int64_t tile_rows, int64_t prefix_splits, int64_t suffix_splits,
                             double scale) {
  using namespace shared_prefix;
  SP_CHECK(kv_cache.scalar_type() == at::kBFloat16 && kv_cache.dim() == 6 && kv_cache.is_contiguous() &&
                  kv_cache.size(2) == 2 && kv_cache.size(4) == PAGE &&
                  (kv_cache.size(5) == 128 || kv_cache.size(5) == 64),
              "kv_cache must be contiguous bf16 [L, NB, 2, KVH, 16, 128 or 64]");
  const int64_t D = kv_cache.size(5), nkv = kv_cache.size(3);
  SP_CHECK(layer >= 0 && layer < kv_cache.size(0), "layer is outside the cache");
  SP_CHECK(q.scalar_type() == at::kBFloat16 && q.dim() == 3 && q.size(2) == D && q.stride(2) == 1 &&
                  q.stride(1) == D && q.stride(0) % 8 == 0 && (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15u) == 0,
              "q must be bf16 [B * q_len, heads, head_dim] with contiguous token rows on 16-byte boundaries");
  SP_CHECK(out.scalar_type() == at::kBFloat16 && out.sizes() == q.sizes() && out.stride(2) == 1 &&
                  out.stride(1) == D && out.stride(0) % 8 == 0 && out.stride(0) >= out.size(1) * D &&
                  (reinterpret_cast<uintptr_t>(out.data_ptr()) & 15u) == 0,
              "out must be like q");
  SP_CHECK(nkv > 0 && q.size(1) > 0 && q.size(1) % nkv == 0, "q heads must be a multiple of KV heads");
  const int64_t B = seq_lens.size(0);
  SP_CHECK(seq_lens.scalar_type() == at::kInt && seq_lens.dim() == 1 && seq_lens.is_contiguous(), "seq_lens must be contiguous int32 [B]");
  SP_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B &&
                  (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              "block_table must be int32 [B, W] with contiguous rows");
  SP_CHECK(q_len >= 1 && q.size(0) == B * q_len, "q must have batch x q_len rows");
  SP_CHECK(seqs.scalar_type() == at::kInt && seqs.dim() == 2 && seqs.size(1) == 2 && seqs.is_contiguous() &&
               seqs.size(0) == B, "the plan is for another number of sequences");
  SP_CHECK(items.scalar_type() == at::kInt && items.dim() == 2 && items.size(1) == 4 && items.is_contiguous() &&
                  groups.scalar_type() == at::kInt && groups.dim() == 2 && groups.size(1) == 4 &&
                  groups.is_contiguous(),
              "items and groups must be a plan's");
  SP_CHECK(tile_rows == 8 || tile_rows == 16 || tile_rows == 32 || tile_rows == 128 || tile_rows == 256, "unknown row tile");
  SP_CHECK(suffix_splits == 1 || suffix_splits == 2 || suffix_splits == 4 || suffix_splits == 8, "suffix_splits must be 1, 2, 4 or 8");
  const uint64_t rows = (uint64_t)kv_cache.size(1) * 2 * nkv * PAGE;
  SP_CHECK(rows < (1ull << 31), "kv_cache has too many rows per layer for 32-bit tile coordinates");
  // the suffix grid's second dimension: KV heads x chunks of up to 32 query rows
  SP_CHECK(nkv * ((q_len * (q.size(1) / nkv) + 31) / 32) <= 65535, "too many heads x query rows");
  SP_CHECK(std::isfinite(float(scale * 1.4426950408889634)), "scale must be a finite number");
  SP_CHECK(q.is_cuda(), "tensors must be on a CUDA device");
  for (const torch::Tensor* t : {&kv_cache, &block_table, &seq_lens, &static_cast<const torch::Tensor&>(out), &items,
                                 &groups, &seqs})
    SP_CHECK(t->device() == q.device(), "tensors must be on one device");
  if (B == 0) return;
  const at::cuda::CUDAGuard guard(q.device());
  const c10::cuda::CUDAStream stream = at::cuda::getCurrentCUDAStream();
  const int64_t T = B * q_len, nq = q.size(1);
  Args a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.q_stride = q.stride(0);
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.out_stride = out.stride(0);
  a.table = block_table.data_ptr<int>();
  a.table_stride = block_table.stride(0);
  a.W = int(block_table.size(1));
  a.lens = seq_lens.data_ptr<int>();
  a.items = reinterpret_cast<const int4*>(items.data_ptr<int>());
  a.groups = reinterpret_cast<const Group*>(groups.data_ptr<int>());
  a.seqs = reinterpret_cast<const int2*>(seqs.data_ptr<int>());
  a.B = int(B);
  a.nq = int(nq);
  a.nkv = int(nkv);
  a.ql = int(q_len);
  const int64_t G = nq / nkv;
  SP_CHECK(T * G * G < (1ll << 32), "too many query rows");
  a.per_g = G > 1 ? uint32_t(((1ull << 32) + G - 1) / G) : 0;
  a.NB = int(kv_cache.size(1));
  a.scale_log2 = float(scale * 1.4426950408889634);
  a.status = status_word(q.get_device());
  a.parts = tile_rows == 128 ? 2 : 1;
  // partial results: every (part, row) that is read has been written, the prefix's by the plan's items
  const int64_t prefix_parts = prefix_splits * a.parts, parts = prefix_parts + (tile_rows == 256 ? suffix_splits : 0);
  auto ws = torch::empty({parts * T * nq * (D + 2)}, q.options().dtype(at::kFloat));
  a.part_o = ws.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part_o + parts * T * nq * D);
  const auto* base = reinterpret_cast<const __nv_bfloat16*>(kv_cache.data_ptr()) + layer * kv_cache.stride(0);
  const CUtensorMap tm = make_tmap_bf16_2d(base, D, rows, D * 2, 64, PAGE);
  const int sms = num_sms(q.get_device());
  if (D == 128) run<128>(tm, a, int(items.size(0)), int(tile_rows), int(prefix_parts), int(suffix_splits), sms, stream);
  else run<64>(tm, a, int(items.size(0)), int(tile_rows), int(prefix_parts), int(suffix_splits), sms, stream);
}

}  // namespace bloom

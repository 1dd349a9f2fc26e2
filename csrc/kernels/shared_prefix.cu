// Decode / verify attention of a batch whose sequences share long prefixes (many completions of one prompt, requests
// behind one system prompt).
//
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q.k_j
//
// splits exactly at any key: with (o1, m1, l1) over the prefix and (o2, m2, l2) over a row's own pages,
// o = (o1 2^(m1-M) + o2 2^(m2-M)) / (l1 2^(m1-M) + l2 2^(m2-M)).  So the prefix of a group is read once for all of its
// members, as a product with members x q_len x (q heads per KV head) rows, and only the rest is read per sequence.
//
// Two kernels.  The prefix kernel (work items: a tile of a group's rows x a range of the prefix) leaves partial sums in
// fp32.  The suffix kernel is one CTA (or a cluster over the pages) per sequence, KV head and chunk of rows; it is
// launched as a dependent of the prefix kernel, runs its own pages beside it, and waits for it only before it adds the
// partial sums and writes the result: two launches, memory and tensor work overlapped.
//
// Slots behind a sequence's last token may hold anything (NaN too): scores there are replaced, and V rows there are
// zeroed in shared memory.  A block id outside the cache sets kStatusBadArgument and page 0 is read instead.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <torch/extension.h>

#include <algorithm>

#include "bloom/common.cuh"
#include "bloom/ops_share.h"
#include "bloom/tma_host.h"

namespace cg = cooperative_groups;

namespace bloom {
namespace shared_prefix {

constexpr int PAGE = 16;
constexpr float kNegBig = -1e30f;
constexpr int kWarps = 4, kStages = 3;  // streaming kernels: warps and ring depth per warp

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
  const int* seq_group;    // [B]
  float* part_o;           // [splits, B * ql, nq, D]
  float2* part_ml;         // [splits, B * ql, nq]
  int B, nq, nkv, ql, NB;
  int parts;               // partial sums per prefix split: 2 where the two streams of a CTA leave one each
  float scale_log2;
  int* status;
};

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
  unsigned long long best = 0;
  for (int i = lane_id(); i < g.members; i += 32) {
    const int n = min(seq_len(a, g.first + i), g.prefix);
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
constexpr int stage_bytes() { return 2 * PAGE * D * 2; }
template <int D, int MT>
constexpr int stream_smem() {
  constexpr int ring = kWarps * kStages * stage_bytes<D>(), merge = kWarps * MT * 16 * (D + 2) * 4;
  return (ring > merge ? ring : merge) + kWarps * kStages * 8 + 1024;
}

// Streams keys [k_begin, k_end) of one KV head past up to MT * 16 packed query rows (row r: token q0 + r / G, q head
// kh * G + r % G; limit(r): the last key that it sees) and leaves, in shared memory, row r's O[D], m, l at
// merged + r * (D + 2).  Each warp streams every kWarps-th page through its own TMA ring; the rows are the M dimension
// of m16n8k16 MMAs, so a page is read once for all of them.
template <int D, int MT, typename Limit>
__device__ float* stream(const CUtensorMap& tm, const Args& a, uint8_t* smem, int* abort_flag, const int* row, int kh,
                         long q0, int r0, int rows, int k_begin, int k_end, Limit&& limit_of) {
  constexpr int kStage = stage_bytes<D>(), kPageB = PAGE * D * 2, RS = D + 2;
  constexpr int ring = kWarps * kStages * kStage, merge = kWarps * MT * 16 * RS * 4;
  const int warp = warp_id(), lane = lane_id(), g = lane >> 2, t4 = lane & 3;
  const int G = a.nq / a.nkv;
  uint8_t* wsm = smem + warp * kStages * kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (ring > merge ? ring : merge)) + warp * kStages;
  const int p0 = k_begin / PAGE, p1 = k_end > k_begin ? (k_end + PAGE - 1) / PAGE : p0;
  const int first = p0 + warp;
  const int my_n = p1 > first ? (p1 - first + kWarps - 1) / kWarps : 0;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bars[s], 1);
    fence_barrier_init();
  }
  __syncthreads();
  auto issue = [&](int i) {
    const int s = i % kStages;
    const int blk = block_id(a, row, first + i * kWarps);
    const int rowK = (blk * 2 * a.nkv + kh) * PAGE, rowV = ((blk * 2 + 1) * a.nkv + kh) * PAGE;
    uint8_t* st = wsm + s * kStage;
    mbar_arrive_expect_tx(&bars[s], kStage);
    tma_load_2d(st, &tm, &bars[s], 0, rowK);
    if constexpr (D == 128) tma_load_2d(st + 2048, &tm, &bars[s], 64, rowK);
    tma_load_2d(st + kPageB, &tm, &bars[s], 0, rowV);
    if constexpr (D == 128) tma_load_2d(st + kPageB + 2048, &tm, &bars[s], 64, rowV);
  };
  if (lane == 0)
    for (int i = 0; i < kStages && i < my_n; ++i) issue(i);

  uint32_t qf[MT][D / 16][4];
  int limit[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      const int r = mt * 16 + g + 8 * hr;
      const __nv_bfloat16* qrow = nullptr;
      limit[mt][hr] = -1;
      if (r < rows) {
        qrow = a.q + (q0 + (r0 + r) / G) * a.q_stride + (kh * G + (r0 + r) % G) * D;
        limit[mt][hr] = min(limit_of(r), k_end - 1);
      }
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int d = ks * 16 + 2 * t4;
        qf[mt][ks][hr] = qrow ? *reinterpret_cast<const uint32_t*>(qrow + d) : 0u;
        qf[mt][ks][hr + 2] = qrow ? *reinterpret_cast<const uint32_t*>(qrow + d + 8) : 0u;
      }
    }
  float m_run[MT][2], l_run[MT][2], o[MT][D / 8][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m_run[mt][0] = m_run[mt][1] = kNegBig;
    l_run[mt][0] = l_run[mt][1] = 0.f;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[mt][n][0] = o[mt][n][1] = o[mt][n][2] = o[mt][n][3] = 0.f;
  }
  int i = 0;
  for (; i < my_n; ++i) {
    const int s = i % kStages;
    if (!mbar_wait(&bars[s], (i / kStages) & 1, abort_flag, a.status, kStatusAttnTimeout)) break;
    const uint32_t sK = smem_u32(wsm + s * kStage), sV = sK + kPageB;
    const int tok0 = (first + i * kWarps) * PAGE;
    if (tok0 + PAGE > k_end) {  // V rows behind the last key: whatever they hold must not meet p = 0
      for (int c = lane; c < PAGE * D / 8; c += 32) {
        const int tok = c & 15, d = (c >> 4) * 8;
        if (tok0 + tok >= k_end)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(page_addr(sV, tok, d)), "r"(0) : "memory");
      }
      __syncwarp();
    }
    float sc[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) sc[mt][nt][0] = sc[mt][nt][1] = sc[mt][nt][2] = sc[mt][nt][3] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        uint32_t b0, b1, b2, b3;
        ldsm_x4(page_addr(sK, 8 * nt + (lane & 7), 32 * j + 8 * (lane >> 3)), b0, b1, b2, b3);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma_bf16_16816(sc[mt][nt], qf[mt][2 * j], b0, b1);
          mma_bf16_16816(sc[mt][nt], qf[mt][2 * j + 1], b2, b3);
        }
      }
    uint32_t pa[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {
        float x[4], mx = kNegBig;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int idx = tok0 + 8 * nt + 2 * t4 + e;
            const bool sees = idx >= k_begin && idx <= limit[mt][hr];
            const float v = sees ? sc[mt][nt][2 * hr + e] * a.scale_log2 : -INFINITY;
            x[nt * 2 + e] = v;
            mx = fmaxf(mx, v);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run[mt][hr], mx);
        const float alpha = exp2f(m_run[mt][hr] - m_new);
        m_run[mt][hr] = m_new;
        float ps = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[k] = exp2f(x[k] - m_new);
          ps += x[k];
        }
        l_run[mt][hr] = l_run[mt][hr] * alpha + ps;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[mt][n][2 * hr] *= alpha;
          o[mt][n][2 * hr + 1] *= alpha;
        }
        // P is rounded to bf16 (2^-8 relative at most) for the tensor cores; l keeps the fp32 sum
        pa[mt][hr] = pack_bf16x2(x[0], x[1]);
        pa[mt][hr + 2] = pack_bf16x2(x[2], x[3]);
      }
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      uint32_t b0, b1, b2, b3;
      ldsm_x4_t(page_addr(sV, (lane & 7) + 8 * ((lane >> 3) & 1), 16 * j + 8 * (lane >> 4)), b0, b1, b2, b3);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mma_bf16_16816(o[mt][2 * j], pa[mt], b0, b1);
        mma_bf16_16816(o[mt][2 * j + 1], pa[mt], b2, b3);
      }
    }
    __syncwarp();
    if (lane == 0 && i + kStages < my_n) {
      fence_proxy_async();
      issue(i + kStages);
    }
  }
  if (i < my_n && lane == 0)  // gave up: the loads in flight must land before the shared memory is reused
    for (int k = i; k < my_n && k < i + kStages; ++k) mbar_drain(&bars[k % kStages], (k / kStages) & 1);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      float l = l_run[mt][hr];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      l_run[mt][hr] = l;
    }
  __syncthreads();
  // the warps' results into the shared memory of the rings, then summed into warp 0's place
  float* cm = reinterpret_cast<float*>(smem);
  float* wbuf = cm + warp * (MT * 16 * RS);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {
      const int r = mt * 16 + g + 8 * hr;
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2*>(wbuf + r * RS + 8 * n + 2 * t4) = make_float2(o[mt][n][2 * hr], o[mt][n][2 * hr + 1]);
      if (t4 == 0) *reinterpret_cast<float2*>(wbuf + r * RS + D) = make_float2(m_run[mt][hr], l_run[mt][hr]);
    }
  __syncthreads();
  // one warp per row: every lane reads the row's (m, l) of all warps before any lane writes the sums back
  for (int r = warp; r < rows; r += kWarps) {
    float m[kWarps], M = kNegBig, L = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 ml = *reinterpret_cast<const float2*>(cm + (w * MT * 16 + r) * RS + D);
      m[w] = ml.x;
      M = fmaxf(M, ml.x);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      m[w] = exp2f(m[w] - M);
      L += cm[(w * MT * 16 + r) * RS + D + 1] * m[w];
    }
    __syncwarp();
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float O = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) O += cm[(w * MT * 16 + r) * RS + c * 32 + lane] * m[w];
      cm[r * RS + c * 32 + lane] = O;
    }
    if (lane == 0) *reinterpret_cast<float2*>(cm + r * RS + D) = make_float2(M, L);
  }
  __syncthreads();
  return cm;
}

// Prefix work of groups with few rows: the keys stream past at most MT * 16 of them.  grid (items, KV heads).
template <int D, int MT>
__global__ void __launch_bounds__(kWarps * 32)
    prefix_stream_kernel(const __grid_constant__ CUtensorMap tm, const Args a) {
  griddep_launch_dependents();
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ int abort_flag;
  if (threadIdx.x == 0) abort_flag = 0;
  const int4 it = a.items[blockIdx.x];
  const Group gr = a.groups[it.x];
  const int kh = blockIdx.y, G = a.nq / a.nkv;
  const int2 hold = prefix_holder(a, gr);
  const int k0 = min(it.z * gr.chunk, hold.y), k1 = min(k0 + gr.chunk, hold.y);
  const int rows = min(MT * 16, gr.members * a.ql * G - it.y);
  const long q0 = (long)gr.first * a.ql;
  const float* res = stream<D, MT>(tm, a, smem, &abort_flag, a.table + hold.x * a.table_stride, kh, q0, it.y, rows, k0,
                                   k1, [&](int r) {
                                     const int tok = (it.y + r) / G;
                                     return seq_len(a, gr.first + tok / a.ql) - a.ql + tok % a.ql;
                                   });
  constexpr int RS = D + 2;
  for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kWarps * 32) {
    const int r = idx / (D / 4), d = idx % (D / 4) * 4;
    const long at = ((long)it.z * a.B * a.ql + q0 + (it.y + r) / G) * a.nq + kh * G + (it.y + r) % G;
    const float* p = res + r * RS + d;
    *reinterpret_cast<float4*>(a.part_o + at * D + d) = make_float4(p[0], p[1], p[2], p[3]);
    if (d == 0) a.part_ml[at] = make_float2(res[r * RS + D], res[r * RS + D + 1]);
  }
}

// ---------------------------------------------------------------- prefix on tcgen05
// Groups with more rows than a streaming CTA holds: S = Q K^T and O += P V on the 5th-generation tensor cores, with
// 128 rows per softmax warpgroup, one thread per row (no exchange between threads).  A CTA runs two such streams that
// take turns on the tensor pipe, one stream's softmax under the other's MMAs:
//   pair   (256-row items)  two row tiles over the same K / V tiles, so each K / V tile serves 256 rows
//   single (128-row items)  one row tile, the streams take alternate K / V tiles and leave one partial sum each
// TMEM: S0, S1, O0, O1 of 128 columns; P (bf16, two keys per column) is written over the first half of its S and
// read from there as the A operand, so it never goes through shared memory.  S(i + 1) of a stream is issued only after
// its P V(i) has completed, which also makes O safe to rescale when S(i + 1) is seen.  The running max is lazy: O is
// rescaled only when a row's max grows by more than 2^8.
// Warps 0-7 softmax and epilogue, warp 8 TMA producer and TMEM owner, warp 9 issues the MMAs of both streams from an
// event loop over their barriers.
namespace tc {

constexpr int kRows = 128, kKv = 128;
constexpr int kThreads = 256 + 64;
constexpr int kTmemCols = 512;
constexpr float kLazy = 8.f;  // log2 units

template <int D>
struct Cfg {
  static constexpr int kRegion = kKv * 128;       // 64 dims of a K or V tile: 128 token rows of 128 bytes
  static constexpr int kTile = kKv * D * 2;
  static constexpr int kQ = kRows * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;  // of the K ring and of the V ring
  static constexpr int kSmem = 2 * kQ + 2 * kStages * kTile + 256 + 1024;
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
  griddep_launch_dependents();
  using C = Cfg<D>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = smem + 2 * C::kQ;
  uint8_t* sV = sK + kStages * C::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kStages * C::kTile);
  uint64_t *fullK = bars, *emptyK = bars + 4, *fullV = bars + 8, *emptyV = bars + 12;
  uint64_t *s_done = bars + 16, *p_ready = bars + 18, *o_done = bars + 20, *q_ready = bars + 22, *drain = bars + 23;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
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
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_done[w], 1);
      mbar_init(&p_ready[w], 4);
      mbar_init(&o_done[w], 1);
    }
    mbar_init(q_ready, kPair ? 8 : 4);
    mbar_init(drain, 1);
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
  const uint32_t tmem = *tmem_slot;  // S_w at 128 w, O_w at 256 + 128 w

  if (warp == 8) {
    if (lane == 0) {
      const int n_pages = (k1 + PAGE - 1) / PAGE;
      auto load = [&](int t, uint8_t* dst, uint64_t* bar, int kv) {
        int ids[kKv / PAGE];
#pragma unroll
        for (int p = 0; p < kKv / PAGE; ++p) {
          const int page = k0 / PAGE + t * (kKv / PAGE) + p;
          ids[p] = block_id(a, table, page < n_pages ? page : k0 / PAGE);  // behind the end: any page, it is masked
        }
        mbar_arrive_expect_tx(bar, C::kTile);
#pragma unroll
        for (int p = 0; p < kKv / PAGE; ++p) {
          const int row = ((ids[p] * 2 + kv) * a.nkv + kh) * PAGE;
#pragma unroll
          for (int r = 0; r < D / 64; ++r) tma_load_2d(dst + r * C::kRegion + p * 2048, &tm, bar, 64 * r, row);
        }
      };
      int nK = 0, nV = 0;
      bool ok = true;
      uint64_t t_prog = globaltimer_ns();
      uint32_t spins = 0;
      while (ok && (nK < n_kt || nV < n_kt)) {  // the rings advance on their own; V never runs ahead of K
        bool progressed = false;
        if (nK < n_kt && mbar_test(&emptyK[nK % kStages], ((nK / kStages) & 1) ^ 1u)) {
          load(nK, sK + nK % kStages * C::kTile, &fullK[nK % kStages], 0);
          ++nK;
          progressed = true;
        }
        if (nV < nK && mbar_test(&emptyV[nV % kStages], ((nV / kStages) & 1) ^ 1u)) {
          load(nV, sV + nV % kStages * C::kTile, &fullV[nV % kStages], 1);
          ++nV;
          progressed = true;
        }
        if (progressed) {
          t_prog = globaltimer_ns();
        } else if ((++spins & 31u) == 0) {
          if (*abort_flag) {
            ok = false;
          } else if (globaltimer_ns() - t_prog > kLocalWaitTimeoutNs) {
            *abort_flag = 1;
            atomicOr(a.status, kStatusAttnTimeout);
            ok = false;
          }
        }
      }
      if (!ok) {  // the loads in flight land before the block leaves (bounded)
        for (int j = max(0, nK - kStages); j < nK; ++j) mbar_drain(&fullK[j % kStages], (j / kStages) & 1);
        for (int j = max(0, nV - kStages); j < nV; ++j) mbar_drain(&fullV[j % kStages], (j / kStages) & 1);
      }
    }
  } else if (warp == 9) {
    if (lane == 0 && n_kt > 0) {
      constexpr uint32_t idS = umma_idesc_bf16(kRows, kKv);
      constexpr uint32_t idO = umma_idesc_bf16(kRows, D) | (1u << 16);  // B is MN-major
      bool ok = mbar_wait(q_ready, 0, abort_flag, a.status, kStatusAttnTimeout), issued = false;
      auto issue_s = [&](int w, int t) {
        tc_fence_after();
        const int s = t % kStages;
        const uint32_t kb = smem_u32(sK + s * C::kTile), qb = smem_u32(sQ + (kPair ? w * C::kQ : 0));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          umma_f16(tmem + 128 * w, umma_desc_sw128(qb + (kk >> 2) * (kRows * 128)) + 2 * (kk & 3),
                   umma_desc_sw128(kb + (kk >> 2) * C::kRegion) + 2 * (kk & 3), idS, kk > 0 ? 1u : 0u);
        umma_commit(&s_done[w]);
        umma_commit(&emptyK[s]);
        issued = true;
      };
      // per stream: the tile in work, and whether its P V has been issued
      int i[2] = {0, 0};
      bool pv[2] = {false, false};
      int left = 0;
      for (int w = 0; w < 2 && ok; ++w)
        if (count(w) > 0) {
          ++left;
          const int t = tile(w, 0);
          ok = mbar_wait(&fullK[t % kStages], (t / kStages) & 1, abort_flag, a.status, kStatusAttnTimeout);
          if (ok) issue_s(w, t);
        }
      uint64_t t_prog = globaltimer_ns();
      uint32_t spins = 0;
      while (ok && left > 0) {
        bool progressed = false;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (i[w] >= count(w)) continue;
          if (!pv[w]) {
            const int t = tile(w, i[w]), s = t % kStages;
            if (!mbar_test(&p_ready[w], i[w] & 1) || !mbar_test(&fullV[s], (t / kStages) & 1)) continue;
            tc_fence_after();
            const uint32_t vb = smem_u32(sV + s * C::kTile);
#pragma unroll
            for (int kk = 0; kk < kKv / 16; ++kk)
              umma_f16_ts(tmem + 256 + 128 * w, tmem + 128 * w + 8 * kk, desc_mn(vb + kk * 16 * 128, C::kRegion), idO,
                          (i[w] > 0 || kk > 0) ? 1u : 0u);
            umma_commit(&o_done[w]);
            umma_commit(&emptyV[s]);
            pv[w] = true;
            if (i[w] + 1 == count(w)) ++i[w], --left;  // the last one: the softmax warps wait for it
          } else {
            const int t = tile(w, i[w] + 1);
            if (!mbar_test(&o_done[w], i[w] & 1) || !mbar_test(&fullK[t % kStages], (t / kStages) & 1)) continue;
            issue_s(w, t);
            ++i[w];
            pv[w] = false;
          }
          progressed = true;
        }
        if (progressed) {
          t_prog = globaltimer_ns();
        } else if ((++spins & 31u) == 0) {
          if (*abort_flag) {
            ok = false;
          } else if (globaltimer_ns() - t_prog > kLocalWaitTimeoutNs) {
            *abort_flag = 1;
            atomicOr(a.status, kStatusAttnTimeout);
            ok = false;
          }
        }
      }
      if (!ok && issued) {  // what was issued completes before TMEM is freed
        umma_commit(drain);
        mbar_drain(drain, 0);
      }
    }
  } else {
    const int w = warp >> 2, t = threadIdx.x & (kRows - 1);
    const int r = it.y + (kPair ? w * kRows : 0) + t;
    const bool valid = r < rows;
    const bool any = __any_sync(0xffffffffu, valid);
    const int tok = (valid ? r : 0) / G;
    const long token = (long)gr.first * a.ql + tok;
    const int h = kh * G + (valid ? r : 0) % G;
    if (kPair || w == 0) {  // this thread's q row, K-major with the 128-byte swizzle
      const uint4* src = reinterpret_cast<const uint4*>(a.q + token * a.q_stride + (long)h * D);
      uint8_t* dst = sQ + (kPair ? w * C::kQ : 0) + t * 128;
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        *reinterpret_cast<uint4*>(dst + (c >> 3) * (kRows * 128) + (((c & 7) ^ (t & 7)) << 4)) =
            valid ? src[c] : make_uint4(0, 0, 0, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
    }
    const int limit =
        valid ? min(k1 - 1, seq_len(a, gr.first + tok / a.ql) - a.ql + tok % a.ql) : 0x7fffffff;  // padding: unmasked
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + 128 * w + lanes, tO = tmem + 256 + 128 * w + lanes;
    float m = kNegBig, l = 0.f;
    bool failed = false;
    const int n = count(w);
    for (int i = 0; i < n; ++i) {
      if (!mbar_wait(&s_done[w], i & 1, abort_flag, a.status, kStatusAttnTimeout)) failed = true;
      if (__any_sync(0xffffffffu, failed)) {
        failed = true;
        break;
      }
      tc_fence_after();
      const int kv0 = k0 + tile(w, i) * kKv;
      if (any) {  // a warp of padding rows only signals
        float v[8][16];
#pragma unroll
        for (int c = 0; c < 8; ++c) tmem_ld_32x32b_x16(tS + 16 * c, v[c]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 8; ++c) pin(v[c]);
        float mx = kNegBig;
        if (__all_sync(0xffffffffu, kv0 + kKv - 1 <= limit)) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              v[c][e] *= a.scale_log2;
              mx = fmaxf(mx, v[c][e]);
            }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              v[c][e] = kv0 + 16 * c + e <= limit ? v[c][e] * a.scale_log2 : -INFINITY;
              mx = fmaxf(mx, v[c][e]);
            }
        }
        const float m_new = fmaxf(m, mx);
        const bool grow = m_new > m + kLazy || i == 0;
        const float alpha = grow ? exp2f(m - m_new) : 1.f;
        if (i > 0 && __any_sync(0xffffffffu, grow)) {
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
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // 32 keys -> 16 columns of P
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p0 = exp2f(v[2 * c + (e >> 3)][(2 * e) & 15] - m);
            const float p1 = exp2f(v[2 * c + (e >> 3)][(2 * e + 1) & 15] - m);
            sum[e & 3] += p0 + p1;
            u[e] = pack_bf16x2(p0, p1);  // rounded by 2^-8 at most; l keeps the fp32 sum
          }
          tmem_st_x16(tS + 16 * c, u);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
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
      if (lane == 0) mbar_arrive(&p_ready[w]);
    }
    if (!failed && n > 0 && !mbar_wait(&o_done[w], (n - 1) & 1, abort_flag, a.status, kStatusAttnTimeout)) failed = true;
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

// Each sequence's own keys, then the sum with the prefix.  grid (B, KV heads x row chunks, page splits), the splits of
// a row one cluster.
template <int D, int MT>
__global__ void __launch_bounds__(kWarps * 32)
    suffix_kernel(const __grid_constant__ CUtensorMap tm, const Args a, int row_chunks) {
  extern __shared__ uint8_t raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  __shared__ int abort_flag;
  if (threadIdx.x == 0) abort_flag = 0;
  const int b = blockIdx.x, kh = blockIdx.y / row_chunks, r0 = blockIdx.y % row_chunks * (MT * 16);
  const int G = a.nq / a.nkv, rows = min(MT * 16, a.ql * G - r0);
  const int splits = gridDim.z, me = blockIdx.z;
  const Group gr = a.groups[a.seq_group[b]];
  const int len = seq_len(a, b);
  // this CTA's pages of [prefix, len)
  const int begin = min(gr.prefix, len), p0 = begin / PAGE, pages = (len + PAGE - 1) / PAGE - p0;
  const int per = (pages + splits - 1) / splits;
  const int k0 = max(begin, (p0 + me * per) * PAGE), k1 = min(len, (p0 + (me + 1) * per) * PAGE);
  float* res = stream<D, MT>(tm, a, smem, &abort_flag, a.table + (long)b * a.table_stride, kh, (long)b * a.ql, r0, rows,
                             min(k0, max(k1, 0)), k1, [&](int r) { return len - a.ql + (r0 + r) / G; });
  constexpr int RS = D + 2;
  cg::cluster_group cl = cg::this_cluster();
  if (splits > 1) cl.sync();
  griddep_wait();
  const int n_prefix = gr.prefix > 0 ? (gr.prefix + gr.chunk - 1) / gr.chunk * a.parts : 0;
  // one warp per row: the weights of all parts, then the sum; the rows are dealt over the CTAs of the cluster
  for (int r = me * kWarps + warp_id(); r < rows; r += splits * kWarps) {
    const int lane = lane_id();
    const long tok = (long)b * a.ql + (r0 + r) / G;
    const int h = kh * G + (r0 + r) % G;
    const long at0 = tok * a.nq + h, step = (long)a.B * a.ql * a.nq;
    float M = kNegBig;
    for (int s = 0; s < splits; ++s) M = fmaxf(M, (splits > 1 ? cl.map_shared_rank(res, s) : res)[r * RS + D]);
    for (int s = lane; s < n_prefix; s += 32) M = fmaxf(M, a.part_ml[at0 + s * step].x);
    M = warp_max(M);
    float L = 0.f, O[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) O[c] = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float* p = (splits > 1 ? cl.map_shared_rank(res, s) : res) + r * RS;
      const float w = exp2f(p[D] - M);
      L += p[D + 1] * w;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) O[c] += p[lane * (D / 32) + c] * w;
    }
    for (int s = 0; s < n_prefix; ++s) {
      const float2 ml = a.part_ml[at0 + s * step];
      const float w = exp2f(ml.x - M);
      L += ml.y * w;
      const float* p = a.part_o + (at0 + s * step) * D + lane * (D / 32);
      if constexpr (D == 128) {
        const float4 v = *reinterpret_cast<const float4*>(p);
        O[0] += v.x * w, O[1] += v.y * w, O[2] += v.z * w, O[3] += v.w * w;
      } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        O[0] += v.x * w, O[1] += v.y * w;
      }
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;  // a row that sees nothing gives zeros
    __nv_bfloat16* dst = a.out + tok * a.out_stride + h * D + lane * (D / 32);
    if constexpr (D == 128)
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack_bf16x2(O[0] * inv, O[1] * inv), pack_bf16x2(O[2] * inv, O[3] * inv));
    else
      *reinterpret_cast<uint32_t*>(dst) = pack_bf16x2(O[0] * inv, O[1] * inv);
  }
  if (splits > 1) cl.sync();  // the others may still read this CTA's result
}

template <int D, int MT>
void launch_prefix(const CUtensorMap& tm, const Args& a, int items, cudaStream_t stream) {
  constexpr int smem = stream_smem<D, MT>();
  C10_CUDA_CHECK(
      cudaFuncSetAttribute(prefix_stream_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  prefix_stream_kernel<D, MT><<<dim3(items, a.nkv), kWarps * 32, smem, stream>>>(tm, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <int D, bool kPair>
void launch_prefix_tc(const CUtensorMap& tm, const Args& a, int items, cudaStream_t stream) {
  constexpr int smem = tc::Cfg<D>::kSmem;
  C10_CUDA_CHECK(
      cudaFuncSetAttribute(tc::prefix_tc_kernel<D, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  tc::prefix_tc_kernel<D, kPair><<<dim3(items, a.nkv), tc::kThreads, smem, stream>>>(tm, a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

template <int D, int MT>
void launch_suffix(const CUtensorMap& tm, const Args& a, int splits, bool dependent, cudaStream_t stream) {
  constexpr int smem = stream_smem<D, MT>();
  C10_CUDA_CHECK(cudaFuncSetAttribute(suffix_kernel<D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int row_chunks = (a.ql * (a.nq / a.nkv) + MT * 16 - 1) / (MT * 16);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.B, a.nkv * row_chunks, splits);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (splits > 1) {
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
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, suffix_kernel<D, MT>, tm, a, row_chunks));
}

template <int D>
void run(const CUtensorMap& tm, const Args& a, int items, int tile_rows, int suffix_splits, cudaStream_t stream) {
  if (items > 0) {
    if (tile_rows == 16) launch_prefix<D, 1>(tm, a, items, stream);
    else if (tile_rows == 32) launch_prefix<D, 2>(tm, a, items, stream);
    else if (tile_rows == 128) launch_prefix_tc<D, false>(tm, a, items, stream);
    else launch_prefix_tc<D, true>(tm, a, items, stream);
  }
  if (a.ql * (a.nq / a.nkv) <= 16) launch_suffix<D, 1>(tm, a, suffix_splits, items > 0, stream);
  else launch_suffix<D, 2>(tm, a, suffix_splits, items > 0, stream);
}

}  // namespace shared_prefix

// The messages are single literals: formatting one needs iostreams, which crash where the extension was linked to a
// libstdc++ of its own.
#define SP_CHECK(cond, msg) TORCH_CHECK(cond, "shared_prefix_attention: " msg)

void shared_prefix_attention(const torch::Tensor& q, const torch::Tensor& kv_cache, int64_t layer,
                             const torch::Tensor& block_table, const torch::Tensor& seq_lens, torch::Tensor& out,
                             const torch::Tensor& items, const torch::Tensor& groups, const torch::Tensor& seq_group,
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
  SP_CHECK(seq_group.scalar_type() == at::kInt && seq_group.is_contiguous() && seq_group.numel() == B, "the plan is for another number of sequences");
  SP_CHECK(items.scalar_type() == at::kInt && items.dim() == 2 && items.size(1) == 4 && items.is_contiguous() &&
                  groups.scalar_type() == at::kInt && groups.dim() == 2 && groups.size(1) == 4 &&
                  groups.is_contiguous(),
              "items and groups must be a plan's");
  SP_CHECK(tile_rows == 16 || tile_rows == 32 || tile_rows == 128 || tile_rows == 256, "unknown row tile");
  SP_CHECK(suffix_splits == 1 || suffix_splits == 2 || suffix_splits == 4 || suffix_splits == 8, "suffix_splits must be 1, 2, 4 or 8");
  const uint64_t rows = (uint64_t)kv_cache.size(1) * 2 * nkv * PAGE;
  SP_CHECK(rows < (1ull << 31), "kv_cache has too many rows per layer for 32-bit tile coordinates");
  SP_CHECK(nkv * q.size(1) * q_len <= 65535, "too many heads");
  SP_CHECK(q.is_cuda(), "tensors must be on a CUDA device");
  for (const torch::Tensor* t : {&kv_cache, &block_table, &seq_lens, &static_cast<const torch::Tensor&>(out), &items,
                                 &groups, &seq_group})
    SP_CHECK(t->device() == q.device(), "tensors must be on one device");
  if (B == 0) return;
  const at::cuda::CUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
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
  a.seq_group = seq_group.data_ptr<int>();
  a.B = int(B);
  a.nq = int(nq);
  a.nkv = int(nkv);
  a.ql = int(q_len);
  a.NB = int(kv_cache.size(1));
  a.scale_log2 = float(scale * 1.4426950408889634);
  a.status = status_word(q.get_device());
  a.parts = tile_rows == 128 ? 2 : 1;
  prefix_splits *= a.parts;
  // partial sums of the prefix: every (split, row) that the suffix kernel reads is written by an item
  auto ws = torch::empty({prefix_splits * T * nq * (D + 2)}, q.options().dtype(at::kFloat));
  a.part_o = ws.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part_o + prefix_splits * T * nq * D);
  const auto* base = reinterpret_cast<const __nv_bfloat16*>(kv_cache.data_ptr()) + layer * kv_cache.stride(0);
  const CUtensorMap tm = make_tmap_bf16_2d(base, D, rows, D * 2, 64, PAGE);
  if (D == 128) run<128>(tm, a, int(items.size(0)), int(tile_rows), int(suffix_splits), stream);
  else run<64>(tm, a, int(items.size(0)), int(tile_rows), int(suffix_splits), stream);
}

}  // namespace bloom

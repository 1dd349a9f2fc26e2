// Tokens from logits and given uniform numbers: temperature, top-k, top-p, min-p, several draws per row.
//
//   w_i = exp((l_i - max) / t)                        (l = NaN counts as -inf)
//   top-k  keeps the k largest, ties to the lowest index
//   top-p  keeps, in falling order, every token with less than p Z ahead of it (Z: the mass that top-k keeps)
//   min-p  keeps w_i >= min_p, i.e. l_i >= max + t ln(min_p)
//   token  the first kept i in vocabulary order whose inclusive sum exceeds u Z_kept
//
// The token is a whole number, so sums decide it at borders: weights are computed in fp64 (error below 1e-10) and summed
// as 64-bit fixed point with 2^45 for the largest.  Integer sums are exact and do not depend on the order of atomics,
// so a call gives the same tokens every time.  Weights below 2^-46 of the largest (32 t below the maximum) count as 0.
//
// One cluster of C CTAs per row, each CTA holding a slice of the row in shared memory, so a row is read from HBM once
// however many passes follow.  The passes are bound by instructions (a weight takes about 20), so the cut of top-k / top-p
// avoids weights where it can:
//   1. counts in 1024 bins over the distance to the maximum, (max - l) / t in steps of 1 / 32
//   2. top-k: the bin that holds the k-th is gathered into one CTA, sorted by (value, index), and cut
//   3. top-p: counts bound the mass of a bin to 3%, which leaves a window of bins for the cut; one pass sums the exact
//      masses before, behind, and per bin of the window; the bin that holds the cut is gathered, sorted and cut
// A bin of more than kList tokens (many equal values) is instead narrowed by histograms over the bits of its values,
// and equal values are counted off in vocabulary order.  Histograms are reduced over the cluster through distributed
// shared memory.  The draw walks vocabulary order: sums of 256 tokens, a scan, and one warp for the chunk that
// holds u Z.
// Measured with 128,256 bf16 logits a row (normal, deviation 3): one row 9 us plain, 16 top-k 50, 29 top-p 0.9 (cluster
// barriers, a sort); 256 rows 69, 95 and 227 us, bound by instructions (40, 60 and 120 a token; reading the row is
// 10 us).  Two CTAs per SM leave 64 registers a thread: 44 bytes of spills for bf16, 20 for fp32.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <cfloat>

#include "bloom/common.cuh"
#include "bloom/ops_share.h"
#include "bloom/tma_host.h"

namespace cg = cooperative_groups;

namespace bloom {
namespace draw {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kChunk = 256;          // tokens of one warp step: 8 consecutive ones per lane
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxVocab = 1 << 18;  // sums of 2^45 stay below 2^63
constexpr int kMaxSliceBytes = 128 * 1024;
constexpr float kRange = 32.f;       // in units of t below the maximum; e^-32 < 2^-46
constexpr float kBinsPerT = kBins / kRange;
constexpr int kTab = 512;
constexpr int kList = 2048;          // tokens that one CTA sorts

using u64 = unsigned long long;

struct Args {
  const void* logits;
  long ld;               // row stride in elements
  int V, slice;          // tokens per CTA, a multiple of kChunk
  const float* u;
  long ldu;
  int draws;
  const float* temp;
  const int* top_k;      // null: off
  const float* top_p;
  const float* min_p;
  int* out;              // [B, draws]
  bool vec;              // rows start on 16-byte boundaries
};

struct Hist {
  unsigned cnt[kBins], lo[kBins], hi[kBins];  // this CTA's counts and masses
  unsigned fine[kBins];                       // the cluster's counts of a finer level, scanned
};
// What top-k / top-p keep: values above `v`, and of those equal to it the ones at or before `last`.
struct Cut {
  float v;
  int last;
};
struct Shared {
  double tab[kTab];                    // 2^45 2^(j / 512)
  union {
    Hist h;
    u64 list[kList];                   // (order-preserving bits of the value, ~index)
  };
  unsigned count[kBins];               // the cluster's counts of the first level, scanned
  u64 mass[kBins];
  u64 wsum[kWarps];
  double wlo[kWarps], whi[kWarps];
  unsigned wcnt[kWarps];
  float cl_max[kMaxCluster];           // written by the CTAs of the cluster
  int cl_arg[kMaxCluster];
  unsigned cl_lo[2][kMaxCluster], cl_hi[2][kMaxCluster];  // one for each of a row's two selections
  unsigned cl_cnt[kMaxCluster];
  u64 cl_above[kMaxCluster], cl_all[kMaxCluster], cl_mass[kMaxCluster];
  Cut cl_cut[2];
  int cl_index;
  unsigned n_list;
  unsigned found, found2;
  float red_f[kWarps];
  unsigned red_a[kWarps], red_b[kWarps];
};

__device__ __forceinline__ unsigned* counts_of(Shared& s, int lv) { return lv == 0 ? s.count : s.h.fine; }

// Order-preserving bits of a float (-0 as +0).
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned b = __float_as_uint(v + 0.f);
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key ^ ((key & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

struct Row {
  float step, top, bins;  // a power of two, the maximum times it, bins per unit of l times it
  float low;           // values below it have no mass
  double mxd, c;       // the maximum, 512 / (t ln 2)
};
// round(2^45 exp((l - max) / t)) for l >= low: y = 512 (l - max) / (t ln 2) = n + f with n = 512 k + j, then
// 2^k 2^(j / 512) e^(f ln 2 / 512): a table of powers, and 1 + x + x^2 / 2 for |x| < 6.8e-4 (remainder < 6e-11).  The
// rounding to n adds 1.5 2^52, whose low bits are n; the rounding to a whole mass adds 2^52.
__device__ __forceinline__ u64 mass_of(float l, const Row& r, const double* tab) {
  constexpr double kMagic = 6755399441055744.0, a = 1.3538030870311430e-3;  // ln 2 / 512
  const double y = (static_cast<double>(l) - r.mxd) * r.c;  // the difference is exact, or nearly: logits may be large
  const double z = y + kMagic;
  const int n = __double2loint(z);
  const double f = y - (z - kMagic);
  const double p = fma(f, fma(f, 0.5 * a * a, a), 1.0);
  const double v = tab[n & (kTab - 1)] * p;
  const double w = __hiloint2double(__double2hiint(v) + ((n & ~(kTab - 1)) << 11), __double2loint(v));
  return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
}
// What a cut keeps, for all values including those below low, and the mass then.  Without a branch: in one, a warp
// runs the 20 instructions of a mass for every token all the same, and as many again to enter and leave it.
__device__ __forceinline__ bool keeps(const Cut& c, float v, int i) { return v > c.v || (v == c.v && i <= c.last); }
__device__ __forceinline__ u64 mass_if(bool keep, float v, const Row& r, const double* tab) {
  const u64 m = mass_of(v, r, tab);
  return keep ? m : 0;
}
// First-level bin of l >= low: monotone in l, because every rounding in it is.  The distance (max - l) step is rounded
// once; the step is 1 unless the distance or the bins per unit could leave fp32's range.
__device__ __forceinline__ int bin_of(float l, const Row& r) {
  return min(static_cast<int>(fmaf(-l, r.step, r.top) * r.bins), kBins - 1);
}

// 8 consecutive tokens from the slice.
template <typename T>
__device__ __forceinline__ void load8(const T* at, float (&v)[8]) {
  const uint4* p = reinterpret_cast<const uint4*>(at);
  if constexpr (sizeof(T) == 2) {
    const uint4 a = p[0];
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const uint4 a = p[0], b = p[1];
    v[0] = __uint_as_float(a.x), v[1] = __uint_as_float(a.y), v[2] = __uint_as_float(a.z);
    v[3] = __uint_as_float(a.w), v[4] = __uint_as_float(b.x), v[5] = __uint_as_float(b.y);
    v[6] = __uint_as_float(b.z), v[7] = __uint_as_float(b.w);
  }
}
// f(first index within the slice, 8 values) for this warp's chunks.
template <typename T, typename F>
__device__ __forceinline__ void for_chunks(const T* sl, int chunks, F&& f) {
  const int lane = lane_id();
  for (int c = warp_id(); c < chunks; c += kWarps) {
    float v[8];
    load8(sl + c * kChunk + lane * 8, v);
    f(c * kChunk + lane * 8, v);
  }
}
__device__ __forceinline__ u64 warp_sum_u64(u64 m) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
  return m;
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename P>
__device__ __forceinline__ P* remote(cg::cluster_group& cl, P* p, int rank) {
  return cl.map_shared_rank(p, rank);
}

__device__ __forceinline__ void clear_hist(Shared& s, bool with_mass) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    s.h.cnt[b] = 0;
    if (with_mass) s.h.lo[b] = s.h.hi[b] = 0;
  }
}
// 64-bit sums as two 32-bit atomics and a carry: integer adds of 64 bits are not native to shared memory
__device__ __forceinline__ void hist_mass(Shared& s, int b, u64 m) {
  const unsigned l = static_cast<unsigned>(m);
  const unsigned before = atomicAdd(&s.h.lo[b], l);
  const unsigned up = static_cast<unsigned>(m >> 32) + (before + l < before ? 1u : 0u);
  if (up) atomicAdd(&s.h.hi[b], up);
}

// The cluster's histogram, inclusively scanned, into count[lv] (counts) / mass (masses) of every CTA.
__device__ void combine(cg::cluster_group& cl, Shared& s, int lv, bool counts, bool masses) {
  const int C = cl.num_blocks(), me = cl.block_rank();
  cl.sync();
  const int share = kBins / C;
  for (int i = threadIdx.x; i < share; i += kThreads) {
    const int b = me * share + i;
    unsigned c = 0;
    u64 m = 0;
    for (int r = 0; r < C; ++r) {
      const Shared* o = remote(cl, &s, r);
      if (counts) c += o->h.cnt[b];
      if (masses) m += (static_cast<u64>(o->h.hi[b]) << 32) + o->h.lo[b];
    }
    for (int r = 0; r < C; ++r) {
      Shared* o = remote(cl, &s, r);
      if (counts) counts_of(*o, lv)[b] = c;
      if (masses) o->mass[b] = m;
    }
  }
  cl.sync();
  // block scan, two bins per thread
  const int lane = lane_id(), w = warp_id(), b0 = 2 * threadIdx.x;
  unsigned* cs = counts_of(s, lv);
  const unsigned c0 = counts ? cs[b0] : 0, c1 = counts ? cs[b0 + 1] : 0;
  const u64 m0 = masses ? s.mass[b0] : 0, m1 = masses ? s.mass[b0 + 1] : 0;
  unsigned c = c0 + c1;
  u64 m = m0 + m1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned c2 = __shfl_up_sync(0xffffffffu, c, o);
    const u64 m2 = __shfl_up_sync(0xffffffffu, m, o);
    if (lane >= o) c += c2, m += m2;
  }
  if (lane == 31) s.wcnt[w] = c, s.wsum[w] = m;
  __syncthreads();
  unsigned cb = 0;
  u64 mb = 0;
  for (int i = 0; i < w; ++i) cb += s.wcnt[i], mb += s.wsum[i];
  c += cb, m += mb;
  if (counts) cs[b0] = c - c1, cs[b0 + 1] = c;
  if (masses) s.mass[b0] = m - m1, s.mass[b0 + 1] = m;
  __syncthreads();
}

// First bin whose inclusive count (lv) or mass (lv < 0) reaches `target`.
__device__ int find(Shared& s, int lv, u64 target) {
  if (threadIdx.x == 0) s.found = kBins - 1;
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    const u64 v = lv < 0 ? s.mass[b] : counts_of(s, lv)[b];
    const u64 p = b == 0 ? 0 : lv < 0 ? s.mass[b - 1] : counts_of(s, lv)[b - 1];
    if (v >= target && p < target) s.found = b;  // at most one bin
  }
  __syncthreads();
  const int r = s.found;
  __syncthreads();
  return r;
}

// The members of first-level bin `bin` that `cut` keeps (there are `inside` <= kList of them), gathered into CTA 0 and
// sorted there by falling value, then index.  The cut moves to the first of them whose inclusive count, or mass after
// `mbefore`, reaches the target.
template <typename T>
__device__ Cut sort_select(cg::cluster_group& cl, Shared& s, const T* sl, int chunks, int s0, const Row& row, int sel,
                           Cut cut, int bin, unsigned inside, bool by_mass, u64 before, u64 target) {
  const int me = cl.block_rank(), lane = lane_id(), w = warp_id();
  Shared* o = remote(cl, &s, 0);
  for_chunks(sl, chunks, [&](int i, const float(&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v[e] >= row.low && bin_of(v[e], row) == bin && (v[e] > cut.v || (v[e] == cut.v && s0 + i + e <= cut.last))) {
        const unsigned at = atomicAdd(&o->n_list, 1u);
        if (at < kList)
          o->list[at] = (static_cast<u64>(key_of(v[e])) << 32) | static_cast<unsigned>(~(s0 + i + e));
      }
  });
  cl.sync();
  if (me == 0) {
    int n = 32;
    while (n < static_cast<int>(inside)) n *= 2;
    for (int i = inside + threadIdx.x; i < n; i += kThreads) s.list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= n; k *= 2)  // bitonic, falling
      for (int j = k / 2; j > 0; j /= 2) {
        for (int i = threadIdx.x; i < n / 2; i += kThreads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const u64 x = s.list[a], y = s.list[b];
          if ((x < y) == ((a & k) == 0)) s.list[a] = y, s.list[b] = x;
        }
        __syncthreads();
      }
    int pick = -1;
    if (!by_mass) {
      pick = static_cast<int>(target - before) - 1;
    } else {  // inclusive masses in order: each thread a run of 4
      const int i0 = threadIdx.x * (kList / kThreads);
      u64 m[kList / kThreads], sum = 0;
#pragma unroll
      for (int q = 0; q < kList / kThreads; ++q) {
        const int i = i0 + q;
        m[q] = i < static_cast<int>(inside) ? mass_of(value_of(static_cast<unsigned>(s.list[i] >> 32)), row, s.tab) : 0;
        sum += m[q];
      }
      u64 x = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (lane == 31) s.wsum[w] = x;
      if (threadIdx.x == 0) s.found2 = inside - 1;
      __syncthreads();
      u64 acc = before + x - sum;
      for (int i = 0; i < w; ++i) acc += s.wsum[i];
#pragma unroll
      for (int q = 0; q < kList / kThreads; ++q) {
        if (acc < target && acc + m[q] >= target) s.found2 = i0 + q;  // at most one
        acc += m[q];
      }
      __syncthreads();
      pick = static_cast<int>(s.found2);
    }
    if (threadIdx.x < cl.num_blocks()) {
      const u64 x = s.list[pick];
      remote(cl, &s, threadIdx.x)->cl_cut[sel] =
          Cut{value_of(static_cast<unsigned>(x >> 32)), static_cast<int>(~static_cast<unsigned>(x))};
    }
    __syncthreads();
    if (threadIdx.x == 0) s.n_list = 0;
  }
  cl.sync();
  return s.cl_cut[sel];
}

// The same for a bin of more tokens: its range of values is narrowed by histograms of their bits until it is one value
// (or all of it is kept), and equal values are counted off in vocabulary order.
template <typename T>
__device__ Cut narrow_select(cg::cluster_group& cl, Shared& s, const T* sl, int chunks, int s0, const Row& row, int sel,
                             Cut cut, int bin, unsigned inside, u64 minside, bool by_mass, unsigned before, u64 mbefore,
                             u64 target) {
  const int C = cl.num_blocks(), me = cl.block_rank();
  const int lane = lane_id(), w = warp_id();
  auto member = [&](float v, int i) {
    return v >= row.low && bin_of(v, row) == bin && (v > cut.v || (v == cut.v && i <= cut.last));
  };
  unsigned lo = 0xffffffffu, hi = 0;
  for_chunks(sl, chunks, [&](int i, const float(&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (member(v[e], s0 + i + e)) {
        const unsigned k = key_of(v[e]);
        lo = min(lo, k);
        hi = max(hi, k);
      }
  });
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) s.red_a[w] = lo, s.red_b[w] = hi;
  __syncthreads();
  if (threadIdx.x < C) {
    for (int i = 0; i < kWarps; ++i) lo = min(lo, s.red_a[i]), hi = max(hi, s.red_b[i]);
    Shared* o = remote(cl, &s, threadIdx.x);
    o->cl_lo[sel][me] = lo;
    o->cl_hi[sel][me] = hi;
  }
  cl.sync();
  for (int r = 0; r < C; ++r) lo = min(lo, s.cl_lo[sel][r]), hi = max(hi, s.cl_hi[sel][r]);
  // all that is left in the range is kept: no need to look inside
  auto whole = [&]() { return inside == 1 || (by_mass ? mbefore + minside == target : before + inside == target); };
  while (hi != lo && !whole()) {
    const int shift = max(0, 32 - __clz(hi - lo) - 10);
    clear_hist(s, by_mass);
    __syncthreads();
    for_chunks(sl, chunks, [&](int i, const float(&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (member(v[e], s0 + i + e)) {
          const unsigned k = key_of(v[e]);
          if (k >= lo && k <= hi) {
            atomicAdd(&s.h.cnt[(hi - k) >> shift], 1u);
            if (by_mass) hist_mass(s, (hi - k) >> shift, mass_of(v[e], row, s.tab));
          }
        }
    });
    combine(cl, s, 1, true, by_mass);
    const int b = by_mass ? find(s, -1, target - mbefore) : find(s, 1, target - before);
    const unsigned cb = b ? s.h.fine[b - 1] : 0;
    inside = s.h.fine[b] - cb;
    before += cb;
    if (by_mass) {
      const u64 mb = b ? s.mass[b - 1] : 0;
      minside = s.mass[b] - mb;
      mbefore += mb;
    }
    const unsigned top = hi - (static_cast<unsigned>(b) << shift);
    lo = max(lo, top - ((1u << shift) - 1u));
    hi = top;
  }
  const float v = value_of(lo);
  const int old = v == cut.v ? cut.last : 0x7fffffff;  // of values equal to the previous cut's, those it kept
  if (whole()) return Cut{v, old};
  // equal values: the first `r` of them by index
  const u64 one = by_mass ? mass_of(v, row, s.tab) : 0;
  const u64 r = by_mass ? (one ? (target - mbefore + one - 1) / one : 1) : target - before;
  if (r >= inside) return Cut{v, old};
  unsigned mine = 0;
  for_chunks(sl, chunks, [&](int, const float(&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mine += x[e] == v;
  });
  mine = __reduce_add_sync(0xffffffffu, mine);
  if (lane == 0) s.red_a[w] = mine;
  __syncthreads();
  if (threadIdx.x < C) {
    unsigned t = 0;
    for (int i = 0; i < kWarps; ++i) t += s.red_a[i];
    remote(cl, &s, threadIdx.x)->cl_cnt[me] = t;
  }
  cl.sync();
  u64 ahead = 0;
  for (int i = 0; i < me; ++i) ahead += s.cl_cnt[i];
  if (r > ahead && r <= ahead + s.cl_cnt[me] && w == 0) {  // this CTA holds the r-th: one warp walks its slice in order
    unsigned left = static_cast<unsigned>(r - ahead);
    for (int c = 0; c < chunks; ++c) {
      unsigned hit = 0;
      const T* p = sl + c * kChunk + lane * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) hit |= (to_float(p[e]) == v ? 1u : 0u) << e;
      unsigned n = __popc(hit), incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      const unsigned all = __shfl_sync(0xffffffffu, incl, 31);
      if (all >= left) {
        if (incl >= left && incl - n < left) {
          for (unsigned k = incl - n + 1; k < left; ++k) hit &= hit - 1;
          const int at = s0 + c * kChunk + lane * 8 + __ffs(hit) - 1;
          for (int i = 0; i < C; ++i) remote(cl, &s, i)->cl_index = at;
        }
        break;
      }
      left -= all;
    }
  }
  cl.sync();
  return Cut{v, s.cl_index};
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) draw_kernel(const Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  cg::cluster_group cl = cg::this_cluster();
  const int C = cl.num_blocks(), me = cl.block_rank();
  Shared& s = *reinterpret_cast<Shared*>(raw);
  T* sl = reinterpret_cast<T*>(raw + ((sizeof(Shared) + 15) & ~size_t(15)));
  u64* csum = reinterpret_cast<u64*>(reinterpret_cast<uint8_t*>(sl) + (size_t)a.slice * sizeof(T));
  const int b = blockIdx.x / C;
  const int lane = lane_id(), w = warp_id();
  const int s0 = me * a.slice;
  const int n = max(0, min(a.slice, a.V - s0));
  const int chunks = (n + kChunk - 1) / kChunk;
  const T* row = static_cast<const T*>(a.logits) + (long)b * a.ld + s0;
  const float t = a.temp[b];
  const int k = a.top_k != nullptr ? a.top_k[b] : 0;
  const float p = a.top_p != nullptr ? a.top_p[b] : 1.f;
  const float mp = a.min_p != nullptr ? a.min_p[b] : 0.f;

  // ---- the slice into shared memory (padding: -inf), its maximum (NaN is never the larger one)
  constexpr int kVec = 16 / sizeof(T);
  float best = -INFINITY;
  int done = 0;
  if (a.vec) {
    const int nv = n / kVec;
    constexpr int kAhead = 8;  // requests in flight per thread
    for (int i0 = threadIdx.x; i0 < nv; i0 += kAhead * kThreads) {
      uint4 x[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i0 + j * kThreads < nv) x[j] = __ldg(reinterpret_cast<const uint4*>(row) + i0 + j * kThreads);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (i0 + j * kThreads < nv) {
          reinterpret_cast<uint4*>(sl)[i0 + j * kThreads] = x[j];
          if constexpr (sizeof(T) == 2) {
            const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&x[j]);
            const __nv_bfloat162 m = __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3]));
            best = fmaxf(best, fmaxf(__low2float(m), __high2float(m)));
          } else {
            const float* e = reinterpret_cast<const float*>(&x[j]);
            best = fmaxf(best, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])));
          }
        }
    }
    done = nv * kVec;
  }
  for (int i = done + threadIdx.x; i < chunks * kChunk; i += kThreads) {
    const T x = i < n ? row[i] : static_cast<T>(-INFINITY);
    sl[i] = x;
    best = fmaxf(best, to_float(x));
  }
  best = warp_max(best);
  if (lane == 0) s.red_f[w] = best;
  if (threadIdx.x == 0) s.n_list = 0;
  cl.sync();  // also: every CTA of the cluster runs, so its shared memory may be written
  if (threadIdx.x < C) {
    for (int i = 0; i < kWarps; ++i) best = fmaxf(best, s.red_f[i]);
    remote(cl, &s, threadIdx.x)->cl_max[me] = best;
  }
  cl.sync();
  for (int r = 0; r < C; ++r) best = fmaxf(best, s.cl_max[r]);

  int* out = a.out + (long)b * a.draws;
  if (best == -INFINITY) {  // nothing to draw from (the whole cluster leaves; nothing of it is written any more)
    if (me == 0)
      for (int d = threadIdx.x; d < a.draws; d += kThreads) out[d] = -1;
    return;
  }
  if (!(t > 0.f)) {  // greedy: the first index of the maximum
    int at = 0x7fffffff;
    for_chunks(sl, chunks, [&](int i, const float(&v)[8]) {
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (v[e] == best) at = min(at, s0 + i + e);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) s.red_a[w] = at;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 0; i < kWarps; ++i) at = min(at, static_cast<int>(s.red_a[i]));
      remote(cl, &s, 0)->cl_arg[me] = at;
    }
    cl.sync();
    if (me == 0) {
      for (int r = 0; r < C; ++r) at = min(at, s.cl_arg[r]);
      for (int d = threadIdx.x; d < a.draws; d += kThreads) out[d] = at;
    }
    return;
  }
  // the table of powers, from 16 and 32 of them
  static_assert(kTab == kThreads, "one entry per thread");
  if (threadIdx.x < 48)
    s.tab[threadIdx.x] = threadIdx.x < 16 ? exp2(45.0 + threadIdx.x / 16.0) : exp2((threadIdx.x - 16) / 512.0);
  __syncthreads();
  const double pw = s.tab[threadIdx.x >> 5] * s.tab[16 + (threadIdx.x & 31)];
  __syncthreads();
  s.tab[threadIdx.x] = pw;
  if (best == INFINITY) {  // the limit of finite ones: infinities share the mass
    for (int i = threadIdx.x; i < chunks * kChunk; i += kThreads)
      sl[i] = static_cast<T>(to_float(sl[i]) == INFINITY ? 0.f : -INFINITY);
    best = 0.f;
  }
  __syncthreads();
  Row r;
  const double td = static_cast<double>(t);
  // max - l may be twice the largest float, which matters where t is as large; 1 / t overflows below 2^-128, and
  // distances of t / 32 are subnormal (0 here) below 2^-121.  With such a t and a maximum of 1 or more, all of l >= low
  // equal the maximum.
  r.step = t > 0x1p64f ? 0.25f : t < 0x1p-100f && fabsf(best) < 1.f ? 0x1p100f : 1.f;
  r.top = best * r.step;
  r.c = 738.65986093514926 / td;  // 512 / ln 2
  r.mxd = static_cast<double>(best);
  r.bins = static_cast<float>(kBinsPerT / (td * static_cast<double>(r.step)));
  r.low = fmaxf(static_cast<float>(static_cast<double>(best) - kRange * td), -FLT_MAX);
  const bool need_k = k > 0 && k < a.V, need_p = p > 0.f && p < 1.f;
  Cut cut{r.low, 0x7fffffff};
  if (need_k || need_p) {
    clear_hist(s, true);
    __syncthreads();
    for_chunks(sl, chunks, [&](int, const float(&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v[e] >= r.low) atomicAdd(&s.h.cnt[bin_of(v[e], r)], 1u);
    });
    combine(cl, s, 0, true, false);
    unsigned total = s.count[kBins - 1];
    if (need_k && static_cast<unsigned>(k) < total) {
      const int bk = find(s, 0, static_cast<u64>(k));
      const unsigned before = bk ? s.count[bk - 1] : 0, inside = s.count[bk] - before;
      cut = inside <= kList
                ? sort_select(cl, s, sl, chunks, s0, r, 0, cut, bk, inside, false, before, static_cast<u64>(k))
                : narrow_select(cl, s, sl, chunks, s0, r, 0, cut, bk, inside, 0ull, false, before, 0ull,
                                static_cast<u64>(k));
      total = static_cast<unsigned>(k);
    }
    if (need_p) {
      // Bounds on the inclusive masses: c_b e^-(b + 1)/32 <= mass of bin b <= c_b e^-b/32, with 1e-4 of room for the
      // roundings of bins and sums.  `total` ends the counts where top-k does.
      const int b0 = 2 * threadIdx.x;
      double up[2], dn[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int i = b0 + q;
        const unsigned prev = i ? min(s.count[i - 1], total) : 0, c = min(s.count[i], total) - prev;
        const double e = exp2f(-static_cast<float>(i) * (1.4426950408889634f / kBinsPerT));
        up[q] = c * e * 1.0001;
        dn[q] = c * e * (0.96923323447634 * 0.9999);  // e^(-1/32)
      }
      double xu = up[0] + up[1], xd = dn[0] + dn[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double yu = __shfl_up_sync(0xffffffffu, xu, o), yd = __shfl_up_sync(0xffffffffu, xd, o);
        if (lane >= o) xu += yu, xd += yd;
      }
      if (lane == 31) s.whi[w] = xu, s.wlo[w] = xd;
      if (threadIdx.x == 0) s.found = 0, s.found2 = kBins - 1;
      __syncthreads();
      double bu = 0, bd = 0, zu = 0, zd = 0;
      for (int i = 0; i < kWarps; ++i) {
        if (i < w) bu += s.whi[i], bd += s.wlo[i];
        zu += s.whi[i], zd += s.wlo[i];
      }
      // the cut's bin is the first whose mass reaches p Z: none whose upper bound is below the lowest p Z, and none
      // after the first whose lower bound reaches the highest
      const double pd = static_cast<double>(p);
      xu += bu, xd += bd;
#pragma unroll
      for (int q = 1; q >= 0; --q) {
        const double iu = q ? xu : xu - up[1], id = q ? xd : xd - dn[1];
        if (iu >= pd * zd && iu - up[q] < pd * zd) s.found = b0 + q;
        if (id >= pd * zu && id - dn[q] < pd * zu) s.found2 = b0 + q;
      }
      clear_hist(s, true);
      __syncthreads();
      const int wlo = static_cast<int>(s.found), whi = static_cast<int>(s.found2);
      // exact masses: above the window, in the window by bins, and of all
      u64 above = 0, all = 0;
      const Cut in{cut.v, cut.last - s0};  // indexes within the slice
      for_chunks(sl, chunks, [&](int i, const float(&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const bool keep = keeps(in, v[e], i + e);
          const u64 m = mass_if(keep, v[e], r, s.tab);
          const int q = bin_of(v[e], r);
          all += m;
          above += q < wlo ? m : 0;
          if (keep && q >= wlo && q <= whi) hist_mass(s, q, m);
        }
      });
      above = warp_sum_u64(above);
      all = warp_sum_u64(all);
      __syncthreads();  // wsum, whi are read no more
      if (lane == 0) s.wsum[w] = above, reinterpret_cast<u64*>(s.whi)[w] = all;
      __syncthreads();
      if (threadIdx.x < C) {
        above = all = 0;
        for (int i = 0; i < kWarps; ++i) above += s.wsum[i], all += reinterpret_cast<u64*>(s.whi)[i];
        Shared* o = remote(cl, &s, threadIdx.x);
        o->cl_above[me] = above;
        o->cl_all[me] = all;
      }
      combine(cl, s, 1, false, true);
      u64 head = 0, z = 0;
      for (int i = 0; i < C; ++i) head += s.cl_above[i], z += s.cl_all[i];
      u64 target = static_cast<u64>(ceil(pd * static_cast<double>(z)));
      if (target < 1) target = 1;
      const int bp = min(max(find(s, -1, target > head ? target - head : 1), wlo), whi);
      const unsigned before = bp ? min(s.count[bp - 1], total) : 0;
      const unsigned inside = min(s.count[bp], total) - before;
      const u64 mbefore = head + (bp ? s.mass[bp - 1] : 0), minside = s.mass[bp] - (bp ? s.mass[bp - 1] : 0);
      if (inside > 0)
        cut = inside <= kList ? sort_select(cl, s, sl, chunks, s0, r, 1, cut, bp, inside, true, mbefore, target)
                              : narrow_select(cl, s, sl, chunks, s0, r, 1, cut, bp, inside, minside, true, before,
                                              mbefore, target);
    }
  }
  if (mp > 0.f) {  // values at or above max + t ln(min_p), as the smallest float that is
    const double thr = static_cast<double>(best) + td * log(fmin(1.0, static_cast<double>(mp)));
    float f = static_cast<float>(thr);
    if (static_cast<double>(f) < thr) f = nextafterf(f, INFINITY);
    if (f > cut.v) cut = Cut{f, 0x7fffffff};
  }
  const Cut in{cut.v, cut.last - s0};  // indexes within the slice
  // ---- sums of 256 tokens in vocabulary order
  for_chunks(sl, chunks, [&](int i, const float(&v)[8]) {
    bool some = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) some |= v[e] >= cut.v;
    u64 m = 0;
    if (__any_sync(0xffffffffu, some)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) m += mass_if(keeps(in, v[e], i + e), v[e], r, s.tab);
      m = warp_sum_u64(m);
    }
    if (lane == 0) csum[i / kChunk] = m;
  });
  __syncthreads();
  if (w == 0) {  // inclusive scan of the sums
    u64 carry = 0;
    for (int c0 = 0; c0 < chunks; c0 += 32) {
      u64 x = c0 + lane < chunks ? csum[c0 + lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      x += carry;
      if (c0 + lane < chunks) csum[c0 + lane] = x;
      carry = __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane < C) remote(cl, &s, lane)->cl_mass[me] = carry;
  }
  cl.sync();
  u64 first = 0, z = 0;
  for (int i = 0; i < C; ++i) {
    if (i < me) first += s.cl_mass[i];
    z += s.cl_mass[i];
  }
  const u64 mine = s.cl_mass[me];
  for (int d = w; d < a.draws; d += kWarps) {
    const double u = static_cast<double>(a.u[(long)b * a.ldu + d]);
    u64 target = u > 0.0 ? static_cast<u64>(fmin(u, 1.0) * static_cast<double>(z)) : 0;
    if (target >= z) target = z - 1;
    if (target < first || target >= first + mine) continue;  // another CTA's
    const u64 at = target - first;
    int c0 = 0, c1 = chunks - 1;  // the first chunk whose inclusive sum exceeds `at`
    while (c0 < c1) {
      const int m = (c0 + c1) / 2;
      if (csum[m] > at) c1 = m;
      else c0 = m + 1;
    }
    const u64 left = at - (c0 ? csum[c0 - 1] : 0);
    u64 m[8], sum = 0;
    const int i = c0 * kChunk + lane * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = to_float(sl[i + e]);
      m[e] = mass_if(keeps(in, v, i + e), v, r, s.tab);
      sum += m[e];
    }
    u64 incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    u64 acc = incl - sum;
    if (incl > left && acc <= left) {
      int token = i;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        acc += m[e];
        if (acc > left) {
          token = i + e;
          break;
        }
      }
      out[d] = s0 + token;
    }
  }
}

template <typename T>
void launch(const Args& a, int B, int C, cudaStream_t stream) {
  const int smem = int((sizeof(Shared) + 15) / 16 * 16 + a.slice * sizeof(T) + a.slice / kChunk * sizeof(u64));
  static std::atomic<uint64_t> configured{0};  // per device: the limit of dynamic shared memory has been raised
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (!(configured.load(std::memory_order_acquire) >> dev & 1u)) {
    constexpr int most = int((sizeof(Shared) + 15) / 16 * 16 + kMaxSliceBytes + kMaxSliceBytes / sizeof(T) / kChunk * sizeof(u64));
    C10_CUDA_CHECK(cudaFuncSetAttribute(draw_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    configured.fetch_or(uint64_t(1) << dev, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(B) * C);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, draw_kernel<T>, a));
}

}  // namespace draw

void sample_uniform(const torch::Tensor& logits, const torch::Tensor& u, const torch::Tensor& temperature,
                    const c10::optional<torch::Tensor>& top_k, const c10::optional<torch::Tensor>& top_p,
                    const c10::optional<torch::Tensor>& min_p, torch::Tensor& out) {
  using namespace draw;
  TORCH_CHECK(logits.dim() == 2 && (logits.scalar_type() == at::kFloat || logits.scalar_type() == at::kBFloat16) &&
                  (logits.size(1) <= 1 || logits.stride(1) == 1),
              "sample_uniform: logits must be f32 or bf16 [B, V] with contiguous rows");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V <= kMaxVocab, "sample_uniform: 1 to 2^18 tokens per row");
  TORCH_CHECK((u.dim() == 1 || u.dim() == 2) && u.size(0) == B && u.scalar_type() == at::kFloat &&
                  (u.dim() == 1 ? u.is_contiguous() : u.size(1) <= 1 || u.stride(1) == 1),
              "sample_uniform: u must be f32 [B] or [B, n] with contiguous rows");
  TORCH_CHECK(out.sizes() == u.sizes() && out.scalar_type() == at::kInt && out.is_contiguous(),
              "sample_uniform: out must be contiguous int32 of u's shape");
  auto per_row = [&](const torch::Tensor& t, at::ScalarType ty) {
    return t.dim() == 1 && t.size(0) == B && t.scalar_type() == ty && t.is_contiguous();
  };
  auto here = [&](const c10::optional<torch::Tensor>& t) { return !t.has_value() || t->device() == logits.device(); };
  TORCH_CHECK(per_row(temperature, at::kFloat), "sample_uniform: temperature must be contiguous f32 [B]");
  TORCH_CHECK(!top_k.has_value() || per_row(*top_k, at::kInt), "sample_uniform: top_k must be contiguous int32 [B]");
  TORCH_CHECK(!top_p.has_value() || per_row(*top_p, at::kFloat), "sample_uniform: top_p must be contiguous f32 [B]");
  TORCH_CHECK(!min_p.has_value() || per_row(*min_p, at::kFloat), "sample_uniform: min_p must be contiguous f32 [B]");
  TORCH_CHECK(u.device() == logits.device() && out.device() == logits.device() && here(temperature) && here(top_k) &&
                  here(top_p) && here(min_p),
              "sample_uniform: tensors must be on one device");
  TORCH_CHECK(logits.is_cuda(), "sample_uniform: tensors must be on a CUDA device");
  const int64_t draws = u.dim() == 2 ? u.size(1) : 1;
  if (B == 0 || draws == 0) return;
  TORCH_CHECK(B * kMaxCluster < (1ll << 31), "sample_uniform: too many rows");
  const at::cuda::CUDAGuard guard(logits.device());
  const int size = int(logits.element_size());
  auto slice_of = [&](int C) { return int(((V + C - 1) / C + kChunk - 1) / kChunk * kChunk); };
  // CTAs per row: enough for a slice of 64 KB (two CTAs per SM), and while the grid leaves SMs idle as many as keep
  // 4096 tokens per CTA
  int C = 1;
  const int sms = num_sms(logits.get_device());
  while (C < kMaxCluster && (slice_of(C) * size > 64 * 1024 || (B * C < sms && slice_of(C) >= 2 * 4096))) C *= 2;
  Args a;
  a.logits = logits.data_ptr();
  a.ld = logits.stride(0);
  a.V = int(V);
  a.slice = slice_of(C);
  TORCH_CHECK(a.slice * size <= kMaxSliceBytes, "sample_uniform: row too long");
  a.u = u.data_ptr<float>();
  a.ldu = u.stride(0);
  a.draws = int(draws);
  a.temp = temperature.data_ptr<float>();
  a.top_k = top_k.has_value() ? top_k->data_ptr<int>() : nullptr;
  a.top_p = top_p.has_value() ? top_p->data_ptr<float>() : nullptr;
  a.min_p = min_p.has_value() ? min_p->data_ptr<float>() : nullptr;
  a.out = out.data_ptr<int>();
  a.vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (B == 1 || a.ld * size % 16 == 0);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (size == 2) launch<__nv_bfloat16>(a, int(B), C, stream);
  else launch<float>(a, int(B), C, stream);
}

}  // namespace bloom

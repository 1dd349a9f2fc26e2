// Tokens from logits and given uniform numbers: temperature, top-k, top-p, min-p, several draws per row.
//
//   w_i = exp((l_i - max) / t)                        (l = NaN counts as -inf)
//   top-k  keeps the k largest, ties to the lowest index
//   top-p  keeps, in falling order, every token with less than p Z ahead of it (Z: the mass that top-k keeps)
//   min-p  keeps w_i >= min_p
//   token  the first kept i in vocabulary order whose inclusive sum exceeds u Z_kept
//
// The token is a whole number, so sums decide it at borders: weights are computed in fp64 (error ~1e-16) and summed as
// 64-bit fixed point with 2^45 for the largest.  Integer sums are exact and do not depend on the order of atomics, so
// a call gives the same tokens every time.  Weights below 2^-46 of the largest count as zero.
//
// One cluster of C CTAs per row, each CTA holding a slice of the row in shared memory, so a row is read from HBM once
// however many passes follow.  The cut of top-k / top-p is found by histograms of 1024 bins: first over the scaled
// distance to the maximum, (max - l) / t in 30 / 1023 steps, which spreads real logits over many bins where their
// floating-point bits would crowd a few; then over the bits of the values inside the bin that holds the cut, until it
// is one value.  Each histogram is reduced over the cluster through distributed shared memory (each CTA sums its
// share of the bins and stores the sums into all CTAs).  Mass sums use two 32-bit shared atomics with a carry.
// The draw walks vocabulary order: sums of 256-token chunks, a scan, and one warp for the chunk that holds u Z.
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
namespace draw {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kChunk = 256;          // tokens of one warp step: 8 consecutive ones per lane
constexpr int kMaxCluster = 8;
constexpr int64_t kMaxVocab = 1 << 18;  // sums of 2^45 stay below 2^63
constexpr int kMaxSliceBytes = 128 * 1024;
constexpr float kRange = 30.f;
constexpr int kTab = 64;

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

struct Shared {
  double tab[kTab];                    // 2^(j / 64)
  unsigned cnt[kBins], lo[kBins], hi[kBins];  // this CTA's histogram
  u64 mass[2][kBins];                  // the cluster's, scanned: [0] first level, [1] the finer ones
  unsigned count[2][kBins];
  u64 wsum[kWarps];
  unsigned wcnt[kWarps];
  float cl_max[kMaxCluster];           // written by the CTAs of the cluster
  int cl_arg[kMaxCluster];
  unsigned cl_lo[2][kMaxCluster], cl_hi[2][kMaxCluster];  // one for each of a row's two selections
  unsigned cl_cnt[kMaxCluster];
  u64 cl_mass[kMaxCluster];
  int cl_index;
  unsigned found;
  float red_f[kWarps];
  int red_i[kWarps];
  unsigned red_a[kWarps], red_b[kWarps];
};

template <typename T>
__device__ __forceinline__ float clean(T v);
// NaN -> -inf, -0 -> +0
template <>
__device__ __forceinline__ float clean<float>(float v) {
  return v == v ? v + 0.f : -INFINITY;
}
template <>
__device__ __forceinline__ float clean<__nv_bfloat16>(__nv_bfloat16 v) {
  return clean<float>(__bfloat162float(v));
}
// Order-preserving bits of a float.
__device__ __forceinline__ unsigned key_of(float v) {
  const unsigned b = __float_as_uint(v);
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key ^ ((key & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// exp(x) for x in (-32, 0] as 2^k 2^(j/64) e^r with |r| <= ln 2 / 128: a table of powers and the Taylor polynomial
// of degree 5 (remainder r^6 / 720 < 4e-17).  The rounding to n = 64 k + j adds 1.5 2^52, whose low bits are n.
__device__ __forceinline__ double exp_neg(double x, const double* tab) {
  constexpr double kMagic = 6755399441055744.0;
  const double z = fma(x, 92.332482616893656877, kMagic);  // 64 / ln 2
  const int n = __double2loint(z);
  const double r = fma(z - kMagic, -0.010830424696249145, x);  // ln 2 / 64
  double p = fma(r, 1.0 / 120, 1.0 / 24);
  p = fma(r, p, 1.0 / 6);
  p = fma(r, p, 0.5);
  p = fma(r, p, 1.0);
  p = fma(r, p, 1.0);
  const double v = tab[n & (kTab - 1)] * p;
  return __hiloint2double(__double2hiint(v) + ((n >> 6) << 20), __double2loint(v));
}

struct Row {
  float mx, inv_tf;
  double mxd, inv_t, min_w;
};
__device__ __forceinline__ double weight(float l, const Row& r, const double* tab) {
  if (l == r.mx) return 1.0;
  if (!(l > -INFINITY)) return 0.0;
  const double x = (static_cast<double>(l) - r.mxd) * r.inv_t;
  return x > -32.0 ? exp_neg(x, tab) : 0.0;
}
// round(w 2^45): the low 52 bits of w 2^45 + 2^52
__device__ __forceinline__ u64 fixed(double w) {
  return static_cast<u64>(__double_as_longlong(fma(w, 35184372088832.0, 4503599627370496.0))) & 0xfffffffffffffull;
}
__device__ __forceinline__ u64 mass_of(float l, const Row& r, const double* tab) { return fixed(weight(l, r, tab)); }
// First-level bin: monotone in l, because every rounding in it is.
__device__ __forceinline__ int bin_of(float l, const Row& r) {
  if (l == r.mx) return 0;
  const float x = (r.mx - l) * r.inv_tf;
  return x < kRange ? static_cast<int>(x * ((kBins - 1) / kRange)) : kBins - 1;
}

// f(chunk, first index within the slice, 8 values) for this warp's chunks.
template <typename T, typename F>
__device__ __forceinline__ void for_chunks(const T* sl, int chunks, F&& f) {
  const int lane = lane_id();
  for (int c = warp_id(); c < chunks; c += kWarps) {
    float v[8];
    const uint4* p = reinterpret_cast<const uint4*>(sl + c * kChunk + lane * 8);
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
    f(c, c * kChunk + lane * 8, v);
  }
}

template <typename P>
__device__ __forceinline__ P* remote(cg::cluster_group& cl, P* p, int rank) {
  return cl.map_shared_rank(p, rank);
}

__device__ __forceinline__ void clear_hist(Shared& s) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) s.cnt[b] = s.lo[b] = s.hi[b] = 0;
}
__device__ __forceinline__ void hist_add(Shared& s, int b, bool with_mass, u64 m) {
  atomicAdd(&s.cnt[b], 1u);
  if (with_mass) {
    const unsigned l = static_cast<unsigned>(m);
    const unsigned before = atomicAdd(&s.lo[b], l);
    const unsigned up = static_cast<unsigned>(m >> 32) + (before + l < before ? 1u : 0u);
    if (up) atomicAdd(&s.hi[b], up);
  }
}

// The cluster's histogram, inclusively scanned, into count[lv] / mass[lv] of every CTA.
__device__ void combine(cg::cluster_group& cl, Shared& s, int lv) {
  const int C = cl.num_blocks(), me = cl.block_rank();
  cl.sync();
  const int share = kBins / C;
  for (int i = threadIdx.x; i < share; i += kThreads) {
    const int b = me * share + i;
    unsigned c = 0;
    u64 m = 0;
    for (int r = 0; r < C; ++r) {
      const Shared* o = remote(cl, &s, r);
      c += o->cnt[b];
      m += (static_cast<u64>(o->hi[b]) << 32) + o->lo[b];
    }
    for (int r = 0; r < C; ++r) {
      Shared* o = remote(cl, &s, r);
      o->count[lv][b] = c;
      o->mass[lv][b] = m;
    }
  }
  cl.sync();
  // block scan, two bins per thread
  const int lane = lane_id(), w = warp_id(), b0 = 2 * threadIdx.x;
  const unsigned c0 = s.count[lv][b0], c1 = s.count[lv][b0 + 1];
  const u64 m0 = s.mass[lv][b0], m1 = s.mass[lv][b0 + 1];
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
  s.count[lv][b0] = c - c1;
  s.count[lv][b0 + 1] = c;
  s.mass[lv][b0] = m - m1;
  s.mass[lv][b0 + 1] = m;
  __syncthreads();
}

// First bin whose inclusive count or mass reaches `target`.
__device__ int find(Shared& s, int lv, bool by_mass, u64 target) {
  if (threadIdx.x == 0) s.found = kBins - 1;
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    const u64 v = by_mass ? s.mass[lv][b] : s.count[lv][b];
    const u64 p = b == 0 ? 0 : by_mass ? s.mass[lv][b - 1] : s.count[lv][b - 1];
    if (v >= target && p < target) s.found = b;  // at most one bin
  }
  __syncthreads();
  const int r = s.found;
  __syncthreads();
  return r;
}

// What top-k / top-p keep: keys above `key`, and of those equal to it the ones at or before `last`.
struct Cut {
  unsigned key;
  int last;
  u64 mass;  // of all that is kept (only with masses)
};

template <typename T>
__device__ Cut select(cg::cluster_group& cl, Shared& s, const T* sl, int chunks, int s0, const Row& row, int sel,
                      bool by_mass, bool with_mass, u64 target) {
  const int C = cl.num_blocks(), me = cl.block_rank();
  const int lane = lane_id(), w = warp_id();
  int b = find(s, 0, by_mass, target);
  unsigned before = b ? s.count[0][b - 1] : 0, inside = s.count[0][b] - before;
  u64 mbefore = b ? s.mass[0][b - 1] : 0, minside = s.mass[0][b] - mbefore;
  // the smallest and largest key in the bin
  unsigned lo = 0xffffffffu, hi = 0;
  for_chunks(sl, chunks, [&](int, int, const float(&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (bin_of(v[e], row) == b) {
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
  // all that is in the bin is kept: no need to look inside
  auto whole = [&]() { return inside == 1 || (by_mass ? mbefore + minside == target : before + inside == target); };
  while (hi != lo && !whole()) {
    const int shift = max(0, 32 - __clz(hi - lo) - 10);
    clear_hist(s);
    __syncthreads();
    for_chunks(sl, chunks, [&](int, int, const float(&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned k = key_of(v[e]);
        if (k >= lo && k <= hi)
          hist_add(s, (hi - k) >> shift, with_mass, with_mass ? mass_of(v[e], row, s.tab) : 0);
      }
    });
    combine(cl, s, 1);
    b = find(s, 1, by_mass, target - (by_mass ? mbefore : before));
    const unsigned cb = b ? s.count[1][b - 1] : 0;
    const u64 mb = b ? s.mass[1][b - 1] : 0;
    inside = s.count[1][b] - cb;
    minside = s.mass[1][b] - mb;
    before += cb;
    mbefore += mb;
    const unsigned top = hi - (static_cast<unsigned>(b) << shift);
    lo = max(lo, top - ((1u << shift) - 1u));
    hi = top;
  }
  Cut cut;
  cut.key = lo;
  cut.last = 0x7fffffff;
  cut.mass = mbefore + minside;
  if (whole()) return cut;
  // equal values: the first `r` of them by index
  const u64 one = with_mass ? mass_of(value_of(lo), row, s.tab) : 0;
  const u64 r = by_mass ? (one ? (target - mbefore + one - 1) / one : 1) : target - before;
  if (r >= inside) return cut;
  cut.mass = mbefore + r * one;
  unsigned mine = 0;
  for_chunks(sl, chunks, [&](int, int, const float(&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mine += key_of(v[e]) == lo;
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
      for (int e = 0; e < 8; ++e) hit |= (key_of(clean<T>(p[e])) == lo ? 1u : 0u) << e;
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
  cut.last = s.cl_index;
  return cut;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) draw_kernel(const Args a) {
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

  // ---- the slice into shared memory (NaN and the padding as -inf), its maximum
  if (threadIdx.x < kTab) s.tab[threadIdx.x] = exp2(threadIdx.x / double(kTab));
  float best = -INFINITY;
  int arg = 0x7fffffff;
  auto take = [&](int i, T raw_v) {
    const float v = clean<T>(raw_v);
    if (v > best) best = v, arg = s0 + i;  // a thread sees rising indexes: the first of equal ones stays
    return static_cast<T>(v);
  };
  constexpr int kVec = 16 / sizeof(T);
  int done = 0;
  if (a.vec) {
    const int nv = n / kVec;
    for (int i = threadIdx.x; i < nv; i += kThreads) {
      uint4 x = __ldg(reinterpret_cast<const uint4*>(row) + i);
      T* e = reinterpret_cast<T*>(&x);
#pragma unroll
      for (int q = 0; q < kVec; ++q) e[q] = take(i * kVec + q, e[q]);
      reinterpret_cast<uint4*>(sl)[i] = x;
    }
    done = nv * kVec;
  }
  for (int i = done + threadIdx.x; i < chunks * kChunk; i += kThreads)
    sl[i] = i < n ? take(i, row[i]) : static_cast<T>(-INFINITY);
  auto better = [&](float v, int i) {
    if (v > best || (v == best && i < arg)) best = v, arg = i;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    better(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, arg, o));
  if (lane == 0) s.red_f[w] = best, s.red_i[w] = arg;
  cl.sync();  // also: every CTA of the cluster runs, so its shared memory may be written
  if (threadIdx.x < C) {
    for (int i = 0; i < kWarps; ++i) better(s.red_f[i], s.red_i[i]);
    Shared* o = remote(cl, &s, threadIdx.x);
    o->cl_max[me] = best;
    o->cl_arg[me] = arg;
  }
  cl.sync();
  for (int r = 0; r < C; ++r) better(s.cl_max[r], s.cl_arg[r]);

  const float t = a.temp[b];
  int* out = a.out + (long)b * a.draws;
  if (!(t > 0.f) || best == -INFINITY) {  // greedy, or nothing to draw from
    if (me == 0)
      for (int d = threadIdx.x; d < a.draws; d += kThreads) out[d] = best == -INFINITY ? -1 : arg;
    return;  // the whole cluster; nothing of it is written any more
  }
  // every thread holds the row's maximum: `best` of other warps saw all of cl_max too
  Row r;
  r.mx = best;
  r.mxd = best;
  r.inv_t = 1.0 / static_cast<double>(t);
  r.inv_tf = static_cast<float>(r.inv_t);
  const float mp = a.min_p != nullptr ? a.min_p[b] : 0.f;
  r.min_w = mp > 0.f ? fmin(1.0, static_cast<double>(mp)) : 0.0;
  const int k = a.top_k != nullptr ? a.top_k[b] : 0;
  const float p = a.top_p != nullptr ? a.top_p[b] : 1.f;
  const bool need_k = k > 0 && k < a.V, need_p = p > 0.f && p < 1.f;
  Cut cut{0u, 0x7fffffff, 0ull};
  if (need_k || need_p) {
    clear_hist(s);
    __syncthreads();
    for_chunks(sl, chunks, [&](int, int, const float(&v)[8]) {
#pragma unroll
      for (int e = 0; e < 8; ++e) hist_add(s, bin_of(v[e], r), need_p, need_p ? mass_of(v[e], r, s.tab) : 0);
    });
    combine(cl, s, 0);
    u64 z = s.mass[0][kBins - 1];
    if (need_k) {
      cut = select(cl, s, sl, chunks, s0, r, 0, false, need_p, static_cast<u64>(k));
      z = cut.mass;
    }
    if (need_p) {
      const u64 target = static_cast<u64>(ceil(static_cast<double>(p) * static_cast<double>(z)));
      cut = select(cl, s, sl, chunks, s0, r, 1, true, true, target > 0 ? target : 1);
    }
  }
  // mass of token `i` of the slice if it is kept
  auto kept = [&](float v, int i) -> u64 {
    const unsigned key = key_of(v);
    if (key < cut.key || (key == cut.key && s0 + i > cut.last)) return 0;
    const double x = weight(v, r, s.tab);
    return x >= r.min_w ? fixed(x) : 0;
  };
  // ---- sums of 256 tokens in vocabulary order
  for_chunks(sl, chunks, [&](int c, int i, const float(&v)[8]) {
    u64 m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m += kept(v[e], i + e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    if (lane == 0) csum[c] = m;
  });
  __syncthreads();
  if (w == 0) {  // inclusive scan of the chunk sums
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
      m[e] = kept(clean<T>(sl[i + e]), i + e);
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
  C10_CUDA_CHECK(cudaFuncSetAttribute(draw_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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

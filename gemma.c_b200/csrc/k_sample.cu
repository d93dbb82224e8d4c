// k_sample.cu -- the next token of each row of logits, from given random numbers.
//
//   w_j = exp((x_j - max) / T);  top-k, top-p, min-p;  the first kept index whose
//   running sum of weights passes u * total.
//
// Weights are 64-bit fixed point, round(w * 2^b) with the largest b up to 51 at
// which n equal logits' sum fits (45 for 262144 logits): their sums are whole
// numbers, the same in every order, so the token does not depend on how the row
// is split.  A weight below 2^-(b + 1) of the largest is zero.
//
// Top-k and top-p both keep the logits down to a cut in the order (value
// descending, index ascending).  A histogram over (max - x) / T in steps of 1/128
// (counts, and for top-p the weights) finds the step that holds the cut.  When all
// that lies above its end is a short list, that list is gathered and sorted, and
// one CTA ends the search on it; otherwise the step's few elements are gathered
// and sorted for the cut (key, index), and all CTAs sum what it keeps.  A step with
// too many elements is split by its float keys until they fit or are all equal,
// and then the cut is an index.
//
// One cluster of 2 to 16 CTAs per row: every CTA scans its contiguous slice, from
// shared memory where it fits (n / CTAs up to 32768) or again from L2, histograms and
// lists meet in distributed shared memory, and the whole search is one launch
// with one read of HBM.  One row is bound by the latency of the passes and their cluster
// barriers.  In batches a slice is longer than what is held and is read from L2 in every
// pass, four loads a thread in flight; the 64-bit weights, 12 instructions of the FP64 units
// each, are about 6.5 us a pass over 65536 logits.
// 262144 logits, top-p 0.9 and min-p: 26 us for a row (16 CTAs), 36 for 8 rows (8), 70 for
// 32 (4; clusters of 8, of which 15 run at once, took 116); top-k 64 and top-p 15 us for a
// row, 19 with every list sorted by exchanges.
#include "gcu_internal.cuh"

#include <cooperative_groups.h>

#include <mutex>
#include <utility>

#define GCU_EXPORT extern "C" __attribute__((visibility("default")))

namespace gcu {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr int kBins = 2048;
constexpr float kBinsPerNat = 128.0f;
constexpr int kCap = 1024;                // elements that are sorted
constexpr int kFew = 256;                 // and up to how many by counting
constexpr int kKeep = 1024;               // logits per warp held in shared memory
constexpr int kTable = 32;                // entries of the 2^(j/32) table, one per lane

typedef unsigned long long u64;

struct SampleArgs {
  int *token;
  float *prob;
  const float *logits;
  long ld;
  const float *u;
  float temperature, top_p, min_p;
  int top_k, m, n;
  double one;  // 2^b, the largest weight
};

// float keys: unsigned order = value order; NaN below every number, -0 = +0
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x == x)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct Shared {
  unsigned int lo[kBins], hi[kBins];  // histogram of this CTA's slice
  u64 sum[kBins];                     // of the row
  u64 found[kCap];                    // what this CTA gathers: (~key, index)
  u64 list[kCap];                     // rank 0: all that is gathered, sorted ascending
  u64 weight[kCap];
  unsigned int order[kCap];
  unsigned int place[kFew];
  u64 warp_sum[kWarps], totals[kMaxCluster];
  float maxes[kMaxCluster];
  u64 cta_sum, before;
  u64 upto;
  unsigned int nfound, klo, khi;
  int bin, cut_idx;
  uint32_t cut_key;
  u64 need;
  float values[kWarps * kKeep];
};

struct Row {
  const float *x;       // the row
  const float *held;    // this warp's slice in shared memory
  bool holds;           // whether it is there
  double table;         // 2^(lane/32)
  int w0, w1;           // this warp's contiguous elements
  float max;
  bool inf;             // the largest logit is +inf: those count as 0, all others as -inf
  double max_d, scale;  // scale: log2(e) / T
  float least;          // logits below it weigh nothing
  double one;
  float half_max, bin_scale;

  // one * 2^((v - max) * log2(e) / T), rounded to a whole number, to 2^-39 of itself;
  // the whole warp calls it.  t = k/32 + r; 2^r by its Taylor series to r^4 (|r| <=
  // 1/64: the rest is below 2^-39); 2^(j/32) from the table (Tang's method), which
  // the lanes hold: two shuffles cost half of a gather from shared memory; the sum
  // with 2^52 leaves the whole number in the low bits.
  __device__ __forceinline__ u64 weight(float v) const {
    constexpr double shift = 6755399441055744.0 / kTable;  // 1.5 * 2^52 / 32: rounds to 32nds
    const double t = ((double)v - max_d) * scale, z = t + shift;
    const int k = __double2loint(z);
    const double r = t - (z - shift);
    double p = 9.6181291076284772e-3;  // ln(2)^i / i!, i = 4 .. 1
    p = fma(p, r, 5.5504108664821580e-2);
    p = fma(p, r, 2.4022650695910071e-1);
    p = fma(p, r, 6.9314718055994531e-1);
    const double w = __shfl_sync(0xffffffffu, table, k & (kTable - 1));
    // one * 2^n through its exponent (2^42 * 2^-64 stays normal)
    const double s = __hiloint2double(__double2hiint(one) + ((k >> 5) << 20), __double2loint(one));
    const u64 f = (u64)__double_as_longlong(fma(fma(w * r, p, w), s, 4503599627370496.0)) & 0xfffffffffffffull;
    return v < least ? 0 : f;
  }
  // steps of 1/128 below the largest; monotone in v.  Half the distance, which fits where
  // the distance of two logits past 1.7e38 does not, times twice the scale.
  __device__ __forceinline__ int bin(float v) const {
    return min((int)(__fmaf_rn(-0.5f, v, half_max) * bin_scale), kBins - 1);
  }
  // About the logit `off` bins above the start of a bin: with 0.01 above all of the
  // bin, with -1.01 below all of it (the last has no end).  bin()'s roundings are
  // 2^-22 of 2048 bins at most, and those of the logits' own size are allowed for.
  __device__ __forceinline__ float edge(int bin, double off) const {
    if (off < 0.0 && bin == kBins - 1) return -INFINITY;
    const double x = max_d - (bin - off) * 2.0 / (double)bin_scale;
    const double slack = (fabs(max_d) + fabs(x)) * 2.4e-7;
    return (float)(off < 0.0 ? x - slack : x + slack);
  }
  // a logit as it counts: NaN as -inf, -0 as +0
  __device__ __forceinline__ float counted(float v) const {
    if (inf) return v == INFINITY ? 0.0f : -INFINITY;
    return v == v ? v + 0.0f : -INFINITY;
  }
  // The warp's elements, 4 x 32 consecutive ones at a time, lane l's j-th at index +
  // 32 j + l: f(index, values), every lane; past the end -inf.  Four at a time so
  // that their arithmetic overlaps.
  template <typename F>
  __device__ __forceinline__ void each4(int lane, F f) const {
    if (holds) {
      for (int b = w0; b < w1; b += 128) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = held[b - w0 + 32 * j + lane];
        f(b + lane, v);
      }
      return;
    }
    float next[4];
    auto fetch = [&](int b) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = b + 32 * j + lane;
        next[j] = i < w1 ? __ldg(x + i) : -INFINITY;
      }
    };
    fetch(w0);
    for (int b = w0; b < w1; b += 128) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = counted(next[j]);
      fetch(b + 128);
      f(b + lane, v);
    }
  }
  // f(index, value), one at a time
  template <typename F>
  __device__ __forceinline__ void each(int lane, F f) const {
    each4(lane, [&](int i, const float (&v)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f(i + 32 * j, v[j]);
    });
  }
};

__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// exclusive prefix over the warps of each one's `v` (lane 0's), in warp order;
// the CTA's total in s.cta_sum after the next barrier
__device__ __forceinline__ u64 cta_prefix(Shared &s, u64 v, int warp, int lane) {
  __syncthreads();
  if (lane == 0) s.warp_sum[warp] = v;
  __syncthreads();
  const u64 mine = s.warp_sum[lane], incl = warp_scan(mine, lane);
  if (threadIdx.x == kThreads - 1) s.cta_sum = incl;
  const u64 p = __shfl_sync(0xffffffffu, incl - mine, warp);
  __syncthreads();
  return p;
}
// inclusive prefix over the CTA's threads
__device__ __forceinline__ u64 cta_scan(Shared &s, u64 v, int warp, int lane) {
  const u64 incl = warp_scan(v, lane);
  return incl + cta_prefix(s, __shfl_sync(0xffffffffu, incl, 31), warp, lane);
}

// A cut: kept are the elements with (v > value) or (v == value and index <= idx); at
// first all but -inf.
struct Cut {
  float value = -INFINITY;
  int idx = -1;
  __device__ __forceinline__ bool keeps(float v, int i) const { return v > value || (v == value && i <= idx); }
};

__device__ __forceinline__ int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}
// ascending sort of n <= kCap different elements.  Up to kFew: an element's place is
// the number of smaller ones, each counted over a share of the list by 1024 / n
// threads (broadcast reads).  More: bitonic, one element per thread, partners within a
// warp by shuffles; the array's places up to the next power of two are filled.
template <typename T>
__device__ void sort(T *a, int n, unsigned int *place) {
  const int tid = threadIdx.x, n2 = max(32, pow2_at_least(n));
  __syncthreads();
  if (n <= kFew) {
    const int e = tid & (n2 - 1), parts = kThreads / n2, share = (n + parts - 1) / parts, from = tid / n2 * share;
    const T x = e < n ? a[e] : T(0);
    if (tid < kFew) place[tid] = 0;
    unsigned int less = 0;
    for (int j = from; j < min(n, from + share); ++j) less += a[j] < x;
    __syncthreads();
    if (e < n && less) atomicAdd(&place[e], less);
    __syncthreads();
    if (tid < n) a[place[tid]] = x;
    __syncthreads();
    return;
  }
  T x = tid < n ? a[tid] : T(~T(0));
  for (int size = 2; size <= n2; size <<= 1)
    for (int d = size >> 1; d > 0; d >>= 1) {
      T y;
      if (d >= 32) {
        __syncthreads();
        if (tid < n2) a[tid] = x;
        __syncthreads();
        y = tid < n2 ? a[tid ^ d] : T(0);
      } else {
        y = __shfl_xor_sync(0xffffffffu, x, d);
      }
      // the lower of a pair keeps the smaller in an ascending block
      if (((tid & d) == 0) == ((tid & size) == 0) ? y < x : y > x) x = y;
    }
  __syncthreads();
  if (tid < n2) a[tid] = x;
  __syncthreads();
}
__device__ __forceinline__ float list_value(u64 e) { return value_of(~(uint32_t)(e >> 32)); }

// The row's histogram of the elements that bin_of(index, value) gives a bin (not
// -1), of their number or (MASS) their weights, in every CTA's sum.
template <int C, bool MASS, typename B>
__device__ void histogram(cg::cluster_group &cl, Shared &s, const Row &r, B bin_of) {
  const int tid = threadIdx.x, lane = tid & 31, rank = cl.block_rank();
  for (int b = tid; b < kBins; b += kThreads) {
    s.lo[b] = 0;
    if (MASS) s.hi[b] = 0;
  }
  __syncthreads();
  r.each4(lane, [&](int i, const float (&v)[4]) {
    u64 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = MASS ? r.weight(v[j]) : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int b = bin_of(i + 32 * j, v[j]);
      if (b < 0 || (MASS && w[j] == 0)) continue;
      const unsigned int lo = MASS ? (unsigned int)w[j] : 1u, old = atomicAdd(&s.lo[b], lo);
      if (MASS) {  // 64-bit additions in shared memory are a compare-and-swap loop: two of 32 bits
        const unsigned int hi = (unsigned int)(w[j] >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&s.hi[b], hi);
      }
    }
  });
  cl.sync();
  // each CTA sums its share of the bins over the cluster and hands it to all
  constexpr int kShare = kBins / C;
  if (tid < kShare) {
    const int b = rank * kShare + tid;
    u64 n = 0;
#pragma unroll
    for (int p = 0; p < C; ++p) {
      const Shared &o = *cl.map_shared_rank(&s, p);
      n += o.lo[b];
      if (MASS) n += (u64)o.hi[b] << 32;
    }
#pragma unroll
    for (int p = 0; p < C; ++p) cl.map_shared_rank(&s, p)->sum[b] = n;
  }
  cl.sync();
}

// The first bin of the row's histogram at which the running sum, which starts at
// `before`, reaches the target: s.bin (-1: none), the sum before it and with it
// (s.before, s.upto).  The same in every CTA.
__device__ void find_bin(Shared &s, u64 before, double target, int warp, int lane) {
  constexpr int J = kBins / kThreads;
  const int tid = threadIdx.x;
  if (tid == 0) s.bin = -1;
  u64 v[J], t = 0;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    v[j] = s.sum[tid * J + j];
    t += v[j];
  }
  u64 run = before + cta_scan(s, t, warp, lane) - t;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    // sums of whole numbers only grow, also rounded to doubles: one bin at most
    if (v[j] && (double)run < target && (double)(run + v[j]) >= target) {
      s.bin = tid * J + j;
      s.before = run;
      s.upto = run + v[j];
    }
    run += v[j];
  }
  __syncthreads();
}

// Elements that pass `in`, to rank 0's list; their number, in every CTA.  More than
// kCap: the list is not made.  None lies outside [lo, hi]: a cheaper test that most
// groups of 128 elements end with.
template <int C, typename P>
__device__ int gather(cg::cluster_group &cl, Shared &s, const Row &r, float lo, float hi, P in) {
  const int tid = threadIdx.x, lane = tid & 31, rank = cl.block_rank();
  if (tid == 0) s.nfound = 0;
  __syncthreads();
  r.each4(lane, [&](int i, const float (&v)[4]) {
    bool may = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) may |= v[j] >= lo && v[j] <= hi;
    if (!__any_sync(0xffffffffu, may)) return;  // the whole warp
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool hit = v[j] >= lo && v[j] <= hi && in(i + 32 * j, v[j]);
      const unsigned int b = __ballot_sync(0xffffffffu, hit);
      if (!b) continue;
      unsigned int at = 0;
      if (lane == 0) at = atomicAdd(&s.nfound, (unsigned int)__popc(b));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(b & ((1u << lane) - 1));
      if (hit && at < kCap) s.found[at] = ((u64)~key_of(v[j]) << 32) | (unsigned int)(i + 32 * j);
    }
  });
  __syncthreads();
  if (tid < C) cl.map_shared_rank(&s, tid)->totals[rank] = s.nfound;
  cl.sync();
  u64 before = 0, all = 0;
  for (int q = 0; q < C; ++q) {
    if (q < rank) before += s.totals[q];
    all += s.totals[q];
  }
  if (all <= kCap && tid < (int)s.nfound) cl.map_shared_rank(&s, 0)->list[before + tid] = s.found[tid];
  cl.sync();
  return all <= kCap ? (int)all : kCap + 1;
}

// rank 0: the first element of the sorted list at which the running sum reaches
// the target; its place in s.cut_idx, or nl when there is none
template <bool MASS>
__device__ int cut_list(Shared &s, int nl, u64 before, double target, int warp, int lane) {
  const int tid = threadIdx.x;
  if (tid == 0) s.cut_idx = nl;
  const u64 v = tid >= nl ? 0 : MASS ? s.weight[tid] : 1;
  const u64 run = before + cta_scan(s, v, warp, lane) - v;
  if (v && (double)run < target && (double)(run + v) >= target) s.cut_idx = tid;
  __syncthreads();
  return s.cut_idx;
}

// rank 0: sorts its list of nl elements and fills in their weights
__device__ void sort_list(Shared &s, const Row &r, int nl) {
  const int tid = threadIdx.x;
  sort(s.list, nl, s.place);
  const u64 w = r.weight(tid < nl ? list_value(s.list[tid]) : r.max);
  if (tid < nl) s.weight[tid] = w;
  __syncthreads();
}

// The search for one cut among the elements that `c` keeps, whatever its size.
// Starts from find_bin's answer over the linear bins.  c is left as it is when the
// elements never reach the target.
template <int C, bool MASS>
__device__ void find_cut(cg::cluster_group &cl, Shared &s, const Row &r, Cut &c, double target) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = cl.block_rank();
  Shared &s0 = *cl.map_shared_rank(&s, 0);
  uint32_t klo = 0, khi = 0xffffffffu, step = 0;  // level 0: linear bins; then keys
  auto key_bin = [&](int i, float v) {
    const uint32_t key = key_of(v);
    return c.keeps(v, i) && key >= klo && key <= khi ? (int)((khi - key) / step) : -1;
  };
  for (int level = 0; s.bin >= 0; ++level) {
    const int bin = s.bin;
    const u64 before = s.before;
    auto here = [&](int i, float v) { return level == 0 ? c.keeps(v, i) && r.bin(v) == bin : key_bin(i, v) == bin; };
    const float top = level == 0 ? r.edge(bin, 0.01) : value_of(khi - bin * step);
    const int nbin = gather<C>(cl, s, r, level == 0 ? r.edge(bin, -1.01) : -INFINITY, top, here);
    if (nbin <= kCap) {
      if (rank == 0) {
        sort_list(s, r, nbin);
        const int at = min(cut_list<MASS>(s, nbin, before, target, warp, lane), nbin - 1);
        if (tid < C) {
          Shared &o = *cl.map_shared_rank(&s, tid);
          o.cut_key = ~(uint32_t)(s.list[at] >> 32);
          o.need = (u64)(uint32_t)s.list[at];
        }
      }
      cl.sync();
      c.value = value_of(s.cut_key);
      c.idx = (int)s.need;
      return;
    }
    // the bin's range of keys
    unsigned int lo = 0xffffffffu, hi = 0;
    r.each(lane, [&](int i, float v) {
      if (here(i, v)) {
        lo = min(lo, key_of(v));
        hi = max(hi, key_of(v));
      }
    });
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) {
      atomicMin(&s0.klo, lo);
      atomicMax(&s0.khi, hi);
    }
    cl.sync();
    klo = s0.klo;
    khi = s0.khi;
    cl.sync();  // read by all
    if (tid == 0) {
      s.klo = 0xffffffffu;
      s.khi = 0;
    }
    if (klo == khi) {
      // all equal: the cut is the index of one of them, counted in index order
      const float tie = value_of(klo);
      u64 need;
      if (MASS) {
        const u64 w = r.weight(tie);
        need = (u64)((target - (double)before) / (double)w);
        while (need && (double)(before + need * w) >= target) --need;
        while ((double)(before + need * w) < target) ++need;
      } else {
        need = (u64)target - before;
      }
      u64 mine = 0;
      r.each(lane, [&](int i, float v) { mine += c.keeps(v, i) && v == tie; });
      mine = warp_total(mine);
      u64 p = cta_prefix(s, mine, warp, lane);
      if (tid < C) cl.map_shared_rank(&s, tid)->totals[rank] = s.cta_sum;
      cl.sync();
      for (int q = 0; q < rank; ++q) p += s.totals[q];
      if (p < need && need <= p + mine) {  // this warp holds it
        r.each(lane, [&](int i, float v) {
          const bool hit = c.keeps(v, i) && v == tie;
          const unsigned int b = __ballot_sync(0xffffffffu, hit);
          if (hit && p + __popc(b & ((2u << lane) - 1)) == need)
            for (int q = 0; q < C; ++q) cl.map_shared_rank(&s, q)->cut_idx = i;
          p += __popc(b);
        });
      }
      cl.sync();
      c.value = tie;
      c.idx = s.cut_idx;
      return;
    }
    step = (khi - klo) / kBins + 1;
    histogram<C, MASS>(cl, s, r, key_bin);
    find_bin(s, before, target, warp, lane);
  }
}

// rank 0: the whole choice on its sorted list of nl elements, which holds all that
// may be kept; all_mass: the sum that top-p's share is of (0: what top-k keeps)
__device__ void choose_from_list(Shared &s, const SampleArgs &a, const Row &r, int row, int nl, u64 all_mass) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  sort_list(s, r, nl);
  if (a.top_k > 0) nl = min(nl, a.top_k);
  if (a.top_p < 1.0f) {
    if (!all_mass) {
      const u64 t = cta_scan(s, tid < nl ? s.weight[tid] : 0, warp, lane);
      if (tid == kThreads - 1) s.need = t;
      __syncthreads();
      all_mass = s.need;
    }
    nl = min(nl, cut_list<true>(s, nl, 0, (double)a.top_p * (double)all_mass, warp, lane) + 1);
  }
  // in index order (index, place), what min-p drops without weight
  if (tid < nl) s.order[tid] = (unsigned int)s.list[tid] << 10 | tid;
  sort(s.order, nl, s.place);
  u64 w = 0;
  if (tid < nl) {
    w = s.weight[s.order[tid] & (kCap - 1)];
    if ((double)w < (double)a.min_p * r.one) w = 0;
  }
  const u64 incl = cta_scan(s, w, warp, lane);
  if (tid == kThreads - 1) s.need = incl;
  __syncthreads();
  const u64 total = s.need;
  const float uf = __ldg(a.u + row);
  const double u = uf > 0.0f ? (double)uf : 0.0;  // NaN and below: 0
  u64 target = (u64)(u * (double)total);
  if (u >= 1.0 || target >= total) target = total - 1;
  if (incl > target && incl - w <= target) {
    a.token[row] = (int)(s.order[tid] >> 10);
    if (a.prob) a.prob[row] = (float)((double)w / (double)total);
  }
}

template <int C>
__global__ void __launch_bounds__(kThreads) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared &s = *reinterpret_cast<Shared *>(raw);
  ptx::griddep_launch();
  cg::cluster_group cl = cg::this_cluster();
  auto started = cl.barrier_arrive();  // waited for before the first access to another CTA
  const int rank = cl.block_rank(), row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // contiguous slices of CTAs and warps, in index order, multiples of 128
  const int per_warp = ((a.n + C * kWarps - 1) / (C * kWarps) + 127) & ~127;
  Row r;
  r.x = a.logits + (long)row * a.ld;
  r.w0 = min(a.n, (rank * kWarps + warp) * per_warp);
  r.w1 = min(a.n, r.w0 + per_warp);
  r.held = s.values + warp * kKeep;
  r.holds = per_warp <= kKeep;
  r.inf = false;
  r.table = exp2((double)lane / kTable);
  if (tid == 0) {
    s.klo = 0xffffffffu;
    s.khi = 0;
  }
  ptx::griddep_wait();
  float top = -INFINITY;
  if (r.holds) {
    float *hold = s.values + warp * kKeep;
    for (int b = lane; b - lane < r.w1 - r.w0; b += 256) {
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = r.w0 + b + 32 * j;
        v[j] = i < r.w1 ? __ldg(r.x + i) : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[j] = r.counted(v[j]);
        top = fmaxf(top, v[j]);
        if (b + 32 * j < kKeep) hold[b + 32 * j] = v[j];
      }
    }
    __syncwarp();
  } else {
    r.each(lane, [&](int, float v) { top = fmaxf(top, v); });
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float *warp_max = reinterpret_cast<float *>(s.warp_sum);
  if (lane == 0) warp_max[warp] = top;
  __syncthreads();
  top = warp_max[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  cl.barrier_wait(std::move(started));
  if (tid < C) cl.map_shared_rank(&s, tid)->maxes[rank] = top;
  cl.sync();
  r.max = s.maxes[0];
  for (int p = 1; p < C; ++p) r.max = fmaxf(r.max, s.maxes[p]);
  if (r.max == -INFINITY) {  // nothing to choose from
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      if (a.prob) a.prob[row] = 0.0f;
    }
    return;
  }
  if (a.temperature == 0.0f) {
    // the first CTA whose slice has the largest logit knows that it is the first
    bool mine = s.maxes[rank] == r.max;
    for (int p = 0; p < rank; ++p) mine &= s.maxes[p] != r.max;
    if (!mine) return;
    int at = 0x7fffffff;
    r.each(lane, [&](int i, float v) {
      if (v == r.max) at = min(at, i);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    __syncthreads();
    int *warp_at = reinterpret_cast<int *>(s.warp_sum);
    if (lane == 0) warp_at[warp] = at;
    __syncthreads();
    at = __reduce_min_sync(0xffffffffu, warp_at[lane]);
    if (tid == 0) {
      a.token[row] = at;
      if (a.prob) a.prob[row] = 1.0f;
    }
    return;
  }
  if (r.max == INFINITY) {
    r.inf = true;
    r.max = 0.0f;
    float *hold = s.values + warp * kKeep;
    if (r.holds)
      for (int i = lane; i < kKeep; i += 32) hold[i] = r.counted(hold[i]);
    __syncwarp();
  }
  r.scale = 1.4426950408889634 / (double)a.temperature;
  r.max_d = (double)r.max;
  r.least = fmaxf((float)(r.max_d - 63.0 / r.scale), -3.4028235e38f);  // -inf lies below it
  r.half_max = 0.5f * r.max;
  r.bin_scale = fminf(2.0f * kBinsPerNat / a.temperature, 3.4028235e38f);  // 0 times it is 0
  r.one = a.one;
  Cut c;
  const bool by_k = a.top_k > 0 && a.top_k < a.n, by_p = a.top_p < 1.0f;
  // all that lies up to the end of the bin, as one list
  auto list_upto = [&](int bin) {
    return gather<C>(cl, s, r, r.edge(bin, -1.01), INFINITY,
                     [&](int, float v) { return v > -INFINITY && r.bin(v) <= bin; });
  };
  if (by_k) {
    histogram<C, false>(cl, s, r, [&](int, float v) { return v > -INFINITY ? r.bin(v) : -1; });
    find_bin(s, 0, (double)a.top_k, warp, lane);
    if (s.bin >= 0 && s.upto <= kCap) {
      const int nl = list_upto(s.bin);
      if (rank == 0) choose_from_list(s, a, r, row, nl, 0);
      return;
    }
    find_cut<C, false>(cl, s, r, c, (double)a.top_k);
  }
  if (by_p) {
    if (by_k) {
      histogram<C, true>(cl, s, r, [&](int i, float v) { return c.keeps(v, i) ? r.bin(v) : -1; });
    } else {
      histogram<C, true>(cl, s, r, [&](int, float v) { return r.bin(v); });
    }
    u64 all = s.sum[tid * 2] + s.sum[tid * 2 + 1];
    cta_scan(s, all, warp, lane);
    all = s.cta_sum;
    const double target = (double)a.top_p * (double)all;
    find_bin(s, 0, target, warp, lane);
    // every element up to the end of the bin weighs at least this: a bound on their number
    const double edge = exp2(-(double)(s.bin + 2) / kBinsPerNat * 1.4426950408889634) * r.one;
    if (!by_k && s.bin >= 0 && s.bin < kBins - 1 && (double)s.upto <= kCap * edge) {
      const int nl = list_upto(s.bin);
      if (rank == 0) choose_from_list(s, a, r, row, nl, all);
      return;
    }
    find_cut<C, true>(cl, s, r, c, target);
  }
  const double least = (double)a.min_p * r.one;
  auto kept = [&](int i, float v) -> u64 {
    const u64 w = r.weight(v);
    return c.keeps(v, i) && (double)w >= least ? w : 0;
  };
  // what the cuts keep, often few, moves to the front of the warp's shared memory
  u64 mine = 0;
  float *hold = s.values + warp * kKeep;
  int n = 0;
  auto weigh = [&]() {
    __syncwarp();
#pragma unroll 4
    for (int b = 0; b < n; b += 32) {
      const u64 w = r.weight(b + lane < n ? hold[b + lane] : -INFINITY);
      mine += (double)w >= least ? w : 0;
    }
    __syncwarp();
    n = 0;
  };
  if (!by_k && !by_p) {  // all but -inf, which weighs nothing
    r.each4(lane, [&](int, const float (&v)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 w = r.weight(v[j]);
        mine += (double)w >= least ? w : 0;
      }
    });
  } else {
    r.each4(lane, [&](int i, const float (&v)[4]) {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = c.keeps(v[j], i + 32 * j);
        const unsigned int b = __ballot_sync(0xffffffffu, in);
        if (in) hold[n + __popc(b & ((1u << lane) - 1))] = v[j];
        n += __popc(b);
      }
      if (!r.holds && n > kKeep - 128) weigh();
    });
    weigh();
  }
  mine = warp_total(mine);
  u64 p = cta_prefix(s, mine, warp, lane);
  if (tid < C) cl.map_shared_rank(&s, tid)->totals[rank] = s.cta_sum;
  cl.sync();
  u64 total = 0;
  for (int q = 0; q < C; ++q) {
    if (q < rank) p += s.totals[q];
    total += s.totals[q];
  }
  const float uf = __ldg(a.u + row);
  const double u = uf > 0.0f ? (double)uf : 0.0;  // NaN and below: 0
  u64 target = (u64)(u * (double)total);
  if (u >= 1.0 || target >= total) target = total - 1;
  // the warp that holds the token hands its elements to the whole CTA
  __syncthreads();
  if (tid == 0) s.bin = -1;
  __syncthreads();
  if (lane == 0 && p <= target && target < p + mine) {
    s.bin = warp;
    s.before = p;
  }
  __syncthreads();
  if (s.bin < 0) return;
  u64 before = s.before;
  const int first = min(a.n, (rank * kWarps + s.bin) * per_warp), last = min(a.n, first + per_warp);
  for (int b = first; b < last && before <= target; b += kThreads) {
    const int i = b + tid;
    const float v = i < last ? r.counted(__ldg(r.x + i)) : -INFINITY;
    const u64 w = kept(i, v), run = before + cta_scan(s, w, warp, lane);
    if (run > target && run - w <= target) {
      a.token[row] = i;
      if (a.prob) a.prob[row] = (float)((double)w / (double)total);
    }
    before += s.cta_sum;
  }
}

// Clusters of C CTAs that run at once on the current device (0: the size is not
// to be had), after the kernel's opt-ins; both once per device.
template <int C>
int resident(int *n) {
  constexpr int kDevices = 64;
  static std::mutex mu;
  static int known[kDevices];  // their number + 1
  int dev = 0;
  GCU_CUDA(cudaGetDevice(&dev));
  if (dev >= kDevices) return set_error("sample: device %d", dev);
  std::lock_guard<std::mutex> lk(mu);
  if (!known[dev]) {
    GCU_CUDA(cudaFuncSetAttribute(k_sample<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
    if (C > 8) GCU_CUDA(cudaFuncSetAttribute(k_sample<C>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3(C);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    int c = 0;
    GCU_CUDA(cudaOccupancyMaxActiveClusters(&c, k_sample<C>, &cfg));
    known[dev] = c + 1;
  }
  *n = known[dev] - 1;
  return 0;
}

template <int C>
int launch(const SampleArgs &a, cudaStream_t st) {
  GCU_CUDA(launch_cluster_k(k_sample<C>, dim3((unsigned)a.m * C), dim3(kThreads), C, sizeof(Shared), st, a));
  return 0;
}

// Few rows are cut finely, many coarsely: a row's time is about that of kFixed
// logits in every CTA (barriers, the histogram's sums, the list) and of its slice, and
// rows beyond the resident clusters wait.
constexpr long kFixed = 16384;

template <int C>
int consider(const SampleArgs &a, long &best, int &size) {
  int n = 0;
  if (resident<C>(&n)) return 1;
  if (n == 0) return 0;
  const long time = ((long)a.m + n - 1) / n * (kFixed + a.n / C);
  if (time < best) best = time, size = C;
  return 0;
}

}  // namespace
}  // namespace gcu

using namespace gcu;

GCU_EXPORT int gcu_dev_sample(int *token, float *prob, const float *logits, long ld, const float *u,
                              float temperature, int top_k, float top_p, float min_p, int m, int nvocab,
                              void *stream) {
  if (m == 0) return 0;
  if (!token || !logits || !u) return set_error("sample: null pointer");
  if (ld == 0) ld = nvocab;
  if (m < 0 || m > (1 << 20) || nvocab < 1 || nvocab > (1 << 20) || ld < nvocab)
    return set_error("sample: %d rows of %d logits at stride %ld (1 to 2^20 of each)", m, nvocab, ld);
  if (!(temperature >= 0.0f) || temperature == INFINITY || top_k < 0 || !(top_p > 0.0f) ||
      !(min_p >= 0.0f && min_p <= 1.0f))
    return set_error("sample: temperature %g, top_k %d, top_p %g, min_p %g (finite and >= 0; >= 0; > 0; 0 to 1)",
                     temperature, top_k, top_p, min_p);
  double one = 9223372036854775808.0;  // 2^63, halved until nvocab of them fit
  for (long n = 1; n < nvocab; n <<= 1) one *= 0.5;
  one = one > 2251799813685248.0 ? 2251799813685248.0 : one;  // and 2^51 at most, a whole number of a double
  SampleArgs a{token, prob, logits, ld, u, temperature, top_p, min_p, top_k, m, nvocab, one};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  long best = 0x7fffffffffffffffl;
  int size = 0;
  if (consider<2>(a, best, size) || consider<4>(a, best, size) || consider<8>(a, best, size) ||
      consider<16>(a, best, size))
    return 1;
  switch (size) {
    case 2: return launch<2>(a, st);
    case 4: return launch<4>(a, st);
    case 8: return launch<8>(a, st);
    case 16: return launch<16>(a, st);
  }
  return set_error("sample: no cluster of %d bytes of shared memory a CTA fits", (int)sizeof(Shared));
}

// k_sample.cu -- the next token of each row of logits, from given random numbers.
//
//   w_j = exp((x_j - max) / T);  top-k, top-p, min-p;  the first kept index whose
//   running sum of weights passes u * total.
//
// Weights are 64-bit fixed point, round(w * 2^b) with the largest b at which n
// equal logits' sum fits (45 for 262144 logits): their sums are whole numbers,
// the same in every order, so the token does not depend on how the row is
// split.  A weight below 2^-(b + 1) of the largest is zero.
//
// Top-k and top-p both keep the logits down to a cut in the order (value
// descending, index ascending), so each is one search for a cut (key, index):
// a histogram over (max - x) / T in steps of 1/64 (counts, and for top-p the
// weights) finds the step that holds the cut, and the step's few elements are
// gathered and sorted.  A step with too many elements is split by its float
// keys until they fit or are all equal, and then the cut is an index.
//
// One cluster per row: every CTA scans its contiguous slice (which stays in
// its L1 after the first pass), the histograms and lists meet in distributed
// shared memory, and the whole search is one launch with one read of HBM.
// Latency-bound for a few rows: each pass is a scan of 16 K logits and a
// cluster barrier.
#include "gcu_internal.cuh"

#include <cooperative_groups.h>

#define GCU_EXPORT extern "C" __attribute__((visibility("default")))

namespace gcu {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 16;
constexpr int kBins = 2048;
constexpr float kBinsPerNat = 64.0f;
constexpr int kCap = 1024;  // elements that are sorted

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
constexpr uint32_t kNegInf = 0x007fffffu;  // key_of(-inf); keys up to it are never kept

struct Shared {
  unsigned int count[kBins];
  unsigned int mass_lo[kBins], mass_hi[kBins];
  u64 sum_count[kBins];  // rank 0: the row's histograms
  u64 sum_mass[kBins];
  u64 list[kCap];  // rank 0: gathered (~key, index), sorted ascending
  u64 weight[kCap];
  u64 warp_sum[kWarps + 1];
  u64 cta_sum;
  unsigned int nlist, kmax, klo, khi;
  // rank 0's answers
  int bin;
  u64 before, nbin;
  uint32_t cut_key;
  int cut_idx;
  int argmax;
};

struct Row {
  const float *x;
  int w0, w1;  // this warp's contiguous elements
  float max;
  bool inf;  // the largest logit is +inf
  double inv_t, one;
  float inv_tf;

  // w as a 64-bit float, of the largest
  __device__ __forceinline__ double weight(float v) const {
    if (inf) return v == max ? 1.0 : 0.0;
    return exp(((double)v - (double)max) * inv_t);
  }
  __device__ __forceinline__ u64 fixed(float v) const { return __double2ull_rn(weight(v) * one); }
  // steps of 1/64 below the largest; monotone in v
  __device__ __forceinline__ int bin(float v) const {
    if (inf) return v == max ? 0 : kBins - 1;
    const float t = (max - v) * inv_tf * kBinsPerNat;
    return t < (float)(kBins - 1) ? (int)t : kBins - 1;
  }
  // f(index, value) over the warp's elements, 32 consecutive ones at a time
  // (every lane calls f; index >= w1 for lanes past the end, with -inf)
  template <typename F>
  __device__ __forceinline__ void each(int lane, F f) const {
    for (int b = w0; b < w1; b += 128) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = b + 32 * j + lane;
        v[j] = i < w1 ? __ldg(x + i) : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (b + 32 * j < w1) f(b + 32 * j + lane, v[j]);
    }
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

// A cut: kept are the elements with (key > cut.key) or (key == cut.key and
// index <= cut.idx).
struct Cut {
  uint32_t key = kNegInf + 1;
  int idx = 0x7fffffff;
  __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= idx); }
};

// exclusive prefix over the warps of each one's `v` (lane 0's), in warp order;
// the CTA's total in cta_sum
__device__ __forceinline__ u64 cta_prefix(Shared &s, u64 v, int warp, int lane) {
  __syncthreads();
  if (lane == 0) s.warp_sum[warp] = v;
  __syncthreads();
  u64 p = 0, t = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) p += s.warp_sum[w];
    t += s.warp_sum[w];
  }
  if (threadIdx.x == 0) s.cta_sum = t;
  return p;
}

__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The search for one cut among the elements that `c` keeps: the first element,
// in (value descending, index ascending) order, at which the running count
// (MASS false) reaches k, or the running weight (MASS) reaches share of the
// total.  c is left as it is when the elements never reach it.
template <bool MASS>
__device__ void find_cut(cg::cluster_group &cl, Shared &s, const Row &r, Cut &c, u64 k, double share) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Shared &s0 = *cl.map_shared_rank(&s, 0);
  const int rank = cl.block_rank();
  uint32_t klo = 0, khi = 0xffffffffu;  // keys of the current range; level 0: all of them, in linear bins
  uint32_t step = 0;
  u64 before = 0;
  double target = (double)k;
  for (int level = 0;; ++level) {
    for (int b = tid; b < kBins; b += kThreads) {
      s.count[b] = 0;
      if (MASS) s.mass_lo[b] = s.mass_hi[b] = 0;
    }
    __syncthreads();
    auto bin_of = [&](uint32_t key, float v) { return level == 0 ? r.bin(v) : (int)((khi - key) / step); };
    auto in_range = [&](uint32_t key) { return key >= klo && key <= khi; };
    r.each(lane, [&](int i, float v) {
      const uint32_t key = key_of(v);
      if (i < r.w1 && c.keeps(key, i) && in_range(key)) {
        const int b = bin_of(key, v);
        atomicAdd(&s.count[b], 1u);
        if (MASS) {
          const u64 w = r.fixed(v);
          const unsigned int lo = (unsigned int)w, old = atomicAdd(&s.mass_lo[b], lo);
          atomicAdd(&s.mass_hi[b], (unsigned int)(w >> 32) + (old + lo < old ? 1u : 0u));
        }
      }
    });
    cl.sync();
    // each CTA sums a share of the bins over the cluster into rank 0
    for (int b = rank * (kBins / kCluster) + tid; b < (rank + 1) * (kBins / kCluster); b += kThreads) {
      u64 n = 0, w = 0;
      for (int p = 0; p < kCluster; ++p) {
        const Shared &o = *cl.map_shared_rank(&s, p);
        n += o.count[b];
        if (MASS) w += ((u64)o.mass_hi[b] << 32) + o.mass_lo[b];
      }
      s0.sum_count[b] = n;
      s0.sum_mass[b] = w;
    }
    cl.sync();
    if (rank == 0) {
      // prefix sums over the bins, four per thread, and the bin that holds the cut
      if (tid == 0) {
        s.bin = -1;
        s.nlist = 0;
        s.klo = 0xffffffffu;
        s.khi = 0;
      }
      u64 v[kBins / kThreads], t = 0;
#pragma unroll
      for (int j = 0; j < kBins / kThreads; ++j) {
        v[j] = MASS ? s.sum_mass[tid * (kBins / kThreads) + j] : s.sum_count[tid * (kBins / kThreads) + j];
        t += v[j];
      }
      const u64 incl = warp_scan(t, lane);
      const u64 base = cta_prefix(s, __shfl_sync(0xffffffffu, incl, 31), warp, lane);
      __syncthreads();
      if (MASS && level == 0) target = share * (double)s.cta_sum;
      u64 run = before + base + incl - t;
#pragma unroll
      for (int j = 0; j < kBins / kThreads; ++j) {
        // the first bin at which the running sum reaches the target; rounding
        // leaves no bin behind: the sums only grow
        if (v[j] && (double)run < target && (double)(run + v[j]) >= target) {
          s.bin = tid * (kBins / kThreads) + j;
          s.before = run;
          s.nbin = s.sum_count[s.bin];
        }
        run += v[j];
      }
    }
    cl.sync();
    const int bin = s0.bin;
    if (bin < 0) {
      cl.sync();  // rank 0's answer has been read by all
      return;
    }
    before = s0.before;
    const u64 nbin = s0.nbin;
    const bool fits = nbin <= kCap;
    // gather the bin's elements, or find its key range
    unsigned int lo = 0xffffffffu, hi = 0;
    r.each(lane, [&](int i, float v) {
      const uint32_t key = key_of(v);
      if (i < r.w1 && c.keeps(key, i) && in_range(key) && bin_of(key, v) == bin) {
        if (fits) {
          const unsigned int at = atomicAdd(&s0.nlist, 1u);
          if (at < kCap) s0.list[at] = ((u64)~key << 32) | (unsigned int)i;
        } else {
          lo = min(lo, key);
          hi = max(hi, key);
        }
      }
    });
    if (!fits) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      if (lane == 0) {
        atomicMin(&s0.klo, lo);
        atomicMax(&s0.khi, hi);
      }
    }
    cl.sync();
    if (fits) {
      if (rank == 0) {
        const int nl = (int)nbin;
        int n2 = 1;
        while (n2 < nl) n2 <<= 1;
        for (int i = nl + tid; i < n2; i += kThreads) s.list[i] = ~0ull;
        __syncthreads();
        for (int size = 2; size <= n2; size <<= 1)
          for (int d = size >> 1; d > 0; d >>= 1) {
            for (int i = tid; i < n2 / 2; i += kThreads) {
              const int p = 2 * i - (i & (d - 1)), q = p + d;
              const u64 x = s.list[p], y = s.list[q];
              if ((x > y) == ((p & size) == 0)) {
                s.list[p] = y;
                s.list[q] = x;
              }
            }
            __syncthreads();
          }
        constexpr int J = kCap / kThreads;
        u64 v[J], t = 0;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int i = tid * J + j;
          v[j] = i >= nl ? 0 : MASS ? r.fixed(value_of(~(uint32_t)(s.list[i] >> 32))) : 1;
          t += v[j];
        }
        const u64 incl = warp_scan(t, lane);
        u64 run = before + cta_prefix(s, __shfl_sync(0xffffffffu, incl, 31), warp, lane) + incl - t;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (v[j] && (double)run < target && (double)(run + v[j]) >= target) {
            s.cut_key = ~(uint32_t)(s.list[tid * J + j] >> 32);
            s.cut_idx = (int)(uint32_t)s.list[tid * J + j];
          }
          run += v[j];
        }
      }
      cl.sync();
      c.key = s0.cut_key;
      c.idx = s0.cut_idx;
      cl.sync();
      return;
    }
    klo = s0.klo;
    khi = s0.khi;
    if (klo == khi) {
      // all equal: the cut is the index of one of them, counted in index order
      if (rank == 0 && tid == 0) {
        u64 need;
        if (MASS) {
          const u64 w = r.fixed(value_of(klo));
          need = (u64)((target - (double)before) / (double)w);
          while (need && (double)(before + need * w) >= target) --need;
          while ((double)(before + need * w) < target) ++need;
        } else {
          need = k - before;
        }
        s.nbin = need;
        s.cut_idx = 0x7fffffff;
      }
      u64 mine = 0;
      r.each(lane, [&](int i, float v) { mine += i < r.w1 && c.keeps(key_of(v), i) && key_of(v) == klo; });
      mine = warp_total(mine);
      u64 p = cta_prefix(s, mine, warp, lane);
      cl.sync();
      const u64 need = s0.nbin;
      for (int q = 0; q < rank; ++q) p += cl.map_shared_rank(&s, q)->cta_sum;
      if (p < need && need <= p + mine) {  // this warp holds it
        r.each(lane, [&](int i, float v) {
          const bool hit = i < r.w1 && c.keeps(key_of(v), i) && key_of(v) == klo;
          const unsigned int b = __ballot_sync(0xffffffffu, hit);
          if (hit && p + __popc(b & ((2u << lane) - 1)) == need) s0.cut_idx = i;
          p += __popc(b);
        });
      }
      cl.sync();
      c.key = klo;
      c.idx = s0.cut_idx;
      cl.sync();
      return;
    }
    step = (khi - klo) / kBins + 1;
    cl.sync();  // rank 0's range has been read by all
  }
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared &s = *reinterpret_cast<Shared *>(raw);
  ptx::griddep_launch();
  cg::cluster_group cl = cg::this_cluster();
  const int rank = cl.block_rank(), row = blockIdx.x / kCluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Shared &s0 = *cl.map_shared_rank(&s, 0);
  // contiguous slices of CTAs and warps, in index order, multiples of 32
  const int per_warp = ((a.n + kCluster * kWarps - 1) / (kCluster * kWarps) + 31) & ~31;
  Row r;
  r.x = a.logits + (long)row * a.ld;
  r.w0 = min(a.n, (rank * kWarps + warp) * per_warp);
  r.w1 = min(a.n, r.w0 + per_warp);
  if (tid == 0) {
    s.kmax = 0;
    s.argmax = 0x7fffffff;
    s.cut_idx = -1;
  }
  ptx::griddep_wait();
  cl.sync();
  uint32_t km = 0;
  r.each(lane, [&](int, float v) { km = max(km, key_of(v)); });
  km = __reduce_max_sync(0xffffffffu, km);
  if (lane == 0) atomicMax(&s0.kmax, km);
  cl.sync();
  const uint32_t kmax = s0.kmax;
  if (kmax <= kNegInf) {  // nothing to choose from
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      if (a.prob) a.prob[row] = 0.0f;
    }
    cl.sync();
    return;
  }
  r.max = value_of(kmax);
  r.inf = r.max == INFINITY;
  if (a.temperature == 0.0f) {
    int at = 0x7fffffff;
    r.each(lane, [&](int i, float v) {
      if (i < r.w1 && key_of(v) == kmax) at = min(at, i);
    });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) atomicMin(&s0.argmax, at);
    cl.sync();
    if (rank == 0 && tid == 0) {
      a.token[row] = s.argmax;
      if (a.prob) a.prob[row] = 1.0f;
    }
    return;
  }
  r.one = a.one;
  r.inv_t = 1.0 / (double)a.temperature;
  r.inv_tf = 1.0f / a.temperature;
  Cut c;
  if (a.top_k > 0 && a.top_k < a.n) find_cut<false>(cl, s, r, c, (u64)a.top_k, 0.0);
  if (a.top_p < 1.0f) find_cut<true>(cl, s, r, c, 0, (double)a.top_p);
  const double min_p = (double)a.min_p;
  auto kept = [&](int i, float v) -> u64 {
    if (i >= r.w1 || !c.keeps(key_of(v), i)) return 0;
    const double w = r.weight(v);
    return w >= min_p ? __double2ull_rn(w * r.one) : 0;
  };
  u64 mine = 0;
  r.each(lane, [&](int i, float v) { mine += kept(i, v); });
  mine = warp_total(mine);
  u64 p = cta_prefix(s, mine, warp, lane);
  cl.sync();
  u64 total = 0;
  for (int q = 0; q < kCluster; ++q) {
    const u64 t = cl.map_shared_rank(&s, q)->cta_sum;
    if (q < rank) p += t;
    total += t;
  }
  const float uf = __ldg(a.u + row);
  const double u = uf > 0.0f ? (double)uf : 0.0;  // NaN and below: 0
  u64 target = (u64)(u * (double)total);
  if (u >= 1.0 || target >= total) target = total - 1;
  if (p <= target && target < p + mine) {  // this warp holds the token
    r.each(lane, [&](int i, float v) {
      const u64 w = kept(i, v), incl = warp_scan(w, lane);
      const u64 run = p + incl;
      if (run > target && run - w <= target) {
        a.token[row] = i;
        if (a.prob) a.prob[row] = (float)((double)w / (double)total);
      }
      p += __shfl_sync(0xffffffffu, incl, 31);
    });
  }
  cl.sync();  // no CTA leaves while another may read its sums
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
  // largest weight exponent: (max - x) / T must not leave fp32 as 0 / 0
  if (temperature > 0.0f && temperature < 1e-30f) temperature = 1e-30f;
  double one = 9223372036854775808.0;  // 2^63
  for (long n = 1; n < nvocab; n <<= 1) one *= 0.5;
  SampleArgs a{token, prob, logits, ld, u, temperature, top_p, min_p, top_k, m, nvocab, one};
  GCU_CUDA(cudaFuncSetAttribute(k_sample, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  GCU_CUDA(cudaFuncSetAttribute(k_sample, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared)));
  GCU_CUDA(launch_k(k_sample, dim3((unsigned)m * kCluster), dim3(kThreads), sizeof(Shared),
                    static_cast<cudaStream_t>(stream), a));
  return 0;
}

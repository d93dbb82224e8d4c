// k_attention_i8.cu -- attention over the 8-bit KV cache: how a call is cut into
// chunks of its key range, the merge of the chunks, and the entry points.  The
// kernels are in k_attention_i8_kt.cu (decode) and k_attention_i8_tc.cu (prompts).
#include "attention_i8.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

#define GCU_EXPORT extern "C" __attribute__((visibility("default")))

namespace gcu {
namespace attn8 {
namespace {

constexpr int kMergeThreads = 128;  // of k_merge_many
constexpr long kManyRows = 512;

// xo = sum_s e_s O_s / sum_s e_s l_s, e_s = 2^(m_s - max m), in slot order.
// For few rows, one CTA each: the slots' factors are formed by all threads at once and
// staged, and each thread keeps eight slots' loads in flight.  Bound by latency: 7.3 us
// cold for the 18 slots of 32768 keys and 16 heads, most of it hidden behind the end of
// the kernel before it.
template <int HD>
__global__ void __launch_bounds__(HD) k_merge_few(const Args a) {
  __shared__ float s_e[HD], s_l[HD], s_red[HD / 32];
  ptx::griddep_launch();
  const int i = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, d = threadIdx.x;
  const size_t row = blockIdx.x, rows = (size_t)a.ni * a.n_heads;
  ptx::griddep_wait();
  if (!row_live(a, i) || a.stat[row].y == kAlone) return;
  float m = -INFINITY;
  for (int s = d; s < a.slots; s += HD) m = fmaxf(m, a.stat[s * rows + row].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((d & 31) == 0) s_red[d >> 5] = m;
  __syncthreads();
  m = s_red[0];
#pragma unroll
  for (int w = 1; w < HD / 32; ++w) m = fmaxf(m, s_red[w]);
  float o = 0.0f, l = 0.0f;
  for (int s0 = 0; s0 < a.slots; s0 += HD) {
    const int ns = min(HD, a.slots - s0);
    __syncthreads();
    if (d < ns) {
      const float2 st = a.stat[(s0 + d) * rows + row];
      // a slot whose keys the row does not see: its sums count for nothing
      const float e = st.x == -INFINITY && st.y == 0.0f ? 0.0f : ex2(st.x - m);
      s_e[d] = e;
      s_l[d] = e * st.y;
    }
    __syncthreads();
    const float *ps = a.part + ((size_t)s0 * rows + row) * HD + d;
    int s = 0;
    for (; s + 8 <= ns; s += 8) {
      float v[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) v[t] = ps[(size_t)(s + t) * rows * HD];
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float e = s_e[s + t];
        l += s_l[s + t];
        o += e == 0.0f ? 0.0f : e * v[t];
      }
    }
    for (; s < ns; ++s) {
      const float e = s_e[s];
      l += s_l[s];
      o += e == 0.0f ? 0.0f : e * ps[(size_t)s * rows * HD];
    }
  }
  a.xo[(long)i * a.o_i + (long)h * HD + d] = o / (l == 0.0f ? 1.0f : l);
}

// The same for many rows, a warp each: lane s holds slot s's (m, l), and a lane HD/32
// columns of kFly slots in flight.  From kManyRows rows, where a CTA for each would
// come in waves: a prompt of 16368 rows in two slots 84.2 -> 72.7 us in all; 64 rows of
// 13 slots 10.0 -> 10.6, 8 rows of 148 slots 16.9 -> 25.3.
template <int HD>
__global__ void __launch_bounds__(kMergeThreads) k_merge_many(const Args a) {
  ptx::griddep_launch();
  constexpr int V = HD == 64 ? 2 : 4, Q = HD / 32 / V, kFly = HD == 256 ? 6 : 8;
  using F = typename std::conditional<V == 4, float4, float2>::type;
  const int lane = threadIdx.x & 31;
  const long row = (long)blockIdx.x * (kMergeThreads / 32) + (threadIdx.x >> 5), rows = (long)a.ni * a.n_heads;
  ptx::griddep_wait();
  if (row >= rows) return;
  const int i = (int)((uint32_t)row / (uint32_t)a.n_heads), h = (int)(row - (long)i * a.n_heads);
  if (!row_live(a, i)) return;
  auto stat = [&](int s) { return s < a.slots ? a.stat[s * rows + row] : make_float2(-INFINITY, 0.0f); };
  float2 st = stat(lane);
  if (__shfl_sync(0xffffffffu, st.y, 0) == kAlone) return;
  float m = st.x;
  for (int s = lane + 32; s < a.slots; s += 32) m = fmaxf(m, a.stat[s * rows + row].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float o[Q * V] = {}, l = 0.0f;
  for (int s0 = 0; s0 < a.slots; s0 += 32) {
    if (s0 > 0) st = stat(s0 + lane);
    // a slot whose keys the row does not see: its sums count for nothing
    const float e = st.x == -INFINITY && st.y == 0.0f ? 0.0f : ex2(st.x - m), le = e * st.y;
    const int ns = min(32, a.slots - s0);
    for (int t0 = 0; t0 < ns; t0 += kFly) {
      F v[kFly][Q];
#pragma unroll
      for (int t = 0; t < kFly; ++t)
#pragma unroll
        for (int q = 0; q < Q; ++q)
          if (t0 + t < ns)
            v[t][q] = *reinterpret_cast<const F *>(a.part + ((size_t)(s0 + t0 + t) * rows + row) * HD + (q * 32 + lane) * V);
#pragma unroll
      for (int t = 0; t < kFly; ++t) {
        if (t0 + t >= ns) break;
        const float f = __shfl_sync(0xffffffffu, e, t0 + t);
        l += __shfl_sync(0xffffffffu, le, t0 + t);
        if (f == 0.0f) continue;  // such a slot may not even be written
#pragma unroll
        for (int c = 0; c < Q * V; ++c) o[c] += f * reinterpret_cast<const float *>(&v[t][c / V])[c % V];
      }
    }
  }
  if (l == 0.0f) l = 1.0f;
  float *xo = a.xo + (long)i * a.o_i + (long)h * HD;
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    F r;
#pragma unroll
    for (int c = 0; c < V; ++c) reinterpret_cast<float *>(&r)[c] = o[q * V + c] / l;
    *reinterpret_cast<F *>(xo + (q * 32 + lane) * V) = r;
  }
}

int max_group(int n_heads, int nkv) { return (n_heads + nkv - 1) / nkv; }

}  // namespace

int launch_merge(const Args &a, cudaStream_t st) {
  const long rows = (long)a.ni * a.n_heads;
  if (rows > 0x7fffffffL) return set_error("attention_i8: %ld rows", rows);
  if (rows < kManyRows) {
    const dim3 grid((unsigned)rows);
    GCU_CUDA(a.kv.hdim == 256   ? launch_k(k_merge_few<256>, grid, dim3(256), 0, st, a)
             : a.kv.hdim == 128 ? launch_k(k_merge_few<128>, grid, dim3(128), 0, st, a)
                                : launch_k(k_merge_few<64>, grid, dim3(64), 0, st, a));
    return 0;
  }
  constexpr int per = kMergeThreads / 32;
  const dim3 grid((unsigned)((rows + per - 1) / per)), block(kMergeThreads);
  GCU_CUDA(a.kv.hdim == 256   ? launch_k(k_merge_many<256>, grid, block, 0, st, a)
           : a.kv.hdim == 128 ? launch_k(k_merge_many<128>, grid, block, 0, st, a)
                              : launch_k(k_merge_many<64>, grid, block, 0, st, a));
  return 0;
}

namespace {

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// A key range of at most n positions in chunks of whole tiles, as many as give
// `ctas` CTAs for `units` independent row groups.
struct Plan {
  int chunk, splits;
};

// Splits of n keys in tiles for `units` CTAs a split, of `ctas` in all.  However many
// units there are, a CTA takes at most kMaxKeys: decode's sums of byte products are
// 32-bit (66,312 keys of 255*127 fit), and a thread's fp32 sum of weights then has
// at most 128 terms in a row.  At 128 tiles the set-up of a further CTA is 1.5%.
constexpr long kMaxKeys = 16384;

Plan plan_range(long n, long units, long ctas, int tile) {
  if (n < 1) n = 1;
  const long tiles = (n + tile - 1) / tile, least = (n + kMaxKeys - 1) / kMaxKeys;
  const long want = std::min(tiles, std::max(least, ctas / units));
  Plan p;
  p.chunk = (int)((tiles + want - 1) / want * tile);
  p.splits = (int)((n + p.chunk - 1) / p.chunk);
  return p;
}

int visible(int n, int slide) { return slide > 0 ? std::min(n, slide) : n; }

struct DecodePlan {
  int rows;  // query rows per CTA
  Plan own, pre;
  bool cluster;  // the chunks' CTAs join their sums themselves
  int slots() const { return cluster ? 1 : own.splits + pre.splits; }
};

// Splits of the prefix: a CTA costs about kSetup tiles' time before and after its
// tiles, and CTAs run one per SM, the prefix's first.  Of the splits that give
// at most one wave of prefix CTAs the one whose last CTA ends first.
constexpr long kSetup = 3;

// Up to kKtCluster chunks are joined in the kernel that makes them, which saves the
// scratch and the merge's launch (5 us of the caller's time) and is worth kJoin
// further tiles a CTA: 2048 keys of one head take 8.6 us either way, 512 keys 7.6
// against 7.7; with three further tiles (4096 keys) 10.6 against 9.4.
constexpr long kJoin = 1;

bool join(Plan &p, long n, long units) {
  const Plan few = plan_range(n, units, std::min((long)num_sms(), kKtCluster * units), kKtKeys);
  if (few.splits < 2 || few.splits > kKtCluster || few.chunk > p.chunk + kJoin * kKtKeys) return false;
  p = few;
  return true;
}

DecodePlan plan_decode(const gcu_kv_i8 &own, int plen, int max_len, int n_heads, int slide) {
  const long G = max_group(n_heads, own.nkv), sms = std::max(1, num_sms());
  DecodePlan p;
  p.rows = plen > 0 && own.nseq * G > 16 ? 32 : 16;
  const long units = (long)own.nkv * own.nseq;
  p.own = plan_range(visible(max_len, slide), units, plen > 0 ? sms / 2 : sms, kKtKeys);
  p.pre = Plan{1, 0};
  p.cluster = plen == 0 && join(p.own, visible(max_len, slide), units);
  if (plen > 0) {
    const long n = visible(plen, slide), tiles = (n + kKtKeys - 1) / kKtKeys;
    const long pre = (own.nseq * G + p.rows - 1) / p.rows * own.nkv;
    const long own_ctas = units * p.own.splits, own_time = kSetup + p.own.chunk / kKtKeys;
    long best = -1, ctas = pre;
    for (long s = 1; s <= std::max(1l, std::min(tiles, sms / pre)); ++s) {
      const long time = kSetup + (tiles + s - 1) / s, idle = sms - std::min(sms, s * pre);
      // own CTAs that fit beside the prefix's, the others after them
      const long beside = std::min(own_ctas, idle * (time / own_time));
      const long end = time + (own_ctas - beside + sms - 1) / sms * own_time;
      if (best < 0 || end < best) best = end, ctas = s * pre;
    }
    p.pre = plan_range(n, pre, ctas, kKtKeys);
  }
  return p;
}

size_t slot_bytes(int slots, long rows, int hdim) {
  return slots > 1 ? (size_t)slots * rows * (hdim + 2) * sizeof(float) : 0;
}

void use_work(Args &a, void *work, long rows) {
  a.part = static_cast<float *>(work);
  a.stat = reinterpret_cast<float2 *>(a.part + (size_t)a.slots * rows * a.kv.hdim);
}

int check_heads(const char *what, int n_heads, int nkv) {
  if (n_heads < 1 || nkv > n_heads || max_group(n_heads, nkv) > kMaxGroup)
    return set_error("%s: %d query heads over %d kv heads (at most %d each)", what, n_heads, nkv, kMaxGroup);
  return 0;
}

int check_work(const char *what, size_t need, const void *work, size_t have) {
  if (need > have || (need && (!work || !aligned16(work))))
    return set_error("%s: %zu bytes of 16-byte aligned scratch needed, %zu given", what, need, have);
  return 0;
}

}  // namespace
}  // namespace attn8
}  // namespace gcu

using namespace gcu;
using namespace gcu::attn8;

GCU_EXPORT size_t gcu_attention_decode_i8_work(const gcu_kv_i8 *, int plen, const gcu_kv_i8 *own, int max_len,
                                               int n_heads, int slide) {
  if (!own || own->nkv < 1 || own->nseq < 1 || n_heads < 1) return 0;
  return slot_bytes(plan_decode(*own, plen, max_len, n_heads, slide).slots(), (long)own->nseq * n_heads, own->hdim);
}

GCU_EXPORT int gcu_dev_attention_decode_i8(float *xo, const float *xq, const gcu_kv_i8 *prefix, int plen,
                                           const gcu_kv_i8 *own, const int *len, int max_len, int n_heads,
                                           int slide, float asc, float sc_att, void *work, size_t work_bytes,
                                           void *stream) {
  const char *what = "attention_decode_i8";
  if (check_kv_i8(what, own) || check_heads(what, n_heads, own->nkv)) return 1;
  if (plen < 0 || slide < 0 || max_len < 0 || max_len > own->clen)
    return set_error("%s: %d of %d own positions, a prefix of %d, window %d", what, max_len, own->clen, plen, slide);
  if (plen > 0) {
    if (check_kv_i8(what, prefix, 1)) return 1;
    if (prefix->nkv != own->nkv || prefix->hdim != own->hdim || plen > prefix->clen)
      return set_error("%s: a prefix of %d positions from a cache of %d heads x %d x %d", what, plen, prefix->nkv,
                       prefix->clen, prefix->hdim);
  }
  if (!xo || !xq) return set_error("%s: null pointer", what);
  if (!aligned16(xo) || !aligned16(xq)) return set_error("%s: buffers must be 16-byte aligned", what);
  const DecodePlan p = plan_decode(*own, plen, max_len, n_heads, slide);
  const long rows = (long)own->nseq * n_heads;
  if (check_work(what, slot_bytes(p.slots(), rows, own->hdim), work, work_bytes)) return 1;
  if (overlap(xo, rows * own->hdim * 4, xq, rows * own->hdim * 4)) return set_error("%s: xo and xq overlap", what);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long qrow = (long)n_heads * own->hdim;
  Args a{xq, qrow, own->hdim, xo, qrow, *own, OWN, n_heads, own->nseq, 0, slide, 1, plen, max_len, len, asc, sc_att,
         p.own.chunk, p.own.splits, p.pre.splits, p.slots(), nullptr, nullptr, dev_error_word(),
         dev_length_word()};
  use_work(a, work, rows);
  Args sets[2] = {a, a};
  int n = 1;
  if (plen > 0) {  // the longer set first
    sets[0].mode = PREFIX;
    sets[0].kv = *prefix;
    sets[0].chunk = p.pre.chunk;
    sets[0].splits = p.pre.splits;
    sets[0].slot0 = 0;
    n = 2;
  }
  if (launch_kt(sets, n, p.rows, st)) return 1;
  return a.slots > 1 ? launch_merge(a, st) : 0;
}

namespace {

// Which kernel takes a prompt chunk, and how its keys are split.  k_kt (32 rows a
// CTA) starts and ends quickly and joins its chunks itself, k_tc (128 rows) moves a
// quarter of the keys per product: 512 tokens of 4 + 1 heads of 256 take 12.8 us
// against 21.5, 2048 of 16 + 8 heads 136 against 93.  The times come from a model
// fitted to both at 64 to 4096 tokens, heads 4 + 1, 8 + 4 and 16 + 8 of 64, 128 and 256:
// `fixed` us a CTA and `tile` us a tile of keys, the longest CTA or the average load
// of an SM, and a merge.  1023 tokens at 777 (16 + 8 heads of 128, capped) in chunks of 20
// tiles take 72.7 us, whole ones (of up to 29) 81.
struct PrefillPlan {
  bool kt, cluster;
  int rows;
  Plan p;
  int slots() const { return cluster ? 1 : p.splits; }
};

// kernel: 0 the faster of the two, 1 k_kt, 2 k_tc
PrefillPlan plan_prefill(const gcu_kv_i8 &kv, int n_heads, int spos, int ntok, int slide, int mask, bool cap,
                         int kernel = 0) {
  const long G = max_group(n_heads, kv.nkv), sms = std::max(1, num_sms()), end = (long)spos + ntok;
  const bool window = mask && slide > 0;
  auto plan = [&](bool kt, double &time) {
    PrefillPlan p;
    p.kt = kt;
    p.rows = !kt ? kTcRows : ntok * G > 16 ? 32 : 16;
    const int keys = kt ? kKtKeys : kTcKeys;
    const long units = (ntok * G + p.rows - 1) / p.rows * kv.nkv;
    // keys that a CTA's rows see when the last of them is at position at - 1: a window
    // and the tokens of the rows past the first
    auto seen = [&](long at) { return !mask ? end : window ? std::min(at, (long)slide + p.rows) : at; };
    const long n = seen(end);
    p.p = plan_range(n, units, sms, keys);
    p.cluster = kt && join(p.p, n, units);
    const double fixed = kt ? (kv.hdim == 256 ? 7.5 : 6.5) : kv.hdim == 256 ? 12.0 : kv.hdim == 128 ? 9.0 : 8.0;
    double tile = kt ? (kv.hdim == 256 ? 1.4 : 1.25) : kv.hdim == 256 ? 2.4 : kv.hdim == 128 ? 1.6 : 1.45;
    if (cap) tile *= kt ? 1.4 : 1.6;
    const long ctas = units * p.p.splits, waves = (ctas + sms - 1) / sms;
    const double mean = (seen(spos + 1) + 2 * seen(spos + ntok / 2 + 1) + n) / 4.0 / keys + 0.5;
    time = std::max(fixed + tile * (p.p.chunk / keys),
                    (kt ? (double)waves : (double)ctas / sms) * fixed + units * mean * tile / sms);
    const double merge = 4.0 + ntok * (double)n_heads / 3000;
    if (p.p.splits > 1 && !p.cluster) time += merge;
    // Fewer CTAs than SMs and row tiles of different lengths: a second chunk for the
    // longest ones, where the idle SMs' time and that of the short ones' takes it.
    const double t1 = (double)n / keys, t0 = (double)seen(spos + 1) / keys;
    if (!kt && !window && units < sms && t1 - t0 > 2.0)
      for (int k = 8; k < 16; ++k) {
        const int c = (int)std::ceil(t1 * k / 16);
        if (c <= t0 || c >= t1) continue;
        const double first = fixed + tile * c, over = (t1 - c) / (t1 - t0) * units;
        const double need = over * (fixed + tile * (t1 - c) / 2);
        const double spare = 0.85 * ((sms - units) * first + (units - over) * (c - t0) / 2 * tile);
        const double all = first + merge + (need > spare ? (need - spare) / sms + fixed + tile : 0.0);
        if (all >= time) continue;
        time = all;
        p.p.chunk = c * keys;
        p.p.splits = (int)((n + p.p.chunk - 1) / p.p.chunk);
      }
    return p;
  };
  double few, many;
  const PrefillPlan kt = plan(true, few), tc = plan(false, many);
  return kernel ? (kernel == 1 ? kt : tc) : few < many ? kt : tc;
}

}  // namespace

GCU_EXPORT size_t gcu_attention_prefill_i8_work(const gcu_kv_i8 *kv, int n_heads, int spos, int ntok, int slide,
                                                float sc_att, int mask) {
  if (!kv || kv->nkv < 1 || n_heads < 1 || ntok < 1 || spos < 0) return 0;
  return slot_bytes(plan_prefill(*kv, n_heads, spos, ntok, slide, mask, sc_att != 0.0f).slots(), (long)ntok * n_heads,
                    kv->hdim);
}

// The public call, and with the kernel given (for tests and measurements; not in the
// public header).
GCU_EXPORT int gcu_dev_attention_prefill_i8_tuned(float *xo, int xostr, const float *xq, const gcu_kv_i8 *kv,
                                                  int n_heads, int spos, int ntok, int slide, float sc_att, int mask,
                                                  void *work, size_t work_bytes, int kernel, void *stream) {
  if (ntok == 0) return 0;
  const char *what = "attention_prefill_i8";
  if (check_kv_i8(what, kv, 1) || check_heads(what, n_heads, kv->nkv)) return 1;
  if (spos < 0 || ntok < 0 || slide < 0 || spos > kv->clen - ntok)
    return set_error("%s: %d positions from %d outside a cache of %d, window %d", what, ntok, spos, kv->clen, slide);
  if (!xo || !xq) return set_error("%s: null pointer", what);
  if (xostr == 0) xostr = n_heads * kv->hdim;
  if (!aligned16(xo) || !aligned16(xq) || xostr % 4 || xostr < n_heads * kv->hdim)
    return set_error("%s: buffers must be 16-byte aligned, xostr a multiple of 4 floats, at least n_heads*hdim", what);
  const PrefillPlan p = plan_prefill(*kv, n_heads, spos, ntok, slide, mask, sc_att != 0.0f, kernel);
  const long rows = (long)ntok * n_heads;
  if (check_work(what, slot_bytes(p.slots(), rows, kv->hdim), work, work_bytes)) return 1;
  if (overlap(xo, ((long)(ntok - 1) * xostr + (long)n_heads * kv->hdim) * 4, xq, rows * kv->hdim * 4))
    return set_error("%s: xo and xq overlap", what);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Args a{xq, kv->hdim, (long)ntok * kv->hdim, xo, xostr, *kv, PREFILL, n_heads, ntok, spos, slide, mask ? 1 : 0, 0, 0,
         nullptr, 1.0f, sc_att, p.p.chunk, p.p.splits, 0, p.slots(), nullptr, nullptr, dev_error_word(),
         dev_length_word()};
  use_work(a, work, rows);
  if (p.kt ? launch_kt(&a, 1, p.rows, st) : launch_tc(a, st)) return 1;
  return a.slots > 1 ? launch_merge(a, st) : 0;
}

GCU_EXPORT int gcu_dev_attention_prefill_i8(float *xo, int xostr, const float *xq, const gcu_kv_i8 *kv, int n_heads,
                                            int spos, int ntok, int slide, float sc_att, int mask, void *work,
                                            size_t work_bytes, void *stream) {
  return gcu_dev_attention_prefill_i8_tuned(xo, xostr, xq, kv, n_heads, spos, ntok, slide, sc_att, mask, work,
                                            work_bytes, 0, stream);
}

// k_cache_i8.cu -- the 8-bit KV cache: rows quantized as they are written, and
// read back.
//
// Per head row x of hdim values (query, key, value heads of a token):
//   query, key: rms = 1 / sqrt(mean(x^2) + eps)         (QK norm, optional)
//               y = (x * rms) * (w + 1)
//               pairs (d, d + hdim/2): (a*c - b*s, a*s + b*c), queries * q_scale
//   key, value: scale = max|y| / 127, code = round(y / scale), per row, in the
//               arithmetic of quantize_acts (ptx::quant_scale, quant_one)
// The codes are what later steps live with, so they are made reproducible: the
// sum of squares is taken in 64 bits (its order cannot show in 32) and every
// fp32 step is rounded by itself.
//
// One warp per head row; lane l holds elements [l*E, l*E + E) of each half
// (E = hdim/64), so both elements of a RoPE pair sit in one lane, loads and
// stores are coalesced and only the two row reductions cross lanes.
// HBM-bound: per token 4*(nh + 2*nkv)*hdim bytes in, 4*nh*hdim + nkv*(2*hdim +
// 8) out.
#include "gcu_internal.cuh"

#define GCU_EXPORT extern "C" __attribute__((visibility("default")))

namespace gcu {
namespace {

constexpr int kThreads = 256;

struct WriteArgs {
  float *xq;
  const float *qkv;
  long ld;
  gcu_kv_i8 kv;
  const int *len;  // null: a chunk of one sequence from position spos
  const float *nq, *nk;
  float eps;
  const float *freqs;
  float q_scale;
  int n_heads, spos, rows;
  unsigned int *err;
};

template <int E>
struct Vec;
template <>
struct Vec<4> {
  using F = float4;
  using C = uint32_t;
};
template <>
struct Vec<2> {
  using F = float2;
  using C = uint16_t;
};
template <>
struct Vec<1> {
  using F = float;
  using C = uint8_t;
};

template <int E>
__device__ __forceinline__ void load(float (&v)[E], const float *p) {
  *reinterpret_cast<typename Vec<E>::F *>(v) = __ldg(reinterpret_cast<const typename Vec<E>::F *>(p));
}
template <int E>
__device__ __forceinline__ void store(float *p, const float (&v)[E]) {
  *reinterpret_cast<typename Vec<E>::F *>(p) = *reinterpret_cast<const typename Vec<E>::F *>(v);
}

// 1 / sqrt(x) to 64-bit rounding: two Newton steps on the fp32 estimate
// (relative error 2^-22 -> 2^-43 -> below 2^-52), a sixth of the 64-bit
// instructions that sqrt and a division take.  x outside fp32's normal range
// (a row of zeros with eps 0, a row past 1e19) takes those.
__device__ __forceinline__ double rsqrt64(double x) {
  if (!(x > 1e-37 && x < 1e37)) return 1.0 / sqrt(x);
  double y = (double)rsqrtf((float)x);
  y = y * (1.5 - 0.5 * x * y * y);
  return y * (1.5 - 0.5 * x * y * y);
}

// a, b: the lane's elements of the first and second half; fr: the lane's table
// entries (cos, sin per element)
template <int E>
__device__ __forceinline__ void norm_rope(float (&a)[E], float (&b)[E], const float *w, float eps, const float *fr,
                                          float scale, int lane) {
  constexpr int HD = 64 * E;
  if (w) {
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) sq += (double)a[i] * a[i] + (double)b[i] * b[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float rms = (float)rsqrt64(sq / HD + (double)eps);
    float wa[E], wb[E];
    load<E>(wa, w + lane * E);
    load<E>(wb, w + HD / 2 + lane * E);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      a[i] = __fmul_rn(__fmul_rn(a[i], rms), __fadd_rn(wa[i], 1.0f));
      b[i] = __fmul_rn(__fmul_rn(b[i], rms), __fadd_rn(wb[i], 1.0f));
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float2 t = __ldg(reinterpret_cast<const float2 *>(fr) + lane * E + i);
    const float x = a[i], y = b[i];
    a[i] = __fmul_rn(__fsub_rn(__fmul_rn(x, t.x), __fmul_rn(y, t.y)), scale);
    b[i] = __fmul_rn(__fadd_rn(__fmul_rn(x, t.y), __fmul_rn(y, t.x)), scale);
  }
}

template <int E>
__device__ __forceinline__ typename Vec<E>::C codes(const float (&v)[E], float inv) {
  uint32_t c = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) c |= (uint32_t)(ptx::quant_one(v[i], inv) & 0xff) << (8 * i);
  return (typename Vec<E>::C)c;
}

template <int E>
__global__ void __launch_bounds__(kThreads) k_write(WriteArgs a) {
  constexpr int HD = 64 * E;
  ptx::griddep_launch();
  const int lane = threadIdx.x & 31;
  const long row = (long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int heads = a.n_heads + 2 * a.kv.nkv;
  ptx::griddep_wait();
  if (row >= (long)a.rows * heads) return;  // whole warp
  const int t = (int)(row / heads), h = (int)(row - (long)t * heads);
  int seq = 0, pos = a.spos + t;
  if (a.len) {
    seq = t;
    const int n = __ldg(a.len + t);
    if (n < 1) return;
    if (n > a.kv.clen) {
      if (lane == 0) ptx::record_err(a.err, DEV_BAD_LENGTH);
      return;
    }
    pos = n - 1;
  }
  float lo[E], hi[E];
  const float *src = a.qkv + t * a.ld + (long)h * HD + lane * E;
  load<E>(lo, src);
  load<E>(hi, src + HD / 2);
  const bool isq = h < a.n_heads, isk = !isq && h < a.n_heads + a.kv.nkv;
  if (isq || isk)
    norm_rope<E>(lo, hi, isq ? a.nq : a.nk, a.eps, a.freqs + (long)t * HD, isq ? a.q_scale : 1.0f, lane);
  if (isq) {
    float *dst = a.xq + (a.len ? ((long)t * a.n_heads + h) * HD : ((long)h * a.rows + t) * HD) + lane * E;
    store<E>(dst, lo);
    store<E>(dst + HD / 2, hi);
    return;
  }
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < E; ++i) amax = fmaxf(amax, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float scale, inv;
  ptx::quant_scale(amax, scale, inv);
  const int hk = h - a.n_heads - (isk ? 0 : a.kv.nkv);
  int8_t *q = (isk ? a.kv.k : a.kv.v) + seq * a.kv.seq_stride + hk * a.kv.kv_stride + (long)pos * HD + lane * E;
  *reinterpret_cast<typename Vec<E>::C *>(q) = codes<E>(lo, inv);
  *reinterpret_cast<typename Vec<E>::C *>(q + HD / 2) = codes<E>(hi, inv);
  if (lane == 0) (isk ? a.kv.ks : a.kv.vs)[seq * a.kv.sc_seq_stride + hk * a.kv.sc_stride + pos] = scale;
}

// 16 lanes x 4 codes a step over a row of the cache, 16-byte stores
template <int HD>
__global__ void __launch_bounds__(kThreads) k_read(float *k, float *v, long out_seq_stride, long out_stride,
                                                   gcu_kv_i8 kv, int spos, int ntok) {
  ptx::griddep_launch();
  constexpr int L = HD / 4;  // threads per row
  const long i = (long)blockIdx.x * kThreads + threadIdx.x;
  ptx::griddep_wait();
  const int c = (int)(i % L);
  long r = i / L;
  const int t = (int)(r % ntok);
  r /= ntok;
  const int h = (int)(r % kv.nkv);
  const long b = r / kv.nkv;
  if (b >= kv.nseq) return;
  const bool isv = blockIdx.y;
  const char4 q = *reinterpret_cast<const char4 *>((isv ? kv.v : kv.k) + b * kv.seq_stride + h * kv.kv_stride +
                                                   (long)(spos + t) * HD + c * 4);
  const float s = (isv ? kv.vs : kv.ks)[b * kv.sc_seq_stride + h * kv.sc_stride + spos + t];
  *reinterpret_cast<float4 *>((isv ? v : k) + b * out_seq_stride + h * out_stride + (long)t * HD + c * 4) =
      make_float4(q.x * s, q.y * s, q.z * s, q.w * s);
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int launch_write(const WriteArgs &a, cudaStream_t st) {
  const long rows = (long)a.rows * (a.n_heads + 2 * a.kv.nkv);
  const long ctas = (rows + kThreads / 32 - 1) / (kThreads / 32);
  if (ctas > 0x7fffffffL) return set_error("qkv_norm_rope_cache_i8: %ld head rows", rows);
  const dim3 grid((unsigned)ctas);
  cudaError_t e = a.kv.hdim == 256   ? launch_k(k_write<4>, grid, dim3(kThreads), 0, st, a)
                  : a.kv.hdim == 128 ? launch_k(k_write<2>, grid, dim3(kThreads), 0, st, a)
                                     : launch_k(k_write<1>, grid, dim3(kThreads), 0, st, a);
  GCU_CUDA(e);
  return 0;
}

int check_write(const char *what, const float *xq, const float *qkv, long ld, const gcu_kv_i8 *kv,
                const float *nq, const float *nk, const float *freqs, int n_heads) {
  if (check_kv_i8(what, kv)) return 1;
  if (!xq || !qkv || !freqs) return set_error("%s: null pointer", what);
  if (n_heads < 1 || n_heads < kv->nkv)
    return set_error("%s: %d query heads over %d kv heads", what, n_heads, kv->nkv);
  const void *ptrs[] = {xq, qkv, freqs, nq, nk};
  for (const void *p : ptrs)
    if (!aligned16(p)) return set_error("%s: buffers must be 16-byte aligned", what);
  if (ld % 4 || ld < (long)(n_heads + 2 * kv->nkv) * kv->hdim)
    return set_error("%s: row stride %ld (a multiple of 4, at least the %ld fused q/k/v columns)", what, ld,
                     (long)(n_heads + 2 * kv->nkv) * kv->hdim);
  return 0;
}

}  // namespace

int check_kv_i8(const char *what, const gcu_kv_i8 *kv, int nseq) {
  if (!kv || !kv->k || !kv->v || !kv->ks || !kv->vs) return set_error("%s: null cache", what);
  if (kv->hdim != 64 && kv->hdim != 128 && kv->hdim != 256)
    return set_error("%s: head size %d (64, 128 or 256 supported)", what, kv->hdim);
  if (kv->nseq < 1 || kv->nkv < 1 || kv->clen < 1 || (nseq && kv->nseq != nseq))
    return set_error("%s: a cache of %d sequences, %d kv heads, %d positions", what, kv->nseq, kv->nkv, kv->clen);
  if (!aligned16(kv->k) || !aligned16(kv->v) || (uintptr_t)kv->ks % 4 || (uintptr_t)kv->vs % 4 ||
      kv->seq_stride % 16 || kv->kv_stride % 16)
    return set_error("%s: cache codes must be 16-byte aligned, their strides multiples of 16", what);
  if ((kv->nkv > 1 && (kv->kv_stride < (long)kv->clen * kv->hdim || kv->sc_stride < kv->clen)) ||
      (kv->nseq > 1 && (kv->seq_stride < (kv->nkv - 1) * kv->kv_stride + (long)kv->clen * kv->hdim ||
                        kv->sc_seq_stride < (kv->nkv - 1) * kv->sc_stride + kv->clen)))
    return set_error("%s: cache strides overlap rows of %d positions x %d", what, kv->clen, kv->hdim);
  return 0;
}

}  // namespace gcu

using namespace gcu;

GCU_EXPORT int gcu_dev_qkv_norm_rope_cache_i8(float *xq, const float *qkv, long ld, const gcu_kv_i8 *kv,
                                              const float *nq, const float *nk, float eps, const float *freqs,
                                              float q_scale, int n_heads, int spos, int ntok, void *stream) {
  if (ntok == 0) return 0;
  const char *what = "qkv_norm_rope_cache_i8";
  if (check_write(what, xq, qkv, ld, kv, nq, nk, freqs, n_heads)) return 1;
  if (kv->nseq != 1) return set_error("%s: a cache of one sequence expected, not of %d", what, kv->nseq);
  if (spos < 0 || ntok < 0 || spos > kv->clen - ntok)
    return set_error("%s: %d positions from %d outside a cache of %d", what, ntok, spos, kv->clen);
  WriteArgs a{xq, qkv, ld, *kv, nullptr, nq, nk, eps, freqs, q_scale, n_heads, spos, ntok, dev_error_word()};
  return launch_write(a, static_cast<cudaStream_t>(stream));
}

GCU_EXPORT int gcu_dev_qkv_norm_rope_cache_i8_seqs(float *xq, const float *qkv, long ld, const gcu_kv_i8 *kv,
                                                   const int *len, const float *nq, const float *nk, float eps,
                                                   const float *freqs, float q_scale, int n_heads,
                                                   void *stream) {
  const char *what = "qkv_norm_rope_cache_i8_seqs";
  if (check_write(what, xq, qkv, ld, kv, nq, nk, freqs, n_heads)) return 1;
  if (!len) return set_error("%s: null pointer", what);
  WriteArgs a{xq, qkv, ld, *kv, len, nq, nk, eps, freqs, q_scale, n_heads, 0, kv->nseq, dev_error_word()};
  return launch_write(a, static_cast<cudaStream_t>(stream));
}

GCU_EXPORT int gcu_dev_cache_i8_read(float *k, float *v, long out_seq_stride, long out_stride, const gcu_kv_i8 *kv,
                                     int spos, int ntok, void *stream) {
  if (ntok == 0) return 0;
  const char *what = "cache_i8_read";
  if (check_kv_i8(what, kv)) return 1;
  if (!k || !v) return set_error("%s: null pointer", what);
  if (spos < 0 || ntok < 0 || spos > kv->clen - ntok)
    return set_error("%s: %d positions from %d outside a cache of %d", what, ntok, spos, kv->clen);
  if (!aligned16(k) || !aligned16(v) || out_stride % 4 || out_seq_stride % 4)
    return set_error("%s: buffers must be 16-byte aligned, strides multiples of 4 floats", what);
  if ((kv->nkv > 1 && out_stride < (long)ntok * kv->hdim) ||
      (kv->nseq > 1 && out_seq_stride < (kv->nkv - 1) * out_stride + (long)ntok * kv->hdim))
    return set_error("%s: output strides overlap rows of %d positions x %d", what, ntok, kv->hdim);
  const long items = (long)kv->nseq * kv->nkv * ntok * (kv->hdim / 4), ctas = (items + kThreads - 1) / kThreads;
  if (ctas > 0x7fffffffL) return set_error("%s: %ld rows", what, items);
  const dim3 grid((unsigned)ctas, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kern = kv->hdim == 256 ? k_read<256> : kv->hdim == 128 ? k_read<128> : k_read<64>;
  GCU_CUDA(launch_k(kern, grid, dim3(kThreads), 0, st, k, v, out_seq_stride, out_stride, *kv, spos, ntok));
  return 0;
}

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
// A warp takes four heads of a token, lane l elements [l*E, l*E + E) of each half of
// each row (E = hdim/64), so both elements of a RoPE pair sit in one lane, loads
// and stores are coalesced, the tables and norm weights are read once for four
// rows, and only the two row reductions cross lanes, for four rows at once.
// HBM-bound: per token 4*(nh + 2*nkv)*hdim bytes in, 4*nh*hdim + nkv*(2*hdim +
// 8) out.  4096 tokens of 16 + 8 + 8 heads of 256: 45 us for 222 MB (4.9 TB/s,
// with an L2 full of another kernel's output to write back); one row per warp took
// 55, with 285 instructions a row against 120.  Reading them back: 20 us, 84 MB.
#include "gcu_internal.cuh"

#define GCU_EXPORT extern "C" __attribute__((visibility("default")))

namespace gcu {
namespace {

constexpr int kThreads = 256;       // of k_read
constexpr int kWriteThreads = 128;  // of k_write
constexpr int kRows = 4;            // head rows of a warp

__host__ __device__ __forceinline__ int groups(int heads) { return (heads + kRows - 1) / kRows; }

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
  unsigned int *bad_len;
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
// a lane's 2*E floats of a RoPE table row
template <int E>
__device__ __forceinline__ void load_table(float (&v)[2 * E], const float *p) {
  using F = typename Vec<E == 1 ? 2 : 4>::F;
#pragma unroll
  for (int i = 0; i < 2 * E; i += sizeof(F) / 4)
    *reinterpret_cast<F *>(v + i) = __ldg(reinterpret_cast<const F *>(p + i));
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

// Lane l of 32 gets row l / 8's total of v[row] over the lanes: the first two
// steps halve the rows that a lane carries, so four rows take 6 exchanges, not 20.
template <typename T, typename F>
__device__ __forceinline__ T reduce_rows(const T (&v)[kRows], int lane, F op) {
  const bool up = lane & 16, odd = lane & 8;
  T a = up ? v[2] : v[0], b = up ? v[3] : v[1];
  a = op(a, __shfl_xor_sync(0xffffffffu, up ? v[0] : v[2], 16));
  b = op(b, __shfl_xor_sync(0xffffffffu, up ? v[1] : v[3], 16));
  T c = odd ? b : a;
  c = op(c, __shfl_xor_sync(0xffffffffu, odd ? a : b, 8));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) c = op(c, __shfl_xor_sync(0xffffffffu, c, o));
  return c;
}

// a, b: the lane's elements of the first and second half of each row; w: the norm's
// weights, or null; t: the lane's table entries (cos, sin per element)
template <int E>
__device__ __forceinline__ void norm_rope(float (&a)[kRows][E], float (&b)[kRows][E], const float *w, float eps,
                                          const float (&t)[2 * E], float scale, int lane) {
  constexpr int HD = 64 * E;
  if (w) {
    float wa[E], wb[E];
    load<E>(wa, w + lane * E);
    load<E>(wb, w + HD / 2 + lane * E);
    double sq[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      sq[r] = 0.0;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const double x = a[r][i], y = b[r][i];
        sq[r] = fma(x, x, fma(y, y, sq[r]));
      }
    }
    const double sum = reduce_rows(sq, lane, [](double x, double y) { return x + y; });
    const float mine = (float)rsqrt64(sum * (1.0 / HD) + (double)eps);
#pragma unroll
    for (int i = 0; i < E; ++i) wa[i] = __fadd_rn(wa[i], 1.0f), wb[i] = __fadd_rn(wb[i], 1.0f);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float rms = __shfl_sync(0xffffffffu, mine, 8 * r);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        a[r][i] = __fmul_rn(__fmul_rn(a[r][i], rms), wa[i]);
        b[r][i] = __fmul_rn(__fmul_rn(b[r][i], rms), wb[i]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float x = a[r][i], y = b[r][i];
      a[r][i] = __fmul_rn(__fsub_rn(__fmul_rn(x, t[2 * i]), __fmul_rn(y, t[2 * i + 1])), scale);
      b[r][i] = __fmul_rn(__fadd_rn(__fmul_rn(x, t[2 * i + 1]), __fmul_rn(y, t[2 * i])), scale);
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
__global__ void __launch_bounds__(kWriteThreads) k_write(WriteArgs a) {
  constexpr int HD = 64 * E;
  ptx::griddep_launch();
  const int lane = threadIdx.x & 31;
  // x is the token, y some of its groups of heads: query, key, then value heads
  const int t = blockIdx.x, qg = groups(a.n_heads), kg = groups(a.kv.nkv);
  const int g = blockIdx.y * (kWriteThreads / 32) + (threadIdx.x >> 5);
  ptx::griddep_wait();
  if (g >= qg + 2 * kg) return;  // whole warp
  const bool isq = g < qg, isk = !isq && g < qg + kg;
  const int h0 = (isq ? g : isk ? g - qg : g - qg - kg) * kRows;
  const int nr = min(kRows, (isq ? a.n_heads : a.kv.nkv) - h0);
  int seq = 0, pos = a.spos + t;
  if (a.len) {
    seq = t;
    const int n = __ldg(a.len + t);
    if (n < 1) return;
    if (n > a.kv.clen) {
      if (lane == 0) ptx::record_err(a.bad_len, DEV_BAD_LENGTH);
      return;
    }
    pos = n - 1;
  }
  float lo[kRows][E], hi[kRows][E];
  const float *src =
      a.qkv + t * a.ld + ((long)h0 + (isq ? 0 : isk ? a.n_heads : a.n_heads + a.kv.nkv)) * HD + lane * E;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (r < nr) {
      load<E>(lo[r], src + r * HD);
      load<E>(hi[r], src + r * HD + HD / 2);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) lo[r][i] = hi[r][i] = 0.0f;
    }
  }
  if (isq || isk) {
    float fr[2 * E];
    load_table<E>(fr, a.freqs + (long)t * HD + lane * 2 * E);
    norm_rope<E>(lo, hi, isq ? a.nq : a.nk, a.eps, fr, isq ? a.q_scale : 1.0f, lane);
  }
  if (isq) {
    const long step = a.len ? HD : (long)a.rows * HD;
    float *dst = a.xq + (a.len ? (long)t * a.n_heads * HD : (long)t * HD) + h0 * step + lane * E;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= nr) break;
      store<E>(dst + r * step, lo[r]);
      store<E>(dst + r * step + HD / 2, hi[r]);
    }
    return;
  }
  float amax[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    amax[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) amax[r] = fmaxf(amax[r], fmaxf(fabsf(lo[r][i]), fabsf(hi[r][i])));
  }
  float scale, inv;
  ptx::quant_scale(reduce_rows(amax, lane, [](float x, float y) { return fmaxf(x, y); }), scale, inv);
  int8_t *q = (isk ? a.kv.k : a.kv.v) + seq * a.kv.seq_stride + h0 * a.kv.kv_stride + (long)pos * HD + lane * E;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float f = __shfl_sync(0xffffffffu, inv, 8 * r);
    if (r >= nr) break;
    *reinterpret_cast<typename Vec<E>::C *>(q + r * a.kv.kv_stride) = codes<E>(lo[r], f);
    *reinterpret_cast<typename Vec<E>::C *>(q + r * a.kv.kv_stride + HD / 2) = codes<E>(hi[r], f);
  }
  if (lane % 8 == 0 && lane / 8 < nr)
    (isk ? a.kv.ks : a.kv.vs)[seq * a.kv.sc_seq_stride + (h0 + lane / 8) * a.kv.sc_stride + pos] = scale;
}

// 4 codes a thread, kReadRows rows at a time so that their loads overlap; a CTA
// reads kReadRows * 1024 / HD positions of one head, K or V (y).
constexpr int kReadRows = 4;

template <int HD>
__global__ void __launch_bounds__(kThreads) k_read(float *k, float *v, long out_seq_stride, long out_stride,
                                                   gcu_kv_i8 kv, int spos, int ntok, int blocks) {
  ptx::griddep_launch();
  constexpr int L = HD / 4, R = kThreads / L;  // threads per row, rows at once
  const int bh = blockIdx.x / blocks, b = bh / kv.nkv, h = bh - b * kv.nkv;
  const int t0 = (blockIdx.x - bh * blocks) * (kReadRows * R) + threadIdx.x / L, c = threadIdx.x % L * 4;
  const int8_t *src = (blockIdx.y ? kv.v : kv.k) + b * kv.seq_stride + h * kv.kv_stride + (long)spos * HD + c;
  const float *sc = (blockIdx.y ? kv.vs : kv.ks) + b * kv.sc_seq_stride + h * kv.sc_stride + spos;
  float *dst = (blockIdx.y ? v : k) + b * out_seq_stride + h * out_stride + c;
  ptx::griddep_wait();
  char4 q[kReadRows];
  float s[kReadRows];
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const int t = min(t0 + i * R, ntok - 1);
    q[i] = *reinterpret_cast<const char4 *>(src + (long)t * HD);
    s[i] = sc[t];
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const int t = t0 + i * R;
    if (t < ntok)
      *reinterpret_cast<float4 *>(dst + (long)t * HD) =
          make_float4(q[i].x * s[i], q[i].y * s[i], q[i].z * s[i], q[i].w * s[i]);
  }
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int launch_write(const WriteArgs &a, cudaStream_t st) {
  if (overlap(a.xq, (long)a.rows * a.n_heads * a.kv.hdim * 4, a.qkv,
              ((a.rows - 1) * a.ld + (long)(a.n_heads + 2 * a.kv.nkv) * a.kv.hdim) * 4))
    return set_error("qkv_norm_rope_cache_i8: xq and qkv overlap");
  if (a.kv.k == a.kv.v || a.kv.ks == a.kv.vs) return set_error("qkv_norm_rope_cache_i8: the cache's k and v overlap");
  constexpr int kWarps = kWriteThreads / 32;
  const int y = (groups(a.n_heads) + 2 * groups(a.kv.nkv) + kWarps - 1) / kWarps;
  if (y > 65535) return set_error("qkv_norm_rope_cache_i8: %d query and %d kv heads", a.n_heads, a.kv.nkv);
  const dim3 grid(a.rows, y);
  cudaError_t e = a.kv.hdim == 256   ? launch_k(k_write<4>, grid, dim3(kWriteThreads), 0, st, a)
                  : a.kv.hdim == 128 ? launch_k(k_write<2>, grid, dim3(kWriteThreads), 0, st, a)
                                     : launch_k(k_write<1>, grid, dim3(kWriteThreads), 0, st, a);
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
  WriteArgs a{xq, qkv, ld, *kv, nullptr, nq, nk, eps, freqs, q_scale, n_heads, spos, ntok, dev_length_word()};
  return launch_write(a, static_cast<cudaStream_t>(stream));
}

GCU_EXPORT int gcu_dev_qkv_norm_rope_cache_i8_seqs(float *xq, const float *qkv, long ld, const gcu_kv_i8 *kv,
                                                   const int *len, const float *nq, const float *nk, float eps,
                                                   const float *freqs, float q_scale, int n_heads,
                                                   void *stream) {
  const char *what = "qkv_norm_rope_cache_i8_seqs";
  if (check_write(what, xq, qkv, ld, kv, nq, nk, freqs, n_heads)) return 1;
  if (!len) return set_error("%s: null pointer", what);
  WriteArgs a{xq, qkv, ld, *kv, len, nq, nk, eps, freqs, q_scale, n_heads, 0, kv->nseq, dev_length_word()};
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
  if (k == v) return set_error("%s: k and v overlap", what);
  const int per = kReadRows * kThreads * 4 / kv->hdim;  // positions of a CTA
  const int blocks = (int)(((long)ntok + per - 1) / per);
  const long ctas = (long)kv->nseq * kv->nkv * blocks;
  if (ctas > 0x7fffffffL) return set_error("%s: %ld CTAs", what, ctas);
  const dim3 grid((unsigned)ctas, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kern = kv->hdim == 256 ? k_read<256> : kv->hdim == 128 ? k_read<128> : k_read<64>;
  GCU_CUDA(launch_k(kern, grid, dim3(kThreads), 0, st, k, v, out_seq_stride, out_stride, *kv, spos, ntok, blocks));
  return 0;
}

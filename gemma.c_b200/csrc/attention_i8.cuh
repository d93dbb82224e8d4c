// attention_i8.cuh -- what the kernels of attention over the 8-bit KV cache
// share: the launch arguments, which positions a query row sees, and the
// three-digit form of the queries.
//
//   s[t]  = asc * ks[t] * sum_d q[d] * kc[t][d]          (kc, vc int8 codes)
//   p[t]  = exp(cap(s[t]) - m)
//   o     = sum_t p[t] * vs[t] * vc[t] / sum_t p[t]
//
// The codes stay integers up to the matrix products: a query row is scaled to
// 24-bit integers (q ~ sq * (65536 d2 + 256 d1 + d0), d signed bytes), so its
// products with int8 keys are int8 x int8 sums, exact in int32.  That is fixed point: every
// element is rounded by up to 2^-24 of the row's largest, as fp32 rounds that one, and
// one 2^-10 of its size keeps 14 bits where fp32 keeps 24.  A score moves by up to
// 2^-24 max|q| * asc * ks * sum |kc|.  The keys' own codes are rounded by 2^-8 of their
// row's largest, far more than that.  A fourth digit would cost a third more product and
// 64 TMEM columns, which k_tc has not left at hdim 256 (192 of scores, 256 of sums, 64
// of weights).
//
// Rows: the query heads of one kv head share its keys, so a row is (i, g):
// token or sequence i, head h0 + g of the group, row index i * G + g.
#pragma once

#include "gcu_internal.cuh"

namespace gcu {
namespace attn8 {

constexpr int kMaxGroup = 8;        // query heads per kv head
constexpr float kQMax = 8355000.0f;  // three signed bytes hold up to 127 * 65793 = 8355711
constexpr float kQLeast = 1e-31f;    // rows of smaller elements are scaled as if by this: 1 / scale stays finite
constexpr float kLog2e = 1.4426950408889634f;

enum Mode {
  PREFILL,  // row i is token spos + i of one sequence, keys at cache positions
  OWN,      // row i is sequence i, its own cache
  PREFIX    // row i is sequence i, the cache that all sequences share
};

constexpr float kAlone = -1.0f;  // where a sum of weights would stand

struct Args {
  const float *xq;  // row (i, h) at xq + i*q_i + h*q_h
  long q_i, q_h;
  float *xo;  // row (i, h) at xo + i*o_i + h*hdim
  long o_i;
  gcu_kv_i8 kv;
  Mode mode;
  int n_heads, ni;  // ni: tokens or sequences
  int spos, slide, mask;
  int plen, max_len;
  const int *len;  // device lengths of the sequences' own caches, or null: max_len
  float asc, sc_att;
  // Key ranges are cut into `splits` chunks; a launch writes slots [slot0,
  // slot0 + splits) of `slots` per row: unnormalised sums part[slot][row][hdim]
  // and (m, l) stat[slot][row] with row = i*n_heads + h, weights 2^(log2e*s - m).
  // slot 0 may hold (0, kAlone): the row is in xo already.
  // slots == 1: the rows go straight to xo, from the chunks' CTAs together (a
  // cluster) when there are several.
  int chunk, splits, slot0, slots;
  float *part;
  float2 *stat;
  unsigned int *err, *bad_len;
};

// query heads [head0(hk), head0(hk + 1)) belong to kv head hk (h * nkv / n_heads)
__host__ __device__ __forceinline__ int head0(int hk, int n_heads, int nkv) {
  return (hk * n_heads + nkv - 1) / nkv;
}

// own length of sequence i; -1: skipped
__device__ __forceinline__ int seq_len(const Args &a, int i) {
  if (!a.len) return a.max_len;
  const int n = __ldg(a.len + i);
  return n < 0 || n > a.max_len ? -1 : n;
}

// cache positions [lo, hi) that row i sees (lo >= hi: none)
__device__ __forceinline__ void row_window(const Args &a, int i, int &lo, int &hi) {
  if (a.mode == PREFILL) {
    const int pos = a.spos + i;
    lo = a.mask && a.slide > 0 ? max(0, pos + 1 - a.slide) : 0;
    hi = a.mask ? pos + 1 : a.spos + a.ni;
    return;
  }
  const int n = seq_len(a, i);
  if (n < 0) {
    lo = hi = 0;
    return;
  }
  // of plen + n positions the last `slide`
  const long skip = a.slide > 0 ? (long)a.plen + n - a.slide : 0;
  if (a.mode == OWN) {
    lo = (int)max(0l, skip - a.plen);
    hi = n;
  } else {
    lo = (int)min((long)a.plen, max(0l, skip));
    hi = a.plen;
  }
}

// whether row i's output is written at all
__device__ __forceinline__ bool row_live(const Args &a, int i) { return a.mode == PREFILL || seq_len(a, i) >= 0; }

// Rows first, first + 1, ... of a kv head as (i, g): one division, and a multiplication
// for each row after that (exact for up to 248 rows and G <= 8).
struct RowSplit {
  int i0, g0, G;
  uint32_t inv;
  __device__ __forceinline__ RowSplit(int first, int G_) : i0(first / G_), g0(first % G_), G(G_), inv(65536u / G_ + 1) {}
  __device__ __forceinline__ int i(int r) const { return i0 + (int)((uint32_t)(g0 + r) * inv >> 16); }
  __device__ __forceinline__ int g(int r) const { return g0 + r - (i(r) - i0) * G; }
};

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// tanh to 2^-22 of itself, without a branch: below 0.6 y + y^3 p(y^2), p a least-squares
// fit of (tanh(y)/y - 1)/y^2 at 400 Chebyshev nodes of [0, 0.36] with relative
// weights (2^-23.7 measured over 200001 points); above, 1 - 2/(1 + e^2|y|).  tanhf's
// branches cost the capped 1023-token prompt three quarters of its time (262 us).
__device__ __forceinline__ float tanh_fast(float y) {
  const float a = fabsf(y), z = y * y;
  float p = __fmaf_rn(z, -5.893945228e-3f, 2.079461701e-2f);
  p = __fmaf_rn(p, z, -5.378329381e-2f);
  p = __fmaf_rn(p, z, 1.333191544e-1f);
  p = __fmaf_rn(p, z, -3.333329856e-1f);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(ex2(a * (2.0f * kLog2e)) + 1.0f));
  return a < 0.6f ? __fmaf_rn(y * z, p, y) : copysignf(__fmaf_rn(-2.0f, r, 1.0f), y);
}

// E consecutive floats of a query row (zeros unless `have`)
template <int E>
__device__ __forceinline__ void load_floats(float (&v)[E], const float *src, bool have) {
  if constexpr (E % 4 == 0) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 f = have ? __ldg(reinterpret_cast<const float4 *>(src + e)) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[e] = f.x;
      v[e + 1] = f.y;
      v[e + 2] = f.z;
      v[e + 3] = f.w;
    }
  } else {
    const float2 f = have ? __ldg(reinterpret_cast<const float2 *>(src)) : make_float2(0.f, 0.f);
    v[0] = f.x;
    v[1] = f.y;
  }
}
// N rows of a warp: their largest |elements| (NaN if there is one; kQLeast at least) and
// the digits of this lane's elements, packed bytes of d0, d1, d2
template <int E, int N>
__device__ __forceinline__ void row_digits(const float (&v)[N][E], uint32_t (&w)[N][3][(E + 3) / 4], float (&amax)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    amax[n] = kQLeast;
#pragma unroll
    for (int e = 0; e < E; ++e) amax[n] = max_nan(amax[n], fabsf(v[n][e]));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) amax[n] = max_nan(amax[n], __shfl_xor_sync(0xffffffffu, amax[n], o));
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float inv = kQMax / amax[n];
    // n + 0x808080 (8421504) has the digits, each plus 128, as its bytes
    uint32_t u[(E + 3) / 4 * 4] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) u[e] = __float2uint_rn(__fmaf_rn(v[n][e], inv, 8421504.0f));
#pragma unroll
    for (int i = 0; i < (E + 3) / 4; ++i) {
      const uint32_t *x = u + 4 * i;
      const uint32_t a = __byte_perm(x[0], x[1], 0x5140), b = __byte_perm(x[2], x[3], 0x5140);
      w[n][0][i] = __byte_perm(a, b, 0x5410) ^ 0x80808080u;
      w[n][1][i] = __byte_perm(a, b, 0x7632) ^ 0x80808080u;
      w[n][2][i] = __byte_perm(__byte_perm(x[0], x[1], 0x0062), __byte_perm(x[2], x[3], 0x0062), 0x5410) ^ 0x80808080u;
    }
  }
}
template <int E>
__device__ __forceinline__ void put_digits(uint8_t *dst, const uint32_t (&w)[(E + 3) / 4]) {
  if constexpr (E == 8) {
    *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
  } else if constexpr (E == 4) {
    *reinterpret_cast<uint32_t *>(dst) = w[0];
  } else {
    *reinterpret_cast<uint16_t *>(dst) = (uint16_t)w[0];
  }
}

// 65536 s2 + 256 s1 + s0 in fp32, two columns at a time.  |s| < 2^22 goes into the
// mantissa of 1.5 * 2^23 by an integer addition (a conversion instruction runs
// at a fraction of the rate); the offsets leave with the next step.  256 s1 + s0
// is rounded at 2^31.6 at most, to 2^8, where the largest possible product of one
// query and key element alone is 127 * 2^23 = 2^30.
__device__ __forceinline__ float2 magic2(const uint32_t *s) {
  return make_float2(__uint_as_float(s[0] + 0x4B400000u), __uint_as_float(s[1] + 0x4B400000u));
}
// 256 s1 + s0 + 12582912
__device__ __forceinline__ float2 low_digits(const uint32_t *s1, const uint32_t *s0) {
  constexpr float off = -12582912.0f * 256.0f;
  return __fadd2_rn(magic2(s0), __ffma2_rn(magic2(s1), make_float2(256.0f, 256.0f), make_float2(off, off)));
}
__device__ __forceinline__ float2 high_digit(const uint32_t *s2, float2 low) {
  constexpr float off = -12582912.0f * 65537.0f;  // the low digits' offset too
  return __fadd2_rn(low, __ffma2_rn(magic2(s2), make_float2(65536.0f, 65536.0f), make_float2(off, off)));
}

// A value row's scale as it goes into the exponent and out of the sum of weights.
// Taken as at least 2^-64 and at most 2^100: reciprocals stay finite, and so do the
// sums of weights over them, up to 2^24 * 2^64 a key.
// NaN makes the weights NaN where the key is seen; where it is not, 1 / vs is
// finite against the zero weight.
constexpr float kScaleLo = 5.421011e-20f, kScaleHi = 1.2676506e30f;
__device__ __forceinline__ void value_scale(float v, float &log2_vs, float &inv_vs) {
  v = v < kScaleLo ? kScaleLo : v > kScaleHi ? kScaleHi : v;
  log2_vs = log2f(v);
  inv_vs = v == v ? 1.0f / v : 1.0f;
}

// A value row of zeros, to which the quantizer gives scale 1, adds nothing to the sum of
// products whatever its scale, but with 1 it could set m and take the bits of rows of
// small values. For m it counts as a row of scale 2^-32 (k_kt), or altogether (k_tc, where
// 2^32 times its weight goes into the sum of weights): its part of that sum then stays a
// normal number beside scales of up to 2^90. Only scales of exactly 1 are looked at.
constexpr float kZeros = 32.0f, kScaleZeros = 2.3283064e-10f;

// The roles of a CTA wait with a limit.  Every wait is on the phase after the last
// one that its waiter knows complete (a parity cannot tell two phases apart): what
// two groups take in turn has one barrier per tile parity.
struct Waiter {
  volatile int *abort;
  unsigned int *err;
  // false once any role of the CTA has given up
  __device__ __forceinline__ bool operator()(uint64_t *bar, uint32_t parity, unsigned int code) const {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = ptx::globaltimer();
    while (!*abort) {
      for (int i = 0; i < 64; ++i)
        if (ptx::mbar_try_wait(bar, parity)) return true;
      if (ptx::globaltimer() - t0 > 2000000000ull) {
        ptx::record_err(err, code);
        *abort = 1;
      }
    }
    return false;
  }
};

// k_attention_i8_tc.cu: 128 rows per CTA, kTcKeys keys at a time
int launch_tc(const Args &a, cudaStream_t st);
constexpr int kTcRows = 128, kTcKeys = 64;
// k_attention_i8_kt.cu: 16 or 32 rows per CTA, kKtKeys keys at a time; one launch
// for one or two sets of rows (a shared prefix, the sequences' own caches)
int launch_kt(const Args *sets, int n, int rows, cudaStream_t st);
constexpr int kKtKeys = 128;
constexpr int kKtCluster = 8;  // chunks that one launch joins
int launch_merge(const Args &a, cudaStream_t st);

}  // namespace attn8
}  // namespace gcu

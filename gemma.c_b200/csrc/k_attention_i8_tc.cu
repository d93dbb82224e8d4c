// k_attention_i8_tc.cu -- attention over the 8-bit KV cache on the tensor cores:
// prompt chunks, and decode rows that share a prefix.
//
// A CTA takes 128 query rows of one kv head (token or sequence i, head of the
// group: the heads that share keys fill the rows) and one chunk of the key
// range, and walks it in tiles of NK keys, keeping the running maximum and sum
// of the softmax:
//   S   three tcgen05.mma kind::i8 products per tile, the query's three digits
//       against the codes as TMA brings them: exact int32 sums in TMEM, put
//       together in fp32 (65536 s2 + 256 s1 + s0).  No conversion of K.
//   P   w = 2^(s + log2 vs[t] - m), m a reference point of the row near the
//       largest exponent so far, split into two fp16 parts in TMEM: w to 2^-22,
//       and to 2^-39 of the row's largest (the weights are placed just below
//       fp16's largest number).
//   T   two kind::f16 products, P's parts against the V codes as fp16 (exact).
//   l   sum of w / vs in fp32.
// vs rides in the exponent, so rows of V of any size keep their precision.  m
// stays where it is until an exponent passes it by kSlack.
//
// The tensor cores add in fp32 by cutting off (measured: 2e-9 of the sum is lost
// per key, 1.7e-5 over 8192 keys), so T holds kFlush tiles at most; then its
// softmax threads add it to the row's sums in their registers, rounded to
// nearest, and the next tile starts T afresh.  The same happens when a row's m
// moves, so the rescaling is a multiplication of registers.
//
// Warpgroups 0 and 1: softmax (two threads per row, half a tile's columns and half
// the output columns each; the row's sums take HD/2 registers of each, which
// the third warpgroup gives up).  Warps 8, 9: V codes to fp16 in the MN-major
// layout that the product reads; 10: loads; 11: products.  While the softmax of
// tile j runs, the tensor cores compute S of tile j + 1 and T of tile j - 1.
// Every wait is bounded; a role that gives up sets the CTA's abort flag, which
// ends the others' waits.
#include "attention_i8.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

namespace gcu {
namespace attn8 {
namespace {

constexpr int kSoftmax = 256;   // warps 0-7
constexpr int kConvert = 64;    // warps 8, 9
constexpr int kLoadWarp = 10, kMmaWarp = 11;
constexpr int kThreads = 384;
constexpr int kRegsSoftmax = 224, kRegsOther = 56;  // 2 * 224 + 56 = 3 * 168
constexpr int kRows = 128;
constexpr int NK = 64;     // keys per tile
constexpr int kFlush = 4;  // tiles per T
// Weights run up to 2^kTop at the reference point and may pass it by 2^kSlack:
// 2^15 stays below fp16's 65504.
constexpr float kTop = 10.0f, kSlack = 5.0f;
// Scales of V rows are taken as at least 2^-100 and at most 2^100: their
// reciprocals and sums stay finite.
constexpr float kVsMin = 7.888609e-31f, kVsMax = 1.2676506e30f;

template <int HD>
struct Cfg {
  static constexpr int SW = HD == 64 ? 64 : 128;  // bytes of a Q / K swizzle row
  static constexpr int KB = HD / SW;              // K blocks of SW bytes
  static constexpr int Q_BLOCK = kRows * SW;      // one digit's K block
  static constexpr int Q_BYTES = 3 * KB * Q_BLOCK;
  static constexpr int K_BLOCK = NK * SW;
  static constexpr int K_BYTES = KB * K_BLOCK;
  static constexpr int V8_BYTES = NK * HD;
  static constexpr int NV8 = HD == 256 ? 1 : 2;  // V code stages
  static constexpr int V16_BLOCK = NK * 128;     // 64 columns of the tile
  static constexpr int V16_BYTES = NK * HD * 2;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = Q_OFF + Q_BYTES;
  static constexpr int V16_OFF = K_OFF + 2 * K_BYTES;
  static constexpr int V8_OFF = V16_OFF + 2 * V16_BYTES;
  static constexpr int SC_OFF = V8_OFF + NV8 * V8_BYTES;      // scales [4][3][NK]: ks, log2 vs, 1 / vs
  static constexpr int MAX_OFF = SC_OFF + 4 * 3 * NK * 4;     // [2][2][128] row maxima (at the end: sums)
  static constexpr int RF_OFF = MAX_OFF + 2 * 2 * kRows * 4;  // [128] score factors
  static constexpr int SMEM = RF_OFF + kRows * 4 + 1024;
  // TMEM columns: S of three digits, T, P (two parts, two keys per column)
  static constexpr int S_COL = 0, T_COL = 3 * NK, P_COL = T_COL + HD;
  static constexpr int HALF = NK / 2;  // score columns per softmax thread
  static_assert(SMEM <= 232448 - 512, "shared memory budget");
  static_assert(P_COL + NK <= 512, "TMEM budget");
};

struct alignas(64) TcArgs {
  CUtensorMap tmK;
  Args a;
  int tiles;  // query tiles per kv head (of the largest group)
};

struct Bars {
  uint64_t kfull[2], kempty[2], v8full[2], v8empty[2], v16full[2], v16empty[2], sfull, sfree, pfull, pvdone, drain;
};

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

// four codes of a word as two fp16 pairs: byte ^ 0x80 into the mantissa of 1024,
// less 1152; exact
__device__ __forceinline__ uint2 to_half4(uint32_t w) {
  w ^= 0x80808080u;
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
  const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
  const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
  return make_uint2(*reinterpret_cast<const uint32_t *>(&x), *reinterpret_cast<const uint32_t *>(&y));
}

// 65536 s2 + 256 s1 + s0 in fp32.  |s| < 2^22 goes into the mantissa of 1.5 *
// 2^23 by an integer addition (a conversion instruction runs at a quarter of
// the rate); the three offsets leave together in the first step, whose result
// is 2^31.6 or more: an error of 2^8 at most, where the largest possible
// product of one query and key element alone is 127 * 8355711 = 2^30.
__device__ __forceinline__ float2 digit_sum2(const uint32_t *s2, const uint32_t *s1, const uint32_t *s0) {
  constexpr float offsets = 12582912.0f * 65793.0f;
  auto in = [](const uint32_t *s) { return make_float2(__uint_as_float(s[0] + 0x4B400000u), __uint_as_float(s[1] + 0x4B400000u)); };
  const float2 t = __ffma2_rn(in(s2), make_float2(65536.0f, 65536.0f), make_float2(-offsets, -offsets));
  return __fadd2_rn(in(s0), __ffma2_rn(in(s1), make_float2(256.0f, 256.0f), t));
}

// thread i < NK puts ks[i], i < 2 NK log2 and reciprocal of vs[i - NK]
__device__ __forceinline__ void put_scale(float *sc, int i, float v) {
  if (i < NK) {
    sc[i] = v;
  } else if (i < 2 * NK) {
    v = v < kVsMin ? kVsMin : v > kVsMax ? kVsMax : v;  // NaN stays
    sc[i] = log2f(v);
    sc[i + NK] = 1.0f / v;
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) k_tc(const __grid_constant__ TcArgs p) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_fresh[2], s_range[4];  // first key, end, last start of a window, first end
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const Args &a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y;
  const int h0 = head0(hk, a.n_heads, a.kv.nkv), G = head0(hk + 1, a.n_heads, a.kv.nkv) - h0;
  // heavy tiles first: the last query rows of a prompt see the most keys
  const int tile = p.tiles - 1 - (int)(blockIdx.x / a.splits), split = blockIdx.x % a.splits;
  const int first = tile * kRows, nrows = min(kRows, a.ni * G - first);
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&bars.kfull[s], 1);
      ptx::mbar_init(&bars.kempty[s], 1);
      ptx::mbar_init(&bars.v8full[s], 1);
      ptx::mbar_init(&bars.v8empty[s], kConvert);
      ptx::mbar_init(&bars.v16full[s], kConvert);
      ptx::mbar_init(&bars.v16empty[s], 1);
    }
    ptx::mbar_init(&bars.sfull, 1);
    ptx::mbar_init(&bars.sfree, kSoftmax);
    ptx::mbar_init(&bars.pfull, kSoftmax);
    ptx::mbar_init(&bars.pvdone, 1);
    ptx::mbar_init(&bars.drain, 1);
    ptx::fence_mbar_init();
    s_abort = 0;
    s_range[0] = s_range[3] = 0x7fffffff;
    s_range[1] = s_range[2] = 0;
    ptx::prefetch_tmap(&p.tmK);
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(&s_tmem, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  // the next kernel may start now: this CTA holds its TMEM
  ptx::griddep_launch();
  ptx::griddep_wait();

  // the rows' windows: the CTA's key range, and the keys that every row sees
  if ((int)threadIdx.x < nrows) {
    int lo, hi;
    row_window(a, (first + threadIdx.x) / G, lo, hi);
    if (lo < hi) {
      atomicMin(&s_range[0], lo);
      atomicMax(&s_range[1], hi);
    }
    atomicMax(&s_range[2], lo);
    atomicMin(&s_range[3], hi);
  }
  __syncthreads();
  const int all_lo = s_range[2], all_hi = s_range[3];
  const long c0 = (long)s_range[0] + (long)split * a.chunk;
  const int n = (int)max(0l, min((long)s_range[1], c0 + a.chunk) - c0);
  const int kbeg = (int)min(c0, 0x7fffffffl), kend = kbeg + n, nt = (n + NK - 1) / NK;
  Waiter wait{&s_abort, a.err};

  const int8_t *vh = a.kv.v + hk * a.kv.kv_stride, *kh = a.kv.k + hk * a.kv.kv_stride;
  // the loads of tile j (one thread)
  auto load_k = [&](int j, uint64_t pol) {
    uint64_t *bar = &bars.kfull[j & 1];
    ptx::mbar_arrive_expect_tx(bar, C::K_BYTES);
#pragma unroll
    for (int b = 0; b < C::KB; ++b)
      ptx::tma_load_3d(&p.tmK, bar, smem + C::K_OFF + (j & 1) * C::K_BYTES + b * C::K_BLOCK, b * C::SW, kbeg + j * NK, hk,
                       pol);
  };
  auto load_v = [&](int j, uint64_t pol) {
    const uint32_t bytes = (uint32_t)min(NK, n - j * NK) * HD;
    uint64_t *bar = &bars.v8full[j % C::NV8];
    ptx::mbar_arrive_expect_tx(bar, bytes);
    ptx::bulk_load(smem + C::V8_OFF + (j % C::NV8) * C::V8_BYTES, vh + (long)(kbeg + j * NK) * HD, bytes, bar, pol);
  };
  const uint64_t pol = ptx::policy_evict_last();  // every query tile of the head reads these tiles
  if (warp == kLoadWarp && lane == 0 && nt > 0) {
    load_k(0, pol);
    load_v(0, pol);
    if (nt > 1) load_k(1, pol);
  }

  // the query rows' digits, a warp per row; rows past the end are zeros
  float *s_rf = reinterpret_cast<float *>(smem + C::RF_OFF);
  if (nt > 0) {
    constexpr int E = HD / 32;
    for (int r = warp; r < kRows; r += kThreads / 32) {
      float v[E], amax = 0.0f;
      const int i = (first + r) / G, g = (first + r) % G;
      const float *src = a.xq + (long)i * a.q_i + (long)(h0 + g) * a.q_h + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = r < nrows ? __ldg(src + e) : 0.0f;
        amax = max_nan(amax, fabsf(v[e]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const float inv = amax > 0.0f ? kQMax / amax : 0.0f;
      uint32_t w[3][(E + 3) / 4] = {};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        int d2, d1, d0;
        digits(v[e], inv, d2, d1, d0);
        w[0][e / 4] |= (uint32_t)(d0 & 0xff) << (8 * (e % 4));
        w[1][e / 4] |= (uint32_t)(d1 & 0xff) << (8 * (e % 4));
        w[2][e / 4] |= (uint32_t)(d2 & 0xff) << (8 * (e % 4));
      }
      const int col = lane * E, in = col % C::SW;
      const int sw = C::SW == 128 ? r & 7 : (r >> 1) & 3;
      uint8_t *dst = smem + C::Q_OFF + (col / C::SW) * C::Q_BLOCK + r * C::SW + (((in >> 4) ^ sw) << 4) + (in & 15);
#pragma unroll
      for (int d = 0; d < 3; ++d) {
        uint8_t *q = dst + d * C::KB * C::Q_BLOCK;
        if constexpr (E == 8) {
          *reinterpret_cast<uint2 *>(q) = make_uint2(w[d][0], w[d][1]);
        } else if constexpr (E == 4) {
          *reinterpret_cast<uint32_t *>(q) = w[d][0];
        } else {
          *reinterpret_cast<uint16_t *>(q) = (uint16_t)w[d][0];
        }
      }
      if (lane == 0) s_rf[r] = amax / kQMax * a.asc;
    }
    // tile 0's scales
    if ((int)threadIdx.x < 2 * NK) {
      const int t = threadIdx.x % NK;
      const float *src = (threadIdx.x < NK ? a.kv.ks : a.kv.vs) + hk * a.kv.sc_stride;
      put_scale(reinterpret_cast<float *>(smem + C::SC_OFF), threadIdx.x, t < n ? __ldg(src + kbeg + t) : 1.0f);
    }
  }
  ptx::fence_proxy_async_smem();
  __syncthreads();

  if (warp >= kSoftmax / 32) ptx::regs_dec<kRegsOther>();
  if (warp == kLoadWarp) {
    // ------------------------------------------------------------ loads
    if (lane == 0 && nt > 0) {
      int nk = min(2, nt), nv = 1;  // tiles issued
      for (int j = 1; j < nt; ++j) {
        // two tiles ahead into L2
        if (j + 2 < nt) {
          const long at = (long)(kbeg + (j + 2) * NK) * HD;
          const uint32_t bytes = (uint32_t)min(NK, n - (j + 2) * NK) * HD;
          ptx::bulk_prefetch_l2(kh + at, bytes);
          ptx::bulk_prefetch_l2(vh + at, bytes);
        }
        if (j + 1 < nt) {
          if (!wait(&bars.kempty[(j + 1) & 1], ((j - 1) >> 1) & 1, DEV_TIMEOUT_EMPTY)) break;
          load_k(j + 1, pol);
          ++nk;
        }
        if (j >= C::NV8 &&
            !wait(&bars.v8empty[j % C::NV8], ((j - C::NV8) / C::NV8) & 1, DEV_TIMEOUT_EMPTY))
          break;
        load_v(j, pol);
        ++nv;
      }
      // every load issued must have landed before the CTA may exit
      for (int j = max(0, nk - 2); j < nk; ++j)
        ptx::mbar_wait(&bars.kfull[j & 1], (j >> 1) & 1, a.err, DEV_TIMEOUT_DRAIN);
      for (int j = max(0, nv - C::NV8); j < nv; ++j)
        ptx::mbar_wait(&bars.v8full[j % C::NV8], (j / C::NV8) & 1, a.err, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ products
    if (lane == 0 && nt > 0) {
      constexpr uint32_t id_s = ptx::idesc_i8(kRows, NK), id_o = ptx::idesc_f16_bt(kRows, HD);
      const uint32_t q0 = ptx::smem_u32(smem + C::Q_OFF), k0 = ptx::smem_u32(smem + C::K_OFF);
      const uint32_t v0 = ptx::smem_u32(smem + C::V16_OFF);
      auto scores = [&](int j) {
#pragma unroll
        for (int d = 0; d < 3; ++d)
#pragma unroll
          for (int b = 0; b < C::KB; ++b)
#pragma unroll
            for (int s = 0; s < C::SW / 32; ++s)
              ptx::mma_i8(tmem + C::S_COL + d * NK,
                          ptx::smem_desc(q0 + (d * C::KB + b) * C::Q_BLOCK + 32 * s, 16, 8 * C::SW, C::SW),
                          ptx::smem_desc(k0 + (j & 1) * C::K_BYTES + b * C::K_BLOCK + 32 * s, 16, 8 * C::SW, C::SW), id_s,
                          b + s > 0 ? 1u : 0u);
        ptx::mma_commit(&bars.kempty[j & 1]);
        ptx::mma_commit(&bars.sfull);
      };
      bool ok = wait(&bars.kfull[0], 0, DEV_TIMEOUT_FULL);
      if (ok) {
        ptx::tc_fence_after();
        scores(0);
      }
      for (int j = 0; j < nt && ok; ++j) {
        if (j + 1 < nt) {
          ok = wait(&bars.kfull[(j + 1) & 1], ((j + 1) >> 1) & 1, DEV_TIMEOUT_FULL) &&
               wait(&bars.sfree, j & 1, DEV_TIMEOUT_TMEM);
          if (!ok) break;
          ptx::tc_fence_after();
          scores(j + 1);
        }
        ok = wait(&bars.v16full[j & 1], (j >> 1) & 1, DEV_TIMEOUT_FULL) && wait(&bars.pfull, j & 1, DEV_TIMEOUT_TMEM);
        if (!ok) break;
        ptx::tc_fence_after();
        const uint32_t keep = *(volatile int *)&s_fresh[j & 1] ? 0u : 1u;
#pragma unroll
        for (int part = 0; part < 2; ++part)
#pragma unroll
          for (int s = 0; s < NK / 16; ++s)
            ptx::mma_f16_ts(tmem + C::T_COL, tmem + C::P_COL + part * (NK / 2) + 8 * s,
                            ptx::smem_desc(v0 + (j & 1) * C::V16_BYTES + s * 2048, C::V16_BLOCK, 1024, 128), id_o,
                            part + s > 0 ? 1u : keep);
        ptx::mma_commit(&bars.v16empty[j & 1]);
        ptx::mma_commit(&bars.pvdone);
      }
      // all products complete before TMEM is freed
      ptx::mma_commit(&bars.drain);
      ptx::mbar_wait(&bars.drain, 0, a.err, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp >= kSoftmax / 32) {
    // ------------------------------------------------------------ V codes to fp16
    const int t = threadIdx.x - kSoftmax;
    constexpr int L = HD / 8, KS = kConvert / L;  // threads per key (8 columns each), keys at a time
    const int c = t % L, key0 = t / L;
    for (int j = 0; j < nt; ++j) {
      if (!wait(&bars.v8full[j % C::NV8], (j / C::NV8) & 1, DEV_TIMEOUT_FULL)) break;
      if (j > 1 && !wait(&bars.v16empty[j & 1], ((j - 2) >> 1) & 1, DEV_TIMEOUT_TMEM)) break;
      const uint8_t *src = smem + C::V8_OFF + (j % C::NV8) * C::V8_BYTES + c * 8;
      uint8_t *dst = smem + C::V16_OFF + (j & 1) * C::V16_BYTES + (c >> 3) * C::V16_BLOCK;
      // keys past the range hold an earlier tile's codes, which weigh nothing
#pragma unroll 8
      for (int k = 0; k < NK; k += KS) {
        const int key = key0 + k;
        const uint2 w = *reinterpret_cast<const uint2 *>(src + key * HD);
        const uint2 x = to_half4(w.x), y = to_half4(w.y);
        *reinterpret_cast<uint4 *>(dst + key * 128 + (((c & 7) ^ (key & 7)) << 4)) = make_uint4(x.x, x.y, y.x, y.y);
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&bars.v8empty[j % C::NV8]);
      ptx::mbar_arrive(&bars.v16full[j & 1]);
    }
  } else {
    // ------------------------------------------------------------ softmax
    ptx::regs_inc<kRegsSoftmax>();
    const int half = warp >> 2, row = (warp & 3) * 32 + lane, tid = threadIdx.x;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float *sc = reinterpret_cast<float *>(smem + C::SC_OFF);
    float *smax = reinterpret_cast<float *>(smem + C::MAX_OFF);
    const bool live = row < nrows;
    const int i = live ? (first + row) / G : 0, h = live ? h0 + (first + row) % G : h0;
    int lo = 0, hi = 0;
    if (live) row_window(a, i, lo, hi);
    const float rf_nat = nt > 0 ? s_rf[row] : 0.0f;
    const bool capped = a.sc_att != 0.0f;
    const float rf = capped ? kLog2e : rf_nat * kLog2e;
    const float *sc_src = (tid < NK ? a.kv.ks : a.kv.vs) + hk * a.kv.sc_stride + kbeg;
    auto fetch_scale = [&](int j) {
      const int t = j * NK + tid % NK;
      return tid < 2 * NK && t < n ? __ldg(sc_src + t) : 1.0f;
    };
    float next = fetch_scale(1);
    float m = -INFINITY, l = 0.0f;
    float acc[HD / 2];  // the row's sums, output columns [half * HD/2, +HD/2)
#pragma unroll
    for (int c = 0; c < HD / 2; ++c) acc[c] = 0.0f;
    // add T (complete) to the row's sums
    auto flush = [&]() {
      ptx::tc_fence_after();
#pragma unroll
      for (int c = 0; c < HD / 2; c += 32) {
        uint32_t t[32];
        ptx::tmem_ld_32x32(lanes + C::T_COL + half * (HD / 2) + c, t);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) acc[c + e] += __uint_as_float(t[e]);
      }
      ptx::tc_fence_before();
    };
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      const float *ks = sc + (j & 3) * 3 * NK + half * C::HALF, *lvs = ks + NK, *rvs = ks + 2 * NK;
      ok = ok && wait(&bars.sfull, j & 1, DEV_TIMEOUT_TMEM);
      ptx::tc_fence_after();
      // exponents: the score in log2 units plus log2 of the value row's scale
      float x[C::HALF];
#pragma unroll
      for (int c = 0; c < C::HALF; c += 16) {
        uint32_t s2[16], s1[16], s0[16];
        const uint32_t at = lanes + C::S_COL + half * C::HALF + c;
        ptx::tmem_ld_32x16(at, s0);
        ptx::tmem_ld_32x16(at + NK, s1);
        ptx::tmem_ld_32x16(at + 2 * NK, s2);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const float4 k = *reinterpret_cast<const float4 *>(ks + c + e);
          float2 u = digit_sum2(s2 + e, s1 + e, s0 + e), v = digit_sum2(s2 + e + 2, s1 + e + 2, s0 + e + 2);
          u = __fmul2_rn(u, make_float2(k.x, k.y));
          v = __fmul2_rn(v, make_float2(k.z, k.w));
          x[c + e] = u.x;
          x[c + e + 1] = u.y;
          x[c + e + 2] = v.x;
          x[c + e + 3] = v.y;
        }
      }
      ptx::tc_fence_before();
      ptx::mbar_arrive(&bars.sfree);
      if (capped) {
#pragma unroll
        for (int c = 0; c < C::HALF; ++c) x[c] = tanhf(x[c] * rf_nat / a.sc_att) * a.sc_att;
      }
#pragma unroll
      for (int c = 0; c < C::HALF; c += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(lvs + c);
        const float2 r2 = make_float2(rf, rf);
        const float2 y = __ffma2_rn(make_float2(x[c], x[c + 1]), r2, make_float2(v.x, v.y));
        const float2 z = __ffma2_rn(make_float2(x[c + 2], x[c + 3]), r2, make_float2(v.z, v.w));
        x[c] = y.x;
        x[c + 1] = y.y;
        x[c + 2] = z.x;
        x[c + 3] = z.y;
      }
      // a tile that some row does not see in full
      const int t0 = kbeg + j * NK;
      const bool masked = t0 < all_lo || t0 + NK > min(all_hi, kend);
      if (masked) {
        const int cl = lo - t0 - half * C::HALF, ch = min(hi, kend) - t0 - half * C::HALF;
#pragma unroll
        for (int c = 0; c < C::HALF; ++c)
          if (c < cl || c >= ch) x[c] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < C::HALF; ++c) mx = fmaxf(mx, x[c]);
      float *sm = smax + (j & 1) * 2 * kRows;
      sm[half * kRows + row] = mx;
      put_scale(sc + ((j + 1) & 3) * 3 * NK, tid, next);
      next = fetch_scale(j + 2);
      float f = 1.0f;
      bool fresh = j % kFlush == 0;
      if (ptx::named_bar_or(1, kSoftmax, mx > m + kSlack || (m == -INFINITY && mx > m) || !ok)) {
        if (ptx::named_bar_or(1, kSoftmax, !ok)) break;
        const float to = fmaxf(m, fmaxf(sm[row], sm[kRows + row]));
        f = to == m ? 1.0f : ex2(m - to);  // m = -inf: 0
        l *= f;
        m = to;
        fresh = true;
      }
      const float ref = m == -INFINITY ? 0.0f : m - kTop;
      uint32_t ph[C::HALF / 2], pl[C::HALF / 2];
      float2 lt = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int c = 0; c < C::HALF; c += 4) {
        const float4 r = *reinterpret_cast<const float4 *>(rvs + c);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 d = __fadd2_rn(make_float2(x[c + e], x[c + e + 1]), make_float2(-ref, -ref));
          const float2 w = make_float2(ex2(d.x), ex2(d.y));
          float2 q = e ? make_float2(r.z, r.w) : make_float2(r.x, r.y);
          if (masked) {  // a key that is not seen weighs nothing, whatever its scales
            q.x = x[c + e] == -INFINITY ? 0.0f : q.x;
            q.y = x[c + e + 1] == -INFINITY ? 0.0f : q.y;
          }
          lt = __ffma2_rn(w, q, lt);
          const __half2 hi2 = __floats2half2_rn(w.x, w.y);
          const float2 back = __half22float2(hi2);
          const __half2 lo2 = __floats2half2_rn(w.x - back.x, w.y - back.y);
          ph[(c + e) / 2] = *reinterpret_cast<const uint32_t *>(&hi2);
          pl[(c + e) / 2] = *reinterpret_cast<const uint32_t *>(&lo2);
        }
      }
      l += lt.x + lt.y;
      // P and T are free once the previous tile's product is done
      if (j > 0) {
        ok = wait(&bars.pvdone, (j - 1) & 1, DEV_TIMEOUT_TMEM) && ok;
        if (fresh) {
          flush();
          if (f != 1.0f) {
#pragma unroll
            for (int c = 0; c < HD / 2; ++c) acc[c] *= f;
          }
        }
      }
      ptx::tmem_st_32x16(lanes + C::P_COL + half * (C::HALF / 2), ph);
      ptx::tmem_st_32x16(lanes + C::P_COL + NK / 2 + half * (C::HALF / 2), pl);
      if (tid == 0) *(volatile int *)&s_fresh[j & 1] = fresh;
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      ptx::mbar_arrive(&bars.pfull);
    }
    if (nt > 0) {
      ok = wait(&bars.pvdone, (nt - 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      flush();
    }
    // the row's sum over both halves
    ptx::named_bar_sync(1, kSoftmax);
    smax[half * kRows + row] = l;
    ptx::named_bar_sync(1, kSoftmax);
    l = smax[row] + smax[kRows + row];
    const size_t at = ((size_t)(a.slot0 + split) * a.ni + i) * a.n_heads + h;
    float *out = (a.slots == 1 ? a.xo + (long)i * a.o_i + (long)h * HD : a.part + at * HD) + half * (HD / 2);
    const float d = a.slots > 1 || l == 0.0f ? 1.0f : l;  // a row that sees nothing: zeros
    if (live && ok && (a.slots > 1 || row_live(a, i))) {
#pragma unroll
      for (int c = 0; c < HD / 2; c += 4)
        *reinterpret_cast<float4 *>(out + c) = make_float4(acc[c] / d, acc[c + 1] / d, acc[c + 2] / d, acc[c + 3] / d);
      if (a.slots > 1 && half == 0) a.stat[at] = make_float2(m == -INFINITY ? m : m - kTop, l);
    }
  }
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, 512);
}

template <int HD>
int launch_tc_hd(const Args &a, cudaStream_t st) {
  using C = Cfg<HD>;
  TcArgs p;
  p.a = a;
  const int gmax = (a.n_heads + a.kv.nkv - 1) / a.kv.nkv;
  p.tiles = (int)(((long)a.ni * gmax + kRows - 1) / kRows);
  if (gemm_tmap_heads_i8(&p.tmK, a.kv.k, HD, a.kv.clen, a.kv.nkv, a.kv.kv_stride, NK)) return 1;
  {
    // the shared-memory opt-in is per device: once for each device this runs on
    static std::mutex mu;
    static unsigned long long done = 0;
    int dev = 0;
    GCU_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (!(done & (1ull << (dev & 63)))) {
      GCU_CUDA(cudaFuncSetAttribute(k_tc<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
      done |= 1ull << (dev & 63);
    }
  }
  if ((long)p.tiles * a.splits > 0x7fffffffL) return set_error("attention_i8: %d x %d CTAs", p.tiles, a.splits);
  GCU_CUDA(launch_k(k_tc<HD>, dim3((unsigned)(p.tiles * a.splits), a.kv.nkv), dim3(kThreads), C::SMEM, st, p));
  return 0;
}

}  // namespace

int launch_tc(const Args &a, cudaStream_t st) {
  return a.kv.hdim == 256 ? launch_tc_hd<256>(a, st) : a.kv.hdim == 128 ? launch_tc_hd<128>(a, st) : launch_tc_hd<64>(a, st);
}

}  // namespace attn8
}  // namespace gcu

// k_attention_i8_tc.cu -- attention over the 8-bit KV cache for prompt chunks of
// many rows.
//
// A CTA takes 128 query rows of one kv head (token i, head of the group: the heads
// that share keys fill the rows) and one chunk of the key range, and walks it in tiles
// of NK keys, keeping the running maximum and sum of the softmax:
//   S   three tcgen05.mma kind::i8 products per tile, the query's three digits
//       against the codes as TMA brings them: exact int32 sums in TMEM, put
//       together in fp32 (65536 s2 + 256 s1 + s0).  No conversion of K.
//   P   w = 2^(s + log2 vs[t] - m), m a reference point of the row near the
//       largest exponent so far, split into two fp16 parts in TMEM: w to 2^-22,
//       and to 2^-35 of the row's largest (that is 2^10 or more, just below fp16's
//       largest number, and the second part ends at fp16's smallest, 2^-24).
//   T   two kind::f16 products, P's parts against the V codes as fp16 (exact).
//   l   sum of w / vs in fp32.
// vs rides in the exponent, so w is of the size that counts for the output.  m
// stays where it is until an exponent passes it by kSlack.
//
// The tensor cores add in fp32 by cutting off (measured: 2e-9 of the sum is lost
// per key, 1.7e-5 over 8192 keys), so T holds kFlush tiles at most; then its
// softmax threads add it to the row's sums in their registers, rounded to
// nearest, and the next tile starts T afresh.  The same happens when a row's m
// moves, so the rescaling is a multiplication of registers.
//
// Warps 0-7 and 8-15: two groups of softmax threads, for even and odd tiles, so
// that one's loads and barriers hide behind the other's arithmetic.  In a group
// two threads share a row, half a tile's columns each; of the row's output
// columns each of its four threads holds a quarter in HD/4 registers (some of
// which the last warpgroup gives up).  The groups agree on m through shared
// memory, tile by tile (a "decision").  A group also turns its tile's V codes
// into fp16, in the MN-major layout that the product reads, while its scores are
// formed.  Warp 16: products, issued by one thread of a warp that computes
// the descriptors uniformly; 17: loads.  While the softmax of tile j runs, the
// tensor cores compute S of tile j + 1 and T of tile j - 1.
// Bound by the softmax threads: 2.5 us a tile at hdim 256 against about 1900 cycles of
// products.  8192 tokens of 16 + 8 heads of 256 take 1180 us, 466 TFLOP/s of the
// attention's own products.
// Every wait is bounded; a role that gives up sets the CTA's abort flag, which
// ends the others' waits.
#include "attention_i8.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

namespace gcu {
namespace attn8 {
namespace {

constexpr int kGroup = 256, kSoftmax = 2 * kGroup;  // warps 0-7, 8-15
constexpr int kMmaWarp = 16, kLoadWarp = 17;
constexpr int kThreads = 640;  // setmaxnreg counts whole warpgroups: two warps of the last one idle
constexpr int kRegsSoftmax = 112, kRegsOther = 32;  // 4 * 112 + 32 = 5 * 96
constexpr int kRows = 128;
constexpr int NK = 64;     // keys per tile
constexpr int kFlush = 4;  // tiles per T
// m is placed kTop below the largest exponent so far, so that weights run up to 2^10 and
// may pass that by 2^kSlack: 2^15 stays below fp16's 65504.  Beside scores whose own
// spacing is more than that, m is rounded up, at most to the largest exponent.
constexpr float kTop = 10.0f, kSlack = 5.0f;

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
  static constexpr int REF_OFF = SC_OFF + 4 * 3 * NK * 4;     // [128] reference points
  static constexpr int MAX_OFF = REF_OFF + kRows * 4;         // [2][2][128] row maxima (at the end: sums)
  static constexpr int RF_OFF = MAX_OFF + 4 * kRows * 4;  // [128] score factors
  static constexpr int SMEM = RF_OFF + kRows * 4 + 1024;
  // TMEM columns: S of three digits, T, P (two parts, two keys per column)
  static constexpr int HALF = NK / 2;  // score columns per softmax thread
  static constexpr int OC = HD / 4;    // output columns per softmax thread
  static constexpr int RB = HD == 256 ? 8 : 16;  // score columns read at a time (registers)
  static constexpr int S_COL = 0, T_COL = 3 * NK, P_COL = T_COL + HD;
  static_assert(V16_OFF - Q_OFF >= kRows * HD * 4, "the output's stage");
  static_assert(SMEM <= 232448 - 512, "shared memory budget");
  static_assert(P_COL + NK <= 512, "TMEM budget");
};

struct alignas(64) TcArgs {
  CUtensorMap tmK;
  Args a;
  int tiles;  // query tiles per kv head (of the largest group)
};

struct Bars {
  uint64_t kfull[2], kempty[2], v8full[2], v8empty[2], v16full[2], dec[2], sfull[2], pvdone[2], sfree, pfull, tfree, drain;
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

__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[8]) { ptx::tmem_ld_32x8(at, r); }
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[16]) { ptx::tmem_ld_32x16(at, r); }

// whether a value row is all zeros; kFly loads at a time once its first 16 codes are
template <int HD>
__device__ __forceinline__ bool row_of_zeros(const int8_t *codes) {
  constexpr int N = HD / 16, kFly = 5;
  const uint4 *p = reinterpret_cast<const uint4 *>(codes);
  const uint4 f = __ldg(p);
  uint32_t any = f.x | f.y | f.z | f.w;
#pragma unroll 1
  for (int i = 1; i < N && !any; i += kFly) {
    uint4 w[kFly];
#pragma unroll
    for (int t = 0; t < kFly; ++t) w[t] = __ldg(p + min(i + t, N - 1));
#pragma unroll
    for (int t = 0; t < kFly; ++t) any |= w[t].x | w[t].y | w[t].z | w[t].w;
  }
  return !any;
}

// thread i < NK puts ks[i], i < 2 NK log2 and reciprocal of vs[i - NK]
__device__ __forceinline__ void put_scale(float *sc, int i, float v) {
  if (i < NK) {
    sc[i] = v;
  } else if (i < 2 * NK) {
    value_scale(v, sc[i], sc[i + NK]);
  }
}

template <int HD, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) k_tc(const __grid_constant__ TcArgs p) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_fresh[2], s_range[4];  // first key, end, last start of a window, first end
  // aligned by an offset: the accesses stay in the shared address space
  uint8_t *smem = smem_raw + ((1024 - (ptx::smem_u32(smem_raw) & 1023)) & 1023);
  const Args &a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // heavy CTAs first: the first chunks, and of each the last query rows, which see
  // the most keys; the heads side by side
  const int hk = blockIdx.x % a.kv.nkv, unit = blockIdx.x / a.kv.nkv, split = unit / p.tiles;
  const int tile = p.tiles - 1 - (unit - split * p.tiles);
  const int h0 = head0(hk, a.n_heads, a.kv.nkv), G = head0(hk + 1, a.n_heads, a.kv.nkv) - h0;
  const int first = tile * kRows, nrows = min(kRows, a.ni * G - first);
  const RowSplit rows(first, G);
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&bars.kfull[s], 1);
      ptx::mbar_init(&bars.kempty[s], 1);
      ptx::mbar_init(&bars.v8full[s], 1);
      ptx::mbar_init(&bars.v8empty[s], kGroup / 32);
      ptx::mbar_init(&bars.v16full[s], kGroup / 32);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&bars.dec[s], kGroup / 32);
      ptx::mbar_init(&bars.sfull[s], 1);
      ptx::mbar_init(&bars.pvdone[s], 1);
    }
    ptx::mbar_init(&bars.sfree, kGroup / 32);
    ptx::mbar_init(&bars.pfull, kGroup / 32);
    ptx::mbar_init(&bars.tfree, 2 * kGroup / 32);
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
    row_window(a, rows.i(threadIdx.x), lo, hi);
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
  // rows whose keys fit into one chunk go straight to xo, and slot 0 tells the merge
  const bool alone = a.slots == 1 || (long)s_range[1] - s_range[0] <= a.chunk;
  Waiter wait{&s_abort, a.err};

  const int8_t *vh = a.kv.v + hk * a.kv.kv_stride, *kh = a.kv.k + hk * a.kv.kv_stride;
  // the loads of tile j (one thread)
  auto load_k = [&](int j, uint64_t pol) {
    uint64_t *bar = &bars.kfull[j & 1];
    ptx::mbar_arrive_expect_tx(bar, C::K_BYTES);
#pragma unroll
    for (int b = 0; b < C::KB; ++b)
      ptx::tma_load_4d(&p.tmK, bar, smem + C::K_OFF + (j & 1) * C::K_BYTES + b * C::K_BLOCK, b * C::SW, kbeg + j * NK, hk,
                       0, pol);
  };
  auto load_v = [&](int j, uint64_t pol) {
    const uint32_t bytes = (uint32_t)min(NK, n - j * NK) * HD;
    uint64_t *bar = &bars.v8full[j & 1];
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
    // a row ahead in flight; one copy of the code, which every CTA fetches anew
    constexpr int E = HD / 32, W = kThreads / 32;
    auto load_row = [&](float (&v)[E], int r) {
      load_floats<E>(v, a.xq + (long)rows.i(r) * a.q_i + (long)(h0 + rows.g(r)) * a.q_h + lane * E, r < nrows);
    };
    float v[2][E], ahead[2][E];  // two rows at a time: their reductions overlap
    load_row(v[0], warp);
    load_row(v[1], warp + W);
#pragma unroll 1
    for (int r0 = warp; r0 < kRows; r0 += 2 * W) {
      load_row(ahead[0], r0 + 2 * W);
      load_row(ahead[1], r0 + 3 * W);
      float amax[2];
      uint32_t w[2][3][(E + 3) / 4];
      row_digits<E, 2>(v, w, amax);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = r0 + t * W, col = lane * E, in = col % C::SW;
        if (r >= kRows) break;
        const int sw = C::SW == 128 ? r & 7 : (r >> 1) & 3;
        uint8_t *dst = smem + C::Q_OFF + (col / C::SW) * C::Q_BLOCK + r * C::SW + (((in >> 4) ^ sw) << 4) + (in & 15);
#pragma unroll
        for (int d = 0; d < 3; ++d) put_digits<E>(dst + d * C::KB * C::Q_BLOCK, w[t][d]);
        if (lane == 0) s_rf[r] = amax[t] / kQMax * a.asc;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[0][e] = ahead[0][e];
        v[1][e] = ahead[1][e];
      }
    }
    // tile 0's scales
    if ((int)threadIdx.x < 2 * NK) {
      const int t = threadIdx.x % NK;
      const float *src = (threadIdx.x < NK ? a.kv.ks : a.kv.vs) + hk * a.kv.sc_stride;
      float v = t < n ? __ldg(src + kbeg + t) : 1.0f;
      if (v == 1.0f && threadIdx.x >= NK && t < n && row_of_zeros<HD>(vh + (long)(kbeg + t) * HD)) v = kScaleZeros;
      put_scale(reinterpret_cast<float *>(smem + C::SC_OFF), threadIdx.x, v);
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
      for (int j = max(0, nv - 2); j < nv; ++j)
        ptx::mbar_wait(&bars.v8full[j & 1], (j >> 1) & 1, a.err, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ products
    const int tiles = __shfl_sync(0xffffffffu, nt, 0);
    if (tiles > 0) {
      constexpr uint32_t id_s = ptx::idesc_i8(kRows, NK), id_o = ptx::idesc_f16_bt(kRows, HD);
      const ptx::Desc dq = ptx::smem_desc(ptx::smem_u32(smem + C::Q_OFF), 16, 8 * C::SW, C::SW);
      const ptx::Desc dk = ptx::smem_desc(ptx::smem_u32(smem + C::K_OFF), 16, 8 * C::SW, C::SW);
      const ptx::Desc dv = ptx::smem_desc(ptx::smem_u32(smem + C::V16_OFF), C::V16_BLOCK, 1024, 128);
      auto scores = [&](int j) {
        if (ptx::elect_one()) {
          const uint32_t k_lo = dk.lo + (j & 1) * (C::K_BYTES >> 4);
#pragma unroll
          for (int b = 0; b < C::KB; ++b)
#pragma unroll
            for (int s = 0; s < C::SW / 32; ++s)
#pragma unroll
              for (int d = 0; d < 3; ++d)
                ptx::mma_i8(tmem + C::S_COL + d * NK,
                            ptx::Desc{dq.lo + (((d * C::KB + b) * C::Q_BLOCK + 32 * s) >> 4), dq.hi},
                            ptx::Desc{k_lo + ((b * C::K_BLOCK + 32 * s) >> 4), dk.hi}, id_s, b + s > 0 ? 1u : 0u);
          ptx::mma_commit(&bars.kempty[j & 1]);
          ptx::mma_commit(&bars.sfull[j & 1]);
        }
        __syncwarp();
      };
      auto values = [&](int j, bool fresh) {
        if (ptx::elect_one()) {
          const uint32_t v_lo = dv.lo + (j & 1) * (C::V16_BYTES >> 4);
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int s = 0; s < NK / 16; ++s)
              ptx::mma_f16_ts(tmem + C::T_COL, tmem + C::P_COL + part * (NK / 2) + 8 * s,
                              ptx::Desc{v_lo + ((s * 2048) >> 4), dv.hi}, id_o, part + s > 0 || !fresh ? 1u : 0u);
          ptx::mma_commit(&bars.pvdone[j & 1]);
        }
        __syncwarp();
      };
      // The two products of a tile wait for different things: T of tile jt for its
      // weights, S of tile js for its keys and for S of tile js - 1 to have been read.
      // Whichever can go goes, T first.
      uint64_t t0 = ptx::globaltimer();
      for (int js = 0, jt = 0, taken = 0; jt < tiles;) {
        bool go = false;
        if (jt < js && __all_sync(0xffffffffu, ptx::mbar_test(&bars.pfull, jt & 1) &&
                                                   ptx::mbar_test(&bars.v16full[jt & 1], (jt >> 1) & 1))) {
          const bool fresh = __shfl_sync(0xffffffffu, *(volatile int *)&s_fresh[jt & 1], 0), taking = fresh && jt > 0;
          if (!taking || __all_sync(0xffffffffu, ptx::mbar_test(&bars.tfree, taken & 1))) {
            ptx::tc_fence_after();
            values(jt++, fresh);
            taken += taking;
            go = true;
          }
        }
        if (js < tiles && __all_sync(0xffffffffu, ptx::mbar_test(&bars.kfull[js & 1], (js >> 1) & 1) &&
                                                      (js == 0 || ptx::mbar_test(&bars.sfree, (js - 1) & 1)))) {
          ptx::tc_fence_after();
          scores(js++);
          go = true;
        }
        if (go) {
          t0 = ptx::globaltimer();
        } else if (*wait.abort || ptx::globaltimer() - t0 > 2000000000ull) {
          if (lane == 0 && !*wait.abort) {
            ptx::record_err(a.err, DEV_TIMEOUT_TMEM);
            *wait.abort = 1;
          }
          break;
        }
      }
      // all products complete before TMEM is freed
      if (ptx::elect_one()) ptx::mma_commit(&bars.drain);
      __syncwarp();
      ptx::mbar_wait(&bars.drain, 0, a.err, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp < kSoftmax / 32) {
    // ------------------------------------------------------------ softmax
    ptx::regs_inc<kRegsSoftmax>();
    const int grp = warp >> 3, half = (warp >> 2) & 1, quarter = warp >> 2;
    const int row = threadIdx.x & (kRows - 1), tid = threadIdx.x & (kGroup - 1);
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    float *sc = reinterpret_cast<float *>(smem + C::SC_OFF);
    volatile float *refs = reinterpret_cast<float *>(smem + C::REF_OFF);
    volatile float *smax = reinterpret_cast<float *>(smem + C::MAX_OFF);
    volatile int *freshp = s_fresh;
    const bool live = row < nrows;
    int lo = 0, hi = 0;
    if (live) row_window(a, rows.i(row), lo, hi);
    // scores from digit sums: natural units over the cap, then times the cap, or log2 units
    float rf_nat = nt > 0 ? s_rf[row] : 0.0f, rf = rf_nat * kLog2e;
    if (CAP) {
      rf_nat /= a.sc_att;
      rf = a.sc_att * kLog2e;
    }
    // scales of the other group's next tile: thread tid of ks (tid < NK) or vs
    auto fetch_scale = [&](int j) {
      const int t = j * NK + (tid & (NK - 1));
      return tid < 2 * NK && t < n ? __ldg((tid < NK ? a.kv.ks : a.kv.vs) + hk * a.kv.sc_stride + kbeg + t) : 1.0f;
    };
    float next = fetch_scale(grp + 1);
    // a scale of tile j that is 1: the row may be zeros.  Looked at after a tile's work, while
    // the other group is at its own.
    auto look = [&](int j) {
      const int t = j * NK + (tid & (NK - 1));
      if (next == 1.0f && tid >= NK && tid < 2 * NK && t < n && row_of_zeros<HD>(vh + (long)(kbeg + t) * HD))
        next = kScaleZeros;
    };
    look(grp + 1);
    float m = -INFINITY, l = 0.0f;
    float acc[C::OC];  // the row's sums, output columns [quarter * OC, +OC)
#pragma unroll
    for (int c = 0; c < C::OC; ++c) acc[c] = 0.0f;
    // add T (complete) to the row's sums, then scale them
    auto flush = [&](float f) {
      ptx::tc_fence_after();
#pragma unroll
      for (int c = 0; c < C::OC; c += 16) {
        uint32_t t[16];
        ptx::tmem_ld_32x16(lanes + C::T_COL + quarter * C::OC + c, t);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[c + e] = (acc[c + e] + __uint_as_float(t[e])) * f;
      }
      ptx::tc_fence_before();
    };
    bool ok = true;
    // take over the decision of tile j (the other group's): its reference point,
    // and T's sums when its product starts T afresh
    auto follow = [&](int j) {
      ok = wait(&bars.dec[j & 1], (j >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      const float to = refs[row];
      const float f = to == m ? 1.0f : ex2(m - to);  // m = -inf: 0
      l *= f;
      m = to;
      if (j > 0 && freshp[j & 1]) {
        ok = wait(&bars.pvdone[(j - 1) & 1], ((j - 1) >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
        flush(f);
        ptx::mbar_arrive_warp(&bars.tfree);
      }
    };
    // V codes of tile j to fp16; 8 columns of a key per thread.  Keys past the range
    // hold an earlier tile's codes, which weigh nothing.  At hdim 256 it fits into the
    // wait for the scores (8192 tokens 1264 -> 1239 us); with shorter score products
    // that wait is short, and it goes between the weights and the wait for the
    // previous product (hdim 128 1000 -> 897 us).
    auto convert = [&](int j) {
      ok = wait(&bars.v8full[j & 1], (j >> 1) & 1, DEV_TIMEOUT_FULL) && ok;
      if (j > 1) ok = wait(&bars.pvdone[j & 1], ((j - 2) >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      {
        constexpr int L = HD / 8, KS = kGroup / L;
        const int c = tid % L, key0 = tid / L;
        const uint8_t *src = smem + C::V8_OFF + (j % C::NV8) * C::V8_BYTES + c * 8;
        uint8_t *dst = smem + C::V16_OFF + (j & 1) * C::V16_BYTES + (c >> 3) * C::V16_BLOCK;
#pragma unroll
        for (int k = 0; k < NK; k += KS) {
          const int key = key0 + k;
          const uint2 w = *reinterpret_cast<const uint2 *>(src + key * HD);
          const uint2 x = to_half4(w.x), y = to_half4(w.y);
          *reinterpret_cast<uint4 *>(dst + key * 128 + (((c & 7) ^ (key & 7)) << 4)) = make_uint4(x.x, x.y, y.x, y.y);
        }
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive_warp(&bars.v8empty[j % C::NV8]);
        ptx::mbar_arrive_warp(&bars.v16full[j & 1]);
      }
    };
    int j = grp;
    for (; j < nt; j += 2) {
      const float *ks = sc + (j & 3) * 3 * NK + half * C::HALF, *lvs = ks + NK, *rvs = ks + 2 * NK;
      if (j > 0) follow(j - 1);
      // while the scores are formed: the scales of the other group's next tile, which it
      // reads after this tile's decision, and the values
      put_scale(sc + ((j + 1) & 3) * 3 * NK, tid, next);
      next = fetch_scale(j + 3);
      if (HD == 256) convert(j);
      ok = wait(&bars.sfull[j & 1], (j >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      ptx::tc_fence_after();
      // exponents: the score in log2 units plus log2 of the value row's scale
      float x[C::HALF];
#pragma unroll
      for (int c = 0; c < C::HALF; c += C::RB) {
        uint32_t s1[C::RB], s0[C::RB];
        const uint32_t at = lanes + C::S_COL + half * C::HALF + c;
        tmem_ld(at, s0);
        tmem_ld(at + NK, s1);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < C::RB; e += 2) {
          const float2 u = low_digits(s1 + e, s0 + e);
          x[c + e] = u.x;
          x[c + e + 1] = u.y;
        }
      }
#pragma unroll
      for (int c = 0; c < C::HALF; c += C::RB) {
        uint32_t s2[C::RB];
        tmem_ld(lanes + C::S_COL + 2 * NK + half * C::HALF + c, s2);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < C::RB; e += 4) {
          const float4 k = *reinterpret_cast<const float4 *>(ks + c + e);
          const float4 v = *reinterpret_cast<const float4 *>(lvs + c + e);
          // q . kc first: digits times a scale of 1e28 would run over
          const float2 f = CAP ? make_float2(rf_nat, rf_nat) : make_float2(rf, rf);
          float2 y = __fmul2_rn(high_digit(s2 + e, make_float2(x[c + e], x[c + e + 1])), f);
          float2 z = __fmul2_rn(high_digit(s2 + e + 2, make_float2(x[c + e + 2], x[c + e + 3])), f);
          if constexpr (CAP) {
            y = __ffma2_rn(make_float2(tanh_fast(y.x * k.x), tanh_fast(y.y * k.y)), make_float2(rf, rf), make_float2(v.x, v.y));
            z = __ffma2_rn(make_float2(tanh_fast(z.x * k.z), tanh_fast(z.y * k.w)), make_float2(rf, rf), make_float2(v.z, v.w));
          } else {
            y = __ffma2_rn(y, make_float2(k.x, k.y), make_float2(v.x, v.y));
            z = __ffma2_rn(z, make_float2(k.z, k.w), make_float2(v.z, v.w));
          }
          x[c + e] = y.x;
          x[c + e + 1] = y.y;
          x[c + e + 2] = z.x;
          x[c + e + 3] = z.y;
        }
      }
      ptx::tc_fence_before();
      ptx::mbar_arrive_warp(&bars.sfree);
      // a tile that some row does not see in full
      const int t0 = kbeg + j * NK;
      if (t0 < all_lo || t0 + NK > min(all_hi, kend)) {
        const int cl = lo - t0 - half * C::HALF, ch = min(hi, kend) - t0 - half * C::HALF;
#pragma unroll
        for (int c = 0; c < C::HALF; ++c)
          if (c < cl || c >= ch) x[c] = -INFINITY;
      }
      float top = -INFINITY, top2 = -INFINITY;
#pragma unroll
      for (int c = 0; c < C::HALF; c += 4) {
        top = fmaxf(fmaxf(top, x[c]), x[c + 1]);
        top2 = fmaxf(fmaxf(top2, x[c + 2]), x[c + 3]);
      }
      top = fmaxf(top, top2);
      smax[(grp * 2 + half) * kRows + row] = top;
      const bool moved = ptx::named_bar_or(1 + grp, kGroup, top > __fadd_rd(m, kTop + kSlack) || !ok);
      if (moved && ptx::named_bar_or(1 + grp, kGroup, !ok)) break;
      const float to =
          moved ? fmaxf(m, __fsub_ru(fmaxf(top, smax[(grp * 2 + (half ^ 1)) * kRows + row]), kTop)) : m;
      const bool fresh = moved || j % kFlush == 0;
      if (half == 0) refs[row] = to;
      if (tid == 0) freshp[j & 1] = fresh;
      ptx::mbar_arrive_warp(&bars.dec[j & 1]);
      const float f = to == m ? 1.0f : ex2(m - to);  // m = -inf: 0
      l *= f;
      m = to;
      const float ref = m == -INFINITY ? 0.0f : m;
      uint32_t ph[C::HALF / 2], pl[C::HALF / 2];
      float2 lt = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int c = 0; c < C::HALF; c += 4) {
        const float4 r = *reinterpret_cast<const float4 *>(rvs + c);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 d = __fadd2_rn(make_float2(x[c + e], x[c + e + 1]), make_float2(-ref, -ref));
          const float2 w = make_float2(ex2(d.x), ex2(d.y));
          lt = __ffma2_rn(w, e ? make_float2(r.z, r.w) : make_float2(r.x, r.y), lt);
          const __half2 hi2 = __floats2half2_rn(w.x, w.y);
          const float2 back = __half22float2(hi2);
          const float2 rest = __fadd2_rn(w, make_float2(-back.x, -back.y));
          const __half2 lo2 = __floats2half2_rn(rest.x, rest.y);
          ph[(c + e) / 2] = *reinterpret_cast<const uint32_t *>(&hi2);
          pl[(c + e) / 2] = *reinterpret_cast<const uint32_t *>(&lo2);
        }
      }
      l += lt.x + lt.y;
      if (HD != 256) convert(j);
      // P and T are free once the previous tile's product is done
      if (j > 0) {
        ok = wait(&bars.pvdone[(j - 1) & 1], ((j - 1) >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
        if (fresh) {
          flush(f);
          ptx::mbar_arrive_warp(&bars.tfree);
        }
      }
      ptx::tc_fence_after();
      ptx::tmem_st_32x16(lanes + C::P_COL + half * (C::HALF / 2), ph);
      ptx::tmem_st_32x16(lanes + C::P_COL + NK / 2 + half * (C::HALF / 2), pl);
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      ptx::mbar_arrive_warp(&bars.pfull);
      look(j + 3);
    }
    // the group without the last tile follows its decision too (j is the tile
    // after it); then both take what is left in T
    if (j == nt && nt > 0) follow(nt - 1);
    if (nt > 0) {
      ok = wait(&bars.pvdone[(nt - 1) & 1], ((nt - 1) >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      flush(1.0f);
    }
    // the row's sum over its four threads, which end with the same m
    ptx::named_bar_sync(3, kSoftmax);
    smax[quarter * kRows + row] = l;
    ptx::named_bar_sync(3, kSoftmax);
    l = (smax[row] + smax[kRows + row]) + (smax[2 * kRows + row] + smax[3 * kRows + row]);
    // Rows go out through shared memory (the queries' and keys' is free now: every
    // product that reads them is done), a warp per row, 512 bytes at a time.
    const float d = !alone || l == 0.0f ? 1.0f : 1.0f / l;  // a row that sees nothing: zeros
    float4 *stage = reinterpret_cast<float4 *>(smem);
#pragma unroll
    for (int c = 0; c < C::OC; c += 4)
      stage[row * (HD / 4) + ((quarter * C::OC + c) / 4 ^ (row & 7))] =
          make_float4(acc[c] * d, acc[c + 1] * d, acc[c + 2] * d, acc[c + 3] * d);
    if (live && ok && a.slots > 1 && quarter == 0 && (!alone || split == 0))
      a.stat[((size_t)(a.slot0 + split) * a.ni + rows.i(row)) * a.n_heads + h0 + rows.g(row)] =
          alone ? make_float2(0.0f, kAlone) : make_float2(m, l);
    ptx::named_bar_sync(3, kSoftmax);
    const bool none = alone ? split > 0 : nt == 0;  // (-inf, 0) says that there is nothing to add
    for (int r = warp; r < nrows && ok && !none; r += kSoftmax / 32) {
      const int i = rows.i(r), h = h0 + rows.g(r);
      float *out = alone ? a.xo + (long)i * a.o_i + (long)h * HD
                         : a.part + (((size_t)(a.slot0 + split) * a.ni + i) * a.n_heads + h) * HD;
#pragma unroll
      for (int c = lane; c < HD / 4; c += 32) reinterpret_cast<float4 *>(out)[c] = stage[r * (HD / 4) + (c ^ (r & 7))];
    }
  }
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, 512);
}

template <int HD, bool CAP>
int launch_tc_hd(const Args &a, cudaStream_t st) {
  using C = Cfg<HD>;
  TcArgs p;
  p.a = a;
  const int gmax = (a.n_heads + a.kv.nkv - 1) / a.kv.nkv;
  p.tiles = (int)(((long)a.ni * gmax + kRows - 1) / kRows);
  const long ctas = (long)p.tiles * a.splits * a.kv.nkv;
  if (ctas > 0x7fffffffL) return set_error("attention_i8: %ld CTAs", ctas);
  if (gemm_tmap_heads_i8(&p.tmK, a.kv.k, a.kv, NK)) return 1;
  {
    // the shared-memory opt-in is per device: once for each device this runs on
    static std::mutex mu;
    static unsigned long long done = 0;
    int dev = 0;
    GCU_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (!(done & (1ull << (dev & 63)))) {
      GCU_CUDA(cudaFuncSetAttribute(k_tc<HD, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
      done |= 1ull << (dev & 63);
    }
  }
  GCU_CUDA(launch_k(k_tc<HD, CAP>, dim3((unsigned)ctas), dim3(kThreads), C::SMEM, st, p));
  return 0;
}

template <bool CAP>
int launch_tc_cap(const Args &a, cudaStream_t st) {
  return a.kv.hdim == 256   ? launch_tc_hd<256, CAP>(a, st)
         : a.kv.hdim == 128 ? launch_tc_hd<128, CAP>(a, st)
                            : launch_tc_hd<64, CAP>(a, st);
}

}  // namespace

int launch_tc(const Args &a, cudaStream_t st) {
  return a.sc_att != 0.0f ? launch_tc_cap<true>(a, st) : launch_tc_cap<false>(a, st);
}

}  // namespace attn8
}  // namespace gcu

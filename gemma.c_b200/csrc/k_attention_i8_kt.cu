// k_attention_i8_kt.cu -- attention over the 8-bit KV cache for few query rows per kv
// head (the heads of one token, of the tokens of several sequences that share a
// prefix, or of a short prompt).  The codes are read once, as they lie, and go
// from TMA into the tensor cores without a conversion.
//
// With few rows the keys take the long side of the products:
//   S^T  [128 keys x 3R]    = K [128 x hdim] * Q^T, the R rows' three digits side
//                             by side (kind::i8, exact)
//   O^T  [hdim x 4R]       += V^T [hdim x 128 keys] * W, the R rows' weights as four
//                             unsigned digits each, the bytes of an integer as they
//                             lie (kind::i8 with both operands MN-major: V's tile
//                             as it lies is V^T)
// Weights are 32-bit fixed point, W = round(2^(s + e - m) * f + d_t) for a value scale
// of 2^e * f, 1 <= f < 2, m placed so that the row's largest weight so far is 2^25 at
// least and below 2^32.  The offset d_t in [-1/2, 1/2) runs through the golden
// ratio's multiples along the keys: of many small weights some gain what others lose
// (of n equal ones a few steps are left, where plain rounding could take all of them),
// so a sum of products is off by about sqrt(n) / 2 steps of 2^-25 of the largest weight, while
// the sum of weights, in fp32, is of the weights as they were.
// O stays in int32 in TMEM (a digit's sum over 66,312 keys fits, and the plan gives a
// CTA fewer), so nothing more is lost, and only moves to fp32 registers when a row's
// m has to move.
//
// Per 128 keys at hdim 256 this is 16 products of N <= 128 (about 1100 cycles)
// against 64 KB of codes, which at the card's copy rate are 2800 cycles of one SM.  A CTA
// costs 5.4 us besides its tiles and, with 16 rows, 1.0 us a tile whose codes are in L2;
// from HBM 148 CTAs of 32 tiles take 50 us for 310 MB.  32768 keys of 8 heads: 29.6 us for
// 136 MB, the merge of 18 chunks 3.6 of them.  32 rows are bound by the softmax, 1.5 us a
// tile: 32 sequences that share 32768 keys 63 us, 52 without keys of their own.
//
// Warps 0-15: softmax, thread = (key, a quarter of the rows); 16: products; 17: loads.
#include "attention_i8.cuh"

#include <cooperative_groups.h>

#include <mutex>

namespace gcu {
namespace attn8 {
namespace {

constexpr int kSoftmax = 512, kMmaWarp = 16, kLoadWarp = 17, kThreads = 576;
constexpr int kKeys = kKtKeys;
// log2 of W at m (over f), and by how much an exponent may pass m: what precision wants
// high and few moves of m want low.  It multiplies f, so that the exponent is x - m for
// scores of any size.  32 sequences that share 32768 keys, prompt of 512: 62.9 and 12.8 us
// with 24, 63.2 and 12.9 with 25, 64.3 and 13.2 with 26, 66.5 and 13.8 with 28.
constexpr int kTop = 25;
constexpr float kSlack = 5.9f, kOne = 1 << kTop;

// A value row's scale 2^e * f, as attn8::value_scale limits it: e (NaN for NaN, which then
// makes the weights NaN where the key is seen; elsewhere the others are finite
// against the zero weight), f * 2^kTop and 2^-e.  Exact, and a quarter of the instructions
// that a logarithm and a reciprocal take (32 sequences that share 32768 keys 63.0
// -> 60.9 us).
__device__ __forceinline__ void split_scale(float v, float &e, float &f, float &inv) {
  v = v < kScaleLo ? kScaleLo : v > kScaleHi ? kScaleHi : v;
  const int b = __float_as_int(v), x = min(b & 0x7f800000, 0x71800000);  // NaN as 2^100
  e = v == v ? (float)((x >> 23) - 127) : v;
  f = __int_as_float((b & 0x007fffff) | (0x3f800000 + (kTop << 23)));
  inv = __int_as_float(0x7f000000 - x);
}

template <int HD, int R>
struct Cfg {
  static constexpr int SW = HD == 64 ? 64 : 128;  // bytes of a Q / K / V swizzle row
  static constexpr int KB = HD / SW;              // blocks of SW bytes
  static constexpr int NS = 3 * R, NP = 4 * R;    // columns of S^T and of W
  static constexpr int MB = HD == 256 ? 2 : 1;    // 128-row blocks of O^T (hdim 64: rows 64-127 repeat)
  static constexpr int Q_BLOCK = NS * SW;
  static constexpr int Q_BYTES = KB * Q_BLOCK;
  static constexpr int T_BLOCK = kKeys * SW;
  static constexpr int T_BYTES = KB * T_BLOCK;  // a K or V tile
  static constexpr int P_ROW = NP;              // bytes of a key: 64 or 128
  static constexpr int P_BYTES = kKeys * P_ROW;
  static constexpr int Q_PAD = (Q_BYTES + 1023) / 1024 * 1024;
  static constexpr int FIXED = Q_PAD + 2 * P_BYTES + 1024 + 6 * 1024;
  static constexpr int FIT = (232448 - FIXED) / (2 * T_BYTES);
  static constexpr int STAGES = FIT > 6 ? 6 : FIT;  // of K and of V
  static constexpr int Q_OFF = 0;
  static constexpr int P_OFF = Q_PAD;
  static constexpr int K_OFF = P_OFF + 2 * P_BYTES;
  static constexpr int V_OFF = K_OFF + STAGES * T_BYTES;
  static constexpr int SMEM = V_OFF + STAGES * T_BYTES + 1024;
  static constexpr int S_COL = 0, O_COL = 2 * NS;
  static constexpr int COLS = O_COL + MB * NP <= 256 ? 256 : 512;
  static constexpr int RQ = R / 4;                      // rows per softmax thread
  static constexpr int OR = HD == 256 ? R / 2 : R / 4;  // output rows per thread (of one column)
  static_assert(STAGES >= 2 && O_COL + MB * NP <= 512, "budget");
};

__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[4]) { ptx::tmem_ld_32x4(at, r); }
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[8]) { ptx::tmem_ld_32x8(at, r); }

// Whether a value row is all zeros, in its tile as TMA left it: 16-byte steps of the
// row's SW bytes in the order that spreads neighbouring keys over the banks.
template <typename C>
__device__ __forceinline__ bool row_of_zeros(const uint8_t *row, int key) {
  uint32_t any = 0;
#pragma unroll 1
  for (int i = 0; i < C::KB * C::SW / 16 && !any; ++i) {
    const int b = i * 16 / C::SW, at = (i ^ (C::SW == 128 ? key : key >> 1)) % (C::SW / 16);
    const uint4 w = *reinterpret_cast<const uint4 *>(row + b * C::T_BLOCK + at * 16);
    any = w.x | w.y | w.z | w.w;
  }
  return !any;
}

struct alignas(64) KtArgs {
  CUtensorMap k[2], v[2];
  Args a[2];
  int first1;  // CTAs of set 0: the longer set's come first
};

template <int HD, int R, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) k_kt(const __grid_constant__ KtArgs p) {
  using C = Cfg<HD, R>;
  constexpr int ST = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t kfull[ST], kempty[ST], vfull[ST], vempty[ST], sfull[2], sfree[2], pfull[2], pvdone[2], drain;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_gone, s_fresh[2], s_lo[R], s_hi[R], s_row[R];
  __shared__ long s_out[R];
  __shared__ float s_part[kKtCluster][R];  // a fused merge's factors
  __shared__ float s_rf[R], s_m[R], s_f[R], s_sum[R], s_red[16][R / 4];
  // aligned by an offset: the accesses stay in the shared address space
  uint8_t *smem = smem_raw + ((1024 - (ptx::smem_u32(smem_raw) & 1023)) & 1023);
  float *part = reinterpret_cast<float *>(smem + C::K_OFF);  // a fused merge's sums, over K's first tile
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int set = (int)blockIdx.x >= p.first1;
  const Args &a = p.a[set];
  const int block = (int)blockIdx.x - (set ? p.first1 : 0);
  const int split = block % a.splits, unit = block / a.splits;
  int group = unit / a.kv.nkv;
  const int hk = unit - group * a.kv.nkv;
  // a prompt's last rows see the most keys: they come first
  if (a.mode == PREFILL) group = (int)gridDim.x / (a.splits * a.kv.nkv) - 1 - group;
  const int h0 = head0(hk, a.n_heads, a.kv.nkv), G = head0(hk + 1, a.n_heads, a.kv.nkv) - h0;
  // rows of this CTA: OWN one sequence's group, else R of the (i, g) rows
  const int first = a.mode == OWN ? group * G : group * R;
  const int nr = max(0, a.mode == OWN ? G : min(R, a.ni * G - first));
  const RowSplit rows(first, G);
  const bool fused = a.slots == 1 && a.splits > 1;  // the splits are a cluster
  // The loads start before anything else: their warp sets up their barriers.
  if (warp == kLoadWarp && lane == 0) {
    ptx::prefetch_tmap(&p.k[set]);
    ptx::prefetch_tmap(&p.v[set]);
    for (int s = 0; s < ST; ++s) {
      ptx::mbar_init(&kfull[s], 1);
      ptx::mbar_init(&kempty[s], 1);
      ptx::mbar_init(&vfull[s], 1);
      ptx::mbar_init(&vempty[s], 1);
    }
    ptx::fence_mbar_init();
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(&sfull[s], 1);
      ptx::mbar_init(&sfree[s], kSoftmax / 32);
      ptx::mbar_init(&pfull[s], kSoftmax / 32);
      ptx::mbar_init(&pvdone[s], 1);
    }
    ptx::mbar_init(&drain, 1);
    ptx::fence_mbar_init();
    s_abort = s_gone = 0;
  }
  ptx::griddep_wait();

  // The rows' windows, lane r of every warp: the CTA's key range, and the keys that
  // every row sees.
  int lo = 0, hi = 0, row = 0;  // row: its place among the i * n_heads + h
  long from = 0, to = 0;        // in xq and xo
  if (lane < nr) {
    const int i = rows.i(lane), h = h0 + rows.g(lane);
    row = i * a.n_heads + h;
    from = i * a.q_i + h * a.q_h;
    to = i * a.o_i + (long)h * HD;
    row_window(a, i, lo, hi);
    if (!row_live(a, i)) row = -1;
  }
  if (threadIdx.x < R) {
    s_row[threadIdx.x] = row;
    s_out[threadIdx.x] = to;
    s_lo[threadIdx.x] = lo;
    s_hi[threadIdx.x] = hi;
    s_m[threadIdx.x] = -INFINITY;
  }
  const int any_lo = __reduce_min_sync(0xffffffffu, lo < hi ? lo : 0x7fffffff);
  const int any_hi = __reduce_max_sync(0xffffffffu, lo < hi ? hi : 0);
  const int all_lo = __reduce_max_sync(0xffffffffu, lo);
  const int all_hi = __reduce_min_sync(0xffffffffu, lane < nr ? hi : 0x7fffffff);
  const long c0 = (long)any_lo + (long)split * a.chunk;
  const int n = (int)max(0l, min((long)any_hi, c0 + a.chunk) - c0);
  const int kbeg = (int)min(c0, 0x7fffffffl), kend = kbeg + n, nt = (n + kKeys - 1) / kKeys;
  const int seq = a.mode == OWN ? group : 0;
  Waiter wait{&s_abort, a.err};
  if (a.mode == OWN && a.len && threadIdx.x == 0 && split == 0 && hk == 0 && __ldg(a.len + group) > a.max_len)
    ptx::record_err(a.bad_len, DEV_BAD_LENGTH);

  const uint64_t pol = ptx::policy_evict_first();
  auto load = [&](const CUtensorMap *m, uint64_t *full, int off, int j) {
    const int st = j % ST;
    ptx::mbar_arrive_expect_tx(&full[st], C::T_BYTES);
#pragma unroll
    for (int b = 0; b < C::KB; ++b)
      ptx::tma_load_4d(m, &full[st], smem + off + st * C::T_BYTES + b * C::T_BLOCK, b * C::SW, kbeg + j * kKeys, hk, seq,
                       pol);
  };
  if (warp == kLoadWarp && lane == 0)
    for (int j = 0; j < min(ST, nt); ++j) {
      load(&p.k[set], kfull, C::K_OFF, j);
      load(&p.v[set], vfull, C::V_OFF, j);
    }

  if (warp == kMmaWarp) {
    ptx::tmem_alloc(&s_tmem, C::COLS);
    ptx::tmem_relinquish();
  }
  // the query rows' digits, row n = d * R + r; rows past the end are zeros
  if (nt > 0) {
    constexpr int E = HD / 32, W = kThreads / 32, N = (R + W - 1) / W;  // rows of a warp
    float vs[N][E];  // of all its rows in flight at once
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = warp + n * W, at = __shfl_sync(0xffffffffu, row, r & 31);
      load_floats<E>(vs[n], a.xq + __shfl_sync(0xffffffffu, from, r & 31) + lane * E, r < nr && at >= 0);
    }
    float amax[N];
    uint32_t w[N][3][(E + 3) / 4];
    row_digits<E, N>(vs, w, amax);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = warp + n * W;
      if (r >= R) break;
      const int col = lane * E, in = col % C::SW;
#pragma unroll
      for (int d = 0; d < 3; ++d) {
        const int line = d * R + r, sw = C::SW == 128 ? line & 7 : (line >> 1) & 3;
        uint8_t *q = smem + C::Q_OFF + (col / C::SW) * C::Q_BLOCK + line * C::SW + (((in >> 4) ^ sw) << 4) + (in & 15);
        put_digits<E>(q, w[n][d]);
      }
      if (lane == 0) s_rf[r] = amax[n] / kQMax * a.asc;
    }
  }
  ptx::fence_proxy_async_smem();
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = s_tmem;
  // the next kernel may start now: this CTA holds its TMEM
  ptx::griddep_launch();

  if (warp == kLoadWarp) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      int nk = min(ST, nt), nv = nk;  // tiles issued
      for (int j = nk; j < nt; ++j) {
        if (!wait(&kempty[j % ST], ((j - ST) / ST) & 1, DEV_TIMEOUT_EMPTY)) break;
        load(&p.k[set], kfull, C::K_OFF, j);
        ++nk;
        if (!wait(&vempty[j % ST], ((j - ST) / ST) & 1, DEV_TIMEOUT_EMPTY)) break;
        load(&p.v[set], vfull, C::V_OFF, j);
        ++nv;
      }
      // every load issued must have landed before the CTA may exit
      for (int j = max(0, nk - ST); j < nk; ++j)
        ptx::mbar_wait(&kfull[j % ST], (j / ST) & 1, a.err, DEV_TIMEOUT_DRAIN);
      for (int j = max(0, nv - ST); j < nv; ++j)
        ptx::mbar_wait(&vfull[j % ST], (j / ST) & 1, a.err, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ products
    if (nt > 0) {
      constexpr uint32_t id_s = ptx::idesc_i8(128, C::NS), id_o = ptx::idesc_i8u_mn(128, C::NP);
      const ptx::Desc dq = ptx::smem_desc(ptx::smem_u32(smem + C::Q_OFF), 16, 8 * C::SW, C::SW);
      const ptx::Desc dk = ptx::smem_desc(ptx::smem_u32(smem + C::K_OFF), 16, 8 * C::SW, C::SW);
      // V^T: atoms of SW columns x 8 keys; hdim 64 repeats its one atom along M (lbo 0)
      const ptx::Desc dv = ptx::smem_desc(ptx::smem_u32(smem + C::V_OFF), 0, 8 * C::SW, C::SW);
      const ptx::Desc dp = ptx::smem_desc(ptx::smem_u32(smem + C::P_OFF), 0, 8 * C::P_ROW, C::P_ROW);
      auto scores = [&](int j) {
        if (ptx::elect_one()) {
          const uint32_t k_lo = dk.lo + (j % ST) * (C::T_BYTES >> 4);
#pragma unroll
          for (int b = 0; b < C::KB; ++b)
#pragma unroll
            for (int s = 0; s < C::SW / 32; ++s)
              ptx::mma_i8(tmem + C::S_COL + (j & 1) * C::NS,
                          ptx::Desc{k_lo + ((b * C::T_BLOCK + 32 * s) >> 4), dk.hi},
                          ptx::Desc{dq.lo + ((b * C::Q_BLOCK + 32 * s) >> 4), dq.hi}, id_s, b + s > 0 ? 1u : 0u);
          ptx::mma_commit(&kempty[j % ST]);
          ptx::mma_commit(&sfull[j & 1]);
        }
        __syncwarp();
      };
      bool ok = wait(&kfull[0], 0, DEV_TIMEOUT_FULL);
      if (__any_sync(0xffffffffu, !ok)) ok = false;
      if (ok) {
        ptx::tc_fence_after();
        scores(0);
      }
      for (int j = 0; j < nt && ok; ++j) {
        if (j + 1 < nt) {
          ok = wait(&kfull[(j + 1) % ST], ((j + 1) / ST) & 1, DEV_TIMEOUT_FULL) &&
               (j < 1 || wait(&sfree[(j + 1) & 1], ((j - 1) >> 1) & 1, DEV_TIMEOUT_TMEM));
          if (__any_sync(0xffffffffu, !ok)) break;
          ptx::tc_fence_after();
          scores(j + 1);
        }
        ok = wait(&vfull[j % ST], (j / ST) & 1, DEV_TIMEOUT_FULL) && wait(&pfull[j & 1], (j >> 1) & 1, DEV_TIMEOUT_TMEM);
        const bool fresh = __shfl_sync(0xffffffffu, *(volatile int *)&s_fresh[j & 1], 0);
        if (__any_sync(0xffffffffu, !ok)) break;
        ptx::tc_fence_after();
        if (ptx::elect_one()) {
          const uint32_t v_lo = dv.lo + (j % ST) * (C::T_BYTES >> 4), p_lo = dp.lo + (j & 1) * (C::P_BYTES >> 4);
#pragma unroll
          for (int s = 0; s < kKeys / 32; ++s)
#pragma unroll
            for (int b = 0; b < C::MB; ++b)
              ptx::mma_i8(tmem + C::O_COL + b * C::NP, ptx::Desc{v_lo + ((b * C::T_BLOCK + s * 32 * C::SW) >> 4), dv.hi},
                          ptx::Desc{p_lo + ((s * 32 * C::P_ROW) >> 4), dp.hi}, id_o, s > 0 || !fresh ? 1u : 0u);
          ptx::mma_commit(&vempty[j % ST]);
          ptx::mma_commit(&pvdone[j & 1]);
        }
        __syncwarp();
      }
      // all products complete before TMEM is freed
      if (ptx::elect_one()) ptx::mma_commit(&drain);
      __syncwarp();
      ptx::mbar_wait(&drain, 0, a.err, DEV_TIMEOUT_DRAIN);
    }
  } else {
    // ------------------------------------------------------------ softmax
    constexpr int RQ = C::RQ;
    const int quarter = warp >> 2, key = threadIdx.x & (kKeys - 1), r0 = quarter * RQ;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float *ksrc = a.kv.ks + seq * a.kv.sc_seq_stride + hk * a.kv.sc_stride;
    const float *vsrc = a.kv.vs + seq * a.kv.sc_seq_stride + hk * a.kv.sc_stride;
    auto fetch = [&](const float *src, int j) {
      const int t = j * kKeys + key;
      return t < n ? __ldg(src + kbeg + t) : 1.0f;
    };
    const float to_unit = CAP ? 1.0f / a.sc_att : kLog2e, unit = a.sc_att * kLog2e;
    // up: what takes an exponent to that of the weight, -m; while m is -inf,
    // whatever is seen at all is too large
    constexpr float kUnseen = 3.4e38f;
    float rf[RQ], l[RQ], up[RQ];
#pragma unroll
    for (int r = 0; r < RQ; ++r) {
      rf[r] = nt > 0 ? s_rf[r0 + r] * to_unit : 0.0f;
      l[r] = 0.0f;
      up[r] = kUnseen;
    }
    // the output column of this thread, a lane of O^T, and its rows of it (hdim 256:
    // two blocks of columns, half of the rows each; else a quarter)
    const int oblock = C::MB == 2 ? quarter & 1 : 0, ocol = oblock * 128 + (warp & 3) * 32 + lane;
    const int orow = C::MB == 2 ? (quarter >> 1) * C::OR : r0;
    float acc[C::OR];
#pragma unroll
    for (int r = 0; r < C::OR; ++r) acc[r] = 0.0f;
    const uint32_t olane = lanes + C::O_COL + oblock * C::NP + 4 * orow;
    // add O^T's digit sums (complete), back at the weights' size, to the column's sums
    auto flush = [&]() {
      ptx::tc_fence_after();
#pragma unroll
      for (int r = 0; r < C::OR; r += 4) {
        uint32_t d[16];
        ptx::tmem_ld_32x16(olane + 4 * r, d);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = (float)(int)d[4 * e + 3] * (16777216.0f / kOne) + (float)(int)d[4 * e + 2] * (65536.0f / kOne);
          v += (float)(int)d[4 * e + 1] * (256.0f / kOne) + (float)(int)d[4 * e] * (1.0f / kOne);
          acc[r + e] += v;
        }
      }
      ptx::tc_fence_before();
    };
    float ks = fetch(ksrc, 0), vs = fetch(vsrc, 0);
    constexpr uint32_t kGolden = 2654435769u;  // 2^32 times the golden ratio's fraction
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      const float ks_next = fetch(ksrc, j + 1), vs_next = fetch(vsrc, j + 1);
      float evs, fvs, rvs;
      split_scale(vs, evs, fvs, rvs);
      ok = wait(&sfull[j & 1], (j >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      ptx::tc_fence_after();
      // exponents: the score in log2 units plus the value scale's
      float x[RQ];
      {
        uint32_t s2[RQ], s1[RQ], s0[RQ];
        const uint32_t at = lanes + C::S_COL + (j & 1) * C::NS + r0;
        tmem_ld(at, s0);
        tmem_ld(at + R, s1);
        tmem_ld(at + 2 * R, s2);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int r = 0; r < RQ; r += 2) {
          // q . kc first: digits times a scale of 1e28 would run over
          const float2 y = __fmul2_rn(high_digit(s2 + r, low_digits(s1 + r, s0 + r)), make_float2(rf[r], rf[r + 1]));
          float2 e;
          if constexpr (CAP) {
            e = __fmul2_rn(y, make_float2(ks, ks));
            e = __ffma2_rn(make_float2(tanh_fast(e.x), tanh_fast(e.y)), make_float2(unit, unit), make_float2(evs, evs));
          } else {
            e = __ffma2_rn(y, make_float2(ks, ks), make_float2(evs, evs));
          }
          x[r] = e.x;
          x[r + 1] = e.y;
        }
      }
      ptx::tc_fence_before();
      ptx::mbar_arrive_warp(&sfree[j & 1]);
      const int t0 = kbeg + j * kKeys;
      if (t0 < all_lo || t0 + kKeys > min(all_hi, kend)) {  // a tile that some row does not see in full
        const int t = t0 + key;
#pragma unroll
        for (int r = 0; r < RQ; ++r)
          if (t < s_lo[r0 + r] || t >= min(s_hi[r0 + r], kend)) x[r] = -INFINITY;
      }
      float e[RQ];  // the weights' exponents
      auto exponents = [&]() {
#pragma unroll
        for (int r = 0; r < RQ; r += 2) {
          const float2 t = __fadd2_rn(make_float2(x[r], x[r + 1]), make_float2(up[r], up[r + 1]));
          e[r] = t.x;
          e[r + 1] = t.y;
        }
      };
      exponents();
      float most = e[0];
#pragma unroll
      for (int r = 1; r < RQ; ++r) most = fmaxf(most, e[r]);
      bool fresh = j == 0, move = ptx::named_bar_or(1, kSoftmax, !ok || most > kSlack);
      float less = 0.0f;
      if (move) {
        // What runs over from a row of zeros may: its W, the largest integer then,
        // multiplies zeros.  (fvs * rvs is kOne for a scale of 1 alone; keeping vs itself up
        // to here cost 0.9 us of 63.4.)
        if (fvs * rvs == kOne && t0 + key < kend) {
          ok = wait(&vfull[j % ST], (j / ST) & 1, DEV_TIMEOUT_FULL) && ok;
          less = row_of_zeros<C>(smem + C::V_OFF + (j % ST) * C::T_BYTES + key * C::SW, key) ? kZeros : 0.0f;
        }
        move = ptx::named_bar_or(1, kSoftmax, !ok || most - less > kSlack);
      }
      if (move) {
        // some row's weights would run over: move every row's m to its largest
        // exponent so far, and take O^T's sums at the old one
        if (!ok) s_gone = 1;
#pragma unroll
        for (int r = 0; r < RQ; ++r) {
          float top = x[r] - less;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          if (lane == 0) s_red[warp][r] = top;
        }
        ptx::named_bar_sync(1, kSoftmax);
        if (threadIdx.x < R) {
          const int hh = threadIdx.x / RQ, r = threadIdx.x % RQ;
          const float m = s_m[threadIdx.x];
          float to = m;
          for (int w = 0; w < 4; ++w) to = fmaxf(to, s_red[hh * 4 + w][r]);
          s_f[threadIdx.x] = to == m ? 1.0f : ex2(m - to);  // m = -inf: 0
          s_m[threadIdx.x] = to;
        }
        ptx::named_bar_sync(1, kSoftmax);
        if (s_gone) break;
        if (j > 0) {
          ok = wait(&pvdone[(j - 1) & 1], ((j - 1) >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
          if (!fresh) flush();
        }
#pragma unroll
        for (int r = 0; r < C::OR; ++r) acc[r] *= s_f[orow + r];
#pragma unroll
        for (int r = 0; r < RQ; ++r) {
          l[r] *= s_f[r0 + r];
          const float m = s_m[r0 + r];
          up[r] = m == -INFINITY ? kUnseen : -m;
        }
        exponents();
        fresh = true;
      }
      // this buffer's last reader is the product of tile j - 2
      if (j > 1) ok = wait(&pvdone[j & 1], ((j - 2) >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      uint32_t w[RQ];
      // a weight of 0 stays 0
      const float off = __uint_as_float((uint32_t)(kbeg + j * kKeys + key) * kGolden >> 9 | 0x3f800000u) - 1.5f;
#pragma unroll
      for (int r = 0; r < RQ; r += 2) {
        const float2 v = make_float2(ex2(e[r]), ex2(e[r + 1]));
        const float2 t = __ffma2_rn(v, make_float2(rvs, rvs), make_float2(l[r], l[r + 1]));
        l[r] = t.x;
        l[r + 1] = t.y;
        const float2 u = __ffma2_rn(v, make_float2(fvs, fvs), make_float2(off, off));
        w[r] = __float2uint_rn(u.x);
        w[r + 1] = __float2uint_rn(u.y);
      }
      uint8_t *dst = smem + C::P_OFF + (j & 1) * C::P_BYTES + key * C::P_ROW;
      const int sw = C::P_ROW == 128 ? key & 7 : (key >> 1) & 3;
#pragma unroll
      for (int r = 0; r < RQ; r += 4)
        *reinterpret_cast<uint4 *>(dst + (((r0 + r) >> 2 ^ sw) << 4)) = make_uint4(w[r], w[r + 1], w[r + 2], w[r + 3]);
      if (threadIdx.x == 0) *(volatile int *)&s_fresh[j & 1] = fresh;
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive_warp(&pfull[j & 1]);
      ks = ks_next;
      vs = vs_next;
    }
    // the rows' sums of weights, over the keys' threads
#pragma unroll
    for (int r = 0; r < RQ; ++r) {
      float v = l[r];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (lane == 0) s_red[warp][r] = v;
    }
    ptx::named_bar_sync(1, kSoftmax);
    const size_t rows_all = (size_t)a.ni * a.n_heads;
    const int slot = a.slot0 + split;
    if (threadIdx.x < nr) {
      const int r = threadIdx.x, q = r / RQ * 4, at = s_row[r];
      const float sum = (s_red[q][r % RQ] + s_red[q + 1][r % RQ]) + (s_red[q + 2][r % RQ] + s_red[q + 3][r % RQ]);
      const float m = s_m[r];
      s_sum[r] = sum;
      if (a.slots > 1 && at >= 0) a.stat[slot * rows_all + at] = make_float2(m, sum);
    }
    if (nt > 0) {
      ok = wait(&pvdone[(nt - 1) & 1], ((nt - 1) >> 1) & 1, DEV_TIMEOUT_TMEM) && ok;
      flush();
    }
    ptx::named_bar_sync(1, kSoftmax);
    if (ok && ocol < HD) {
      float *to_part = a.part + (size_t)slot * rows_all * HD + ocol;
#pragma unroll
      for (int r = 0; r < C::OR; ++r) {
        const int rr = orow + r;
        if (rr >= nr) break;
        const int at = s_row[rr];
        if (fused) {
          part[rr * HD + ocol] = acc[r];
        } else if (at < 0) {
          continue;
        } else if (a.slots == 1) {  // a row that sees nothing: zeros
          const float sum = s_sum[rr];
          a.xo[s_out[rr] + ocol] = acc[r] / (sum == 0.0f ? 1.0f : sum);
        } else if (nt > 0) {
          to_part[(size_t)at * HD] = acc[r];
        }
      }
    }
    ptx::tc_fence_before();
  }
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, C::COLS);
  if (fused) {
    // o = sum_s e_s O_s / sum_s e_s l_s, e_s = 2^(m_s - max m), in chunk order from the
    // CTAs' shared memory, each CTA a share of the elements
    auto cl = cooperative_groups::this_cluster();
    cl.sync();
    if ((int)threadIdx.x < nr) {
      const int r = threadIdx.x;
      float ms[kKtCluster], ls[kKtCluster], m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int s = 0; s < kKtCluster; ++s) {
        ms[s] = s < a.splits ? cl.map_shared_rank(s_m, s)[r] : -INFINITY;
        ls[s] = s < a.splits ? cl.map_shared_rank(s_sum, s)[r] : 0.0f;
      }
#pragma unroll
      for (int s = 0; s < kKtCluster; ++s) m = fmaxf(m, ms[s]);
#pragma unroll
      for (int s = 0; s < kKtCluster; ++s) {
        const float f = ms[s] == -INFINITY && ls[s] == 0.0f ? 0.0f : ex2(ms[s] - m);  // 0: sees none of the chunk
        s_part[s][r] = f;
        l += f * ls[s];
      }
      s_lo[r] = __float_as_int(l == 0.0f ? 1.0f : l);
    }
    __syncthreads();
    for (int e = split * kThreads + threadIdx.x; e < nr * (HD / 4); e += a.splits * kThreads) {
      const int rr = e / (HD / 4);
      float4 v[kKtCluster];
#pragma unroll
      for (int s = 0; s < kKtCluster; ++s)
        v[s] = s < a.splits && s_part[s][rr] != 0.0f ? reinterpret_cast<const float4 *>(cl.map_shared_rank(part, s))[e]
                                                    : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int s = 0; s < kKtCluster; ++s) {
        const float f = s_part[s][rr];
        o.x += f * v[s].x;
        o.y += f * v[s].y;
        o.z += f * v[s].z;
        o.w += f * v[s].w;
      }
      const float l = __int_as_float(s_lo[rr]);
      if (s_row[rr] >= 0)
        *reinterpret_cast<float4 *>(a.xo + s_out[rr] + e % (HD / 4) * 4) = make_float4(o.x / l, o.y / l, o.z / l, o.w / l);
    }
    cl.sync();  // read by all
  }
}

template <int HD, int R, bool CAP>
int launch_kt_r(const Args *sets, int n, cudaStream_t st) {
  using C = Cfg<HD, R>;
  KtArgs p;
  long blocks = 0;
  for (int s = 0; s < 2; ++s) {
    const Args &a = sets[s < n ? s : 0];
    const int G = (a.n_heads + a.kv.nkv - 1) / a.kv.nkv;
    p.a[s] = a;
    if (s == 1) p.first1 = (int)(n > 1 ? blocks : 0x7fffffff);
    if (s >= n) continue;
    blocks += (a.mode == OWN ? (long)a.ni : ((long)a.ni * G + R - 1) / R) * a.kv.nkv * a.splits;
    if (blocks > 0x7fffffffL - 1) return set_error("attention_i8: %ld CTAs", blocks);
    if (gemm_tmap_heads_i8(&p.k[s], a.kv.k, a.kv, kKeys) || gemm_tmap_heads_i8(&p.v[s], a.kv.v, a.kv, kKeys)) return 1;
  }
  {
    // the shared-memory opt-in is per device: once for each device this runs on
    static std::mutex mu;
    static unsigned long long done = 0;
    int dev = 0;
    GCU_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (!(done & (1ull << (dev & 63)))) {
      GCU_CUDA(cudaFuncSetAttribute(k_kt<HD, R, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
      done |= 1ull << (dev & 63);
    }
  }
  const unsigned cluster = sets[0].slots == 1 ? sets[0].splits : 1;
  GCU_CUDA(launch_cluster_k(k_kt<HD, R, CAP>, dim3((unsigned)blocks), dim3(kThreads), cluster, C::SMEM,
                            st, p));
  return 0;
}

template <int HD, int R>
int launch_kt_cap(const Args *sets, int n, cudaStream_t st) {
  return sets[0].sc_att != 0.0f ? launch_kt_r<HD, R, true>(sets, n, st) : launch_kt_r<HD, R, false>(sets, n, st);
}

}  // namespace

int launch_kt(const Args *sets, int n, int rows, cudaStream_t st) {
  const int hd = sets[0].kv.hdim;
  if (rows == 16)
    return hd == 256   ? launch_kt_cap<256, 16>(sets, n, st)
           : hd == 128 ? launch_kt_cap<128, 16>(sets, n, st)
                       : launch_kt_cap<64, 16>(sets, n, st);
  return hd == 256   ? launch_kt_cap<256, 32>(sets, n, st)
         : hd == 128 ? launch_kt_cap<128, 32>(sets, n, st)
                     : launch_kt_cap<64, 32>(sets, n, st);
}

}  // namespace attn8
}  // namespace gcu

// k_attention_i8.cu -- attention over the 8-bit KV cache on the CUDA cores, the
// merge of split key ranges, and the entry points.
//
// k_rows: a CTA takes up to GM query rows of one kv head and one chunk of the
// key range, and streams that chunk's codes once: K tiles (scores of all rows
// against a key row that is read once), a softmax over the chunk, V tiles.
// Bound by HBM for a few rows: 2*(hdim + 4) bytes per position and kv head.
//   K: dp4a on the codes as they lie, three per 4 codes and row (the query's
//      digits), exact; 16 lanes share a key row and reduce by halving the rows
//      each lane keeps.
//   V: codes to fp32 by a byte permute into the mantissa of 2^23 and one
//      subtraction, multiply-adds with the weights p * vs.
#include "attention_i8.cuh"

#include <algorithm>
#include <mutex>

#define GCU_EXPORT extern "C" __attribute__((visibility("default")))

namespace gcu {
namespace attn8 {
namespace {

constexpr int kThreads = 256;
constexpr int kTR = 32;          // cache rows per copy
constexpr int kStages = 8;       // copies in flight per CTA
constexpr int kMaxChunk = 1024;  // positions per CTA

template <int HD, int GM>
struct Smem {
  static constexpr int C4 = HD / 4;          // 4-code columns of a row
  static constexpr int R = kThreads / C4;    // row groups of the value phase
  static constexpr size_t ring = (size_t)kStages * kTR * HD;
  static constexpr size_t red = (size_t)R * GM * HD * sizeof(float);
  static constexpr size_t region = ring > red ? ring : red;
  // the ring (at the end: the row groups' sums), scores [GM][chunk], scales [2][chunk]
  static size_t bytes(int chunk) { return region + (size_t)(GM + 2) * chunk * sizeof(float); }
};

// four codes of a word as floats: byte ^ 0x80 into 2^23's mantissa
__device__ __forceinline__ float4 to_float4(uint32_t w) {
  w ^= 0x80808080u;
  const uint32_t m = 0x4B000000u;
  return make_float4(__int_as_float(__byte_perm(w, m, 0x7540)) - 8388736.0f,
                     __int_as_float(__byte_perm(w, m, 0x7541)) - 8388736.0f,
                     __int_as_float(__byte_perm(w, m, 0x7542)) - 8388736.0f,
                     __int_as_float(__byte_perm(w, m, 0x7543)) - 8388736.0f);
}

// sums v[0..N) over 16 lanes, halving the values a lane keeps while it has
// more than one: lane l ends with the sum of value reduced_index<N>(l)
template <int N>
__device__ __forceinline__ int reduce16(int (&v)[N], int lane) {
  int n = N;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const int send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
  return v[0];
}
template <int N>
__device__ __forceinline__ int reduced_index(int lane) {
  int g = 0;
#pragma unroll
  for (int o = 8, n = N; o > 0; o >>= 1)
    if (n > 1) {
      n >>= 1;
      if (lane & o) g += n;
    }
  return g;
}

template <int HD, int GM>
__global__ void __launch_bounds__(kThreads, GM <= 2 ? 3 : 2) k_rows(const Args a) {
  using S = Smem<HD, GM>;
  constexpr int W = HD / 64;  // words of a key row per lane
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ __align__(16) int8_t qd[3][GM][HD];
  __shared__ __align__(8) uint64_t full[kStages];
  __shared__ float s_rf[GM], s_red[kThreads / 32][GM], s_m[GM], s_l[GM];
  __shared__ int s_lo[GM], s_hi[GM];
  float *sc = reinterpret_cast<float *>(sm + S::region);
  ptx::griddep_launch();
  const int split = blockIdx.x % a.splits, group = blockIdx.x / a.splits, hk = blockIdx.y;
  const int h0 = head0(hk, a.n_heads, a.kv.nkv), G = head0(hk + 1, a.n_heads, a.kv.nkv) - h0;
  // rows of this CTA: OWN one sequence's group, else GM of the (i, g) rows
  const int first = a.mode == OWN ? group * G : group * GM;
  const int nr = a.mode == OWN ? G : min(GM, a.ni * G - first);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) ptx::mbar_init(&full[s], 1);
    ptx::fence_mbar_init();
  }
  ptx::griddep_wait();
  if (nr <= 0) return;
  if (a.mode == OWN && a.len && threadIdx.x == 0 && split == 0 && hk == 0 && __ldg(a.len + group) > a.max_len)
    ptx::record_err(a.err, DEV_BAD_LENGTH);
  if (threadIdx.x < GM) {
    int lo = 0, hi = 0;
    if ((int)threadIdx.x < nr) row_window(a, (first + threadIdx.x) / G, lo, hi);
    s_lo[threadIdx.x] = lo;
    s_hi[threadIdx.x] = hi;
  }
  __syncthreads();
  int base = 0x7fffffff, end = 0;
  for (int r = 0; r < nr; ++r)
    if (s_lo[r] < s_hi[r]) {
      base = min(base, s_lo[r]);
      end = max(end, s_hi[r]);
    }
  const long c0 = (long)base + (long)split * a.chunk;
  const int n = (int)max(0l, min((long)end, c0 + a.chunk) - c0);
  const int nt = (n + kTR - 1) / kTR, nload = 2 * nt;
  const int seq = a.mode == OWN ? group : 0;
  const long off = seq * a.kv.seq_stride + hk * a.kv.kv_stride + c0 * HD;
  const long soff = seq * a.kv.sc_seq_stride + hk * a.kv.sc_stride + c0;
  const int8_t *kh = a.kv.k + off, *vh = a.kv.v + off;
  const uint64_t pol = ptx::policy_evict_first();
  int issued = 0;  // thread 0 only
  auto issue = [&](int j) {
    const int tile = j < nt ? j : j - nt;
    const uint32_t bytes = (uint32_t)min(kTR, n - tile * kTR) * HD;
    ptx::mbar_arrive_expect_tx(&full[j % kStages], bytes);
    ptx::bulk_load(sm + (size_t)(j % kStages) * kTR * HD, (j < nt ? kh : vh) + (size_t)tile * kTR * HD, bytes,
                   &full[j % kStages], pol);
  };
  if (threadIdx.x == 0)
    for (; issued < kStages && issued < nload; ++issued) issue(issued);
  float *kss = sc + GM * a.chunk, *vss = kss + a.chunk;
  for (int t = threadIdx.x; t < n; t += kThreads) {
    kss[t] = __ldg(a.kv.ks + soff + t);
    vss[t] = __ldg(a.kv.vs + soff + t);
  }
  // the rows' digits, one warp per row
  for (int r = warp; r < GM; r += kThreads / 32) {
    constexpr int E = HD / 32;
    float v[E], amax = 0.0f;
    const float *src = a.xq + (long)((first + r) / G) * a.q_i + (long)(h0 + (first + r) % G) * a.q_h + lane * E;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      v[i] = r < nr ? __ldg(src + i) : 0.0f;
      amax = max_nan(amax, fabsf(v[i]));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const float inv = amax > 0.0f ? kQMax / amax : 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      int d2, d1, d0;
      digits(v[i], inv, d2, d1, d0);
      qd[2][r][lane * E + i] = (int8_t)d2;
      qd[1][r][lane * E + i] = (int8_t)d1;
      qd[0][r][lane * E + i] = (int8_t)d0;
    }
    if (lane == 0) s_rf[r] = amax / kQMax * a.asc;
  }
  __syncthreads();
  const int half = lane >> 4, l16 = lane & 15;
  int q[GM][3][W];
#pragma unroll
  for (int g = 0; g < GM; ++g)
#pragma unroll
    for (int d = 0; d < 3; ++d)
#pragma unroll
      for (int i = 0; i < W; ++i) q[g][d][i] = reinterpret_cast<const int *>(qd[d][g])[l16 * W + i];
  const int mine = reduced_index<GM>(l16);       // the row whose sums this lane ends with
  const bool writer = (l16 & (16 / GM - 1)) == 0;  // one lane per row
  const float rf = s_rf[mine];
  const int my_lo = s_lo[mine], my_hi = s_hi[mine];
  float wmax = -INFINITY;
  const int c = threadIdx.x % S::C4, r = threadIdx.x / S::C4;  // value phase
  float4 acc[GM];
#pragma unroll
  for (int g = 0; g < GM; ++g) acc[g] = make_float4(0.f, 0.f, 0.f, 0.f);

  int j = 0;
  for (; j < nload; ++j) {
    const bool ok = ptx::mbar_wait(&full[j % kStages], (j / kStages) & 1, a.err, DEV_TIMEOUT_FULL);
    if (__syncthreads_or(!ok)) break;  // also: every thread is done with tile j - 1
    if (threadIdx.x == 0 && j >= 1 && issued < nload) {
      ptx::fence_proxy_async_smem();
      issue(issued++);
    }
    const uint8_t *tl = sm + (size_t)(j % kStages) * kTR * HD;
    const int tile = j < nt ? j : j - nt;
    const int rows = min(kTR, n - tile * kTR);
    if (j < nt) {
#pragma unroll
      for (int rr = 0; rr < kTR / (kThreads / 16); ++rr) {
        const int row = warp * 2 + half + rr * (kThreads / 16);
        const int *kp = reinterpret_cast<const int *>(tl + row * HD) + l16 * W;
        int k[W];
        if constexpr (W == 4) {
          *reinterpret_cast<int4 *>(k) = *reinterpret_cast<const int4 *>(kp);
        } else if constexpr (W == 2) {
          *reinterpret_cast<int2 *>(k) = *reinterpret_cast<const int2 *>(kp);
        } else {
          k[0] = *kp;
        }
        int hi[GM], lo[GM];
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          int d2 = 0, d1 = 0, d0 = 0;
#pragma unroll
          for (int i = 0; i < W; ++i) {
            d2 = __dp4a(q[g][2][i], k[i], d2);
            d1 = __dp4a(q[g][1][i], k[i], d1);
            d0 = __dp4a(q[g][0][i], k[i], d0);
          }
          hi[g] = d2 * 256 + d1;  // |d| <= hdim * 127 * 128: the 16 lanes' sum stays below 2^30
          lo[g] = d0;
        }
        const int sh = reduce16<GM>(hi, l16), sl = reduce16<GM>(lo, l16);
        const int at = tile * kTR + row;
        if (writer && row < rows) {
          float s = ((float)sh * 256.0f + (float)sl) * kss[at] * rf;
          if (a.sc_att != 0.0f) s = tanhf(s / a.sc_att) * a.sc_att;
          s *= kLog2e;
          const long t = c0 + at;
          if (t < my_lo || t >= my_hi) s = -INFINITY;
          wmax = fmaxf(wmax, s);
          sc[mine * a.chunk + at] = s;
        }
      }
      if (j == nt - 1) {
        // the chunk's softmax: weights p * vs in place of the scores, their sums
        if (threadIdx.x < 8 * GM) s_red[threadIdx.x / GM][threadIdx.x % GM] = -INFINITY;
        wmax = fmaxf(wmax, __shfl_xor_sync(0xffffffffu, wmax, 16));
        __syncthreads();
        if (writer && half == 0) s_red[warp][mine] = wmax;
        __syncthreads();
        if (threadIdx.x < GM) {
          float m = -INFINITY;
          for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, s_red[w][threadIdx.x]);
          s_m[threadIdx.x] = m;
        }
        __syncthreads();
        for (int g = 0; g < nr; ++g) {
          const float m = s_m[g] == -INFINITY ? 0.0f : s_m[g];
          float l = 0.0f;
          for (int t = threadIdx.x; t < n; t += kThreads) {
            const float s = sc[g * a.chunk + t];
            const float p = ex2(s - m);
            // a position the row does not see weighs nothing, whatever its scale
            sc[g * a.chunk + t] = s == -INFINITY ? 0.0f : p * vss[t];
            l += p;
          }
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
          if (lane == 0) s_red[warp][g] = l;
        }
        __syncthreads();
        if ((int)threadIdx.x < nr) {
          float l = 0.0f;
          for (int w = 0; w < kThreads / 32; ++w) l += s_red[w][threadIdx.x];
          s_l[threadIdx.x] = l;
        }
      }
    } else {
#pragma unroll 2
      for (int row = r; row < rows; row += S::R) {
        const float4 v = to_float4(*reinterpret_cast<const uint32_t *>(tl + row * HD + c * 4));
        const int t = tile * kTR + row;
#pragma unroll
        for (int g = 0; g < GM; ++g) {
          const float p = g < nr ? sc[g * a.chunk + t] : 0.0f;
          acc[g].x += p * v.x;
          acc[g].y += p * v.y;
          acc[g].z += p * v.z;
          acc[g].w += p * v.w;
        }
      }
    }
  }
  if (j < nload) {
    // a copy never completed: the error word says so; wait (bounded) for the
    // copies still in flight into this CTA's shared memory, then leave
    if (threadIdx.x == 0)
      for (int jj = j; jj < issued; ++jj)
        ptx::mbar_wait(&full[jj % kStages], (jj / kStages) & 1, a.err, DEV_TIMEOUT_DRAIN);
    return;
  }
  if (n == 0 && (int)threadIdx.x < nr) {
    s_m[threadIdx.x] = -INFINITY;
    s_l[threadIdx.x] = 0.0f;
  }
  __syncthreads();
  float *rs = reinterpret_cast<float *>(sm);  // [R][GM][HD] (the ring is free now)
#pragma unroll
  for (int g = 0; g < GM; ++g)
    if (g < nr) *reinterpret_cast<float4 *>(rs + ((size_t)r * GM + g) * HD + c * 4) = acc[g];
  __syncthreads();
  for (int g = r; g < nr; g += S::R) {
    float4 s = *reinterpret_cast<const float4 *>(rs + (size_t)g * HD + c * 4);
    for (int rr = 1; rr < S::R; ++rr) {
      const float4 u = *reinterpret_cast<const float4 *>(rs + ((size_t)rr * GM + g) * HD + c * 4);
      s.x += u.x;
      s.y += u.y;
      s.z += u.z;
      s.w += u.w;
    }
    const int i = (first + g) / G, h = h0 + (first + g) % G;
    const float l = s_l[g];
    if (a.slots == 1) {
      if (!row_live(a, i)) continue;
      const float d = l == 0.0f ? 1.0f : l;  // a row that sees nothing: zeros
      *reinterpret_cast<float4 *>(a.xo + (long)i * a.o_i + (long)h * HD + c * 4) =
          make_float4(s.x / d, s.y / d, s.z / d, s.w / d);
    } else {
      const size_t at = ((size_t)(a.slot0 + split) * a.ni + i) * a.n_heads + h;
      *reinterpret_cast<float4 *>(a.part + at * HD + c * 4) = s;
      if (c == 0) a.stat[at] = make_float2(s_m[g], l);
    }
  }
}

// xo = sum_s e_s O_s / sum_s e_s l_s, e_s = 2^(m_s - max m), in slot order.
// One CTA per row; the slots' factors are formed by all threads at once and
// staged, and each thread keeps eight slots' loads in flight.
template <int HD>
__global__ void __launch_bounds__(HD) k_merge(const Args a) {
  __shared__ float s_e[HD], s_l[HD], s_red[HD / 32];
  ptx::griddep_launch();
  const int i = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, d = threadIdx.x;
  const size_t row = blockIdx.x, rows = (size_t)a.ni * a.n_heads;
  ptx::griddep_wait();
  if (!row_live(a, i)) return;
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

// the shared-memory opt-in is per device: once for each device a kernel runs on
template <typename K>
cudaError_t opt_in(K kern, size_t bytes, unsigned long long &done_mask) {
  static std::mutex mu;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lk(mu);
  if (done_mask & (1ull << (dev & 63))) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done_mask |= 1ull << (dev & 63);
  return e;
}

template <int HD, int GM>
cudaError_t launch_rows_gm(const Args &a, int groups, cudaStream_t st) {
  static unsigned long long done = 0;
  cudaError_t e = opt_in(k_rows<HD, GM>, Smem<HD, GM>::bytes(kMaxChunk), done);
  if (e != cudaSuccess) return e;
  return launch_k(k_rows<HD, GM>, dim3((unsigned)(a.splits * groups), a.kv.nkv), dim3(kThreads),
                  Smem<HD, GM>::bytes(a.chunk), st, a);
}

template <int HD>
cudaError_t launch_rows_hd(const Args &a, int gm, int groups, cudaStream_t st) {
  return gm == 1   ? launch_rows_gm<HD, 1>(a, groups, st)
         : gm == 2 ? launch_rows_gm<HD, 2>(a, groups, st)
         : gm == 4 ? launch_rows_gm<HD, 4>(a, groups, st)
                   : launch_rows_gm<HD, 8>(a, groups, st);
}

int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

int max_group(int n_heads, int nkv) { return (n_heads + nkv - 1) / nkv; }

// rows per CTA and row groups of a launch
void row_groups(const Args &a, int &gm, int &groups) {
  const int G = max_group(a.n_heads, a.kv.nkv);
  gm = pow2_at_least(a.mode == OWN ? G : (int)std::min((long)kMaxGroup, (long)a.ni * G));
  groups = a.mode == OWN ? a.ni : (int)(((long)a.ni * G + gm - 1) / gm);
}

}  // namespace

int launch_rows(const Args &a, cudaStream_t st) {
  int gm, groups;
  row_groups(a, gm, groups);
  if ((long)a.splits * groups > 0x7fffffffL) return set_error("attention_i8: %d x %d CTAs", a.splits, groups);
  GCU_CUDA(a.kv.hdim == 256   ? launch_rows_hd<256>(a, gm, groups, st)
           : a.kv.hdim == 128 ? launch_rows_hd<128>(a, gm, groups, st)
                              : launch_rows_hd<64>(a, gm, groups, st));
  return 0;
}

int launch_merge(const Args &a, cudaStream_t st) {
  const long rows = (long)a.ni * a.n_heads;
  if (rows > 0x7fffffffL) return set_error("attention_i8: %ld rows", rows);
  const dim3 grid((unsigned)rows);
  GCU_CUDA(a.kv.hdim == 256   ? launch_k(k_merge<256>, grid, dim3(256), 0, st, a)
           : a.kv.hdim == 128 ? launch_k(k_merge<128>, grid, dim3(128), 0, st, a)
                              : launch_k(k_merge<64>, grid, dim3(64), 0, st, a));
  return 0;
}

namespace {

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// How one launch covers its key ranges: which kernel, and chunks of the range.
struct Plan {
  bool tc;
  int chunk, splits;
};

// ni x G rows per kv head over at most n positions each.  More rows than one
// CTA of k_rows takes go to the tensor cores.
Plan plan_rows(const gcu_kv_i8 &kv, Mode mode, long ni, int G, int n) {
  Plan p{mode != OWN && ni * G > kMaxGroup, 1, 0};
  if (n < 1) n = 1;
  if (p.tc) {
    // one CTA per SM: as many chunks as make one wave of them
    const long units = (ni * G + kTcRows - 1) / kTcRows * kv.nkv, nk = kTcKeys;
    const long tiles = (n + nk - 1) / nk, want = std::min(tiles, std::max(1l, num_sms() / units));
    p.chunk = (int)((tiles + want - 1) / want * nk);
  } else {
    // enough CTAs to fill the SMs twice, 32 to kMaxChunk positions each
    const long units = mode == OWN ? ni * kv.nkv : (ni * G + kMaxGroup - 1) / kMaxGroup * kv.nkv;
    long want = std::max(1l, (2l * num_sms() + units - 1) / units);
    want = std::min(want, ((long)n + 31) / 32);
    want = std::max(want, ((long)n + kMaxChunk - 1) / kMaxChunk);
    p.chunk = (int)((n + want - 1) / want);
  }
  p.splits = (int)(((long)n + p.chunk - 1) / p.chunk);
  return p;
}

int visible(int n, int slide) { return slide > 0 ? std::min(n, slide) : n; }

struct DecodePlan {
  Plan own, pre;
  int slots() const { return own.splits + pre.splits; }
};

DecodePlan plan_decode(const gcu_kv_i8 &own, int plen, int max_len, int n_heads, int slide) {
  const int G = max_group(n_heads, own.nkv);
  DecodePlan p{plan_rows(own, OWN, own.nseq, G, visible(max_len, slide)), Plan{false, 1, 0}};
  if (plen > 0) p.pre = plan_rows(own, PREFIX, own.nseq, G, visible(plen, slide));
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
  if (!own || own->nkv < 1 || n_heads < 1) return 0;
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long qrow = (long)n_heads * own->hdim;
  Args a{xq, qrow, own->hdim, xo, qrow, *own, OWN, n_heads, own->nseq, 0, slide, 1, plen, max_len, len, asc, sc_att,
         p.own.chunk, p.own.splits, p.pre.splits, p.slots(), nullptr, nullptr, dev_error_word()};
  use_work(a, work, rows);
  if (plen > 0) {
    Args b = a;
    b.mode = PREFIX;
    b.kv = *prefix;
    b.chunk = p.pre.chunk;
    b.splits = p.pre.splits;
    b.slot0 = 0;
    if (p.pre.tc ? launch_tc(b, st) : launch_rows(b, st)) return 1;
  }
  if (launch_rows(a, st)) return 1;
  return a.slots > 1 ? launch_merge(a, st) : 0;
}

namespace {

Plan plan_prefill(const gcu_kv_i8 &kv, int n_heads, int spos, int ntok, int slide, int mask) {
  // a window's width, and the tokens of one CTA's rows past its first
  const long n = mask && slide > 0 ? std::min((long)spos + ntok, (long)slide + kTcRows) : (long)spos + ntok;
  return plan_rows(kv, PREFILL, ntok, max_group(n_heads, kv.nkv), (int)n);
}

}  // namespace

GCU_EXPORT size_t gcu_attention_prefill_i8_work(const gcu_kv_i8 *kv, int n_heads, int spos, int ntok, int slide,
                                                int mask) {
  if (!kv || kv->nkv < 1 || n_heads < 1 || ntok < 1 || spos < 0) return 0;
  return slot_bytes(plan_prefill(*kv, n_heads, spos, ntok, slide, mask).splits, (long)ntok * n_heads, kv->hdim);
}

GCU_EXPORT int gcu_dev_attention_prefill_i8(float *xo, int xostr, const float *xq, const gcu_kv_i8 *kv, int n_heads,
                                            int spos, int ntok, int slide, float sc_att, int mask, void *work,
                                            size_t work_bytes, void *stream) {
  if (ntok == 0) return 0;
  const char *what = "attention_prefill_i8";
  if (check_kv_i8(what, kv, 1) || check_heads(what, n_heads, kv->nkv)) return 1;
  if (spos < 0 || ntok < 0 || slide < 0 || spos > kv->clen - ntok)
    return set_error("%s: %d positions from %d outside a cache of %d, window %d", what, ntok, spos, kv->clen, slide);
  if (!xo || !xq) return set_error("%s: null pointer", what);
  if (xostr == 0) xostr = n_heads * kv->hdim;
  if (!aligned16(xo) || !aligned16(xq) || xostr % 4 || xostr < n_heads * kv->hdim)
    return set_error("%s: buffers must be 16-byte aligned, xostr a multiple of 4 floats, at least n_heads*hdim", what);
  const Plan p = plan_prefill(*kv, n_heads, spos, ntok, slide, mask);
  const long rows = (long)ntok * n_heads;
  if (check_work(what, slot_bytes(p.splits, rows, kv->hdim), work, work_bytes)) return 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Args a{xq, kv->hdim, (long)ntok * kv->hdim, xo, xostr, *kv, PREFILL, n_heads, ntok, spos, slide, mask ? 1 : 0, 0, 0,
         nullptr, 1.0f, sc_att, p.chunk, p.splits, 0, p.splits, nullptr, nullptr, dev_error_word()};
  use_work(a, work, rows);
  if (p.tc ? launch_tc(a, st) : launch_rows(a, st)) return 1;
  return a.slots > 1 ? launch_merge(a, st) : 0;
}

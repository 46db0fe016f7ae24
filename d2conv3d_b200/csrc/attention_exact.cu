// Cross attention on CUDA cores: fp32, fp16 and bf16 tensors, any head width up to 128, all arithmetic fp32.
//
//   s_ij = scale q_i . k_j (j below the clip's length), p = softmax_j s, o_i = sum_j p_ij v_j
//   delta_i = grad_o_i . o_i,  ds_ij = p_ij (grad_o_i . v_j - delta_i)
//   grad_q_i = scale sum_j ds_ij k_j,  grad_k_j = scale sum_i ds_ij q_i,  grad_v_j = sum_i p_ij grad_o_i
//
// One pass over the keys with the running maximum and sum of the softmax; scores live in registers and one shared tile only.
// The backward is two kernels, one with a tile of queries that runs over the keys, one with a tile of keys that runs over the
// queries of all heads that share them: each gradient has one writer, so that there are no atomics and every call gives the
// same bits, for 7 products a score instead of 5.  Bound by the FMA pipe: a thread forms 4 x 4 scores from 16-byte
// shared-memory reads.  1215 x 3240, 4 heads of 64 in fp32: 165 us forward, 225 (queries) and 333 us (keys), 24, 27 and 24 TFLOP/s.
#include "attention.h"

#include <algorithm>

namespace d2c {
namespace attn {
namespace {

constexpr int kThreads = 256;
constexpr int kPitch = kTile + 4;

// 64 rows x DP channels of `src` (row stride `stride`) as fp32; rows from `rows` on and channels from D on are zero.
template <typename T, int DP>
__device__ __forceinline__ void load_tile(float* dst, const T* src, long long stride, int rows, int D, float mul) {
  constexpr int P = DP + 4;
  if (D % 4 == 0 && stride % 4 == 0 && (reinterpret_cast<uintptr_t>(src) & (4 * sizeof(T) - 1)) == 0) {
    for (int i = threadIdx.x; i < kTile * DP / 4; i += kThreads) {
      const int r = i / (DP / 4), c = (i % (DP / 4)) * 4;
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows && c < D) {
        const Vec<T, 4> v = load_vec<T, 4>(src + r * stride + c);
        f = make_float4(to_f32(v.v[0]) * mul, to_f32(v.v[1]) * mul, to_f32(v.v[2]) * mul, to_f32(v.v[3]) * mul);
      }
      *reinterpret_cast<float4*>(dst + r * P + c) = f;
    }
  } else {
    for (int i = threadIdx.x; i < kTile * DP; i += kThreads) {
      const int r = i / DP, c = i % DP;
      dst[r * P + c] = (r < rows && c < D) ? to_f32(src[r * stride + c]) * mul : 0.f;
    }
  }
}

// s[i][j] = a row (ty * 4 + i) . b row (tx + 16 j)
template <int DP>
__device__ __forceinline__ void scores(float (&s)[4][4], const float* a, const float* b, int ty, int tx) {
  constexpr int P = DP + 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
  for (int c = 0; c < DP; c += 4) {
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty * 4 + i) * P + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * P + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = fmaf(x[i].x, y[j].x, s[i][j]);
        s[i][j] = fmaf(x[i].y, y[j].y, s[i][j]);
        s[i][j] = fmaf(x[i].z, y[j].z, s[i][j]);
        s[i][j] = fmaf(x[i].w, y[j].w, s[i][j]);
      }
  }
}

// acc[i][..] += sum_k w row (ty * 4 + i)[k] * b row k; a thread's channels: DP / 16, as vectors of up to 4, 16 vectors apart.
template <int DP>
struct Channels {
  static constexpr int kN = DP / 16, kV = kN < 4 ? kN : 4;
  static __device__ __forceinline__ int at(int e, int tx) { return (e / kV) * 16 * kV + tx * kV + e % kV; }
};
template <int DP>
__device__ __forceinline__ void weigh(float (&acc)[4][DP / 16], const float* w, const float* b, int ty, int tx) {
  constexpr int P = DP + 4, N = Channels<DP>::kN, V = Channels<DP>::kV;
#pragma unroll 2
  for (int k = 0; k < kTile; k += 4) {
    float4 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(w + (ty * 4 + i) * kPitch + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      float y[N];
#pragma unroll
      for (int m = 0; m < N / V; ++m) {
        const Vec<float, V> t = *reinterpret_cast<const Vec<float, V>*>(b + (k + kk) * P + m * 16 * V + tx * V);
#pragma unroll
        for (int e = 0; e < V; ++e) y[m * V + e] = t.v[e];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = kk == 0 ? p[i].x : (kk == 1 ? p[i].y : (kk == 2 ? p[i].z : p[i].w));
#pragma unroll
        for (int e = 0; e < N; ++e) acc[i][e] = fmaf(f, y[e], acc[i][e]);
      }
    }
  }
}

struct Where {
  int tile, head, b, split;
};
__device__ __forceinline__ Where where(int tiles, int heads, int splits) {
  Where w;
  long long i = blockIdx.x;
  w.tile = (int)(i % tiles); i /= tiles;
  w.split = (int)(i % splits); i /= splits;
  w.head = (int)(i % heads);
  w.b = (int)(i / heads);
  return w;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) fwd_kernel(Args a) {
  constexpr int P = DP + 4;
  extern __shared__ __align__(16) float sm[];
  float *sq = sm, *skv = sq + kTile * P, *sp = skv + kTile * P;
  const Where w = where((a.Lq + kTile - 1) / kTile, a.Hq, a.splits);
  const int q0 = w.tile * kTile, rows = min(kTile, a.Lq - q0), hk = w.head / (a.Hq / a.Hkv);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int len = key_length(a, w.b);
  int t0, t1;
  share((len + kTile - 1) / kTile, a.splits, w.split, t0, t1);
  const T* q = reinterpret_cast<const T*>(a.q) + w.b * a.qs[0] + (long long)q0 * a.qs[1] + w.head * a.qs[2];
  const T* k = reinterpret_cast<const T*>(a.k) + w.b * a.ks[0] + hk * a.ks[2];
  const T* v = reinterpret_cast<const T*>(a.v) + w.b * a.vs[0] + hk * a.vs[2];
  load_tile<T, DP>(sq, q, a.qs[1], rows, a.D, a.scale * kLog2e);
  float m[4], l[4], acc[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) acc[i][e] = 0.f;
  }
  for (int t = t0; t < t1; ++t) {
    const int n = min(kTile, len - t * kTile);
    __syncthreads();
    load_tile<T, DP>(skv, k + (long long)t * kTile * a.ks[1], a.ks[1], n, a.D, 1.f);
    __syncthreads();
    float s[4][4];
    scores<DP>(s, sq, skv, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (tx + 16 * j >= n) s[i][j] = -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int o = 8; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      mx = fmaxf(mx, m[i]);
      const float shift = mx == -INFINITY ? 0.f : mx, f = exp2f(m[i] - shift);
      m[i] = mx;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - shift);
        sum += s[i][j];
        sp[(ty * 4 + i) * kPitch + tx + 16 * j] = s[i][j];
      }
      l[i] = l[i] * f + sum;
#pragma unroll
      for (int e = 0; e < DP / 16; ++e) acc[i][e] *= f;
    }
    __syncthreads();
    load_tile<T, DP>(skv, v + (long long)t * kTile * a.vs[1], a.vs[1], n, a.D, 1.f);
    __syncthreads();
    weigh<DP>(acc, sp, skv, ty, tx);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float sum = l[i];
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const int r = ty * 4 + i;
    if (r >= rows) continue;
    // a share without keys, or whose keys all score -inf, weighs nothing
    const float inv = t1 == t0 || (a.splits > 1 && sum == 0.f) ? 0.f : 1.f / sum;
    const float lse = t1 > t0 ? m[i] + log2f(sum) : -INFINITY;
    const long long row = ((long long)w.b * a.Lq + q0 + r) * a.Hq + w.head;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int c = Channels<DP>::at(e, tx);
      if (c >= a.D) continue;
      if (a.splits > 1)
        a.part[((long long)w.split * a.B * a.Lq * a.Hq + row) * a.D + c] = acc[i][e] * inv;
      else
        reinterpret_cast<T*>(a.o)[row * a.D + c] = from_f32<T>(acc[i][e] * inv);
    }
    if (tx == 0) {
      if (a.splits > 1) a.part_lse[(long long)w.split * a.B * a.Lq * a.Hq + row] = lse;
      else if (a.lse) a.lse[((long long)w.b * a.Hq + w.head) * a.Lq + q0 + r] = lse;
    }
  }
}

// grad_q of 64 queries of a head, over the keys.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) bwd_q_kernel(Args a) {
  constexpr int P = DP + 4;
  extern __shared__ __align__(16) float sm[];
  float *sq = sm, *sg = sq + kTile * P, *sk = sg + kTile * P, *sv = sk + kTile * P, *sd = sv + kTile * P;
  const Where w = where((a.Lq + kTile - 1) / kTile, a.Hq, a.splits);
  const int q0 = w.tile * kTile, rows = min(kTile, a.Lq - q0), hk = w.head / (a.Hq / a.Hkv);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int len = key_length(a, w.b);
  int t0, t1;
  share((len + kTile - 1) / kTile, a.splits, w.split, t0, t1);
  const T* k = reinterpret_cast<const T*>(a.k) + w.b * a.ks[0] + hk * a.ks[2];
  const T* v = reinterpret_cast<const T*>(a.v) + w.b * a.vs[0] + hk * a.vs[2];
  load_tile<T, DP>(sq, reinterpret_cast<const T*>(a.q) + w.b * a.qs[0] + (long long)q0 * a.qs[1] + w.head * a.qs[2], a.qs[1],
                   rows, a.D, a.scale * kLog2e);
  load_tile<T, DP>(sg, reinterpret_cast<const T*>(a.g) + w.b * a.gs[0] + (long long)q0 * a.gs[1] + w.head * a.gs[2], a.gs[1],
                   rows, a.D, 1.f);
  float lse[4], delta[4], acc[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    const long long at = ((long long)w.b * a.Hq + w.head) * a.Lq + q0 + r;
    lse[i] = r < rows ? a.lse[at] : INFINITY;                    // rows that are not there: p = 0
    delta[i] = r < rows ? a.delta[at] : 0.f;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) acc[i][e] = 0.f;
  }
  for (int t = t0; t < t1; ++t) {
    const int n = min(kTile, len - t * kTile);
    __syncthreads();
    load_tile<T, DP>(sk, k + (long long)t * kTile * a.ks[1], a.ks[1], n, a.D, 1.f);
    load_tile<T, DP>(sv, v + (long long)t * kTile * a.vs[1], a.vs[1], n, a.D, 1.f);
    __syncthreads();
    float s[4][4], dp[4][4];
    scores<DP>(s, sq, sk, ty, tx);
    scores<DP>(dp, sg, sv, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = tx + 16 * j;
        sd[(ty * 4 + i) * kPitch + c] = c < n ? exp2f(s[i][j] - lse[i]) * (dp[i][j] - delta[i]) : 0.f;
      }
    __syncthreads();
    weigh<DP>(acc, sd, sk, ty, tx);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    if (r >= rows) continue;
    const long long row = ((long long)w.b * a.Lq + q0 + r) * a.Hq + w.head;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int c = Channels<DP>::at(e, tx);
      if (c >= a.D) continue;
      const float f = acc[i][e] * a.scale;
      if (a.splits > 1) a.part[((long long)w.split * a.B * a.Lq * a.Hq + row) * a.D + c] = f;
      else reinterpret_cast<T*>(a.gq)[row * a.D + c] = from_f32<T>(f);
    }
  }
}

// grad_k, grad_v of 64 keys of a head, over the queries of the heads that read it.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) bwd_kv_kernel(Args a) {
  constexpr int P = DP + 4;
  extern __shared__ __align__(16) float sm[];
  float *sk = sm, *sv = sk + kTile * P, *sq = sv + kTile * P, *sg = sq + kTile * P, *sp = sg + kTile * P,
        *sd = sp + kTile * kPitch, *srow = sd + kTile * kPitch;
  const Where w = where((a.Lk + kTile - 1) / kTile, a.Hkv, a.splits);
  const int k0 = w.tile * kTile, group = a.Hq / a.Hkv;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int len = key_length(a, w.b), n = min(kTile, len - k0);   // valid keys of the tile (may be <= 0)
  const int qtiles = (a.Lq + kTile - 1) / kTile;
  int i0, i1;
  share(qtiles * group, a.splits, w.split, i0, i1);
  if (n <= 0) i1 = i0;
  load_tile<T, DP>(sk, reinterpret_cast<const T*>(a.k) + w.b * a.ks[0] + (long long)k0 * a.ks[1] + w.head * a.ks[2], a.ks[1],
                   n, a.D, a.scale * kLog2e);
  load_tile<T, DP>(sv, reinterpret_cast<const T*>(a.v) + w.b * a.vs[0] + (long long)k0 * a.vs[1] + w.head * a.vs[2], a.vs[1],
                   n, a.D, 1.f);
  float ak[4][DP / 16], av[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) ak[i][e] = av[i][e] = 0.f;
  for (int it = i0; it < i1; ++it) {
    const int h = w.head * group + it / qtiles, q0 = (it % qtiles) * kTile, rows = min(kTile, a.Lq - q0);
    __syncthreads();
    load_tile<T, DP>(sq, reinterpret_cast<const T*>(a.q) + w.b * a.qs[0] + (long long)q0 * a.qs[1] + h * a.qs[2], a.qs[1], rows,
                     a.D, 1.f);
    load_tile<T, DP>(sg, reinterpret_cast<const T*>(a.g) + w.b * a.gs[0] + (long long)q0 * a.gs[1] + h * a.gs[2], a.gs[1], rows,
                     a.D, 1.f);
    if (threadIdx.x < kTile) {
      const long long at = ((long long)w.b * a.Hq + h) * a.Lq + q0 + threadIdx.x;
      const bool live = threadIdx.x < rows;
      srow[threadIdx.x] = live ? a.lse[at] : INFINITY;
      srow[kTile + threadIdx.x] = live ? a.delta[at] : 0.f;
    }
    __syncthreads();
    float s[4][4], dp[4][4];
    scores<DP>(s, sk, sq, ty, tx);
    scores<DP>(dp, sv, sg, ty, tx);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = tx + 16 * j, r = ty * 4 + i;
        const float p = (r < n && c < rows) ? exp2f(s[i][j] - srow[c]) : 0.f;
        sp[r * kPitch + c] = p;
        sd[r * kPitch + c] = (r < n && c < rows) ? p * (dp[i][j] - srow[kTile + c]) : 0.f;
      }
    __syncthreads();
    weigh<DP>(av, sp, sg, ty, tx);
    weigh<DP>(ak, sd, sq, ty, tx);
  }
  const int there = min(kTile, a.Lk - k0);
  const long long all = (long long)a.B * a.Lk * a.Hkv * a.D;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty * 4 + i;
    if (r >= there) continue;
    const long long row = ((long long)w.b * a.Lk + k0 + r) * a.Hkv + w.head;
#pragma unroll
    for (int e = 0; e < DP / 16; ++e) {
      const int c = Channels<DP>::at(e, tx);
      if (c >= a.D) continue;
      const float fk = ak[i][e] * a.scale, fv = av[i][e];
      if (a.splits > 1) {
        a.part[w.split * all + row * a.D + c] = fk;
        a.part[(a.splits + w.split) * all + row * a.D + c] = fv;
      } else {
        reinterpret_cast<T*>(a.gk)[row * a.D + c] = from_f32<T>(fk);
        reinterpret_cast<T*>(a.gv)[row * a.D + c] = from_f32<T>(fv);
      }
    }
  }
}

// ---- a few queries ------------------------------------------------------------------------------------------

// R query rows (heads that share keys, times queries) against a share of the keys, which are read once.  LPK lanes hold a key's
// channels, 16 bytes each; every such group of lanes runs a softmax of its own over some of the keys, four or eight at a time, so
// that 8 or 16 16-byte loads are in flight; the groups meet in shuffles and shared memory.  Bound by HBM where the GPU is filled.
// One query, 12960 keys, 8 / 2 heads of 64 in bf16: 8.5 us of launch and two waits for memory (the bytes take 1).
constexpr int kFewThreads = 256;
template <typename T, int LPK, int R>
__global__ void __launch_bounds__(kFewThreads) few_kernel(Args a) {
  constexpr int V = 16 / (int)sizeof(T), kGroups = kFewThreads / LPK, kU = sizeof(T) == 2 && R <= 4 && LPK <= 8 ? 8 : 4;
  next_kernel_may_start();
  const int group = a.Hq / a.Hkv, all_rows = group * a.Lq, row_sets = (all_rows + R - 1) / R;
  long long id = blockIdx.x;
  const int set = (int)(id % row_sets); id /= row_sets;          // blocks that read the same keys run beside one another
  const int split = (int)(id % a.splits); id /= a.splits;
  const int hk = (int)(id % a.Hkv), b = (int)(id / a.Hkv);
  const int lane = threadIdx.x % LPK, grp = threadIdx.x / LPK, c = lane * V;
  const bool has = c < a.D;
  const int len = key_length(a, b);
  int j0, j1;
  share(len, a.splits, split, j0, j1);
  float q[R][V], acc[R][V], m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = set * R + r;
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) q[r][e] = acc[r][e] = 0.f;
    if (has && row < all_rows) {
      const T* p = reinterpret_cast<const T*>(a.q) + b * a.qs[0] + (long long)(row / group) * a.qs[1] + (hk * group + row % group) * a.qs[2] + c;
      const Vec<T, V> t = load_vec<T, V>(p);
#pragma unroll
      for (int e = 0; e < V; ++e) q[r][e] = to_f32(t.v[e]) * (a.scale * kLog2e);
    }
  }
  const T* k = reinterpret_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2] + c;
  const T* v = reinterpret_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2] + c;
  for (int j = j0 + grp - (threadIdx.x & 31) / LPK; j < j1; j += kGroups * kU) {   // the same for all lanes of a warp
    const int jl = j + (threadIdx.x & 31) / LPK;
    Vec<T, V> kv[kU], vv[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int ju = jl + u * kGroups;
      const bool in = has && ju < j1;
#pragma unroll
      for (int e = 0; e < V; ++e) kv[u].v[e] = vv[u].v[e] = from_f32<T>(0.f);
      if (in) {
        kv[u] = load_vec<T, V>(k + ju * a.ks[1]);
        vv[u] = load_vec<T, V>(v + ju * a.vs[1]);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s[kU], mx = m[r];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        s[u] = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) s[u] = fmaf(q[r][e], to_f32(kv[u].v[e]), s[u]);
#pragma unroll
        for (int o = LPK / 2; o >= 1; o >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], o);
        if (jl + u * kGroups >= j1) s[u] = -INFINITY;
        mx = fmaxf(mx, s[u]);
      }
      const float shift = mx == -INFINITY ? 0.f : mx, f = exp2f(m[r] - shift);
      m[r] = mx;
      l[r] *= f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[r][e] *= f;
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const float p = exp2f(s[u] - shift);
        l[r] += p;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r][e] = fmaf(p, to_f32(vv[u].v[e]), acc[r][e]);
      }
    }
  }
  // the lane groups of a warp, then the warps
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int o = LPK; o < 32; o <<= 1) {
      const float om = __shfl_xor_sync(0xffffffffu, m[r], o), mx = fmaxf(m[r], om), shift = mx == -INFINITY ? 0.f : mx;
      const float f = exp2f(m[r] - shift), of = exp2f(om - shift);
      m[r] = mx;
      l[r] = l[r] * f + __shfl_xor_sync(0xffffffffu, l[r], o) * of;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[r][e] = acc[r][e] * f + __shfl_xor_sync(0xffffffffu, acc[r][e], o) * of;
    }
  constexpr int kWarps = kFewThreads / 32, kWidth = LPK * V;
  __shared__ float sm[R][kWarps], sl[R][kWarps], so[R][kWarps][kWidth];
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) < LPK) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (lane == 0) {
        sm[r][warp] = m[r];
        sl[r][warp] = l[r];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) so[r][warp][c + e] = acc[r][e];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R * kWidth; i += kFewThreads) {
    const int r = i / kWidth, d = i % kWidth, row = set * R + r;
    if (row >= all_rows || d >= a.D) continue;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm[r][w]);
    const float shift = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(sm[r][w] - shift);
      sum += sl[r][w] * f;
      o = fmaf(so[r][w][d], f, o);
    }
    const float inv = j1 == j0 || (a.splits > 1 && sum == 0.f) ? 0.f : 1.f / sum;
    const float lse = j1 > j0 ? mx + log2f(sum) : -INFINITY;
    const int qi = row / group, h = hk * group + row % group;
    const long long out = ((long long)b * a.Lq + qi) * a.Hq + h;
    if (a.splits > 1) a.part[((long long)split * a.B * a.Lq * a.Hq + out) * a.D + d] = o * inv;
    else reinterpret_cast<T*>(a.o)[out * a.D + d] = from_f32<T>(o * inv);
    if (d == 0) {
      if (a.splits > 1) a.part_lse[(long long)split * a.B * a.Lq * a.Hq + out] = lse;
      else if (a.lse) a.lse[((long long)b * a.Hq + h) * a.Lq + qi] = lse;
    }
  }
}

// ---- joining shares -----------------------------------------------------------------------------------------

// Place of a row of [B, Lq, Hq]; there are fewer than 2^31 of them.
struct RowAt {
  int head, query, clip;
};
__device__ __forceinline__ RowAt row_at(const Args& a, unsigned row) {
  const unsigned t = row / (unsigned)a.Hq, b = t / (unsigned)a.Lq;
  return {(int)(row - t * (unsigned)a.Hq), (int)(t - b * (unsigned)a.Lq), (int)b};
}

// o = sum_s 2^(lse_s - m) o_s / sum_s 2^(lse_s - m).  A block of 8 warps; W of them share a row's parts (1, or 8 where a few rows
// have many parts: their loads then wait for memory at the same time).  Launched beside the kernel that writes the parts, which it
// waits for: nothing here is read before that, and nothing through the read-only path.
template <typename T, int W>
__global__ void __launch_bounds__(256) combine_kernel(Args a) {
  wait_for_kernels_before();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = warp % W;
  const long long rows = (long long)a.B * a.Lq * a.Hq, row = (long long)blockIdx.x * (8 / W) + warp / W;
  if (row >= rows) return;                                       // W = 8: the whole block
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, a.part_lse[s * rows + row]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float shift = m == -INFINITY ? 0.f : m;
  float acc[4] = {}, sum = 0.f;
  constexpr int kU = W == 1 ? 4 : 8;                             // parts on their way at the same time
  for (int s0 = first; s0 < a.splits; s0 += kU * W) {
    float f[kU], v[kU][4];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const long long at = (s0 + u * W) * rows + row;
      const bool in = s0 + u * W < a.splits;
      f[u] = in ? a.part_lse[at] : -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[u][e] = in && lane + 32 * e < a.D ? a.part[at * a.D + lane + 32 * e] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      f[u] = exp2f(f[u] - shift);
      sum += f[u];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(f[u], v[u][e], acc[e]);
    }
  }
  if constexpr (W > 1) {
    __shared__ float sh[W][4][32], sums[W];
#pragma unroll
    for (int e = 0; e < 4; ++e) sh[warp][e][lane] = acc[e];
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    if (warp) return;
    for (int w = 1; w < W; ++w) {
      sum += sums[w];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += sh[w][e][lane];
    }
  }
  const RowAt r = row_at(a, (unsigned)row);
  const int h = r.head, qi = r.query, b = r.clip;
  const bool any = key_length(a, b) > 0;
  const float inv = any ? 1.f / sum : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 32 * e < a.D) reinterpret_cast<T*>(a.o)[row * a.D + lane + 32 * e] = from_f32<T>(acc[e] * inv);
  if (lane == 0 && a.lse) a.lse[((long long)b * a.Hq + h) * a.Lq + qi] = any ? m + log2f(sum) : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(256) delta_kernel(Args a) {
  const long long rows = (long long)a.B * a.Lq * a.Hq, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const RowAt r = row_at(a, (unsigned)row);
  const int h = r.head, qi = r.query, b = r.clip;
  const T* g = reinterpret_cast<const T*>(a.g) + b * a.gs[0] + (long long)qi * a.gs[1] + h * a.gs[2];
  const T* o = reinterpret_cast<const T*>(a.o_in) + row * a.D;
  float s = 0.f, most = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (lane + 32 * e < a.D) {
      const float f = to_f32(g[lane + 32 * e]);
      s = fmaf(f, to_f32(o[lane + 32 * e]), s);
      if (fabsf(f) < INFINITY) most = fmaxf(most, fabsf(f));     // as largest_sizes takes them
    }
  }
#pragma unroll
  for (int k = 16; k >= 1; k >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, k);
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, k));
  }
  if (lane == 0) {
    const long long at = ((long long)b * a.Hq + h) * a.Lq + qi;
    a.delta[at] = s;
    // a row of zeros: the largest exponent, so that no other row is measured by it
    if (a.g_exp) a.g_exp[at] = most > 0.f ? scale_exponent(__float_as_uint(most)) : 126;
  }
}

// out[y] = sum of `splits` parts of n values each, part[y]'s one behind the other; y = blockIdx.y.  Launched beside the kernel that
// writes the parts.
template <typename T>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* part, int splits, long long n, T* out0, T* out1) {
  wait_for_kernels_before();
  T* out = blockIdx.y ? out1 : out0;
  part += (long long)blockIdx.y * splits * n;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float s = 0.f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) s += part[k * n + i];
    out[i] = from_f32<T>(s);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------

template <int DP>
constexpr int smem_bytes(int tiles, int squares, int rows) {
  return (int)sizeof(float) * (tiles * kTile * (DP + 4) + squares * kTile * kPitch + rows * kTile);
}
int grid_of(long long n, unsigned* out) {
  if (n < 1 || n > 0x7fffffffLL) return D2C_ERR_TOO_LARGE;
  *out = (unsigned)n;
  return D2C_OK;
}

enum class Kind { fwd, bwd_q, bwd_kv };
template <typename T, int DP>
int launch(Kind kind, const Args& a, cudaStream_t st) {
  unsigned grid = 0;
  const long long tiles = ((kind == Kind::bwd_kv ? a.Lk : a.Lq) + kTile - 1) / kTile;
  int rc = grid_of(tiles * a.splits * (kind == Kind::bwd_kv ? a.Hkv : a.Hq) * a.B, &grid);
  if (rc) return rc;
  if (kind == Kind::fwd) {
    constexpr int smem = smem_bytes<DP>(2, 1, 0);
    if ((rc = allow_dynamic_smem<fwd_kernel<T, DP>>(smem))) return rc;
    fwd_kernel<T, DP><<<grid, kThreads, smem, st>>>(a);
  } else if (kind == Kind::bwd_q) {
    constexpr int smem = smem_bytes<DP>(4, 1, 0);
    if ((rc = allow_dynamic_smem<bwd_q_kernel<T, DP>>(smem))) return rc;
    bwd_q_kernel<T, DP><<<grid, kThreads, smem, st>>>(a);
  } else {
    constexpr int smem = smem_bytes<DP>(4, 2, 2);
    if ((rc = allow_dynamic_smem<bwd_kv_kernel<T, DP>>(smem))) return rc;
    bwd_kv_kernel<T, DP><<<grid, kThreads, smem, st>>>(a);
  }
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
template <typename T>
int by_width(Kind kind, const Args& a, cudaStream_t st) {
  if (a.D <= 32) return launch<T, 32>(kind, a, st);
  if (a.D <= 64) return launch<T, 64>(kind, a, st);
  return launch<T, 128>(kind, a, st);
}
int by_type(Kind kind, int dtype, const Args& a, cudaStream_t st) {
  switch (dtype) {
    case D2C_F32: return by_width<float>(kind, a, st);
    case D2C_F16: return by_width<__half>(kind, a, st);
    default: return by_width<__nv_bfloat16>(kind, a, st);
  }
}

template <typename T, int LPK>
int few_rows(const Args& a, cudaStream_t st) {
  const int rows = a.Hq / a.Hkv * a.Lq, R = rows >= 3 ? 4 : rows;
  unsigned grid = 0;
  if (const int rc = grid_of((long long)((rows + R - 1) / R) * a.splits * a.Hkv * a.B, &grid)) return rc;
  if (R == 1) few_kernel<T, LPK, 1><<<grid, kFewThreads, 0, st>>>(a);
  else if (R == 2) few_kernel<T, LPK, 2><<<grid, kFewThreads, 0, st>>>(a);
  else few_kernel<T, LPK, 4><<<grid, kFewThreads, 0, st>>>(a);
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
template <typename T>
int few_typed(const Args& a, cudaStream_t st) {
  const int lanes = a.D * (int)sizeof(T) / 16;
  if (lanes <= 4) return few_rows<T, 4>(a, st);
  if (lanes <= 8) return few_rows<T, 8>(a, st);
  if (lanes <= 16) return few_rows<T, 16>(a, st);
  return few_rows<T, 32>(a, st);
}

}  // namespace

int exact_fwd(int dtype, const Args& a, cudaStream_t st) { return by_type(Kind::fwd, dtype, a, st); }
int exact_bwd_q(int dtype, const Args& a, cudaStream_t st) { return by_type(Kind::bwd_q, dtype, a, st); }
int exact_bwd_kv(int dtype, const Args& a, cudaStream_t st) { return by_type(Kind::bwd_kv, dtype, a, st); }

int few_fwd(int dtype, const Args& a, cudaStream_t st) {
  switch (dtype) {
    case D2C_F32: return few_typed<float>(a, st);
    case D2C_F16: return few_typed<__half>(a, st);
    default: return few_typed<__nv_bfloat16>(a, st);
  }
}

template <typename T>
static int combine_typed(const Args& a, cudaStream_t st) {
  const long long rows = (long long)a.B * a.Lq * a.Hq;
  const bool wide = a.splits >= 16 && rows <= 148 * 16;          // 8 rows, 102 parts: 22.7 us with a warp a row
  unsigned grid = 0;
  if (const int rc = grid_of(wide ? rows : (rows + 7) / 8, &grid)) return rc;
  D2C_CUDA_TRY(launch_beside(wide ? combine_kernel<T, 8> : combine_kernel<T, 1>, dim3(grid), dim3(256), 0, st, a));
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
int combine(int dtype, const Args& a, cudaStream_t st) {
  switch (dtype) {
    case D2C_F32: return combine_typed<float>(a, st);
    case D2C_F16: return combine_typed<__half>(a, st);
    default: return combine_typed<__nv_bfloat16>(a, st);
  }
}

int delta_rows(int dtype, const Args& a, cudaStream_t st) {
  unsigned grid = 0;
  if (const int rc = grid_of(((long long)a.B * a.Lq * a.Hq + 7) / 8, &grid)) return rc;
  switch (dtype) {
    case D2C_F32: delta_kernel<float><<<grid, 256, 0, st>>>(a); break;
    case D2C_F16: delta_kernel<__half><<<grid, 256, 0, st>>>(a); break;
    default: delta_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a); break;
  }
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}

template <typename T>
static int sum_parts_typed(const float* part, int splits, long long n, void* out0, void* out1, cudaStream_t st) {
  const unsigned grid = (unsigned)std::min<long long>((n + 255) / 256, 148 * 8);
  D2C_CUDA_TRY(launch_beside(sum_parts_kernel<T>, dim3(grid, out1 ? 2 : 1), dim3(256), 0, st, part, splits, n, (T*)out0, (T*)out1));
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
int sum_parts(int dtype, const float* part, int splits, long long n, void* out0, void* out1, cudaStream_t st) {
  switch (dtype) {
    case D2C_F32: return sum_parts_typed<float>(part, splits, n, out0, out1, st);
    case D2C_F16: return sum_parts_typed<__half>(part, splits, n, out0, out1, st);
    default: return sum_parts_typed<__nv_bfloat16>(part, splits, n, out0, out1, st);
  }
}

}  // namespace attn
}  // namespace d2c

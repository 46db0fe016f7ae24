// Layer norm over the channels of a position, forward and backward:
//   mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  h = (x - mu) r,  y = w h + b
//   grad_x = r (g w - mean_c(g w) - h mean_c(g w h)),  grad_w = sum_positions g h,  grad_b = sum_positions g
// for three layouts: token rows [positions, C]; volumes [B, C, V] (channels first); and volumes whose result (and whose
// gradient) is token rows [B, V, C], which is the transposition that a projection or an attention behind it needs.
//
// Bound by HBM: x is read once and y written once (backward: x and g read, grad_x written), so every kernel keeps a
// position's channels in registers between the statistics and the result.  Variance: sums of squares around the mean, in
// registers (rows), or per thread and then merged (volumes) -- never a difference of large sums.  Parameter gradients: fp32
// per thread over the positions of a persistent block, written as one partial row per block, added up in a fixed order by
// a second kernel: no atomics, so that a call gives the same bits every time.
#include <algorithm>
#include <type_traits>

#include "token_common.cuh"

namespace d2c {
namespace {

struct NormArgs {
  int C;
  int batch;
  long long V;                 // positions per batch entry
  const void *x, *g, *w, *b;   // g: gradient of y (backward)
  void* y;                     // y, or grad_x
  float2* stats;               // [batch * V] (mean, 1 / sqrt(var + eps)); written by the forward if not NULL
  float* partial;              // [blocks][2][C]: sums for grad_w, grad_b of one block; NULL if neither is asked for
  float eps;
  int param_f32;               // w and b are fp32 (otherwise of x's type)
  int vec_tokens;              // token rows are whole vectors, of 32 bytes (fewer where a thread holds fewer)
};

template <typename T>
__device__ __forceinline__ float param(const void* p, int c, int f32, float none) {
  if (!p) return none;
  return f32 ? __ldg(reinterpret_cast<const float*>(p) + c) : to_f32(reinterpret_cast<const T*>(p)[c]);
}

// w and b as fp32 in shared memory: read once per block, whatever their type (51840 rows of 512 channels in fp16: 28 us; read from
// global memory for every row, element by element: 49).  b may be NULL.
template <typename T>
__device__ __forceinline__ void stage_params(const NormArgs& a, float* w, float* b, int padded) {
  for (int c = threadIdx.x; c < padded; c += blockDim.x) {
    w[c] = c < a.C ? param<T>(a.w, c, a.param_f32, 1.f) : 0.f;
    if (b) b[c] = c < a.C ? param<T>(a.b, c, a.param_f32, 0.f) : 0.f;
  }
  __syncthreads();
}
// VEC neighbouring channels of them.
template <int VEC>
__device__ __forceinline__ void params_at(const float* p, float (&f)[VEC]) {
  if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + e);
      f[e] = v.x; f[e + 1] = v.y; f[e + 2] = v.z; f[e + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = p[e];
  }
}

// VEC neighbouring values as pairs (one instruction for two operations), where there are pairs.
template <typename T, int VEC>
__device__ __forceinline__ F2 value_pair(const Vec<T, VEC>& v, int i) {
  if constexpr (sizeof(T) == 4) return f2(v.v[2 * i], v.v[2 * i + 1]);
  else return unpack_word<T>(reinterpret_cast<const uint32_t*>(&v)[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void set_pair(Vec<T, VEC>& v, int i, F2 f) {
  float a, b;
  f2_split(f, a, b);
  if constexpr (sizeof(T) == 4) {
    v.v[2 * i] = a;
    v.v[2 * i + 1] = b;
  } else {
    reinterpret_cast<uint32_t*>(&v)[i] = pack_word<T>(a, b);
  }
}
__device__ __forceinline__ float both_halves(F2 f) {
  float a, b;
  f2_split(f, a, b);
  return a + b;
}

// ---- token rows -------------------------------------------------------------------------------------------

// Sum of a and b over the TPR threads of a row (TPR lanes of a warp, or the whole block).
template <int TPR>
__device__ __forceinline__ void row_sum(float& a, float& b, float2* red) {
  constexpr int kLanes = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = kLanes / 2; o >= 1; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if constexpr (TPR > 32) {
    __syncthreads();                       // the last call's sums have been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(a, b);
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) { a += red[i].x; b += red[i].y; }
  }
}

// TPR threads a row, each with EPT channels as EPT / VEC vectors that lie TPR vectors apart.  The next rows are asked for before
// these are worked on.  51840 rows of 512 in fp16: 29 us (3.7 TB/s), bound by issue slots (60 %) and the reads of w and b; two rows at a
// time, which read them half as often, keep fewer warps on a SM and took 35.
template <typename T, int VEC, int EPT, int TPR>
__global__ void __launch_bounds__(256) norm_rows_fwd_kernel(NormArgs a) {
  constexpr int kChunks = EPT / VEC, kRows = 256 / TPR;
  __shared__ float2 red[8];
  extern __shared__ __align__(16) float wb[];
  const int t = threadIdx.x % TPR, C = a.C, cpad = (C + 3) & ~3;
  const long long rows = a.V * a.batch, step = (long long)gridDim.x * kRows;
  auto ask = [&](long long row, Vec<T, VEC> (&v)[kChunks]) {
    const T* x = reinterpret_cast<const T*>(a.x) + row * C;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = (k * TPR + t) * VEC;
      if (row < rows && c < C) v[k] = load_vec<T, VEC>(x + c);
    }
  };
  Vec<T, VEC> v[kChunks], next[kChunks];
  long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
  ask(row, next);
  stage_params<T>(a, wb, wb + cpad, cpad);
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < rows; r0 += step, row += step) {
    const bool live = row < rows;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) v[k] = next[k];
    ask(row + step, next);
    float s = 0.f, q = 0.f;
    F2 acc = 0ull;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = (k * TPR + t) * VEC;
      if (live && c < C) {
        if constexpr (VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) acc = add2(acc, value_pair<T, VEC>(v[k], i));
        } else {
          s += to_f32(v[k].v[0]);
        }
      }
    }
    s += both_halves(acc);
    row_sum<TPR>(s, q, red);
    const float mean = s / (float)C;
    const F2 off = f2(-mean, -mean);
    s = q = 0.f;
    acc = 0ull;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = (k * TPR + t) * VEC;
      if (live && c < C) {
        if constexpr (VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const F2 d = add2(value_pair<T, VEC>(v[k], i), off);
            acc = fma2(d, d, acc);
          }
        } else {
          const float d = to_f32(v[k].v[0]) - mean;
          q = fmaf(d, d, q);
        }
      }
    }
    q += both_halves(acc);
    row_sum<TPR>(s, q, red);
    const float rstd = 1.f / sqrtf(q / (float)C + a.eps);
    if (!live) continue;                   // no barrier follows in a block of several rows; a block of one row is all live
    if (a.stats && t == 0) a.stats[row] = make_float2(mean, rstd);
    T* y = reinterpret_cast<T*>(a.y) + row * C;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = (k * TPR + t) * VEC;
      if (c < C) {
        float w[VEC], b[VEC];
        params_at<VEC>(wb + c, w);
        params_at<VEC>(wb + cpad + c, b);
        Vec<T, VEC> o;
        if constexpr (VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i)
            set_pair<T, VEC>(o, i, fma2(mul2(add2(value_pair<T, VEC>(v[k], i), off), f2(rstd, rstd)), f2(w[2 * i], w[2 * i + 1]), f2(b[2 * i], b[2 * i + 1])));
        } else {
          o.v[0] = from_f32<T>(fmaf((to_f32(v[k].v[0]) - mean) * rstd, w[0], b[0]));
        }
        store_vec<T, VEC>(y + c, o);
      }
    }
  }
}

// (51840 rows of 512 in fp16: 43 us, 3.7 TB/s; 16 warps a SM by registers wait for loads.)
// A thread meets the same channels in every row of its block, so that the parameter gradients are sums of its own; the rows
// that a block works on at the same time are added at the end, in shared memory.
template <typename T, int VEC, int EPT, int TPR>
__global__ void __launch_bounds__(256) norm_rows_bwd_kernel(NormArgs a) {
  constexpr int kChunks = EPT / VEC, kRows = 256 / TPR;
  __shared__ float2 red[8];
  extern __shared__ __align__(16) float sums[];   // [kRows][C] at the end, w before
  const int t = threadIdx.x % TPR, C = a.C;
  const long long rows = a.V * a.batch, step = (long long)gridDim.x * kRows;
  constexpr int kPair = VEC > 1 ? 2 : 1;   // sums of one channel, or of two in one register pair
  F2 aw[EPT / kPair], ab[EPT / kPair];
#pragma unroll
  for (int i = 0; i < EPT / kPair; ++i) aw[i] = ab[i] = 0ull;
  constexpr bool kAhead = EPT <= 16;       // the next rows are asked for before these are worked on, where registers allow
  Vec<T, VEC> xv[kChunks], gv[kChunks], xn[kAhead ? kChunks : 1], gn[kAhead ? kChunks : 1];
  float2 st, stn = make_float2(0.f, 0.f);
  auto ask = [&](long long row, Vec<T, VEC>* x, Vec<T, VEC>* g, float2& s) {
    const T* px = reinterpret_cast<const T*>(a.x) + row * C;
    const T* pg = reinterpret_cast<const T*>(a.g) + row * C;
    if (row < rows) s = a.stats[row];
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = (k * TPR + t) * VEC;
      if (row < rows && c < C) {
        x[k] = load_vec<T, VEC>(px + c);
        g[k] = load_vec<T, VEC>(pg + c);
      }
    }
  };
  long long row = (long long)blockIdx.x * kRows + threadIdx.x / TPR;
  if constexpr (kAhead) ask(row, xn, gn, stn);
  stage_params<T>(a, sums, nullptr, (C + 3) & ~3);
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < rows; r0 += step, row += step) {
    const bool live = row < rows;
    if constexpr (kAhead) {
      st = stn;
#pragma unroll
      for (int k = 0; k < kChunks; ++k) { xv[k] = xn[k]; gv[k] = gn[k]; }
      ask(row + step, xn, gn, stn);
    } else {
      ask(row, xv, gv, st);
    }
    float s1, s2;
    F2 p1 = 0ull, p2 = 0ull;
    const F2 off = f2(-st.x, -st.x), mul = f2(st.y, st.y);
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = (k * TPR + t) * VEC;
      if (live && c < C) {
        float w[VEC];
        params_at<VEC>(sums + c, w);
#pragma unroll
        for (int i = 0; i < VEC / kPair; ++i) {
          const int at = k * (VEC / kPair) + i;
          F2 x, gg, ww;
          if constexpr (VEC > 1) {
            x = value_pair<T, VEC>(xv[k], i);
            gg = value_pair<T, VEC>(gv[k], i);
            ww = f2(w[2 * i], w[2 * i + 1]);
          } else {
            x = f2(to_f32(xv[k].v[0]), st.x);
            gg = f2(to_f32(gv[k].v[0]), 0.f);
            ww = f2(w[0], 0.f);
          }
          const F2 h = mul2(add2(x, off), mul), gw = mul2(gg, ww);
          p1 = add2(p1, gw);
          p2 = fma2(gw, h, p2);
          aw[at] = fma2(gg, h, aw[at]);
          ab[at] = add2(ab[at], gg);
        }
      }
    }
    s1 = both_halves(p1);
    s2 = both_halves(p2);
    row_sum<TPR>(s1, s2, red);
    if (!live || !a.y) continue;           // see the forward
    s1 /= (float)C;
    s2 /= (float)C;
    T* gx = reinterpret_cast<T*>(a.y) + row * C;
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
      const int c = (k * TPR + t) * VEC;
      if (c < C) {
        float w[VEC];
        params_at<VEC>(sums + c, w);
        Vec<T, VEC> o;
        if constexpr (VEC > 1) {
          const F2 n1 = f2(-s1, -s1), n2 = f2(-s2, -s2);
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const F2 h = mul2(add2(value_pair<T, VEC>(xv[k], i), off), mul);
            set_pair<T, VEC>(o, i, mul2(fma2(h, n2, fma2(value_pair<T, VEC>(gv[k], i), f2(w[2 * i], w[2 * i + 1]), n1)), mul));
          }
        } else {
          const float h = (to_f32(xv[k].v[0]) - st.x) * st.y;
          o.v[0] = from_f32<T>(st.y * (to_f32(gv[k].v[0]) * w[0] - s1 - h * s2));
        }
        store_vec<T, VEC>(gx + c, o);
      }
    }
  }
  if (!a.partial) return;
  auto sum_of = [&](int part, int i) {
    float u, v;
    f2_split(part ? ab[i / kPair] : aw[i / kPair], u, v);
    return kPair == 1 || i % 2 == 0 ? u : v;
  };
  float* out = a.partial + (long long)blockIdx.x * 2 * C;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    if constexpr (kRows == 1) {
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const int c = ((i / VEC) * TPR + t) * VEC + i % VEC;
        if (c < C) out[part * C + c] = sum_of(part, i);
      }
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const int c = ((i / VEC) * TPR + t) * VEC + i % VEC;
        if (c < C) sums[(threadIdx.x / TPR) * C + c] = sum_of(part, i);
      }
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += 256) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < kRows; ++r) s += sums[r * C + c];
        out[part * C + c] = s;
      }
    }
  }
}

// ---- volumes ----------------------------------------------------------------------------------------------

// Adds N values over the LV lanes that differ in the low bits of the lane; lane l ends with the sums of values
// (l % LV) * N / LV + k, k < N / LV (N < LV: value (l % LV) * N / LV).  N - 1 exchanges instead of N log2(LV): every step
// passes half of the values on.
template <int N, int LV>
__device__ __forceinline__ void spread_sum(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int n = N;
#pragma unroll
  for (int o = LV / 2; o >= 1; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool upper = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const float keep = upper ? v[i + n] : v[i], send = upper ? v[i] : v[i + n];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
}

// VV neighbouring positions of one channel: one register (16-bit positions apart would take one each).
template <typename T, int VV>
struct Cell {
  static constexpr bool kPair = VV == 2;
  using Raw = std::conditional_t<kPair, uint32_t, T>;
  Raw raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void clear() {
    if constexpr (kPair) raw = 0u;
    else raw = from_f32<T>(0.f);
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (!kPair) {
      return to_f32(raw);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return __uint_as_float(i ? raw & 0xffff0000u : raw << 16);
    } else {
      const __half2 h = *reinterpret_cast<const __half2*>(&raw);
      return i ? __high2float(h) : __low2float(h);
    }
  }
  // both positions (VV = 2)
  __device__ __forceinline__ F2 get2() const {
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return f2(__uint_as_float(raw << 16), __uint_as_float(raw & 0xffff0000u));
    } else {
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&raw));
      return f2(h.x, h.y);
    }
  }
  // v[0], v[1] rounded
  __device__ __forceinline__ void set(const float (&v)[VV]) {
    if constexpr (!kPair) {
      raw = from_f32<T>(v[0]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[VV - 1]);
      raw = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __half2 h = __floats2half2_rn(v[0], v[VV - 1]);
      raw = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};
// kW channels of a token row, moved as 32-bit words where they can be.
template <typename T, int kW>
struct RowPiece {
  static constexpr int kWords = kW * (int)sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void get(const uint8_t* p) {             // from shared memory
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const uint4 v = reinterpret_cast<const uint4*>(p)[i / 4];
      w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void put(uint8_t* p) const {
#pragma unroll
    for (int i = 0; i < kWords; i += 4) reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
  __device__ __forceinline__ void load(const T* p, int n) {          // the first n channels, element by element
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = i < n ? reinterpret_cast<const uint32_t*>(p)[i] : 0u;
      } else {
        const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
        w[i] = (2 * i < n ? q[2 * i] : 0u) | ((uint32_t)(2 * i + 1 < n ? q[2 * i + 1] : 0u) << 16);
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int n) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (sizeof(T) == 4) {
        if (i < n) reinterpret_cast<uint32_t*>(p)[i] = w[i];
      } else {
        uint16_t* q = reinterpret_cast<uint16_t*>(p);
        if (2 * i < n) q[2 * i] = (uint16_t)w[i];
        if (2 * i + 1 < n) q[2 * i + 1] = (uint16_t)(w[i] >> 16);
      }
    }
  }
};

// A tile is LV * VV neighbouring positions with all their channels: LV threads, of VV positions each, by groups of EPT
// neighbouring channels.  A warp's access to one channel is a contiguous run of positions.  Token rows pass through shared memory, where a
// warp moves whole rows; rows whose channels are not whole vectors move element by element.
// 2 x 256 x 51360 in fp32: forward 36 us (5.8 TB/s), backward 62 us (5.1 TB/s).  2 x 1024 x 12960 in bf16, to and from rows: 40 us
// (2.6 TB/s) and 66 us (2.4 TB/s): 16 warps a SM hold two tiles, whose loads, barrier and stores follow one another.
// Arithmetic goes by pairs of values (one instruction for two): the two positions of a channel (VV = 2), or two channels.
template <typename T, int EPT, int VV>
__device__ __forceinline__ F2 pair_of(const Cell<T, VV> (&v)[EPT], int i) {
  if constexpr (VV == 2) return v[i].get2();
  else return f2(v[2 * i].get(0), v[2 * i + 1].get(0));
}
template <int VV>
__device__ __forceinline__ F2 param_pair(const float (&w)[4], int i) {     // i-th pair of four channels (VV = 2: of 4 pairs, else of 2)
  if constexpr (VV == 2) return f2(w[i], w[i]);
  else return f2(w[2 * i], w[2 * i + 1]);
}
// One value a position of the thread from a pair's two halves.
template <int VV>
__device__ __forceinline__ void per_position(F2 v, float (&out)[VV]) {
  float a, b;
  f2_split(v, a, b);
  if constexpr (VV == 2) { out[0] = a; out[1] = b; }
  else out[0] = a + b;
}
template <int VV>
__device__ __forceinline__ F2 both(const float (&v)[VV]) { return f2(v[0], v[VV - 1]); }

// EPT channels of a thread's positions, `stride` apart; what is not there is zero.
template <typename T, int EPT, int VV>
__device__ __forceinline__ void load_cells(Cell<T, VV> (&v)[EPT], const T* p, long long stride, bool live, bool whole, int n) {
  if (live && whole) {
#pragma unroll
    for (int e = 0; e < EPT; ++e, p += stride) v[e].load(p);
  } else {
#pragma unroll
    for (int e = 0; e < EPT; ++e, p += stride) {
      if (live && e < n) v[e].load(p);
      else v[e].clear();
    }
  }
}

template <typename T, int EPT, int LV, int VV, bool kTokens, bool kBackward>
__global__ void __launch_bounds__(512, kBackward || VV == 2 ? 1 : 2) norm_volume_kernel(NormArgs a) {
  extern __shared__ float shared[];
  const int C = a.C, groups = blockDim.x / LV;
  float* wb = shared;                                                     // [2][C rounded up to whole groups]
  const int cpad = groups * EPT;
  float2* red = reinterpret_cast<float2*>(wb + 2 * cpad);                 // [2][groups][LV * VV]
  uint8_t* rows = reinterpret_cast<uint8_t*>(red + 2 * groups * LV * VV); // token rows of a tile, 16 bytes apart from a whole power of two
  const int pitch = C * (int)sizeof(T) + 16;
  stage_params<T>(a, wb, kBackward ? nullptr : wb + cpad, cpad);
  const int lv = threadIdx.x % LV, grp = threadIdx.x / LV, c0 = grp * EPT;
  const int n = min(max(C - c0, 0), EPT);                                 // channels that this thread has
  constexpr int kTile = LV * VV;
  constexpr int kW = (32 / (int)sizeof(T)) < EPT ? (32 / (int)sizeof(T)) : EPT;   // channels per token access
  const long long tiles_b = (a.V + kTile - 1) / kTile, tiles = tiles_b * a.batch;
  constexpr int kKeep = kBackward ? (EPT > LV ? EPT / LV : 1) : 1;
  float aw[kKeep] = {}, ab[kKeep] = {};
  // tile -> clip, place in it: divided once, then stepped
  const long long step_b = gridDim.x / tiles_b, step_t = gridDim.x % tiles_b;
  long long b = blockIdx.x / tiles_b, tb = blockIdx.x % tiles_b;
  const bool whole = n == EPT;
  // groups of a warp meet in shuffles, warps in shared memory: 32 groups read one after the other took longer than the tile's loads
  constexpr int kSteps = LV == 32 ? 0 : (LV == 16 ? 1 : 2), kOfWarp = 32 / LV * EPT;      // steps; channels of a warp
  const int warps = (C + kOfWarp - 1) / kOfWarp, warp = threadIdx.x >> 5;                 // warps that have channels
  float toward[kSteps + 1], apart[kSteps + 1];                            // of two groups' means: n_b / (n_a + n_b), n_a n_b / (n_a + n_b)
  {
    int na = n;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int nb = __shfl_xor_sync(0xffffffffu, na, LV << k);
      const float inv = na + nb ? 1.f / (float)(na + nb) : 0.f;
      toward[k] = (float)nb * inv;
      apart[k] = (float)na * (float)nb * inv;
      na += nb;
    }
  }
  int turn = 0;
  for (long long tile = blockIdx.x; tile < tiles;
       tile += gridDim.x, turn ^= 1, b += step_b, tb += step_t, b += tb >= tiles_b, tb -= tb >= tiles_b ? tiles_b : 0) {
    const long long p = tb * kTile + lv * VV;
    const bool live = p < a.V;             // VV > 1 only where it divides V
    const long long vol = (b * C + c0) * a.V + p, tok = (b * a.V + p) * C + c0;
    const T* x = reinterpret_cast<const T*>(a.x) + vol;
    if constexpr (kTokens && kBackward) {
      if (a.vec_tokens) {                                                 // asked for before x
        const T* g = reinterpret_cast<const T*>(a.g) + (b * a.V + tb * kTile) * C;
        const int there = (int)min((long long)kTile, a.V - tb * kTile);
        for (int r = threadIdx.x >> 5; r < there; r += blockDim.x >> 5)
          for (int c = threadIdx.x & 31; c < pitch / 16 - 1; c += 32)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(rows + r * pitch + c * 16)),
                         "l"(reinterpret_cast<const uint4*>(g + (long long)r * C) + c)
                         : "memory");
      }
    }
    Cell<T, VV> xv[EPT];
    load_cells<T, EPT, VV>(xv, x, a.V, live, whole, n);
    float2* slot = red + turn * groups * kTile;    // the other half is still read by threads that are behind
    if constexpr (!kBackward) {
      // mean and sum of squares around it, of each thread's channels; merged: the squares of the means' distances come in too
      const float inv = n ? 1.f / (float)n : 0.f;
      constexpr int kPairs = EPT * VV / 2;
      F2 total = 0ull;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) total = add2(total, pair_of<T, EPT, VV>(xv, i));
      float m[VV], q[VV];
      per_position<VV>(total, m);
#pragma unroll
      for (int i = 0; i < VV; ++i) m[i] *= inv;
      if (whole) {
        F2 sq = 0ull;
        const F2 off = f2(-m[0], -m[VV - 1]);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const F2 d = add2(pair_of<T, EPT, VV>(xv, i), off);
          sq = fma2(d, d, sq);
        }
        per_position<VV>(sq, q);
      } else {
#pragma unroll
        for (int i = 0; i < VV; ++i) {
          q[i] = 0.f;
#pragma unroll
          for (int e = 0; e < EPT; ++e) {
            const float d = xv[e].get(i) - m[i];
            if (e < n) q[i] = fmaf(d, d, q[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < VV; ++i) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          const float d = __shfl_xor_sync(0xffffffffu, m[i], LV << k) - m[i], oq = __shfl_xor_sync(0xffffffffu, q[i], LV << k);
          m[i] = fmaf(d, toward[k], m[i]);
          q[i] = fmaf(d * d, apart[k], q[i] + oq);
        }
        if ((threadIdx.x & 31) < LV) slot[warp * kTile + lv * VV + i] = make_float2(m[i], q[i]);
      }
      __syncthreads();
      float mean[VV], rstd[VV];
#pragma unroll
      for (int i = 0; i < VV; ++i) {
        float m = 0.f, q = 0.f;
        const float2* all = slot + lv * VV + i;
        auto count = [&](int w) { return (float)min(C - w * kOfWarp, kOfWarp); };
#pragma unroll 4
        for (int w = 0; w < warps; ++w) m = fmaf(all[w * kTile].x, count(w), m);
        m /= (float)C;
#pragma unroll 4
        for (int w = 0; w < warps; ++w) {
          const float2 s = all[w * kTile];
          const float d = s.x - m;
          q = fmaf(d * count(w), d, q) + s.y;
        }
        mean[i] = m;
        rstd[i] = 1.f / sqrtf(q / (float)C + a.eps);
        if (live && a.stats && grp == 0) a.stats[b * a.V + p + i] = make_float2(m, rstd[i]);
      }
      if (live) {
        const F2 off = f2(-mean[0], -mean[VV - 1]), mul = both<VV>(rstd);
        constexpr int kStep = 4 * VV / 2;                                 // pairs of four channels
        if constexpr (kTokens) {
#pragma unroll
          for (int e0 = 0; e0 < EPT; e0 += kW) {
            float f[VV][kW];
#pragma unroll
            for (int e1 = 0; e1 < kW; e1 += 4) {
              float w[4], bb[4];
              params_at<4>(wb + c0 + e0 + e1, w);
              params_at<4>(wb + cpad + c0 + e0 + e1, bb);
#pragma unroll
              for (int k = 0; k < kStep; ++k) {
                const F2 h = mul2(add2(pair_of<T, EPT, VV>(xv, (e0 + e1) * VV / 2 + k), off), mul);
                const F2 y2 = fma2(h, param_pair<VV>(w, k), param_pair<VV>(bb, k));
                if constexpr (VV == 2) f2_split(y2, f[0][e1 + k], f[VV - 1][e1 + k]);
                else f2_split(y2, f[0][e1 + 2 * k], f[0][e1 + 2 * k + 1]);
              }
            }
#pragma unroll
            for (int i = 0; i < VV; ++i) {
              T* y = reinterpret_cast<T*>(a.y) + tok + (long long)i * C + e0;
              RowPiece<T, kW> o;
#pragma unroll
              for (int k = 0; k < RowPiece<T, kW>::kWords; ++k) {
                constexpr int kPer = 4 / (int)sizeof(T);
                float pair[kPer];
#pragma unroll
                for (int j = 0; j < kPer; ++j) pair[j] = f[i][k * kPer + j];
                Cell<T, kPer> c;
                c.set(pair);
                o.w[k] = *reinterpret_cast<const uint32_t*>(&c.raw);
              }
              if (!a.vec_tokens) o.store(y, n - e0);
              else if (e0 < n) o.put(rows + (lv * VV + i) * pitch + (c0 + e0) * (int)sizeof(T));
            }
          }
        } else {
          T* y = reinterpret_cast<T*>(a.y) + vol;
#pragma unroll
          for (int e0 = 0; e0 < EPT; e0 += 4) {
            float w[4], bb[4], f[4][VV];
            params_at<4>(wb + c0 + e0, w);
            params_at<4>(wb + cpad + c0 + e0, bb);
#pragma unroll
            for (int k = 0; k < kStep; ++k) {
              const F2 h = mul2(add2(pair_of<T, EPT, VV>(xv, e0 * VV / 2 + k), off), mul);
              const F2 y2 = fma2(h, param_pair<VV>(w, k), param_pair<VV>(bb, k));
              if constexpr (VV == 2) f2_split(y2, f[k][0], f[k][VV - 1]);
              else f2_split(y2, f[2 * k][0], f[2 * k + 1][0]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k, y += a.V) {
              Cell<T, VV> o;
              o.set(f[k]);
              if (whole || e0 + k < n) o.store(y);
            }
          }
        }
      }
      if constexpr (kTokens) {
        if (a.vec_tokens) {
          __syncthreads();
          T* y = reinterpret_cast<T*>(a.y) + (b * a.V + tb * kTile) * C;
          const int there = (int)min((long long)kTile, a.V - tb * kTile);
          for (int r = threadIdx.x >> 5; r < there; r += blockDim.x >> 5)
            for (int c = threadIdx.x & 31; c < pitch / 16 - 1; c += 32)
              reinterpret_cast<uint4*>(y + (long long)r * C)[c] = *reinterpret_cast<const uint4*>(rows + r * pitch + c * 16);
        }
      }
    } else {
      Cell<T, VV> gv[EPT];
      if constexpr (kTokens) {
        constexpr int kPer = 4 / (int)sizeof(T);                          // channels of a word
        if (a.vec_tokens) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncthreads();
        }
#pragma unroll
        for (int e0 = 0; e0 < EPT; e0 += kW) {
          RowPiece<T, kW> o[VV];
#pragma unroll
          for (int i = 0; i < VV; ++i) {
            const T* g = reinterpret_cast<const T*>(a.g) + tok + (long long)i * C + e0;
            if (a.vec_tokens && live && e0 < n) o[i].get(rows + (lv * VV + i) * pitch + (c0 + e0) * (int)sizeof(T));
            else o[i].load(g, live ? n - e0 : 0);
          }
#pragma unroll
          for (int e = 0; e < kW; ++e) {
            if constexpr (sizeof(T) == 4) {
              gv[e0 + e].raw = __uint_as_float(o[0].w[e]);
            } else if constexpr (VV == 2) {
              gv[e0 + e].raw = __byte_perm(o[0].w[e / kPer], o[VV - 1].w[e / kPer], e % 2 ? 0x7632 : 0x5410);
            } else {
              const uint16_t h = (uint16_t)(e % 2 ? o[0].w[e / kPer] >> 16 : o[0].w[e / kPer]);
              gv[e0 + e].raw = *reinterpret_cast<const T*>(&h);
            }
          }
        }
      } else {
        const T* g = reinterpret_cast<const T*>(a.g) + vol;
        load_cells<T, EPT, VV>(gv, g, a.V, live, whole, n);
      }
      float mean[VV], rstd[VV];
#pragma unroll
      for (int i = 0; i < VV; ++i) {
        const float2 st = live ? a.stats[b * a.V + p + i] : make_float2(0.f, 0.f);
        mean[i] = st.x;
        rstd[i] = st.y;
      }
      const F2 off = f2(-mean[0], -mean[VV - 1]), mul = both<VV>(rstd);
      constexpr int kStep = 4 * VV / 2;                                   // pairs of four channels
      {
        F2 s1 = 0ull, s2 = 0ull;
#pragma unroll
        for (int e0 = 0; e0 < EPT; e0 += 4) {
          float w[4];
          params_at<4>(wb + c0 + e0, w);
#pragma unroll
          for (int k = 0; k < kStep; ++k) {                               // channels that are not there: g = w = 0
            const int i = e0 * VV / 2 + k;
            const F2 gw = mul2(pair_of<T, EPT, VV>(gv, i), param_pair<VV>(w, k));
            s1 = add2(s1, gw);
            s2 = fma2(gw, mul2(add2(pair_of<T, EPT, VV>(xv, i), off), mul), s2);
          }
        }
        float t1[VV], t2[VV];
        per_position<VV>(s1, t1);
        per_position<VV>(s2, t2);
#pragma unroll
        for (int i = 0; i < VV; ++i) {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            t1[i] += __shfl_xor_sync(0xffffffffu, t1[i], LV << k);
            t2[i] += __shfl_xor_sync(0xffffffffu, t2[i], LV << k);
          }
          if ((threadIdx.x & 31) < LV) slot[warp * kTile + lv * VV + i] = make_float2(t1[i], t2[i]);
        }
      }
      if (a.partial) {
        float v[EPT];
#pragma unroll
        for (int part = 0; part < 2; ++part) {
#pragma unroll
          for (int i = 0; i < EPT * VV / 2; ++i) {
            const F2 g2 = pair_of<T, EPT, VV>(gv, i);
            const F2 t = part ? g2 : mul2(g2, mul2(add2(pair_of<T, EPT, VV>(xv, i), off), mul));
            if constexpr (VV == 2) {
              float sum[1];
              per_position<1>(t, sum);
              v[i] = sum[0];
            } else {
              f2_split(t, v[2 * i], v[2 * i + 1]);
            }
          }
          spread_sum<EPT, LV>(v);
#pragma unroll
          for (int k = 0; k < kKeep; ++k) (part ? ab : aw)[k] += v[k];
        }
      }
      __syncthreads();
      if (a.y) {
        float m1[VV], m2[VV];
#pragma unroll
        for (int i = 0; i < VV; ++i) {
          float s1 = 0.f, s2 = 0.f;
#pragma unroll 4
          for (int w = 0; w < warps; ++w) {
            const float2 s = slot[w * kTile + lv * VV + i];
            s1 += s.x;
            s2 += s.y;
          }
          m1[i] = -s1 / (float)C;
          m2[i] = -s2 / (float)C;
        }
        const F2 n1 = both<VV>(m1), n2 = both<VV>(m2);
        T* gx = reinterpret_cast<T*>(a.y) + vol;
#pragma unroll
        for (int e0 = 0; e0 < EPT; e0 += 4) {
          float w[4], f[4][VV];
          params_at<4>(wb + c0 + e0, w);
#pragma unroll
          for (int k = 0; k < kStep; ++k) {
            const int i = e0 * VV / 2 + k;
            const F2 h = mul2(add2(pair_of<T, EPT, VV>(xv, i), off), mul);
            const F2 r = mul2(fma2(h, n2, fma2(pair_of<T, EPT, VV>(gv, i), param_pair<VV>(w, k), n1)), mul);
            if constexpr (VV == 2) f2_split(r, f[k][0], f[k][VV - 1]);
            else f2_split(r, f[2 * k][0], f[2 * k + 1][0]);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k, gx += a.V) {
            Cell<T, VV> o;
            o.set(f[k]);
            if (live && (whole || e0 + k < n)) o.store(gx);
          }
        }
      }
    }
  }
  if constexpr (kBackward) {
    if (a.partial) {
      float* out = a.partial + (long long)blockIdx.x * 2 * C;
      constexpr int kPer = EPT < LV ? LV / EPT : 1;                       // lanes that hold the same sum
      if (lv % kPer == 0) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k) {
          const int c = c0 + lv * EPT / LV + k;
          if (c < C) {
            out[c] = aw[k];
            out[C + c] = ab[k];
          }
        }
      }
    }
  }
}

// ---- any number of channels, any layout -------------------------------------------------------------------

struct Strides {
  long long batch, position, channel;
};

// One block per position, the channels read again for every pass: wider than what a block can hold.
template <typename T, bool kBackward>
__global__ void __launch_bounds__(256) norm_wide_kernel(NormArgs a, Strides sx, Strides sy) {
  __shared__ float2 red[8];
  const long long rows = a.V * a.batch;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
    const long long b = row / a.V, p = row % a.V;
    const T* x = reinterpret_cast<const T*>(a.x) + b * sx.batch + p * sx.position;
    float s1 = 0.f, s2 = 0.f;
    if constexpr (!kBackward) {
      T* y = reinterpret_cast<T*>(a.y) + b * sy.batch + p * sy.position;
      for (int c = threadIdx.x; c < a.C; c += 256) s1 += to_f32(x[c * sx.channel]);
      row_sum<256>(s1, s2, red);
      const float mean = s1 / (float)a.C;
      s1 = s2 = 0.f;
      for (int c = threadIdx.x; c < a.C; c += 256) {
        const float d = to_f32(x[c * sx.channel]) - mean;
        s2 = fmaf(d, d, s2);
      }
      row_sum<256>(s1, s2, red);
      const float rstd = 1.f / sqrtf(s2 / (float)a.C + a.eps);
      if (a.stats && threadIdx.x == 0) a.stats[row] = make_float2(mean, rstd);
      for (int c = threadIdx.x; c < a.C; c += 256)
        y[c * sy.channel] = from_f32<T>(fmaf((to_f32(x[c * sx.channel]) - mean) * rstd, param<T>(a.w, c, a.param_f32, 1.f),
                                             param<T>(a.b, c, a.param_f32, 0.f)));
    } else {
      const T* g = reinterpret_cast<const T*>(a.g) + b * sy.batch + p * sy.position;
      T* gx = reinterpret_cast<T*>(a.y) + b * sx.batch + p * sx.position;
      const float2 st = a.stats[row];
      for (int c = threadIdx.x; c < a.C; c += 256) {
        const float gw = to_f32(g[c * sy.channel]) * param<T>(a.w, c, a.param_f32, 1.f);
        s1 += gw;
        s2 = fmaf(gw, (to_f32(x[c * sx.channel]) - st.x) * st.y, s2);
      }
      row_sum<256>(s1, s2, red);
      s1 /= (float)a.C;
      s2 /= (float)a.C;
      for (int c = threadIdx.x; c < a.C; c += 256) {
        const float gw = to_f32(g[c * sy.channel]) * param<T>(a.w, c, a.param_f32, 1.f);
        gx[c * sx.channel] = from_f32<T>(st.y * (gw - s1 - (to_f32(x[c * sx.channel]) - st.x) * st.y * s2));
      }
    }
  }
}

// Sums for grad_w and grad_b of a share of the positions, a thread per channel.
template <typename T>
__global__ void __launch_bounds__(256) norm_wide_sums_kernel(NormArgs a, Strides sx, Strides sy) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  const long long rows = a.V * a.batch;
  float s1 = 0.f, s2 = 0.f;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const long long b = row / a.V, p = row % a.V;
    const float gg = to_f32(reinterpret_cast<const T*>(a.g)[b * sy.batch + p * sy.position + c * sy.channel]);
    const float2 st = a.stats[row];
    s1 = fmaf(gg, (to_f32(reinterpret_cast<const T*>(a.x)[b * sx.batch + p * sx.position + c * sx.channel]) - st.x) * st.y, s1);
    s2 += gg;
  }
  float* out = a.partial + (long long)blockIdx.y * 2 * a.C;
  out[c] = s1;
  out[a.C + c] = s2;
}

// grad_w[c], grad_b[c]: the blocks' partial sums, added in a fixed order.  32 channels by 16 shares of the blocks.
template <typename T>
__global__ void __launch_bounds__(512) norm_fold_kernel(const float* __restrict__ partial, int blocks, int C, int param_f32,
                                                        void* gw, void* gb) {
  __shared__ float sh[16][33];
  const int cx = threadIdx.x & 31, share = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx, part = blockIdx.y;
  float s = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int i = share; i < blocks; i += 16) s += partial[((long long)i * 2 + part) * C + c];
  }
  sh[share][cx] = s;
  __syncthreads();
  if (share == 0 && c < C) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += sh[i][cx];
    void* out = part ? gb : gw;
    if (!out) return;
    if (param_f32) reinterpret_cast<float*>(out)[c] = s;
    else reinterpret_cast<T*>(out)[c] = from_f32<T>(s);
  }
}

// ---- host -------------------------------------------------------------------------------------------------

enum class Path { rows, volume, wide };
struct Plan {
  Path path;
  int vec, ept, tpr;         // rows
  int lv, vv, threads;       // volume (and ept)
  int blocks;                // of the main kernel: rows of `partial`
  size_t smem;
};

// Rows: one of three thread groups per row (8 lanes, a warp, a block) with at most 32 channels a thread.
// Volumes: 32 channels a thread from 256 channels on (16 bytes of a narrower row would still be whole vectors), as many
// positions a tile as the block has threads left for; fewer where the tiles would not fill the GPU.
Plan make_plan(const d2c_layer_norm_desc& d, bool backward, bool aligned, int sms) {
  Plan p{};
  const int size = (int)token_dtype_size(d.dtype), C = d.channels;
  const long long rows = (long long)d.batch * d.positions;
  if (d.layout == D2C_NORM_ROWS) {
    p.vec = aligned && C % (16 / size) == 0 ? 16 / size : 1;
    if (C > 8192) {
      p.path = Path::wide;
    } else {
      p.path = Path::rows;
      if (C <= 64) { p.tpr = 8; p.ept = 8; }
      else if (C <= 256) { p.tpr = 32; p.ept = 8; }
      else if (C <= 1024) { p.tpr = 32; p.ept = C <= 512 ? 16 : 32; }
      else { p.tpr = 256; p.ept = C <= 2048 ? 8 : 32; }
      const int per = 256 / p.tpr;
      const long long groups = (rows + per - 1) / per, most = (long long)sms * (backward ? 2 : 4);
      p.blocks = (int)(groups < most ? groups : most);
      const int cpad = (C + 3) / 4 * 4;
      p.smem = sizeof(float) * (backward ? std::max(per > 1 ? per * C : 0, cpad) : 2 * cpad);
    }
  } else {
    // two pairs of positions a thread take 100 registers and more: blocks of 256 threads, so that a SM has several to switch
    // between (1024 channels in bf16: 46 and 66 us instead of 56 and 72 in blocks of 512)
    p.ept = C <= 64 ? 8 : 32;
    const int groups = (C + p.ept - 1) / p.ept;
    p.vv = (size == 2 && d.positions % 2 == 0 && aligned) ? 2 : 1;
    const int most_threads = p.vv == 2 && groups <= 32 ? 256 : 512;
    p.lv = 32;
    while (p.lv > 8 && (p.lv * groups > most_threads ||
                        ((d.positions + p.lv * p.vv - 1) / (p.lv * p.vv)) * d.batch < 2 * sms))
      p.lv >>= 1;
    p.threads = (p.lv * groups + 31) / 32 * 32;
    if (p.threads > most_threads) {
      p.path = Path::wide;
    } else {
      p.path = Path::volume;
      const int g = p.threads / p.lv;
      p.smem = sizeof(float) * 2 * g * p.ept + sizeof(float2) * 2 * g * p.lv * p.vv;
      if (d.layout == D2C_NORM_VOLUME_TO_ROWS) p.smem += (size_t)p.lv * p.vv * (C * size + 16);
      const long long tiles = (d.positions + p.lv * p.vv - 1) / (p.lv * p.vv) * d.batch;
      const long long most = (long long)sms * std::min(8, std::max(1, (backward ? 512 : 1024) / p.threads));
      p.blocks = (int)(tiles < most ? tiles : most);
    }
  }
  if (p.path == Path::wide) p.blocks = (int)(rows < sms * 8 ? rows : sms * 8);
  if (p.blocks < 1) p.blocks = 1;
  return p;
}
constexpr int kWideShares = 64;   // partial rows of the wide parameter gradient

int plan_checked(const d2c_layer_norm_desc* d) {
  if (!d) return D2C_ERR_NULL;
  if (!token_dtype_ok(d->dtype)) return D2C_ERR_DTYPE;
  if (d->param_dtype != D2C_F32 && d->param_dtype != d->dtype) return D2C_ERR_DTYPE;
  if (d->layout != D2C_NORM_ROWS && d->layout != D2C_NORM_VOLUME && d->layout != D2C_NORM_VOLUME_TO_ROWS) return D2C_ERR_MODE;
  if (d->batch < 1 || d->channels < 1 || d->positions < 1) return D2C_ERR_SHAPE;
  if (d->positions > 0x7fffffffffffLL / d->batch / d->channels) return D2C_ERR_TOO_LARGE;
  return D2C_OK;
}

void wide_strides(const d2c_layer_norm_desc& d, Strides* in, Strides* out) {
  const Strides rows{d.positions * d.channels, d.channels, 1}, volume{d.positions * d.channels, 1, d.positions};
  *in = d.layout == D2C_NORM_ROWS ? rows : volume;
  *out = d.layout == D2C_NORM_VOLUME ? volume : rows;
}

template <typename T, int VEC, int EPT, int TPR>
int launch_rows(const NormArgs& a, const Plan& p, bool backward, cudaStream_t st) {
  if (backward) {
    const int rc = allow_dynamic_smem<norm_rows_bwd_kernel<T, VEC, EPT, TPR>>((int)p.smem);
    if (rc) return rc;
    norm_rows_bwd_kernel<T, VEC, EPT, TPR><<<p.blocks, 256, p.smem, st>>>(a);
  } else {
    const int rc = allow_dynamic_smem<norm_rows_fwd_kernel<T, VEC, EPT, TPR>>((int)p.smem);
    if (rc) return rc;
    norm_rows_fwd_kernel<T, VEC, EPT, TPR><<<p.blocks, 256, p.smem, st>>>(a);
  }
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
template <typename T, int VEC>
int rows_path(const NormArgs& a, const Plan& p, bool backward, cudaStream_t st) {
  if (p.tpr == 8) return launch_rows<T, VEC, 8, 8>(a, p, backward, st);
  if (p.tpr == 32)
    return p.ept == 8 ? launch_rows<T, VEC, 8, 32>(a, p, backward, st)
                      : (p.ept == 16 ? launch_rows<T, VEC, 16, 32>(a, p, backward, st)
                                     : launch_rows<T, VEC, 32, 32>(a, p, backward, st));
  return p.ept == 8 ? launch_rows<T, VEC, 8, 256>(a, p, backward, st) : launch_rows<T, VEC, 32, 256>(a, p, backward, st);
}

template <typename T, int EPT, int LV, int VV, bool kTokens, bool kBackward>
int launch_volume(const NormArgs& a, const Plan& p, cudaStream_t st) {
  const int rc = allow_dynamic_smem<norm_volume_kernel<T, EPT, LV, VV, kTokens, kBackward>>((int)p.smem);
  if (rc) return rc;
  norm_volume_kernel<T, EPT, LV, VV, kTokens, kBackward><<<p.blocks, p.threads, p.smem, st>>>(a);
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
template <typename T, int EPT, int LV, int VV>
int volume_dir(const NormArgs& a, const Plan& p, bool tokens, bool backward, cudaStream_t st) {
  if (tokens)
    return backward ? launch_volume<T, EPT, LV, VV, true, true>(a, p, st) : launch_volume<T, EPT, LV, VV, true, false>(a, p, st);
  return backward ? launch_volume<T, EPT, LV, VV, false, true>(a, p, st) : launch_volume<T, EPT, LV, VV, false, false>(a, p, st);
}
template <typename T, int EPT, int LV>
int volume_vv(const NormArgs& a, const Plan& p, bool tokens, bool backward, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (p.vv == 2) return volume_dir<T, EPT, LV, 2>(a, p, tokens, backward, st);
  }
  return volume_dir<T, EPT, LV, 1>(a, p, tokens, backward, st);
}
template <typename T, int EPT>
int volume_lv(const NormArgs& a, const Plan& p, bool tokens, bool backward, cudaStream_t st) {
  if (p.lv == 32) return volume_vv<T, EPT, 32>(a, p, tokens, backward, st);
  if (p.lv == 16) return volume_vv<T, EPT, 16>(a, p, tokens, backward, st);
  return volume_vv<T, EPT, 8>(a, p, tokens, backward, st);
}

template <typename T>
int run_typed(const d2c_layer_norm_desc& d, NormArgs a, const Plan& p, bool backward, void* gw, void* gb, cudaStream_t st) {
  int partials = p.blocks;
  if (p.path == Path::rows) {
    constexpr int kVec = 16 / (int)sizeof(T);
    const int rc = p.vec == kVec ? rows_path<T, kVec>(a, p, backward, st) : rows_path<T, 1>(a, p, backward, st);
    if (rc) return rc;
  } else if (p.path == Path::volume) {
    const bool tokens = d.layout == D2C_NORM_VOLUME_TO_ROWS;
    const int w = std::min<int>(32 / (int)sizeof(T), p.ept);
    a.vec_tokens = tokens && d.channels % w == 0 && aligned_to(backward ? a.g : a.y, 16);
    const int rc = p.ept == 8 ? volume_lv<T, 8>(a, p, tokens, backward, st) : volume_lv<T, 32>(a, p, tokens, backward, st);
    if (rc) return rc;
  } else {
    Strides in, out;
    wide_strides(d, &in, &out);
    if (!backward) {
      norm_wide_kernel<T, false><<<p.blocks, 256, 0, st>>>(a, in, out);
      D2C_LAUNCH_CHECK();
    } else {
      if (a.y) {
        norm_wide_kernel<T, true><<<p.blocks, 256, 0, st>>>(a, in, out);
        D2C_LAUNCH_CHECK();
      }
      if (a.partial) {
        partials = kWideShares;
        norm_wide_sums_kernel<T><<<dim3((d.channels + 255) / 256, kWideShares), 256, 0, st>>>(a, in, out);
        D2C_LAUNCH_CHECK();
      }
    }
  }
  if (backward && a.partial) {
    norm_fold_kernel<T><<<dim3((d.channels + 31) / 32, 2), 512, 0, st>>>(a.partial, partials, d.channels, a.param_f32, gw, gb);
    D2C_LAUNCH_CHECK();
  }
  return D2C_OK;
}

int run(const d2c_layer_norm_desc& d, const NormArgs& a, bool backward, void* gw, void* gb, cudaStream_t st) {
  int sms = 0, rc = device_sm_count(&sms);
  if (rc) return rc;
  const bool al = aligned_to(a.x, 16) && (!a.y || aligned_to(a.y, 16)) && (!a.g || aligned_to(a.g, 16));
  const Plan p = make_plan(d, backward, al, sms);
  switch (d.dtype) {
    case D2C_F32: return run_typed<float>(d, a, p, backward, gw, gb, st);
    case D2C_F16: return run_typed<__half>(d, a, p, backward, gw, gb, st);
    default: return run_typed<__nv_bfloat16>(d, a, p, backward, gw, gb, st);
  }
}

}  // namespace
}  // namespace d2c

extern "C" {

int d2c_layer_norm_check(const d2c_layer_norm_desc* desc) { return d2c::plan_checked(desc); }

size_t d2c_layer_norm_bwd_workspace_bytes(const d2c_layer_norm_desc* desc) {
  using namespace d2c;
  int sms = 0;
  if (plan_checked(desc) || device_sm_count(&sms)) return 0;
  // whatever the pointers' alignment, and so the plan, turns out to be
  size_t rows = kWideShares;
  for (int al = 0; al < 2; ++al) rows = std::max<size_t>(rows, make_plan(*desc, true, al, sms).blocks);
  return align_up(sizeof(float) * 2 * rows * (size_t)desc->channels, 256);
}

int d2c_layer_norm_fwd(const d2c_layer_norm_desc* desc, const void* x, const void* w, const void* b, void* y, void* stats,
                       d2c_stream_t stream) {
  using namespace d2c;
  if (const int rc = take_device_status()) return rc;
  if (const int rc = plan_checked(desc)) return rc;
  if (!x || !y) return D2C_ERR_NULL;
  NormArgs a{desc->channels, desc->batch, desc->positions, x, nullptr, w, b, y, (float2*)stats, nullptr, desc->eps,
             desc->param_dtype == D2C_F32, 0};
  prof_mark((cudaStream_t)stream, "layer_norm");
  const int rc = run(*desc, a, false, nullptr, nullptr, (cudaStream_t)stream);
  prof_mark((cudaStream_t)stream, nullptr);
  return rc;
}

int d2c_layer_norm_bwd(const d2c_layer_norm_desc* desc, const void* grad_y, const void* x, const void* w, const void* stats,
                       void* grad_x, void* grad_w, void* grad_b, void* workspace, size_t workspace_bytes, d2c_stream_t stream) {
  using namespace d2c;
  if (const int rc = take_device_status()) return rc;
  if (const int rc = plan_checked(desc)) return rc;
  if (!grad_y || !x || !stats) return D2C_ERR_NULL;
  const bool params = grad_w || grad_b;
  if (!grad_x && !params) return D2C_OK;
  if (params && (!workspace || !aligned_to(workspace, 256) || workspace_bytes < d2c_layer_norm_bwd_workspace_bytes(desc)))
    return D2C_ERR_WORKSPACE;
  NormArgs a{desc->channels, desc->batch, desc->positions, x, grad_y, w, nullptr, grad_x, (float2*)stats,
             params ? (float*)workspace : nullptr, desc->eps, desc->param_dtype == D2C_F32, 0};
  prof_mark((cudaStream_t)stream, "layer_norm_bwd");
  const int rc = run(*desc, a, true, grad_w, grad_b, (cudaStream_t)stream);
  prof_mark((cudaStream_t)stream, nullptr);
  return rc;
}

}  // extern "C"

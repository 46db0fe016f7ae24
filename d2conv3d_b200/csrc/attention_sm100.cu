// Cross attention on tensor cores: fp16 and bf16 tensors whose head width is a multiple of 8, and fp32 tensors staged in 16 bits
// (split_rows: two fp16 parts, three products, for fp32 parity; or one bf16 part), up to 128 channels.
//
// Forward: a block has two tiles of 128 queries of a head and runs over tiles of 128 keys.  S_t = Q_t K^T lands in tensor memory;
// four warps a tile (a thread a row) form p = 2^(s scale log2 e - m) with the running maximum and sum, and write it over S as the
// 16-bit A operand of O_t += P_t V, whose accumulator stays in tensor memory too.  While one tile's warps work on their scores the
// tensor cores work for the other tile.  The maximum that p refers to is raised, and O rescaled, only when the row's maximum has
// outgrown it by 2^8: p is then at most 256, which both types hold, and most tiles skip the pass over O.  fp16 p are scaled by 2^7 besides:
// what lies 2^-32 below a row's largest is still there (many keys alike, 17 nats below one: 6 % of what they add were lost at 2^-25).
// 51360 queries, 12960 keys, 4 heads of 128 in bf16: 1.10 ms (1240 TFLOP/s) in a few calls, 1.25 ms (1090) in a long run, where the power
// cap holds; 2 clips of 3240 queries and up to 12960 keys, 4 heads of 64: 136 us.  The chain of a tile (scores, exponentials, product)
// bounds it: two tiles in flight keep the special-function pipe 61 .. 65 % and the tensor pipe 26 .. 58 % busy.
// Operands in two parts of 128 channels: one tile of queries, shared memory has no room for more.
#include <algorithm>
#include <type_traits>

#include "attention_tc.cuh"

namespace d2c {
namespace attn {
namespace {

struct TcParams {
  int B, Lq, Lk, Hq, Hkv, D;
  int width;                     // channels of the operands: D, or D rounded up to 8 where they are staged
  float c;                       // scale * log2(e), not negative
  int splits, qblocks;
  void* o;
  float *lse, *part, *part_lse;
  Args a;                        // lengths
  const uint32_t* bounds;        // two parts: see largest_sizes
  int* status;
};

constexpr int kFwdThreads = 384;                  // 8 softmax warps; MMA issuer, loader, two idle (see registers_up)
constexpr int kFwdMmaWarp = 8, kFwdLoadWarp = 9;
template <int DP, int kParts>
constexpr int kQTiles = DP * kParts > 128 ? 1 : 2;
template <int DP, int kParts>
constexpr int kFwdStages = DP * kParts == 64 ? 6 : (DP * kParts == 128 ? 4 : 2);
template <int DP, int kParts>
constexpr int kFwdSmem = kTileBytes<DP> * kParts * (kQTiles<DP, kParts> + kFwdStages<DP, kParts>) + 1024;

template <typename T, typename Out, int DP, int kParts>
__global__ void __launch_bounds__(kFwdThreads, 1)
fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
              const __grid_constant__ TcParams p) {
  constexpr float kUp = std::is_same_v<T, __half> ? 7.f : 0.f;   // p is scaled by 2^kUp
  constexpr int kStages = kFwdStages<DP, kParts>, kTB = kTileBytes<DP> * kParts, kQ = kQTiles<DP, kParts>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kStages + 9];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t base = (ptx::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t sq = base, ring = base + kQ * kTB;
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (kStages + s); };
  const uint32_t q_full = bar0 + 8 * (2 * kStages), tail = q_full + 8, done = q_full + 16;
  auto s_full = [&](int t) { return q_full + 24 + 8 * t; };
  auto p_ready = [&](int t, int h) { return q_full + 40 + 16 * t + 8 * h; };   // a half of the keys each
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  long long id = blockIdx.x;
  const int qb = (int)(id % p.qblocks); id /= p.qblocks;
  const int split = (int)(id % p.splits); id /= p.splits;
  const int head = (int)(id % p.Hq), b = (int)(id / p.Hq), hk = head / (p.Hq / p.Hkv);
  const int q0 = qb * kQ * kRows, nt = kQ == 2 && p.Lq - q0 > kRows ? 2 : 1;
  const int len = key_length(p.a, b), tiles = (len + kRows - 1) / kRows;
  int j0, j1;
  share(tiles, p.splits, split, j0, j1);
  const int n = j1 - j0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { ptx::mbar_init(full(i), 1); ptx::mbar_init(empty(i), 1); }
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(tail, 1);
    ptx::mbar_init(done, 1);
    for (int t = 0; t < 2; ++t) { ptx::mbar_init(s_full(t), 1); ptx::mbar_init(p_ready(t, 0), 4); ptx::mbar_init(p_ready(t, 1), 4); }
    abort_word = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kFwdMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const uint32_t tS = tmem, tO = tmem + 256;      // S_t at 128 t (P_t over it), O_t at DP t (two parts: the lo sums 128 columns further)

  if (warp >= 8) {
  registers_down();
  if (warp == kFwdLoadWarp) {
    int i = 0;                                    // tiles asked for: K_0 V_0 K_1 V_1 ...
    bool q_asked = false;
    if (n > 0) {
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(q_full, nt * kTB);
        for (int t = 0; t < nt; ++t) tma_tile<DP, kParts>(sq + t * kTB, &mq, head, q0 + t * kRows, b, p.B, q_full);
      }
      q_asked = true;
      for (; i < 2 * n; ++i) {
        const int s = i % kStages, j = j0 + (i >> 1);
        const bool value = i & 1;
        const int valid = len - j * kRows;
        if (!warp_wait(empty(s), ((i / kStages) & 1) ^ 1, abort_flag)) break;
        // rows behind the clip's length may hold anything, and 0 * NaN is NaN
        const bool patch = value && valid < kRows && len < p.Lk;
        const uint32_t bar = patch ? tail : full(s), dst = ring + s * kTB;
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(bar, kTB);
          tma_tile<DP, kParts>(dst, value ? &mv : &mk, hk, j * kRows, b, p.B, bar);
        }
        if (patch) {                              // the last tile: once per block
          drain(tail, 0);
          clear_rows<DP, kParts>(dst, valid);
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(full(s));
        }
      }
    }
    if (lane == 0) {
      if (q_asked) drain(q_full, 0);
      for (int w = i > kStages ? i - kStages : 0; w < i; ++w) drain(full(w % kStages), (w / kStages) & 1);
    }
  } else if (warp == kFwdMmaWarp) {
    if (n > 0 && elect_one()) {
      const uint64_t d_q = ptx::umma_desc_kmajor_sw128(sq), d_k = ptx::umma_desc_kmajor_sw128(ring),
                     d_v = ptx::umma_desc_mnmajor_sw128(ring, kHalfBytes, 1024);
      const uint32_t id_s = idesc_of<T>(kRows, false), id_o = idesc_of<T>((p.width + 15) & ~15, true);
      const int ksteps = (p.width + 15) >> 4;
      auto run = [&]() {
        if (!ptx::mbar_wait(q_full, 0, abort_flag) || !ptx::mbar_wait(full(0), 0, abort_flag)) return;
        ptx::tc_fence_after();
        for (int t = 0; t < nt; ++t) {
          mma_scores<DP, kParts>(tS + 128 * t, d_q + (t * kTB >> 4), d_k, id_s, ksteps);
          ptx::umma_commit(s_full(t));
        }
        ptx::umma_commit(empty(0));
        for (int j = 0; j < n; ++j) {
          const int iv = 2 * j + 1, ik = 2 * j + 2, sv = iv % kStages, sk = ik % kStages;
          const bool more = j + 1 < n;
          if (!ptx::mbar_wait(full(sv), (iv / kStages) & 1, abort_flag)) return;      // what is there long before p
          if (more && !ptx::mbar_wait(full(sk), (ik / kStages) & 1, abort_flag)) return;
          for (int t = 0; t < nt; ++t) {
            for (int h = 0; h < 2; ++h) {         // the first half of the keys while the second's p is formed
              if (!ptx::mbar_wait(p_ready(t, h), j & 1, abort_flag)) return;
              ptx::tc_fence_after();
              mma_weigh<DP, kParts, kParts == 2>(tO + DP * t, tS + 128 * t + 32 * h, 64, d_v + (sv * kTB >> 4) + 512 * h, id_o, j > 0 || h > 0);
            }
            if (more) {
              mma_scores<DP, kParts>(tS + 128 * t, d_q + (t * kTB >> 4), d_k + (sk * kTB >> 4), id_s, ksteps);
            }
            ptx::umma_commit(s_full(t));          // after the last tile: O_t is complete
          }
          ptx::umma_commit(empty(sv));
          if (more) ptx::umma_commit(empty(sk));
        }
      };
      run();
      ptx::umma_commit(done);
      drain(done, 0);
    }
  }
  } else {
    registers_up();
    const int t = warp >> 2, row = (warp & 3) * 32 + lane, qi = q0 + t * kRows + row;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tS + 128 * t + lanes, o_at = tO + DP * t + lanes;
    const int dcols = (p.width + 15) & ~15;
    float c = p.c, o_mul = 1.f;
    if constexpr (kParts == 2) {                  // the operands are scaled by powers of two
      const uint32_t* q = p.bounds + (long long)b * p.Hkv + hk;
      const int n_heads = p.B * p.Hkv;
      c = ldexpf(c, -scale_exponent(q[0]) - scale_exponent(q[n_heads]));
      o_mul = pow2(-scale_exponent(q[2 * n_heads]));
    }
    float m = -INFINITY, l = 0.f;                 // p = 2^(s c - m), 0 as long as all scores are -inf
    bool ok = t < nt;
    for (int j = 0; ok && j < n; ++j) {
      if (!warp_wait(s_full(t), j & 1, abort_flag)) { ok = false; break; }
      ptx::tc_fence_after();
      // scores, 32 columns at a time: the next are on their way while the maximum of these is taken
      uint32_t s[4][32];
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      const int valid = len - (j0 + j) * kRows;
      ptx::tmem_ld_32x32(s_at, s[0]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        ptx::tmem_ld_wait();
        if (k < 3) ptx::tmem_ld_32x32(s_at + 32 * (k + 1), s[k + 1]);
        if (valid < kRows) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * k + e >= valid) s[k][e] = 0xff800000u;
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            mx4[i] = fmaxf(fmaxf(mx4[i], __uint_as_float(s[k][e + 2 * i])), __uint_as_float(s[k][e + 2 * i + 1]));
      }
      float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      mx *= c;
      if (j == 0) {
        m = mx - kUp;
      } else if (__any_sync(0xffffffffu, mx > m + (kUp + 8.f))) {
        const float to = fmaxf(mx - kUp, m), f = m == -INFINITY ? 0.f : exp2_fast(m - to);
        m = to;
        l *= f;
        for (int part = 0; part < kParts; ++part)
          for (int c0 = 0; c0 < dcols; c0 += 32) {
            uint32_t o[32];
            ptx::tmem_ld_32x32(o_at + 128 * part + c0, o);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st_32x32(o_at + 128 * part + c0, o);
          }
      }
      F2 sum[2] = {0ull, 0ull};
      const float shift = m == -INFINITY ? 0.f : m;
      const F2 c2 = f2(c, c), m2 = f2(-shift, -shift);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[32], rest[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int i0 = 64 * h + 2 * e;
          float x, y;
          f2_split(fma2(f2(__uint_as_float(s[i0 >> 5][i0 & 31]), __uint_as_float(s[i0 >> 5][(i0 & 31) + 1])), c2, m2), x, y);
          x = exp2_fast(x);
          y = exp2_fast(y);
          sum[e & 1] = add2(sum[e & 1], f2(x, y));
          w[e] = pack2<T>(x, y);
          if constexpr (kParts == 2) rest[e] = pack2_rest(x, y, w[e]);
        }
        tmem_st_32x32(s_at + 32 * h, w);
        if constexpr (kParts == 2) tmem_st_32x32(s_at + 64 + 32 * h, rest);
        tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_ready(t, h));
      }
      float sa, sb;
      f2_split(add2(sum[0], sum[1]), sa, sb);
      l += sa + sb;
    }
    if (ok && n > 0) {
      ok = warp_wait(s_full(t), n & 1, abort_flag);
      ptx::tc_fence_after();
    }
    if (ok) {
      const long long rows = (long long)p.B * p.Lq * p.Hq, out = ((long long)b * p.Lq + qi) * p.Hq + head;
      const bool live = qi < p.Lq;
      // a share without keys, or whose keys all score -inf, weighs nothing
      const float inv = n == 0 || (p.splits > 1 && l == 0.f) ? 0.f : 1.f / l;
      const float lse = n > 0 ? m + log2f(l) : -INFINITY;
      for (int c0 = 0; c0 < p.D; c0 += 32) {
        uint32_t o[32];
        if (n > 0) {
          load_sums<kParts == 2>(o_at + c0, o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0u;
        }
        if (!live) continue;
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          if (c0 + e >= p.D) break;
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(o[e + i]) * inv * o_mul;
          if (p.splits > 1) store8(p.part + ((long long)split * rows + out) * p.D + c0 + e, f, p.D - c0 - e, p.D % 4 == 0);
          else store8(reinterpret_cast<Out*>(p.o) + out * p.D + c0 + e, f, p.D - c0 - e, p.D * sizeof(Out) % 16 == 0);
        }
      }
      if (live) {
        if (p.splits > 1) p.part_lse[(long long)split * rows + out] = lse;
        else if (p.lse) p.lse[((long long)b * p.Hq + head) * p.Lq + qi] = lse;
      }
    }
    ptx::tc_fence_before();
  }
  __syncthreads();
  report(p.status, abort_flag);
  if (warp == kFwdMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encoder(EncodeTiled* out) {
  static std::atomic<EncodeTiled> known{nullptr};
  EncodeTiled f = known.load(std::memory_order_acquire);
  if (!f) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    D2C_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found));
    if (!p || found != cudaDriverEntryPointSuccess) return check_cuda(cudaErrorNotSupported);
    f = reinterpret_cast<EncodeTiled>(p);
    known.store(f, std::memory_order_release);
  }
  *out = f;
  return D2C_OK;
}

template <typename T, typename Out, int DP, int kParts>
int launch_fwd(const CUtensorMap (&m)[3], TcParams p, cudaStream_t st) {
  p.qblocks = (p.Lq + kQTiles<DP, kParts> * kRows - 1) / (kQTiles<DP, kParts> * kRows);
  const long long blocks = (long long)p.qblocks * p.splits * p.Hq * p.B;
  if (blocks > 0x7fffffffLL) return D2C_ERR_TOO_LARGE;
  constexpr int smem = kFwdSmem<DP, kParts>;
  if (const int rc = allow_dynamic_smem<fwd_tc_kernel<T, Out, DP, kParts>>(smem)) return rc;
  fwd_tc_kernel<T, Out, DP, kParts><<<(unsigned)blocks, kFwdThreads, smem, st>>>(m[0], m[1], m[2], p);
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
template <typename T, typename Out, int kParts>
int fwd_by_width(const CUtensorMap (&m)[3], const TcParams& p, cudaStream_t st) {
  return p.width <= 64 ? launch_fwd<T, Out, 64, kParts>(m, p, st) : launch_fwd<T, Out, 128, kParts>(m, p, st);
}

// Up to four tensors [B, L, H, D] of one launch: q, k, v, grad_o (which: their places in `bounds`).
struct RowsArgs {
  const void* x[4];
  void* out[4];
  long long s[4][3];
  int L[4], H[4], which[4], keys[4];
  int B, D, width, parts;
  Args a;                        // lengths
  uint32_t* bounds;              // [4][B, Hkv]
};

// Largest size of an element among the valid rows of a clip and key head.  Bits of a float that is not negative order like the float, so
// that the maximum does not depend on the order of the atomics, one per block.  Elements that are not finite are left out: what they
// touch is lost anyway, the rest is not.  A warp a row, four rows at a time.
template <typename T>
__global__ void __launch_bounds__(256) bound_kernel(const __grid_constant__ RowsArgs p) {
  constexpr int kU = 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = blockIdx.z, H = p.H[i];
  __shared__ float all[8];
  for (long long head = blockIdx.y; head < (long long)p.B * H; head += gridDim.y) {
    const int h = (int)(head % H), b = (int)(head / H), hk = h / (H / p.a.Hkv);
    const int len = p.keys[i] ? key_length(p.a, b) : p.L[i], step = gridDim.x * 8;
    const T* x = reinterpret_cast<const T*>(p.x[i]) + b * p.s[i][0] + h * p.s[i][2];
    float most = 0.f;
    for (int r = blockIdx.x * 8 + warp; r < len; r += step * kU) {
      float v[kU][4];
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[u][e] = r + u * step < len && lane + 32 * e < p.D ? fabsf(to_f32(x[(long long)(r + u * step) * p.s[i][1] + lane + 32 * e])) : 0.f;
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (v[u][e] < INFINITY) most = fmaxf(most, v[u][e]);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    __syncthreads();                                             // the last head's values have been read
    if (lane == 0) all[warp] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) most = fmaxf(most, all[w]);
      if (most > 0.f) atomicMax(p.bounds + ((long long)p.which[i] * p.B + b) * p.a.Hkv + hk, __float_as_uint(most));
    }
  }
}

// x fp32 with any strides -> [parts][B, L, H, width]: fp16 hi and lo of x 2^e (e of the clip and key head, grad_o: of the row), or bf16;
// zeros from D on.  A thread writes 8 channels.
__global__ void __launch_bounds__(256) split_rows_kernel(const __grid_constant__ RowsArgs a) {
  const int t = blockIdx.y, L = a.L[t], H = a.H[t], per = a.width / 8;
  const long long n = (long long)a.B * L * H * per;
  const float* x = reinterpret_cast<const float*>(a.x[t]);
  uint4* out = reinterpret_cast<uint4*>(a.out[t]);
  const bool wide = a.D % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0 && a.s[t][0] % 4 == 0 && a.s[t][1] % 4 == 0 &&
                    a.s[t][2] % 4 == 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int c = (int)(i % per) * 8;
    long long r = i / per;
    const int h = (int)(r % H);
    r /= H;
    const int l = (int)(r % L), b = (int)(r / L);
    const float* src = x + b * a.s[t][0] + l * a.s[t][1] + h * a.s[t][2] + c;
    float f[8];
    if (wide && c + 8 <= a.D) {
      const float4 p = *reinterpret_cast<const float4*>(src), q = *reinterpret_cast<const float4*>(src + 4);
      f[0] = p.x; f[1] = p.y; f[2] = p.z; f[3] = p.w; f[4] = q.x; f[5] = q.y; f[6] = q.z; f[7] = q.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = c + e < a.D ? src[e] : 0.f;
    }
    uint32_t hi[4], lo[4];
    if (a.parts == 2) {
      const float up = pow2(a.which[t] == 3 ? a.a.g_exp[((long long)b * H + h) * L + l]
                                            : scale_exponent(a.bounds[((long long)a.which[t] * a.B + b) * a.a.Hkv + h / (H / a.a.Hkv)]));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = f[2 * e] * up, x1 = f[2 * e + 1] * up;
        hi[e] = pack2<__half>(x0, x1);
        const float2 h2 = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
        lo[e] = pack2<__half>(fabsf(h2.x) == INFINITY ? 0.f : x0 - h2.x, fabsf(h2.y) == INFINITY ? 0.f : x1 - h2.y);   // infinity has no rest
      }
      out[n + i] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) hi[e] = ptx::pack_bf16x2(f[2 * e], f[2 * e + 1]);
    }
    out[i] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  }
}

RowsArgs rows_args(const Args& a, uint32_t* bounds) {
  RowsArgs s{};
  s.B = a.B; s.D = a.D; s.width = (a.D + 7) / 8 * 8;
  s.a = a;
  s.bounds = bounds;
  return s;
}
void add_rows(RowsArgs& s, int i, const Args& a, int which) {
  const void* src[4] = {a.q, a.k, a.v, a.g};
  const long long* strides[4] = {a.qs, a.ks, a.vs, a.gs};
  const bool keys = which == 1 || which == 2;
  s.x[i] = src[which];
  s.which[i] = which;
  s.keys[i] = keys;
  s.L[i] = keys ? a.Lk : a.Lq;
  s.H[i] = keys ? a.Hkv : a.Hq;
  for (int d = 0; d < 3; ++d) s.s[i][d] = strides[which][d];
}

}  // namespace

// The device's status word.  The first call registers it, which a capture in progress on this thread must not mind.
int status_pointer(int** out) {
  static std::atomic<int*> known[64];
  int dev = -1;
  D2C_CUDA_TRY(cudaGetDevice(&dev));
  const bool kept = dev >= 0 && dev < 64;
  if (kept && (*out = known[dev].load(std::memory_order_acquire))) return D2C_OK;
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  D2C_CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
  const int rc = status_word_device_ptr(out);
  const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
  if (rc) return rc;
  if (kept) known[dev].store(*out, std::memory_order_release);
  return check_cuda(back);
}

// [clips, tokens, heads, D] 16-bit; a dimension of one element has no stride.
int tile_map(CUtensorMap* map, const Operand& o, int dtype, int D, int heads, int tokens, int clips, int rows) {
  EncodeTiled f;
  if (const int rc = encoder(&f)) return rc;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)clips};
  auto bytes = [&](long long st, int n) { return (cuuint64_t)(n == 1 ? 256 : 2 * st); };
  const cuuint64_t strides[3] = {bytes(o.s[2], heads), bytes(o.s[1], tokens), bytes(o.s[0], clips)};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult rc = f(map, dtype == D2C_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                        const_cast<void*>(o.p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? D2C_OK : check_cuda(cudaErrorInvalidValue);
}

size_t split_bytes(int B, int L, int H, int D, int parts) {
  return align_up((size_t)2 * parts * B * L * H * ((D + 7) / 8 * 8), 256);
}

// [4][B, Hkv]: the largest sizes of elements of q, k, v and, if it is there, grad_o; with `values_only` of v and grad_o alone.
int largest_sizes(int dtype, const Args& a, bool values_only, uint32_t* bounds, cudaStream_t st) {
  D2C_CUDA_TRY(cudaMemsetAsync(bounds, 0, sizeof(uint32_t) * 4 * a.B * a.Hkv, st));
  RowsArgs s = rows_args(a, bounds);
  int n = 0;
  for (int which = values_only ? 2 : 0; which < (a.g ? 4 : 3); ++which) add_rows(s, n++, a, which);
  const long long heads = (long long)a.B * a.Hq;                 // not fewer than the key heads
  const long long rows = (std::max(a.Lq, a.Lk) + 31) / 32;       // steps of a block
  const unsigned x = (unsigned)std::max<long long>(1, std::min<long long>(rows, (148 * 4 + heads * n - 1) / (heads * n)));
  const dim3 grid(x, (unsigned)std::min<long long>(heads, 65535), n);
  switch (dtype) {
    case D2C_F32: bound_kernel<float><<<grid, 256, 0, st>>>(s); break;
    case D2C_F16: bound_kernel<__half><<<grid, 256, 0, st>>>(s); break;
    default: return D2C_ERR_DTYPE;
  }
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}

// Stages fp32 q, k, v and, if it is there, grad_o; o[0..3] become the staged operands.  Two parts: largest_sizes, and delta_rows for
// grad_o, before.
int split_rows(const Args& a, int parts, uint32_t* bounds, void* workspace, Operand (&o)[4], cudaStream_t st) {
  RowsArgs s = rows_args(a, bounds);
  s.parts = parts;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  const int n = a.g ? 4 : 3;
  long long most = 0;
  for (int i = 0; i < n; ++i) {
    add_rows(s, i, a, i);
    s.out[i] = ws;
    o[i] = {ws, {(long long)s.L[i] * s.H[i] * s.width, (long long)s.H[i] * s.width, s.width}};
    ws += split_bytes(a.B, s.L[i], s.H[i], a.D, parts);
    most = std::max(most, (long long)a.B * s.L[i] * s.H[i] * (s.width / 8));
  }
  const unsigned blocks = (unsigned)std::min<long long>((most + 255) / 256, 148 * 8);
  split_rows_kernel<<<dim3(blocks, n), 256, 0, st>>>(s);
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}

int tc_fwd(int dtype, const Args& a, const Operand (&x)[4], int parts, const uint32_t* bounds, cudaStream_t st) {
  TcParams p{};
  p.B = a.B; p.Lq = a.Lq; p.Lk = a.Lk; p.Hq = a.Hq; p.Hkv = a.Hkv; p.D = a.D;
  p.width = (a.D + 7) / 8 * 8;
  CUtensorMap m[3];
  int rc;
  bool staged = false;                           // from fp32
  if (dtype == D2C_F32) dtype = parts == 2 ? D2C_F16 : D2C_BF16, staged = true;
  if ((rc = tile_map(&m[0], x[0], dtype, p.width, a.Hq, a.Lq, a.B * parts))) return rc;
  if ((rc = tile_map(&m[1], x[1], dtype, p.width, a.Hkv, a.Lk, a.B * parts))) return rc;
  if ((rc = tile_map(&m[2], x[2], dtype, p.width, a.Hkv, a.Lk, a.B * parts))) return rc;
  p.c = a.scale * kLog2e;
  p.splits = a.splits;
  p.o = a.o; p.lse = a.lse; p.part = a.part; p.part_lse = a.part_lse;
  p.a = a;
  p.bounds = bounds;
  if ((rc = status_pointer(&p.status))) return rc;
  if (staged) return parts == 2 ? fwd_by_width<__half, float, 2>(m, p, st) : fwd_by_width<__nv_bfloat16, float, 1>(m, p, st);
  return dtype == D2C_BF16 ? fwd_by_width<__nv_bfloat16, __nv_bfloat16, 1>(m, p, st) : fwd_by_width<__half, __half, 1>(m, p, st);
}

}  // namespace attn
}  // namespace d2c

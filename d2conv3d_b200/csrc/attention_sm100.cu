// Cross attention on tensor cores (fp16 and bf16 tensors, head widths that are multiples of 8 up to 128).
//
// Forward: a block has two tiles of 128 queries of a head and runs over tiles of 128 keys.  S_t = Q_t K^T lands in tensor memory;
// four warps a tile (a thread a row) form p = 2^(s scale log2 e - m) with the running maximum and sum, and write it over S as the
// 16-bit A operand of O_t += P_t V, whose accumulator stays in tensor memory too.  While one tile's warps work on their scores the
// tensor cores work for the other tile.  The maximum that p refers to is raised, and O rescaled, only when the row's maximum has
// outgrown it by 2^8: p is then at most 256, which both types hold, and most tiles skip the pass over O.
#include <algorithm>
#include <type_traits>

#include "attention_tc.cuh"

namespace d2c {
namespace attn {
namespace {

struct TcParams {
  int B, Lq, Lk, Hq, Hkv, D;
  float c;                       // scale * log2(e), not negative
  int splits, qblocks;
  void* o;
  float *lse, *part, *part_lse;
  Args a;                        // lengths
  int* status;
};

constexpr int kFwdThreads = 384;                  // 8 softmax warps; MMA issuer, loader, two idle (see registers_up)
constexpr int kFwdMmaWarp = 8, kFwdLoadWarp = 9;
template <int DP>
constexpr int kFwdStages = DP == 64 ? 6 : 4;
template <int DP>
constexpr int kFwdSmem = kTileBytes<DP> * (2 + kFwdStages<DP>) + 1024 + 256;

template <typename T, int DP>
__global__ void __launch_bounds__(kFwdThreads, 1)
fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
              const __grid_constant__ TcParams p) {
  constexpr int kStages = kFwdStages<DP>, kTB = kTileBytes<DP>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kStages + 8];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t base = (ptx::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t sq = base, ring = base + 2 * kTB;
  const uint32_t bar0 = ptx::smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (kStages + s); };
  const uint32_t q_full = bar0 + 8 * (2 * kStages), tail = q_full + 8, done = q_full + 16;
  auto s_full = [&](int t) { return q_full + 24 + 8 * t; };
  auto p_ready = [&](int t) { return q_full + 40 + 8 * t; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  long long id = blockIdx.x;
  const int qb = (int)(id % p.qblocks); id /= p.qblocks;
  const int split = (int)(id % p.splits); id /= p.splits;
  const int head = (int)(id % p.Hq), b = (int)(id / p.Hq), hk = head / (p.Hq / p.Hkv);
  const int q0 = qb * 2 * kRows, nt = p.Lq - q0 > kRows ? 2 : 1;
  const int len = key_length(p.a, b), tiles = (len + kRows - 1) / kRows;
  int j0, j1;
  share(tiles, p.splits, split, j0, j1);
  const int n = j1 - j0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) { ptx::mbar_init(full(i), 1); ptx::mbar_init(empty(i), 1); }
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(tail, 1);
    ptx::mbar_init(done, 1);
    for (int t = 0; t < 2; ++t) { ptx::mbar_init(s_full(t), 1); ptx::mbar_init(p_ready(t), 4); }
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
  const uint32_t tS = tmem, tO = tmem + 256;      // S_t at 128 t (P_t over it), O_t at DP t

  if (warp >= 8) {
  registers_down();
  if (warp == kFwdLoadWarp) {
    int i = 0;                                    // tiles asked for: K_0 V_0 K_1 V_1 ...
    bool q_asked = false;
    if (n > 0) {
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(q_full, nt * kTB);
        for (int t = 0; t < nt; ++t) tma_tile<DP>(sq + t * kTB, &mq, head, q0 + t * kRows, b, q_full);
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
          tma_tile<DP>(dst, value ? &mv : &mk, hk, j * kRows, b, bar);
        }
        if (patch) {                              // the last tile: once per block
          drain(tail, 0);
          clear_rows<DP>(dst, valid);
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
    if (lane == 0 && n > 0) {
      const uint32_t id_s = idesc_of<T>(kRows, false), id_o = idesc_of<T>((p.D + 15) & ~15, true);
      const int ksteps = (p.D + 15) >> 4;
      auto run = [&]() {
        if (!ptx::mbar_wait(q_full, 0, abort_flag) || !ptx::mbar_wait(full(0), 0, abort_flag)) return;
        ptx::tc_fence_after();
        for (int t = 0; t < nt; ++t) {
          mma_scores(tS + 128 * t, sq + t * kTB, ring, id_s, ksteps);
          ptx::umma_commit(s_full(t));
        }
        ptx::umma_commit(empty(0));
        for (int j = 0; j < n; ++j) {
          const int iv = 2 * j + 1, ik = 2 * j + 2, sv = iv % kStages, sk = ik % kStages;
          const bool more = j + 1 < n;
          if (!ptx::mbar_wait(full(sv), (iv / kStages) & 1, abort_flag)) return;
          for (int t = 0; t < nt; ++t) {
            if (!ptx::mbar_wait(p_ready(t), j & 1, abort_flag)) return;
            ptx::tc_fence_after();
            mma_weigh(tO + DP * t, tS + 128 * t, ring + sv * kTB, id_o, j > 0);
            if (more) {
              if (t == 0 && !ptx::mbar_wait(full(sk), (ik / kStages) & 1, abort_flag)) return;
              mma_scores(tS + 128 * t, sq + t * kTB, ring + sk * kTB, id_s, ksteps);
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
    const int dcols = (p.D + 15) & ~15;
    float m = 0.f, l = 0.f;
    bool ok = t < nt;
    for (int j = 0; ok && j < n; ++j) {
      if (!warp_wait(s_full(t), j & 1, abort_flag)) { ok = false; break; }
      ptx::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int k = 0; k < 4; ++k) ptx::tmem_ld_32x32(s_at + 32 * k, s[k]);
      ptx::tmem_ld_wait();
      const int valid = len - (j0 + j) * kRows;
      if (valid < kRows) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * k + e >= valid) s[k][e] = 0xff800000u;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(s[k][e]));
      mx *= p.c;
      if (j == 0) {
        m = mx == -INFINITY ? 0.f : mx;
      } else if (__any_sync(0xffffffffu, mx > m + 8.f)) {
        const float to = fmaxf(mx, m), f = exp2_fast(m - to);
        m = to;
        l *= f;
        for (int c0 = 0; c0 < dcols; c0 += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32(o_at + c0, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st_32x32(o_at + c0, o);
        }
      }
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int i0 = 64 * h + 2 * e;
          const float x = exp2_fast(fmaf(__uint_as_float(s[i0 >> 5][i0 & 31]), p.c, -m));
          const float y = exp2_fast(fmaf(__uint_as_float(s[i0 >> 5][(i0 & 31) + 1]), p.c, -m));
          sum[e & 1] += x;
          sum[2 + (e & 1)] += y;
          w[e] = pack2<T>(x, y);
        }
        tmem_st_32x32(s_at + 32 * h, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(p_ready(t));
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
          ptx::tmem_ld_32x32(o_at + c0, o);
          ptx::tmem_ld_wait();
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
          for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(o[e + i]) * inv;
          if (p.splits > 1) {
            float* dst = p.part + ((long long)split * rows + out) * p.D + c0 + e;
            *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
            *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
          } else {
            uint4 w = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
            *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.o) + out * p.D + c0 + e) = w;
          }
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

template <typename T, int DP>
int launch_fwd(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TcParams& p, unsigned grid, cudaStream_t st) {
  if (const int rc = allow_dynamic_smem<fwd_tc_kernel<T, DP>>(kFwdSmem<DP>)) return rc;
  fwd_tc_kernel<T, DP><<<grid, kFwdThreads, kFwdSmem<DP>, st>>>(mq, mk, mv, p);
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}

}  // namespace

// The device's status word.  The first call registers it, which a capture in progress on this thread must not mind.
int status_pointer(int** out) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  D2C_CUDA_TRY(cudaThreadExchangeStreamCaptureMode(&mode));
  const int rc = status_word_device_ptr(out);
  const cudaError_t back = cudaThreadExchangeStreamCaptureMode(&mode);
  return rc ? rc : check_cuda(back);
}

// [clips, tokens, heads, D] with element strides s (clip, token, head); a dimension of one element has no stride.
int tile_map(CUtensorMap* map, int dtype, const void* p, int D, int heads, int tokens, int clips, const long long (&s)[3]) {
  EncodeTiled f;
  if (const int rc = encoder(&f)) return rc;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens, (cuuint64_t)clips};
  auto bytes = [&](long long st, int n) { return (cuuint64_t)(n == 1 ? 256 : 2 * st); };
  const cuuint64_t strides[3] = {bytes(s[2], heads), bytes(s[1], tokens), bytes(s[0], clips)};
  const cuuint32_t box[4] = {64, 1, kRows, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult rc = f(map, dtype == D2C_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                        const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? D2C_OK : check_cuda(cudaErrorInvalidValue);
}

int tc_fwd(int dtype, const Args& a, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  int rc;
  if ((rc = tile_map(&mq, dtype, a.q, a.D, a.Hq, a.Lq, a.B, a.qs))) return rc;
  if ((rc = tile_map(&mk, dtype, a.k, a.D, a.Hkv, a.Lk, a.B, a.ks))) return rc;
  if ((rc = tile_map(&mv, dtype, a.v, a.D, a.Hkv, a.Lk, a.B, a.vs))) return rc;
  TcParams p{};
  p.B = a.B; p.Lq = a.Lq; p.Lk = a.Lk; p.Hq = a.Hq; p.Hkv = a.Hkv; p.D = a.D;
  p.c = a.scale * kLog2e;
  p.splits = a.splits;
  p.qblocks = (a.Lq + 2 * kRows - 1) / (2 * kRows);
  p.o = a.o; p.lse = a.lse; p.part = a.part; p.part_lse = a.part_lse;
  p.a = a;
  if ((rc = status_pointer(&p.status))) return rc;
  const long long blocks = (long long)p.qblocks * p.splits * p.Hq * p.B;
  if (blocks > 0x7fffffffLL) return D2C_ERR_TOO_LARGE;
  const unsigned grid = (unsigned)blocks;
  if (dtype == D2C_BF16)
    return a.D <= 64 ? launch_fwd<__nv_bfloat16, 64>(mq, mk, mv, p, grid, st) : launch_fwd<__nv_bfloat16, 128>(mq, mk, mv, p, grid, st);
  return a.D <= 64 ? launch_fwd<__half, 64>(mq, mk, mv, p, grid, st) : launch_fwd<__half, 128>(mq, mk, mv, p, grid, st);
}

}  // namespace attn
}  // namespace d2c

// Gradients of cross attention on tensor cores: fp16 and bf16 tensors whose head width is a multiple of 8, up to 128 channels; fp32
// tensors staged in 16 bits (attention_sm100.cu: split_rows), in one part or two; up to 128 channels.
//
// One kernel, two uses.  A block keeps a tile of 128 rows X (X1, X2) and runs over tiles of 128 rows Y (Y1, Y2):
//   S = X1 Y1^T,  dP = X2 Y2^T,  P = 2^(S scale log2 e - lse),  dS = P (dP - delta)
//   queries:  X = (q, grad_o), Y = (k, v):        grad_q += dS Y1
//   keys:     X = (k, v),      Y = (q, grad_o):   grad_v += P Y2, grad_k += dS Y1      (S, P, dS are transposed; over all heads
//                                                                                       that share the keys)
// so that every gradient has one writer: no atomics, the same bits in every call, for 7 products a score instead of 5.  S, dP and
// the accumulators stay in tensor memory; P and dS go back over S and dP as 16-bit A operands.  The order of the issued products lets
// the tensor cores work on the next S while the warps form dS, and on the next dP while they form P.
//
// A tile's products, exponentials and gradients wait for one another: what a SM does at a time is what it has of independent tiles.  Up
// to 64 channels Y tiles have 64 rows (kY), so that tensor memory (64 + 64 + 64 + 64 columns) and shared memory hold two blocks a SM, of
// 4 working warps, a thread a row.  With operands twice as large (128 channels, or two parts) Y tiles have 128 rows and the one block has
// 8 working warps, a thread a row and half of the columns.  With both, shared memory holds X and one Y1 and one Y2 of 64 rows: the next
// are loaded when these are done.
//
// 2 clips of 3240 queries and up to 12960 keys, 4 heads of 64 in bf16: keys 183 us, queries 152 us, with tiles of 128 x 64 and two blocks a
// SM; with one block of 128 x 128 tiles 212 and 162.
//
// fp16 operands: a probability is of the order of 1 / keys, score gradients are smaller still, and both go with what a loss makes of its
// queries, which may differ by any power of two.  So a row of X has a power of two of its own, 2^lift, that follows the largest of its
// P_xy g_y so far, or a tile's sum of them (g_y: the size of that query's grad_o against the largest; 1 in the queries' kernel, where the
// row is the query): a tile that brings far more takes the row's sums back by the difference, as a running softmax does.  Under that
// scale |dS| <= 2^15, since |dP - delta| <= 2 D max|g_y| max|v|; dS typically lies 2^7 below that, and the second part ends at 2^-24.  fp32
// tensors are staged with every query's grad_o at its own exponent: P g_y takes P's place and is scaled alike.  P itself, for fp16
// tensors, is scaled by 2^14.  Whatever the sizes of grad_o in fp32's normal range and the number of keys (3240 .. 1000000), fp32
// gradients are 0.6e-6 .. 1.9e-6 (2-norm) from 64 bits; one scale for all rows lost the queries 2^-20 below the largest altogether, and 4e-5 at 1000000 keys.  It
// costs 6 % of these kernels in two parts of 64 channels and 12 % of the fp16 keys' kernel of 64 (208 us with one scale, 233 with
// the rows').
#include <algorithm>
#include <type_traits>

#include "attention_tc.cuh"

namespace d2c {
namespace attn {
namespace {

struct BwdParams {
  int B, Lq, Lk, Hq, Hkv, D;
  int width;                     // channels of the operands
  float c, scale;
  int splits, blocks_x;          // tiles of X per head
  const float *lse, *delta;
  const uint32_t* bounds;        // fp16: see largest_sizes
  const int* g_exp;              // fp16: see Args
  void *g1, *g2;                 // keys: grad_v, grad_k; queries: g2 = grad_q
  float* part;                   // queries [splits][B, Lq, Hq][D]; keys [grad_k, grad_v][splits][B, Lk, Hkv][D]
  Args a;                        // lengths
  int* status;
};

// P of a row adds up to 1 over its keys, so that dS_j = p_j ((1 - p_j) dP_j - sum of the other p_k dP_k) is at most max|dP| / 2, a quarter of
// what 2^e_one brings to 1: 2^17 keep it within 2^15.  With one part that does for the queries' kernel: 11 bits of dS down to p =
// 2^-24 where dP is 2^7 below its bound.
constexpr int kFixedLift = 17;

constexpr int y_rows(int size) { return size == 128 ? 128 : 64; }    // size: channels (64, 128) times parts
template <int DP, int kParts>
constexpr int kYRows = y_rows(DP * kParts);
template <int DP, int kParts>
constexpr int kThreads = kYRows<DP, kParts> == 64 ? 256 : 384;       // working warps; MMA issuer, loader, two idle (see registers_up)
template <int DP, int kParts>
constexpr int kStages = DP * kParts == 64 ? 8 : (DP * kParts == 128 ? 4 : 2);
template <int DP, int kParts>
constexpr int kYBytes = kYRows<DP, kParts> * DP * 2 * kParts;
template <int DP, int kParts>
constexpr int kSmem = 2 * kTileBytes<DP> * kParts + kStages<DP, kParts> * kYBytes<DP, kParts> + 1024;

__device__ __forceinline__ void lift_row(uint32_t (&s)[2][32], int lift) {
  const F2 mul = f2(pow2(lift), pow2(lift));
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int e = 0; e < 32; e += 2) {
      float x, y;
      f2_split(mul2(f2(__uint_as_float(s[k][e]), __uint_as_float(s[k][e + 1])), mul), x, y);
      s[k][e] = __float_as_uint(x);
      s[k][e + 1] = __float_as_uint(y);
    }
}

template <typename T, typename Out, int DP, int kParts, bool kKeys>
__global__ void __launch_bounds__(kThreads<DP, kParts>, DP * kParts == 64 ? 2 : 1)
bwd_tc_kernel(const __grid_constant__ CUtensorMap mx1, const __grid_constant__ CUtensorMap mx2, const __grid_constant__ CUtensorMap my1,
              const __grid_constant__ CUtensorMap my2, const __grid_constant__ BwdParams p) {
  constexpr int kY = kYRows<DP, kParts>, kWork = kY / 16;        // rows of a Y tile, working warps
  constexpr int kSt = kStages<DP, kParts>, kTB = kTileBytes<DP> * kParts, kYB = kYBytes<DP, kParts>;
  constexpr int kMmaWarp = kWork, kLoadWarp = kWork + 1, kCols = kY == 64 && DP == 64 ? 256 : 512;
  constexpr bool kApart = kParts == 2 && DP == 64;                        // tensor memory has room for sums of lo parts
  constexpr bool kHalf = std::is_same_v<T, __half>;
  constexpr int kUp = kHalf && kKeys && kParts == 1 ? 14 : 0;             // P is scaled by 2^kUp
  constexpr bool kLift = kHalf && (kKeys || kParts == 2);                 // a row's scale follows what it meets; else it is 2^kFixedLift
  constexpr bool kShared = kLift && kY == 128;    // a row's columns belong to two threads
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kSt + 12];
  __shared__ __align__(16) float rows_of_y[kKeys ? kSt / 2 : 1][kHalf && kParts == 1 ? 3 : 2][kY];   // of a Y tile's queries: lse, delta, g_y
  __shared__ float row_top[kShared ? 2 : 1][kShared ? 2 : 1][kShared ? kRows : 1];    // by turns: what either half of the columns has
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const uint32_t base = (ptx::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t sx = base, ring = base + 2 * kTB, bar0 = ptx::smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (kSt + s); };
  const uint32_t x_full = bar0 + 16 * kSt, tail = x_full + 8, done = x_full + 16, s_full = x_full + 24, dp_full = x_full + 32,
                 p_ready = x_full + 40, ds_ready = x_full + 48;
  auto pair = [&](int w) { return x_full + 56 + 8 * w; };                 // the two warps of 32 rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  long long id = blockIdx.x;
  const int xb = (int)(id % p.blocks_x); id /= p.blocks_x;
  const int split = (int)(id % p.splits); id /= p.splits;
  const int heads = kKeys ? p.Hkv : p.Hq, head = (int)(id % heads), b = (int)(id / heads);
  const int group = p.Hq / p.Hkv, hk = kKeys ? head : head / group;
  const int x0 = xb * kRows;
  const int len = key_length(p.a, b);
  const int qtiles = (p.Lq + kY - 1) / kY;
  int i0, i1;
  share(kKeys ? qtiles * group : (len + kY - 1) / kY, p.splits, split, i0, i1);
  if (kKeys && x0 >= len) i1 = i0;                // keys that are not there
  const int n = i1 - i0;
  // powers of two: of the operands (two parts; e_v and e_g bound them in one part too), and of dP - delta, which they bring to 1 at most
  int e_q = 0, e_k = 0, e_v = 0, e_g = 0, e_one = 0;
  if constexpr (kHalf) {
    const uint32_t* q = p.bounds + (long long)b * p.Hkv + hk;
    const int n_heads = p.B * p.Hkv;
    e_v = scale_exponent(q[2 * n_heads]);
    e_g = scale_exponent(q[3 * n_heads]);         // not above any row's
    e_one = -31 - (32 - __clz(p.D - 1));          // |g 2^e_g| < 2^15, |v 2^e_v| < 2^15, D products, and delta is no larger
    if constexpr (kParts == 2) {
      e_q = scale_exponent(q[0]);
      e_k = scale_exponent(q[n_heads]);
    }
  }
  // tile i of Y: head, first row
  auto y_head = [&](int i) { return kKeys ? head * group + i / qtiles : hk; };
  auto y_row = [&](int i) { return (kKeys ? i % qtiles : i) * kY; };

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSt; ++i) { ptx::mbar_init(full(i), 1); ptx::mbar_init(empty(i), 1); }
    ptx::mbar_init(x_full, 1);
    ptx::mbar_init(tail, 1);
    ptx::mbar_init(done, 1);
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(dp_full, 1);
    ptx::mbar_init(p_ready, kWork);
    ptx::mbar_init(ds_ready, kWork);
    for (int w = 0; w < 4; ++w) ptx::mbar_init(pair(w), 2);
    abort_word = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), kCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_slot, tS = tmem, tD = tmem + kY, tA1 = tmem + 2 * kY, tA2 = tA1 + DP;

  if (warp >= kWork) {
    if constexpr (kCols == 256) registers_down_4();                       // (8 warps alone on a SM have registers enough)
    else if constexpr (kY == 128) registers_down();
    if (warp == kLoadWarp) {
      int i = 0;                                  // Y tiles asked for: Y1 Y2 Y1 Y2 ...
      if (n > 0) {
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(x_full, 2 * kTB);
          tma_tile<DP, kParts>(sx, &mx1, head, x0, b, p.B, x_full);
          tma_tile<DP, kParts>(sx + kTB, &mx2, head, x0, b, p.B, x_full);
        }
        for (; i < 2 * n; ++i) {
          const int s = i % kSt, y = i0 + (i >> 1), h = y_head(y), r0 = y_row(y);
          const bool second = i & 1;
          // the queries' values are asked for before the wait
          float row_lse[kKeys ? kY / 32 : 1], row_delta[kKeys ? kY / 32 : 1];
          int row_exp[kKeys && kHalf ? kY / 32 : 1];
          if constexpr (kKeys) {
            if (!second) {
              const long long at = ((long long)b * p.Hq + h) * p.Lq;
#pragma unroll
              for (int e = 0; e < kY / 32; ++e) {
                const int r = min(r0 + lane + 32 * e, p.Lq - 1);
                row_lse[e] = p.lse[at + r];
                row_delta[e] = p.delta[at + r];
                if constexpr (kHalf) row_exp[e] = p.g_exp[at + r];
              }
            }
          }
          if (!warp_wait(empty(s), ((i / kSt) & 1) ^ 1, abort_flag)) break;
          if constexpr (kKeys) {
            if (!second) {
#pragma unroll
              for (int e = 0; e < kY / 32; ++e) {
                const int r = lane + 32 * e;
                const bool live = r0 + r < p.Lq;  // queries that are not there: P = 0
                float l = row_lse[e] - (float)kUp, d = row_delta[e];
                if constexpr (kHalf) {
                  const int ge = row_exp[e];
                  d = d * pow2(e_v) * pow2(kParts == 2 ? ge : e_g) * pow2(e_one);
                  if constexpr (kParts == 2) l += (float)(ge - e_g);      // P g_y
                  else rows_of_y[s >> 1][2][r] = live && e_g - ge >= -126 ? pow2(e_g - ge) : 0.f;
                }
                rows_of_y[s >> 1][0][r] = live ? l : INFINITY;
                rows_of_y[s >> 1][1][r] = live ? d : 0.f;
              }
              __syncwarp();
            }
          }
          // keys behind the clip's length may hold anything: dS is 0 there, and 0 * NaN is NaN
          const bool patch = !kKeys && !second && len - r0 < kY && len < p.Lk;
          const uint32_t bar = patch ? tail : full(s), dst = ring + s * kYB;
          if (lane == 0) {
            ptx::mbar_arrive_expect_tx(bar, kYB);
            tma_tile<DP, kParts, kY>(dst, second ? &my2 : &my1, h, r0, b, p.B, bar);
          }
          if (patch) {                            // the last tile: once per block
            drain(tail, 0);
            clear_rows<DP, kParts, kY>(dst, len - r0);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(full(s));
          }
        }
        if (lane == 0) {
          drain(x_full, 0);
          for (int w = i > kSt ? i - kSt : 0; w < i; ++w) drain(full(w % kSt), (w / kSt) & 1);
        }
      }
    } else if (warp == kMmaWarp && n > 0 && elect_one()) {
      const uint64_t d_x = ptx::umma_desc_kmajor_sw128(sx), d_y = ptx::umma_desc_kmajor_sw128(ring),
                     d_yt = ptx::umma_desc_mnmajor_sw128(ring, kY * 128, 1024);
      const uint32_t id_s = idesc_of<T>(kY, false), id_a = idesc_of<T>((p.width + 15) & ~15, true);
      const int ksteps = (p.width + 15) >> 4;
      auto slot = [&](int i) { return (uint32_t)((i % kSt) * kYB) >> 4; };
      auto there = [&](int i) { return ptx::mbar_wait(full(i % kSt), (i / kSt) & 1, abort_flag); };
      auto weigh = [&](uint32_t acc, uint32_t w, uint32_t y, bool more) {   // each half of the columns has its parts at its own start
        mma_weigh<DP, kParts, kApart, kY>(acc, w, 32, d_yt + y, id_a, more);
        if constexpr (kY == 128) mma_weigh<DP, kParts, kApart, kY>(acc, w + 64, 32, d_yt + y + 512, id_a, true);
      };
      auto run = [&]() {
        if (!ptx::mbar_wait(x_full, 0, abort_flag) || !there(0)) return;
        ptx::tc_fence_after();
        mma_scores<DP, kParts, kY>(tS, d_x, d_y + slot(0), id_s, ksteps);
        ptx::umma_commit(s_full);
        if (!there(1)) return;
        mma_scores<DP, kParts, kY>(tD, d_x + (kTB >> 4), d_y + slot(1), id_s, ksteps);
        ptx::umma_commit(dp_full);
        if (!kKeys) ptx::umma_commit(empty(1));
        for (int i = 0; i < n; ++i) {
          const int y1 = 2 * i, y2 = y1 + 1;
          const bool more = i + 1 < n;
          if (kSt > 2 && more && !there(y1 + 2)) return;                  // what is there long before P
          if (!ptx::mbar_wait(p_ready, i & 1, abort_flag)) return;
          ptx::tc_fence_after();
          if constexpr (kKeys) {
            weigh(tA1, tS, slot(y2), i > 0);
            ptx::umma_commit(empty(y2 % kSt));    // before the next S: a short ring waits for this tile's place
          }
          if (kSt > 2 && more) {
            mma_scores<DP, kParts, kY>(tS, d_x, d_y + slot(y1 + 2), id_s, ksteps);
            ptx::umma_commit(s_full);
            if (!there(y2 + 2)) return;
          }
          if (!ptx::mbar_wait(ds_ready, i & 1, abort_flag)) return;
          ptx::tc_fence_after();
          weigh(tA2, tD, slot(y1), i > 0);
          ptx::umma_commit(empty(y1 % kSt));
          if (kSt == 2 && more) {                 // the next tiles take the places of these
            if (!there(y1 + 2)) return;
            mma_scores<DP, kParts, kY>(tS, d_x, d_y + slot(y1 + 2), id_s, ksteps);
            ptx::umma_commit(s_full);
            if (!there(y2 + 2)) return;
          }
          if (more) {
            mma_scores<DP, kParts, kY>(tD, d_x + (kTB >> 4), d_y + slot(y2 + 2), id_s, ksteps);
            ptx::umma_commit(dp_full);
            if (!kKeys) ptx::umma_commit(empty((y2 + 2) % kSt));
          }
        }
      };
      run();
      ptx::umma_commit(done);
      drain(done, 0);
    }
  } else {
    if constexpr (kCols == 256) registers_up_4();
    else if constexpr (kY == 128) registers_up();
    const int half = warp >> 2, row = (warp & 3) * 32 + lane, xi = x0 + row;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tS + 64 * half + lanes, d_at = tD + 64 * half + lanes;
    float lse = INFINITY, delta = 0.f;            // queries: this row's
    int e_row = e_g;                              // exponent of grad_o
    if (!kKeys && xi < p.Lq) {
      const long long at = ((long long)b * p.Hq + head) * p.Lq + xi;
      lse = p.lse[at];
      if constexpr (kHalf) e_row = p.g_exp[at];
      delta = p.delta[at];
      if constexpr (kHalf) delta = delta * pow2(e_v) * pow2(e_row) * pow2(e_one);
    }
    float dp_mul = !kHalf ? 1.f : pow2(min(126, e_one + (kParts == 2 ? 0 : e_row + e_v)));   // (126: a row of zeros)
    if constexpr (kHalf && !kLift) {
      dp_mul *= pow2(kFixedLift);
      delta *= pow2(kFixedLift);
    }
    int lift = kHalf && !kLift ? kFixedLift : 0;  // of this row: P 2^lift
    const bool row_in = kKeys ? xi < len : true, x_ragged = kKeys && x0 + kRows > len;
    constexpr bool kZeroEach = kKeys && kParts == 2;   // keys that are not there value by value: at the end, both parts spill
    float c = p.c;
    if constexpr (kParts == 2) c = ldexpf(c, -e_q - e_k);
    const F2 c2 = f2(c, c);
    // a sum's columns that this thread takes back: all of its row, or half of them
    auto take_back = [&](uint32_t acc, float f) {
      constexpr int kOwn = kShared ? DP / 2 : DP;
      acc += lanes + (kShared ? half * kOwn : 0);
#pragma unroll 1
      for (int c0 = 0; c0 < (kApart ? 2 : 1) * kOwn; c0 += 32) {
        const uint32_t at = acc + (c0 < kOwn ? c0 : 128 + c0 - kOwn);
        uint32_t r[32];
        ptx::tmem_ld_32x32(at, r);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * f);
        tmem_st_32x32(at, r);
      }
      tmem_st_wait();
    };
    // The row's `lift` goes by the exponent of tile i's largest value or sum: what this thread has of the row, and what the row has.  It is
    // brought to 2^kTop, and may grow to 2^15 afterwards (above 2^35 it is not finite).
    constexpr int kTop = kKeys && kParts == 2 ? 9 : 11;
    bool lower = false;                           // the warp's sums are to be taken back, by `fall`
    float fall = 1.f, own_top = 0.f;
    auto post = [&](int i, float top) {
      own_top = top;
      if constexpr (kShared) {
        row_top[i & 1][half][row] = top;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(pair(warp & 3));
      }
    };
    auto follow = [&](int i) {
      float top = own_top;
      if constexpr (kShared) {
        if (!warp_wait(pair(warp & 3), i & 1, abort_flag)) return false;
        top = fmaxf(top, row_top[i & 1][half ^ 1][row]);
      }
      const int to = kTop - __float2int_rd(fminf(fmaxf(top, -89.f), 35.f));
      lower = false;
      fall = 1.f;
      if (i == 0) {
        lift = to;
      } else if (__any_sync(0xffffffffu, lift - to >= 15 - kTop)) {
        lower = true;
        if (lift - to >= 15 - kTop) {
          fall = pow2(to - lift);
          lift = to;
        }
      }
      return true;
    };
    bool ok = true;
    for (int i = 0; ok && i < n; ++i) {
      if (!warp_wait(s_full, i & 1, abort_flag)) { ok = false; break; }
      ptx::tc_fence_after();
      uint32_t s[2][32];
#pragma unroll
      for (int k = 0; k < 2; ++k) ptx::tmem_ld_32x32(s_at + 32 * k, s[k]);
      ptx::tmem_ld_wait();
      if constexpr (!kKeys) {                     // S has been read
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_ready);
      }
      const int valid = kKeys ? kY : len - y_row(i0 + i);   // columns from there on are masked
      const bool ragged = valid < kY;
      const float* ly = kKeys ? &rows_of_y[(2 * i % kSt) >> 1][0][64 * half] : nullptr;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float4 l4 = make_float4(lse, lse, lse, lse);
          if constexpr (kKeys) l4 = *reinterpret_cast<const float4*>(ly + 32 * k + e);
          const F2 lv[2] = {f2(-l4.x, -l4.y), f2(-l4.z, -l4.w)};
#pragma unroll
          for (int u = 0; u < 4; u += 2) {
            float x, y;
            f2_split(fma2(f2(__uint_as_float(s[k][e + u]), __uint_as_float(s[k][e + u + 1])), c2, lv[u / 2]), x, y);
            if constexpr (kKeys && kParts == 2) {
              s[k][e + u] = row_in ? __float_as_uint(x) : 0xff800000u;    // keys that are not there
              s[k][e + u + 1] = row_in ? __float_as_uint(y) : 0xff800000u;
            } else {
              s[k][e + u] = __float_as_uint(exp2_fast(x));
              s[k][e + u + 1] = __float_as_uint(exp2_fast(y));
            }
          }
        }
      if constexpr (kKeys && kParts == 2) {
        // P waits for its scale: from the largest exponent, which the other warp has before the exponentials are formed
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 64; e += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            top4[u] = fmaxf(fmaxf(top4[u], __uint_as_float(s[e >> 5][(e & 31) + u])), __uint_as_float(s[e >> 5][(e & 31) + 4 + u]));
        post(i, fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])));
#pragma unroll
        for (int e = 0; e < 64; ++e) s[e >> 5][e & 31] = __float_as_uint(exp2_fast(__uint_as_float(s[e >> 5][e & 31])));
        if (!follow(i)) { ok = false; break; }
        if (lower) take_back(tA1, fall);
        lift_row(s, lift);
      } else if constexpr (kLift) {
        // only dS waits for it: from the sum, which is at least the largest.  (64 maxima, of half the additions' rate, took a fifth of the
        // queries' kernel.)
        if (ragged) {
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (64 * half + e >= valid) s[e >> 5][e & 31] = 0u;
        }
        F2 sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const uint32_t* v = &s[e >> 5][e & 31];
          const F2 a = f2(__uint_as_float(v[0]), __uint_as_float(v[1])), b = f2(__uint_as_float(v[2]), __uint_as_float(v[3]));
          F2 &sa = sum[e / 2 & 2], &sb = sum[(e / 2 & 2) + 1];
          if constexpr (kKeys) {
            const float4 g4 = *reinterpret_cast<const float4*>(ly + 2 * kY + e);
            sa = fma2(a, f2(g4.x, g4.y), sa);
            sb = fma2(b, f2(g4.z, g4.w), sb);
          } else {
            sa = add2(sa, a);
            sb = add2(sb, b);
          }
        }
        float x, y;
        f2_split(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), x, y);
        post(i, row_in ? (float)((int)(__float_as_uint(x + y) >> 23) - 127) : -INFINITY);
        if constexpr (!kKeys) {
          if (!follow(i)) { ok = false; break; }
        }
      }
      if constexpr (kKeys) {
        uint32_t w[32], rest[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = __uint_as_float(s[e >> 4][2 * e & 31]), y = __uint_as_float(s[e >> 4][(2 * e & 31) + 1]);
          w[e] = pack2<T>(x, y);
          if constexpr (kParts == 2) rest[e] = pack2_rest(x, y, w[e]);
        }
        if (!kZeroEach && x_ragged && !row_in) {  // keys that are not there: whatever S is
#pragma unroll
          for (int e = 0; e < 32; ++e) w[e] = 0u;
        }
        tmem_st_32x32(s_at, w);
        if constexpr (kParts == 2) tmem_st_32x32(s_at + 32, rest);
        tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_ready);
        if constexpr (kLift && kParts == 1) {
          if (!follow(i)) { ok = false; break; }
          lift_row(s, lift);
        }
      }
      if (!warp_wait(dp_full, i & 1, abort_flag)) { ok = false; break; }
      ptx::tc_fence_after();
      float dm = dp_mul, dd = delta;
      if constexpr (kLift) {
        if constexpr (!kKeys) {
          dm *= pow2(lift);
          dd *= pow2(lift);
        }
        if (lower) take_back(tA2, fall);
      }
      uint32_t w[32], rest[kParts == 2 ? 32 : 1];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t d[32];
        ptx::tmem_ld_32x32(d_at + 32 * k, d);
        ptx::tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float4 d4 = make_float4(dd, dd, dd, dd);
          if constexpr (kKeys) d4 = *reinterpret_cast<const float4*>(ly + kY + 32 * k + e);
          const F2 dv[2] = {f2(-d4.x, -d4.y), f2(-d4.z, -d4.w)};
          float v[4];
#pragma unroll
          for (int u = 0; u < 4; u += 2) {
            const F2 dp = f2(__uint_as_float(d[e + u]), __uint_as_float(d[e + u + 1]));
            const F2 t = mul2(f2(__uint_as_float(s[k][e + u]), __uint_as_float(s[k][e + u + 1])),
                              kHalf ? fma2(dp, f2(dm, dm), dv[u / 2]) : add2(dp, dv[u / 2]));
            f2_split(t, v[u], v[u + 1]);
          }
          if constexpr (kZeroEach) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (!row_in) v[u] = 0.f;
          }
          if (!kKeys && ragged) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (64 * half + 32 * k + e + u >= valid) v[u] = 0.f;
          }
          w[16 * k + e / 2] = pack2<T>(v[0], v[1]);
          w[16 * k + e / 2 + 1] = pack2<T>(v[2], v[3]);
          if constexpr (kParts == 2) {
            rest[16 * k + e / 2] = pack2_rest(v[0], v[1], w[16 * k + e / 2]);
            rest[16 * k + e / 2 + 1] = pack2_rest(v[2], v[3], w[16 * k + e / 2 + 1]);
          }
        }
      }
      if (kKeys && !kZeroEach && x_ragged && !row_in) {
#pragma unroll
        for (int e = 0; e < 32; ++e) w[e] = 0u;
      }
      tmem_st_32x32(d_at, w);
      if constexpr (kParts == 2) tmem_st_32x32(d_at + 32, rest);
      tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ds_ready);
    }
    if (ok && n > 0) {
      ok = warp_wait(done, 0, abort_flag);
      ptx::tc_fence_after();
    }
    if (ok) {
      // keys: grad_v and grad_k, by four warps each or one after the other; queries: all channels, or half of them
      const int there = kKeys ? p.Lk : p.Lq;
      const long long rows = (long long)p.B * there * heads, out = ((long long)b * there + xi) * heads + head;
      auto write = [&](bool first, int c0, int c_end) {
        // what the sums were scaled by: P (by kUp, or lift) and grad_o; P, dP - delta and the other factor
        const int up = first ? (kParts == 2 ? lift + e_g : kUp) : kUp + lift + e_row + e_v + e_one + (kKeys ? e_q : e_k);
        // (three factors: together they may be beyond a float's exponents)
        const int down = max(-378, min(378, -up));
        const float m1 = pow2(down / 3), m2 = pow2((down + 1) / 3), m3 = pow2(down - down / 3 - (down + 1) / 3);
        const uint32_t acc = (first ? tA1 : tA2) + lanes;
        Out* dst = reinterpret_cast<Out*>(first ? p.g1 : p.g2) + out * p.D;
        float* part = p.splits > 1 ? p.part + (((long long)(first ? p.splits : 0) + split) * rows + out) * p.D : nullptr;
        for (; c0 < c_end; c0 += 32) {
          uint32_t r[32];
          if (n > 0) {
            load_sums<kApart>(acc + c0, r);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0u;
          }
          if (xi >= there) continue;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (c0 + e >= c_end) break;
            float f[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              f[u] = __uint_as_float(r[e + u]) * (first ? 1.f : p.scale);
              if constexpr (kHalf) f[u] = f[u] * m1 * m2 * m3;
            }
            if (part) store8(part + c0 + e, f, p.D - c0 - e, p.D % 4 == 0);
            else store8(dst + c0 + e, f, p.D - c0 - e, p.D * sizeof(Out) % 16 == 0);
          }
        }
      };
      if (kY == 64) {
        if (kKeys) write(true, 0, p.D);
        write(false, 0, p.D);
      } else if (kKeys) {
        write(half == 0, 0, p.D);
      } else {
        write(false, half * (DP / 2), min(p.D, (half + 1) * (DP / 2)));
      }
    }
    ptx::tc_fence_before();
  }
  __syncthreads();
  report(p.status, abort_flag);
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kCols);
  }
}

template <typename T, typename Out, int DP, int kParts, bool kKeys>
int launch(const CUtensorMap (&m)[4], const BwdParams& p, cudaStream_t st) {
  const long long blocks = (long long)p.blocks_x * p.splits * (kKeys ? p.Hkv : p.Hq) * p.B;
  if (blocks > 0x7fffffffLL) return D2C_ERR_TOO_LARGE;
  constexpr int smem = kSmem<DP, kParts>;
  if (const int rc = allow_dynamic_smem<bwd_tc_kernel<T, Out, DP, kParts, kKeys>>(smem)) return rc;
  bwd_tc_kernel<T, Out, DP, kParts, kKeys><<<(unsigned)blocks, kThreads<DP, kParts>, smem, st>>>(m[0], m[1], m[2], m[3], p);
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}
template <typename T, typename Out, int DP, int kParts>
int by_side(const CUtensorMap (&m)[4], const BwdParams& p, bool keys, cudaStream_t st) {
  return keys ? launch<T, Out, DP, kParts, true>(m, p, st) : launch<T, Out, DP, kParts, false>(m, p, st);
}
template <typename T, typename Out, int kParts>
int by_width(const CUtensorMap (&m)[4], const BwdParams& p, bool keys, cudaStream_t st) {
  return p.width <= 64 ? by_side<T, Out, 64, kParts>(m, p, keys, st) : by_side<T, Out, 128, kParts>(m, p, keys, st);
}

}  // namespace

int tc_bwd(int dtype, const Args& a, const Operand (&x)[4], int parts, bool keys, const uint32_t* bounds, cudaStream_t st) {
  BwdParams p{};
  p.B = a.B; p.Lq = a.Lq; p.Lk = a.Lk; p.Hq = a.Hq; p.Hkv = a.Hkv; p.D = a.D;
  p.width = (a.D + 7) / 8 * 8;
  CUtensorMap q, k, v, g;
  int rc;
  const bool staged = dtype == D2C_F32;
  if (staged) dtype = parts == 2 ? D2C_F16 : D2C_BF16;
  const int rows = y_rows((p.width <= 64 ? 64 : 128) * parts), q_rows = keys ? rows : kRows, k_rows = keys ? kRows : rows;
  if ((rc = tile_map(&q, x[0], dtype, p.width, a.Hq, a.Lq, a.B * parts, q_rows))) return rc;
  if ((rc = tile_map(&k, x[1], dtype, p.width, a.Hkv, a.Lk, a.B * parts, k_rows))) return rc;
  if ((rc = tile_map(&v, x[2], dtype, p.width, a.Hkv, a.Lk, a.B * parts, k_rows))) return rc;
  if ((rc = tile_map(&g, x[3], dtype, p.width, a.Hq, a.Lq, a.B * parts, q_rows))) return rc;
  const CUtensorMap maps[4] = {keys ? k : q, keys ? v : g, keys ? q : k, keys ? g : v};
  p.c = a.scale * kLog2e; p.scale = a.scale;
  p.splits = a.splits;
  p.blocks_x = ((keys ? a.Lk : a.Lq) + kRows - 1) / kRows;
  p.lse = a.lse; p.delta = a.delta; p.bounds = bounds; p.g_exp = a.g_exp;
  p.g1 = a.gv; p.g2 = keys ? a.gk : a.gq;
  p.part = a.part;
  p.a = a;
  if ((rc = status_pointer(&p.status))) return rc;
  if (staged) return parts == 2 ? by_width<__half, float, 2>(maps, p, keys, st) : by_width<__nv_bfloat16, float, 1>(maps, p, keys, st);
  return dtype == D2C_BF16 ? by_width<__nv_bfloat16, __nv_bfloat16, 1>(maps, p, keys, st) : by_width<__half, __half, 1>(maps, p, keys, st);
}

}  // namespace attn
}  // namespace d2c

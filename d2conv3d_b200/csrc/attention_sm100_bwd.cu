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
// fp16 operands: a probability is of the order of 1 / keys, score gradients are smaller still, and both go with the sizes of grad_o and v,
// which may differ by any power of two from query to query and from key to key.  fp32 tensors are staged with every query's grad_o at its
// own exponent; in the keys' kernel P g_y takes P's place (g_y: the size of that query's grad_o against the largest), and has, row by row,
// a power of two of its own that follows the largest that the row has met: a tile that brings far more takes the row's sums back by the
// difference, as a running softmax does.  (P of fp16 tensors, and of the queries' kernel, is at most 1 and scaled by a constant.)  dS is
// scaled by what |dP - delta| <= 2 D max|g_y| max|v| allows, less what dS usually lies below that.  How large it was is added up beside its
// rounding, and if a row of the block was beyond fp16, or so small that its last bits were lost, the block runs over its tiles again, each row
// with a scale of its own.  Ordinary tensors hardly ever need that; one value 2^10 times the others that nobody looks at does, and then costs
// twice the time instead of 1e-4 of every query's gradient.
// fp32 gradients are 0.6e-6 .. 1.9e-6 (2-norm) from 64 bits whatever the sizes of grad_o in fp32's normal range and the number of keys
// (3240 .. 1000000); one scale for all rows lost the queries 2^-20 below the largest altogether, and 4e-5 at 1000000 keys.  Against that
// (2 x 3240 x 12960, 4 heads, keys + queries): two parts of 64 channels 586 + 416 us for 547 + 378; fp16 of 64 channels 217 + 192 for 208 +
// 167, of 128 channels 325 + 265 for 380 + 257 (a tile's values of the queries are asked for before its place is free).
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
  constexpr bool kLift = kKeys && kParts == 2;    // a row's scale of P follows what it meets
  constexpr bool kShared = kHalf && kY == 128;    // a row's columns belong to two threads
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kSt + 12];
  __shared__ __align__(16) float rows_of_y[kKeys ? kSt / 2 : 1][2][kY];   // of a Y tile's queries: lse, delta
  __shared__ float row_top[kShared ? 2 : 1][kShared ? 2 : 1][kShared ? kRows : 1];    // by turns: what either half of a row's columns has
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, again_word;
  volatile int *abort_flag = &abort_word, *again = &again_word;
  const uint32_t base = (ptx::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t sx = base, ring = base + 2 * kTB, bar0 = ptx::smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (kSt + s); };
  const uint32_t x_full = bar0 + 16 * kSt, tail = x_full + 8, done = x_full + 16, s_full = x_full + 24, dp_full = x_full + 32,
                 p_ready = x_full + 40, ds_ready = x_full + 48;
  auto pair = [&](int w) { return x_full + 56 + 8 * w; };                 // the two warps of 32 rows
  const uint32_t verdict = x_full + 88;           // whether the tiles are run over again (fp16)
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
  // powers of two: of the operands (two parts; e_v and e_g bound them in one part too), and of dP - delta
  int e_q = 0, e_k = 0, e_v = 0, e_g = 0, e_one = 0, e_first = 0;
  bool nothing = false;                           // grad_o or v are zero: so is dS
  if constexpr (kHalf) {
    const uint32_t* q = p.bounds + (long long)b * p.Hkv + hk;
    const int n_heads = p.B * p.Hkv;
    e_v = scale_exponent(q[2 * n_heads]);
    e_g = scale_exponent(q[3 * n_heads]);         // not above any row's
    nothing = q[2 * n_heads] == 0u || q[3 * n_heads] == 0u;
    // |g 2^e_g| < 2^15, |v 2^e_v| < 2^15, D products, and delta is no larger: 1 at most, and then what dS is scaled by
    e_one = -31 - (32 - __clz(p.D - 1));
    const int bits = 32 - __clz(max(len, 2) - 1); // p is of the order of 2^-bits, dP - delta of 2^-7
    e_first = kLift ? 5 : (kParts == 2 ? max(22, bits + 3) : max(17, bits));
    e_one += e_first - kUp;
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
    ptx::mbar_init(verdict, kWork);
    abort_word = again_word = 0;
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
        for (int pass = 0; ; ++i) {
          if (i == 2 * n * (pass + 1)) {
            if (!kHalf || pass || !warp_wait(verdict, 0, abort_flag) || !*again) break;
            pass = 1;
          }
          const int s = i % kSt, y = i0 + (i >> 1) - pass * n, h = y_head(y), r0 = y_row(y);
          const bool second = i & 1;
          // the queries' values are asked for before the wait
          float row_lse[kKeys ? kY / 32 : 1], row_delta[kKeys ? kY / 32 : 1];
          int row_exp[kKeys && kParts == 2 ? kY / 32 : 1];
          if constexpr (kKeys) {
            if (!second) {
              const long long at = ((long long)b * p.Hq + h) * p.Lq;
#pragma unroll
              for (int e = 0; e < kY / 32; ++e) {
                const int r = min(r0 + lane + 32 * e, p.Lq - 1);
                row_lse[e] = p.lse[at + r];
                row_delta[e] = p.delta[at + r];
                if constexpr (kParts == 2) row_exp[e] = p.g_exp[at + r];
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
                if constexpr (kHalf) d = d * pow2(e_v) * pow2(kParts == 2 ? row_exp[e] : e_g) * pow2(e_one);
                if constexpr (kParts == 2) l += (float)(row_exp[e] - e_g);        // P g_y
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
          if (patch) {                            // the last tile: once a pass
            drain(tail, pass);
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
      auto run = [&](int first) {                 // tiles [first, first + n) of the ring's count
        if (!ptx::mbar_wait(x_full, 0, abort_flag) || !there(2 * first)) return;
        ptx::tc_fence_after();
        mma_scores<DP, kParts, kY>(tS, d_x, d_y + slot(2 * first), id_s, ksteps);
        ptx::umma_commit(s_full);
        if (!there(2 * first + 1)) return;
        mma_scores<DP, kParts, kY>(tD, d_x + (kTB >> 4), d_y + slot(2 * first + 1), id_s, ksteps);
        ptx::umma_commit(dp_full);
        if (!kKeys) ptx::umma_commit(empty((2 * first + 1) % kSt));
        for (int i = first; i < first + n; ++i) {
          const int y1 = 2 * i, y2 = y1 + 1;
          const bool more = i + 1 < first + n;
          if (kSt > 2 && more && !there(y1 + 2)) return;                  // what is there long before P
          if (!ptx::mbar_wait(p_ready, i & 1, abort_flag)) return;
          ptx::tc_fence_after();
          if constexpr (kKeys) {
            weigh(tA1, tS, slot(y2), i > first);
            ptx::umma_commit(empty(y2 % kSt));    // before the next S: a short ring waits for this tile's place
          }
          if (kSt > 2 && more) {
            mma_scores<DP, kParts, kY>(tS, d_x, d_y + slot(y1 + 2), id_s, ksteps);
            ptx::umma_commit(s_full);
            if (!there(y2 + 2)) return;
          }
          if (!ptx::mbar_wait(ds_ready, i & 1, abort_flag)) return;
          ptx::tc_fence_after();
          weigh(tA2, tD, slot(y1), i > first);
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
      run(0);
      ptx::umma_commit(done);
      if (kHalf && ptx::mbar_wait(verdict, 0, abort_flag) && *again) {
        drain(done, 0);
        run(n);
        ptx::umma_commit(done);
        drain(done, 1);
      } else {
        drain(done, 0);
      }
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
    const float dp_mul = !kHalf ? 1.f : pow2(min(126, e_one + (kParts == 2 ? 0 : e_row + e_v)));   // (126: a row of zeros)
    int lift = 0, scale = 0;                      // of this row: P 2^lift (kLift); dS 2^scale besides the constant one, kLift: 2^(lift + scale)
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
    // What the other half of a row's columns has of a value that this half posts.
    int turn = 0;
    auto post = [&](float x) {
      if constexpr (kShared) {
        row_top[turn & 1][half][row] = x;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(pair(warp & 3));
      }
    };
    auto other = [&](float mine, float& x) {
      x = mine;
      if constexpr (kShared) {
        if (!warp_wait(pair(warp & 3), turn & 1, abort_flag)) return false;
        x = row_top[turn & 1][half ^ 1][row];
        ++turn;
      }
      return true;
    };
    float most = 0.f, most_free = 0.f;            // largest sum of a tile's |dS|, as it is scaled; without 2^lift
    bool ok = true;
    int pass = 0;
    for (bool run = true; run;) {                 // once, or twice: the body keeps its indentation
    run = false;
    for (int i = 0; ok && i < n; ++i) {
      const int at = pass * n + i;
      if (!warp_wait(s_full, at & 1, abort_flag)) { ok = false; break; }
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
      const float* ly = kKeys ? &rows_of_y[(2 * at % kSt) >> 1][0][64 * half] : nullptr;
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
      bool lower = false;                         // the warp's sums are taken back, by `fall`
      float fall = 1.f;
      if constexpr (kLift) {
        // P waits for its scale: from the largest exponent, which the other warp has before the exponentials are formed.  It is brought to
        // 2^9 .. 2^10, and may grow to 2^15 afterwards (above 2^35 it is not finite).
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, theirs;
#pragma unroll
        for (int e = 0; e < 64; e += 8)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            top4[u] = fmaxf(fmaxf(top4[u], __uint_as_float(s[e >> 5][(e & 31) + u])), __uint_as_float(s[e >> 5][(e & 31) + 4 + u]));
        const float largest = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
        post(largest);
#pragma unroll
        for (int e = 0; e < 64; ++e) s[e >> 5][e & 31] = __float_as_uint(exp2_fast(__uint_as_float(s[e >> 5][e & 31])));
        if (!other(largest, theirs)) { ok = false; break; }
        const int to = 9 - __float2int_rd(fminf(fmaxf(fmaxf(largest, theirs), -89.f), 35.f));
        if (i == 0) {
          lift = to;
        } else if (__any_sync(0xffffffffu, lift - to >= 6)) {
          lower = true;
          if (lift - to >= 6) {
            fall = pow2(to - lift);
            lift = to;
          }
          take_back(tA1, fall);
        }
        lift_row(s, lift);
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
        if constexpr (kHalf) {                    // the second pass has the row's own scale: with kLift, whatever P's is
          if (pass) lift_row(s, kLift ? max(-126, scale - lift) : scale);
        }
      }
      if (!warp_wait(dp_full, at & 1, abort_flag)) { ok = false; break; }
      ptx::tc_fence_after();
      float dm = dp_mul, dd = delta;
      if constexpr (kHalf && !kKeys) {
        dm *= pow2(scale);
        dd *= pow2(scale);
      }
      if constexpr (kLift) {
        if (lower && !pass) take_back(tA2, fall);
      }
      __half2 sizes[4];                           // sums of |dS| as they are rounded
#pragma unroll
      for (int u = 0; u < 4; ++u) sizes[u] = __float2half2_rn(0.f);
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
          if constexpr (kHalf) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              __half2& a = sizes[u + (e & 4) / 2];
              a = __hadd2(a, __habs2(*reinterpret_cast<const __half2*>(&w[16 * k + e / 2 + u])));
            }
          }
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
      if constexpr (kHalf) {
        const float2 x = __half22float2(__hadd2(__hadd2(sizes[0], sizes[1]), __hadd2(sizes[2], sizes[3])));
        most = fmaxf(most, x.x + x.y);
        if constexpr (kLift) most_free = fmaxf(most_free, (x.x + x.y) * pow2(-lift));
      }
    }
    if (ok && n > 0) {
      ok = warp_wait(done, pass, abort_flag);
      ptx::tc_fence_after();
    }
    if constexpr (kHalf) {
      if (ok && n > 0 && !pass) {
        float theirs;
        post(most);
        ok = other(most, theirs);
        most = fmaxf(most, theirs);
        if constexpr (kLift) {
          post(most_free);
          ok = ok && other(most_free, theirs);
          most_free = fmaxf(most_free, theirs) * pow2(lift);     // as it would be with the last lift
        } else {
          most_free = most;
        }
        // What rounding to fp16's smallest step, 2^-24, takes from such a sum: nothing that 22 bits have left, in two parts from 2^0 on, or
        // 11 bits, in one part from 2^-5 on; nor what a fp16 result shows (|q| or |k| times the scale up to 2^4).  A sum of zero is taken
        // for 2^-25 where it may be less.
        const int up = kUp + e_row + e_v + e_one, size = most_free > 0.f ? ilogbf(most_free) : -25;
        const bool none = nothing || (!kKeys && (e_row == 126 || xi >= p.Lq)), over = most >= 32768.f;
        const bool under = !none && size < (kParts == 2 ? 0 : -5) && (kParts == 2 || 3 + (31 - __clz(n * kY)) / 2 >= up);
        const bool off = row_in && (over || under);
        scale = lift + (over ? (kLift ? 0 : 15) - e_first : (under ? min(100, 11 - size) : 0));
        if (__any_sync(0xffffffffu, off) && lane == 0) *again = 1;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(verdict);
        ok = ok && warp_wait(verdict, 0, abort_flag);
        run = ok && *again;
        if (run) pass = 1;
        else scale = 0;
      }
    }
    }
    if (ok) {
      // keys: grad_v and grad_k, by four warps each or one after the other; queries: all channels, or half of them
      const int there = kKeys ? p.Lk : p.Lq;
      const long long rows = (long long)p.B * there * heads, out = ((long long)b * there + xi) * heads + head;
      auto write = [&](bool first, int c0, int c_end) {
        // what the sums were scaled by: P and grad_o; dS and the other factor
        const int up = first ? (kParts == 2 ? lift + e_g : kUp) : kUp + (kLift && pass ? scale : lift + scale) + e_row + e_v + e_one + (kKeys ? e_q : e_k);
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

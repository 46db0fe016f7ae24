// Pieces that the tensor-core attention kernels share: TMA tile loads, tensor-memory stores, MMAs whose A operand lies in tensor
// memory, and the shared-memory operand tile.
//
// Operand tile: 128 rows (queries or keys) of one head, as 64-channel halves of [128][128 bytes] with the 128-byte swizzle: what one
// tensor-map box delivers.  Read with the channels as the reduction (K-major) it is an operand of q k^T; read with the rows as the
// reduction (MN-major) the same bytes are the B operand of p v.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "attention.h"
#include "sm100_ptx.cuh"

namespace d2c {
namespace attn {

constexpr int kRows = 128;                       // rows of a tile
constexpr int kHalfBytes = kRows * 128;          // 64 channels of it
template <int DP>
constexpr int kTileBytes = kHalfBytes * (DP / 64);

// fp32 tensors are staged (split_rows) in `kParts` = 2 operand tiles behind one another: fp16, hi = fp16(x 2^e) and lo = fp16(x 2^e - hi),
// whose products hi hi + lo hi + hi lo keep 22 bits of each factor, with 2^e from the largest element of the clip and key head (grad_o: of
// the query's row, whose sizes differ by what a loss makes of them): an element keeps its 22 bits down to 2^-18 of that largest one, and
// is off by 2^-40 of it below.  Or in one part, bf16.  The parts are the outer half of a tensor map's clips.
//
// One box of 64 channels x 1 head x 128 (R) tokens x 1 clip; what lies outside the tensor arrives as zeros.  x is 0 or 64.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int head, int token, int clip, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(map), "r"(x), "r"(head), "r"(token), "r"(clip), "r"(bar)
               : "memory");
}
template <int DP, int kParts, int R = kRows>
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int head, int token, int clip, int clips, uint32_t bar) {
#pragma unroll
  for (int part = 0; part < kParts; ++part)
#pragma unroll
    for (int h = 0; h < DP / 64; ++h)
      tma_box(dst + (part * DP / 64 + h) * R * 128, map, h * 64, head, token, part * clips + clip, bar);
}

// Zeroes rows [from, R) of a tile of R rows (one warp).
template <int DP, int kParts, int R = kRows>
__device__ __forceinline__ void clear_rows(uint32_t tile, int from) {
  const int lane = threadIdx.x & 31;
  for (int i = from * 8 + lane; i < R * 8; i += 32) {            // 16-byte pieces: the swizzle stays inside a row
#pragma unroll
    for (int h = 0; h < kParts * DP / 64; ++h) ptx::sts_v4(tile + h * R * 128 + i * 16, make_uint4(0u, 0u, 0u, 0u));
  }
}

// 32 lanes x 32 consecutive 32-bit columns of tensor memory.
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D[tmem] (+)= A[tmem] * B[smem], A 128 rows (lanes) x 16 of the reduction (8 columns of pairs).  Issued by one thread.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor: A and B fp16 or bf16 alike, fp32 accumulator, 128 x N.  b_mn: B's rows are the reduction (MN-major).
template <typename T>
__device__ __forceinline__ uint32_t idesc_of(int N, bool b_mn) {
  const uint32_t fmt = std::is_same_v<T, __nv_bfloat16> ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// One thread of the (converged) warp.  Inside `if (elect_one())` the compiler knows that a single thread runs and feeds the MMAs from
// uniform registers; inside `if (lane == 0)` a 128 x 64 x 16 product issued every 51 clocks instead of 34.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// Operand descriptors are formed once per buffer; tiles, halves and steps are constant distances (in 16 bytes) on the address field:
// with a descriptor built for each product in a rolled loop, the products issued 200 clocks apart instead of their 64.
//
// D (128 x RY) = X Y^T over the channels, both K-major (descriptors of the first part's first step); ksteps = channels / 16 rounded up
// (zero-filled above D).
// The products with a lo part come first: the tensor cores truncate the sum at every product, by the size that it has then.
template <int DP, int kParts, int RY = kRows>
__device__ __forceinline__ void mma_scores(uint32_t d_tmem, uint64_t x, uint64_t y, uint32_t idesc, int ksteps) {
#pragma unroll
  for (int pass = kParts == 2 ? 2 : 0; pass >= 0; --pass) {              // hi lo, lo hi, hi hi
    const uint32_t xp = pass == 1 ? kTileBytes<DP> >> 4 : 0, yp = pass == 2 ? RY * DP * 2 >> 4 : 0;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const uint32_t in = (k & 3) * 2, h = k >> 2;
      if (k < ksteps)
        ptx::umma_bf16(d_tmem, x + (xp + in + h * (kHalfBytes >> 4)), y + (yp + in + h * (RY * 128 >> 4)), idesc,
                       (kParts == 2 && pass < 2) || k > 0);
    }
  }
}
// D (128 x N) (+)= A Y, A 128 x 64 in tensor memory (32 columns; its lo part `lo` columns further), 64 rows of Y, MN-major, the reduction.
// kApart: what has a lo part adds up in 128 columns further on, so that the large sum is truncated a third as often.
template <int DP, int kParts, bool kApart, int RY = kRows>
__device__ __forceinline__ void mma_weigh(uint32_t d_tmem, uint32_t a_tmem, int lo, uint64_t y, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int pass = 0; pass < (kParts == 2 ? 3 : 1); ++pass) {
    const uint32_t ap = a_tmem + (pass == 1 ? lo : 0), yp = pass == 2 ? RY * DP * 2 >> 4 : 0;
    const uint32_t d = d_tmem + (kApart && pass > 0 ? 128 : 0);
    const bool fresh = pass == 0 || (kApart && pass == 1);
#pragma unroll
    for (int k = 0; k < 4; ++k) umma_ts(d, ap + 8 * k, y + (yp + 128 * k), idesc, accumulate || !fresh || k > 0);
  }
}
// 32 columns of such an accumulator, both parts added.
template <bool kApart>
__device__ __forceinline__ void load_sums(uint32_t at, uint32_t (&r)[32]) {
  ptx::tmem_ld_32x32(at, r);
  if constexpr (kApart) {
    uint32_t q[32];
    ptx::tmem_ld_32x32(at + 128, q);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(q[e]));
  } else {
    ptx::tmem_ld_wait();
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return ptx::pack_bf16x2(lo, hi);
  } else {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
}
// What fp16 rounding left over of two values, rounded again.
__device__ __forceinline__ uint32_t pack2_rest(float lo, float hi, uint32_t packed) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&packed));
  return pack2<__half>(lo - h.x, hi - h.y);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // |e| <= 126
// Eight neighbouring results of a row, the first `n` of them (16-byte stores where all are there; dst is then 16-byte aligned).
template <typename Out>
__device__ __forceinline__ void store8(Out* dst, const float (&f)[8], int n, bool wide) {
  if (wide && n >= 8) {
    if constexpr (sizeof(Out) == 4) {
      reinterpret_cast<float4*>(dst)[0] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(dst)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack2<Out>(f[0], f[1]), pack2<Out>(f[2], f[3]), pack2<Out>(f[4], f[5]), pack2<Out>(f[6], f[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) dst[i] = from_f32<Out>(f[i]);
  }
}
// (A polynomial on the FMA pipe for a share of the values made no kernel faster: they wait for one another, not for this pipe.)
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Register split of a block of 12 warps launched with 168 registers a thread: 8 working warps take 208, the 4 others keep 80
// (8 * 208 + 4 * 80 <= 12 * 168).  Executed by every warp of a group of four.
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 208;"); }
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 80;"); }
// The same for a block of 8 warps launched with 128 registers a thread (two blocks a SM): 4 * 184 + 4 * 72 = 8 * 128.
__device__ __forceinline__ void registers_up_4() { asm volatile("setmaxnreg.inc.sync.aligned.u32 184;"); }
__device__ __forceinline__ void registers_down_4() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }

// Called by all threads at a kernel's end: reports a wait that gave up to the host.
__device__ __forceinline__ void report(int* status, volatile int* abort_flag) {
  if (threadIdx.x == 0 && *abort_flag && status) {
    *reinterpret_cast<volatile int*>(status) = 1;
    __threadfence_system();
  }
}

// A wait of a whole warp: all lanes go on, or none (the warp's next step needs them all).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, abort_flag));
}

// Bounded wait of a thread that may not leave with copies or MMAs in flight, whatever else happened.
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!ptx::mbar_try_wait(bar, parity))
    if (clock64() - t0 > ptx::kWaitBudgetCycles) break;
}

// attention_sm100.cu: host helpers
int status_pointer(int** out);
int tile_map(CUtensorMap* map, const Operand& o, int dtype, int D, int heads, int tokens, int clips, int rows = kRows);

}  // namespace attn
}  // namespace d2c

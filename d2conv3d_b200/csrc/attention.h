// Cross attention: what its kernels share (attention_exact.cu: CUDA cores, any type and head width; attention_sm100.cu: tensor
// cores, 16-bit types) and the host side that chooses between them (attention_api.cu).
#pragma once

#include "token_common.cuh"

namespace d2c {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void *q, *k, *v, *g, *o_in;      // g, o_in: gradient of the output and the output (backward)
  void *o, *gq, *gk, *gv;
  float* lse;                            // [B, Hq, Lq]: log2 of the sum of exp2(scores in log2 units); -inf without keys
  float* delta;                          // [B, Hq, Lq]: sum_d grad_o * o
  int* g_exp;                            // [B, Hq, Lq]: grad_o 2^g_exp has its largest element in 2^14 .. 2^15; NULL where operands are bf16
  const void* lengths;
  int lengths_i64;
  int B, Lq, Lk, Hq, Hkv, D;
  float scale;
  long long qs[3], ks[3], vs[3], gs[3];  // batch, token, head
  int splits;                            // shares of the inner loop; > 1: partial results
  float* part;                           // forward [splits][B, Lq, Hq][D]; grad_q the same; grad_k, then grad_v [splits][B, Lk, Hkv][D]
  float* part_lse;                       // forward [splits][B, Lq, Hq]
};

// Valid keys of clip b.
__device__ __forceinline__ int key_length(const Args& a, int b) {
  if (!a.lengths) return a.Lk;
  const long long n = a.lengths_i64 ? reinterpret_cast<const long long*>(a.lengths)[b]
                                    : (long long)reinterpret_cast<const int*>(a.lengths)[b];
  return (int)(n < 0 ? 0 : (n > a.Lk ? a.Lk : n));
}

// Exponent e that brings a largest element to 2^14 .. 2^15 (bits of a float, as largest_sizes writes it; 0: all are zero).
__device__ __forceinline__ int scale_exponent(uint32_t size) {
  const float f = __uint_as_float(size);
  return f > 0.f ? max(-126, min(126, 14 - ilogbf(f))) : 0;
}

// Share [begin, end) of n items, of `splits`.
__device__ __forceinline__ void share(int n, int splits, int s, int& begin, int& end) {
  begin = (int)((long long)n * s / splits);
  end = (int)((long long)n * (s + 1) / splits);
}

// ---- attention_exact.cu
enum { kTile = 64, kFewRows = 4 };
int exact_fwd(int dtype, const Args& a, cudaStream_t st);
int few_fwd(int dtype, const Args& a, cudaStream_t st);          // needs 16-byte rows: see few_fits
int exact_bwd_q(int dtype, const Args& a, cudaStream_t st);
int exact_bwd_kv(int dtype, const Args& a, cudaStream_t st);
int combine(int dtype, const Args& a, cudaStream_t st);          // partial outputs -> o, lse
int delta_rows(int dtype, const Args& a, cudaStream_t st);       // delta, g_exp
int sum_parts(int dtype, const float* part, int splits, long long n, void* out0, void* out1, cudaStream_t st);   // out1: NULL, or a second sum

// ---- tensor cores: operands with positive strides and 16-byte rows, scale > 0
struct Operand {
  const void* p;
  long long s[3];                        // clip, token, head
};
// attention_sm100.cu.  fp32: operands staged by split_rows, in `parts` parts.  bounds [4][B, Hkv]: by largest_sizes, for two parts and for
// the gradients of fp16 tensors
int largest_sizes(int dtype, const Args& a, bool values_only, uint32_t* bounds, cudaStream_t st);
size_t split_bytes(int B, int L, int H, int D, int parts);
int split_rows(const Args& a, int parts, uint32_t* bounds, void* workspace, Operand (&o)[4], cudaStream_t st);   // q, k, v, and g if there is one
int tc_fwd(int dtype, const Args& a, const Operand (&x)[4], int parts, const uint32_t* bounds, cudaStream_t st);
// attention_sm100_bwd.cu
int tc_bwd(int dtype, const Args& a, const Operand (&x)[4], int parts, bool keys, const uint32_t* bounds, cudaStream_t st);

}  // namespace attn
}  // namespace d2c

// Rotary positions with three axes (time, height, width): the channels of a head are cut into one section per axis and a
// rest; pair i of section a turns by the angle p_a * base^(-2 i / n_a), n_a the section's channels, p_a the token's
// position on that axis; the rest stays.  The gradient is the same with the angle's sign changed.
//
// HBM-bound: 2 * sizeof(T) bytes per element.  A block forms the frequencies once, a thread holds the same pairs of every token it
// meets; the angle is formed once per token and used for all heads.  Angles: position times
// frequency in turns, in 64 bits, its whole turns taken off, then sin and cos in 32 bits: at position 100 000 a 32-bit
// product would be off by thousandths of a turn.
// 25920 tokens of 8 heads of 64 in fp32: 21 us (5.1 TB/s).  205440 tokens of 8 heads of 32 in bf16, neighbouring pairs: 36 us (5.8 TB/s);
// with every 16-bit value converted by itself 54.
#include <algorithm>

#include "token_common.cuh"

namespace d2c {
namespace {

struct RotaryArgs {
  const void *x, *positions;
  void* y;
  long long tokens;                  // batch * length
  long long sb, sl, sh;              // strides of x; y is contiguous
  long long pos_batch;               // positions' elements between two batch entries (0: shared)
  int length, heads, dim;
  int n[3];                          // channels of the sections
  int pos_kind;
  int grid_h, grid_w;
  double step[3], first[3];          // grid positions: index * step + first
  double log2_base;
  float sign;
};

// V pairs of a thread: channels u0 .. and v0 .. (halves of a section, which V divides), or 2 V neighbouring channels (which may
// belong to two sections).  The first heads are asked for before the angles are formed.
template <typename T, int V, bool kInterleaved>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 2) rotary_kernel(RotaryArgs a) {
  constexpr int kHeads = 4;                                      // in flight
  __shared__ double freqs[256];                                  // turns per position of every pair
  const int pairs = a.dim / 2, j = threadIdx.x * V;              // first pair of this thread
  int axis[V], u0 = 0, v0 = 0;                                   // 3: the rest, which stays
  auto place = [&](int pair, int& start, int& i) {
    int x = 0;
    start = 0;
    i = pair;
    while (x < 3 && i >= a.n[x] / 2) {
      i -= a.n[x] / 2;
      start += a.n[x];
      ++x;
    }
    return x;
  };
  for (int k = threadIdx.y * blockDim.x + threadIdx.x; k < pairs; k += blockDim.x * blockDim.y) {
    int start, i;
    const int x = place(k, start, i);
    freqs[k] = x < 3 ? exp2(-2.0 * i / a.n[x] * a.log2_base) * 0.15915494309189533577 : 0.0;
  }
  __syncthreads();
  double freq[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    int start, i;
    axis[e] = place(j + e, start, i);
    freq[e] = freqs[j + e];
    if (e == 0) {
      u0 = kInterleaved ? 2 * j : start + i;
      v0 = start + i + (axis[0] < 3 ? a.n[axis[0]] : a.dim - start) / 2;
    }
  }
  const bool turns = axis[0] < 3, all_turn = axis[V - 1] < 3;    // sections come in order
  for (long long tok = (long long)blockIdx.x * blockDim.y + threadIdx.y; tok < a.tokens; tok += (long long)gridDim.x * blockDim.y) {
    const long long b = tok / a.length;
    const int l = (int)(tok - b * a.length);
    const T* x = reinterpret_cast<const T*>(a.x) + b * a.sb + (long long)l * a.sl;
    T* y = reinterpret_cast<T*>(a.y) + tok * a.heads * a.dim;
    float c[V], s[V];
    for (int h0 = 0; h0 < a.heads; h0 += kHeads, x += kHeads * a.sh, y += kHeads * a.dim) {
      constexpr int kW = kInterleaved ? 2 * V : V;
      Vec<T, kW> p[kHeads], q[kInterleaved ? 1 : kHeads];
#pragma unroll
      for (int h = 0; h < kHeads; ++h)
        if (h0 + h < a.heads) {
          p[h] = load_vec<T, kW>(x + h * a.sh + u0);
          if constexpr (!kInterleaved) q[h] = load_vec<T, kW>(x + h * a.sh + v0);
        }
      if (h0 == 0 && turns) {
        double pos[3];
        if (a.pos_kind == D2C_POS_GRID) {
          const int row = l / a.grid_w;
          pos[0] = (row / a.grid_h) * a.step[0] + a.first[0];
          pos[1] = (row % a.grid_h) * a.step[1] + a.first[1];
          pos[2] = (l - row * a.grid_w) * a.step[2] + a.first[2];
        } else {
          const long long at = b * a.pos_batch + (long long)l * 3;
#pragma unroll
          for (int k = 0; k < 3; ++k)
            pos[k] = a.pos_kind == D2C_POS_I32   ? (double)reinterpret_cast<const int*>(a.positions)[at + k]
                     : a.pos_kind == D2C_POS_I64 ? (double)reinterpret_cast<const long long*>(a.positions)[at + k]
                                                 : (double)reinterpret_cast<const float*>(a.positions)[at + k];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const double t = (axis[e] == 0 ? pos[0] : (axis[e] == 1 ? pos[1] : pos[2])) * freq[e];
          sincospif(2.f * (float)(t - rint(t)), &s[e], &c[e]);
          s[e] *= a.sign;
        }
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        if (h0 + h >= a.heads) break;
        if (turns) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if constexpr (kInterleaved && sizeof(T) == 2) {        // a pair is a word
              uint32_t& w = reinterpret_cast<uint32_t*>(&p[h])[e];
              float u, v;
              f2_split(unpack_word<T>(w), u, v);
              const uint32_t r = pack_word<T>(u * c[e] - v * s[e], u * s[e] + v * c[e]);
              if (all_turn || axis[e] < 3) w = r;                  // what stays keeps its bits
            } else if constexpr (!kInterleaved && sizeof(T) == 2 && V % 2 == 0) {
              if (e % 2 == 0) {                                    // two pairs are two words
                uint32_t& wu = reinterpret_cast<uint32_t*>(&p[h])[e / 2];
                uint32_t& wv = reinterpret_cast<uint32_t*>(&q[h])[e / 2];
                float u0, u1, v0, v1;
                f2_split(unpack_word<T>(wu), u0, u1);
                f2_split(unpack_word<T>(wv), v0, v1);
                wu = pack_word<T>(u0 * c[e] - v0 * s[e], u1 * c[e + 1] - v1 * s[e + 1]);
                wv = pack_word<T>(u0 * s[e] + v0 * c[e], u1 * s[e + 1] + v1 * c[e + 1]);
              }
            } else {
              T& ru = kInterleaved ? p[h].v[2 * e] : p[h].v[e];
              T& rv = kInterleaved ? p[h].v[2 * e + 1] : q[kInterleaved ? 0 : h].v[e];
              const float u = to_f32(ru), v = to_f32(rv);
              if (!kInterleaved || all_turn || axis[e] < 3) {
                ru = from_f32<T>(u * c[e] - v * s[e]);
                rv = from_f32<T>(u * s[e] + v * c[e]);
              }
            }
          }
        }
        store_vec<T, kW>(y + h * a.dim + u0, p[h]);
        if constexpr (!kInterleaved) store_vec<T, kW>(y + h * a.dim + v0, q[h]);
      }
    }
  }
}

template <typename T, int V, bool kInterleaved>
int launch(const RotaryArgs& a, cudaStream_t st) {
  int sms = 0;
  if (const int rc = device_sm_count(&sms)) return rc;
  const int px = a.dim / 2 / V, py = std::max(1, 256 / px);      // px <= 256
  const long long blocks = std::min<long long>((a.tokens + py - 1) / py, (long long)sms * 16);
  rotary_kernel<T, V, kInterleaved><<<(unsigned)blocks, dim3(px, py), 0, st>>>(a);
  D2C_LAUNCH_CHECK();
  return D2C_OK;
}

template <typename T>
int run(const d2c_rotary_desc& d, const RotaryArgs& a, cudaStream_t st) {
  // pairs a thread: as many as every section, the strides and the pointers allow, 16 bytes an access at most
  auto fits = [&](int v) {
    const int run = d.interleaved ? 2 * v : v;                   // contiguous channels of one access
    for (int k = 0; k < 3; ++k)
      if (!d.interleaved && (a.n[k] / 2) % v) return false;
    return (a.dim / 2) % v == 0 && a.sb % run == 0 && a.sl % run == 0 && a.sh % run == 0 &&
           run * (int)sizeof(T) <= 16 && aligned_to(a.x, run * sizeof(T)) && aligned_to(a.y, run * sizeof(T));
  };
  if (d.interleaved) {
    if (fits(4)) return launch<T, 4, true>(a, st);
    if (fits(2)) return launch<T, 2, true>(a, st);
    if (fits(1)) return launch<T, 1, true>(a, st);
    return D2C_ERR_ALIGN;
  }
  if (fits(4)) return launch<T, 4, false>(a, st);
  if (fits(2)) return launch<T, 2, false>(a, st);
  return launch<T, 1, false>(a, st);
}

int checked(const d2c_rotary_desc* d) {
  if (!d) return D2C_ERR_NULL;
  if (!token_dtype_ok(d->dtype)) return D2C_ERR_DTYPE;
  if (d->batch < 1 || d->length < 1 || d->heads < 1 || d->dim < 2 || d->dim % 2 || d->dim > 512) return D2C_ERR_SHAPE;
  int sum = 0;
  for (int k = 0; k < 3; ++k) {
    if (d->axis_dims[k] < 0 || d->axis_dims[k] % 2 || d->axis_dims[k] > d->dim) return D2C_ERR_SHAPE;
    sum += d->axis_dims[k];
  }
  if (sum > d->dim || !(d->base > 0)) return D2C_ERR_SHAPE;
  if (d->pos_kind < D2C_POS_GRID || d->pos_kind > D2C_POS_F32) return D2C_ERR_MODE;
  if (d->pos_kind == D2C_POS_GRID) {
    long long n = 1;
    for (int k = 0; k < 3; ++k) {
      if (d->grid[k] < 1) return D2C_ERR_SHAPE;
      n *= d->grid[k];
      if (n > d->length) return D2C_ERR_SHAPE;
    }
    if (n != d->length) return D2C_ERR_SHAPE;
  }
  return D2C_OK;
}

}  // namespace
}  // namespace d2c

extern "C" int d2c_rotary_check(const d2c_rotary_desc* desc) { return d2c::checked(desc); }

extern "C" int d2c_rotary(const d2c_rotary_desc* desc, const void* x, const void* positions, void* y, d2c_stream_t stream) {
  using namespace d2c;
  if (const int rc = take_device_status()) return rc;
  if (const int rc = checked(desc)) return rc;
  if (!x || !y || (desc->pos_kind != D2C_POS_GRID && !positions)) return D2C_ERR_NULL;
  RotaryArgs a{};
  a.x = x; a.positions = positions; a.y = y;
  a.tokens = (long long)desc->batch * desc->length;
  a.sb = desc->stride_batch; a.sl = desc->stride_token; a.sh = desc->stride_head;
  a.pos_batch = desc->pos_batch_stride;
  a.length = desc->length; a.heads = desc->heads; a.dim = desc->dim;
  a.pos_kind = desc->pos_kind;
  a.grid_h = desc->grid[1]; a.grid_w = desc->grid[2];
  for (int k = 0; k < 3; ++k) {
    a.n[k] = desc->axis_dims[k];
    // centres of cells: (index + 1/2) * step - 1/2
    a.step[k] = desc->grid_step[k];
    a.first[k] = 0.5 * desc->grid_step[k] - 0.5;
  }
  a.log2_base = log2(desc->base);
  a.sign = desc->inverse ? -1.f : 1.f;
  cudaStream_t st = (cudaStream_t)stream;
  prof_mark(st, "rotary");
  int rc;
  switch (desc->dtype) {
    case D2C_F32: rc = run<float>(*desc, a, st); break;
    case D2C_F16: rc = run<__half>(*desc, a, st); break;
    default: rc = run<__nv_bfloat16>(*desc, a, st); break;
  }
  prof_mark(st, nullptr);
  return rc;
}

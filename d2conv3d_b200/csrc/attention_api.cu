// Cross attention: entry points, checks, and the choice of kernels.
#include <algorithm>

#include "attention.h"

namespace d2c {
namespace attn {
namespace {

enum class Path { few, exact, tensor };
struct Plan {
  Path path;
  int splits;
  int parts;           // tensor: parts of an operand
};

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Shares of an inner loop of `steps` steps: what costs least in steps, where `slots` blocks run at the same time, a block costs
// `start` steps besides its loop, and joining costs `join` per share.  (A wave that is not full costs as much as a full one: 64
// blocks of 102 steps on 148 SMs take 102 steps whole, 4 * 28.5 in 9 shares.)  At least `fewest` of them.
int shares(long long blocks, int steps, int slots, double start, double join, int fewest) {
  fewest = std::max(1, std::min(fewest, steps));
  const int most = std::min(steps, fewest + 127);
  int best = fewest;
  double least = 0;
  auto look = [&](long long s) {
    if (s < fewest || s > most) return;
    const double cost = (double)((blocks * s + slots - 1) / slots) * (ceil_div(steps, s) + start) + (s > 1 ? start + join * s : 0.0);
    if (least == 0 || cost < least) {
      best = (int)s;
      least = cost;
    }
  };
  look(fewest);
  look(fewest + 1);
  for (int waves = 1; waves <= 16; ++waves) {
    const long long s = (long long)waves * slots / blocks;        // the most that these waves hold
    look(std::min<long long>(s, most));
    if (s >= most) break;
  }
  return best;
}

long long q_rows(const d2c_attention_desc& d) { return (long long)d.batch * d.queries * d.q_heads; }
long long kv_rows(const d2c_attention_desc& d) { return (long long)d.batch * d.keys * d.kv_heads; }

// What writing and reading one share's fp32 results takes, in steps of about 1.5 us, at 5 TB/s.
double join_steps(long long rows, int dim) { return 8.0 * rows * dim / 5e6 / 1.5; }

// 16-byte pieces of every row
bool rows_fit(const d2c_attention_desc& d, const int64_t (&s)[3]) {
  const int v = 16 / (int)token_dtype_size(d.dtype);
  return s[0] % v == 0 && s[1] % v == 0 && s[2] % v == 0;
}
bool few_fits(const d2c_attention_desc& d) {
  const int v = 16 / (int)token_dtype_size(d.dtype);
  return d.dim % v == 0 && rows_fit(d, d.q_stride) && rows_fit(d, d.k_stride) && rows_fit(d, d.v_stride);
}

// What the tensor-core kernels' tensor maps take: 16-byte rows, no dimension that repeats its elements, strides under 2^40 bytes.
bool tensor_rows(const d2c_attention_desc& d, const int64_t (&s)[3], int tokens, int heads) {
  const int n[3] = {d.batch, tokens, heads};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 || s[i] >= 1LL << 39)) return false;
  return true;
}

// Parts of the tensor-core kernels' operands; 0 where they do not apply.  fp32 goes by the math mode: two parts for parity, one, or CUDA
// cores.  The running maximum is that of the raw
// scores, so the scale has to be above zero.
int tensor_parts(const d2c_attention_desc& d, int mode, bool aligned, bool backward) {
  if (!aligned || !(d.scale > 1e-30f)) return 0;
  if (d.dtype == D2C_F32) {
    if (mode == D2C_MATH_FP32) return 0;
    if (mode == D2C_MATH_BF16) return 1;
    // staging and joining are launches of their own: 2 x 1015 x 179, 4 heads of 32 channels, trains in 84 us on CUDA cores and in 113
    // in two parts; 2 x 400 x 400, 4 heads of 64, in 118 and 107
    const double products = (double)d.batch * d.q_heads * d.queries * d.keys * d.dim;
    return mode == D2C_MATH_AUTO && products < (double)(1 << 26) ? 0 : 2;
  }
  return d.dim % 8 == 0 && tensor_rows(d, d.q_stride, d.queries, d.q_heads) && tensor_rows(d, d.k_stride, d.keys, d.kv_heads) &&
         tensor_rows(d, d.v_stride, d.keys, d.kv_heads) && (!backward || tensor_rows(d, d.g_stride, d.queries, d.q_heads));
}

// The tensor cores add into their accumulator with truncation: a chain of n accumulating products loses about n * 2^-27 of the
// result.  With two parts (24 products a tile, 8 of them into the sum of the hi parts where those of lo parts have one of their own) a
// share ends after 8 tiles, or 3, 0.5e-6, and the shares are added in fp32 -- unless their results would take more than 2 GB.
int fewest_shares(int parts, bool apart, int steps, long long rows, int dim) {
  if (parts != 2) return 1;
  return (int)std::min<long long>(ceil_div(steps, apart ? 8 : 3), std::max(1LL, (2LL << 30) / (4 * rows * dim)));
}

// `slots` blocks at a time on the tensor cores.
Plan make_plan(const d2c_attention_desc& d, int parts, int rows_x, int heads_x, long long rows_out, int per_block, long long steps_rows, int slots,
               int sms, bool apart) {
  const bool tensor = parts > 0;
  const int tile = tensor ? 128 : kTile;
  const int steps = ceil_div(steps_rows, tile);
  return {tensor ? Path::tensor : Path::exact,
          shares((long long)ceil_div(rows_x, tile * per_block) * heads_x * d.batch, steps, tensor ? slots : 2 * sms, tensor ? 3.0 : 1.0,
                 join_steps(rows_out, d.dim), fewest_shares(parts, apart, steps, rows_out, d.dim)),
          parts};
}

// few: up to 16 query rows on a head's keys; every four rows read the keys once, from L2 after the first.
Plan plan_fwd(const d2c_attention_desc& d, int mode, bool aligned, int sms) {
  const long long rows = (long long)d.q_heads / d.kv_heads * d.queries;
  if (rows <= 16 && few_fits(d) && aligned) {
    const long long blocks = (long long)ceil_div(rows, kFewRows) * d.kv_heads * d.batch;
    return {Path::few, std::max(1, std::min({ceil_div(2LL * sms, blocks), ceil_div(d.keys, 256), 128})), 0};
  }
  const int parts = tensor_parts(d, mode, aligned, false);
  const bool two_tiles = parts > 0 && !(parts == 2 && d.dim > 64);
  return make_plan(d, parts, d.queries, d.q_heads, q_rows(d), two_tiles ? 2 : 1, d.keys, sms, sms, true);
}
// A gradient kernel's block has a tile of one side and runs over the other.
Plan plan_bwd(const d2c_attention_desc& d, int mode, bool keys, bool aligned, int sms) {
  const int parts = tensor_parts(d, mode, aligned, true);
  const int slots = parts == 1 && d.dim <= 64 ? 2 * sms : sms;
  if (!keys) return make_plan(d, parts, d.queries, d.q_heads, q_rows(d), 1, d.keys, slots, sms, d.dim <= 64);
  const int tile = parts ? 128 : kTile;
  return make_plan(d, parts, d.keys, d.kv_heads, 2 * kv_rows(d), 1, (long long)ceil_div(d.queries, tile) * tile * (d.q_heads / d.kv_heads), slots, sms, d.dim <= 64);
}

size_t bound_bytes(const d2c_attention_desc& d) { return align_up(sizeof(uint32_t) * 4 * d.batch * d.kv_heads, 256); }
size_t fwd_bytes(const d2c_attention_desc& d, const Plan& p) {
  size_t n = 0;
  if (p.path == Path::tensor && d.dtype == D2C_F32)
    n += bound_bytes(d) + split_bytes(d.batch, d.queries, d.q_heads, d.dim, p.parts) + 2 * split_bytes(d.batch, d.keys, d.kv_heads, d.dim, p.parts);
  if (p.splits > 1)
    n += align_up(sizeof(float) * p.splits * q_rows(d) * d.dim, 256) + align_up(sizeof(float) * p.splits * q_rows(d), 256);
  return n;
}
size_t fwd_workspace(const d2c_attention_desc& d, int mode, int sms) {
  size_t n = 0;                       // whatever the pointers' alignment, and so the plan, turns out to be
  for (int al = 0; al < 2; ++al) n = std::max(n, fwd_bytes(d, plan_fwd(d, mode, al, sms)));
  return n;
}

size_t delta_bytes(const d2c_attention_desc& d) { return align_up(sizeof(float) * q_rows(d), 256); }
// Rows' exponents, where operands are fp16.
bool scaled_rows(const d2c_attention_desc& d, int parts) { return parts == 2 || (parts && d.dtype == D2C_F16); }
size_t exponent_bytes(const d2c_attention_desc& d, int parts) { return scaled_rows(d, parts) ? align_up(sizeof(int) * q_rows(d), 256) : 0; }
size_t staged_bytes(const d2c_attention_desc& d, int parts) {
  if (d.dtype != D2C_F32 || !parts) return 0;
  return 2 * split_bytes(d.batch, d.queries, d.q_heads, d.dim, parts) + 2 * split_bytes(d.batch, d.keys, d.kv_heads, d.dim, parts);
}
size_t bwd_bytes(const d2c_attention_desc& d, const Plan& pq, const Plan& pk) {
  size_t part = 0;                    // one gradient kernel's shares at a time
  if (pq.splits > 1) part = std::max<size_t>(part, sizeof(float) * pq.splits * q_rows(d) * d.dim);
  if (pk.splits > 1) part = std::max<size_t>(part, sizeof(float) * 2 * pk.splits * kv_rows(d) * d.dim);
  return delta_bytes(d) + exponent_bytes(d, pq.parts) + bound_bytes(d) + staged_bytes(d, pq.parts) + align_up(part, 256);
}
size_t bwd_workspace(const d2c_attention_desc& d, int mode, int sms) {
  size_t n = 0;
  for (int al = 0; al < 2; ++al) n = std::max(n, bwd_bytes(d, plan_bwd(d, mode, false, al, sms), plan_bwd(d, mode, true, al, sms)));
  return n;
}

int checked(const d2c_attention_desc* d) {
  if (!d) return D2C_ERR_NULL;
  if (!token_dtype_ok(d->dtype)) return D2C_ERR_DTYPE;
  if (d->batch < 1 || d->queries < 1 || d->keys < 1 || d->q_heads < 1 || d->kv_heads < 1 || d->dim < 1 || d->dim > 128)
    return D2C_ERR_SHAPE;
  if (d->q_heads % d->kv_heads) return D2C_ERR_GROUPS;
  // grids, row indexes and the kernels' 32-bit steps over tokens
  if (q_rows(*d) > 0x7fffffffLL || kv_rows(*d) > 0x7fffffffLL || d->queries > 1 << 30 || d->keys > 1 << 30) return D2C_ERR_TOO_LARGE;
  return D2C_OK;
}

Args make_args(const d2c_attention_desc& d, const void* q, const void* k, const void* v, const void* lengths) {
  Args a{};
  a.q = q; a.k = k; a.v = v;
  a.lengths = lengths; a.lengths_i64 = d.lengths_i64;
  a.B = d.batch; a.Lq = d.queries; a.Lk = d.keys; a.Hq = d.q_heads; a.Hkv = d.kv_heads; a.D = d.dim;
  a.scale = d.scale;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = d.q_stride[i]; a.ks[i] = d.k_stride[i]; a.vs[i] = d.v_stride[i]; a.gs[i] = d.g_stride[i];
  }
  a.splits = 1;
  return a;
}

bool ws_ok(const void* ws, size_t have, size_t need) { return need == 0 || (ws && aligned_to(ws, 256) && have >= need); }

// The tensors themselves as operands (16-bit types).
void own_operands(const Args& a, Operand (&o)[4]) {
  const void* p[4] = {a.q, a.k, a.v, a.g};
  const long long* s[4] = {a.qs, a.ks, a.vs, a.gs};
  for (int i = 0; i < 4; ++i) o[i] = {p[i], {s[i][0], s[i][1], s[i][2]}};
}

int run_fwd(const d2c_attention_desc& d, Args a, int mode, void* workspace, int sms, cudaStream_t st) {
  const Plan p = plan_fwd(d, mode, aligned_to(a.q, 16) && aligned_to(a.k, 16) && aligned_to(a.v, 16) && aligned_to(a.o, 16), sms);
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  a.splits = p.splits;
  if (p.splits > 1) {
    a.part = reinterpret_cast<float*>(ws);
    ws += align_up(sizeof(float) * p.splits * q_rows(d) * d.dim, 256);
    a.part_lse = reinterpret_cast<float*>(ws);
    ws += align_up(sizeof(float) * p.splits * q_rows(d), 256);
  }
  int rc;
  if (p.path == Path::tensor) {
    Operand x[4];
    own_operands(a, x);
    uint32_t* bounds = reinterpret_cast<uint32_t*>(ws);
    if (d.dtype == D2C_F32) {
      if (p.parts == 2 && (rc = largest_sizes(d.dtype, a, false, bounds, st))) return rc;
      if ((rc = split_rows(a, p.parts, bounds, ws + bound_bytes(d), x, st))) return rc;
    }
    rc = tc_fwd(d.dtype, a, x, p.parts, bounds, st);
  } else {
    rc = p.path == Path::few ? few_fwd(d.dtype, a, st) : exact_fwd(d.dtype, a, st);
  }
  if (rc || p.splits == 1) return rc;
  return combine(d.dtype, a, st);
}

int run_bwd(const d2c_attention_desc& d, Args a, int mode, void* workspace, int sms, cudaStream_t st) {
  const bool aligned = aligned_to(a.q, 16) && aligned_to(a.k, 16) && aligned_to(a.v, 16) && aligned_to(a.g, 16) &&
                       aligned_to(a.gq, 16) && aligned_to(a.gk, 16) && aligned_to(a.gv, 16);
  const Plan pk = plan_bwd(d, mode, true, aligned, sms), pq = plan_bwd(d, mode, false, aligned, sms);
  const bool tensor = pk.path == Path::tensor;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  a.delta = reinterpret_cast<float*>(ws);
  ws += delta_bytes(d);
  if (scaled_rows(d, pk.parts)) {
    a.g_exp = reinterpret_cast<int*>(ws);
    ws += exponent_bytes(d, pk.parts);
  }
  uint32_t* bounds = reinterpret_cast<uint32_t*>(ws);
  ws += bound_bytes(d);
  Operand x[4];
  own_operands(a, x);
  int rc;
  if ((rc = delta_rows(d.dtype, a, st))) return rc;
  if (scaled_rows(d, pk.parts) && (rc = largest_sizes(d.dtype, a, d.dtype == D2C_F16, bounds, st))) return rc;
  if (tensor && d.dtype == D2C_F32) {
    if ((rc = split_rows(a, pk.parts, bounds, ws, x, st))) return rc;
    ws += staged_bytes(d, pk.parts);
  }
  a.part = reinterpret_cast<float*>(ws);
  a.splits = pk.splits;
  if ((rc = tensor ? tc_bwd(d.dtype, a, x, pk.parts, true, bounds, st) : exact_bwd_kv(d.dtype, a, st))) return rc;
  if (a.splits > 1) {
    if ((rc = sum_parts(d.dtype, a.part, a.splits, kv_rows(d) * d.dim, a.gk, a.gv, st))) return rc;
  }
  a.splits = pq.splits;
  if ((rc = tensor ? tc_bwd(d.dtype, a, x, pq.parts, false, bounds, st) : exact_bwd_q(d.dtype, a, st))) return rc;
  if (a.splits > 1) return sum_parts(d.dtype, a.part, a.splits, q_rows(d) * d.dim, a.gq, nullptr, st);
  return D2C_OK;
}

}  // namespace
}  // namespace attn
}  // namespace d2c

extern "C" {

int d2c_attention_check(const d2c_attention_desc* desc) { return d2c::attn::checked(desc); }

size_t d2c_attention_fwd_workspace_bytes(const d2c_attention_desc* desc) {
  using namespace d2c;
  int sms = 0;
  if (attn::checked(desc) || device_sm_count(&sms)) return 0;
  return attn::fwd_workspace(*desc, d2c_get_math_mode(), sms);
}

int d2c_attention_fwd(const d2c_attention_desc* desc, const void* q, const void* k, const void* v, const void* key_lengths,
                      void* o, void* lse, void* workspace, size_t workspace_bytes, d2c_stream_t stream) {
  using namespace d2c;
  if (const int rc = take_device_status()) return rc;
  if (const int rc = attn::checked(desc)) return rc;
  if (!q || !k || !v || !o) return D2C_ERR_NULL;
  int sms = 0;
  if (const int rc = device_sm_count(&sms)) return rc;
  const int mode = d2c_get_math_mode();
  if (!attn::ws_ok(workspace, workspace_bytes, attn::fwd_workspace(*desc, mode, sms))) return D2C_ERR_WORKSPACE;
  attn::Args a = attn::make_args(*desc, q, k, v, key_lengths);
  a.o = o; a.lse = reinterpret_cast<float*>(lse);
  prof_mark((cudaStream_t)stream, "attention");
  const int rc = attn::run_fwd(*desc, a, mode, workspace, sms, (cudaStream_t)stream);
  prof_mark((cudaStream_t)stream, nullptr);
  return rc;
}

size_t d2c_attention_bwd_workspace_bytes(const d2c_attention_desc* desc) {
  using namespace d2c;
  int sms = 0;
  if (attn::checked(desc) || device_sm_count(&sms)) return 0;
  return attn::bwd_workspace(*desc, d2c_get_math_mode(), sms);
}

int d2c_attention_bwd(const d2c_attention_desc* desc, const void* grad_o, const void* q, const void* k, const void* v,
                      const void* key_lengths, const void* o, const void* lse, void* grad_q, void* grad_k, void* grad_v,
                      void* workspace, size_t workspace_bytes, d2c_stream_t stream) {
  using namespace d2c;
  if (const int rc = take_device_status()) return rc;
  if (const int rc = attn::checked(desc)) return rc;
  if (!grad_o || !q || !k || !v || !o || !lse || !grad_q || !grad_k || !grad_v) return D2C_ERR_NULL;
  int sms = 0;
  if (const int rc = device_sm_count(&sms)) return rc;
  const int mode = d2c_get_math_mode();
  if (!attn::ws_ok(workspace, workspace_bytes, attn::bwd_workspace(*desc, mode, sms))) return D2C_ERR_WORKSPACE;
  attn::Args a = attn::make_args(*desc, q, k, v, key_lengths);
  a.g = grad_o; a.o_in = o; a.lse = const_cast<float*>(reinterpret_cast<const float*>(lse));
  a.gq = grad_q; a.gk = grad_k; a.gv = grad_v;
  prof_mark((cudaStream_t)stream, "attention_bwd");
  const int rc = attn::run_bwd(*desc, a, mode, workspace, sms, (cudaStream_t)stream);
  prof_mark((cudaStream_t)stream, nullptr);
  return rc;
}

}  // extern "C"

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
};

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Shares of an inner loop of `steps` steps: what costs least in steps, where `slots` blocks run at the same time, a block costs
// `start` steps besides its loop, and joining costs `join` per share.  (A wave that is not full costs as much as a full one: 64
// blocks of 102 steps on 148 SMs take 102 steps whole, 4 * 28.5 in 9 shares.)
int shares(long long blocks, int steps, int slots, double start, double join) {
  int best = 1;
  double least = 0;
  for (int s = 1; s <= std::min(steps, 128); ++s) {
    const long long waves = (blocks * s + slots - 1) / slots;
    const double cost = waves * (ceil_div(steps, s) + start) + (s > 1 ? start + join * s : 0.0);
    if (s == 1 || cost < least) { best = s; least = cost; }
    if (s > 1 && waves > 16) break;
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

// What the tensor-core kernels' tensor maps take: 16-bit types, 16-byte rows, no dimension that repeats its elements, strides under
// 2^40 bytes; and, for the running maximum to be that of the raw scores, a scale above zero.
bool tensor_rows(const d2c_attention_desc& d, const int64_t (&s)[3], int tokens, int heads) {
  const int n[3] = {d.batch, tokens, heads};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 || s[i] >= 1LL << 39)) return false;
  return true;
}
bool tensor_fits(const d2c_attention_desc& d) {
  if (d.dtype == D2C_F32 || d.dim % 8 || !(d.scale > 1e-30f)) return false;
  return tensor_rows(d, d.q_stride, d.queries, d.q_heads) && tensor_rows(d, d.k_stride, d.keys, d.kv_heads) &&
         tensor_rows(d, d.v_stride, d.keys, d.kv_heads);
}

// few: up to 16 query rows on a head's keys; every four rows read the keys once, from L2 after the first.
Plan plan_fwd(const d2c_attention_desc& d, bool aligned, int sms) {
  Plan p{Path::exact, 1};
  const long long rows = (long long)d.q_heads / d.kv_heads * d.queries;
  if (rows <= 16 && few_fits(d) && aligned) {
    p.path = Path::few;
    const long long blocks = (long long)ceil_div(rows, kFewRows) * d.kv_heads * d.batch;
    p.splits = std::max(1, std::min({ceil_div(4LL * sms, blocks), ceil_div(d.keys, 128), 128}));
  } else if (aligned && tensor_fits(d)) {
    p.path = Path::tensor;
    p.splits = shares((long long)ceil_div(d.queries, 256) * d.q_heads * d.batch, ceil_div(d.keys, 128), sms, 3.0, join_steps(q_rows(d), d.dim));
  } else {
    p.splits = shares((long long)ceil_div(d.queries, kTile) * d.q_heads * d.batch, ceil_div(d.keys, kTile), 2 * sms, 1.0, join_steps(q_rows(d), d.dim));
  }
  return p;
}
// A gradient kernel's block has a tile of one side and runs over the other.
Plan plan_bwd(const d2c_attention_desc& d, bool keys, bool aligned, int sms) {
  Plan p{Path::exact, 1};
  int tile = kTile;
  if (aligned && tensor_fits(d) && tensor_rows(d, d.g_stride, d.queries, d.q_heads)) {
    p.path = Path::tensor;
    tile = 128;
  }
  const int q = ceil_div(d.queries, tile), k = ceil_div(d.keys, tile);
  const int slots = p.path == Path::tensor ? sms : 2 * sms;
  const double start = p.path == Path::tensor ? 3.0 : 1.0;
  p.splits = keys ? shares((long long)k * d.kv_heads * d.batch, q * (d.q_heads / d.kv_heads), slots, start, join_steps(2 * kv_rows(d), d.dim))
                  : shares((long long)q * d.q_heads * d.batch, k, slots, start, join_steps(q_rows(d), d.dim));
  return p;
}

size_t fwd_bytes(const d2c_attention_desc& d, const Plan& p) {
  if (p.splits == 1) return 0;
  return align_up(sizeof(float) * p.splits * q_rows(d) * d.dim, 256) + align_up(sizeof(float) * p.splits * q_rows(d), 256);
}
size_t bwd_part_bytes(const d2c_attention_desc& d, int sms) {
  size_t most = 0;                    // whatever the pointers' alignment, and so the plan, turns out to be
  for (int al = 0; al < 2; ++al) {
    const int sq = plan_bwd(d, false, al, sms).splits, skv = plan_bwd(d, true, al, sms).splits;
    if (sq > 1) most = std::max<size_t>(most, sizeof(float) * sq * q_rows(d) * d.dim);
    if (skv > 1) most = std::max<size_t>(most, sizeof(float) * 2 * skv * kv_rows(d) * d.dim);
  }
  return align_up(most, 256);
}
size_t delta_bytes(const d2c_attention_desc& d) { return align_up(sizeof(float) * q_rows(d), 256); }
size_t bound_bytes(const d2c_attention_desc& d) { return align_up(sizeof(uint32_t) * 2 * d.batch * d.kv_heads, 256); }

int checked(const d2c_attention_desc* d) {
  if (!d) return D2C_ERR_NULL;
  if (!token_dtype_ok(d->dtype)) return D2C_ERR_DTYPE;
  if (d->batch < 1 || d->queries < 1 || d->keys < 1 || d->q_heads < 1 || d->kv_heads < 1 || d->dim < 1 || d->dim > 128)
    return D2C_ERR_SHAPE;
  if (d->q_heads % d->kv_heads) return D2C_ERR_GROUPS;
  // grids and row indexes of the kernels
  if (q_rows(*d) > 0x7fffffffLL || kv_rows(*d) > 0x7fffffffLL || (long long)d->batch * d->q_heads > 65535) return D2C_ERR_TOO_LARGE;
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

int run_fwd(const d2c_attention_desc& d, Args a, void* workspace, int sms, cudaStream_t st) {
  const Plan p = plan_fwd(d, aligned_to(a.q, 16) && aligned_to(a.k, 16) && aligned_to(a.v, 16) && aligned_to(a.o, 16), sms);
  a.splits = p.splits;
  if (p.splits > 1) {
    a.part = reinterpret_cast<float*>(workspace);
    a.part_lse = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(workspace) +
                                          align_up(sizeof(float) * p.splits * q_rows(d) * d.dim, 256));
  }
  const int rc = p.path == Path::few      ? few_fwd(d.dtype, a, st)
                 : p.path == Path::tensor ? tc_fwd(d.dtype, a, st)
                                          : exact_fwd(d.dtype, a, st);
  if (rc || p.splits == 1) return rc;
  return combine(d.dtype, a, st);
}

int run_bwd(const d2c_attention_desc& d, Args a, void* workspace, int sms, cudaStream_t st) {
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  a.delta = reinterpret_cast<float*>(ws);
  uint32_t* bounds = reinterpret_cast<uint32_t*>(ws + delta_bytes(d));
  a.part = reinterpret_cast<float*>(ws + delta_bytes(d) + bound_bytes(d));
  const bool aligned = aligned_to(a.q, 16) && aligned_to(a.k, 16) && aligned_to(a.v, 16) && aligned_to(a.g, 16) &&
                       aligned_to(a.gq, 16) && aligned_to(a.gk, 16) && aligned_to(a.gv, 16);
  int rc = delta_rows(d.dtype, a, st);
  if (rc) return rc;
  const Plan pk = plan_bwd(d, true, aligned, sms), pq = plan_bwd(d, false, aligned, sms);
  const bool tensor = pk.path == Path::tensor;
  if (tensor && d.dtype == D2C_F16 && (rc = tc_bounds(a, bounds, st))) return rc;
  a.splits = pk.splits;
  if ((rc = tensor ? tc_bwd(d.dtype, a, true, bounds, st) : exact_bwd_kv(d.dtype, a, st))) return rc;
  if (a.splits > 1) {
    const long long n = kv_rows(d) * d.dim;
    if ((rc = sum_parts(d.dtype, a.part, a.splits, n, a.gk, st))) return rc;
    if ((rc = sum_parts(d.dtype, a.part + a.splits * n, a.splits, n, a.gv, st))) return rc;
  }
  a.splits = pq.splits;
  if ((rc = tensor ? tc_bwd(d.dtype, a, false, bounds, st) : exact_bwd_q(d.dtype, a, st))) return rc;
  if (a.splits > 1) return sum_parts(d.dtype, a.part, a.splits, q_rows(d) * d.dim, a.gq, st);
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
  size_t n = 0;                       // whatever the pointers' alignment, and so the plan, turns out to be
  for (int al = 0; al < 2; ++al) n = std::max(n, attn::fwd_bytes(*desc, attn::plan_fwd(*desc, al, sms)));
  return n;
}

int d2c_attention_fwd(const d2c_attention_desc* desc, const void* q, const void* k, const void* v, const void* key_lengths,
                      void* o, void* lse, void* workspace, size_t workspace_bytes, d2c_stream_t stream) {
  using namespace d2c;
  if (const int rc = take_device_status()) return rc;
  if (const int rc = attn::checked(desc)) return rc;
  if (!q || !k || !v || !o) return D2C_ERR_NULL;
  if (!attn::ws_ok(workspace, workspace_bytes, d2c_attention_fwd_workspace_bytes(desc))) return D2C_ERR_WORKSPACE;
  int sms = 0;
  if (const int rc = device_sm_count(&sms)) return rc;
  attn::Args a = attn::make_args(*desc, q, k, v, key_lengths);
  a.o = o; a.lse = reinterpret_cast<float*>(lse);
  prof_mark((cudaStream_t)stream, "attention");
  const int rc = attn::run_fwd(*desc, a, workspace, sms, (cudaStream_t)stream);
  prof_mark((cudaStream_t)stream, nullptr);
  return rc;
}

size_t d2c_attention_bwd_workspace_bytes(const d2c_attention_desc* desc) {
  using namespace d2c;
  int sms = 0;
  if (attn::checked(desc) || device_sm_count(&sms)) return 0;
  return attn::delta_bytes(*desc) + attn::bound_bytes(*desc) + attn::bwd_part_bytes(*desc, sms);
}

int d2c_attention_bwd(const d2c_attention_desc* desc, const void* grad_o, const void* q, const void* k, const void* v,
                      const void* key_lengths, const void* o, const void* lse, void* grad_q, void* grad_k, void* grad_v,
                      void* workspace, size_t workspace_bytes, d2c_stream_t stream) {
  using namespace d2c;
  if (const int rc = take_device_status()) return rc;
  if (const int rc = attn::checked(desc)) return rc;
  if (!grad_o || !q || !k || !v || !o || !lse || !grad_q || !grad_k || !grad_v) return D2C_ERR_NULL;
  if (!attn::ws_ok(workspace, workspace_bytes, d2c_attention_bwd_workspace_bytes(desc))) return D2C_ERR_WORKSPACE;
  int sms = 0;
  if (const int rc = device_sm_count(&sms)) return rc;
  attn::Args a = attn::make_args(*desc, q, k, v, key_lengths);
  a.g = grad_o; a.o_in = o; a.lse = const_cast<float*>(reinterpret_cast<const float*>(lse));
  a.gq = grad_q; a.gk = grad_k; a.gv = grad_v;
  prof_mark((cudaStream_t)stream, "attention_bwd");
  const int rc = attn::run_bwd(*desc, a, workspace, sms, (cudaStream_t)stream);
  prof_mark((cudaStream_t)stream, nullptr);
  return rc;
}

}  // extern "C"

// Logits of token policies: the rules that shape them and their gradient, neglogp and entropy of an action, the clipped
// objective with its gradient.  Semantics in include/ppo_xp.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "ops_common.h"

namespace {

using namespace ppoxp_ops;

constexpr float kLog2e = 1.44269504088896340736f;

// ---- rules ----------------------------------------------------------------------------------------------------------------

struct ShapeArgs {
  const void *in;        // logits, or the gradient of the shaped logits
  const void *logits;    // backward: the logits, for the sign of tokens that were seen
  void *out;
  int64_t in_stride, logits_stride, out_stride;
  unsigned vocab, chunks;
  ppo_xp_logit_rules r;
};

constexpr int kShapeVecs = 4;                        // 8-element vectors a thread
constexpr unsigned kShapeChunk = 256 * 8 * kShapeVecs;
constexpr unsigned kPromptOnly = 0x80000000u;        // table word: occurrences in the generated part, this bit: in the rest

// One workgroup shapes one chunk of one row's vocabulary.  With a history it counts the row's tokens that fall into its chunk
// in LDS first (integer atomics: the order does not matter), while its logits are already on their way into registers.
template <typename T, bool HIST, bool BACKWARD>
__global__ __launch_bounds__(256) void shape_logits_kernel(ShapeArgs a) {
  __shared__ __attribute__((aligned(16))) unsigned table[HIST ? kShapeChunk : 4];
  const ppo_xp_logit_rules &r = a.r;
  const size_t row = blockIdx.x / a.chunks;
  const unsigned c0 = (blockIdx.x % a.chunks) * kShapeChunk, tid = threadIdx.x;
  const T *in = (const T *)a.in + (int64_t)row * a.in_stride;
  T *out = (T *)a.out + (int64_t)row * a.out_stride;

  Raw8<T> raw[kShapeVecs];
#pragma unroll
  for (int k = 0; k < kShapeVecs; ++k) {
    const unsigned e = c0 + (k * 256 + tid) * 8;
    if (e < a.vocab) load8(raw[k], in + e, (long)(a.vocab - e), 0.f);
  }
  if (HIST) {
    for (unsigned i = tid * 4; i < kShapeChunk; i += 1024) *(u32x4 *)(table + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    const int64_t h = r.hist_row ? r.hist_row[row] : (int64_t)row;
    if (h >= 0 && h < r.hist_rows) {
      const int64_t end = r.hist_end ? min((int64_t)r.hist_end[row], r.hist_len) : r.hist_len;
      const int64_t begin = r.hist_begin ? max((int64_t)r.hist_begin[row], (int64_t)0) : 0;
      const int64_t gen = r.gen_begin ? (int64_t)r.gen_begin[row] : begin;
      const int64_t base = h * r.hist_row_stride;
      for (int64_t k = begin + tid; k < end; k += 256) {
        const int64_t at = base + k * r.hist_tok_stride;
        const int64_t tok = r.history_bits == 64 ? ((const int64_t *)r.history)[at] : (int64_t)((const int32_t *)r.history)[at];
        const int64_t slot = tok - c0;
        if (slot < 0 || slot >= kShapeChunk || tok >= a.vocab) continue;
        if (k >= gen) atomicAdd(&table[slot], 1u);
        else atomicOr(&table[slot], kPromptOnly);
      }
    }
    __syncthreads();
  }
  const float rep = r.repetition_rows ? r.repetition_rows[row] : r.repetition;
  const float pres = r.presence_rows ? r.presence_rows[row] : r.presence;
  const float freq = r.frequency_rows ? r.frequency_rows[row] : r.frequency;
  const float inv_t = 1.f / (r.temperature_rows ? r.temperature_rows[row] : r.temperature);
  const float *bias = r.bias ? r.bias + (int64_t)row * r.bias_stride : nullptr;
  const uint8_t *mask = nullptr;
  if (r.mask_kind != PPO_XP_MASK_NONE) {
    const int64_t m = r.mask_row ? r.mask_row[row] : (r.mask_stride == 0 ? 0 : (int64_t)row);
    if (m >= 0 && m < r.mask_rows) mask = (const uint8_t *)r.mask + m * r.mask_stride * (r.mask_kind == PPO_XP_MASK_BITS ? 4 : 1);
  }
#pragma unroll
  for (int k = 0; k < kShapeVecs; ++k) {
    const unsigned e = c0 + (k * 256 + tid) * 8;
    if (e >= a.vocab) break;
    const int n = (int)min(8u, a.vocab - e);
    unsigned allowed = 0xffu;
    if (mask) {
      if (r.mask_kind == PPO_XP_MASK_BITS) allowed = mask[e / 8];
      else {
        allowed = 0;
        for (int i = 0; i < n; ++i) allowed |= (mask[e + i] ? 1u : 0u) << i;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x = raw[k].get(i);
      unsigned c = 0;
      if (HIST) c = table[e - c0 + i];
      if (BACKWARD) {
        x *= inv_t;
        if (HIST && c && i < n) x = (float)((const T *)a.logits)[(int64_t)row * a.logits_stride + e + i] > 0.f ? x / rep : x * rep;
        if (!((allowed >> i) & 1)) x = 0.f;
      } else {
        if (HIST && c) {
          x = x > 0.f ? x / rep : x * rep;
          const unsigned cnt = c & ~kPromptOnly;
          if (cnt) x -= freq * (float)cnt + pres;
        }
        if (bias && i < n) x += bias[e + i];
        x *= inv_t;
        if (!((allowed >> i) & 1)) x = -__builtin_inff();
      }
      raw[k].set(i, x);
    }
    store8(raw[k], out + e, n);
  }
}

// ---- softmax statistics and the objective ---------------------------------------------------------------------------------

struct PolicyArgs {
  const void *logits;
  int64_t stride;
  const int64_t *actions;
  float *neglogps, *entropies;
  unsigned vocab;
  size_t rows;
  // the objective only
  const float *old_values, *old_neglogps, *returns, *advantages, *values;
  float clip, ent_coef, vf_coef, inv_denom;
  void *dlogits;
  int64_t dstride;
  float *dvalues;
  double *partials;      // [rows][5]: policy, value, entropy, kl, clipped
};

// m = max l, s = sum e^(l-m), t = sum e^(l-m) (l-m)
struct Softmax { float m, s, t; };

__device__ __forceinline__ float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }   // d <= 0
// l - m, kept finite: e^-150 is 0 in 32 bits, and 0 * -150 is 0 where 0 * -inf is not
__device__ __forceinline__ float below(float l, float m) { return __builtin_fmaxf(l - m, -150.f); }

// Brings (s, t) from maximum `m` to the larger or equal `to`.
__device__ __forceinline__ void rebase(float m, float to, float &s, float &t) {
  if (s == 0.f) return;
  const float d = below(m, to), f = exp_neg(d);
  t = (t + s * d) * f;
  s *= f;
}

// What one row's statistics mean for its action.
struct RowTerms {
  bool padding, dead;    // dead: -inf throughout | NaN rows have nan set
  bool nan;
  float nlp, ent, ln_s, rs, t;
};

__device__ __forceinline__ RowTerms row_terms(const Softmax &w, int64_t action, unsigned vocab, float l_a) {
  RowTerms o{};
  o.padding = action == -1;
  if (o.padding) return o;
  o.nan = !(w.m < __builtin_inff()) || action < 0 || action >= (int64_t)vocab;
  if (o.nan) { o.nlp = o.ent = __builtin_nanf(""); return o; }
  o.dead = w.m == -__builtin_inff();
  if (o.dead) { o.nlp = __builtin_inff(); return o; }
  o.ln_s = logf(w.s);
  o.rs = 1.f / w.s;
  o.t = w.t;
  o.nlp = o.ln_s - (l_a - w.m);
  o.ent = o.ln_s - w.t * o.rs;
  return o;
}

// The row's share of the objective; `g` = d(policy term) / d(neglogp).
__device__ __forceinline__ float row_objective(const PolicyArgs &a, size_t row, const RowTerms &o, double part[5]) {
  if (o.padding) {
    a.dvalues[row] = 0.f;
    for (int i = 0; i < 5; ++i) part[i] = 0.;
    return 0.f;
  }
  const float A = a.advantages[row], old = a.old_neglogps[row];
  const float v = a.values[row], v0 = a.old_values[row], ret = a.returns[row];
  const float ratio = expf(old - o.nlp);
  const float lo = 1.f - a.clip, hi = 1.f + a.clip;
  const float held = ratio < lo ? lo : (ratio > hi ? hi : ratio);   // NaN stays NaN
  const float plain = -A * ratio, clipped = -A * held;
  const float dvv = v - v0;
  const float e1 = v - ret, e2 = v0 + (dvv < -a.clip ? -a.clip : (dvv > a.clip ? a.clip : dvv)) - ret;
  const float q1 = e1 * e1, q2 = e2 * e2;
  const float dv = q2 > q1 ? (__builtin_fabsf(dvv) <= a.clip ? e2 : 0.f) : e1;
  a.dvalues[row] = a.vf_coef * a.inv_denom * dv;
  const float kl = o.nlp - old;
  part[0] = plain >= clipped ? plain : (clipped > plain ? clipped : plain + clipped);
  part[1] = 0.5f * __builtin_elementwise_maximum(q1, q2);
  part[2] = o.ent;
  part[3] = 0.5f * kl * kl;
  part[4] = __builtin_fabsf(ratio - 1.f) > a.clip ? 1. : 0.;
  return plain >= clipped ? A * ratio : (clipped > plain ? 0.f : plain + clipped);
}

template <int WAVES>
__device__ __forceinline__ Softmax block_softmax(Softmax w, float *red) {   // red: 3 * WAVES floats; every thread gets the result
  const unsigned wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const float m = wave_max_nan(w.m);
  if (lane == 0) red[wave] = m;
  __syncthreads();
  float top = red[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) top = __builtin_elementwise_maximum(top, red[i]);
  rebase(w.m, top, w.s, w.t);
  const float s = wave_sum(w.s), t = wave_sum(w.t);
  if (lane == 0) { red[WAVES + wave] = s; red[2 * WAVES + wave] = t; }
  __syncthreads();
  Softmax o{top, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < WAVES; ++i) { o.s += red[WAVES + i]; o.t += red[2 * WAVES + i]; }
  return o;
}

template <typename T>
__device__ __forceinline__ void online(Softmax &w, const Raw8<T> &r, int n) {
  float top = w.m;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) top = __builtin_elementwise_maximum(top, r.get(i));
  if (!(top > w.m) && w.s == 0.f) { w.m = top; return; }     // nothing but -inf so far, or NaN
  rebase(w.m, top, w.s, w.t);
  w.m = top;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) {
      const float d = below(r.get(i), top), e = exp_neg(d);
      w.s += e;
      w.t = __builtin_fmaf(e, d, w.t);
    }
}

// One workgroup per row, the row read once (statistics) or twice (with the gradient, the second time out of the caches).
template <typename T, bool LOSS>
__global__ __launch_bounds__(256) void policy_row_kernel(PolicyArgs a) {
  __shared__ float red[12];
  __shared__ float share[4];
  const size_t row = blockIdx.x;
  const unsigned tid = threadIdx.x;
  const T *in = (const T *)a.logits + (int64_t)row * a.stride;
  const int64_t action = a.actions[row];
  const bool inside = action >= 0 && action < (int64_t)a.vocab;
  const float l_a = inside ? (float)in[action] : 0.f;
  Softmax w{-__builtin_inff(), 0.f, 0.f};
  if (action != -1)
    for (unsigned e = tid * 8; e < a.vocab; e += 2048) {
      Raw8<T> r;
      load8(r, in + e, (long)(a.vocab - e), 0.f);
      online(w, r, (int)min(8u, a.vocab - e));
    }
  w = block_softmax<4>(w, red);
  const RowTerms o = row_terms(w, action, a.vocab, l_a);
  if (tid == 0) { a.neglogps[row] = o.nlp; a.entropies[row] = o.ent; }
  if (!LOSS) return;
  if (tid == 0) {
    double part[5];
    share[0] = row_objective(a, row, o, part);
    for (int i = 0; i < 5; ++i) a.partials[row * 5 + i] = part[i];
  }
  __syncthreads();
  const float g = share[0];
  T *out = (T *)a.dlogits + (int64_t)row * a.dstride;
  // dl_j = (g (p_j - 1{j = a}) + ent p_j (ln p_j + H)) / n,  p_j = e_j / s,  ln p_j + H = d_j - t / s
  const float c1 = o.rs * a.ent_coef * a.inv_denom;
  const float c0 = o.rs * a.inv_denom * (g - a.ent_coef * o.t * o.rs);
  for (unsigned e = tid * 8; e < a.vocab; e += 2048) {
    const int n = (int)min(8u, a.vocab - e);
    Raw8<T> r;
    load8(r, in + e, n, 0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float d = below(r.get(i), w.m);
      float y = exp_neg(d) * __builtin_fmaf(d, c1, c0);
      if ((int64_t)(e + i) == action) y -= g * a.inv_denom;
      if (o.nan) y = __builtin_nanf("");
      if (o.padding || o.dead) y = 0.f;
      r.set(i, y);
    }
    store8(r, out + e, n);
  }
}

// Sums the rows' terms in a fixed order, in 64 bits.
__global__ __launch_bounds__(1024) void policy_stats_kernel(const double *partials, size_t n, double denom, float vf, float ent, float *stats) {
  __shared__ double red[16][5];
  double s[5] = {0, 0, 0, 0, 0};
  for (size_t i = threadIdx.x; i < n; i += 1024)
    for (int k = 0; k < 5; ++k) s[k] += partials[i * 5 + k];
  for (int k = 0; k < 5; ++k) {
    s[k] = wave_sum(s[k]);
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64][k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x) return;
  for (int k = 0; k < 5; ++k) {
    s[k] = 0;
    for (int w = 0; w < 16; ++w) s[k] += red[w][k];
    s[k] /= denom;
  }
  stats[0] = (float)(s[0] + (double)vf * s[1] - (double)ent * s[2]);
  for (int k = 0; k < 5; ++k) stats[1 + k] = (float)s[k];
}

// ---- host -----------------------------------------------------------------------------------------------------------------

bool finite_positive(float x) { return x > 0.f && std::isfinite(x); }

int check_rows(const char *who, int dtype, const void *p, int64_t stride, size_t rows, size_t vocab) {
  if (!is_dtype(dtype)) return ppoxp_fail(PPO_XP_EINVAL, "%s: unknown element type %d", who, dtype);
  if (vocab > kMaxVocab) return ppoxp_fail(PPO_XP_EINVAL, "%s: %zu tokens (2^30 at most)", who, vocab);
  if (rows == 0 || vocab == 0) return 0;
  if (!p) return ppoxp_fail(PPO_XP_EINVAL, "%s: NULL array", who);
  if (rows > 1 && stride < (int64_t)vocab) return ppoxp_fail(PPO_XP_EINVAL, "%s: rows of %zu elements lie %lld apart", who, vocab, (long long)stride);
  return 0;
}

int check_rules(const char *who, const ppo_xp_logit_rules *r, size_t rows, size_t vocab) {
  if (!r) return ppoxp_fail(PPO_XP_EINVAL, "%s: rules is NULL", who);
  if (!finite_positive(r->repetition) || !finite_positive(r->temperature))
    return ppoxp_fail(PPO_XP_EINVAL, "%s: repetition %g and temperature %g must be finite and > 0", who, r->repetition, r->temperature);
  if (!std::isfinite(r->presence) || !std::isfinite(r->frequency))
    return ppoxp_fail(PPO_XP_EINVAL, "%s: presence %g and frequency %g must be finite", who, r->presence, r->frequency);
  if (r->history) {
    if (r->history_bits != 32 && r->history_bits != 64) return ppoxp_fail(PPO_XP_EINVAL, "%s: history of %d-bit tokens", who, r->history_bits);
    if (r->hist_rows < 0 || r->hist_len < 0 || r->hist_len > 0x7fffffff || r->hist_row_stride < 0 || r->hist_tok_stride < 0)
      return ppoxp_fail(PPO_XP_EINVAL, "%s: bad history shape", who);
    if (!r->hist_row && (size_t)r->hist_rows < rows)
      return ppoxp_fail(PPO_XP_EINVAL, "%s: %lld history rows for %zu rows of logits", who, (long long)r->hist_rows, rows);
  }
  if (r->bias && r->bias_stride != 0 && r->bias_stride < (int64_t)vocab)
    return ppoxp_fail(PPO_XP_EINVAL, "%s: bias rows of %zu lie %lld apart", who, vocab, (long long)r->bias_stride);
  if (r->mask_kind != PPO_XP_MASK_NONE) {
    if (r->mask_kind != PPO_XP_MASK_BITS && r->mask_kind != PPO_XP_MASK_BYTES) return ppoxp_fail(PPO_XP_EINVAL, "%s: unknown mask kind %d", who, r->mask_kind);
    if (!r->mask) return ppoxp_fail(PPO_XP_EINVAL, "%s: mask is NULL", who);
    const int64_t need = r->mask_kind == PPO_XP_MASK_BITS ? (int64_t)((vocab + 31) / 32) : (int64_t)vocab;
    if (r->mask_rows < 1 || (r->mask_stride != 0 && r->mask_stride < need))
      return ppoxp_fail(PPO_XP_EINVAL, "%s: mask rows of %lld do not fit a stride of %lld", who, (long long)need, (long long)r->mask_stride);
    if (!r->mask_row && r->mask_stride != 0 && (size_t)r->mask_rows < rows)
      return ppoxp_fail(PPO_XP_EINVAL, "%s: %lld mask rows for %zu rows of logits", who, (long long)r->mask_rows, rows);
  }
  return 0;
}

template <typename T>
void launch_shape(const ShapeArgs &a, dim3 grid, hipStream_t s, bool hist, bool backward) {
  if (backward) {
    if (hist) hipLaunchKernelGGL((shape_logits_kernel<T, true, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((shape_logits_kernel<T, false, true>), grid, dim3(256), 0, s, a);
  } else {
    if (hist) hipLaunchKernelGGL((shape_logits_kernel<T, true, false>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((shape_logits_kernel<T, false, false>), grid, dim3(256), 0, s, a);
  }
}

int shape(const char *who, int device, void *stream, int dtype, ShapeArgs &a, size_t rows, size_t vocab, const ppo_xp_logit_rules *rules,
          bool backward) {
  if (int rc = check_rules(who, rules, rows, vocab)) return rc;
  if (rows == 0 || vocab == 0) return 0;
  a.vocab = (unsigned)vocab;
  a.chunks = (unsigned)((vocab + kShapeChunk - 1) / kShapeChunk);
  a.r = *rules;
  if (rows > kMaxGrid / a.chunks) return ppoxp_fail(PPO_XP_EINVAL, "%s: %zu rows of %zu are too many for one launch", who, rows, vocab);
  DeviceGuard dev(device, who);
  if (dev.rc()) return dev.rc();
  const dim3 grid((unsigned)(rows * a.chunks));
  const bool hist = rules->history && rules->hist_rows > 0 && rules->hist_len > 0;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_shape<float>(a, grid, s, hist, backward);
  else if (dtype == PPO_XP_BF16) launch_shape<__bf16>(a, grid, s, hist, backward);
  else launch_shape<_Float16>(a, grid, s, hist, backward);
  return launched(who);
}

template <bool LOSS>
void launch_policy(int dtype, const PolicyArgs &a, hipStream_t s) {
  const dim3 grid((unsigned)a.rows);
  if (dtype == PPO_XP_F32) hipLaunchKernelGGL((policy_row_kernel<float, LOSS>), grid, dim3(256), 0, s, a);
  else if (dtype == PPO_XP_BF16) hipLaunchKernelGGL((policy_row_kernel<__bf16, LOSS>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((policy_row_kernel<_Float16, LOSS>), grid, dim3(256), 0, s, a);
}

int check_workspace(const char *who, int dtype, size_t rows, size_t vocab, const void *ws, size_t bytes) {
  const size_t need = ppo_xp_policy_workspace(dtype, rows, vocab);
  if (need && (!ws || bytes < need || (uintptr_t)ws % 16))
    return ppoxp_fail(PPO_XP_EINVAL, "%s: workspace of %zu bytes, 16-byte aligned, expected (%zu given)", who, need, bytes);
  return 0;
}

}  // namespace

extern "C" {

int ppo_xp_shape_logits(int device, void *stream, int dtype, const void *logits, int64_t logits_stride, void *out, int64_t out_stride,
                        size_t rows, size_t vocab, const ppo_xp_logit_rules *rules) {
  if (int rc = check_rows("shape_logits", dtype, logits, logits_stride, rows, vocab)) return rc;
  if (int rc = check_rows("shape_logits", dtype, out, out_stride, rows, vocab)) return rc;
  ShapeArgs a{};
  a.in = logits; a.in_stride = logits_stride; a.out = out; a.out_stride = out_stride;
  return shape("shape_logits", device, stream, dtype, a, rows, vocab, rules, false);
}

int ppo_xp_shape_logits_backward(int device, void *stream, int dtype, const void *grad, int64_t grad_stride, const void *logits,
                                 int64_t logits_stride, void *out, int64_t out_stride, size_t rows, size_t vocab,
                                 const ppo_xp_logit_rules *rules) {
  if (int rc = check_rows("shape_logits_backward", dtype, grad, grad_stride, rows, vocab)) return rc;
  if (int rc = check_rows("shape_logits_backward", dtype, logits, logits_stride, rows, vocab)) return rc;
  if (int rc = check_rows("shape_logits_backward", dtype, out, out_stride, rows, vocab)) return rc;
  ShapeArgs a{};
  a.in = grad; a.in_stride = grad_stride; a.logits = logits; a.logits_stride = logits_stride; a.out = out; a.out_stride = out_stride;
  return shape("shape_logits_backward", device, stream, dtype, a, rows, vocab, rules, true);
}

size_t ppo_xp_policy_workspace(int dtype, size_t rows, size_t vocab) {
  (void)dtype; (void)vocab;
  return rows * 5 * sizeof(double);
}

int ppo_xp_action_stats(int device, void *stream, int dtype, const void *logits, int64_t logits_stride, const int64_t *actions,
                        float *neglogps, float *entropies, size_t rows, size_t vocab, void *workspace, size_t workspace_bytes) {
  if (int rc = check_rows("action_stats", dtype, logits, logits_stride, rows, vocab)) return rc;
  if (rows == 0 || vocab == 0) return 0;
  if (!actions || !neglogps || !entropies) return ppoxp_fail(PPO_XP_EINVAL, "action_stats: NULL argument");
  if (rows > kMaxGrid) return ppoxp_fail(PPO_XP_EINVAL, "action_stats: %zu rows are too many for one launch", rows);
  if (int rc = check_workspace("action_stats", dtype, rows, vocab, workspace, workspace_bytes)) return rc;
  PolicyArgs a{};
  a.logits = logits; a.stride = logits_stride; a.actions = actions; a.neglogps = neglogps; a.entropies = entropies;
  a.vocab = (unsigned)vocab; a.rows = rows;
  DeviceGuard dev(device, "action_stats");
  if (dev.rc()) return dev.rc();
  launch_policy<false>(dtype, a, (hipStream_t)stream);
  return launched("action_stats");
}

int ppo_xp_policy_loss(int device, void *stream, int dtype, const void *logits, int64_t logits_stride, const ppo_xp_policy_batch *b,
                       float clip, float ent_coef, float vf_coef, double denom, void *dlogits, int64_t dlogits_stride, float *dvalues,
                       float *neglogps, float *entropies, float *stats, size_t rows, size_t vocab, void *workspace, size_t workspace_bytes) {
  if (int rc = check_rows("policy_loss", dtype, logits, logits_stride, rows, vocab)) return rc;
  if (int rc = check_rows("policy_loss", dtype, dlogits, dlogits_stride, rows, vocab)) return rc;
  if (!(clip >= 0.f) || !std::isfinite(clip) || !std::isfinite(ent_coef) || !std::isfinite(vf_coef))
    return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: clip %g (>= 0), ent_coef %g and vf_coef %g must be finite", clip, ent_coef, vf_coef);
  if (!(denom > 0.) || !std::isfinite(denom)) return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: denom %g must be finite and > 0", denom);
  if (rows == 0 || vocab == 0) return 0;
  if (!b || !b->actions || !b->old_values || !b->old_neglogps || !b->returns || !b->advantages || !b->values || !dvalues || !neglogps ||
      !entropies || !stats)
    return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: NULL argument");
  if (rows > kMaxGrid) return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: %zu rows are too many for one launch", rows);
  if (int rc = check_workspace("policy_loss", dtype, rows, vocab, workspace, workspace_bytes)) return rc;
  PolicyArgs a{};
  a.logits = logits; a.stride = logits_stride; a.actions = b->actions; a.neglogps = neglogps; a.entropies = entropies;
  a.vocab = (unsigned)vocab; a.rows = rows;
  a.old_values = b->old_values; a.old_neglogps = b->old_neglogps; a.returns = b->returns; a.advantages = b->advantages; a.values = b->values;
  a.clip = clip; a.ent_coef = ent_coef; a.vf_coef = vf_coef; a.inv_denom = (float)(1. / denom);
  a.dlogits = dlogits; a.dstride = dlogits_stride; a.dvalues = dvalues; a.partials = (double *)workspace;
  DeviceGuard dev(device, "policy_loss");
  if (dev.rc()) return dev.rc();
  launch_policy<true>(dtype, a, (hipStream_t)stream);
  if (int rc = launched("policy_loss")) return rc;
  hipLaunchKernelGGL(policy_stats_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const double *)workspace, rows, denom, vf_coef, ent_coef, stats);
  return launched("policy_loss");
}

}  // extern "C"

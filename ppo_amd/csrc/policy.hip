// Logits of token policies: the rules that shape them and their gradient, neglogp and entropy of an action, the clipped
// objective with its gradient.  Semantics in include/ppo_xp.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ops_common.h"

namespace {

using namespace ppoxp_ops;

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// ---- rules ----------------------------------------------------------------------------------------------------------------

struct ShapeArgs {
  const void *in;        // logits, or the gradient of the shaped logits
  const void *logits;    // backward: the logits, for the sign of tokens that were seen
  void *out;
  int64_t in_stride, logits_stride, out_stride;
  size_t rows;
  unsigned vocab, chunks, part;                 // chunks of a row and their elements, where a row fills a workgroup
  unsigned rows_per, units, magic, scan_log2;   // else rows of a workgroup, 8-element units of a row, 2^20 / units, lanes that scan a row
  ppo_xp_logit_rules r;
};

enum ShapeMode { kForward, kGather, kReadAll };
// Elements of a workgroup, with VECS vectors of 8 a thread.
constexpr unsigned shape_chunk(int vecs) { return 256 * 8 * vecs; }
constexpr unsigned kPromptOnly = 0x80000000u;        // table word: occurrences in the generated part, this bit: in the rest

// Where element e of a workgroup's chunk has its table word: the lower and the upper halves of the vectors lie apart, so that a
// wave reads each half without bank conflicts.
template <int VECS>
__device__ __forceinline__ unsigned table_slot(unsigned e) { return ((e & 4) ? shape_chunk(VECS) / 2 : 0) + (e >> 3) * 4 + (e & 3); }

struct RowRules {
  float rep, inv_rep, pres, freq, inv_t;
  const float *bias;
  const uint8_t *mask;
};

// Divisors from the least normal number on have a finite reciprocal (of smaller ones it is infinite, and 0 times that NaN): a
// row's own value below it counts as that number, a scalar was refused.
constexpr float kLeastDivisor = 0x1p-126f;
__device__ __forceinline__ float divisor(float x) { return x < kLeastDivisor ? kLeastDivisor : x; }   // NaN stays NaN

__device__ __forceinline__ RowRules row_rules(const ppo_xp_logit_rules &r, size_t row) {
  RowRules q;
  q.rep = divisor(r.repetition_rows ? r.repetition_rows[row] : r.repetition);
  q.inv_rep = 1.f / q.rep;
  q.pres = r.presence_rows ? r.presence_rows[row] : r.presence;
  q.freq = r.frequency_rows ? r.frequency_rows[row] : r.frequency;
  q.inv_t = 1.f / divisor(r.temperature_rows ? r.temperature_rows[row] : r.temperature);
  q.bias = r.bias ? r.bias + (int64_t)row * r.bias_stride : nullptr;
  q.mask = nullptr;
  if (r.mask_kind != PPO_XP_MASK_NONE) {
    const int64_t m = r.mask_row ? r.mask_row[row] : (r.mask_stride == 0 ? 0 : (int64_t)row);
    if (m >= 0 && m < r.mask_rows) q.mask = (const uint8_t *)r.mask + m * r.mask_stride * (r.mask_kind == PPO_XP_MASK_BITS ? 4 : 1);
  }
  return q;
}

// Bit i: element e + i of a row is allowed.
__device__ __forceinline__ unsigned allowed8(const RowRules &q, int kind, unsigned e, unsigned vocab) {
  if (!q.mask) return 0xffu;
  if (kind == PPO_XP_MASK_BITS) return q.mask[e / 8];
  unsigned ok = 0;
  if (e + 8 <= vocab) {
    typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
    const u32x2 w = *(const u32x2_a1 *)(q.mask + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) ok |= ((w[i >> 2] >> (8 * (i & 3))) & 0xffu) ? 1u << i : 0u;
  } else {
    for (unsigned i = 0; e + i < vocab; ++i) ok |= (q.mask[e + i] ? 1u : 0u) << i;
  }
  return ok;
}

// One workgroup shapes one chunk of one row's vocabulary, or several whole rows (MULTI).  With a history it enters the tokens that
// fall into its part in an LDS table first, while its logits are already on their way into registers: their counts (integer
// atomics, the order does not matter), or in the backward pass the slope, which every occurrence knows from the token's logit
// (kGather), or only that it was seen, where all logits are read (kReadAll).
// Every workgroup of a row reads the row's whole history; that is cheaper than sorting it while the history is shorter than the
// vocabulary.  Of a lane's 8 elements those take their word for which some lane of the wave has one (at a token in 64 seen 63 % of
// them).  256 x 131072 bf16 with 2048 tokens a row, a shared bias and mask bits: 34 us a call, 152 MB, of which the bias fetched ahead
// of the second barrier saves 1.4 us; the same without a history or bias 22 us.  Memory bounds it, then the table.
template <typename T, bool HIST, int MODE, bool MULTI, int VECS>
__global__ __launch_bounds__(256) void shape_logits_kernel(ShapeArgs a) {
  constexpr bool BACKWARD = MODE != kForward;
  constexpr unsigned CHUNK = shape_chunk(VECS);
  __shared__ __attribute__((aligned(16))) unsigned table[HIST ? CHUNK : 4];
  const ppo_xp_logit_rules &r = a.r;
  const unsigned tid = threadIdx.x;
  const size_t row0 = MULTI ? (size_t)blockIdx.x * a.rows_per : blockIdx.x / a.chunks;
  const unsigned c0 = MULTI ? 0 : (blockIdx.x % a.chunks) * a.part;
  const unsigned here = MULTI ? (unsigned)min((size_t)a.rows_per, a.rows - row0) : 1;    // rows of this workgroup
  const unsigned c1 = MULTI ? a.vocab : min(a.vocab, c0 + a.part);
  RowRules one;
  if (!MULTI) one = row_rules(r, row0);
  // unit k of this thread: its row and first element, and whether there is one
  auto place = [&](int k, size_t &row, unsigned &e) {
    const unsigned u = k * 256 + tid;
    if (!MULTI) { row = row0; e = c0 + u * 8; return e < c1; }
    const unsigned rl = (u * a.magic) >> 20;
    row = row0 + rl;
    e = (u - rl * a.units) * 8;
    return rl < here;
  };

  auto fetch = [&](Raw8<T> *to, const void *from, int64_t stride) {
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      size_t row; unsigned e;
      if (!place(k, row, e)) { row = row0; e = 0; }   // nothing here: the whole wave stays on the wide load
      const T *p = (const T *)from + (int64_t)row * stride;
      if (e + 8 <= a.vocab) {
        to[k].load(p + e);
      } else {                                       // a row's end: clamped addresses, no further branch
        T q[8];
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = p[min(e + i, a.vocab - 1)];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (float)q[i];
        to[k].set8(y);
      }
    }
  };
  Raw8<T> raw[VECS], own[MODE == kReadAll ? VECS : 1];
  fetch(raw, a.in, a.in_stride);
  if (MODE == kReadAll) fetch(own, a.logits, a.logits_stride);
  unsigned ok[VECS];                                 // with one row a workgroup the mask's bits are on their way as well
  if (!MULTI) {
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      const unsigned e = c0 + (k * 256 + tid) * 8;
      ok[k] = one.mask && r.mask_kind == PPO_XP_MASK_BITS ? one.mask[min(e, a.vocab - 1) / 8] : 0xffu;
    }
  }
  // ... and so is the bias, once the history has left its registers
  Raw8<float> bias[MULTI || BACKWARD ? 1 : VECS];
  auto fetch_bias = [&]() {
    if (MULTI || BACKWARD || !one.bias) return;
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      size_t row; unsigned e;
      if (!place(k, row, e)) e = 0;
      if (e + 8 <= a.vocab) {
        bias[k].load(one.bias + e);
      } else {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = one.bias[min(e + i, a.vocab - 1)];
        bias[k].set8(y);
      }
    }
  };
  if (HIST) {
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      unsigned word = 0;
      if (MODE == kGather) {
        float inv_t = one.inv_t;
        if (MULTI) {
          size_t row; unsigned e;
          const bool live = place(k, row, e);
          inv_t = row_rules(r, live ? row : row0).inv_t;
        }
        word = __builtin_bit_cast(unsigned, inv_t);
      }
      *(u32x4 *)(table + (k * 256 + tid) * 4) = u32x4(word);
      *(u32x4 *)(table + CHUNK / 2 + (k * 256 + tid) * 4) = u32x4(word);
    }
    __syncthreads();
    const unsigned lanes = MULTI ? 1u << a.scan_log2 : 256u;
    for (unsigned rl = MULTI ? tid >> a.scan_log2 : 0; rl < here; rl += MULTI ? 256u >> a.scan_log2 : 1u) {
      const size_t row = row0 + rl;
      const int64_t h = r.hist_row ? r.hist_row[row] : (int64_t)row;
      if (h < 0 || h >= r.hist_rows) continue;
      const int end = (int)min(r.hist_end ? (int64_t)r.hist_end[row] : r.hist_len, r.hist_len);
      // 64 bits: a first position near the type's end plus the thread's own must not wrap round to in front of the history
      const int64_t begin = r.hist_begin ? min((int64_t)max(r.hist_begin[row], 0), r.hist_len) : 0;
      const int64_t gen = r.gen_begin ? r.gen_begin[row] : begin;
      const int64_t base = h * r.hist_row_stride;
      const T *logits = MODE == kGather ? (const T *)a.logits + (int64_t)row * a.logits_stride : nullptr;
      float up = 0.f, down = 0.f;                    // backward: the slope at positive logits and at others
      if (MODE == kGather) {
        const RowRules q = MULTI ? row_rules(r, row) : one;
        up = q.inv_rep * q.inv_t;
        down = q.rep * q.inv_t;
      }
      constexpr int kTokens = 8;                     // on their way at a time
      for (int64_t k0 = begin + (MULTI ? tid & (lanes - 1) : tid); k0 < end; k0 += kTokens * lanes) {
        int64_t tok[kTokens];
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
          const int64_t at = base + min(k0 + j * lanes, (int64_t)end - 1) * r.hist_tok_stride;
          tok[j] = r.history_bits == 64 ? ((const int64_t *)r.history)[at] : (int64_t)((const int32_t *)r.history)[at];
        }
        float l[kTokens];
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
          const bool in_chunk = tok[j] >= c0 && tok[j] < (int64_t)c1 && k0 + j * lanes < end;
          if (!in_chunk) tok[j] = -1;
          if (MODE == kGather) l[j] = in_chunk ? (float)logits[tok[j]] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
          if (tok[j] < 0) continue;
          unsigned *word = table + table_slot<VECS>((unsigned)tok[j] - c0 + rl * a.units * 8);
          if (MODE == kGather) *word = __builtin_bit_cast(unsigned, l[j] > 0.f ? up : down);   // the same from every occurrence
          else if (MODE == kReadAll) *word = 1;
          else if (k0 + j * lanes >= gen) atomicAdd(word, 1u);
          else atomicOr(word, kPromptOnly);
        }
      }
    }
    fetch_bias();
    __syncthreads();
  } else {
    fetch_bias();
  }
#pragma unroll
  for (int k = 0; k < VECS; ++k) {
    size_t row; unsigned e;
    if (!place(k, row, e)) continue;
    const RowRules q = MULTI ? row_rules(r, row) : one;
    const unsigned allowed = !MULTI && r.mask_kind != PPO_XP_MASK_BYTES ? ok[k] : allowed8(q, r.mask_kind, e, a.vocab);
    u32x4 c[2] = {u32x4(0), u32x4(0)};
    if (HIST) {
      c[0] = *(const u32x4 *)(table + (k * 256 + tid) * 4);
      c[1] = *(const u32x4 *)(table + CHUNK / 2 + (k * 256 + tid) * 4);
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = raw[k].get(i);
    if (BACKWARD) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned w = c[i >> 2][i & 3];
        if (MODE == kReadAll) x[i] *= q.inv_t * (w ? (own[k].get(i) > 0.f ? q.inv_rep : q.rep) : 1.f);
        else x[i] *= HIST ? __builtin_bit_cast(float, w) : q.inv_t;
      }
    } else {
      if (HIST) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned w = c[i >> 2][i & 3];
          if (!__any(w != 0)) continue;
          const float n = (float)(w & ~kPromptOnly);
          x[i] *= w ? (x[i] > 0.f ? q.inv_rep : q.rep) : 1.f;
          x[i] -= n > 0.f ? q.freq * n + q.pres : 0.f;    // not freq * 0: it may be infinite
        }
      }
      if (!MULTI && q.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += bias[k].get(i);
      } else if (q.bias) {
        if (e + 8 <= a.vocab) {
          Raw8<float> b;
          b.load(q.bias + e);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] += b.get(i);
        } else {
          for (int i = 0; i < 8; ++i)
            if (e + i < a.vocab) x[i] += q.bias[e + i];
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= q.inv_t;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (allowed >> i) & 1 ? x[i] : (BACKWARD ? 0.f : -__builtin_inff());
    raw[k].set8(x);
    store8(raw[k], (T *)a.out + (int64_t)row * a.out_stride + e, (long)a.vocab - (long)e);
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
  double *partials;      // [5][records]: policy, value, entropy, kl, clipped
  unsigned *ticket;      // of policy_stats_kernel; the launch before it sets it to 0
};

// A row in powers of two: m = max l, x = (l - m) log2(e), s = sum 2^x, t = sum 2^x x;  ln softmax(l)_j = ln2 (x_j - log2 s).
// (One fma of l with a rounded m log2(e) would save an instruction, but its error grows with |m| until 2^x overflows.)
struct Softmax { float m, s, t; };

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float power(float l, float m) { return (l - m) * kLog2e; }
// ... kept finite: 2^-200 is 0 in 32 bits, and 0 * -200 is 0 where 0 * -inf is not
__device__ __forceinline__ float finite_power(float l, float m) { return __builtin_fmaxf(power(l, m), -200.f); }

// Brings (s, t) from maximum `m` to the larger or equal `to`.
__device__ __forceinline__ void rebase(float m, float to, float &s, float &t) {
  if (s == 0.f) return;
  const float d = finite_power(m, to), f = exp2_fast(d);
  t = (t + s * d) * f;
  s *= f;
}

// What one row's statistics mean for its action.
struct RowTerms {
  bool padding, dead, nan;   // dead: -inf throughout
  float nlp, ent, rs, ts;    // rs = 1 / s, ts = t / s
};

__device__ __forceinline__ RowTerms row_terms(const Softmax &w, int64_t action, unsigned vocab, float l_a) {
  RowTerms o{};
  o.padding = action == -1;
  if (o.padding) return o;
  o.nan = !(w.m < __builtin_inff()) || action < 0 || action >= (int64_t)vocab;
  if (o.nan) { o.nlp = o.ent = __builtin_nanf(""); return o; }
  o.dead = w.m == -__builtin_inff();
  if (o.dead) { o.nlp = __builtin_inff(); return o; }
  const float log2_s = log2f(w.s);
  o.rs = 1.f / w.s;
  o.ts = w.t * o.rs;
  o.nlp = kLn2 * (log2_s - power(l_a, w.m));
  o.ent = kLn2 * (log2_s - o.ts);
  return o;
}

// The row's entries of the batch, loaded while the logits are on their way.
struct RowInputs { float A, old, v, v0, ret; };

__device__ __forceinline__ RowInputs row_inputs(const PolicyArgs &a, size_t row) {
  return RowInputs{a.advantages[row], a.old_neglogps[row], a.values[row], a.old_values[row], a.returns[row]};
}

// The row's share of the objective.
struct RowShare { float g, dvalue, part[5]; };       // g = d(policy term) / d(neglogp)

__device__ __forceinline__ RowShare row_objective(const PolicyArgs &a, const RowInputs &q, const RowTerms &o) {
  RowShare r{};
  if (o.padding) return r;
  const float ratio = expf(q.old - o.nlp);
  const float lo = 1.f - a.clip, hi = 1.f + a.clip;
  const float held = ratio < lo ? lo : (ratio > hi ? hi : ratio);   // NaN stays NaN
  const float plain = -q.A * ratio, clipped = -q.A * held;
  const float dvv = q.v - q.v0;
  const float e1 = q.v - q.ret, e2 = q.v0 + (dvv < -a.clip ? -a.clip : (dvv > a.clip ? a.clip : dvv)) - q.ret;
  const float q1 = e1 * e1, q2 = e2 * e2;
  const float kl = o.nlp - q.old;
  r.dvalue = a.vf_coef * a.inv_denom * (q2 > q1 ? (__builtin_fabsf(dvv) <= a.clip ? e2 : 0.f) : e1);
  r.part[0] = plain >= clipped ? plain : (clipped > plain ? clipped : plain + clipped);
  r.part[1] = 0.5f * __builtin_elementwise_maximum(q1, q2);
  r.part[2] = o.ent;
  r.part[3] = 0.5f * kl * kl;
  r.part[4] = __builtin_fabsf(ratio - 1.f) > a.clip ? 1.f : 0.f;
  r.g = plain >= clipped ? q.A * ratio : (clipped > plain ? 0.f : plain + clipped);
  return r;
}

// One lane of a row's workgroup writes what the row gives.
__device__ __forceinline__ void put_row(const PolicyArgs &a, size_t row, const RowTerms &o, const RowShare &r) {
  a.neglogps[row] = o.nlp;
  a.entropies[row] = o.ent;
  a.dvalues[row] = r.dvalue;
  for (int i = 0; i < 5; ++i) a.partials[i * a.rows + row] = r.part[i];
  if (row == 0) *a.ticket = 0;
}

// Joins the lanes' statistics, each relative to its own maximum, over a workgroup of up to 16 waves with one barrier; every
// thread gets the result.  A maximum of NaN stays NaN.
__device__ __forceinline__ Softmax wave_softmax(Softmax w) {
  const float m = wave_max_nan(w.m);
  rebase(w.m, m, w.s, w.t);
  return Softmax{m, wave_sum(w.s), wave_sum(w.t)};
}
__device__ __forceinline__ Softmax block_softmax(Softmax w, Softmax *red) {   // red: 16
  w = wave_softmax(w);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = w;
  __syncthreads();
  const unsigned lane = threadIdx.x % 64;
  w = lane < blockDim.x / 64 ? red[lane] : Softmax{-__builtin_inff(), 0.f, 0.f};
  return wave_softmax(w);
}

// Elements beyond the row read as -inf and add nothing.
template <typename T>
__device__ __forceinline__ float max8(float m, const Raw8<T> &r) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __builtin_elementwise_maximum(m, r.get(i));
  return m;
}
__device__ __forceinline__ void add_term(Softmax &w, float l) {
  const float x = finite_power(l, w.m), e = exp2_fast(x);
  w.s += e;
  w.t = __builtin_fmaf(e, x, w.t);
}
template <typename T>
__device__ __forceinline__ void sums8(Softmax &w, const Raw8<T> &r) {
#pragma unroll
  for (int i = 0; i < 8; ++i) add_term(w, r.fresh(i));
}

// What an element costs in the vector unit is what bounds rows of 16-bit logits, so rows that allow it take a shorter way: with
// the reference m of moderate size and every logit finite, x = l log2(e) - m2 is one fma against m2 = fl(m log2(e)) and needs no
// clamp.  (m2's rounding shifts all x by `shift`, which is known exactly and taken out afterwards; its size grows with |m|.)
constexpr float kPlainMost = 4096.f, kPlainLeast = -1e30f;

struct Plain {
  float m2, shift;       // x of the row's definition = x here - shift
  __device__ __forceinline__ explicit Plain(float m) {
    m2 = m * kLog2e;
    shift = __builtin_fmaf(m, kLog2e, -m2);
  }
};

__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c)); return d; }
__device__ __forceinline__ float min3(float a, float b, float c) { float d; asm("v_minimum3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c)); return d; }

// What the place beyond a row's end holds: so small that its power is 0, finite so that the row's last wave need not go the long
// way.  Where the row itself is as small, row_softmax reads its own elements once more instead.
template <typename T> constexpr float kBeyond = -9e29f;
template <> constexpr float kBeyond<_Float16> = -65504.f;

// Elements first .. end of an array: a row, seen from the last 4-byte boundary at or before its start.  Sixteen bytes at a multiple of
// two bytes only cost the row kernels 15 % (50 001 against 50 000 bf16 tokens); at a multiple of four they are free.
struct Span { unsigned first, end; };

template <typename T>
__device__ __forceinline__ Span span_of(const T *&in, unsigned vocab, bool room = true) {   // room: for an element in front
  const unsigned odd = sizeof(T) == 2 && room ? (unsigned)((uintptr_t)in >> 1) & 1u : 0u;
  in -= odd;
  return Span{odd, vocab + odd};
}

// A row over `lanes` lanes: lane i holds vectors i, i + lanes, ...  All of them are on their way before anything waits (which is
// why the row's ends are one straight block with clamped addresses: another merge of values would make the compiler wait for each).
template <int NV, typename T>
__device__ __forceinline__ void load_row(Raw8<T> *r, const T *in, unsigned lane, unsigned lanes, Span at) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const unsigned e = (k * lanes + lane) * 8;
    if (e >= at.first && e + 8 <= at.end) {
      r[k].load(in + e);
    } else {
      T q[8];
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = in[max(min(e + i, at.end - 1), at.first)];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = e + i >= at.first && e + i < at.end ? (float)q[i] : kBeyond<T>;
      r[k].set8(y);
    }
  }
}

// NV vectors in registers, `step` elements apart from element e0 on.  Returns whether the whole wave went the short way, which
// its gradient may then go as well.  KEEP: few enough vectors to hold their floats from the maximum to the sums, one conversion an
// element less (statistics of 4096 x 32768 bf16 49.0 us against 51.0).
template <int NV, bool KEEP = false, typename T>
__device__ __forceinline__ bool row_softmax(Softmax &w, const Raw8<T> *r, const T *in, unsigned e0, unsigned step, Span at) {
  float least = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = r[k].get(i), b = r[k].get(i + 1);
      w.m = max3(w.m, a, b);
      least = min3(least, a, b);
    }
  }
  if (__all(least >= kPlainLeast && __builtin_fabsf(w.m) <= kPlainMost)) {
    const Plain p(w.m);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = __builtin_fmaf(KEEP ? r[k].get(i) : r[k].fresh(i), kLog2e, -p.m2), e = exp2_fast(x);
        w.s += e;
        w.t = __builtin_fmaf(e, x, w.t);
      }
    }
    const float f = exp2_fast(-p.shift);
    w.t = (w.t - p.shift * w.s) * f;
    w.s *= f;
    return true;
  }
  if (w.m <= kBeyond<T> / 2) {                                // the row's own logits are as small as what lies beyond it, or -inf
    w.m = -__builtin_inff();
#pragma unroll 1
    for (unsigned j = 0; j < NV * 8; ++j) {
      const unsigned e = e0 + j / 8 * step + j % 8;
      if (e >= at.first && e < at.end) w.m = __builtin_elementwise_maximum(w.m, (float)in[e]);
    }
    if (w.m == -__builtin_inff()) return false;
#pragma unroll 1
    for (unsigned j = 0; j < NV * 8; ++j) {
      const unsigned e = e0 + j / 8 * step + j % 8;
      if (e >= at.first && e < at.end) add_term(w, (float)in[e]);
    }
    return false;
  }
#pragma unroll
  for (int k = 0; k < NV; ++k) sums8(w, r[k]);
  return false;
}

// One pass with a running maximum.
template <typename T>
__device__ __forceinline__ void online(Softmax &w, const Raw8<T> &r) {
  const float top = max8(w.m, r);
  if (!(top > w.m) && w.s == 0.f) { w.m = top; return; }     // nothing but -inf so far, or NaN
  rebase(w.m, top, w.s, w.t);
  w.m = top;
  sums8(w, r);
}

// Gradient of one row's logits r (in place): dl_j = (g (p_j - 1{j = a}) + ent p_j (ln p_j + H)) / n with p_j = e_j / s and
// ln p_j + H = ln2 (x_j - t / s), so dl_j = e_j (c1 x_j + c0) - 1{j = a} g / n.
struct GradTerms {
  float m, c0, c1, hit;
  bool nan, zero;
};

__device__ __forceinline__ GradTerms grad_terms(const PolicyArgs &a, float m, const RowTerms &o, float g) {
  GradTerms k;
  k.m = m;
  k.c1 = o.rs * (kLn2 * a.ent_coef) * a.inv_denom;
  k.c0 = o.rs * a.inv_denom * (g - (kLn2 * a.ent_coef) * o.ts);
  k.hit = g * a.inv_denom;
  k.nan = o.nan;
  k.zero = o.padding || o.dead;
  return k;
}

// ... as the short way has it: k.m holds m2.
__device__ __forceinline__ GradTerms plain_terms(GradTerms k) {
  const Plain p(k.m);
  const float f = exp2_fast(-p.shift);
  k.c0 = (k.c0 - k.c1 * p.shift) * f;
  k.c1 *= f;
  k.m = p.m2;
  return k;
}

template <bool PLAIN, typename T>
__device__ __forceinline__ void gradient8(Raw8<T> &r, const GradTerms &k, int at) {   // at: the action's place in r, if 0..7
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float l = r.fresh(i), x = PLAIN ? __builtin_fmaf(l, kLog2e, -k.m) : finite_power(l, k.m);
    y[i] = exp2_fast(x) * __builtin_fmaf(x, k.c1, k.c0);
  }
  if ((unsigned)at < 8u) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i == at) y[i] -= k.hit;
  }
  if (!PLAIN && (k.nan || k.zero)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = k.zero ? 0.f : __builtin_nanf("");
  }
  r.set8(y);
}

// The gradient of a row that load_row brought, written.
template <bool PLAIN, int NV, typename T>
__device__ __forceinline__ void write_gradient(Raw8<T> *r, const GradTerms &k, T *out, unsigned lane, unsigned lanes, Span at, int64_t action) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const unsigned e = (v * lanes + lane) * 8;
    if (e >= at.end) break;
    gradient8<PLAIN>(r[v], k, (int)(action - e));
    if (e >= at.first && e + 8 <= at.end) r[v].store(out + e);
    else
      for (int i = 0; i < 8; ++i)
        if (e + i >= at.first && e + i < at.end) out[e + i] = (T)r[v].get(i);
  }
}
// The short way only where every lane's row allows it and has a distribution.
template <int NV, typename T>
__device__ __forceinline__ void write_gradient(Raw8<T> *r, const GradTerms &k, T *out, unsigned lane, unsigned lanes, Span at, int64_t action, bool plain) {
  if (plain && __all(__builtin_fabsf(k.m) <= kPlainMost && !k.nan && !k.zero)) write_gradient<true, NV>(r, plain_terms(k), out, lane, lanes, at, action);
  else write_gradient<false, NV>(r, k, out, lane, lanes, at, action);
}

// One record of the objective a workgroup that walks over several rows, its waves' sums added in order.
__device__ __forceinline__ void put_block(const PolicyArgs &a, const double sum[5], double (*red)[5]) {
  for (int i = 0; i < 5; ++i) {
    const double x = wave_sum(sum[i]);
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64][i] = x;
  }
  __syncthreads();
  if (threadIdx.x < 5) a.partials[threadIdx.x * (size_t)gridDim.x + blockIdx.x] = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
}

// Action sets of ordinary environments, and rows of some hundred tokens that do not fill the lanes of policy_group_kernel: a wave's rows
// come in and leave as one run of elements, 64 neighbours an access, and are turned in shared memory, where they lie an odd number of
// floats apart, free of bank conflicts.  Up to 48 tokens a lane has a row, since what a row costs beside its elements is as much as 15 of
// them; longer ones are SPREAD over 2, 4, ... lanes, element i with lane i of them.  SLOTS elements a lane, the last of them perhaps
// beyond the row.  Memory bounds it (objective of 1048576 x 32 f32: 306 MB in 59 us, of 262144 x 18 f32: 49 MB in 15 us).
constexpr unsigned kGroupBlocks = 1536;

__device__ __forceinline__ void wave_lds_fence() {            // what the wave's lanes wrote to LDS, its other lanes read afterwards
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T, bool LOSS, int SLOTS, bool SPREAD>
__global__ __launch_bounds__(256, SLOTS <= 32 ? 4 : 2) void policy_small_kernel(PolicyArgs a, unsigned magic, unsigned lanes_log2) {   // magic: 2^22 / vocab, rounded up
  constexpr int LEAST = SLOTS <= 32 && !SPREAD ? SLOTS - 3 : SLOTS - 7, FULL = SPREAD ? LEAST - 1 : LEAST;   // slots in use at least, and up to their end
  __shared__ double red[4][5];
  __shared__ float turn[4][64 * (SLOTS + 1)];
  const unsigned vocab = a.vocab, even = vocab % 2 ? 0 : magic;
  const unsigned lg = SPREAD ? lanes_log2 : 0, lanes = 1u << lg, wave_rows = 64u >> lg;
  const int slots = (int)((vocab + lanes - 1) >> lg);
  unsigned lane = threadIdx.x % 64;
  float *all = turn[threadIdx.x / 64];
  auto place = [&]() { return all + (lane >> lg) * (vocab | 1) + (lane & (lanes - 1)); };   // of the lane's first element
  auto slot = [&](unsigned i) { return i + (__umul24(i, even) >> 22); };    // of element i of the run
  double sum[5] = {0, 0, 0, 0, 0};
  for (size_t row0 = ((size_t)blockIdx.x * 4 + threadIdx.x / 64) * wave_rows; row0 < a.rows; row0 += (size_t)gridDim.x * 4 * wave_rows) {
    const unsigned here = (unsigned)min((size_t)wave_rows, a.rows - row0), end = here * vocab;
    const T *in = (const T *)a.logits + (int64_t)row0 * a.stride;
    asm volatile("" : "+v"(lane));                   // or the compiler holds every element's place across the rows: 256 registers
    T raw[SLOTS];
    if (a.stride == (int64_t)vocab) {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k)
        if (k < LEAST || k < slots) raw[k] = in[min(k * 64 + lane, end - 1)];
    } else {
#pragma unroll
      for (int k = 0; k < SLOTS; ++k) {
        const unsigned i = min(k * 64 + lane, end - 1), r = __umul24(i, magic) >> 22;
        if (k < LEAST || k < slots) raw[k] = in[(int64_t)r * a.stride + (i - r * vocab)];
      }
    }
    const unsigned own = lane >> lg, sub = lane & (lanes - 1);
    const size_t row = row0 + min(own, here - 1);
    const bool puts = own < here && sub == 0;
    const int64_t action = a.actions[row];
    RowInputs q{};
    if (LOSS) q = row_inputs(a, row);
#pragma unroll
    for (int k = 0; k < SLOTS; ++k)
      if (k < LEAST || k < slots) all[slot(k * 64 + lane)] = (float)raw[k];
    wave_lds_fence();
    const unsigned pick = action >= 0 && action < (int64_t)vocab ? (unsigned)action : 0;
    float *mine = place();
    const float l_a = mine[(int)pick - (int)sub];
    float x[SLOTS], e[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) x[i] = i < FULL || (i << lg) + sub < vocab ? mine[i << lg] : -__builtin_inff();
    Softmax w{-__builtin_inff(), 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SLOTS; i += 2) w.m = max3(w.m, x[i], x[i + 1]);
    if (SPREAD) w.m = group_max_nan(w.m, lanes);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      x[i] = finite_power(x[i], w.m);
      e[i] = exp2_fast(x[i]);
      w.s += e[i];
      w.t = __builtin_fmaf(e[i], x[i], w.t);
    }
    if (SPREAD) {
      w.s = group_sum(w.s, lanes);
      w.t = group_sum(w.t, lanes);
    }
    const RowTerms o = row_terms(w, action, vocab, l_a);
    if (puts) { a.neglogps[row] = o.nlp; a.entropies[row] = o.ent; }
    if (LOSS) {
      const RowShare share = row_objective(a, q, o);
      if (puts) {
        a.dvalues[row] = share.dvalue;
        for (int i = 0; i < 5; ++i) sum[i] += share.part[i];
      }
      GradTerms k = grad_terms(a, w.m, o, share.g);
      if (k.nan) k.c0 = __builtin_nanf("");
      if (SPREAD) asm volatile("" : "+v"(lane));
      mine = place();
#pragma unroll
      for (int i = 0; i < SLOTS; ++i)
        if (i < FULL || (i << lg) + sub < vocab) mine[i << lg] = k.zero ? 0.f : e[i] * __builtin_fmaf(x[i], k.c1, k.c0);
      if (!k.zero && (pick & (lanes - 1)) == sub) mine[pick - sub] -= k.hit;   // after a NaN it stays one
      wave_lds_fence();
      T *out = (T *)a.dlogits + (int64_t)row0 * a.dstride;
      asm volatile("" : "+v"(lane));
      if (a.dstride == (int64_t)vocab) {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
          const unsigned i = k * 64 + lane;
          if ((k < LEAST || k < slots) && i < end) out[i] = (T)all[slot(i)];
        }
      } else {
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
          const unsigned i = k * 64 + lane, r = __umul24(i, magic) >> 22;
          if ((k < LEAST || k < slots) && i < end) out[(int64_t)r * a.dstride + (i - r * vocab)] = (T)all[slot(i)];
        }
      }
    }
    wave_lds_fence();
  }
  if (LOSS) put_block(a, sum, red);
}

// Up to kGroupVocab tokens: `lanes` neighbouring lanes hold one row, NV vectors of 8 each, and a wave as many rows as it can: what a
// row costs beside its elements (some 200 instructions) is paid once a wave.  Memory bounds it where rows fill their lanes (objective of
// 131072 x 256 f32 277 MB in 60 us, bf16 143 MB in 33 us), the row's cost and its odd ends where they do not (222214 x 151 bf16 52 us).
constexpr unsigned kGroupVocab = 2048;

template <typename T, bool LOSS, int NV>
__global__ __launch_bounds__(256, 4) void policy_group_kernel(PolicyArgs a, unsigned lanes_log2) {
  __shared__ double red[4][5];
  const unsigned lanes = 1u << lanes_log2, sub = threadIdx.x & (lanes - 1);
  const size_t per_block = 256u >> lanes_log2;
  double sum[5] = {0, 0, 0, 0, 0};
  for (size_t row0 = blockIdx.x * per_block; row0 < a.rows; row0 += gridDim.x * per_block) {
    const size_t place = row0 + (threadIdx.x >> lanes_log2), row = min(place, a.rows - 1);   // every lane stays, for the permutations
    const bool live = place < a.rows;
    const T *in = (const T *)a.logits + (int64_t)row * a.stride;
    const Span at = span_of(in, a.vocab, a.vocab < NV * 8 * lanes);
    Raw8<T> r[NV];
    load_row<NV>(r, in, sub, lanes, at);
    const int64_t action = a.actions[row];
    RowInputs q{};
    if (LOSS) q = row_inputs(a, row);
    const float l_a = action >= 0 && action < (int64_t)a.vocab ? (float)in[at.first + action] : 0.f;
    Softmax w{-__builtin_inff(), 0.f, 0.f};
    const bool plain = row_softmax<NV>(w, r, in, sub * 8, lanes * 8, at);
    const float m = group_max_nan(w.m, lanes);
    rebase(w.m, m, w.s, w.t);
    w = Softmax{m, group_sum(w.s, lanes), group_sum(w.t, lanes)};
    const RowTerms o = row_terms(w, action, a.vocab, l_a);
    if (live && sub == 0) { a.neglogps[row] = o.nlp; a.entropies[row] = o.ent; }
    if (!LOSS) continue;
    const RowShare share = row_objective(a, q, o);
    if (live && sub == 0) {
      a.dvalues[row] = share.dvalue;
      for (int i = 0; i < 5; ++i) sum[i] += share.part[i];
    }
    const GradTerms k = grad_terms(a, w.m, o, share.g);
    write_gradient<NV>(r, k, (T *)a.dlogits + (int64_t)row * a.dstride - at.first, sub, lanes, live ? at : Span{0, 0}, action + at.first, plain);
  }
  if (LOSS) put_block(a, sum, red);
}

// One workgroup per row, statistics only: the row streams through registers once, a few vectors a thread at a time.
template <typename T, int THREADS, int kStatsVecs>
__global__ __launch_bounds__(THREADS) void policy_stats_row_kernel(PolicyArgs a) {
  __shared__ Softmax red[16];
  const size_t row = blockIdx.x;
  const T *in = (const T *)a.logits + (int64_t)row * a.stride;
  const int64_t action = a.actions[row];
  const float l_a = action >= 0 && action < (int64_t)a.vocab ? (float)in[action] : 0.f;
  const Span at = span_of(in, a.vocab);
  Softmax w{-__builtin_inff(), 0.f, 0.f};
  if (action != -1)
    for (unsigned e0 = 0; e0 < at.end; e0 += kStatsVecs * THREADS * 8) {
      Raw8<T> r[kStatsVecs];
      const Span part{e0 ? 0u : at.first, min(at.end - e0, kStatsVecs * THREADS * 8u)};
      load_row<kStatsVecs>(r, in + e0, threadIdx.x, THREADS, part);
      Softmax q{-__builtin_inff(), 0.f, 0.f};
      row_softmax<kStatsVecs, true>(q, r, in + e0, threadIdx.x * 8, THREADS * 8, part);
      const float m = __builtin_elementwise_maximum(w.m, q.m);
      rebase(w.m, m, w.s, w.t);
      rebase(q.m, m, q.s, q.t);
      w = Softmax{m, w.s + q.s, w.t + q.t};
    }
  w = block_softmax(w, red);
  const RowTerms o = row_terms(w, action, a.vocab, l_a);
  if (threadIdx.x == 0) { a.neglogps[row] = o.nlp; a.entropies[row] = o.ent; }
}

// One workgroup per row, the whole row in registers (NV vectors of 8 a thread): read once, the gradient written from there.
// Rows of up to half the registers leave room for a second workgroup, which loads while the first computes.  4096 x 50001 bf16 with
// padding rows: 148 us, 761 MB; the vector unit is busy for 68 % of it, two powers an element.
template <typename T, int NV>
__global__ __launch_bounds__(1024, NV * sizeof(Raw8<T>) <= 128 ? 8 : 4) void policy_loss_row_kernel(PolicyArgs a) {
  __shared__ Softmax red[16];
  const size_t row = blockIdx.x;
  const unsigned tid = threadIdx.x, threads = blockDim.x;
  const T *in = (const T *)a.logits + (int64_t)row * a.stride;
  const int64_t action = a.actions[row];
  const float l_a = action >= 0 && action < (int64_t)a.vocab ? (float)in[action] : 0.f;
  const RowInputs q = row_inputs(a, row);
  const Span at = span_of(in, a.vocab);
  Raw8<T> r[NV];
  bool plain = false;
  Softmax w{-__builtin_inff(), 0.f, 0.f};
  if (action != -1) {
    load_row<NV>(r, in, tid, threads, at);
    plain = row_softmax<NV>(w, r, in, tid * 8, threads * 8, at);
  }
  w = block_softmax(w, red);
  const RowTerms o = row_terms(w, action, a.vocab, l_a);
  const RowShare share = row_objective(a, q, o);
  if (tid == 0) put_row(a, row, o, share);
  const GradTerms k = grad_terms(a, w.m, o, share.g);
  write_gradient<NV>(r, k, (T *)a.dlogits + (int64_t)row * a.dstride - at.first, tid, threads, at, action + at.first, plain);
}

// Rows too long for the registers of a workgroup: read a second time for the gradient, out of the caches as far as they hold it
// (256 x 262144 f32 167 us, 4.8 TB/s with the second read; bf16 75 us).
template <typename T>
__global__ __launch_bounds__(1024) void policy_loss_long_kernel(PolicyArgs a) {
  __shared__ Softmax red[16];
  const size_t row = blockIdx.x;
  const unsigned tid = threadIdx.x;
  const T *in = (const T *)a.logits + (int64_t)row * a.stride;
  const int64_t action = a.actions[row];
  const float l_a = action >= 0 && action < (int64_t)a.vocab ? (float)in[action] : 0.f;
  const RowInputs q = row_inputs(a, row);
  Softmax w{-__builtin_inff(), 0.f, 0.f};
  if (action != -1)
    for (unsigned e = tid * 8; e < a.vocab; e += 8192) {
      Raw8<T> r;
      load8(r, in + e, (long)(a.vocab - e), -__builtin_inff());
      online(w, r);
    }
  w = block_softmax(w, red);
  const RowTerms o = row_terms(w, action, a.vocab, l_a);
  const RowShare share = row_objective(a, q, o);
  if (tid == 0) put_row(a, row, o, share);
  const GradTerms k = grad_terms(a, w.m, o, share.g);
  T *out = (T *)a.dlogits + (int64_t)row * a.dstride;
  for (unsigned e = tid * 8; e < a.vocab; e += 8192) {
    Raw8<T> r;
    load8(r, in + e, (long)(a.vocab - e), -__builtin_inff());
    gradient8<false>(r, k, (int)(action - e));
    store8(r, out + e, (long)(a.vocab - e));
  }
}

// Few long rows: every row is cut into chunks of kSplitChunk tokens, a workgroup each; the chunks' (m, s, t) meet in a second
// launch, whose workgroups join all chunks of their row themselves.
constexpr unsigned kSplitChunk = 4096;
constexpr int kSplitVecs = kSplitChunk / 2048;

template <typename T>
__global__ __launch_bounds__(256) void policy_split_kernel(PolicyArgs a, unsigned chunks, Softmax *parts, float *picked) {
  __shared__ Softmax red[16];
  const size_t row = blockIdx.x / chunks;
  const unsigned c0 = (blockIdx.x % chunks) * kSplitChunk;
  const T *in = (const T *)a.logits + (int64_t)row * a.stride;
  Raw8<T> r[kSplitVecs];
  Softmax w{-__builtin_inff(), 0.f, 0.f};
  const unsigned len = min(a.vocab - c0, kSplitChunk);
  load_row<kSplitVecs>(r, in + c0, threadIdx.x, 256, Span{0, len});
  row_softmax<kSplitVecs, true>(w, r, in + c0, threadIdx.x * 8, 2048, Span{0, len});
  w = block_softmax(w, red);
  if (threadIdx.x == 0) {
    parts[blockIdx.x] = w;
    const int64_t action = a.actions[row];           // its logit is put aside here: the gradient may be written over the logits
    if (action >= (int64_t)c0 && action < (int64_t)min(a.vocab, c0 + kSplitChunk)) picked[row] = (float)in[action];
    if (blockIdx.x == 0) *a.ticket = 0;
  }
}

__device__ __forceinline__ Softmax join_chunks(const Softmax *parts, unsigned chunks) {   // one wave, every lane gets the result
  Softmax w{-__builtin_inff(), 0.f, 0.f};
  for (unsigned c = threadIdx.x % 64; c < chunks; c += 64) {
    Softmax q = parts[c];
    const float m = __builtin_elementwise_maximum(w.m, q.m);
    rebase(w.m, m, w.s, w.t);
    rebase(q.m, m, q.s, q.t);
    w = Softmax{m, w.s + q.s, w.t + q.t};
  }
  return wave_softmax(w);
}

__global__ __launch_bounds__(64) void policy_join_kernel(PolicyArgs a, unsigned chunks, const Softmax *parts, const float *picked) {
  const size_t row = blockIdx.x;
  const RowTerms o = row_terms(join_chunks(parts + row * chunks, chunks), a.actions[row], a.vocab, picked[row]);
  if (threadIdx.x == 0) { a.neglogps[row] = o.nlp; a.entropies[row] = o.ent; }
}

template <typename T>
__global__ __launch_bounds__(256) void policy_split_loss_kernel(PolicyArgs a, unsigned chunks, const Softmax *parts, const float *picked) {
  const size_t row = blockIdx.x / chunks;
  const unsigned chunk = blockIdx.x % chunks, c0 = chunk * kSplitChunk, tid = threadIdx.x;
  const T *in = (const T *)a.logits + (int64_t)row * a.stride;
  T *out = (T *)a.dlogits + (int64_t)row * a.dstride;
  Raw8<T> r[kSplitVecs];
  const unsigned len = min(a.vocab - c0, kSplitChunk);
  load_row<kSplitVecs>(r, in + c0, tid, 256, Span{0, len});
  const RowInputs q = row_inputs(a, row);
  const int64_t action = a.actions[row];
  const Softmax w = join_chunks(parts + row * chunks, chunks);
  const RowTerms o = row_terms(w, action, a.vocab, picked[row]);
  const RowShare share = row_objective(a, q, o);
  if (chunk == 0 && tid == 0) put_row(a, row, o, share);
  const GradTerms k = grad_terms(a, w.m, o, share.g);
  write_gradient<false, kSplitVecs>(r, k, out + c0, tid, 256, Span{0, len}, action - c0);
}

// Sums the records in a fixed order, in 64 bits: each workgroup a slice, three waves a column; the last workgroup to finish adds
// the slices.
constexpr unsigned kStatsBlocks = 64, kStatsSlice = 8192;

__device__ __forceinline__ void sum_records(const double *p, size_t stride, size_t begin, size_t end, double s[5], double *red) {
  const unsigned wave = threadIdx.x / 64, column = wave / 3;
  double x = 0;
  for (size_t i = begin + (wave % 3) * 64 + threadIdx.x % 64; i < end; i += 8 * 192) {   // eight loads on their way at a time
    double v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = p[column * stride + min(i + j * 192, end - 1)];
#pragma unroll
    for (int j = 0; j < 8; ++j) x += i + j * 192 < end ? v[j] : 0.;
  }
  x = wave_sum(x);
  __syncthreads();
  if (threadIdx.x % 64 == 0) red[wave] = x;
  __syncthreads();
  for (int k = 0; k < 5; ++k) s[k] = red[3 * k] + red[3 * k + 1] + red[3 * k + 2];
}

__global__ __launch_bounds__(960) void policy_stats_kernel(const double *partials, size_t n, double *slices, unsigned *ticket, double denom, float vf,
                                                           float ent, float *stats) {
  __shared__ double red[15];
  __shared__ unsigned last;
  double s[5];
  const size_t per = (n + gridDim.x - 1) / gridDim.x;
  sum_records(partials, n, min(n, blockIdx.x * per), min(n, (blockIdx.x + 1) * per), s, red);
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) {
      for (int k = 0; k < 5; ++k) slices[k * kStatsBlocks + blockIdx.x] = s[k];
      __threadfence();
      last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    sum_records(slices, kStatsBlocks, 0, gridDim.x, s, red);
  }
  if (threadIdx.x >= 6) return;                      // a division each, side by side
  double x = s[0] + (double)vf * s[1] - (double)ent * s[2];
#pragma unroll
  for (int k = 0; k < 5; ++k) x = threadIdx.x == 1 + k ? s[k] : x;
  stats[threadIdx.x] = (float)(x / denom);
}

// ---- host -----------------------------------------------------------------------------------------------------------------

bool is_divisor(float x) { return x >= kLeastDivisor && std::isfinite(x); }

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
  if (!is_divisor(r->repetition) || !is_divisor(r->temperature))
    return ppoxp_fail(PPO_XP_EINVAL, "%s: repetition %g and temperature %g must be finite and at least 2^-126", who, r->repetition, r->temperature);
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

template <typename T, bool HIST, int MODE>
void launch_shape(const ShapeArgs &a, dim3 grid, bool narrow, hipStream_t s) {
  constexpr int WIDE = std::is_same<T, float>::value && !HIST ? 1 : 4;       // never wide: see shape()
  if (narrow && a.rows_per > 1) hipLaunchKernelGGL((shape_logits_kernel<T, HIST, MODE, true, 1>), grid, dim3(256), 0, s, a);
  else if (narrow) hipLaunchKernelGGL((shape_logits_kernel<T, HIST, MODE, false, 1>), grid, dim3(256), 0, s, a);
  else if (a.rows_per > 1) hipLaunchKernelGGL((shape_logits_kernel<T, HIST, MODE, true, WIDE>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((shape_logits_kernel<T, HIST, MODE, false, WIDE>), grid, dim3(256), 0, s, a);
}
template <typename T>
void launch_shape(const ShapeArgs &a, dim3 grid, bool narrow, hipStream_t s, bool hist, bool backward) {
  if (!backward) hist ? launch_shape<T, true, kForward>(a, grid, narrow, s) : launch_shape<T, false, kForward>(a, grid, narrow, s);
  else if (!hist) launch_shape<T, false, kGather>(a, grid, narrow, s);
  // Fetching the logits of seen tokens one by one costs as much as reading them all at about a token in 50 (2048 x 50001 bf16, us one
  // by one against all: 133 and 132 at 1024 tokens a row, 164 and 134 at 2048, 232 and 157 at 4096); histories may be partly filled.
  else if ((uint64_t)a.r.hist_len * 32 < a.vocab) launch_shape<T, true, kGather>(a, grid, narrow, s);
  else launch_shape<T, true, kReadAll>(a, grid, narrow, s);
}

int shape(const char *who, int device, void *stream, int dtype, ShapeArgs &a, size_t rows, size_t vocab, const ppo_xp_logit_rules *rules,
          bool backward) {
  if (int rc = check_rules(who, rules, rows, vocab)) return rc;
  if (rows == 0 || vocab == 0) return 0;
  a.rows = rows;
  a.vocab = (unsigned)vocab;
  a.units = (unsigned)((vocab + 7) / 8);
  const bool hist = rules->history && rules->hist_rows > 0 && rules->hist_len > 0;
  // A workgroup's part is 8192 elements, or 2048 where a row is no longer than that, where 8192 leave CUs idle, and for f32 without a
  // history, whose wider elements fill a wave's loads by themselves.  In us a call, parts of 8192 | 2048: f32 without a history
  // 4096 x 151 8.2 | 4.1, 16384 x 4000 102 | 96, 2048 x 50001 158 | 149; bf16 with a history of 1024 tokens 4096 x 151 13.8 | 6.6,
  // 65536 x 1000 143 | 134, 8 x 131072 5.8 | 4.3, 64 x 32768 (256 workgroups of 8192) 6.0 | 5.3, 32 x 131072 (512) 6.7 | 7.8,
  // 16384 x 4000 80 | 91, 1024 x 131072 117 | 168.
  const unsigned long_chunks = (a.units + shape_chunk(4) / 8 - 1) / (shape_chunk(4) / 8);
  const bool narrow = a.units <= shape_chunk(1) / 8 || (dtype == PPO_XP_F32 && !hist) || rows * long_chunks <= 256;
  const unsigned part = shape_chunk(narrow ? 1 : 4) / 8;
  a.chunks = (a.units + part - 1) / part;
  // rows that fill less than half a workgroup's part share one (one workgroup a row: 113 us at 262144 x 32 bf16)
  a.rows_per = (unsigned)std::min<size_t>(part / std::min(a.units, part), rows);
  // workgroups go to the 8 XCDs in turn, and of an even number of chunks a short last one is always the same XCDs': equal parts then
  // (4096 x 10000 f32 with a history, 8192 and 1808: 91 us, 5056 and 4944: 71; with an odd number they cost 2048 x 50001 bf16 16 %)
  a.part = a.chunks % 2 ? part * 8 : ((a.units + a.chunks - 1) / a.chunks + 7) / 8 * 64;
  const size_t blocks = a.rows_per > 1 ? rows / a.rows_per + (rows % a.rows_per != 0) : rows * a.chunks;
  if (rows > kMaxRows || !one_launch(blocks, 256)) return ppoxp_fail(PPO_XP_EINVAL, "%s: %zu rows of %zu are too many for one launch", who, rows, vocab);
  a.magic = ((1u << 20) + a.units - 1) / a.units;
  a.scan_log2 = 8;
  while (a.scan_log2 && (256u >> a.scan_log2) < a.rows_per) --a.scan_log2;
  a.r = *rules;
  DeviceGuard dev(device, who);
  if (dev.rc()) return dev.rc();
  const dim3 grid((unsigned)blocks);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_shape<float>(a, grid, narrow, s, hist, backward);
  else if (dtype == PPO_XP_BF16) launch_shape<__bf16>(a, grid, narrow, s, hist, backward);
  else launch_shape<_Float16>(a, grid, narrow, s, hist, backward);
  return launched(who);
}

// Which kernels a call takes, and what they need.
enum Route { kSmall, kGroup, kRow, kSplit };

struct Plan {
  Route route = kRow;
  unsigned lanes_log2 = 0, chunks = 0;             // kGroup: lanes of a row; kSplit: chunks of a row
  unsigned blocks = 0;                             // kSmall, kGroup: workgroups, which walk over the rows
  size_t records = 0;                              // of the objective
  size_t o_slices = 0, o_ticket = 0, o_parts = 0, o_picked = 0, bytes = 0;
};

// Few long rows leave most of the 256 CUs idle with a workgroup each; the split costs a launch more (2 us of the host's time, which
// bounds all of these up to 32 rows) and a second read out of the caches.  Measured in us a call, one workgroup a row | split:
// statistics of 8 x 65536 f32 6.2 | 8.3, bf16 6.7 | 8.4, 8 x 131072 f32 8.9 | 8.3, bf16 10.6 | 8.1, 100 x 131072 f32 13.4 | 12.4,
// 128 x 131072 bf16 11.9 | 11.8; objective of 8 x 50001 f32 11.6 | 12.4, bf16 13.0 | 12.2, 8 x 131072 f32 27.6 | 12.5,
// 100 x 131072 bf16 22.0 | 20.1, 128 x 131072 bf16 22.8 | 23.7.
constexpr size_t kSplitRows = 128, kSplitLoss = 65536, kSplitStats = 98304;   // rows, tokens

constexpr size_t kTurnedVocab = 768, kTurnedWork = size_t(1) << 24;   // tokens, elements

Plan plan_of(size_t rows, size_t vocab, bool loss, bool wide) {   // wide: f32
  Plan p;
  if (vocab <= kGroupVocab) {
    unsigned lanes = 1;
    while (32 * lanes < vocab) lanes *= 2;
    // Rows whose vectors of 8 the lanes of policy_group_kernel share out evenly are its own; others are cheaper turned, for 16 bits up to 128
    // tokens only (a lane reads less at a time there).  us for 2^25 elements, in groups | turned: objective f32 x 64 75 | 59, x 100 94 | 64,
    // x 128 61 | 58, x 151 77 | 61, x 192 57 | 72, x 600 62 | 61, bf16 x 64 62 | 49, x 100 74 | 58, x 128 35 | 50, x 151 52 | 53,
    // x 300 47 | 53; statistics f32 x 64 31 | 30, x 100 35 | 32, x 151 37 | 31, x 256 25 | 29, x 600 37 | 30, bf16 x 64 17 | 21,
    // x 100 22 | 26, x 151 24 | 24.  For 2^22 elements: objective f32 x 100 16.8 | 16.6, x 151 15.6 | 16.8, for 2^20 10.2 | 10.8, 9.6 | 11.8.
    const bool even = vocab % (8 * lanes) == 0;
    const bool turned = vocab <= 48 || (loss && vocab <= 64) || (!even && vocab <= (wide ? kTurnedVocab : loss ? 128 : 0) && rows >= kTurnedWork / vocab);
    p.route = turned ? kSmall : kGroup;
    while ((turned ? 48u : 32u) << p.lanes_log2 < vocab) ++p.lanes_log2;
    const size_t per = 256u >> p.lanes_log2;
    p.blocks = (unsigned)std::min<size_t>((rows + per - 1) / per, kGroupBlocks);
  } else if (rows < kSplitRows && vocab > (loss ? kSplitLoss : kSplitStats)) {
    p.route = kSplit;
    p.chunks = (unsigned)((vocab + kSplitChunk - 1) / kSplitChunk);
  }
  p.records = p.blocks ? p.blocks : rows;
  if (loss) p.bytes = p.records * 5 * sizeof(double);
  p.o_slices = p.bytes;
  if (loss) p.bytes += kStatsBlocks * 5 * sizeof(double);
  p.o_ticket = p.bytes;
  if (loss || p.route == kSplit) p.bytes += 16;
  p.o_parts = p.bytes;
  if (p.route == kSplit) p.bytes += rows * p.chunks * sizeof(Softmax);
  p.o_picked = p.bytes;
  if (p.route == kSplit) p.bytes += rows * sizeof(float);
  return p;
}

template <typename T, bool LOSS>
void launch_group(const Plan &p, const PolicyArgs &a, hipStream_t s) {
  const dim3 grid(p.blocks), block(256);
  if (p.route == kGroup) {
    const unsigned vecs = ((a.vocab + 7) / 8 + (1u << p.lanes_log2) - 1) >> p.lanes_log2;
    if (vecs <= 3) hipLaunchKernelGGL((policy_group_kernel<T, LOSS, 3>), grid, block, 0, s, a, p.lanes_log2);
    else hipLaunchKernelGGL((policy_group_kernel<T, LOSS, 4>), grid, block, 0, s, a, p.lanes_log2);
    return;
  }
  const unsigned magic = ((1u << 22) + a.vocab - 1) / a.vocab;       // exact for the 64 * 48 elements of a wave, at most, and 768 tokens
  const unsigned slots = (a.vocab + (1u << p.lanes_log2) - 1) >> p.lanes_log2;
  if (p.lanes_log2) {
    if constexpr (LOSS || std::is_same<T, float>::value) {      // see plan_of
      if (slots <= 32) hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 32, true>), grid, block, 0, s, a, magic, p.lanes_log2);
      else if (slots <= 40) hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 40, true>), grid, block, 0, s, a, magic, p.lanes_log2);
      else hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 48, true>), grid, block, 0, s, a, magic, p.lanes_log2);
    }
    return;
  }
  switch (slots <= 32 ? (slots + 3) / 4 : (slots + 7) / 8 * 2) {
    case 1: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 4, false>), grid, block, 0, s, a, magic, 0); break;
    case 2: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 8, false>), grid, block, 0, s, a, magic, 0); break;
    case 3: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 12, false>), grid, block, 0, s, a, magic, 0); break;
    case 4: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 16, false>), grid, block, 0, s, a, magic, 0); break;
    case 5: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 20, false>), grid, block, 0, s, a, magic, 0); break;
    case 6: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 24, false>), grid, block, 0, s, a, magic, 0); break;
    case 7: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 28, false>), grid, block, 0, s, a, magic, 0); break;
    case 8: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 32, false>), grid, block, 0, s, a, magic, 0); break;
    case 10: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 40, false>), grid, block, 0, s, a, magic, 0); break;
    default: hipLaunchKernelGGL((policy_small_kernel<T, LOSS, 48, false>), grid, block, 0, s, a, magic, 0);
  }
}

template <typename T>
void launch_stats(const Plan &p, const PolicyArgs &a, Softmax *parts, float *picked, hipStream_t s) {
  const unsigned rows = (unsigned)a.rows;
  if (p.blocks) launch_group<T, false>(p, a, s);
  else if (p.route == kSplit) {
    hipLaunchKernelGGL(policy_split_kernel<T>, dim3(rows * p.chunks), dim3(256), 0, s, a, p.chunks, parts, picked);
    hipLaunchKernelGGL(policy_join_kernel, dim3(rows), dim3(64), 0, s, a, p.chunks, (const Softmax *)parts, (const float *)picked);
  } else if (a.vocab < kSplitChunk) hipLaunchKernelGGL((policy_stats_row_kernel<T, 256, 1>), dim3(rows), dim3(256), 0, s, a);
  else if (a.vocab < 2 * kSplitChunk) hipLaunchKernelGGL((policy_stats_row_kernel<T, 256, 2>), dim3(rows), dim3(256), 0, s, a);
  else if (rows < 256 && a.vocab <= 32768) hipLaunchKernelGGL((policy_stats_row_kernel<T, 1024, 4>), dim3(rows), dim3(1024), 0, s, a);
  else if (rows < 256) hipLaunchKernelGGL((policy_stats_row_kernel<T, 1024, 8>), dim3(rows), dim3(1024), 0, s, a);
  else hipLaunchKernelGGL((policy_stats_row_kernel<T, 256, 4>), dim3(rows), dim3(256), 0, s, a);
}

// Vectors a thread: the choice that keeps most rows in a CU at once, whose phases then overlap; of equal ones the smallest.
// `kWaves`: waves a CU holds of the kernel with that many vectors (its registers: 22 and 4 a vector, 8 of floats).
constexpr int row_waves(int regs) { return 512 / ((regs + 7) / 8 * 8) >= 8 ? 32 : 512 / ((regs + 7) / 8 * 8) * 4; }

struct RowChoice { int registers; unsigned threads; };    // 16-byte registers of a thread's vectors; 0: the row is too long for them

template <typename T>
RowChoice row_choice(const PolicyArgs &a) {
  constexpr int kScale = sizeof(T) / 2;                 // 16-byte registers of 8 elements
  static const int choices[] = {4, 6, 8, 10, 12, 14, 16};
  const bool odd = (uintptr_t)a.logits % 4 || (a.rows > 1 && a.stride * sizeof(T) % 4);   // some row starts with half a word
  const unsigned vecs = (a.vocab + odd + 7) / 8;
  RowChoice best{0, 1024};
  int rows = 0;
  for (int c : choices) {
    const unsigned waves = (vecs + c / kScale * 64 - 1) / (c / kScale * 64);
    const int held = waves <= 16 ? row_waves(22 + 4 * c) / (int)waves : 0;
    if (held > rows) { rows = held; best = RowChoice{c, waves * 64}; }
  }
  return best;
}

template <typename T, int NV>
void launch_row_as(const PolicyArgs &a, unsigned threads, hipStream_t s) {
  hipLaunchKernelGGL((policy_loss_row_kernel<T, NV>), dim3((unsigned)a.rows), dim3(threads), 0, s, a);
}

template <typename T>
void launch_row(const PolicyArgs &a, hipStream_t s) {
  constexpr int kScale = sizeof(T) / 2;
  const RowChoice r = row_choice<T>(a);
  switch (r.registers) {
    case 4: launch_row_as<T, 4 / kScale>(a, r.threads, s); break;
    case 6: launch_row_as<T, 6 / kScale>(a, r.threads, s); break;
    case 8: launch_row_as<T, 8 / kScale>(a, r.threads, s); break;
    case 10: launch_row_as<T, 10 / kScale>(a, r.threads, s); break;
    case 12: launch_row_as<T, 12 / kScale>(a, r.threads, s); break;
    case 14: launch_row_as<T, 14 / kScale>(a, r.threads, s); break;
    case 16: launch_row_as<T, 16 / kScale>(a, r.threads, s); break;
    default: hipLaunchKernelGGL(policy_loss_long_kernel<T>, dim3((unsigned)a.rows), dim3(r.threads), 0, s, a); break;
  }
}

// Whether the call's largest launch can be dispatched; `threads`: of a row's workgroup where it has one.
bool fits(const Plan &p, size_t rows, unsigned threads) {
  if (rows > kMaxRows) return false;
  return p.blocks || (p.route == kSplit ? one_launch(rows * p.chunks, 256) : one_launch(rows, threads));
}

template <typename T>
void launch_loss(const Plan &p, const PolicyArgs &a, Softmax *parts, float *picked, hipStream_t s) {
  const unsigned rows = (unsigned)a.rows;
  if (p.blocks) launch_group<T, true>(p, a, s);
  else if (p.route == kSplit) {
    hipLaunchKernelGGL(policy_split_kernel<T>, dim3(rows * p.chunks), dim3(256), 0, s, a, p.chunks, parts, picked);
    hipLaunchKernelGGL(policy_split_loss_kernel<T>, dim3(rows * p.chunks), dim3(256), 0, s, a, p.chunks, (const Softmax *)parts, (const float *)picked);
  } else launch_row<T>(a, s);
}

int check_workspace(const char *who, const Plan &p, const void *ws, size_t bytes) {
  if (p.bytes && (!ws || bytes < p.bytes || (uintptr_t)ws % 16))
    return ppoxp_fail(PPO_XP_EINVAL, "%s: workspace of %zu bytes, 16-byte aligned, expected (%zu given)", who, p.bytes, bytes);
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

size_t ppo_xp_policy_workspace(size_t rows, size_t vocab, int loss) {
  return rows && vocab ? std::max(plan_of(rows, vocab, loss != 0, false).bytes, plan_of(rows, vocab, loss != 0, true).bytes) : 0;
}

int ppo_xp_action_stats(int device, void *stream, int dtype, const void *logits, int64_t logits_stride, const int64_t *actions,
                        float *neglogps, float *entropies, size_t rows, size_t vocab, void *workspace, size_t workspace_bytes) {
  if (int rc = check_rows("action_stats", dtype, logits, logits_stride, rows, vocab)) return rc;
  if (rows == 0 || vocab == 0) return 0;
  if (!actions || !neglogps || !entropies) return ppoxp_fail(PPO_XP_EINVAL, "action_stats: NULL argument");
  const Plan p = plan_of(rows, vocab, false, dtype == PPO_XP_F32);
  if (!fits(p, rows, 256))                                   // 1024 threads a row only below 256 rows
    return ppoxp_fail(PPO_XP_EINVAL, "action_stats: %zu rows of %zu are too many for one launch", rows, vocab);
  if (int rc = check_workspace("action_stats", p, workspace, workspace_bytes)) return rc;
  PolicyArgs a{};
  a.logits = logits; a.stride = logits_stride; a.actions = actions; a.neglogps = neglogps; a.entropies = entropies;
  a.vocab = (unsigned)vocab; a.rows = rows;
  DeviceGuard dev(device, "action_stats");
  if (dev.rc()) return dev.rc();
  char *ws = (char *)workspace;
  a.ticket = (unsigned *)(ws + p.o_ticket);
  Softmax *parts = (Softmax *)(ws + p.o_parts);
  float *picked = (float *)(ws + p.o_picked);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_stats<float>(p, a, parts, picked, s);
  else if (dtype == PPO_XP_BF16) launch_stats<__bf16>(p, a, parts, picked, s);
  else launch_stats<_Float16>(p, a, parts, picked, s);
  return launched("action_stats");
}

int ppo_xp_policy_loss(int device, void *stream, int dtype, const void *logits, int64_t logits_stride, const ppo_xp_policy_batch *b,
                       float clip, float ent_coef, float vf_coef, double denom, void *dlogits, int64_t dlogits_stride, float *dvalues,
                       float *neglogps, float *entropies, float *stats, size_t rows, size_t vocab, void *workspace, size_t workspace_bytes) {
  if (int rc = check_rows("policy_loss", dtype, logits, logits_stride, rows, vocab)) return rc;
  if (int rc = check_rows("policy_loss", dtype, dlogits, dlogits_stride, rows, vocab)) return rc;
  if (!(clip >= 0.f) || !std::isfinite(clip) || !std::isfinite(ent_coef) || !std::isfinite(vf_coef))
    return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: clip %g (>= 0), ent_coef %g and vf_coef %g must be finite", clip, ent_coef, vf_coef);
  if (!(denom > 0.) || !std::isfinite(denom) || !std::isfinite((float)(1. / denom)))     // gradients are scaled by the 32-bit 1 / denom
    return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: denom %g must be finite and at least 2^-127", denom);
  if (rows == 0 || vocab == 0) return 0;
  if (!b || !b->actions || !b->old_values || !b->old_neglogps || !b->returns || !b->advantages || !b->values || !dvalues || !neglogps ||
      !entropies || !stats)
    return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: NULL argument");
  const Plan p = plan_of(rows, vocab, true, dtype == PPO_XP_F32);
  PolicyArgs a{};
  a.logits = logits; a.stride = logits_stride; a.actions = b->actions; a.neglogps = neglogps; a.entropies = entropies;
  a.vocab = (unsigned)vocab; a.rows = rows;
  a.old_values = b->old_values; a.old_neglogps = b->old_neglogps; a.returns = b->returns; a.advantages = b->advantages; a.values = b->values;
  a.clip = clip; a.ent_coef = ent_coef; a.vf_coef = vf_coef; a.inv_denom = (float)(1. / denom);
  a.dlogits = dlogits; a.dstride = dlogits_stride; a.dvalues = dvalues; a.partials = (double *)workspace;
  // threads of a row: 1024 at most, which fewer rows fit with; of the type its size matters
  const unsigned threads = rows >> 22 == 0 ? 1024 : (dtype == PPO_XP_F32 ? row_choice<float>(a) : row_choice<__bf16>(a)).threads;
  if (!fits(p, rows, threads))
    return ppoxp_fail(PPO_XP_EINVAL, "policy_loss: %zu rows of %zu are too many for one launch", rows, vocab);
  if (int rc = check_workspace("policy_loss", p, workspace, workspace_bytes)) return rc;
  DeviceGuard dev(device, "policy_loss");
  if (dev.rc()) return dev.rc();
  char *ws = (char *)workspace;
  a.ticket = (unsigned *)(ws + p.o_ticket);
  Softmax *parts = (Softmax *)(ws + p.o_parts);
  float *picked = (float *)(ws + p.o_picked);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_loss<float>(p, a, parts, picked, s);
  else if (dtype == PPO_XP_BF16) launch_loss<__bf16>(p, a, parts, picked, s);
  else launch_loss<_Float16>(p, a, parts, picked, s);
  const unsigned slices = (unsigned)std::min<size_t>((p.records + kStatsSlice - 1) / kStatsSlice, kStatsBlocks);
  hipLaunchKernelGGL(policy_stats_kernel, dim3(slices), dim3(960), 0, s, (const double *)a.partials, p.records, (double *)(ws + p.o_slices), a.ticket,
                     denom, vf_coef, ent_coef, stats);
  return launched("policy_loss");
}

}  // extern "C"

// Observation rows in 8 or 4 bits: quantised as they are written, gathered and read back by a minibatch's indices.
// Formats and the rounding are defined in include/ppo_xp.h.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ops_common.h"

namespace {

using namespace ppoxp_ops;

typedef u32x2 u32x2_a1 __attribute__((aligned(1)));
typedef unsigned u32_a1 __attribute__((aligned(1)));
typedef unsigned short u16_a1 __attribute__((aligned(1)));

// Units of a launch (16 bytes of output or 8 elements) lie row after row, `slots` to a row; a workgroup takes 256 * U of them.
struct Units {
  size_t total, row0;
  unsigned slots, off;       // the workgroup's first unit is unit `off` of row0
  float inv;
  __device__ __forceinline__ Units(size_t total_, unsigned slots_, unsigned per_block) : total(total_), slots(slots_) {
    const size_t first = (size_t)blockIdx.x * per_block;
    row0 = total >> 32 ? first / slots : (unsigned)first / slots;
    off = (unsigned)(first - row0 * slots);
    inv = 1.f / (float)slots;
  }
  // Unit k * 256 + thread: its row and its place there; false beyond the last one.  (Exact: off + k * 256 + thread < 2^24.)
  __device__ __forceinline__ bool at(int k, size_t &row, unsigned &slot) const {
    const unsigned t = off + k * 256 + threadIdx.x;
    unsigned q = (unsigned)((float)t * inv), r = t - q * slots;
    if ((int)r < 0) { --q; r += slots; }
    if (r >= slots) { ++q; r -= slots; }
    row = row0 + q;
    slot = r;
    return (row0 * slots + t) < total;
  }
};

struct QuantArgs {
  const void *rows;
  uint8_t *codes;
  float *scales;
  int64_t rows_stride, codes_stride, scales_stride;   // elements, bytes, floats
  size_t total;                                       // n * slots
  unsigned width, slots, lanes_log2;                  // slots of 8 elements per row (whole groups), lanes of one group
  size_t at;
};

// Nearest integer to x / s, ties to even, exactly: the product with the rounded reciprocal can be on the wrong side of a
// border; the remainder x - q s is exact in one fma (|q| <= 127, |remainder| <= s / 2 up to one rounding of q) and says so.
__device__ __forceinline__ int round_quotient(float x, float s, float inv, float half) {
  float q = __builtin_rintf(x * inv);
  const float r = __builtin_fmaf(-q, s, x);
  if (__builtin_fabsf(r) >= half) {
    const float up = r > 0.f ? 1.f : -1.f;
    if (__builtin_fabsf(r) > half || ((int)q & 1)) q += up;
  }
  return (int)q;
}

// One lane holds 8 elements, group / 8 neighbouring lanes one group: the group's largest magnitude is found with lane
// shuffles and the row is read once.  Magnitudes are compared as integers, which puts NaN and inf above every number.
template <typename T, int FORMAT, int U>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
  const Units units(a.total, a.slots, 256 * U);
  Raw8<T> raw[U];
  size_t row[U];
  unsigned e[U], top[U];
  long left[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const bool live = units.at(k, row[k], e[k]);
    e[k] *= 8;
    left[k] = live ? (long)a.width - (long)e[k] : 0;
    const T *p = (const T *)a.rows + (int64_t)row[k] * a.rows_stride;
    if (left[k] >= 8) {
      raw[k].load(p + e[k]);
    } else {                                           // a row's end, or beyond it: clamped addresses, no further branch
      p = (const T *)a.rows + (int64_t)(live ? row[k] : 0) * a.rows_stride;
      T q[8];
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = p[min(e[k] + i, a.width - 1)];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = i < left[k] ? (float)q[i] : 0.f;
      raw[k].set8(y);
    }
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    top[k] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top[k] = max(top[k], __builtin_bit_cast(unsigned, raw[k].get(i)) & 0x7fffffffu);
    top[k] = group_max_bits(top[k], 1u << a.lanes_log2);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const bool empty = top[k] < (17u << 23), bad = top[k] >= 0x7f800000u;   // below 2^-110 | NaN or inf
    float s, inv;
    if (FORMAT == PPO_XP_Q_E4M3) {
      // top = 1.m 2^E <= 448 2^k = 1.75 2^(8+k)
      const unsigned k127 = (top[k] >> 23) - 8 + ((top[k] & 0x7fffffu) > 0x600000u ? 1 : 0);
      s = __builtin_bit_cast(float, k127 << 23);
      inv = __builtin_bit_cast(float, (254 - k127) << 23);
    } else {
      s = __builtin_bit_cast(float, top[k]) / (FORMAT == PPO_XP_Q_INT8 ? 127.f : 7.f);
      inv = 1.f / s;
    }
    if (empty || bad) { s = bad ? __builtin_nanf("") : 0.f; inv = 0.f; }
    if (left[k] <= 0) continue;
    if (((e[k] >> 3) & ((1u << a.lanes_log2) - 1)) == 0)
      a.scales[(int64_t)(a.at + row[k]) * a.scales_stride + (e[k] >> (a.lanes_log2 + 3))] = s;
    uint8_t *dst = a.codes + (int64_t)(a.at + row[k]) * a.codes_stride;
    u32x2 w = {0, 0};
    if (inv != 0.f) {
      if (FORMAT == PPO_XP_Q_E4M3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int p = __builtin_amdgcn_cvt_pk_fp8_f32(raw[k].get(4 * h) * inv, raw[k].get(4 * h + 1) * inv, 0, false);
          p = __builtin_amdgcn_cvt_pk_fp8_f32(raw[k].get(4 * h + 2) * inv, raw[k].get(4 * h + 3) * inv, p, true);
          w[h] = (unsigned)p;
        }
      } else {
        const float half = 0.5f * s;
        int q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = round_quotient(raw[k].get(i), s, inv, half);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (FORMAT == PPO_XP_Q_INT4) w[0] |= ((unsigned)q[i] & 15u) << (4 * i);
          else w[i >> 2] |= ((unsigned)q[i] & 255u) << (8 * (i & 3));
        }
      }
    }
    if (FORMAT == PPO_XP_Q_INT4) {
      dst += e[k] / 2;
      if (left[k] >= 8) *(u32_a1 *)dst = w[0];
      else for (int i = 0; i < (int)(left[k] + 1) / 2; ++i) dst[i] = (uint8_t)(w[0] >> (8 * i));
    } else {
      dst += e[k];
      if (left[k] >= 8) *(u32x2_a1 *)dst = w;
      else for (int i = 0; i < (int)left[k]; ++i) dst[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
  }
}

struct DequantArgs {
  const uint8_t *codes;
  const float *scales;
  const void *index;
  void *out;
  int64_t codes_stride, scales_stride, out_stride;
  size_t total, store_rows, at;                       // total = n * slots
  unsigned width, slots, group_log2, index_bits;      // slots of 16 / sizeof(T) elements per row
};

// N codes from element 0 of p on (N 4 or 8, p at an even element), as they lie: 4 bits or 8 each.
template <int FORMAT, int N>
struct Codes {
  static constexpr int kBits = FORMAT == PPO_XP_Q_INT4 ? 4 : 8, kBytes = N * kBits / 8;
  unsigned w[kBytes > 4 ? 2 : 1];
  __device__ __forceinline__ void load(const uint8_t *p) {
    if constexpr (kBytes == 8) { const u32x2 v = *(const u32x2_a1 *)p; w[0] = v.x; w[1] = v.y; }
    else if constexpr (kBytes == 4) w[0] = *(const u32_a1 *)p;
    else w[0] = *(const u16_a1 *)p;
  }
  __device__ __forceinline__ void load(const uint8_t *p, int left) {   // `left` elements, at least one; what is beyond is not read
    const int last = (left * kBits + 7) / 8 - 1;
    unsigned b[kBytes];
#pragma unroll
    for (int i = 0; i < kBytes; ++i) b[i] = p[min(i, last)];
#pragma unroll
    for (unsigned &x : w) x = 0;
#pragma unroll
    for (int i = 0; i < kBytes; ++i) w[i / 4] |= b[i] << (8 * (i % 4));
  }
  __device__ __forceinline__ void values(float v[N]) const {
    if constexpr (FORMAT == PPO_XP_Q_E4M3) {
      typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int h = 0; h < N / 4; ++h) {
        const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
        v[4 * h] = lo.x; v[4 * h + 1] = lo.y; v[4 * h + 2] = hi.x; v[4 * h + 3] = hi.y;
      }
    } else {
      constexpr int kPer = 32 / kBits;
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)((int)(w[i / kPer] << (32 - kBits - kBits * (i % kPer))) >> (32 - kBits));
    }
  }
};

// A code's value as T: the product rounded to 32 bits, then to T.  Left to itself the compiler rounds some of a vector's f16 products
// once, others twice.
template <typename T>
__device__ __forceinline__ T scaled(float v, float s) {
  float p = v * s;
  if constexpr (__is_same(T, _Float16)) asm("" : "+v"(p));
  return (T)p;
}

// One lane writes U times 16 bytes of output, its index entries, codes and scales on their way together.  An index beyond the store
// reads its last row, as the gathers of a pass do.  The output goes past the caches, which keep the store (16384 x 4100 int4 to bf16:
// 35 us, through them 46).
template <typename T, int FORMAT, int U>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(DequantArgs a) {
  constexpr int E = 16 / sizeof(T);
  const Units units(a.total, a.slots, 256 * U);
  size_t row[U], src[U];
  unsigned e[U];
  bool live[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    live[k] = units.at(k, row[k], e[k]);
    e[k] *= E;
    if (!live[k]) { row[k] = 0; e[k] = 0; }
    src[k] = a.at + row[k];
    if (a.index) src[k] = a.index_bits == 32 ? (size_t)((const uint32_t *)a.index)[row[k]] : (size_t)((const uint64_t *)a.index)[row[k]];
  }
  Codes<FORMAT, E> codes[U];
  float s[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    src[k] = min(src[k], a.store_rows - 1);
    const uint8_t *p = a.codes + (int64_t)src[k] * a.codes_stride + (FORMAT == PPO_XP_Q_INT4 ? e[k] / 2 : e[k]);
    s[k] = a.scales[(int64_t)src[k] * a.scales_stride + (e[k] >> a.group_log2)];
    if (e[k] + E <= a.width) codes[k].load(p);
    else codes[k].load(p, (int)(a.width - e[k]));
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    if (!live[k]) continue;
    T *dst = (T *)a.out + (int64_t)row[k] * a.out_stride + e[k];
    float v[E];
    codes[k].values(v);
    if (e[k] + E <= a.width) {
      typedef T vec __attribute__((ext_vector_type(E)));
      typedef vec vec_u __attribute__((aligned(sizeof(T))));
      vec o;
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] = scaled<T>(v[i], s[k]);
      __builtin_nontemporal_store(o, (vec_u *)dst);
    } else {
      for (int i = 0; i < E; ++i)
        if (e[k] + i < a.width) dst[i] = scaled<T>(v[i], s[k]);
    }
  }
}

int log2_of_group(size_t g) {   // 16 .. 512, a power of two; else -1
  for (int k = 4; k <= 9; ++k)
    if (g == (size_t(1) << k)) return k;
  return -1;
}

int check_store(const char *who, int dtype, size_t width, int format, size_t group, const void *codes, int64_t codes_stride,
                const float *scales, int64_t scales_stride) {
  if (!is_dtype(dtype)) return ppoxp_fail(PPO_XP_EINVAL, "%s: unknown element type %d", who, dtype);
  if (format != PPO_XP_Q_INT8 && format != PPO_XP_Q_E4M3 && format != PPO_XP_Q_INT4)
    return ppoxp_fail(PPO_XP_EINVAL, "%s: unknown format %d", who, format);
  if (log2_of_group(group) < 0) return ppoxp_fail(PPO_XP_EINVAL, "%s: group %zu is not a power of two in 16..512", who, group);
  if (width == 0 || width > (size_t(1) << 24)) return ppoxp_fail(PPO_XP_EINVAL, "%s: width %zu (1 .. 2^24 expected)", who, width);
  if (!codes || !scales) return ppoxp_fail(PPO_XP_EINVAL, "%s: NULL store", who);
  const size_t row_bytes = format == PPO_XP_Q_INT4 ? (width + 1) / 2 : width;
  if (codes_stride < (int64_t)row_bytes || scales_stride < (int64_t)((width + group - 1) / group))
    return ppoxp_fail(PPO_XP_EINVAL, "%s: rows of %zu code bytes and %zu scales do not fit strides %lld and %lld", who, row_bytes,
                      (width + group - 1) / group, (long long)codes_stride, (long long)scales_stride);
  return 0;
}

// Several units a lane hide the latency of large calls (a small one would not reach every CU): two where rows are read whole (32768 x
// 4096 bf16: 70 us, with four 88, with one 83), four where they are gathered.
constexpr size_t kManyUnits = size_t(256) * 256 * 4;
constexpr int kWriteUnits = 2, kReadUnits = 4;
size_t blocks_of(size_t total, int units) {      // `units` a lane, where there are many
  const size_t per = 256 * (total >= kManyUnits ? units : 1);
  return total / per + (total % per != 0);
}

template <typename T, int U>
void launch_quant(int format, hipStream_t s, const QuantArgs &a) {
  const dim3 grid((unsigned)blocks_of(a.total, kWriteUnits));
  if (format == PPO_XP_Q_INT8) hipLaunchKernelGGL((quantize_rows_kernel<T, PPO_XP_Q_INT8, U>), grid, dim3(256), 0, s, a);
  else if (format == PPO_XP_Q_E4M3) hipLaunchKernelGGL((quantize_rows_kernel<T, PPO_XP_Q_E4M3, U>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quantize_rows_kernel<T, PPO_XP_Q_INT4, U>), grid, dim3(256), 0, s, a);
}
template <typename T>
void launch_quant(int format, hipStream_t s, const QuantArgs &a) {
  if (a.total >= kManyUnits) launch_quant<T, kWriteUnits>(format, s, a);
  else launch_quant<T, 1>(format, s, a);
}
template <typename T, int U>
void launch_dequant(int format, hipStream_t s, const DequantArgs &a) {
  const dim3 grid((unsigned)blocks_of(a.total, kReadUnits));
  if (format == PPO_XP_Q_INT8) hipLaunchKernelGGL((dequantize_rows_kernel<T, PPO_XP_Q_INT8, U>), grid, dim3(256), 0, s, a);
  else if (format == PPO_XP_Q_E4M3) hipLaunchKernelGGL((dequantize_rows_kernel<T, PPO_XP_Q_E4M3, U>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((dequantize_rows_kernel<T, PPO_XP_Q_INT4, U>), grid, dim3(256), 0, s, a);
}
template <typename T>
void launch_dequant(int format, hipStream_t s, const DequantArgs &a) {
  if (a.total >= kManyUnits) launch_dequant<T, kReadUnits>(format, s, a);
  else launch_dequant<T, 1>(format, s, a);
}

}  // namespace

extern "C" {

int ppo_xp_quantize_rows(int device, void *stream, int dtype, const void *rows, int64_t rows_stride, size_t n, size_t width,
                         int format, size_t group, void *codes, int64_t codes_stride, float *scales, int64_t scales_stride,
                         size_t store_rows, size_t at) {
  if (int rc = check_store("quantize_rows", dtype, width, format, group, codes, codes_stride, scales, scales_stride)) return rc;
  if (n == 0) return 0;
  if (!rows) return ppoxp_fail(PPO_XP_EINVAL, "quantize_rows: NULL rows");
  if (at > store_rows || n > store_rows - at)
    return ppoxp_fail(PPO_XP_EINVAL, "quantize_rows: rows %zu .. %zu of a store of %zu", at, at + n, store_rows);
  if (n > 1 && rows_stride < (int64_t)width) return ppoxp_fail(PPO_XP_EINVAL, "quantize_rows: rows of %zu elements lie %lld apart", width, (long long)rows_stride);
  QuantArgs a{};
  a.rows = rows; a.codes = (uint8_t *)codes; a.scales = scales;
  a.rows_stride = rows_stride; a.codes_stride = codes_stride; a.scales_stride = scales_stride;
  a.width = (unsigned)width; a.at = at; a.lanes_log2 = (unsigned)log2_of_group(group) - 3;
  a.slots = (unsigned)(((width + group - 1) / group) * (group / 8));
  if (n > (~size_t(0)) / a.slots || !one_launch(blocks_of(n * a.slots, kWriteUnits), 256))
    return ppoxp_fail(PPO_XP_EINVAL, "quantize_rows: %zu rows of %zu are too many for one launch", n, width);
  a.total = n * a.slots;
  DeviceGuard dev(device, "quantize_rows");
  if (dev.rc()) return dev.rc();
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_quant<float>(format, s, a);
  else if (dtype == PPO_XP_BF16) launch_quant<__bf16>(format, s, a);
  else launch_quant<_Float16>(format, s, a);
  return launched("quantize_rows");
}

int ppo_xp_dequantize_rows(int device, void *stream, int dtype, const void *codes, int64_t codes_stride, const float *scales,
                           int64_t scales_stride, size_t store_rows, size_t width, int format, size_t group, const void *index,
                           int index_bits, size_t at, size_t n, void *out, int64_t out_stride) {
  if (int rc = check_store("dequantize_rows", dtype, width, format, group, codes, codes_stride, scales, scales_stride)) return rc;
  if (n == 0) return 0;
  if (!out) return ppoxp_fail(PPO_XP_EINVAL, "dequantize_rows: NULL out");
  if (store_rows == 0) return ppoxp_fail(PPO_XP_EINVAL, "dequantize_rows: %zu rows asked of an empty store", n);
  if (index && index_bits != 32 && index_bits != 64) return ppoxp_fail(PPO_XP_EINVAL, "dequantize_rows: index of %d bits", index_bits);
  if (!index && (at > store_rows || n > store_rows - at))
    return ppoxp_fail(PPO_XP_EINVAL, "dequantize_rows: rows %zu .. %zu of a store of %zu", at, at + n, store_rows);
  if (n > 1 && out_stride < (int64_t)width) return ppoxp_fail(PPO_XP_EINVAL, "dequantize_rows: rows of %zu elements do not fit a stride of %lld", width, (long long)out_stride);
  DequantArgs a{};
  a.codes = (const uint8_t *)codes; a.scales = scales; a.index = index; a.out = out;
  a.codes_stride = codes_stride; a.scales_stride = scales_stride; a.out_stride = out_stride;
  a.store_rows = store_rows; a.at = at; a.width = (unsigned)width; a.index_bits = (unsigned)index_bits;
  a.group_log2 = (unsigned)log2_of_group(group);
  const size_t E = 16 / dtype_bytes(dtype);
  a.slots = (unsigned)((width + E - 1) / E);
  if (n > (~size_t(0)) / a.slots || !one_launch(blocks_of(n * a.slots, kReadUnits), 256))
    return ppoxp_fail(PPO_XP_EINVAL, "dequantize_rows: %zu rows of %zu are too many for one launch", n, width);
  a.total = n * a.slots;
  DeviceGuard dev(device, "dequantize_rows");
  if (dev.rc()) return dev.rc();
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_dequant<float>(format, s, a);
  else if (dtype == PPO_XP_BF16) launch_dequant<__bf16>(format, s, a);
  else launch_dequant<_Float16>(format, s, a);
  return launched("dequantize_rows");
}

}  // extern "C"

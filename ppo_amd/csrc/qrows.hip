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
template <typename T, int FORMAT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs a) {
  const size_t first = (size_t)blockIdx.x * 256;
  const size_t row0 = first / a.slots;
  const unsigned t = (unsigned)(first - row0 * a.slots) + threadIdx.x;
  const bool live = first + threadIdx.x < a.total;
  const size_t row = row0 + t / a.slots;
  const unsigned e = (t % a.slots) * 8;
  const long left = live ? (long)a.width - (long)e : 0;
  Raw8<T> raw;
  load8(raw, (const T *)a.rows + (int64_t)row * a.rows_stride + e, left, 0.f);
  float x[8];
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = raw.get(i);
    top = max(top, __builtin_bit_cast(unsigned, x[i]) & 0x7fffffffu);
  }
  for (unsigned off = 1; off < (1u << a.lanes_log2); off <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, (int)off, 64));

  const bool empty = top < (17u << 23), bad = top >= 0x7f800000u;   // below 2^-110 | NaN or inf
  float s, inv;
  if (FORMAT == PPO_XP_Q_E4M3) {
    // top = 1.m 2^E <= 448 2^k = 1.75 2^(8+k)
    const unsigned k127 = (top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    s = __builtin_bit_cast(float, k127 << 23);
    inv = __builtin_bit_cast(float, (254 - k127) << 23);
  } else {
    s = __builtin_bit_cast(float, top) / (FORMAT == PPO_XP_Q_INT8 ? 127.f : 7.f);
    inv = 1.f / s;
  }
  if (empty || bad) { s = bad ? __builtin_nanf("") : 0.f; inv = 0.f; }
  if (left > 0 && ((t % a.slots) & ((1u << a.lanes_log2) - 1)) == 0)
    a.scales[(int64_t)(a.at + row) * a.scales_stride + (e >> (a.lanes_log2 + 3))] = s;

  if (left <= 0) return;
  uint8_t *dst = a.codes + (int64_t)(a.at + row) * a.codes_stride;
  if (FORMAT == PPO_XP_Q_INT4) {
    unsigned w = 0;
    if (inv != 0.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w |= ((unsigned)round_quotient(x[i], s, inv, 0.5f * s) & 15u) << (4 * i);
    }
    dst += e / 2;
    if (left >= 8) *(u32_a1 *)dst = w;
    else for (int i = 0; i < (int)(left + 1) / 2; ++i) dst[i] = (uint8_t)(w >> (8 * i));
    return;
  }
  u32x2 w = {0, 0};
  if (inv != 0.f) {
    if (FORMAT == PPO_XP_Q_E4M3) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] * inv, x[4 * h + 1] * inv, 0, false);
        p = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] * inv, x[4 * h + 3] * inv, p, true);
        w[h] = (unsigned)p;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i >> 2] |= ((unsigned)round_quotient(x[i], s, inv, 0.5f * s) & 255u) << (8 * (i & 3));
    }
  }
  dst += e;
  if (left >= 8) *(u32x2_a1 *)dst = w;
  else for (int i = 0; i < (int)left; ++i) dst[i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
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

template <int FORMAT>
__device__ __forceinline__ void decode4(const uint8_t *p, int left, float v[4]) {   // 4 codes from element 0 of p on
  unsigned w = 0;
  if (FORMAT == PPO_XP_Q_INT4) {
    if (left >= 4) w = *(const u16_a1 *)p;
    else for (int i = 0; i < (left + 1) / 2; ++i) w |= (unsigned)p[i] << (8 * i);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)((int)(w << (28 - 4 * i)) >> 28);
    return;
  }
  if (left >= 4) w = *(const u32_a1 *)p;
  else for (int i = 0; i < left; ++i) w |= (unsigned)p[i] << (8 * i);
  if (FORMAT == PPO_XP_Q_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)((int)(w << (24 - 8 * i)) >> 24);
  } else {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
  }
}

// One lane writes 16 bytes of output.  An index beyond the store reads its last row, as the gathers of a pass do.
template <typename T, int FORMAT>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(DequantArgs a) {
  constexpr int E = 16 / sizeof(T);
  const size_t first = (size_t)blockIdx.x * 256;
  if (first + threadIdx.x >= a.total) return;
  const size_t row0 = first / a.slots;
  const unsigned t = (unsigned)(first - row0 * a.slots) + threadIdx.x;
  const size_t row = row0 + t / a.slots;
  const unsigned e = (t % a.slots) * E;
  size_t src = a.at + row;
  if (a.index) src = a.index_bits == 32 ? (size_t)((const uint32_t *)a.index)[row] : (size_t)((const uint64_t *)a.index)[row];
  src = min(src, a.store_rows - 1);
  const int left = (int)(a.width - e);
  const float s = a.scales[(int64_t)src * a.scales_stride + (e >> a.group_log2)];
  const uint8_t *p = a.codes + (int64_t)src * a.codes_stride + (FORMAT == PPO_XP_Q_INT4 ? e / 2 : e);
  T *dst = (T *)a.out + (int64_t)row * a.out_stride + e;
  float v[E];
#pragma unroll
  for (int h = 0; h < E / 4; ++h) decode4<FORMAT>(p + h * (FORMAT == PPO_XP_Q_INT4 ? 2 : 4), left - 4 * h, v + 4 * h);
  if (left >= E) {
    typedef T vec __attribute__((ext_vector_type(E)));
    typedef vec vec_u __attribute__((aligned(sizeof(T))));
    vec o;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = (T)(v[i] * s);
    *(vec_u *)dst = o;
  } else {
    for (int i = 0; i < E; ++i)
      if (i < left) dst[i] = (T)(v[i] * s);
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

template <typename T>
void launch_quant(int format, dim3 grid, hipStream_t s, const QuantArgs &a) {
  if (format == PPO_XP_Q_INT8) hipLaunchKernelGGL((quantize_rows_kernel<T, PPO_XP_Q_INT8>), grid, dim3(256), 0, s, a);
  else if (format == PPO_XP_Q_E4M3) hipLaunchKernelGGL((quantize_rows_kernel<T, PPO_XP_Q_E4M3>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((quantize_rows_kernel<T, PPO_XP_Q_INT4>), grid, dim3(256), 0, s, a);
}
template <typename T>
void launch_dequant(int format, dim3 grid, hipStream_t s, const DequantArgs &a) {
  if (format == PPO_XP_Q_INT8) hipLaunchKernelGGL((dequantize_rows_kernel<T, PPO_XP_Q_INT8>), grid, dim3(256), 0, s, a);
  else if (format == PPO_XP_Q_E4M3) hipLaunchKernelGGL((dequantize_rows_kernel<T, PPO_XP_Q_E4M3>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((dequantize_rows_kernel<T, PPO_XP_Q_INT4>), grid, dim3(256), 0, s, a);
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
  if (n > (~size_t(0)) / a.slots || (n * a.slots + 255) / 256 > kMaxGrid)
    return ppoxp_fail(PPO_XP_EINVAL, "quantize_rows: %zu rows of %zu are too many for one launch", n, width);
  a.total = n * a.slots;
  DeviceGuard dev(device, "quantize_rows");
  if (dev.rc()) return dev.rc();
  const dim3 grid((unsigned)((a.total + 255) / 256));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_quant<float>(format, grid, s, a);
  else if (dtype == PPO_XP_BF16) launch_quant<__bf16>(format, grid, s, a);
  else launch_quant<_Float16>(format, grid, s, a);
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
  if (n > (~size_t(0)) / a.slots || (n * a.slots + 255) / 256 > kMaxGrid)
    return ppoxp_fail(PPO_XP_EINVAL, "dequantize_rows: %zu rows of %zu are too many for one launch", n, width);
  a.total = n * a.slots;
  DeviceGuard dev(device, "dequantize_rows");
  if (dev.rc()) return dev.rc();
  const dim3 grid((unsigned)((a.total + 255) / 256));
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PPO_XP_F32) launch_dequant<float>(format, grid, s, a);
  else if (dtype == PPO_XP_BF16) launch_dequant<__bf16>(format, grid, s, a);
  else launch_dequant<_Float16>(format, grid, s, a);
  return launched("dequantize_rows");
}

}  // extern "C"

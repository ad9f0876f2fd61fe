// Shared pieces of the token-policy operators (policy.hip, qrows.hip): element types, 8-wide unaligned loads and stores,
// wave reductions, and the host side's checks.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/ppo_xp.h"
#include "errors.h"

namespace ppoxp_ops {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
// gfx950 global memory takes 16-byte accesses at any element address: rows of odd length need no peeling
typedef u32x4 u32x4_a4 __attribute__((aligned(4)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// Eight consecutive elements as they lie in memory, and as floats.
template <typename T>
struct Raw8;

template <>
struct Raw8<float> {
  u32x4 lo, hi;
  __device__ __forceinline__ void load(const float *p) { lo = *(const u32x4_a4 *)p; hi = *(const u32x4_a4 *)(p + 4); }
  __device__ __forceinline__ float get(int i) const { return __builtin_bit_cast(float, i < 4 ? lo[i & 3] : hi[i & 3]); }
  __device__ __forceinline__ void set(int i, float x) {
    if (i < 4) lo[i & 3] = __builtin_bit_cast(unsigned, x);
    else hi[i & 3] = __builtin_bit_cast(unsigned, x);
  }
  __device__ __forceinline__ void store(float *p) const { *(u32x4_a4 *)p = lo; *(u32x4_a4 *)(p + 4) = hi; }
  __device__ __forceinline__ void set8(const float y[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) set(i, y[i]);
  }
  __device__ __forceinline__ void fill(float x) { lo = hi = u32x4(__builtin_bit_cast(unsigned, x)); }
  __device__ __forceinline__ float fresh(int i) const { return get(i); }
};

template <typename T>   // 16-bit elements: two to a register
struct Raw8 {
  u32x4 v;
  __device__ __forceinline__ void load(const T *p) { v = *(const u32x4_a2 *)p; }
  __device__ __forceinline__ float get(int i) const {
    const unsigned short h = (unsigned short)(v[i >> 1] >> ((i & 1) * 16));
    return (float)__builtin_bit_cast(T, h);
  }
  __device__ __forceinline__ void set(int i, float x) {
    const unsigned h = __builtin_bit_cast(unsigned short, (T)x);
    v[i >> 1] = (i & 1) ? ((v[i >> 1] & 0xffffu) | (h << 16)) : ((v[i >> 1] & 0xffff0000u) | h);
  }
  // Past the caches: whole lines from a wave, which nothing here reads again (5 % at 4096 x 65536).  The halves of eight floats fill
  // lines in two instructions and lose a third that way.
  __device__ __forceinline__ void store(T *p) const { __builtin_nontemporal_store(v, (u32x4_a2 *)p); }
  __device__ __forceinline__ void set8(const float y[8]) {
    typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const pair q = {(T)y[2 * i], (T)y[2 * i + 1]};
      v[i] = __builtin_bit_cast(unsigned, q);
    }
  }
  __device__ __forceinline__ void fill(float x) { v = u32x4((unsigned)__builtin_bit_cast(unsigned short, (T)x) * 0x10001u); }
  // get() that is computed here and now: left to itself the compiler keeps the floats of an earlier use, twice the registers.
  __device__ __forceinline__ float fresh(int i) const {
    float x;
    const unsigned w = v[i >> 1];
    if constexpr (__is_same(T, __bf16)) {
      if (i & 1) asm volatile("v_and_b32 %0, 0xffff0000, %1" : "=v"(x) : "v"(w));
      else asm volatile("v_lshlrev_b32 %0, 16, %1" : "=v"(x) : "v"(w));
    } else {
      if (i & 1) asm volatile("v_cvt_f32_f16_sdwa %0, %1 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:WORD_1" : "=v"(x) : "v"(w));
      else asm volatile("v_cvt_f32_f16 %0, %1" : "=v"(x) : "v"(w));
    }
    return x;
  }
};

// The same with the end of the row in sight: elements at or beyond `left` read as `fill` and are not written.  The loads of a
// last partial vector are all on their way before the first is waited for.
template <typename T>
__device__ __forceinline__ void load8(Raw8<T> &r, const T *p, long left, float fill) {
  if (left >= 8) { r.load(p); return; }
  r.fill(fill);
  if (left <= 0) return;
  T q[8];
#pragma unroll
  for (int i = 0; i < 7; ++i) q[i] = p[min((long)i, left - 1)];
  float y[8];
#pragma unroll
  for (int i = 0; i < 7; ++i) y[i] = i < left ? (float)q[i] : fill;
  y[7] = fill;
  r.set8(y);
}
template <typename T>
__device__ __forceinline__ void store8(const Raw8<T> &r, T *p, long left) {
  if (left >= 8) { r.store(p); return; }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < left) p[i] = (T)r.get(i);
}

// Wave reductions in the vector unit (rotations within 16 lanes, then the row broadcasts): lane 63 ends with the whole wave's
// value, which every lane gets.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float other, float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, other), __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float last_lane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
__device__ __forceinline__ float wave_max_nan(float x) {   // a NaN anywhere makes the result NaN
  x = __builtin_elementwise_maximum(x, dpp<0x128, 0xf>(x, x));
  x = __builtin_elementwise_maximum(x, dpp<0x124, 0xf>(x, x));
  x = __builtin_elementwise_maximum(x, dpp<0x122, 0xf>(x, x));
  x = __builtin_elementwise_maximum(x, dpp<0x121, 0xf>(x, x));
  x = __builtin_elementwise_maximum(x, dpp<0x142, 0xa>(x, x));
  x = __builtin_elementwise_maximum(x, dpp<0x143, 0xc>(x, x));
  return last_lane(x);
}
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0x128, 0xf>(0.f, x);
  x += dpp<0x124, 0xf>(0.f, x);
  x += dpp<0x122, 0xf>(0.f, x);
  x += dpp<0x121, 0xf>(0.f, x);
  x += dpp<0x142, 0xa>(0.f, x);
  x += dpp<0x143, 0xc>(0.f, x);
  return last_lane(x);
}
// Over `lanes` (a power of two) neighbouring lanes, the same in each of them: inside 16 lanes by permutations of the vector unit.
template <typename Op>
__device__ __forceinline__ float group_reduce(float x, unsigned lanes, Op op) {
  if (lanes > 1) x = op(x, dpp<0xb1, 0xf>(x, x));      // the other lane of a pair
  if (lanes > 2) x = op(x, dpp<0x4e, 0xf>(x, x));      // the other pair of four
  if (lanes > 4) x = op(x, dpp<0x141, 0xf>(x, x));     // mirrored within eight
  if (lanes > 8) x = op(x, dpp<0x140, 0xf>(x, x));     // mirrored within sixteen
  if (lanes > 16) x = op(x, __shfl_xor(x, 16, 64));
  if (lanes > 32) x = op(x, __shfl_xor(x, 32, 64));
  return x;
}
__device__ __forceinline__ float group_max_nan(float x, unsigned lanes) {
  return group_reduce(x, lanes, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
}
__device__ __forceinline__ float group_sum(float x, unsigned lanes) {
  return group_reduce(x, lanes, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ unsigned group_max_bits(unsigned x, unsigned lanes) {   // of bit patterns, as integers
  return __builtin_bit_cast(unsigned, group_reduce(__builtin_bit_cast(float, x), lanes, [](float a, float b) {
    return __builtin_bit_cast(float, max(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, b)));
  }));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
  const u32x2 v = __builtin_bit_cast(u32x2, x);
  const u32x2 o = {(unsigned)__builtin_amdgcn_update_dpp(0, (int)v.x, CTRL, ROWS, 0xf, false),
                   (unsigned)__builtin_amdgcn_update_dpp(0, (int)v.y, CTRL, ROWS, 0xf, false)};
  return x + __builtin_bit_cast(double, o);
}
__device__ __forceinline__ double wave_sum(double x) {
  x = dpp_add<0x128, 0xf>(x);
  x = dpp_add<0x124, 0xf>(x);
  x = dpp_add<0x122, 0xf>(x);
  x = dpp_add<0x121, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);
  x = dpp_add<0x143, 0xc>(x);
  const u32x2 v = __builtin_bit_cast(u32x2, x);
  const u32x2 last = {(unsigned)__builtin_amdgcn_readlane((int)v.x, 63), (unsigned)__builtin_amdgcn_readlane((int)v.y, 63)};
  return __builtin_bit_cast(double, last);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

// Makes `device` current for a call and puts the caller's device back.
class DeviceGuard {
 public:
  explicit DeviceGuard(int device, const char *who) {
    int n = 0;
    if (hipGetDevice(&prev_) != hipSuccess || (device != prev_ && (hipGetDeviceCount(&n) != hipSuccess || device < 0 || device >= n))) {
      prev_ = -1;
      rc_ = ppoxp_fail(PPO_XP_ENODEV, "%s: no HIP device %d (this library has no CPU path)", who, device);
      return;
    }
    if (device == prev_) { prev_ = -1; return; }
    hipError_t e = hipSetDevice(device);
    if (e != hipSuccess) { prev_ = -1; rc_ = ppoxp_fail(PPO_XP_EIO, "%s: hipSetDevice(%d): %s", who, device, hipGetErrorString(e)); }
  }
  ~DeviceGuard() { if (prev_ >= 0) (void)hipSetDevice(prev_); }
  DeviceGuard(const DeviceGuard &) = delete;
  DeviceGuard &operator=(const DeviceGuard &) = delete;
  int rc() const { return rc_; }

 private:
  int prev_ = -1, rc_ = 0;
};

inline int launched(const char *who) {
  hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : ppoxp_fail(PPO_XP_EIO, "%s: launch failed: %s", who, hipGetErrorString(e));
}

inline bool is_dtype(int d) { return d == PPO_XP_F32 || d == PPO_XP_BF16 || d == PPO_XP_F16; }
inline size_t dtype_bytes(int d) { return d == PPO_XP_F32 ? 4 : 2; }
// A dispatch counts its work items in 32 bits, and more of them wrap round without an error: 2^24 + 8 workgroups of 256 ran as 8.
inline bool one_launch(size_t workgroups, size_t threads) { return workgroups <= size_t(0xffffffff) / threads; }
constexpr size_t kMaxRows = 0x7fffffff;
constexpr size_t kMaxVocab = size_t(1) << 30;

}  // namespace ppoxp_ops

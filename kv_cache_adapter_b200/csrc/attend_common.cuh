// What the paged attention kernels share: their arguments, which tokens a
// query sees, and the PTX forms they use.
//
// For a query at position p of its sequence (the new token's own position),
//   out = sum_j softmax_j(scale * q . k_j) v_j   over the visible j:
//   j <= p  and  (no window, or j > p - window, or j < sinks).
// Scores are held in units of log2 (scale * key_scale * log2 e folded into
// one factor), so that every exponential is one ex2.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "kvca_device.cuh"
#include "kvca_launch.h"

namespace kvca {
namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLog2e = 1.4426950408889634f;

// Storage types of the cache, and what its matrix products run in: e4m3
// widens to fp16, which holds every e4m3 value.
struct CacheF16 {
  static constexpr int kBytes = 2;
  static constexpr bool kBf16 = false;
};
struct CacheBf16 {
  static constexpr int kBytes = 2;
  static constexpr bool kBf16 = true;
};
struct CacheE4m3 {
  static constexpr int kBytes = 1;
  static constexpr bool kBf16 = false;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The larger of two; NaN when either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Two floats cut off to 16 bits (towards 0), in one register, the first in the
// low half.
template <bool kBf16>
__device__ __forceinline__ uint32_t cut2(float lo, float hi) {
  if constexpr (kBf16) return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632);
  uint32_t r;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes from global to shared memory; zeros when `read` is false (then
// nothing is read from `src`).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two floats to one register of two 16-bit values, the first in the low half.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  } else {
    __half2 h;
    memcpy(&h, &v, 4);
    return __half22float2(h);
  }
}

// Two e4m3 values (low 16 bits) to two fp16 values.
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(v)));
  return r;
}

// Powers of two that bring a row of queries, whose largest magnitude is
// `big`, into fp16 for the products with e4m3 keys: the largest value falls
// into [2^12, 2^13), so a bf16 row keeps its bits (values 2^-27 of the largest
// and less fall among fp16's subnormals).  The inverse goes into the factor of
// the scores.
__device__ __forceinline__ int power_up(float big) {
  const int exponent = static_cast<int>(__float_as_uint(big) >> 23);  // 0: zero or subnormal, 255: not finite
  return exponent == 0 || exponent == 255 ? 0 : min(max(12 + 127 - exponent, -120), 120);
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// The tokens that the query at the end of a sequence of `len` tokens sees,
// numbered 0 .. count - 1: the first `sinks` ones, then those of the window.
struct Visible {
  int count;
  int sinks;
  int skip;  // tokens between the sinks and the window
  __device__ __forceinline__ int position(int v) const { return v < sinks ? v : v + skip; }
};

__device__ __forceinline__ Visible visible_tokens(int len, int window, int sinks) {
  Visible r;
  if (window > 0 && len > window) {
    r.sinks = min(sinks, len - window);
    r.count = window + r.sinks;
    r.skip = len - r.count;
  } else {
    r.count = len;
    r.sinks = len;
    r.skip = 0;
  }
  return r;
}

// Length of a sequence, at most what its page table holds (a longer one is
// reported); negative for an idle row, which is left as it was.
__device__ __forceinline__ int sequence_length(const AttendArgs& a, int seq) {
  const int64_t len = __ldg(a.lens + seq);
  if (len > a.capacity) {
    report(a.status, KVCA_ERR_BAD_INDEX, len);
    return a.capacity;
  }
  return len < 0 ? -1 : static_cast<int>(len);
}

}  // namespace
}  // namespace kvca

// Device helpers that the kernel files share: the status word, the packed
// slot metadata word and a block-wide scan.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace kvca {
namespace {

// ---------------------------------------------------------------------------
// Status reporting
// ---------------------------------------------------------------------------

__device__ __forceinline__ void report(int64_t* status, int64_t code, int64_t value) {
  if (status == nullptr) return;
  const unsigned long long prev = atomicCAS(reinterpret_cast<unsigned long long*>(status), 0ull,
                                            static_cast<unsigned long long>(code));
  if (prev == 0ull) status[1] = value;
}

// ---------------------------------------------------------------------------
// Packed slot metadata: pin count in the low half of the word, usage count in
// the high half (adapter.py:1419-1432).
// ---------------------------------------------------------------------------

template <typename MetaT>
struct Meta {
  static constexpr int kFieldBits = static_cast<int>(sizeof(MetaT)) * 4;
  static constexpr unsigned kFieldMask = (1u << kFieldBits) - 1u;
  static constexpr int kUsageMax = static_cast<int>(kFieldMask);
  static constexpr int kSlotsPerVec = 16 / static_cast<int>(sizeof(MetaT));

  __device__ __forceinline__ static unsigned pin(unsigned w) { return w & kFieldMask; }
  __device__ __forceinline__ static unsigned usage(unsigned w) {
    return (w >> kFieldBits) & kFieldMask;
  }
  // Masks both fields exactly like _pack_slot_meta: pins above the field
  // maximum and negative pins wrap.
  __device__ __forceinline__ static MetaT pack(int64_t pin_count, int64_t usage_count) {
    const uint64_t p = static_cast<uint64_t>(pin_count) & kFieldMask;
    const uint64_t u = static_cast<uint64_t>(usage_count) & kFieldMask;
    return static_cast<MetaT>(p | (u << kFieldBits));
  }
  __device__ __forceinline__ static unsigned sat_inc(unsigned usage_count) {
    return usage_count + 1u > kFieldMask ? kFieldMask : usage_count + 1u;
  }
};

// ---------------------------------------------------------------------------
// Block-wide exclusive scan (blockDim.x a multiple of 32, at most 1024).
// `sm` holds 33 ints.  Contains three __syncthreads.
// ---------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ T block_excl_scan(T x, T* total, T* sm) {
  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  T incl = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T y = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 31) sm[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    const int nwarps = static_cast<int>(blockDim.x >> 5);
    const T w = lane < nwarps ? sm[lane] : T(0);
    T wi = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, wi, d);
      if (lane >= d) wi += y;
    }
    if (lane < nwarps) sm[lane] = wi - w;
    if (lane == 31) sm[32] = wi;
  }
  __syncthreads();
  const T result = sm[warp] + incl - x;
  *total = sm[32];
  __syncthreads();
  return result;
}

}  // namespace
}  // namespace kvca

// Rows of new tokens: rotary positions, the append to a paged cache of 16, 8
// or 4 bits, and the way back from a cache of 8 or 4 bits.
//
// The rotation turns pairs of a head's first rotary dims, (i, i + rotary / 2)
// or (2 i, 2 i + 1), by an angle of the token's position and of i:
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s
// with c and s from a table of fp32 rows (cosines, then sines), one row per
// position; its transpose has -s.  Every product and sum is rounded by itself
// (no fused multiply-add), so that the values to be stored in few bits do not
// depend on how an expression was compiled.
//
// A warp takes some rows (heads) of one token at a time, a lane 8 neighbouring
// dims (16 where they are stored in 4 bits: one group with a scale) and keeps
// its angles for the next rows of the token.  Each output is computed from its
// own value and its pair's, both loaded (the second comes from the first-level
// cache), so that one form does for every layout; a row never leaves its warp,
// so its place may be its result's.

#include <cuda_runtime.h>
#include <stdint.h>

#include "attend_common.cuh"
#include "kvca_host.cuh"

namespace kvca {
namespace {

constexpr int kTokenWarps = 4;  // of a CTA

struct InF32 {
  static constexpr int kBytes = 4;
};

// 8 neighbouring values, 16-byte aligned.
template <typename In>
__device__ __forceinline__ void load8(const char* p, float (&x)[8]) {
  if constexpr (In::kBytes == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 16);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2<In::kBf16>(w[j]);
      x[2 * j] = f.x, x[2 * j + 1] = f.y;
    }
  }
}

template <typename In>
__device__ __forceinline__ float load1(const char* p) {
  if constexpr (In::kBytes == 4)
    return *reinterpret_cast<const float*>(p);
  else
    return unpack2<In::kBf16>(*reinterpret_cast<const uint16_t*>(p)).x;
}

template <typename Out>
__device__ __forceinline__ void store8(char* p, const float (&x)[8]) {
  if constexpr (Out::kBytes == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 16) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<Out::kBf16>(x[0], x[1]), pack2<Out::kBf16>(x[2], x[3]),
                                              pack2<Out::kBf16>(x[4], x[5]), pack2<Out::kBf16>(x[6], x[7]));
  }
}

// ---------------------------------------------------------------------------
// Rotation
// ---------------------------------------------------------------------------

enum TurnMode {
  kTurnNone,
  kTurnHalves,       // pairs (i, i + rotary / 2), rotary / 2 a multiple of 8
  kTurnHalvesLoose,  // the same, any rotary / 2
  kTurnPairs,        // pairs (2 i, 2 i + 1)
};

// The angles of dims d0 .. d0 + 7 and where their pairs are.
template <int kMode>
struct Turn8 {
  static constexpr int kAngles = kMode == kTurnPairs ? 4 : 8;
  float c[kAngles], s[kAngles];  // s with the sign that an output's pair takes
  int other[kMode == kTurnHalvesLoose ? 8 : 1];  // dims to the pair's value
  unsigned on;                                   // a bit per angle: rotated

  __device__ __forceinline__ void load(const TokenArgs& a, const float* angles, int d0) {
    const int half = a.rotary / 2;
    const float sign = a.transpose ? -1.f : 1.f;
    on = 0;
    if constexpr (kMode == kTurnHalves) {
      const bool second = d0 >= half;
      other[0] = second ? -half : half;
      if (d0 >= a.rotary) return;
      on = 0xffu;
      const int i = second ? d0 - half : d0;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4 cc = __ldg(reinterpret_cast<const float4*>(angles + i + e));
        const float4 ss = __ldg(reinterpret_cast<const float4*>(angles + half + i + e));
        c[e] = cc.x, c[e + 1] = cc.y, c[e + 2] = cc.z, c[e + 3] = cc.w;
        const float side = second ? sign : -sign;
        s[e] = ss.x * side, s[e + 1] = ss.y * side, s[e + 2] = ss.z * side, s[e + 3] = ss.w * side;
      }
    } else if constexpr (kMode == kTurnHalvesLoose) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        const bool second = d >= half;
        const int i = second ? d - half : d;
        other[e] = second ? -half : half;
        c[e] = 1.f, s[e] = 0.f;
        if (d >= a.rotary) continue;
        on |= 1u << e;
        c[e] = __ldg(angles + i);
        s[e] = __ldg(angles + half + i) * (second ? sign : -sign);
      }
    } else if constexpr (kMode == kTurnPairs) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = d0 / 2 + e;
        c[e] = 1.f, s[e] = 0.f;
        if (i >= half) continue;
        on |= 1u << e;
        c[e] = __ldg(angles + i);
        s[e] = __ldg(angles + half + i) * sign;
      }
    }
  }
};

__device__ __forceinline__ float turned(float own, float c, float pair, float s) {
  return __fadd_rn(__fmul_rn(own, c), __fmul_rn(pair, s));
}

// x: dims d0 .. d0 + 7 of the row at p, rotated.
template <typename In, int kMode>
__device__ __forceinline__ void load_turned(const char* row, int d0, const Turn8<kMode>& t, float (&x)[8]) {
  load8<In>(row + d0 * In::kBytes, x);
  if constexpr (kMode == kTurnHalves) {
    if (t.on == 0) return;
    float y[8];
    load8<In>(row + (d0 + t.other[0]) * In::kBytes, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = turned(x[e], t.c[e], y[e], t.s[e]);
  } else if constexpr (kMode == kTurnHalvesLoose) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((t.on >> e) & 1u) x[e] = turned(x[e], t.c[e], load1<In>(row + (d0 + e + t.other[e]) * In::kBytes), t.s[e]);
  } else if constexpr (kMode == kTurnPairs) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = turned(x[2 * e], t.c[e], x[2 * e + 1], -t.s[e]);
      const float z = turned(x[2 * e + 1], t.c[e], x[2 * e], t.s[e]);
      const bool on = (t.on >> e) & 1u;
      x[2 * e] = on ? y : x[2 * e];
      x[2 * e + 1] = on ? z : x[2 * e + 1];
    }
  }
}

// ---------------------------------------------------------------------------
// 8 and 4 bits
// ---------------------------------------------------------------------------

// Two values to e4m3 (to the nearest, ties to even; beyond 448 to 448, NaN
// stays), the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two values to e2m1, the first in the low half of the byte.
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n.reg .b8 b;\ncvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\ncvt.u32.u8 %0, b;\n}" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float e4m3_to_float(uint32_t byte) { return unpack2<false>(e4m3_to_f16x2(byte)).x; }

// 16 values as codes with one scale, which is chosen so that the largest
// becomes 6, the largest code.  A NaN makes the scale and so all of them NaN;
// what lies beyond 6 times the largest scale is cut off.
__device__ __forceinline__ uint2 to_codes(const float (&x)[2][8], float factor, uint32_t* scale) {
  float big = 0.f;
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) big = max_nan(big, fabsf(x[j][e]));
  *scale = to_e4m3x2(__fdiv_rn(big, 6.f * factor), 0.f) & 0xffu;
  const float unit = e4m3_to_float(*scale) * factor;
  uint32_t word[2] = {0, 0};
  if (unit > 0.f) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        word[j] |= to_e2m1x2(__fdiv_rn(x[j][e], unit), __fdiv_rn(x[j][e + 1], unit)) << (4 * e);
  }
  return make_uint2(word[0], word[1]);
}

// ---------------------------------------------------------------------------
// The append, and the rotation alone
// ---------------------------------------------------------------------------

struct TokenPlace {
  bool live;       // not padding, nothing out of range
  int64_t block;
  int offset;
  const float* angles;
};

template <bool kStores>
__device__ __forceinline__ TokenPlace place_of(const TokenArgs& a, int64_t token) {
  TokenPlace t{false, 0, 0, nullptr};
  if constexpr (kStores) {
    const int64_t slot = __ldg(a.slots + token);
    if (slot < 0) return t;
    if (slot >= a.num_slots) {
      report(a.status, KVCA_ERR_BAD_INDEX, slot);
      return t;
    }
    t.block = a.block_shift >= 0 ? slot >> a.block_shift : slot / a.block_size;
    t.offset = static_cast<int>(slot - t.block * a.block_size);
  }
  if (a.table != nullptr) {
    const int64_t position = __ldg(a.positions + token);
    if (!kStores && position < 0) return t;
    if (position < 0 || position >= a.table_rows) {
      report(a.status, KVCA_ERR_BAD_INDEX, position);
      return t;
    }
    t.angles = a.table + position * a.rotary;
  }
  t.live = true;
  return t;
}

// Cache: the type that keys and values are stored in; In where nothing is.
template <typename In, typename Cache, int kMode, bool kStores>
__global__ void __launch_bounds__(32 * kTokenWarps) token_rows_kernel(const __grid_constant__ TokenArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = static_cast<int64_t>(blockIdx.x) * kTokenWarps + (threadIdx.x >> 5);
  const int64_t token = warp / a.token_warps;
  const int part = static_cast<int>(warp - token * a.token_warps);
  if (token >= a.rows) return;
  const TokenPlace place = place_of<kStores>(a, token);
  if (!place.live) return;
  constexpr bool kFour = kStores && Cache::kBytes == 0;

  {
    // rows of 8 dims per lane: queries, then (unless stored in 4 bits) keys
    const int lanes = a.dim / 8, rows = 32 / lanes;
    const int row_of = lane / lanes, d0 = (lane - row_of * lanes) * 8;
    const int heads = a.q_heads + (kStores && !kFour ? a.kv_heads : 0);
    if (part * rows < heads) {
      Turn8<kMode> turn;
      turn.load(a, place.angles, d0);
      for (int r = part * rows; r < heads; r += a.token_warps * rows) {
        const int h = r + row_of;
        const bool mine = row_of < rows && h < heads;
        const bool is_query = h < a.q_heads;
        float x[8];
        const char* const from = is_query ? a.query + token * a.query_row + h * a.query_head
                                          : a.key + token * a.key_row + (h - a.q_heads) * a.key_head;
        if (mine) load_turned<In, kMode>(from, d0, turn, x);
        __syncwarp();  // a row's place may be its result's
        if (!mine) continue;
        if (is_query) {
          store8<In>(a.query_out + token * a.query_out_row + h * a.query_out_head + d0 * In::kBytes, x);
        } else if constexpr (kStores && !kFour) {
          char* const to = a.key_cache + place.block * a.key_cache_block + place.offset * a.key_cache_token +
                           (h - a.q_heads) * a.key_cache_head + d0 * Cache::kBytes;
          if constexpr (Cache::kBytes == 1) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = to_e4m3x2(__fdiv_rn(x[2 * e], a.key_scale), __fdiv_rn(x[2 * e + 1], a.key_scale));
            *reinterpret_cast<uint2*>(to) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
          } else {
            store8<Cache>(to, x);
          }
        }
      }
    }
    if constexpr (kStores && !kFour) {
      for (int r = part * rows; r < a.kv_heads; r += a.token_warps * rows) {
        const int h = r + row_of;
        if (row_of >= rows || h >= a.kv_heads) continue;
        const char* const from = a.value + token * a.value_row + h * a.value_head + d0 * In::kBytes;
        char* const to = a.value_cache + place.block * a.value_cache_block + place.offset * a.value_cache_token +
                         h * a.value_cache_head + d0 * Cache::kBytes;
        if constexpr (Cache::kBytes == 1) {
          float x[8];
          load8<In>(from, x);
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = to_e4m3x2(__fdiv_rn(x[2 * e], a.value_scale), __fdiv_rn(x[2 * e + 1], a.value_scale));
          *reinterpret_cast<uint2*>(to) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
        } else {
          *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
        }
      }
    }
  }
  if constexpr (kFour) {
    // a group of 16 dims per lane, keys and then values
    const int lanes = a.dim / 16, rows = 32 / lanes;
    const int row_of = lane / lanes, group = lane - row_of * lanes;
    const int64_t codes = static_cast<int64_t>(a.kv_heads) * (a.dim / 2);
    if (part * rows >= 2 * a.kv_heads) return;
    Turn8<kMode> turn[2];
    turn[0].load(a, place.angles, group * 16);
    turn[1].load(a, place.angles, group * 16 + 8);
    for (int r = part * rows; r < 2 * a.kv_heads; r += a.token_warps * rows) {
      int h = r + row_of;
      if (row_of >= rows || h >= 2 * a.kv_heads) continue;
      const bool is_key = h < a.kv_heads;
      float x[2][8];
      char* to;
      if (is_key) {
        const char* const from = a.key + token * a.key_row + h * a.key_head;
        load_turned<In, kMode>(from, group * 16, turn[0], x[0]);
        load_turned<In, kMode>(from, group * 16 + 8, turn[1], x[1]);
        to = a.key_cache + place.block * a.key_cache_block + place.offset * a.key_cache_token;
      } else {
        h -= a.kv_heads;
        const char* const from = a.value + token * a.value_row + h * a.value_head + group * 16 * In::kBytes;
        load8<In>(from, x[0]);
        load8<In>(from + 8 * In::kBytes, x[1]);
        to = a.value_cache + place.block * a.value_cache_block + place.offset * a.value_cache_token;
      }
      uint32_t scale;
      const uint2 word = to_codes(x, is_key ? a.key_scale : a.value_scale, &scale);
      *reinterpret_cast<uint2*>(to + h * (a.dim / 2) + group * 8) = word;
      *reinterpret_cast<uint8_t*>(to + codes + h * (a.dim / 16) + group) = static_cast<uint8_t>(scale);
    }
  }
}

struct CacheE2m1Rows {
  static constexpr int kBytes = 0;  // less than one
};

template <typename In, typename Cache, bool kStores>
cudaError_t launch_rows(const TokenArgs& a, cudaStream_t stream) {
  const int64_t warps = a.rows * a.token_warps;
  const dim3 grid(static_cast<unsigned>((warps + kTokenWarps - 1) / kTokenWarps));
  const int half = a.rotary / 2;
  if (a.table == nullptr) {
    if constexpr (kStores) token_rows_kernel<In, Cache, kTurnNone, kStores><<<grid, 32 * kTokenWarps, 0, stream>>>(a);
  } else if (a.interleaved) {
    token_rows_kernel<In, Cache, kTurnPairs, kStores><<<grid, 32 * kTokenWarps, 0, stream>>>(a);
  } else if (half % 8 == 0) {
    token_rows_kernel<In, Cache, kTurnHalves, kStores><<<grid, 32 * kTokenWarps, 0, stream>>>(a);
  } else {
    token_rows_kernel<In, Cache, kTurnHalvesLoose, kStores><<<grid, 32 * kTokenWarps, 0, stream>>>(a);
  }
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Back from 8 or 4 bits
// ---------------------------------------------------------------------------

template <typename Out, bool kFour>
__global__ void __launch_bounds__(256) read_rows_kernel(const __grid_constant__ ReadArgs a) {
  const int lanes = a.heads * (a.dim / 8);  // of 8 values each, per token
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t token = i / lanes;
  if (token >= a.rows) return;
  const int at = static_cast<int>(i - token * lanes);
  const int64_t slot = __ldg(a.slots + token);
  if (slot < 0) return;
  if (slot >= a.num_slots) {
    report(a.status, KVCA_ERR_BAD_INDEX, slot);
    return;
  }
  const int64_t block = a.block_shift >= 0 ? slot >> a.block_shift : slot / a.block_size;
  const char* const row = a.cache + block * a.cache_block + (slot - block * a.block_size) * a.cache_token;
  const int h = at / (a.dim / 8), d0 = (at - h * (a.dim / 8)) * 8;
  float x[8];
  if constexpr (kFour) {
    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(row) + at);
    const float unit =
        e4m3_to_float(__ldg(reinterpret_cast<const uint8_t*>(row) + a.heads * (a.dim / 2) + at / 2)) * a.scale;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 f = unpack2<false>(e2m1_to_f16x2(word >> (4 * e)));
      x[e] = f.x * unit, x[e + 1] = f.y * unit;
    }
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(row + h * a.cache_head + d0));
    const uint32_t w[4] = {v.x, v.x >> 16, v.y, v.y >> 16};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack2<false>(e4m3_to_f16x2(w[e]));
      x[2 * e] = f.x * a.scale, x[2 * e + 1] = f.y * a.scale;
    }
  }
  store8<Out>(a.out + (token * lanes + at) * 8 * Out::kBytes, x);
}

template <typename Out>
cudaError_t launch_read_to(const ReadArgs& a, cudaStream_t stream) {
  const int64_t threads = a.rows * a.heads * (a.dim / 8);
  const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
  if (a.cache_type == KVCA_TYPE_E2M1)
    read_rows_kernel<Out, true><<<grid, 256, 0, stream>>>(a);
  else
    read_rows_kernel<Out, false><<<grid, 256, 0, stream>>>(a);
  return cudaGetLastError();
}

// Warps that share a token's heads, each with several rows of them.
int warps_of(const TokenArgs& a, bool four, bool stores) {
  const int rows = 32 / (a.dim / 8);
  const int wide = a.q_heads + (stores && !four ? a.kv_heads : 0);
  int items = (wide + rows - 1) / rows;
  if (four) {
    const int narrow = 32 / (a.dim / 16);
    const int more = (2 * a.kv_heads + narrow - 1) / narrow;
    items = items > more ? items : more;
  }
  return items;
}

}  // namespace

cudaError_t launch_append_tokens(const TokenArgs& args, int type, int cache_type, cudaStream_t stream) {
  TokenArgs a = args;
  a.token_warps = warps_of(a, cache_type == KVCA_TYPE_E2M1, true);
  if (type == KVCA_TYPE_F16) {
    if (cache_type == KVCA_TYPE_E4M3) return launch_rows<CacheF16, CacheE4m3, true>(a, stream);
    if (cache_type == KVCA_TYPE_E2M1) return launch_rows<CacheF16, CacheE2m1Rows, true>(a, stream);
    return launch_rows<CacheF16, CacheF16, true>(a, stream);
  }
  if (cache_type == KVCA_TYPE_E4M3) return launch_rows<CacheBf16, CacheE4m3, true>(a, stream);
  if (cache_type == KVCA_TYPE_E2M1) return launch_rows<CacheBf16, CacheE2m1Rows, true>(a, stream);
  return launch_rows<CacheBf16, CacheBf16, true>(a, stream);
}

cudaError_t launch_rotate_tokens(const TokenArgs& args, int type, cudaStream_t stream) {
  TokenArgs a = args;
  a.token_warps = warps_of(a, false, false);
  switch (type) {
    case KVCA_TYPE_F16: return launch_rows<CacheF16, CacheF16, false>(a, stream);
    case KVCA_TYPE_BF16: return launch_rows<CacheBf16, CacheBf16, false>(a, stream);
    default: return launch_rows<InF32, InF32, false>(a, stream);
  }
}

cudaError_t launch_read_tokens(const ReadArgs& a, int type, cudaStream_t stream) {
  switch (type) {
    case KVCA_TYPE_F16: return launch_read_to<CacheF16>(a, stream);
    case KVCA_TYPE_BF16: return launch_read_to<CacheBf16>(a, stream);
    default: return launch_read_to<InF32>(a, stream);
  }
}

}  // namespace kvca

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
// A warp takes some rows (heads) of one token at a time and keeps the angles for
// its next rows.  Where pairs are half the rotary dims apart, a lane holds both
// sides of 8 of them, so each value is loaded once and its place may be its
// result's; neighbouring pairs (and pairs at odd distances) lie 8 dims to a lane,
// 16 where they are stored in 4 bits: a group with its scale.
//
// Bytes bound the large calls with pairs at distances of a multiple of 8 dims, and of
// neighbouring pairs to 16 bits: each row is read and written once, so a turn of 8 dims
// costs 32 bytes and some 20 instructions.  A warp takes up to 12 turns, two loaded at a
// time.  16,384 tokens (32 query and 2 x 8 K/V heads of 128, bf16): 67 us, 64 of bytes
// at the copy's rate (91 us with three turns to a warp, all loaded at once), 65 to e4m3
// (58 of bytes); the gradient of 8,192 x 32 fp32 heads, neighbouring pairs: 47 us, 43 of
// bytes.  To 4 bits, 8,191 such tokens and their way back: 53 us, 33 of bytes; there the
// registers that rows in flight lie in bound it (7 blocks per SM, with 16 bytes spilled;
// 6 blocks 59 us, 8 with more spills 57; fewer instructions per group the same).
//
// The other forms are far from their bytes, for their registers (90-138 neighbouring
// pairs, 142-255 the loose mode: 8-20 warps per SM) and, in the loose mode, three loads
// of single values per rotated one, for each head again.  us, and of bytes, for 16,384
// tokens (to 4 bits 8,191): neighbouring pairs to e4m3 102 (58), to 4 bits 74 (28; pairs
// of halves 40); no table, 2 x 8 heads of 128: to 16 bits 49 (21), to e4m3 74 (16), to 4
// bits 30 (7); 84 of 112 dims, 32 heads, rotated: 121 (37); 72 of 96 dims to 4 bits: 133
// (21).  Few tokens: the host's 8-12 us, in a replayed graph 4.

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

// 8 values as they lie in memory, and as floats.
template <typename In>
struct Raw8 {
  uint4 w[In::kBytes / 2 > 0 ? In::kBytes / 2 : 1];

  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int j = 0; j < In::kBytes / 2; ++j) w[j] = *reinterpret_cast<const uint4*>(p + 16 * j);
  }
  __device__ __forceinline__ void store(char* p) const {
#pragma unroll
    for (int j = 0; j < In::kBytes / 2; ++j) *reinterpret_cast<uint4*>(p + 16 * j) = w[j];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (In::kBytes == 4) {
      x[0] = __uint_as_float(w[0].x), x[1] = __uint_as_float(w[0].y);
      x[2] = __uint_as_float(w[0].z), x[3] = __uint_as_float(w[0].w);
      x[4] = __uint_as_float(w[1].x), x[5] = __uint_as_float(w[1].y);
      x[6] = __uint_as_float(w[1].z), x[7] = __uint_as_float(w[1].w);
    } else {
      const uint32_t v[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2<In::kBf16>(v[j]);
        x[2 * j] = f.x, x[2 * j + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    if constexpr (In::kBytes == 4) {
      w[0] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      w[1] = make_uint4(__float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7]));
    } else {
      w[0] = make_uint4(pack2<In::kBf16>(x[0], x[1]), pack2<In::kBf16>(x[2], x[3]), pack2<In::kBf16>(x[4], x[5]),
                        pack2<In::kBf16>(x[6], x[7]));
    }
  }
};

template <typename In>
__device__ __forceinline__ float load1(const char* p) {
  if constexpr (In::kBytes == 4)
    return *reinterpret_cast<const float*>(p);
  else
    return unpack2<In::kBf16>(*reinterpret_cast<const uint16_t*>(p)).x;
}

// ---------------------------------------------------------------------------
// Rotation
// ---------------------------------------------------------------------------

enum TurnMode {
  kTurnHalves,  // pairs (i, i + rotary / 2) with rotary / 2 a multiple of 8 (4 bits: of 16): a lane has both sides
  kTurnLoose,   // the same at any distance, or no rotation (far from its bytes: above)
  kTurnPairs,   // pairs (2 i, 2 i + 1)
};

__device__ __forceinline__ float turned(float own, float c, float pair, float s) {
  return __fadd_rn(__fmul_rn(own, c), __fmul_rn(pair, s));
}

// A lane's share of a row: 8 dims from `first` on, and in kTurnHalves the 8 that
// they turn with (4 bits, other modes: the 8 after them).
template <int kMode, bool kWide>
struct Lane8 {
  static constexpr int kParts = kMode == kTurnHalves || kWide ? 2 : 1;  // of 8 dims
  static constexpr int kAngles = kMode == kTurnPairs ? 4 * kParts : 8;
  int lanes;    // per row
  int first;
  int second;   // dims of the other part, or -1
  bool turns;   // (kTurnHalves) both parts by the angles
  float c[kAngles], s[kAngles];
  unsigned on;  // (other modes) a bit per angle or dim: rotated

  __device__ __forceinline__ void place(const TokenArgs& a, int lane) {
    const int half = a.rotary / 2;
    if constexpr (kMode == kTurnHalves) {
      const int pairs = half / 8;
      lanes = pairs + (a.dim - a.rotary) / 8;
      const int at = lane % lanes;
      turns = at < pairs;
      first = turns ? at * 8 : a.rotary + (at - pairs) * 8;
      second = turns ? first + half : -1;
    } else {
      lanes = a.dim / (8 * kParts);
      first = lane % lanes * 8 * kParts;
      second = kParts == 2 ? first + 8 : -1;
    }
  }
  __device__ __forceinline__ void load(const TokenArgs& a, const float* angles) {
    const int half = a.rotary / 2;
    on = 0;
    if constexpr (kMode == kTurnHalves) {
      if (!turns) return;
      const float sign = a.transpose ? -1.f : 1.f;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4 cc = __ldg(reinterpret_cast<const float4*>(angles + first + e));
        const float4 ss = __ldg(reinterpret_cast<const float4*>(angles + half + first + e));
        c[e] = cc.x, c[e + 1] = cc.y, c[e + 2] = cc.z, c[e + 3] = cc.w;
        s[e] = ss.x * sign, s[e + 1] = ss.y * sign, s[e + 2] = ss.z * sign, s[e + 3] = ss.w * sign;
      }
    } else if constexpr (kMode == kTurnPairs) {
#pragma unroll
      for (int e = 0; e < kAngles; ++e) {
        const int i = first / 2 + e;
        c[e] = 1.f, s[e] = 0.f;
        if (i >= half) continue;
        on |= 1u << e;
        c[e] = __ldg(angles + i);
        s[e] = a.transpose ? -__ldg(angles + half + i) : __ldg(angles + half + i);
      }
    }
  }

  // The parts of the row at p, rotated; those that stay, as they were.
  template <typename In>
  __device__ __forceinline__ void rotate(const TokenArgs& a, const char* p, const float* angles,
                                         Raw8<In> (&raw)[kParts], float (&x)[kParts][8], bool keep_floats) {
#pragma unroll
    for (int j = 0; j < kParts; ++j) raw[j].get(x[j]);
    if constexpr (kMode == kTurnHalves) {
      if (!turns) return;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = turned(x[0][e], c[e], x[1][e], -s[e]);
        x[1][e] = turned(x[1][e], c[e], x[0][e], s[e]);
        x[0][e] = y;
      }
      if (keep_floats) return;
      raw[0].set(x[0]);
      raw[1].set(x[1]);
    } else if constexpr (kMode == kTurnPairs) {
#pragma unroll
      for (int j = 0; j < kParts; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = j * 4 + e;
          const float y = turned(x[j][2 * e], c[k], x[j][2 * e + 1], -s[k]);
          const float z = turned(x[j][2 * e + 1], c[k], x[j][2 * e], s[k]);
          const bool turn = (on >> k) & 1u;
          x[j][2 * e] = turn ? y : x[j][2 * e];
          x[j][2 * e + 1] = turn ? z : x[j][2 * e + 1];
        }
      if (keep_floats) return;
#pragma unroll
      for (int j = 0; j < kParts; ++j)
        if ((on >> (4 * j)) & 15u) raw[j].set(x[j]);
    } else {
      if (angles == nullptr) return;
      const int half = a.rotary / 2;
#pragma unroll
      for (int j = 0; j < kParts; ++j) {
        if (first + 8 * j >= a.rotary) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = first + 8 * j + e;
          if (d >= a.rotary) continue;
          const bool back = d >= half;
          const float sine = __ldg(angles + (back ? d : d + half));
          x[j][e] = turned(x[j][e], __ldg(angles + (back ? d - half : d)),
                           load1<In>(p + (back ? d - half : d + half) * In::kBytes),
                           back != a.transpose ? sine : -sine);
        }
        if (!keep_floats) raw[j].set(x[j]);
      }
    }
  }
};

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

// x / b for a rounding to few bits, from r, the rounded reciprocal of b: the
// product's remainder corrects it (Markstein's correction).  A quotient that is
// a midpoint of the few bits comes out exactly: with x = t b the remainder of
// q = t + d is -d b, exactly, and the correction leaves d r b, 2^-24 of d.  Any
// other is off by 2^-46 before its rounding.  Where q is past `most`, which the
// rounding cuts off anyway, it stays, as it may be infinite.
__device__ __forceinline__ float quotient(float x, float b, float r, float most) {
  const float q = x * r;
  const float better = __fmaf_rn(__fmaf_rn(-q, b, x), r, q);
  return fabsf(q) < most ? better : q;
}

__device__ __forceinline__ uint2 to_e4m3x8(const float (&x)[8], float scale, float reciprocal) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = to_e4m3x2(quotient(x[2 * e], scale, reciprocal, 512.f), quotient(x[2 * e + 1], scale, reciprocal, 512.f));
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

__device__ __forceinline__ float largest8(const float (&x)[8]) {
  float big = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) big = max_nan(big, fabsf(x[e]));
  return big;
}

// The scale of a group whose largest magnitude is `big`: that one becomes 6, the
// largest code.  A NaN makes it, and so all values of the group, NaN; what lies
// beyond 6 times the largest scale is cut off.
__device__ __forceinline__ uint32_t scale_of(float big, float factor) {
  return to_e4m3x2(__fdiv_rn(big, 6.f * factor), 0.f) & 0xffu;
}

// 8 values as codes; zeros where the scale is 0 or NaN.
__device__ __forceinline__ uint32_t to_codes(const float (&x)[8], float unit, float reciprocal) {
  uint32_t word = 0;
#pragma unroll
  for (int e = 0; e < 8; e += 2)
    word |= to_e2m1x2(quotient(x[e], unit, reciprocal, 8.f), quotient(x[e + 1], unit, reciprocal, 8.f)) << (4 * e);
  return unit > 0.f ? word : 0u;
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

struct CacheE2m1Rows {
  static constexpr int kBytes = 0;  // less than one
};

// Cache: the type that keys and values are stored in; In where nothing is.
// kWide: 16 dims to a lane, for the keys and values of a 4-bit cache; its
// queries then are rows of a warp of their own kind (8 dims to a lane).
template <typename In, typename Cache, int kMode, bool kStores, bool kWide, int kBatch>
__device__ __forceinline__ void token_rows(const TokenArgs& a, int64_t token, int part, int parts) {
  constexpr bool kFour = kStores && Cache::kBytes == 0;
  using Lane = Lane8<kMode, kWide>;
  constexpr int kParts = Lane::kParts;
  const int lane = threadIdx.x & 31;
  Lane at;
  at.place(a, lane);
  const int rows = 32 / at.lanes, row_of = lane / at.lanes;
  // heads of queries, keys and values in turn
  const int begin = kWide && kMode != kTurnHalves ? a.q_heads : 0;
  const int keys = a.q_heads, values = keys + a.kv_heads;
  const int end = kFour && !kWide && kMode != kTurnHalves ? a.q_heads : kStores ? values + a.kv_heads : a.q_heads;
  if (begin + part * rows >= end) return;
  TokenPlace place;
  float key_reciprocal = 0.f, value_reciprocal = 0.f;
  if constexpr (kStores && Cache::kBytes == 1) {
    key_reciprocal = __frcp_rn(a.key_scale);
    value_reciprocal = __frcp_rn(a.value_scale);
  }
  // The rows of kBatch turns are on their way together, the first ones before the
  // token's slot and position are known.
  const int step = parts * rows;
#pragma unroll 1
  for (int r0 = begin + part * rows; r0 < end; r0 += kBatch * step) {
    Raw8<In> batch[kBatch][kParts];
    const char* from[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int h = r0 + b * step + row_of;
      if (row_of >= rows || h >= end) continue;
      from[b] = h < keys     ? a.query + token * a.query_row + h * a.query_head
                : h >= values ? a.value + token * a.value_row + (h - values) * a.value_head
                              : a.key + token * a.key_row + (h - keys) * a.key_head;
      batch[b][0].load(from[b] + at.first * In::kBytes);
      if constexpr (kParts == 2)
        if (at.second >= 0) batch[b][1].load(from[b] + at.second * In::kBytes);
    }
    if (r0 == begin + part * rows) {
      place = place_of<kStores>(a, token);
      if (!place.live) return;
      at.load(a, place.angles);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (r0 + b * step >= end) break;
      const int h = r0 + b * step + row_of;
      const bool mine = row_of < rows && h < end;
      const bool is_query = h < keys, is_value = h >= values;
      Raw8<In>(&raw)[kParts] = batch[b];
      float x[kParts][8];
      if (mine) {
        if (!is_value) {
          at.template rotate<In>(a, from[b], place.angles, raw, x,
                                 !is_query && (kFour || (kStores && Cache::kBytes == 1)));
        } else if constexpr (kStores && Cache::kBytes < 2) {
#pragma unroll
          for (int j = 0; j < kParts; ++j) raw[j].get(x[j]);
        }
      }
      // another lane's values have been read: their place may be the result's
      if constexpr (kMode == kTurnLoose) __syncwarp();
      if constexpr (!kStores) {
        if (!mine) continue;
        char* const to = a.query_out + token * a.query_out_row + h * a.query_out_head;
        raw[0].store(to + at.first * In::kBytes);
        if constexpr (kParts == 2)
          if (at.second >= 0) raw[1].store(to + at.second * In::kBytes);
      } else {
        float big[kParts];
        if constexpr (kFour && (kMode == kTurnHalves || kWide)) {
          if constexpr (kMode == kTurnHalves) {
            // a group is two neighbouring lanes' parts
  #pragma unroll
            for (int j = 0; j < kParts; ++j) {
              big[j] = mine && !is_query ? largest8(x[j]) : 0.f;
              big[j] = max_nan(big[j], __shfl_xor_sync(0xffffffffu, big[j], 1));
            }
          } else {
            big[0] = mine ? max_nan(largest8(x[0]), largest8(x[1])) : 0.f;
            big[1] = big[0];
          }
        }
        if (!mine) continue;
        if (is_query) {
          char* const to = a.query_out + token * a.query_out_row + h * a.query_out_head;
          raw[0].store(to + at.first * In::kBytes);
          if constexpr (kParts == 2)
            if (at.second >= 0) raw[1].store(to + at.second * In::kBytes);
          continue;
        }
        const int head = is_value ? h - values : h - keys;
        char* const row = is_value
                              ? a.value_cache + place.block * a.value_cache_block + place.offset * a.value_cache_token
                              : a.key_cache + place.block * a.key_cache_block + place.offset * a.key_cache_token;
        const float scale = is_value ? a.value_scale : a.key_scale;
        if constexpr (kFour) {
          if constexpr (kMode == kTurnHalves || kWide) {
            const int64_t codes = static_cast<int64_t>(a.kv_heads) * (a.dim / 2);
  #pragma unroll
            for (int j = 0; j < kParts; ++j) {
              const int d = j == 0 ? at.first : at.second;
              if (d < 0) continue;
              const uint32_t byte = scale_of(big[j], scale);
              const float unit = e4m3_to_float(byte) * scale;
              *reinterpret_cast<uint32_t*>(row + head * (a.dim / 2) + d / 2) = to_codes(x[j], unit, __frcp_rn(unit));
              if (d % 16 == 0)
                *reinterpret_cast<uint8_t*>(row + codes + head * (a.dim / 16) + d / 16) = static_cast<uint8_t>(byte);
            }
          }
        } else {
          char* const to = row + head * (is_value ? a.value_cache_head : a.key_cache_head);
          if constexpr (Cache::kBytes == 1) {
            const float reciprocal = is_value ? value_reciprocal : key_reciprocal;
            *reinterpret_cast<uint2*>(to + at.first) = to_e4m3x8(x[0], scale, reciprocal);
            if constexpr (kParts == 2)
              if (at.second >= 0) *reinterpret_cast<uint2*>(to + at.second) = to_e4m3x8(x[1], scale, reciprocal);
          } else {
            raw[0].store(to + at.first * In::kBytes);
            if constexpr (kParts == 2)
              if (at.second >= 0) raw[1].store(to + at.second * In::kBytes);
          }
        }
      }
    }
  }
}

// Blocks per SM that the registers leave room for: bound by how many rows are on
// their way, so 28 warps with two turns each at 72 registers beat 20 with three at
// 96 (prompt of 16,384 tokens, 48 heads: 74 us and 77, before what brought it to 67).
// The other modes take what they need.
template <int kMode>
constexpr int kTokenBlocks = kMode == kTurnHalves ? 7 : 1;

template <typename In, typename Cache, int kMode, bool kStores, int kBatch>
__global__ void __launch_bounds__(32 * kTokenWarps, kTokenBlocks<kMode>)
    token_rows_kernel(const __grid_constant__ TokenArgs a) {
  const uint32_t warp = blockIdx.x * kTokenWarps + (threadIdx.x >> 5);  // below 2^32
  const uint32_t token = warp / a.token_warps;
  const int part = static_cast<int>(warp - token * a.token_warps);
  if (token >= a.rows) return;
  if constexpr (kStores && Cache::kBytes == 0 && kMode != kTurnHalves) {
    if (part < a.query_warps)
      token_rows<In, Cache, kMode, kStores, false, kBatch>(a, token, part, a.query_warps);
    else
      token_rows<In, Cache, kMode, kStores, true, kBatch>(a, token, part - a.query_warps,
                                                          a.token_warps - a.query_warps);
  } else {
    token_rows<In, Cache, kMode, kStores, false, kBatch>(a, token, part, a.token_warps);
  }
}

// Turns of a warp at most, for which the token's angles are loaded once and its
// slot and position looked up (the prompt of 16,384 tokens, 12 turns to a token:
// one turn to a warp 150 us, 3 88, 12 74, before what brought it to 67).
constexpr int kTurns = 12;

template <typename In, typename Cache, int kMode, bool kStores>
cudaError_t launch_mode(TokenArgs a, int sms, cudaStream_t stream) {
  constexpr bool kFour = kStores && Cache::kBytes == 0;
  const int kv = kStores ? 2 * a.kv_heads : 0;
  // Turns of a token's heads, `rows` at a time; of queries by themselves, and of
  // what is stored in 4 bits (16 dims to a lane).
  const auto turns_of = [](int heads, int rows) { return (heads + rows - 1) / rows; };
  int turns = 0, query_turns = 0;
  if constexpr (kMode == kTurnHalves) {
    turns = turns_of(a.q_heads + kv, 32 / (a.rotary / 16 + (a.dim - a.rotary) / 8));
  } else if constexpr (kFour) {
    query_turns = turns_of(a.q_heads, 32 / (a.dim / 8));
    turns = turns_of(kv, 32 / (a.dim / 16));
  } else {
    turns = turns_of(a.q_heads + kv, 32 / (a.dim / 8));
  }
  // Fewer turns while that leaves SMs with fewer than 16 warps.
  const int64_t share = a.rows * (turns + query_turns) / (static_cast<int64_t>(sms) * 16);
  const int each = static_cast<int>(share < 1 ? 1 : share < kTurns ? share : kTurns);
  a.query_warps = (query_turns + each - 1) / each;
  a.token_warps = a.query_warps + (turns + each - 1) / each;
  const int64_t warps = a.rows * a.token_warps;
  const dim3 grid(static_cast<unsigned>((warps + kTokenWarps - 1) / kTokenWarps));
  if (each == 1)
    token_rows_kernel<In, Cache, kMode, kStores, 1><<<grid, 32 * kTokenWarps, 0, stream>>>(a);
  else
    token_rows_kernel<In, Cache, kMode, kStores, 2><<<grid, 32 * kTokenWarps, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename In, typename Cache, bool kStores>
cudaError_t launch_rows(const TokenArgs& a, int sms, cudaStream_t stream) {
  const int step = kStores && Cache::kBytes == 0 ? 16 : 8;
  if (a.table != nullptr && a.interleaved) return launch_mode<In, Cache, kTurnPairs, kStores>(a, sms, stream);
  if (a.table != nullptr && a.rotary / 2 % step == 0)
    return launch_mode<In, Cache, kTurnHalves, kStores>(a, sms, stream);
  return launch_mode<In, Cache, kTurnLoose, kStores>(a, sms, stream);
}

// ---------------------------------------------------------------------------
// Back from 8 or 4 bits
// ---------------------------------------------------------------------------

constexpr int kReadThreads = 128;
constexpr int kReadUnits = 2;  // of 16 values, of a thread at a time

// 16 values to `p`, in 32-byte pieces where it is aligned to them.
template <typename Out>
__device__ __forceinline__ void store16(char* p, const float (&x)[16], bool wide) {
  uint32_t w[Out::kBytes * 4];
#pragma unroll
  for (int e = 0; e < 16; e += Out::kBytes == 4 ? 1 : 2) {
    if constexpr (Out::kBytes == 4)
      w[e] = __float_as_uint(x[e]);
    else
      w[e / 2] = pack2<Out::kBf16>(x[e], x[e + 1]);
  }
#pragma unroll
  for (int k = 0; k < Out::kBytes * 4; k += 8) {
    char* const at = p + 4 * k;
    if (wide) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[k]), "r"(w[k + 1]),
                   "r"(w[k + 2]), "r"(w[k + 3]), "r"(w[k + 4]), "r"(w[k + 5]), "r"(w[k + 6]), "r"(w[k + 7])
                   : "memory");
    } else {
      *reinterpret_cast<uint4*>(at) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
      *reinterpret_cast<uint4*>(at + 16) = make_uint4(w[k + 4], w[k + 5], w[k + 6], w[k + 7]);
    }
  }
}

// A block reads `tokens` rows, a thread 16 values of one at a time (4 bits: a group
// with its scale).  Bound by HBM, once enough rows are on their way: 65,536 tokens
// of 8 heads of 128 from 4 bits to bf16 (172 MB) 31 us; with 8 values to a unit a fifth more.
template <typename Out, bool kFour>
__global__ void __launch_bounds__(kReadThreads) read_rows_kernel(const __grid_constant__ ReadArgs a, int tokens,
                                                                uint32_t reciprocal) {
  const uint32_t lanes = a.heads * (a.dim / 16);  // units of a token
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens;
  const uint32_t units = static_cast<uint32_t>(min(static_cast<int64_t>(tokens), a.rows - first)) * lanes;
  const bool wide = reinterpret_cast<uint64_t>(a.out) % 32 == 0;
#pragma unroll 1
  for (uint32_t base = threadIdx.x; base < units; base += kReadThreads * kReadUnits) {
    uint4 raw[kReadUnits];
    uint32_t scale[kReadUnits];
    bool live[kReadUnits];
#pragma unroll
    for (int u = 0; u < kReadUnits; ++u) {
      const uint32_t i = base + u * kReadThreads;
      live[u] = false;
      if (i >= units) continue;
      const uint32_t token = lanes > 1 ? __umulhi(i, reciprocal) : i;  // i / lanes
      const uint32_t at = i - token * lanes;
      const int64_t slot = __ldg(a.slots + first + token);
      if (slot < 0) continue;
      if (slot >= a.num_slots) {
        report(a.status, KVCA_ERR_BAD_INDEX, slot);
        continue;
      }
      live[u] = true;
      const int64_t block = a.block_shift >= 0 ? slot >> a.block_shift : slot / a.block_size;
      const char* const row = a.cache + block * a.cache_block + (slot - block * a.block_size) * a.cache_token;
      if constexpr (kFour) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(row) + at);
        raw[u].x = v.x, raw[u].y = v.y;
        scale[u] = __ldg(reinterpret_cast<const uint8_t*>(row) + a.heads * (a.dim / 2) + at);
      } else {
        const uint32_t h = at / (a.dim / 16);
        raw[u] = __ldg(reinterpret_cast<const uint4*>(row + h * a.cache_head) + (at - h * (a.dim / 16)));
      }
    }
#pragma unroll
    for (int u = 0; u < kReadUnits; ++u) {
      if (!live[u]) continue;
      float x[16];
      if constexpr (kFour) {
        const float unit = e4m3_to_float(scale[u]) * a.scale;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          uint32_t w[4];
          e2m1x8_to_f16x2(w, k == 0 ? raw[u].x : raw[u].y);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack2<false>(w[e]);
            x[8 * k + 2 * e] = f.x * unit, x[8 * k + 2 * e + 1] = f.y * unit;
          }
        }
      } else {
        const uint32_t v[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 f = unpack2<false>(e4m3_to_f16x2(v[e / 2] >> (16 * (e & 1))));
          x[2 * e] = f.x * a.scale, x[2 * e + 1] = f.y * a.scale;
        }
      }
      store16<Out>(a.out + (first * lanes + base + u * kReadThreads) * 16 * Out::kBytes, x, wide);
    }
  }
}

template <typename Out>
cudaError_t launch_read_to(const ReadArgs& a, int sms, cudaStream_t stream) {
  const int64_t lanes = static_cast<int64_t>(a.heads) * (a.dim / 16);  // 16,384 at most
  // kReadUnits rounds of a block where there are rows enough for all SMs
  int64_t tokens = kReadThreads * kReadUnits / lanes;
  while (tokens > 1 && (a.rows + tokens - 1) / tokens < 4 * sms) tokens /= 2;
  if (tokens < 1) tokens = 1;
  const dim3 grid(static_cast<unsigned>((a.rows + tokens - 1) / tokens));
  // exact for i below 2^16 (or a token's own 2^14): i * lanes < 2^32
  const uint32_t reciprocal = static_cast<uint32_t>(((int64_t{1} << 32) + lanes - 1) / lanes);
  if (a.cache_type == KVCA_TYPE_E2M1)
    read_rows_kernel<Out, true><<<grid, kReadThreads, 0, stream>>>(a, static_cast<int>(tokens), reciprocal);
  else
    read_rows_kernel<Out, false><<<grid, kReadThreads, 0, stream>>>(a, static_cast<int>(tokens), reciprocal);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_append_tokens(const TokenArgs& a, int type, int cache_type, int sms, cudaStream_t stream) {
  if (type == KVCA_TYPE_F16) {
    if (cache_type == KVCA_TYPE_E4M3) return launch_rows<CacheF16, CacheE4m3, true>(a, sms, stream);
    if (cache_type == KVCA_TYPE_E2M1) return launch_rows<CacheF16, CacheE2m1Rows, true>(a, sms, stream);
    return launch_rows<CacheF16, CacheF16, true>(a, sms, stream);
  }
  if (cache_type == KVCA_TYPE_E4M3) return launch_rows<CacheBf16, CacheE4m3, true>(a, sms, stream);
  if (cache_type == KVCA_TYPE_E2M1) return launch_rows<CacheBf16, CacheE2m1Rows, true>(a, sms, stream);
  return launch_rows<CacheBf16, CacheBf16, true>(a, sms, stream);
}

cudaError_t launch_rotate_tokens(const TokenArgs& a, int type, int sms, cudaStream_t stream) {
  switch (type) {
    case KVCA_TYPE_F16: return launch_rows<CacheF16, CacheF16, false>(a, sms, stream);
    case KVCA_TYPE_BF16: return launch_rows<CacheBf16, CacheBf16, false>(a, sms, stream);
    default: return launch_rows<InF32, InF32, false>(a, sms, stream);
  }
}

cudaError_t launch_read_tokens(const ReadArgs& a, int type, int sms, cudaStream_t stream) {
  switch (type) {
    case KVCA_TYPE_F16: return launch_read_to<CacheF16>(a, sms, stream);
    case KVCA_TYPE_BF16: return launch_read_to<CacheBf16>(a, sms, stream);
    default: return launch_read_to<InF32>(a, sms, stream);
  }
}

}  // namespace kvca

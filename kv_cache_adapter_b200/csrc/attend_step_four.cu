// Attention of one new token per sequence over a paged cache of 4-bit values:
// e2m1 codes with an e4m3 scale for each 16 dims.
//
// HBM would bound it (144 bytes per token and K/V head of 128 dims, for both
// sides), were there not 64 conversions, 64 multiplications by scales and 16
// products per 16 tokens and warp to issue in the time that these bytes take.
// So everything else is kept off the warps that compute:
//
// * A token's row holds all heads, so the warps that take neighbouring heads (a
//   run) share a ring of token rows, filled by bulk copies: one for each stretch
//   of tokens side by side in memory, a page at least as a rule.  One warp of the
//   run, in turn, looks up the pages of a tile of 32 tokens and starts its copies.
//   (With a ring per warp, filled by 16-byte copies of its head's part, the copies
//   and their addresses were 45 % of all instructions, and each 64-byte piece and
//   each scale a cache line to look up: 257 us for the windowed sequences.)
// * A code's two halves of a byte are converted at once; a value is the code
//   times its scale, which fp16 holds exactly.
// * The running maximum is raised only when a score exceeds it by 2^8, so most
//   tiles need no look across the lanes.  Weights are held times 2^7 of it: those
//   of 2^-21 of the largest keep fp16's 11 bits, those of 2^-31 some.  One term: a
//   weight is off by 2^-12, a value has 2 bits.
//
// Both products run transposed on m16n8k16, tokens (dims) as rows and up to 8
// query heads as columns, as in the step over wider caches, with whose numbering,
// runs and places of partial results this one's agree.
//
// 256 sequences of 500-16,384 tokens, window 4,096 (64 query heads on 8, head dim
// 128): 174-188 us, of which some 27 are fixed (lengths, queries, joins; the last
// run's wait), the rest 2.1 us per tile of 16 warps: 5.0 TB/s, issue slots 60 %,
// ALU 51 %.  (121 us of bytes at the copy's rate; e4m3, twice the bytes, 277.)
//
// Where a run has a part of the heads only, a token's row takes four copies of that
// part's codes and scales.  For the bytes of 94 us at the copy's rate (128 sequences,
// head dim 128): 8 K/V heads 141 us, 16 149; 17 (runs of one head) 560, 32 (of 16)
// 372, 40 (of 10) 302, where e4m3 takes 196-230 for its 167.

#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "attend_step_common.cuh"
#include "kvca_host.cuh"

namespace kvca {
namespace {

constexpr int kRows = 16;        // tokens of one m16n8k16
constexpr int kTile = 32;        // tokens whose rows are fetched together
constexpr int kSegmentCost = 1;  // tiles' worth of a segment's queries and output
constexpr int kRingBytes = 216 * 1024;
constexpr int kMaxStages = 6;    // of a ring
constexpr int kScanGroups = 512; // sequences (or runs of them) in the shared tile counts
constexpr float kShift = 7.f;    // log2 of the weights' factor
constexpr float kGrowth = 8.f;   // log2 of how far a maximum may lag
constexpr float kNoMaximum = -3.4028234e38f;  // of no score yet: any finite one exceeds it by far

using Position = Cursor<kTile, kSegmentCost>;

// DP: head dim padded to 64, 128 or 256; NG: tiles of 8 query heads.
template <int DP, int NG>
struct FourShape {
  static constexpr int kWarps = DP > 128 || (NG > 1 && DP > 64) ? 8 : 16;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kHeads = 8 * NG;
  static constexpr int kSteps = DP / 16;
  static constexpr int kAcc = DP * kHeads;        // floats of a partial output
  static constexpr int kVecs = kAcc / 128;        // float4 of it per lane: NG x kSteps
  static constexpr int kSmem = kRingBytes + 128;  // a lane may read past a row
};

// How a call's work lies on the warps: `span` warps side by side share a run,
// each for a head group of its own: the largest divisor of the head groups that
// there are warps for.  Warps that make no whole run are left out: of 16, one with 3
// or 5 head groups, 4 with 6, 7 with 9, 6 with 10, 5 with 11, 4 with 12; of 8, two
// with 3 and 3 with 5.  Whole rows make up for it (bytes of 94 us: 6 K/V heads 148 us,
// 11 155, 12 144, against 141 with 8), at 9 (185) and 10 (166) not quite; a prime
// above the warps gives runs of one head.
struct FourLayout {
  int parts;   // head groups of a sequence: K/V heads x tiles of query heads
  int span;    // of them in a run
  int chunks;  // runs' worth of them, one after the other in the numbering
  int groups;  // runs of a CTA at a time

  __device__ __forceinline__ FourLayout(int kv_heads, int head_groups, int warps) {
    parts = kv_heads * head_groups;
    span = min(parts, warps);
    while (parts % span != 0) --span;
    chunks = parts / span;
    groups = warps / span;
  }
  // The warp (of the grid) that has run r for the j-th of a run's heads.
  __device__ __forceinline__ int warp_of(int r, int j, int warps) const {
    const int cta = r / groups;
    return cta * warps + (r - cta * groups) * span + j;
  }
};

// The ring of token rows that the warps of a run share.  A stage holds the rows of
// a tile's tokens, keys and then values; where a run has part of the heads only,
// their codes, and then the 16-byte pieces that their scales lie in.
struct RunRing {
  int stages, stage_bytes;
  int pitch;  // of rows
  int codes;  // bytes of them before the scales
  int ahead;  // tiles fetched before the one that is computed

  __device__ __forceinline__ RunRing(const AttendArgs& a, const FourLayout& layout, int head_groups) {
    if (layout.chunks == 1) {
      codes = a.kv_heads * (a.dim / 2);
      pitch = a.row_bytes;
    } else {
      const int heads = min(a.kv_heads, (layout.span + head_groups - 2) / head_groups + 1);  // at most
      codes = heads * (a.dim / 2);
      pitch = codes + ((heads * (a.dim / 16) + 30) & ~15);
    }
    stage_bytes = 2 * kTile * pitch;
    stages = min(kMaxStages, ring_bytes(layout) / stage_bytes);  // two at least: 16 heads of 128, 8 of 256
    ahead = stages > 3 ? stages - 2 : stages - 1;
  }
  static __device__ __forceinline__ int ring_bytes(const FourLayout& layout) {
    return kRingBytes / layout.groups & ~127;
  }
};

// What a warp keeps in shared memory of the tiles that it has to fetch.
struct alignas(16) Fetch {
  Position at;         // the next one
  int stage, round;    // of the ring, for it
  uint32_t mine, parity;  // stages that this warp has filled, and the phase that its copies end
};

// Token of a row of the products: rows side by side, which a quarter of a warp
// reads together, are an odd number of tokens apart (rows of memory that begin 64
// bytes apart, modulo 128, lie on different banks).
__device__ __forceinline__ int row_token(int row) { return row & 1 ? 4 + ((row >> 1) ^ 1) : row >> 1; }

// N = 1, 2 or 4 words of shared memory.
template <int N>
__device__ __forceinline__ void load_shared(uint32_t (&w)[N], uint32_t addr) {
  if constexpr (N == 1)
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr) : "memory");
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t load_shared16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ uint32_t load_shared8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Both halves of a register alike (the multiplication's operand takes one half
// twice).
__device__ __forceinline__ uint32_t low_twice(uint32_t v) {
  uint32_t r;
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %1;\nmov.b32 %0, {a, a};\n}" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t high_twice(uint32_t v) {
  uint32_t r;
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %1;\nmov.b32 %0, {b, b};\n}" : "=r"(r) : "r"(v));
  return r;
}

// d = a b, with nothing before it.
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
               "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// The scales of kGroups groups of a row from group `first` on, at `addr`, each
// twice in a register; groups from `groups` on, which are padding of odd head
// dims, have none.
template <int kGroups, bool kOdd>
__device__ __forceinline__ void read_scales(uint32_t (&unit)[kGroups], uint32_t addr, int first, int groups) {
  if constexpr (kGroups == 1) {
    unit[0] = low_twice(e4m3_to_f16x2(load_shared8(addr)));
  } else {
#pragma unroll
    for (int j = 0; j < kGroups; j += 2) {
      const uint32_t v = e4m3_to_f16x2(load_shared16(addr + j));
      unit[j] = low_twice(v);
      unit[j + 1] = high_twice(v);
    }
  }
  if constexpr (kOdd) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
      if (first + j >= groups) unit[j] = 0;
  }
}

// The same scales of two rows, side by side in a register.
template <int kGroups, bool kOdd>
__device__ __forceinline__ void read_scale_pairs(uint32_t (&unit)[kGroups], uint32_t one, uint32_t other, int first,
                                                 int groups) {
  if constexpr (kGroups == 1) {
    unit[0] = e4m3_to_f16x2(__byte_perm(load_shared8(one), load_shared8(other), 0x0040));
  } else {
    const uint32_t a = load_shared16(one), b = load_shared16(other);
    unit[0] = e4m3_to_f16x2(__byte_perm(a, b, 0x0040));
    unit[1] = e4m3_to_f16x2(__byte_perm(a, b, 0x0051));
  }
  if constexpr (kOdd) {
#pragma unroll
    for (int j = 0; j < kGroups; ++j)
      if (first + j >= groups) unit[j] = 0;
  }
}

// kOdd: the head dim is not DP.
template <int DP, int NG, bool kOdd>
__global__ void __launch_bounds__(FourShape<DP, NG>::kThreads, 1)
    attend_step_four_kernel(const __grid_constant__ AttendArgs a, void* workspace, uint32_t* arrived) {
  using Shape = FourShape<DP, NG>;
  constexpr int kHeads = Shape::kHeads;
  constexpr int kSteps = Shape::kSteps;
  constexpr int kWarps = Shape::kWarps;
  extern __shared__ __align__(128) unsigned char rings[];
  __shared__ int64_t prefix[kScanGroups + 1];
  __shared__ int64_t scan[33];
  __shared__ uint64_t bars[kWarps * 2 * kMaxStages];  // full and empty stages of each run's ring
  __shared__ Fetch fetches[kWarps];
  __shared__ StepJoin leaves[kWarps][2];  // segments whose results a warp leaves in its places
  __shared__ int held[kWarps];
  __shared__ __align__(16) float held_ml[kWarps][2 * kHeads];
  __shared__ StepJoin joins[2 * kWarps];
  __shared__ int join_count;
  __shared__ int gave_up;

  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int head_groups = (a.group + kHeads - 1) / kHeads;
  const FourLayout layout(a.kv_heads, head_groups, kWarps);
  const int chunks = layout.chunks, span = layout.span;
  StepWorkspace<kHeads, Shape::kAcc> ws(workspace, static_cast<int64_t>(gridDim.x) * kWarps);

  // Tile counts of the sequences, or of runs of `per` of them.
  const int per = (a.num_seqs + kScanGroups - 1) / kScanGroups;
  const int scanned = (a.num_seqs + per - 1) / per;
  int64_t tiles = 0;
  for (int base = 0; base < scanned; base += Shape::kThreads) {
    const int g = base + threadIdx.x;
    int64_t n = 0;
    if (g < scanned) {
      const int end = min(a.num_seqs, (g + 1) * per);
      for (int seq = g * per; seq < end; ++seq) {
        Position c;
        c.seq = seq;
        c.load(a);
        n += sequence_share<kSegmentCost>(c.tiles, chunks);
      }
    }
    int64_t total;
    const int64_t before = block_excl_scan(n, &total, scan);
    if (g < scanned) prefix[g] = tiles + before;
    tiles += total;
  }
  const int64_t runs = min(static_cast<int64_t>(gridDim.x) * layout.groups, tiles);
  if (threadIdx.x == 0) {
    join_count = 0;
    gave_up = 0;
  }
  if (threadIdx.x < layout.groups * kMaxStages) {
    barrier_init(smem_addr(bars) + 16 * threadIdx.x, 1);
    barrier_init(smem_addr(bars) + 16 * threadIdx.x + 8, span);
  }
  if (threadIdx.x < 2 * kWarps) leaves[threadIdx.x / 2][threadIdx.x % 2].segment = -1;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();

  // Sequences without tokens: the sum over nothing.
  for (int seq = blockIdx.x; seq < a.num_seqs; seq += gridDim.x) {
    if (__ldg(a.lens + seq) != 0) continue;
    const int64_t row = static_cast<int64_t>(seq) * a.kv_heads * a.group;
    const int n = a.kv_heads * a.group;
    for (int i = threadIdx.x; i < n * a.dim; i += Shape::kThreads)
      static_cast<uint16_t*>(a.out)[row * a.dim + i] = 0;
    if (a.lse != nullptr)
      for (int i = threadIdx.x; i < n; i += Shape::kThreads) a.lse[row + i] = -INFINITY;
  }

  const int64_t own = static_cast<int64_t>(blockIdx.x) * kWarps + warp;  // where this warp leaves results
  const int64_t my_run = static_cast<int64_t>(blockIdx.x) * layout.groups + warp / span;
  const int lane_of_heads = warp % span;
  const Patience patience{&gave_up, a.wait_limit};
  int held_segment = -1;
  bool held_starts = false;
  StepJoin held_runs{-1, 0, 0};

  // Lane 4 i + t has of the heads 2 t and 2 t + 1 of each tile of 8 the maxima, its
  // share of the sums, and the dims i DP / 8 and on of the outputs: acc[][b] are dims
  // 2 b of those (both heads), then 2 b + 1.
  float acc[NG][kSteps][4];
  float m[NG][2], l[NG][2];

  // The output of a segment from acc, m and the whole sums l.
  auto write_out = [&](int seq, int part) {
    const int kv_head = part / head_groups;
    const int first = (part - kv_head * head_groups) * kHeads;
    const int64_t row = (static_cast<int64_t>(seq) * a.kv_heads + kv_head) * a.group;
    const bool bf16 = a.query_type == KVCA_TYPE_BF16;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const float r0 = a.value_scale / l[n][0], r1 = a.value_scale / l[n][1];
      const int h = first + n * 8 + (lane >> 2);
      uint16_t* const out = static_cast<uint16_t*>(a.out) + (row + h) * a.dim;
#pragma unroll
      for (int r = 0; r < kSteps / 2; ++r) {
        uint32_t w[2][2];  // dims 4 r + 2 p + j
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = acc[n][2 * r + p][2 * j] * r0, y = acc[n][2 * r + p][2 * j + 1] * r1;
            // now of head i, the dims of lanes 4 (2 t) and 4 (2 t + 1)
            w[p][j] = transpose8x8(bf16 ? pack2<true>(x, y) : pack2<false>(x, y));
          }
        if (h >= a.group) continue;
        const int d = (lane & 3) * (DP / 4) + 4 * r;
        if (d < a.dim)
          *reinterpret_cast<uint2*>(out + d) =
              make_uint2(__byte_perm(w[0][0], w[0][1], 0x5410), __byte_perm(w[1][0], w[1][1], 0x5410));
        if (d + DP / 8 < a.dim)
          *reinterpret_cast<uint2*>(out + d + DP / 8) =
              make_uint2(__byte_perm(w[0][0], w[0][1], 0x7632), __byte_perm(w[1][0], w[1][1], 0x7632));
      }
      if (a.lse != nullptr && lane < 4) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int hh = first + n * 8 + 2 * lane + j;
          if (hh < a.group) a.lse[row + hh] = (m[n][j] - kShift) * kLn2 + logf(l[n][j]);
        }
      }
    }
  };
  // Partial results lie as the lanes hold them, a float4 each.
  auto leave = [&](int slot) {
    float* const ml = ws.ml_of(own, slot);
    float4* const to = reinterpret_cast<float4*>(ws.acc_of(own, slot)) + lane;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      if (lane < 4) {
        *reinterpret_cast<float2*>(ml + n * 8 + 2 * lane) = make_float2(m[n][0], m[n][1]);
        *reinterpret_cast<float2*>(ml + kHeads + n * 8 + 2 * lane) = make_float2(l[n][0], l[n][1]);
      }
#pragma unroll
      for (int t = 0; t < kSteps; ++t)
        to[(n * kSteps + t) * 32] = make_float4(acc[n][t][0], acc[n][t][1], acc[n][t][2], acc[n][t][3]);
    }
  };
  // Another partial result into acc, m and l.
  auto fold = [&](const float2 (&top)[NG], const float2 (&sum)[NG], const float4 (&from)[Shape::kVecs]) {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const float tops[2] = {top[n].x, top[n].y}, sums[2] = {sum[n].x, sum[n].y};
      float keep[2], weight[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float best = fmaxf(m[n][j], tops[j]);
        keep[j] = exp2_approx(m[n][j] - best);
        weight[j] = exp2_approx(tops[j] - best);
        m[n][j] = best;
        l[n][j] = l[n][j] * keep[j] + sums[j] * weight[j];
      }
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        const float4 v = from[n * kSteps + t];
        acc[n][t][0] = acc[n][t][0] * keep[0] + v.x * weight[0];
        acc[n][t][1] = acc[n][t][1] * keep[1] + v.y * weight[1];
        acc[n][t][2] = acc[n][t][2] * keep[0] + v.z * weight[0];
        acc[n][t][3] = acc[n][t][3] * keep[1] + v.w * weight[1];
      }
    }
  };
  auto clear = [&]() {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
#pragma unroll
      for (int t = 0; t < kSteps; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][t][j] = 0.f;
      m[n][0] = m[n][1] = kNoMaximum;
      l[n][0] = l[n][1] = 0.f;
    }
  };

  if (warp < layout.groups * span && my_run < runs) {
    const RunRing ring(a, layout, head_groups);
    const uint32_t ring_base = smem_addr(rings) + warp / span * RunRing::ring_bytes(layout);
    const uint32_t ring_bars = smem_addr(bars) + warp / span * (16 * kMaxStages);
    bool ok = true;  // no wait has given up
    // With a limit of 0, whether the phase is over now.
    auto await = [&](uint32_t bar, uint32_t parity) {
      if (a.wait_limit > 0) {
        ok = warp_wait(bar, parity, patience) && ok;
      } else if (!__all_sync(0xffffffffu, barrier_test(bar, parity))) {
        *patience.gave_up = 1;
        ok = false;
      }
    };

    Position at;  // the tile computed next
    {
      const int64_t begin = run_begin(tiles, runs, my_run), finish = run_begin(tiles, runs, my_run + 1);
      int lo = 0, hi = scanned;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= begin) lo = mid; else hi = mid;
      }
      int64_t rest = begin - prefix[lo];
      at.seq = lo * per;
      at.load(a);
      while (rest >= sequence_share<kSegmentCost>(at.tiles, chunks) && at.seq + 1 < a.num_seqs) {
        rest -= sequence_share<kSegmentCost>(at.tiles, chunks);
        ++at.seq;
        at.load(a);
      }
      const int segment = at.tiles + kSegmentCost;
      at.chunk = static_cast<int>(rest / segment);
      at.tile = static_cast<int>(rest - static_cast<int64_t>(at.chunk) * segment) - kSegmentCost;
      at.left = static_cast<int>(finish - begin);
      if (at.tile < 0) {  // the costs of the first segment
        at.left += at.tile;
        at.tile = 0;
      }
    }

    // The tiles that this warp fetches: one of `span`.  A lane looks up the page of
    // one token, a turn before its rows are copied.
    constexpr int64_t kHidden = -1ll << 62;  // no token of this tile
    int64_t page = kHidden;
    int offset = 0;
    auto look_up = [&](const Position& p) {
      const int v = p.tile * kTile + lane;
      page = kHidden;
      if (lane < kTile && v < p.vis.count) {
        const int pos = p.vis.position(v);
        const int block = a.block_shift >= 0 ? pos >> a.block_shift : pos / a.block_size;
        offset = pos - block * a.block_size;
        page = __ldg(a.tables + static_cast<int64_t>(p.seq) * a.table_stride + block);
      }
      if (p.tile < span) {
        // the segment's queries, on their way to the first-level cache
        const int part = p.chunk * span + lane_of_heads, kv_head = part / head_groups;
        const int h = (part - kv_head * head_groups) * kHeads + (lane >> 1);
        if (lane < 2 * kHeads && h < a.group)
          asm volatile("prefetch.global.L1 [%0];" ::"l"(
              static_cast<const uint16_t*>(a.query) + static_cast<int64_t>(p.seq) * a.query_row +
              static_cast<int64_t>(kv_head * a.group + h) * a.query_head + (lane & 1) * min(64, a.dim - 1)));
      }
    };
    int done = -ring.ahead;  // tiles computed; before the first, tiles until then
    int due = lane_of_heads; // the next one to fetch, counted alike
    {
      Fetch f;
      f.at = at;
      f.stage = lane_of_heads % ring.stages;
      f.round = lane_of_heads / ring.stages;
      f.mine = f.parity = 0;
      if (f.at.skip(a, chunks, lane_of_heads))
        look_up(f.at);
      else
        due = 1 << 30;
      if (lane == 0) fetches[warp] = f;
      __syncwarp();
    }
    // Starts the copies of the rows of the tile that is due.  Rows of hidden tokens,
    // and of a page outside the cache, are left out.
    auto fetch = [&]() {
      Fetch f = fetches[warp];
      const bool good = page >= 0 && page < a.num_blocks;
      if (!good && page != kHidden) report(a.status, KVCA_ERR_BAD_INDEX, page);
      const uint32_t full = ring_bars + 16 * f.stage;
      if (f.round > 0) await(full + 8, static_cast<uint32_t>(f.round - 1) & 1u);
      if (ok) {
        const unsigned seen = __ballot_sync(0xffffffffu, good);
        // K/V heads of which the run has parts, and the pieces of their scales
        const int first = f.at.chunk * span / head_groups;
        const int heads = (f.at.chunk * span + span - 1) / head_groups + 1 - first;
        const int in_row = a.kv_heads * (a.dim / 2) + first * (a.dim / 16);
        const int scales = in_row & ~15, scale_bytes = ((in_row + heads * (a.dim / 16) + 15) & ~15) - scales;
        const uint32_t row_bytes = chunks == 1 ? ring.pitch : heads * (a.dim / 2) + scale_bytes;
        if (lane == 0) barrier_arrive_expect(full, 2u * __popc(seen) * row_bytes);
        f.mine |= 1u << f.stage;
        f.parity = (f.parity & ~(1u << f.stage)) | (static_cast<uint32_t>(f.round) & 1u) << f.stage;
        __syncwarp();
        const int64_t block = good ? page : 0;
        const char* const key_row = a.key + block * a.key_block + offset * a.key_token;
        const char* const value_row = a.value + block * a.value_block + offset * a.value_token;
        const uint32_t to = ring_base + f.stage * ring.stage_bytes + lane * ring.pitch;
        const uint32_t values = kTile * ring.pitch;
        if (chunks == 1) {
          const unsigned long long k = reinterpret_cast<unsigned long long>(key_row);
          const unsigned long long v = reinterpret_cast<unsigned long long>(value_row);
          const unsigned long long k_before = __shfl_up_sync(0xffffffffu, k, 1);
          const unsigned long long v_before = __shfl_up_sync(0xffffffffu, v, 1);
          const bool follows = lane > 0 && ((seen >> (lane - 1)) & 1u) && k_before + ring.pitch == k &&
                               v_before + ring.pitch == v;
          const unsigned ends = ~seen | __ballot_sync(0xffffffffu, !follows);
          if (good && !follows) {
            const unsigned behind = lane < 31 ? ends >> (lane + 1) : 0u;
            const uint32_t bytes = (behind != 0 ? __ffs(behind) : 32 - lane) * ring.pitch;
            copy_bulk(to, key_row, bytes, full);
            copy_bulk(to + values, value_row, bytes, full);
          }
        } else if (good) {
          const int codes = first * (a.dim / 2);
          copy_bulk(to, key_row + codes, heads * (a.dim / 2), full);
          copy_bulk(to + ring.codes, key_row + scales, scale_bytes, full);
          copy_bulk(to + values, value_row + codes, heads * (a.dim / 2), full);
          copy_bulk(to + values + ring.codes, value_row + scales, scale_bytes, full);
        }
      }
      f.stage += span;
      while (f.stage >= ring.stages) {
        f.stage -= ring.stages;
        ++f.round;
      }
      due += span;
      if (f.at.skip(a, chunks, span))
        look_up(f.at);
      else
        due = 1 << 30;
      __syncwarp();
      if (lane == 0) fetches[warp] = f;
      __syncwarp();
    };
#pragma unroll 1
    for (; done < 0; ++done)
      if (done + ring.ahead >= due) fetch();

    uint32_t q[NG][kSteps][2];
    float unit[NG][2];  // score factor of the heads 2 * (lane % 4), + 1
    const int my_token = row_token(lane >> 2);
    // Where this lane reads in a stage: keys of row lane / 4, and values of row 2
    // (lane % 4); their scales; from one row to the next.
    uint32_t key_at = 0, key_scale_at = 0, value_at = 0, value_scale_at = 0;
    const int next_row = (row_token(2 * (lane & 3) + 1) - row_token(2 * (lane & 3))) * ring.pitch;
    bool starts = at.tile == 0;
    bool fresh = true;
    int stage = 0;
    uint32_t phase = 0;
#pragma unroll 1
    for (bool go = at.left > 0; go;) {
      if (fresh) {
        // the segment's queries as the B operand: column (head) lane / 4, dims
        // (lane % 4) DP / 4 and on, four per step; fp16 products, each row times a
        // power of two (power_up)
        const int part = at.chunk * span + lane_of_heads;
        const int kv_head = part / head_groups;
        const int first = (part - kv_head * head_groups) * kHeads;
        const bool bf16 = a.query_type == KVCA_TYPE_BF16;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const int h = first + n * 8 + (lane >> 2);
          const bool live = h < a.group;
          const uint16_t* row = static_cast<const uint16_t*>(a.query) + static_cast<int64_t>(at.seq) * a.query_row +
                                static_cast<int64_t>(kv_head * a.group + (live ? h : 0)) * a.query_head;
          float big = 0.f;
          uint2 raw[kSteps];
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const int d = (lane & 3) * (DP / 4) + 4 * k;
            raw[k] = live && d < a.dim ? *reinterpret_cast<const uint2*>(row + d) : make_uint2(0, 0);
            const float2 x = bf16 ? unpack2<true>(raw[k].x) : unpack2<false>(raw[k].x);
            const float2 y = bf16 ? unpack2<true>(raw[k].y) : unpack2<false>(raw[k].y);
            big = fmaxf(big, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
          }
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          const int e = power_up(big);
          const float up = power_of_two(e);
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            const float2 x = bf16 ? unpack2<true>(raw[k].x) : unpack2<false>(raw[k].x);
            const float2 y = bf16 ? unpack2<true>(raw[k].y) : unpack2<false>(raw[k].y);
            q[n][k][0] = pack2<false>(x.x * up, x.y * up);
            q[n][k][1] = pack2<false>(y.x * up, y.y * up);
          }
          const float mine = a.scale_log2 * power_of_two(-e);
          unit[n][0] = __shfl_sync(0xffffffffu, mine, (2 * (lane & 3)) * 4);
          unit[n][1] = __shfl_sync(0xffffffffu, mine, (2 * (lane & 3) + 1) * 4);
        }
        clear();
        const int leading = at.chunk * span / head_groups;  // K/V head of the rows in the ring
        const int codes_at = (kv_head - leading) * (a.dim / 2);
        const int scales_at = ring.codes + ((a.kv_heads * (a.dim / 2) + leading * (a.dim / 16)) & 15) +
                              (kv_head - leading) * (a.dim / 16);
        key_at = my_token * ring.pitch + codes_at + (lane & 3) * (DP / 8);
        key_scale_at = my_token * ring.pitch + scales_at + (lane & 3) * (DP / 64);
        const int value_row = (kTile + row_token(2 * (lane & 3))) * ring.pitch;
        value_at = value_row + codes_at + (lane >> 2) * (DP / 16);
        value_scale_at = value_row + scales_at + (lane >> 2) * (DP / 8) / 16;
        fresh = false;
      }

      await(ring_bars + 16 * stage, phase);
      const uint32_t rows = ring_base + stage * ring.stage_bytes;
      const int count = at.vis.count - at.tile * kTile;

#pragma unroll 1
      for (int sub = 0; sub < min(count, kTile); sub += kRows) {
        const uint32_t own_rows = rows + sub * ring.pitch;
        const int left = count - sub;
        // S^T = K Q^T: row i is token row_token(i), lane 4 i + t has its dims t DP / 4
        // and on, four per step, as the query's are above
        float s[NG][2][4];
        {
          constexpr int kWords = DP / 32, kRead = kWords > 4 ? 4 : kWords;
          constexpr int kGroups = DP / 64;  // of 16 dims, of a lane
          uint32_t w[2][kWords], scale[2][kGroups];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int part = 0; part < kWords / kRead; ++part) {
              uint32_t x[kRead];
              load_shared(x, own_rows + key_at + 8 * i * ring.pitch + part * 16);
#pragma unroll
              for (int j = 0; j < kRead; ++j) w[i][part * kRead + j] = x[j];
            }
            read_scales<kGroups, kOdd>(scale[i], own_rows + key_scale_at + 8 * i * ring.pitch, (lane & 3) * kGroups,
                                       a.dim / 16);
          }
#pragma unroll
          for (int k = 0; k < kSteps; k += 2) {
            uint32_t x[4], y[4];
            e2m1x8_to_f16x2(x, w[0][k / 2]);
            e2m1x8_to_f16x2(y, w[1][k / 2]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[j] = mul_f16x2(x[j], scale[0][k / 4]);
              y[j] = mul_f16x2(y[j], scale[1][k / 4]);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t f[4] = {x[2 * j], y[2 * j], x[2 * j + 1], y[2 * j + 1]};
#pragma unroll
              for (int n = 0; n < NG; ++n) {
                if (k == 0)
                  mma16816_first(s[n][j], f, q[n][k + j][0], q[n][k + j][1]);
                else
                  mma16816<false>(s[n][j], f, q[n][k + j][0], q[n][k + j][1]);
              }
            }
          }
        }

        // softmax; y: log2 of the weights
        float y[NG][4];
        float most = -INFINITY;
        const bool cut = left < kRows;
        const bool hidden0 = my_token >= left, hidden1 = my_token + 8 >= left;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[n][0][j] += s[n][1][j];
            y[n][j] = fmaf(s[n][0][j], unit[n][j & 1], kShift - m[n][j & 1]);
          }
          if (cut) {  // whatever the ring held there
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (j < 2 ? hidden0 : hidden1) y[n][j] = -INFINITY;
          }
          most = max3(max3(most, y[n][0], y[n][1]), y[n][2], y[n][3]);
        }
        if (__any_sync(0xffffffffu, most > kShift + kGrowth)) {
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            float decay[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float top = fmaxf(hidden0 ? -INFINITY : s[n][0][j] * unit[n][j],
                                hidden1 ? -INFINITY : s[n][0][j + 2] * unit[n][j]);
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
              top = fmaxf(top, m[n][j]);
              decay[j] = exp2_approx(m[n][j] - top);
              m[n][j] = top;
              l[n][j] *= decay[j];
            }
#pragma unroll
            for (int t = 0; t < kSteps; ++t)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[n][t][j] *= decay[j & 1];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              y[n][j] = (j < 2 ? hidden0 : hidden1)
                            ? -INFINITY
                            : fmaf(s[n][0][j], unit[n][j & 1], kShift - m[n][j & 1]);
          }
        }
        uint32_t p[NG][2];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
#pragma unroll
          for (int j = 0; j < 4; ++j) y[n][j] = exp2_approx(y[n][j]);
          l[n][0] += y[n][0] + y[n][2];
          l[n][1] += y[n][1] + y[n][3];
          p[n][0] = transpose8x8(pack2<false>(y[n][0], y[n][1]));
          p[n][1] = transpose8x8(pack2<false>(y[n][2], y[n][3]));
        }

        // O^T += V^T P^T.  Lane 4 i + t: dims i DP / 8 and on of the tokens of rows 2 t,
        // 2 t + 1, 2 t + 8 and 2 t + 9.  A byte is two dims of one token, the operand wants
        // one dim of two tokens in a register: the codes of two tokens are paired before
        // they are converted, 16 operations for 32 registers.  (With a product each for
        // the even and the odd dims instead, tokens' weights beside zeros, the
        // multiplications by scales wait for the tensor cores: 203 us for 187.)
        constexpr int kWords = DP / 64;  // of a lane's dims of a token
        constexpr int kGroups = DP > 128 ? 2 : 1;
        uint32_t w[4][kWords], scale[2][kGroups];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          load_shared(w[i], own_rows + value_at + 8 * (i / 2) * ring.pitch + (i % 2) * next_row);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t first_row = own_rows + value_scale_at + 8 * i * ring.pitch;
          read_scale_pairs<kGroups, kOdd>(scale[i], first_row, first_row + next_row, (lane >> 2) * (DP / 8) / 16,
                                          a.dim / 16);
          if (cut) {  // nothing of what the ring held there
            const uint32_t keep = (row_token(2 * (lane & 3)) + 8 * i < left ? 0xffffu : 0u) |
                                  (row_token(2 * (lane & 3) + 1) + 8 * i < left ? 0xffff0000u : 0u);
#pragma unroll
            for (int j = 0; j < kGroups; ++j) scale[i][j] &= keep;
          }
        }
#pragma unroll
        for (int r = 0; r < kWords; ++r) {
          uint32_t x[4][4];  // even dims of the first two tokens, odd ones, and of the others
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t one = w[2 * i][r], other = w[2 * i + 1][r];
            e2m1x8_to_f16x2(x[2 * i], (one & 0x0f0f0f0fu) | (other << 4 & 0xf0f0f0f0u));
            e2m1x8_to_f16x2(x[2 * i + 1], (one >> 4 & 0x0f0f0f0fu) | (other & 0xf0f0f0f0u));
          }
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const uint32_t f[4] = {mul_f16x2(x[0][b], scale[0][r / 2]), mul_f16x2(x[1][b], scale[0][r / 2]),
                                   mul_f16x2(x[2][b], scale[1][r / 2]), mul_f16x2(x[3][b], scale[1][r / 2])};
#pragma unroll
            for (int n = 0; n < NG; ++n) mma16816<false>(acc[n][4 * r + b], f, p[n][0], p[n][1]);
          }
        }
        // in the middle of a tile, when the other warps have long left the stage of
        // the tile before it
        if (sub == 0 && done + ring.ahead >= due) fetch();
      }
      __syncwarp();
      if (lane == 0) barrier_arrive(ring_bars + 16 * stage + 8);
      if (++stage == ring.stages) {
        stage = 0;
        phase ^= 1u;
      }
      ++done;

      const bool ends = at.ends();
      go = !at.last();
      if (!ends && go) {
        ++at.tile;
        --at.left;
        continue;
      }
      // the segment, or this run's share of it, is done
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 4);
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 8);
          l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 16);
        }
      const int part = at.chunk * span + lane_of_heads;
      const int segment = at.seq * layout.parts + part;
      // the segment's first tile in the numbering
      const int64_t here = run_begin(tiles, runs, my_run + 1) - at.left - at.tile;
      const int this_run = static_cast<int>(my_run);
      if (ends && starts) {
        write_out(at.seq, part);
      } else if (ends) {
        // the end of a segment that an earlier run began
        if (lane == 0) leaves[warp][0] = StepJoin{segment, run_of(tiles, runs, here), this_run};
        leave(0);
      } else {
        held_segment = segment;
        held_starts = starts;
        held_runs = StepJoin{segment, starts ? this_run : run_of(tiles, runs, here),
                             run_of(tiles, runs, here + at.tiles - 1)};
      }
      if (go) {
        at.advance(a, chunks);
        go = at.left > 0;
        starts = true;
        fresh = true;
      }
    }
    // After a wait that gave up, copies of this warp may still run: they end before
    // the ring is used again (bounded, 80 ms each).
    if (*patience.gave_up != 0) {
      const Fetch f = fetches[warp];
      for (int i = 0; i < ring.stages; ++i)
        if ((f.mine >> i) & 1u)
          for (int k = 0; k < 4096 && !barrier_try_for(ring_bars + 16 * i, (f.parity >> i) & 1u, kTryTime); ++k) {
          }
      __syncwarp();
    }
  }

  // Partial results that the CTA's warps still hold: of warps of following runs
  // with the same segment, the first takes the others' through the rings, which are
  // free now, and leaves their sum.
  if (lane == 0) held[warp] = held_segment;
  if (held_segment >= 0 && lane < 4) {
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        held_ml[warp][n * 8 + 2 * lane + j] = m[n][j];
        held_ml[warp][kHeads + n * 8 + 2 * lane + j] = l[n][j];
      }
  }
  __syncthreads();
  if (threadIdx.x == 0 && gave_up != 0) report(a.status, KVCA_ERR_DEVICE_TIMEOUT, blockIdx.x);
  float4* const parked = reinterpret_cast<float4*>(rings) + lane;  // [warp][kVecs][lane]
  auto park = [&]() {
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int t = 0; t < kSteps; ++t)
        parked[(warp * Shape::kVecs + n * kSteps + t) * 32] =
            make_float4(acc[n][t][0], acc[n][t][1], acc[n][t][2], acc[n][t][3]);
  };
  auto take = [&](int from) {  // what warp `from` has parked
    float2 top[NG], sum[NG];
    float4 v[Shape::kVecs];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      top[n] = *reinterpret_cast<const float2*>(&held_ml[from][n * 8 + 2 * (lane & 3)]);
      sum[n] = *reinterpret_cast<const float2*>(&held_ml[from][kHeads + n * 8 + 2 * (lane & 3)]);
    }
#pragma unroll
    for (int t = 0; t < Shape::kVecs; ++t) v[t] = parked[(from * Shape::kVecs + t) * 32];
    fold(top, sum, v);
  };
  const bool follows = held_segment >= 0 && warp >= span && held[warp - span] == held_segment;
  if (follows) park();
  __syncthreads();
  if (held_segment >= 0 && !follows) {
#pragma unroll 1
    for (int k = warp + span; k < kWarps && held[k] == held_segment; k += span) take(k);
    leave(held_starts ? 1 : 0);
    if (lane == 0) leaves[warp][held_starts ? 1 : 0] = held_runs;
  }

  // Whoever leaves the last result of a segment joins them, in run order: a warp
  // alone while they are few, the CTA when they are many (a long sequence over all
  // SMs).  The count of a segment's results is kept at its first run's warp, and is
  // zero again then.
  constexpr int kWarpResults = 8;
  auto gather = [&](const StepJoin& join, int results, int first_result, int stride) {
    clear();
#pragma unroll 1
    for (int k = first_result; k < results; k += stride) {
      const int r = result_run(k, join.first_run, join.last_run, layout.groups);
      const int w = layout.warp_of(r, join.segment % layout.parts % span, kWarps);
      const int slot = k == 0 ? 1 : 0;
      float2 top[NG], sum[NG];
      float4 v[Shape::kVecs];
      const float4* const from = reinterpret_cast<const float4*>(ws.acc_of(w, slot)) + lane;
#pragma unroll
      for (int t = 0; t < Shape::kVecs; ++t) v[t] = __ldcg(from + t * 32);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        top[n] = __ldcg(reinterpret_cast<const float2*>(ws.ml_of(w, slot) + n * 8 + 2 * (lane & 3)));
        sum[n] = __ldcg(reinterpret_cast<const float2*>(ws.ml_of(w, slot) + kHeads + n * 8 + 2 * (lane & 3)));
      }
      fold(top, sum, v);
    }
  };

  __threadfence();
  __syncwarp();
  bool mine_last = false;
  if (lane < 2) {
    const StepJoin mine = leaves[warp][lane];
    if (mine.segment >= 0) {
      uint32_t* const count = arrived + layout.warp_of(mine.first_run, lane_of_heads, kWarps);
      const int results = result_count(mine.first_run, mine.last_run, layout.groups);
      if (atomicAdd(count, 1u) == static_cast<uint32_t>(results) - 1) {
        *count = 0;
        if (results <= kWarpResults)
          mine_last = true;
        else
          joins[atomicAdd(&join_count, 1)] = mine;
      }
    }
  }
  __threadfence();
  const unsigned alone = __ballot_sync(0xffffffffu, mine_last);
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    if (!((alone >> which) & 1u)) continue;
    const StepJoin join = leaves[warp][which];
    gather(join, result_count(join.first_run, join.last_run, layout.groups), 0, 1);
    write_out(join.segment / layout.parts, join.segment % layout.parts);
  }
  __syncthreads();
  const int join_total = join_count;
#pragma unroll 1
  for (int j = 0; j < join_total; ++j) {
    const StepJoin join = joins[j];
    gather(join, result_count(join.first_run, join.last_run, layout.groups), warp, kWarps);
    if (lane < 4) {
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          held_ml[warp][n * 8 + 2 * lane + i] = m[n][i];
          held_ml[warp][kHeads + n * 8 + 2 * lane + i] = l[n][i];
        }
    }
    park();
    __syncthreads();
    if (warp == 0) {
#pragma unroll 1
      for (int k = 1; k < kWarps; ++k) take(k);
      write_out(join.segment / layout.parts, join.segment % layout.parts);
    }
    __syncthreads();
  }
}

template <int DP, int NG, bool kOdd>
cudaError_t launch_typed(const AttendArgs& a, void* workspace, uint32_t* arrived, int sms, cudaStream_t stream) {
  using Shape = FourShape<DP, NG>;
  auto kernel = attend_step_four_kernel<DP, NG, kOdd>;
  static DeviceFlags configured;
  int dev = -1;
  if (needs_setup(configured, &dev)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
    if (e != cudaSuccess) return e;
    mark_setup(configured, dev);
  }
  kernel<<<sms, Shape::kThreads, Shape::kSmem, stream>>>(a, workspace, arrived);
  return cudaGetLastError();
}

template <int DP, int NG>
cudaError_t launch_dims(const AttendArgs& a, void* workspace, uint32_t* arrived, int sms, cudaStream_t stream) {
  return a.dim == DP ? launch_typed<DP, NG, false>(a, workspace, arrived, sms, stream)
                     : launch_typed<DP, NG, true>(a, workspace, arrived, sms, stream);
}

template <int DP, int NG>
size_t workspace_of(int sms) {
  using Shape = FourShape<DP, NG>;
  return StepWorkspace<Shape::kHeads, Shape::kAcc>::bytes(static_cast<int64_t>(sms) * Shape::kWarps);
}

}  // namespace

size_t attend_step_four_workspace(const AttendArgs& a, int tiles, int sms) {
  if (a.dim <= 64) return tiles == 1 ? workspace_of<64, 1>(sms) : workspace_of<64, 2>(sms);
  if (a.dim <= 128) return tiles == 1 ? workspace_of<128, 1>(sms) : workspace_of<128, 2>(sms);
  return workspace_of<256, 1>(sms);
}

cudaError_t launch_attend_step_four(const AttendArgs& a, int tiles, void* workspace, uint32_t* arrived, int sms,
                                    cudaStream_t stream) {
  if (a.dim <= 64)
    return tiles == 1 ? launch_dims<64, 1>(a, workspace, arrived, sms, stream)
                      : launch_dims<64, 2>(a, workspace, arrived, sms, stream);
  if (a.dim <= 128)
    return tiles == 1 ? launch_dims<128, 1>(a, workspace, arrived, sms, stream)
                      : launch_dims<128, 2>(a, workspace, arrived, sms, stream);
  return launch_dims<256, 1>(a, workspace, arrived, sms, stream);
}

}  // namespace kvca

// Attention of one new token per sequence over a paged cache.
//
// Bound by HBM: every visible K and V row is read once, for 4 operations per
// element and query head.  Work is cut into tiles of 16 visible tokens of one
// (sequence, head group), numbered sequence by sequence; the tiles of all
// sequences are dealt out evenly, a contiguous run to each warp of one CTA per
// SM, so ragged batches and single long sequences load every SM alike.  Warps
// side by side take the same run for different heads, whose rows lie side by
// side in memory (256 windowed sequences with 8 e4m3 K/V heads: a run per warp
// and head takes 18 % more).  A warp streams its run through a ring of its own in
// shared memory (cp.async, no barrier with other warps) and keeps the running
// maximum and sum of the softmax and the output in registers.  A (sequence,
// head group) that lies inside one run is written directly; one that several
// runs share leaves a partial result per CTA; the CTA that leaves the last of a
// segment's results joins them, in run order (a second kernel for that cost 6
// us of 94 with 96 ragged sequences, and a launch).
//
// 96 ragged sequences of 37-8,191 tokens, 8 K/V heads of 128 in fp16 (495 MB):
// 95 us, 5.2 TB/s, 79 % of the measured copy bandwidth; 256 sequences with a
// window of 4,096 tokens in e4m3 (1.34 GB): 260-277 us, 4.8-5.1 TB/s, issue
// slots 65 % (as many instructions per token as fp16, and the conversions).
//
// Both products run transposed on m16n8k16: S^T = K Q^T has the 16 tokens as
// rows and up to 8 query heads that share the K/V head as columns, O^T = V^T
// P^T the head dim as rows, so that 8 heads cost no padding and the transposed
// probabilities move between the two with one movmatrix per 8 x 8.

#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "attend_common.cuh"
#include "kvca_host.cuh"

namespace kvca {
namespace {

constexpr int kTile = 16;         // tokens per tile: the rows of one m16n8k16
constexpr int kScanGroups = 1024; // sequences (or runs of them) in the shared tile counts
// What a segment costs a warp beside its tiles (queries, the output), in
// tiles.  It counts when the tiles are dealt out, as tiles before the first.
constexpr int kSegmentCost = 2;

// Warps of a CTA, which share 192 KiB of rings: stages of 32 rows, three of
// them or more in a ring, two at 256-byte rows (96 ragged sequences: 8 warps
// with three stages 94.5 us, 12 with two 92).
__host__ __device__ constexpr int step_warps(int row_bytes, int head_tiles) {
  return row_bytes > 256 ? 4 : row_bytes > 128 ? 12 : head_tiles > 1 && row_bytes > 64 ? 8 : 16;
}

// DP: head dim padded to 64, 128 or 256; NG: tiles of 8 query heads.
template <typename Cache, int DP, int NG>
struct StepShape {
  static constexpr int kRowBytes = DP * Cache::kBytes;
  static constexpr int kChunks = kRowBytes / 16;       // 16-byte chunks of a row
  static constexpr int kStageBytes = 2 * kTile * kRowBytes;
  static constexpr int kWarps = step_warps(kRowBytes, NG);
  static constexpr int kThreads = 32 * kWarps;
  // 192 KiB of rings per SM
  static constexpr int kRingBytes = 192 * 1024 / kWarps;
  static constexpr int kStages = kRingBytes / kStageBytes < 8 ? kRingBytes / kStageBytes : 8;
  static constexpr int kHeads = 8 * NG;
  static constexpr int kAcc = DP * kHeads;  // floats of a partial output
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  // Weights of the values and their sum are held times 2^kShift of the running
  // maximum's own: fp16 ones then keep 11 bits to 2^-29 of the largest and some
  // to 2^-39 (to 2^-14 and 2^-24 without, where 2,000 tokens at 2^-26 of a
  // first one were lost); the largest, 2^15, is within fp16's range.  bf16 ones
  // are held 2^16 times smaller, so that sums of 65,536 of the type's largest
  // values do not overflow.
  static constexpr float kShift = Cache::kBf16 ? -16.f : 15.f;
  // An infinite value at a token that the query sees is the result, however
  // small its weight: a visible token's weight is never 0 (0 x inf is NaN),
  // nor is that of a partial result.  What the least ones add is below a value's
  // 2^-39 (fp16) or 2^-110 (bf16).  e4m3 has no infinities.
  static constexpr bool kInfinities = Cache::kBytes == 2;
  static constexpr float kLeast = Cache::kBf16 ? 0x1p-126f : 0x1p-24f;
};

// Shared memory address of 16-byte chunk c of row r: chunks are permuted
// within 128 bytes so that the 8 rows an ldmatrix reads fall on distinct banks.
template <int kChunks>
__device__ __forceinline__ uint32_t chunk_offset(int r, int c) {
  if constexpr (kChunks >= 8)
    return static_cast<uint32_t>((r * kChunks + (c ^ (r & 7))) * 16);
  else
    return static_cast<uint32_t>((r * kChunks + (c ^ ((r >> 1) & 3))) * 16);
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// How a call's work lies on the warps: `span` warps side by side share a run,
// each for a head group of its own.
struct StepLayout {
  int parts;   // head groups of a sequence: K/V heads x tiles of query heads
  int span;    // of them in a run
  int chunks;  // runs' worth of them, one after the other in the numbering
  int groups;  // runs of a CTA at a time

  __host__ __device__ StepLayout(int kv_heads, int group, int heads, int warps) {
    parts = kv_heads * ((group + heads - 1) / heads);
    int a = parts, b = warps;
    while (b != 0) {
      const int r = a % b;
      a = b;
      b = r;
    }
    span = a;  // the greatest common divisor: no warp is left out
    chunks = parts / span;
    groups = warps / span;
  }
  // The warp (of the grid) that has run r for the j-th of a run's heads.
  __device__ __forceinline__ int warp_of(int r, int j, int warps) const {
    const int cta = r / groups;
    return cta * warps + (r - cta * groups) * span + j;
  }
};

// A segment that several runs share leaves one result per CTA (its first run's
// place) and one from the run that ends it, unless that is a CTA's first.
__device__ __forceinline__ int result_count(int first_run, int last_run, int groups) {
  const int cta = first_run / groups, last_cta = last_run / groups;
  return last_cta - cta + 1 + (cta == last_cta || last_run != last_cta * groups ? 1 : 0);
}

__device__ __forceinline__ int result_run(int k, int first_run, int last_run, int groups) {
  const int cta = first_run / groups, last_cta = last_run / groups;
  return k == 0 ? first_run : k <= last_cta - cta ? (cta + k) * groups : last_run;
}

// The workspace: two partial results per warp, slot 0 for a segment that an
// earlier run began, slot 1 for one that this warp's run began.
template <int kHeads, int kAcc>
struct StepWorkspace {
  float* ml;   // [warp][slot][2][heads]: maxima, then sums
  float* acc;  // [warp][slot][dim][heads]

  static __host__ __device__ size_t bytes(int64_t warps) {
    return static_cast<size_t>(warps) * 2 * (2 * kHeads + kAcc) * sizeof(float);
  }
  __host__ __device__ StepWorkspace(void* base, int64_t warps) {
    acc = static_cast<float*>(base);
    ml = acc + warps * 2 * kAcc;
  }
  __device__ __forceinline__ float* ml_of(int64_t warp, int slot) const { return ml + (warp * 2 + slot) * 2 * kHeads; }
  __device__ __forceinline__ float* acc_of(int64_t warp, int slot) const { return acc + (warp * 2 + slot) * kAcc; }
};

// A segment to join.
struct StepJoin {
  int segment;
  int first_run, last_run;
};

__device__ __forceinline__ int64_t run_begin(int64_t tiles, int64_t runs, int64_t r) {
  return tiles * r / runs;  // below 2^31 tiles x a few thousand runs
}

__device__ __forceinline__ int run_of(int64_t tiles, int64_t runs, int64_t t) {
  return static_cast<int>((runs * (t + 1) - 1) / tiles);
}

// A position in the numbering of tiles: sequence, chunk of head groups, tile.
struct Cursor {
  int seq;
  int chunk;
  int tile;
  int tiles;  // of this sequence's visible tokens
  int left;   // of the run, this tile included; none when <= 0
  Visible vis;

  __device__ __forceinline__ void load(const AttendArgs& a) {
    vis = visible_tokens(max(sequence_length(a, seq), 0), a.window, a.sinks);
    tiles = (vis.count + kTile - 1) / kTile;
  }
  __device__ __forceinline__ bool ends() const { return tile + 1 == tiles; }
  __device__ __forceinline__ bool last() const { return left <= (ends() ? 1 + kSegmentCost : 1); }
  // To the next tile; only when this one is not the last.
  __device__ __forceinline__ void advance(const AttendArgs& a, int chunks) {
    --left;
    if (++tile < tiles) return;
    tile = 0;
    left -= kSegmentCost;
    if (++chunk < chunks) return;
    chunk = 0;
    do {
      if (++seq >= a.num_seqs) {  // not while the lengths stay as they were counted
        left = 0;
        --seq;
        return;
      }
      load(a);
    } while (tiles == 0);
  }
};

// The shares a sequence's segments take of the numbering.
__device__ __forceinline__ int64_t sequence_share(int tiles, int chunks) {
  return tiles > 0 ? static_cast<int64_t>(tiles + kSegmentCost) * chunks : 0;
}

template <typename Cache, int DP, int NG>
__global__ void __launch_bounds__(StepShape<Cache, DP, NG>::kThreads, 1)
    attend_step_kernel(const __grid_constant__ AttendArgs a, void* workspace, uint32_t* arrived) {
  using Shape = StepShape<Cache, DP, NG>;
  constexpr bool kBf16 = Cache::kBf16;
  constexpr bool kE4m3 = Cache::kBytes == 1;
  constexpr bool kTwoTerms = !kE4m3;  // of a probability
  constexpr int kChunks = Shape::kChunks;
  constexpr int kStages = Shape::kStages;
  constexpr int kHeads = Shape::kHeads;
  constexpr int kSteps = DP / 16;
  constexpr int kWarps = Shape::kWarps;
  extern __shared__ __align__(128) unsigned char rings[];
  __shared__ int64_t prefix[kScanGroups + 1];
  __shared__ int64_t scan[33];
  __shared__ int held[kWarps];
  __shared__ bool held_begins[kWarps];
  __shared__ __align__(16) float held_ml[kWarps][2 * kHeads];
  __shared__ StepJoin joins[2 * kWarps];
  __shared__ int join_count;

  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const int head_groups = (a.group + kHeads - 1) / kHeads;
  const StepLayout layout(a.kv_heads, a.group, kHeads, kWarps);
  const int chunks = layout.chunks, span = layout.span;
  StepWorkspace<kHeads, Shape::kAcc> ws(workspace, static_cast<int64_t>(gridDim.x) * kWarps);

  // Tile counts of the sequences, or of runs of `per` of them.
  const int per = (a.num_seqs + kScanGroups - 1) / kScanGroups;
  const int groups = (a.num_seqs + per - 1) / per;
  int64_t run = 0;
  for (int base = 0; base < groups; base += Shape::kThreads) {
    const int g = base + threadIdx.x;
    int64_t n = 0;
    if (g < groups) {
      const int end = min(a.num_seqs, (g + 1) * per);
      for (int seq = g * per; seq < end; ++seq) {
        Cursor c;
        c.seq = seq;
        c.load(a);
        n += sequence_share(c.tiles, chunks);
      }
    }
    int64_t total;
    const int64_t before = block_excl_scan(n, &total, scan);
    if (g < groups) prefix[g] = run + before;
    run += total;
  }
  const int64_t tiles = run;
  const int64_t all = static_cast<int64_t>(gridDim.x) * layout.groups;
  const int64_t runs = min(all, tiles);
  if (threadIdx.x == 0) join_count = 0;
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
  int held_segment = -1;
  bool held_starts = false;
  StepJoin held_runs{-1, 0, 0};
  // what this warp leaves, and the runs of its segment: of a segment that an
  // earlier run began (slot 0), and of one that this run began (slot 1)
  StepJoin leaves[2] = {{-1, 0, 0}, {-1, 0, 0}};

  float acc[NG][kSteps][4];
  float m[NG][2], l[NG][2];  // of the heads 2 * (lane % 4), + 1 of each tile of 8
  // Weight of a token of score s, and of sums whose maximum is `behind` (<= 0) the whole's.
  auto token_weight = [](float s, float base) {
    const float w = exp2_approx(s - (base - Shape::kShift));
    if constexpr (!Shape::kInfinities) return w;
    return s == -INFINITY ? 0.f : max_nan(w, Shape::kLeast);
  };
  auto partial_weight = [](float behind) {
    const float w = exp2_approx(behind);
    if constexpr (!Shape::kInfinities) return w;
    return max_nan(w, 0x1p-126f);
  };

  if (my_run < runs) {
    const int64_t begin = run_begin(tiles, runs, my_run), finish = run_begin(tiles, runs, my_run + 1);

    Cursor at;  // the tile computed next
    {
      int lo = 0, hi = groups;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= begin) lo = mid; else hi = mid;
      }
      int64_t rest = begin - prefix[lo];
      at.seq = lo * per;
      at.load(a);
      while (rest >= sequence_share(at.tiles, chunks) && at.seq + 1 < a.num_seqs) {
        rest -= sequence_share(at.tiles, chunks);
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

    const uint32_t ring = smem_addr(rings) + warp * (kStages * Shape::kStageBytes);
    const int row_chunks = a.dim * Cache::kBytes / 16;
    if (row_chunks < kChunks) {  // the padded dims stay zero: no copy writes them
      for (int i = lane; i < kStages * Shape::kStageBytes / 16; i += 32)
        *reinterpret_cast<uint4*>(rings + warp * (kStages * Shape::kStageBytes) + i * 16) = make_uint4(0, 0, 0, 0);
      __syncwarp();
    }

    // Lane i holds K's row of token i % 16, lane 16 + i V's.  The page of the
    // next tile is read one iteration before its rows.
    const int token = lane & 15;
    const bool value_side = lane >= 16;
    const char* const plane = value_side ? a.value : a.key;
    const int64_t block_stride = value_side ? a.value_block : a.key_block;
    const int64_t token_stride = value_side ? a.value_token : a.key_token;
    const int64_t head_stride = value_side ? a.value_head : a.key_head;
    constexpr int64_t kHidden = -1ll << 62;  // no token of this tile
    Cursor ahead = at;
    bool more = at.left > 0;  // tiles to issue
    int64_t page = kHidden;
    int offset = 0, page_head = 0;
    bool in_page = false;  // all 16 tokens of the tile, one after the other in one page
    auto look_up = [&]() {
      const int v0 = ahead.tile * kTile, v = v0 + token;
      const int first = ahead.vis.position(v0);
      const int first_offset = a.block_shift >= 0 ? first & (a.block_size - 1) : first % a.block_size;
      in_page = v0 + kTile <= ahead.vis.count && first_offset + kTile <= a.block_size &&
                ahead.vis.position(v0 + kTile - 1) == first + kTile - 1;
      page = kHidden;
      const int part = ahead.chunk * span + lane_of_heads;
      page_head = part / head_groups;
      if (v < ahead.vis.count) {
        const int pos = ahead.vis.position(v);
        const int block = a.block_shift >= 0 ? pos >> a.block_shift : pos / a.block_size;
        offset = pos - block * a.block_size;
        page = __ldg(a.tables + static_cast<int64_t>(ahead.seq) * a.table_stride + block);
      }
      if (ahead.tile == 0) {
        // the segment's queries, on their way to the first-level cache
        const int h = (part - page_head * head_groups) * kHeads + (lane >> 1);
        if (lane < 2 * kHeads && h < a.group)
          asm volatile("prefetch.global.L1 [%0];" ::"l"(
              static_cast<const uint16_t*>(a.query) + static_cast<int64_t>(ahead.seq) * a.query_row +
              static_cast<int64_t>(page_head * a.group + h) * a.query_head + (lane & 1) * min(64, a.dim - 1)));
      }
    };
    int stage_of = 0;  // ring entry of the next tile issued
    auto issue = [&]() {
      if (more) {
        const bool good = page >= 0 && page < a.num_blocks;
        if (!good && page != kHidden) report(a.status, KVCA_ERR_BAD_INDEX, page);  // its rows read as zeros
        const unsigned long long row = reinterpret_cast<unsigned long long>(
            plane + (good ? page : 0) * block_stride + offset * token_stride + page_head * head_stride);
        const unsigned seen = __ballot_sync(0xffffffffu, good);
        const uint32_t stage = ring + stage_of * Shape::kStageBytes;
        constexpr int kPerInstr = 32 / kChunks > 0 ? 32 / kChunks : 1;
        const int r0 = kChunks >= 32 ? 0 : lane / kChunks;
        const int c = lane % kChunks;
        if (in_page && seen == 0xffffffffu) {
          // one page: rows at a fixed distance
#pragma unroll
          for (int side = 0; side < 2; ++side) {
            const int64_t stride = side == 0 ? a.key_token : a.value_token;
            const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, row, side * kTile)) + r0 * stride + c * 16;
            if (c < row_chunks) {
#pragma unroll
              for (int r = 0; r < kTile; r += kPerInstr) {
                cp_async16(stage + chunk_offset<kChunks>(side * kTile + r + r0, c), src);
                src += kPerInstr * stride;
              }
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 2 * kTile; r += kPerInstr) {
            const char* src = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, row, r + r0)) + c * 16;
            if (c < row_chunks) cp_async16(stage + chunk_offset<kChunks>(r + r0, c), src, (seen >> (r + r0)) & 1u);
          }
        }
        if (++stage_of == kStages) stage_of = 0;
        more = !ahead.last();
        if (more) {
          ahead.advance(a, chunks);
          more = ahead.left > 0;
          look_up();
        }
      }
      cp_async_commit();
    };
    if (more) {
      look_up();
#pragma unroll 1
      for (int s = 0; s < kStages - 1; ++s) issue();
    }

    uint32_t q[NG][kSteps][2];
    float unit[NG][2];  // score factor of the heads 2 * (lane % 4), + 1
    bool starts = at.tile == 0;
    bool fresh = true;
    int stage_at = 0;  // ring entry of the tile computed
#pragma unroll 1
    for (bool go = at.left > 0; go;) {
      if (fresh) {
        // the segment's queries as the B operand: column (head) lane / 4
        const int part = at.chunk * span + lane_of_heads;
        const int kv_head = part / head_groups;
        const int first = (part - kv_head * head_groups) * kHeads;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const int h = first + n * 8 + (lane >> 2);
          const bool live = h < a.group;
          const uint16_t* row = static_cast<const uint16_t*>(a.query) + static_cast<int64_t>(at.seq) * a.query_row +
                                static_cast<int64_t>(kv_head * a.group + (live ? h : 0)) * a.query_head;
          if constexpr (!kE4m3) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int d = k * 16 + j * 8 + 2 * (lane & 3);
                q[n][k][j] = live && d < a.dim ? *reinterpret_cast<const uint32_t*>(row + d) : 0u;
              }
            unit[n][0] = unit[n][1] = a.scale_log2;
          } else {
            // fp16 products, each row times a power of two (power_up)
            float big = 0.f;
            const bool bf16 = a.query_type == KVCA_TYPE_BF16;
            uint2 raw[kSteps];
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              const int d = k * 16 + 4 * (lane & 3);
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
#pragma unroll
          for (int t = 0; t < kSteps; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][t][j] = 0.f;
          m[n][0] = m[n][1] = -INFINITY;
          l[n][0] = l[n][1] = 0.f;
        }
        fresh = false;
      }

      cp_async_wait<kStages - 2>();
      __syncwarp();
      const uint32_t keys = ring + stage_at * Shape::kStageBytes;
      if (++stage_at == kStages) stage_at = 0;
      issue();  // into the stage that the tile before this one left

      // S^T = K Q^T, even and odd steps apart for two shorter chains
      float s[NG][2][4];
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][0][j] = s[n][1][j] = 0.f;
#pragma unroll
      for (int k = 0; k < kSteps; k += kE4m3 ? 2 : 1) {
        uint32_t f[4];
        if constexpr (!kE4m3) {
          ldmatrix4(f, keys + chunk_offset<kChunks>(lane & 15, 2 * k + (lane >> 4)));
#pragma unroll
          for (int n = 0; n < NG; ++n) mma16816<kBf16>(s[n][k & 1], f, q[n][k][0], q[n][k][1]);
        } else {
          // a chunk holds the 16 dims of one step; a thread's four bytes of
          // it are the columns 2t, 2t + 1 and 2t + 8, 2t + 9 of the operand,
          // as the query's are above
          ldmatrix4(f, keys + chunk_offset<kChunks>(lane & 15, k + (lane >> 4)));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t w[4] = {e4m3_to_f16x2(f[2 * j]), e4m3_to_f16x2(f[2 * j + 1]),
                                   e4m3_to_f16x2(f[2 * j] >> 16), e4m3_to_f16x2(f[2 * j + 1] >> 16)};
#pragma unroll
            for (int n = 0; n < NG; ++n) mma16816<false>(s[n][j], w, q[n][k + j][0], q[n][k + j][1]);
          }
        }
      }

      // softmax over the tile's tokens (rows lane / 4 and + 8)
      const int left = at.vis.count - at.tile * kTile;
      const bool row0 = (lane >> 2) < left, row1 = (lane >> 2) + 8 < left;
      uint32_t p[NG][2], p_low[NG][2];
      bool grew = false;
      float decay[NG][2];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[j] = (j < 2 ? row0 : row1) ? (s[n][0][j] + s[n][1][j]) * unit[n][j & 1] : -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = fmaxf(x[j], x[j + 2]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float next = fmaxf(m[n][j], top);
          const float base = next == -INFINITY ? 0.f : next;
          decay[n][j] = partial_weight(m[n][j] - base);
          grew |= next != m[n][j];
          m[n][j] = next;
          x[j] = token_weight(x[j], base);
          x[j + 2] = token_weight(x[j + 2], base);
          l[n][j] = l[n][j] * decay[n][j] + (x[j] + x[j + 2]);
        }
        if constexpr (kTwoTerms) {
          // 16 bits would leave 8 (bf16) or 11 (fp16) of a probability: the
          // remainder goes in as a second product (the tensor cores idle here
          // anyway), to 2^-15 (2^-21) in all.  The first term is cut off, so that
          // the remainder is not negative, and like it never 0 (inf - inf, 0 x
          // inf).
          const uint32_t top = cut2<kBf16>(x[0], x[1]), bottom = cut2<kBf16>(x[2], x[3]);
          const float2 t = unpack2<kBf16>(top), b = unpack2<kBf16>(bottom);
          p[n][0] = transpose8x8(top);
          p[n][1] = transpose8x8(bottom);
          p_low[n][0] = transpose8x8(pack2<kBf16>(max_nan(x[0] - t.x, Shape::kLeast), max_nan(x[1] - t.y, Shape::kLeast)));
          p_low[n][1] = transpose8x8(pack2<kBf16>(max_nan(x[2] - b.x, Shape::kLeast), max_nan(x[3] - b.y, Shape::kLeast)));
        } else {
          // one term, to 2^-11: an e4m3 cache is bound by instructions, and its
          // values have 4 bits
          p[n][0] = transpose8x8(pack2<false>(x[0], x[1]));
          p[n][1] = transpose8x8(pack2<false>(x[2], x[3]));
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
          for (int t = 0; t < kSteps; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[n][t][j] *= decay[n][j & 1];
      }

      // O^T += V^T P^T
      const uint32_t values = keys + kTile * Shape::kRowBytes;
#pragma unroll
      for (int t = 0; t < kSteps; t += kE4m3 ? 2 : 1) {
        uint32_t f[4];
        if constexpr (!kE4m3) {
          // 8 x 8 pieces: dims 0-7 and 8-15 of tokens 0-7, then of 8-15
          ldmatrix4_trans(f, values + chunk_offset<kChunks>((lane & 7) + (lane >> 4) * 8, 2 * t + ((lane >> 3) & 1)));
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            mma16816<kBf16>(acc[n][t], f, p[n][0], p[n][1]);
            if constexpr (kTwoTerms) mma16816<kBf16>(acc[n][t], f, p_low[n][0], p_low[n][1]);
          }
        } else {
          // pieces: chunk t of tokens 0-7 and 8-15, then chunk t + 1; a
          // transposed 16-bit element is two dims of one token, so row g of
          // the operand is dim 2 g of the chunk and row g + 8 dim 2 g + 1
          ldmatrix4_trans(f, values + chunk_offset<kChunks>(lane & 15, t + (lane >> 4)));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t v = __byte_perm(f[2 * j + half], 0, 0x3120);
              w[2 * half] = e4m3_to_f16x2(v);
              w[2 * half + 1] = e4m3_to_f16x2(v >> 16);
            }
#pragma unroll
            for (int n = 0; n < NG; ++n) mma16816<false>(acc[n][t + j], w, p[n][0], p[n][1]);
          }
        }
      }

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
      const int segment = at.seq * layout.parts + at.chunk * span + lane_of_heads;
      const int64_t here = finish - at.left - at.tile;  // the segment's first tile in the numbering
      const int this_run = static_cast<int>(my_run);
      if (ends && starts) {
        const int part = at.chunk * span + lane_of_heads;
        const int kv_head = part / head_groups;
        const int first = (part - kv_head * head_groups) * kHeads;
        const int64_t row = (static_cast<int64_t>(at.seq) * a.kv_heads + kv_head) * a.group;
        const bool bf16 = a.query_type == KVCA_TYPE_BF16;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const float r0 = a.value_scale / l[n][0], r1 = a.value_scale / l[n][1];
          const int h = first + n * 8 + (lane >> 2);
          uint16_t* const out = static_cast<uint16_t*>(a.out) + (row + h) * a.dim;
#pragma unroll
          for (int t = 0; t < kSteps; ++t) {
            uint32_t top, bottom;
            if (bf16) {
              top = pack2<true>(acc[n][t][0] * r0, acc[n][t][1] * r1);
              bottom = pack2<true>(acc[n][t][2] * r0, acc[n][t][3] * r1);
            } else {
              top = pack2<false>(acc[n][t][0] * r0, acc[n][t][1] * r1);
              bottom = pack2<false>(acc[n][t][2] * r0, acc[n][t][3] * r1);
            }
            top = transpose8x8(top);  // now head lane / 4, rows 2 * (lane % 4), + 1
            bottom = transpose8x8(bottom);
            if (h >= a.group) continue;
            if constexpr (!kE4m3) {
              const int d = t * 16 + 2 * (lane & 3);
              if (d < a.dim) *reinterpret_cast<uint32_t*>(out + d) = top;
              if (d + 8 < a.dim) *reinterpret_cast<uint32_t*>(out + d + 8) = bottom;
            } else {
              const int d = t * 16 + 4 * (lane & 3);
              if (d < a.dim)
                *reinterpret_cast<uint2*>(out + d) =
                    make_uint2(__byte_perm(top, bottom, 0x5410), __byte_perm(top, bottom, 0x7632));
            }
          }
          if (a.lse != nullptr && lane < 4) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const int hh = first + n * 8 + 2 * lane + j;
              if (hh < a.group) a.lse[row + hh] = (m[n][j] - Shape::kShift) * kLn2 + logf(l[n][j]);
            }
          }
        }
      } else if (ends) {
        // the end of a segment that an earlier run began
        leaves[0] = StepJoin{segment, run_of(tiles, runs, here), this_run};
        float* const ml = ws.ml_of(own, 0);
        float* const part = ws.acc_of(own, 0);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
          const int h = n * 8 + 2 * (lane & 3);
          if (lane < 4) {
            *reinterpret_cast<float2*>(ml + h) = make_float2(m[n][0], m[n][1]);
            *reinterpret_cast<float2*>(ml + kHeads + h) = make_float2(l[n][0], l[n][1]);
          }
#pragma unroll
          for (int t = 0; t < kSteps; ++t) {
            const int d0 = kE4m3 ? t * 16 + 2 * (lane >> 2) : t * 16 + (lane >> 2);
            const int d1 = kE4m3 ? d0 + 1 : d0 + 8;
            *reinterpret_cast<float2*>(part + d0 * kHeads + h) = make_float2(acc[n][t][0], acc[n][t][1]);
            *reinterpret_cast<float2*>(part + d1 * kHeads + h) = make_float2(acc[n][t][2], acc[n][t][3]);
          }
        }
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
    cp_async_wait<0>();
  }

  // Partial results that the CTA's warps still hold, joined where runs that
  // follow each other hold the same segment: the rings are free now.
  if (lane == 0) {
    held[warp] = held_segment;
    held_begins[warp] = held_starts;
  }
  __syncthreads();
  float* const parked = reinterpret_cast<float*>(rings);
  if (held_segment >= 0) {
    float* const mine = parked + warp * Shape::kAcc;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int h = n * 8 + 2 * (lane & 3);
      if (lane < 4) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          held_ml[warp][h + j] = m[n][j];
          held_ml[warp][kHeads + h + j] = l[n][j];
        }
      }
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        const int d0 = kE4m3 ? t * 16 + 2 * (lane >> 2) : t * 16 + (lane >> 2);
        const int d1 = kE4m3 ? d0 + 1 : d0 + 8;
        *reinterpret_cast<float2*>(mine + d0 * kHeads + h) = make_float2(acc[n][t][0], acc[n][t][1]);
        *reinterpret_cast<float2*>(mine + d1 * kHeads + h) = make_float2(acc[n][t][2], acc[n][t][3]);
      }
    }
    const bool leads = warp < span || held[warp - span] != held_segment;
    if (leads && held_starts) leaves[1] = held_runs;
    if (leads && !held_starts) leaves[0] = held_runs;
  }
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    const int segment = held[w];
    if (segment < 0 || (w >= span && held[w - span] == segment)) continue;
    int end = w + span;
    while (end < kWarps && held[end] == segment) end += span;
    // a run whose only tiles continue a segment leads with slot 0, one that
    // began it with slot 1
    const int64_t leader = static_cast<int64_t>(blockIdx.x) * kWarps + w;
    const bool begins = held_begins[w];
    float* const out = ws.acc_of(leader, begins ? 1 : 0);
    float* const ml = ws.ml_of(leader, begins ? 1 : 0);
    for (int i = threadIdx.x; i < Shape::kAcc; i += Shape::kThreads) {
      const int h = i % kHeads;
      float top = -INFINITY;
      for (int k = w; k < end; k += span) top = fmaxf(top, held_ml[k][h]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, total = 0.f;
      for (int k = w; k < end; k += span) {
        const float weight = partial_weight(held_ml[k][h] - base);
        sum += weight * parked[k * Shape::kAcc + i];
        total += weight * held_ml[k][kHeads + h];
      }
      out[i] = sum;
      if (i < kHeads) {
        ml[i] = top;
        ml[kHeads + i] = total;
      }
    }
  }

  // Whoever leaves the last result of a segment joins them: a warp alone while
  // they are few, the CTA when they are many (a long sequence over all SMs).
  // The count of a segment's results is kept at its first run's warp, and is
  // zero again then.
  constexpr int kVecs = Shape::kAcc / 128;  // float4 per lane
  constexpr int kWarpResults = 8;
  const int h4 = lane * 4 % kHeads;         // a lane's four heads
  float4 top, total, sum[kVecs];
  auto fold = [&](float& old, float next, float& keep, float& weight) {
    const float best = fmaxf(old, next), base = best == -INFINITY ? 0.f : best;
    keep = partial_weight(old - base);
    weight = partial_weight(next - base);
    old = best;
  };
  const int groups_of = layout.groups;
  auto gather = [&](const StepJoin& join, int results, int first_result, int stride) {
    top = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    total = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int v = 0; v < kVecs; ++v) sum[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k = first_result; k < results; k += stride) {
      const int r = result_run(k, join.first_run, join.last_run, groups_of);
      const int w = layout.warp_of(r, join.segment % layout.parts % span, kWarps);
      const int slot = k == 0 ? 1 : 0;
      const float4 mk = __ldcg(reinterpret_cast<const float4*>(ws.ml_of(w, slot) + h4));
      const float4 lk = __ldcg(reinterpret_cast<const float4*>(ws.ml_of(w, slot) + kHeads + h4));
      const float4* const from = reinterpret_cast<const float4*>(ws.acc_of(w, slot)) + lane;
      float4 o[kVecs];
#pragma unroll
      for (int v = 0; v < kVecs; ++v) o[v] = __ldcg(from + 32 * v);
      float4 keep, weight;
      fold(top.x, mk.x, keep.x, weight.x);
      fold(top.y, mk.y, keep.y, weight.y);
      fold(top.z, mk.z, keep.z, weight.z);
      fold(top.w, mk.w, keep.w, weight.w);
      total.x = total.x * keep.x + lk.x * weight.x;
      total.y = total.y * keep.y + lk.y * weight.y;
      total.z = total.z * keep.z + lk.z * weight.z;
      total.w = total.w * keep.w + lk.w * weight.w;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        sum[v].x = sum[v].x * keep.x + o[v].x * weight.x;
        sum[v].y = sum[v].y * keep.y + o[v].y * weight.y;
        sum[v].z = sum[v].z * keep.z + o[v].z * weight.z;
        sum[v].w = sum[v].w * keep.w + o[v].w * weight.w;
      }
    }
  };
  // The joined output from the results of warps [from, to) in shared memory, by
  // `threads` threads, two dims each at a time.
  auto put = [&](const StepJoin& join, int from, int to, int thread, int threads) {
    const int part = join.segment % layout.parts;
    const int kv_head = part / head_groups;
    const int first = (part - kv_head * head_groups) * kHeads;
    const int heads = min(kHeads, a.group - first);
    const int64_t row =
        (static_cast<int64_t>(join.segment / layout.parts) * a.kv_heads + kv_head) * a.group + first;
#pragma unroll 1
    for (int i = thread; i < kHeads * (DP / 2); i += threads) {
      const int h = i / (DP / 2), d = i % (DP / 2) * 2;
      if (h >= heads || d >= a.dim) continue;
      float best = -INFINITY;
#pragma unroll 1
      for (int w = from; w < to; ++w) best = fmaxf(best, held_ml[w][h]);
      const float base = best == -INFINITY ? 0.f : best;
      float x = 0.f, y = 0.f, l2 = 0.f;
#pragma unroll 1
      for (int w = from; w < to; ++w) {
        const float weight = partial_weight(held_ml[w][h] - base);
        x += weight * parked[w * Shape::kAcc + d * kHeads + h];
        y += weight * parked[w * Shape::kAcc + (d + 1) * kHeads + h];
        l2 += weight * held_ml[w][kHeads + h];
      }
      const float factor = a.value_scale / l2;
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + (row + h) * a.dim + d) =
          a.query_type == KVCA_TYPE_BF16 ? pack2<true>(x * factor, y * factor) : pack2<false>(x * factor, y * factor);
      if (a.lse != nullptr && d == 0) a.lse[row + h] = (base - Shape::kShift) * kLn2 + logf(l2);
    }
  };
  auto park = [&]() {
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
      *reinterpret_cast<float4*>(parked + warp * Shape::kAcc + (lane + 32 * v) * 4) = sum[v];
    if (lane * 4 < kHeads) {
      *reinterpret_cast<float4*>(&held_ml[warp][h4]) = top;
      *reinterpret_cast<float4*>(&held_ml[warp][kHeads + h4]) = total;
    }
  };

  __threadfence();
  __syncthreads();
  bool mine_last = false;
  if (lane < 2) {
    const StepJoin mine = lane == 0 ? leaves[0] : leaves[1];
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
    const StepJoin join = which == 0 ? leaves[0] : leaves[1];
    gather(join, result_count(join.first_run, join.last_run, layout.groups), 0, 1);
    park();
    __syncwarp();
    put(join, warp, warp + 1, lane, 32);
    __syncwarp();
  }
  __syncthreads();
  const int join_total = join_count;
#pragma unroll 1
  for (int j = 0; j < join_total; ++j) {
    const StepJoin join = joins[j];
    gather(join, result_count(join.first_run, join.last_run, layout.groups), warp, kWarps);
    park();
    __syncthreads();
    put(join, 0, kWarps, threadIdx.x, Shape::kThreads);
    __syncthreads();
  }
}

template <typename Cache, int DP, int NG>
cudaError_t launch_typed(const AttendArgs& a, void* workspace, uint32_t* arrived, int sms, cudaStream_t stream) {
  using Shape = StepShape<Cache, DP, NG>;
  auto kernel = attend_step_kernel<Cache, DP, NG>;
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

template <typename Cache, int DP>
size_t workspace_of(int tiles, int sms) {
  const int64_t warps = static_cast<int64_t>(sms) * step_warps(DP * Cache::kBytes, tiles);
  return tiles == 1 ? StepWorkspace<8, DP * 8>::bytes(warps) : StepWorkspace<16, DP * 16>::bytes(warps);
}

// Tiles of 8 query heads that share one pass over the rows: two for groups
// above 8, except at head dims above 128, whose outputs fill the registers;
// larger groups pass over the rows once per 16 (8) heads.
int head_tiles(const AttendArgs& a) { return a.group > 8 && a.dim <= 128 ? 2 : 1; }

}  // namespace

size_t attend_step_workspace(const AttendArgs& a, int sms) {
  const int n = head_tiles(a);
  const bool e4m3 = a.cache_type == KVCA_TYPE_E4M3;
  if (a.dim <= 64) return e4m3 ? workspace_of<CacheE4m3, 64>(n, sms) : workspace_of<CacheF16, 64>(n, sms);
  if (a.dim <= 128) return e4m3 ? workspace_of<CacheE4m3, 128>(n, sms) : workspace_of<CacheF16, 128>(n, sms);
  return e4m3 ? workspace_of<CacheE4m3, 256>(n, sms) : workspace_of<CacheF16, 256>(n, sms);
}

template <typename Cache>
static cudaError_t launch_cache(const AttendArgs& a, void* workspace, uint32_t* arrived, int sms,
                                cudaStream_t stream) {
  const int n = head_tiles(a);
  if (a.dim <= 64)
    return n == 1 ? launch_typed<Cache, 64, 1>(a, workspace, arrived, sms, stream)
                  : launch_typed<Cache, 64, 2>(a, workspace, arrived, sms, stream);
  if (a.dim <= 128)
    return n == 1 ? launch_typed<Cache, 128, 1>(a, workspace, arrived, sms, stream)
                  : launch_typed<Cache, 128, 2>(a, workspace, arrived, sms, stream);
  return launch_typed<Cache, 256, 1>(a, workspace, arrived, sms, stream);
}

cudaError_t launch_attend_step(const AttendArgs& a, void* workspace, uint32_t* arrived, int sms,
                               cudaStream_t stream) {
  switch (a.cache_type) {
    case KVCA_TYPE_F16: return launch_cache<CacheF16>(a, workspace, arrived, sms, stream);
    case KVCA_TYPE_BF16: return launch_cache<CacheBf16>(a, workspace, arrived, sms, stream);
    default: return launch_cache<CacheE4m3>(a, workspace, arrived, sms, stream);
  }
}

}  // namespace kvca

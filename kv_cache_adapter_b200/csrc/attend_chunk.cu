// Attention of a ragged chunk of new tokens per sequence over a paged cache.
//
// For one K/V head, the chunk's rows are its (token, query head of the group)
// pairs, token by token; a block of up to 256 of them (two tiles of 128, one
// per softmax warpgroup) shares a pass over the keys that any of them sees.
// Those keys, numbered without the gap between sinks and window, are cut into
// tiles of 128.  The tiles of all blocks and heads are dealt out evenly, a
// contiguous run to each SM, so causal triangles, ragged chunks and a few rows
// over a long cache all load the SMs alike; a block that several SMs share
// leaves one partial result per SM, which a last kernel joins.
//
// One persistent CTA per SM, 16 warps:
//   warps 0-3, 4-7  softmax of row tile 0 and 1, a thread per row: scores from
//                   tensor memory, running maximum and sum in registers,
//                   probabilities back to tensor memory, output at the end
//   warps 8-11      rows of the pages to shared memory (cp.async per 16 bytes,
//                   so that any block size and stride does; e4m3 and e2m1 are widened
//                   on the way), 128-byte swizzled as the tensor cores read them
//   warp 12         issues tcgen05.mma: S = Q K^T, O += P V
//   warp 13         finds the CTA's next segments (block, head, tiles)
//   warps 14, 15    queries to shared memory
// The two tiles alternate: while one's softmax runs, the tensor cores work on
// the other's products.  The output is rescaled only when a row's maximum grew
// by more than 2^8, so that most tiles leave it alone; a probability is then at
// most 2^8.
//
// All are bound by the latency of the chain scores, softmax, probabilities,
// product of each row tile, with two tiles to overlap; no unit is busy half of
// the time.  10,494 new tokens in 5 sequences (32 query heads of 128, bf16)
// 970-1,030 us by the GPU's clock, 0.80-0.85 PFLOP/s: tensor cores 46 % active,
// exponentials 48 %, issue slots 45 %.  16,167 tokens, window 1,024, head dim
// 64, e4m3, 275-279 us: 19, 41 and 46 %.  24 sequences with 1-8 tokens over
// 27,000 keys 51-53 us (2.1 TB/s): at most 32 rows of a block's 256.
//
// 4-bit rows are bytes to shared memory first (kAhead tiles in flight), from
// where the same four warps widen a tile once it has arrived: code times scale,
// exact in fp16.  bf16 queries are lifted to fp16 (with a power of two per row)
// by blocks of the planning kernel, to be copied like fp16 ones: converted by
// warps 14 and 15 they held up each segment (691 us for 6,465 prompt tokens, now
// 433-441; the same ones over a 16-bit cache take 370, the rest is the widening).
//
// Probabilities go into the second product as the 16-bit type that the tensor
// cores multiply values in, rounded to half a step: 2^-11 of each as fp16 (fp16
// and e4m3 caches), 2^-8 as bf16, as much as the result's own rounding and
// averaged over the keys (error against 64 bits 1.35 times that of fp32
// probabilities on the bf16 prompts, 1.33 times on the fp16 drafts).  A second
// term would double the second product, half of the tensor cores' work.  The
// sums of the softmax take the fp32 ones.
//
// The softmax reads its scores twice from tensor memory, in loops of 32
// columns: held in registers in one pass (128 of them, unrolled) the prompts
// took 2 % less and the window 11 % more.  Scores in halves of 64 keys, so that the
// next half comes while a softmax runs, cost the tensor cores more than it
// gave (19 % more time), as did an issuing warp per row tile (27 %).

#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "attend_common.cuh"
#include "kvca_host.cuh"

namespace kvca {
namespace {

constexpr int kRows = 256;      // rows of a block
constexpr int kKeys = 128;      // keys of a tile
constexpr int kThreads = 512;
constexpr int kPlanThreads = 1024;
constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 16;   // rows per block of the join
constexpr int kSlots = 4;       // segments announced ahead
constexpr int kReaders = 15;    // warps that read them
constexpr uint32_t kAhead = 2;  // tiles (of keys or values) in flight behind the one being issued
static_assert(kSlots == 4, "marks of tiles in flight hold a slot in two bits");
// What a segment costs beside its tiles, in tiles: queries, first loads, the
// output.  It counts when the tiles are dealt out, as tiles before the first.
constexpr int kSegmentCost = 3;
constexpr float kGrowth = 8.f;  // log2 of how far a maximum may lag
// Probabilities, and their sum, are held times 2^7 where they are fp16 (the
// largest, 2^15, is within its range): those of 2^-21 of the maximum keep 11
// bits, those of 2^-31 some (2^-14 and 2^-24 without: 2,000 tokens at 2^-26 of a
// first one were lost).  bf16 has fp32's exponents: there they are 2^24 times
// smaller, 2^-16 at most, so that sums of 65,536 of the type's largest values
// do not overflow.
template <typename Cache>
constexpr float kShift = Cache::kBf16 ? -24.f : 7.f;

template <int DP>
struct ChunkShape {
  static constexpr int kHalves = DP / 64;                 // 64 dims (128 bytes) each
  static constexpr int kTileBytes = kHalves * kKeys * 128;  // 128 rows of DP 16-bit values
  static constexpr int kStages = 128 * 1024 / kTileBytes;
  static constexpr int kQueries = DP == 64 ? 2 : 1;        // segments whose queries are there at once
  static constexpr int kSmem = 1024 + (2 * kQueries + kStages) * kTileBytes;
  // 4 bits: rows as they lie in memory, of kAhead + 1 sides (keys or values) per
  // loading warp: 32 rows of values, then of up to 8 bytes with their scales.
  static constexpr int kFourSide = 32 * (DP / 2 + 8);
  static constexpr int kFourBytes = 4 * (kAhead + 1) * kFourSide;
};

// ---------------------------------------------------------------------------
// Plan: the blocks of all chunks and their tiles
// ---------------------------------------------------------------------------

struct ChunkHeader {
  int64_t tiles;  // of all blocks and heads, segment costs included
  int64_t ctas;   // that get tiles
  int32_t blocks;
  int32_t unused;
};

struct ChunkBlock {
  int32_t seq;
  int32_t row;    // first (token, head) row within the chunk
  int32_t rows;
  int32_t tiles;  // per head
};

struct ChunkPiece {
  int32_t tail;  // segment (block * heads + head) whose continuation slot 0 holds, or -1
  int32_t head;  // segment whose beginning slot 1 holds, or -1
  int32_t last;  // CTA with the last tile of `head`
  int32_t unused;
};

struct ChunkWorkspace {
  ChunkHeader* header;
  float* acc;        // [cta][slot][row][dim]
  float* ml;         // [cta][slot][2][row]
  ChunkPiece* pieces;
  int64_t* first;    // tiles before each block
  ChunkBlock* blocks;

  static __host__ __device__ size_t bytes(int dp, int64_t ctas, int64_t max_blocks) {
    return 256 + static_cast<size_t>(ctas) * (sizeof(ChunkPiece) + 2 * kRows * (dp + 2) * sizeof(float)) +
           static_cast<size_t>(max_blocks + 1) * (sizeof(int64_t) + sizeof(ChunkBlock));
  }
  __host__ __device__ ChunkWorkspace(void* base, int dp, int64_t ctas, int64_t max_blocks) {
    char* p = static_cast<char*>(base);
    header = reinterpret_cast<ChunkHeader*>(p);
    acc = reinterpret_cast<float*>(p + 256);
    ml = acc + ctas * 2 * kRows * dp;
    pieces = reinterpret_cast<ChunkPiece*>(ml + ctas * 2 * 2 * kRows);
    blocks = reinterpret_cast<ChunkBlock*>(pieces + ctas);
    first = reinterpret_cast<int64_t*>(blocks + max_blocks + 1);
  }
};

// What a block's rows see.  v numbers the keys without the gap: v < sinks is
// key v, any other key v + skip.
struct BlockView {
  int seq, row, rows;
  int context;  // position of the chunk's first token
  int skip, sinks, count;

  __device__ __forceinline__ int key(int v) const { return v < sinks ? v : v + skip; }
};

__device__ __forceinline__ BlockView view_of(const AttendArgs& a, int seq, int row, int rows, int tokens, int len) {
  BlockView b;
  b.seq = seq;
  b.row = row;
  b.rows = rows;
  b.context = len - tokens;
  const int first = b.context + row / a.group, last = b.context + (row + rows - 1) / a.group;
  const int low = a.window > 0 ? max(0, first - a.window + 1) : 0;
  b.sinks = min(a.sinks, low);
  b.skip = low - b.sinks;
  b.count = last + 1 - b.skip;
  return b;
}

// Tokens of sequence `seq`'s chunk (0: none, or an idle or bad sequence).
__device__ __forceinline__ int chunk_tokens(const AttendArgs& a, const ChunkArgs& c, int seq, int* len) {
  const int64_t begin = __ldg(c.offsets + seq), end = __ldg(c.offsets + seq + 1);
  *len = sequence_length(a, seq);
  if (end == begin || *len < 0) return 0;
  if (begin < 0 || end < begin || end > c.rows) {
    report(a.status, KVCA_ERR_BAD_INDEX, end);
    return 0;
  }
  if (end - begin > *len) {
    report(a.status, KVCA_ERR_BAD_INDEX, __ldg(a.lens + seq));
    return 0;
  }
  return static_cast<int>(end - begin);
}

// The largest x of this and the threads before it; `sm` holds kPlanThreads.
__device__ __noinline__ int64_t block_incl_max(int64_t x, int64_t* sm) {
#pragma unroll 1
  for (int d = 1; d < kPlanThreads; d <<= 1) {
    sm[threadIdx.x] = x;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) >= d) x = max(x, sm[threadIdx.x - d]);
    __syncthreads();
  }
  return x;
}

// bf16 queries for the products with 4-bit keys: fp16 times a power of two per
// row (power_up), whose inverse goes into its score factor, with the sign or the
// zeros of the scores' factor; by all warps of blocks 1 and on, a row on dim / 8
// lanes.  (By the two warps that fetch queries, as with e4m3 keys, it held up every
// segment: prompts 691 us, not 433-441.)
__device__ __forceinline__ void lift_queries(const AttendArgs& a, const ChunkArgs& c) {
  const int lanes = a.dim / 8, per_warp = 32 / lanes;
  const int lane = threadIdx.x & 31, row_of = lane / lanes, chunk = lane - row_of * lanes;
  const int heads = a.kv_heads * a.group;
  const int64_t total = c.rows * heads, warps = static_cast<int64_t>(gridDim.x - 1) * (kPlanThreads / 32);
  const int64_t warp = static_cast<int64_t>(blockIdx.x - 1) * (kPlanThreads / 32) + (threadIdx.x >> 5);
  constexpr int kBatch = 4;
#pragma unroll 1
  for (int64_t first = warp * per_warp; first < total; first += warps * per_warp * kBatch) {
    uint4 x[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t at = first + b * warps * per_warp + row_of;
      x[b] = make_uint4(0, 0, 0, 0);
      if (row_of >= per_warp || at >= total) continue;
      const int64_t row = at / heads;
      x[b] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.query) + row * a.query_row +
                                                  (at - row * heads) * a.query_head) + chunk);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int64_t at = first + b * warps * per_warp + row_of;
      uint32_t word[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
      float2 f[4];
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j] = unpack2<true>(word[j]);
        big = fmaxf(big, fmaxf(fabsf(f[j].x), fabsf(f[j].y)));
      }
      float all = big;  // of the row's lanes, wherever they begin
#pragma unroll 1
      for (int o = 1; o < lanes; ++o) {
        const int from = row_of * lanes + (chunk + o >= lanes ? chunk + o - lanes : chunk + o);
        all = fmaxf(all, __shfl_sync(0xffffffffu, big, from & 31));
      }
      const int e = power_up(all);
      const float up = power_of_two(e);
      if (row_of >= per_warp || at >= total) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) word[j] = (pack2<false>(f[j].x * up, f[j].y * up) & c.query_and) ^ c.query_xor;
      reinterpret_cast<uint4*>(c.queries + at * a.dim)[chunk] = make_uint4(word[0], word[1], word[2], word[3]);
      if (chunk == 0) c.units[at] = power_of_two(-e);
    }
  }
}

__global__ void __launch_bounds__(kPlanThreads) attend_chunk_plan_kernel(const __grid_constant__ AttendArgs a,
                                                                        const __grid_constant__ ChunkArgs c,
                                                                        void* workspace, int dp, int64_t ctas) {
  if (blockIdx.x > 0) {
    lift_queries(a, c);
    return;
  }
  __shared__ int64_t scan[33];
  __shared__ int64_t highest[kPlanThreads];
  ChunkWorkspace ws(workspace, dp, ctas, c.max_blocks);
  int64_t run = 0;
  auto rows_of = [&](int seq) {
    int len;
    return seq < a.num_seqs ? chunk_tokens(a, c, seq, &len) * a.group : 0;
  };
  int next_rows = rows_of(threadIdx.x);
  // Offsets that go back somewhere: a sequence that begins before one of the
  // offsets ahead of it is bad, so that the others keep their rows to themselves.
  bool back = false;
  for (int seq = threadIdx.x; seq < a.num_seqs; seq += kPlanThreads)
    back |= __ldg(c.offsets + seq + 1) < __ldg(c.offsets + seq);
  back = __syncthreads_or(back) != 0;
  int64_t ahead = 0;  // the largest offset within the rows so far
  for (int base = 0; base < a.num_seqs; base += kPlanThreads) {
    const int seq = base + threadIdx.x;
    int rows = next_rows;
    next_rows = rows_of(seq + kPlanThreads);
    if (back) {
      const int64_t begin = seq < a.num_seqs ? __ldg(c.offsets + seq) : 0;
      const int64_t high = max(ahead, block_incl_max(begin <= c.rows ? begin : 0, highest));
      if (rows > 0 && begin < high) {
        report(a.status, KVCA_ERR_BAD_INDEX, begin);
        rows = 0;
      }
      highest[threadIdx.x] = high;
      __syncthreads();
      ahead = highest[kPlanThreads - 1];
      __syncthreads();
    }
    const int n = (rows + kRows - 1) / kRows;
    int64_t total;
    const int64_t at = run + block_excl_scan(static_cast<int64_t>(n), &total, scan);
    // (the good sequences' rows do not overlap, so their blocks fit)
    for (int b = 0; b < n && at + b < c.max_blocks; ++b)
      ws.blocks[at + b] = ChunkBlock{seq, b * kRows, min(kRows, rows - b * kRows), 0};
    run += total;
  }
  const int blocks = static_cast<int>(min(run, static_cast<int64_t>(c.max_blocks)));
  __syncthreads();
  run = 0;
  for (int base = 0; base < blocks; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int tiles = 0;
    if (i < blocks) {
      const ChunkBlock b = ws.blocks[i];
      int len;
      const int tokens = chunk_tokens(a, c, b.seq, &len);
      tiles = (view_of(a, b.seq, b.row, b.rows, tokens, len).count + kKeys - 1) / kKeys;
      ws.blocks[i].tiles = tiles;
    }
    int64_t total;
    const int64_t cost = tiles > 0 ? static_cast<int64_t>(tiles + kSegmentCost) * a.kv_heads : 0;
    const int64_t before = run + block_excl_scan(cost, &total, scan);
    if (i < blocks) ws.first[i] = before;
    run += total;
  }
  if (threadIdx.x == 0) {
    ws.first[blocks] = run;
    *ws.header = ChunkHeader{run, run < ctas ? run : ctas, blocks, 0};
  }
}

__device__ __forceinline__ int64_t share_begin(int64_t tiles, int64_t ctas, int64_t c) { return tiles * c / ctas; }

// ---------------------------------------------------------------------------
// Tensor memory
// ---------------------------------------------------------------------------

__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Arrives on `bar` when the tensor core work issued so far is done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// One 128 x n x 16 product; operands given by the low words of their
// descriptors (kOperandHigh above them).
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nmov.b64 a, {%1, %3};\nmov.b64 b, {%2, %3};\n"
               "setp.ne.u32 p, %5, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n}"
               ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(accumulate) : "memory");
}

// The same with `a` in tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\n.reg .b64 b;\nmov.b64 b, {%2, %3};\n"
               "setp.ne.u32 p, %5, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}"
               ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(accumulate) : "memory");
}

// Shared memory operands with 128-byte swizzle; 8 rows of 128 bytes are 1 KiB.
// K-major (queries, keys): groups of 8 rows 1 KiB apart.  MN-major (values:
// tokens are the reduced dim): groups of 8 tokens 1 KiB apart, 64 dims
// `leading` bytes apart.
constexpr uint32_t kOperandHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ constexpr uint32_t operand_low(uint32_t addr, uint32_t leading) {
  return (addr >> 4) | ((leading >> 4) << 16);  // shared memory ends below 2^18
}

// fp32 accumulators; both operands fp16 or both bf16; m x n.
__device__ __forceinline__ constexpr uint32_t mma_shape(bool bf16, int m, int n, bool values) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (values ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// 32 columns of this warp's 32 lanes: a thread gets its lane's.
__device__ __forceinline__ void tmem_load32(float (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(addr));
}

__device__ __forceinline__ void tmem_store32(uint32_t addr, const float (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
      "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]),
      "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]),
      "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Two floats at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\n"
      "fma.rn.f32x2 d, a, b, c;\nmov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nadd.rn.f32x2 d, a, b;\n"
      "mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Keeps the uses of loaded values behind the wait before this.
__device__ __forceinline__ void tmem_landed(float (&r)[32]) {
  asm volatile(""
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
                 "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
                 "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]),
                 "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]),
                 "+f"(r[30]), "+f"(r[31]));
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---------------------------------------------------------------------------
// The CTA's share of the tiles, segment by segment
// ---------------------------------------------------------------------------

struct Share {
  int64_t left;    // of the share from this segment's first cost or tile on
  int block, head;
  int from;        // where in the segment (costs, then tiles) the share begins
  int tile;        // first tile of the segment that is this CTA's
  int end;         // past the last one; `tile` when the share is done
  int tiles;       // of the segment
  int last_cta;    // that has the segment's last tile
  BlockView view;
  int seen_last;   // keys up to here, and
  int seen_low;    // those behind here or among the sinks, are seen by every row
  int64_t out_row;  // the chunk's first row of query and out

  // Whether a row of the block does not see a key of the tile at v0.
  __device__ __forceinline__ bool cut(int v0, int sinks) const {
    return v0 + kKeys - 1 > seen_last || (v0 + kKeys > sinks && max(v0, sinks) <= seen_low);
  }
  __device__ __forceinline__ int row_tiles() const { return view.rows > 128 ? 2 : 1; }

  // The tiles of (block, head) that are this CTA's, none perhaps.
  __device__ __forceinline__ void place() {
    const int64_t stop = min(static_cast<int64_t>(tiles) + kSegmentCost, from + left);
    tile = max(0, from - kSegmentCost);
    end = max(tile, static_cast<int>(stop) - kSegmentCost);
  }
  __device__ __forceinline__ void load(const AttendArgs& a, const ChunkArgs& c, const ChunkWorkspace& ws) {
    const ChunkBlock b = ws.blocks[block];
    out_row = __ldg(c.offsets + b.seq);
    const int tokens = static_cast<int>(__ldg(c.offsets + b.seq + 1) - out_row);
    view = view_of(a, b.seq, b.row, b.rows, tokens, sequence_length(a, b.seq));
    tiles = b.tiles;
    seen_last = view.context + view.row / a.group - view.skip;
    seen_low = a.window > 0 ? view.context + (view.row + view.rows - 1) / a.group - a.window - view.skip : -1;
  }
  // To the next segment with tiles of this CTA; without one, end == tile.
  __device__ __forceinline__ void next(const AttendArgs& a, const ChunkArgs& c, const ChunkWorkspace& ws) {
    do {
      left -= tiles + kSegmentCost - from;
      from = 0;
      if (left <= kSegmentCost) {
        end = tile;
        return;
      }
      if (++head == a.kv_heads) {
        head = 0;
        do {
          ++block;
        } while (ws.blocks[block].tiles == 0);
        load(a, c, ws);
      }
      place();
    } while (end == tile);
  }
};

// ---------------------------------------------------------------------------
// Infinite and NaN values
// ---------------------------------------------------------------------------
//
// The tensor cores multiply every value of a tile by every row's probability,
// and 0 times an infinity or a NaN is NaN.  So the values of a tile that is cut
// (a row of the block does not see one of its keys) go in with 0 in their
// places, noted per segment, and are added to the rows that see them at the
// end.  Any other tile is seen by all rows alike: there a row's output shows
// them, and what they make of it is found from the values alone.  Neither takes
// a second product; a segment without such values pays one look at the values
// of its cut tiles.

template <bool kBf16>
__device__ __forceinline__ bool is_finite16(uint32_t half) {
  constexpr uint32_t kExponent = kBf16 ? 0x7f80u : 0x7c00u;
  return (half & kExponent) != kExponent;
}

// Where 16-byte chunk `ch` of row r of a tile lies.
__device__ __forceinline__ uint32_t place(int r, int ch) {
  return static_cast<uint32_t>((ch >> 3) * (kKeys * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
}

// Zeros for the infinite and NaN values among the chunks of 32 rows of a tile
// that this lane copied (chunk lane % kRowChunks of every kPerInstr-th row);
// whether this lane found one.
template <bool kBf16, int DP>
__device__ __noinline__ bool drop_non_finite(unsigned char* tile, int first_row, int row_chunks) {
  constexpr int kRowChunks = DP / 8, kPerInstr = 32 / kRowChunks;
  const int lane = threadIdx.x & 31, chunk = lane % kRowChunks, sub = lane / kRowChunks;
  if (chunk >= row_chunks) return false;
  uint32_t sum = 0;  // of the values times 0: NaN with one that is not finite
#pragma unroll
  for (int i = 0; i < 32 / kPerInstr; ++i) {
    const uint4 x = *reinterpret_cast<const uint4*>(tile + place(first_row + i * kPerInstr + sub, chunk));
    const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (kBf16)
        asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(word[j]), "r"(0u));
      else
        asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(word[j]), "r"(0u));
    }
  }
  if ((sum & 0x7fff7fffu) == 0) return false;
#pragma unroll 1
  for (int i = 0; i < 32 / kPerInstr; ++i) {
    uint32_t* const word = reinterpret_cast<uint32_t*>(tile + place(first_row + i * kPerInstr + sub, chunk));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      word[j] &= (is_finite16<kBf16>(word[j]) ? 0xffffu : 0u) | (is_finite16<kBf16>(word[j] >> 16) ? 0xffff0000u : 0u);
  }
  return true;
}

// The same for four e4m3 values, which have NaN only (all bits but the sign).
__device__ __forceinline__ uint32_t drop_nan4(uint32_t word, uint32_t* found) {
  const uint32_t tops = ((word & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  *found |= tops;
  return word & ~((tops >> 7) * 255u);
}

// Bytes from a head's 4-bit values in a token's row to its scales.
__device__ __forceinline__ int scales_after(const AttendArgs& a, int head) {
  return (a.kv_heads - head) * (a.dim / 2) + head * (a.dim / 16);
}

// Puts the infinite and NaN values of a segment's tiles into the outputs of a
// softmax warp's rows, one per lane: `out` (16 bits, a whole segment) or `part`
// (fp32, a share of one).  Of uncut tiles (`uncut`) they take an output's
// place, of cut ones (`cut`) they are added for rows that see the key (`mine`:
// the lane has a row, and its sum is a number).  A key that is not finite
// itself has a score of NaN or an infinity: then the row is NaN already, or the
// value's weight is 0 and its product NaN.
template <typename Cache, int DP>
__device__ __noinline__ void put_non_finite(const AttendArgs& a, const Share& s, bool uncut, bool cut, bool mine,
                                            int v_last, int v_low, uint16_t* out, float* part) {
  constexpr int kOwn = DP / 32;  // a lane's values of a row
  constexpr int kBatch = 8;
  const int lane = threadIdx.x & 31;
  const bool has = lane * kOwn < a.dim;
  const bool bf16 = a.query_type == KVCA_TYPE_BF16;
  auto own_of = [&](unsigned long long row, float (&x)[kOwn]) {
    if constexpr (Cache::kBytes == 0) {
      const uint8_t* const p = reinterpret_cast<const uint8_t*>(row);
      const float unit = unpack2<false>(e4m3_to_f16x2(p[scales_after(a, s.head) + lane * kOwn / 16])).x;
#pragma unroll
      for (int e = 0; e < kOwn; e += 2) {
        const float2 f = unpack2<false>(e2m1_to_f16x2(p[(lane * kOwn + e) / 2]));
        x[e] = f.x * unit, x[e + 1] = f.y * unit;
      }
      return;
    }
    const char* const p = reinterpret_cast<const char*>(row) + lane * kOwn * Cache::kBytes;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      if constexpr (Cache::kBytes < 2)
        x[e] = unpack2<false>(e4m3_to_f16x2(reinterpret_cast<const uint8_t*>(p)[e])).x;
      else
        x[e] = unpack2<Cache::kBf16>(reinterpret_cast<const uint16_t*>(p)[e]).x;
    }
  };
  auto any_non_finite = [&](const float (&x)[kOwn]) {
    bool bad = false;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) bad |= !(fabsf(x[e]) < INFINITY);
    return __ballot_sync(0xffffffffu, has && bad);
  };
  // y into place d of this lane's row
  auto put = [&](int d, float y, bool add) {
    if (out != nullptr) {
      y *= a.value_scale;
      if (add) y += bf16 ? unpack2<true>(out[d]).x : unpack2<false>(out[d]).x;
      out[d] = static_cast<uint16_t>(bf16 ? pack2<true>(y, 0.f) : pack2<false>(y, 0.f));
    } else {
      part[d] = add ? part[d] + y : y;
    }
  };
#pragma unroll 1
  for (int pass = uncut ? 0 : 1; pass < (cut ? 2 : 1); ++pass) {
    float special[kOwn];  // their sum
#pragma unroll
    for (int e = 0; e < kOwn; ++e) special[e] = 0.f;
#pragma unroll 1
    for (int tile = s.tile; tile < s.end; ++tile) {
      if (s.cut(tile * kKeys, a.sinks) != (pass == 1)) continue;
#pragma unroll 1
      for (int v0 = tile * kKeys; v0 < min(s.view.count, (tile + 1) * kKeys); v0 += 32) {
        // a lane finds the rows of one key
        unsigned long long key_row = 0, value_row = 0;
        if (v0 + lane < s.view.count) {
          const int key = s.view.key(v0 + lane), block = key / a.block_size, offset = key - block * a.block_size;
          const int64_t page = __ldg(a.tables + static_cast<int64_t>(s.view.seq) * a.table_stride + block);
          if (page >= 0 && page < a.num_blocks) {
            key_row = reinterpret_cast<unsigned long long>(a.key + page * a.key_block + offset * a.key_token +
                                                           s.head * a.key_head);
            value_row = reinterpret_cast<unsigned long long>(a.value + page * a.value_block + offset * a.value_token +
                                                             s.head * a.value_head);
          }
        }
#pragma unroll 1
        for (int k0 = 0; k0 < 32; k0 += kBatch) {
          float x[kBatch][kOwn];
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            const unsigned long long row = __shfl_sync(0xffffffffu, value_row, k0 + k);
#pragma unroll
            for (int e = 0; e < kOwn; ++e) x[k][e] = 0.f;
            if (row != 0 && has) own_of(row, x[k]);
          }
#pragma unroll
          for (int k = 0; k < kBatch; ++k) {
            unsigned lanes = any_non_finite(x[k]);
            if (lanes == 0) continue;
            float of_key[kOwn];
#pragma unroll
            for (int e = 0; e < kOwn; ++e) of_key[e] = 0.f;
            const unsigned long long row = __shfl_sync(0xffffffffu, key_row, k0 + k);
            if (has) own_of(row, of_key);
            const bool bad_key = any_non_finite(of_key) != 0;
#pragma unroll
            for (int e = 0; e < kOwn; ++e)
              x[k][e] = fabsf(x[k][e]) < INFINITY ? 0.f : bad_key ? NAN : x[k][e];
            if (pass == 0) {
#pragma unroll
              for (int e = 0; e < kOwn; ++e) special[e] += x[k][e];
              continue;
            }
            const int v = v0 + k0 + k;
            const bool sees = mine && v <= v_last && !(v >= a.sinks && v <= v_low);
#pragma unroll 1
            for (; lanes != 0; lanes &= lanes - 1) {
              const int from = __ffs(lanes) - 1;
#pragma unroll
              for (int e = 0; e < kOwn; ++e) {
                const float y = __shfl_sync(0xffffffffu, x[k][e], from);
                if (sees && y != 0.f) put(from * kOwn + e, y, true);
              }
            }
          }
        }
      }
    }
    if (pass == 0) {
#pragma unroll 1
      for (unsigned lanes = any_non_finite(special); lanes != 0; lanes &= lanes - 1) {
        const int from = __ffs(lanes) - 1;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const float y = __shfl_sync(0xffffffffu, special[e], from);
          if (mine && y != 0.f) put(from * kOwn + e, y, false);
        }
      }
    }
  }
}

template <typename Cache, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attend_chunk_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ ChunkArgs c, void* workspace) {
  using Shape = ChunkShape<DP>;
  constexpr bool kBf16 = Cache::kBf16;
  constexpr bool kE4m3 = Cache::kBytes == 1;
  constexpr bool kFour = Cache::kBytes == 0;
  constexpr bool kNarrow = Cache::kBytes < 2;  // widened on the way
  constexpr int kStages = Shape::kStages;
  constexpr int kTileBytes = Shape::kTileBytes;
  constexpr int kQueries = Shape::kQueries;
  extern __shared__ unsigned char dynamic[];
  __shared__ uint64_t bars[2 * kStages + 2 * kSlots + 2 * kQueries + 7];
  __shared__ float row_unit[kQueries][kRows];
  __shared__ uint32_t tmem_base;
  __shared__ int start_block;
  __shared__ Share shares[kSlots];
  __shared__ int gave_up;
  __shared__ int dropped[kSlots];  // values left out of a segment's cut tiles

  const int lane = threadIdx.x & 31;
  const int warp = threadIdx.x >> 5;
  const uint32_t smem = (smem_addr(dynamic) + 1023u) & ~1023u;
  unsigned char* const smem_ptr = dynamic + (smem - smem_addr(dynamic));
  const uint32_t kv_smem = smem + 2 * kQueries * kTileBytes;
  const uint32_t full = smem_addr(bars), empty = full + 8 * kStages;
  const uint32_t q_full = empty + 8 * kStages, q_empty = q_full + 8 * kQueries;
  const uint32_t s_full = q_empty + 8 * kQueries, p_ready = s_full + 16, o_full = s_full + 32;  // per row tile
  const uint32_t drained = s_full + 48, announced = s_full + 56, released = announced + 8 * kSlots;
  const Patience patience{&gave_up, c.wait_limit};

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      barrier_init(full + 8 * i, 128);
      barrier_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kQueries; ++i) {
      barrier_init(q_full + 8 * i, 64);
      barrier_init(q_empty + 8 * i, 1 + kRows);
    }
    for (int i = 0; i < 2; ++i) {
      barrier_init(s_full + 8 * i, 1);
      barrier_init(p_ready + 8 * i, 128);
      barrier_init(o_full + 8 * i, 1);
    }
    barrier_init(drained, 1);
    for (int i = 0; i < kSlots; ++i) {
      barrier_init(announced + 8 * i, 1);
      barrier_init(released + 8 * i, kReaders);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    gave_up = 0;
    start_block = 0;
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_base))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // Padded dims stay zero: no copy writes them.
  const int row_chunks = a.dim / 8;  // 16-byte chunks of 16-bit values
  if (row_chunks < DP / 8)
    for (int i = threadIdx.x; i < (kStages + 2 * kQueries) * kTileBytes / 16; i += kThreads)
      reinterpret_cast<uint4*>(smem_ptr)[i] = make_uint4(0, 0, 0, 0);
  fence_async_proxy();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  ChunkWorkspace ws(workspace, DP, gridDim.x, c.max_blocks);
  const ChunkHeader plan = *ws.header;
  const bool working = blockIdx.x < plan.ctas;
  const int64_t begin = working ? share_begin(plan.tiles, plan.ctas, blockIdx.x) : 0;
  const int64_t share = working ? share_begin(plan.tiles, plan.ctas, blockIdx.x + 1) - begin : 0;
  __syncthreads();
  if (working)
    for (int i = threadIdx.x; i < plan.blocks; i += kThreads)
      if (ws.first[i] <= begin && begin < ws.first[i + 1]) start_block = i;
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = tmem_base;

  auto queries_barrier = [&](uint32_t bar, uint32_t n) { return bar + 8 * (n % kQueries); };
  auto queries_parity = [&](uint32_t n) { return (n / kQueries) & 1u; };
  // The segment that a warp turns to, and the end of its use of one.
  auto announced_segment = [&](uint32_t n) {
    return warp_wait(announced + 8 * (n % kSlots), (n / kSlots) & 1, patience);
  };
  auto release_segment = [&](uint32_t n) {
    __syncwarp();
    if (lane == 0) barrier_arrive(released + 8 * (n % kSlots));
  };

  if (warp >= 12) {
    // ------------------------------------------------------------------ MMA
    if (warp == 12 && working) {
      // the whole warp keeps step, one lane issues
      constexpr uint32_t kScores = mma_shape(kBf16, 128, kKeys, false);
      constexpr uint32_t kOutput = mma_shape(kBf16, 128, DP, true);
      constexpr uint32_t kHalf = kKeys * 128 >> 4;  // between 64 dims, in descriptor units
      uint32_t q_low = 0;  // this segment's queries
      const uint32_t k_low = operand_low(kv_smem, 16);
      const uint32_t v_low = operand_low(kv_smem, kKeys * 128);
      const bool issues = lane == 0;
      uint32_t stage = 0, round = 0;  // of the next ring entry
      uint32_t segment = 0;
      uint32_t p_phase = 0;  // a bit per row tile
      bool ok = true;
      auto step = [&]() {
        if (++stage == kStages) {
          stage = 0;
          round ^= 1;
        }
      };
      auto scores = [&](int q, uint32_t at) {  // S_q = Q_q K^T, K in ring entry `at`
        const uint32_t keys = k_low + at * (kTileBytes >> 4), queries = q_low + q * (kTileBytes >> 4);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = (k >> 2) * kHalf + (k & 3) * 2;
          mma_ss(tmem + q * 128, queries + off, keys + off, kOperandHigh, kScores, k > 0);
        }
        mma_commit(s_full + 8 * q);
      };
      for (;; ++segment) {
        ok = announced_segment(segment);
        if (!ok) break;
        const Share& s = shares[segment % kSlots];
        const int n = s.end - s.tile;
        const int row_tiles = s.row_tiles();
        release_segment(segment);
        if (n == 0) break;
        q_low = operand_low(smem, 16) + 2 * (segment % kQueries) * (kTileBytes >> 4);
        ok = warp_wait(queries_barrier(q_full, segment), queries_parity(segment), patience) && warp_wait(full + 8 * stage, round, patience);
        if (!ok) break;
        fence_after_sync();
        if (issues) {
#pragma unroll 1
          for (int q = 0; q < row_tiles; ++q) scores(q, stage);
          mma_commit(empty + 8 * stage);
          if (n == 1) mma_commit(queries_barrier(q_empty, segment));
        }
        step();
        for (int i = 0; i < n; ++i) {
          const uint32_t values_at = stage;
          const bool more = i + 1 < n;
          ok = ok && warp_wait(full + 8 * stage, round, patience);
          step();
          const uint32_t keys_at = stage;
#pragma unroll 1
          for (int q = 0; q < row_tiles; ++q) {
            ok = ok && warp_wait(p_ready + 8 * q, (p_phase >> q) & 1, patience);
            p_phase ^= 1u << q;
            if (more && q == 0) ok = ok && warp_wait(full + 8 * stage, round, patience);
            if (!ok) break;
            fence_after_sync();
            if (issues) {
              const uint32_t values = v_low + values_at * (kTileBytes >> 4);
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)
                mma_ts(tmem + 256 + q * 128, tmem + q * 128 + k * 8, values + k * 128, kOperandHigh, kOutput,
                       k > 0 ? 1u : static_cast<uint32_t>(i));
              if (more)
                scores(q, keys_at);
              else
                mma_commit(o_full + 8 * q);
            }
          }
          if (!ok) break;
          if (issues) {
            mma_commit(empty + 8 * values_at);
            if (more) mma_commit(empty + 8 * keys_at);
            if (i + 2 == n) mma_commit(queries_barrier(q_empty, segment));  // the last scores of the segment were just issued
          }
          if (more) step();
        }
        if (!ok) break;
      }
    }
    __syncwarp();
    if (warp == 13 && lane == 0 && working) {
      // -------------------------------------------------------- next segments
      Share s;
      s.left = share;
      s.block = start_block;
      const int64_t rest = begin - ws.first[s.block];
      const int span = ws.blocks[s.block].tiles + kSegmentCost;
      s.head = static_cast<int>(rest / span);
      s.from = static_cast<int>(rest - static_cast<int64_t>(s.head) * span);
      s.load(a, c, ws);
      s.place();
      if (s.end == s.tile) s.next(a, c, ws);
      for (uint32_t n = 0;; ++n) {
        if (n >= kSlots && !barrier_wait(released + 8 * (n % kSlots), (n / kSlots - 1) & 1, patience)) break;
        // the CTA of the segment's last tile
        const int64_t last = ws.first[s.block] + static_cast<int64_t>(s.head + 1) * (s.tiles + kSegmentCost) - 1;
        s.last_cta = static_cast<int>((plan.ctas * (last + 1) - 1) / plan.tiles);
        shares[n % kSlots] = s;
        dropped[n % kSlots] = 0;
        barrier_arrive(announced + 8 * (n % kSlots));
        if (s.end == s.tile) break;
        s.next(a, c, ws);
      }
    }
    __syncwarp();
    if (warp >= 14 && working) {
      // -------------------------------------------------------------- queries
      const int w = warp - 14;
      constexpr int kRowChunks = DP / 8;
      constexpr int kPerInstr = 32 / kRowChunks;
      const int chunk = lane % kRowChunks, sub = lane / kRowChunks;
      constexpr int kBatch = 8;  // rows of a lane in flight through registers; kBatch * kPerInstr divides 32
      bool ok = true;
      for (uint32_t segment = 0;; ++segment) {
        ok = announced_segment(segment);
        if (!ok) break;
        const Share& s = shares[segment % kSlots];
        if (s.end == s.tile) break;
        // Queries.  With e4m3 they go through registers, times a power of two
        // per row (power_up); so they do when the sign of a negative
        // scale or the zeros of a zero one go into them.
        if (segment >= kQueries)
          ok = warp_wait(queries_barrier(q_empty, segment), queries_parity(segment - kQueries), patience);
        if (!ok) break;
        const uint32_t tile = (2 * (segment % kQueries) + w) * kTileBytes;  // of this warp's 128 rows
        float* const unit_of = row_unit[segment % kQueries] + w * 128;
        const bool as_is = Cache::kLifted || (!kE4m3 && c.query_and == 0xffffffffu && c.query_xor == 0u);
#pragma unroll 1
        for (int r0 = 0; r0 < 128 && w < s.row_tiles(); r0 += 32) {  // a lane finds one of 32 rows
          const int r = w * 128 + r0 + lane;
          const int row = s.view.row + r, token = row / a.group;
          const int q_head = s.head * a.group + row - token * a.group;
          const int64_t lifted = (s.out_row + token) * (static_cast<int64_t>(a.kv_heads) * a.group) + q_head;
          const uint16_t* own = Cache::kLifted ? c.queries + lifted * a.dim
                                               : static_cast<const uint16_t*>(a.query) +
                                                     (s.out_row + token) * a.query_row +
                                                     static_cast<int64_t>(q_head) * a.query_head;
          const bool live = r < s.view.rows;
          const unsigned lives = __ballot_sync(0xffffffffu, live);
          const unsigned long long row_at =
              reinterpret_cast<unsigned long long>(live ? static_cast<const void*>(own) : a.query);
          if (Cache::kLifted)
            unit_of[r0 + lane] = live ? c.scale_log2 * __ldg(c.units + lifted) : 1.f;
          else if (!kE4m3)
            unit_of[r0 + lane] = c.scale_log2;
          if (as_is) {
            const char* src[32 / kPerInstr];
#pragma unroll
            for (int i = 0; i < 32 / kPerInstr; ++i)
              src[i] = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, row_at, i * kPerInstr + sub)) + chunk * 16;
            if (chunk < row_chunks) {
#pragma unroll
              for (int i = 0; i < 32 / kPerInstr; ++i)
                cp_async16(smem + tile + place(r0 + i * kPerInstr + sub, chunk), src[i],
                           (lives >> (i * kPerInstr + sub)) & 1u);
            }
            continue;
          }
          if constexpr (!Cache::kLifted) {
#pragma unroll 1
            for (int r1 = 0; r1 < 32; r1 += kBatch * kPerInstr) {
              uint4 x[kBatch];
#pragma unroll
              for (int i = 0; i < kBatch; ++i) {
                const int from = r1 + i * kPerInstr + sub;
                const uint4* src = reinterpret_cast<const uint4*>(__shfl_sync(0xffffffffu, row_at, from)) + chunk;
                x[i] = ((lives >> from) & 1u) && chunk < row_chunks ? __ldg(src) : make_uint4(0, 0, 0, 0);
              }
#pragma unroll
              for (int i = 0; i < kBatch; ++i) {
                const int at = r0 + r1 + i * kPerInstr + sub;
                uint32_t word[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                float unit = c.scale_log2;
                if constexpr (kE4m3) {
                  const bool bf16 = a.query_type == KVCA_TYPE_BF16;
                  float2 f[4];
                  float big = 0.f;
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    f[j] = bf16 ? unpack2<true>(word[j]) : unpack2<false>(word[j]);
                    big = fmaxf(big, fmaxf(fabsf(f[j].x), fabsf(f[j].y)));
                  }
#pragma unroll
                  for (int o = kRowChunks / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                  const int e = power_up(big);
                  const float up = power_of_two(e);
#pragma unroll
                  for (int j = 0; j < 4; ++j) word[j] = pack2<false>(f[j].x * up, f[j].y * up);
                  unit *= power_of_two(-e);
                }
                if (kE4m3 && chunk == 0) unit_of[at] = unit;
#pragma unroll
                for (int j = 0; j < 4; ++j) word[j] = (word[j] & c.query_and) ^ c.query_xor;
                if (chunk < row_chunks)
                  *reinterpret_cast<uint4*>(smem_ptr + tile + place(at, chunk)) =
                      make_uint4(word[0], word[1], word[2], word[3]);
              }
            }
          }
        }
        cp_async_wait_all();
        fence_async_proxy();
        barrier_arrive(queries_barrier(q_full, segment));
        release_segment(segment);
      }
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- loads
    if (working) {
      const int w = warp - 8;
      [[maybe_unused]] const uint32_t four_smem =
          kv_smem + kStages * kTileBytes + w * ((kAhead + 1) * Shape::kFourSide);
      constexpr int kRowChunks = DP / 8;             // of a row in shared memory
      constexpr int kPerInstr = 32 / kRowChunks;     // rows per instruction (16-bit rows)
      const int chunk = lane % kRowChunks, sub = lane / kRowChunks;
      bool ok = true;
      uint32_t issued = 0, arrived = 0;
      uint32_t segment = 0;
      // Of each tile in flight four bits: values of a cut tile, and the
      // segment's slot (nobody reuses it before its softmax, thus these, is done).
      uint32_t marks = 0;
      // Hands over the oldest of the tiles in flight.
      auto complete = [&]() {
        if constexpr (!kNarrow) {
          const uint32_t mark = marks >> (4 * (arrived & 7u));
          if (mark & 1u) {
            unsigned char* const tile = smem_ptr + 2 * kQueries * kTileBytes + (arrived % kStages) * kTileBytes;
            if (drop_non_finite<kBf16, DP>(tile, w * 32, row_chunks)) *const_cast<volatile int*>(&dropped[(mark >> 1) & 3u]) = 1;
            __syncwarp();
          }
        }
        fence_async_proxy();
        barrier_arrive(full + 8 * (arrived % kStages));
        ++arrived;
      };
      // The same with 4-bit rows: widens them into the next tile.  A lane has 32 values
      // with their two scales of one row at a time; the lanes of a quarter warp, two
      // pieces of four rows, read and write distinct banks.
      [[maybe_unused]] auto complete_four = [&]() {
        constexpr int kPieces = DP / 32;
        const uint32_t src = four_smem + (arrived % (kAhead + 1)) * Shape::kFourSide;
        const uint32_t mark = marks >> (4 * (arrived & 7u));
        __syncwarp();
        if (arrived >= kStages)
          ok = warp_wait(empty + 8 * (arrived % kStages), ((arrived / kStages) - 1) & 1, patience) && ok;
        if (!ok) return;
        unsigned char* const dst = smem_ptr + 2 * kQueries * kTileBytes + (arrived % kStages) * kTileBytes;
        uint32_t found = 0;
        auto part_of = [lane](int i) { return kPieces > 2 ? (lane & 1) + 2 * (i & 1) : lane & 1; };
        auto row_of = [lane](int i) { return (lane >> 1) + 16 * (kPieces > 2 ? i >> 1 : i); };
        uint4 raw[kPieces];
        uint16_t bytes[kPieces];
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {  // all of them before the first store
          const int part = part_of(i), r = row_of(i);
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(raw[i].x), "=r"(raw[i].y), "=r"(raw[i].z), "=r"(raw[i].w)
                       : "r"(src + r * (DP / 2) + ((part ^ (kPieces > 2 ? r & 2 : 0)) * 16)) : "memory");
          asm volatile("ld.shared.u16 %0, [%1];"
                       : "=h"(bytes[i]) : "r"(src + 32 * (DP / 2) + r * 8 + ((mark >> 2) & 2u) + 2 * part) : "memory");
        }
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int part = part_of(i), r = row_of(i);
          if (part * 32 >= a.dim) continue;
          const uint4 x = raw[i];
          uint32_t scales = bytes[i];
          if (mark & 1u) scales = drop_nan4(scales, &found);
          const uint32_t both = e4m3_to_f16x2(scales);
          const uint32_t factor[2] = {__byte_perm(both, 0, 0x1010), __byte_perm(both, 0, 0x3232)};
          const uint32_t in[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t wide[4];
            e2m1x8_to_f16x2(wide, in[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) wide[e] = mul_f16x2(wide[e], factor[j / 2]);
            *reinterpret_cast<uint4*>(dst + place(w * 32 + r, 4 * part + j)) =
                make_uint4(wide[0], wide[1], wide[2], wide[3]);
          }
        }
        if (found != 0) *const_cast<volatile int*>(&dropped[(mark >> 1) & 3u]) = 1;
        __syncwarp();  // the place may be filled again
        fence_async_proxy();
        barrier_arrive(full + 8 * (arrived % kStages));
        ++arrived;
      };
      auto drain = [&]() {
        while (arrived < issued && (!kFour || ok)) {
          if (issued - arrived == kAhead)
            cp_async_wait<kAhead - 1>();
          else
            cp_async_wait<0>();
          if constexpr (kFour)
            complete_four();
          else
            complete();
        }
      };
      // The ring entry of the next tile.  Before it waits for one, a warp
      // hands over what it has in flight.
      auto claim = [&]() {
        if (issued < kStages || !ok) return;
        const uint32_t bar = empty + 8 * (issued % kStages), parity = ((issued / kStages) - 1) & 1;
        if (__all_sync(0xffffffffu, barrier_test(bar, parity))) return;
        if constexpr (!kNarrow) drain();
        ok = warp_wait(bar, parity, patience);
      };
      constexpr int64_t kHidden = -1ll << 62;
      for (; ok; ++segment) {
        if constexpr (!kNarrow || kFour) {
          // nothing in flight is held back while the next segment is awaited
          if (arrived < issued &&
              !__all_sync(0xffffffffu, barrier_test(announced + 8 * (segment % kSlots), (segment / kSlots) & 1)))
            drain();
        }
        ok = announced_segment(segment);
        if (!ok) break;
        const Share& s = shares[segment % kSlots];
        if (s.end == s.tile) break;
        // keys and values, tile by tile; a lane looks up the page of one token
        int64_t page;
        int offset = 0;
        auto look_up = [&](int tile) {
          const int v = tile * kKeys + w * 32 + lane;
          page = kHidden;
          if (v < s.view.count) {
            const int key = s.view.key(v);
            const int block = a.block_shift >= 0 ? key >> a.block_shift : key / a.block_size;
            offset = key - block * a.block_size;
            page = __ldg(a.tables + static_cast<int64_t>(s.view.seq) * a.table_stride + block);
          }
        };
        look_up(s.tile);
        for (int tile = s.tile; tile < s.end && ok; ++tile) {
          // rows of hidden tokens, and of a page outside the cache, read as zeros
          const bool good = page >= 0 && page < a.num_blocks;
          if (!good && page != kHidden) report(a.status, KVCA_ERR_BAD_INDEX, page);
          const int64_t block = good ? page : 0;
          const unsigned seen = __ballot_sync(0xffffffffu, good);
          const char* const key_row = a.key + block * a.key_block + offset * a.key_token + s.head * a.key_head;
          const char* const value_row = a.value + block * a.value_block + offset * a.value_token + s.head * a.value_head;
          if (tile + 1 < s.end) look_up(tile + 1);
          const bool cut = s.cut(tile * kKeys, a.sinks);
#pragma unroll 1
          for (int side = 0; side < 2; ++side) {
            const unsigned long long row = reinterpret_cast<unsigned long long>(side == 0 ? key_row : value_row);
            if constexpr (!kNarrow) {
              claim();
              if (!ok) break;
              const uint32_t dst = kv_smem + (issued % kStages) * kTileBytes;
              const char* src[32 / kPerInstr];
#pragma unroll
              for (int i = 0; i < 32 / kPerInstr; ++i)
                src[i] = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, row, i * kPerInstr + sub)) + chunk * 16;
              if (chunk < row_chunks) {
#pragma unroll
                for (int i = 0; i < 32 / kPerInstr; ++i)
                  cp_async16(dst + place(w * 32 + i * kPerInstr + sub, chunk), src[i],
                             (seen >> (i * kPerInstr + sub)) & 1u);
              }
              cp_async_commit();
              const uint32_t mark = (side == 1 && cut ? 1u : 0u) | (segment % kSlots) << 1;
              marks = (marks & ~(15u << (4 * (issued & 7u)))) | mark << (4 * (issued & 7u));
              ++issued;
              if (issued - arrived > kAhead) {
                cp_async_wait<kAhead>();
                complete();
              }
            } else if constexpr (kFour) {
              // to the warp's own place, in 16-byte pieces of 32 values (pieces of rows
              // 2 and 3 of 4 with halves exchanged: see complete_four); a lane copies its
              // row's scales, at most two 4-byte words
              constexpr int kPieces = DP / 32, kRowsPer = 32 / kPieces;
              const int part = lane % kPieces, which = lane / kPieces;
              const uint32_t dst = four_smem + (issued % (kAhead + 1)) * Shape::kFourSide;
#pragma unroll
              for (int i = 0; i < kPieces; ++i) {
                const int r = i * kRowsPer + which;
                const char* const from = reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, row, r)) + part * 16;
                if (part * 32 < a.dim)
                  cp_async16(dst + r * (DP / 2) + ((part ^ (kPieces > 2 ? r & 2 : 0)) * 16), from, (seen >> r) & 1u);
              }
              const int scales = scales_after(a, s.head);
              const int off = scales & 2;  // rows and their values are multiples of 16
              const char* const from = reinterpret_cast<const char*>(row) + (scales - off);
              const uint32_t to = dst + 32 * (DP / 2) + lane * 8;
              const bool read = (seen >> lane) & 1u;
              cp_async4(to, from, read);
              if (off + a.dim / 16 > 4) cp_async4(to + 4, from + 4, read);
              cp_async_commit();
              const uint32_t mark =
                  (side == 1 && cut ? 1u : 0u) | (segment % kSlots) << 1 | static_cast<uint32_t>(off) << 2;
              marks = (marks & ~(15u << (4 * (issued & 7u)))) | mark << (4 * (issued & 7u));
              ++issued;
              if (issued - arrived > kAhead) {
                cp_async_wait<kAhead>();
                complete_four();
                if (!ok) break;
              }
            } else {
              // 16 e4m3 values per load become two chunks
              constexpr int kLoads = kRowChunks / 2;       // per row
              constexpr int kRowsPer = 32 / kLoads;
              const int part = lane % kLoads, which = lane / kLoads;
              uint4 x[32 / kRowsPer];
#pragma unroll
              for (int i = 0; i < 32 / kRowsPer; ++i) {
                const int r = i * kRowsPer + which;
                const uint4* from = reinterpret_cast<const uint4*>(__shfl_sync(0xffffffffu, row, r)) + part;
                x[i] = ((seen >> r) & 1u) && part * 16 < a.dim ? __ldg(from) : make_uint4(0, 0, 0, 0);
              }
              if (side == 1 && cut) {
                uint32_t found = 0;
#pragma unroll
                for (int i = 0; i < 32 / kRowsPer; ++i)
                  x[i] = make_uint4(drop_nan4(x[i].x, &found), drop_nan4(x[i].y, &found), drop_nan4(x[i].z, &found),
                                    drop_nan4(x[i].w, &found));
                if (found != 0) *const_cast<volatile int*>(&dropped[segment % kSlots]) = 1;
                __syncwarp();
              }
              claim();
              if (!ok) break;
              unsigned char* const dst = smem_ptr + 2 * kQueries * kTileBytes + (issued % kStages) * kTileBytes;
#pragma unroll
              for (int i = 0; i < 32 / kRowsPer; ++i) {
                const int r = w * 32 + i * kRowsPer + which;
                const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                uint32_t wide[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  wide[2 * j] = e4m3_to_f16x2(in[j]);
                  wide[2 * j + 1] = e4m3_to_f16x2(in[j] >> 16);
                }
                *reinterpret_cast<uint4*>(dst + place(r, 2 * part)) = make_uint4(wide[0], wide[1], wide[2], wide[3]);
                *reinterpret_cast<uint4*>(dst + place(r, 2 * part + 1)) =
                    make_uint4(wide[4], wide[5], wide[6], wide[7]);
              }
              ++issued;
              complete();
            }
          }
        }
        release_segment(segment);
      }
      if constexpr (!kNarrow || kFour) drain();
      cp_async_wait<0>();
    }
  } else {
    // -------------------------------------------------------------- softmax
    const int q = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t scores = tmem + lanes + q * 128, output = tmem + lanes + 256 + q * 128;
    const int r = q * 128 + (warp & 3) * 32 + lane;  // this thread's row of the block
    ChunkPiece piece{-1, -1, -1, 0};
    if (working) {
      bool ok = true;
      uint32_t segment = 0, phase = 0, o_phase = 0;
      for (;; ++segment) {
        ok = announced_segment(segment);
        if (!ok) break;
        const Share& s = shares[segment % kSlots];
        if (s.end == s.tile) break;
        ok = warp_wait(queries_barrier(q_full, segment), queries_parity(segment), patience);
        if (!ok) break;
        const float unit = row_unit[segment % kQueries][r];
        barrier_arrive(queries_barrier(q_empty, segment));
        const int n = s.end - s.tile;
        const bool starts = s.tile == 0, ends = s.end == s.tiles;
        if (q < s.row_tiles()) {
          // what this row sees, in numbers of the block's keys
          const int own = min(s.view.row + r, s.view.row + s.view.rows - 1);
          const int p = s.view.context + own / a.group;
          const int v_last = p - s.view.skip;
          const int v_low = a.window > 0 ? p - a.window - s.view.skip : -1;
          // the same for the tile's first and last row
          const int row_first = s.view.row + q * 128, row_last = min(row_first + 127, s.view.row + s.view.rows - 1);
          const int all_last = s.view.context + row_first / a.group - s.view.skip;
          const int all_low = a.window > 0 ? s.view.context + row_last / a.group - a.window - s.view.skip : -1;

          float m = -INFINITY, l = 0.f;  // m in units of the raw scores
          int v0 = s.tile * kKeys;
#pragma unroll 1
          for (int i = 0; i < n; ++i, v0 += kKeys) {
            ok = ok && warp_wait(s_full + 8 * q, phase & 1, patience);
            if (!ok) break;
            ++phase;
            fence_after_sync();
            // Hidden keys, behind the row's own token (only the block's last
            // tiles have any) or between the sinks and the window, are
            // overwritten before anything reads them.
            if (v0 + kKeys - 1 > all_last || (v0 + kKeys > a.sinks && max(v0, a.sinks) <= all_low)) {
#pragma unroll 1
              for (int j = 0; j < 4; ++j) {
                float x[32];
                tmem_load32(x, scores + j * 32);
                tmem_wait_load();
                tmem_landed(x);
                const int last = v_last - v0 - j * 32, first = a.sinks - v0 - j * 32;
                const unsigned gap = max(v_low - v0 - j * 32 + 1 - first, 0);
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  x[k] = (k > last) | (static_cast<unsigned>(k - first) < gap) ? -INFINITY : x[k];
                tmem_store32(scores + j * 32, x);
              }
              tmem_wait_store();
            }
            float xa[32], xb[32];
            float best = -INFINITY;
            auto largest = [&](const float (&x)[32]) {
              float top[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) top[k] = fmaxf(x[2 * k], x[2 * k + 1]);
#pragma unroll
              for (int k = 8; k < 32; k += 8)
#pragma unroll
                for (int i = 0; i < 4; ++i) top[i] = max3(top[i], x[k + 2 * i], x[k + 2 * i + 1]);
              best = fmaxf(best, fmaxf(max3(top[0], top[1], top[2]), top[3]));
            };
            tmem_load32(xa, scores);
#pragma unroll 1
            for (int j = 0; j < 4; j += 2) {
              tmem_wait_load();
              tmem_landed(xa);
              tmem_load32(xb, scores + j * 32 + 32);
              largest(xa);
              tmem_wait_load();
              tmem_landed(xb);
              tmem_load32(xa, scores + ((j * 32 + 64) & 127));  // around to the first for the second pass
              largest(xb);
            }
            const float old = m;
            // (-inf) - (-inf) is no growth
            if ((best - m) * unit > kGrowth) m = best;
            const float base = m == -INFINITY ? 0.f : m * unit;
            const float decay = m != old ? exp2_approx(old * unit - base) : 1.f;
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
            const float low = kShift<Cache> - base;
            const float2 units = make_float2(unit, unit), bases = make_float2(low, low);
            auto weigh = [&](const float (&x)[32], int j) {
              uint32_t packed[16];
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                float2 e = fma2(make_float2(x[k], x[k + 1]), units, bases);
                e = make_float2(exp2_approx(e.x), exp2_approx(e.y));
                sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], e);
                packed[k >> 1] = pack2<kBf16>(e.x, e.y);
              }
              tmem_store16(scores + j * 16, packed);
            };
#pragma unroll 1
            for (int j = 0; j < 4; j += 2) {
              tmem_wait_load();
              tmem_landed(xa);
              tmem_load32(xb, scores + j * 32 + 32);
              weigh(xa, j);
              tmem_wait_load();
              tmem_landed(xb);
              if (j == 0) tmem_load32(xa, scores + 64);
              weigh(xb, j + 1);
            }
            l = l * decay + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
            if (i > 0 && __any_sync(0xffffffffu, m != old)) {
#pragma unroll 1
              for (int j = 0; j < DP / 32; ++j) {
                float o[32];
                tmem_load32(o, output + j * 32);
                tmem_wait_load();
                tmem_landed(o);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] *= decay;
                tmem_store32(output + j * 32, o);
              }
            }
            tmem_wait_store();
            fence_before_sync();
            barrier_arrive(p_ready + 8 * q);
          }
          ok = ok && warp_wait(o_full + 8 * q, o_phase & 1, patience);
          if (!ok) break;
          ++o_phase;
          fence_after_sync();

          const float base = m == -INFINITY ? 0.f : m * unit;
          const bool live = r < s.view.rows;
          const bool whole = starts && ends;
          const float factor = whole ? a.value_scale / l : 1.f;
          const int token = own / a.group;
          const int64_t row = s.out_row + token;
          const int head = s.head * a.group + own - token * a.group;
          const int64_t out_row = row * (static_cast<int64_t>(a.kv_heads) * a.group) + head;
          const int64_t slot = static_cast<int64_t>(blockIdx.x) * 2 + (starts ? 1 : 0);
          float* const part = ws.acc + (slot * kRows + r) * DP;
          uint16_t* const out = static_cast<uint16_t*>(a.out) + out_row * a.dim;
          bool finite = true;
#pragma unroll 1
          for (int j = 0; j < DP / 32; ++j) {
            float o[32];
            __syncwarp();
            tmem_load32(o, output + j * 32);
            tmem_wait_load();
            tmem_landed(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) finite &= fabsf(o[k]) < INFINITY;
            if (live && whole) {
              const bool bf16 = a.query_type == KVCA_TYPE_BF16;
#pragma unroll
              for (int k = 0; k < 32; k += 8) {
                if (j * 32 + k >= a.dim) break;
                uint4 w;
                uint32_t* const word = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                  const float x0 = o[k + 2 * h] * factor, x1 = o[k + 2 * h + 1] * factor;
                  word[h] = bf16 ? pack2<true>(x0, x1) : pack2<false>(x0, x1);
                }
                *reinterpret_cast<uint4*>(out + j * 32 + k) = w;
              }
            } else if (live) {
#pragma unroll
              for (int k = 0; k < 32; k += 4)
                *reinterpret_cast<float4*>(part + j * 32 + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
          }
          if (live) {
            if (whole) {
              if (a.lse != nullptr) a.lse[out_row] = (base - kShift<Cache>) * kLn2 + logf(l);
            } else {
              float* const ml = ws.ml + slot * 2 * kRows;
              ml[r] = m == -INFINITY ? -INFINITY : base;
              ml[kRows + r] = l;
            }
          }
          // the outputs of rows whose sum is a number show values that are not
          const bool mine = live && l < INFINITY;
          const bool uncut = __any_sync(0xffffffffu, mine && !finite);
          const bool cut = *const_cast<volatile int*>(&dropped[segment % kSlots]) != 0;
          if (uncut || cut)
            put_non_finite<Cache, DP>(a, s, uncut, cut, mine, v_last, v_low, whole ? out : nullptr, part);
          fence_before_sync();
        }
        if (!(starts && ends)) {
          const int id = s.block * a.kv_heads + s.head;
          if (starts) {
            piece.head = id;
            piece.last = s.last_cta;
          } else {
            piece.tail = id;
          }
        }
        release_segment(segment);
      }
    }
    if (threadIdx.x == 0 && working) ws.pieces[blockIdx.x] = piece;
  }
  fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && gave_up != 0) report(a.status, KVCA_ERR_DEVICE_TIMEOUT, blockIdx.x);
  if (warp == 12) {
    fence_after_sync();
    if (gave_up != 0) {
      // products that nobody waited for may still run: they end before their
      // memory goes (bounded, 80 ms)
      if (lane == 0) mma_commit(drained);
      for (int i = 0; i < 4096 && !barrier_try_for(drained, 0, kTryTime); ++i) {
      }
      __syncwarp();
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the partial results of the blocks that several CTAs share: a column
// of blocks of the grid per CTA that began one, kJoinRows rows each.
template <int DP>
__global__ void __launch_bounds__(kJoinThreads) attend_chunk_join_kernel(const __grid_constant__ AttendArgs a,
                                                                        const __grid_constant__ ChunkArgs c,
                                                                        void* workspace, int64_t ctas) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  ChunkWorkspace ws(workspace, DP, ctas, c.max_blocks);
  const int64_t owner = blockIdx.x;
  if (owner >= ws.header->ctas) return;
  const ChunkPiece own = ws.pieces[owner];
  if (own.head < 0) return;
  const int block = own.head / a.kv_heads, kv_head = own.head - block * a.kv_heads;
  const ChunkBlock b = ws.blocks[block];
  constexpr int kPerRow = kJoinThreads / kJoinRows;  // threads per row
  const int r = blockIdx.y * kJoinRows + threadIdx.x / kPerRow;
  if (r >= b.rows) return;
  const int t = threadIdx.x % kPerRow;
  float top = -INFINITY;
  for (int64_t p = owner; p <= own.last; ++p)
    top = fmaxf(top, __ldcg(ws.ml + (p * 2 + (p == owner)) * 2 * kRows + r));
  const float base = top == -INFINITY ? 0.f : top;
  constexpr int kVecs = DP / 4 / kPerRow;
  float4 sum[kVecs];
#pragma unroll
  for (int v = 0; v < kVecs; ++v) sum[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.f;
#pragma unroll 4
  for (int64_t p = owner; p <= own.last; ++p) {
    const int64_t slot = p * 2 + (p == owner);
    const float* const ml = ws.ml + slot * 2 * kRows;
    // never 0: an infinite value is the result, however small its weight
    const float w = max_nan(exp2_approx(__ldcg(ml + r) - base), 0x1p-126f);
    total += w * __ldcg(ml + kRows + r);
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const float4 o = __ldcg(reinterpret_cast<const float4*>(ws.acc + (slot * kRows + r) * DP) + t + v * kPerRow);
      sum[v].x += w * o.x;
      sum[v].y += w * o.y;
      sum[v].z += w * o.z;
      sum[v].w += w * o.w;
    }
  }
  const int flat = b.row + r;
  const int token = flat / a.group;
  const int64_t out_row = (__ldg(c.offsets + b.seq) + token) * (static_cast<int64_t>(a.kv_heads) * a.group) +
                          kv_head * a.group + flat - token * a.group;
  const float factor = a.value_scale / total;
  const bool bf16 = a.query_type == KVCA_TYPE_BF16;
#pragma unroll
  for (int v = 0; v < kVecs; ++v) {
    const int d = (t + v * kPerRow) * 4;
    if (d >= a.dim) continue;
    uint2 w;
    w.x = bf16 ? pack2<true>(sum[v].x * factor, sum[v].y * factor) : pack2<false>(sum[v].x * factor, sum[v].y * factor);
    w.y = bf16 ? pack2<true>(sum[v].z * factor, sum[v].w * factor) : pack2<false>(sum[v].z * factor, sum[v].w * factor);
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + out_row * a.dim + d) = w;
  }
  if (a.lse != nullptr && t == 0) a.lse[out_row] = (base - c.shift) * kLn2 + logf(total);
}

template <typename Cache, int DP>
cudaError_t launch_typed(const AttendArgs& a, const ChunkArgs& c, void* workspace, int sms, cudaStream_t stream) {
  auto kernel = attend_chunk_kernel<Cache, DP>;
  constexpr int kSmem = ChunkShape<DP>::kSmem + (Cache::kBytes == 0 ? ChunkShape<DP>::kFourBytes : 0);
  static DeviceFlags configured;
  int dev = -1;
  if (needs_setup(configured, &dev)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return e;
    mark_setup(configured, dev);
  }
  const int64_t ctas = sms;
  // a block to plan, and with queries to lift as many as their rows keep busy
  int64_t lifting = 0;
  if (Cache::kLifted) lifting = (c.rows * a.kv_heads * a.group + 4 * kPlanThreads / 32 - 1) / (4 * kPlanThreads / 32);
  attend_chunk_plan_kernel<<<1 + static_cast<int>(lifting < 2 * sms ? lifting : 2 * sms), kPlanThreads, 0, stream>>>(
      a, c, workspace, DP, ctas);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  e = launch_dependent(kernel, dim3(sms), kThreads, kSmem, stream, a, c, workspace);
  if (e != cudaSuccess) return e;
  return launch_dependent(attend_chunk_join_kernel<DP>, dim3(sms, kRows / kJoinRows), kJoinThreads, 0, stream, a, c,
                          workspace, ctas);
}

template <typename Cache>
cudaError_t launch_cache(const AttendArgs& a, const ChunkArgs& c, void* workspace, int sms, cudaStream_t stream) {
  return a.dim <= 64 ? launch_typed<Cache, 64>(a, c, workspace, sms, stream)
                     : launch_typed<Cache, 128>(a, c, workspace, sms, stream);
}

}  // namespace

int64_t attend_chunk_max_blocks(const AttendArgs& a, int64_t rows) {
  return rows * a.group / kRows + a.num_seqs;  // each sequence's last block may be short
}

// Bytes of the workspace before the lifted queries.
static size_t chunk_workspace_plan(const AttendArgs& a, int64_t rows, int sms) {
  return (ChunkWorkspace::bytes(a.dim <= 64 ? 64 : 128, sms, attend_chunk_max_blocks(a, rows)) + 15) / 16 * 16;
}

static bool lifts_queries(const AttendArgs& a) {
  return a.cache_type == KVCA_TYPE_E2M1 && a.query_type == KVCA_TYPE_BF16;
}

size_t attend_chunk_workspace(const AttendArgs& a, int64_t rows, int sms) {
  const size_t query_rows = lifts_queries(a) ? static_cast<size_t>(rows) * a.kv_heads * a.group : 0;
  return chunk_workspace_plan(a, rows, sms) + query_rows * (a.dim * sizeof(uint16_t) + sizeof(float));
}

cudaError_t launch_attend_chunk(const AttendArgs& args, const int64_t* offsets, int64_t rows, int64_t wait_limit,
                                void* workspace, int sms, cudaStream_t stream) {
  AttendArgs a = args;
  ChunkArgs c;
  c.offsets = offsets;
  c.rows = rows;
  c.wait_limit = wait_limit;
  c.max_blocks = static_cast<int>(attend_chunk_max_blocks(a, rows));
  // the softmax takes the maximum of the raw scores, so their factor is positive
  c.scale_log2 = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
  c.query_and = a.scale_log2 == 0.f ? 0u : 0xffffffffu;
  c.query_xor = a.scale_log2 < 0.f ? 0x80008000u : 0u;
  c.queries = nullptr;
  c.units = nullptr;
  if (lifts_queries(a)) {
    c.queries = reinterpret_cast<uint16_t*>(static_cast<char*>(workspace) + chunk_workspace_plan(a, rows, sms));
    c.units = reinterpret_cast<float*>(c.queries + rows * a.kv_heads * a.group * a.dim);
  }
  c.shift = a.cache_type == KVCA_TYPE_BF16 ? kShift<CacheBf16> : kShift<CacheF16>;
  switch (a.cache_type) {
    case KVCA_TYPE_F16: return launch_cache<CacheF16>(a, c, workspace, sms, stream);
    case KVCA_TYPE_BF16: return launch_cache<CacheBf16>(a, c, workspace, sms, stream);
    case KVCA_TYPE_E2M1:
      return a.query_type == KVCA_TYPE_BF16 ? launch_cache<CacheE2m1<true>>(a, c, workspace, sms, stream)
                                            : launch_cache<CacheE2m1<false>>(a, c, workspace, sms, stream);
    default: return launch_cache<CacheE4m3>(a, c, workspace, sms, stream);
  }
}

}  // namespace kvca

// What the decode step's kernels share: their products, how a call's tiles are
// numbered and dealt out to runs, and where runs that share a segment leave their
// results.
//
// The tiles of all sequences, each for all chunks of head groups, are numbered
// one after the other, with a segment's fixed cost as tiles before its first; a
// run is an even share of the numbering.
#pragma once

#include "attend_common.cuh"

namespace kvca {
namespace {

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
template <int kTile, int kSegmentCost>
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
  // `count` tiles on; whether the run has one there.
  __device__ __forceinline__ bool skip(const AttendArgs& a, int chunks, int count) {
    while (count > 0 && left > 0) {
      const int here = min(count, tiles - 1 - tile);
      tile += here;
      left -= here;
      count -= here;
      if (count == 0 || left <= 0) break;
      if (last()) {
        left = 0;
        break;
      }
      advance(a, chunks);
      --count;
    }
    return left > 0;
  }
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
template <int kSegmentCost>
__device__ __forceinline__ int64_t sequence_share(int tiles, int chunks) {
  return tiles > 0 ? static_cast<int64_t>(tiles + kSegmentCost) * chunks : 0;
}

}  // namespace
}  // namespace kvca

// Sharing, dropping and moving the pages of a cache's sequences.
//
// A page table row names the slots of a sequence's pages in order; a slot's
// pin count says how many sequences hold it.  All three operators are bound
// by their launches and the dependent reads in them (table entry, then slot
// word) until many pages' bytes move, and then by HBM.  Each is a chain of
// small launches, the later ones programmatic dependents, instead of one
// kernel with grid barriers, because the work of each part is spread over the
// whole GPU differently.  240 children of 48 sequences (64 planes, 60 MB): 54 us;
// 128 sequences with 75,000 pages freed: 40 us; 1.85 GB of pages compacted: 310
// us, 91 % of the measured copy bandwidth.

#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "kvca_device.cuh"
#include "kvca_host.cuh"
#include "kvca_launch.h"

namespace kvca {
namespace {

constexpr int kPageThreads = 256;
constexpr int kEntriesPerBlock = 4 * kPageThreads;  // table entries
constexpr int kScanSlots = 4096;                    // slots per block of the compaction's passes
constexpr int kCopyBytes = 4096;                    // of one warp's item

__device__ __forceinline__ void dependent_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependent_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Adds `delta` (1 or -1) to the pin count of a slot; false, and nothing
// added, when the slot has none and `held` or the field would wrap.  Other
// slots of the 32-bit word may change at the same time.
template <typename MetaT>
__device__ __forceinline__ bool add_pin(MetaT* meta, int64_t slot, int delta, bool held) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(meta + slot);
  unsigned* const word = reinterpret_cast<unsigned*>(at & ~uintptr_t{3});
  const unsigned shift = static_cast<unsigned>(at & 3) * 8;
  unsigned old = *reinterpret_cast<volatile unsigned*>(word);
  for (;;) {
    const unsigned pin = (old >> shift) & Meta<MetaT>::kFieldMask;
    if ((held && pin == 0) || (delta > 0 && pin == Meta<MetaT>::kFieldMask)) return false;
    const unsigned seen = atomicCAS(word, old, delta > 0 ? old + (1u << shift) : old - (1u << shift));
    if (seen == old) return true;
    old = seen;
  }
}

// One warp copies bytes [begin, begin + kCopyBytes) of `rows` rows of
// row_bytes (stride row_stride) laid end to end.
template <typename V>
__device__ __forceinline__ void copy_part(char* dst, const char* src, int64_t begin, int64_t total, int64_t row_bytes,
                                          int64_t row_stride) {
  constexpr int kPerLane = kCopyBytes / 32 / static_cast<int>(sizeof(V));
  constexpr int kBatch = kPerLane < 8 ? kPerLane : 8;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int first = 0; first < kPerLane; first += kBatch) {
    V v[kBatch];
    int64_t at[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int64_t byte = begin + static_cast<int64_t>((first + i) * 32 + lane) * sizeof(V);
      at[i] = -1;
      if (byte < total) {
        at[i] = row_stride == row_bytes ? byte : byte / row_bytes * row_stride + byte % row_bytes;
        v[i] = __ldcs(reinterpret_cast<const V*>(src + at[i]));
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (at[i] >= 0) __stcs(reinterpret_cast<V*>(dst + at[i]), v[i]);
  }
}

// ---------------------------------------------------------------------------
// Fork
// ---------------------------------------------------------------------------

// Workspace of fork and free: the checks' verdicts, then a byte per table
// entry whose pin was changed (to take back when a later check fails).
struct PageHeader {
  int32_t refused;         // by the pass over the entries
  int32_t verdicts[63];    // of the first checks, one per block of 1,024 sequences
};
static_assert(kPageOpMaxSequences == 63 * 1024, "one verdict per block of 1,024");

__device__ __forceinline__ bool checks_passed(const PageHeader* h, int blocks) {
  for (int i = 0; i < blocks; ++i)
    if (h->verdicts[i] != 0) return false;
  return true;
}

__device__ __forceinline__ int64_t pages_of(int64_t len, int64_t block_size) {
  return (len + block_size - 1) / block_size;
}

constexpr int kCheckThreads = 1024;

// What the pairs of a fork are compared with, a block's worth at a time.
struct ForkTile {
  int64_t parent[kCheckThreads], child[kCheckThreads], fresh[kCheckThreads], id[kCheckThreads];
  bool partial[kCheckThreads];
};

// Everything about pair j that does not concern single pages; the block's
// threads take pairs side by side (those past the last one help with the
// tiles).  True when the pair is refused (and reported).
template <typename MetaT>
__device__ bool fork_refused(const ForkArgs& f, int64_t j, ForkTile& tile) {
  const PageTable& t = f.table;
  int64_t code = 0, value = 0;
  auto refuse = [&](int64_t c, int64_t v) {
    if (code == 0) {
      code = c;
      value = v;
    }
  };
  int64_t child = -1, fresh = -1, id = -1;
  bool partial = false;
  if (j < f.count) {
    const int64_t parent = f.parents[j];
    child = f.children[j];
    if (parent < 0 || parent >= t.num_seqs)
      refuse(KVCA_ERR_BAD_INDEX, parent);
    else if (child < 0 || child >= t.num_seqs)
      refuse(KVCA_ERR_BAD_INDEX, child);
    else {
      const int64_t len = t.lens[parent];
      if (len < 0 || t.lens[child] > 0) refuse(KVCA_ERR_BAD_ARGUMENT, len < 0 ? parent : child);
      if (len > t.width * t.block_size) refuse(KVCA_ERR_BAD_INDEX, len);
      partial = code == 0 && len % t.block_size != 0;
      if (partial) {
        fresh = f.fresh_slots[j];
        id = f.fresh_ids[j];
        const int64_t source = t.tables[parent * t.stride + len / t.block_size];
        if (source < 0 || source >= f.pool.num_slots)
          refuse(KVCA_ERR_BAD_INDEX, source);
        else if (fresh < 0 || fresh >= f.pool.num_slots)
          refuse(KVCA_ERR_BAD_INDEX, fresh);
        else if (id < 0 || id >= f.pool.num_logical)
          refuse(KVCA_ERR_BAD_INDEX, id);
        else if (Meta<MetaT>::pin(static_cast<const MetaT*>(f.pool.slot_meta)[source]) == 0)
          refuse(KVCA_ERR_BAD_ARGUMENT, source);
        else if (Meta<MetaT>::pin(static_cast<const MetaT*>(f.pool.slot_meta)[fresh]) != 0)
          refuse(KVCA_ERR_BAD_ARGUMENT, fresh);
        else if (f.pool.l2p[id] >= 0)
          refuse(KVCA_ERR_BAD_ARGUMENT, id);
        else if (f.pool.p2l[fresh] >= f.pool.num_logical)
          refuse(KVCA_ERR_BAD_INDEX, f.pool.p2l[fresh]);
      }
    }
  }
  // against every other pair
  for (int64_t base = 0; base < f.count; base += kCheckThreads) {
    const int64_t k = base + threadIdx.x;
    __syncthreads();
    if (k < f.count) {
      const int64_t other = f.parents[k];
      tile.parent[threadIdx.x] = other;
      tile.child[threadIdx.x] = f.children[k];
      tile.fresh[threadIdx.x] = f.fresh_slots[k];
      tile.id[threadIdx.x] = f.fresh_ids[k];
      // it counts if it needs its slot, too
      const bool known = other >= 0 && other < t.num_seqs;
      tile.partial[threadIdx.x] = known && t.lens[other] > 0 && t.lens[other] % t.block_size != 0;
    }
    __syncthreads();
    if (j >= f.count) continue;
    const int n = static_cast<int>(min(static_cast<int64_t>(kCheckThreads), f.count - base));
    const int self = static_cast<int>(min(max(j - base, int64_t{-1}), int64_t{kCheckThreads}));
    bool same_child = false, same_slot = false, same_id = false;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const bool other = i != self, copies = other & tile.partial[i];
      same_child |= (tile.parent[i] == child) | (other & (tile.child[i] == child));
      same_slot |= copies & (tile.fresh[i] == fresh);
      same_id |= copies & (tile.id[i] == id);
    }
    if (same_child) refuse(KVCA_ERR_BAD_ARGUMENT, child);
    if (partial && same_slot) refuse(KVCA_ERR_BAD_ARGUMENT, fresh);
    if (partial && same_id) refuse(KVCA_ERR_BAD_ARGUMENT, id);
  }
  if (code != 0) report(f.pool.status, code, value);
  return code != 0;
}

template <typename MetaT>
__global__ void __launch_bounds__(kCheckThreads) fork_check_kernel(const __grid_constant__ ForkArgs f,
                                                                  PageHeader* header) {
  __shared__ ForkTile tile;
  dependent_trigger();
  const int bad = __syncthreads_or(fork_refused<MetaT>(f, static_cast<int64_t>(blockIdx.x) * kCheckThreads + threadIdx.x, tile));
  if (threadIdx.x == 0) {
    header->verdicts[blockIdx.x] = bad;
    if (blockIdx.x == 0) header->refused = 0;
  }
}

// Pins page i of pair j's parent; false (and reported) when it cannot.
template <typename MetaT>
__device__ __forceinline__ bool fork_pin(const ForkArgs& f, int64_t j, int64_t i, int64_t parent, uint8_t* pinned) {
  const int64_t slot = f.table.tables[parent * f.table.stride + i];
  bool done = false, fine = true;
  if (slot >= f.pool.num_slots) {
    report(f.pool.status, KVCA_ERR_BAD_INDEX, slot);
    fine = false;
  } else if (slot >= 0) {
    done = fine = add_pin(static_cast<MetaT*>(f.pool.slot_meta), slot, 1, true);
    if (!done) report(f.pool.status, KVCA_ERR_BAD_ARGUMENT, slot);  // held by nobody, or as often as its field counts
  }
  pinned[j * f.table.width + i] = done;
  return fine;
}

// Page i of pair j's child, or the pin back.
template <typename MetaT>
__device__ __forceinline__ void fork_page(const ForkArgs& f, int64_t j, int64_t i, int64_t parent, int64_t child,
                                          bool refused, const uint8_t* pinned) {
  const PageTable& t = f.table;
  const int64_t slot = t.tables[parent * t.stride + i];
  if (!refused)
    t.tables[child * t.stride + i] = slot;
  else if (pinned[j * t.width + i])
    add_pin(static_cast<MetaT*>(f.pool.slot_meta), slot, -1, true);
}

// The rest of pair j's child: its last page's metadata and its length.
template <typename MetaT>
__device__ __forceinline__ void fork_child(const ForkArgs& f, int64_t j, int64_t len, int64_t child) {
  const PageTable& t = f.table;
  if (len % t.block_size != 0) {
    const int64_t fresh = f.fresh_slots[j], id = f.fresh_ids[j];
    t.tables[child * t.stride + len / t.block_size] = fresh;
    const int64_t old = f.pool.p2l[fresh];
    if (old >= 0) f.pool.l2p[old] = -1;
    f.pool.l2p[id] = fresh;
    f.pool.p2l[fresh] = id;
    static_cast<MetaT*>(f.pool.slot_meta)[fresh] = Meta<MetaT>::pack(1, 1);
  }
  t.lens[child] = len;
}

// A small fork's checks, pins and tables by one block (the bytes follow).
template <typename MetaT>
__global__ void __launch_bounds__(kCheckThreads) fork_small_kernel(const __grid_constant__ ForkArgs f,
                                                                  PageHeader* header, uint8_t* pinned) {
  __shared__ ForkTile tile;
  dependent_trigger();
  const int bad = __syncthreads_or(fork_refused<MetaT>(f, threadIdx.x, tile));
  if (threadIdx.x == 0) {
    header->verdicts[0] = bad;
    header->refused = 0;
  }
  if (bad) return;
  const PageTable& t = f.table;
  const int lanes = 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  bool fine = true;
  for (int64_t j = warp; j < f.count; j += kCheckThreads / lanes) {
    const int64_t parent = f.parents[j];
    const int64_t full = t.lens[parent] / t.block_size;
    for (int64_t i = lane; i < full; i += lanes) fine &= fork_pin<MetaT>(f, j, i, parent, pinned);
  }
  const bool refused = __syncthreads_or(!fine) != 0;
  if (threadIdx.x == 0) header->refused = refused;
  for (int64_t j = warp; j < f.count; j += kCheckThreads / lanes) {
    const int64_t parent = f.parents[j], child = f.children[j];
    const int64_t len = t.lens[parent];
    for (int64_t i = lane; i < len / t.block_size; i += lanes) fork_page<MetaT>(f, j, i, parent, child, refused, pinned);
    if (!refused && lane == 0) fork_child<MetaT>(f, j, len, child);
  }
}

// Pins the shared pages, one more per child.
template <typename MetaT>
__global__ void __launch_bounds__(kPageThreads) fork_pin_kernel(const __grid_constant__ ForkArgs f, PageHeader* header,
                                                                uint8_t* pinned, int checks) {
  dependent_wait();
  dependent_trigger();
  if (!checks_passed(header, checks)) return;
  const PageTable& t = f.table;
  const int64_t j = blockIdx.x;
  const int64_t parent = f.parents[j];
  const int64_t full = t.lens[parent] / t.block_size;
  const int64_t base = static_cast<int64_t>(blockIdx.y) * kEntriesPerBlock;
  for (int64_t i = base + threadIdx.x; i < full && i < base + kEntriesPerBlock; i += kPageThreads)
    if (!fork_pin<MetaT>(f, j, i, parent, pinned)) header->refused = 1;
}

// The children's tables, their last pages' metadata and bytes; or, when a
// page was refused, the pins back.  Blocks of the grid's last row copy.
template <typename MetaT, typename V>
__global__ void __launch_bounds__(kPageThreads) fork_commit_kernel(const __grid_constant__ ForkArgs f,
                                                                   const __grid_constant__ PagedSide cache,
                                                                   int num_planes, int64_t row_bytes,
                                                                   const PageHeader* header, const uint8_t* pinned,
                                                                   int checks, int copy_blocks) {
  dependent_wait();
  if (!checks_passed(header, checks)) return;
  const bool refused = header->refused != 0;
  const PageTable& t = f.table;
  if (static_cast<int>(blockIdx.x) < copy_blocks) {
    if (refused) return;
    const int64_t block_bytes = t.block_size * row_bytes;
    const int64_t parts = (block_bytes + kCopyBytes - 1) / kCopyBytes;
    const int64_t items = f.count * num_planes * parts;
    const int64_t warps = static_cast<int64_t>(copy_blocks) * (kPageThreads / 32);
    for (int64_t it = static_cast<int64_t>(blockIdx.x) * (kPageThreads / 32) + (threadIdx.x >> 5); it < items;
         it += warps) {
      const int64_t part = it % parts, rest = it / parts;
      const int64_t j = rest / num_planes;
      const int plane = static_cast<int>(rest - j * num_planes);
      const int64_t parent = f.parents[j];
      const int64_t len = t.lens[parent];
      const int64_t total = len % t.block_size * row_bytes;
      if (part * kCopyBytes >= total) continue;
      const int64_t source = t.tables[parent * t.stride + len / t.block_size];
      char* const base = reinterpret_cast<char*>(cache.planes[plane]);
      copy_part<V>(base + f.fresh_slots[j] * cache.block_stride, base + source * cache.block_stride, part * kCopyBytes,
                   total, row_bytes, cache.row_stride);
    }
    return;
  }
  const int64_t chunks = (t.width + kEntriesPerBlock - 1) / kEntriesPerBlock;
  const int64_t at = blockIdx.x - copy_blocks;
  const int64_t j = at / chunks, chunk = at - j * chunks;
  const int64_t parent = f.parents[j], child = f.children[j];
  const int64_t len = t.lens[parent];
  const int64_t full = len / t.block_size;
  const int64_t base = chunk * kEntriesPerBlock;
  for (int64_t i = base + threadIdx.x; i < full && i < base + kEntriesPerBlock; i += kPageThreads)
    fork_page<MetaT>(f, j, i, parent, child, refused, pinned);
  if (!refused && chunk == 0 && threadIdx.x == 0) fork_child<MetaT>(f, j, len, child);
}

// ---------------------------------------------------------------------------
// Free
// ---------------------------------------------------------------------------

// Everything about sequence j of the call that does not concern single pages;
// keeps its length.  True when it is refused (and reported).
__device__ bool free_refused(const FreeArgs& f, int64_t j, int64_t (&tile)[kCheckThreads]) {
  const PageTable& t = f.table;
  int64_t code = 0, value = 0, seq = -1;
  if (j < f.count) {
    value = seq = f.sequences[j];
    if (seq < 0 || seq >= t.num_seqs) {
      code = KVCA_ERR_BAD_INDEX;
    } else {
      const int64_t len = t.lens[seq];
      f.lens_before[j] = len;
      if (len > t.width * t.block_size) {
        code = KVCA_ERR_BAD_INDEX;
        value = len;
      }
    }
  }
  for (int64_t base = 0; base < f.count; base += kCheckThreads) {  // twice in the list
    __syncthreads();
    if (base + threadIdx.x < f.count) tile[threadIdx.x] = f.sequences[base + threadIdx.x];
    __syncthreads();
    if (j >= f.count || code != 0) continue;
    const int n = static_cast<int>(min(static_cast<int64_t>(kCheckThreads), f.count - base));
    bool twice = false;
#pragma unroll 4
    for (int k = 0; k < n; ++k) twice |= (tile[k] == seq) & (base + k != j);
    if (twice) code = KVCA_ERR_BAD_ARGUMENT;
  }
  if (code != 0) report(f.pool.status, code, value);
  return code != 0;
}

__global__ void __launch_bounds__(kCheckThreads) free_check_kernel(const __grid_constant__ FreeArgs f,
                                                                  PageHeader* header) {
  __shared__ int64_t tile[kCheckThreads];
  dependent_trigger();
  const int bad = __syncthreads_or(free_refused(f, static_cast<int64_t>(blockIdx.x) * kCheckThreads + threadIdx.x, tile));
  if (threadIdx.x == 0) {
    header->verdicts[blockIdx.x] = bad;
    if (blockIdx.x == 0) header->refused = 0;
  }
}

// One holder less of page i of sequence j; false (and reported) when it cannot.
template <typename MetaT>
__device__ __forceinline__ bool free_unpin(const FreeArgs& f, int64_t j, int64_t i, int64_t seq, uint8_t* unpinned) {
  const int64_t slot = f.table.tables[seq * f.table.stride + i];
  bool done = false, fine = true;
  if (slot >= f.pool.num_slots) {
    report(f.pool.status, KVCA_ERR_BAD_INDEX, slot);
    fine = false;
  } else if (slot >= 0) {
    done = fine = add_pin(static_cast<MetaT*>(f.pool.slot_meta), slot, -1, true);
    if (!done) report(f.pool.status, KVCA_ERR_BAD_ARGUMENT, slot);  // held by fewer sequences than name it
  }
  unpinned[j * f.table.width + i] = done;
  return fine;
}

// Entry i of sequence j cleared, and with `discard` its page unmapped if
// nobody holds it any more (every sequence that held it writes the same
// words); or the pin back.
template <typename MetaT>
__device__ __forceinline__ void free_page(const FreeArgs& f, int64_t j, int64_t i, int64_t seq, bool refused,
                                          const uint8_t* unpinned) {
  const PageTable& t = f.table;
  MetaT* const meta = static_cast<MetaT*>(f.pool.slot_meta);
  const int64_t slot = t.tables[seq * t.stride + i];
  if (refused) {
    if (unpinned[j * t.width + i]) add_pin(meta, slot, 1, false);
    return;
  }
  t.tables[seq * t.stride + i] = -1;
  if (slot < 0 || !f.discard) return;
  if (Meta<MetaT>::pin(*reinterpret_cast<volatile MetaT*>(meta + slot)) != 0) return;
  const int64_t id = *reinterpret_cast<volatile int64_t*>(f.pool.p2l + slot);
  if (id >= 0 && id < f.pool.num_logical) f.pool.l2p[id] = -1;
  f.pool.p2l[slot] = -1;
  meta[slot] = 0;
}

// A small call by one block.
template <typename MetaT>
__global__ void __launch_bounds__(kCheckThreads) free_small_kernel(const __grid_constant__ FreeArgs f,
                                                                  uint8_t* unpinned) {
  __shared__ int64_t tile[kCheckThreads];
  if (__syncthreads_or(free_refused(f, threadIdx.x, tile))) return;
  const PageTable& t = f.table;
  // a sequence's pages to as many warps as there are for it
  const int warps = kCheckThreads / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = f.count >= warps ? 1 : warps / static_cast<int>(f.count);
  const int teams = warps / team;
  const bool plays = warp < team * teams;
  const int64_t first = warp % team * 32 + lane;
  bool fine = true;
  for (int64_t j = warp / team; plays && j < f.count; j += teams) {
    const int64_t pages = f.lens_before[j] > 0 ? pages_of(f.lens_before[j], t.block_size) : 0;
    for (int64_t i = first; i < pages; i += team * 32) fine &= free_unpin<MetaT>(f, j, i, f.sequences[j], unpinned);
  }
  const bool refused = __syncthreads_or(!fine) != 0;
  for (int64_t j = warp / team; plays && j < f.count; j += teams) {
    const int64_t len = f.lens_before[j], pages = len > 0 ? pages_of(len, t.block_size) : 0;
    for (int64_t i = first; i < pages; i += team * 32) free_page<MetaT>(f, j, i, f.sequences[j], refused, unpinned);
    if (!refused && first == 0 && len > 0) t.lens[f.sequences[j]] = 0;
  }
}

template <typename MetaT>
__global__ void __launch_bounds__(kPageThreads) free_unpin_kernel(const __grid_constant__ FreeArgs f,
                                                                  PageHeader* header, uint8_t* unpinned, int checks) {
  dependent_wait();
  dependent_trigger();
  if (!checks_passed(header, checks)) return;
  const PageTable& t = f.table;
  const int64_t j = blockIdx.x;
  const int64_t seq = f.sequences[j], len = f.lens_before[j];
  const int64_t pages = len > 0 ? pages_of(len, t.block_size) : 0;
  const int64_t base = static_cast<int64_t>(blockIdx.y) * kEntriesPerBlock;
  for (int64_t i = base + threadIdx.x; i < pages && i < base + kEntriesPerBlock; i += kPageThreads)
    if (!free_unpin<MetaT>(f, j, i, seq, unpinned)) header->refused = 1;
}

template <typename MetaT>
__global__ void __launch_bounds__(kPageThreads) free_commit_kernel(const __grid_constant__ FreeArgs f,
                                                                   const PageHeader* header, const uint8_t* unpinned,
                                                                   int checks) {
  dependent_wait();
  if (!checks_passed(header, checks)) return;
  const bool refused = header->refused != 0;
  const PageTable& t = f.table;
  const int64_t j = blockIdx.x;
  const int64_t seq = f.sequences[j], len = f.lens_before[j];
  const int64_t pages = len > 0 ? pages_of(len, t.block_size) : 0;
  const int64_t base = static_cast<int64_t>(blockIdx.y) * kEntriesPerBlock;
  for (int64_t i = base + threadIdx.x; i < pages && i < base + kEntriesPerBlock; i += kPageThreads)
    free_page<MetaT>(f, j, i, seq, refused, unpinned);
  if (!refused && blockIdx.y == 0 && threadIdx.x == 0 && len > 0) t.lens[seq] = 0;
}

// ---------------------------------------------------------------------------
// Compaction
// ---------------------------------------------------------------------------

// Workspace: the header, the live slots of each run of kScanSlots, then the
// slots of holes by rank and of live slots past the last kept one by rank.
struct CompactHeader {
  int64_t live;    // slots
  int64_t kept;    // live slots among the first `live` ones
};

template <typename MetaT>
__device__ __forceinline__ bool slot_live(const PagePool& p, int64_t slot) {
  return p.p2l[slot] >= 0 || Meta<MetaT>::pin(static_cast<const MetaT*>(p.slot_meta)[slot]) != 0;
}

template <typename MetaT>
__global__ void __launch_bounds__(1024) compact_count_kernel(const __grid_constant__ CompactArgs c, int32_t* counts) {
  dependent_trigger();
  int n = 0;
#pragma unroll
  for (int i = 0; i < kScanSlots / 1024; ++i) {
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * kScanSlots + i * 1024 + threadIdx.x;
    n += __syncthreads_count(slot < c.pool.num_slots && slot_live<MetaT>(c.pool, slot));
  }
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// remap of the slots that stay or are dead; -2 - r for the live slot of rank
// r that will move; holes and movers listed by rank.
template <typename MetaT>
__global__ void __launch_bounds__(1024) compact_rank_kernel(const __grid_constant__ CompactArgs c,
                                                            CompactHeader* header, const int32_t* counts, int runs,
                                                            int32_t* holes, int32_t* movers) {
  __shared__ int64_t scan[33];
  __shared__ int small[33];
  dependent_wait();
  dependent_trigger();
  int64_t before = 0, all = 0;
  if (runs == 1) {  // counted here
    for (int64_t slot = threadIdx.x; slot < c.pool.num_slots; slot += 1024) all += slot_live<MetaT>(c.pool, slot) ? 1 : 0;
  } else {
    for (int i = threadIdx.x; i < runs; i += 1024) {
      all += counts[i];
      if (i < static_cast<int>(blockIdx.x)) before += counts[i];
    }
  }
  int64_t rank, live;
  block_excl_scan(before, &rank, scan);
  block_excl_scan(all, &live, scan);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    header->live = live;
    *c.live = live;
    if (live == c.pool.num_slots) header->kept = live;
  }
#pragma unroll 1
  for (int i = 0; i < kScanSlots / 1024; ++i) {
    const int64_t slot = static_cast<int64_t>(blockIdx.x) * kScanSlots + i * 1024 + threadIdx.x;
    const bool in = slot < c.pool.num_slots;
    const bool alive = in && slot_live<MetaT>(c.pool, slot);
    int total;
    const int64_t r = rank + block_excl_scan(alive ? 1 : 0, &total, small);
    rank += total;
    if (!in) continue;
    if (slot == live) header->kept = r;
    if (alive && slot >= live) {
      movers[r] = static_cast<int32_t>(slot);
      c.remap[slot] = -2 - r;
    } else {
      if (!alive && slot < live) holes[slot - r] = static_cast<int32_t>(slot);
      c.remap[slot] = alive ? slot : -1;
    }
  }
}

// Bytes, metadata and page tables: blocks in that order.
template <typename MetaT, typename V>
__global__ void __launch_bounds__(kPageThreads) compact_move_kernel(const __grid_constant__ CompactArgs c,
                                                                    const __grid_constant__ PagedSide cache,
                                                                    int num_planes, int64_t row_bytes,
                                                                    const CompactHeader* header, const int32_t* holes,
                                                                    const int32_t* movers, int copy_blocks,
                                                                    int meta_blocks) {
  dependent_wait();
  const int64_t kept = header->kept, moves = header->live - kept;
  if (static_cast<int>(blockIdx.x) < copy_blocks) {
    const int64_t total = c.table.block_size * row_bytes;
    const int64_t parts = (total + kCopyBytes - 1) / kCopyBytes;
    const int64_t items = moves * num_planes * parts;
    const int64_t warps = static_cast<int64_t>(copy_blocks) * (kPageThreads / 32);
    for (int64_t it = static_cast<int64_t>(blockIdx.x) * (kPageThreads / 32) + (threadIdx.x >> 5); it < items;
         it += warps) {
      const int64_t part = it % parts, rest = it / parts;
      const int64_t plane = rest / moves, k = rest - plane * moves;
      char* const base = reinterpret_cast<char*>(cache.planes[plane]);
      copy_part<V>(base + holes[k] * cache.block_stride, base + movers[kept + k] * cache.block_stride,
                   part * kCopyBytes, total, row_bytes, cache.row_stride);
    }
    return;
  }
  if (static_cast<int>(blockIdx.x) < copy_blocks + meta_blocks) {
    MetaT* const meta = static_cast<MetaT*>(c.pool.slot_meta);
    for (int64_t k = static_cast<int64_t>(blockIdx.x - copy_blocks) * kPageThreads + threadIdx.x; k < moves;
         k += static_cast<int64_t>(meta_blocks) * kPageThreads) {
      const int64_t to = holes[k], from = movers[kept + k];
      c.remap[from] = to;
      const int64_t id = c.pool.p2l[from];
      c.pool.p2l[to] = id;
      c.pool.p2l[from] = -1;
      meta[to] = meta[from];
      meta[from] = 0;
      if (id >= c.pool.num_logical)
        report(c.pool.status, KVCA_ERR_BAD_INDEX, id);
      else if (id >= 0)
        c.pool.l2p[id] = to;
    }
    return;
  }
  const PageTable& t = c.table;
  const int64_t chunks = (t.width + kEntriesPerBlock - 1) / kEntriesPerBlock;
  const int64_t at = blockIdx.x - copy_blocks - meta_blocks;
  const int64_t seq = at / chunks, base = (at - seq * chunks) * kEntriesPerBlock;
  const int64_t len = t.lens[seq];
  int64_t pages = len > 0 ? pages_of(len, t.block_size) : 0;
  if (pages > t.width) {
    if (base == 0 && threadIdx.x == 0) report(c.pool.status, KVCA_ERR_BAD_INDEX, len);
    pages = t.width;
  }
  for (int64_t i = base + threadIdx.x; i < pages && i < base + kEntriesPerBlock; i += kPageThreads) {
    const int64_t slot = t.tables[seq * t.stride + i];
    if (slot < 0) continue;
    if (slot >= c.pool.num_slots) {
      report(c.pool.status, KVCA_ERR_BAD_INDEX, slot);
      continue;
    }
    // a mover's entry turns from its rank into its new slot meanwhile
    const int64_t r = *reinterpret_cast<volatile int64_t*>(c.remap + slot);
    t.tables[seq * t.stride + i] = r <= -2 ? holes[-2 - r - kept] : r;
  }
}

int page_chunks(int64_t width) { return static_cast<int>((width + kEntriesPerBlock - 1) / kEntriesPerBlock); }

// Copy blocks: enough for every item to have a warp, at most eight blocks per SM.
int copy_grid(int64_t items, int sms) {
  const int64_t blocks = (items + kPageThreads / 32 - 1) / (kPageThreads / 32);
  const int64_t most = static_cast<int64_t>(sms > 0 ? sms : 1) * 8;
  return static_cast<int>(blocks < most ? blocks : most);
}

// Calls whose checks, pins and tables one block does in one launch, against
// three (two with a fork's bytes): each launch costs 4-5 us of the host's time
// and 2-3 of the GPU's, a block 1,024 entries each few us.
bool is_small(int64_t count, int64_t width) { return count <= kCheckThreads && count * width <= 8 * 1024; }

template <typename MetaT>
cudaError_t launch_fork_typed(const ForkArgs& f, const PagedSide& cache, int num_planes, int64_t row_bytes, int vec,
                              void* workspace, cudaStream_t stream) {
  PageHeader* const header = static_cast<PageHeader*>(workspace);
  uint8_t* const pinned = static_cast<uint8_t*>(workspace) + sizeof(PageHeader);
  const int checks = static_cast<int>((f.count + kCheckThreads - 1) / kCheckThreads);
  const int chunks = page_chunks(f.table.width);
  const unsigned count = static_cast<unsigned>(f.count);
  const bool small = is_small(f.count, f.table.width);
  if (small)
    fork_small_kernel<MetaT><<<1, kCheckThreads, 0, stream>>>(f, header, pinned);
  else
    fork_check_kernel<MetaT><<<checks, kCheckThreads, 0, stream>>>(f, header);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  if (!small && chunks > 0) {
    e = launch_dependent(fork_pin_kernel<MetaT>, dim3(count, chunks), kPageThreads, 0, stream, f, header, pinned,
                         checks);
    if (e != cudaSuccess) return e;
  }
  const int64_t parts = (f.table.block_size * row_bytes + kCopyBytes - 1) / kCopyBytes;
  const int copies = copy_grid(f.count * num_planes * parts, device_sm_count());
  const unsigned grid =
      static_cast<unsigned>(copies) + (small ? 0u : count * static_cast<unsigned>(chunks > 0 ? chunks : 1));
  auto go = [&](auto kernel) {
    return launch_dependent(kernel, dim3(grid), kPageThreads, 0, stream, f, cache, num_planes, row_bytes,
                            static_cast<const PageHeader*>(header), static_cast<const uint8_t*>(pinned), checks,
                            copies);
  };
  switch (vec) {
    case 16: return go(fork_commit_kernel<MetaT, uint4>);
    case 8: return go(fork_commit_kernel<MetaT, uint2>);
    case 4: return go(fork_commit_kernel<MetaT, uint32_t>);
    case 2: return go(fork_commit_kernel<MetaT, uint16_t>);
    default: return go(fork_commit_kernel<MetaT, uint8_t>);
  }
}

template <typename MetaT>
cudaError_t launch_compact_typed(const CompactArgs& c, const PagedSide& cache, int num_planes, int64_t row_bytes,
                                 int vec, void* workspace, cudaStream_t stream) {
  const int runs = static_cast<int>((c.pool.num_slots + kScanSlots - 1) / kScanSlots);
  CompactHeader* const header = static_cast<CompactHeader*>(workspace);
  int32_t* const counts = reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + 256);
  int32_t* const holes = counts + runs;
  int32_t* const movers = holes + c.pool.num_slots;
  if (runs > 1) {
    compact_count_kernel<MetaT><<<runs, 1024, 0, stream>>>(c, counts);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  // (alone, the ranks wait for the work before this call)
  const cudaError_t e = launch_dependent(compact_rank_kernel<MetaT>, dim3(runs), 1024, 0, stream, c, header,
                                         static_cast<const int32_t*>(counts), runs, holes, movers);
  if (e != cudaSuccess) return e;
  const int sms = device_sm_count();
  const int64_t parts = (c.table.block_size * row_bytes + kCopyBytes - 1) / kCopyBytes;
  const int copies = copy_grid(c.pool.num_slots / 2 * num_planes * parts, sms);
  const int64_t most = (c.pool.num_slots / 2 + kPageThreads - 1) / kPageThreads;
  const int metas = static_cast<int>(most < sms ? most : sms);
  const unsigned grid = static_cast<unsigned>(copies + metas) +
                        static_cast<unsigned>(c.table.num_seqs) * static_cast<unsigned>(page_chunks(c.table.width));
  if (grid == 0) return cudaSuccess;
  auto go = [&](auto kernel) {
    return launch_dependent(kernel, dim3(grid), kPageThreads, 0, stream, c, cache, num_planes, row_bytes,
                            static_cast<const CompactHeader*>(header), static_cast<const int32_t*>(holes),
                            static_cast<const int32_t*>(movers), copies, metas);
  };
  switch (vec) {
    case 16: return go(compact_move_kernel<MetaT, uint4>);
    case 8: return go(compact_move_kernel<MetaT, uint2>);
    case 4: return go(compact_move_kernel<MetaT, uint32_t>);
    case 2: return go(compact_move_kernel<MetaT, uint16_t>);
    default: return go(compact_move_kernel<MetaT, uint8_t>);
  }
}

template <typename MetaT>
cudaError_t launch_free_typed(const FreeArgs& args, void* workspace, cudaStream_t stream) {
  FreeArgs f = args;
  PageHeader* const header = static_cast<PageHeader*>(workspace);
  f.lens_before = reinterpret_cast<int64_t*>(header + 1);
  uint8_t* const unpinned = reinterpret_cast<uint8_t*>(f.lens_before + f.count);
  if (is_small(f.count, f.table.width)) {
    free_small_kernel<MetaT><<<1, kCheckThreads, 0, stream>>>(f, unpinned);
    return cudaGetLastError();
  }
  const int checks = static_cast<int>((f.count + kCheckThreads - 1) / kCheckThreads);
  free_check_kernel<<<checks, kCheckThreads, 0, stream>>>(f, header);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int chunks = page_chunks(f.table.width);
  const dim3 grid(static_cast<unsigned>(f.count), chunks > 0 ? chunks : 1);
  e = launch_dependent(free_unpin_kernel<MetaT>, grid, kPageThreads, 0, stream, f, header, unpinned, checks);
  if (e != cudaSuccess) return e;
  return launch_dependent(free_commit_kernel<MetaT>, grid, kPageThreads, 0, stream, f,
                          static_cast<const PageHeader*>(header), static_cast<const uint8_t*>(unpinned), checks);
}

}  // namespace

size_t fork_workspace(int64_t count, int64_t table_width) {
  return sizeof(PageHeader) + static_cast<size_t>(count) * static_cast<size_t>(table_width);
}

size_t free_workspace(int64_t count, int64_t table_width) {
  return sizeof(PageHeader) + static_cast<size_t>(count) * (sizeof(int64_t) + static_cast<size_t>(table_width));
}

size_t compact_workspace(int64_t num_slots) {
  const int64_t runs = (num_slots + kScanSlots - 1) / kScanSlots;
  return 256 + static_cast<size_t>(runs + 2 * num_slots) * sizeof(int32_t);
}

cudaError_t launch_fork(int meta_bits, const ForkArgs& f, const PagedSide& cache, int num_planes, int64_t row_bytes,
                        int vec, void* workspace, cudaStream_t stream) {
  return meta_bits == 8 ? launch_fork_typed<uint8_t>(f, cache, num_planes, row_bytes, vec, workspace, stream)
                        : launch_fork_typed<uint16_t>(f, cache, num_planes, row_bytes, vec, workspace, stream);
}

cudaError_t launch_free(int meta_bits, const FreeArgs& f, void* workspace, cudaStream_t stream) {
  return meta_bits == 8 ? launch_free_typed<uint8_t>(f, workspace, stream)
                        : launch_free_typed<uint16_t>(f, workspace, stream);
}

cudaError_t launch_compact(int meta_bits, const CompactArgs& c, const PagedSide& cache, int num_planes,
                           int64_t row_bytes, int vec, void* workspace, cudaStream_t stream) {
  return meta_bits == 8 ? launch_compact_typed<uint8_t>(c, cache, num_planes, row_bytes, vec, workspace, stream)
                        : launch_compact_typed<uint16_t>(c, cache, num_planes, row_bytes, vec, workspace, stream);
}

}  // namespace kvca

// Sharing, dropping and moving the pages of a cache's sequences.
//
// A page table row names the slots of a sequence's pages in order; a slot's
// pin count says how many sequences hold it.  All three operators are bound
// by their launches and the dependent reads in them (table entry, then slot
// word) until many pages' bytes move, and then by HBM.  Each is a chain of
// small launches, the later ones programmatic dependents, instead of one
// kernel with grid barriers, because the work of each part is spread over the
// whole GPU differently.

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

// Everything about the call that does not concern single pages.
template <typename MetaT>
__global__ void __launch_bounds__(1024) fork_check_kernel(const __grid_constant__ ForkArgs f, PageHeader* header) {
  dependent_trigger();
  const PageTable& t = f.table;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
  int64_t code = 0, value = 0;
  auto refuse = [&](int64_t c, int64_t v) {
    if (code == 0) {
      code = c;
      value = v;
    }
  };
  if (j < f.count) {
    const int64_t parent = f.parents[j], child = f.children[j];
    if (parent < 0 || parent >= t.num_seqs)
      refuse(KVCA_ERR_BAD_INDEX, parent);
    else if (child < 0 || child >= t.num_seqs)
      refuse(KVCA_ERR_BAD_INDEX, child);
    else {
      const int64_t len = t.lens[parent];
      if (len < 0 || t.lens[child] > 0) refuse(KVCA_ERR_BAD_ARGUMENT, len < 0 ? parent : child);
      if (len > t.width * t.block_size) refuse(KVCA_ERR_BAD_INDEX, len);
      const bool partial = code == 0 && len % t.block_size != 0;
      int64_t fresh = -1, id = -1;
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
      for (int64_t k = 0; k < f.count && code == 0; ++k) {
        if (f.parents[k] == child || (k != j && f.children[k] == child)) refuse(KVCA_ERR_BAD_ARGUMENT, child);
        if (k == j || !partial) continue;
        if (f.fresh_slots[k] != fresh && f.fresh_ids[k] != id) continue;
        // the other one counts if it needs its slot, too
        const int64_t other = f.parents[k];
        if (other >= 0 && other < t.num_seqs && t.lens[other] > 0 && t.lens[other] % t.block_size != 0)
          refuse(KVCA_ERR_BAD_ARGUMENT, f.fresh_slots[k] == fresh ? fresh : id);
      }
    }
  }
  if (code != 0) report(f.pool.status, code, value);
  const int bad = __syncthreads_or(code != 0);
  if (threadIdx.x == 0) {
    header->verdicts[blockIdx.x] = bad;
    if (blockIdx.x == 0) header->refused = 0;
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
  for (int64_t i = base + threadIdx.x; i < full && i < base + kEntriesPerBlock; i += kPageThreads) {
    const int64_t slot = t.tables[parent * t.stride + i];
    bool done = false;
    if (slot >= f.pool.num_slots) {
      report(f.pool.status, KVCA_ERR_BAD_INDEX, slot);
      header->refused = 1;
    } else if (slot >= 0) {
      done = add_pin(static_cast<MetaT*>(f.pool.slot_meta), slot, 1, true);
      if (!done) {
        report(f.pool.status, KVCA_ERR_BAD_ARGUMENT, slot);  // held by nobody, or as often as its field counts
        header->refused = 1;
      }
    }
    pinned[j * t.width + i] = done;
  }
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
  MetaT* const meta = static_cast<MetaT*>(f.pool.slot_meta);
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
  for (int64_t i = base + threadIdx.x; i < full && i < base + kEntriesPerBlock; i += kPageThreads) {
    const int64_t slot = t.tables[parent * t.stride + i];
    if (!refused)
      t.tables[child * t.stride + i] = slot;
    else if (pinned[j * t.width + i])
      add_pin(meta, slot, -1, true);
  }
  if (refused || chunk != 0 || threadIdx.x != 0) return;
  if (len % t.block_size != 0) {
    const int64_t fresh = f.fresh_slots[j], id = f.fresh_ids[j];
    t.tables[child * t.stride + full] = fresh;
    const int64_t old = f.pool.p2l[fresh];
    if (old >= 0) f.pool.l2p[old] = -1;
    f.pool.l2p[id] = fresh;
    f.pool.p2l[fresh] = id;
    meta[fresh] = Meta<MetaT>::pack(1, 1);
  }
  t.lens[child] = len;
}

// ---------------------------------------------------------------------------
// Free
// ---------------------------------------------------------------------------

__global__ void __launch_bounds__(1024) free_check_kernel(const __grid_constant__ FreeArgs f, PageHeader* header) {
  dependent_trigger();
  const PageTable& t = f.table;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x;
  int64_t code = 0, value = 0;
  if (j < f.count) {
    const int64_t seq = f.sequences[j];
    value = seq;
    if (seq < 0 || seq >= t.num_seqs) {
      code = KVCA_ERR_BAD_INDEX;
    } else if (t.lens[seq] > t.width * t.block_size) {
      code = KVCA_ERR_BAD_INDEX;
      value = t.lens[seq];
    } else {
      for (int64_t k = 0; k < j && code == 0; ++k)
        if (f.sequences[k] == seq) code = KVCA_ERR_BAD_ARGUMENT;
    }
  }
  if (code != 0)
    report(f.pool.status, code, value);
  else if (j < f.count)
    f.lens_before[j] = t.lens[f.sequences[j]];
  const int bad = __syncthreads_or(code != 0);
  if (threadIdx.x == 0) {
    header->verdicts[blockIdx.x] = bad;
    if (blockIdx.x == 0) header->refused = 0;
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
  const int64_t seq = f.sequences[j];
  const int64_t len = t.lens[seq];
  const int64_t pages = len > 0 ? pages_of(len, t.block_size) : 0;
  const int64_t base = static_cast<int64_t>(blockIdx.y) * kEntriesPerBlock;
  for (int64_t i = base + threadIdx.x; i < pages && i < base + kEntriesPerBlock; i += kPageThreads) {
    const int64_t slot = t.tables[seq * t.stride + i];
    bool done = false;
    if (slot >= f.pool.num_slots) {
      report(f.pool.status, KVCA_ERR_BAD_INDEX, slot);
      header->refused = 1;
    } else if (slot >= 0) {
      done = add_pin(static_cast<MetaT*>(f.pool.slot_meta), slot, -1, true);
      if (!done) {
        report(f.pool.status, KVCA_ERR_BAD_ARGUMENT, slot);  // held by fewer sequences than name it
        header->refused = 1;
      }
    }
    unpinned[j * t.width + i] = done;
  }
}

// Entries and lengths cleared, and with `discard` the pages that nobody holds
// any more unmapped (by every sequence that held one: the same words); or the
// pins back.
template <typename MetaT>
__global__ void __launch_bounds__(kPageThreads) free_commit_kernel(const __grid_constant__ FreeArgs f,
                                                                   const PageHeader* header, const uint8_t* unpinned,
                                                                   int checks) {
  dependent_wait();
  if (!checks_passed(header, checks)) return;
  const bool refused = header->refused != 0;
  const PageTable& t = f.table;
  MetaT* const meta = static_cast<MetaT*>(f.pool.slot_meta);
  const int64_t j = blockIdx.x;
  const int64_t seq = f.sequences[j];
  const int64_t len = f.lens_before[j];
  const int64_t pages = len > 0 ? pages_of(len, t.block_size) : 0;
  const int64_t base = static_cast<int64_t>(blockIdx.y) * kEntriesPerBlock;
  for (int64_t i = base + threadIdx.x; i < pages && i < base + kEntriesPerBlock; i += kPageThreads) {
    const int64_t slot = t.tables[seq * t.stride + i];
    if (refused) {
      if (unpinned[j * t.width + i]) add_pin(meta, slot, 1, false);
      continue;
    }
    t.tables[seq * t.stride + i] = -1;
    if (slot < 0 || !f.discard) continue;
    if (Meta<MetaT>::pin(*reinterpret_cast<volatile MetaT*>(meta + slot)) != 0) continue;
    const int64_t id = *reinterpret_cast<volatile int64_t*>(f.pool.p2l + slot);
    if (id >= 0 && id < f.pool.num_logical) f.pool.l2p[id] = -1;
    f.pool.p2l[slot] = -1;
    meta[slot] = 0;
  }
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
  for (int i = threadIdx.x; i < runs; i += 1024) {
    all += counts[i];
    if (i < static_cast<int>(blockIdx.x)) before += counts[i];
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

template <typename MetaT>
cudaError_t launch_fork_typed(const ForkArgs& f, const PagedSide& cache, int num_planes, int64_t row_bytes, int vec,
                              void* workspace, cudaStream_t stream) {
  PageHeader* const header = static_cast<PageHeader*>(workspace);
  uint8_t* const pinned = static_cast<uint8_t*>(workspace) + sizeof(PageHeader);
  const int checks = static_cast<int>((f.count + 1023) / 1024);
  fork_check_kernel<MetaT><<<checks, 1024, 0, stream>>>(f, header);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  const int chunks = page_chunks(f.table.width);
  const unsigned count = static_cast<unsigned>(f.count);
  if (chunks > 0) {
    e = launch_dependent(fork_pin_kernel<MetaT>, dim3(count, chunks), kPageThreads, 0, stream, f, header, pinned,
                         checks);
    if (e != cudaSuccess) return e;
  }
  const int64_t parts = (f.table.block_size * row_bytes + kCopyBytes - 1) / kCopyBytes;
  const int copies = copy_grid(f.count * num_planes * parts, device_sm_count());
  const unsigned grid = static_cast<unsigned>(copies) + count * static_cast<unsigned>(chunks > 0 ? chunks : 1);
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
  compact_count_kernel<MetaT><<<runs, 1024, 0, stream>>>(c, counts);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  e = launch_dependent(compact_rank_kernel<MetaT>, dim3(runs), 1024, 0, stream, c, header,
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
  const int checks = static_cast<int>((f.count + 1023) / 1024);
  free_check_kernel<<<checks, 1024, 0, stream>>>(f, header);
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

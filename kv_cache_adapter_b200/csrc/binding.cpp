// C ABI of the adapter hot path (declared in include/kvca.h).
//
// This layer checks host-visible arguments (sizes, null pointers, word
// widths, plane counts), picks the widest vector access that every address
// and stride allows, and hands off to the sm_100a launchers.  It allocates
// nothing and never synchronises the stream.

#include <atomic>
#include <chrono>

#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include "kvca.h"
#include "kvca_launch.h"

namespace {

constexpr int kAbiVersion = 1;

int status_of(cudaError_t e) { return e == cudaSuccess ? KVCA_OK : KVCA_ERR_CUDA; }

bool valid_meta_bits(int bits) { return bits == 8 || bits == 16; }

// Largest power-of-two access width (<= 16) dividing x.
int align_of(uint64_t x) {
  if (x % 16 == 0) return 16;
  if (x % 8 == 0) return 8;
  if (x % 4 == 0) return 4;
  if (x % 2 == 0) return 2;
  return 1;
}

int min_align(int a, uint64_t x) {
  const int b = align_of(x);
  return a < b ? a : b;
}

bool check_paged(const kvca_paged_desc* d, int64_t num_planes, int64_t row_bytes, int* vec) {
  if (d == nullptr || d->plane_ptrs == nullptr) return false;
  if (d->num_blocks < 0 || d->block_size < 1 || d->block_stride < 0 || d->row_stride < 0)
    return false;
  if (d->block_size > 1 && d->row_stride < row_bytes) return false;
  for (int64_t p = 0; p < num_planes; ++p) {
    if (d->plane_ptrs[p] == 0) return false;
    *vec = min_align(*vec, d->plane_ptrs[p]);
  }
  *vec = min_align(*vec, static_cast<uint64_t>(d->block_stride));
  *vec = min_align(*vec, static_cast<uint64_t>(d->row_stride));
  return true;
}

bool check_chunk(const kvca_chunk_desc* d, int* vec) {
  if (d == nullptr || d->base == 0) return false;
  if (d->rows_per_chunk < 1 || d->chunk_stride < 0 || d->row_stride < 0 || d->plane_stride < 0)
    return false;
  *vec = min_align(*vec, d->base);
  *vec = min_align(*vec, static_cast<uint64_t>(d->chunk_stride));
  *vec = min_align(*vec, static_cast<uint64_t>(d->row_stride));
  *vec = min_align(*vec, static_cast<uint64_t>(d->plane_stride));
  return true;
}

void to_side(const kvca_paged_desc* d, int64_t num_planes, kvca::PagedSide* s) {
  memset(s, 0, sizeof(*s));
  for (int64_t p = 0; p < num_planes; ++p) s->planes[p] = d->plane_ptrs[p];
  s->index = d->index;
  s->num_blocks = d->num_blocks;
  s->block_size = d->block_size;
  s->block_stride = d->block_stride;
  s->row_stride = d->row_stride;
}

void to_side(const kvca_chunk_desc* d, kvca::ChunkSide* s) {
  s->base = d->base;
  s->rows_per_chunk = d->rows_per_chunk;
  s->chunk_stride = d->chunk_stride;
  s->row_stride = d->row_stride;
  s->plane_stride = d->plane_stride;
}

bool aligned16(uint64_t x) { return x % 16 == 0; }

// The checked arguments of an attention call as the kernels take them.
int to_attend(const kvca_attend_desc* d, int64_t* d_status, kvca::AttendArgs* a) {
  if (d == nullptr || d->num_seqs < 0 || d->num_blocks < 0 || d->block_size < 1 || d->table_width < 0 ||
      d->table_stride < 0 || d->window < 0 || d->sinks < 0 || d->kv_heads < 1 || d->q_heads < 1 ||
      d->q_heads % d->kv_heads != 0 || d->head_dim < 8 || d->head_dim > 256)
    return KVCA_ERR_BAD_ARGUMENT;
  if (d->query_type != KVCA_TYPE_F16 && d->query_type != KVCA_TYPE_BF16) return KVCA_ERR_BAD_ARGUMENT;
  const bool e4m3 = d->cache_type == KVCA_TYPE_E4M3;
  if (!e4m3 && d->cache_type != d->query_type) return KVCA_ERR_BAD_ARGUMENT;
  if (d->head_dim % (e4m3 ? 16 : 8) != 0) return KVCA_ERR_BAD_ARGUMENT;
  const uint64_t strides[] = {d->key, d->value, static_cast<uint64_t>(d->key_block_stride),
                              static_cast<uint64_t>(d->key_token_stride), static_cast<uint64_t>(d->key_head_stride),
                              static_cast<uint64_t>(d->value_block_stride),
                              static_cast<uint64_t>(d->value_token_stride),
                              static_cast<uint64_t>(d->value_head_stride), d->query,
                              static_cast<uint64_t>(d->query_row_stride),
                              static_cast<uint64_t>(d->query_head_stride), d->out};
  for (uint64_t x : strides)
    if (!aligned16(x)) return KVCA_ERR_BAD_ARGUMENT;
  const int64_t limit = int64_t{1} << 30;
  if (d->table_width > limit / d->block_size || d->num_seqs > limit / d->q_heads || d->q_heads > 65536)
    return KVCA_ERR_SIZE_LIMIT;
  memset(a, 0, sizeof(*a));
  a->key = reinterpret_cast<const char*>(d->key);
  a->value = reinterpret_cast<const char*>(d->value);
  a->key_block = d->key_block_stride;
  a->key_token = d->key_token_stride;
  a->key_head = d->key_head_stride;
  a->value_block = d->value_block_stride;
  a->value_token = d->value_token_stride;
  a->value_head = d->value_head_stride;
  a->num_blocks = d->num_blocks;
  a->block_size = static_cast<int>(d->block_size < limit ? d->block_size : limit);
  a->block_shift = -1;
  for (int b = 0; b < 31; ++b)
    if (a->block_size == 1 << b) a->block_shift = b;
  a->tables = d->block_tables;
  a->table_stride = d->table_stride;
  a->capacity = static_cast<int>(d->table_width * d->block_size);
  a->lens = d->seq_lens;
  a->num_seqs = static_cast<int>(d->num_seqs);
  a->kv_heads = d->kv_heads;
  a->group = d->q_heads / d->kv_heads;
  a->dim = d->head_dim;
  a->scale_log2 = static_cast<float>(static_cast<double>(d->scale) * d->key_scale * 1.4426950408889634);
  a->value_scale = d->value_scale;
  a->window = static_cast<int>(d->window < limit ? d->window : limit);
  a->sinks = static_cast<int>(d->sinks < limit ? d->sinks : limit);
  a->query = reinterpret_cast<const void*>(d->query);
  a->query_row = d->query_row_stride / 2;
  a->query_head = d->query_head_stride / 2;
  a->out = reinterpret_cast<void*>(d->out);
  a->lse = d->lse;
  a->query_type = d->query_type;
  a->cache_type = d->cache_type;
  a->status = d_status;
  // without blocks no row is read, but rows that are not read get an address
  if (d->num_blocks == 0) a->key = a->value = static_cast<const char*>(a->query);
  return KVCA_OK;
}

// Pointers that a call which has work to do cannot go without.
bool attend_pointers_ok(const kvca::AttendArgs& a) {
  return a.lens != nullptr && a.query != nullptr && a.out != nullptr &&
         (a.capacity == 0 || a.num_blocks == 0 ||
          (a.key != nullptr && a.value != nullptr && a.tables != nullptr));
}

bool common_move_args_ok(int64_t num_planes, int64_t num_rows, int64_t row_bytes) {
  return num_planes >= 1 && num_planes <= KVCA_MAX_PLANES && num_rows >= 0 && row_bytes >= 1;
}

// A device-store call whose rows total at most this many bytes runs as one
// single-CTA launch (plan, finish and row copies): its cost is launches and
// dependent round trips, not bandwidth.  Over the host link one CTA moves
// less, so the limit is lower for a pinned store.
constexpr int64_t kSmallStoreBytes = 256 * 1024;
constexpr int64_t kSmallHostStoreBytes = 64 * 1024;

bool small_store_call(int64_t count, int64_t row_bytes, int32_t move_flags) {
  const int64_t limit = (move_flags & KVCA_FLAG_HOST_MEMORY) ? kSmallHostStoreBytes : kSmallStoreBytes;
  return count <= limit / (row_bytes > 0 ? row_bytes : 1);
}

}  // namespace

extern "C" {

int kvca_abi_version(void) { return kAbiVersion; }

int kvca_device_sm_count(void) {
  // looked up once per device: launchers ask on every call
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const bool tracked = dev >= 0 && dev < 64;
  int sms = tracked ? known[dev].load(std::memory_order_relaxed) : 0;
  if (sms > 0) return sms;
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (tracked) known[dev].store(sms, std::memory_order_relaxed);
  return sms;
}

int kvca_inspect_load_requests(int meta_bits, const int64_t* d_l2p, int64_t num_logical,
                               const void* d_slot_meta, int64_t num_slots,
                               const int64_t* d_ids, int64_t count, int64_t* d_cur_out,
                               uint8_t* d_resident_out, int64_t* d_pin_out, void* d_usage_out,
                               int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) || count < 0 || num_logical < 0 || num_slots < 0)
    return KVCA_ERR_BAD_ARGUMENT;
  if (count == 0) return KVCA_OK;
  if (!d_l2p || !d_slot_meta || !d_ids || !d_cur_out || !d_resident_out || !d_pin_out ||
      !d_usage_out)
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_inspect_load(meta_bits, d_l2p, num_logical, d_slot_meta,
                                             num_slots, d_ids, count, d_cur_out, d_resident_out,
                                             d_pin_out, d_usage_out, d_status, stream));
}

int kvca_inspect_save_requests(int meta_bits, const int64_t* d_l2p, int64_t num_logical,
                               const void* d_slot_meta, int64_t num_slots,
                               const int64_t* d_ids, int64_t count, int64_t* d_cur_out,
                               uint8_t* d_existing_out, void* d_usage_out, int64_t* d_status,
                               kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) || count < 0 || num_logical < 0 || num_slots < 0)
    return KVCA_ERR_BAD_ARGUMENT;
  if (count == 0) return KVCA_OK;
  if (!d_l2p || !d_slot_meta || !d_ids || !d_cur_out || !d_existing_out || !d_usage_out)
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_inspect_save(meta_bits, d_l2p, num_logical, d_slot_meta,
                                             num_slots, d_ids, count, d_cur_out, d_existing_out,
                                             d_usage_out, d_status, stream));
}

size_t kvca_pop_scratch_bytes(int64_t num_slots) { return kvca::pop_scratch_bytes(num_slots); }

int kvca_pop_reusable_slots(int meta_bits, int order, void* d_slot_meta, int64_t num_slots,
                            int64_t* d_search_start, const int64_t* d_blocked,
                            int64_t num_blocked, int64_t count, int64_t* d_out,
                            uint32_t* d_scratch_bitmap, int64_t* d_status,
                            kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits)) return KVCA_ERR_BAD_ARGUMENT;
  if (order != KVCA_POP_ORDER_GROUPED && order != KVCA_POP_ORDER_PREFIX)
    return KVCA_ERR_BAD_ARGUMENT;
  if (num_slots <= 0 || count < 0 || num_blocked < 0) return KVCA_ERR_BAD_ARGUMENT;
  if (count == 0) return KVCA_OK;
  if (!d_slot_meta || !d_search_start || !d_out || !d_scratch_bitmap) return KVCA_ERR_BAD_ARGUMENT;
  if (num_blocked > 0 && !d_blocked) return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_pop(meta_bits, order, d_slot_meta, num_slots, d_search_start,
                                    d_blocked, num_blocked, count, d_out, d_scratch_bitmap,
                                    d_status, stream));
}

int64_t kvca_choose_pop_launch_warps(int64_t num_slots) {
  if (num_slots <= 0) return 0;
  return kvca::pop_threads_for(8, num_slots) / 32;
}

int kvca_commit_load_metadata(int meta_bits, int64_t* d_l2p, int64_t num_logical, int64_t* d_p2l,
                              void* d_slot_meta, int64_t num_slots, const int64_t* d_evicted,
                              int64_t num_evicted, const int64_t* d_miss_ids,
                              const int64_t* d_miss_slots, int64_t num_miss,
                              const int64_t* d_hit_slots, const int64_t* d_hit_pins,
                              const void* d_hit_usage, int64_t num_hit, const void* d_miss_usage,
                              int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) || num_evicted < 0 || num_miss < 0 || num_hit < 0 ||
      num_logical < 0 || num_slots < 0)
    return KVCA_ERR_BAD_ARGUMENT;
  if (num_evicted == 0 && num_miss == 0 && num_hit == 0) return KVCA_OK;
  if (!d_l2p || !d_p2l || !d_slot_meta) return KVCA_ERR_BAD_ARGUMENT;
  if (num_evicted > 0 && !d_evicted) return KVCA_ERR_BAD_ARGUMENT;
  if (num_miss > 0 && (!d_miss_ids || !d_miss_slots || !d_miss_usage)) return KVCA_ERR_BAD_ARGUMENT;
  if (num_hit > 0 && (!d_hit_slots || !d_hit_pins || !d_hit_usage)) return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_commit_load(
      meta_bits, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots, d_evicted, num_evicted,
      d_miss_ids, d_miss_slots, num_miss, d_hit_slots, d_hit_pins, d_hit_usage, num_hit,
      d_miss_usage, d_status, stream));
}

int kvca_commit_save_metadata(int meta_bits, int64_t* d_l2p, int64_t num_logical, int64_t* d_p2l,
                              void* d_slot_meta, int64_t num_slots, const int64_t* d_evicted,
                              int64_t num_evicted, const int64_t* d_ids, const int64_t* d_slots,
                              const void* d_final_pins, const void* d_final_usage, int64_t count,
                              int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) || num_evicted < 0 || count < 0 || num_logical < 0 ||
      num_slots < 0)
    return KVCA_ERR_BAD_ARGUMENT;
  if (num_evicted == 0 && count == 0) return KVCA_OK;
  if (!d_l2p || !d_p2l || !d_slot_meta) return KVCA_ERR_BAD_ARGUMENT;
  if (num_evicted > 0 && !d_evicted) return KVCA_ERR_BAD_ARGUMENT;
  if (count > 0 && (!d_ids || !d_slots || !d_final_pins || !d_final_usage))
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_commit_save(meta_bits, d_l2p, num_logical, d_p2l, d_slot_meta,
                                            num_slots, d_evicted, num_evicted, d_ids, d_slots,
                                            d_final_pins, d_final_usage, count, d_status,
                                            stream));
}

int kvca_release_metadata(int meta_bits, const int64_t* d_l2p, int64_t num_logical,
                          void* d_slot_meta, int64_t num_slots, const int64_t* d_ids,
                          int64_t count, int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) || count < 0 || num_logical < 0 || num_slots < 0)
    return KVCA_ERR_BAD_ARGUMENT;
  if (count == 0) return KVCA_OK;
  if (!d_l2p || !d_slot_meta || !d_ids) return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_release(meta_bits, d_l2p, num_logical, d_slot_meta, num_slots,
                                        d_ids, count, d_status, stream));
}

int kvca_clock_stream(int meta_bits, int order, void* d_slot_meta, int64_t num_slots,
                      int64_t* d_search_start, int64_t num_steps, int64_t alloc_per_step,
                      const int64_t* d_reaccess, int64_t reaccess_per_step, int64_t* d_victims,
                      int64_t* d_steps_done, int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits)) return KVCA_ERR_BAD_ARGUMENT;
  if (order != KVCA_POP_ORDER_GROUPED && order != KVCA_POP_ORDER_PREFIX)
    return KVCA_ERR_BAD_ARGUMENT;
  if (num_slots <= 0 || num_steps < 0 || alloc_per_step < 1 || reaccess_per_step < 0 ||
      reaccess_per_step > 8192)
    return KVCA_ERR_BAD_ARGUMENT;
  if (!d_slot_meta || !d_search_start || !d_steps_done) return KVCA_ERR_BAD_ARGUMENT;
  if (num_steps == 0)  // nothing to run: no victims buffer needed
    return status_of(cudaMemsetAsync(d_steps_done, 0, sizeof(int64_t), stream));
  if (!d_victims) return KVCA_ERR_BAD_ARGUMENT;
  if (reaccess_per_step > 0 && !d_reaccess) return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_clock_stream(meta_bits, order, d_slot_meta, num_slots,
                                             d_search_start, num_steps, alloc_per_step,
                                             d_reaccess, reaccess_per_step, d_victims,
                                             d_steps_done, d_status, stream));
}

size_t kvca_clock_stream_scratch_bytes(int64_t num_slots) {
  if (num_slots <= 0) return 0;
  return static_cast<size_t>(num_slots) * 32 + kvca::kClockStreamGridBytes;
}

int kvca_clock_stream_batched(int meta_bits, int order, void* d_slot_meta, int64_t num_slots,
                              int64_t* d_search_start, int64_t num_steps, int64_t alloc_per_step,
                              const int64_t* d_reaccess, int64_t reaccess_per_step,
                              int64_t* d_victims, int64_t* d_steps_done, void* d_scratch,
                              int ctas, int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) || ctas < 0) return KVCA_ERR_BAD_ARGUMENT;
  if (order != KVCA_POP_ORDER_GROUPED && order != KVCA_POP_ORDER_PREFIX)
    return KVCA_ERR_BAD_ARGUMENT;
  const int64_t limit = INT32_MAX - 2;
  if (num_slots <= 0 || num_slots > limit || num_steps < 0 || num_steps > limit ||
      alloc_per_step < 1 || alloc_per_step > limit || reaccess_per_step < 0 ||
      reaccess_per_step > 8192 || num_steps * alloc_per_step > limit)
    return KVCA_ERR_BAD_ARGUMENT;
  if (!d_slot_meta || !d_search_start || !d_steps_done || !d_scratch) return KVCA_ERR_BAD_ARGUMENT;
  if ((reinterpret_cast<uintptr_t>(d_scratch) & 7u) != 0u) return KVCA_ERR_BAD_ARGUMENT;
  if (num_steps == 0)  // nothing to run: no victims buffer needed
    return status_of(cudaMemsetAsync(d_steps_done, 0, sizeof(int64_t), stream));
  if (!d_victims) return KVCA_ERR_BAD_ARGUMENT;
  if (reaccess_per_step > 0 && !d_reaccess) return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_clock_stream_batched(
      meta_bits, order, d_slot_meta, num_slots, d_search_start, num_steps, alloc_per_step,
      d_reaccess, reaccess_per_step, d_victims, d_steps_done,
      reinterpret_cast<unsigned char*>(d_scratch), ctas, d_status, stream));
}

static bool plan_args_ok(int meta_bits, int order, const int64_t* l2p, int64_t num_logical,
                         const int64_t* p2l, const void* meta, int64_t num_slots,
                         const int64_t* search_start, const int64_t* ids, int64_t count,
                         const uint32_t* bitmap, const int64_t* counts) {
  return valid_meta_bits(meta_bits) &&
         (order == KVCA_POP_ORDER_GROUPED || order == KVCA_POP_ORDER_PREFIX) && num_logical > 0 &&
         num_slots > 0 && count > 0 && l2p && p2l && meta && search_start && ids && bitmap && counts;
}

int kvca_plan_load(int meta_bits, int order, const int64_t* d_l2p, int64_t num_logical,
                   const int64_t* d_p2l, void* d_slot_meta, int64_t num_slots,
                   int64_t* d_search_start, const int64_t* d_ids, int64_t count,
                   uint32_t* d_scratch_bitmap, int64_t* d_result, int64_t* d_hit_slots,
                   int64_t* d_hit_pins, void* d_hit_usage, int64_t* d_miss_ids,
                   int64_t* d_victims, int64_t* d_evict_ids, int64_t* d_evict_slots,
                   int64_t* d_counts, int64_t* d_status, kvca_stream_t stream) {
  if (!plan_args_ok(meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots,
                    d_search_start, d_ids, count, d_scratch_bitmap, d_counts) ||
      !d_result || !d_hit_slots || !d_hit_pins || !d_hit_usage || !d_miss_ids || !d_victims ||
      !d_evict_ids || !d_evict_slots)
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_plan_load(
      meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots, d_search_start, d_ids,
      count, d_scratch_bitmap, d_result, d_hit_slots, d_hit_pins, d_hit_usage, d_miss_ids,
      d_victims, d_evict_ids, d_evict_slots, d_counts, d_status, stream));
}

int kvca_plan_save(int meta_bits, int order, const int64_t* d_l2p, int64_t num_logical,
                   const int64_t* d_p2l, void* d_slot_meta, int64_t num_slots,
                   int64_t* d_search_start, const int64_t* d_ids, int64_t count,
                   uint32_t* d_scratch_bitmap, int64_t* d_selected, int64_t* d_move_slots,
                   void* d_final_pins, void* d_final_usage, int64_t* d_allocated,
                   int64_t* d_evict_ids, int64_t* d_evict_slots, int64_t* d_counts,
                   int64_t* d_status, kvca_stream_t stream) {
  if (!plan_args_ok(meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots,
                    d_search_start, d_ids, count, d_scratch_bitmap, d_counts) ||
      !d_selected || !d_move_slots || !d_final_pins || !d_final_usage || !d_allocated || !d_evict_ids ||
      !d_evict_slots)
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_plan_save(
      meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots, d_search_start, d_ids,
      count, d_scratch_bitmap, d_selected, d_move_slots, d_final_pins, d_final_usage, d_allocated,
      d_evict_ids, d_evict_slots, d_counts, d_status, stream));
}

// One-plane paged side: slot s at base + s * row_stride.
static void one_plane(uint64_t base, int64_t rows, int64_t row_stride, const int64_t* index,
                      kvca::PagedSide* out) {
  out->planes[0] = base;
  out->index = index;
  out->num_blocks = rows;
  out->block_size = 1;
  out->block_stride = row_stride;
  out->row_stride = row_stride;
}

static bool store_ok(const kvca_device_store* store, uint64_t actual, int64_t actual_row_stride,
                     int64_t row_bytes) {
  return store && store->storage && store->present && store->scratch && actual &&
         row_bytes > 0 && actual_row_stride >= row_bytes && store->storage_row_stride >= row_bytes &&
         (store->move_flags & ~KVCA_FLAG_HOST_MEMORY) == 0;
}

int kvca_host_memory_usable(const void* p, int64_t bytes) {
  if (p == nullptr || bytes <= 0) return 0;
  const char* last = static_cast<const char*>(p) + (bytes - 1);
  for (const void* q : {p, static_cast<const void*>(last)}) {
    cudaPointerAttributes attr;
    if (cudaPointerGetAttributes(&attr, q) != cudaSuccess) {
      cudaGetLastError();  // clear the sticky-free error of an unknown pointer
      return 0;
    }
    if (attr.type != cudaMemoryTypeHost || attr.devicePointer != q) return 0;
  }
  return 1;
}

// host_counts (session calls): when the call is one launch, that launch
// ends by writing the counts and seq to host_counts (*signalled = true).
static int load_device_store_impl(int meta_bits, int order, int64_t* d_l2p, int64_t num_logical,
                                  int64_t* d_p2l, void* d_slot_meta, int64_t num_slots,
                                  int64_t* d_search_start, const int64_t* d_ids, int64_t count,
                                  uint32_t* d_scratch_bitmap, const kvca_device_store* store,
                                  uint64_t d_actual, int64_t actual_row_stride, int64_t row_bytes,
                                  int64_t* d_work, void* d_work_meta, int64_t* d_result,
                                  int64_t* d_counts, int64_t* d_status, kvca_stream_t stream,
                                  int64_t* host_counts, int64_t seq, bool* signalled) {
  if (!plan_args_ok(meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots,
                    d_search_start, d_ids, count, d_scratch_bitmap, d_counts) ||
      !store_ok(store, d_actual, actual_row_stride, row_bytes) || !d_work || !d_work_meta ||
      !d_result)
    return KVCA_ERR_BAD_ARGUMENT;
  int vec = align_of(static_cast<uint64_t>(row_bytes));
  vec = min_align(vec, d_actual);
  vec = min_align(vec, static_cast<uint64_t>(actual_row_stride));
  vec = min_align(vec, store->storage);
  vec = min_align(vec, static_cast<uint64_t>(store->storage_row_stride));
  if (small_store_call(count, row_bytes, store->move_flags)) {
    const kvca::StoreRowArgs rows{d_actual, actual_row_stride, store->storage, store->storage_row_stride, 0,
                                  row_bytes, vec};
    *signalled = host_counts != nullptr;
    return status_of(kvca::launch_store_load_small(
        meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots, d_search_start, d_ids, count,
        d_scratch_bitmap, store->scratch, store->present, d_work, d_work_meta, d_result, d_counts, d_status,
        rows, stream, host_counts, seq));
  }
  int rc = status_of(kvca::launch_store_load_meta(
      meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots, d_search_start, d_ids,
      count, d_scratch_bitmap, store->scratch, store->present, d_work, d_work_meta, d_result,
      d_counts, d_status, stream));
  if (rc != KVCA_OK) return rc;
  const int64_t k = count;
  const int32_t flags = KVCA_FLAG_SKIP_NEGATIVE | store->move_flags;
  const int64_t* xslot = d_work + 6 * k;
  const int64_t* spill_to = d_work + 7 * k;
  const int64_t* fill_from = d_work + 8 * k;
  const int64_t* gate = d_counts + 7;
  kvca::PagedSide slots, store_out, store_in, slots_in;
  one_plane(d_actual, num_slots, actual_row_stride, xslot, &slots);
  one_plane(store->storage, num_logical, store->storage_row_stride, spill_to, &store_out);
  kvca::ExchangeArgs x{&slots, &store_out, fill_from, gate, k, row_bytes, vec, flags, d_status};
  rc = status_of(kvca::launch_exchange(x, stream));
  if (rc != KVCA_OK) return rc;
  // a miss that this call also spills is filled after every spill (gate set)
  one_plane(store->storage, num_logical, store->storage_row_stride, fill_from, &store_in);
  one_plane(d_actual, num_slots, actual_row_stride, xslot, &slots_in);
  kvca::MoveArgs fill{kvca::MoveKind::kCopyPaged, &store_in, nullptr, &slots_in, nullptr, 1, k,
                      row_bytes, vec, flags, d_status, gate};
  return status_of(kvca::launch_move(fill, stream));
}

int kvca_load_device_store(int meta_bits, int order, int64_t* d_l2p, int64_t num_logical,
                           int64_t* d_p2l, void* d_slot_meta, int64_t num_slots,
                           int64_t* d_search_start, const int64_t* d_ids, int64_t count,
                           uint32_t* d_scratch_bitmap, const kvca_device_store* store,
                           uint64_t d_actual, int64_t actual_row_stride, int64_t row_bytes,
                           int64_t* d_work, void* d_work_meta, int64_t* d_result,
                           int64_t* d_counts, int64_t* d_status, kvca_stream_t stream) {
  bool signalled = false;
  return load_device_store_impl(meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots,
                                d_search_start, d_ids, count, d_scratch_bitmap, store, d_actual,
                                actual_row_stride, row_bytes, d_work, d_work_meta, d_result, d_counts, d_status,
                                stream, nullptr, 0, &signalled);
}

static int save_device_store_impl(int meta_bits, int order, int64_t* d_l2p, int64_t num_logical,
                                  int64_t* d_p2l, void* d_slot_meta, int64_t num_slots,
                                  int64_t* d_search_start, const int64_t* d_ids, int64_t count,
                                  uint32_t* d_scratch_bitmap, const kvca_device_store* store,
                                  uint64_t d_actual, int64_t actual_row_stride, int64_t row_bytes,
                                  uint64_t d_block_data, int64_t* d_work, void* d_work_meta,
                                  int64_t* d_counts, int64_t* d_status, kvca_stream_t stream,
                                  int64_t* host_counts, int64_t seq, bool* signalled) {
  if (!plan_args_ok(meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots,
                    d_search_start, d_ids, count, d_scratch_bitmap, d_counts) ||
      !store_ok(store, d_actual, actual_row_stride, row_bytes) || !d_block_data || !d_work ||
      !d_work_meta)
    return KVCA_ERR_BAD_ARGUMENT;
  int vec = align_of(static_cast<uint64_t>(row_bytes));
  vec = min_align(vec, d_actual);
  vec = min_align(vec, static_cast<uint64_t>(actual_row_stride));
  vec = min_align(vec, store->storage);
  vec = min_align(vec, static_cast<uint64_t>(store->storage_row_stride));
  vec = min_align(vec, d_block_data);
  if (small_store_call(count, row_bytes, store->move_flags)) {
    const kvca::StoreRowArgs rows{d_actual, actual_row_stride, store->storage, store->storage_row_stride,
                                  d_block_data, row_bytes, vec};
    *signalled = host_counts != nullptr;
    return status_of(kvca::launch_store_save_small(
        meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots, d_search_start, d_ids, count,
        d_scratch_bitmap, store->scratch, store->present, d_work, d_work_meta, d_counts, d_status, rows,
        stream, host_counts, seq));
  }
  int rc = status_of(kvca::launch_store_save_meta(
      meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots, d_search_start, d_ids,
      count, d_scratch_bitmap, store->scratch, store->present, d_work, d_work_meta, d_counts,
      d_status, stream));
  if (rc != KVCA_OK) return rc;
  const int64_t k = count;
  kvca::PagedSide actual_evicted, store_evicted, actual_selected;
  one_plane(d_actual, num_slots, actual_row_stride, d_work + 3 * k, &actual_evicted);
  one_plane(store->storage, num_logical, store->storage_row_stride, d_work + 2 * k, &store_evicted);
  one_plane(d_actual, num_slots, actual_row_stride, d_work + 4 * k, &actual_selected);
  kvca::MoveArgs spill{kvca::MoveKind::kCopyPaged, &actual_evicted, nullptr, &store_evicted,
                       nullptr, 1, k, row_bytes, vec, KVCA_FLAG_SKIP_NEGATIVE | store->move_flags,
                       d_status};
  rc = status_of(kvca::launch_move(spill, stream));
  if (rc != KVCA_OK) return rc;
  kvca::ChunkSide data;
  data.base = d_block_data;
  data.rows_per_chunk = k;
  data.chunk_stride = k * row_bytes;
  data.row_stride = row_bytes;
  data.plane_stride = k * row_bytes;
  kvca::MoveArgs scatter{kvca::MoveKind::kScatter, nullptr, &data, &actual_selected, nullptr, 1,
                         k, row_bytes, vec, KVCA_FLAG_SKIP_NEGATIVE, d_status};
  return status_of(kvca::launch_move(scatter, stream));
}

int kvca_save_device_store(int meta_bits, int order, int64_t* d_l2p, int64_t num_logical,
                           int64_t* d_p2l, void* d_slot_meta, int64_t num_slots,
                           int64_t* d_search_start, const int64_t* d_ids, int64_t count,
                           uint32_t* d_scratch_bitmap, const kvca_device_store* store,
                           uint64_t d_actual, int64_t actual_row_stride, int64_t row_bytes,
                           uint64_t d_block_data, int64_t* d_work, void* d_work_meta,
                           int64_t* d_counts, int64_t* d_status, kvca_stream_t stream) {
  bool signalled = false;
  return save_device_store_impl(meta_bits, order, d_l2p, num_logical, d_p2l, d_slot_meta, num_slots,
                                d_search_start, d_ids, count, d_scratch_bitmap, store, d_actual,
                                actual_row_stride, row_bytes, d_block_data, d_work, d_work_meta, d_counts,
                                d_status, stream, nullptr, 0, &signalled);
}

// Ends a session call: when its one launch signals the host, waits for the
// sequence number in host memory (bounded; after about a second the stream's
// own synchronisation decides); otherwise copies the counts to the host and
// waits for the stream.  Either way the call returns with its work done.
static int session_finish(kvca_adapter_session* s, int rc, bool signalled) {
  if (rc != KVCA_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(s->stream);
  if (signalled) {
    volatile int64_t* done = s->counts_host + 8;
    const auto t0 = std::chrono::steady_clock::now();
    for (uint32_t spins = 0;; ++spins) {
      if (*done == s->sequence) return KVCA_OK;
      if ((spins & 4095u) == 4095u && std::chrono::steady_clock::now() - t0 > std::chrono::seconds(1)) break;
    }
    if (cudaStreamSynchronize(st) != cudaSuccess) return KVCA_ERR_CUDA;
    return *done == s->sequence ? KVCA_OK : KVCA_ERR_CUDA;
  }
  if (cudaMemcpyAsync(s->counts_host, s->counts, 8 * sizeof(int64_t), cudaMemcpyDeviceToHost, st) !=
          cudaSuccess ||
      cudaStreamSynchronize(st) != cudaSuccess)
    return KVCA_ERR_CUDA;
  return KVCA_OK;
}

int kvca_session_load(kvca_adapter_session* s, const int64_t* d_ids, int64_t count, int64_t* d_result) {
  if (!s || !s->counts_host || count < 0 || count > s->work_ids) return KVCA_ERR_BAD_ARGUMENT;
  bool signalled = false;
  ++s->sequence;
  const int rc = load_device_store_impl(
      s->meta_bits, s->order, s->l2p, s->num_logical, s->p2l, s->slot_meta, s->num_slots, s->search_start, d_ids,
      count, s->scratch_bitmap, &s->store, s->actual, s->actual_row_stride, s->row_bytes, s->work, s->work_meta,
      d_result, s->counts, s->status, s->stream, s->counts_host, s->sequence, &signalled);
  return session_finish(s, rc, signalled);
}

int kvca_session_save(kvca_adapter_session* s, const int64_t* d_ids, int64_t count, uint64_t d_block_data) {
  if (!s || !s->counts_host || count < 0 || count > s->work_ids) return KVCA_ERR_BAD_ARGUMENT;
  bool signalled = false;
  ++s->sequence;
  const int rc = save_device_store_impl(
      s->meta_bits, s->order, s->l2p, s->num_logical, s->p2l, s->slot_meta, s->num_slots, s->search_start, d_ids,
      count, s->scratch_bitmap, &s->store, s->actual, s->actual_row_stride, s->row_bytes, d_block_data, s->work,
      s->work_meta, s->counts, s->status, s->stream, s->counts_host, s->sequence, &signalled);
  return session_finish(s, rc, signalled);
}

int kvca_exchange(const kvca_paged_desc* slots, const kvca_paged_desc* store,
                  const int64_t* d_fill_rows, int64_t num_rows, int64_t row_bytes, int32_t flags,
                  int64_t* d_status, kvca_stream_t stream) {
  if (!common_move_args_ok(1, num_rows, row_bytes)) return KVCA_ERR_BAD_ARGUMENT;
  if (num_rows == 0) return KVCA_OK;
  if (slots == nullptr || store == nullptr || slots->index == nullptr || store->index == nullptr ||
      d_fill_rows == nullptr || slots->block_size != 1 || store->block_size != 1)
    return KVCA_ERR_BAD_ARGUMENT;
  int vec = align_of(static_cast<uint64_t>(row_bytes));
  if (!check_paged(slots, 1, row_bytes, &vec) || !check_paged(store, 1, row_bytes, &vec))
    return KVCA_ERR_BAD_ARGUMENT;
  kvca::PagedSide a, st;
  to_side(slots, 1, &a);
  to_side(store, 1, &st);
  kvca::ExchangeArgs x{&a, &st, d_fill_rows, nullptr, num_rows, row_bytes, vec, flags, d_status};
  return status_of(kvca::launch_exchange(x, stream));
}

int kvca_append_step(int meta_bits, int order, void* d_slot_meta, int64_t num_slots,
                     int64_t* d_search_start, int64_t* d_l2p, int64_t num_logical, int64_t* d_p2l,
                     const int64_t* d_need, int64_t num_need, int64_t* d_cur_block,
                     int64_t* d_cur_logical, int64_t* d_pos, int64_t num_seqs, int64_t block_size,
                     int64_t* d_next_logical, int64_t* d_victims, int64_t* d_slot_mapping,
                     uint32_t* d_scratch_bitmap, int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) ||
      (order != KVCA_POP_ORDER_GROUPED && order != KVCA_POP_ORDER_PREFIX) || num_slots <= 0 ||
      num_logical <= 0 || num_seqs <= 0 || block_size <= 0 || num_need < 0 ||
      num_need > num_seqs || !d_slot_meta || !d_search_start || !d_l2p || !d_p2l ||
      !d_cur_block || !d_cur_logical || !d_pos || !d_next_logical || !d_slot_mapping ||
      !d_scratch_bitmap || (num_need > 0 && (!d_need || !d_victims)))
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_append_step(
      meta_bits, order, d_slot_meta, num_slots, d_search_start, d_l2p, num_logical, d_p2l, d_need,
      num_need, d_cur_block, d_cur_logical, d_pos, num_seqs, block_size, d_next_logical,
      d_scratch_bitmap, d_victims, d_slot_mapping, d_status, stream));
}

int kvca_append_steps(int meta_bits, int order, void* d_slot_meta, int64_t num_slots,
                      int64_t* d_search_start, int64_t* d_l2p, int64_t num_logical, int64_t* d_p2l,
                      const int64_t* d_need, const int64_t* d_need_offsets, int64_t num_need,
                      int64_t num_steps, int64_t* d_cur_block, int64_t* d_cur_logical,
                      int64_t* d_pos, int64_t num_seqs, int64_t block_size,
                      int64_t* d_next_logical, int64_t* d_victims, int64_t* d_slot_mapping,
                      int64_t* d_status, kvca_stream_t stream) {
  if (!valid_meta_bits(meta_bits) ||
      (order != KVCA_POP_ORDER_GROUPED && order != KVCA_POP_ORDER_PREFIX) || num_slots <= 0 ||
      num_logical <= 0 || num_seqs <= 0 || block_size <= 0 || num_need < 0 || num_steps < 0 ||
      !d_slot_meta || !d_search_start || !d_l2p || !d_p2l || !d_cur_block || !d_cur_logical ||
      !d_pos || !d_next_logical || !d_status || (num_steps > 0 && (!d_need_offsets || !d_slot_mapping)) ||
      (num_need > 0 && (!d_need || !d_victims)))
    return KVCA_ERR_BAD_ARGUMENT;
  if (num_steps == 0) return KVCA_OK;
  return status_of(kvca::launch_append_steps(
      meta_bits, order, d_slot_meta, num_slots, d_search_start, d_l2p, num_logical, d_p2l, d_need,
      d_need_offsets, num_need, num_steps, d_cur_block, d_cur_logical, d_pos, num_seqs, block_size,
      d_next_logical, d_victims, d_slot_mapping, d_status, stream));
}

int kvca_wait_selftest(const uint32_t* d_flag, uint32_t from, int64_t* d_status, kvca_stream_t stream) {
  if (!d_flag || !d_status) return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_wait_selftest(d_flag, from, d_status, stream));
}

int kvca_gather(const kvca_paged_desc* src, const kvca_chunk_desc* dst, int64_t num_planes,
                int64_t num_rows, int64_t row_bytes, int32_t flags, int64_t* d_status,
                kvca_stream_t stream) {
  if (!common_move_args_ok(num_planes, num_rows, row_bytes)) return KVCA_ERR_BAD_ARGUMENT;
  if (num_rows == 0) return KVCA_OK;
  int vec = align_of(static_cast<uint64_t>(row_bytes));
  if (!check_paged(src, num_planes, row_bytes, &vec) || !check_chunk(dst, &vec))
    return KVCA_ERR_BAD_ARGUMENT;
  kvca::PagedSide sp;
  kvca::ChunkSide dc;
  to_side(src, num_planes, &sp);
  to_side(dst, &dc);
  kvca::MoveArgs a{kvca::MoveKind::kGather, &sp, nullptr, nullptr, &dc, num_planes, num_rows,
                   row_bytes, vec, flags, d_status};
  return status_of(kvca::launch_move(a, stream));
}

int kvca_scatter(const kvca_chunk_desc* src, const kvca_paged_desc* dst, int64_t num_planes,
                 int64_t num_rows, int64_t row_bytes, int32_t flags, int64_t* d_status,
                 kvca_stream_t stream) {
  if (!common_move_args_ok(num_planes, num_rows, row_bytes)) return KVCA_ERR_BAD_ARGUMENT;
  if (num_rows == 0) return KVCA_OK;
  int vec = align_of(static_cast<uint64_t>(row_bytes));
  if (!check_chunk(src, &vec) || !check_paged(dst, num_planes, row_bytes, &vec))
    return KVCA_ERR_BAD_ARGUMENT;
  kvca::ChunkSide sc;
  kvca::PagedSide dp;
  to_side(src, &sc);
  to_side(dst, num_planes, &dp);
  kvca::MoveArgs a{kvca::MoveKind::kScatter, nullptr, &sc, &dp, nullptr, num_planes, num_rows,
                   row_bytes, vec, flags, d_status};
  return status_of(kvca::launch_move(a, stream));
}

int kvca_scatter_gather(const kvca_chunk_desc* s_src, const kvca_paged_desc* s_dst, int64_t s_planes,
                        int64_t s_rows, int64_t s_row_bytes, const kvca_paged_desc* g_src,
                        const kvca_chunk_desc* g_dst, int64_t g_planes, int64_t g_rows,
                        int64_t g_row_bytes, int32_t s_flags, int32_t g_flags, int64_t* d_status,
                        kvca_stream_t stream) {
  if (!common_move_args_ok(s_planes, s_rows, s_row_bytes) || !common_move_args_ok(g_planes, g_rows, g_row_bytes))
    return KVCA_ERR_BAD_ARGUMENT;
  kvca::ChunkSide sc{}, gc{};
  kvca::PagedSide sp{}, gp{};
  int s_vec = align_of(static_cast<uint64_t>(s_row_bytes));
  int g_vec = align_of(static_cast<uint64_t>(g_row_bytes));
  if (s_rows > 0) {
    if (!check_chunk(s_src, &s_vec) || !check_paged(s_dst, s_planes, s_row_bytes, &s_vec))
      return KVCA_ERR_BAD_ARGUMENT;
    to_side(s_src, &sc);
    to_side(s_dst, s_planes, &sp);
  }
  if (g_rows > 0) {
    if (!check_paged(g_src, g_planes, g_row_bytes, &g_vec) || !check_chunk(g_dst, &g_vec))
      return KVCA_ERR_BAD_ARGUMENT;
    to_side(g_src, g_planes, &gp);
    to_side(g_dst, &gc);
  }
  if (s_rows == 0 && g_rows == 0) return KVCA_OK;
  kvca::MoveArgs s{kvca::MoveKind::kScatter, nullptr, &sc, &sp, nullptr, s_planes, s_rows,
                   s_row_bytes, s_vec, s_flags, d_status};
  kvca::MoveArgs g{kvca::MoveKind::kGather, &gp, nullptr, nullptr, &gc, g_planes, g_rows,
                   g_row_bytes, g_vec, g_flags, d_status};
  return status_of(kvca::launch_scatter_gather(s, g, stream));
}

int64_t kvca_move_cycle_scratch_bytes(int64_t num_blocks) {
  if (num_blocks < 0) return -1;
  return static_cast<int64_t>(kvca::move_cycle_scratch_bytes(num_blocks));
}

int kvca_move_cycle(const kvca_chunk_desc* tokens, const kvca_paged_desc* token_dst, int64_t token_row_bytes,
                    const kvca_paged_desc* block_src, int64_t num_victims, const kvca_chunk_desc* spill,
                    int64_t block_row_bytes, int64_t num_planes, const int64_t* d_offsets, int64_t num_steps,
                    int64_t num_seqs, int64_t spill_rows, int32_t flags, void* d_scratch, int64_t* d_status,
                    kvca_stream_t stream) {
  if (!common_move_args_ok(num_planes, num_seqs, token_row_bytes) || block_row_bytes < 1 || num_seqs < 1 ||
      num_steps < 1 || num_steps > kvca::kMoveCycleMaxSteps || spill_rows < 0 || num_victims < 0 ||
      d_offsets == nullptr || d_scratch == nullptr || d_status == nullptr)
    return KVCA_ERR_BAD_ARGUMENT;
  int vec = 16;
  vec = min_align(vec, static_cast<uint64_t>(token_row_bytes));
  vec = min_align(vec, static_cast<uint64_t>(block_row_bytes));
  if (!check_chunk(tokens, &vec) || !check_chunk(spill, &vec) ||
      !check_paged(token_dst, num_planes, token_row_bytes, &vec) ||
      !check_paged(block_src, num_planes, block_row_bytes, &vec) || vec != 16)
    return KVCA_ERR_BAD_ARGUMENT;
  if (token_dst->index == nullptr || (num_victims > 0 && block_src->index == nullptr) ||
      block_src->block_size != 1 || token_dst->num_blocks != block_src->num_blocks ||
      token_dst->block_stride != block_src->block_stride || block_row_bytes > block_src->block_stride ||
      (token_dst->block_size - 1) * token_dst->row_stride + token_row_bytes > token_dst->block_stride)
    return KVCA_ERR_BAD_ARGUMENT;
  for (int64_t p = 0; p < num_planes; ++p)
    if (token_dst->plane_ptrs[p] != block_src->plane_ptrs[p]) return KVCA_ERR_BAD_ARGUMENT;
  // item numbers and per-item vector counts stay below 2^31
  const int64_t s_group = kvca::move_cycle_group(token_row_bytes, num_planes);
  const int64_t g_group = kvca::move_cycle_group(block_row_bytes, num_planes);
  const int64_t items = num_steps * num_seqs * ((num_planes + s_group - 1) / s_group) *
                            kvca::move_cycle_segments(token_row_bytes) +
                        spill_rows * ((num_planes + g_group - 1) / g_group) * kvca::move_cycle_segments(block_row_bytes);
  if (num_seqs > (int64_t{1} << 26) || spill_rows > (int64_t{1} << 26) || num_victims > (int64_t{1} << 40) ||
      items >= (int64_t{1} << 31) ||
      s_group * (token_row_bytes / 16) >= (int64_t{1} << 31) || g_group * (block_row_bytes / 16) >= (int64_t{1} << 31))
    return KVCA_ERR_SIZE_LIMIT;
  kvca::PagedSide cache;
  kvca::ChunkSide src, dst;
  to_side(token_dst, num_planes, &cache);
  to_side(tokens, &src);
  to_side(spill, &dst);
  kvca::CycleArgs a{&cache, block_src->index, num_victims, d_offsets, &src, &dst, num_planes, num_steps,
                    num_seqs, spill_rows, token_row_bytes, block_row_bytes, flags,
                    static_cast<unsigned char*>(d_scratch), d_status};
  return status_of(kvca::launch_move_cycle(a, stream));
}

namespace {

int to_pages(const kvca_page_pool* p, int64_t* d_status, kvca::PagePool* pool, kvca::PageTable* table) {
  if (p == nullptr || !valid_meta_bits(p->meta_bits) || p->num_slots < 0 || p->num_logical < 0 || p->table_width < 0 ||
      p->table_stride < 0 || p->num_seqs < 0 || p->block_size < 1 ||
      (p->num_seqs > 1 && p->table_stride < p->table_width))
    return KVCA_ERR_BAD_ARGUMENT;
  if (p->num_slots >= (int64_t{1} << 31) || p->table_width > (int64_t{1} << 25) || p->block_size > (int64_t{1} << 30) ||
      p->num_seqs >= (int64_t{1} << 31))
    return KVCA_ERR_SIZE_LIMIT;
  *pool = kvca::PagePool{p->slot_meta, p->num_slots, p->l2p, p->num_logical, p->p2l, d_status};
  *table = kvca::PageTable{p->block_tables, p->table_stride, p->table_width, p->seq_lens, p->num_seqs, p->block_size};
  return KVCA_OK;
}

bool page_pointers_ok(const kvca::PagePool& pool, const kvca::PageTable& t) {
  return (pool.num_slots == 0 || (pool.slot_meta != nullptr && pool.p2l != nullptr)) &&
         (pool.num_logical == 0 || pool.l2p != nullptr) &&
         (t.num_seqs == 0 || (t.lens != nullptr && (t.width == 0 || t.tables != nullptr)));
}

// The cache side of a page operator: whole blocks of block_size token rows.
bool check_pages(const kvca_paged_desc* d, const kvca_page_pool* p, int64_t num_planes, int64_t row_bytes, int* vec) {
  if (num_planes < 1 || num_planes > KVCA_MAX_PLANES || row_bytes < 1) return false;
  *vec = align_of(static_cast<uint64_t>(row_bytes));
  return check_paged(d, num_planes, row_bytes, vec) && d->num_blocks == p->num_slots &&
         d->block_size == p->block_size && (d->block_size == 1 || d->row_stride >= row_bytes) &&
         (d->num_blocks <= 1 || d->block_stride >= (d->block_size - 1) * d->row_stride + row_bytes);
}

}  // namespace

size_t kvca_fork_workspace_bytes(int64_t count, int64_t table_width) {
  return count < 0 || table_width < 0 ? 0 : kvca::fork_workspace(count, table_width);
}

size_t kvca_free_workspace_bytes(int64_t count, int64_t table_width) {
  return count < 0 || table_width < 0 ? 0 : kvca::free_workspace(count, table_width);
}

size_t kvca_compact_workspace_bytes(int64_t num_slots) { return num_slots < 0 ? 0 : kvca::compact_workspace(num_slots); }

int kvca_fork_sequences(const kvca_page_pool* pool, const int64_t* d_parents, const int64_t* d_children,
                        const int64_t* d_fresh_slots, const int64_t* d_fresh_ids, int64_t count,
                        const kvca_paged_desc* cache, int64_t num_planes, int64_t row_bytes, void* d_workspace,
                        int64_t workspace_bytes, int64_t* d_status, kvca_stream_t stream) {
  kvca::ForkArgs f;
  const int rc = to_pages(pool, d_status, &f.pool, &f.table);
  if (rc != KVCA_OK) return rc;
  int vec = 16;
  if (count < 0 || !check_pages(cache, pool, num_planes, row_bytes, &vec)) return KVCA_ERR_BAD_ARGUMENT;
  if (count == 0) return KVCA_OK;
  if (count > kvca::kPageOpMaxSequences || count * pool->table_width > (int64_t{1} << 38)) return KVCA_ERR_SIZE_LIMIT;
  if (!page_pointers_ok(f.pool, f.table) || !d_parents || !d_children || !d_fresh_slots || !d_fresh_ids || !d_status ||
      !d_workspace || !aligned16(reinterpret_cast<uint64_t>(d_workspace)) ||
      workspace_bytes < static_cast<int64_t>(kvca::fork_workspace(count, pool->table_width)))
    return KVCA_ERR_BAD_ARGUMENT;
  f.parents = d_parents;
  f.children = d_children;
  f.fresh_slots = d_fresh_slots;
  f.fresh_ids = d_fresh_ids;
  f.count = count;
  kvca::PagedSide side;
  to_side(cache, num_planes, &side);
  return status_of(kvca::launch_fork(pool->meta_bits, f, side, static_cast<int>(num_planes), row_bytes, vec,
                                     d_workspace, stream));
}

int kvca_free_sequences(const kvca_page_pool* pool, const int64_t* d_sequences, int64_t count, int32_t discard,
                        void* d_workspace, int64_t workspace_bytes, int64_t* d_status, kvca_stream_t stream) {
  kvca::FreeArgs f;
  const int rc = to_pages(pool, d_status, &f.pool, &f.table);
  if (rc != KVCA_OK) return rc;
  if (count < 0) return KVCA_ERR_BAD_ARGUMENT;
  if (count == 0) return KVCA_OK;
  if (count > kvca::kPageOpMaxSequences || count * pool->table_width > (int64_t{1} << 38)) return KVCA_ERR_SIZE_LIMIT;
  if (!page_pointers_ok(f.pool, f.table) || !d_sequences || !d_status || !d_workspace ||
      !aligned16(reinterpret_cast<uint64_t>(d_workspace)) ||
      workspace_bytes < static_cast<int64_t>(kvca::free_workspace(count, pool->table_width)))
    return KVCA_ERR_BAD_ARGUMENT;
  f.sequences = d_sequences;
  f.count = count;
  f.discard = discard != 0;
  f.lens_before = nullptr;
  return status_of(kvca::launch_free(pool->meta_bits, f, d_workspace, stream));
}

int kvca_compact_pages(const kvca_page_pool* pool, const kvca_paged_desc* cache, int64_t num_planes,
                       int64_t row_bytes, int64_t* d_remap, int64_t* d_live, void* d_workspace,
                       int64_t workspace_bytes, int64_t* d_status, kvca_stream_t stream) {
  kvca::CompactArgs c;
  const int rc = to_pages(pool, d_status, &c.pool, &c.table);
  if (rc != KVCA_OK) return rc;
  int vec = 16;
  if (!check_pages(cache, pool, num_planes, row_bytes, &vec)) return KVCA_ERR_BAD_ARGUMENT;
  if (pool->num_slots == 0) return KVCA_OK;
  if (pool->num_seqs * ((pool->table_width + 1023) / 1024) > (int64_t{1} << 30)) return KVCA_ERR_SIZE_LIMIT;
  if (!page_pointers_ok(c.pool, c.table) || !d_remap || !d_live || !d_status || !d_workspace ||
      !aligned16(reinterpret_cast<uint64_t>(d_workspace)) ||
      workspace_bytes < static_cast<int64_t>(kvca::compact_workspace(pool->num_slots)))
    return KVCA_ERR_BAD_ARGUMENT;
  c.remap = d_remap;
  c.live = d_live;
  kvca::PagedSide side;
  to_side(cache, num_planes, &side);
  return status_of(kvca::launch_compact(pool->meta_bits, c, side, static_cast<int>(num_planes), row_bytes, vec,
                                        d_workspace, stream));
}

int64_t kvca_attend_step_workspace_bytes(const kvca_attend_desc* desc) {
  kvca::AttendArgs a;
  if (to_attend(desc, nullptr, &a) != KVCA_OK) return -1;
  return static_cast<int64_t>(kvca::attend_step_workspace(a, kvca_device_sm_count()));
}

uint64_t kvca_stream_id(kvca_stream_t stream) {
  unsigned long long id = 0;
  return cudaStreamGetId(stream, &id) == cudaSuccess ? id : ~uint64_t{0};
}

int64_t kvca_attend_step_counters(void) {
  return static_cast<int64_t>(kvca_device_sm_count()) * kvca::kStepMaxWarps;
}

int kvca_attend_step(const kvca_attend_desc* desc, void* d_workspace, int64_t workspace_bytes, uint32_t* d_counters,
                     int64_t* d_status, kvca_stream_t stream) {
  kvca::AttendArgs a;
  const int rc = to_attend(desc, d_status, &a);
  if (rc != KVCA_OK) return rc;
  if (a.num_seqs == 0) return KVCA_OK;
  if (!attend_pointers_ok(a)) return KVCA_ERR_BAD_ARGUMENT;
  const int sms = kvca_device_sm_count();
  if (sms < 1) return KVCA_ERR_CUDA;
  if (d_workspace == nullptr || !aligned16(reinterpret_cast<uint64_t>(d_workspace)) || d_counters == nullptr ||
      workspace_bytes < static_cast<int64_t>(kvca::attend_step_workspace(a, sms)))
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_attend_step(a, d_workspace, d_counters, sms, stream));
}

namespace {

std::atomic<int64_t> attend_wait_limit{2000000000};

int to_chunk(const kvca_attend_desc* desc, int64_t num_rows, int64_t* d_status, kvca::AttendArgs* a) {
  const int rc = to_attend(desc, d_status, a);
  if (rc != KVCA_OK) return rc;
  if (num_rows < 0 || a->dim > kvca::kChunkMaxDim) return KVCA_ERR_BAD_ARGUMENT;
  if (num_rows > (int64_t{1} << 30) / desc->q_heads) return KVCA_ERR_SIZE_LIMIT;
  return KVCA_OK;
}

}  // namespace

int64_t kvca_attend_wait_limit(int64_t nanoseconds) {
  return nanoseconds < 0 ? attend_wait_limit.load() : attend_wait_limit.exchange(nanoseconds);
}

int64_t kvca_attend_chunk_workspace_bytes(const kvca_attend_desc* desc, int64_t num_rows) {
  kvca::AttendArgs a;
  if (to_chunk(desc, num_rows, nullptr, &a) != KVCA_OK) return -1;
  return static_cast<int64_t>(kvca::attend_chunk_workspace(a, num_rows, kvca_device_sm_count()));
}

int kvca_attend_chunk(const kvca_attend_desc* desc, const int64_t* d_query_offsets, int64_t num_rows,
                      void* d_workspace, int64_t workspace_bytes, int64_t* d_status, kvca_stream_t stream) {
  kvca::AttendArgs a;
  const int rc = to_chunk(desc, num_rows, d_status, &a);
  if (rc != KVCA_OK) return rc;
  if (a.num_seqs == 0 || num_rows == 0) return KVCA_OK;
  if (!attend_pointers_ok(a) || d_query_offsets == nullptr) return KVCA_ERR_BAD_ARGUMENT;
  const int sms = kvca_device_sm_count();
  if (sms < 1) return KVCA_ERR_CUDA;
  if (d_workspace == nullptr || !aligned16(reinterpret_cast<uint64_t>(d_workspace)) ||
      workspace_bytes < static_cast<int64_t>(kvca::attend_chunk_workspace(a, num_rows, sms)))
    return KVCA_ERR_BAD_ARGUMENT;
  return status_of(kvca::launch_attend_chunk(a, d_query_offsets, num_rows, attend_wait_limit.load(), d_workspace, sms,
                                             stream));
}

int kvca_copy_paged(const kvca_paged_desc* src, const kvca_paged_desc* dst, int64_t num_planes,
                    int64_t num_rows, int64_t row_bytes, int32_t flags, int64_t* d_status,
                    kvca_stream_t stream) {
  if (!common_move_args_ok(num_planes, num_rows, row_bytes)) return KVCA_ERR_BAD_ARGUMENT;
  if (num_rows == 0) return KVCA_OK;
  int vec = align_of(static_cast<uint64_t>(row_bytes));
  if (!check_paged(src, num_planes, row_bytes, &vec) ||
      !check_paged(dst, num_planes, row_bytes, &vec))
    return KVCA_ERR_BAD_ARGUMENT;
  kvca::PagedSide sp;
  kvca::PagedSide dp;
  to_side(src, num_planes, &sp);
  to_side(dst, num_planes, &dp);
  kvca::MoveArgs a{kvca::MoveKind::kCopyPaged, &sp, nullptr, &dp, nullptr, num_planes, num_rows,
                   row_bytes, vec, flags, d_status};
  return status_of(kvca::launch_move(a, stream));
}

}  // extern "C"

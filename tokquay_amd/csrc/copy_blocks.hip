// Copies of whole or partly filled blocks of the pool, all layers at once.
//
// A block is num_layers * 2 * num_kv_heads slabs of block_size slots; the first n slots of each are copied. The copies of one call
// run beside each other, so none may read what another writes: a pair whose destination is another pair's source, or the
// destination of an earlier one, is left out and flagged, which every workgroup of the pair finds out by itself. Past 256 pairs that takes
// longer, and a workgroup copies more.
//
// Bound by memory: whole blocks run as a large copy does, of 8 KiB a workgroup whose loads and stores pass the caches by (128 blocks of
// 1 MiB 48 us, 5.6 TB/s read and written; by ordinary ones and 16 KiB 59 us; a device copy of 128 MiB 50).
#include "tq_internal.h"

namespace tq {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr int kPer = 2;  // pieces of a thread at a time
// Every workgroup goes through all pairs (of 256 bytes: 4,096 28 us, 65,536 4.1 ms, 262,144 63): these take about a second, a hundred times
// as many hours.
constexpr int kMaxPairs = 1 << 20;

struct CopyArgs {
  char* pool;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* num_slots;  // or null: whole blocks
  int32_t* d_error;
  int64_t block_bytes;
  int64_t slab_bytes;
  int32_t slot_pieces;  // 16-byte pieces of a slot in a slab
  int32_t slabs;
  int32_t num_blocks;
  int32_t block_size;
  int32_t pairs;
  int32_t slices;  // workgroups of a pair
  int32_t turns;   // of a workgroup
};

__global__ __launch_bounds__(kThreads) void copy_blocks_kernel(const CopyArgs a) {
  __shared__ int s_clash;
  const int slice = blockIdx.x % a.slices, pair = blockIdx.x / a.slices;
  const int32_t src = a.src[pair], dst = a.dst[pair];
  const int32_t n = a.num_slots != nullptr ? a.num_slots[pair] : a.block_size;
  if (src < 0 || dst < 0 || src == dst || n == 0) return;
  const bool lead = slice == 0 && threadIdx.x == 0;
  if (src >= a.num_blocks || dst >= a.num_blocks) {
    if (lead) flag_error(a.d_error, TQ_DEVERR_BLOCK_ID);
    return;
  }
  if (n < 0 || n > a.block_size) {
    if (lead) flag_error(a.d_error, TQ_DEVERR_LENGTH);
    return;
  }
  if (threadIdx.x == 0) s_clash = 0;
  __syncthreads();
  bool clash = false;
  for (int p = threadIdx.x; p < a.pairs; p += kThreads) {
    const int32_t s = a.src[p], d = a.dst[p];
    const bool copies = s >= 0 && d >= 0 && s != d && (a.num_slots == nullptr || a.num_slots[p] != 0);
    clash |= copies && (s == dst || (d == dst && p < pair));
  }
  if (clash) s_clash = 1;
  __syncthreads();
  if (s_clash != 0) {
    if (lead) flag_error(a.d_error, TQ_DEVERR_OVERLAP);
    return;
  }
  const char* from = a.pool + src * a.block_bytes;
  char* to = a.pool + dst * a.block_bytes;
  // Pieces of a slab and of the block that are copied; of whole blocks they follow each other.
  const uint32_t run = (uint32_t)n * a.slot_pieces, all = run * (uint32_t)a.slabs;
#pragma unroll 1
  for (int turn = 0; turn < a.turns; ++turn) {
    const uint32_t first = ((uint32_t)slice * a.turns + turn) * kThreads * kPer + threadIdx.x;
    u32x4 v[kPer];
    uint64_t at[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const uint32_t i = first + j * kThreads;
      at[j] = n == a.block_size ? (uint64_t)i * 16 : (uint64_t)(i / run) * a.slab_bytes + i % run * 16;
      if (i < all) v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(from + at[j]));
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (first + j * kThreads < all) __builtin_nontemporal_store(v[j], reinterpret_cast<u32x4*>(to + at[j]));
  }
}

}  // namespace
}  // namespace tq

extern "C" tq_status tq_copy_blocks(void* pool, int64_t num_blocks, int32_t num_layers, int32_t num_kv_heads,
                                    int32_t block_size, int32_t head_dim, int32_t dtype, const int32_t* src_blocks,
                                    const int32_t* dst_blocks, const int32_t* num_slots, int32_t num_pairs,
                                    int32_t* d_error, void* stream) {
  using namespace tq;
  if (num_pairs < 0 || num_blocks < 1 || num_blocks > 0x7fffffffLL || num_layers < 1 || num_kv_heads < 1 || block_size < 1)
    return TQ_ERR_INVALID_ARGUMENT;
  if ((head_dim != 64 && head_dim != 128) || block_size > kMaxBlockSize ||
      (dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16))
    return TQ_ERR_UNSUPPORTED;
  if (num_pairs == 0) return TQ_OK;
  if (num_pairs > kMaxPairs) return TQ_ERR_UNSUPPORTED;
  if (pool == nullptr || src_blocks == nullptr || dst_blocks == nullptr || (uintptr_t)pool % 16 != 0)
    return TQ_ERR_INVALID_ARGUMENT;
  const int64_t slot = (int64_t)head_dim * (dtype == TQ_F32 ? 4 : 2), slabs = 2LL * num_layers * num_kv_heads;
  CopyArgs a;
  a.pool = static_cast<char*>(pool);
  a.src = src_blocks;
  a.dst = dst_blocks;
  a.num_slots = num_slots;
  a.d_error = d_error;
  a.slab_bytes = slot * block_size;
  a.block_bytes = slabs * a.slab_bytes;
  a.turns = (num_pairs + kThreads - 1) / kThreads;
  const int64_t turn = (int64_t)kThreads * kPer * a.turns, slices = (a.block_bytes / 16 + turn - 1) / turn;
  if (a.block_bytes / 16 > 0x7fffffffLL || !grid_fits(slices * num_pairs, kThreads)) return TQ_ERR_UNSUPPORTED;
  a.slot_pieces = (int32_t)(slot / 16);
  a.slabs = (int32_t)slabs;
  a.num_blocks = (int32_t)num_blocks;
  a.block_size = block_size;
  a.pairs = num_pairs;
  a.slices = (int32_t)slices;
  hipLaunchKernelGGL(copy_blocks_kernel, dim3((unsigned)(slices * num_pairs)), dim3(kThreads), 0, (hipStream_t)stream, a);
  return check_launch();
}

// Trees of drafted tokens: their layout (positions and masks) from the nodes' parents, and the path of a tree that the sampled
// tokens take, with its keys and values moved behind the sequence's own.
//
// Node i of a sequence is its i-th row; a node's parent comes before it, -1 has none. A node's mask has a bit for itself and for each
// of its ancestors, its depth is the number of these, its position q_start + depth.
#include "tq_internal.h"

namespace tq {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------------- layout
struct LayoutArgs {
  int64_t* positions;
  uint64_t* masks;
  const int32_t* parents;
  const int32_t* cu;
  const int32_t* q_start;
  int32_t* d_error;
  int64_t words;
  int32_t num_rows;
  int32_t num_seqs;
  int32_t max_query_len;
};

// One workgroup a sequence, a wave 64 of its nodes. Inside these the ancestors are joined in six steps, each over twice as many links as
// the one before, by all waves at once; what lies above comes, wave after wave, from the mask of the one node further up that the links
// lead to, which LDS holds (of trees of more than kLayoutNodes nodes: the masks themselves). The last workgroup clears the rows of no
// sequence. Bound by its latency: the loads of lengths and parents, and the stores (one tree of 26 nodes 1.9 us, 128 of 65-256 nodes 5.3;
// with one wave a sequence, 64 nodes after the other, 8.5).
constexpr int kLayoutWaves = 8, kLayoutNodes = kWave * kLayoutWaves;

__global__ __launch_bounds__(kLayoutNodes) void tree_layout_kernel(const LayoutArgs a) {
  __shared__ uint64_t s_masks[kLayoutNodes * kLayoutWaves];  // [word][node]: of nodes below kLayoutNodes
  const int tid = threadIdx.x, lane = tid & (kWave - 1), b = blockIdx.x, threads = blockDim.x;
  if (b == a.num_seqs) {
    const int first = min(max(a.cu[0], 0), a.num_rows), last = min(max(a.cu[a.num_seqs], first), a.num_rows);
    for (int64_t i = tid; i < (int64_t)first + a.num_rows - last; i += threads) {
      const int64_t r = i < first ? i : i - first + last;
      a.positions[r] = 0;
      for (int64_t w = 0; w < a.words; ++w) a.masks[r * a.words + w] = 0;
    }
    return;
  }
  const int lo = a.cu[b], start = a.q_start[b];
  const int64_t n = (int64_t)a.cu[b + 1] - lo;
  if (n == 0) return;
  if (n < 0 || lo < 0 || lo + n > a.num_rows || n > a.max_query_len || start < 0) {
    if (tid == 0) flag_error(a.d_error, TQ_DEVERR_LENGTH);
    return;
  }
  for (int base = 0; base < n; base += threads) {
    const int i = base + tid, own = i / kWave;  // the word of this wave's nodes
    int parent = i < n ? a.parents[lo + i] : -1;
    if (parent < -1 || parent >= i) {
      if (i < n) flag_error(a.d_error, TQ_DEVERR_PARENT);
      parent = -1;
    }
    uint64_t mine = 1ull << lane;
    int up = parent >= own * kWave ? parent - own * kWave : -1, top = lane;  // a lane; the furthest one that was reached
#pragma unroll
    for (int step = 0; step < 6; ++step) {
      if (__builtin_amdgcn_ballot_w64(up >= 0) == 0) break;
      const int from = up < 0 ? lane : up;
      const uint64_t more = __shfl(mine, from);
      const int there = __shfl(top, from), next = __shfl(up, from);
      if (up >= 0) {
        mine |= more;
        top = there;
        up = next;
      }
    }
    const int above = __shfl(parent, top);  // below this wave's nodes
    uint64_t* mask = a.masks + (int64_t)(lo + i) * a.words;
    int depth = __builtin_popcountll(mine) - 1;
    if (i < n && own < kLayoutWaves) s_masks[own * kLayoutNodes + i] = mine;
    // Wave after wave: words before its own.
    const int waves = (int)min((int64_t)threads, n - base + kWave - 1) / kWave;
    for (int turn = 0; turn < waves; ++turn) {
      if (tid / kWave == turn && i < n) {
        for (int w = 0; w < own; ++w) {
          uint64_t word = 0;
          if (w <= above / kWave && above >= 0) {
            if (i < kLayoutNodes)
              word = s_masks[w * kLayoutNodes + above];
            else  // written by this workgroup before
              word = __hip_atomic_load(a.masks + (int64_t)(lo + above) * a.words + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
          depth += __builtin_popcountll(word);
          if (i < kLayoutNodes) s_masks[w * kLayoutNodes + i] = word;
          __hip_atomic_store(mask + w, word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __hip_atomic_store(mask + own, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int64_t w = own + 1; w < a.words; ++w) mask[w] = 0;
        a.positions[lo + i] = (int64_t)start + depth;
      }
      if (n > kLayoutNodes) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
      }
      if (waves > 1 || n > threads) __syncthreads();
    }
  }
}

// ---------------------------------------------------------------------------------------------- acceptance
constexpr int kMoveThreads = 256;

struct AcceptArgs {
  int64_t* tokens;
  int32_t* path;
  int32_t* counts;
  const int64_t* sampled;
  const int64_t* drafts;
  const int32_t* parents;
  const int32_t* cu;
  const int32_t* q_start;
  const int32_t* block_tables;
  int64_t bt_stride;
  char* pool;  // or null: nothing is moved
  int64_t block_bytes;
  int64_t slab_bytes;  // of a block's K or V of one head of one layer
  int32_t* d_error;
  int32_t slot_pieces;  // 16-byte pieces of a slot's K or V of one head
  int32_t pieces;       // of a slot, in all layers
  int32_t num_blocks;
  int32_t block_size;
  int32_t num_rows;
  int32_t num_seqs;
  int32_t max_path;
  int32_t slices;
  int64_t max_context;  // positions of a block table, at most 2^31 - 1: they are counted in 32 bits
};

// A workgroup takes 256 16-byte pieces of the slots of one sequence. Each of its waves walks the tree by itself; a piece's
// moves are all made by one thread, and a node's place on the path is never behind the node, so moving the path in order from the top
// reads every source before it is written over. Bound by its latency too: lengths, nodes, tables, rows (one tree in a pool of 12 layers
// 4.2 us, 64 in one of 16 layers 5.8; with each node of the path looked up in memory 5.3 and 7.3).
__global__ __launch_bounds__(kMoveThreads) void accept_tree_kernel(const AcceptArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int slice = blockIdx.x % a.slices, b = blockIdx.x / a.slices;
  const bool lead = slice == 0 && threadIdx.x < kWave;  // the wave that writes the outputs
  const int lo = a.cu[b];
  const int64_t n = (int64_t)a.cu[b + 1] - lo;
  int start = 0;
  bool fits = lo >= 0 && n > 0 && lo + n <= a.num_rows;
  if (a.pool != nullptr) {
    start = a.q_start[b];
    fits = fits && start >= 0 && start + n <= a.max_context;
  }
  int64_t* tokens = a.tokens + (int64_t)b * a.max_path;
  int32_t* path = a.path + (int64_t)b * a.max_path;
  if (!fits) {
    if (lead) {
      if (n != 0 && lane == 0) flag_error(a.d_error, TQ_DEVERR_LENGTH);
      for (int j = lane; j < a.max_path; j += kWave) tokens[j] = path[j] = -1;
      if (lane == 0) a.counts[b] = 0;
    }
    return;
  }
  const int32_t* table = a.block_tables + (int64_t)b * a.bt_stride;
  const int piece = slice * kMoveThreads + threadIdx.x;
  char* mine = a.pool + (int64_t)(piece / a.slot_pieces) * a.slab_bytes + piece % a.slot_pieces * 16;
  // The first 64 nodes, one a lane.
  const int there = lo + min(lane, (int)n - 1);
  const int32_t parent = lane < n ? a.parents[there] : -2;
  const int64_t draft = a.drafts[there], after = a.sampled[there];
  int node = 0, count = 0;
  while (node >= 0 && count < a.max_path) {
    // Up to 64 nodes of the path, one a lane.
    int here = 0, many = 0;
    int64_t token = -1;
    while (node >= 0 && many < kWave && count + many < a.max_path) {
      int64_t t;
      if (node < kWave)
        t = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(after >> 32), node) << 32 |
                      (uint32_t)__builtin_amdgcn_readlane((int)after, node));
      else
        t = a.sampled[lo + node];
      if (lane == many) {
        here = node;
        token = t;
      }
      ++many;
      int next = -1;
      if (t >= 0) {
        const uint64_t hit = __builtin_amdgcn_ballot_w64(parent == node && draft == t && lane > node);
        if (hit != 0) next = __builtin_ctzll(hit);
        for (int i0 = max(node + 1, kWave); i0 < n && next < 0; i0 += kWave) {
          const int i = min(i0 + lane, (int)n - 1);
          const uint64_t more = __builtin_amdgcn_ballot_w64(i0 + lane < n && a.parents[lo + i] == node && a.drafts[lo + i] == t);
          if (more != 0) next = i0 + __builtin_ctzll(more);
        }
      }
      node = next;
    }
    if (lead && lane < many) {
      tokens[count + lane] = token;
      path[count + lane] = here;
    }
    if (a.pool != nullptr) {
      // Lane j finds the places of node j of these.
      bool moves = lane < many && here != count + lane;
      const int sp = start + (moves ? here : 0), dp = start + (moves ? count + lane : 0);
      int32_t sb = 0, db = 0;
      if (moves) {
        sb = table[sp / a.block_size];
        db = table[dp / a.block_size];
        if ((uint32_t)sb >= (uint32_t)a.num_blocks || (uint32_t)db >= (uint32_t)a.num_blocks) {
          if (lead) flag_error(a.d_error, TQ_DEVERR_BLOCK_ID);
          moves = false;
        }
      }
      const int64_t slot = (int64_t)a.slot_pieces * 16;
      const int64_t src = sb * a.block_bytes + sp % a.block_size * slot, dst = db * a.block_bytes + dp % a.block_size * slot;
      auto of = [&](int64_t v, int j) {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), j) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)v, j));
      };
      // Four at a time: none of them is written before a later one is read from the same place (above).
      uint64_t left = __builtin_amdgcn_ballot_w64(moves);
      while (left != 0) {
        u32x4 v[4];
        int j[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          j[e] = left != 0 ? __builtin_ctzll(left) : -1;
          left &= left - 1;
          if (j[e] >= 0 && piece < a.pieces) v[e] = *reinterpret_cast<const u32x4*>(mine + of(src, j[e]));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j[e] >= 0 && piece < a.pieces) *reinterpret_cast<u32x4*>(mine + of(dst, j[e])) = v[e];
      }
    }
    count += many;
  }
  if (lead) {
    for (int j = count + lane; j < a.max_path; j += kWave) tokens[j] = path[j] = -1;
    if (lane == 0) a.counts[b] = count;
  }
}

}  // namespace
}  // namespace tq

extern "C" tq_status tq_tree_layout(int64_t* positions, int64_t* masks, int64_t mask_words, const int32_t* parents,
                                    const int32_t* cu_seqlens_q, const int32_t* q_start, int32_t num_seqs,
                                    int32_t num_rows, int32_t max_query_len, int32_t* d_error, void* stream) {
  using namespace tq;
  if (num_seqs < 0 || num_rows < 0 || max_query_len < 0 || mask_words < 0) return TQ_ERR_INVALID_ARGUMENT;
  if (num_rows == 0) return TQ_OK;
  if (positions == nullptr || cu_seqlens_q == nullptr || (masks == nullptr && mask_words > 0) ||
      (num_seqs > 0 && (parents == nullptr || q_start == nullptr)) || mask_words > 0x3fffffffLL ||
      mask_words * 64 < max_query_len)
    return TQ_ERR_INVALID_ARGUMENT;
  const int waves = max_query_len > kLayoutNodes - kWave ? kLayoutWaves : max_query_len > kWave ? (max_query_len + kWave - 1) / kWave : 1;
  if (!grid_fits((int64_t)num_seqs + 1, kWave * waves)) return TQ_ERR_UNSUPPORTED;
  LayoutArgs a;
  a.positions = positions;
  a.masks = reinterpret_cast<uint64_t*>(masks);
  a.parents = parents;
  a.cu = cu_seqlens_q;
  a.q_start = q_start;
  a.d_error = d_error;
  a.words = mask_words;
  a.num_rows = num_rows;
  a.num_seqs = num_seqs;
  a.max_query_len = max_query_len;
  hipLaunchKernelGGL(tree_layout_kernel, dim3((unsigned)num_seqs + 1), dim3(kWave * waves), 0, (hipStream_t)stream, a);
  return check_launch();
}

extern "C" tq_status tq_accept_tree(int64_t* tokens, int32_t* path, int32_t* counts, int32_t max_path,
                                    const int64_t* sampled, const int64_t* draft_tokens, const int32_t* parents,
                                    const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t num_rows, void* pool,
                                    int64_t num_blocks, int32_t num_layers, int32_t num_kv_heads, int32_t block_size,
                                    int32_t head_dim, int32_t dtype, const int32_t* block_tables,
                                    int64_t block_table_stride, int32_t max_blocks_per_seq, const int32_t* q_start,
                                    int32_t* d_error, void* stream) {
  using namespace tq;
  if (num_seqs < 0 || num_rows < 0 || max_path < 0) return TQ_ERR_INVALID_ARGUMENT;
  if (num_seqs == 0) return TQ_OK;
  if (max_path < 1 || tokens == nullptr || path == nullptr || counts == nullptr || cu_seqlens_q == nullptr ||
      (num_rows > 0 && (sampled == nullptr || draft_tokens == nullptr || parents == nullptr)))
    return TQ_ERR_INVALID_ARGUMENT;
  AcceptArgs a = {};
  a.slices = 1;
  if (pool != nullptr) {
    if (num_blocks < 1 || num_blocks > 0x7fffffffLL || num_layers < 1 || num_kv_heads < 1 || block_size < 1 ||
        max_blocks_per_seq < 0 || block_tables == nullptr || q_start == nullptr || block_table_stride < max_blocks_per_seq ||
        (uintptr_t)pool % 16 != 0)
      return TQ_ERR_INVALID_ARGUMENT;
    if ((head_dim != 64 && head_dim != 128) || block_size > kMaxBlockSize ||
        (dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16))
      return TQ_ERR_UNSUPPORTED;
    const int64_t slot = (int64_t)head_dim * (dtype == TQ_F32 ? 4 : 2), slabs = 2LL * num_layers * num_kv_heads;
    if (slabs * (slot / 16) > 0x7fffffffLL - kMoveThreads) return TQ_ERR_UNSUPPORTED;
    a.pool = static_cast<char*>(pool);
    a.slab_bytes = slot * block_size;
    a.block_bytes = slabs * a.slab_bytes;
    a.slot_pieces = (int32_t)(slot / 16);
    a.pieces = (int32_t)(slabs * (slot / 16));
    a.slices = (a.pieces + kMoveThreads - 1) / kMoveThreads;
    a.num_blocks = (int32_t)num_blocks;
    a.block_size = block_size;
    const int64_t positions = (int64_t)max_blocks_per_seq * block_size;
    a.max_context = positions < 0x7fffffffLL ? positions : 0x7fffffffLL;
    a.block_tables = block_tables;
    a.bt_stride = block_table_stride;
    a.q_start = q_start;
  } else {
    a.slot_pieces = 1;
  }
  if (!grid_fits((int64_t)num_seqs * a.slices, kMoveThreads)) return TQ_ERR_UNSUPPORTED;
  a.tokens = tokens;
  a.path = path;
  a.counts = counts;
  a.sampled = sampled;
  a.drafts = draft_tokens;
  a.parents = parents;
  a.cu = cu_seqlens_q;
  a.d_error = d_error;
  a.num_rows = num_rows;
  a.num_seqs = num_seqs;
  a.max_path = max_path;
  hipLaunchKernelGGL(accept_tree_kernel, dim3((unsigned)(num_seqs * a.slices)), dim3(kMoveThreads), 0, (hipStream_t)stream, a);
  return check_launch();
}

// Attention of chunks of new tokens over a paged 16-bit cache, heads grouped: G = H / Hkv query
// heads read each K/V head.
//
//   out[t, h] = sum_j p_j V[j, h / G] / sum_j p_j,   p_j = 2^(c (q[t, h] . K[j, h / G]) - m),   j <= q_start + t
//
// with c = scale log2(e) and m a running maximum less kLift (any m gives the same quotient; it is raised when a score
// passes the maximum by more than kSlack, so p stays below 2^(kLift + kSlack) and the sums are rescaled rarely). The G heads of a
// token read the same keys, so (token, head of the group) pairs are the rows of one matrix product: row r
// is token r / G, head r % G of the group, and a 16-row tile holds 16 / G tokens.
//
// Per 16 rows and 32 keys, on the 16x16x32 matrix instructions (fp32 sums):
//
//   S^T[key][row] = K[key][:] . Q[row][:]            D / 32 depth steps for each 16 keys
//   O^T[dim][row] += V^T[dim][key] P^T[key][row]     one depth step for each 16 dims
//
// The transposed scores leave lane (i, g) = (lane % 16, lane / 16) with row i and the keys 4 g + 0..3 and
// 16 + 4 g + 0..3, so one lane's scores belong to one row (its position is one register, its maximum
// is taken in the lane and across four lanes) and are, rounded to 16 bits, the B operand
// of the second product with no exchange: that product may take the keys in any order, and V^T is read in
// the same one (two transposing LDS reads of 4 keys each). Rounding p to the cache's type costs each weight half a
// step, about as much as the rounding of the output; the rounded weights are summed, so equal values come out exactly. float16
// has no full step below 2^-14, so its weights are lifted by 2^7: those below 2^-21 of the row's largest are off by up to 2^-32 of
// that one, where half a step would be less (without the lift 2^-25: 4,000 equal keys 17 nats below one without value came
// out 44 % too heavy, and not at all at 17.4).
//
// K and V come in tiles straight from HBM into LDS (16 bytes a lane, no registers), a tile ahead of the products.
// 16-byte pieces are permuted inside a row as they arrive (swizzled), so that what an LDS read takes in a clock
// lies in different banks.
//
// Two kernels. Up to 64 rows a K/V head (tokens, drafted tokens) the bytes of K and V bound it: chunk_rows_kernel streams them,
// each wave its own keys (128 tokens at 511-4,094 positions, 8 heads of 128: 1.21 GB in 218 us, 5.5 TB/s, where a device copy
// moves 5.07). More rows share tiles (chunk_tiles_kernel; chunk_queue_kernel over long contexts), and the matrix cores beside
// the exponentials bound it: 4 x 2,048 tokens behind 768-5,376 cached ones run 550 GFLOP in 495-540 us (1,020-1,110 TFLOP/s from
// card to card; a large bf16 library product reaches 1,370), with the matrix cores busy for 57 % of the time and the vector units
// for 55. The longest sequence decides for all (plan_of): beside 259 tokens behind 32,500, three single tokens at 300 take 818 us
// with them, where the two calls take 175 and 9.
//
// TREE (tq_paged_tree): the new tokens are nodes of a tree of drafts, and a row sees of them those that its mask names and that are not
// behind itself, so a part of what it would see in a line: tiles, parts and maxima are those of a line, and tiles with new keys are
// masked by bits. A row that sees nothing has a sum of zero and gets zeros (inverse). 64 trees of 64 nodes behind 511-4,094 tokens, 32 / 8
// heads of 128: 0.62 GB and 155 GFLOP in 202 us (as a line 196), matrix cores busy for 46 % of the time and vector units for 47.
#include <float.h>

#include <utility>

#include "half_types.h"

namespace tq {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTileKeys = 32;  // keys of a tile
constexpr int kCus = 256, kXcds = 8;
constexpr int kTileRows = 16;  // rows of a tile
constexpr int kWaves = 4;

struct ChunkArgs {
  uint16_t* out;
  int64_t out_stride;
  const uint16_t* q;
  int64_t q_stride;
  const uint16_t* pool_layer;
  uint32_t block_stride;
  int64_t kv_stride;
  int64_t head_stride;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu_q;
  const int32_t* q_start;
  float* part_o;   // [num_q_rows][num_heads][parts][D] sums of each part, or null: one part
  float* part_ml;  // [num_q_rows][num_heads][parts][2] maximum and weight sum
  int32_t* queue;  // kQueueHead words, then (sequence, row tile) pairs: chunk_order_kernel; or null
  int32_t* d_error;
  float c;         // |scale| log2(e)
  uint32_t q_sign; // 0x80008000 where the scale is negative: the queries' signs are flipped
  int32_t num_blocks;
  int32_t num_heads;
  int32_t kv_heads;
  int32_t group;
  int32_t block_size;
  uint32_t inv_block;  // ceil(2^21 / block_size)
  int32_t max_blocks;
  int32_t num_q_rows;
  int32_t max_query_len;
  int32_t max_context;
  int32_t num_seqs;
  int32_t row_tiles;    // workgroup row tiles per (sequence, K/V head)
  int32_t parts;        // key parts per row tile
  int32_t part_tokens;  // keys of a part, a multiple of kWaves * kTileKeys
  // tq_paged_tree: row r's bits from masks + r mask_words on. Behind all others, so that those lie where they do without masks: further
  // up, the kernels without masks fetched them otherwise (one token behind 4,000 12.1 -> 12.4 us, 32 x 5 drafted tokens 42.9 -> 43.5).
  const uint32_t* masks;
  int64_t mask_words;
};

__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A sequence's rows and positions, or why it has none here.
struct Seq {
  int row0, nq, start;
};

__device__ __forceinline__ bool fits(const ChunkArgs& a, const Seq& s, int64_t nq) {
  const int64_t end = (int64_t)s.start + nq;
  return nq > 0 && nq <= a.max_query_len && s.row0 >= 0 && s.row0 + nq <= a.num_q_rows && s.start >= 0 &&
         end <= a.max_context && end <= (int64_t)a.max_blocks * a.block_size;
}

// False where the sequence has no rows or its lengths do not fit (flagged by the workgroup that `reports`).
__device__ __forceinline__ bool seq_of(const ChunkArgs& a, int b, bool reports, Seq& s) {
  s.row0 = __builtin_amdgcn_readfirstlane(a.cu_q[b]);
  const int64_t nq = (int64_t)__builtin_amdgcn_readfirstlane(a.cu_q[b + 1]) - s.row0;
  s.start = __builtin_amdgcn_readfirstlane(a.q_start[b]);
  s.nq = (int)nq;
  if (nq == 0) return false;
  const bool ok = fits(a, s, nq);
  if (!ok && reports && threadIdx.x == 0) flag_error(a.d_error, TQ_DEVERR_LENGTH);
  return ok;
}

// 16-byte piece p of a tile's key `key` lies at piece p ^ swizzle(key) of the key's row in LDS, so that the banks (64 of 4
// bytes) are each met once a clock: a read of K takes one piece of 16 keys, 16 lanes a clock (quads of lanes 0, 3 of one lane
// group and 1, 2 of the next); one of V two neighbouring pieces of 8 consecutive keys. The first asks for distinct
// swizzle(key) ^ group, the second for distinct swizzle(key) / 2 (at D = 64 with the key's lowest bit above, which picks
// the half of the 256 bytes). No conflicts counted; with key & 15 a quarter of the reading clocks.
template <int D>
__device__ __forceinline__ int swizzle(int key) {
  return D == 128 ? (key & 7) << 1 ^ (key & 8 ? 9 : 0) : (key & 6) ^ (key & 8 ? 5 : 0);
}

// Zeros in place of the infinities and NaN among a wave's `pieces` 16-byte pieces of V in LDS; whether there were any (uniform).
// For tiles with keys that some row does not see: a weight of zero times infinity is NaN. The rows that do see them get them
// back at the end (add_left_out).
template <typename T>
__device__ __forceinline__ bool clean_values(uint16_t* s_v, int pieces) {
  bool any = false;
#pragma unroll 1
  for (int j = threadIdx.x & (kWave - 1); j < pieces; j += kWave) {
    u32x4 v = reinterpret_cast<const u32x4*>(s_v)[j];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = v[e];
      const bool lo = (x & T::kExponent) == T::kExponent, hi = ((x >> 16) & T::kExponent) == T::kExponent;
      v[e] = (lo ? 0u : x & 0xffffu) | (hi ? 0u : x & 0xffff0000u);
      bad |= lo || hi;
    }
    if (bad) reinterpret_cast<u32x4*>(s_v)[j] = v;
    any |= bad;
  }
  return __builtin_amdgcn_ballot_w64(any) != 0;
}

// Which of the keys from .. from + 31 a tree's row at position qpos sees: every key before `start`, of those from there on the ones
// its mask names, none behind its own.
__device__ __forceinline__ uint32_t seen_bits(const ChunkArgs& a, int64_t row, int start, int qpos, int from) {
  const uint32_t* m = a.masks + row * a.mask_words;
  const int rel = from - start, w = rel >> 5, own = qpos - from;
  const int words = (int)a.mask_words;
  auto word = [&](int i) {  // no branches: the loads of all rows are on their way together
    const uint32_t v = m[min(max(i, 0), words - 1)];
    return i < 0 ? ~0u : i < words ? v : 0u;
  };
  const uint32_t bits = __builtin_amdgcn_alignbit(word(w + 1), word(w), rel & 31);
  return own >= 31 ? bits : own < 0 ? 0u : bits & ((2u << own) - 1u);
}

// Values of four dims of a row that the products left out, added to `o`: those of keys from..to - 1 (to: past the row's last
// key) that are infinities or NaN. head_base is at the first of the dims in the K slab. TREE: of those the row sees.
template <typename T, bool TREE>
__device__ __forceinline__ void add_left_out(const ChunkArgs& a, const int32_t* bt, const uint16_t* head_base, int D,
                                             int from, int to, const Seq& s, int t, f32x4& o) {
#pragma unroll 1
  for (int key = from; key < to; ++key) {
    if (TREE && !(seen_bits(a, s.row0 + t, s.start, s.start + t, key) & 1u)) continue;
    const int ti = key / a.block_size;
    const int32_t blk = bt[ti];
    if ((uint32_t)blk >= (uint32_t)a.num_blocks) continue;  // flagged by the loads
    const u32x2 v = *reinterpret_cast<const u32x2*>(head_base + (int64_t)blk * a.block_stride + a.kv_stride +
                                                    (int64_t)(key - ti * a.block_size) * D);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t x = (v[e >> 1] >> (16 * (e & 1))) & 0xffffu;
      if ((x & T::kExponent) == T::kExponent) o[e] += T::load((uint16_t)x);
    }
  }
}

// A block-table entry, or block 0 for a bad one, which is flagged.
__device__ __forceinline__ int32_t checked(const ChunkArgs& a, int32_t id) {
  if ((uint32_t)id < (uint32_t)a.num_blocks) return id;
  flag_error(a.d_error, TQ_DEVERR_BLOCK_ID);
  return 0;
}

// A tile's first key and its place in the sequence's blocks. Keys from `stop` on are the last one before it again:
// finite wherever that one is, and masked.
struct Cursor {
  int kt, stop;          // uniform, as is all of it
  int q, r;              // kt = q block_size + r
  int end_q, end_r;      // stop - 1
  int step_q, step_r;    // the step to the next tile

  __device__ __forceinline__ void init(const ChunkArgs& a, int first, int until, int step) {
    kt = first;
    stop = until;
    q = kt / a.block_size;
    r = kt - q * a.block_size;
    end_q = (stop - 1) / a.block_size;
    end_r = stop - 1 - end_q * a.block_size;
    step_q = step / a.block_size;
    step_r = step - step_q * a.block_size;
  }
  __device__ __forceinline__ void next(const ChunkArgs& a, int step) {
    kt += step;
    q += step_q;
    r += step_r;
    if (r >= a.block_size) {
      r -= a.block_size;
      ++q;
    }
  }
  __device__ __forceinline__ int first_entry() const { return kt < stop ? q : end_q; }
  // Table entry and slot in its block of the tile's key `local` (below 64). With x below 1024 + 64 and inv_block =
  // ceil(2^21 / block_size), x inv_block / 2^21 exceeds x / block_size by less than 1 / block_size.
  __device__ __forceinline__ void place(const ChunkArgs& a, int local, int& entry, int& slot) const {
    const bool in = kt < stop;
    const uint32_t x = (uint32_t)((in ? r : end_r) + min(local, in ? stop - 1 - kt : 0));
    const uint32_t b = __umul24(x, a.inv_block) >> 21;
    entry = (in ? q : end_q) + (int)b;
    slot = (int)(x - __umul24(b, a.block_size));
  }
};

// The block ids of one wave's tiles: 64 consecutive table entries in its lanes, and the 64 that come next on their
// way, so that a tile waits for none.
struct Window {
  int base, next_base;
  int32_t ids, next;

  __device__ __forceinline__ int32_t entries(const int32_t* bt, const Cursor& c, int from) const {
    return bt[min(from + (int)(threadIdx.x & (kWave - 1)), c.end_q)];
  }
  // The entries from the first later tile on that passes these.
  __device__ __forceinline__ void ahead(const ChunkArgs& a, const int32_t* bt, const Cursor& c, int step) {
    const int64_t left = (int64_t)(base + kWave) * a.block_size - (kTileKeys - 1) - c.kt;
    const int64_t at = c.kt + (left <= 0 ? step : (left + step - 1) / step * step);
    next_base = (int)(min(at, (int64_t)c.stop - 1) / a.block_size);
    next = entries(bt, c, next_base);
  }
  __device__ __forceinline__ void init(const ChunkArgs& a, const int32_t* bt, const Cursor& c, int step) {
    base = c.first_entry();
    ids = entries(bt, c, base);
    ahead(a, bt, c, step);
    ids = checked(a, ids);
  }
  // Moves on where the cursor's tile passes the entries at hand.
  __device__ __forceinline__ void move(const ChunkArgs& a, const int32_t* bt, const Cursor& c, int step) {
    if (min(c.kt + kTileKeys, c.stop) - 1 < (int64_t)(base + kWave) * a.block_size) return;  // uniform
    base = next_base;
    ids = checked(a, next);
    asm volatile("" : "+v"(ids));  // waited for here, not by every tile
    ahead(a, bt, c, step);
  }
};

// The copy of J times 1024 bytes of a tile of one K/V head into LDS by one wave, from key `first` of the tile on. kLanes lanes
// take a key's row, so instruction j copies the keys first + j kKeys + lane / kLanes; lane l looks up the key of
// instruction l % J, and hands where its row lies to the others that copy it (a broadcast in rows of 16 or 4 lanes).
template <int D, int J>
struct Loader {
  static constexpr int kLanes = D / 8;
  static constexpr int kKeys = kWave / kLanes;
  static_assert(J <= 4 || (J == 8 && kLanes == 16), "J lanes that copy the same keys lie in one row");
  const uint16_t* src[J];  // K; V is kv_stride on

  static __device__ __forceinline__ int own_key(int first) {
    const int lane = threadIdx.x & (kWave - 1);
    return first + kKeys * (lane % J) + lane / kLanes;
  }
  template <int FROM>
  static __device__ __forceinline__ uint32_t broadcast(uint32_t v) {
    constexpr int kRowBroadcast = 0x150;  // of the row's lane FROM; else of the quad's
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, J == 8 ? kRowBroadcast + FROM : 0x55 * FROM, 0xF, 0xF, true);
  }
  // `id`, `slot`: block and slot of this lane's own_key.
  __device__ __forceinline__ void aim(const ChunkArgs& a, const uint16_t* head_base, int first, int32_t id, int slot) {
    const uint64_t row = (uint64_t)head_base + ((uint64_t)(uint32_t)id * (2 * a.block_stride) + (uint32_t)slot * (2 * D));
    aim_each(first, row, std::make_integer_sequence<int, J>());
  }
  template <int... j>
  __device__ __forceinline__ void aim_each(int first, uint64_t row, std::integer_sequence<int, j...>) {
    const int lane = threadIdx.x & (kWave - 1);
    ((src[j] = reinterpret_cast<const uint16_t*>(
          ((uint64_t)broadcast<j>((uint32_t)(row >> 32)) << 32 | broadcast<j>((uint32_t)row)) +
          16 * (uint32_t)((lane % kLanes) ^ swizzle<D>(first + j * kKeys + lane / kLanes)))),
     ...);
  }

  // `to`: the tile's row `first` in LDS.
  __device__ __forceinline__ void start(uint16_t* to, int64_t offset) const {
    typedef const __attribute__((address_space(1))) void* Global;
    typedef __attribute__((address_space(3))) void* Lds;
#pragma unroll
    for (int j = 0; j < J; ++j)
      __builtin_amdgcn_global_load_lds((Global)(src[j] + offset), (Lds)(to + j * kKeys * D), 16, 0, 0);
  }
};

// The rows of one wave: queries, sums, running maxima. KS: 32-key steps of a tile.
template <int D, int NT, int KS, typename T, bool TREE>
struct Rows {
  u32x4 q[NT][D / 32];
  f32x4 o[NT][D / 16];
  f32x4 l[NT];  // sum of the weights, four times
  float m[NT];
  int qpos[NT];
  int lo, hi;  // every row sees the keys up to lo, none those past hi (uniform)
  int start;   // of the sequence, with TREE
  int64_t row_at;  // a row at position p is row p + row_at of the call, with TREE

  typedef f32x4 Scores[2 * KS][NT];  // of keys 16 h + 4 g + 0..3 with row i of row tile n
  typedef u32x4 Weights[KS][NT];     // rounded: of keys 32 k + 4 g + 0..3 and 32 k + 16 + 4 g + 0..3

  __device__ __forceinline__ void init(const ChunkArgs& a, const Seq& s, int kvh, int r0) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
    const int last = s.nq * a.group - 1;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = min(r0 + kTileRows * n + i, last), t = r / a.group;
      const uint16_t* qp = a.q + (int64_t)(s.row0 + t) * a.q_stride + (kvh * a.group + r - t * a.group) * D + 8 * g;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) q[n][k] = *reinterpret_cast<const u32x4*>(qp + 32 * k);
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      qpos[n] = s.start + t;
      m[n] = -FLT_MAX;
      l[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    lo = TREE ? s.start - 1 : __builtin_amdgcn_readfirstlane(s.start + min(r0, last) / a.group);
    if constexpr (TREE) {
      start = s.start;
      row_at = (int64_t)s.row0 - s.start;
    }
    hi = __builtin_amdgcn_readfirstlane(s.start + min(r0 + kTileRows * NT - 1, last) / a.group);
  }

  __device__ __forceinline__ void flip(uint32_t sign) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < D / 32; ++k) q[n][k] ^= sign;
  }

  // K of keys 16 h + 0..15 as the first operand of D / 32 products.
  static __device__ __forceinline__ void read_k(const uint16_t* s_k, int h, u32x4 (&kf)[D / 32]) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
    const int key = 16 * h + i;
#pragma unroll
    for (int k = 0; k < D / 32; ++k)
      kf[k] = *reinterpret_cast<const u32x4*>(s_k + key * D + 8 * ((4 * k + g) ^ swizzle<D>(key)));
  }

  // The same beside loads into LDS (values_beside_loads).
  static __device__ __forceinline__ void read_k_beside_loads(const uint16_t* s_k, int h, u32x4 (&kf)[D / 32]) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
    const int key = 16 * h + i;
    typedef __attribute__((address_space(3))) const u32x4* Lds;
    Lds at[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) at[k] = (Lds)(s_k + key * D + 8 * ((4 * k + g) ^ swizzle<D>(key)));
    if constexpr (D == 128)
      asm volatile(
          "ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(kf[0]), "=&v"(kf[1]), "=&v"(kf[2]), "=&v"(kf[3])
          : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
          : "memory");
    else
      asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(kf[0]), "=&v"(kf[1])
                   : "v"(at[0]), "v"(at[1])
                   : "memory");
  }

  __device__ __forceinline__ void scores(const u32x4 (&kf)[D / 32], f32x4 (&s)[NT]) const {
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < D / 32; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n] = T::mfma(kf[k], q[n][k], s[n]);
  }

  // Whether some row does not see some key of the tile (uniform).
  __device__ __forceinline__ bool masked(int kt) const { return kt + 32 * KS - 1 > lo; }

  // Masks the scores of the tile of keys kt .. and raises the running maxima where they are passed.
  __device__ __forceinline__ void maxima(const ChunkArgs& a, int kt, Scores& s) {
    const int g = (threadIdx.x & (kWave - 1)) >> 4;
    if (TREE && masked(kt)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const uint32_t bits = seen_bits(a, qpos[n] + row_at, start, qpos[n], kt + 32 * k) >> (4 * g);
#pragma unroll
          for (int h = 2 * k; h < 2 * k + 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[h][n][e] = bits >> (16 * (h % 2) + e) & 1u ? s[h][n][e] : -INFINITY;
        }
    } else if (masked(kt)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2 * KS; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[h][n][e] = kt + 16 * h + 4 * g + e <= qpos[n] ? s[h][n][e] : -INFINITY;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = max2(max2(s[0][n][0], s[0][n][1]), max2(s[0][n][2], s[0][n][3]));
#pragma unroll
      for (int h = 1; h < 2 * KS; ++h)
        top = max2(max2(max2(top, s[h][n][0]), s[h][n][1]), max2(s[h][n][2], s[h][n][3]));
      top *= a.c;
      // By the difference, which is exact where it is near: a limit of its own would be rounded, at scores from 2^24 on past
      // what a float16 weight holds.
      if (__builtin_amdgcn_ballot_w64(top - m[n] > T::kLift + T::kSlack) != 0) {
        top = max2(top, __shfl_xor(top, 16));
        top = max2(top, __shfl_xor(top, 32));
        const bool grow = top - m[n] > T::kLift + T::kSlack;
        const float next = grow ? top - T::kLift : m[n];
        const float corr = grow ? __builtin_amdgcn_exp2f(m[n] - next) : 1.f;
        l[n] *= corr;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[n][d] *= corr;
        m[n] = next;
      }
    }
  }

  // The weights of keys 16 h + 0..15.
  __device__ __forceinline__ void weights(const ChunkArgs& a, int h, const f32x4 (&s)[NT], Weights& w) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[n][e], a.c, -m[n]));
      w[h / 2][n][2 * (h % 2)] = pack2<T>(p[0], p[1]);
      w[h / 2][n][2 * (h % 2) + 1] = pack2<T>(p[2], p[3]);
    }
  }

  // Adds the weights to their rows' sums, by a product with ones: on the matrix cores, which have the time (4 instructions
  // for 32 additions and their joining across lanes), and of the rounded weights that meet V.
  __device__ __forceinline__ void sums(const Weights& w) {
    const u32x4 ones = {T::kOnes, T::kOnes, T::kOnes, T::kOnes};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n) l[n] = T::mfma(ones, w[k][n], l[n]);
  }

  // Four dim tiles' V at a time, the next four's on their way.
  __device__ __forceinline__ void values(const uint16_t* s_v, const Weights& w) {
    u32x4 vf[2][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) vf[0][e] = read_v(s_v, e);
#pragma unroll
    for (int j = 0; j < KS * D / 64; ++j) {
      const int k = j / (D / 64), d = j % (D / 64) * 4, jn = j + 1;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (jn < KS * D / 64) vf[jn & 1][e] = read_v(s_v + 32 * (jn / (D / 64)) * D, jn % (D / 64) * 4 + e);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[n][d + e] = T::mfma(vf[j & 1][e], w[k][n], o[n][d + e]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // The same for callers with loads into LDS on their way, for all of which the compiler waits before the builtin's reads (it
  // cannot tell them apart): the reads and the wait for them in one block, four dim tiles at a time.
  __device__ __forceinline__ void values_beside_loads(const uint16_t* s_v, const Weights& w) {
#pragma unroll
    for (int j = 0; j < KS * D / 64; ++j) {
      const int k = j / (D / 64), d = j % (D / 64) * 4;
      const uint16_t* base = s_v + 32 * k * D;
      u32x2 lo[4], hi[4];
      asm volatile(
          "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %4, %8 offset:%12\n\t"
          "ds_read_b64_tr_b16 %1, %9\n\tds_read_b64_tr_b16 %5, %9 offset:%12\n\t"
          "ds_read_b64_tr_b16 %2, %10\n\tds_read_b64_tr_b16 %6, %10 offset:%12\n\t"
          "ds_read_b64_tr_b16 %3, %11\n\tds_read_b64_tr_b16 %7, %11 offset:%12\n\t"
          "s_waitcnt lgkmcnt(0)"
          : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
          : "v"(v_address(base, d)), "v"(v_address(base, d + 1)), "v"(v_address(base, d + 2)),
            "v"(v_address(base, d + 3)), "n"(16 * D * 2)
          : "memory");
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          o[n][d + e] = T::mfma(u32x4{lo[e][0], lo[e][1], hi[e][0], hi[e][1]}, w[k][n], o[n][d + e]);
    }
  }

  // V^T of dims 16 d + 0..15: dim 16 d + i, keys 4 g + 0..3 and 16 + 4 g + 0..3. Of 16 lanes, lane 4 a + b names
  // four values of key a and gets value (its own index) of keys 0..3.
  static __device__ __forceinline__ u32x4 read_v(const uint16_t* s_v, int d) {
    u32x2 half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)  // 16 keys on, the swizzle is the same
      half[h] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(v_address(s_v, d) + 4 * h * D));
    return u32x4{half[0][0], half[0][1], half[1][0], half[1][1]};
  }

  typedef __attribute__((address_space(3))) s16x4* Lds;
  static __device__ __forceinline__ Lds v_address(const uint16_t* s_v, int d) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
    const int key = 4 * g + (i >> 2), piece = 2 * d + ((i >> 1) & 1);
    return (Lds)(s_v + key * D + 8 * (piece ^ swizzle<D>(key)) + 4 * (i & 1));
  }
};

// Waits until at most N loads are on their way (they end in order); the compiler does not know which loads into LDS a read
// of LDS needs.
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "vmcnt has six bits");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// Waits until what was read of LDS is in registers: its place is free for other loads.
__device__ __forceinline__ void wait_reads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_sched_barrier(0);
}

// The workgroup's waves meet, with their LDS accesses done; loads may be on their way.
__device__ __forceinline__ void barrier() {
  wait_reads();
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// One over a row's sum of weights; 0 for a tree's row (token t of the sequence) that sees nothing, whose output is zero. A row that
// sees keys, but with scores of -infinity alone, has no softmax: NaN, with or without TREE.
template <bool TREE>
__device__ __forceinline__ float inverse(const ChunkArgs& a, const Seq& s, int t, float l) {
  if constexpr (TREE) {
    if (l == 0.f && s.start == 0) {
      const uint32_t* m = a.masks + (s.row0 + t) * a.mask_words;
      uint32_t any = m[t / 32] & ((2u << t % 32) - 1u);  // none behind its own
#pragma unroll 1
      for (int w = 0; w < t / 32; ++w) any |= m[w];
      if (any == 0) return 0.f;
    }
  }
  return 1.f / l;
}

// Few rows: a workgroup takes 16 NT rows and one part of the keys; its waves take every fourth tile of the
// part, each with its own two K and two V buffers in LDS and no barrier, and join their sums in LDS at the end.
//
// K and V of the next tile and V of this one are on their way while a tile's scores are computed: 24 KB a wave, 96 KB a CU
// (12 KB and two workgroups at D = 64), which covers the latency of HBM at its full rate. With the tile loaded only when the one
// before was done: 128 tokens at 511-4,094 positions 557 us instead of 218. Tiles of 64 keys at D = 64 changed nothing on average
// (32 x 5 drafted tokens 39.7 -> 39.2 us, 64 tokens of 12 heads 38 -> 42, 16 x 4 of 28 heads 32 -> 28).
template <int D, int NT, typename T, bool TREE>
__global__ __launch_bounds__(kWave* kWaves) void chunk_rows_kernel(const ChunkArgs a) {
  constexpr int kTileElems = kTileKeys * D;
  __shared__ __attribute__((aligned(16))) uint16_t s_k0[kWaves * kTileElems], s_v0[kWaves * kTileElems],
      s_k1[kWaves * kTileElems], s_v1[kWaves * kTileElems];
  __shared__ float s_ml[kWaves][kTileRows * NT][2];
  __shared__ int s_dirty[kWaves];
  const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int idx = blockIdx.x;
  const int part = idx % a.parts;
  idx /= a.parts;
  const int tile = idx % a.row_tiles;
  idx /= a.row_tiles;
  const int kvh = idx % a.kv_heads, b = idx / a.kv_heads;
  Seq s;
  if (!seq_of(a, b, part == 0 && tile == 0 && kvh == 0, s)) return;
  const int r0 = tile * kTileRows * NT, rows = min(kTileRows * NT, s.nq * a.group - r0);
  if (rows <= 0) return;
  const int last = (s.start + min(r0 + kTileRows * NT - 1, s.nq * a.group - 1) / a.group);
  const int kend = last + 1, kbeg = part * a.part_tokens;
  if (kbeg >= kend) return;
  const int kstop = min(kend, kbeg + a.part_tokens);

  const int32_t* bt = a.block_tables + (int64_t)b * a.bt_stride;
  const uint16_t* head_base = a.pool_layer + (int64_t)kvh * a.head_stride;
  constexpr int kStep = kWaves * kTileKeys;
  constexpr int J = kTileElems * 2 / 1024;
  typedef Rows<D, NT, 1, T, TREE> R;
  R w;
  Loader<D, J> load;
  uint16_t *k0 = s_k0 + wave * kTileElems, *v0 = s_v0 + wave * kTileElems, *k1 = s_k1 + wave * kTileElems,
           *v1 = s_v1 + wave * kTileElems;
  int kt = kbeg + wave * kTileKeys;
  w.init(a, s, kvh, r0);
  Cursor c;
  c.init(a, kt, kstop, kStep);
  Window ids;
  ids.init(a, bt, c, kStep);
  // Tiles past the part's end are loaded too (its last key again and again), so that the count of loads behind the
  // one that is waited for stays the same: K and V of two tiles are always on their way, of which a wait takes the first.
  auto aim = [&] {
    ids.move(a, bt, c, kStep);
    int entry, slot;
    c.place(a, Loader<D, J>::own_key(0), entry, slot);
    load.aim(a, head_base, 0, __shfl(ids.ids, entry - ids.base), slot);
    c.next(a, kStep);
  };
  aim();
  load.start(k0, 0);
  load.start(v0, a.kv_stride);
  aim();
  load.start(k1, 0);
  load.start(v1, a.kv_stride);
  w.flip(a.q_sign);
  bool dirty = false;
  auto step = [&](uint16_t* s_k, uint16_t* s_v) {
    typename R::Scores sc;
    typename R::Weights wt;
    u32x4 kf[2][D / 32];
    wait_loads<3 * J>();  // behind K of this tile: V, K and V of the next
    R::read_k_beside_loads(s_k, 0, kf[0]);
    R::read_k_beside_loads(s_k, 1, kf[1]);
    w.scores(kf[0], sc[0]);
    w.scores(kf[1], sc[1]);
    wait_reads();
    aim();
    load.start(s_k, 0);
    w.maxima(a, kt, sc);
    w.weights(a, 0, sc[0], wt);
    w.weights(a, 1, sc[1], wt);
    wait_loads<3 * J>();
    if (w.masked(kt)) dirty |= clean_values<T>(s_v, kTileElems / 8);
    w.sums(wt);
    w.values_beside_loads(s_v, wt);
    wait_reads();
    load.start(s_v, a.kv_stride);
    kt += kStep;
  };
  while (kt < kstop) {
    step(k0, v0);
    if (kt >= kstop) break;
    step(k1, v1);
  }

  // Join: wave v's sums go to the v-th array, 16-byte pieces permuted by row.
  wait_loads<0>();  // of tiles that were not needed
  if (lane == 0) s_dirty[wave] = dirty;
  __syncthreads();
  float* s_o[kWaves] = {reinterpret_cast<float*>(s_k0), reinterpret_cast<float*>(s_v0), reinterpret_cast<float*>(s_k1),
                        reinterpret_cast<float*>(s_v1)};
  float* mine = wave == 0 ? s_o[0] : wave == 1 ? s_o[1] : wave == 2 ? s_o[2] : s_o[3];
  static_assert(kTileRows * NT * D * 4 <= kWaves * kTileElems * 2, "a wave's sums fit one array");
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float l = w.l[n][0];
    const int r = kTileRows * n + i;
    if (g == 0) {
      s_ml[wave][r][0] = w.m[n];
      s_ml[wave][r][1] = l;
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
      *reinterpret_cast<f32x4*>(mine + r * D + 4 * ((4 * d + g) ^ (r & (D / 4 - 1)))) = w.o[n][d];
  }
  __syncthreads();
  dirty = (s_dirty[0] | s_dirty[1] | s_dirty[2] | s_dirty[3]) != 0;
  for (int e = threadIdx.x; e < rows * (D / 4); e += kWave * kWaves) {
    const int r = e / (D / 4), piece = e % (D / 4), d = 4 * piece;
    float top = s_ml[0][r][0];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) top = fmaxf(top, s_ml[v][r][0]);
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f(s_ml[v][r][0] - top);
      l = fmaf(f, s_ml[v][r][1], l);
      const f32x4 ov = *reinterpret_cast<const f32x4*>(s_o[v] + r * D + 4 * (piece ^ (r & (D / 4 - 1))));
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fmaf(f, ov[k], o[k]);
    }
    const int t = (r0 + r) / a.group, h = kvh * a.group + (r0 + r) - t * a.group;
    if (dirty)
      add_left_out<T, TREE>(a, bt, head_base + d, D, max(kbeg, (w.lo + 1) / kTileKeys * kTileKeys), min(kstop, s.start + t + 1),
                            s, t, o);
    if (a.parts == 1) {
      const float inv = inverse<TREE>(a, s, t, l);
      *reinterpret_cast<u32x2*>(a.out + (int64_t)(s.row0 + t) * a.out_stride + h * D + d) =
          u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
    } else {
      const int64_t at = ((int64_t)(s.row0 + t) * a.num_heads + h) * a.parts + part;
      *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = o;
      if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + at * 2) = f32x2{top, l};
    }
  }
}

// Many rows: a workgroup takes 64 NT rows, 16 NT a wave, and one part of the keys; its waves share the tiles of 64 keys
// in LDS, each loading a quarter. The scores of tile t + 1 are computed beside the weights of tile t (matrix and
// vector instructions of one iteration do not depend on each other), so one barrier a tile is enough: behind it K of t + 1
// and V of t are in LDS, and the buffers of K of t and V of t - 1 are free for K of t + 2 and V of t + 1.
// Workgroups of a CU: as many as have the registers (168 a wave at D = 64, 256 at 128). A third at D = 64: 64 chunks of 100-300
// tokens 85 -> 78 us, 8 x 1,024 behind 4,000-8,000 293 -> 279.
constexpr int tiles_per_cu(int head_dim) { return head_dim == 64 ? 3 : 2; }

template <int D, int NT, typename T, bool TREE>
__device__ __forceinline__ void row_tile(const ChunkArgs& a, const Seq& s, int b, int tile, int kvh, int part,
                                         uint16_t* s_k0, uint16_t* s_v0, uint16_t* s_k1, uint16_t* s_v1, int& s_dirty) {
  constexpr int kKeys = 64, kTileElems = kKeys * D;
  constexpr int J = kTileElems * 2 / 1024 / kWaves;  // load instructions of a wave for K, and for V
  const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  constexpr int kRows = kTileRows * NT;
  const int r0 = tile * kRows * kWaves, total = s.nq * a.group;
  if (r0 >= total) return;
  const int kend = s.start + min(r0 + kRows * kWaves - 1, total - 1) / a.group + 1, kbeg = part * a.part_tokens;
  if (kbeg >= kend) return;
  const int kstop = min(kend, kbeg + a.part_tokens);
  const int tiles = (kstop - kbeg + kKeys - 1) / kKeys;

  const int32_t* bt = a.block_tables + (int64_t)b * a.bt_stride;
  const uint16_t* head_base = a.pool_layer + (int64_t)kvh * a.head_stride;
  typedef Rows<D, NT, 2, T, TREE> R;
  R w;
  const int wr0 = r0 + wave * kRows;  // the wave's first row; from total on: it only loads
  w.init(a, s, kvh, wr0);
  const bool has_rows = wr0 < total;
  const int lo = TREE ? s.start - 1 : s.start + r0 / a.group;  // every row of the workgroup sees the keys up to it
  if (threadIdx.x == 0) s_dirty = 0;
  Loader<D, J> load;
  const int first = wave * (kKeys / kWaves);
  const int at = first * D;
  Cursor c;  // the tile to fetch block ids of
  c.init(a, kbeg, kstop, kKeys);
  struct Place {
    int32_t id;
    int slot;
  };
  auto fetch = [&] {
    int entry;
    Place at;
    c.place(a, Loader<D, J>::own_key(first), entry, at.slot);
    c.next(a, kKeys);
    at.id = bt[entry];
    return at;
  };
  auto aim = [&](const Place& at) { load.aim(a, head_base, first, checked(a, at.id), at.slot); };
  // Tiles past the last one repeat its last key.
  Place at2, at3;
  {
    const Place at0 = fetch(), at1 = fetch();
    at2 = fetch();
    at3 = fetch();
    aim(at0);
    load.start(s_k0 + at, 0);
    load.start(s_v0 + at, a.kv_stride);
    aim(at1);
    load.start(s_k1 + at, 0);
  }
  w.flip(a.q_sign);
  typename R::Scores sc;
  wait_loads<0>();
  barrier();
  if (has_rows) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      u32x4 kf[D / 32];
      R::read_k(s_k0, h, kf);
      w.scores(kf, sc[h]);
    }
  }
  // The loader is aimed at tile t + 1 at the start.
  auto step = [&](int t, uint16_t* k_next, uint16_t* k_free, uint16_t* v_this, uint16_t* v_free) {
    wait_loads<0>();
    const int kt = kbeg + t * kKeys;
    if (kt + kKeys - 1 > lo && clean_values<T>(v_this + at, kTileElems / 8 / kWaves)) s_dirty = 1;
    barrier();
    load.start(v_free + at, a.kv_stride);
    aim(at2);
    load.start(k_free + at, 0);
    at2 = at3;
    at3 = fetch();
    if (has_rows && kt <= w.hi) {
      u32x4 kf[2][D / 32];
      R::read_k(k_next, 0, kf[0]);
      w.maxima(a, kt, sc);
      typename R::Weights wt;
#pragma unroll
      for (int h = 0; h < 4; ++h) {  // scores of the next tile beside the weights of this one
        if (h < 3) R::read_k(k_next, h + 1, kf[(h + 1) & 1]);
        f32x4 sn[NT];
        w.scores(kf[h & 1], sn);
        w.weights(a, h, sc[h], wt);
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[h][n] = sn[n];
        __builtin_amdgcn_sched_barrier(0);
      }
      w.sums(wt);
      w.values(v_this, wt);
    }
  };
  for (int t = 0; t < tiles; t += 2) {
    step(t, s_k1, s_k0, s_v0, s_v1);
    if (t + 1 >= tiles) break;
    step(t + 1, s_k0, s_k1, s_v1, s_v0);
  }
  wait_loads<0>();  // of tiles that were not needed
  if (!has_rows) return;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float l = w.l[n][0];
    const int r = wr0 + kTileRows * n + i;
    if (r >= total) continue;
    const int t = r / a.group, h = kvh * a.group + r - t * a.group;
    if (a.parts == 1) {
      const float inv = inverse<TREE>(a, s, t, l);
      uint16_t* op = a.out + (int64_t)(s.row0 + t) * a.out_stride + h * D + 4 * g;
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
        *reinterpret_cast<u32x2*>(op + 16 * d) =
            u32x2{pack2<T>(w.o[n][d][0] * inv, w.o[n][d][1] * inv), pack2<T>(w.o[n][d][2] * inv, w.o[n][d][3] * inv)};
    } else {
      const int64_t to = ((int64_t)(s.row0 + t) * a.num_heads + h) * a.parts + part;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) *reinterpret_cast<f32x4*>(a.part_o + to * D + 16 * d + 4 * g) = w.o[n][d];
      if (g == 0) *reinterpret_cast<f32x2*>(a.part_ml + to * 2) = f32x2{w.m[n], l};
    }
  }
  if (s_dirty == 0) return;
  // What was left out goes into what was just written, by the lane that wrote it.
  const int from = max(kbeg, (lo + 1) / kKeys * kKeys);
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {
    const int r = wr0 + kTileRows * n + i;
    if (r >= total) continue;
    const int t = r / a.group, h = kvh * a.group + r - t * a.group;
#pragma unroll 1
    for (int d = 4 * g; d < D; d += 16) {
      f32x4 more = {0.f, 0.f, 0.f, 0.f};
      add_left_out<T, TREE>(a, bt, head_base + d, D, from, min(kstop, s.start + t + 1), s, t, more);
      if (a.parts == 1) {
        uint16_t* op = a.out + (int64_t)(s.row0 + t) * a.out_stride + h * D + d;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (more[e] != 0.f) op[e] = (uint16_t)pack2<T>(more[e] + T::load(op[e]), 0.f);
      } else {
        float* op = a.part_o + (((int64_t)(s.row0 + t) * a.num_heads + h) * a.parts + part) * D + d;
#pragma unroll
        for (int e = 0; e < 4; ++e) op[e] += more[e];
      }
    }
  }
}

// One workgroup a (sequence, K/V head, part, row tile). The last row tiles see the most keys and go first. Tiles of one K/V
// head and part follow each other every 8th workgroup, so on one XCD, where these are a multiple of 8.
//
// Workgroups go to CUs in turn, so every other 256 of them are dealt backwards on each XCD: the CU with the longest gets
// the shortest of those beside it (8 x 1,023 tokens of 12 heads of 64 30.0 -> 28.3 us, 8 x 100-1,900 44 -> 42, 2 x 2,000 of
// 32 heads of 128 84 -> 81; 4 x 1,023 of these 55 -> 57).
template <int D, int NT, typename T, bool TREE>
__global__ __launch_bounds__(kWave* kWaves, tiles_per_cu(D)) void chunk_tiles_kernel(const ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t s_k0[64 * D], s_v0[64 * D], s_k1[64 * D], s_v1[64 * D];
  __shared__ int s_dirty;
  int idx = blockIdx.x;
  const int turn = idx / kCus;
  if (turn % 2 == 1 && (turn + 1) * kCus <= (int)gridDim.x)
    idx = turn * kCus + (kCus / kXcds - 1 - idx % kCus / kXcds) * kXcds + idx % kXcds;
  const int units = a.num_seqs * a.kv_heads * a.parts;
  const int tile = a.row_tiles - 1 - idx / units;
  idx %= units;
  const int kvh = idx % a.kv_heads;
  idx /= a.kv_heads;
  const int part = idx % a.parts, b = idx / a.parts;
  Seq s;
  if (!seq_of(a, b, part == 0 && tile == 0 && kvh == 0, s)) return;
  row_tile<D, NT, T, TREE>(a, s, b, tile, kvh, part, s_k0, s_v0, s_k1, s_v1, s_dirty);
}

// With more row tiles than run at once, workgroups that stay and take them from a queue, the most keys first: dispatched
// workgroups go to an XCD's CUs in turn, and one that has to wait for its CU holds up those behind it (4 x 2,048 tokens behind 768
// to 5,376: 330 of 512 workgroups at work on average).
constexpr int kQueueLine = 32;                           // words between counters: a 128-byte line each
constexpr int kQueueHead = (kXcds + 1) * kQueueLine;     // [0] pairs, then the counter of each XCD's share
constexpr int kOrderThreads = 1024, kBuckets = 2048;

__host__ __device__ inline int64_t queue_pairs(int64_t num_q_rows, int group, int rows_per_tile, int num_seqs) {
  return num_q_rows * group / rows_per_tile + num_seqs;  // a sequence's last row tile may be partly filled
}

// The (sequence, row tile) pairs by keys, most first (to 1 / kBuckets of the longest context), and the counters at zero.
__global__ __launch_bounds__(kOrderThreads) void chunk_order_kernel(const ChunkArgs a, int rows_per_tile) {
  __shared__ int s_count[kBuckets];
  __shared__ int s_wave[kOrderThreads / kWave];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  for (int i = tid; i < kBuckets; i += kOrderThreads) s_count[i] = 0;
  if (tid < kXcds) a.queue[(tid + 1) * kQueueLine] = 0;
  __syncthreads();
  const int64_t all = (int64_t)a.num_seqs * a.row_tiles;
  // The pair's bucket, or -1: no such tile.
  auto bucket = [&](int64_t i, int& b, int& tile) {
    b = (int)(i / a.row_tiles);
    tile = (int)(i - (int64_t)b * a.row_tiles);
    Seq s;
    s.row0 = a.cu_q[b];
    s.start = a.q_start[b];
    const int64_t nq = (int64_t)a.cu_q[b + 1] - s.row0;
    if (!fits(a, s, nq)) {
      if (nq != 0 && tile == 0) flag_error(a.d_error, TQ_DEVERR_LENGTH);
      return -1;
    }
    const int64_t r0 = (int64_t)tile * rows_per_tile, total = nq * a.group;
    if (r0 >= total) return -1;
    const int64_t keys = s.start + (min(r0 + rows_per_tile, total) - 1) / a.group;  // below max_context
    return kBuckets - 1 - (int)(keys * kBuckets / a.max_context);
  };
  int b, tile;
  for (int64_t i = tid; i < all; i += kOrderThreads) {
    const int k = bucket(i, b, tile);
    if (k >= 0) atomicAdd(&s_count[k], 1);
  }
  __syncthreads();
  // Counts to starts: two buckets a thread, summed over the wave, then over the waves.
  static_assert(kBuckets == 2 * kOrderThreads, "two buckets a thread");
  const int c0 = s_count[2 * tid], c1 = s_count[2 * tid + 1];
  int sum = c0 + c1;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int up = __shfl_up(sum, off);
    if (lane >= off) sum += up;
  }
  if (lane == kWave - 1) s_wave[wave] = sum;
  __syncthreads();
  int before = 0;
  for (int v = 0; v < wave; ++v) before += s_wave[v];
  s_count[2 * tid] = before + sum - c0 - c1;
  s_count[2 * tid + 1] = before + sum - c1;
  // More only where sequences share rows (cu_seqlens_q falls somewhere): those are left out.
  const int64_t room = queue_pairs(a.num_q_rows, a.group, rows_per_tile, a.num_seqs);
  if (tid == kOrderThreads - 1) {
    a.queue[0] = (int)min((int64_t)(before + sum), room);
    if (before + sum > room) flag_error(a.d_error, TQ_DEVERR_LENGTH);
  }
  __syncthreads();
  for (int64_t i = tid; i < all; i += kOrderThreads) {
    const int k = bucket(i, b, tile);
    if (k < 0) continue;
    const int at = atomicAdd(&s_count[k], 1);
    if (at >= room) continue;
    a.queue[kQueueHead + 2 * (int64_t)at] = b;
    a.queue[kQueueHead + 2 * (int64_t)at + 1] = tile;
  }
}

// Item f is pair f / kv_heads with K/V head f % kv_heads. XCD x takes the items f % 8 = x (with a multiple of 8 heads, heads of
// its own), then those that others left.
template <int D, int NT, typename T, bool TREE>
__global__ __launch_bounds__(kWave* kWaves, tiles_per_cu(D)) void chunk_queue_kernel(const ChunkArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t s_k0[64 * D], s_v0[64 * D], s_k1[64 * D], s_v1[64 * D];
  __shared__ int s_dirty;
  __shared__ int64_t s_item;
  const int64_t items = (int64_t)a.queue[0] * a.kv_heads;
  int turn = 0;  // shares that were found empty
  for (;;) {
    if (threadIdx.x == 0) {
      int64_t item = -1;
      while (turn < kXcds && item < 0) {
        const int x = (blockIdx.x + turn) % kXcds;
        const int64_t f = x + (int64_t)kXcds * atomicAdd(&a.queue[(x + 1) * kQueueLine], 1);
        if (f < items)
          item = f;
        else
          ++turn;
      }
      s_item = item;
    }
    __syncthreads();
    const int64_t item = s_item;
    if (item < 0) return;
    const int pair = __builtin_amdgcn_readfirstlane((int)(item / a.kv_heads));
    const int kvh = __builtin_amdgcn_readfirstlane((int)(item - (int64_t)pair * a.kv_heads));
    const int b = __builtin_amdgcn_readfirstlane(a.queue[kQueueHead + 2 * (int64_t)pair]);
    const int tile = __builtin_amdgcn_readfirstlane(a.queue[kQueueHead + 2 * (int64_t)pair + 1]);
    Seq s;
    seq_of(a, b, false, s);
    row_tile<D, NT, T, TREE>(a, s, b, tile, kvh, 0, s_k0, s_v0, s_k1, s_v1, s_dirty);
    __syncthreads();  // the buffers and s_item are free
  }
}

// Joins the parts of each (row, head). A lane first takes a part's maximum and weight sum, then some dims of all parts, whose loads
// do not depend on each other. 16 lanes a pair at D = 64, a wave at 128, where the pair's place is worked out once a wave (4 x 256
// rows of 12 heads of 64 in two parts: whole launch 24.6 us, with a wave a pair 35.5; 512 rows of 32 heads of 128: 21.7, with 32
// lanes a pair 25.6).
template <int D>
constexpr int kJoinLanes = D == 64 ? 16 : kWave;
template <int D>
constexpr int kJoinPairs = 256 / kJoinLanes<D>;

template <int D, typename T, bool TREE>
__global__ __launch_bounds__(256) void chunk_join_kernel(const ChunkArgs a) {
  constexpr int kLanes = kJoinLanes<D>, kDims = D / kLanes;
  typedef float Dims __attribute__((ext_vector_type(kDims)));
  const int lane = threadIdx.x % kLanes;
  const int tiles = (a.max_query_len * a.num_heads + kJoinPairs<D> - 1) / kJoinPairs<D>;
  const int b = blockIdx.x / tiles;
  int pair = (blockIdx.x - b * tiles) * kJoinPairs<D> + threadIdx.x / kLanes;
  if constexpr (kLanes == kWave) pair = __builtin_amdgcn_readfirstlane(pair);
  Seq s;
  if (!seq_of(a, b, false, s)) return;
  const int t = pair / a.num_heads, h = pair - t * a.num_heads;
  if (t >= s.nq) return;
  const int parts = (s.start + t) / a.part_tokens + 1;  // parts that the row sees
  const int64_t at = ((int64_t)(s.row0 + t) * a.num_heads + h) * a.parts;
  float top = -FLT_MAX, l = 0.f;
  Dims o = {};
  for (int p0 = 0; p0 < parts; p0 += kLanes) {
    const int n = min(kLanes, parts - p0);
    const f32x2 ml = lane < n ? *reinterpret_cast<const f32x2*>(a.part_ml + (at + p0 + lane) * 2) : f32x2{-FLT_MAX, 0.f};
    float most = ml[0];
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off));
    const float next = fmaxf(top, most), f = __builtin_amdgcn_exp2f(top - next);
    const float fp = lane < n ? __builtin_amdgcn_exp2f(ml[0] - next) : 0.f;
    float sum = lane < n ? fp * ml[1] : 0.f;
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    l = fmaf(l, f, sum);
    top = next;
#pragma unroll
    for (int k = 0; k < kDims; ++k) o[k] *= f;
    auto weight = [&](int p) {
      if constexpr (kLanes == kWave) return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, fp), p));
      return __shfl(fp, p, kLanes);
    };
    const float* op = a.part_o + (at + p0) * D + lane * kDims;
    int p = 0;
    for (; p + 8 <= n; p += 8) {
      Dims x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = *reinterpret_cast<const Dims*>(op + (int64_t)(p + e) * D);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float w = weight(p + e);
#pragma unroll
        for (int k = 0; k < kDims; ++k) o[k] = fmaf(w, x[e][k], o[k]);
      }
    }
    for (; p < n; ++p) {
      const float w = weight(p);
      const Dims x = *reinterpret_cast<const Dims*>(op + (int64_t)p * D);
#pragma unroll
      for (int k = 0; k < kDims; ++k) o[k] = fmaf(w, x[k], o[k]);
    }
  }
  const float inv = inverse<TREE>(a, s, t, l);
  uint16_t* to = a.out + (int64_t)(s.row0 + t) * a.out_stride + h * D + lane * kDims;
#pragma unroll
  for (int k = 0; k < kDims; k += 2) reinterpret_cast<uint32_t*>(to)[k / 2] = pack2<T>(o[k] * inv, o[k + 1] * inv);
}

// How a call is split: row tiles of `rows` rows per (sequence, K/V head), key parts of part_tokens.
struct Plan {
  int rows, row_tiles, parts, part_tokens;
  bool tiles;  // chunk_tiles_kernel or chunk_queue_kernel, else chunk_rows_kernel
  bool queue;
};

constexpr int kMaxContext = 1 << 30;  // positions a few tiles past it are still ints
// 16-row tiles of a wave of chunk_tiles_kernel. Three spill at D = 128 and are slower at 64 (16 x 100-1,900 tokens 190 -> 198 us).
constexpr int kTilesNt = 2;
// Row tiles of contexts up to this differ too little for the queue and its launch (direct -> queue): 16 prompts of 17-1,023 tokens
// 31 -> 38 us, 16 x 512 behind 512 151 -> 165, 4 x 2,048 168 -> 173; but 16 of 100-1,900 behind up to 2,000 224 -> 199, 64 of
// 100-500 behind up to 2,000 325 -> 267, 4 x 2,048 behind up to 6,144 696 -> 535.
constexpr int kQueueFrom = 2048;

// A tree has few rows, and the sequences of a batch have contexts of all lengths: parts of the longest one are empty for most others
// and their workgroups end at once. So trees are split into as many parts as would fit in four rounds (one round -> four: 32 trees of 9-33
// nodes behind 1,001-8,007 tokens, 32 / 4 heads of 64, 88 -> 75 us; 16 of 20-40 behind 100-12,000, 32 / 8 of 128, 174 -> 126; but 4 of
// 130 behind 3,000-6,000 72 -> 79). With equal lengths the parts are those that pay in both (8 of 64 nodes behind 4,000: 58). Parts
// worked out on the device from the lengths took as long as this, and 6 us more of every call.
constexpr int kTreeRounds = 4;

Plan plan_of(int num_seqs, int kv_heads, int group, int head_dim, int num_q_rows, int max_query_len, int max_context, bool tree) {
  Plan p;
  const int64_t rows = (int64_t)max_query_len * group;
  p.tiles = rows > 64;
  p.rows = p.tiles ? kTileRows * kTilesNt * kWaves : rows > 48 ? 64 : rows > 32 ? 48 : rows > 16 ? 32 : 16;
  p.row_tiles = (int)((rows + p.rows - 1) / p.rows);
  constexpr int kStep = kWaves * kTileKeys;
  const int64_t steps = ((int64_t)max_context + kStep - 1) / kStep;
  const int64_t groups = (int64_t)num_seqs * kv_heads * p.row_tiles;
  const int64_t want = kCus * (p.tiles ? tiles_per_cu(head_dim) : head_dim == 64 ? 2 : 1);
  // No second round for a few (259 tokens behind 32,500: 8 parts 220 us, 7 175), and no more parts than pay: steps go on beside
  // each other, but a launch is added and every pair of row and head has its sums written and read a part (us: measured on this
  // card). 16 x 256 tokens of 12 heads of 64 in one part 12 us, in two 25; 4 x 1,023 23 and 32; one token at 300 8.9 and 10.7; but
  // 300 tokens at 4,000 66 in one part, 23 in eight; one token at 4,000 30 in one, 12 in 32.
  const float step = (p.tiles ? 2.0f : 0.6f) * (head_dim == 64 ? 1.f : 1.3f), launch = 4.5f;
  const float pairs = 2e-6f * head_dim * num_q_rows * kv_heads * group;
  const float best = __builtin_sqrtf(steps * step / __builtin_fmaxf(pairs, 1e-6f));
  int64_t parts = (tree ? kTreeRounds : 1) * want / groups;
  if ((float)parts > best) parts = (int64_t)best;
  parts = parts < 1 ? 1 : parts > steps ? steps : parts;
  if (steps * step <= (float)((steps + parts - 1) / parts) * step + launch + pairs * parts) parts = 1;
  const int64_t per = (steps + parts - 1) / parts;
  p.part_tokens = (int)(per * kStep > 0x7fffffff - kStep ? 0x7fffffff / kStep * kStep : per * kStep);
  p.parts = (int)((steps + per - 1) / per);
  p.queue = p.tiles && p.parts == 1 && groups > want && max_context >= kQueueFrom;
  return p;
}

bool sizes_ok(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_q_rows,
              int32_t max_query_len, int32_t max_context) {
  return num_seqs >= 0 && num_heads >= 1 && num_kv_heads >= 1 && num_heads % num_kv_heads == 0 && head_dim >= 1 &&
         num_q_rows >= 0 && max_query_len >= 0 && max_context >= 0;
}

size_t workspace_of(const Plan& p, int32_t num_seqs, int32_t num_q_rows, int32_t num_heads, int32_t group,
                    int32_t head_dim) {
  if (p.queue) return (kQueueHead + 2 * (size_t)queue_pairs(num_q_rows, group, p.rows, num_seqs)) * sizeof(int32_t);
  return p.parts <= 1 ? 0 : (size_t)num_q_rows * num_heads * p.parts * (head_dim + 2) * sizeof(float);
}

template <int D, typename T, bool TREE>
tq_status launch(const ChunkArgs& a, const Plan& p, hipStream_t stream) {
  const int64_t grid = (int64_t)a.num_seqs * a.kv_heads * a.row_tiles * a.parts;
  const int64_t join = (int64_t)a.num_seqs * (((int64_t)a.max_query_len * a.num_heads + kJoinPairs<D> - 1) / kJoinPairs<D>);
  if (grid > 0x7fffffffLL || (!p.queue && !grid_fits(grid, kWave * kWaves)) || (a.parts > 1 && !grid_fits(join, 256)))
    return TQ_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid), t(kWave * kWaves);
  if (p.queue) {
    hipLaunchKernelGGL(chunk_order_kernel, dim3(1), dim3(kOrderThreads), 0, stream, a, p.rows);
    const tq_status st = check_launch();
    if (st != TQ_OK) return st;
    hipLaunchKernelGGL((chunk_queue_kernel<D, kTilesNt, T, TREE>), dim3(tiles_per_cu(D) * kCus), t, 0, stream, a);
  } else if (p.tiles)
    hipLaunchKernelGGL((chunk_tiles_kernel<D, kTilesNt, T, TREE>), g, t, 0, stream, a);
  else
    switch (p.rows) {
      case 16: hipLaunchKernelGGL((chunk_rows_kernel<D, 1, T, TREE>), g, t, 0, stream, a); break;
      case 32: hipLaunchKernelGGL((chunk_rows_kernel<D, 2, T, TREE>), g, t, 0, stream, a); break;
      case 48: hipLaunchKernelGGL((chunk_rows_kernel<D, 3, T, TREE>), g, t, 0, stream, a); break;
      default: hipLaunchKernelGGL((chunk_rows_kernel<D, 4, T, TREE>), g, t, 0, stream, a); break;
    }
  tq_status st = check_launch();
  if (st != TQ_OK || a.parts == 1) return st;
  hipLaunchKernelGGL((chunk_join_kernel<D, T, TREE>), dim3((unsigned)join), dim3(256), 0, stream, a);
  return check_launch();
}

template <bool TREE>
size_t workspace_size(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_q_rows,
                      int32_t max_query_len, int32_t max_context_len) {
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, num_q_rows, max_query_len, max_context_len) ||
      num_seqs == 0 || num_q_rows == 0 || max_query_len == 0 || max_context_len == 0 || max_context_len > kMaxContext)
    return 0;
  const int32_t group = num_heads / num_kv_heads;
  const Plan p = plan_of(num_seqs, num_kv_heads, group, head_dim, num_q_rows, max_query_len, max_context_len, TREE);
  return workspace_of(p, num_seqs, num_q_rows, num_heads, group, head_dim);
}

template <bool TREE>
tq_status attend(void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, const void* pool,
                 int64_t num_blocks, int32_t num_layers, int32_t num_heads, int32_t num_kv_heads, int32_t block_size,
                 int32_t head_dim, int32_t layer, const int32_t* block_tables, int64_t block_table_stride,
                 int32_t max_blocks_per_seq, const int32_t* cu_seqlens_q, const int32_t* q_start, const int64_t* masks,
                 int64_t mask_words, int32_t num_seqs, int32_t num_q_rows, int32_t max_query_len, int32_t max_context_len,
                 float scale, int32_t dtype, void* workspace, size_t workspace_bytes, int32_t* d_error, void* stream) {
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, num_q_rows, max_query_len, max_context_len) ||
      num_blocks < 1 || num_blocks > 0x7fffffffLL || num_layers < 1 || block_size < 1 || layer < 0 ||
      layer >= num_layers || max_blocks_per_seq < 0 || !(scale - scale == 0.f))
    return TQ_ERR_INVALID_ARGUMENT;
  if ((head_dim != 64 && head_dim != 128) || block_size > kMaxBlockSize || (dtype != TQ_F16 && dtype != TQ_BF16) ||
      max_context_len > kMaxContext)
    return TQ_ERR_UNSUPPORTED;
  if (num_seqs == 0 || num_q_rows == 0 || max_query_len == 0) return TQ_OK;
  const int64_t width = (int64_t)num_heads * head_dim;
  if (out == nullptr || q == nullptr || pool == nullptr || block_tables == nullptr || cu_seqlens_q == nullptr ||
      q_start == nullptr || block_table_stride < max_blocks_per_seq || out_row_stride < width ||
      q_row_stride < width || max_context_len < 1)
    return TQ_ERR_INVALID_ARGUMENT;
  if (TREE && (masks == nullptr || mask_words > 0x3fffffffLL || mask_words * 64 < max_query_len)) return TQ_ERR_INVALID_ARGUMENT;
  // 16-byte loads of q and the pool, 8-byte stores of out.
  if (((uintptr_t)q | (uintptr_t)pool) % 16 != 0 || (uintptr_t)out % 8 != 0 || q_row_stride % 8 != 0 ||
      out_row_stride % 4 != 0)
    return TQ_ERR_INVALID_ARGUMENT;
  if ((int64_t)max_query_len * num_heads > 0x7fffffffLL - 65536) return TQ_ERR_UNSUPPORTED;

  const int32_t group = num_heads / num_kv_heads;
  const Plan p = plan_of(num_seqs, num_kv_heads, group, head_dim, num_q_rows, max_query_len, max_context_len, TREE);
  const size_t need = workspace_of(p, num_seqs, num_q_rows, num_heads, group, head_dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0))
    return TQ_ERR_WORKSPACE;

  const PoolGeom g = pool_geom(num_layers, num_kv_heads, block_size, head_dim, layer);
  if (g.block_stride > 0x7fffffffLL) return TQ_ERR_UNSUPPORTED;
  ChunkArgs a;
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_row_stride;
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_row_stride;
  a.pool_layer = static_cast<const uint16_t*>(pool) + g.layer_offset;
  a.block_stride = (uint32_t)g.block_stride;
  a.kv_stride = g.kv_stride;
  a.head_stride = g.head_stride;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.cu_q = cu_seqlens_q;
  a.q_start = q_start;
  a.masks = reinterpret_cast<const uint32_t*>(masks);
  a.mask_words = 2 * mask_words;
  a.queue = p.queue ? static_cast<int32_t*>(workspace) : nullptr;
  a.part_o = p.parts > 1 ? static_cast<float*>(workspace) : nullptr;
  a.part_ml = a.part_o == nullptr ? nullptr : a.part_o + (size_t)num_q_rows * num_heads * p.parts * head_dim;
  a.d_error = d_error;
  // A scale of zero weighs every visible key alike: the smallest positive factor does the same, and keeps
  // the masked scores' -inf from becoming NaN.
  const float c = scale * kLog2e;
  a.c = c == 0.f ? FLT_MIN : c < 0.f ? -c : c;
  a.q_sign = c < 0.f ? 0x80008000u : 0u;
  a.num_blocks = (int32_t)num_blocks;
  a.num_heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.group = group;
  a.block_size = block_size;
  a.inv_block = ((1u << 21) + block_size - 1) / block_size;
  a.max_blocks = max_blocks_per_seq;
  a.num_q_rows = num_q_rows;
  a.max_query_len = max_query_len;
  a.max_context = max_context_len;
  a.num_seqs = num_seqs;
  a.row_tiles = p.row_tiles;
  a.parts = p.parts;
  a.part_tokens = p.part_tokens;
  const hipStream_t st = (hipStream_t)stream;
  if (head_dim == 64)
    return dtype == TQ_BF16 ? launch<64, Bf16, TREE>(a, p, st) : launch<64, Fp16, TREE>(a, p, st);
  return dtype == TQ_BF16 ? launch<128, Bf16, TREE>(a, p, st) : launch<128, Fp16, TREE>(a, p, st);
}

}  // namespace
}  // namespace tq

extern "C" size_t tq_paged_chunk_workspace_size(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                                int32_t head_dim, int32_t num_q_rows, int32_t max_query_len,
                                                int32_t max_context_len) {
  return tq::workspace_size<false>(num_seqs, num_heads, num_kv_heads, head_dim, num_q_rows, max_query_len, max_context_len);
}

extern "C" size_t tq_paged_tree_workspace_size(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                               int32_t head_dim, int32_t num_q_rows, int32_t max_query_len,
                                               int32_t max_context_len) {
  return tq::workspace_size<true>(num_seqs, num_heads, num_kv_heads, head_dim, num_q_rows, max_query_len, max_context_len);
}

extern "C" tq_status tq_paged_chunk(void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride,
                                    const void* pool, int64_t num_blocks, int32_t num_layers, int32_t num_heads,
                                    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, int32_t layer,
                                    const int32_t* block_tables, int64_t block_table_stride,
                                    int32_t max_blocks_per_seq, const int32_t* cu_seqlens_q, const int32_t* q_start,
                                    int32_t num_seqs, int32_t num_q_rows, int32_t max_query_len,
                                    int32_t max_context_len, float scale, int32_t dtype, void* workspace,
                                    size_t workspace_bytes, int32_t* d_error, void* stream) {
  return tq::attend<false>(out, out_row_stride, q, q_row_stride, pool, num_blocks, num_layers, num_heads, num_kv_heads, block_size,
                           head_dim, layer, block_tables, block_table_stride, max_blocks_per_seq, cu_seqlens_q, q_start, nullptr, 0,
                           num_seqs, num_q_rows, max_query_len, max_context_len, scale, dtype, workspace, workspace_bytes,
                           d_error, stream);
}

extern "C" tq_status tq_paged_tree(void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride,
                                    const void* pool, int64_t num_blocks, int32_t num_layers, int32_t num_heads,
                                    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, int32_t layer,
                                    const int32_t* block_tables, int64_t block_table_stride,
                                    int32_t max_blocks_per_seq, const int32_t* cu_seqlens_q, const int32_t* q_start,
                                    const int64_t* masks, int64_t mask_words,
                                    int32_t num_seqs, int32_t num_q_rows, int32_t max_query_len,
                                    int32_t max_context_len, float scale, int32_t dtype, void* workspace,
                                    size_t workspace_bytes, int32_t* d_error, void* stream) {
  return tq::attend<true>(out, out_row_stride, q, q_row_stride, pool, num_blocks, num_layers, num_heads, num_kv_heads, block_size,
                          head_dim, layer, block_tables, block_table_stride, max_blocks_per_seq, cu_seqlens_q, q_start, masks, mask_words,
                          num_seqs, num_q_rows, max_query_len, max_context_len, scale, dtype, workspace, workspace_bytes,
                          d_error, stream);
}

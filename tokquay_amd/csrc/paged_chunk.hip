// Attention of chunks of new tokens over a paged 16-bit cache, heads grouped: G = H / Hkv query
// heads read each K/V head.
//
//   out[t, h] = sum_j p_j V[j, h / G] / sum_j p_j,   p_j = 2^(c (q[t, h] . K[j, h / G]) - m),   j <= q_start + t
//
// with c = scale log2(e) and m a running maximum (any m gives the same quotient; it is raised when a score
// passes it by more than kSlack, so p stays below 2^8 and the sums are rescaled rarely). The G heads of a
// token read the same keys, so (token, head of the group) pairs are the rows of one matrix product: row r
// is token r / G, head r % G of the group, and a 16-row tile holds 16 / G tokens.
//
// Per 16 rows and 32 keys, on the 16x16x32 matrix instructions (fp32 sums):
//
//   S^T[key][row] = K[key][:] . Q[row][:]            D / 32 depth steps for each 16 keys
//   O^T[dim][row] += V^T[dim][key] P^T[key][row]     one depth step for each 16 dims
//
// The transposed scores leave lane (i, g) = (lane % 16, lane / 16) with row i and the keys 4 g + 0..3 and
// 16 + 4 g + 0..3, so one lane's scores belong to one row (its position is one register, its maximum and
// sum are taken in the lane and across four lanes at the end) and are, rounded to 16 bits, the B operand
// of the second product with no exchange: that product may take the keys in any order, and V^T is read in
// the same one (two transposing LDS reads of 4 keys each). Rounding p to the cache's type costs each weight half a
// step, as much as the rounding of the output; its sum is taken before the rounding.
//
// K and V come in 32-key tiles straight from HBM into LDS (16 bytes a lane, no registers), a tile ahead
// of the products. 16-byte pieces are permuted inside a row as they arrive (swizzled), so that the 16 keys
// that one LDS read takes lie in different banks.
#include <float.h>

#include "half_types.h"

namespace tq {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;  // log2 units a score may exceed the running maximum by
constexpr int kTileKeys = 32;  // keys of a tile
constexpr int kTileRows = 16;  // rows of a tile
constexpr int kWaves = 4;

struct ChunkArgs {
  uint16_t* out;
  int64_t out_stride;
  const uint16_t* q;
  int64_t q_stride;
  const uint16_t* pool_layer;
  int64_t block_stride;
  int64_t kv_stride;
  int64_t head_stride;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* cu_q;
  const int32_t* q_start;
  float* part_o;   // [num_q_rows][num_heads][parts][D] sums of each part, or null: one part
  float* part_ml;  // [num_q_rows][num_heads][parts][2] maximum and weight sum
  int32_t* d_error;
  float c;         // |scale| log2(e)
  uint32_t q_sign; // 0x80008000 where the scale is negative: the queries' signs are flipped
  int32_t num_blocks;
  int32_t num_heads;
  int32_t kv_heads;
  int32_t group;
  int32_t block_size;
  int32_t max_blocks;
  int32_t num_q_rows;
  int32_t max_query_len;
  int32_t max_context;
  int32_t num_seqs;
  int32_t row_tiles;    // workgroup row tiles per (sequence, K/V head)
  int32_t parts;        // key parts per row tile
  int32_t part_tokens;  // keys of a part, a multiple of kWaves * kTileKeys
};

__device__ __forceinline__ float max2(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A sequence's rows and positions, or why it has none here.
struct Seq {
  int row0, nq, start;
};

// False where the sequence has no rows or its lengths do not fit (flagged by the workgroup that `reports`).
__device__ __forceinline__ bool seq_of(const ChunkArgs& a, int b, bool reports, Seq& s) {
  s.row0 = __builtin_amdgcn_readfirstlane(a.cu_q[b]);
  const int64_t nq = (int64_t)__builtin_amdgcn_readfirstlane(a.cu_q[b + 1]) - s.row0;
  s.start = __builtin_amdgcn_readfirstlane(a.q_start[b]);
  if (nq == 0) return false;
  const int64_t end = (int64_t)s.start + nq;
  const bool ok = nq > 0 && nq <= a.max_query_len && s.row0 >= 0 && s.row0 + nq <= a.num_q_rows && s.start >= 0 &&
                  end <= a.max_context && end <= (int64_t)a.max_blocks * a.block_size;
  if (!ok && reports && threadIdx.x == 0) flag_error(a.d_error, TQ_DEVERR_LENGTH);
  s.nq = (int)nq;
  return ok;
}

// 16-byte piece p of a tile's key `key` lies at piece p ^ swizzle(key) of the key's row in LDS: reads take
// the same piece of 16 consecutive keys, or two neighbouring ones, and 256 bytes cover all banks once.
template <int D>
__device__ __forceinline__ int swizzle(int key) {
  return D == 128 ? key & 15 : (key >> 1) & 7;
}

// Starts the copy of keys kt .. kt + 31 of one K/V head into LDS (K, then V), by one wave. Keys from kend on
// are the last one again: finite wherever it is, and masked.
template <int D>
__device__ __forceinline__ void load_tile(const ChunkArgs& a, const int32_t* bt, const uint16_t* head_base, int kt,
                                          int kend, uint16_t* s_k, uint16_t* s_v) {
  constexpr int kLanes = D / 8;             // lanes a key row takes, 16 bytes each
  constexpr int kKeys = kWave / kLanes;     // keys of one instruction
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int j = 0; j < kTileKeys / kKeys; ++j) {
    const int local = j * kKeys + lane / kLanes;
    const int key = min(kt + local, kend - 1);
    const int ti = key / a.block_size;
    int32_t blk = bt[ti];
    if ((uint32_t)blk >= (uint32_t)a.num_blocks) {
      flag_error(a.d_error, TQ_DEVERR_BLOCK_ID);
      blk = 0;
    }
    const uint16_t* src = head_base + (int64_t)blk * a.block_stride + (int64_t)(key - ti * a.block_size) * D +
                          8 * ((lane % kLanes) ^ swizzle<D>(local));
    typedef const __attribute__((address_space(1))) void* Global;
    typedef __attribute__((address_space(3))) void* Lds;
    __builtin_amdgcn_global_load_lds((Global)src, (Lds)(s_k + j * kKeys * D), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((Global)(src + a.kv_stride), (Lds)(s_v + j * kKeys * D), 16, 0, 0);
  }
}

// s_waitcnt vmcnt(0) lgkmcnt(0): the tile that was loaded is in LDS, and what was read of the other one is in registers.
__device__ __forceinline__ void wait_tile() {
  __builtin_amdgcn_s_waitcnt(0x0070);
  __builtin_amdgcn_sched_barrier(0);
}

// The rows of one wave: queries, sums, running maxima.
template <int D, int NT, typename T>
struct Rows {
  u32x4 q[NT][D / 32];
  f32x4 o[NT][D / 16];
  float m[NT], mthr[NT], l[NT];
  int qpos[NT];
  int lo, hi;  // positions of the first and last row (uniform)

  __device__ __forceinline__ void init(const ChunkArgs& a, const Seq& s, int kvh, int r0) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
    const int last = s.nq * a.group - 1;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = min(r0 + kTileRows * n + i, last), t = r / a.group;
      const uint16_t* qp = a.q + (int64_t)(s.row0 + t) * a.q_stride + (kvh * a.group + r - t * a.group) * D + 8 * g;
#pragma unroll
      for (int k = 0; k < D / 32; ++k)
        q[n][k] = *reinterpret_cast<const u32x4*>(qp + 32 * k) ^ a.q_sign;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      qpos[n] = s.start + t;
      m[n] = -FLT_MAX;
      mthr[n] = -FLT_MAX;
      l[n] = 0.f;
    }
    lo = s.start + min(r0, last) / a.group;
    hi = s.start + min(r0 + kTileRows * NT - 1, last) / a.group;
  }

  // One tile of keys kt .. kt + 31, of which those from kend on are not there.
  __device__ __forceinline__ void tile(const ChunkArgs& a, int kt, const uint16_t* s_k, const uint16_t* s_v) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
    f32x4 s[2][NT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[h][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const int key = 16 * h + i;
        const u32x4 kf = *reinterpret_cast<const u32x4*>(s_k + key * D + 8 * ((4 * k + g) ^ swizzle<D>(key)));
#pragma unroll
        for (int n = 0; n < NT; ++n) s[h][n] = T::mfma(kf, q[n][k], s[h][n]);
      }
    }
    const bool masked = kt + kTileKeys - 1 > lo;  // uniform: some row does not see some key
    if (masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[h][n][e] = kt + 16 * h + 4 * g + e <= qpos[n] ? s[h][n][e] : -INFINITY;
    }
    float p[NT][8];
    u32x4 pf[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = max2(max2(max2(s[0][n][0], s[0][n][1]), max2(s[0][n][2], s[0][n][3])),
                       max2(max2(s[1][n][0], s[1][n][1]), max2(s[1][n][2], s[1][n][3])));
      top *= a.c;
      if (__builtin_amdgcn_ballot_w64(top > mthr[n]) != 0) {
        top = max2(top, __shfl_xor(top, 16));
        top = max2(top, __shfl_xor(top, 32));
        const bool grow = top > mthr[n];
        const float next = grow ? top : m[n];
        const float corr = grow ? __builtin_amdgcn_exp2f(m[n] - next) : 1.f;
        l[n] *= corr;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[n][d] *= corr;
        m[n] = next;
        mthr[n] = next + kSlack;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) p[n][e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][n][e & 3], a.c, -m[n]));
      l[n] += ((p[n][0] + p[n][1]) + (p[n][2] + p[n][3])) + ((p[n][4] + p[n][5]) + (p[n][6] + p[n][7]));
#pragma unroll
      for (int e = 0; e < 4; ++e) pf[n][e] = pack2<T>(p[n][2 * e], p[n][2 * e + 1]);
    }
    if (masked && not_finite(s_v)) {
      visible_values(kt, s_v, p);
      return;
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const u32x4 vf = read_v(s_v, d);
#pragma unroll
      for (int n = 0; n < NT; ++n) o[n][d] = T::mfma(vf, pf[n], o[n][d]);
    }
  }

  // V^T of dims 16 d + 0..15: dim 16 d + i, keys 4 g + 0..3 and 16 + 4 g + 0..3. Of 16 lanes, lane 4 a + b names
  // four values of key a and gets value (its own index) of keys 0..3.
  static __device__ __forceinline__ u32x4 read_v(const uint16_t* s_v, int d) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
    u32x2 half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = 16 * h + 4 * g + (i >> 2), piece = 2 * d + ((i >> 1) & 1);
      const uint16_t* at = s_v + key * D + 8 * (piece ^ swizzle<D>(key)) + 4 * (i & 1);
      half[h] = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at)));
    }
    return u32x4{half[0][0], half[0][1], half[1][0], half[1][1]};
  }

  // Whether the tile's V holds an infinity or a NaN (uniform).
  static __device__ __forceinline__ bool not_finite(const uint16_t* s_v) {
    const int lane = threadIdx.x & (kWave - 1);
    bool bad = false;
#pragma unroll 1
    for (int j = lane; j < kTileKeys * D / 8; j += kWave) {
      const u32x4 v = reinterpret_cast<const u32x4*>(s_v)[j];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        bad |= (v[e] & T::kExponent) == T::kExponent || ((v[e] >> 16) & T::kExponent) == T::kExponent;
    }
    return __builtin_amdgcn_ballot_w64(bad) != 0;
  }

  // The second product of a tile whose V is not finite and that some row does not see all of: a weight of
  // zero times infinity is NaN, so each key's values reach only the rows that see it.
  __device__ __forceinline__ void visible_values(int kt, const uint16_t* s_v, const float (&p)[NT][8]) {
    const int lane = threadIdx.x & (kWave - 1), i = lane & 15, g = lane >> 4;
#pragma unroll 1
    for (int key = 0; key < kTileKeys; ++key) {
      const int from = 16 * ((key >> 2) & 3) + i, slot = 4 * (key >> 4) + (key & 3);
      float w[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        w[n] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[n] = e == slot ? p[n][e] : w[n];
        w[n] = __shfl(w[n], from);
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const int dim = 16 * d + 4 * g;
        const u32x2 v = *reinterpret_cast<const u32x2*>(s_v + key * D + 8 * ((dim >> 3) ^ swizzle<D>(key)) + (dim & 7));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float f = T::load((uint16_t)(v[r >> 1] >> (16 * (r & 1))));
#pragma unroll
          for (int n = 0; n < NT; ++n) o[n][d][r] = kt + key <= qpos[n] ? fmaf(w[n], f, o[n][d][r]) : o[n][d][r];
        }
      }
    }
  }
};

// Few rows: a workgroup takes 16 NT rows and one part of the keys; its waves take every fourth tile of the
// part, each with its own two tile buffers in LDS and no barrier, and join their sums in LDS at the end.
template <int D, int NT, typename T>
__global__ __launch_bounds__(kWave* kWaves) void chunk_rows_kernel(const ChunkArgs a) {
  constexpr int kTileElems = kTileKeys * D;
  // Two buffers of K and V for each wave; at the end the waves' sums (D + 4 floats a row keep rows apart).
  constexpr int kSumFloats = kWaves * kTileRows * NT * (D + 4);
  constexpr int kBytes = kWaves * 4 * kTileElems * 2 > kSumFloats * 4 ? kWaves * 4 * kTileElems * 2 : kSumFloats * 4;
  __shared__ __attribute__((aligned(16))) char s_mem[kBytes];
  __shared__ float s_ml[kWaves][kTileRows * NT][2];
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
  Rows<D, NT, T> w;
  w.init(a, s, kvh, r0);
  const int kend = w.hi + 1, kbeg = part * a.part_tokens;
  if (kbeg >= kend) return;
  const int kstop = min(kend, kbeg + a.part_tokens);

  const int32_t* bt = a.block_tables + (int64_t)b * a.bt_stride;
  const uint16_t* head_base = a.pool_layer + (int64_t)kvh * a.head_stride;
  uint16_t* s_tile = reinterpret_cast<uint16_t*>(s_mem) + wave * 4 * kTileElems;
  constexpr int kStep = kWaves * kTileKeys;
  int kt = kbeg + wave * kTileKeys, buf = 0;
  if (kt < kstop) load_tile<D>(a, bt, head_base, kt, kend, s_tile, s_tile + kTileElems);
  for (; kt < kstop; kt += kStep) {
    wait_tile();
    const int nbuf = buf ^ 1;
    if (kt + kStep < kstop)
      load_tile<D>(a, bt, head_base, kt + kStep, kend, s_tile + nbuf * 2 * kTileElems,
                   s_tile + nbuf * 2 * kTileElems + kTileElems);
    w.tile(a, kt, s_tile + buf * 2 * kTileElems, s_tile + buf * 2 * kTileElems + kTileElems);
    buf = nbuf;
  }

  // Join: m is the same in the four lanes of a row, l is each lane's own keys'.
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(s_mem);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float l = w.l[n];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = kTileRows * n + i;
    if (g == 0) {
      s_ml[wave][r][0] = w.m[n];
      s_ml[wave][r][1] = l;
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
      *reinterpret_cast<f32x4*>(s_o + (wave * kTileRows * NT + r) * (D + 4) + 16 * d + 4 * g) = w.o[n][d];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < rows * (D / 4); e += kWave * kWaves) {
    const int r = e / (D / 4), d = 4 * (e % (D / 4));
    float top = s_ml[0][r][0];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) top = fmaxf(top, s_ml[v][r][0]);
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f(s_ml[v][r][0] - top);
      l = fmaf(f, s_ml[v][r][1], l);
      const f32x4 ov = *reinterpret_cast<const f32x4*>(s_o + (v * kTileRows * NT + r) * (D + 4) + d);
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = fmaf(f, ov[k], o[k]);
    }
    const int t = (r0 + r) / a.group, h = kvh * a.group + (r0 + r) - t * a.group;
    if (a.parts == 1) {
      const float inv = 1.f / l;
      *reinterpret_cast<u32x2*>(a.out + (int64_t)(s.row0 + t) * a.out_stride + h * D + d) =
          u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
    } else {
      const int64_t at = ((int64_t)(s.row0 + t) * a.num_heads + h) * a.parts + part;
      *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = o;
      if (d == 0) *reinterpret_cast<f32x2*>(a.part_ml + at * 2) = f32x2{top, l};
    }
  }
}

// Joins the parts of each (row, head): D / 4 lanes a pair, four dims each.
template <int D, typename T>
__global__ __launch_bounds__(256) void chunk_join_kernel(const ChunkArgs a) {
  constexpr int kLanes = D / 4, kPairs = 256 / kLanes;
  const int tiles = (a.max_query_len * a.num_heads + kPairs - 1) / kPairs;
  const int b = blockIdx.x / tiles, pair = (blockIdx.x - b * tiles) * kPairs + threadIdx.x / kLanes;
  Seq s;
  if (!seq_of(a, b, false, s)) return;
  const int t = pair / a.num_heads, h = pair - t * a.num_heads;
  if (t >= s.nq) return;
  const int d = 4 * (threadIdx.x % kLanes);
  const int parts = (s.start + t) / a.part_tokens + 1;  // parts that the row sees
  const int64_t at = ((int64_t)(s.row0 + t) * a.num_heads + h) * a.parts;
  float top = -FLT_MAX, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < parts; ++p) {
    const f32x2 ml = *reinterpret_cast<const f32x2*>(a.part_ml + (at + p) * 2);
    const f32x4 op = *reinterpret_cast<const f32x4*>(a.part_o + (at + p) * D + d);
    const float next = fmaxf(top, ml[0]);
    const float f = __builtin_amdgcn_exp2f(top - next), fp = __builtin_amdgcn_exp2f(ml[0] - next);
    l = fmaf(fp, ml[1], l * f);
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = fmaf(fp, op[k], o[k] * f);
    top = next;
  }
  const float inv = 1.f / l;
  *reinterpret_cast<u32x2*>(a.out + (int64_t)(s.row0 + t) * a.out_stride + h * D + d) =
      u32x2{pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv)};
}

// How a call is split: row tiles of 16 nt rows per (sequence, K/V head), key parts of part_tokens.
struct Plan {
  int nt, row_tiles, parts, part_tokens;
};

constexpr int kCus = 256;

Plan plan_of(int num_seqs, int kv_heads, int group, int max_query_len, int max_context) {
  Plan p;
  const int64_t rows = (int64_t)max_query_len * group;
  p.nt = rows > 48 ? 4 : rows > 32 ? 3 : rows > 16 ? 2 : 1;
  p.row_tiles = (int)((rows + kTileRows * p.nt - 1) / (kTileRows * p.nt));
  constexpr int kStep = kWaves * kTileKeys;
  const int64_t steps = ((int64_t)max_context + kStep - 1) / kStep;
  const int64_t groups = (int64_t)num_seqs * kv_heads * p.row_tiles;
  int64_t parts = (kCus + groups - 1) / groups;
  if (parts > steps) parts = steps;
  const int64_t per = (steps + parts - 1) / parts;
  p.part_tokens = (int)(per * kStep > 0x7fffffff - kStep ? 0x7fffffff / kStep * kStep : per * kStep);
  p.parts = (int)((steps + per - 1) / per);
  return p;
}

bool sizes_ok(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_q_rows,
              int32_t max_query_len, int32_t max_context) {
  return num_seqs >= 0 && num_heads >= 1 && num_kv_heads >= 1 && num_heads % num_kv_heads == 0 && head_dim >= 1 &&
         num_q_rows >= 0 && max_query_len >= 0 && max_context >= 0;
}

size_t workspace_of(const Plan& p, int32_t num_q_rows, int32_t num_heads, int32_t head_dim) {
  return p.parts <= 1 ? 0 : (size_t)num_q_rows * num_heads * p.parts * (head_dim + 2) * sizeof(float);
}

template <int D, typename T>
tq_status launch(const ChunkArgs& a, const Plan& p, hipStream_t stream) {
  const int64_t grid = (int64_t)a.num_seqs * a.kv_heads * a.row_tiles * a.parts;
  const int64_t join = (int64_t)a.num_seqs * (((int64_t)a.max_query_len * a.num_heads + 1024 / D - 1) / (1024 / D));
  if (grid > 0x7fffffffLL || (a.parts > 1 && join > 0x7fffffffLL)) return TQ_ERR_UNSUPPORTED;
  const dim3 g((unsigned)grid), t(kWave * kWaves);
  switch (p.nt) {
    case 1: hipLaunchKernelGGL((chunk_rows_kernel<D, 1, T>), g, t, 0, stream, a); break;
    case 2: hipLaunchKernelGGL((chunk_rows_kernel<D, 2, T>), g, t, 0, stream, a); break;
    case 3: hipLaunchKernelGGL((chunk_rows_kernel<D, 3, T>), g, t, 0, stream, a); break;
    default: hipLaunchKernelGGL((chunk_rows_kernel<D, 4, T>), g, t, 0, stream, a); break;
  }
  tq_status st = check_launch();
  if (st != TQ_OK || a.parts == 1) return st;
  hipLaunchKernelGGL((chunk_join_kernel<D, T>), dim3((unsigned)join), dim3(256), 0, stream, a);
  return check_launch();
}

}  // namespace
}  // namespace tq

extern "C" size_t tq_paged_chunk_workspace_size(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                                int32_t head_dim, int32_t num_q_rows, int32_t max_query_len,
                                                int32_t max_context_len) {
  using namespace tq;
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, num_q_rows, max_query_len, max_context_len) ||
      num_seqs == 0 || num_q_rows == 0 || max_query_len == 0 || max_context_len == 0)
    return 0;
  return workspace_of(plan_of(num_seqs, num_kv_heads, num_heads / num_kv_heads, max_query_len, max_context_len),
                      num_q_rows, num_heads, head_dim);
}

extern "C" tq_status tq_paged_chunk(void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride,
                                    const void* pool, int64_t num_blocks, int32_t num_layers, int32_t num_heads,
                                    int32_t num_kv_heads, int32_t block_size, int32_t head_dim, int32_t layer,
                                    const int32_t* block_tables, int64_t block_table_stride,
                                    int32_t max_blocks_per_seq, const int32_t* cu_seqlens_q, const int32_t* q_start,
                                    int32_t num_seqs, int32_t num_q_rows, int32_t max_query_len,
                                    int32_t max_context_len, float scale, int32_t dtype, void* workspace,
                                    size_t workspace_bytes, int32_t* d_error, void* stream) {
  using namespace tq;
  if (!sizes_ok(num_seqs, num_heads, num_kv_heads, head_dim, num_q_rows, max_query_len, max_context_len) ||
      num_blocks < 1 || num_blocks > 0x7fffffffLL || num_layers < 1 || block_size < 1 || layer < 0 ||
      layer >= num_layers || max_blocks_per_seq < 0 || !(scale - scale == 0.f))
    return TQ_ERR_INVALID_ARGUMENT;
  if ((head_dim != 64 && head_dim != 128) || block_size > kMaxBlockSize || (dtype != TQ_F16 && dtype != TQ_BF16))
    return TQ_ERR_UNSUPPORTED;
  if (num_seqs == 0 || num_q_rows == 0 || max_query_len == 0) return TQ_OK;
  const int64_t width = (int64_t)num_heads * head_dim;
  if (out == nullptr || q == nullptr || pool == nullptr || block_tables == nullptr || cu_seqlens_q == nullptr ||
      q_start == nullptr || block_table_stride < max_blocks_per_seq || out_row_stride < width ||
      q_row_stride < width || max_context_len < 1)
    return TQ_ERR_INVALID_ARGUMENT;
  // 16-byte loads of q and the pool, 8-byte stores of out.
  if (((uintptr_t)q | (uintptr_t)pool) % 16 != 0 || (uintptr_t)out % 8 != 0 || q_row_stride % 8 != 0 ||
      out_row_stride % 4 != 0)
    return TQ_ERR_INVALID_ARGUMENT;
  if ((int64_t)max_query_len * num_heads > 0x7fffffffLL - 65536) return TQ_ERR_UNSUPPORTED;

  const int32_t group = num_heads / num_kv_heads;
  const Plan p = plan_of(num_seqs, num_kv_heads, group, max_query_len, max_context_len);
  const size_t need = workspace_of(p, num_q_rows, num_heads, head_dim);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0))
    return TQ_ERR_WORKSPACE;

  const PoolGeom g = pool_geom(num_layers, num_kv_heads, block_size, head_dim, layer);
  ChunkArgs a;
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_row_stride;
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_row_stride;
  a.pool_layer = static_cast<const uint16_t*>(pool) + g.layer_offset;
  a.block_stride = g.block_stride;
  a.kv_stride = g.kv_stride;
  a.head_stride = g.head_stride;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.cu_q = cu_seqlens_q;
  a.q_start = q_start;
  a.part_o = static_cast<float*>(workspace);
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
    return dtype == TQ_BF16 ? launch<64, Bf16>(a, p, st) : launch<64, Fp16>(a, p, st);
  return dtype == TQ_BF16 ? launch<128, Bf16>(a, p, st) : launch<128, Fp16>(a, p, st);
}

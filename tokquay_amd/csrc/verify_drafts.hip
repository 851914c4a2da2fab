// Verification of drafted tokens: speculative sampling's accept / resample rule on given random numbers.
//
// Sequence b has rows lo .. last of logits: row lo + i judges its i-th drafted token x_i, the last row follows them
// all. With p the row's distribution, softmax(logits / T) (all of it on the largest logit where T = 0), and q the
// one the draft was drawn from (all of it on the draft where none is given):
//
//   token i stands while u_i q(x_i) < p(x_i); at the first that does not, the next token is drawn from
//   max(p - q, 0); after the last one from p. The draw: the lowest j with w_0 + .. + w_j > u_last sum(w).
//
// Which side of a border of that running sum u_last falls on decides a token, and 100,000 borders lie
// close: sums are fp64, of exponentials that are off by at most 2.2e-12 (fp64 FMAs run at the fp32 rate here). A chunk's sum
// is made of two of them, its columns' to its maximum and that one's to the row's, so p and its running sums are right to 1e-11 of
// them (those of p - q to 1e-11 of 1). Whether a draft stands and which token is drawn can differ from the exact rule only where a
// uniform is that close, for every order of a sum.
//
// 1. stats: one workgroup per row and chunk of columns keeps its logits in registers and leaves their maximum and their
//    sum of exponentials. The logits are read once, 21 vector instructions each, which take about as long as their
//    bytes in fp32, twice as long in 16 bits: 640 rows of 128,000 fp32 logits 72 us (4.6 TB/s), 288 of 50,257 bf16 ones 16 us.
// 2. decide: one workgroup per sequence joins the rows' statistics, finds the first token that does not stand and, but for draws
//    from max(p - q, 0), the chunk the next token falls in, from the statistics again, and the column in that.
// 3. draw, where q is given: one workgroup per sequence and chunk sums its chunk of max(p - q, 0); the last workgroup of a
//    sequence to finish finds chunk and column. A few sequences do without 2: each workgroup decides, all draw (one sequence of
//    4 drafts: 10 us, dependent steps of 1-2 us).

#include <type_traits>

#include "half_types.h"

namespace tq {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

struct Stat {  // of one row's chunk
  double sum;      // of exp((logit - max) / T); 0 at T = 0
  uint64_t key;    // argmax_key of its largest logit (the column: where T = 0 or the maximum is not finite)
};

struct VerifyArgs {
  int64_t* tokens;
  int32_t* accepted;
  const void* logits;
  int64_t logits_stride;
  const float* probs;
  int64_t probs_stride;
  const int64_t* drafts;
  const float* uniforms;
  const float* temperature;
  const int32_t* cu;
  Stat* stats;        // [num_rows][chunks]
  struct Decision* decisions;  // [num_seqs]
  double* sums;       // [num_seqs][draw_chunks]
  uint32_t* arrived;  // [num_seqs]
  int32_t* d_error;
  int32_t num_seqs;
  int32_t num_rows;
  int32_t max_rows;
  int32_t vocab;
  int32_t chunks;
  int32_t draw_chunks;
};

// 2^t for t <= 0: 2^k 2^f with k the nearest integer (read off the low bits of t + 1.5 2^52), the second factor by the polynomial
// that meets 2^f at 0 and at the 8 Chebyshev points of [-1/2, 1/2]; off by at most 2.2e-12, and 1 for 0, so that equal logits
// have equal, whole weights. Below -1000, and for NaN: 2^-1000, which no sum of theirs notices.
__device__ __forceinline__ double exp2_neg(double t) {
  t = __builtin_fmax(t, -1000.0);
  const double shifted = t + 0x1.8p52;
  const double f = t - (shifted - 0x1.8p52);
  double r = 1.3250805512080399e-06;
  r = __builtin_fma(r, f, 1.5303700711214572e-05);
  r = __builtin_fma(r, f, 1.5403475186561525e-04);
  r = __builtin_fma(r, f, 1.333347847368613e-03);
  r = __builtin_fma(r, f, 9.618129135236088e-03);
  r = __builtin_fma(r, f, 5.550410906325866e-02);
  r = __builtin_fma(r, f, 2.4022650695888503e-01);
  r = __builtin_fma(r, f, 6.931471805568324e-01);
  r = __builtin_fma(r, f, 1.0);
  u32x2 bits = __builtin_bit_cast(u32x2, r);
  bits[1] += __builtin_bit_cast(u32x2, shifted)[0] << 20;
  return __builtin_bit_cast(double, bits);
}

template <typename T>
__device__ __forceinline__ float logit_at(const void* row, int64_t j) {
  if constexpr (__is_same(T, float))
    return static_cast<const float*>(row)[j];
  else
    return T::load(static_cast<const uint16_t*>(row)[j]);
}

template <typename T>
__device__ __forceinline__ const void* row_of(const VerifyArgs& a, int64_t row) {
  return static_cast<const char*>(a.logits) + row * a.logits_stride * (__is_same(T, float) ? 4 : 2);
}

// The value an argmax_key stands for (NaN: every NaN).
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  if (u == 0xFFFFFFFFu) return __builtin_nanf("");
  return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

// Reductions of a wave, through DPP in rows of 16 lanes and lanes 0, 16, 32, 48 (a 64-bit shuffle through LDS takes five times as
// long, and they lie on the path of a small call). Every lane gets the result; all orders of the lanes give the same.
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_move64(uint64_t v) {
  const uint32_t lo = __float_as_uint(dpp_move<CTRL>(__uint_as_float((uint32_t)v)));
  const uint32_t hi = __float_as_uint(dpp_move<CTRL>(__uint_as_float((uint32_t)(v >> 32))));
  return (uint64_t)hi << 32 | lo;
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}
template <typename F>
__device__ __forceinline__ uint64_t wave_reduce(uint64_t v, F&& join) {
  v = join(v, dpp_move64<kDppQuadXor1>(v));
  v = join(v, dpp_move64<kDppQuadXor2>(v));
  v = join(v, dpp_move64<kDppRowHalfMirror>(v));
  v = join(v, dpp_move64<kDppRowMirror>(v));
  return join(join(lane_of(v, 0), lane_of(v, 16)), join(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ double wave_sum(double v) {
  return __builtin_bit_cast(double, wave_reduce(__builtin_bit_cast(uint64_t, v), [](uint64_t a, uint64_t b) {
                              return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b));
                            }));
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  return wave_reduce(v, [](uint64_t a, uint64_t b) { return max_u64(a, b); });
}
__device__ __forceinline__ float wave_maximum(float v) {  // NaN, if any is
  v = __builtin_elementwise_maximum(v, dpp_move<kDppQuadXor1>(v));
  v = __builtin_elementwise_maximum(v, dpp_move<kDppQuadXor2>(v));
  v = __builtin_elementwise_maximum(v, dpp_move<kDppRowHalfMirror>(v));
  v = __builtin_elementwise_maximum(v, dpp_move<kDppRowMirror>(v));
  auto lane = [&](int l) { return __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(v), l)); };
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(lane(0), lane(16)),
                                       __builtin_elementwise_maximum(lane(32), lane(48)));
}

template <typename T>
constexpr int kVec = __is_same(T, float) ? 4 : 8;  // logits in 16 bytes

// Thread t's column i of a chunk: pieces of VEC columns t, t + N, .. (of N threads), or (RUNS) PER columns in a row.
template <int VEC, int N, int PER, bool RUNS>
__device__ __forceinline__ int column_of(int i) {
  return RUNS ? (int)threadIdx.x * PER + i : (i / VEC * N + (int)threadIdx.x) * VEC + i % VEC;
}

// Those columns of a row of T as floats, columns past n as -inf. Rows start at any element.
template <typename T, int VEC, int N, int PER, bool RUNS>
__device__ __forceinline__ void columns(const void* row, int base, int n, float (&x)[PER]) {
  constexpr int kSize = __is_same(T, float) ? 4 : 2;
#pragma unroll
  for (int v = 0; v < PER; v += VEC) {
    const int at = column_of<VEC, N, PER, RUNS>(v);
    if (at + VEC <= n) {
      u32x4 w[VEC * kSize / 16];
      __builtin_memcpy(w, static_cast<const char*>(row) + (int64_t)(base + at) * kSize, VEC * kSize);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if constexpr (__is_same(T, float))
          x[v + e] = __uint_as_float(w[e / 4][e % 4]);
        else
          x[v + e] = T::load((uint16_t)(w[e / 8][e % 8 / 2] >> (16 * (e & 1))));
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) x[v + e] = at + e < n ? logit_at<T>(row, base + at + e) : -INFINITY;
    }
  }
}

constexpr double kLog2e = 1.4426950408889634;

// The sequence that a row belongs to: the last one with cu[b] <= row (empty sequences hold no row), among 64 parts at a time.
// Its temperature, asked for before the logits, arrives before them. (Counted through all 1,024 sequences of 5 rows, 50,257 bf16
// logits each, the call took 328 us instead of 259.) Where cu falls somewhere this may be another one, still below num_seqs; every
// count grows with the row, so if it is b for two rows it is for those between them.
__device__ __forceinline__ int64_t owner_of(const VerifyArgs& a, int row) {
  const int lane = threadIdx.x & (kWave - 1);
  int64_t b = 0, n = a.num_seqs;
  while (n > 1) {
    const int64_t step = (n + kWave - 1) / kWave, at = b + lane * step;
    const int k = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane * step < n && a.cu[at] <= row));
    const int64_t skip = max(k - 1, 0) * step;
    b += skip;
    n = min(step, n - skip);
  }
  return b;
}

template <typename T, int PER>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(const VerifyArgs a) {
  __shared__ float s_top[kWaves];
  __shared__ double s_sum[kWaves];
  __shared__ int s_col;
  const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks;
  if (row < a.num_seqs && chunk == 0 && threadIdx.x == 0) a.arrived[row] = 0;  // for the second launch
  if (row >= a.num_rows) return;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int base = chunk * kThreads * PER, n = min(kThreads * PER, a.vocab - base);
  float x[PER], top = -INFINITY;
  const float temp = a.temperature[owner_of(a, row)];
  columns<T, kVec<T>, kThreads, PER, false>(row_of<T>(a, row), base, n, x);
#pragma unroll
  for (int i = 0; i < PER; ++i) top = __builtin_elementwise_maximum(top, x[i]);  // NaN, if any is
  top = wave_maximum(top);
  if (lane == 0) s_top[wave] = top;
  if (threadIdx.x == 0) s_col = 0x7fffffff;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kWaves; ++v) top = __builtin_elementwise_maximum(top, s_top[v]);
  double sum = 0.0;
  int col = 0;
  if (temp > 0.f && top > -INFINITY && top < INFINITY) {  // uniform
    const double c = kLog2e / (double)temp, t0 = (double)top;
#pragma unroll
    for (int i = 0; i < PER; ++i) sum += exp2_neg(((double)x[i] - t0) * c);
    sum = wave_sum(sum);
    if (lane == 0) s_sum[wave] = sum;
  } else {  // no distribution, or none needed: the first column that holds the maximum
    int mine = 0x7fffffff;
#pragma unroll
    for (int i = PER - 1; i >= 0; --i) {
      const int at = column_of<kVec<T>, kThreads, PER, false>(i);
      if (at < n && (top != top ? x[i] != x[i] : x[i] == top)) mine = at;
    }
    atomicMin(&s_col, mine);
    if (lane == 0) s_sum[wave] = 0.0;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = s_sum[0];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) sum += s_sum[v];
    if (s_col != 0x7fffffff) col = s_col;
    a.stats[(int64_t)row * a.chunks + chunk] = Stat{sum, argmax_key(top, base + col)};
  }
}

// A row's distribution: 2^((logit - top) c) / sum, or all of it on column best.
struct Dist {
  double sum, c;
  int64_t best;
  float top;
  bool peak;
};

// By one wave; every lane gets it.
__device__ __forceinline__ Dist dist_of(const VerifyArgs& a, int row, float temp) {
  const Stat* st = a.stats + (int64_t)row * a.chunks;
  const int lane = threadIdx.x & (kWave - 1);
  uint64_t key = 0;
  for (int c = lane; c < a.chunks; c += kWave) key = max_u64(key, st[c].key);
  key = wave_max(key);
  Dist d;
  d.top = key_value(key);
  d.best = argmax_key_column(key);
  d.c = kLog2e / (double)temp;
  d.peak = !(temp > 0.f) || !(d.top > -INFINITY && d.top < INFINITY);
  d.sum = 0.0;
  if (!d.peak) {
    for (int c = lane; c < a.chunks; c += kWave) {
      const float m = key_value(st[c].key);
      if (m > -INFINITY) d.sum += st[c].sum * exp2_neg(((double)m - (double)d.top) * d.c);
    }
    d.sum = wave_sum(d.sum);
  }
  return d;
}

// p of a column times sum (the draw needs no division), of a distribution without peak. A logit of -inf has none.
__device__ __forceinline__ double mass_of(const Dist& d, float logit) {
  const double t = ((double)logit - (double)d.top) * d.c;
  return t >= -1000.0 ? exp2_neg(t) : 0.0;
}

enum Mode { kAll, kLess, kWithout };  // the draw is from p, from p - q where positive, from p without the draft

// The draw's weight of a column, times sum.
__device__ __forceinline__ double weight_of(const Dist& d, float logit, double q, int64_t draft, int mode, int64_t col) {
  const double p = mass_of(d, logit);
  if (mode == kAll) return p;
  if (mode == kWithout) return col == draft ? 0.0 : p;
  const double w = p - q * d.sum;
  return w > 0.0 ? w : 0.0;
}

// The weights of a thread's columns of a chunk.
template <typename T, int N, int PER, bool RUNS, typename F>
__device__ __forceinline__ void weights(const Dist& d, const void* row, const float* qrow, int64_t draft, int mode,
                                        int base, int n, F&& put) {
  float x[PER], q[PER];
  columns<T, kVec<T>, N, PER, RUNS>(row, base, n, x);
  if (mode == kLess) {
    columns<float, kVec<T>, N, PER, RUNS>(qrow, base, n, q);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) q[i] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int at = column_of<kVec<T>, N, PER, RUNS>(i);
    put(i, at < n ? weight_of(d, x[i], (double)q[i], draft, mode, base + at) : 0.0);
  }
}

// Inclusive sums over the workgroup's N threads, in order; s_part: a word a wave.
template <int N>
__device__ __forceinline__ double scan(double v, double* s_part) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  auto up = [&](auto ctrl) {  // from a lane further down in the row of 16; 0 past its start
    return __builtin_bit_cast(double, dpp_move64<decltype(ctrl)::value>(__builtin_bit_cast(uint64_t, v)));
  };
  v += up(std::integral_constant<int, 0x111>());  // row_shr:1, 2, 4, 8
  v += up(std::integral_constant<int, 0x112>());
  v += up(std::integral_constant<int, 0x114>());
  v += up(std::integral_constant<int, 0x118>());
  double before = 0.0;  // the rows before this one
#pragma unroll
  for (int r = 1; r < kWave / 16; ++r) {
    const double row = __builtin_bit_cast(double, lane_of(__builtin_bit_cast(uint64_t, v), 16 * r - 1));
    before += lane >= 16 * r ? row : 0.0;
  }
  v += before;
  if (lane == kWave - 1) s_part[wave] = v;
  __syncthreads();
  before = 0.0;
#pragma unroll
  for (int u = 0; u < N / kWave - 1; ++u) before += u < wave ? s_part[u] : 0.0;
  __syncthreads();
  return before + v;
}

// The first thread with `over`, or the last with `has` where there is none; -1: none either. s_pick: two words a wave.
template <int N>
__device__ __forceinline__ int pick(bool over, bool has, int (*s_pick)[2]) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const uint64_t overs = __builtin_amdgcn_ballot_w64(over), those = __builtin_amdgcn_ballot_w64(has);
  if (lane == 0) {
    s_pick[wave][0] = overs != 0 ? wave * kWave + __builtin_ctzll(overs) : 0x7fffffff;
    s_pick[wave][1] = those != 0 ? wave * kWave + 63 - __builtin_clzll(those) : -1;
  }
  __syncthreads();
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int v = 0; v < N / kWave; ++v) {
    first = min(first, s_pick[v][0]);
    last = max(last, s_pick[v][1]);
  }
  __syncthreads();
  return first != 0x7fffffff ? first : last;
}

// What became of a sequence's drafts: how many stand, and the distribution of the row that the next token is drawn from.
struct Decision {
  Dist dist;
  int first;  // -1: the sequence has no rows (or is refused)
};

constexpr int kDists = 16;  // rows whose distributions are kept in LDS
struct DecideShared {
  Dist dist[kDists];
  int first, bad;
  bool refused;
};

// By one workgroup of N threads. `lead`: it also writes the tokens that stand, and the flags.
template <typename T, int N>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, int b, bool lead, DecideShared& sh) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int lo = a.cu[b];
  const int64_t rows = (int64_t)a.cu[b + 1] - lo;
  int64_t* out = a.tokens + (int64_t)b * a.max_rows;
  Decision r;
  const bool fits = lo >= 0 && rows > 0 && lo + rows <= a.num_rows && rows <= a.max_rows;
  const int drafts = fits ? (int)rows - 1 : -1;
  const float temp = a.temperature[b];
  if (threadIdx.x == 0) {
    sh.first = drafts;
    sh.bad = drafts + 1;
  }
  __syncthreads();
  // Rows that another sequence claims too may have statistics of its temperature. The last wave has the fewest rows.
  if (wave == N / kWave - 1) {
    const bool refused = !fits || owner_of(a, lo) != b || owner_of(a, lo + drafts) != b;
    if (lane == 0) sh.refused = refused;
  }
  // A wave a row, after a lane a row has fetched what it needs of 64 rows. (Rows behind one that does not stand are left out.)
  for (int i0 = 0; i0 <= drafts && i0 <= *(volatile int*)&sh.first; i0 += kWave) {
    float lx = 0.f, qx = 1.f, ux = 0.f;
    bool in = false;
    int64_t x = 0;
    if (i0 + lane < drafts) {
      x = a.drafts[lo + i0 + lane];
      ux = a.uniforms[lo + i0 + lane];
      in = x >= 0 && x < a.vocab;
      if (in) {
        lx = logit_at<T>(row_of<T>(a, lo + i0 + lane), x);
        if (a.probs != nullptr) qx = a.probs[(int64_t)(lo + i0 + lane) * a.probs_stride + x];
      }
    }
    for (int i = i0 + wave; i <= drafts && i < i0 + kWave && i <= *(volatile int*)&sh.first; i += N / kWave) {
      const Dist d = dist_of(a, lo + i, temp);
      if (lane == 0 && i < kDists) sh.dist[i] = d;
      if (d.peak && temp > 0.f && lane == 0) atomicMin(&sh.bad, i);
      if (lane == i - i0 && i < drafts) {
        bool stands = false;
        if (in) {
          const double p = d.peak ? (x == d.best ? 1.0 : 0.0) : mass_of(d, lx) / d.sum;
          stands = (double)ux * (double)qx < p;
        }
        if (!stands) atomicMin(&sh.first, i);
      }
    }
  }
  __syncthreads();
  if (sh.refused) {
    if (lead) {
      if (rows != 0 && threadIdx.x == 0) flag_error(a.d_error, TQ_DEVERR_LENGTH);
      for (int i = threadIdx.x; i < a.max_rows; i += N) out[i] = -1;
      if (threadIdx.x == 0) a.accepted[b] = 0;
    }
    r.first = -1;
    return r;
  }
  r.first = sh.first;
  if (r.first >= kDists) {  // uniform
    if (wave == 0) {
      const Dist d = dist_of(a, lo + r.first, temp);
      if (lane == 0) sh.dist[0] = d;
    }
    __syncthreads();
  }
  r.dist = sh.dist[r.first < kDists ? r.first : 0];
  if (lead) {
    for (int i = threadIdx.x; i < a.max_rows; i += N)
      if (i != r.first) out[i] = i < r.first ? a.drafts[lo + i] : -1;
    if (threadIdx.x == 0) {
      a.accepted[b] = r.first;
      if (sh.bad <= r.first) flag_error(a.d_error, TQ_DEVERR_VALUE);
      if (r.first < drafts && (a.drafts[lo + r.first] < 0 || a.drafts[lo + r.first] >= a.vocab))
        flag_error(a.d_error, TQ_DEVERR_TOKEN);
    }
  }
  return r;
}

template <int N>
struct DrawShared {
  double part[N / kWave], goal;
  int turn, pick[N / kWave][2];
};

// The sum of a chunk's weights, by the workgroup.
template <typename T, int N, int PER>
__device__ __forceinline__ double chunk_sum(const VerifyArgs& a, const Dist& d, const void* row, const float* qrow,
                                            int64_t draft, int mode, int chunk, DrawShared<N>& sh) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave, at = chunk * N * PER;
  double w = 0.0;
  weights<T, N, PER, false>(d, row, qrow, draft, mode, at, min(N * PER, a.vocab - at), [&](int, double v) { w += v; });
  w = wave_sum(w);
  if (lane == 0) sh.part[wave] = w;
  __syncthreads();
  w = 0.0;
#pragma unroll
  for (int v = 0; v < N / kWave; ++v) w += sh.part[v];
  __syncthreads();
  return w;
}

// The workgroup's sum of mine, in all of its threads; upto: up to this one.
template <int N>
__device__ __forceinline__ double total_of(double mine, double& upto, DrawShared<N>& sh) {
  upto = scan<N>(mine, sh.part);
  if (threadIdx.x == N - 1) sh.goal = upto;
  __syncthreads();
  return sh.goal;
}

// The draw, from the chunks' sums (thread c's: of chunk c, and up to it): the chunk it falls in, the last one with weight where
// rounding leaves none above the goal, and the column in that.
template <typename T, int N, int PER>
__device__ __forceinline__ void draw(const VerifyArgs& a, const Dist& d, const void* row, const float* qrow, int64_t draft,
                                     int mode, double mine, double upto, double goal, int64_t* token, DrawShared<N>& sh) {
  const int c = threadIdx.x;
  const int chosen = pick<N>(mine > 0.0 && upto > goal, mine > 0.0, sh.pick);
  if (chosen < 0) {  // no weight anywhere: draft probabilities that are not numbers
    if (c == 0) *token = d.best;
    return;
  }
  if (c == chosen) sh.goal = goal - (upto - mine);
  // Runs of PER columns a thread.
  const int at = chosen * N * PER;
  double ws[PER], run = 0.0;
  weights<T, N, PER, true>(d, row, qrow, draft, mode, at, min(N * PER, a.vocab - at), [&](int i, double v) {
    ws[i] = v;
    run += v;
  });
  upto = scan<N>(run, sh.part);
  const double rest = sh.goal;
  if (c == pick<N>(run > 0.0 && upto > rest, run > 0.0, sh.pick)) {
    double cum = upto - run;
    int col = -1;
    bool done = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      cum += ws[i];
      if (!done && ws[i] > 0.0) {
        col = at + c * PER + i;
        done = cum > rest;
      }
    }
    *token = col;
  }
}

// One workgroup a sequence. Where the draw is not from a difference, the statistics hold its chunks' sums already, less the draft
// (whose chunk is summed again without it: the rest may be far below it; only doing so where it has more than half of the weight
// saves nothing), and the sequence ends here; the others' decisions are left for verify_draw_kernel. A chunk of the statistics
// is 8 columns a thread: 64 sequences of 50,257 columns 13.8 us with 1,024 threads, 19.2 with 256 of 32 columns.
template <typename T, int N>
__global__ __launch_bounds__(N) void verify_decide_kernel(const VerifyArgs a) {
  __shared__ DecideShared s_decide;
  __shared__ DrawShared<N> sh;
  constexpr int kPer = 8;  // columns of a thread in a chunk of the statistics
  const int b = blockIdx.x, c = threadIdx.x;
  Decision r = decide<T, N>(a, b, true, s_decide);
  const int lo = a.cu[b], drafts = a.cu[b + 1] - lo - 1, row = lo + r.first;
  const bool less = r.first >= 0 && r.first < drafts && a.probs != nullptr && !r.dist.peak;
  if (a.probs != nullptr && c == 0) {
    a.decisions[b] = r;
    if (!less) a.decisions[b].first = -1;
  }
  if (r.first < 0 || less) return;
  const Dist d = r.dist;
  int64_t* token = a.tokens + (int64_t)b * a.max_rows + r.first;
  if (d.peak) {  // whatever q is
    if (c == 0) *token = d.best;
    return;
  }
  const Stat* st = a.stats + (int64_t)row * a.chunks;
  const void* lp = row_of<T>(a, row);
  const double u = (double)a.uniforms[lo + drafts];
  const int64_t draft = r.first < drafts ? a.drafts[row] : -1;
  double all = 0.0;
  if (c < a.chunks) {
    const double t = ((double)key_value(st[c].key) - (double)d.top) * d.c;
    if (t >= -1000.0) all = st[c].sum * exp2_neg(t);  // else no column of it has weight
  }
  double mine = all, upto;
  int mode = kAll;
  if (draft >= 0 && draft < a.vocab) {
    mode = kWithout;
    const int skip = (int)draft / (N * kPer);
    const double sum = chunk_sum<T, N, kPer>(a, d, lp, nullptr, draft, mode, skip, sh);
    if (c == skip) mine = sum;
  }
  double total = total_of<N>(mine, upto, sh);
  if (!(total > 0.0)) {  // p is all on the draft (to rounding): the draw is from p itself
    mode = kAll;
    mine = all;
    total = total_of<N>(mine, upto, sh);
  }
  draw<T, N, kPer>(a, d, lp, nullptr, draft, mode, mine, upto, u * total, token, sh);
}

// One workgroup a sequence and chunk. DECIDED: by verify_decide_kernel; else each decides for itself.
template <typename T, int PER, bool DECIDED>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(const VerifyArgs a) {
  __shared__ DrawShared<kThreads> sh;
  const int chunk = blockIdx.x % a.draw_chunks, b = blockIdx.x / a.draw_chunks;
  Decision r;
  if constexpr (DECIDED) {
    r = a.decisions[b];
  } else {
    __shared__ DecideShared s_decide;
    r = decide<T, kThreads>(a, b, chunk == 0, s_decide);
  }
  if (r.first < 0) return;
  const Dist d = r.dist;
  const int lo = a.cu[b], drafts = a.cu[b + 1] - lo - 1, row = lo + r.first;
  const void* lp = row_of<T>(a, row);
  const float* qrow = a.probs + (int64_t)row * a.probs_stride;
  int64_t* token = a.tokens + (int64_t)b * a.max_rows + r.first;
  if (!DECIDED && d.peak) {
    if (chunk == 0 && threadIdx.x == 0) *token = d.best;
    return;
  }
  int mode = r.first == drafts ? kAll : kLess;
  const double w = chunk_sum<T, kThreads, PER>(a, d, lp, qrow, -1, mode, chunk, sh);
  double* sums = a.sums + (int64_t)b * a.draw_chunks;
  if (threadIdx.x == 0) {
    // The sums are all that workgroups hand each other, by accesses of agent scope, which are done where all XCDs meet: the
    // count has to follow the store, which has ended after the wait. (Release and acquire of everything else would write this
    // XCD's L2 back and drop it.)
    __hip_atomic_store(&sums[chunk], w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    sh.turn = (int)__hip_atomic_fetch_add(&a.arrived[b], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (sh.turn != a.draw_chunks - 1) return;

  // The last workgroup of the sequence, a chunk a thread.
  const int c = threadIdx.x;
  double mine = c < a.draw_chunks ? __hip_atomic_load(&sums[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0.0, upto;
  double total = total_of<kThreads>(mine, upto, sh);
  if (!(total > 0.0)) {
    // Nothing left where q covers p (to rounding): the draw is from p itself.
    mode = kAll;
    mine = 0.0;
    __syncthreads();
    for (int k = 0; k < a.draw_chunks; ++k) {
      const double sum = chunk_sum<T, kThreads, PER>(a, d, lp, qrow, -1, mode, k, sh);
      mine = c == k ? sum : mine;
    }
    total = total_of<kThreads>(mine, upto, sh);
  }
  draw<T, kThreads, PER>(a, d, lp, qrow, -1, mode, mine, upto, (double)a.uniforms[lo + drafts] * total, token, sh);
}

constexpr int kMaxVocab = kThreads * kThreads * 32;  // a chunk a thread
// Workgroups of the draw up to which 2,048 columns each end sooner than 4,096 (sequences of 4 drafts with q, both launches: 8 over
// 50,257 bf16 columns 15.6 and 17.3 us, 16 20.3 and 20.6, 32 26.8 and 24.8; 8,192 columns 23.2, 25.3, 29.1), and from which a
// decision launch pays (32 over 128,000 fp32 columns 47 us with, 42 without; 128 over 50,257 55 and 55; 64 over 128,000 63 and 69;
// 128 108 and 133).
constexpr int kFewDraws = 400;
constexpr int kDecideFrom = 1664;
static_assert(kFewDraws < kDecideFrom, "draws of 8 columns a thread have no decision launch");

// How a call is split, and its workspace.
struct Plan {
  int per, draw_per;  // columns of a thread in stats (8 or 32) and draw (8, 16, or 32 where 256 chunks ask for it)
  int chunks, draw_chunks;
  bool decide;  // a launch between them, where q is given
  size_t stats, decisions, sums, arrived, bytes;  // offsets
};

Plan plan_of(int32_t num_seqs, int32_t num_rows, int32_t vocab) {
  Plan p;
  auto chunks = [&](int per) { return (vocab + kThreads * per - 1) / (kThreads * per); };
  // 32 columns a thread keep the loads of a row in flight (640 rows of 128,000 fp32 logits 73 us, with 16 82, with 8 95); 8 spread
  // few rows over more CUs (5 rows of 50,257: 3.6 us, with 16 4.0).
  p.per = (int64_t)num_rows * chunks(32) < 512 && chunks(8) <= kThreads ? 8 : 32;
  p.draw_per = chunks(8) <= kThreads && (int64_t)num_seqs * chunks(8) <= kFewDraws ? 8 : chunks(16) <= kThreads ? 16 : 32;
  p.chunks = chunks(p.per);
  p.draw_chunks = chunks(p.draw_per);
  p.decide = (int64_t)num_seqs * p.draw_chunks >= kDecideFrom;
  p.stats = 0;
  p.decisions = p.stats + (size_t)num_rows * p.chunks * sizeof(Stat);
  p.sums = p.decisions + (size_t)num_seqs * sizeof(Decision);
  p.arrived = p.sums + (size_t)num_seqs * p.draw_chunks * sizeof(double);
  p.bytes = p.arrived + (size_t)num_seqs * sizeof(uint32_t);
  return p;
}

template <typename T, int PER>
tq_status launch_draw(const VerifyArgs& a, bool decided, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.num_seqs * a.draw_chunks));
  if constexpr (PER > 8) {
    if (decided) {
      hipLaunchKernelGGL((verify_draw_kernel<T, PER, true>), grid, dim3(kThreads), 0, stream, a);
      return check_launch();
    }
  }
  hipLaunchKernelGGL((verify_draw_kernel<T, PER, false>), grid, dim3(kThreads), 0, stream, a);
  return check_launch();
}

template <typename T>
tq_status launch(const VerifyArgs& a, const Plan& p, hipStream_t stream) {
  const int64_t rows = a.num_rows > a.num_seqs ? a.num_rows : a.num_seqs;
  const int64_t stats = rows * a.chunks;
  if (stats > 0x7fffffffLL || (int64_t)a.num_seqs * a.draw_chunks > 0x7fffffffLL) return TQ_ERR_UNSUPPORTED;
  if (p.per == 8)
    hipLaunchKernelGGL((verify_stats_kernel<T, 8>), dim3((unsigned)stats), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((verify_stats_kernel<T, 32>), dim3((unsigned)stats), dim3(kThreads), 0, stream, a);
  tq_status st = check_launch();
  if (st != TQ_OK) return st;
  const bool decided = p.decide || a.probs == nullptr;
  if (decided) {
    if (p.per == 8)
      hipLaunchKernelGGL((verify_decide_kernel<T, kThreads>), dim3((unsigned)a.num_seqs), dim3(kThreads), 0, stream, a);
    else
      hipLaunchKernelGGL((verify_decide_kernel<T, 4 * kThreads>), dim3((unsigned)a.num_seqs), dim3(4 * kThreads), 0, stream, a);
    st = check_launch();
    if (st != TQ_OK || a.probs == nullptr) return st;
  }
  switch (p.draw_per) {
    case 8: return launch_draw<T, 8>(a, decided, stream);
    case 16: return launch_draw<T, 16>(a, decided, stream);
    default: return launch_draw<T, 32>(a, decided, stream);
  }
}

}  // namespace
}  // namespace tq

extern "C" size_t tq_verify_drafts_workspace_size(int32_t num_seqs, int32_t num_rows, int32_t vocab) {
  using namespace tq;
  if (num_seqs < 1 || num_rows < 0 || vocab < 1 || vocab > kMaxVocab) return 0;
  return plan_of(num_seqs, num_rows, vocab).bytes;
}

extern "C" tq_status tq_verify_drafts(int64_t* tokens, int32_t* accepted, const void* logits,
                                      int64_t logits_row_stride, const float* draft_probs, int64_t probs_row_stride,
                                      const int64_t* draft_tokens, const float* uniforms, const float* temperature,
                                      const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t num_rows,
                                      int32_t max_query_len, int32_t vocab, int32_t dtype, void* workspace,
                                      size_t workspace_bytes, int32_t* d_error, void* stream) {
  using namespace tq;
  if (num_seqs < 0 || num_rows < 0 || max_query_len < 0 || vocab < 1) return TQ_ERR_INVALID_ARGUMENT;
  if ((dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) || vocab > kMaxVocab) return TQ_ERR_UNSUPPORTED;
  if (num_seqs == 0) return TQ_OK;
  if (max_query_len < 1 || tokens == nullptr || accepted == nullptr || cu_seqlens_q == nullptr ||
      temperature == nullptr || (num_rows > 0 && (logits == nullptr || draft_tokens == nullptr || uniforms == nullptr)) ||
      (num_rows > 1 && (logits_row_stride < vocab || (draft_probs != nullptr && probs_row_stride < vocab))))
    return TQ_ERR_INVALID_ARGUMENT;
  const Plan p = plan_of(num_seqs, num_rows, vocab);
  if (workspace == nullptr || workspace_bytes < p.bytes || (uintptr_t)workspace % 16 != 0) return TQ_ERR_WORKSPACE;
  VerifyArgs a;
  a.tokens = tokens;
  a.accepted = accepted;
  a.logits = logits;
  a.logits_stride = logits_row_stride;
  a.probs = draft_probs;
  a.probs_stride = probs_row_stride;
  a.drafts = draft_tokens;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.cu = cu_seqlens_q;
  a.num_seqs = num_seqs;
  a.num_rows = num_rows;
  a.max_rows = max_query_len;
  a.vocab = vocab;
  a.chunks = p.chunks;
  a.draw_chunks = p.draw_chunks;
  char* ws = static_cast<char*>(workspace);
  a.stats = reinterpret_cast<Stat*>(ws + p.stats);
  a.decisions = reinterpret_cast<Decision*>(ws + p.decisions);
  a.sums = reinterpret_cast<double*>(ws + p.sums);
  a.arrived = reinterpret_cast<uint32_t*>(ws + p.arrived);
  a.d_error = d_error;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TQ_F32) return launch<float>(a, p, st);
  return dtype == TQ_BF16 ? launch<Bf16>(a, p, st) : launch<Fp16>(a, p, st);
}

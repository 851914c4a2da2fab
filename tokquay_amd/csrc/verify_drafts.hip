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
// close: exponentials and sums are fp64 (fp64 FMAs run at the fp32 rate here), which also makes the order of a sum
// not matter. Two launches:
//
// 1. stats: one workgroup per row and kChunk columns keeps its logits in registers and leaves their maximum, its
//    lowest column and their sum of exponentials. The logits are read once: HBM bound.
// 2. draw: one workgroup per sequence and kChunk columns joins the rows' statistics, finds the first token that
//    does not stand and sums its chunk's weights of that row; the last workgroup of a sequence to finish
//    finds the chunk the draw falls in, and the column in it.

#include <float.h>

#include "half_types.h"

namespace tq {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 32;                 // columns of a thread
constexpr int kChunk = kThreads * kPer;  // columns of a workgroup

struct Stat {  // of one row's chunk
  double sum;      // of exp((logit - max) / T); 0 at T = 0
  uint64_t key;    // argmax_key of its largest logit
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
  double* sums;       // [num_seqs][chunks]
  uint32_t* arrived;  // [num_seqs]
  int32_t* d_error;
  int32_t num_seqs;
  int32_t num_rows;
  int32_t max_rows;
  int32_t vocab;
  int32_t chunks;
};

// e^x for x <= 0 (0 for NaN): 2^k 2^f, the second factor by its Taylor series (|f ln 2| < 0.35: the first term left
// out is below 7e-15).
__device__ __forceinline__ double exp_neg(double x) {
  const double t = __builtin_fmax(x * 1.4426950408889634, -1100.0);  // below it: 0
  const double k = __builtin_rint(t);
  const double f = (t - k) * 0.6931471805599453;
  double r = 2.505210838544172e-08;                // 1 / 11!
  r = __builtin_fma(r, f, 2.755731922398589e-07);  // 1 / 10!
  r = __builtin_fma(r, f, 2.755731922398589e-06);
  r = __builtin_fma(r, f, 2.48015873015873e-05);
  r = __builtin_fma(r, f, 1.984126984126984e-04);
  r = __builtin_fma(r, f, 1.388888888888889e-03);
  r = __builtin_fma(r, f, 8.333333333333333e-03);
  r = __builtin_fma(r, f, 4.1666666666666664e-02);
  r = __builtin_fma(r, f, 1.6666666666666666e-01);
  r = __builtin_fma(r, f, 0.5);
  r = __builtin_fma(r, f, 1.0);
  r = __builtin_fma(r, f, 1.0);
  return __builtin_ldexp(r, (int)k);
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

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// The sequence that a row belongs to: the last with cu[b] <= row (empty sequences hold no row).
__device__ __forceinline__ int sequence_of(const VerifyArgs& a, int row) {
  int lo = 0, hi = a.num_seqs;  // cu[lo] <= row < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.cu[mid] <= row)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(const VerifyArgs a) {
  __shared__ uint64_t s_key[kThreads / kWave];
  __shared__ double s_sum[kThreads / kWave];
  const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks;
  if (row < a.num_seqs && chunk == 0 && threadIdx.x == 0) a.arrived[row] = 0;  // for the second launch
  if (row >= a.num_rows) return;
  const int b = sequence_of(a, row);
  const float temp = a.temperature[b];
  const void* lp = row_of<T>(a, row);
  const int base = chunk * kChunk, n = min(kChunk, a.vocab - base);
  float x[kPer];
  uint64_t key = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int j = i * kThreads + threadIdx.x;
    x[i] = j < n ? logit_at<T>(lp, base + j) : -INFINITY;
    if (j < n) key = max_u64(key, argmax_key(x[i], base + j));
  }
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) key = max_u64(key, __shfl_xor(key, off));
  if (lane == 0) s_key[wave] = key;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kThreads / kWave; ++v) key = max_u64(key, s_key[v]);
  const float top = key_value(key);
  double sum = 0.0;
  if (temp > 0.f && top > -INFINITY && top < INFINITY) {  // else no distribution, or none needed
    const double inv = 1.0 / (double)temp;
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += exp_neg(((double)x[i] - (double)top) * inv);
  }
  sum = wave_sum(sum);
  if (lane == 0) s_sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int v = 1; v < kThreads / kWave; ++v) sum += s_sum[v];
    a.stats[(int64_t)row * a.chunks + chunk] = Stat{sum, key};
  }
}

// A row's distribution: exp((logit - top) / T) / sum, or all of it on column best.
struct Dist {
  double sum, inv;
  float top;
  int64_t best;
  bool peak;
};

__device__ __forceinline__ Dist dist_of(const VerifyArgs& a, int row, float temp) {
  const Stat* st = a.stats + (int64_t)row * a.chunks;
  uint64_t key = 0;
  for (int c = 0; c < a.chunks; ++c) key = max_u64(key, st[c].key);
  Dist d;
  d.top = key_value(key);
  d.best = argmax_key_column(key);
  d.inv = 1.0 / (double)temp;
  d.peak = !(temp > 0.f) || !(d.top > -INFINITY && d.top < INFINITY);
  d.sum = 0.0;
  if (!d.peak) {
    for (int c = 0; c < a.chunks; ++c) {
      const float m = key_value(st[c].key);
      if (m > -INFINITY) d.sum += st[c].sum * exp_neg(((double)m - (double)d.top) * d.inv);
    }
  }
  return d;
}

// p of column j, times sum (the draw needs no division).
template <typename T>
__device__ __forceinline__ double mass_at(const Dist& d, const void* row, int64_t j) {
  if (d.peak) return j == d.best ? 1.0 : 0.0;
  return exp_neg(((double)logit_at<T>(row, j) - (double)d.top) * d.inv);
}

// The draw's weight of column j: all of p's (mode 0), p - q where positive (1), p without the draft (2). Times d.sum.
template <typename T>
__device__ __forceinline__ double weight_at(const Dist& d, const void* row, const float* qrow, int64_t draft, int mode,
                                            int64_t j) {
  const double p = mass_at<T>(d, row, j);
  if (mode == 0) return p;
  if (mode == 2) return j == draft ? 0.0 : p;
  const double w = d.peak ? p - (double)qrow[j] : p - (double)qrow[j] * d.sum;
  return w > 0.0 ? w : 0.0;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(const VerifyArgs a) {
  __shared__ int s_first, s_bad;
  __shared__ Dist s_dist;
  __shared__ double s_sum[kThreads];
  __shared__ int s_last;
  const int chunk = blockIdx.x % a.chunks, b = blockIdx.x / a.chunks;
  const int lo = a.cu[b];
  const int64_t rows64 = (int64_t)a.cu[b + 1] - lo;
  int64_t* out = a.tokens + (int64_t)b * a.max_rows;
  const bool lead = chunk == 0;
  if (lo < 0 || rows64 < 0 || lo + rows64 > a.num_rows || rows64 > a.max_rows || rows64 == 0) {
    if (lead) {
      if (rows64 != 0 && threadIdx.x == 0) flag_error(a.d_error, TQ_DEVERR_LENGTH);
      for (int i = threadIdx.x; i < a.max_rows; i += kThreads) out[i] = -1;
      if (threadIdx.x == 0) a.accepted[b] = 0;
    }
    return;
  }
  const int rows = (int)rows64, drafts = rows - 1;
  const float temp = a.temperature[b];
  if (threadIdx.x == 0) {
    s_first = drafts;
    s_bad = rows;
  }
  __syncthreads();
  // The first drafted token that does not stand.
  for (int i = threadIdx.x; i < drafts; i += kThreads) {
    const Dist d = dist_of(a, lo + i, temp);
    const int64_t x = a.drafts[lo + i];
    const bool in = x >= 0 && x < a.vocab;
    if (!in && lead) flag_error(a.d_error, TQ_DEVERR_TOKEN);
    bool stands = false;
    if (in) {
      const double p = d.peak ? (x == d.best ? 1.0 : 0.0) : mass_at<T>(d, row_of<T>(a, lo + i), x) / d.sum;
      const double q = a.probs == nullptr ? 1.0 : (double)a.probs[(int64_t)(lo + i) * a.probs_stride + x];
      stands = (double)a.uniforms[lo + i] * q < p;
    }
    if (!stands) atomicMin(&s_first, i);
    if (d.peak && temp > 0.f) atomicMin(&s_bad, i);
  }
  __syncthreads();
  const int first = s_first, row = lo + first;
  if (threadIdx.x == 0) {
    s_dist = dist_of(a, row, temp);
    if (lead && temp > 0.f && (s_dist.peak || s_bad < first)) flag_error(a.d_error, TQ_DEVERR_VALUE);
  }
  __syncthreads();
  const Dist d = s_dist;
  const void* lp = row_of<T>(a, row);
  const float* qrow = a.probs == nullptr ? nullptr : a.probs + (int64_t)row * a.probs_stride;
  const int64_t draft = first < drafts ? a.drafts[row] : -1;
  int mode = first == drafts ? 0 : a.probs != nullptr ? 1 : 2;
  if (lead) {
    for (int i = threadIdx.x; i < a.max_rows; i += kThreads)
      if (i != first) out[i] = i < first ? a.drafts[lo + i] : -1;
    if (threadIdx.x == 0) a.accepted[b] = first;
  }
  // This chunk's weights, a run of kPer columns a thread.
  const int base = chunk * kChunk + threadIdx.x * kPer;
  double w = 0.0;
  for (int i = 0; i < kPer; ++i)
    if (base + i < a.vocab) w += weight_at<T>(d, lp, qrow, draft, mode, base + i);
  w = wave_sum(w);
  if (threadIdx.x % kWave == 0) s_sum[threadIdx.x / kWave] = w;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = s_sum[0];
    for (int v = 1; v < kThreads / kWave; ++v) total += s_sum[v];
    __hip_atomic_store(&a.sums[(int64_t)b * a.chunks + chunk], total, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = __hip_atomic_fetch_add(&a.arrived[b], 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
             (uint32_t)a.chunks - 1;
  }
  __syncthreads();
  if (!s_last) return;

  // The last workgroup of the sequence: the chunk, then the thread's run, then the column.
  __shared__ double s_goal;
  __shared__ int s_chunk;
  const double u = (double)a.uniforms[lo + drafts];
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int c = 0; c < a.chunks; ++c)
      total += __hip_atomic_load(&a.sums[(int64_t)b * a.chunks + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_chunk = -1;
    s_goal = u * total;
    if (total > 0.0) {
      double before = 0.0;
      int pick = -1;
      double pick_before = 0.0;
      for (int c = 0; c < a.chunks; ++c) {
        const double part =
            __hip_atomic_load(&a.sums[(int64_t)b * a.chunks + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (part > 0.0) {  // the last one with weight, should rounding leave none above the goal
          pick = c;
          pick_before = before;
        }
        before += part;
        if (part > 0.0 && before > s_goal) break;
      }
      s_chunk = pick;
      s_goal -= pick_before;
    }
  }
  __syncthreads();
  int c0 = s_chunk, c1 = c0 + 1;
  double goal = s_goal;
  bool whole = false;
  if (c0 < 0) {
    // Nothing left where q covers p (to rounding): the draw is from p itself, over all chunks.
    mode = 0;
    c0 = 0;
    c1 = a.chunks;
    whole = true;
    goal = d.peak ? u : u * d.sum;
  }
  __shared__ int64_t s_token;
  for (int c = c0; c < c1; ++c) {
    const int at = c * kChunk + threadIdx.x * kPer;
    double run = 0.0;
    for (int i = 0; i < kPer; ++i)
      if (at + i < a.vocab) run += weight_at<T>(d, lp, qrow, draft, mode, at + i);
    s_sum[threadIdx.x] = run;
    __syncthreads();
    if (threadIdx.x == 0) {
      double before = 0.0;
      int64_t token = -1;
      for (int v = 0; v < kThreads && token < 0; ++v) {
        if (!(s_sum[v] > 0.0)) continue;
        // The column: inside this run if the goal falls in it; the last weighted column where the chunk ends first.
        double cum = before;
        int64_t lastw = -1;
        const int from = c * kChunk + v * kPer;
        const bool inside = before + s_sum[v] > goal;
        bool more = false;
        for (int vv = v + 1; vv < kThreads && !more; ++vv) more = s_sum[vv] > 0.0;
        if (inside || (!more && (!whole || c == c1 - 1))) {
          for (int i = 0; i < kPer && from + i < a.vocab; ++i) {
            const double wi = weight_at<T>(d, lp, qrow, draft, mode, from + i);
            if (!(wi > 0.0)) continue;
            cum += wi;
            lastw = from + i;
            if (cum > goal) break;
          }
          token = lastw;
        }
        before += s_sum[v];
      }
      s_token = token;
      s_goal = goal - before;
    }
    __syncthreads();
    if (s_token >= 0) break;
    goal = s_goal;
    __syncthreads();
  }
  if (threadIdx.x == 0) out[first] = s_token >= 0 ? s_token : d.best;
}

int64_t chunks_of(int32_t vocab) { return ((int64_t)vocab + kChunk - 1) / kChunk; }

template <typename T>
tq_status launch(const VerifyArgs& a, hipStream_t stream) {
  const int64_t rows = a.num_rows > a.num_seqs ? a.num_rows : a.num_seqs;
  const int64_t stats = rows * a.chunks, draw = (int64_t)a.num_seqs * a.chunks;
  if (stats > 0x7fffffffLL || draw > 0x7fffffffLL) return TQ_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((verify_stats_kernel<T>), dim3((unsigned)stats), dim3(kThreads), 0, stream, a);
  const tq_status st = check_launch();
  if (st != TQ_OK) return st;
  hipLaunchKernelGGL((verify_draw_kernel<T>), dim3((unsigned)draw), dim3(kThreads), 0, stream, a);
  return check_launch();
}

}  // namespace
}  // namespace tq

extern "C" size_t tq_verify_drafts_workspace_size(int32_t num_seqs, int32_t num_rows, int32_t vocab) {
  using namespace tq;
  if (num_seqs < 1 || num_rows < 0 || vocab < 1) return 0;
  const size_t chunks = (size_t)chunks_of(vocab);
  return num_rows * chunks * sizeof(Stat) + num_seqs * chunks * sizeof(double) + num_seqs * sizeof(uint32_t);
}

extern "C" tq_status tq_verify_drafts(int64_t* tokens, int32_t* accepted, const void* logits,
                                      int64_t logits_row_stride, const float* draft_probs, int64_t probs_row_stride,
                                      const int64_t* draft_tokens, const float* uniforms, const float* temperature,
                                      const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t num_rows,
                                      int32_t max_query_len, int32_t vocab, int32_t dtype, void* workspace,
                                      size_t workspace_bytes, int32_t* d_error, void* stream) {
  using namespace tq;
  if (num_seqs < 0 || num_rows < 0 || max_query_len < 0 || vocab < 1) return TQ_ERR_INVALID_ARGUMENT;
  if ((dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) || vocab > 1 << 30) return TQ_ERR_UNSUPPORTED;
  if (num_seqs == 0) return TQ_OK;
  if (max_query_len < 1 || tokens == nullptr || accepted == nullptr || cu_seqlens_q == nullptr ||
      temperature == nullptr || (num_rows > 0 && (logits == nullptr || draft_tokens == nullptr || uniforms == nullptr)) ||
      (num_rows > 1 && (logits_row_stride < vocab || (draft_probs != nullptr && probs_row_stride < vocab))))
    return TQ_ERR_INVALID_ARGUMENT;
  const size_t need = tq_verify_drafts_workspace_size(num_seqs, num_rows, vocab);
  if (workspace == nullptr || workspace_bytes < need || (uintptr_t)workspace % 16 != 0) return TQ_ERR_WORKSPACE;
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
  a.chunks = (int32_t)chunks_of(vocab);
  a.stats = static_cast<Stat*>(workspace);
  a.sums = reinterpret_cast<double*>(a.stats + (size_t)num_rows * a.chunks);
  a.arrived = reinterpret_cast<uint32_t*>(a.sums + (size_t)num_seqs * a.chunks);
  a.d_error = d_error;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TQ_F32) return launch<float>(a, st);
  return dtype == TQ_BF16 ? launch<Bf16>(a, st) : launch<Fp16>(a, st);
}

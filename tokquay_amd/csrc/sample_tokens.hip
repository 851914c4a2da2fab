// Tokens drawn from rows of logits with temperature, top-k, top-p and min-p, from given random numbers.
//
// A row's columns are ranked by logit, the largest first, equal ones by column. With w_j = exp((x_j - max) / T):
//
//   top-k leaves the first k ranks; top-p of these every rank before which less than p of their weight lies (one at least);
//   min-p of these the columns with w_j >= min_p; the token is the lowest of the columns that are left with
//   w_0 + .. + w_j > u (sum of w), in the order of columns.
//
// Ranks are found by value: with d the distance of a column's ordered key (argmax_key) from the row's largest, the first
// ranks are those with d below some d*, and the first columns of those with d = d*. d* is found by counting (and weighing) columns in
// 2,048 intervals of d, then in the intervals of the one that it lies in. Weights are counted there in fixed point, so that the order of
// the additions changes nothing.
//
// 1. stats: one workgroup per row and chunk of columns reads the logits, once, and leaves the chunk's maximum, its sum of
//    exponentials where the settings need it, and the maximum of each group of 32 columns.
// 2. pick: one workgroup per row. Columns that can be among the first ranks lie in groups whose maximum can: the k-th largest of
//    these maxima is a lower bound of the k-th largest logit, and where the maxima's own weights reach p of the row's
//    the least of them bounds top-p. Of the groups above the bound, a few more than k, the columns above it are listed in LDS.
#include "draw.h"

namespace tq {
namespace {

constexpr int kThreads = 256;       // of a chunk's workgroup
constexpr int kGroup = 32;          // columns of a group
constexpr int kPick = 1024;         // threads of a row's workgroup
constexpr int kPickWaves = kPick / kWave;
constexpr int kBins = 2 * kPick;
constexpr int kListed = 8192;       // columns that are kept in LDS; rows of which more matter are read again
constexpr int kSelected = 4096;     // groups whose columns are listed; if more reach the limit, all are looked at
constexpr int kMaxVocab = 1 << 21;
constexpr int kMaxRounds = kMaxVocab / (4 * kPick);

struct SampleArgs {
  int64_t* tokens;
  const void* logits;
  int64_t logits_stride;
  const float* uniforms;
  const float* temperature;
  const int32_t* top_k;  // this and the next two: or null
  const float* top_p;
  const float* min_p;
  const int32_t* cu;  // or null: a setting a row
  Stat* stats;        // [num_rows][chunks]
  float* maxima;      // [num_rows][groups]
  int32_t* d_error;
  int32_t num_rows;
  int32_t num_seqs;
  int32_t vocab;
  int32_t chunks;
  int32_t chunk_columns;
  int32_t groups;
  int32_t mass_bits;  // weights are counted in units of 2^-mass_bits
};

// A row's settings.
struct Settings {
  float temp, p, least;
  int k;      // 0: off
  bool none;  // the row is in no sequence

  __device__ __forceinline__ bool nucleus() const { return p < 1.f; }
  __device__ __forceinline__ bool all() const { return k == 0 && !nucleus() && !(least > 0.f); }
  // Whether the sum of the whole row's weights is asked for.
  __device__ __forceinline__ bool sums() const { return k == 0 && (nucleus() || !(least > 0.f)); }
};

__device__ __forceinline__ Settings settings_of(const SampleArgs& a, int row) {
  Settings s;
  int64_t at = row;
  s.none = false;
  if (a.cu != nullptr) {
    s.none = row < a.cu[0] || row >= a.cu[a.num_seqs];
    at = owner_of(a.cu, a.num_seqs, row);
  }
  s.temp = a.temperature[at];
  const int k = a.top_k != nullptr ? a.top_k[at] : 0;
  s.k = k > 0 && k < a.vocab ? k : 0;
  s.p = a.top_p != nullptr ? a.top_p[at] : 1.f;
  const float low = a.min_p != nullptr ? a.min_p[at] : 0.f;
  s.least = low > 0.f ? low < 1.f ? low : 1.f : 0.f;
  return s;
}

template <typename T>
__device__ __forceinline__ const char* row_of(const SampleArgs& a, int64_t row) {
  return static_cast<const char*>(a.logits) + row * a.logits_stride * (__is_same(T, float) ? 4 : 2);
}

// Lanes that hold a group of 32 columns, 16 bytes each; also a thread's pieces of 32 columns.
template <typename T>
constexpr int kTeam = kGroup / kVec<T>;

template <typename T, int PER>
__global__ __launch_bounds__(kThreads) void sample_stats_kernel(const SampleArgs a) {
  __shared__ StatShared<kThreads> sh;
  constexpr int V = kVec<T>, L = kTeam<T>, kPieces = PER / V;
  const int chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks;
  const int base = chunk * kThreads * PER, n = min(kThreads * PER, a.vocab - base);
  const Settings s = settings_of(a, row);
  if (s.none) return;
  float x[PER];
  columns<T, V, kThreads, PER, false>(row_of<T>(a, row), base, n, x);
  chunk_stat<T>(x, s.temp, s.sums(), base, n, a.stats + (int64_t)row * a.chunks + chunk, sh);
  if (!(s.temp > 0.f) || s.all()) return;  // uniform
  // Lane l of a team stores the maximum of piece l.
  const int member = threadIdx.x % L, team = threadIdx.x / L;
  float mine = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    float top = x[i * V];
#pragma unroll
    for (int e = 1; e < V; ++e) top = fmaxf(top, x[i * V + e]);
    top = fmaxf(top, dpp_move<kDppQuadXor1>(top));
    top = fmaxf(top, dpp_move<kDppQuadXor2>(top));
    if constexpr (L == 8) top = fmaxf(top, dpp_move<kDppRowHalfMirror>(top));
    mine = member == i ? top : mine;
  }
  const int group = base / kGroup + member * (kThreads / L) + team;
  if (member < kPieces && group < a.groups) a.maxima[(int64_t)row * a.groups + group] = mine;
}

struct PickShared {
  uint32_t n[kBins];
  uint64_t m[kBins];
  uint64_t part[kPickWaves], part_m[kPickWaves];
  double sum[kPickWaves], goal;
  double round[kMaxRounds];
  uint32_t distance[kListed], column[kListed];  // the columns that matter
  uint16_t group[kSelected];                    // the groups that they lie in
  uint64_t before_n, before_m, bin_n;
  uint32_t member;
  int found, pick[kPickWaves][2], last;
};

// Where the count of columns, or their weight, first reaches a goal: at distance lo .. hi, with n columns of weight m before.
struct Cut {
  uint32_t lo, hi;
  uint64_t n, m, ties;  // ties: columns in the interval
  bool found;
};

template <typename T>
__global__ __launch_bounds__(kPick) void sample_pick_kernel(const SampleArgs a) {
  __shared__ PickShared sh;
  constexpr int V = kVec<T>, L = kTeam<T>, kRound = kPick * V;
  // Keys of different values of the type are at least this far apart.
  constexpr uint32_t kApart = __is_same(T, float) ? 1u : __is_same(T, Bf16) ? 1u << 16 : 1u << 13;
  constexpr uint32_t kNone = 0xffffffffu;  // no column's distance
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const Settings s = settings_of(a, row);
  if (s.none) return;
  const char* at = row_of<T>(a, row);
  const Stat* st = a.stats + (int64_t)row * a.chunks;

  // The row's largest logit, each wave by itself.
  uint64_t best = 0;
  for (int c = lane; c < a.chunks; c += kWave) best = max_u64(best, st[c].key);
  best = wave_max(best);
  const float top = key_value(best);
  if (!(s.temp > 0.f) || !(top > -INFINITY && top < INFINITY)) {
    if (tid == 0) {
      a.tokens[row] = argmax_key_column(best);
      if (s.temp > 0.f) flag_error(a.d_error, TQ_DEVERR_VALUE);
    }
    return;
  }
  const double c = kLog2e / (double)s.temp, t0 = (double)top;
  const uint32_t key = (uint32_t)(argmax_key(top, 0) >> 32);
  auto distance_of = [&](float v) { return key - (uint32_t)(argmax_key(v, 0) >> 32); };
  auto weight = [&](uint32_t d) {
    const double t = ((double)key_value((uint64_t)(key - d) << 32) - t0) * c;
    return t >= -1000.0 ? exp2_neg(t) : 0.0;
  };
  const double unit = __builtin_ldexp(1.0, a.mass_bits);
  auto fixed = [&](double w) {  // w below 2^(52 - mass_bits)
    return __builtin_bit_cast(uint64_t, __builtin_fma(w, unit, 0x1p52)) & 0xfffffffffffffull;
  };
  const double u = (double)a.uniforms[row];

  // The columns at hand: those from `first` to `end`, or the list's, V in a row a thread, a round at a time.
  int first = 0, end = a.vocab, listed = -1, rounds = (a.vocab + kRound - 1) / kRound;
  uint32_t limit = kNone - 1;  // no column past this distance is among the first ranks
  uint32_t d[V];
  auto load = [&](int r) {
    const int i0 = r * kRound + tid * V;
    if (listed >= 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = i0 + e < listed ? sh.distance[i0 + e] : kNone;
    } else {
      float x[V];
      columns<T, V, kPick, V, true>(at, first + r * kRound, end - first - r * kRound, x);
#pragma unroll
      for (int e = 0; e < V; ++e) d[e] = first + i0 + e < end ? distance_of(x[e]) : kNone;
    }
  };
  auto column = [&](int r, int e) {
    const int i = r * kRound + tid * V + e;
    return listed >= 0 ? (int)sh.column[min(i, kListed - 1)] : first + i;
  };
  auto each_column = [&](auto&& use) {
    for (int r = 0; r < rounds; ++r) {
      load(r);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (d[e] <= limit) use(d[e]);
    }
  };
  const float* maxima = a.maxima + (int64_t)row * a.groups;
  auto each_maximum = [&](auto&& use) {
    for (int i = tid; i < a.groups; i += kPick) use(distance_of(maxima[i]));
  };
  // Lists the columns within the limit, in order, if there is room; those of the `many` selected groups, or (-1) of all.
  auto list = [&](int many) {
    const int groups = many >= 0 ? many : a.groups;
    int count = 0;
    for (int g0 = 0; g0 < groups && count <= kListed; g0 += kPick / L) {
      const int slot = g0 + tid / L;
      const int col = (slot < groups ? many >= 0 ? (int)sh.group[slot] : slot : 0) * kGroup + tid % L * V;
      float x[V];
      uint32_t near[V];
      columns<T, V, kPick, V, true>(at, col - tid * V, slot < groups ? a.vocab - col + tid * V : 0, x);
      int mine = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        near[e] = slot < groups && col + e < a.vocab ? distance_of(x[e]) : kNone;
        mine += near[e] <= limit;
      }
      const int upto = (int)scan<kPick>((uint64_t)mine, sh.part);
      int place = count + upto - mine;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (near[e] <= limit) {
          if (place < kListed) {
            sh.distance[place] = near[e];
            sh.column[place] = col + e;
          }
          ++place;
        }
      if (tid == kPick - 1) sh.found = upto;
      __syncthreads();
      count += sh.found;
      __syncthreads();
    }
    if (count <= kListed) {
      listed = count;
      rounds = (count + kRound - 1) / kRound;
    }
  };

  // `apart`: the interval is narrowed down until its columns have one value; 0: as it was found.
  auto find = [&](auto&& each, bool weigh, bool by_mass, double goal, uint32_t apart) {
    Cut r = {0, 0, 0, 0, 0, false};
    int shift = 14;
    for (;;) {
      for (int i = tid; i < kBins; i += kPick) {
        sh.n[i] = 0;
        sh.m[i] = 0;
      }
      if (tid == 0) sh.found = -1;
      __syncthreads();
      each([&](uint32_t v) {
        const uint32_t b = (v - r.lo) >> shift;
        if (v >= r.lo && b < kBins) {
          atomicAdd(&sh.n[b], 1u);
          if (weigh) atomicAdd((unsigned long long*)&sh.m[b], (unsigned long long)fixed(weight(v)));
        }
      });
      __syncthreads();
      const uint64_t na = sh.n[2 * tid], nb = sh.n[2 * tid + 1], ma = sh.m[2 * tid], mb = sh.m[2 * tid + 1];
      const uint64_t n = r.n + scan<kPick>(na + nb, sh.part), m = weigh ? r.m + scan<kPick>(ma + mb, sh.part_m) : 0;
      auto reaches = [&](uint64_t n, uint64_t m) { return by_mass ? (double)m >= goal : (double)n >= goal; };
      const uint64_t n1 = n - na - nb, m1 = m - ma - mb;  // before this thread's
      if (reaches(n, m) && (tid == 0 || !reaches(n1, m1))) {
        const bool one = reaches(n1 + na, m1 + ma);
        sh.found = 2 * tid + (one ? 0 : 1);
        sh.before_n = one ? n1 : n1 + na;
        sh.before_m = one ? m1 : m1 + ma;
        sh.bin_n = one ? na : nb;
      } else if (tid == kPick - 1 && !reaches(n, m)) {
        sh.before_n = n;
        sh.before_m = m;
      }
      __syncthreads();
      const int found = sh.found;
      r.n = sh.before_n;
      r.m = sh.before_m;
      if (found < 0) {
        if (shift == 21) return r;
        r.lo += (uint32_t)kBins << shift;
        shift = 21;
        __syncthreads();
        continue;
      }
      r.found = true;
      r.ties = sh.bin_n;
      r.lo += (uint32_t)found << shift;
      r.hi = r.lo + ((1u << shift) - 1);
      __syncthreads();
      if (apart == 0) return r;
      if (listed < 0 && r.n + r.ties <= kListed) {
        limit = r.hi;
        list(-1);
      }
      if (r.ties == 1 || (1u << shift) <= apart) {
        each([&](uint32_t v) {
          if (v >= r.lo && v <= r.hi) sh.member = v;
        });
        __syncthreads();
        r.lo = r.hi = sh.member;
        return r;
      }
      shift = shift == 14 ? 3 : shift == 21 ? 10 : 0;
    }
  };

  // The sum of the row's weights, and for draws from all of them the chunk that the token falls in.
  double total = 0.0, rest = -1.0;
  if (s.sums()) {
    double mine = 0.0;
    if (tid < a.chunks) {
      const double t = ((double)key_value(st[tid].key) - t0) * c;
      if (t >= -1000.0) mine = st[tid].sum * exp2_neg(t);
    }
    const double upto = scan<kPick>(mine, sh.sum);
    if (tid == kPick - 1) sh.goal = upto;
    __syncthreads();
    total = sh.goal;
    if (s.all()) {
      const double goal = u * total;
      const int chosen = pick<kPick>(mine > 0.0 && upto > goal, mine > 0.0, sh.pick);
      if (tid == chosen) sh.goal = goal - (upto - mine);
      __syncthreads();
      rest = sh.goal;
      first = chosen * a.chunk_columns;
      end = min(first + a.chunk_columns, a.vocab);
      rounds = (end - first + kRound - 1) / kRound;
    }
  }

  // A limit from the groups' maxima, and the groups that reach it.
  if (!s.all()) {
    if (s.k > 0) {
      if (s.k <= a.groups) {
        const Cut cut = find(each_maximum, false, false, (double)s.k, 0);
        if (cut.found) limit = cut.hi;
      }
    } else if (s.nucleus()) {
      const Cut cut = find(each_maximum, true, true, (s.p > 0.f ? (double)s.p : 0.0) * (total * unit), 0);
      if (cut.found) limit = cut.hi;
    } else {
      // Where the weight is `least`, and a little further: the columns are weighed again.
      const double edge = t0 + ((double)__builtin_amdgcn_logf(s.least) - 1e-4) / c;
      const float low = (float)(edge - 1e-6 * __builtin_fabs(edge));
      if (low > -INFINITY) limit = distance_of(low);
    }
    if (limit < kNone - 1) {
      int many = 0;
      for (int i0 = 0; i0 < a.groups; i0 += kPick) {
        const bool in = i0 + tid < a.groups && distance_of(maxima[i0 + tid]) <= limit;
        const uint64_t those = __builtin_amdgcn_ballot_w64(in);
        if (lane == 0) sh.pick[wave][0] = __builtin_popcountll(those);
        __syncthreads();
        int place = many + __builtin_popcountll(those & ((1ull << lane) - 1));
        for (int v = 0; v < kPickWaves; ++v) {
          place += v < wave ? sh.pick[v][0] : 0;
          many += sh.pick[v][0];
        }
        if (in && place < kSelected) sh.group[place] = (uint16_t)(i0 + tid);
        __syncthreads();
      }
      list(many <= kSelected ? many : -1);
    }
  }

  // The first ranks: columns with distance below cut.lo, and the first `ties` of those at it.
  Cut cut = {kNone - 1, kNone - 1, 0, 0, 0, false};
  uint64_t ties = 0;
  bool some = false;  // whether `ties` is less than there are
  if (s.k > 0) {
    cut = find(each_column, s.nucleus(), false, (double)s.k, kApart);
    ties = s.k - cut.n;
    some = cut.found && ties < cut.ties;
  }
  if (s.nucleus()) {
    const double whole = s.k > 0 ? (double)(cut.m + ties * fixed(weight(cut.lo))) : total * unit;
    const double goal = (s.p > 0.f ? (double)s.p : 0.0) * whole;
    const Cut nucleus = find(each_column, true, true, goal, kApart);
    if (nucleus.found) {
      const double each = (double)fixed(weight(nucleus.lo)), need = __builtin_ceil((goal - (double)nucleus.m) / each);
      uint64_t want = need >= 1.0 && need < (double)nucleus.ties ? (uint64_t)need : need < 1.0 ? 1 : nucleus.ties;
      if (s.k > 0 && nucleus.lo == cut.lo && want > ties) want = ties;
      cut = nucleus;
      ties = want;
      some = ties < cut.ties;
    }
  }
  // The column of the last tie that is kept.
  int last = 0x7fffffff;
  if (some) {
    uint64_t before = 0;
    for (int r = 0; r < rounds && before < ties; ++r) {
      load(r);
      uint64_t mine = 0;
#pragma unroll
      for (int e = 0; e < V; ++e) mine += d[e] == cut.lo;
      const uint64_t upto = before + scan<kPick>(mine, sh.part);
      if (upto >= ties && upto - mine < ties) {
        uint64_t left = ties - (upto - mine);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (d[e] == cut.lo && left-- == 1) sh.last = column(r, e);
      }
      if (tid == kPick - 1) sh.before_n = upto;
      __syncthreads();
      before = sh.before_n;
      __syncthreads();
    }
    if (before >= ties) last = sh.last;
  }

  // The draw: the round, then the column.
  const double least = (double)s.least;
  double w[V];
  auto weigh = [&](int r) {
    load(r);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[e] = 0.0;
      if (d[e] < cut.lo || (d[e] == cut.lo && column(r, e) <= last)) {
        const double v = weight(d[e]);
        w[e] = v >= least ? v : 0.0;
      }
      sum += w[e];
    }
    return sum;
  };
  int r = 0;
  double mine = 0.0, upto = 0.0;
  if (rounds > 1) {
    for (r = 0; r < rounds; ++r) {
      const double sum = wave_sum(weigh(r));
      if (lane == 0) sh.sum[wave] = sum;
      __syncthreads();
      if (tid == 0) {
        double all = 0.0;
        for (int v = 0; v < kPickWaves; ++v) all += sh.sum[v];
        sh.round[r] = all;
      }
      __syncthreads();
    }
    mine = tid < rounds ? sh.round[tid] : 0.0;
    upto = scan<kPick>(mine, sh.sum);
    if (tid == kPick - 1) sh.goal = upto;
    __syncthreads();
    const double goal = rest < 0.0 ? u * sh.goal : rest;
    r = max(pick<kPick>(mine > 0.0 && upto > goal, mine > 0.0, sh.pick), 0);
    if (tid == r) sh.goal = goal - (upto - mine);
    __syncthreads();
    rest = sh.goal;
  }
  mine = weigh(r);
  upto = scan<kPick>(mine, sh.sum);
  if (rest < 0.0) {
    if (tid == kPick - 1) sh.goal = upto;
    __syncthreads();
    rest = u * sh.goal;
  }
  if (tid == pick<kPick>(mine > 0.0 && upto > rest, mine > 0.0, sh.pick)) {
    double cum = upto - mine;
    int col = -1;
    bool done = false;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      cum += w[e];
      if (!done && w[e] > 0.0) {
        col = column(r, e);
        done = cum > rest;
      }
    }
    a.tokens[row] = col;
  }
}

struct Plan {
  int per;  // columns of a thread in stats: 8 or 32
  int chunks, groups;
  size_t maxima, bytes;  // offset, size
};

Plan plan_of(int32_t num_rows, int32_t vocab) {
  Plan p;
  auto chunks = [&](int per) { return (vocab + kThreads * per - 1) / (kThreads * per); };
  p.per = (int64_t)num_rows * chunks(32) < 512 && chunks(8) <= kPick ? 8 : 32;
  p.chunks = chunks(p.per);
  p.groups = (vocab + kGroup - 1) / kGroup;
  p.maxima = (size_t)num_rows * p.chunks * sizeof(Stat);
  p.bytes = p.maxima + (size_t)num_rows * p.groups * sizeof(float);
  return p;
}

template <typename T>
tq_status launch(const SampleArgs& a, const Plan& p, hipStream_t stream) {
  const int64_t stats = (int64_t)a.num_rows * a.chunks;
  if (stats > 0x7fffffffLL) return TQ_ERR_UNSUPPORTED;
  if (p.per == 8)
    hipLaunchKernelGGL((sample_stats_kernel<T, 8>), dim3((unsigned)stats), dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((sample_stats_kernel<T, 32>), dim3((unsigned)stats), dim3(kThreads), 0, stream, a);
  const tq_status st = check_launch();
  if (st != TQ_OK) return st;
  hipLaunchKernelGGL((sample_pick_kernel<T>), dim3((unsigned)a.num_rows), dim3(kPick), 0, stream, a);
  return check_launch();
}

}  // namespace
}  // namespace tq

extern "C" size_t tq_sample_tokens_workspace_size(int32_t num_rows, int32_t vocab) {
  using namespace tq;
  if (num_rows < 1 || vocab < 1 || vocab > kMaxVocab) return 0;
  return plan_of(num_rows, vocab).bytes;
}

extern "C" tq_status tq_sample_tokens(int64_t* tokens, const void* logits, int64_t logits_row_stride,
                                      const float* uniforms, const float* temperature, const int32_t* top_k,
                                      const float* top_p, const float* min_p, const int32_t* cu_seqlens_q,
                                      int32_t num_seqs, int32_t num_rows, int32_t vocab, int32_t dtype, void* workspace,
                                      size_t workspace_bytes, int32_t* d_error, void* stream) {
  using namespace tq;
  if (num_seqs < 0 || num_rows < 0 || vocab < 1) return TQ_ERR_INVALID_ARGUMENT;
  if ((dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) || vocab > kMaxVocab) return TQ_ERR_UNSUPPORTED;
  if (num_rows == 0 || num_seqs == 0) return TQ_OK;
  if (tokens == nullptr || logits == nullptr || uniforms == nullptr || temperature == nullptr ||
      (cu_seqlens_q == nullptr && num_seqs < num_rows) || (num_rows > 1 && logits_row_stride < vocab))
    return TQ_ERR_INVALID_ARGUMENT;
  const Plan p = plan_of(num_rows, vocab);
  if (workspace == nullptr || workspace_bytes < p.bytes || (uintptr_t)workspace % 16 != 0) return TQ_ERR_WORKSPACE;
  SampleArgs a;
  a.tokens = tokens;
  a.logits = logits;
  a.logits_stride = logits_row_stride;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.cu = cu_seqlens_q;
  a.stats = static_cast<Stat*>(workspace);
  a.maxima = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.maxima);
  a.d_error = d_error;
  a.num_rows = num_rows;
  a.num_seqs = num_seqs;
  a.vocab = vocab;
  a.chunks = p.chunks;
  a.chunk_columns = kThreads * p.per;
  a.groups = p.groups;
  int bits = 0;
  while (1 << bits < vocab) ++bits;
  a.mass_bits = bits > 12 ? 63 - bits : 51;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == TQ_F32) return launch<float>(a, p, st);
  return dtype == TQ_BF16 ? launch<Bf16>(a, p, st) : launch<Fp16>(a, p, st);
}

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
//    the least of them bounds top-p. Of the groups above the bound, a few more than k, the columns above it are listed in LDS. Where
//    there is no bound (top-p of a flat row), the row is read again to find one.
//
// 1 is bound by HBM (256 rows of 128,000 fp32 logits 23 us, 5.6 TB/s, of which the sums of exponentials, where all rows need them,
// make 31), 2 by its dependent steps of 1-3 us: one row of 50,257 with top-k 50 and top-p 11 us, from the temperature alone 5.6, with top-k
// 1,000 23; 256 rows of 128,000 with settings of all kinds 24. Read and ranked by one workgroup a row in passes over all of its columns, one row
// took 103 us and the 256 273. Top-p 0.9 of 256 x 128,000 normal logits, some 5,700 columns each, takes 96.
#include <type_traits>

#include "draw.h"

namespace tq {
namespace {

constexpr int kThreads = 256;       // of a chunk's workgroup
constexpr int kGroup = 32;          // columns of a group
constexpr int kPick = 1024;         // threads of a row's workgroup
constexpr int kPickWaves = kPick / kWave;
constexpr int kBins = 2 * kPick;
constexpr int kListed = 8192;       // columns that are kept in LDS; rows of which more matter are read again
constexpr int kRanked = 1024;       // of them, those that are ranked by comparing each with each; at most kPick
constexpr int kSelected = 4096;     // groups whose columns are listed; if more reach the limit, all are looked at
constexpr int kMaxVocab = 1 << 21;
constexpr int kFewRanks = 4096;     // of top-k: their weights' roundings in units of the vocabulary's stay below those of the row's
constexpr int kRound = 4 * kPick;
constexpr int kMaxRounds = kMaxVocab / kRound;
static_assert(kMaxRounds <= kPick && kRanked <= kPick && kMaxVocab / kGroup <= 1 << 16, "an entry a thread, groups in 16 bits");

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
  int32_t mass_bits;  // weights are counted in units of 2^-mass_bits, where the row's sum is not known
};

// A row's settings.
struct Settings {
  float temp, p, least;
  int k;      // 0: off
  bool none;  // the row is in no sequence

  __device__ __forceinline__ bool nucleus() const { return p < 1.f; }
  __device__ __forceinline__ bool all() const { return k == 0 && !nucleus() && !(least > 0.f); }
  // Whether the sum of the whole row's weights is asked for.
  __device__ __forceinline__ bool sums() const { return nucleus() ? k == 0 || k > kFewRanks : k == 0 && !(least > 0.f); }
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

// Inclusive sums over the row's workgroup, in order, of 32- or 64-bit values. The waves' sums are added up in a row of 16 lanes, by every
// wave. One barrier: calls that follow each other take turns with s_part (16 words each), and so does `first_of`.
template <int CTRL, typename V>
__device__ __forceinline__ V dpp_of(V v) {
  if constexpr (sizeof(V) == 4)
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
  else
    return __builtin_bit_cast(V, dpp_move64<CTRL>(__builtin_bit_cast(uint64_t, v)));
}
template <typename V>
__device__ __forceinline__ V lane_value(V v, int lane) {
  if constexpr (sizeof(V) == 4)
    return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  else
    return __builtin_bit_cast(V, lane_of(__builtin_bit_cast(uint64_t, v), lane));
}
template <typename V>
__device__ __forceinline__ V row_sums(V v) {  // inclusive, in rows of 16 lanes
  v += dpp_of<0x111>(v);  // row_shr:1, 2, 4, 8
  v += dpp_of<0x112>(v);
  v += dpp_of<0x114>(v);
  v += dpp_of<0x118>(v);
  return v;
}
template <typename V>
__device__ __forceinline__ V wave_sums(V v) {
  const int lane = threadIdx.x & (kWave - 1);
  v = row_sums(v);
  V before = 0;
#pragma unroll
  for (int r = 1; r < kWave / 16; ++r) {
    const V row = lane_value(v, 16 * r - 1);
    before += lane >= 16 * r ? row : 0;
  }
  return v + before;
}
// all: the sum of all threads' values.
template <typename V>
__device__ __forceinline__ V sums(V v, uint64_t* s_part, V& all) {
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  v = wave_sums(v);
  V* part = reinterpret_cast<V*>(s_part);
  if (lane == kWave - 1) part[wave] = v;
  __syncthreads();
  static_assert(kPickWaves == 16, "the waves' sums in a row of lanes");
  const V mine = part[lane & 15], upto = row_sums(mine);
  all = lane_value(upto, 15);
  return v + lane_value(upto - mine, wave);
}
// The first thread with `over`, or the last with `has` where there is none; -1: none either.
__device__ __forceinline__ int first_of(bool over, bool has, uint64_t* s_part) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const uint64_t overs = __builtin_amdgcn_ballot_w64(over), those = __builtin_amdgcn_ballot_w64(has);
  int* part = reinterpret_cast<int*>(s_part);
  if (lane == 0) {
    part[2 * wave] = overs != 0 ? wave * kWave + __builtin_ctzll(overs) : -1;
    part[2 * wave + 1] = those != 0 ? wave * kWave + 63 - __builtin_clzll(those) : -1;
  }
  __syncthreads();
  const int2 mine = reinterpret_cast<const int2*>(part)[lane & 15];
  const uint64_t first = __builtin_amdgcn_ballot_w64(mine.x >= 0) & 0xffff, last = __builtin_amdgcn_ballot_w64(mine.y >= 0) & 0xffff;
  if (first != 0) return __builtin_amdgcn_readlane(mine.x, __builtin_ctzll(first));
  return last != 0 ? __builtin_amdgcn_readlane(mine.y, 63 - __builtin_clzll(last)) : -1;
}

struct PickShared {
  uint32_t n[kBins];
  uint64_t m[kBins];
  uint64_t part[2][kPickWaves];
  double sum[kPickWaves], goal;
  double round[kMaxRounds];
  alignas(16) uint32_t distance[kListed + 4], column[kListed];  // the columns that matter
  uint16_t group[kSelected];                                    // the groups that they lie in
  uint64_t before_n, before_m, bin_n;
  uint32_t member;
  int found, last;
};

// What is gone through, four items in a row a thread, a round of all threads at a time: the maxima of the groups, the columns of the
// selected groups, those of the row (or of one chunk), those listed in LDS.
enum Source { kMaxima, kGroups, kColumns, kList };

// One code for all steps and sources, rolled where few items go through it: a row's workgroup runs most of it once, and is held up by the
// fetching of instructions, a microsecond a kilobyte (unrolled over four rounds everywhere: top-k 50 of one row 13.5 -> 20 us), and by
// scratch memory (with registers spilled there, 12 us more of every call).
template <typename T>
__global__ __launch_bounds__(kPick) void sample_pick_kernel(const SampleArgs a) {
  __shared__ PickShared sh;
  // Keys of different values of the type are at least this far apart.
  constexpr uint32_t kApart = __is_same(T, float) ? 1u : __is_same(T, Bf16) ? 1u << 16 : 1u << 13;
  constexpr uint32_t kNone = 0xffffffffu;  // no column's distance
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const Settings s = settings_of(a, row);
  if (s.none) return;
  const char* at = row_of<T>(a, row);
  const float* maxima = a.maxima + (int64_t)row * a.groups;
  const Stat* st = a.stats + (int64_t)row * a.chunks;
  const double u = (double)a.uniforms[row];
  int turn = 0;
  auto part = [&] { return sh.part[turn ^= 1]; };

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
  int mass_bits = a.mass_bits;
  double unit = __builtin_ldexp(1.0, mass_bits);
  auto fixed = [&](double w) {  // w at most 1, mass_bits at most 51
    return __builtin_bit_cast(uint64_t, __builtin_fma(w, unit, 0x1p52)) & 0xfffffffffffffull;
  };

  // The same nearly, for a search that is made again with exact ones where it ends: by an exponential that is off by 2e-6 (of
  // exponents up to 30), in units of 2^-31; `slack` is more than both. Not where T is so small that c is infinite in 32 bits: then
  // there is no such search.
  const float cf = (float)c;
  auto nearly = [&](uint32_t d) {
    const float w = __builtin_amdgcn_exp2f((key_value((uint64_t)(key - d) << 32) - top) * cf);
    return (uint64_t)(uint32_t)(w * 0x1p31f) << (mass_bits - 31);
  };
  const double slack = 1.0 + 1e-4 + a.vocab * 0x1p-31;

  Source source = kColumns;
  int first = 0, items = a.vocab;  // of the source; columns from `first` on
  auto column = [&](Source from, int i) {
    return from == kList ? (int)sh.column[i] : from == kGroups ? sh.group[i / kGroup] * kGroup + i % kGroup : first + i;
  };
  // Items i .. i + 3 of `many`, NaN past them: no other item is. Not of kList.
  auto load = [&](Source from, int i, int many, float (&x)[4]) {
    const bool wide = __is_same(T, float) || from == kMaxima;
    int j = i, end = many;  // places in the array
    if (from == kGroups) {
      j = column(kGroups, min(i, many - 1));
      end = i < many ? a.vocab : j;
    } else if (from == kColumns) {
      j += first;
      end += first;
    }
    const char* p = from == kMaxima ? reinterpret_cast<const char*>(maxima) : at;
    if (j + 4 <= end) {
      if (wide) {
        u32x4 v;
        __builtin_memcpy(&v, p + 4 * (int64_t)j, 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
      } else if constexpr (!__is_same(T, float)) {
        u32x2 v;
        __builtin_memcpy(&v, p + 2 * (int64_t)j, 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = T::load((uint16_t)(v[e / 2] >> (16 * (e & 1))));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = j + e < end ? wide ? reinterpret_cast<const float*>(p)[j + e] : logit_at<T>(p, j + e) : __builtin_nanf("");
    }
  };

  // The same of N rounds, whose loads are on their way together: of columns, where N > 1.
  auto load_rounds = [&](Source from, int i0, int many, auto& x) {
    constexpr int N = sizeof(x) / sizeof(x[0]);
    typedef typename std::conditional<__is_same(T, float), u32x4, u32x2>::type Raw;
    if constexpr (N == 1) {
      load(from, i0, many, x[0]);
      return;
    }
    Raw v[N];
    bool full[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int i = i0 + j * kRound, col = column(from, min(i, many - 4));
      full[j] = i + 4 <= many && col + 4 <= a.vocab;
      const char* p = full[j] ? at + (int64_t)col * (sizeof(Raw) / 4) : reinterpret_cast<const char*>(a.stats);
      __builtin_memcpy(&v[j], p, sizeof(Raw));
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (full[j]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (__is_same(T, float))
            x[j][e] = __uint_as_float(v[j][e]);
          else
            x[j][e] = T::load((uint16_t)(v[j][e / 2] >> (16 * (e & 1))));
        }
      } else {
        load(from, i0 + j * kRound, many, x[j]);
      }
    }
  };

  // Their distances; kNone past the last.
  auto fetch = [&](Source from, int i, int many, auto& d) {
    constexpr int N = sizeof(d) / sizeof(d[0]);
    if (N == 1 && from == kList) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(&sh.distance[min(i, kListed)]);
#pragma unroll
      for (int e = 0; e < 4; ++e) d[0][e] = i + e < many ? v[e] : kNone;
      return;
    }
    float x[N][4];
    load_rounds(from, i, many, x);
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) d[j][e] = x[j][e] == x[j][e] ? distance_of(x[j][e]) : kNone;
  };

  // What is left of the goal behind what lies before a thread: `upto - mine` is not the sum before it bit for bit, and may be a few
  // roundings past a goal that meets this border. Below 0 means that there is no goal yet.
  auto behind = [](double goal, double before) { return goal < before ? 0.0 : goal - before; };

  // The sum of the row's weights, and for draws from all of them the chunk that the token falls in.
  double total = 0.0, rest = -1.0;
  if (s.sums()) {
    double mine = 0.0;
    if (tid < a.chunks) {
      const double t = ((double)key_value(st[tid].key) - t0) * c;
      if (t >= -1000.0) mine = st[tid].sum * exp2_neg(t);
    }
    const double upto = sums(mine, part(), total);
    // As fine as the sum allows, that of all weights below 2^63 units: a peaked row's many tiny weights are not rounded away together.
    // Off by half a unit each, they are off by less than vocab 2^-51 of the sum; so are up to kFewRanks in units of the vocabulary's.
    mass_bits = min(51, 63 - __builtin_amdgcn_frexp_exp(total));
    unit = __builtin_ldexp(1.0, mass_bits);
    if (s.all()) {
      const double goal = u * total;
      const int chosen = first_of(mine > 0.0 && upto > goal, mine > 0.0, part());
      if (tid == chosen) sh.goal = behind(goal, upto - mine);
      __syncthreads();
      rest = sh.goal;
      first = chosen * a.chunk_columns;
      items = min(a.chunk_columns, a.vocab - first);
    }
  }

  // 0: a limit from the maxima, past which no column is among the first ranks, and a list of those up to it. 1: top-k, 2: top-p: columns with
  // distance below `cut`, and the first `ties` of those at it.
  uint32_t limit = kNone - 1, cut = kNone - 1;
  uint64_t ties = 0, cut_m = 0;
  bool some = false;  // whether `ties` is less than there are
  double whole = total * unit;
#pragma unroll 1
  for (int job = s.all() ? 3 : 0; job < 3; ++job) {
    bool run = job == 0 ? s.k > 0 ? s.k <= a.groups : s.nucleus() : job == 1 ? s.k > 0 : s.nucleus();
    const bool by_mass = job == 0 ? s.k == 0 : job == 2, weigh = by_mass || (job == 1 && s.nucleus());
    if (job == 2 && s.k > 0) whole = (double)(cut_m + ties * fixed(weight(cut)));
    const double goal = by_mass ? (s.p > 0.f ? (double)s.p : 0.0) * whole : (double)s.k;
    int make = -1;  // the source to be listed
    if (job == 0 && !run && s.k == 0) {
      // Where the weight is `least`, and a little further: the columns are weighed again.
      const double edge = t0 + ((double)__builtin_amdgcn_logf(s.least) - 1e-4) / c;
      const float low = (float)(edge - 1e-6 * __builtin_fabs(edge));
      if (low > -INFINITY) {
        limit = distance_of(low);
        make = kMaxima;
      }
    }
    bool scouted = !(cf < INFINITY);
    uint32_t lo = 0;
    uint64_t n0 = 0, m0 = 0;  // before lo
    int shift = 14;
#pragma unroll 1
    while (run || make >= 0) {
      if (make >= 0) {
        // Items up to the limit, in order: the waves count theirs, and each adds up all counts.
        const Source from = (Source)make;
        const int many = from == kMaxima ? a.groups : from == kGroups ? items * kGroup : a.vocab;
        const int room = from == kMaxima ? kSelected : kListed;
        int count = 0, side = 0;
        // The least value up to the limit (past the last key: -inf).
        float low = limit <= key ? key_value((uint64_t)(key - limit) << 32) : -INFINITY;
        low = low == low ? low : -INFINITY;
        auto take = [&](int i0, auto& x) {
          constexpr int N = sizeof(x) / sizeof(x[0]);
          load_rounds(from, i0 + 4 * tid, many, x);
          int place[N];
#pragma unroll
          for (int j = 0; j < N; ++j) {
            int all = 0;
            place[j] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t those = __builtin_amdgcn_ballot_w64(x[j][e] >= low);
              all += __builtin_popcountll(those);
              place[j] = __builtin_amdgcn_mbcnt_hi((uint32_t)(those >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)those, place[j]));
            }
            if (lane == 0) sh.n[side * kWave + j * kPickWaves + wave] = all;
          }
          static_assert(4 * kPickWaves == kWave, "a count a lane");
          __syncthreads();
          const int mine = lane < N * kPickWaves ? sh.n[side * kWave + lane] : 0;
          int upto = mine;
          auto up = [&](auto ctrl) { return __builtin_amdgcn_update_dpp(0, upto, decltype(ctrl)::value, 0xF, 0xF, true); };
          upto += up(std::integral_constant<int, 0x111>());  // in rows of 16: row_shr:1, 2, 4, 8
          upto += up(std::integral_constant<int, 0x112>());
          upto += up(std::integral_constant<int, 0x114>());
          upto += up(std::integral_constant<int, 0x118>());
#pragma unroll
          for (int j = 0; j < N; ++j) {
            static_assert(kPickWaves == 16, "a round a row of lanes");
            int to = count + place[j] + __builtin_amdgcn_readlane(upto - mine, j * kPickWaves + wave);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (x[j][e] >= low) {
                const int i = i0 + j * kRound + 4 * tid + e;
                if (to < room) {
                  if (from == kMaxima) {
                    sh.group[to] = (uint16_t)i;
                  } else {
                    sh.distance[to] = distance_of(x[j][e]);
                    sh.column[to] = column(from, i);
                  }
                }
                ++to;
              }
            count += __builtin_amdgcn_readlane(upto, j * kPickWaves + kPickWaves - 1);
          }
          side ^= 1;
        };
        int i0 = 0;
        float one[1][4], four[4][4];
#pragma unroll 1
        for (; from != kMaxima && i0 + 2 * kRound < many && count <= room; i0 += 4 * kRound) take(i0, four);
#pragma unroll 1
        for (; i0 < many && count <= room; i0 += kRound) take(i0, one);
        __syncthreads();
        if (from == kMaxima) {
          make = count <= kSelected ? kGroups : kColumns;
          items = count <= kSelected ? count : items;
        } else {
          make = -1;
          source = count <= kListed ? kList : kColumns;
          items = count <= kListed ? count : a.vocab;
        }
        continue;
      }
      const Source from = job == 0 ? kMaxima : source;
      const int many = job == 0 ? a.groups : items;
      for (int i = tid; i < kBins; i += kPick) {
        sh.n[i] = 0;
        sh.m[i] = 0;
      }
      if (tid == 0) sh.found = -1;
      __syncthreads();
      const bool scout = from == kColumns && !scouted;
      auto tally = [&](int i0, auto& d) {
        constexpr int N = sizeof(d) / sizeof(d[0]);
        fetch(from, i0 + 4 * tid, many, d);
#pragma unroll
        for (int j = 0; j < N; ++j) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = d[j][e], b = (v - lo) >> shift;
            if (v >= lo && v <= limit && b < kBins) {
              atomicAdd(&sh.n[b], 1u);
              if (scout ? by_mass : weigh)
                atomicAdd((unsigned long long*)&sh.m[b], (unsigned long long)(scout ? nearly(v) : fixed(weight(v))));
            }
          }
        }
      };
      int i0 = 0;
      uint32_t one[1][4], four[4][4];
      if (from == kColumns)
#pragma unroll 1
        for (; i0 + 2 * kRound < many; i0 += 4 * kRound) tally(i0, four);
#pragma unroll 1
      for (; i0 < many; i0 += kRound) tally(i0, one);
      __syncthreads();
      const uint32_t na = sh.n[2 * tid], nb = sh.n[2 * tid + 1];
      uint32_t all_n;
      const uint32_t n = (uint32_t)n0 + sums(na + nb, part(), all_n);
      uint64_t ma = 0, mb = 0, m = 0, all_m = 0;
      if (scout ? by_mass : weigh) {
        ma = sh.m[2 * tid];
        mb = sh.m[2 * tid + 1];
        m = m0 + sums(ma + mb, part(), all_m);
      }
      const double aim = scout && by_mass ? goal * slack : goal;
      auto reaches = [&](uint32_t n, uint64_t m) { return (by_mass ? (double)m : (double)n) >= aim; };
      const uint32_t n1 = n - na - nb;  // before this thread's
      const uint64_t m1 = m - ma - mb;
      if (reaches(n, m) && (tid == 0 || !reaches(n1, m1))) {
        const bool one = reaches(n1 + na, m1 + ma);
        sh.found = 2 * tid + (one ? 0 : 1);
        sh.before_n = one ? n1 : n1 + na;
        sh.before_m = one ? m1 : m1 + ma;
        sh.bin_n = one ? na : nb;
      }
      __syncthreads();
      const int found = sh.found;
      n0 = found < 0 ? n0 + all_n : sh.before_n;
      m0 = found < 0 ? m0 + all_m : sh.before_m;
      const uint64_t there = sh.bin_n;
      __syncthreads();
      if (scout) {
        // Few enough up to the interval: the search begins again among them; else with all, and exact weights.
        if (found >= 0 && n0 + there <= kListed) {
          limit = lo + ((uint32_t)(found + 1) << shift) - 1;
          make = kColumns;
        }
        if (found >= 0 || shift == 21) {
          scouted = true;
          lo = 0;
          n0 = m0 = 0;
          shift = 14;
          continue;
        }
      }
      if (found < 0) {
        run = shift != 21;
        lo += (uint32_t)kBins << shift;
        shift = 21;
        continue;
      }
      lo += (uint32_t)found << shift;
      const uint32_t hi = lo + ((1u << shift) - 1);
      if (job == 0) {
        limit = hi;
        make = kMaxima;
        run = false;
        continue;
      }
      if (there > 1 && (1u << shift) > kApart) {
        shift = shift == 14 ? 3 : shift == 21 ? 10 : 0;
        continue;
      }
      // The interval holds one value.
#pragma unroll 1
      for (int i = 4 * tid; i < many; i += kRound) {
        uint32_t d[1][4];
        fetch(from, i, many, d);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d[0][e] >= lo && d[0][e] <= hi) sh.member = d[0][e];
      }
      __syncthreads();
      const uint32_t value = sh.member;
      uint64_t want = there;
      if (job == 1) {
        want = s.k - n0;
      } else {
        const double each = (double)fixed(weight(value)), need = __builtin_ceil((goal - (double)m0) / each);
        want = need >= 1.0 && need < (double)there ? (uint64_t)need : need < 1.0 ? 1 : there;
        if (s.k > 0 && value == cut && want > ties) want = ties;
      }
      cut = value;
      cut_m = m0;
      ties = want;
      some = want < there;
      run = false;
    }

    // Few: each column's rank is counted, and the ranks are weighed in their order.
    if (job == 0 && source == kList && items <= kRanked) {
      // Up to 16 neighbouring lanes take a column, each every so many-th four of the others.
      if (tid < 4) sh.distance[items + tid] = kNone;
      __syncthreads();
      int lanes = 1;
      while (lanes < 16 && 2 * lanes * items <= kPick) lanes *= 2;
      const int of = tid / lanes;
      if (of < items) {
        const uint32_t its = sh.distance[of];
        float count = 0.f;
#pragma unroll 2
        for (int i = 4 * (tid % lanes); i < items; i += 4 * lanes) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(&sh.distance[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) count += v[e] < its + (i + e < of ? 1u : 0u) ? 1.f : 0.f;
        }
        if (lanes > 1) count += dpp_move<kDppQuadXor1>(count);
        if (lanes > 2) count += dpp_move<kDppQuadXor2>(count);
        if (lanes > 4) count += dpp_move<kDppRowHalfMirror>(count);
        if (lanes > 8) count += dpp_move<kDppRowMirror>(count);
        if (tid % lanes == 0) sh.n[of] = (uint32_t)count;
      }
      __syncthreads();
      const int rank = tid < items ? (int)sh.n[tid] : 0;
      const double w = tid < items ? weight(sh.distance[tid]) : 0.0;
      if (tid < items) sh.m[rank] = fixed(w);
      __syncthreads();
      const int k = s.k > 0 ? s.k : items;
      const uint64_t m = tid < min(k, items) ? sh.m[tid] : 0;
      uint64_t all_m;
      const uint64_t upto = sums(m, part(), all_m);
      const double edge = (s.p > 0.f ? (double)s.p : 0.0) * (s.k > 0 ? (double)all_m : whole);
      sh.n[tid] = tid == 0 || (tid < k && (!s.nucleus() || (double)(upto - m) < edge));
      __syncthreads();
      const double kept = tid < items && sh.n[rank] != 0 && w >= (double)s.least ? w : 0.0;
      double all;
      const double cum = sums(kept, part(), all);
      if (tid == first_of(kept > 0.0 && cum > u * all, kept > 0.0, part())) a.tokens[row] = sh.column[tid];
      return;
    }
  }

  const int rounds = (items + kRound - 1) / kRound;
  // The column of the last tie that is kept.
  int last = 0x7fffffff;
  if (some) {
    uint64_t before = 0;
#pragma unroll 1
    for (int i0 = 0; i0 < items && before < ties; i0 += kRound) {
      uint32_t d[1][4];
      fetch(source, i0 + 4 * tid, items, d);
      uint32_t mine = 0, all;
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += d[0][e] == cut;
      const uint64_t upto = before + sums(mine, part(), all);
      if (upto >= ties && upto - mine < ties) {
        uint64_t left = ties - (upto - mine);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d[0][e] == cut && left-- == 1) sh.last = column(source, i0 + 4 * tid + e);
      }
      before += all;
    }
    __syncthreads();
    if (before >= ties) last = sh.last;
  }

  // The draw: the round, then the column.
  double mine = 0.0, upto = 0.0, w[4];
  int r = 0;
  bool found = rounds == 1;
#pragma unroll 1
  for (;;) {
    const int i = r * kRound + 4 * tid;
    uint32_t d[1][4];
    fetch(source, i, items, d);
    mine = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = 0.0;
      if (d[0][e] < cut || (d[0][e] == cut && column(source, min(i + e, items - 1)) <= last)) w[e] = weight(d[0][e]);
      w[e] = w[e] >= (double)s.least ? w[e] : 0.0;
      mine += w[e];
    }
    if (found) break;
    const double sum = wave_sum(mine);
    if (lane == 0) sh.sum[wave] = sum;
    __syncthreads();
    if (tid == 0) {
      double all = 0.0;
      for (int v = 0; v < kPickWaves; ++v) all += sh.sum[v];
      sh.round[r] = all;
    }
    __syncthreads();
    if (++r < rounds) continue;
    mine = tid < rounds ? sh.round[tid] : 0.0;
    double all;
    upto = sums(mine, part(), all);
    const double goal = rest < 0.0 ? u * all : rest;
    r = max(first_of(mine > 0.0 && upto > goal, mine > 0.0, part()), 0);
    if (tid == r) sh.goal = behind(goal, upto - mine);
    __syncthreads();
    rest = sh.goal;
    found = true;
  }
  double all;
  upto = sums(mine, part(), all);
  if (rest < 0.0) rest = u * all;
  if (tid == first_of(mine > 0.0 && upto > rest, mine > 0.0, part())) {
    double cum = upto - mine;
    int at_item = -1;
    bool done = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      cum += w[e];
      if (!done && w[e] > 0.0) {
        at_item = r * kRound + 4 * tid + e;
        done = cum > rest;
      }
    }
    a.tokens[row] = column(source, at_item);
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
  if (!grid_fits(stats, kThreads) || !grid_fits(a.num_rows, kPick)) return TQ_ERR_UNSUPPORTED;
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
  if (num_rows == 0 || (num_seqs == 0 && cu_seqlens_q != nullptr)) return TQ_OK;
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

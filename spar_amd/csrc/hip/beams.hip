// Beam search's choice: the best tokens of a group of rows of logits, and the rows of
// states in the order of the beams they go on from.
//
// The total of token k of row r is score[r] + x[r][k] - lse(x[r]).  Within a row totals are
// in the order of the logits, so that a wave keeps the best `picks` logits of the part of a
// row it reads, together with the part's maximum and sum of exponentials, before lse is
// known: one pass over the logits.  A workgroup per group then joins the parts' sums, forms
// the totals of what was kept, in double, and chooses.  The exponentials and a lane's sums of
// them within a chunk are of the logits' type: in float32 a log-sum was off by 2e-7 at most and
// 2e-8 at the median (rows of 700 to 131072 normal logits times 3), less than a total's rounding
// to it.  Such rows are read at 4.3 TB/s (1024 of 32000), rows of doubles, with exponentials in
// double, at 2.3 (128 of 50000).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "common.hpp"

namespace spar_hip {
namespace beams {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kPieces = 8;               // 16-byte pieces of a lane's share of a chunk
constexpr uint32_t kMostParts = kWave;   // of a row
constexpr uint32_t kNone = ~0U;          // no token

template <typename T>
constexpr uint32_t kChunk = kWave * kPieces * Vec16<T>::width;

// Candidates a wave holds: what half a chunk brings at most behind the best so far.
template <typename T>
constexpr uint32_t kKept = kChunk<T> / 2 + SPAR_HIP_MAX_BEAMS;

// Whole numbers in the order of the values (of any but NaN; -0 before +0).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000U ? ~u : u | 0x80000000U;
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
  return u >> 63 ? ~u : u | uint64_t{1} << 63;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000U ? key & 0x7fffffffU : ~key);
}
__device__ __forceinline__ double value_of(uint64_t key) {
  return __longlong_as_double(
      static_cast<int64_t>(key >> 63 ? key & ~(uint64_t{1} << 63) : ~key));
}
// -0 and +0 are equal logits.
template <typename T>
__device__ __forceinline__ auto key_of(T x) {
  return ordered(x == T(0) ? T(0) : x);
}

__device__ __forceinline__ float exp_of(float x) {
  return __builtin_amdgcn_exp2f(x * 1.44269504088896340736F);
}
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

template <typename T>
__device__ __forceinline__ T infinity() {
  return static_cast<T>(__builtin_huge_val());
}

// Passes over NaN.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }

__device__ __forceinline__ uint32_t count_of(bool flag) {
  return static_cast<uint32_t>(__popcll(__ballot(flag)));
}

// The largest key that at least `wanted` of the wave's keys reach, of its BITS highest bits:
// bit by bit, from the top.  counted(key) is how many reach it.
template <typename Key, int BITS = 8 * sizeof(Key), typename Counted>
__device__ __forceinline__ Key kth_largest(uint32_t wanted, Counted&& counted) {
  Key found = 0;
  Key bit = Key{1} << (8 * sizeof(Key) - 1);
#pragma unroll 1
  for (int i = 0; i < BITS; ++i, bit >>= 1) {
    if (counted(found | bit) >= wanted) found |= bit;
  }
  return found;
}

template <typename T>
struct Rows {
  const T* logits;
  uint64_t stride;
  const int32_t* ended;
  uint32_t vocabulary;
  uint32_t parts;   // of a row
  uint32_t picks;
  uint32_t slots;   // of a part's candidates, at least picks
  double* maxima;   // [row][part]
  double* sums;     // the same
  T* values;        // [row][part][slot], in no order
  uint32_t* tokens; // the same, kNone behind the last
};

// What a wave has kept, in LDS: the candidates in the order of their finding.
template <typename T>
struct Kept {
  T value[kKept<T>];
  uint32_t token[kKept<T>];
};

// Keeps the best `picks` of `count` candidates (more than picks): those above the
// picks-th largest value, and of those equal to it the lowest tokens.  Returns that value.
// The loops over bits stay loops: unrolled, they would be most of a kernel that runs its
// code once.
template <typename T, int SHARE>
__device__ __forceinline__ T compact(Kept<T>& kept, uint32_t count, uint32_t picks, int lane) {
  using Key = decltype(key_of(T(0)));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  Key key[SHARE];
  uint32_t token[SHARE];
#pragma unroll
  for (int i = 0; i < SHARE; ++i) {
    const uint32_t at = lane + i * kWave;
    token[i] = at < count ? kept.token[at] : kNone;
    key[i] = at < count ? key_of(kept.value[at]) : Key{0};
  }
  const auto counted = [&](auto&& flag) {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < SHARE; ++i) n += count_of(flag(i));
    return n;
  };
  const Key border = kth_largest<Key>(
      picks, [&](Key at) { return counted([&](int i) { return key[i] >= at; }); });
  const uint32_t above = counted([&](int i) { return key[i] > border; });
  // Of the tokens at the border the (picks - above) lowest: those whose complement is
  // among the largest.  Mostly there is one.
  const uint32_t reached = counted([&](int i) { return key[i] >= border; });
  uint32_t last = kNone;
  if (reached != picks) {
    last = ~kth_largest<uint32_t>(picks - above, [&](uint32_t at) {
      return counted([&](int i) { return (key[i] == border) & (~token[i] >= at); });
    });
  }
  uint32_t next = 0;
#pragma unroll
  for (int i = 0; i < SHARE; ++i) {
    const bool stays = (key[i] > border) | ((key[i] == border) & (token[i] <= last));
    const uint64_t mask = __ballot(stays);
    if (stays) {
      const uint32_t to = next + __popcll(mask & ((uint64_t{1} << lane) - 1));
      kept.value[to] = value_of(key[i]);
      kept.token[to] = token[i];
    }
    next += static_cast<uint32_t>(__popcll(mask));
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return value_of(border);
}
// Most waves hold few candidates, all a wave has room for hardly any.
constexpr int kFew = 2, kMore = 5;
// Lanes with a candidate that are worth a higher bar.  Without one a chunk brings as many
// candidates as the first: 1024 rows of 32000 with 32 picks took 54 us for 31.  Where every
// chunk looks for one, 256 rows with 8 picks take 28 for 25.
constexpr uint32_t kWorth = 16;
template <typename T>
constexpr int kAll = kKept<T> / kWave;
static_assert(kKept<float> % kWave == 0 && kKept<double> % kWave == 0);

// The largest value below x.
template <typename T>
__device__ __forceinline__ T below(T x) {
  const auto key = key_of(x);
  return value_of(static_cast<decltype(key_of(x))>(key - (key == key_of(T(0)) ? 2 : 1)));
}

// A wave per part of a row: chunks of the part one after the other, the next one's loads in
// flight.  Bound by memory: 1024 rows of 32000 with 32 picks in 31 us, 4.3 TB/s, and by the
// start and the end of 8 chunks a wave.  A candidate is what exceeds `bar`, below which the
// row's picks-th best cannot lie; it comes from the lanes' maxima so far, and waves of a
// workgroup that read the same row share the highest of theirs.
template <typename T>
__global__ __launch_bounds__(kThreads, 2) void row_kernel(Rows<T> rows, uint32_t waves,
                                                          FastDiv by_parts) {
  constexpr int W = Vec16<T>::width;
  constexpr int E = kPieces * W;
  using Key = decltype(key_of(T(0)));
  __shared__ Kept<T> all_kept[kWaves];
  __shared__ T bars[kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const uint32_t id = blockIdx.x * kWaves + wave;
  bars[wave] = -infinity<T>();
  __syncthreads();
  if (id >= waves) return;
  const uint32_t row = by_parts.div(id);
  const uint32_t part = id - row * rows.parts;
  if (rows.ended != nullptr && rows.ended[row] != 0) return;
  bool shares[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) shares[w] = by_parts.div(blockIdx.x * kWaves + w) == row;
  Kept<T>& kept = all_kept[wave];
  const T* logits = rows.logits + row * rows.stride;
  const uint32_t chunks = (rows.vocabulary + kChunk<T> - 1) / kChunk<T>;
  const uint32_t begin =
      static_cast<uint32_t>(static_cast<uint64_t>(chunks) * part / rows.parts);
  const uint32_t end =
      static_cast<uint32_t>(static_cast<uint64_t>(chunks) * (part + 1) / rows.parts);
  const uint32_t picks = rows.picks;

  // Element i of the lane: token chunk + (i / W * 64 + lane) * W + i % W.
  const auto load = [&](T (&x)[E], uint32_t chunk) {
    const uint32_t first = chunk * kChunk<T> + lane * W;
    if ((chunk + 1) * static_cast<uint64_t>(kChunk<T>) <= rows.vocabulary) {
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const auto piece = loose_load(logits + first + p * kWave * W);
#pragma unroll
        for (int j = 0; j < W; ++j) x[p * W + j] = piece[j];
      }
    } else {  // and the row's last token in the place of those behind
#pragma unroll
      for (int i = 0; i < E; ++i) {
        x[i] = logits[min(first + i / W * kWave * W + i % W, rows.vocabulary - 1)];
      }
    }
  };
  T top = sizeof(T) == 4 ? static_cast<T>(-__FLT_MAX__) : static_cast<T>(-__DBL_MAX__);
  double sum = 0.0;
  T best = -infinity<T>();  // of the lane
  T bar = -infinity<T>();
  uint32_t count = 0;
  T x[E], next[E];
  load(x, begin);
  // Waited for here (vmcnt(0)), or the loop's first use of it would wait for the next chunk's
  // loads in every round.
  __builtin_amdgcn_s_waitcnt(0x0f70);
  for (uint32_t chunk = begin; chunk < end; ++chunk) {
    if (chunk + 1 < end) load(next, chunk + 1);
    if ((chunk + 1) * static_cast<uint64_t>(kChunk<T>) > rows.vocabulary) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const uint32_t token = chunk * kChunk<T> + (i / W * kWave + lane) * W + i % W;
        if (token >= rows.vocabulary) x[i] = -infinity<T>();
      }
    }
    T highs[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      highs[h] = x[h * E / 2];
#pragma unroll
      for (int i = 1; i < E / 2; ++i) highs[h] = larger(highs[h], x[h * E / 2 + i]);
    }
    const T high = larger(highs[0], highs[1]);
    if (high > top) {
      sum *= static_cast<double>(exp_of(top - high));
      top = high;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      T part_sum = T(0);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) part_sum += exp_of(x[h * E / 2 + i] - top);
      sum += static_cast<double>(part_sum);
    }

    best = larger(best, high);
    if (chunk == begin || count_of(high > bar) >= kWorth) {
      // picks lanes hold a value of this size or more each; sign, exponent and 7 bits do.
      const Key key = best > -infinity<T>() ? key_of(best) : Key{0};
      const Key border = kth_largest<Key, sizeof(T) == 4 ? 16 : 19>(
          picks, [&](Key at) { return count_of(key >= at); });
      if (border != 0) {
        const T under = below(value_of(border));
        bar = larger(bar, under);
        if (lane == 0) {
          __hip_atomic_store(&bars[wave], under, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
    }
    // A bar that another wave has not set yet is -infinity, one that it has raised meanwhile
    // lower than it need be: no harm but more candidates.
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const T other =
          __hip_atomic_load(&bars[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      bar = shares[w] ? larger(bar, other) : bar;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!__any(highs[h] > bar)) continue;
      if (count + count_of(highs[h] > bar) * (E / 2) > kKept<T>) {
        // Tokens to come are larger than those before: an equal value does not count.
        bar = compact<T, kAll<T>>(kept, count, picks, lane);
        count = picks;
      }
#pragma unroll
      for (int i = h * E / 2; i < (h + 1) * E / 2; ++i) {
        const uint64_t mask = __ballot(x[i] > bar);
        if (mask == 0) continue;
        if (x[i] > bar) {
          const uint32_t to = count + __popcll(mask & ((uint64_t{1} << lane) - 1));
          kept.value[to] = x[i];
          kept.token[to] = chunk * kChunk<T> + (i / W * kWave + lane) * W + i % W;
        }
        count += static_cast<uint32_t>(__popcll(mask));
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = next[i];
  }
  if (count > rows.slots) {
    if (count <= kFew * kWave) {
      compact<T, kFew>(kept, count, picks, lane);
    } else if (count <= kMore * kWave) {
      compact<T, kMore>(kept, count, picks, lane);
    } else {
      compact<T, kAll<T>>(kept, count, picks, lane);
    }
    count = picks;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // The lanes' sums over the largest maximum.
  T most = top;
#pragma unroll
  for (int mask = kWave / 2; mask > 0; mask >>= 1) {
    const T other = __shfl_xor(most, mask, kWave);
    most = other > most ? other : most;
  }
  sum = wave_sum(sum * static_cast<double>(exp_of(top - most)));
  if (lane == 0) {
    rows.maxima[id] = static_cast<double>(most);
    rows.sums[id] = sum;
  }
  const uint64_t base = static_cast<uint64_t>(id) * rows.slots;
  if (static_cast<uint32_t>(lane) < rows.slots) {
    const bool held = static_cast<uint32_t>(lane) < count;
    rows.values[base + lane] = held ? kept.value[lane] : T(0);
    rows.tokens[base + lane] = held ? kept.token[lane] : kNone;
  }
}

// A candidate of a group.
struct Candidate {
  double total;
  double logit;
  uint32_t row, token;  // row of the group
};

// Whether a comes before b.
__device__ __forceinline__ bool precedes(const Candidate& a, const Candidate& b) {
  if (a.total != b.total) return a.total > b.total;
  if (a.row != b.row) return a.row < b.row;
  if (a.logit != b.logit) return a.logit > b.logit;
  return a.token < b.token;
}

constexpr int kGroupThreads = 512;
constexpr int kGroupWaves = kGroupThreads / kWave;
constexpr uint32_t kBatch = 4096;   // candidates whose totals are held
constexpr uint32_t kListed = 1024;  // candidates in LDS that may be the best
// Up to this many picks the best wave's lanes alone set the bar (32 groups of 8 picks 36 us
// for 38 with all waves' lanes); of more picks too many would pass (32: 18 us for 27).
constexpr uint32_t kFewPicks = 16;

template <typename T>
struct Picked {
  T* scores;
  int64_t* parents;
  int64_t* tokens;
  int32_t* ended;  // or nullptr
};

// A workgroup per group.  Candidates are read while the rows' sums are joined; the picks-th
// best of the lanes bounds what can be among the group's best, which few pass, and those are
// ranked by counting.  Bound by latency, one step behind the other: 7 us for 32 groups of
// 1024 candidates, 18 for one of 8192.
template <typename T>
__global__ __launch_bounds__(kGroupThreads) void group_kernel(Picked<T> picked, Rows<T> rows,
                                                              const T* scores, uint32_t beams,
                                                              int64_t end_token,
                                                              FastDiv by_row) {
  __shared__ Candidate list[kListed], best[SPAR_HIP_MAX_BEAMS];
  __shared__ double score_of[SPAR_HIP_MAX_BEAMS], log_sum[SPAR_HIP_MAX_BEAMS];
  __shared__ bool has_ended[SPAR_HIP_MAX_BEAMS];
  __shared__ uint32_t keys[kBatch], passed[kBatch];
  __shared__ uint32_t bars[kGroupWaves];
  __shared__ uint32_t listed, count;
  const uint32_t group = blockIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const uint32_t picks = rows.picks;
  const uint32_t per_row = by_row.divisor;  // parts * slots
  const uint32_t all = beams * per_row;
  const uint64_t first_row = static_cast<uint64_t>(group) * beams;

  // A thread's share of a batch of candidates, all on their way at once.
  constexpr int kShare = kBatch / kGroupThreads;
  T value[kShare];
  uint32_t token[kShare];
  const auto fetch = [&](uint32_t base) {
#pragma unroll
    for (int j = 0; j < kShare; ++j) {
      const uint32_t i = base + j * kGroupThreads + threadIdx.x;
      const uint64_t from = first_row * per_row + (i < all ? i : 0);
      value[j] = rows.values[from];
      token[j] = rows.tokens[from];
    }
  };
  fetch(0);  // they arrive while the rows' sums are joined
  for (uint32_t r = wave; r < beams; r += kGroupWaves) {
    const uint64_t row = first_row + r;
    const bool ended = rows.ended != nullptr && rows.ended[row] != 0;
    double top = -__DBL_MAX__, sum = 0.0;
    if (!ended && static_cast<uint32_t>(lane) < rows.parts) {
      top = rows.maxima[row * rows.parts + lane];
      sum = rows.sums[row * rows.parts + lane];
    }
    const T score = scores[row];
    double most = top;
#pragma unroll 1
    for (int mask = kWave / 2; mask > 0; mask >>= 1) {
      most = fmax(most, __shfl_xor(most, mask, kWave));
    }
    sum *= exp(top - most);
#pragma unroll 1
    for (int mask = kWave / 2; mask > 0; mask >>= 1) sum += __shfl_xor(sum, mask, kWave);
    if (lane == 0) {
      score_of[r] = static_cast<double>(score);
      log_sum[r] = most + log(sum);
      has_ended[r] = ended;
    }
  }
  if (threadIdx.x == 0) listed = count = 0;
  __syncthreads();

  // Candidate i, of these; its total is -infinity where there is none.
  const auto made = [&](uint32_t i, T value, uint32_t token) {
    Candidate c{-infinity<double>(), static_cast<double>(value), by_row.div(i), token};
    if (has_ended[c.row]) {
      if (i != c.row * per_row) return c;
      c.token = static_cast<uint32_t>(end_token);
      c.total = score_of[c.row];
    } else if (token != kNone) {
      c.total = score_of[c.row] + (c.logit - log_sum[c.row]);
    }
    if (c.total != c.total) c.total = -infinity<double>();
    return c;
  };
  // Totals in single precision: rounding keeps the order, so that what lies below the
  // picks-th largest of these is not among the best; of its bits the first do.
  const uint32_t nothing = key_of(-infinity<float>());
  const auto coarse = [&](uint32_t base, int j) {
    const uint32_t i = base + j * kGroupThreads + threadIdx.x;
    return i < all ? key_of(static_cast<float>(made(i, value[j], token[j]).total)) : 0;
  };

  uint32_t high = nothing;
#pragma unroll
  for (int j = 0; j < kShare; ++j) {
    if (j * kGroupThreads >= all) break;
    keys[j * kGroupThreads + threadIdx.x] = coarse(0, j);
    high = max(high, keys[j * kGroupThreads + threadIdx.x]);
  }
#pragma unroll 1
  for (uint32_t base = kBatch; base < all; base += kBatch) {
    fetch(base);
#pragma unroll
    for (int j = 0; j < kShare; ++j) high = max(high, coarse(base, j));
  }
  uint32_t bar = nothing;
  if (picks <= kFewPicks) {
    const uint32_t border =
        kth_largest<uint32_t, 20>(picks, [&](uint32_t at) { return count_of(high >= at); });
    if (lane == 0) bars[wave] = border;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) bar = max(bar, bars[w]);
  } else {  // of all waves' lanes, in every wave
    passed[threadIdx.x] = high;
    __syncthreads();
    uint32_t highs[kGroupWaves];
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) highs[w] = passed[w * kWave + lane];
    const uint32_t border = kth_largest<uint32_t, 20>(picks, [&](uint32_t at) {
      uint32_t n = 0;
#pragma unroll
      for (int w = 0; w < kGroupWaves; ++w) n += count_of(highs[w] >= at);
      return n;
    });
    bar = max(bar, border);
    __syncthreads();
  }

  // Keeps the best picks of the list; all threads.  Returns how many it keeps.
  const auto choose = [&]() {
    __syncthreads();
    const uint32_t count = listed;  // of all, the best so far among them
    constexpr uint32_t kLanes = 8;  // to rank a candidate
    const uint32_t part = threadIdx.x % kLanes;
    for (uint32_t first = 0; first < count; first += kGroupThreads / kLanes) {
      const uint32_t i = first + threadIdx.x / kLanes;
      const Candidate c = list[i < count ? i : 0];
      uint32_t before = 0;
#pragma unroll 2
      for (uint32_t j = part; j < count; j += kLanes) before += precedes(list[j], c);
      before += __shfl_xor(before, 1, kWave);
      before += __shfl_xor(before, 2, kWave);
      before += __shfl_xor(before, 4, kWave);
      if (part == 0 && i < count && before < picks) best[before] = c;
    }
    const uint32_t kept = count < picks ? count : picks;
    __syncthreads();
    if (threadIdx.x < kept) list[threadIdx.x] = best[threadIdx.x];
    if (threadIdx.x == 0) listed = kept;
    __syncthreads();
    return kept;
  };
  // A batch's candidates that may be the best, first by number and then as they are; the
  // choice waits until the list is full.
  uint32_t held = 0;  // in the list
#pragma unroll 1
  for (uint32_t base = 0; base < all; base += kBatch) {
    if (base != 0) {
      fetch(base);
#pragma unroll
      for (int j = 0; j < kShare; ++j) keys[j * kGroupThreads + threadIdx.x] = coarse(base, j);
    }
    const uint32_t end = min(kBatch, all - base);
#pragma unroll 1
    for (uint32_t first = 0; first < end; first += kGroupThreads) {
      const uint32_t i = first + threadIdx.x;
      const bool taken = i < end && keys[i] >= bar;
      const uint64_t mask = __ballot(taken);
      if (mask == 0) continue;
      uint32_t to = 0;
      if (lane == 0) to = atomicAdd(&count, static_cast<uint32_t>(__popcll(mask)));
      to = __builtin_amdgcn_readfirstlane(to) + __popcll(mask & ((uint64_t{1} << lane) - 1));
      if (taken) passed[to] = base + i;
    }
    __syncthreads();
    const uint32_t found = count;
    for (uint32_t first = 0; first < found; first += kListed - SPAR_HIP_MAX_BEAMS) {
      const uint32_t last = min(first + kListed - SPAR_HIP_MAX_BEAMS, found);
      if (held + (last - first) > kListed) choose();
      for (uint32_t at = first + threadIdx.x; at < last; at += kGroupThreads) {
        const uint32_t i = passed[at];
        const uint64_t from = first_row * per_row + i;
        const Candidate c = made(i, rows.values[from], rows.tokens[from]);
        if (c.total > -infinity<double>()) list[atomicAdd(&listed, 1U)] = c;
      }
      __syncthreads();
      held = listed;
      __syncthreads();
    }
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
  }
  const uint32_t chosen = choose();

  const auto write = [&](uint32_t i, double total, uint32_t r, uint32_t token) {
    const uint64_t at = static_cast<uint64_t>(group) * picks + i;
    picked.scores[at] = static_cast<T>(total);
    picked.parents[at] = static_cast<int64_t>(group) * beams + r;
    picked.tokens[at] = token;
    if (picked.ended != nullptr) {
      picked.ended[at] = has_ended[r] || static_cast<int64_t>(token) == end_token;
    }
  };
  if (threadIdx.x < chosen) {
    const Candidate& c = list[threadIdx.x];
    write(threadIdx.x, c.total, c.row, c.token);
  }
  // The rest: the first tokens of the first rows whose totals are -infinity, which are all
  // but those chosen.
  const uint64_t flat = threadIdx.x;
  if (chosen < picks && flat < static_cast<uint64_t>(beams) * rows.vocabulary) {
    uint32_t before = 0;
    bool among = false;
    for (uint32_t i = 0; i < chosen; ++i) {
      const uint64_t at = static_cast<uint64_t>(list[i].row) * rows.vocabulary + list[i].token;
      before += at < flat;
      among |= at == flat;
    }
    const uint32_t place = chosen + static_cast<uint32_t>(flat) - before;
    if (!among && place < picks) {
      const uint32_t r = static_cast<uint32_t>(flat) / rows.vocabulary;
      write(place, -infinity<double>(), r, static_cast<uint32_t>(flat) - r * rows.vocabulary);
    }
  }
}
static_assert(kGroupThreads >= 2 * SPAR_HIP_MAX_BEAMS);

// ------------------------------------------------------------------ reorder

constexpr uint32_t kStates = 32;  // of one launch

struct State {
  char* output;
  const char* input;
  uint64_t output_pitch, input_pitch;  // bytes between rows
  uint64_t row_bytes;
  uint32_t first_group;                // of its workgroups
  uint32_t row_groups;                 // workgroups of a row
  int unit;                            // bytes a lane moves at once: 16, 8 or 4
};

struct States {
  State state[kStates];
  uint32_t count;
};

// A workgroup moves this much of a row, four pieces of a lane on their way at once.  Bound by
// memory for large states (160 rows of 65536 floats, 42 MB written, in 10 us), by the launch
// for small ones.
constexpr uint64_t kGroupBytes = 4 * kThreads * 16;

// from: nullptr for zeros.
template <typename V>
__device__ __forceinline__ void move_row(char* to, const char* from, uint64_t begin,
                                         uint64_t end) {
  constexpr int kAtOnce = 4;
  for (uint64_t at = begin + threadIdx.x * sizeof(V); at < end;
       at += kAtOnce * kThreads * sizeof(V)) {
    V x[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint64_t place = at + i * kThreads * sizeof(V);
      x[i] = from == nullptr ? V{} : *reinterpret_cast<const V*>(from + (place < end ? place : at));
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint64_t place = at + i * kThreads * sizeof(V);
      if (place < end) *reinterpret_cast<V*>(to + place) = x[i];
    }
  }
}

__global__ __launch_bounds__(kThreads) void reorder_kernel(States states, const int64_t* parents,
                                                           uint64_t source_rows) {
  uint32_t which = 0;
  for (uint32_t i = 1; i < states.count; ++i) {
    if (blockIdx.x >= states.state[i].first_group) which = i;
  }
  const State& state = states.state[which];
  const uint32_t group = blockIdx.x - state.first_group;
  const uint32_t row = group / state.row_groups;
  const uint64_t begin = static_cast<uint64_t>(group - row * state.row_groups) * kGroupBytes;
  const int64_t parent = parents[row];
  const bool known = parent >= 0 && static_cast<uint64_t>(parent) < source_rows;
  char* to = state.output + row * state.output_pitch;
  const char* from =
      known ? state.input + static_cast<uint64_t>(parent) * state.input_pitch : nullptr;
  const uint64_t end =
      begin + kGroupBytes < state.row_bytes ? begin + kGroupBytes : state.row_bytes;
  if (state.unit == 16) {
    move_row<i32x4>(to, from, begin, end);
  } else if (state.unit == 8) {
    move_row<int64_t>(to, from, begin, end);
  } else {
    move_row<int32_t>(to, from, begin, end);
  }
}

// ---------------------------------------------------------------- launchers

// Waves that a call's rows are split up to: eight for each of the 256 CUs, which are as many
// as a CU holds.
constexpr uint64_t kFullWaves = 2048;
// Candidates of a group, which one workgroup goes through: 16 rows of 200000 with 32 picks
// take 46 us with 4096, 42 with 8192, 47 with 16384 and 183 without a bound.
constexpr uint64_t kMostCandidates = 8192;
constexpr uint64_t kMostGroups = (uint64_t{1} << 32) / kGroupThreads - 1;

struct Plan {
  uint64_t rows, parts, slots;
  uint64_t bytes;
};

Plan plan_of(const SparHipBeams& b) {
  Plan plan{};
  plan.rows = b.groups * b.beams;
  const uint64_t size = b.dtype == SPAR_HIP_FLOAT32 ? sizeof(float) : sizeof(double);
  const uint64_t chunk = b.dtype == SPAR_HIP_FLOAT32 ? kChunk<float> : kChunk<double>;
  const uint64_t chunks = (b.vocabulary + chunk - 1) / chunk;
  // Room for a few more than the picks, which a part of one chunk mostly finds: they need
  // not be told apart before the group's choice (10 picks: 27 us for 29).  Many picks are,
  // where the group's choice would take longer (32: 45 us for 46, 42 for 52).
  plan.slots = std::max<uint64_t>(b.picks, std::min<uint64_t>(2 * b.picks, 32));
  plan.parts = std::max<uint64_t>(
      1, std::min({chunks, uint64_t{kMostParts}, kFullWaves / std::max<uint64_t>(1, plan.rows),
                   kMostCandidates / (b.beams * plan.slots)}));
  const uint64_t waves = plan.rows * plan.parts;
  plan.bytes = waves * 2 * sizeof(double) + waves * plan.slots * (size + sizeof(uint32_t));
  return plan;
}

bool valid(const SparHipBeams* b) {
  return b != nullptr && valid_float_dtype(b->dtype) && b->beams >= 1 &&
         b->beams <= SPAR_HIP_MAX_BEAMS && b->picks >= 1 && b->picks <= SPAR_HIP_MAX_BEAMS &&
         b->vocabulary >= 1 && b->vocabulary <= kIndex32Limit &&
         b->picks <= b->beams * b->vocabulary && b->row_stride >= b->vocabulary &&
         b->groups * b->beams <= kMostGroups && b->groups <= kMostGroups &&
         b->end_token < static_cast<int64_t>(b->vocabulary) &&
         (b->ended == nullptr || b->end_token >= 0);
}

template <typename T>
void start(const SparHipBeams& b, const Plan& plan, void* picked_scores, int64_t* parents,
           int64_t* tokens, int32_t* picked_ended, const void* logits, const void* scores,
           void* workspace, hipStream_t stream) {
  const uint64_t waves = plan.rows * plan.parts;
  Rows<T> rows{};
  rows.logits = static_cast<const T*>(logits);
  rows.stride = b.row_stride;
  rows.ended = b.ended;
  rows.vocabulary = static_cast<uint32_t>(b.vocabulary);
  rows.parts = static_cast<uint32_t>(plan.parts);
  rows.picks = static_cast<uint32_t>(b.picks);
  rows.slots = static_cast<uint32_t>(plan.slots);
  rows.maxima = static_cast<double*>(workspace);
  rows.sums = rows.maxima + waves;
  rows.values = reinterpret_cast<T*>(rows.sums + waves);
  rows.tokens = reinterpret_cast<uint32_t*>(rows.values + waves * plan.slots);
  FastDiv by_parts, by_row;
  by_parts.init(rows.parts);
  by_row.init(rows.parts * rows.slots);
  row_kernel<T><<<ceil_div_u32(waves, kWaves), kThreads, 0, stream>>>(
      rows, static_cast<uint32_t>(waves), by_parts);
  const Picked<T> picked{static_cast<T*>(picked_scores), parents, tokens, picked_ended};
  group_kernel<T><<<static_cast<uint32_t>(b.groups), kGroupThreads, 0, stream>>>(
      picked, rows, static_cast<const T*>(scores), static_cast<uint32_t>(b.beams), b.end_token,
      by_row);
}

}  // namespace
}  // namespace beams
}  // namespace spar_hip

using namespace spar_hip;

extern "C" SparHipStatus spar_hip_beam_select_workspace(uint64_t* bytes,
                                                        const SparHipBeams* shape) {
  if (bytes == nullptr || !beams::valid(shape)) return invalid();
  *bytes = beams::plan_of(*shape).bytes;
  return ok();
}

extern "C" SparHipStatus spar_hip_launch_beam_select(void* picked_scores, int64_t* parents,
                                                     int64_t* tokens, int32_t* picked_ended,
                                                     const void* logits, const void* scores,
                                                     const SparHipBeams* shape, void* workspace,
                                                     uint64_t workspace_bytes, int device) {
  if (!beams::valid(shape)) return invalid();
  if (shape->groups == 0) return ok();
  const beams::Plan plan = beams::plan_of(*shape);
  if (picked_scores == nullptr || parents == nullptr || tokens == nullptr || logits == nullptr ||
      scores == nullptr || workspace == nullptr || workspace_bytes < plan.bytes ||
      !aligned16(workspace)) {
    return invalid();
  }
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  if (shape->dtype == SPAR_HIP_FLOAT32) {
    beams::start<float>(*shape, plan, picked_scores, parents, tokens, picked_ended, logits, scores,
                        workspace, guard.stream);
  } else {
    beams::start<double>(*shape, plan, picked_scores, parents, tokens, picked_ended, logits,
                         scores, workspace, guard.stream);
  }
  return finish(guard);
}

extern "C" SparHipStatus spar_hip_launch_reorder(const SparHipReorder* states,
                                                 uint64_t state_count, const int64_t* parents,
                                                 uint64_t rows, uint64_t source_rows, int device) {
  if (state_count > (uint64_t{1} << 16) || rows > kIndex32Limit ||
      (state_count != 0 && states == nullptr)) {
    return invalid();
  }
  if (state_count == 0 || rows == 0) return ok();
  if (parents == nullptr) return invalid();
  constexpr uint64_t kMost = uint64_t{1} << 40;  // elements: beyond memory, and no product wraps
  for (uint64_t i = 0; i < state_count; ++i) {
    const SparHipReorder& s = states[i];
    if ((s.element_size != 4 && s.element_size != 8) || s.output_stride < s.row_elements ||
        s.row_elements > kMost || s.output_stride > kMost || s.input_stride > kMost) {
      return invalid();
    }
    if (s.row_elements == 0) continue;
    if (s.output == nullptr || (s.input == nullptr && source_rows != 0) ||
        (s.row_elements * s.element_size + beams::kGroupBytes - 1) / beams::kGroupBytes * rows >
            beams::kMostGroups) {
      return invalid();
    }
  }
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  beams::States batch{};
  uint64_t groups = 0;
  const auto launch = [&]() {
    if (batch.count == 0) return;
    beams::reorder_kernel<<<static_cast<uint32_t>(groups), beams::kThreads, 0, guard.stream>>>(
        batch, parents, source_rows);
    batch.count = 0;
    groups = 0;
  };
  for (uint64_t i = 0; i < state_count; ++i) {
    const SparHipReorder& s = states[i];
    if (s.row_elements == 0) continue;
    const uint64_t size = s.element_size;
    beams::State state{};
    state.output = static_cast<char*>(s.output);
    state.input = static_cast<const char*>(s.input);
    state.output_pitch = s.output_stride * size;
    state.input_pitch = s.input_stride * size;
    state.row_bytes = s.row_elements * size;
    state.row_groups = ceil_div_u32(state.row_bytes, beams::kGroupBytes);
    const uint64_t mixed = reinterpret_cast<uintptr_t>(s.output) |
                           reinterpret_cast<uintptr_t>(s.input) | state.output_pitch |
                           state.input_pitch | state.row_bytes;
    state.unit = mixed % 16 == 0 ? 16 : mixed % 8 == 0 ? 8 : 4;
    const uint64_t own = state.row_groups * rows;
    if (batch.count == beams::kStates || groups + own > beams::kMostGroups) launch();
    state.first_group = static_cast<uint32_t>(groups);
    batch.state[batch.count++] = state;
    groups += own;
  }
  launch();
  return finish(guard);
}

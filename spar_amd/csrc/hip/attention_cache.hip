// Attention of new tokens over a cache in pages, behind a prefix that several sequences
// share: o = softmax(scale q [K_prefix; K_own]^T) [V_prefix; V_own].
//
// The softmax's sums are joined by base and total (attention_join.hpp), so that the keys
// fall into two sides that are computed apart: the prefix, whose rows are the queries of
// all sequences that share it -- one read of its keys and values serves them all, and
// their products fill the matrix units -- and each sequence's own tokens.  On either side
// the kernels are those of attention_forward.hip with keys found through a table of pages:
// tiles in LDS shared by 64 rows (bound by the matrix units), or 16 rows whose four waves
// take different keys straight from memory (bound by reading the cache).
//
// Pages.  Where a page holds whole blocks of keys, a block is found with one look into the
// table; otherwise every lane looks for the key that it loads, a block ahead of its use.
// A key of a page that holds nothing is read from zeros and masked.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attention_join.hpp"
#include "pages.hpp"

namespace spar_hip {
namespace attention {
namespace {

// What stands in the place of a key that is not there.
alignas(16) __device__ const double kNothing[SPAR_HIP_ATTENTION_MAX_EXTENT] = {};

// One side of the keys: row u of its cache is read by `sharers` sequences from u *
// sharers on, whose queries are the rows of its products: row r = (s * queries + t) *
// group + g.
template <typename T>
struct Side {
  Pages<const T> cache;
  const void* lengths;
  bool wide_lengths;
  bool own;              // causal: a sequence's own tokens
  uint32_t units;        // rows of the cache times key heads
  uint32_t sharers;
  FastDiv per_sequence;  // rows of a sequence
  uint32_t rows;         // of a unit
  uint32_t row_tiles;
  uint32_t splits;
  uint32_t first_part;

  __device__ __forceinline__ int32_t length(uint32_t u) const {
    if (lengths == nullptr) return static_cast<int32_t>(cache.room);
    const int64_t n = wide_lengths ? static_cast<const int64_t*>(lengths)[u]
                                   : static_cast<const int32_t*>(lengths)[u];
    return static_cast<int32_t>(n < 0 ? 0 : n > cache.room ? cache.room : n);
  }
};

// A row of a side: its sequence, query and head, and the last key it sees.
struct RowAt {
  uint32_t b, t, head;
  int32_t limit;  // -1 where it sees nothing
};

template <typename T>
__device__ __forceinline__ RowAt row_at(const Call& call, const Side<T>& side, uint32_t u,
                                        uint32_t key_head, uint32_t r, int32_t side_length) {
  RowAt row;
  const uint32_t s = side.per_sequence.div(r);
  const uint32_t rest = r - s * side.per_sequence.divisor;
  row.t = call.group.div(rest);
  row.head = key_head * call.group.divisor + (rest - row.t * call.group.divisor);
  row.b = u * side.sharers + s;
  const int32_t p = call.length(row.b) - static_cast<int32_t>(call.queries) +
                    static_cast<int32_t>(row.t);
  row.limit = p < 0 ? -1 : side.own ? p : side_length - 1;
  return row;
}

// Writes a row's part, or the row itself where it is the only one.
template <typename T>
__device__ __forceinline__ T* part_row(const Call& call, const Results<T>& results,
                                       const RowAt& row, uint32_t part, T top, T sum, bool first) {
  const uint64_t place =
      (static_cast<uint64_t>(row.b) * call.key_heads * call.group.divisor + row.head) *
          call.queries + row.t;
  if (results.splits == 1) {
    return results.output.data + row.b * results.output.batch + row.head * results.output.head +
           row.t * results.output.token;
  }
  const uint64_t at = part * results.all_rows + place;
  if (first) {
    results.part_top[at] = top;
    results.part_total[at] = sum;
  }
  return results.part_output + at * results.pitch;
}

// The keys of a block of SIZE from `begin` on, found through the table.  `page` is what the
// lane found for key begin + lane (WHOLE: the block's only page).
template <typename T, int SIZE, bool WHOLE>
struct Finder {
  const Pages<const T>& cache;
  uint32_t u;

  __device__ __forceinline__ int32_t look(int32_t begin, int32_t end, int lane) const {
    const int32_t key = WHOLE ? begin : begin + lane;
    if (key >= end || (!WHOLE && lane >= SIZE)) return -1;
    return cache.page_at(u, cache.page_tokens.div(static_cast<uint32_t>(key)));
  }
  // Which of the block's keys are there, a bit each.
  __device__ __forceinline__ uint64_t present(int32_t page, int32_t begin, int32_t end) const {
    constexpr uint64_t kAll = (uint64_t{1} << SIZE) - 1;
    if constexpr (WHOLE) {
      const int32_t count = end - begin;
      const uint64_t inside = count >= SIZE ? kAll : (uint64_t{1} << count) - 1;
      return page < 0 ? 0 : inside;
    }
    return __ballot(page >= 0) & kAll;
  }
  __device__ __forceinline__ uint32_t slot(int32_t key) const {
    const uint32_t k = static_cast<uint32_t>(key);
    return k - cache.page_tokens.div(k) * cache.page_tokens.divisor;
  }
  __device__ __forceinline__ const T* head(const PageHeads<const T>& heads, uint32_t key_head,
                                           int32_t page, uint32_t slot) const {
    return heads.data + static_cast<uint64_t>(page) * heads.page + key_head * heads.head +
           slot * heads.token;
  }
};

template <typename T, int DP, int KB, Reads READS, bool WHOLE>
__global__ __launch_bounds__(kThreads, (tile_waves<T, DP>())) void cache_tile_kernel(
    Call call, Results<T> results, Heads<const T> query, Side<T> side) {
  constexpr int KT = KB * kBlock;
  constexpr int W = Vec16<T>::width;
  constexpr uint32_t kRows = kWaves * kBlock;
  __shared__ Tile<T, KT, DP, READS> keys, values;
  const uint32_t unit = blockIdx.x % side.units;
  const uint32_t rest = blockIdx.x / side.units;
  // Row tiles side by side: they read the same keys.
  const uint32_t split = rest / side.row_tiles;
  const uint32_t row_tile = side.row_tiles - 1 - (rest - split * side.row_tiles);
  const uint32_t u = unit / call.key_heads, key_head = unit % call.key_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wave_lane = threadIdx.x % kWave;
  const Lane<T, DP> lane(wave_lane);

  const int32_t side_length = side.length(u);
  const uint32_t begin_row = row_tile * kRows;
  const uint32_t end_row = begin_row + kRows < side.rows ? begin_row + kRows : side.rows;
  // A sequence's later queries see more.
  const int32_t high =
      side.own ? row_at(call, side, u, key_head, end_row - 1, side_length).limit + 1
               : side_length;
  const uint32_t tiles = static_cast<uint32_t>(high + KT - 1) / KT;
  const uint32_t begin_tile =
      static_cast<uint32_t>(static_cast<uint64_t>(tiles) * split / side.splits);
  const uint32_t end_tile =
      static_cast<uint32_t>(static_cast<uint64_t>(tiles) * (split + 1) / side.splits);

  const Finder<T, KT, WHOLE> finder{side.cache, u};
  typename Tile<T, KT, DP, READS>::Stage next_keys, next_values;
  if constexpr (WHOLE) {
    keys.prepare(next_keys, call.extent, [&](uint32_t j) { return j * side.cache.key.token; });
    values.prepare(next_values, call.extent,
                   [&](uint32_t j) { return j * side.cache.value.token; });
  }
  int32_t page = -1;          // found for the next tile to start
  uint64_t present = 0, next_present = 0;
  const auto look = [&](uint32_t i) {
    page = i < end_tile ? finder.look(static_cast<int32_t>(i) * KT, high, wave_lane) : -1;
  };
  // Starts tile i, whose pages have been looked up, and looks for those of the next.
  const auto start = [&](uint32_t i) {
    const int32_t begin = static_cast<int32_t>(i) * KT;
    next_present = finder.present(page, begin, high);
    if constexpr (WHOLE) {
      const int32_t at = __builtin_amdgcn_readfirstlane(page);
      if (at >= 0) {
        const uint32_t slot = finder.slot(begin);
        const uint32_t count = static_cast<uint32_t>(high - begin);
        // Rows behind the last key repeat the tile's first, and no row sees them.
        const auto in = [&](uint32_t j) { return static_cast<uint64_t>(j < count ? j : 0); };
        keys.start(next_keys, i % 2, finder.head(side.cache.key, key_head, at, slot),
                   count >= KT, call.extent,
                   [&](uint32_t j) { return in(j) * side.cache.key.token; });
        values.start(next_values, i % 2, finder.head(side.cache.value, key_head, at, slot),
                     count >= KT, call.extent,
                     [&](uint32_t j) { return in(j) * side.cache.value.token; });
      }
    } else {
      const uint32_t slot = finder.slot(begin + wave_lane % KT);
      const auto row = [&](const PageHeads<const T>& heads) {
        return [&](int, uint32_t j) {
          const int32_t at = __shfl(page, j, kWave);
          const uint32_t in = __shfl(slot, j, kWave);
          return at < 0 ? reinterpret_cast<const T*>(kNothing)
                        : finder.head(heads, key_head, at, in);
        };
      };
      keys.start_rows(next_keys, i % 2, call.extent, row(side.cache.key));
      values.start_rows(next_values, i % 2, call.extent, row(side.cache.value));
    }
    look(i + 1);
  };
  const auto finish = [&](uint32_t i) {
    keys.finish(next_keys, i % 2);
    values.finish(next_values, i % 2);
    present = next_present;
  };
  look(begin_tile);
  if (begin_tile < end_tile) start(begin_tile);

  const uint32_t wave_row = begin_row + wave * kBlock;
  const uint32_t r = wave_row + lane.column;
  const bool held = r < side.rows;
  const RowAt row_place = row_at(call, side, u, key_head, held ? r : side.rows - 1, side_length);
  const int32_t limit = held ? row_place.limit : -1;
  // The wave's rows see all keys up to `oldest`, none behind `newest`.
  int32_t newest = limit, oldest = held ? limit : INT32_MAX;
#pragma unroll
  for (int mask = kBlock / 2; mask > 0; mask >>= 1) {
    newest = max(newest, __shfl_xor(newest, mask, kWave));
    oldest = min(oldest, __shfl_xor(oldest, mask, kWave));
  }
  newest = __builtin_amdgcn_readfirstlane(newest);
  oldest = __builtin_amdgcn_readfirstlane(oldest);
  Operand<T, DP> q;
  q.template load<READS == Reads::Single ? Reads::Single : Reads::Pieces>(
      query.data + row_place.b * query.batch + row_place.head * query.head +
          row_place.t * query.token,
      call.extent, lane.quarter);
  q.finish(limit >= 0, call.extent, lane.quarter, static_cast<T>(call.scale * kLog2E));
  Row<T, DP> row;
  row.out.clear();
  if (begin_tile < end_tile) finish(begin_tile);

  for (uint32_t i = begin_tile; i < end_tile; ++i) {
    const int32_t begin = static_cast<int32_t>(i) * KT;
    __syncthreads();
    if (i + 1 < end_tile) start(i + 1);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int32_t k0 = begin + kb * kBlock, k1 = k0 + kBlock - 1;
      const uint32_t there = static_cast<uint32_t>(present >> (kb * kBlock)) & 0xffffU;
      if (there == 0 || k0 > newest) continue;
      const T* key_rows = keys.value[i % 2] + kb * kBlock * DP;
      const T* value_rows = values.value[i % 2] + kb * kBlock * DP;
      typename Mma<T>::Acc s{0, 0, 0, 0};
      const auto read = [&](int p) { return lane.along(key_rows, p); };
      Queue<2, typename Vec16<T>::type> queue;
      fill_queue(queue, read);
      run_queue<DP / (4 * W)>(queue, read, [&](int p, const typename Vec16<T>::type& piece) {
#pragma unroll
        for (int x = 0; x < W; ++x) s = Mma<T>::step(piece[x], q.value[p * W + x], s);
      });
      Across<T, DP> across(lane, value_rows);
      const bool whole = (k1 <= oldest) & (there == 0xffffU);
      T score[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) score[v] = s[v];
      if (!whole) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int n = Mma<T>::row_of(v, lane.quarter);
          const bool visible = (k0 + n <= limit) & ((there >> n & 1U) != 0);
          score[v] = visible ? score[v] : lowest<T>();
        }
      }
      row.take(score);
      across.run(row.out, score);
    }
    if (i + 1 < end_tile) finish(i + 1);
  }
  const T total = quarter_sum(row.total);
  if (!held) return;
  T* target = part_row(call, results, row_place, side.first_part + split, row.base, total,
                       lane.quarter == 0);
  const T over = total == T(0) ? T(0) : T(1) / total;
  row.out.visit(lane.quarter, [&](uint32_t d, auto& run) {
    // No weights: nothing, also where what they would have met is not finite.
    for (auto& x : run) x = total == T(0) ? T(0) : x * over;
    store_piece(target, d, call.extent, run);
  });
}

template <typename T, int DP, Reads READS, bool WHOLE>
__global__ __launch_bounds__(kThreads) void cache_token_kernel(Call call, Results<T> results,
                                                               Heads<const T> query,
                                                               Side<T> side) {
  constexpr int W = Vec16<T>::width;
  constexpr int kPitch = DP + W;
  __shared__ T outs[kWaves][kBlock][kPitch];
  __shared__ T tops[kWaves][kBlock], totals[kWaves][kBlock];
  const uint32_t unit = blockIdx.x % side.units;
  const uint32_t rest = blockIdx.x / side.units;
  const uint32_t split = rest / side.row_tiles;
  const uint32_t row_tile = side.row_tiles - 1 - (rest - split * side.row_tiles);
  const uint32_t u = unit / call.key_heads, key_head = unit % call.key_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int quarter = lane / kBlock, column = lane % kBlock;

  const int32_t side_length = side.length(u);
  const uint32_t begin_row = row_tile * kBlock;
  const uint32_t end_row = begin_row + kBlock < side.rows ? begin_row + kBlock : side.rows;
  const int32_t high =
      side.own ? row_at(call, side, u, key_head, end_row - 1, side_length).limit + 1
               : side_length;
  const uint32_t blocks = static_cast<uint32_t>(high + kBlock - 1) / kBlock;
  const uint32_t begin_block =
      static_cast<uint32_t>(static_cast<uint64_t>(blocks) * split / side.splits);
  const uint32_t end_block =
      static_cast<uint32_t>(static_cast<uint64_t>(blocks) * (split + 1) / side.splits);

  const Finder<T, kBlock, WHOLE> finder{side.cache, u};
  const auto look = [&](uint32_t i) {
    return i < end_block ? finder.look(static_cast<int32_t>(i) * kBlock, high, lane % kBlock)
                         : -1;
  };
  int32_t page = look(begin_block + wave);

  const uint32_t r = begin_row + column;
  const bool held = r < side.rows;
  const RowAt row_place = row_at(call, side, u, key_head, held ? r : side.rows - 1, side_length);
  const int32_t limit = held ? row_place.limit : -1;
  int32_t oldest = held ? limit : INT32_MAX;
#pragma unroll
  for (int mask = kBlock / 2; mask > 0; mask >>= 1) {
    oldest = min(oldest, __shfl_xor(oldest, mask, kWave));
  }
  oldest = __builtin_amdgcn_readfirstlane(oldest);
  Operand<T, DP> q;
  q.template load<READS>(query.data + row_place.b * query.batch + row_place.head * query.head +
                             row_place.t * query.token,
                         call.extent, quarter);
  q.finish(limit >= 0, call.extent, quarter, static_cast<T>(call.scale * kLog2E));
  Row<T, DP> row;
  row.out.clear();

  for (uint32_t i = begin_block + wave; i < end_block; i += kWaves) {
    const int32_t begin = static_cast<int32_t>(i) * kBlock;
    const uint32_t there =
        static_cast<uint32_t>(finder.present(page, begin, high)) & 0xffffU;
    const int32_t found = page;
    page = look(i + kWaves);
    if (there == 0) continue;
    Operand<T, DP> k;
    AcrossOperand<T, DP> v;
    if constexpr (WHOLE) {
      const int32_t at = __builtin_amdgcn_readfirstlane(found);
      const uint32_t slot = finder.slot(begin);
      const uint32_t count = static_cast<uint32_t>(high - begin);
      const auto in = [&](uint32_t n) { return static_cast<uint64_t>(n < count ? n : 0); };
      const T* key_base = finder.head(side.cache.key, key_head, at, slot);
      const T* value_base = finder.head(side.cache.value, key_head, at, slot);
      k.template load<READS>(key_base + in(column) * side.cache.key.token, call.extent, quarter);
      v.template load<READS>(call.extent, quarter, column, [&](int n) {
        return value_base + in(n) * side.cache.value.token;
      });
    } else {
      const uint32_t slot = finder.slot(begin + column);
      const T* nothing = reinterpret_cast<const T*>(kNothing);
      k.template load<READS>(
          found < 0 ? nothing : finder.head(side.cache.key, key_head, found, slot), call.extent,
          quarter);
      v.template load<READS>(call.extent, quarter, column, [&](int n) {
        const int32_t at = __shfl(found, n, kWave);
        const uint32_t in = __shfl(slot, n, kWave);
        return at < 0 ? nothing : finder.head(side.cache.value, key_head, at, in);
      });
    }
    typename Mma<T>::Acc s{0, 0, 0, 0};
#pragma unroll
    for (int step = 0; step < DP / 4; ++step) {
      s = Mma<T>::step(k.value[step], q.value[step], s);
    }
    const bool whole = (begin + kBlock - 1 <= oldest) & (there == 0xffffU);
    T score[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int at = Mma<T>::row_of(n, quarter);
      const bool visible = whole | ((begin + at <= limit) & ((there >> at & 1U) != 0));
      score[n] = visible ? s[n] : lowest<T>();
    }
    row.take(score);
    v.add_to(row.out, score);
  }
  const T total = quarter_sum(row.total);
  if (quarter == 0) {
    tops[wave][column] = row.base;
    totals[wave][column] = total;
  }
  row.out.visit(quarter, [&](uint32_t d, auto& run) {
    for (auto& x : run) {
      outs[wave][column][d] = x;
      ++d;
    }
  });
  __syncthreads();
  // Lane by lane over the rows' pieces: the waves in order.
  constexpr int kPieces = DP / W;
  for (int at = threadIdx.x; at < kBlock * kPieces; at += kThreads) {
    const int c = at / kPieces, d = at % kPieces * W;
    const uint32_t out_row = begin_row + c;
    if (out_row >= side.rows) continue;
    T top = tops[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = larger(tops[w][c], top);
    T sum = T(0);
    T run[W] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const T shrink = exp2_of(tops[w][c] - top);
      const T part = totals[w][c];
      sum += part * shrink;
#pragma unroll
      for (int j = 0; j < W; ++j) run[j] += part == T(0) ? T(0) : outs[w][c][d + j] * shrink;
    }
    const T over = sum == T(0) ? T(0) : T(1) / sum;
#pragma unroll
    for (int j = 0; j < W; ++j) run[j] *= over;
    const RowAt place = row_at(call, side, u, key_head, out_row, side_length);
    T* target = part_row(call, results, place, side.first_part + split, top, sum, d == 0);
    store_piece(target, d, call.extent, run);
  }
}

// ---------------------------------------------------------------- launchers

// As in the forward over a contiguous cache: up to this many rows of a unit the waves share
// rows and split keys; workgroups that row tiles are split up to, and the fewest keys that
// repay a part.
constexpr uint64_t kTokenRows = 32;
constexpr uint64_t kFullGrid = 768;
constexpr uint64_t kTokenGrid = 1024;
constexpr uint64_t kFewestKeys = 256;
constexpr uint64_t kFewestTokenKeys = 128;

struct SidePlan {
  bool token;
  uint64_t units, rows, row_tiles, splits;
  uint64_t groups() const { return units * row_tiles * splits; }
};

struct Plan {
  SidePlan own, prefix;
  uint32_t parts;
  uint32_t pitch;
  uint64_t rows;  // batch * query heads * queries
  uint64_t bytes;
};

uint64_t room_of(const SparHipPages* cache) {
  return cache == nullptr || cache->pages == 0 ? 0 : cache->table_pages * cache->page_tokens;
}

SidePlan side_plan(const SparHipCacheAttention& a, uint64_t rows_of_cache, uint64_t sharers,
                   uint64_t room) {
  SidePlan plan{};
  plan.units = rows_of_cache * a.key_heads;
  plan.rows = sharers * a.queries * (a.query_heads / a.key_heads);
  constexpr uint64_t kRows = kWaves * kBlock;
  plan.token = plan.rows <= kTokenRows ||
               spreads((plan.rows + kRows - 1) / kRows * plan.units *
                       std::max<uint64_t>(1, room / kFewestKeys));
  const uint64_t tile_rows = plan.token ? kBlock : kRows;
  plan.row_tiles = (plan.rows + tile_rows - 1) / tile_rows;
  const uint64_t wanted = (plan.token ? kTokenGrid : kFullGrid) /
                          std::max<uint64_t>(1, plan.row_tiles * plan.units);
  plan.splits = std::max<uint64_t>(
      1, std::min({wanted, room / (plan.token ? kFewestTokenKeys : kFewestKeys),
                   uint64_t{kMostParts / 2}}));
  return plan;
}

Plan plan_of(const SparHipCacheAttention& a, const SparHipPages& cache,
             const SparHipPages* prefix) {
  Plan plan{};
  plan.rows = a.batch * a.query_heads * a.queries;
  plan.own = side_plan(a, a.batch, 1, room_of(&cache));
  if (room_of(prefix) != 0) {
    plan.prefix = side_plan(a, a.prefixes, a.batch / a.prefixes, room_of(prefix));
  }
  plan.parts = static_cast<uint32_t>(plan.own.splits + plan.prefix.splits);
  const uint64_t size = a.dtype == SPAR_HIP_FLOAT32 ? sizeof(float) : sizeof(double);
  const uint64_t piece = 16 / size;
  plan.pitch = static_cast<uint32_t>((a.extent + piece - 1) / piece * piece);
  if (plan.parts > 1) plan.bytes = plan.parts * plan.rows * (plan.pitch + 2) * size;
  return plan;
}

// A launch counts its workgroups in 32 bits of work-items.
bool fits(const Plan& plan) {
  return plan.own.groups() <= kMostGroups && plan.prefix.groups() <= kMostGroups &&
         plan.rows <= kMostGroups;
}

// Whether a cache's keys and values go to LDS directly.
template <typename T>
bool pages_aligned(const SparHipPages& cache) {
  return reads_aligned<T>(cache.key, 1) && reads_aligned<T>(cache.value, 1);
}

template <typename T>
void start_side(const SparHipCacheAttention& a, const SparHipPages& cache, const SidePlan& plan,
                const Call& call, const Results<T>& results, const Heads<const T>& query,
                bool own, uint32_t first_part, hipStream_t stream) {
  Side<T> side{};
  side.cache = pages_of<const T>(cache);
  side.lengths = own ? a.lengths : a.prefix_lengths;
  side.wide_lengths = a.length_dtype == SPAR_HIP_INT64;
  side.own = own;
  side.units = static_cast<uint32_t>(plan.units);
  side.sharers = static_cast<uint32_t>(own ? 1 : a.batch / a.prefixes);
  side.per_sequence.init(static_cast<uint32_t>(a.queries * (a.query_heads / a.key_heads)));
  side.rows = static_cast<uint32_t>(plan.rows);
  side.row_tiles = static_cast<uint32_t>(plan.row_tiles);
  side.splits = static_cast<uint32_t>(plan.splits);
  side.first_part = first_part;
  const uint32_t grid = static_cast<uint32_t>(plan.groups());
  const bool pieces = a.extent % Vec16<T>::width == 0;
  with_padded_width(a.extent, [&](auto width) {
    constexpr int DP = decltype(width)::value;
    if (plan.token) {
      const bool whole = cache.table == nullptr || cache.page_tokens % kBlock == 0;
      if (pieces && whole) {
        cache_token_kernel<T, DP, Reads::Pieces, true>
            <<<grid, kThreads, 0, stream>>>(call, results, query, side);
      } else if (pieces) {
        cache_token_kernel<T, DP, Reads::Pieces, false>
            <<<grid, kThreads, 0, stream>>>(call, results, query, side);
      } else {
        cache_token_kernel<T, DP, Reads::Single, false>
            <<<grid, kThreads, 0, stream>>>(call, results, query, side);
      }
      return;
    }
    constexpr int KB = tile_blocks<T, DP>();
    const bool whole = cache.table == nullptr || cache.page_tokens % (KB * kBlock) == 0;
    if (pieces && pages_aligned<T>(cache) && whole) {
      cache_tile_kernel<T, DP, KB, Reads::Aligned, true>
          <<<grid, kThreads, 0, stream>>>(call, results, query, side);
    } else if (pieces && pages_aligned<T>(cache)) {
      cache_tile_kernel<T, DP, KB, Reads::Aligned, false>
          <<<grid, kThreads, 0, stream>>>(call, results, query, side);
    } else {
      cache_tile_kernel<T, DP, KB, Reads::Single, false>
          <<<grid, kThreads, 0, stream>>>(call, results, query, side);
    }
  });
}

template <typename T>
void start(const SparHipCacheAttention& a, const Plan& plan, const SparHipHeads& output,
           const SparHipHeads& query, const SparHipPages& cache, const SparHipPages* prefix,
           void* workspace, hipStream_t stream) {
  Call call{};
  const uint64_t group = a.query_heads / a.key_heads;
  call.lengths = a.lengths;
  call.wide_lengths = a.length_dtype == SPAR_HIP_INT64;
  call.group.init(static_cast<uint32_t>(group));
  call.key_heads = static_cast<uint32_t>(a.key_heads);
  call.batch_heads = static_cast<uint32_t>(a.batch * a.key_heads);
  call.queries = static_cast<uint32_t>(a.queries);
  call.rows = static_cast<uint32_t>(a.queries * group);
  call.keys = static_cast<uint32_t>(cache.table_pages * cache.page_tokens);
  call.extent = static_cast<uint32_t>(a.extent);
  call.window = kNoWindow;
  call.scale = a.scale;
  Results<T> results{heads_of<T>(output), nullptr, nullptr, nullptr, nullptr, plan.parts,
                     plan.pitch, plan.rows};
  if (plan.parts > 1) {
    results.part_output = static_cast<T*>(workspace);
    results.part_top = results.part_output + plan.parts * plan.rows * plan.pitch;
    results.part_total = results.part_top + plan.parts * plan.rows;
  }
  const auto q = heads_of<const T>(query);
  if (plan.prefix.splits != 0) {
    start_side<T>(a, *prefix, plan.prefix, call, results, q, false, 0, stream);
  }
  start_side<T>(a, cache, plan.own, call, results, q, true,
                static_cast<uint32_t>(plan.prefix.splits), stream);
  if (plan.parts > 1) join_parts(call, results, stream);
}

bool valid_call(const SparHipCacheAttention* a, const SparHipPages* cache,
                const SparHipPages* prefix) {
  constexpr uint64_t kMost = kIndex32Limit;
  if (a == nullptr || !valid_pages(cache) || (prefix != nullptr && !valid_pages(prefix)) ||
      !valid_float_dtype(a->dtype) || a->key_heads == 0 || a->query_heads == 0 ||
      a->extent == 0 || a->extent > SPAR_HIP_ATTENTION_MAX_EXTENT ||
      a->query_heads % a->key_heads != 0 || !__builtin_isfinite(a->scale) || a->batch > kMost ||
      a->query_heads > kMost || a->queries > kMost || a->batch * a->key_heads > kMost ||
      a->queries * a->query_heads >= kMostKeys) {
    return false;
  }
  if (prefix != nullptr &&
      (a->prefixes == 0 || a->batch % a->prefixes != 0 ||
       a->batch / a->prefixes > kMostKeys / std::max<uint64_t>(1, a->queries * a->query_heads))) {
    return false;
  }
  return (a->lengths == nullptr && a->prefix_lengths == nullptr) ||
         a->length_dtype == SPAR_HIP_INT32 || a->length_dtype == SPAR_HIP_INT64;
}

bool complete(const SparHipPages* cache) {
  return room_of(cache) == 0 || (cache->key.data != nullptr && cache->value.data != nullptr);
}

}  // namespace
}  // namespace attention
}  // namespace spar_hip

using namespace spar_hip;

extern "C" SparHipStatus spar_hip_cache_attention_workspace(
    uint64_t* bytes, const SparHipPages* cache, const SparHipPages* prefix,
    const SparHipCacheAttention* attention) {
  if (bytes == nullptr || !attention::valid_call(attention, cache, prefix)) return invalid();
  *bytes = 0;
  if (attention->batch == 0 || attention->queries == 0) return ok();
  const attention::Plan plan = attention::plan_of(*attention, *cache, prefix);
  if (!attention::fits(plan)) return invalid();
  *bytes = plan.bytes;
  return ok();
}

extern "C" SparHipStatus spar_hip_launch_cache_attention(
    const SparHipHeads* output, const SparHipHeads* query, const SparHipPages* cache,
    const SparHipPages* prefix, const SparHipCacheAttention* attention, void* workspace,
    uint64_t workspace_bytes, int device) {
  if (!attention::valid_call(attention, cache, prefix)) return invalid();
  const SparHipCacheAttention& a = *attention;
  if (a.batch == 0 || a.queries == 0) return ok();
  if (output == nullptr || query == nullptr || output->data == nullptr ||
      query->data == nullptr || !attention::complete(cache) || !attention::complete(prefix)) {
    return invalid();
  }
  const attention::Plan plan = attention::plan_of(a, *cache, prefix);
  if (!attention::fits(plan) ||
      (plan.bytes != 0 &&
       (workspace == nullptr || workspace_bytes < plan.bytes || !aligned16(workspace)))) {
    return invalid();
  }
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  if (a.dtype == SPAR_HIP_FLOAT32) {
    attention::start<float>(a, plan, *output, *query, *cache, prefix, workspace, guard.stream);
  } else {
    attention::start<double>(a, plan, *output, *query, *cache, prefix, workspace, guard.stream);
  }
  return finish(guard);
}

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

// What stands in the place of a key that is not there: zeros.  Not const, for which it would
// lie in another address space than the caches, and pointers to either could be followed by
// flat loads alone.
alignas(16) __device__ double kNothing[SPAR_HIP_ATTENTION_MAX_EXTENT] = {};

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
  uint32_t least;        // blocks of 16 keys that are worth a part
  uint32_t first_part;
  bool whole;            // a page holds whole blocks of keys

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

// The run of blocks of SIZE keys that part `split` of a side takes of the first `high`:
// equal shares, of fewer parts where those would be small.
template <int SIZE, typename T>
__device__ __forceinline__ void share_of(const Side<T>& side, int32_t high, uint32_t split,
                                         uint32_t& begin, uint32_t& end) {
  const uint32_t blocks = static_cast<uint32_t>(high + SIZE - 1) / SIZE;
  const uint32_t share = max((blocks + side.splits - 1) / side.splits,
                             (side.least * kBlock + SIZE - 1) / SIZE);
  begin = min(split * share, blocks);
  end = min(begin + share, blocks);
}

// The keys of a block of SIZE from `begin` on, below `end`, found through the table.
template <typename T, int SIZE>
struct Finder {
  const Pages<const T>& cache;
  uint32_t u;
  bool whole;
  // Where a page holds whole blocks: the next 64 entries of the row, one in each lane.  A
  // block's page is then known without a load of its own, behind which loads of keys
  // would have to be waited for.
  int32_t window = 0;
  uint32_t window_first = 0, window_end = 0;

  __device__ __forceinline__ Finder(const Pages<const T>& cache_, uint32_t u_, bool whole_)
      : cache(cache_), u(u_), whole(whole_) {}

  __device__ __forceinline__ int32_t only_page(int32_t begin) {
    if (cache.table == nullptr) return static_cast<int32_t>(u);
    const uint32_t entry = cache.page_tokens.div(static_cast<uint32_t>(begin));
    if (entry >= window_end) {
      const uint32_t last = cache.page_tokens.div(cache.room) - 1;
      window_first = entry;
      window_end = entry + kWave;
      window = cache.page_at(u, min(entry + threadIdx.x % kWave, last));
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), here and not at every use
    }
    return __builtin_amdgcn_readlane(window, entry - window_first);
  }
  // Where it does not: what the table names for key begin + lane of the block (for its last
  // key where that is behind it), asked for a block ahead.
  __device__ __forceinline__ int32_t page_of(int32_t begin, int32_t end, int lane) const {
    const int32_t key = min(begin + lane % SIZE, end - 1);
    return cache.page_at(u, cache.page_tokens.div(static_cast<uint32_t>(key)));
  }
  // Which of the block's keys are there, a bit each; `page` as found by either.
  __device__ __forceinline__ uint64_t present(int32_t page, int32_t begin, int32_t end) const {
    constexpr uint64_t kAll = (uint64_t{1} << SIZE) - 1;
    const int32_t count = end - begin;
    const uint64_t inside = count >= SIZE ? kAll : (uint64_t{1} << count) - 1;
    return __ballot(cache.held(page)) & inside;
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

template <typename T, int DP, Reads READS>
struct TileSpace {
  static constexpr int KB = tile_blocks<T, DP>();
  // Three tiles, two of them on their way, where a CU's 160 KB hold them for all workgroups
  // that its registers hold, and every wave has as many loads of a tile.
  static constexpr int kTileBytes = 2 * KB * kBlock * DP * sizeof(T);
  static constexpr int kBuffers =
      READS == Reads::Aligned && KB * kBlock * DP * sizeof(T) / 16 % kThreads == 0 &&
              3 * kTileBytes * tile_waves<T, DP>() <= 160 * 1024
          ? 3
          : 2;
  Tile<T, KB * kBlock, DP, READS, kBuffers> keys, values;
};

// A workgroup's 64 rows and its share of the keys, in tiles that its waves share: every key
// read once for 64 rows.  Bound by the matrix units: 256 rows a key head over 16384 keys, 8
// heads of 128, take 152 us, 113 TFLOP/s (the units are busy in 87% of the waves' lives and
// the softmax's vector instructions take the rest); 4 * 256 tokens behind 4096, 673 us, 115
// TFLOP/s.  Pages of 5 and 100 tokens, found key by key, take 782; so are pages of 16 where
// tiles are 32 keys, at heads up to 64 (256 tokens behind 8192: 714 us, in pages of 32 620).
template <typename T, int DP, Reads READS>
__device__ __forceinline__ void tile_part(TileSpace<T, DP, READS>& space, const Call& call,
                                          const Results<T>& results, const Heads<const T>& query,
                                          const Side<T>& side, uint32_t index) {
  constexpr int KB = TileSpace<T, DP, READS>::KB;
  constexpr int KT = KB * kBlock;
  constexpr int W = Vec16<T>::width;
  constexpr uint32_t kRows = kWaves * kBlock;
  auto& keys = space.keys;
  auto& values = space.values;
  const uint32_t unit = index % side.units;
  const uint32_t rest = index / side.units;
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
  uint32_t begin_tile, end_tile;
  share_of<KT>(side, high, split, begin_tile, end_tile);

  constexpr int B = TileSpace<T, DP, READS>::kBuffers;
  using KeyTile = Tile<T, KT, DP, READS, B>;
  Finder<T, KT> finder(side.cache, u, side.whole);
  typename KeyTile::Stage next_keys, next_values;
  keys.prepare(next_keys, call.extent, [&](uint32_t j) { return j * side.cache.key.token; });
  values.prepare(next_values, call.extent, [&](uint32_t j) { return j * side.cache.value.token; });
  int32_t page = 0;                           // found for the next tile to start
  // Where pages hold whole tiles: the next tile's place in its page.
  const T* key_at = nullptr;
  const T* value_at = nullptr;
  int32_t page_left = 0;  // tokens
  bool page_held = false;
  constexpr uint64_t kAll = (uint64_t{1} << KT) - 1;
  uint64_t present[B] = {};                   // of the current tile and those behind it
  int to = 0;                                 // buffer of the next tile to start
  const auto look = [&](uint32_t i) {
    if (!side.whole && i < end_tile) {
      page = finder.page_of(static_cast<int32_t>(i) * KT, high, wave_lane);
    }
  };
  // Starts tile i, whose pages have been looked up, and looks for those of the next.
  const auto start = [&](uint32_t i) {
    const int32_t begin = static_cast<int32_t>(i) * KT;
    uint64_t there;
    if (side.whole) {
      if (page_left <= 0) {
        const int32_t only = finder.only_page(begin);
        const uint32_t slot = finder.slot(begin);
        page_held = side.cache.held(only);
        page_left = static_cast<int32_t>(side.cache.page_tokens.divisor - slot);
        key_at = finder.head(side.cache.key, key_head, only, slot);
        value_at = finder.head(side.cache.value, key_head, only, slot);
      }
      const uint32_t count = static_cast<uint32_t>(high - begin);
      there = !page_held ? 0 : count >= KT ? kAll : (uint64_t{1} << count) - 1;
      if (page_held) {
        // Rows behind the last key repeat the tile's first, and no row sees them.
        const auto in = [&](uint32_t j) { return static_cast<uint64_t>(j < count ? j : 0); };
        keys.start(next_keys, to, key_at, count >= KT, call.extent,
                   [&](uint32_t j) { return in(j) * side.cache.key.token; });
        values.start(next_values, to, value_at, count >= KT, call.extent,
                     [&](uint32_t j) { return in(j) * side.cache.value.token; });
      }
      key_at += KT * side.cache.key.token;
      value_at += KT * side.cache.value.token;
      page_left -= KT;
    } else {
      there = finder.present(page, begin, high);
      const uint32_t slot = finder.slot(begin + wave_lane % KT);
      const auto row = [&](const PageHeads<const T>& heads) {
        return [&](int, uint32_t j) {
          const int32_t at = __shfl(page, j, kWave);
          const uint32_t in = __shfl(slot, j, kWave);
          return (there >> j & 1U) != 0 ? finder.head(heads, key_head, at, in)
                                        : reinterpret_cast<const T*>(kNothing);
        };
      };
      keys.start_rows(next_keys, to, call.extent, row(side.cache.key));
      values.start_rows(next_values, to, call.extent, row(side.cache.value));
    }
    present[B - 1] = there;
    to = to + 1 < B ? to + 1 : 0;
    look(i + 1);
  };
  // Waits for the tile behind the current one, which becomes the current one: for all loads
  // but those of a tile started after it.
  const auto finish = [&](int at) {
    if constexpr (B > 2) {
      if (present[B - 1] != 0) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"i"(2 * KeyTile::kShare) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
    } else {
      keys.finish(next_keys, at);
      values.finish(next_values, at);
    }
#pragma unroll
    for (int n = 0; n + 1 < B; ++n) present[n] = present[n + 1];
    present[B - 1] = 0;
  };
  look(begin_tile);
#pragma unroll
  for (int n = 0; n + 1 < B; ++n) {
    if (n != 0) {
#pragma unroll
      for (int m = 0; m + 1 < B; ++m) present[m] = present[m + 1];
      present[B - 1] = 0;
    }
    if (begin_tile + n < end_tile) start(begin_tile + n);
  }

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
  int at = 0;  // buffer of the current tile
  if (begin_tile < end_tile) finish(at);

  for (uint32_t i = begin_tile; i < end_tile; ++i) {
    const int32_t begin = static_cast<int32_t>(i) * KT;
    __syncthreads();
    if (i + B - 1 < end_tile) start(i + B - 1);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int32_t k0 = begin + kb * kBlock, k1 = k0 + kBlock - 1;
      const uint32_t there = static_cast<uint32_t>(present[0] >> (kb * kBlock)) & 0xffffU;
      if (there == 0 || k0 > newest) continue;
      const T* key_rows = keys.value[at] + kb * kBlock * DP;
      const T* value_rows = values.value[at] + kb * kBlock * DP;
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
    at = at + 1 < B ? at + 1 : 0;
    if (i + 1 < end_tile) finish(at);
  }
  const T total = quarter_sum(row.total);
  if (!held) return;
  T* target = part_row(call, results, row_place, side.first_part + split, row.base, total,
                       lane.quarter == 0);
  if (begin_tile >= end_tile && results.splits != 1) return;
  const T over = total == T(0) ? T(0) : T(1) / total;
  row.out.visit(lane.quarter, [&](uint32_t d, auto& run) {
    // No weights: nothing, also where what they would have met is not finite.
    for (auto& x : run) x = total == T(0) ? T(0) : x * over;
    store_piece(target, d, call.extent, run);
  });
}

template <typename T, int DP>
struct TokenSpace {
  T outs[kWaves][kBlock][DP + Vec16<T>::width];
  T tops[kWaves][kBlock], totals[kWaves][kBlock];
};

// A workgroup's 16 rows and its share of the keys, of which each wave takes every fourth
// block from memory.  Bound by reading the cache: 16 sequences of up to 4096 tokens, 4 key
// heads of 128 and 8 rows each, 46 us, 3.7 TB/s: a block's loads are waited for before its
// products.
template <typename T, int DP, Reads READS>
__device__ __forceinline__ void token_part(TokenSpace<T, DP>& space, const Call& call,
                                           const Results<T>& results,
                                           const Heads<const T>& query, const Side<T>& side,
                                           uint32_t index) {
  constexpr int W = Vec16<T>::width;
  auto& outs = space.outs;
  auto& tops = space.tops;
  auto& totals = space.totals;
  const uint32_t unit = index % side.units;
  const uint32_t rest = index / side.units;
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
  uint32_t begin_block, end_block;
  share_of<kBlock>(side, high, split, begin_block, end_block);
  if (begin_block >= end_block && results.splits != 1) {
    if (threadIdx.x < end_row - begin_row) {
      part_row(call, results, row_at(call, side, u, key_head, begin_row + threadIdx.x, side_length),
               side.first_part + split, lowest_finite<T>(), T(0), true);
    }
    return;
  }

  Finder<T, kBlock> finder(side.cache, u, side.whole);
  int32_t next = 0;  // page found for the wave's next block
  const auto look = [&](uint32_t i) {
    if (!side.whole && i < end_block) {
      next = finder.page_of(static_cast<int32_t>(i) * kBlock, high, lane);
    }
  };
  look(begin_block + wave);

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
    const int32_t found = side.whole ? finder.only_page(begin) : next;
    const uint32_t there = static_cast<uint32_t>(finder.present(found, begin, high));
    look(i + kWaves);
    if (there == 0) continue;
    Operand<T, DP> k;
    AcrossOperand<T, DP> v;
    if (side.whole) {
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
          (there >> column & 1U) != 0 ? finder.head(side.cache.key, key_head, found, slot)
                                      : nothing,
          call.extent, quarter);
      v.template load<READS>(call.extent, quarter, column, [&](int n) {
        const int32_t at = __shfl(found, n, kWave);
        const uint32_t in = __shfl(slot, n, kWave);
        return (there >> n & 1U) != 0 ? finder.head(side.cache.value, key_head, at, in)
                                      : nothing;
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

// Up to four rows (a token of a group of four query heads): products of 4 keys with 4 rows,
// sixteen of them side by side in the 4x4x1 matrix instruction, where 16x16x4 would leave
// three quarters or more of its columns unused.  The instruction takes one value per lane of
// each operand (lane l: block l / 4, row or column l % 4) and adds one product to each of a
// block's 4x4 results (lane l: column l % 4; the lane's four values are the rows).
//   Scores: block b contracts d = 64 c + 4 b + i, i < 4, of keys 4 g + l % 4; the blocks'
//   sums are added up across the wave and leave key 4 g + l / 16 of row l % 4 in each lane.
//   Values: that lane's weight meets d = 64 c + 4 (l % 16) + i of its key as it stands.  The
//   quarters' sums over their keys are added up once at the end.
// Bound by reading the cache: the own tokens of 64 sequences (up to 2048 of 8 heads of 128)
// take 115 us alone, 5.2 TB/s; in token_part they and their prefix took 294 together, here
// (and in one launch) 200.
constexpr int kFewRows = 4;

__device__ __forceinline__ f32x4 few_step(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_4x4x1f32(a, b, c, 0, 0, 0);
}

// Of four values in every lane, value l / 16, summed over the lanes of all quarters with
// this l % 16.
__device__ __forceinline__ float scattered_sum(const f32x4& x) {
  const auto swapped = [](float a, float b, auto&& swap) {
    const auto both = swap(__float_as_uint(a), __float_as_uint(b));
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
  };
  const auto halves = [](uint32_t a, uint32_t b) {
    return __builtin_amdgcn_permlane32_swap(a, b, false, false);
  };
  const auto quarters = [](uint32_t a, uint32_t b) {
    return __builtin_amdgcn_permlane16_swap(a, b, false, false);
  };
  const float even = swapped(x[0], x[2], halves), odd = swapped(x[1], x[3], halves);
  return swapped(even, odd, quarters);
}

// x of the lane that is LANES further in its row of 16, around its end.
template <int LANES>
__device__ __forceinline__ float rotated(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + LANES, 0xf,
                                                     0xf, true));
}

template <int DP>
constexpr int kFewChunks = (DP + 63) / 64;

template <int DP>
struct FewSpace {
  float outs[kWaves][kFewRows][kFewChunks<DP> * 64 + 4];
  float tops[kWaves][kFewRows], totals[kWaves][kFewRows];
};

// A workgroup's rows and its share of the keys, of which each wave takes every fourth block
// from memory: the next block's loads are in flight while one is used.
template <int DP, Reads READS>
__device__ __forceinline__ void few_part(FewSpace<DP>& space, const Call& call,
                                         const Results<float>& results,
                                         const Heads<const float>& query,
                                         const Side<float>& side, uint32_t index) {
  constexpr int C = kFewChunks<DP>;
  constexpr int SIZE = C == 1 ? 16 : 8;  // keys of a block
  constexpr int G = SIZE / 4;            // groups of four keys
  // Beside tiles, whose products fill the matrix units whenever they may: the short work
  // between two reads goes first (199 us for 210).
  __builtin_amdgcn_s_setprio(3);
  const uint32_t unit = index % side.units, split = index / side.units;
  const uint32_t u = unit / call.key_heads, key_head = unit % call.key_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int quarter = lane / kBlock, column = lane % 4;

  const int32_t side_length = side.length(u);
  const int32_t high =
      side.own ? row_at(call, side, u, key_head, side.rows - 1, side_length).limit + 1
               : side_length;
  uint32_t begin_block, end_block;
  share_of<SIZE>(side, high, split, begin_block, end_block);
  const bool held = static_cast<uint32_t>(column) < side.rows;
  const RowAt row_place =
      row_at(call, side, u, key_head, held ? column : side.rows - 1, side_length);
  if (begin_block >= end_block && results.splits != 1) {
    if (threadIdx.x < side.rows) {
      part_row(call, results, row_place, side.first_part + split, lowest_finite<float>(), 0.0F,
               true);
    }
    return;
  }

  const int32_t limit = held ? row_place.limit : -1;
  int32_t oldest = held ? limit : INT32_MAX;
  oldest = min(oldest, __shfl_xor(oldest, 1, kWave));
  oldest = min(oldest, __shfl_xor(oldest, 2, kWave));
  oldest = __builtin_amdgcn_readfirstlane(oldest);
  const uint32_t key_d = lane / 4 * 4, value_d = lane % kBlock * 4;
  const float* query_row = query.data + row_place.b * query.batch +
                           row_place.head * query.head + row_place.t * query.token;
  f32x4 q[C], out[C][4];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    q[c] = load_piece<READS>(query_row, 64 * c + key_d, call.extent);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool inside = (limit >= 0) & (64 * c + key_d + i < call.extent);
      q[c][i] = inside ? q[c][i] * static_cast<float>(call.scale * kLog2E) : 0.0F;
      out[c][i] = f32x4{0, 0, 0, 0};
    }
  }
  float base = lowest_finite<float>(), total = 0.0F;

  // A block of keys and values on its way.  However few of its keys there are, it is as
  // many loads: in the place of those that are not, ones that are harmless.
  struct Stage {
    f32x4 k[G][C], v[G][C];
    int32_t begin;
    uint32_t there;
  };
  const float* nothing = reinterpret_cast<const float*>(kNothing);
  Finder<float, SIZE> finder(side.cache, u, side.whole);
  int32_t next = 0;  // page found for the next block to fetch
  const auto look = [&](uint32_t i) {
    next = finder.page_of(static_cast<int32_t>(min(i, end_block - 1)) * SIZE, high, lane);
  };
  const auto load = [&](Stage& stage, auto&& key_of, auto&& value_of) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float* head = key_of(4 * g + column);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        stage.k[g][c] = load_piece<READS>(head, 64 * c + key_d, call.extent);
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float* head = value_of(4 * g + quarter);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        stage.v[g][c] = load_piece<READS>(head, 64 * c + value_d, call.extent);
      }
    }
  };
  const auto fetch = [&](auto whole, Stage& stage, uint32_t i) {
    const int32_t begin = static_cast<int32_t>(i) * SIZE;
    stage.begin = begin;
    if constexpr (decltype(whole)::value) {
      const int32_t page = finder.only_page(begin);
      stage.there = static_cast<uint32_t>(finder.present(page, begin, high));
      const uint32_t slot = finder.slot(begin);
      const uint32_t count = stage.there != 0 ? static_cast<uint32_t>(high - begin) : 1;
      const auto in = [&](uint32_t n) { return static_cast<uint64_t>(n < count ? n : 0); };
      const float* key_base =
          stage.there != 0 ? finder.head(side.cache.key, key_head, page, slot) : nothing;
      const float* value_base =
          stage.there != 0 ? finder.head(side.cache.value, key_head, page, slot) : nothing;
      load(
          stage, [&](int n) { return key_base + in(n) * side.cache.key.token; },
          [&](int n) { return value_base + in(n) * side.cache.value.token; });
    } else {
      const int32_t page = next;
      stage.there = static_cast<uint32_t>(finder.present(page, begin, high));
      look(i + kWaves);
      const uint32_t slot = finder.slot(begin + lane % SIZE);
      const auto head_of = [&](const PageHeads<const float>& heads, int n) {
        const int32_t at = __shfl(page, n, kWave);
        const uint32_t in = __shfl(slot, n, kWave);
        return (stage.there >> n & 1U) != 0 ? finder.head(heads, key_head, at, in) : nothing;
      };
      load(
          stage, [&](int n) { return head_of(side.cache.key, n); },
          [&](int n) { return head_of(side.cache.value, n); });
    }
  };
  const auto use = [&](const Stage& stage) {
    constexpr uint32_t kAll = (1U << SIZE) - 1;
    const bool whole = (stage.begin + SIZE - 1 <= oldest) & (stage.there == kAll);
    float score[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      f32x4 s{0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int n = 0; n < 4; ++n) s = few_step(stage.k[g][c][n], q[c][n], s);
      }
      float sum = scattered_sum(s);
      sum += rotated<8>(sum);
      sum += rotated<4>(sum);
      const int at = 4 * g + quarter;
      const bool visible =
          whole | ((stage.begin + at <= limit) & ((stage.there >> at & 1U) != 0));
      score[g] = visible ? sum : lowest<float>();
    }
    float top = score[0];
#pragma unroll
    for (int g = 1; g < G; ++g) top = larger(top, score[g]);
    constexpr float kSlack = Row<float, DP>::kSlack;
    if (__any(top > base + kSlack)) {
      top = quarter_max(top);
      const float risen = top > base + kSlack ? top : base;
      const float shrink = exp2_of(base - risen);
      total *= shrink;
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
          for (int m = 0; m < 4; ++m) out[c][n][m] *= shrink;
        }
      }
      base = risen;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float weight = exp2_of(score[g] - base);
      total += weight;
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int n = 0; n < 4; ++n) out[c][n] = few_step(stage.v[g][c][n], weight, out[c][n]);
      }
    }
  };
  // Two blocks in turn; the last ones apart, and the two ways to find pages too: where a
  // load may or may not have been made, the compiler waits for all.
  const auto run_over = [&](auto whole) {
    uint32_t i = begin_block + wave;
    if (i >= end_block) return;
    uint32_t left = (end_block - i + kWaves - 1) / kWaves;
    Stage one, other;
    if constexpr (!decltype(whole)::value) look(i);
    fetch(whole, one, i);
    for (; left > 2; left -= 2, i += 2 * kWaves) {
      fetch(whole, other, i + kWaves);
      use(one);
      fetch(whole, one, i + 2 * kWaves);
      use(other);
    }
    if (left == 2) {
      fetch(whole, other, i + kWaves);
      use(one);
      use(other);
    } else {
      use(one);
    }
  };
  if (side.whole) {
    run_over(std::true_type{});
  } else {
    run_over(std::false_type{});
  }
  total = quarter_sum(total);
  if (lane < kFewRows) {
    space.tops[wave][lane] = base;
    space.totals[wave][lane] = total;
  }
  // out[c][n][m] is d = 64 c + 16 (l % 16 / 4) + 4 m + n of row l % 4, over the quarter's keys.
#pragma unroll
  for (int c = 0; c < C; ++c) {
    f32x4 piece;
#pragma unroll
    for (int n = 0; n < 4; ++n) piece[n] = scattered_sum(out[c][n]);
    const int d = 64 * c + lane % kBlock / 4 * 16 + 4 * quarter;
    *reinterpret_cast<f32x4*>(&space.outs[wave][column][d]) = piece;
  }
  __syncthreads();
  // Lane by lane over the rows' pieces: the waves in order.
  constexpr int kPieces = C * 16;
  const int r = threadIdx.x / kPieces, d = threadIdx.x % kPieces * 4;
  if (static_cast<uint32_t>(r) >= side.rows || static_cast<uint32_t>(d) >= call.extent) return;
  float most = space.tops[0][r];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) most = larger(space.tops[w][r], most);
  float sum = 0.0F;
  float run[4] = {};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float shrink = exp2_of(space.tops[w][r] - most);
    const float part = space.totals[w][r];
    sum += part * shrink;
#pragma unroll
    for (int j = 0; j < 4; ++j) run[j] += part == 0.0F ? 0.0F : space.outs[w][r][d + j] * shrink;
  }
  const float over = sum == 0.0F ? 0.0F : 1.0F / sum;
#pragma unroll
  for (int j = 0; j < 4; ++j) run[j] *= over;
  const RowAt place = row_at(call, side, u, key_head, r, side_length);
  float* target = part_row(call, results, place, side.first_part + split, most, sum, d == 0);
  store_piece(target, d, call.extent, run);
}
static_assert(kThreads >= kFewRows * kFewChunks<SPAR_HIP_ATTENTION_MAX_EXTENT> * 16);

// How a side is computed.
enum class Kind { Few, Tokens, Tiles };

template <typename T, int DP, Reads READS, Kind KIND>
struct Space {
  using type = TokenSpace<T, DP>;
};
template <typename T, int DP, Reads READS>
struct Space<T, DP, READS, Kind::Tiles> {
  using type = TileSpace<T, DP, READS>;
};
template <typename T, int DP, Reads READS>
struct Space<T, DP, READS, Kind::Few> {
  using type = FewSpace<DP>;
};

template <typename T, int DP, Reads READS, Kind KIND>
__device__ __forceinline__ void side_part(char* space, const Call& call, const Results<T>& results,
                                          const Heads<const T>& query, const Side<T>& side,
                                          uint32_t index) {
  constexpr Reads kReads = READS == Reads::Aligned ? Reads::Pieces : READS;
  auto& mine = *reinterpret_cast<typename Space<T, DP, READS, KIND>::type*>(space);
  if constexpr (KIND == Kind::Tiles) {
    tile_part<T, DP, READS>(mine, call, results, query, side, index);
  } else if constexpr (KIND == Kind::Tokens) {
    token_part<T, DP, kReads>(mine, call, results, query, side, index);
  } else {
    few_part<DP, kReads>(mine, call, results, query, side, index);
  }
}

// The prefixes' workgroups come first: their products keep the matrix units busy while the
// others, which fill what room they leave on a CU, read the sequences' own keys.  64 sequences
// behind 16384 tokens: 152 us for the prefix and 115 for the rest apart, 187 to 204 together
// (from card to card).  In turn by eights all prefix groups came to lie on half of the CUs
// (1141 us for 673 with 256 tokens of 4 sequences).  With registers for a wave more per SIMD
// 204 us where this took 193.
template <typename T, int DP, Reads READS, Kind PREFIX, Kind OWN>
__global__ __launch_bounds__(kThreads, (tile_waves<T, DP>())) void cache_kernel(
    Call call, Results<T> results, Heads<const T> query, Side<T> prefix, Side<T> own,
    uint32_t prefix_groups) {
  constexpr size_t kPrefixBytes = sizeof(typename Space<T, DP, READS, PREFIX>::type);
  constexpr size_t kOwnBytes = sizeof(typename Space<T, DP, READS, OWN>::type);
  __shared__ alignas(16) char space[kPrefixBytes > kOwnBytes ? kPrefixBytes : kOwnBytes];
  const bool mine = blockIdx.x >= prefix_groups;
  const uint32_t index = mine ? blockIdx.x - prefix_groups : blockIdx.x;
  if constexpr (PREFIX == OWN) {
    const Side<T>& side = mine ? own : prefix;
    side_part<T, DP, READS, OWN>(space, call, results, query, side, index);
  } else if (mine) {
    side_part<T, DP, READS, OWN>(space, call, results, query, own, index);
  } else {
    side_part<T, DP, READS, PREFIX>(space, call, results, query, prefix, index);
  }
}

// ---------------------------------------------------------------- launchers

// Up to this many rows of a unit (and where tiles would be few) the waves of a workgroup share
// rows and split keys; the fewest keys that repay a part: 64, 128 and 256 are within a tenth
// of each other, now one now the other ahead; of tiles 128 take 88 us for 82 (heads of 256).
// With 256 a prefix of 8192 tokens and 8 key heads is 256 workgroups at most, a wave per SIMD
// (16 sequences, heads of 128: the prefix alone 38 us with the join, 14 at the units' rate).
constexpr uint64_t kTokenRows = 32;
constexpr uint64_t kFewestKeys = 256;
constexpr uint64_t kFewestTokenKeys = 64;
constexpr uint64_t kCus = 256;

struct SidePlan {
  Kind kind;
  uint64_t units, rows, row_tiles, splits, least;
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
  const bool tiles = plan.rows > kTokenRows &&
                     !spreads((plan.rows + kRows - 1) / kRows * plan.units *
                              std::max<uint64_t>(1, room / kFewestKeys));
  const bool few = a.dtype == SPAR_HIP_FLOAT32 && plan.rows <= kFewRows;
  plan.kind = tiles ? Kind::Tiles : few ? Kind::Few : Kind::Tokens;
  return plan;
}

// Keys that a side's workgroups read at most, one after the other.
uint64_t reads_of(const SidePlan& plan, uint64_t room) {
  return plan.units * ((plan.rows + kBlock - 1) / kBlock) * room;
}

// Workgroups that a side's rows are split up to, by what a CU holds of them (`waves` per
// SIMD).
//   Tiles: all that a CU holds where they are alone there or the other side is tiles too
//   (256 tokens of 4 sequences, heads of 64, 602 us, half as many 658; but 16 tokens of 16
//   sequences, heads of 128, 361 us, with one less 346); otherwise one less, which leaves room
//   for those that read (64 sequences behind 16384 tokens: heads of 128 200 us, all that it
//   holds 264; of 64 121 and 136; of 192 195 and 220).
//   Few rows: one for each CU, whose four waves have enough loads in flight between them;
//   three take 46 us for 39 (one sequence of 4096 behind 16384) to 37 for 34 (16 sequences,
//   heads of 64), and are equal for 16 sequences with heads of 128.
//   16 rows: one less than a CU holds (8 rows, heads of 128: two 60 us, three 68, one 65).
//   Where a CU holds one, all at once: half of them for each side, or all for one that reads
//   far more than the other (heads of 256: half 70 us, all 82, twice as many 96; without a
//   prefix all 41, half 55).
uint64_t grid_of(const SparHipCacheAttention& a, Kind kind, Kind other, uint64_t reads,
                 uint64_t other_reads) {
  uint64_t waves = 0;
  with_padded_width(a.extent, [&](auto width) {
    constexpr int DP = decltype(width)::value;
    waves = a.dtype == SPAR_HIP_FLOAT32 ? tile_waves<float, DP>() : tile_waves<double, DP>();
  });
  const bool alone = other_reads < reads / 4;
  if (kind == Kind::Tiles) {
    return kCus * (alone || other == Kind::Tiles ? waves : std::max<uint64_t>(1, waves - 1));
  }
  if (waves == 1) return alone ? kCus : kCus / 2;
  return kind == Kind::Few ? kCus : kCus * (waves - 1);
}

// Workgroups of a side whose kind is settled.
void divide(SidePlan& plan, uint64_t room, uint64_t grid) {
  constexpr uint64_t kRows = kWaves * kBlock;
  const bool tiles = plan.kind == Kind::Tiles;
  const uint64_t tile_rows = tiles ? kRows : kBlock;
  const uint64_t least = tiles ? kFewestKeys : kFewestTokenKeys;
  plan.row_tiles = (plan.rows + tile_rows - 1) / tile_rows;
  const uint64_t wanted = grid / std::max<uint64_t>(1, plan.row_tiles * plan.units);
  plan.splits =
      std::max<uint64_t>(1, std::min({wanted, room / least, uint64_t{kMostParts / 2}}));
  plan.least = least / kBlock;
}

Plan plan_of(const SparHipCacheAttention& a, const SparHipPages& cache,
             const SparHipPages* prefix) {
  Plan plan{};
  plan.rows = a.batch * a.query_heads * a.queries;
  plan.own = side_plan(a, a.batch, 1, room_of(&cache));
  if (room_of(prefix) != 0) {
    plan.prefix = side_plan(a, a.prefixes, a.batch / a.prefixes, room_of(prefix));
    // There is no launch of fewer rows before more: a prefix has the more rows.
    if (plan.prefix.kind < plan.own.kind) plan.prefix.kind = plan.own.kind;
  }
  const uint64_t own_reads = reads_of(plan.own, room_of(&cache));
  const uint64_t prefix_reads = reads_of(plan.prefix, room_of(prefix));
  if (plan.prefix.units != 0) {
    divide(plan.prefix, room_of(prefix),
           grid_of(a, plan.prefix.kind, plan.own.kind, prefix_reads, own_reads));
  }
  divide(plan.own, room_of(&cache),
         grid_of(a, plan.own.kind, plan.prefix.kind, own_reads, prefix_reads));
  plan.parts = static_cast<uint32_t>(plan.own.splits + plan.prefix.splits);
  const uint64_t size = a.dtype == SPAR_HIP_FLOAT32 ? sizeof(float) : sizeof(double);
  const uint64_t piece = 16 / size;
  plan.pitch = static_cast<uint32_t>((a.extent + piece - 1) / piece * piece);
  if (plan.parts > 1) plan.bytes = plan.parts * plan.rows * (plan.pitch + 2) * size;
  return plan;
}

// A launch counts its workgroups in 32 bits of work-items.  (Rows are many only where neither
// side is split: with a prefix they have two parts, without one a single one.)
bool fits(const Plan& plan) {
  return plan.own.groups() <= kMostGroups && plan.prefix.groups() <= kMostGroups &&
         plan.own.groups() + plan.prefix.groups() <= kMostGroups && joins(plan.rows, plan.parts);
}

// Whether a cache's keys and values go to LDS directly.
template <typename T>
bool pages_aligned(const SparHipPages& cache) {
  return reads_aligned<T>(cache.key, 1) && reads_aligned<T>(cache.value, 1);
}

template <typename T>
Side<T> side_of(const SparHipCacheAttention& a, const SparHipPages& cache, const SidePlan& plan,
                bool own, uint32_t first_part, int block) {
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
  side.least = static_cast<uint32_t>(plan.least);
  side.first_part = first_part;
  // Few rows take blocks of 8 keys or of kBlock: in pages of 8 they look for every key too, at
  // no loss (16 sequences 61 us, in pages of 16 as well).
  side.whole = cache.table == nullptr ||
               cache.page_tokens % (plan.kind == Kind::Tiles ? block : kBlock) == 0;
  return side;
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
  const bool shared = plan.prefix.splits != 0;
  // Only tiles ask for heads at multiples of 16 bytes.  Where theirs are not, everything is read
  // element by element (one token of 16 sequences behind 8192 102 us for 62, of 64 behind 16384
  // 334 for 211, 256 of 4 behind 4096 876 for 669).
  const auto reads_pieces = [&](const SparHipPages& pages, const SidePlan& side) {
    return side.kind != Kind::Tiles || pages_aligned<T>(pages);
  };
  const bool pieces = a.extent % Vec16<T>::width == 0 && reads_pieces(cache, plan.own) &&
                      (!shared || reads_pieces(*prefix, plan.prefix));
  const uint32_t before_own = static_cast<uint32_t>(plan.prefix.groups());
  const uint32_t grid = static_cast<uint32_t>(plan.prefix.groups() + plan.own.groups());
  with_padded_width(a.extent, [&](auto width) {
    constexpr int DP = decltype(width)::value;
    constexpr int block = tile_blocks<T, DP>() * kBlock;
    const Side<T> before =
        shared ? side_of<T>(a, *prefix, plan.prefix, false, 0, block) : Side<T>{};
    const Side<T> own = side_of<T>(a, cache, plan.own, true,
                                   static_cast<uint32_t>(plan.prefix.splits), block);
    const auto launch = [&](auto kernel) {
      kernel<<<grid, kThreads, 0, stream>>>(call, results, q, before, own, before_own);
    };
    const auto with_kinds = [&](auto reads) {
      constexpr Reads READS = decltype(reads)::value;
      const Kind kind = plan.own.kind, prefix_kind = shared ? plan.prefix.kind : kind;
      if (kind == Kind::Tiles) {
        launch(cache_kernel<T, DP, READS, Kind::Tiles, Kind::Tiles>);
      } else if (kind == Kind::Tokens && prefix_kind == Kind::Tiles) {
        launch(cache_kernel<T, DP, READS, Kind::Tiles, Kind::Tokens>);
      } else if (kind == Kind::Tokens) {
        launch(cache_kernel<T, DP, READS, Kind::Tokens, Kind::Tokens>);
      } else if constexpr (std::is_same_v<T, float>) {
        if (prefix_kind == Kind::Tiles) {
          launch(cache_kernel<T, DP, READS, Kind::Tiles, Kind::Few>);
        } else if (prefix_kind == Kind::Tokens) {
          launch(cache_kernel<T, DP, READS, Kind::Tokens, Kind::Few>);
        } else {
          launch(cache_kernel<T, DP, READS, Kind::Few, Kind::Few>);
        }
      }
    };
    if (pieces) {
      with_kinds(std::integral_constant<Reads, Reads::Aligned>{});
    } else {
      with_kinds(std::integral_constant<Reads, Reads::Single>{});
    }
  });
  if (plan.parts > 1) join_parts<T, true>(call, results, stream);
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

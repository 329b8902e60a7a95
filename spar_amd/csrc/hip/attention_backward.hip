// Attention backward from the saved output: with P the weights, dP = do v^T and
// delta = do . o per row,
//   dS = P (dP - delta),  dq = scale dS k,  dk = scale dS^T q,  dv = P^T do.
//
// Two kernels (each in a form for large and one for small grids), so that every gradient
// has one writer and sums in a fixed order.
// query_kernel keeps 16 rows per wave and walks the keys they see (as the forward
// does, with the running maximum and sum of the softmax); it also leaves delta and the
// softmax's base and sum behind.  key_kernel keeps 16 keys per wave and walks
// the rows that see them, the heads of a group among them.  Each recomputes S and
// dP: seven products instead of the five that one kernel with shared sums of dq
// would need, for results that do not depend on the order of workgroups.  In both,
// P and dS pass from the products that yield them into those that consume them in
// registers (attention.hpp).
//
// Weights.  P = 2^(s - base) / sum with scores of the very same bits in both kernels, so
// that a weight is at most 1 whatever a score's size.  (From the forward's logsumexp it
// would be 2^(what rounding s and logsumexp has lost): off by 1e-4 at scores of 1000,
// by half at 1e6, 0 or infinite from 1e9 on.)  The query is the one operand that both
// kernels could not scale alike, resident in one and in LDS in the other: of
// scale * log2(e) the power of two, exact in either operand, goes into the resident one
// and the rest, between 1 and 2, is multiplied into the finished score.  Finding
// maximum and sum again costs some 16 vector instructions a block in query_kernel and the
// factors 8 in key_kernel: 229 against 223 us and 312 against 308 at heads of 64, 0.7%
// of either at heads of 128.
//
// Rows of a tile of keys are split over several workgroups where the tiles alone do
// not fill the chip; and the sinks, which every later row sees, have thousands of
// rows where other keys have the window's: those behind a tile's own window are split
// too; so are the keys of few rows.  Splits write parts, which join_kernel and
// query_join_kernel add in their order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "attention.hpp"

namespace spar_hip {
namespace attention {
namespace {

template <typename T>
struct Saved {
  Heads<const T> query, key, value, output, output_gradient;
  T* statistics;  // [kStatistics][batch][query head][query]
  T power, rest;  // scale * log2(e), its power of two and what remains

  __device__ __forceinline__ T& of(int statistic, const Call& call, uint64_t row) const {
    return statistics[statistic * call.all_rows() + row];
  }
};

// Of a row: do . o, what its weights are powers of two over, and 1 / their sum (0 where
// there is none).
constexpr int kDelta = 0, kBase = 1, kOver = 2, kStatistics = 3;

// 1 / a sum of weights.
template <typename T>
__device__ __forceinline__ T over_of(T sum) {
  return sum == T(0) ? T(0) : T(1) / sum;
}

// How the rows of tiles of keys are split, and where the parts lie: of every tile's
// window (none for one split), then of the rows behind the windows of the sinks' tiles.
template <typename T>
struct Splits {
  // [batch head][tile][split][dk, dv][tile_keys][extent], and the same of the sinks
  T* parts;
  uint32_t tile_keys;
  uint32_t key_tiles, main;    // splits of a tile's window: at least 1
  uint32_t sink_tiles, later;  // splits of the rows behind it
  uint32_t extent;

  __device__ __forceinline__ uint64_t size() const {  // of a part
    return static_cast<uint64_t>(2 * tile_keys) * extent;
  }
  __device__ __forceinline__ T* main_part(uint32_t batch_head, uint32_t tile,
                                          uint32_t split) const {
    return parts + ((static_cast<uint64_t>(batch_head) * key_tiles + tile) * main + split) * size();
  }
  __device__ __forceinline__ T* later_part(uint32_t batch_heads, uint32_t batch_head,
                                           uint32_t tile, uint32_t split) const {
    T* const behind =
        main == 1 ? parts : parts + static_cast<uint64_t>(batch_heads) * key_tiles * main * size();
    return behind +
           ((static_cast<uint64_t>(batch_head) * sink_tiles + tile) * later + split) * size();
  }
};

// Query head, query and place among [batch][query head][query] of a row.
struct Place {
  uint32_t head, t;
  uint64_t at;

  __device__ __forceinline__ Place(const Call& call, uint32_t b, uint32_t key_head, uint32_t r) {
    t = call.group.div(r);
    head = key_head * call.group.divisor + (r - t * call.group.divisor);
    at = (static_cast<uint64_t>(b) * call.key_heads * call.group.divisor + head) * call.queries +
         t;
  }
  template <typename T>
  __device__ __forceinline__ T* of(const Heads<T>& heads, uint32_t b) const {
    return heads.data + b * heads.batch + head * heads.head + t * heads.token;
  }
};

// What dq of a row is made from, as the row's four lanes hold it.
template <typename T, int DP>
struct QueryRow {
  Operand<T, DP> q, g;  // scaled by saved.power; the output gradient
  T delta = T(0);       // do . o

  template <Reads READS>
  __device__ __forceinline__ void load(const Call& call, const Saved<T>& saved,
                                       const Place& place, uint32_t b, bool held, int quarter) {
    Operand<T, DP> out;
    q.template load<READS>(place.of(saved.query, b), call.extent, quarter);
    g.template load<READS>(place.of(saved.output_gradient, b), call.extent, quarter);
    out.template load<READS>(place.of(saved.output, b), call.extent, quarter);
    q.finish(held, call.extent, quarter, saved.power);
    g.finish(held, call.extent, quarter, T(1));
#pragma unroll
    for (int i = 0; i < DP / 4; ++i) delta += out.value[i] * g.value[i];
    delta = quarter_sum(delta);
  }
};

// s += a_rows a and dp += b_rows b of a block of 16 rows each, side by side: two sums
// take turns in the matrix units.
template <typename T, int DP>
__device__ __forceinline__ void products(const Lane<T, DP>& lane, const T* a_rows,
                                         const Operand<T, DP>& a, typename Mma<T>::Acc& s,
                                         const T* b_rows, const Operand<T, DP>& b,
                                         typename Mma<T>::Acc& dp) {
  constexpr int W = Vec16<T>::width;
  struct Pair {
    typename Vec16<T>::type a, b;
  };
  const auto read = [&](int i) { return Pair{lane.along(a_rows, i), lane.along(b_rows, i)}; };
  Queue<1, Pair> queue;
  fill_queue(queue, read);
  run_queue<DP / (4 * W)>(queue, read, [&](int i, const Pair& pair) {
#pragma unroll
    for (int n = 0; n < W; ++n) {
      s = Mma<T>::step(pair.a[n], a.value[i * W + n], s);
      dp = Mma<T>::step(pair.b[n], b.value[i * W + n], dp);
    }
  });
}

// dq and delta of 64 rows, 16 per wave, over tiles of the keys they see.  Bound by the
// matrix units, busy in 88% of the CUs' cycles at heads of 128 (6 extent operations per
// visible pair): 32 heads of 128 with 8192 tokens, window 1024 and 4 sinks in 1.49 ms,
// 130 TFLOP/s of visible pairs; 256 heads of 64 with 1024 tokens and window 256 in
// 228 us, 100 TFLOP/s and 73%, where the blocks of 16 keys that the window's edges cut and
// a block of sinks are a tenth of the work and the vector instructions weigh twice as much.
template <typename T, int DP, int KB, Reads READS>
__global__ __launch_bounds__(kThreads, (tile_waves<T, DP>())) void query_kernel(
    Call call, Saved<T> saved, Heads<T> gradient, uint32_t row_tiles) {
  constexpr int KT = KB * kBlock;
  constexpr uint32_t kRows = kWaves * kBlock;
  __shared__ Tile<T, KT, DP, READS> keys, values;
  const uint32_t batch_head = blockIdx.x % call.batch_heads;
  const uint32_t row_tile = row_tiles - 1 - blockIdx.x / call.batch_heads;
  const uint32_t b = batch_head / call.key_heads, key_head = batch_head % call.key_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const Lane<T, DP> lane(threadIdx.x % kWave);
  const int quarter = lane.quarter, column = lane.column;

  const int32_t first = call.length(b) - call.queries;
  const uint32_t begin_row = row_tile * kRows;
  const uint32_t end_row = begin_row + kRows < call.rows ? begin_row + kRows : call.rows;
  const int32_t low_token = call.token(begin_row, first);
  const Keys seen(call, low_token < 0 ? 0 : low_token, call.token(end_row - 1, first));
  const uint32_t tiles = seen.tiles(KT);

  const uint32_t wave_row = begin_row + wave * kBlock;
  const uint32_t wave_end = wave_row + kBlock < call.rows ? wave_row + kBlock : call.rows;
  const int32_t oldest = call.token(wave_row, first);
  const int32_t newest = wave_row < wave_end ? call.token(wave_end - 1, first) : -1;
  const uint32_t r = wave_row + column;
  const int32_t token = call.token(r, first);
  const Place place(call, b, key_head, r < call.rows ? r : 0);
  QueryRow<T, DP> own;
  own.template load<READS>(call, saved, place, b, token >= 0, quarter);
  Row<T, DP> row;  // its sum is dq
  row.out.clear();
  const T* key_base = saved.key.data + b * saved.key.batch + key_head * saved.key.head;
  const T* value_base = saved.value.data + b * saved.value.batch + key_head * saved.value.head;

  // Rows of a tile behind its run repeat the tile's first key; no row sees them.
  typename Tile<T, KT, DP, READS>::Stage next_keys, next_values;
  keys.prepare(next_keys, call.extent, [&](uint32_t j) { return j * saved.key.token; });
  values.prepare(next_values, call.extent, [&](uint32_t j) { return j * saved.value.token; });
  const auto start = [&](uint32_t i) {
    int32_t begin, end;
    seen.tile(i, KT, begin, end);
    const uint64_t rows = end - begin;
    const auto at = [&](uint64_t j) { return j < rows ? j : 0; };
    keys.start(next_keys, i % 2, key_base + begin * saved.key.token, rows >= KT, call.extent,
               [&](uint32_t j) { return at(j) * saved.key.token; });
    values.start(next_values, i % 2, value_base + begin * saved.value.token, rows >= KT,
                 call.extent, [&](uint32_t j) { return at(j) * saved.value.token; });
  };
  const auto finish = [&](uint32_t i) {
    keys.finish(next_keys, i % 2);
    values.finish(next_values, i % 2);
  };
  if (tiles != 0) {
    start(0);
    finish(0);
  }

  for (uint32_t i = 0; i < tiles; ++i) {
    int32_t begin, end;
    seen.tile(i, KT, begin, end);
    __syncthreads();
    if (i + 1 < tiles) start(i + 1);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int32_t k0 = begin + kb * kBlock, k1 = k0 + kBlock - 1;
      const bool any = k0 < end && k0 <= newest &&
                       ((oldest < 0 ? 0 : oldest) - k1 < call.window || k0 < call.sinks);
      if (!any) continue;
      const bool whole = k1 <= oldest && k1 < end &&
                         (newest - k0 < call.window || k1 < call.sinks);
      const T* key_rows = keys.value[i % 2] + kb * kBlock * DP;
      const T* value_rows = values.value[i % 2] + kb * kBlock * DP;
      typename Mma<T>::Acc s{0, 0, 0, 0}, dp{0, 0, 0, 0};
      products(lane, key_rows, own.q, s, value_rows, own.g, dp);
      Across<T, DP> across(lane, key_rows);
      T weight[4], ds[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        weight[v] = s[v] * saved.rest;
        ds[v] = dp[v] - own.delta;
      }
      if (!whole) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int32_t at = k0 + Mma<T>::row_of(v, quarter);
          const bool visible = (at < end) & call.sees(token, at);
          weight[v] = visible ? weight[v] : lowest<T>();
          ds[v] = visible ? ds[v] : T(0);
        }
      }
      row.take(weight);
#pragma unroll
      for (int v = 0; v < 4; ++v) ds[v] *= weight[v];
      across.run(row.out, ds);
    }
    if (i + 1 < tiles) finish(i + 1);
  }
  const T over = over_of(quarter_sum(row.total));
  if (r >= call.rows) return;
  if (quarter == 0) {
    saved.of(kDelta, call, place.at) = own.delta;
    saved.of(kBase, call, place.at) = row.base;
    saved.of(kOver, call, place.at) = over;
  }
  T* target = place.of(gradient, b);
  row.out.visit(quarter, [&](uint32_t d, auto& run) {
    for (auto& x : run) x = x * over * static_cast<T>(call.scale);
    store_piece(target, d, call.extent, run);
  });
}

// The spread kernels' operands and sums stay in registers up to this many bytes of a head
// (key_spread_kernel for 4 heads of 160 with 210 float64 tokens 81 us against key_kernel's
// 65).
constexpr uint64_t kMostSpreadBytes = 1024;

// Parts of dq [split][batch][query head][query][extent], without the scale and the
// weights' sum, and their bases and sums [split][batch][query head][query].
template <typename T>
struct QueryParts {
  T *dq, *top, *total;
  uint32_t splits;
};

// The same for grids that tiles of 64 rows do not fill: a workgroup's waves share 16
// rows and take every fourth block of 16 keys, straight from memory; their sums meet
// in LDS.  18 heads of 72 with 333 float64 tokens and a window of 100 in 23 us, five
// blocks a wave with the latency of their loads (query_kernel: 31 us).
template <typename T, int DP, Reads READS>
__global__ __launch_bounds__(kThreads) void query_spread_kernel(Call call, Saved<T> saved,
                                                                Heads<T> gradient,
                                                                uint32_t row_tiles,
                                                                QueryParts<T> parts) {
  constexpr int W = Vec16<T>::width;
  // A block's keys, values and keys again are asked for at once where registers hold them,
  // and eight pieces at a time where not (4 heads of 160 with 210 float64
  // tokens: forward and backward 153 us against 181).
  constexpr bool kTogether = DP * sizeof(T) <= kMostSpreadBytes;
  __shared__ alignas(16) T sums[kWaves][kBlock][DP + W];
  __shared__ T tops[kWaves][kBlock], totals[kWaves][kBlock];
  const uint32_t splits = parts.splits;
  const uint32_t batch_head = blockIdx.x % call.batch_heads;
  const uint32_t rest = blockIdx.x / call.batch_heads;
  uint32_t split = 0, row_tile = row_tiles - 1 - rest;
  if (splits != 1) {
    split = rest % splits;
    row_tile = row_tiles - 1 - rest / splits;
  }
  const uint32_t b = batch_head / call.key_heads, key_head = batch_head % call.key_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int quarter = threadIdx.x % kWave / kBlock, column = threadIdx.x % kBlock;

  const int32_t first = call.length(b) - call.queries;
  const uint32_t begin_row = row_tile * kBlock;
  const uint32_t end_row = begin_row + kBlock < call.rows ? begin_row + kBlock : call.rows;
  const int32_t oldest = call.token(begin_row, first);
  const int32_t newest = call.token(end_row - 1, first);
  const Keys seen(call, oldest < 0 ? 0 : oldest, newest);
  uint32_t begin_block = 0, end_block = seen.tiles(kBlock);
  if (splits != 1) {
    const uint64_t blocks = end_block;
    begin_block = static_cast<uint32_t>(blocks * split / splits);
    end_block = static_cast<uint32_t>(blocks * (split + 1) / splits);
  }
  const uint32_t r = begin_row + column;
  const int32_t token = call.token(r, first);
  const Place place(call, b, key_head, r < call.rows ? r : 0);
  QueryRow<T, DP> held;
  held.template load<READS>(call, saved, place, b, token >= 0, quarter);
  if (split == 0 && wave == 0 && quarter == 0 && r < call.rows) {
    saved.of(kDelta, call, place.at) = held.delta;
  }
  Row<T, DP> row;
  row.out.clear();
  const T* key_base = saved.key.data + b * saved.key.batch + key_head * saved.key.head;
  const T* value_base = saved.value.data + b * saved.value.batch + key_head * saved.value.head;

  for (uint32_t i = begin_block + wave; i < end_block; i += kWaves) {
    int32_t begin, end;
    seen.tile(i, kBlock, begin, end);
    // Keys behind the run repeat its block's first; no row sees them.
    const auto at_key = [&](int32_t k) { return static_cast<uint64_t>(k < end ? k : begin); };
    const uint64_t own = at_key(begin + column);
    typename Mma<T>::Acc s{0, 0, 0, 0}, dp{0, 0, 0, 0};
    AcrossOperand<T, DP> across;
    const auto load_across = [&]() {
      across.template load<READS>(call.extent, quarter, column, [&](int n) {
        return key_base + at_key(begin + n) * saved.key.token;
      });
    };
    if constexpr (kTogether) {
      Operand<T, DP> k, x;
      k.template load<READS>(key_base + own * saved.key.token, call.extent, quarter);
      x.template load<READS>(value_base + own * saved.value.token, call.extent, quarter);
      load_across();
#pragma unroll
      for (int step = 0; step < DP / 4; ++step) {
        s = Mma<T>::step(k.value[step], held.q.value[step], s);
        dp = Mma<T>::step(x.value[step], held.g.value[step], dp);
      }
    } else {
      const auto product = [&](const T* head, const Operand<T, DP>& with,
                               typename Mma<T>::Acc& sum) {
#pragma unroll
        for (int n = 0; n < DP / (4 * W); ++n) {
          const auto piece = load_piece<READS>(head, 4 * W * n + W * quarter, call.extent);
#pragma unroll
          for (int w = 0; w < W; ++w) sum = Mma<T>::step(piece[w], with.value[n * W + w], sum);
          if (READS != Reads::Single && n % 8 == 7) keep_order();
        }
      };
      product(key_base + own * saved.key.token, held.q, s);
      product(value_base + own * saved.value.token, held.g, dp);
    }
    T weight[4], ds[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int32_t at = begin + Mma<T>::row_of(v, quarter);
      const bool visible = (at < end) & call.sees(token, at);
      weight[v] = visible ? s[v] * saved.rest : lowest<T>();
      ds[v] = visible ? dp[v] - held.delta : T(0);
    }
    row.take(weight);
#pragma unroll
    for (int v = 0; v < 4; ++v) ds[v] *= weight[v];
    if constexpr (!kTogether) load_across();
    across.add_to(row.out, ds);
  }
  const T total = quarter_sum(row.total);
  if (quarter == 0) {
    tops[wave][column] = row.base;
    totals[wave][column] = total;
  }
  row.out.visit(quarter, [&](uint32_t d, auto& run) {
    for (auto& y : run) sums[wave][column][d++] = y;
  });
  __syncthreads();
  constexpr int kPieces = DP / W;
  for (int at = threadIdx.x; at < kBlock * kPieces; at += kThreads) {
    const int c = at / kPieces, d = at % kPieces * W;
    if (begin_row + c >= call.rows) continue;
    T top = tops[0][c];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = larger(tops[w][c], top);
      T sum = T(0);
    T run[W] = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const T shrink = exp2_of(tops[w][c] - top);
      sum += totals[w][c] * shrink;
#pragma unroll
      for (int j = 0; j < W; ++j) run[j] += sums[w][c][d + j] * shrink;
    }
    const Place to(call, b, key_head, begin_row + c);
    if (splits == 1) {
      const T over = over_of(sum);
      if (d == 0) {
        saved.of(kBase, call, to.at) = top;
        saved.of(kOver, call, to.at) = over;
      }
#pragma unroll
      for (int j = 0; j < W; ++j) run[j] = run[j] * over * static_cast<T>(call.scale);
      store_piece(to.of(gradient, b), d, call.extent, run);
    } else {
      const uint64_t part = split * call.all_rows() + to.at;
      if (d == 0) {
        parts.top[part] = top;
        parts.total[part] = sum;
      }
      store_piece(parts.dq + part * call.extent, d, call.extent, run);
    }
  }
}

// dq from its parts, in their order, and the row's base and sum: a lane per element.
template <typename T>
__global__ __launch_bounds__(kThreads) void query_join_kernel(Call call, Saved<T> saved,
                                                              Heads<T> gradient,
                                                              QueryParts<T> parts) {
  const uint64_t at = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const uint64_t rows = call.all_rows(), all = rows * call.extent;
  if (at >= all) return;
  const uint64_t row = at / call.extent, batch_head = row / call.queries;
  T top = parts.top[row];
#pragma unroll 4
  for (uint32_t s = 1; s < parts.splits; ++s) top = larger(parts.top[s * rows + row], top);
  T sum = T(0), total = T(0);
#pragma unroll 4
  for (uint32_t s = 0; s < parts.splits; ++s) {
    const T shrink = exp2_of(parts.top[s * rows + row] - top);
    total += parts.total[s * rows + row] * shrink;
    sum += parts.dq[s * all + at] * shrink;
  }
  const T over = over_of(total);
  if (at == row * call.extent) {
    saved.of(kBase, call, row) = top;
    saved.of(kOver, call, row) = over;
  }
  const uint32_t heads = call.key_heads * call.group.divisor;
  const uint64_t b = batch_head / heads, head = batch_head - b * heads;
  gradient.data[b * gradient.batch + head * gradient.head +
                (row - batch_head * call.queries) * gradient.token + (at - row * call.extent)] =
      sum * over * static_cast<T>(call.scale);
}

// A token's bits as a value of the heads' type, and back.
template <typename T>
__device__ __forceinline__ T bits_of(int32_t token) {
  if constexpr (sizeof(T) == 4) {
    return __int_as_float(token);
  } else {
    return __longlong_as_double(token);
  }
}
__device__ __forceinline__ int32_t token_of(float bits) { return __float_as_int(bits); }
__device__ __forceinline__ int32_t token_of(double bits) {
  return static_cast<int32_t>(__double_as_longlong(bits));
}

constexpr uint32_t kKeyTile = kWaves * kBlock;

// Its operands and sums take a third more registers than the other kernels'; float32
// tiles that go to LDS directly leave room for a fourth wave.
template <typename T, int DP, Reads READS>
constexpr int key_waves() {
  constexpr int row = DP * sizeof(T);
  if (row <= 256) return sizeof(T) == 4 && READS == Reads::Aligned ? 4 : 3;
  return row <= 512 ? 2 : 1;
}

// Blocks of 16 keys that share a tile's waves, for so many sinks in the tile.
__host__ __device__ inline int sink_blocks(int32_t sinks) {
  return sinks <= kBlock ? 1 : sinks <= 2 * kBlock ? 2 : kWaves;
}

// What a workgroup of either key kernel has to do: a tile of keys, and the rows that see
// one of them, through the window or behind it as sinks.
struct KeyTile {
  uint32_t batch_head, b, key_head;
  uint32_t tile, split, parts;
  bool behind;
  int32_t length, first;  // tokens of the sequence; the token of query 0
  int32_t begin_key;
  uint32_t begin_row, end_row;

  // The tiles of keys come first, the short splits of the sinks' later rows last.
  template <typename T>
  __device__ __forceinline__ KeyTile(const Call& call, const Splits<T>& splits,
                                     int32_t tile_keys) {
    batch_head = blockIdx.x % call.batch_heads;
    const uint32_t rest = blockIdx.x / call.batch_heads;
    const uint32_t main_groups = splits.key_tiles * splits.main;
    behind = rest >= main_groups;
    parts = behind ? splits.later : splits.main;
    tile = (behind ? rest - main_groups : rest) / parts;
    split = (behind ? rest - main_groups : rest) % parts;
    b = batch_head / call.key_heads;
    key_head = batch_head % call.key_heads;
    length = call.length(b);
    first = length - call.queries;
    begin_key = static_cast<int32_t>(tile) * tile_keys;
    const int32_t end_key = begin_key + tile_keys < length ? begin_key + tile_keys : length;
    int32_t low = begin_key, high = end_key - 1 + call.window;  // tokens [low, high)
    if (high > length) high = length;
    if (behind) {
      low = high;
      high = length;
      if (begin_key >= call.sinks) low = high;
    }
    if (low < first) low = first;
    if (low < 0) low = 0;
    if (high < low || begin_key >= length) high = low;
    begin_row = static_cast<uint32_t>(low - first) * call.group.divisor;
    end_row = static_cast<uint32_t>(high - first) * call.group.divisor;
    if (begin_row >= end_row) begin_row = end_row = 0;
  }
  // This split's share of so many blocks of rows.
  __device__ __forceinline__ uint32_t share(uint32_t blocks, uint32_t of) const {
    return static_cast<uint32_t>(static_cast<uint64_t>(blocks) * of / parts);
  }
  // Keys whose gradients it yields end here.
  __device__ __forceinline__ int32_t end_key(const Call& call) const {
    return behind ? call.sinks : static_cast<int32_t>(call.keys);
  }
  // Where the gradients of key `at` of the tile go: a part, or the result.
  template <typename T>
  __device__ __forceinline__ void targets(const Call& call, const Splits<T>& splits,
                                          const Heads<T>& key_gradient,
                                          const Heads<T>& value_gradient, uint32_t at,
                                          uint32_t own, T*& dk, T*& dv) const {
    if (behind || splits.main > 1) {
      T* part = behind ? splits.later_part(call.batch_heads, batch_head, tile, split)
                       : splits.main_part(batch_head, tile, split);
      dk = part + static_cast<uint64_t>(at) * call.extent;
      dv = dk + static_cast<uint64_t>(splits.tile_keys) * call.extent;
    } else {
      dk = key_gradient.data + b * key_gradient.batch + key_head * key_gradient.head +
           own * key_gradient.token;
      dv = value_gradient.data + b * value_gradient.batch + key_head * value_gradient.head +
           own * value_gradient.token;
    }
  }
};

// dk and dv of 64 keys, 16 per wave, over tiles of the rows that see them.  Bound by the
// matrix units, busy in 81% of the CUs' cycles at heads of 128 (8 extent operations per
// visible pair; two waves per SIMD, all that the two sums' registers leave room for): the calls
// at query_kernel in 2.18 ms, 119 TFLOP/s, and 311 us, 98 TFLOP/s and 70%.
template <typename T, int DP, int RB, Reads READS>
__global__ __launch_bounds__(kThreads, (key_waves<T, DP, READS>())) void key_kernel(
    Call call, Saved<T> saved, Heads<T> key_gradient, Heads<T> value_gradient,
    Splits<T> splits) {
  constexpr int RT = RB * kBlock;
  __shared__ Tile<T, RT, DP, READS> queries, output_gradients;
  // Of the tile's rows, and their tokens' bits behind.
  __shared__ alignas(16) T statistics[2][kStatistics + 1][RT];
  const KeyTile work(call, splits, kKeyTile);
  const uint32_t b = work.b, key_head = work.key_head;
  const bool behind = work.behind;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const Lane<T, DP> lane(threadIdx.x % kWave);
  const int quarter = lane.quarter, column = lane.column;

  const int32_t length = work.length, first = work.first, begin_key = work.begin_key;
  const uint32_t begin_row = work.begin_row, end_row = work.end_row;
  uint32_t tiles = (end_row - begin_row + RT - 1) / RT;
  const uint32_t begin_tile = work.share(tiles, work.split);
  tiles = work.share(tiles, work.split + 1);

  // Behind the window a tile with few sinks gives its waves the same keys and every
  // second or fourth block of rows.
  const int key_blocks = behind ? sink_blocks(call.sinks - begin_key) : kWaves;
  const int32_t wave_key = begin_key + wave % key_blocks * kBlock;
  const uint32_t turns = kWaves / key_blocks, turn = wave / key_blocks;
  const int32_t own = wave_key + column;
  const bool keeps = own < length;
  const T* key_base = saved.key.data + b * saved.key.batch + key_head * saved.key.head;
  const T* value_base = saved.value.data + b * saved.value.batch + key_head * saved.value.head;
  Operand<T, DP> k, x;
  {
    const uint64_t at = static_cast<uint32_t>(own) < call.keys ? own : 0;
    k.template load<READS>(key_base + at * saved.key.token, call.extent, quarter);
    x.template load<READS>(value_base + at * saved.value.token, call.extent, quarter);
    k.finish(keeps, call.extent, quarter, saved.power);
    x.finish(keeps, call.extent, quarter, T(1));
  }
  Along<T, DP> dk, dv;
  dk.clear();
  dv.clear();

  // Rows of a tile behind the last repeat the tile's first; their token sees nothing.
  typename Tile<T, RT, DP, READS>::Stage next_queries, next_gradients;
  // A thread brings one of a row's statistics, or its token.
  static_assert((kStatistics + 1) * RT <= kThreads);
  const uint32_t which = threadIdx.x / RT, its_row = threadIdx.x % RT;
  T next_statistic;
  // Offsets of a tile's rows from the first head of the query of its first row,
  // `extra` heads behind which that row is.
  const uint32_t group = call.group.divisor;
  const T* query_base = saved.query.data + b * saved.query.batch +
                        static_cast<uint64_t>(key_head) * group * saved.query.head;
  const T* gradient_base = saved.output_gradient.data + b * saved.output_gradient.batch +
                           static_cast<uint64_t>(key_head) * group * saved.output_gradient.head;
  const auto offset = [&](const Heads<const T>& heads, uint32_t j) {
    const uint32_t t = call.group.div(j);
    return t * heads.token + (j - t * group) * heads.head;
  };
  const bool even = RT % group == 0;
  queries.prepare(next_queries, call.extent,
                  [&](uint32_t j) { return offset(saved.query, j); });
  output_gradients.prepare(next_gradients, call.extent,
                           [&](uint32_t j) { return offset(saved.output_gradient, j); });
  const auto start = [&](uint32_t i) {
    const uint32_t row0 = begin_row + i * RT;
    if (which <= kStatistics) {
      const bool row = row0 + its_row < end_row;
      const Place place(call, b, key_head, row ? row0 + its_row : row0);
      if (which == kStatistics) {
        next_statistic = bits_of<T>(row ? first + static_cast<int32_t>(place.t) : -1);
      } else {
        next_statistic = saved.of(which, call, place.at);
      }
    }
    const uint32_t t0 = call.group.div(row0), extra = row0 - t0 * group;
    const bool whole = even && row0 + RT <= end_row;
    const auto at = [&](uint32_t j) { return extra + (row0 + j < end_row ? j : 0); };
    queries.start(next_queries, i % 2, query_base + t0 * saved.query.token, whole, call.extent,
                  [&](uint32_t j) { return offset(saved.query, at(j)); });
    output_gradients.start(next_gradients, i % 2,
                           gradient_base + t0 * saved.output_gradient.token, whole, call.extent,
                           [&](uint32_t j) { return offset(saved.output_gradient, at(j)); });
  };
  const auto finish = [&](uint32_t i) {
    if (which <= kStatistics) statistics[i % 2][which][its_row] = next_statistic;
    queries.finish(next_queries, i % 2);
    output_gradients.finish(next_gradients, i % 2);
  };
  if (begin_tile < tiles) {
    start(begin_tile);
    finish(begin_tile);
  }

  for (uint32_t i = begin_tile; i < tiles; ++i) {
    const uint32_t row0 = begin_row + i * RT;
    __syncthreads();
    if (i + 1 < tiles) start(i + 1);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const uint32_t block_row = row0 + rb * kBlock;
      if (block_row >= end_row) break;
      if ((i * RB + rb) % turns != turn) continue;
      const uint32_t block_end =
          block_row + kBlock < end_row ? block_row + kBlock : end_row;
      const int32_t oldest = call.token(block_row, first);
      const int32_t newest = call.token(block_end - 1, first);
      const int32_t last_key = wave_key + kBlock - 1;
      const bool any = wave_key < length && wave_key <= newest &&
                       (oldest - last_key < call.window || wave_key < call.sinks);
      if (!any) continue;
      const bool whole = last_key <= oldest && block_end - block_row == kBlock &&
                         (newest - wave_key < call.window || last_key < call.sinks);
      const T* query_rows = queries.value[i % 2] + rb * kBlock * DP;
      const T* gradient_rows = output_gradients.value[i % 2] + rb * kBlock * DP;
      typename Mma<T>::Acc s{0, 0, 0, 0}, dp{0, 0, 0, 0};
      products(lane, query_rows, k, s, gradient_rows, x, dp);
      Across<T, DP> across_gradients(lane, gradient_rows);
      T p[4], ds[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int row = rb * kBlock + Mma<T>::row_of(v, quarter);
        p[v] = exp2_of(s[v] * saved.rest - statistics[i % 2][kBase][row]) *
               statistics[i % 2][kOver][row];
        ds[v] = p[v] * (dp[v] - statistics[i % 2][kDelta][row]);
      }
      if (!whole) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int row = rb * kBlock + Mma<T>::row_of(v, quarter);
          const bool visible = call.sees(token_of(statistics[i % 2][kStatistics][row]), own);
          p[v] = visible ? p[v] : T(0);
          ds[v] = visible ? ds[v] : T(0);
        }
      }
      across_gradients.run(dv, p);
      Across<T, DP> across_queries(lane, query_rows);
      across_queries.run(dk, ds);
    }
    if (i + 1 < tiles) finish(i + 1);
  }

  if (own >= work.end_key(call)) return;
  T *dk_target, *dv_target;
  work.targets(call, splits, key_gradient, value_gradient, wave * kBlock + column, own, dk_target,
               dv_target);
  dk.visit(quarter, [&](uint32_t d, auto& run) {
    for (auto& y : run) y *= static_cast<T>(call.scale);
    store_piece(dk_target, d, call.extent, run);
  });
  dv.visit(quarter, [&](uint32_t d, auto& run) { store_piece(dv_target, d, call.extent, run); });
}

// The same for grids that tiles of 64 keys do not fill: a workgroup's waves share 16
// keys and take every fourth block of 16 rows, straight from memory; their sums meet
// in LDS.  Bound by the latency of a block's loads, about 3 us a block.
template <typename T, int DP, Reads READS>
__global__ __launch_bounds__(kThreads) void key_spread_kernel(Call call, Saved<T> saved,
                                                              Heads<T> key_gradient,
                                                              Heads<T> value_gradient,
                                                              Splits<T> splits) {
  constexpr int W = Vec16<T>::width;
  __shared__ alignas(16) T sums[kWaves][kBlock][DP + W];
  const KeyTile work(call, splits, kBlock);
  const uint32_t b = work.b, key_head = work.key_head;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int quarter = threadIdx.x % kWave / kBlock, column = threadIdx.x % kBlock;
  const uint32_t begin_row = work.begin_row, end_row = work.end_row;
  const uint32_t blocks = (end_row - begin_row + kBlock - 1) / kBlock;
  const uint32_t end_block = work.share(blocks, work.split + 1);

  const int32_t own = work.begin_key + column;
  const bool keeps = own < work.length;
  Operand<T, DP> k, x;
  {
    const uint64_t at = static_cast<uint32_t>(own) < call.keys ? own : 0;
    k.template load<READS>(
        saved.key.data + b * saved.key.batch + key_head * saved.key.head + at * saved.key.token,
        call.extent, quarter);
    x.template load<READS>(saved.value.data + b * saved.value.batch +
                               key_head * saved.value.head + at * saved.value.token,
                           call.extent, quarter);
    k.finish(keeps, call.extent, quarter, saved.power);
    x.finish(keeps, call.extent, quarter, T(1));
  }
  Along<T, DP> dk, dv;
  dk.clear();
  dv.clear();

  for (uint32_t i = work.share(blocks, work.split) + wave; i < end_block; i += kWaves) {
    const uint32_t row0 = begin_row + i * kBlock;
    // Rows behind the last repeat the block's first; their token sees nothing.
    const auto place_of = [&](uint32_t j) {
      return Place(call, b, key_head, row0 + j < end_row ? row0 + j : row0);
    };
    const Place read = place_of(column);
    Operand<T, DP> q, g;
    q.template load<READS>(read.of(saved.query, b), call.extent, quarter);
    g.template load<READS>(read.of(saved.output_gradient, b), call.extent, quarter);
    T base[4], over[4], delta[4];
    int32_t token[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const uint32_t j = Mma<T>::row_of(v, quarter);
      const Place place = place_of(j);
      base[v] = saved.of(kBase, call, place.at);
      over[v] = saved.of(kOver, call, place.at);
      delta[v] = saved.of(kDelta, call, place.at);
      token[v] = row0 + j < end_row ? work.first + static_cast<int32_t>(place.t) : -1;
    }
    typename Mma<T>::Acc s{0, 0, 0, 0}, dp{0, 0, 0, 0};
#pragma unroll
    for (int step = 0; step < DP / 4; ++step) {
      s = Mma<T>::step(q.value[step], k.value[step], s);
      dp = Mma<T>::step(g.value[step], x.value[step], dp);
    }
    T p[4], ds[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const bool visible = call.sees(token[v], own);
      p[v] = exp2_of(s[v] * saved.rest - base[v]) * over[v];
      ds[v] = p[v] * (dp[v] - delta[v]);
      p[v] = visible ? p[v] : T(0);
      ds[v] = visible ? ds[v] : T(0);
    }
    AcrossOperand<T, DP> across;
    across.template load<READS>(call.extent, quarter, column, [&](int n) {
      return place_of(n).of(saved.output_gradient, b);
    });
    across.add_to(dv, p);
    across.template load<READS>(call.extent, quarter, column,
                                [&](int n) { return place_of(n).of(saved.query, b); });
    across.add_to(dk, ds);
  }

  const auto join = [&](const Along<T, DP>& sum, bool keys, T factor) {
    sum.visit(quarter, [&](uint32_t d, auto& run) {
      for (auto& y : run) sums[wave][column][d++] = y;
    });
    __syncthreads();
    constexpr int kPieces = DP / W;
    for (int at = threadIdx.x; at < kBlock * kPieces; at += kThreads) {
      const int c = at / kPieces, d = at % kPieces * W;
      if (work.begin_key + c >= work.end_key(call)) continue;
      T run[W];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        run[j] = sums[0][c][d + j];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) run[j] += sums[w][c][d + j];
        run[j] *= factor;
      }
      T *dk_target, *dv_target;
      work.targets(call, splits, key_gradient, value_gradient, c, work.begin_key + c, dk_target,
                   dv_target);
      store_piece(keys ? dk_target : dv_target, d, call.extent, run);
    }
    __syncthreads();
  };
  join(dk, true, static_cast<T>(call.scale));
  join(dv, false, T(1));
}

// dk and dv of the first `keys` keys from their parts in a fixed order, of a launch's
// elements from `first` on: eight lanes to an element take every eighth part each, and
// their sums meet in a tree (4 to 7 us).
constexpr uint32_t kJoinRuns = 8;
constexpr uint64_t kJoinGroups = uint64_t{1} << 22;  // of a launch

template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(Call call, Heads<T> key_gradient,
                                                        Heads<T> value_gradient,
                                                        Splits<T> splits, uint32_t keys,
                                                        uint64_t first) {
  constexpr uint32_t kRuns = kJoinRuns, kLanes = kThreads / kRuns;
  __shared__ T sums[2][kRuns][kLanes];
  const uint32_t lane = threadIdx.x % kLanes, run = threadIdx.x / kLanes;
  const uint64_t per_head = static_cast<uint64_t>(keys) * call.extent;
  const uint64_t at = first + static_cast<uint64_t>(blockIdx.x) * kLanes + lane;
  const bool inside = at < per_head * call.batch_heads;
  const uint32_t batch_head = inside ? static_cast<uint32_t>(at / per_head) : 0;
  const uint64_t within = inside ? at - batch_head * per_head : 0;  // may pass 32 bits
  const uint32_t key = static_cast<uint32_t>(within / call.extent);
  const uint32_t d = static_cast<uint32_t>(within - static_cast<uint64_t>(key) * call.extent);
  const uint32_t b = batch_head / call.key_heads, key_head = batch_head % call.key_heads;
  const bool spread = splits.tile_keys == kBlock;
  const uint32_t tile = spread ? key / kBlock : key / kKeyTile;
  const uint32_t at_key = spread ? key % kBlock : key % kKeyTile;
  const uint64_t row = static_cast<uint64_t>(call.extent);
  const uint64_t value_part = splits.tile_keys * row;
  T* dk = key_gradient.data + b * key_gradient.batch + key_head * key_gradient.head +
          key * key_gradient.token + d;
  T* dv = value_gradient.data + b * value_gradient.batch + key_head * value_gradient.head +
          key * value_gradient.token + d;
  T sum_k = T(0), sum_v = T(0);
  if (splits.main > 1) {
    const T* from = splits.main_part(batch_head, tile, 0) + at_key * row + d;
#pragma unroll 4
    for (uint32_t s = run; s < splits.main; s += kRuns) {
      sum_k += from[s * splits.size()];
      sum_v += from[s * splits.size() + value_part];
    }
  } else if (run == 0 && inside) {
    sum_k = *dk;
    sum_v = *dv;
  }
  if (splits.later != 0 && key < static_cast<uint32_t>(call.sinks)) {
    // key_kernel's waves that take turns leave a part each.
    const int blocks =
        spread ? kWaves : sink_blocks(call.sinks - static_cast<int32_t>(tile * kKeyTile));
    const uint32_t turns = kWaves / blocks;
    const T* from =
        splits.later_part(call.batch_heads, batch_head, tile, 0) + at_key * row + d;
#pragma unroll 4
    for (uint32_t s = run; s < splits.later * turns; s += kRuns) {
      const uint64_t part = s / turns * splits.size() + s % turns * blocks * kBlock * row;
      sum_k += from[part];
      sum_v += from[part + value_part];
    }
  }
  sums[0][run][lane] = sum_k;
  sums[1][run][lane] = sum_v;
  for (uint32_t half = kRuns / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (run < half) {
      sums[0][run][lane] += sums[0][run + half][lane];
      sums[1][run][lane] += sums[1][run + half][lane];
    }
  }
  if (run == 0 && inside) {
    *dk = sums[0][0][lane];
    *dv = sums[1][0][lane];
  }
}

// ---------------------------------------------------------------- launchers

struct Plan {
  bool spread;      // query_spread_kernel
  uint32_t query_splits;
  bool key_spread;  // key_spread_kernel
  uint32_t tile_keys;
  uint32_t row_tiles, key_tiles, main, sink_tiles, later;
  uint64_t rows;             // batch * query heads * queries
  uint64_t statistic_bytes;  // a multiple of 16
  uint64_t bytes;
};

// Splits of the rows behind a sink tile's window: each of this part of the rows that a
// tile of keys has in its window, at most so many, and no more in all than keep the
// chip busy several times over (their parts take memory).
constexpr uint64_t kLaterShare = 2;
constexpr uint64_t kMostLater = 256;
constexpr uint64_t kMostLaterGroups = 2000;
// Workgroups that fill the chip, and the fewest rows that repay a part of either kernel:
// two parts of 256 rows of key_spread_kernel (8 heads of 128) 15 + 9 us against 20 us
// for one, of 348 float64 rows (heads of 72) 28 + 7 us against 38.
constexpr uint64_t kFullGrid = 512;
constexpr uint64_t kFewestRows = 64;
constexpr uint64_t kFewestSpreadRows = 160;
// Keys that repay a part of query_spread_kernel: 2 heads of 64 with 634 queries of 3057
// keys 67 us in one part, 27 + 5 in six; 4 heads of 128 that share a key head with 1024
// tokens 49 and 38 + 5 in two; 2 heads of 64 that see 516 keys 19 and 19 + 4 in two.
constexpr uint64_t kFewestQueryKeys = 384;
// key_spread_kernel is for tiles of 16 keys whose rows are at most so many for each tile:
// more rows want the rows shared in LDS and more parts.  Kernel and join, key_kernel's
// first: 48 heads of 64 with 128 tokens 24 and 10 us; 16 heads of 64 with 512 tokens and
// a window of 128 35 and 21 us; 8 heads of 64 with 1472 tokens 101 and 81 us; 2 key
// heads, each for 4 heads of 128, with 1024 keys and 256 tokens 42 and 46 us; 8 such key
// heads with 512 tokens 81 and 103 us.
constexpr uint64_t kMostSpreadRows = 4;

Plan plan_of(const SparHipAttention& a) {
  Plan plan{};
  const uint64_t element = a.dtype == SPAR_HIP_FLOAT32 ? sizeof(float) : sizeof(double);
  const uint64_t group = a.query_heads / a.key_heads;
  const uint64_t batch_heads = a.batch * a.key_heads;
  plan.row_tiles = ceil_div_u32(a.queries * group, kWaves * kBlock);
  plan.spread = spreads(plan.row_tiles * batch_heads);
  plan.query_splits = 1;
  if (plan.spread) {
    plan.row_tiles = ceil_div_u32(a.queries * group, kBlock);
    plan.query_splits = static_cast<uint32_t>(std::max<uint64_t>(
        1, std::min(kFullGrid / std::max<uint64_t>(1, plan.row_tiles * batch_heads),
                    most_seen(a) / kFewestQueryKeys)));
  }
  const auto rows_of = [&](uint64_t tile_keys) {  // that see a tile through the window
    return group * (a.window == 0 ? a.queries : std::min(a.queries, a.window + tile_keys));
  };
  plan.key_spread = spreads(ceil_div_u32(a.keys, kKeyTile) * batch_heads) &&
                    rows_of(kBlock) <=
                        kMostSpreadRows * ceil_div_u32(a.keys, kBlock) * batch_heads &&
                    a.extent * element <= kMostSpreadBytes;
  plan.tile_keys = plan.key_spread ? kBlock : kKeyTile;
  plan.key_tiles = ceil_div_u32(a.keys, plan.tile_keys);
  plan.main = 1;
  plan.rows = a.batch * a.query_heads * a.queries;
  plan.statistic_bytes = (kStatistics * plan.rows * element + 15) / 16 * 16;
  const uint64_t fewest = plan.key_spread ? kFewestSpreadRows : kFewestRows;
  if (plan.key_tiles != 0) {
    plan.main = static_cast<uint32_t>(
        std::max<uint64_t>(1, std::min(kFullGrid / (plan.key_tiles * batch_heads),
                                       rows_of(plan.tile_keys) / fewest)));
  }
  const uint64_t sinks = std::min(a.sinks, a.keys);
  if (a.window != 0 && sinks != 0 && a.keys > a.window) {
    plan.sink_tiles = ceil_div_u32(sinks, plan.tile_keys);
    const uint64_t behind = std::min(a.queries, a.keys - a.window);
    const uint64_t share = (a.window + plan.tile_keys) / kLaterShare;
    plan.later = static_cast<uint32_t>(std::min(
        kMostLater, std::max((behind + share - 1) / share,
                             std::min<uint64_t>(plan.main, behind * group / fewest))));
    plan.later = static_cast<uint32_t>(std::min<uint64_t>(
        plan.later,
        std::max<uint64_t>(1, kMostLaterGroups / std::max<uint64_t>(
                                                     1, plan.sink_tiles * batch_heads))));
  }
  const uint64_t parts = (plan.main > 1 ? uint64_t{plan.key_tiles} * plan.main : 0) +
                         uint64_t{plan.sink_tiles} * plan.later;
  // The parts of dq and those of dk and dv take turns in one place.
  const uint64_t query_parts =
      plan.query_splits > 1 ? plan.query_splits * plan.rows * (a.extent + 2) : 0;
  plan.bytes = plan.statistic_bytes +
               std::max(batch_heads * parts * 2 * plan.tile_keys * a.extent, query_parts) * element;
  return plan;
}

// scale * log2(e) as a power of two and a rest in [1, 2).
template <typename T>
void split_scale(double scale, T& power, T& rest) {
  const T whole = static_cast<T>(scale * kLog2E);
  power = whole;
  rest = T(1);
  if (whole == T(0) || !__builtin_isfinite(whole)) return;
  int exponent;
  rest = 2 * std::frexp(whole, &exponent);
  power = std::ldexp(T(1), exponent - 1);
}

template <typename T>
void start(const SparHipAttention& a, const Plan& plan, const SparHipHeads& query_gradient,
           const SparHipHeads& key_gradient, const SparHipHeads& value_gradient,
           const SparHipHeads& output_gradient, const SparHipHeads& output,
           const SparHipHeads& query, const SparHipHeads& key, const SparHipHeads& value,
           void* workspace, hipStream_t stream) {
  const Call call = call_of(a);
  Saved<T> saved{heads_of<const T>(query), heads_of<const T>(key), heads_of<const T>(value),
                 heads_of<const T>(output), heads_of<const T>(output_gradient),
                 static_cast<T*>(workspace), T(0), T(0)};
  split_scale(a.scale, saved.power, saved.rest);
  const Heads<T> dk = heads_of<T>(key_gradient), dv = heads_of<T>(value_gradient);
  const Splits<T> splits{
      reinterpret_cast<T*>(static_cast<char*>(workspace) + plan.statistic_bytes),
      plan.tile_keys,
      plan.key_tiles, plan.main, plan.sink_tiles, plan.later, call.extent};
  T* const query_tops = splits.parts + plan.query_splits * plan.rows * a.extent;
  const QueryParts<T> query_parts{splits.parts, query_tops,
                                  query_tops + plan.query_splits * plan.rows, plan.query_splits};
  const uint32_t key_groups = plan.key_tiles * plan.main + plan.sink_tiles * plan.later;
  with_width<T>(a, {&output_gradient, &output, &query, &key, &value},
                [&](auto width, auto reads) {
    constexpr int DP = decltype(width)::value;
    constexpr Reads READS = decltype(reads)::value;
    constexpr int kBlocks = tile_blocks<T, DP>();
    constexpr int kKeyBlocks = sizeof(T) == 4 && DP <= 128 ? 2 : 1;
    if (call.rows != 0 && plan.spread) {
      // It reads pieces at any address alike.
      constexpr Reads kReads = READS == Reads::Aligned ? Reads::Pieces : READS;
      query_spread_kernel<T, DP, kReads>
          <<<plan.row_tiles * call.batch_heads * plan.query_splits, kThreads, 0, stream>>>(
              call, saved, heads_of<T>(query_gradient), plan.row_tiles, query_parts);
      if (plan.query_splits > 1) {
        query_join_kernel<T>
            <<<ceil_div_u32(call.all_rows() * call.extent, kThreads), kThreads, 0, stream>>>(
                call, saved, heads_of<T>(query_gradient), query_parts);
      }
    } else if (call.rows != 0) {
      query_kernel<T, DP, kBlocks, READS>
          <<<plan.row_tiles * call.batch_heads, kThreads, 0, stream>>>(
              call, saved, heads_of<T>(query_gradient), plan.row_tiles);
    }
    if (call.keys != 0 && plan.key_spread) {
      if constexpr (DP * sizeof(T) <= kMostSpreadBytes) {
        constexpr Reads kReads = READS == Reads::Aligned ? Reads::Pieces : READS;
        key_spread_kernel<T, DP, kReads>
            <<<key_groups * call.batch_heads, kThreads, 0, stream>>>(call, saved, dk, dv, splits);
      }
    } else if (call.keys != 0) {
      key_kernel<T, DP, kKeyBlocks, READS>
          <<<key_groups * call.batch_heads, kThreads, 0, stream>>>(call, saved, dk, dv, splits);
    }
  });
  const uint32_t joined = plan.main > 1     ? call.keys
                          : plan.later != 0 ? static_cast<uint32_t>(std::min(a.sinks, a.keys))
                                            : 0;
  const uint64_t elements = static_cast<uint64_t>(call.batch_heads) * joined * a.extent;
  constexpr uint64_t kLaunch = kJoinGroups * (kThreads / kJoinRuns);
  for (uint64_t at = 0; at < elements; at += kLaunch) {
    join_kernel<T><<<ceil_div_u32(std::min(kLaunch, elements - at), kThreads / kJoinRuns),
                     kThreads, 0, stream>>>(call, dk, dv, splits, joined, at);
  }
}

bool fits(const SparHipAttention& a, const Plan& plan) {
  const uint64_t batch_heads = a.batch * a.key_heads;
  return (static_cast<uint64_t>(plan.key_tiles) * plan.main +
          static_cast<uint64_t>(plan.sink_tiles) * plan.later) * batch_heads <= kMostGroups &&
         static_cast<uint64_t>(plan.row_tiles) * batch_heads * plan.query_splits <= kMostGroups;
}

}  // namespace

uint64_t forward_workspace(const SparHipAttention& a);  // attention_forward.hip

}  // namespace attention
}  // namespace spar_hip

using namespace spar_hip;

extern "C" SparHipStatus spar_hip_attention_workspace(uint64_t* bytes,
                                                      const SparHipAttention* attention,
                                                      int backward) {
  if (bytes == nullptr || backward < 0 || backward > 1 || !attention::valid(attention)) {
    return invalid();
  }
  *bytes = 0;
  if (attention->batch == 0 || attention->query_heads == 0) return ok();
  if (backward != 0) {
    *bytes = attention::plan_of(*attention).bytes;
  } else if (attention->queries != 0) {
    *bytes = attention::forward_workspace(*attention);
  }
  return ok();
}

extern "C" SparHipStatus spar_hip_launch_attention_backward(
    const SparHipHeads* query_gradient, const SparHipHeads* key_gradient,
    const SparHipHeads* value_gradient, const SparHipHeads* output_gradient,
    const SparHipHeads* output, const void* logsumexp, const SparHipHeads* query,
    const SparHipHeads* key, const SparHipHeads* value, const SparHipAttention* attention,
    void* workspace, uint64_t workspace_bytes, int device) {
  if (!attention::valid(attention)) return invalid();
  const SparHipAttention& a = *attention;
  if (a.batch == 0 || a.query_heads == 0 || (a.queries == 0 && a.keys == 0)) return ok();
  for (const SparHipHeads* heads :
       {query_gradient, key_gradient, value_gradient, output_gradient, output, query, key, value}) {
    if (heads == nullptr) return invalid();
  }
  if (a.queries != 0 &&
      (query_gradient->data == nullptr || output_gradient->data == nullptr ||
       output->data == nullptr || query->data == nullptr || logsumexp == nullptr)) {
    return invalid();
  }
  if (a.keys != 0 && (key_gradient->data == nullptr || value_gradient->data == nullptr ||
                      key->data == nullptr || value->data == nullptr)) {
    return invalid();
  }
  const attention::Plan plan = attention::plan_of(a);
  if (!attention::fits(a, plan) ||
      (plan.bytes != 0 &&
       (workspace == nullptr || workspace_bytes < plan.bytes || !aligned16(workspace)))) {
    return invalid();
  }
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  if (a.dtype == SPAR_HIP_FLOAT32) {
    attention::start<float>(a, plan, *query_gradient, *key_gradient, *value_gradient,
                            *output_gradient, *output, *query, *key, *value, workspace,
                            guard.stream);
  } else {
    attention::start<double>(a, plan, *query_gradient, *key_gradient, *value_gradient,
                             *output_gradient, *output, *query, *key, *value, workspace,
                             guard.stream);
  }
  return finish(guard);
}

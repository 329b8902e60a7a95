// Attention forward: o = softmax(scale q k^T over the visible keys) v in one pass
// over the keys, with the running maximum and sum of the softmax per row.
//
// Scores are formed transposed, S^T = K Q^T, and so is the output, O^T = V^T P^T:
// a lane then holds scores of one row only (its column), the row's maximum and sum
// stay in that lane, the exponentials of S^T are the second product's operand as
// they lie, and rescaling O takes no exchange between lanes (attention.hpp).
// Scores carry scale * log2(e), folded into q, so that weights are powers of two.
//
// Two kernels.  tile_kernel: a workgroup of four waves with 16 rows each
// shares tiles of keys and values in LDS; bound by the matrix units (4 extent
// operations per visible pair).  token_kernel, for up to kTokenRows rows (a token
// or a few per sequence) and where tiles would leave the chip idle: a workgroup's
// waves take different keys of the same 16 rows straight from memory into registers;
// bound by reading the visible cache.
// Either splits the keys of a row tile over several workgroups where the rows alone
// do not fill the chip; combine_kernel joins the parts in their order.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention_join.hpp"

namespace spar_hip {
namespace attention {
namespace {

// Writes a finished row: `sum` is its whole total.
template <typename T, int DP>
__device__ __forceinline__ void write_row(const Call& call, const Results<T>& results, uint32_t b,
                                          uint32_t key_head, uint32_t r, uint32_t split, T top,
                                          T sum, const Along<T, DP>& out, int quarter) {
  if (r >= call.rows) return;
  const uint32_t t = call.group.div(r);
  const uint32_t head = key_head * call.group.divisor + (r - t * call.group.divisor);
  const T over = sum == T(0) ? T(0) : T(1) / sum;
  const uint64_t row =
      (static_cast<uint64_t>(b) * call.key_heads * call.group.divisor + head) * call.queries + t;
  T* target;
  if (results.splits == 1) {
    target = results.output.data + b * results.output.batch + head * results.output.head +
             t * results.output.token;
    if (quarter == 0 && results.logsumexp != nullptr) {
      results.logsumexp[row] = logsumexp_of(top, sum);
    }
  } else {
    const uint64_t at = split * results.all_rows + row;
    target = results.part_output + at * results.pitch;
    if (quarter == 0) {
      results.part_top[at] = top;
      results.part_total[at] = sum;
    }
  }
  out.visit(quarter, [&](uint32_t d, auto& run) {
    for (auto& x : run) x *= over;
    store_piece(target, d, call.extent, run);
  });
}

// The head of row r, of some row where r is behind the last.
template <typename T>
__device__ __forceinline__ const T* head_row(const Heads<const T>& heads, const Call& call,
                                             uint32_t b, uint32_t key_head, uint32_t r) {
  r = r < call.rows ? r : call.rows - 1;
  const uint32_t t = call.group.div(r);
  const uint32_t head = key_head * call.group.divisor + (r - t * call.group.divisor);
  return heads.data + b * heads.batch + head * heads.head + t * heads.token;
}

// Workgroups of one key head follow each other at a distance of batch * key heads,
// a multiple of the 8 dies in common sizes, so that they share a die's cache; the
// last rows, which see most, come first.  A wave passes over blocks of 16 keys that none
// of its rows sees, and forms masks only for those that an edge of the window, of the
// sinks or of the diagonal cuts.  The matrix units are busy in 87% of the CUs'
// cycles at heads of 128: 32 of them with 8192 tokens, window 1024 and 4 sinks in 1.02 ms,
// 127 TFLOP/s of visible pairs; in 68% at heads of 64, 256 of them with 1024 tokens and
// window 256 in 163 us, 94 TFLOP/s, where cut blocks are a tenth of the work and the
// vector instructions, some 57 a block, weigh twice as much.
template <typename T, int DP, int KB, Reads READS>
__global__ __launch_bounds__(kThreads, (tile_waves<T, DP>())) void tile_kernel(
    Call call, Results<T> results, Heads<const T> query, Heads<const T> key, Heads<const T> value,
    uint32_t row_tiles) {
  constexpr int KT = KB * kBlock;
  constexpr int W = Vec16<T>::width;
  constexpr uint32_t kRows = kWaves * kBlock;
  __shared__ Tile<T, KT, DP, READS> keys, values;
  const uint32_t batch_head = blockIdx.x % call.batch_heads;
  const uint32_t rest = blockIdx.x / call.batch_heads;
  const uint32_t split = rest % results.splits;
  const uint32_t row_tile = row_tiles - 1 - rest / results.splits;
  const uint32_t b = batch_head / call.key_heads, key_head = batch_head % call.key_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const Lane<T, DP> lane(threadIdx.x % kWave);

  const int32_t first = call.length(b) - call.queries;  // token of query 0
  const uint32_t begin_row = row_tile * kRows;
  const uint32_t end_row = begin_row + kRows < call.rows ? begin_row + kRows : call.rows;
  const int32_t low_token = call.token(begin_row, first);
  const Keys seen(call, low_token < 0 ? 0 : low_token, call.token(end_row - 1, first));
  const uint32_t tiles = seen.tiles(KT);
  const uint32_t begin_tile =
      static_cast<uint32_t>(static_cast<uint64_t>(tiles) * split / results.splits);
  const uint32_t end_tile =
      static_cast<uint32_t>(static_cast<uint64_t>(tiles) * (split + 1) / results.splits);
  const T* key_base = key.data + b * key.batch + key_head * key.head;
  const T* value_base = value.data + b * value.batch + key_head * value.head;
  // Rows of a tile behind its run repeat the tile's first key; no row sees them.
  typename Tile<T, KT, DP, READS>::Stage next_keys, next_values;
  keys.prepare(next_keys, call.extent, [&](uint32_t j) { return j * key.token; });
  values.prepare(next_values, call.extent, [&](uint32_t j) { return j * value.token; });
  const auto start = [&](uint32_t i) {
    int32_t begin, end;
    seen.tile(i, KT, begin, end);
    const uint64_t rows = end - begin;
    const auto at = [&](uint64_t j) { return j < rows ? j : 0; };
    keys.start(next_keys, i % 2, key_base + begin * key.token, rows >= KT, call.extent,
               [&](uint32_t j) { return at(j) * key.token; });
    values.start(next_values, i % 2, value_base + begin * value.token, rows >= KT,
                 call.extent, [&](uint32_t j) { return at(j) * value.token; });
  };
  const auto finish = [&](uint32_t i) {
    keys.finish(next_keys, i % 2);
    values.finish(next_values, i % 2);
  };
  if (begin_tile < end_tile) start(begin_tile);

  // This wave's rows and their tokens: all of them in the wave between `oldest`
  // and `newest`.
  const uint32_t wave_row = begin_row + wave * kBlock;
  const uint32_t wave_end =
      wave_row + kBlock < call.rows ? wave_row + kBlock : call.rows;
  const int32_t oldest = call.token(wave_row, first);
  const int32_t newest = wave_row < wave_end ? call.token(wave_end - 1, first) : -1;
  const uint32_t r = wave_row + lane.column;
  const int32_t token = call.token(r, first);
  Operand<T, DP> q;
  q.template load<READS>(head_row(query, call, b, key_head, r), call.extent, lane.quarter);
  q.finish(token >= 0, call.extent, lane.quarter, static_cast<T>(call.scale * kLog2E));
  Row<T, DP> row;
  row.out.clear();
  if (begin_tile < end_tile) finish(begin_tile);

  for (uint32_t i = begin_tile; i < end_tile; ++i) {
    int32_t begin, end;
    seen.tile(i, KT, begin, end);
    __syncthreads();
    if (i + 1 < end_tile) start(i + 1);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int32_t k0 = begin + kb * kBlock, k1 = k0 + kBlock - 1;
      const bool any = k0 < end && k0 <= newest &&
                       ((oldest < 0 ? 0 : oldest) - k1 < call.window || k0 < call.sinks);
      if (!any) continue;
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
      const bool whole = k1 <= oldest && k1 < end &&
                         (newest - k0 < call.window || k1 < call.sinks);
      T score[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) score[v] = s[v];
      if (!whole) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int32_t at = k0 + Mma<T>::row_of(v, lane.quarter);
          const bool visible = (at < end) & call.sees(token, at);
          score[v] = visible ? score[v] : lowest<T>();
        }
      }
      row.take(score);
      across.run(row.out, score);
    }
    if (i + 1 < end_tile) finish(i + 1);
  }
  write_row(call, results, b, key_head, r, split, row.base, quarter_sum(row.total), row.out,
            lane.quarter);
}

// Four waves with the same 16 rows and every fourth block of 16 keys, read into
// the operands' layout from memory; at the end the waves' rows meet in LDS.  Nothing is
// shared between waves before that, so no wave waits for another.  Bound by reading the
// cache: 4 sequences of about 50000 tokens in 8 key heads of 128 in 340 us, 5.5 TB/s;
// 16 sequences with a window of 1024 in 4 key heads of 64 in 10.4 us, 3.3 TB/s, where the
// launch, a few blocks per wave and their latency show (16 waves a workgroup without
// splits and their join: 17.7 us against 10.4 + 3).
template <typename T, int DP, Reads READS>
__global__ __launch_bounds__(kThreads) void token_kernel(Call call, Results<T> results,
                                                         Heads<const T> query, Heads<const T> key,
                                                         Heads<const T> value,
                                                         uint32_t row_tiles) {
  constexpr int W = Vec16<T>::width;
  constexpr int kPitch = DP + W;
  __shared__ T outs[kWaves][kBlock][kPitch];
  __shared__ T tops[kWaves][kBlock], totals[kWaves][kBlock];
  const uint32_t batch_head = blockIdx.x % call.batch_heads;
  const uint32_t rest = blockIdx.x / call.batch_heads;
  const uint32_t split = rest % results.splits;
  const uint32_t row_tile = row_tiles - 1 - rest / results.splits;
  const uint32_t b = batch_head / call.key_heads, key_head = batch_head % call.key_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int lane = threadIdx.x % kWave;
  const int quarter = lane / kBlock, column = lane % kBlock;

  const int32_t first = call.length(b) - call.queries;
  const uint32_t begin_row = row_tile * kBlock;
  const uint32_t end_row = begin_row + kBlock < call.rows ? begin_row + kBlock : call.rows;
  const int32_t oldest = call.token(begin_row, first);
  const int32_t newest = call.token(end_row - 1, first);
  const Keys seen(call, oldest < 0 ? 0 : oldest, newest);
  const uint32_t blocks = seen.tiles(kBlock);
  const uint32_t begin_block =
      static_cast<uint32_t>(static_cast<uint64_t>(blocks) * split / results.splits);
  const uint32_t end_block =
      static_cast<uint32_t>(static_cast<uint64_t>(blocks) * (split + 1) / results.splits);

  const uint32_t r = begin_row + column;
  const int32_t token = call.token(r, first);
  Operand<T, DP> q;
  q.template load<READS>(head_row(query, call, b, key_head, r), call.extent, quarter);
  q.finish(token >= 0, call.extent, quarter, static_cast<T>(call.scale * kLog2E));
  Row<T, DP> row;
  row.out.clear();
  const T* key_base = key.data + b * key.batch + key_head * key.head;
  const T* value_base = value.data + b * value.batch + key_head * value.head;

  for (uint32_t i = begin_block + wave; i < end_block; i += kWaves) {
    int32_t begin, end;
    seen.tile(i, kBlock, begin, end);
    // Keys behind the run repeat its block's first; no row sees them.
    const auto at_key = [&](int32_t k) { return static_cast<uint64_t>(k < end ? k : begin); };
    Operand<T, DP> k;
    k.template load<READS>(key_base + at_key(begin + column) * key.token, call.extent, quarter);
    AcrossOperand<T, DP> v;
    v.template load<READS>(call.extent, quarter, column, [&](int n) {
      return value_base + at_key(begin + n) * value.token;
    });
    typename Mma<T>::Acc s{0, 0, 0, 0};
#pragma unroll
    for (int step = 0; step < DP / 4; ++step) {
      s = Mma<T>::step(k.value[step], q.value[step], s);
    }
    const int32_t last = begin + kBlock - 1;
    const bool whole = last <= oldest && last < end &&
                       (newest - begin < call.window || last < call.sinks);
    T score[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int32_t at = begin + Mma<T>::row_of(n, quarter);
      const bool visible = whole | ((at < end) & call.sees(token, at));
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
    if (out_row >= call.rows) continue;
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
      for (int j = 0; j < W; ++j) run[j] += outs[w][c][d + j] * shrink;
    }
    const T over = sum == T(0) ? T(0) : T(1) / sum;
#pragma unroll
    for (int j = 0; j < W; ++j) run[j] *= over;
    const uint32_t t = call.group.div(out_row);
    const uint32_t head = key_head * call.group.divisor + (out_row - t * call.group.divisor);
    const uint64_t place =
        (static_cast<uint64_t>(b) * call.key_heads * call.group.divisor + head) * call.queries + t;
    T* target;
    if (results.splits == 1) {
      target = results.output.data + b * results.output.batch + head * results.output.head +
               t * results.output.token;
      if (d == 0 && results.logsumexp != nullptr) {
        results.logsumexp[place] = logsumexp_of(top, sum);
      }
    } else {
      const uint64_t part = split * results.all_rows + place;
      target = results.part_output + part * results.pitch;
      if (d == 0) {
        results.part_top[part] = top;
        results.part_total[part] = sum;
      }
    }
    store_piece(target, d, call.extent, run);
  }
}

// ---------------------------------------------------------------- launchers

// Up to this many rows per key head the waves share rows and split keys: a tile
// of 64 rows would leave half of its matrix work unused.
constexpr uint64_t kTokenRows = 32;

// Workgroups that row tiles are split up to, and the fewest keys that repay the writing
// and reading of a part: three tiles and four tokens to each of the 256 CUs.  (Of
// token_kernel a CU holds as many in float32 up to heads of 64, three at 96, two at 128
// and one above, and the others wait for them to end.)
constexpr uint64_t kFullGrid = 768;
constexpr uint64_t kTokenGrid = 1024;
constexpr uint64_t kFewestKeys = 256;
constexpr uint64_t kFewestTokenKeys = 128;

// Keys of a token that one workgroup takes in less time than splits and their join:
// 64 heads of 64 with 256 keys 6.9 us against 6.2 + 3.9, with 384 keys 6.4 + 4.2 us.
constexpr uint64_t kUnsplitKeys = 320;

struct Plan {
  bool token;
  uint32_t row_tiles;
  uint32_t splits;
  uint32_t pitch;
  uint64_t rows;       // batch * query heads * queries
  uint64_t bytes;
};

uint64_t element_size(const SparHipAttention& a) {
  return a.dtype == SPAR_HIP_FLOAT32 ? sizeof(float) : sizeof(double);
}

Plan plan_of(const SparHipAttention& a) {
  Plan plan{};
  const uint64_t rows = a.queries * (a.query_heads / a.key_heads);
  const uint64_t batch_heads = a.batch * a.key_heads;
  plan.rows = a.batch * a.query_heads * a.queries;
  plan.token = rows <= kTokenRows ||
               spreads((rows + kWaves * kBlock - 1) / (kWaves * kBlock) * batch_heads *
                       std::max<uint64_t>(1, most_seen(a) / kFewestKeys));
  uint64_t grid = kTokenGrid;
  uint64_t seen = most_seen(a);
  if (plan.token) {
    plan.row_tiles = ceil_div_u32(rows, kBlock);
  } else {
    constexpr uint64_t kRows = kWaves * kBlock;
    plan.row_tiles = ceil_div_u32(rows, kRows);
    grid = kFullGrid;
    seen = std::min(a.keys, seen + kRows / (a.query_heads / a.key_heads));
  }
  uint64_t wanted = grid / std::max<uint64_t>(1, plan.row_tiles * batch_heads);
  if (plan.token && seen <= kUnsplitKeys) wanted = 1;
  plan.splits = static_cast<uint32_t>(
      std::max<uint64_t>(1, std::min({wanted, seen / (plan.token ? kFewestTokenKeys : kFewestKeys),
                                          uint64_t{kMostParts}})));
  const uint64_t piece = 16 / element_size(a);
  plan.pitch = static_cast<uint32_t>((a.extent + piece - 1) / piece * piece);
  if (plan.splits > 1) {
    plan.bytes = plan.splits * plan.rows * (plan.pitch + 2) * element_size(a);
  }
  return plan;
}

template <typename T>
void start(const SparHipAttention& a, const Plan& plan, const SparHipHeads& output,
           void* logsumexp, const SparHipHeads& query, const SparHipHeads& key,
           const SparHipHeads& value, void* workspace, hipStream_t stream) {
  const Call call = call_of(a);
  Results<T> results{heads_of<T>(output), static_cast<T*>(logsumexp), nullptr, nullptr, nullptr,
                     plan.splits, plan.pitch, plan.rows};
  if (plan.splits > 1) {
    results.part_output = static_cast<T*>(workspace);
    results.part_top = results.part_output + plan.splits * plan.rows * plan.pitch;
    results.part_total = results.part_top + plan.splits * plan.rows;
  }
  const uint32_t grid = plan.row_tiles * call.batch_heads * plan.splits;
  const auto q = heads_of<const T>(query), k = heads_of<const T>(key),
             v = heads_of<const T>(value);
  with_width<T>(a, {&query, &key, &value}, [&](auto width, auto reads) {
    constexpr int DP = decltype(width)::value;
    constexpr Reads READS = decltype(reads)::value;
    if (plan.token) {
      // It reads pieces at any address alike.
      constexpr Reads kReads = READS == Reads::Aligned ? Reads::Pieces : READS;
      token_kernel<T, DP, kReads>
          <<<grid, kThreads, 0, stream>>>(call, results, q, k, v, plan.row_tiles);
      return;
    }
    tile_kernel<T, DP, tile_blocks<T, DP>(), READS>
        <<<grid, kThreads, 0, stream>>>(call, results, q, k, v, plan.row_tiles);
  });
  if (plan.splits > 1) join_parts<T, false>(call, results, stream);
}

}  // namespace

uint64_t forward_workspace(const SparHipAttention& a) { return plan_of(a).bytes; }

}  // namespace attention
}  // namespace spar_hip

using namespace spar_hip;

extern "C" SparHipStatus spar_hip_launch_attention_forward(
    const SparHipHeads* output, void* logsumexp, const SparHipHeads* query,
    const SparHipHeads* key, const SparHipHeads* value, const SparHipAttention* attention,
    void* workspace, uint64_t workspace_bytes, int device) {
  if (!attention::valid(attention)) return invalid();
  const SparHipAttention& a = *attention;
  if (a.batch == 0 || a.query_heads == 0 || a.queries == 0) return ok();
  if (output == nullptr || query == nullptr || key == nullptr || value == nullptr ||
      output->data == nullptr || query->data == nullptr ||
      (a.keys != 0 && (key->data == nullptr || value->data == nullptr))) {
    return invalid();
  }
  const attention::Plan plan = attention::plan_of(a);
  if (static_cast<uint64_t>(plan.row_tiles) * a.batch * a.key_heads * plan.splits >
          attention::kMostGroups ||
      (plan.bytes != 0 &&
       (workspace == nullptr || workspace_bytes < plan.bytes || !aligned16(workspace)))) {
    return invalid();
  }
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  if (a.dtype == SPAR_HIP_FLOAT32) {
    attention::start<float>(a, plan, *output, logsumexp, *query, *key, *value, workspace,
                            guard.stream);
  } else {
    attention::start<double>(a, plan, *output, logsumexp, *query, *key, *value, workspace,
                             guard.stream);
  }
  return finish(guard);
}

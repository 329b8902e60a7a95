// Parts of the rows of an attention whose keys several workgroups share, and the kernels
// that join them.
#pragma once

#include <hip/hip_runtime.h>

#include "attention.hpp"

namespace spar_hip {
namespace attention {
namespace {

// Where results go: the output itself, or one part per split of the keys.
template <typename T>
struct Results {
  Heads<T> output;
  T* logsumexp;
  T* part_output;  // [split][batch][query head][query][pitch]
  T* part_top;     // [split][batch][query head][query]: the row's base
  T* part_total;   // the same: its sum.  Two numbers, since the sum is lost in the
                   // rounding of a large base
  uint32_t splits;
  uint32_t pitch;     // the extent rounded up to whole pieces
  uint64_t all_rows;  // batch * query heads * queries
};

// At most this many parts of a row: one for each thread that joins them.
constexpr uint32_t kMostParts = kThreads;

// ln of a sum of powers of two over a base; no sum where no key is seen.
template <typename T>
__device__ __forceinline__ T logsumexp_of(T top, T sum) {
  return sum == T(0) ? lowest<T>() : (top + log2_of(sum)) * static_cast<T>(kLn2);
}

// The parts of a row: o = sum w o_part / sum w, w = 2^(part's base - largest base) times
// the part's sum.  Few parts: kLanes lanes side by side along a row's head take them in
// their order, all loaded before the first is used (16384 rows of 128 in 3 parts 7.5 us,
// 256 rows of 64 in 8 parts 3 us).
constexpr uint32_t kFewParts = 8;
constexpr uint32_t kFewLanes = 32;

template <typename T>
__device__ __forceinline__ T* output_row(const Call& call, const Results<T>& results,
                                         uint64_t row) {
  const uint64_t batch_head = row / call.queries;
  const uint32_t t = static_cast<uint32_t>(row - batch_head * call.queries);
  const uint32_t heads = call.key_heads * call.group.divisor;
  const uint64_t b = batch_head / heads, head = batch_head % heads;
  return results.output.data + b * results.output.batch + head * results.output.head +
         t * results.output.token;
}

// EMPTY: parts of no weight (a total of 0) hold nothing but that.
template <typename T, bool EMPTY>
__global__ __launch_bounds__(kThreads) void combine_few_kernel(Call call, Results<T> results) {
  constexpr int W = Vec16<T>::width;
  constexpr uint32_t kLanes = kFewLanes;
  const uint64_t row = static_cast<uint64_t>(blockIdx.x) * (kThreads / kLanes) +
                       threadIdx.x / kLanes;
  if (row >= results.all_rows) return;
  // All loads first, of the last part again where there are fewer.
  constexpr int kPieces = SPAR_HIP_ATTENTION_MAX_EXTENT / (kLanes * W);
  const uint32_t lane = threadIdx.x % kLanes;
  T weight[kFewParts], part_total[kFewParts];
  typename Vec16<T>::type piece[kFewParts];
  const auto part_of = [&](uint32_t s) {
    return (s < results.splits ? s : results.splits - 1) * results.all_rows + row;
  };
  const auto load = [&](uint32_t d) {
#pragma unroll
    for (uint32_t s = 0; s < kFewParts; ++s) {
      piece[s] = *reinterpret_cast<const typename Vec16<T>::type*>(
          results.part_output + part_of(s) * results.pitch + (d < call.extent ? d : 0));
    }
  };
#pragma unroll
  for (uint32_t s = 0; s < kFewParts; ++s) {
    weight[s] = results.part_top[part_of(s)];
    part_total[s] = results.part_total[part_of(s)];
  }
  load(lane * W);
  T top = lowest_finite<T>();
#pragma unroll
  for (uint32_t s = 0; s < kFewParts; ++s) {
    top = larger(weight[s], top);
  }
  T sum = T(0);
#pragma unroll
  for (uint32_t s = 0; s < kFewParts; ++s) {
    weight[s] = s < results.splits ? exp2_of(weight[s] - top) * part_total[s] : T(0);
    sum += weight[s];
  }
  const T over = sum == T(0) ? T(0) : T(1) / sum;
  T* target = output_row(call, results, row);
#pragma unroll
  for (int j = 0; j < kPieces; ++j) {
    const uint32_t d = (lane + j * kLanes) * W;
    if (d >= call.extent) break;
    if (j != 0) load(d);
    typename Vec16<T>::type x = {};
#pragma unroll
    for (uint32_t s = 0; s < kFewParts; ++s) {
      if (s < results.splits && !(EMPTY && part_total[s] == T(0))) x += piece[s] * weight[s];
    }
    T run[W];
#pragma unroll
    for (int i = 0; i < W; ++i) run[i] = x[i] * over;
    store_piece(target, d, call.extent, run);
  }
  if (lane == 0 && results.logsumexp != nullptr) {
    results.logsumexp[row] = logsumexp_of(top, sum);
  }
}

// Many parts: a workgroup per row, the parts dealt out to its runs of lanes, whose
// sums meet in a tree (128 rows of 128 in 32 parts 6 us, latency).
template <typename T, bool EMPTY>
__global__ __launch_bounds__(kThreads) void combine_kernel(Call call, Results<T> results) {
  constexpr int W = Vec16<T>::width;
  constexpr uint32_t kLanes = SPAR_HIP_ATTENTION_MAX_EXTENT / W / 2;  // two pieces each
  constexpr uint32_t kRuns = kThreads / kLanes;
  __shared__ T weights[kMostParts];
  __shared__ T totals[EMPTY ? kMostParts : 1];
  __shared__ alignas(16) T outs[kRuns][SPAR_HIP_ATTENTION_MAX_EXTENT];
  __shared__ T waves[kWaves];
  const uint64_t row = blockIdx.x;
  const uint32_t split = threadIdx.x;
  T part_top = lowest_finite<T>(), part_total = T(0);
  if (split < results.splits) {
    part_top = results.part_top[split * results.all_rows + row];
    part_total = results.part_total[split * results.all_rows + row];
  }
  T top = part_top;
#pragma unroll
  for (int mask = kWave / 2; mask > 0; mask >>= 1) {
    top = larger(__shfl_xor(top, mask, kWave), top);
  }
  if (threadIdx.x % kWave == 0) waves[threadIdx.x / kWave] = top;
  __syncthreads();
  top = waves[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = larger(waves[w], top);
  weights[split] = exp2_of(part_top - top) * part_total;
  if constexpr (EMPTY) totals[split] = part_total;
  __syncthreads();
  T sum = T(0);
  for (uint32_t s = 0; s < results.splits; ++s) sum += weights[s];
  const T over = sum == T(0) ? T(0) : T(1) / sum;
  const uint32_t lane = threadIdx.x % kLanes, run = threadIdx.x / kLanes;
  typename Vec16<T>::type x[2] = {};
#pragma unroll 4
  for (uint32_t s = run; s < results.splits; s += kRuns) {
    if (EMPTY && totals[s] == T(0)) continue;
    const T* part = results.part_output + (s * results.all_rows + row) * results.pitch;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t d = (lane + j * kLanes) * W;
      if (d < results.pitch) {
        x[j] += *reinterpret_cast<const typename Vec16<T>::type*>(part + d) * weights[s];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    *reinterpret_cast<typename Vec16<T>::type*>(&outs[run][(lane + j * kLanes) * W]) = x[j];
  }
  for (uint32_t half = kRuns / 2; half > 0; half >>= 1) {
    __syncthreads();
    if (run < half) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t d = (lane + j * kLanes) * W;
        x[j] += *reinterpret_cast<const typename Vec16<T>::type*>(&outs[run + half][d]);
        *reinterpret_cast<typename Vec16<T>::type*>(&outs[run][d]) = x[j];
      }
    }
  }
  __syncthreads();
  T* target = output_row(call, results, row);
  if (threadIdx.x < call.extent) target[threadIdx.x] = outs[0][threadIdx.x] * over;
  if (threadIdx.x == 0 && results.logsumexp != nullptr) {
    results.logsumexp[row] = logsumexp_of(top, sum);
  }
}
static_assert(kThreads >= SPAR_HIP_ATTENTION_MAX_EXTENT);

// Whether a launch counts the workgroups that join so many parts of `rows` rows.  One part
// is the output itself and is not joined.
inline bool joins(uint64_t rows, uint64_t parts) {
  constexpr uint64_t kRows = kThreads / kFewLanes;  // of a workgroup, few parts
  return parts <= 1 || rows <= (parts <= kFewParts ? kMostGroups * kRows : kMostGroups);
}

template <typename T, bool EMPTY>
void join_parts(const Call& call, const Results<T>& results, hipStream_t stream) {
  if (results.splits <= kFewParts) {
    combine_few_kernel<T, EMPTY>
        <<<ceil_div_u32(results.all_rows, kThreads / kFewLanes), kThreads, 0, stream>>>(call,
                                                                                        results);
  } else {
    combine_kernel<T, EMPTY>
        <<<static_cast<uint32_t>(results.all_rows), kThreads, 0, stream>>>(call, results);
  }
}

}  // namespace
}  // namespace attention
}  // namespace spar_hip

// Keys and values of new tokens written to the pages of a cache, the keys turned by their
// positions on the way, and the queries turned in the same launch.
//
// The rotation is that of rotary.hip: pair (x, y) of a token at position p becomes
// (x c - y s, y c + x s), c and s the cosine and sine of p times the pair's frequency.  A lane
// takes a unit of four pairs (or eight elements behind them) of one or several heads of one
// token.  Bound by memory for prompts: every element is read once and written once, [4, 4096]
// tokens of 32 + 2 * 8 heads of 128 in 149 us, 5.4 TB/s, the rate of the rotation alone.
// For single tokens the launch counts, so that queries, keys and values share it: 64 tokens of
// those heads take 5.2 us.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "pages.hpp"
#include "rotary.hpp"

namespace spar_hip {
namespace rotary {
namespace {

template <typename T>
struct Append {
  Pages<T> cache;
  Heads<T> query_output;
  Heads<const T> query, key, value;
  uint32_t query_heads, key_heads;
  uint32_t query_groups, key_groups;  // of K heads a lane
  const void* places;
  uint64_t place_stride;
  bool wide_places;

  // Token of its row that token t of sequence b becomes, less than 0 where none.
  __device__ __forceinline__ int64_t place(uint64_t b, uint64_t t) const {
    const uint64_t at = b * place_stride + t;
    return wide_places ? static_cast<const int64_t*>(places)[at]
                       : static_cast<const int32_t*>(places)[at];
  }
};

// A lane per unit of K heads of one token: the groups of heads count through the queries',
// the keys' and the values'.
template <typename T, bool HALF, bool NT, int K>
__global__ __launch_bounds__(kThreads) void append_kernel(Append<T> append, Turn turn, Rows rows,
                                                          uint32_t items, FastDiv by_units,
                                                          FastDiv by_groups) {
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
  if (item >= items) return;
  const uint32_t group_item = by_units.div(item);
  const Unit unit =
      unit_at<HALF>(item - group_item * by_units.divisor, turn.half, turn.extent);
  const uint32_t row = by_groups.div(group_item);
  uint32_t group = group_item - row * by_groups.divisor;
  uint64_t b, t;
  rows.split(row, b, t);
  const bool query = group < append.query_groups;
  if (!query) group -= append.query_groups;
  const bool value = !query && group >= append.key_groups;
  if (value) group -= append.key_groups;
  const Heads<const T>& from = query ? append.query : value ? append.value : append.key;
  const uint32_t heads = query ? append.query_heads : append.key_heads;
  const uint32_t groups = query ? append.query_groups : append.key_groups;
  const T* source = from.data + b * from.batch + t * from.token;
  T* target;
  uint64_t pitch;  // between the target's heads
  if (query) {
    target = append.query_output.data + b * append.query_output.batch +
             t * append.query_output.token;
    pitch = append.query_output.head;
  } else {
    const int64_t place = append.place(b, t);
    if (place < 0 || place >= append.cache.room) return;
    const uint32_t at = static_cast<uint32_t>(place);
    const uint32_t entry = append.cache.page_tokens.div(at);
    const int32_t page = append.cache.page_at(static_cast<uint32_t>(b), entry);
    if (!append.cache.held(page)) return;
    const PageHeads<T>& to = value ? append.cache.value : append.cache.key;
    target = to.data + static_cast<uint64_t>(page) * to.page +
             (at - entry * append.cache.page_tokens.divisor) * to.token;
    pitch = to.head;
  }
  T x[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t head = group + k * groups;
    if (head < heads) load_unit<T, NT>(x[k], source + head * from.head, unit);
  }
  T c[4], s[4];
  if (!value) unit_turn(turn, unit, b, t, c, s);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t head = group + k * groups;
    if (head < heads) {
      if (!value) turn_unit<T, HALF>(x[k], unit, c, s);
      store_unit<T, NT>(target + head * pitch, x[k], unit);
    }
  }
}

template <typename T, bool HALF, bool NT, int K>
void launch_append(Append<T> append, uint64_t batch, uint64_t tokens, const Turn& turn,
                   hipStream_t stream) {
  append.query_groups = (append.query_heads + K - 1) / K;
  append.key_groups = (append.key_heads + K - 1) / K;
  const uint32_t units = units_of(turn.half, turn.extent);
  const uint32_t groups = append.query_groups + 2 * append.key_groups;
  FastDiv by_units, by_groups;
  by_units.init(units);
  by_groups.init(groups);
  const uint64_t per_row = static_cast<uint64_t>(units) * groups;
  const uint64_t most = kIndex32Limit / per_row;  // rows of one launch
  for (uint64_t first = 0, all = batch * tokens; first < all; first += most) {
    const uint64_t count = all - first < most ? all - first : most;
    const uint32_t items = static_cast<uint32_t>(count * per_row);
    append_kernel<T, HALF, NT, K><<<ceil_div_u32(items, kThreads), kThreads, 0, stream>>>(
        append, turn, rows_at(first, batch, tokens), items, by_units, by_groups);
  }
}

template <typename T>
void start_append(const Append<T>& append, uint64_t batch, uint64_t tokens, const Turn& turn,
                  int layout, hipStream_t stream) {
  const uint64_t heads = append.query_heads + 2 * static_cast<uint64_t>(append.key_heads);
  const uint64_t lanes = batch * tokens * units_of(turn.half, turn.extent) * heads;
  // Past the caches where much is written in whole lines: halves of float32 heads whose lanes
  // lie side by side ([4, 4096] tokens of 32 + 2 * 8 heads of 128 150 us, through the caches
  // 160).  Elsewhere a store writes every second 16 bytes or ends in the middle of a line, which
  // the caches put together: neighbouring pairs 114 us, past the caches 133, in float64 130 and
  // 255, half of a head of 100 62 and 84.
  const bool stream_out =
      2 * turn.half == turn.extent && turn.half * sizeof(T) % 128 == 0 &&
      stream_output(batch * tokens * heads * static_cast<uint64_t>(turn.extent) * sizeof(T));
  // Two heads a lane, so that cos and sin serve twice: four take 156 us and eight 154 where
  // two take 149.  One head of doubles: a lane's loads are as wide.
  constexpr int kMany = 8 / sizeof(T);
  const bool many = lanes >= kMany * kFullLanes;
  // What goes past the caches is more than that many lanes' share.
  static_assert(kStreamStoreBytes / (8 * sizeof(T)) >= kMany * kFullLanes);
  if constexpr (std::is_same_v<T, float>) {
    if (layout == SPAR_HIP_ROTARY_HALF && stream_out) {
      launch_append<T, true, true, kMany>(append, batch, tokens, turn, stream);
      return;
    }
  }
  const auto launch_heads = [&](auto half) {
    if (many) {
      launch_append<T, decltype(half)::value, false, kMany>(append, batch, tokens, turn, stream);
    } else {
      launch_append<T, decltype(half)::value, false, 1>(append, batch, tokens, turn, stream);
    }
  };
  if (layout == SPAR_HIP_ROTARY_HALF) {
    launch_heads(std::true_type{});
  } else {
    launch_heads(std::false_type{});
  }
}

}  // namespace
}  // namespace rotary
}  // namespace spar_hip

using namespace spar_hip;

extern "C" SparHipStatus spar_hip_launch_cache_append(
    const SparHipPages* cache, const SparHipHeads* query_output, const SparHipHeads* query,
    uint64_t query_heads, const SparHipHeads* key, const SparHipHeads* value, uint64_t batch,
    uint64_t key_heads, uint64_t tokens, uint64_t extent, const void* places,
    uint64_t place_stride, int place_dtype, const SparHipRotary* rotary, int dtype, int device) {
  if (!valid_float_dtype(dtype) || !valid_pages(cache) ||
      (place_dtype != SPAR_HIP_INT32 && place_dtype != SPAR_HIP_INT64) ||
      (rotary != nullptr && !rotary::valid_rotary(rotary, extent)) ||
      (query == nullptr) != (query_output == nullptr) || batch > kIndex32Limit ||
      !rotary::sane(batch, query_heads, tokens, extent) ||
      !rotary::sane(batch, key_heads, tokens, extent)) {
    return invalid();
  }
  const uint64_t queries = query == nullptr ? 0 : query_heads;
  if (batch == 0 || tokens == 0 || extent == 0 || queries + key_heads == 0) return ok();
  const bool keeps = key_heads != 0;
  if ((queries != 0 && (query->data == nullptr || query_output->data == nullptr)) ||
      (keeps && (key == nullptr || value == nullptr || key->data == nullptr ||
                 value->data == nullptr || places == nullptr)) ||
      (keeps && has_room(*cache) &&
       (cache->key.data == nullptr || cache->value.data == nullptr)) ||
      (rotary != nullptr && !rotary::complete_rotary(rotary))) {
    return invalid();
  }
  const rotary::Turn turn =
      rotary != nullptr
          ? rotary::turn_of(*rotary, extent, false)
          : rotary::Turn{nullptr, 0, nullptr, 1.0, 0, static_cast<uint32_t>(extent), false, false};
  const int layout = rotary != nullptr ? rotary->layout : SPAR_HIP_ROTARY_HALF;
  const uint64_t units = rotary::units_of(turn.half, turn.extent);
  if (units * (queries + 2 * key_heads) > kIndex32Limit / 2) return invalid();
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  const auto start = [&](auto zero) {
    using T = decltype(zero);
    rotary::Append<T> append{};
    append.cache = pages_of<T>(*cache);
    if (queries != 0) {
      append.query_output = rotary::heads_of<T>(*query_output);
      append.query = rotary::heads_of<const T>(*query);
    }
    if (keeps) {
      append.key = rotary::heads_of<const T>(*key);
      append.value = rotary::heads_of<const T>(*value);
    }
    append.query_heads = static_cast<uint32_t>(queries);
    append.key_heads = static_cast<uint32_t>(key_heads);
    append.places = places;
    append.place_stride = place_stride;
    append.wide_places = place_dtype == SPAR_HIP_INT64;
    rotary::start_append<T>(append, batch, tokens, turn, layout, guard.stream);
  };
  if (dtype == SPAR_HIP_FLOAT32) {
    start(0.0F);
  } else {
    start(0.0);
  }
  return finish(guard);
}

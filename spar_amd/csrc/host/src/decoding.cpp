// The paged cache, attention over it behind a shared prefix, and beam selection over the
// kernels of cache.hip, attention_cache.hip and beams.hip (additions; the reference's
// decoding concatenates its cache and chooses tokens on the host).
#include <cmath>
#include <cstdint>
#include <limits>
#include <string>
#include <vector>

#include "heads_internal.hpp"
#include "spar/decoding.hpp"

namespace spar {
namespace {

using namespace detail::heads;
using detail::HipTensorAccess;
namespace hip = detail::hip;

void validate_detached(const Tensor& tensor, const char* name) {
  if (tensor.requires_grad()) refuse(name, "has no gradient: detach its tensors");
}

void validate_new_heads(const Tensor& tensor, const char* name, const char* which) {
  validate_heads(tensor, name, which);
  validate_detached(tensor, name);
}

// Checks a cache against the heads it goes with and returns its rows.
std::size_t validate_cache(const PagedCache& cache, const Tensor& heads, const char* name,
                           const char* which) {
  for (const Tensor* tensor : {&cache.key, &cache.value}) {
    validate_new_heads(*tensor, name, which);
    validate_like(*tensor, heads, name);
    if (tensor->numel() != 0 && tensor->shape()[3] != 1 && tensor->strides()[3] != 1) {
      refuse(name, "needs caches whose last axis is contiguous");
    }
  }
  if (cache.key.shape() != cache.value.shape()) {
    refuse(name, "needs keys and values of one shape in a cache");
  }
  if (extent_of(cache.key, 3) != extent_of(heads, 3)) refuse(name, "cache and head extents differ");
  if (extent_of(cache.key, 2) == 0) refuse(name, "needs pages of at least one token");
  if (!cache.table) return extent_of(cache.key, 0);
  const Tensor& table{*cache.table};
  if (table.rank() != 2 || table.dtype() != DType::Int32) {
    refuse(name, "tables must be Int32 [rows, entries]");
  }
  if (table.device() != heads.device()) refuse(name, "tensors are on different devices");
  return extent_of(table, 0);
}

// A cache that is written: every element has a place of its own.
void validate_written(const PagedCache& cache, const char* name) {
  if (cache.key.numel() == 0) return;
  for (const Tensor* tensor : {&cache.key, &cache.value}) {
    for (std::size_t axis{0}; axis < 3; ++axis) {
      if (extent_of(*tensor, axis) > 1 && tensor->strides()[axis] == 0) {
        refuse(name, "needs caches whose tokens have places of their own");
      }
    }
  }
  if (first_element(cache.key) == first_element(cache.value)) {
    refuse(name, "needs keys and values at places of their own");
  }
}

// A cache as kernels read it; `table` is what keeps a packed table alive.
SparHipPages pages_of(const PagedCache& cache, std::optional<Tensor>& table) {
  SparHipPages pages{heads_of(cache.key), heads_of(cache.value), extent_of(cache.key, 0),
                     extent_of(cache.key, 2), nullptr, 0, 1};
  if (cache.table) {
    const bool dense{cache.table->numel() == 0 || cache.table->shape()[1] == 1 ||
                     cache.table->strides()[1] == 1};
    table = dense ? *cache.table : cache.table->contiguous();
    pages.table = static_cast<const std::int32_t*>(first_element(*table));
    pages.table_stride = static_cast<std::uint64_t>(table->strides()[0]);
    pages.table_pages = pages.table == nullptr ? 0 : extent_of(*table, 1);
  }
  return pages;
}

Tensor workspace_of(std::uint64_t bytes, Device device) {
  return Tensor{Shape{static_cast<Shape::dimension_type>((bytes + 3) / 4)}, DType::Int32, device};
}

}  // namespace

std::optional<Tensor> cache_append(const PagedCache& cache, const Tensor& key,
                                   const Tensor& value, const Tensor& places,
                                   const std::optional<CacheRotation>& rotation,
                                   const std::optional<Tensor>& query) {
  constexpr const char* name{"cache_append"};
  validate_new_heads(key, name, "key");
  validate_new_heads(value, name, "value");
  validate_like(value, key, name);
  if (key.shape() != value.shape()) refuse(name, "key and value must have one shape");
  const std::size_t rows{validate_cache(cache, key, name, "cache")};
  const std::size_t batch{extent_of(key, 0)}, key_heads{extent_of(key, 1)},
      tokens{extent_of(key, 2)}, extent{extent_of(key, 3)};
  if (rows != batch) refuse(name, "needs a cache row for every sequence");
  if (extent_of(cache.key, 1) != key_heads) refuse(name, "cache and key heads differ");
  validate_integers(places, key, name, "places");
  if (places.rank() != 2 || extent_of(places, 0) != batch || extent_of(places, 1) != tokens) {
    refuse(name, "places must be [batch, tokens]");
  }
  std::optional<Rotation> turn;
  if (rotation) {
    turn = rotation_of(key, rotation->positions, rotation->frequencies, rotation->layout,
                       rotation->magnitude, name);
  }
  std::optional<Tensor> q, output;
  if (query) {
    if (!turn) refuse(name, "needs a rotation to turn queries");
    validate_new_heads(*query, name, "query");
    validate_like(*query, key, name);
    if (extent_of(*query, 0) != batch || extent_of(*query, 2) != tokens ||
        extent_of(*query, 3) != extent) {
      refuse(name, "query and key may differ in their heads alone");
    }
    q = readable(*query);
    output = ordered_like(*q);
  }
  validate_written(cache, name);
  const Tensor k{readable(key)}, v{readable(value)};
  const bool dense{places.numel() == 0 || tokens == 1 || places.strides()[1] == 1};
  const Tensor at{dense ? places : places.contiguous()};
  std::optional<Tensor> table;
  const SparHipPages pages{pages_of(cache, table)};
  const SparHipHeads k_heads{heads_of(k)}, v_heads{heads_of(v)};
  SparHipHeads q_heads{}, target{};
  if (q) {
    q_heads = heads_of(*q);
    target = heads_of(*output);
  }
  SparHipRotary argument{};
  if (turn) argument = turn->argument();
  hip::check(spar_hip_launch_cache_append(
                 &pages, q ? &target : nullptr, q ? &q_heads : nullptr, q ? extent_of(*q, 1) : 0,
                 &k_heads, &v_heads, batch, key_heads, tokens, extent, first_element(at),
                 at.numel() == 0 ? 0 : static_cast<std::uint64_t>(at.strides()[0]),
                 hip::dtype_tag(at.dtype()), turn ? &argument : nullptr,
                 hip::dtype_tag(key.dtype()), key.device().index()),
             name, key.device());
  return output;
}

Tensor cache_attention(const Tensor& query, const PagedCache& cache,
                       const std::optional<Tensor>& lengths,
                       const std::optional<PagedCache>& prefix,
                       const std::optional<Tensor>& prefix_lengths, std::optional<double> scale) {
  constexpr const char* name{"cache_attention"};
  validate_new_heads(query, name, "query");
  const std::size_t batch{extent_of(query, 0)}, query_heads{extent_of(query, 1)},
      extent{extent_of(query, 3)};
  if (extent < 1 || extent > SPAR_HIP_ATTENTION_MAX_EXTENT) {
    refuse(name, "takes heads of 1 to 256 elements");
  }
  if (validate_cache(cache, query, name, "cache") != batch) {
    refuse(name, "needs a cache row for every sequence");
  }
  const std::size_t key_heads{extent_of(cache.key, 1)};
  if (key_heads == 0 || query_heads == 0 || query_heads % key_heads != 0) {
    refuse(name, "query heads must be a multiple of key heads");
  }
  std::size_t prefixes{0};
  if (prefix) {
    prefixes = validate_cache(*prefix, query, name, "prefix");
    if (extent_of(prefix->key, 1) != key_heads) refuse(name, "cache and prefix heads differ");
    if (prefixes == 0 ? batch != 0 : batch % prefixes != 0) {
      refuse(name, "sequences must be a multiple of prefixes");
    }
  } else if (prefix_lengths) {
    refuse(name, "got prefix lengths without a prefix");
  }
  if (scale && !std::isfinite(*scale)) refuse(name, "scale must be finite");
  std::optional<Tensor> counts, prefix_counts;
  const auto counted{[&](const Tensor& tensor, std::size_t rows) {
    validate_integers(tensor, query, name, "lengths");
    if (tensor.rank() != 1 || extent_of(tensor, 0) != rows) {
      refuse(name, "lengths must be [batch] and [prefix rows]");
    }
    return tensor.contiguous();
  }};
  if (lengths) counts = counted(*lengths, batch);
  if (prefix_lengths) prefix_counts = counted(*prefix_lengths, prefixes);
  if (counts && prefix_counts && counts->dtype() != prefix_counts->dtype()) {
    refuse(name, "lengths must have one dtype");
  }
  const Tensor q{readable(query)};
  Tensor output{ordered_like(q)};
  if (batch == 0) return output;
  const Device device{query.device()};
  const int length_dtype{counts          ? hip::dtype_tag(counts->dtype())
                         : prefix_counts ? hip::dtype_tag(prefix_counts->dtype())
                                         : SPAR_HIP_INT32};
  const SparHipCacheAttention shape{
      batch,
      prefixes,
      query_heads,
      key_heads,
      extent_of(query, 2),
      extent,
      scale ? *scale : 1.0 / std::sqrt(static_cast<double>(extent)),
      counts ? first_element(*counts) : nullptr,
      prefix_counts ? first_element(*prefix_counts) : nullptr,
      length_dtype,
      hip::dtype_tag(query.dtype())};
  std::optional<Tensor> table, prefix_table;
  const SparHipPages pages{pages_of(cache, table)};
  SparHipPages shared{};
  if (prefix) shared = pages_of(*prefix, prefix_table);
  std::uint64_t bytes{0};
  hip::check(spar_hip_cache_attention_workspace(&bytes, &pages, prefix ? &shared : nullptr, &shape),
             name, device);
  Tensor workspace{workspace_of(bytes, device)};
  const SparHipHeads target{heads_of(output)}, q_heads{heads_of(q)};
  hip::check(spar_hip_launch_cache_attention(&target, &q_heads, &pages, prefix ? &shared : nullptr,
                                             &shape, first_element(workspace), bytes,
                                             device.index()),
             name, device);
  return output;
}

BeamSelection beam_select(const Tensor& logits, const Tensor& scores, std::size_t picks,
                          std::optional<std::int64_t> end_token,
                          const std::optional<Tensor>& ended) {
  constexpr const char* name{"beam_select"};
  if (logits.rank() != 3) refuse(name, "logits must be [groups, beams, vocabulary]");
  if (!is_floating(logits.dtype())) refuse(name, "requires a floating-point dtype");
  detail::require_hip(logits, name);
  validate_detached(logits, name);
  validate_detached(scores, name);
  validate_like(scores, logits, name);
  const std::size_t groups{extent_of(logits, 0)}, beams{extent_of(logits, 1)},
      vocabulary{extent_of(logits, 2)};
  const auto by_beam{[&](const Tensor& tensor) {
    return tensor.rank() == 2 && extent_of(tensor, 0) == groups && extent_of(tensor, 1) == beams;
  }};
  if (!by_beam(scores)) refuse(name, "scores must be [groups, beams]");
  if (beams < 1 || beams > SPAR_HIP_MAX_BEAMS) refuse(name, "takes 1 to 64 beams");
  if (vocabulary < 1 || vocabulary > std::numeric_limits<std::int32_t>::max()) {
    refuse(name, "takes vocabularies of 1 to 2^31 - 1 tokens");
  }
  if (picks < 1 || picks > SPAR_HIP_MAX_BEAMS || picks > beams * vocabulary) {
    refuse(name, "takes 1 to 64 picks, at most beams * vocabulary");
  }
  if (end_token && (*end_token < 0 || static_cast<std::uint64_t>(*end_token) >= vocabulary)) {
    refuse(name, "end token is outside the vocabulary");
  }
  if (ended) {
    if (ended->dtype() != DType::Int32 || !by_beam(*ended)) {
      refuse(name, "ended must be Int32 [groups, beams]");
    }
    if (ended->device() != logits.device()) refuse(name, "tensors are on different devices");
    if (!end_token) refuse(name, "needs the end token of beams that have ended");
  }
  const Device device{logits.device()};
  // Rows at one distance, tokens side by side.
  const auto strides{logits.strides()};
  const bool rows{logits.numel() == 0 ||
                  ((vocabulary == 1 || strides[2] == 1) &&
                   (beams == 1 || groups == 1 || strides[0] == strides[1] * beams))};
  std::size_t row_stride{vocabulary};
  if (rows && logits.numel() != 0) {
    row_stride = static_cast<std::size_t>(beams > 1 ? strides[1] : groups > 1 ? strides[0]
                                                                              : vocabulary);
  }
  const bool in_place{rows && row_stride >= vocabulary};
  const Tensor x{in_place ? logits : logits.contiguous()};
  if (!in_place) row_stride = vocabulary;
  const Tensor totals{scores.contiguous()};
  std::optional<Tensor> flags;
  if (ended) flags = ended->contiguous();
  const SparHipBeams shape{groups,
                           beams,
                           vocabulary,
                           picks,
                           row_stride,
                           flags ? static_cast<const std::int32_t*>(first_element(*flags)) : nullptr,
                           end_token ? *end_token : -1,
                           hip::dtype_tag(logits.dtype())};
  const Shape picked{static_cast<Shape::dimension_type>(groups),
                     static_cast<Shape::dimension_type>(picks)};
  BeamSelection made{Tensor{picked, logits.dtype(), device}, Tensor{picked, DType::Int64, device},
                     Tensor{picked, DType::Int64, device}, Tensor{picked, DType::Int32, device}};
  if (groups == 0) return made;
  std::uint64_t bytes{0};
  hip::check(spar_hip_beam_select_workspace(&bytes, &shape), name, device);
  Tensor workspace{workspace_of(bytes, device)};
  hip::check(spar_hip_launch_beam_select(
                 first_element(made.scores), static_cast<std::int64_t*>(first_element(made.parents)),
                 static_cast<std::int64_t*>(first_element(made.tokens)),
                 static_cast<std::int32_t*>(first_element(made.ended)), first_element(x),
                 first_element(totals), &shape, first_element(workspace), bytes, device.index()),
             name, device);
  return made;
}

std::vector<Tensor> reorder(const std::vector<Tensor>& states, const Tensor& parents) {
  constexpr const char* name{"reorder"};
  if (parents.dtype() != DType::Int64) refuse(name, "parents must have Int64 dtype");
  detail::require_hip(parents, name);
  const Tensor order{parents.contiguous()};
  const std::size_t rows{order.numel()};
  std::vector<Tensor> read, made;
  std::size_t source_rows{0};
  for (const Tensor& state : states) {
    if (state.rank() == 0) refuse(name, "needs states with rows");
    validate_detached(state, name);
    if (state.device() != parents.device()) refuse(name, "tensors are on different devices");
    if (read.empty()) source_rows = extent_of(state, 0);
    if (extent_of(state, 0) != source_rows) refuse(name, "needs states of equally many rows");
    read.push_back(state.contiguous());
    std::vector<Shape::dimension_type> extents;
    for (std::size_t k{0}; k < state.rank(); ++k) extents.push_back(state.shape()[k]);
    extents[0] = static_cast<Shape::dimension_type>(rows);
    made.emplace_back(Shape{extents}, state.dtype(), state.device());
  }
  std::vector<SparHipReorder> moves;
  for (std::size_t i{0}; i < read.size(); ++i) {
    std::uint64_t row{1};
    for (std::size_t k{1}; k < read[i].rank(); ++k) row *= extent_of(read[i], k);
    moves.push_back({first_element(made[i]), row, first_element(read[i]), row, row,
                     size_of(read[i].dtype())});
  }
  if (rows == 0 || moves.empty()) return made;
  hip::check(spar_hip_launch_reorder(moves.data(), moves.size(),
                                     static_cast<const std::int64_t*>(first_element(order)), rows,
                                     source_rows, parents.device().index()),
             name, parents.device());
  return made;
}

}  // namespace spar

// What a decoder layer does with the heads of its queries, keys and values, on
// HIP tensors with autograd: rotary positions, RMSNorm of every query and key
// head with the rotation in the same pass, and causal attention with a sliding
// window and sinks.  The reference's nn layer has interleaved rotation of whole
// heads and attention over whole score matrices (src/nn/attention.cpp:122-135).
//
// Heads are [batch, heads, tokens, extent] tensors, Float32 or Float64.  Any view
// whose last axis is contiguous is read in place: the transpose of a projection's
// [batch, tokens, heads, extent], a narrowed part of a packed projection, a cache.
// Outputs and gradients lie in the order of the tensor they belong to: where an
// input holds a token's heads side by side, so does its output, whose transpose
// back to [batch, tokens, heads, extent] is contiguous.
#pragma once

#include <cstddef>
#include <optional>
#include <utility>

#include "spar/tensor.hpp"

namespace spar {

/// which elements of a head's first 2 n form the n pairs of a rotation: j with
/// j + n, or 2j with 2j + 1.
enum class RotaryLayout { Half, Interleaved };

/// how the frequencies of a model trained on `trained_tokens` positions are
/// changed for contexts `factor` times as long.
struct RotaryScaling final {
  enum class Kind {
    None,
    /// every frequency divided by the factor.
    Linear,
    /// the base stretched so that the slowest pair's frequency is divided by the
    /// factor and the fastest pair's kept: base * factor^(r / (r - 2)).
    Base,
    /// pairs that turn less than `slow_turns` times within trained_tokens
    /// divided by the factor, those that turn more than `fast_turns` times kept,
    /// a blend linear in the turns between.
    Parts,
  };
  Kind kind{Kind::None};
  double factor{1.0};
  double trained_tokens{0.0};
  double slow_turns{1.0};
  double fast_turns{32.0};
};

/// radians per position of the pairs of a head's first `rotary_extent` elements,
/// base^(-2 j / rotary_extent) as `scaling` changes them: a Float64 CPU tensor
/// [rotary_extent / 2], to be moved to the heads' device once.
[[nodiscard]] Tensor rotary_frequencies(std::size_t rotary_extent, double base = 10000.0,
                                        const RotaryScaling& scaling = {});
/// the factor 0.1 ln(factor) + 1 that usually goes with Parts scaling.
[[nodiscard]] double rotary_magnitude(double factor);

/// heads turned by their positions.  positions: Int32 or Int64, [tokens] or
/// [batch, tokens]; frequencies: Float64 [n], 2 n <= extent: the rest of a head
/// is passed on.  Turned elements are multiplied by `magnitude`.  The gradient
/// is the opposite rotation.
[[nodiscard]] Tensor rotary_embedding(const Tensor& heads, const Tensor& positions,
                                      const Tensor& frequencies,
                                      RotaryLayout layout = RotaryLayout::Half,
                                      double magnitude = 1.0);

/// rms_norm of every query and key head over its extent (weights [extent], at most
/// 256), each followed by rotary_embedding, in one launch.  Queries and keys may
/// have different numbers of heads.
[[nodiscard]] std::pair<Tensor, Tensor> query_key_norm_rotary(
    const Tensor& query, const Tensor& key, const Tensor& query_weight, const Tensor& key_weight,
    const Tensor& positions, const Tensor& frequencies, RotaryLayout layout = RotaryLayout::Half,
    double magnitude = 1.0, double epsilon = 1.0e-5);

/// Causal attention.  query [batch, query heads, queries, extent], key and value
/// [batch, key heads, keys, extent], extent at most 256; query head h reads key
/// head h / (query heads / key heads).  Query i of a sequence of `length` keys is
/// its token p = length - queries + i and sees the keys j <= p with p - j < window
/// (window 0: all of them) or j < sinks.
///   output = softmax(scale * query key^T) value
/// over the visible keys; zeros for queries that see none (p < 0).
///   scale    1 / sqrt(extent) where not given
///   lengths  Int32 or Int64 [batch], the tokens of each sequence in the keys,
///            clamped to [0, keys]; all keys where not given.  Keys and values
///            behind them have no part in any result, whatever they hold (their
///            memory may be read).
/// A query or key of another sequence or head never changes a result; a NaN or
/// infinity in a key or value that some query of its head sees may also reach
/// other queries of that head, and one in any input that takes part the gradients
/// of its key head and of the query heads that read it.
[[nodiscard]] Tensor window_attention(const Tensor& query, const Tensor& key, const Tensor& value,
                                      std::size_t window = 0, std::size_t sinks = 0,
                                      std::optional<double> scale = std::nullopt,
                                      const std::optional<Tensor>& lengths = std::nullopt);

}  // namespace spar

// Decoding of sequences that share a prompt, on HIP tensors: a cache of keys and values in
// pages that grows token by token, attention over it that reads the shared prompt once, and
// beam search's choice of the next tokens.  The reference's cache is a concatenation of
// tensors and its decoding greedy or sampled on the host.
//
// These operators serve and have no gradients: tensors that require them are refused
// (detach() them).  Heads are [batch, heads, tokens, extent] tensors as in attention.hpp,
// Float32 or Float64, read in place where their last axis is contiguous.
#pragma once

#include <cstddef>
#include <cstdint>
#include <optional>
#include <utility>
#include <vector>

#include "spar/attention.hpp"
#include "spar/tensor.hpp"

namespace spar {

/// Keys and values of several sequences, or of several prefixes, in pages: key and value
/// [pages, key heads, page tokens, extent] with a contiguous last axis (any other strides:
/// a layer's part of a larger cache), written in place.
///   table  Int32 [rows, entries]: token t of row b is token t % page_tokens of page
///          table[b, t / page_tokens].  A page number that is not one of the cache's
///          (-1 behind a sequence's last page) holds nothing: its tokens are neither
///          seen nor written.  Without a table row b is page b: a contiguous cache.
struct PagedCache final {
  Tensor key;
  Tensor value;
  std::optional<Tensor> table{};
};

/// The rotation of a step's new tokens: rotary_embedding's arguments.
struct CacheRotation final {
  Tensor positions;    // Int32 or Int64 [tokens] or [batch, tokens]
  Tensor frequencies;  // Float64 [n]
  RotaryLayout layout{RotaryLayout::Half};
  double magnitude{1.0};
};

/// Writes the keys and values of new tokens, [batch, key heads, tokens, extent] each, to the
/// cache, whose rows are the batch's sequences; with a rotation the keys are turned on the
/// way, and with queries [batch, query heads, tokens, extent] these are turned in the same
/// launch and returned, in the order of their tokens and heads (nothing without queries,
/// which need a rotation).  The cache's keys and values must not overlap each other (nor be
/// expanded) or what is written to them; an operation with gradients that has read them reads
/// them again, as they are then, in its backward.
///   places  Int32 or Int64 [batch, tokens]: the token of its sequence's row that each new
///           token becomes; negative or behind the row's room for one that is not written
///           (padding).  The rest of the cache stays as it is.  Two tokens must not share a
///           place in the pages: rows whose tables name one page, as beams' do that go on
///           from one parent, need pages of their own for new tokens (see reorder).
std::optional<Tensor> cache_append(const PagedCache& cache, const Tensor& key,
                                   const Tensor& value, const Tensor& places,
                                   const std::optional<CacheRotation>& rotation = std::nullopt,
                                   const std::optional<Tensor>& query = std::nullopt);

/// softmax(scale * query [prefix keys; own keys]^T) [prefix values; own values]: query
/// [batch, query heads, queries, extent], extent at most 256; query head h reads key head
/// h / (query heads / key heads).  The last `queries` tokens of sequence b ask: query i is
/// its own token p = length - queries + i in row b of the cache, and sees its own tokens
/// up to p and all of its prefix; zeros where p < 0.
///   prefix   rows shared by batch / rows neighbouring sequences each, whose keys and
///            values are read once for all of them; none where not given
///   lengths, prefix_lengths
///            Int32 or Int64 (one dtype) [batch] and [prefix rows], clamped to [0, what a
///            row has room for], which they are where not given
///   scale    1 / sqrt(extent) where not given
/// Keys and values that no query sees have no part, whatever they hold; a NaN or
/// infinity in one that some query sees may also reach other queries of its head, in a
/// prefix those of all sequences that share it.  Refused are calls of more than 2^27 - 8
/// queries of all heads and sequences behind a prefix, of some 2^30 without one (spar_hip.h).
[[nodiscard]] Tensor cache_attention(const Tensor& query, const PagedCache& cache,
                                     const std::optional<Tensor>& lengths = std::nullopt,
                                     const std::optional<PagedCache>& prefix = std::nullopt,
                                     const std::optional<Tensor>& prefix_lengths = std::nullopt,
                                     std::optional<double> scale = std::nullopt);

/// The picks of a step, [groups, picks] each, best first.
struct BeamSelection final {
  Tensor scores;   // totals, of the logits' dtype
  Tensor parents;  // Int64: row of all groups * beams that each goes on from
  Tensor tokens;   // Int64
  Tensor ended;    // Int32: 1 where the row had ended or the token is the end token
};

/// The best continuations of every group of beams: logits [groups, beams, vocabulary],
/// scores [groups, beams] the log-probabilities of the beams so far.  The total of a token
/// is its beam's score plus log_softmax(logits), -infinity where that is NaN; picks (at most
/// 64, as beams) are the largest totals of a group, of equal ones the lowest beam, its largest
/// logit and lowest token first.  Totals are added in double to a log-sum whose exponentials
/// are of the logits' dtype: of Float32 logits it is mostly off by less than 1e-7 (spar_hip.h
/// has the bound), and two beams' totals that are closer may come in either order.
///   end_token  ends a sequence; none where not given
///   ended      Int32 [groups, beams]: beams that are not 0 have ended and go on with the
///              end token alone (which must be given), at their score
/// At the first step, with all beams alike, scores are 0 for a group's first beam and
/// -infinity for the others.
[[nodiscard]] BeamSelection beam_select(const Tensor& logits, const Tensor& scores,
                                        std::size_t picks,
                                        std::optional<std::int64_t> end_token = std::nullopt,
                                        const std::optional<Tensor>& ended = std::nullopt);

/// New tensors with the states' rows (along axis 0) in the order of `parents`, Int64 of any
/// shape: row i of each is row parents[i] of its state, zeros where there is none.  States of
/// any dtype and shape, moved in one launch; those that are not contiguous are copied first.
/// Where a cache's table is moved and a parent comes twice, both rows name its pages.  They
/// may share pages that are only read.  Before cache_append the page of the next token must
/// be another for each: one that no row names and, in the middle of a page, with a copy of
/// the shared one's tokens, which reorder({key, value}, page numbers) yields as heads [rows,
/// key heads, page tokens, extent] for cache_append to write (-1 for places to come).
[[nodiscard]] std::vector<Tensor> reorder(const std::vector<Tensor>& states,
                                          const Tensor& parents);

}  // namespace spar

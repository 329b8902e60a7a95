// Rotary positions, normed query and key heads with the rotation, and windowed
// attention over the kernels of rotary.hip and attention_*.hip (additions; the
// reference has RoPE and full attention among its nn layers).
#include <cmath>
#include <cstdint>
#include <memory>
#include <numbers>
#include <stdexcept>
#include <string>
#include <vector>

#include "autograd_internal.hpp"
#include "heads_internal.hpp"
#include "spar/attention.hpp"
#include "spar/ops.hpp"

namespace spar {
namespace {

using namespace detail::heads;
namespace hip = detail::hip;

// For a backward: what the program changes in the positions later has no part in it.
Rotation snapshot_of(const Rotation& rotation) {
  Rotation copy{rotation};
  copy.positions = rotation.positions.clone();
  copy.frequencies = rotation.frequencies.clone();
  if (copy.position_stride != 0) {
    copy.position_stride = static_cast<std::size_t>(copy.positions.strides()[0]);
  }
  return copy;
}

Tensor turned(const Tensor& heads, const Rotation& rotation, bool inverse, const char* name) {
  const Tensor x{readable(heads.detach())};
  Tensor output{ordered_like(x)};
  const SparHipHeads target{heads_of(output)}, source{heads_of(x)};
  const SparHipRotary argument{rotation.argument()};
  hip::check(spar_hip_launch_rotary(&target, &source, extent_of(x, 0), extent_of(x, 1),
                                    extent_of(x, 2), extent_of(x, 3), &argument, inverse ? 1 : 0,
                                    hip::dtype_tag(x.dtype()), x.device().index()),
             name, x.device());
  return output;
}

// --------------------------------------------------- head norm and rotation

// What the backward of one normed tensor keeps.
struct SavedHeadNorm {
  Tensor x;
  Tensor weight;
  Tensor denominator;
  Rotation rotation;
  bool grad_x;
  bool grad_weight;
};

std::vector<Tensor> head_norm_backward(const SavedHeadNorm& saved, const Tensor& gradient) {
  const Tensor dy{readable(gradient.detach())};
  Tensor dx{ordered_like(saved.x)};
  Tensor dw{saved.weight.shape(), saved.x.dtype(), saved.x.device()};
  const std::size_t batch{extent_of(saved.x, 0)}, heads{extent_of(saved.x, 1)},
      tokens{extent_of(saved.x, 2)}, extent{extent_of(saved.x, 3)};
  const int dtype{hip::dtype_tag(saved.x.dtype())};
  const Device device{saved.x.device()};
  std::uint64_t bytes{0};
  hip::check(spar_hip_head_norm_rotary_workspace(&bytes, batch, tokens, heads, extent, dtype),
             "query_key_norm_rotary backward", device);
  Tensor workspace{Shape{static_cast<Shape::dimension_type>((bytes + 3) / 4)}, DType::Int32,
                   device};
  const SparHipHeadNormGradient part{heads_of(dx),
                                     first_element(dw),
                                     heads_of(dy),
                                     heads_of(saved.x),
                                     first_element(saved.weight),
                                     first_element(saved.denominator),
                                     heads};
  const SparHipRotary argument{saved.rotation.argument()};
  hip::check(spar_hip_launch_head_norm_rotary_backward(&part, 1, batch, tokens, extent, &argument,
                                                       first_element(workspace), bytes, dtype,
                                                       device.index()),
             "query_key_norm_rotary backward", device);
  std::vector<Tensor> contributions;
  if (saved.grad_x) contributions.push_back(dx);
  if (saved.grad_weight) contributions.push_back(dw);
  return contributions;
}

void record_head_norm(Tensor& output, const Tensor& x, const Tensor& weight,
                      const Tensor& packed_weight, const Tensor& denominator,
                      const Rotation& rotation) {
  const bool grad_x{x.requires_grad()}, grad_weight{weight.requires_grad()};
  if (!grad_x && !grad_weight) return;
  std::vector<Tensor> parents;
  if (grad_x) parents.push_back(x);
  if (grad_weight) parents.push_back(weight);
  auto saved{std::make_shared<const SavedHeadNorm>(SavedHeadNorm{
      x.detach(), packed_weight.detach(), denominator, rotation, grad_x, grad_weight})};
  detail::record_operation(output, std::move(parents), [saved](const Tensor& gradient) {
    return head_norm_backward(*saved, gradient);
  });
}

// ---------------------------------------------------------------- attention

struct SavedAttention {
  Tensor query, key, value, output, logsumexp;
  std::optional<Tensor> lengths;
  SparHipAttention shape;
  bool grad_query, grad_key, grad_value;
};

std::vector<Tensor> attention_backward(const SavedAttention& saved, const Tensor& gradient) {
  const Tensor dy{readable(gradient.detach())};
  Tensor dq{ordered_like(saved.query)}, dk{ordered_like(saved.key)},
      dv{ordered_like(saved.value)};
  const Device device{saved.query.device()};
  std::uint64_t bytes{0};
  hip::check(spar_hip_attention_workspace(&bytes, &saved.shape, 1), "window_attention backward",
             device);
  Tensor workspace{Shape{static_cast<Shape::dimension_type>((bytes + 3) / 4)}, DType::Int32,
                   device};
  const SparHipHeads query_gradient{heads_of(dq)}, key_gradient{heads_of(dk)},
      value_gradient{heads_of(dv)}, output_gradient{heads_of(dy)}, output{heads_of(saved.output)},
      query{heads_of(saved.query)}, key{heads_of(saved.key)}, value{heads_of(saved.value)};
  hip::check(spar_hip_launch_attention_backward(&query_gradient, &key_gradient, &value_gradient,
                                                &output_gradient, &output,
                                                first_element(saved.logsumexp), &query, &key,
                                                &value, &saved.shape, first_element(workspace),
                                                bytes, device.index()),
             "window_attention backward", device);
  std::vector<Tensor> contributions;
  if (saved.grad_query) contributions.push_back(dq);
  if (saved.grad_key) contributions.push_back(dk);
  if (saved.grad_value) contributions.push_back(dv);
  return contributions;
}

}  // namespace

Tensor rotary_frequencies(std::size_t rotary_extent, double base, const RotaryScaling& scaling) {
  constexpr const char* name{"rotary_frequencies"};
  if (rotary_extent == 0 || rotary_extent % 2 != 0) {
    refuse(name, "requires an even, positive rotary extent");
  }
  if (!std::isfinite(base) || base <= 0.0) refuse(name, "base must be finite and positive");
  using Kind = RotaryScaling::Kind;
  const bool scaled{scaling.kind != Kind::None};
  if (scaled && (!std::isfinite(scaling.factor) || scaling.factor <= 0.0)) {
    refuse(name, "scaling factor must be finite and positive");
  }
  if (scaling.kind == Kind::Base && rotary_extent == 2) {
    refuse(name, "cannot stretch the base of a single pair");
  }
  if (scaling.kind == Kind::Parts &&
      !(std::isfinite(scaling.trained_tokens) && scaling.trained_tokens > 0.0 &&
        std::isfinite(scaling.fast_turns) && scaling.slow_turns >= 0.0 &&
        scaling.fast_turns > scaling.slow_turns)) {
    refuse(name, "scaling by parts needs the trained tokens and slow_turns < fast_turns");
  }
  const auto extent{static_cast<double>(rotary_extent)};
  if (scaling.kind == Kind::Base) base *= std::pow(scaling.factor, extent / (extent - 2.0));
  std::vector<double> values(rotary_extent / 2);
  for (std::size_t j{0}; j < values.size(); ++j) {
    double f{std::pow(base, -2.0 * static_cast<double>(j) / extent)};
    if (scaling.kind == Kind::Linear) f /= scaling.factor;
    if (scaling.kind == Kind::Parts) {
      const double turns{scaling.trained_tokens * f / (2.0 * std::numbers::pi)};
      const double share{(turns - scaling.slow_turns) / (scaling.fast_turns - scaling.slow_turns)};
      const double keep{share < 0.0 ? 0.0 : share > 1.0 ? 1.0 : share};
      f = f * keep + f / scaling.factor * (1.0 - keep);
    }
    values[j] = f;
  }
  return from_values<double>(Shape{static_cast<Shape::dimension_type>(values.size())},
                             std::span<const double>{values});
}

double rotary_magnitude(double factor) {
  if (!std::isfinite(factor) || factor <= 0.0) {
    refuse("rotary_magnitude", "factor must be finite and positive");
  }
  return 0.1 * std::log(factor) + 1.0;
}

Tensor rotary_embedding(const Tensor& heads, const Tensor& positions, const Tensor& frequencies,
                        RotaryLayout layout, double magnitude) {
  constexpr const char* name{"rotary_embedding"};
  validate_heads(heads, name, "heads");
  const Rotation rotation{rotation_of(heads, positions, frequencies, layout, magnitude, name)};
  Tensor output{turned(heads, rotation, false, name)};
  if (heads.requires_grad()) {
    detail::record_operation(
        output, {heads}, [saved = snapshot_of(rotation)](const Tensor& gradient) {
          return std::vector<Tensor>{turned(gradient, saved, true, "rotary_embedding backward")};
        });
  }
  return output;
}

std::pair<Tensor, Tensor> query_key_norm_rotary(const Tensor& query, const Tensor& key,
                                                const Tensor& query_weight,
                                                const Tensor& key_weight, const Tensor& positions,
                                                const Tensor& frequencies, RotaryLayout layout,
                                                double magnitude, double epsilon) {
  constexpr const char* name{"query_key_norm_rotary"};
  validate_heads(query, name, "query");
  validate_heads(key, name, "key");
  validate_like(key, query, name);
  if (extent_of(key, 0) != extent_of(query, 0) || extent_of(key, 2) != extent_of(query, 2) ||
      extent_of(key, 3) != extent_of(query, 3)) {
    refuse(name, "query and key may differ in their heads alone");
  }
  const std::size_t batch{extent_of(query, 0)}, tokens{extent_of(query, 2)},
      extent{extent_of(query, 3)};
  if (extent < 1 || extent > SPAR_HIP_HEAD_NORM_MAX_EXTENT) {
    refuse(name, "takes heads of 1 to 256 elements");
  }
  for (const Tensor* weight : {&query_weight, &key_weight}) {
    if (weight->rank() != 1 || extent_of(*weight, 0) != extent) {
      refuse(name, "weights must have a head's extent");
    }
    validate_like(*weight, query, name);
  }
  if (!std::isfinite(epsilon) || epsilon <= 0.0) {
    refuse(name, "epsilon must be finite and positive");
  }
  const Rotation rotation{rotation_of(query, positions, frequencies, layout, magnitude, name)};
  const Tensor q{readable(query)}, k{readable(key)};
  const Tensor qw{query_weight.contiguous()}, kw{key_weight.contiguous()};
  const auto rows{[&](const Tensor& x) {
    return Tensor{Shape{x.shape()[0], x.shape()[1], x.shape()[2]}, x.dtype(), x.device()};
  }};
  Tensor q_output{ordered_like(q)}, k_output{ordered_like(k)};
  const Tensor q_rows{rows(q)}, k_rows{rows(k)};
  const SparHipHeadNorm parts[2]{{heads_of(q_output), first_element(q_rows), heads_of(q),
                                  first_element(qw), extent_of(q, 1)},
                                 {heads_of(k_output), first_element(k_rows), heads_of(k),
                                  first_element(kw), extent_of(k, 1)}};
  const SparHipRotary argument{rotation.argument()};
  hip::check(spar_hip_launch_head_norm_rotary_forward(parts, 2, batch, tokens, extent, &argument,
                                                      epsilon, hip::dtype_tag(query.dtype()),
                                                      query.device().index()),
             name, query.device());
  const bool tracked{q.requires_grad() || k.requires_grad() || query_weight.requires_grad() ||
                     key_weight.requires_grad()};
  const Rotation saved{tracked ? snapshot_of(rotation) : rotation};
  record_head_norm(q_output, q, query_weight, qw, q_rows, saved);
  record_head_norm(k_output, k, key_weight, kw, k_rows, saved);
  return {q_output, k_output};
}

Tensor window_attention(const Tensor& query, const Tensor& key, const Tensor& value,
                        std::size_t window, std::size_t sinks, std::optional<double> scale,
                        const std::optional<Tensor>& lengths) {
  constexpr const char* name{"window_attention"};
  validate_heads(query, name, "query");
  validate_heads(key, name, "key");
  validate_heads(value, name, "value");
  validate_like(key, query, name);
  validate_like(value, query, name);
  if (key.shape() != value.shape()) refuse(name, "key and value must have one shape");
  if (extent_of(key, 0) != extent_of(query, 0)) refuse(name, "key and query batches differ");
  const std::size_t extent{extent_of(query, 3)};
  if (extent_of(key, 3) != extent) refuse(name, "key and query extents differ");
  if (extent < 1 || extent > SPAR_HIP_ATTENTION_MAX_EXTENT) {
    refuse(name, "takes heads of 1 to 256 elements");
  }
  const std::size_t query_heads{extent_of(query, 1)}, key_heads{extent_of(key, 1)};
  if (key_heads == 0 || query_heads == 0 || query_heads % key_heads != 0) {
    refuse(name, "query heads must be a multiple of key heads");
  }
  if (scale && !std::isfinite(*scale)) refuse(name, "scale must be finite");
  std::optional<Tensor> tokens;
  if (lengths) {
    validate_integers(*lengths, query, name, "lengths");
    if (lengths->rank() != 1 || extent_of(*lengths, 0) != extent_of(query, 0)) {
      refuse(name, "lengths must be [batch]");
    }
    tokens = lengths->contiguous().detach();
  }
  const Tensor q{readable(query)}, k{readable(key)}, v{readable(value)};
  const bool grad_query{q.requires_grad()}, grad_key{k.requires_grad()},
      grad_value{v.requires_grad()};
  const bool tracked{grad_query || grad_key || grad_value};
  // The backward's own: the program may go on counting in its lengths.
  if (tokens && tracked) tokens = tokens->clone();
  Tensor output{ordered_like(q)};
  const Device device{query.device()};
  const SparHipAttention shape{
      extent_of(query, 0),
      query_heads,
      key_heads,
      extent_of(query, 2),
      extent_of(key, 2),
      extent,
      window,
      sinks,
      scale ? *scale : 1.0 / std::sqrt(static_cast<double>(extent)),
      tokens ? first_element(*tokens) : nullptr,
      tokens ? hip::dtype_tag(tokens->dtype()) : SPAR_HIP_INT32,
      hip::dtype_tag(query.dtype())};
  Tensor logsumexp{tracked ? Shape{query.shape()[0], query.shape()[1], query.shape()[2]}
                           : Shape{0},
                   query.dtype(), device};
  std::uint64_t bytes{0};
  hip::check(spar_hip_attention_workspace(&bytes, &shape, 0), name, device);
  Tensor workspace{Shape{static_cast<Shape::dimension_type>((bytes + 3) / 4)}, DType::Int32,
                   device};
  const SparHipHeads target{heads_of(output)}, q_heads{heads_of(q)}, k_heads{heads_of(k)},
      v_heads{heads_of(v)};
  hip::check(spar_hip_launch_attention_forward(&target, first_element(logsumexp), &q_heads,
                                               &k_heads, &v_heads, &shape,
                                               first_element(workspace), bytes, device.index()),
             name, device);
  if (tracked) {
    std::vector<Tensor> parents;
    if (grad_query) parents.push_back(q);
    if (grad_key) parents.push_back(k);
    if (grad_value) parents.push_back(v);
    auto saved{std::make_shared<const SavedAttention>(
        SavedAttention{q.detach(), k.detach(), v.detach(), output.detach(), logsumexp, tokens,
                       shape, grad_query, grad_key, grad_value})};
    detail::record_operation(output, std::move(parents), [saved](const Tensor& gradient) {
      return attention_backward(*saved, gradient);
    });
  }
  return output;
}

}  // namespace spar

// What the operators on heads share: their checks of arguments, heads as kernels read
// them, and the rotation's arguments.
#pragma once

#include <cmath>
#include <cstddef>
#include <stdexcept>
#include <string>

#include "bridge.hpp"
#include "spar/attention.hpp"

namespace spar::detail::heads {

inline std::size_t extent_of(const Tensor& tensor, std::size_t axis) {
  return static_cast<std::size_t>(tensor.shape()[axis]);
}

inline void* first_element(const Tensor& tensor) {
  if (tensor.numel() == 0) return nullptr;
  const auto* base{static_cast<const std::byte*>(HipTensorAccess::storage_base(tensor))};
  return const_cast<std::byte*>(base + tensor.storage_offset() * size_of(tensor.dtype()));
}

[[noreturn]] inline void refuse(const char* name, const char* what) {
  throw std::invalid_argument{std::string{name} + " " + what};
}

inline void validate_heads(const Tensor& tensor, const char* name, const char* which) {
  if (tensor.rank() != 4) {
    throw std::invalid_argument{std::string{name} + " " + which +
                                " must be [batch, heads, tokens, extent]"};
  }
  if (!is_floating(tensor.dtype())) refuse(name, "requires a floating-point dtype");
  require_hip(tensor, name);
}

inline void validate_like(const Tensor& tensor, const Tensor& heads, const char* name) {
  if (tensor.dtype() != heads.dtype()) refuse(name, "tensors must have one dtype");
  if (tensor.device() != heads.device()) refuse(name, "tensors are on different devices");
}

inline void validate_integers(const Tensor& tensor, const Tensor& heads, const char* name,
                              const char* which) {
  if (tensor.dtype() != DType::Int32 && tensor.dtype() != DType::Int64) {
    throw std::invalid_argument{std::string{name} + " " + which +
                                " must have Int32 or Int64 dtype"};
  }
  if (tensor.device() != heads.device()) refuse(name, "tensors are on different devices");
}

// The tensor as kernels read heads: itself where its last axis is contiguous.
inline Tensor readable(const Tensor& tensor) {
  if (tensor.numel() == 0) return tensor;
  return tensor.strides()[3] == 1 || tensor.shape()[3] == 1 ? tensor : tensor.contiguous();
}

inline SparHipHeads heads_of(const Tensor& tensor) {
  const auto strides{tensor.strides()};
  return {first_element(tensor), {strides[0], strides[1], strides[2]}};
}

// A new tensor of `like`'s shape whose tokens lie as `like`'s do: a token's heads
// side by side, or a head's tokens.
inline Tensor ordered_like(const Tensor& like) {
  const Shape& shape{like.shape()};
  if (like.strides()[2] > like.strides()[1]) {
    return Tensor{Shape{shape[0], shape[2], shape[1], shape[3]}, like.dtype(), like.device()}
        .transpose(1, 2);
  }
  return Tensor{shape, like.dtype(), like.device()};
}

// ----------------------------------------------------------------- rotation

struct Rotation {
  Tensor positions;  // contiguous tokens
  Tensor frequencies;
  std::size_t position_stride;
  double magnitude;
  RotaryLayout layout;

  [[nodiscard]] SparHipRotary argument() const {
    return {first_element(positions), position_stride, hip::dtype_tag(positions.dtype()),
            static_cast<const double*>(first_element(frequencies)), 2 * frequencies.numel(),
            magnitude,
            layout == RotaryLayout::Half ? SPAR_HIP_ROTARY_HALF : SPAR_HIP_ROTARY_INTERLEAVED};
  }
};

inline Rotation rotation_of(const Tensor& heads, const Tensor& positions, const Tensor& frequencies,
                     RotaryLayout layout, double magnitude, const char* name) {
  validate_integers(positions, heads, name, "positions");
  const std::size_t batch{extent_of(heads, 0)}, tokens{extent_of(heads, 2)};
  const bool shared{positions.rank() == 1};
  if (positions.rank() < 1 || positions.rank() > 2 ||
      extent_of(positions, positions.rank() - 1) != tokens ||
      (!shared && extent_of(positions, 0) != batch)) {
    refuse(name, "positions must be [tokens] or [batch, tokens]");
  }
  if (frequencies.rank() != 1 || frequencies.dtype() != DType::Float64) {
    refuse(name, "frequencies must be a Float64 vector");
  }
  if (frequencies.requires_grad()) refuse(name, "frequencies must not require gradients");
  if (frequencies.device() != heads.device()) refuse(name, "tensors are on different devices");
  if (2 * frequencies.numel() > extent_of(heads, 3)) {
    refuse(name, "frequencies turn more elements than a head has");
  }
  if (!std::isfinite(magnitude)) refuse(name, "magnitude must be finite");
  if (layout != RotaryLayout::Half && layout != RotaryLayout::Interleaved) {
    refuse(name, "received an unknown RotaryLayout");
  }
  const bool dense{positions.numel() <= 1 || tokens == 1 ||
                   positions.strides()[positions.rank() - 1] == 1};
  const Tensor read{dense ? positions : positions.contiguous()};
  return {read.detach(), frequencies.contiguous().detach(),
          shared ? 0 : static_cast<std::size_t>(read.strides()[0]), magnitude, layout};
}

}  // namespace spar::detail::heads

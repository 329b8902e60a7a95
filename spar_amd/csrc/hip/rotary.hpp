// What the kernels that turn heads by their positions share: a lane's share of a head,
// its loads and stores, cos and sin, and the rows of a launch.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"

namespace spar_hip {
namespace rotary {

constexpr int kThreads = 256;

// A lane's share of a head: four pairs, or eight elements behind the pairs, as
// two runs of up to four neighbours.
struct Unit {
  uint32_t first, second;              // elements the runs start at
  uint32_t first_count, second_count;  // their lengths
  uint32_t pair;                       // of the first pair; kPassed: not turned
};
constexpr uint32_t kPassed = ~0U;

__host__ __device__ inline uint32_t turning_units(uint32_t half) { return (half + 3) / 4; }
__host__ __device__ inline uint32_t units_of(uint32_t half, uint32_t extent) {
  return turning_units(half) + (extent - 2 * half + 7) / 8;
}

__device__ __forceinline__ uint32_t at_most_4(uint32_t n) { return n < 4 ? n : 4; }

template <bool HALF>
__device__ __forceinline__ Unit unit_at(uint32_t u, uint32_t half, uint32_t extent) {
  Unit unit;
  const uint32_t turning = turning_units(half);
  uint32_t end;
  if (u < turning) {
    unit.pair = 4 * u;
    if constexpr (HALF) {
      unit.first = unit.pair;
      unit.second = unit.pair + half;
      unit.first_count = unit.second_count = at_most_4(half - unit.pair);
      return unit;
    }
    unit.first = 2 * unit.pair;
    end = 2 * half;
  } else {
    unit.pair = kPassed;
    unit.first = 2 * half + 8 * (u - turning);
    end = extent;
  }
  unit.second = unit.first + 4;
  unit.first_count = at_most_4(end - unit.first);
  unit.second_count = unit.second < end ? at_most_4(end - unit.second) : 0;
  return unit;
}

template <typename T, bool NT>
__device__ __forceinline__ void load_run(T (&x)[8], int at, const T* source, uint32_t count) {
  constexpr int W = Vec16<T>::width;
  if (count == 4) {
#pragma unroll
    for (int i = 0; i < 4; i += W) {
      typename Vec16<T>::type v;
      if constexpr (NT) {
        v = __builtin_nontemporal_load(
            reinterpret_cast<const typename Loose16<T>::type*>(source + i));
      } else {
        v = loose_load(source + i);
      }
#pragma unroll
      for (int k = 0; k < W; ++k) x[at + i + k] = v[k];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[at + i] = static_cast<uint32_t>(i) < count ? source[i] : T(0);
  }
}

template <typename T, bool NT>
__device__ __forceinline__ void store_run(T* target, const T (&x)[8], int at, uint32_t count) {
  constexpr int W = Vec16<T>::width;
  if (count == 4) {
#pragma unroll
    for (int i = 0; i < 4; i += W) {
      typename Vec16<T>::type v;
#pragma unroll
      for (int k = 0; k < W; ++k) v[k] = x[at + i + k];
      loose_store<NT, T>(target + i, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (static_cast<uint32_t>(i) < count) target[i] = x[at + i];
    }
  }
}

template <typename T, bool NT>
__device__ __forceinline__ void load_unit(T (&x)[8], const T* head, const Unit& unit) {
  load_run<T, NT>(x, 0, head + unit.first, unit.first_count);
  load_run<T, NT>(x, 4, head + unit.second, unit.second_count);
}

template <typename T, bool NT>
__device__ __forceinline__ void store_unit(T* head, const T (&x)[8], const Unit& unit) {
  store_run<T, NT>(head + unit.first, x, 0, unit.first_count);
  store_run<T, NT>(head + unit.second, x, 4, unit.second_count);
}

// cos and sin of an angle in double.  For float32 the angle is reduced to
// [-pi/4, pi/4] in double -- n * (pi/2) as the product with pi/2's first 53 bits,
// exact in the fused subtraction, and its next 53 -- and evaluated in single:
// the reduced angle's rounding costs 2^-25, as rounding the result does.
__device__ __forceinline__ void cos_sin(double angle, float& c, float& s) {
  if (!(fabs(angle) < 0x1p30)) {
    double dc, ds;
    sincos(angle, &ds, &dc);
    c = static_cast<float>(dc);
    s = static_cast<float>(ds);
    return;
  }
  const double n = rint(angle * 0.63661977236758134308);
  const double reduced =
      __builtin_fma(-n, 0x1.1a62633145c07p-54, __builtin_fma(-n, 0x1.921fb54442d18p+0, angle));
  float rs, rc;
  sincosf(static_cast<float>(reduced), &rs, &rc);
  const int quarter = static_cast<int>(n) & 3;
  const float swapped_c = (quarter & 1) ? rs : rc;
  const float swapped_s = (quarter & 1) ? rc : rs;
  c = (quarter == 1 || quarter == 2) ? -swapped_c : swapped_c;
  s = (quarter & 2) ? -swapped_s : swapped_s;
}

__device__ __forceinline__ void cos_sin(double angle, double& c, double& s) {
  sincos(angle, &s, &c);
}

template <typename T>
struct Heads {
  T* data;
  uint64_t batch, head, token;  // strides
};

template <typename T>
Heads<T> heads_of(const SparHipHeads& heads) {
  return {static_cast<T*>(heads.data), heads.strides[0], heads.strides[1], heads.strides[2]};
}

// The rotation and the shape every head of the call shares.
struct Turn {
  const void* positions;
  uint64_t position_stride;
  const double* frequencies;
  double magnitude;
  uint32_t half;
  uint32_t extent;
  bool wide_positions;  // Int64
  bool inverse;
};

// cos and sin of a unit's four pairs for one token, times the magnitude.
template <typename T>
__device__ __forceinline__ void unit_turn(const Turn& turn, const Unit& unit, uint64_t b,
                                          uint64_t t, T (&c)[4], T (&s)[4]) {
  if (unit.pair == kPassed) return;
  const uint64_t at = b * turn.position_stride + t;
  const double position =
      turn.wide_positions
          ? static_cast<double>(static_cast<const int64_t*>(turn.positions)[at])
          : static_cast<double>(static_cast<const int32_t*>(turn.positions)[at]);
  const T magnitude = static_cast<T>(turn.magnitude);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (unit.pair + i < turn.half) {
      cos_sin(position * turn.frequencies[unit.pair + i], c[i], s[i]);
      c[i] *= magnitude;
      s[i] *= turn.inverse ? -magnitude : magnitude;
    } else {
      c[i] = s[i] = T(0);
    }
  }
}

template <typename T, bool HALF>
__device__ __forceinline__ void turn_unit(T (&x)[8], const Unit& unit, const T (&c)[4],
                                          const T (&s)[4]) {
  if (unit.pair == kPassed) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int a = HALF ? i : 2 * i, b = HALF ? i + 4 : 2 * i + 1;
    const T first = x[a], second = x[b];
    x[a] = first * c[i] - second * s[i];
    x[b] = second * c[i] + first * s[i];
  }
}

// Rows (one token of one sequence) of a launch: the quotient by the sequence
// length in 32 bits where all rows allow it.
struct Rows {
  uint64_t first;  // row of the launch's first
  uint64_t tokens;
  FastDiv by_tokens;
  bool narrow;

  __device__ __forceinline__ void split(uint64_t row, uint64_t& b, uint64_t& t) const {
    if (narrow) {
      const uint32_t at = static_cast<uint32_t>(first + row);
      const uint32_t q = by_tokens.div(at);
      b = q;
      t = at - q * by_tokens.divisor;
    } else {
      b = (first + row) / tokens;
      t = (first + row) - b * tokens;
    }
  }
};

// ---------------------------------------------------------------- launchers

// Heads a lane turns with one cos and sin: as many as leave the chip full.
constexpr uint64_t kFullLanes = 1 << 16;

inline bool valid_rotary(const SparHipRotary* rotary, uint64_t extent) {
  return rotary != nullptr && rotary->rotary_extent % 2 == 0 && rotary->rotary_extent <= extent &&
         std::isfinite(rotary->magnitude) &&
         (rotary->layout == SPAR_HIP_ROTARY_HALF ||
          rotary->layout == SPAR_HIP_ROTARY_INTERLEAVED) &&
         (rotary->position_dtype == SPAR_HIP_INT32 || rotary->position_dtype == SPAR_HIP_INT64);
}

inline bool complete_rotary(const SparHipRotary* rotary) {
  return rotary->rotary_extent == 0 ||
         (rotary->positions != nullptr && rotary->frequencies != nullptr);
}

inline Turn turn_of(const SparHipRotary& rotary, uint64_t extent, bool inverse) {
  return {rotary.positions, rotary.position_stride, rotary.frequencies, rotary.magnitude,
          static_cast<uint32_t>(rotary.rotary_extent / 2), static_cast<uint32_t>(extent),
          rotary.position_dtype == SPAR_HIP_INT64, inverse};
}

inline bool overflows(uint64_t a, uint64_t b) { return b != 0 && a > UINT64_MAX / b; }

// The largest of a call's extents, far beyond memory, so that products of two
// fit 64 bits and a head's element index 32.
inline bool sane(uint64_t batch, uint64_t heads, uint64_t tokens, uint64_t extent) {
  return heads < (uint64_t{1} << 24) && extent < (uint64_t{1} << 24) &&
         tokens < (uint64_t{1} << 40) && !overflows(batch, tokens) &&
         batch * tokens < (uint64_t{1} << 56);
}

inline Rows rows_at(uint64_t first, uint64_t batch, uint64_t tokens) {
  Rows rows{};
  rows.first = first;
  rows.tokens = tokens;
  rows.narrow = batch * tokens <= kIndex32Limit;
  if (rows.narrow) rows.by_tokens.init(static_cast<uint32_t>(tokens));
  return rows;
}

}  // namespace rotary
}  // namespace spar_hip

// Rotary positions, alone and behind a per-head RMSNorm.
//
// A head's first r elements form r / 2 pairs (a, b); the rotation by the angle
// t = position * frequency[pair], times a magnitude m, is
//   a' = m (a cos t - b sin t),  b' = m (b cos t + a sin t),
// and its transpose (the gradient) the same with -t.  The fused form turns
// y = x / d * w, d = sqrt(mean(x * x) + eps), whose gradient for g = turned back
// output gradient, h = x / d is
//   dw = sum g h,  dx = (g w - h mean(g w h)) / d.
//
// All of it is bound by memory: an element takes about four operations per
// eight to twelve bytes.  What the layouts follow from is the price of cos and
// sin, about 40 instructions per pair: they are computed in the kernel, from an
// angle in double, by lanes that keep them for several heads of one token, so
// that there is no table to read, to size or to keep.  The reference computes
// them in double for every element (cuda_kernels.cu:663-687).
#include <hip/hip_runtime.h>

#include <cmath>

#include "common.hpp"

namespace spar_hip {
namespace {

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

// A lane per unit of K heads of one token (heads `groups` apart, so that lanes
// next to each other read neighbouring heads): cos and sin once for the K.
template <typename T, bool HALF, bool NT, int K>
__global__ __launch_bounds__(kThreads) void rotary_kernel(Heads<T> output, Heads<const T> input,
                                                          Turn turn, Rows rows, uint32_t items,
                                                          FastDiv by_units, FastDiv by_groups,
                                                          uint32_t heads) {
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x;
  if (item >= items) return;
  const uint32_t group_item = by_units.div(item);
  const Unit unit =
      unit_at<HALF>(item - group_item * by_units.divisor, turn.half, turn.extent);
  const uint32_t row = by_groups.div(group_item);
  const uint32_t group = group_item - row * by_groups.divisor;
  uint64_t b, t;
  rows.split(row, b, t);
  const T* source = input.data + b * input.batch + t * input.token;
  T* target = output.data + b * output.batch + t * output.token;
  T x[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t head = group + k * by_groups.divisor;
    if (head < heads) load_unit<T, NT>(x[k], source + head * input.head, unit);
  }
  T c[4], s[4];
  unit_turn(turn, unit, b, t, c, s);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t head = group + k * by_groups.divisor;
    if (head < heads) {
      turn_unit<T, HALF>(x[k], unit, c, s);
      store_unit<T, NT>(target + head * output.head, x[k], unit);
    }
  }
}

// ------------------------------------------------------ head norm and rotation

template <typename T>
struct NormPart {
  Heads<T> output;
  T* denominator;
  Heads<const T> input;
  const T* weight;
};

template <typename T>
struct NormParts {
  NormPart<T> part[2];
  uint32_t heads[2];  // of each; heads[1] is 0 for one part
};

template <typename T, int LANES>
__device__ __forceinline__ T group_sum(T value) {
#pragma unroll
  for (int mask = LANES / 2; mask > 0; mask >>= 1) value += __shfl_xor(value, mask, kWave);
  return value;
}

template <typename T>
__device__ __forceinline__ T square_sum(const T (&x)[8]) {
  return ((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) +
         ((x[4] * x[4] + x[5] * x[5]) + (x[6] * x[6] + x[7] * x[7]));
}

// LANES lanes per head, a unit each (none where a head has fewer), for K heads
// of one token: the heads of both parts counted through, so that a token's
// queries and keys share cos, sin and the launch.
template <typename T, bool HALF, bool NT, int LANES, int K>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(NormParts<T> parts, Turn turn,
                                                                Rows rows, uint32_t items,
                                                                uint32_t units, FastDiv by_groups,
                                                                T epsilon) {
  const uint32_t item = (blockIdx.x * kThreads + threadIdx.x) / LANES;
  const uint32_t u = threadIdx.x % LANES;
  if (item >= items) return;
  const uint32_t row = by_groups.div(item);
  const uint32_t group = item - row * by_groups.divisor;
  uint64_t b, t;
  rows.split(row, b, t);
  const bool holds = u < units;
  Unit unit{0, 0, 0, 0, kPassed};
  if (holds) unit = unit_at<HALF>(u, turn.half, turn.extent);
  const uint32_t heads = parts.heads[0] + parts.heads[1];
  T x[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t head = group + k * by_groups.divisor;
    if (head < heads) {
      const bool other = head >= parts.heads[0];
      const NormPart<T>& part = parts.part[other ? 1 : 0];
      const uint32_t own = other ? head - parts.heads[0] : head;
      load_unit<T, NT>(x[k], part.input.data + b * part.input.batch + t * part.input.token +
                                 own * part.input.head, unit);
    }
  }
  T c[4], s[4];
  unit_turn(turn, unit, b, t, c, s);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t head = group + k * by_groups.divisor;
    if (head >= heads) break;  // the same for all lanes of a head
    const bool other = head >= parts.heads[0];
    const NormPart<T>& part = parts.part[other ? 1 : 0];
    const uint32_t own = other ? head - parts.heads[0] : head;
    const T mean = group_sum<T, LANES>(square_sum(x[k])) / static_cast<T>(turn.extent);
    const T d = sqrt(mean + epsilon);
    const T over = T(1) / d;
    if (u == 0 && part.denominator != nullptr) {
      part.denominator[(b * parts.heads[other ? 1 : 0] + own) * rows.tokens + t] = d;
    }
    T w[8];
    load_unit<T, false>(w, part.weight, unit);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[k][i] = (x[k][i] * over) * w[i];
    turn_unit<T, HALF>(x[k], unit, c, s);
    store_unit<T, NT>(part.output.data + b * part.output.batch + t * part.output.token +
                          own * part.output.head, x[k], unit);
  }
}

template <typename T>
struct NormGradientPart {
  Heads<T> input_gradient;
  Heads<const T> output_gradient;
  Heads<const T> input;
  const T* weight;
  const T* denominator;
};

template <typename T>
struct NormGradientParts {
  NormGradientPart<T> part[2];
  uint32_t heads[2];
};

// The same lanes walk the rows in a grid-stride; each keeps the weight gradients
// of its unit for both parts, which the workgroup adds up at the end into one
// row [2, extent] of `partials`.
template <typename T, bool HALF, bool NT, int LANES, int K>
__global__ __launch_bounds__(kThreads) void norm_backward_kernel(NormGradientParts<T> parts,
                                                                 Turn turn, Rows rows,
                                                                 uint64_t items, uint32_t units,
                                                                 uint32_t groups, T* partials) {
  constexpr uint32_t kGroups = kThreads / LANES;
  const uint32_t u = threadIdx.x % LANES;
  const bool holds = u < units;
  Unit unit{0, 0, 0, 0, kPassed};
  if (holds) unit = unit_at<HALF>(u, turn.half, turn.extent);
  const uint32_t heads = parts.heads[0] + parts.heads[1];
  const T per_extent = T(1) / static_cast<T>(turn.extent);
  T sums[2][8] = {};
  // Items of a group lie a stride apart: its row and head group advance by the
  // stride's quotient and remainder, with no division in the loop.
  const uint64_t stride = static_cast<uint64_t>(gridDim.x) * kGroups;
  uint64_t item = static_cast<uint64_t>(blockIdx.x) * kGroups + threadIdx.x / LANES;
  uint64_t row = item / groups;
  uint32_t group = static_cast<uint32_t>(item - row * groups);
  const uint64_t row_step = stride / groups;
  const uint32_t group_step = static_cast<uint32_t>(stride - row_step * groups);
  for (; item < items; item += stride) {
    uint64_t b, t;
    rows.split(row, b, t);
    T c[4], s[4];
    T x[K][8], g[K][8];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t head = group + k * groups;
      if (head < heads) {
        const bool other = head >= parts.heads[0];
        const NormGradientPart<T>& part = parts.part[other ? 1 : 0];
        const uint32_t own = other ? head - parts.heads[0] : head;
        load_unit<T, NT>(x[k], part.input.data + b * part.input.batch + t * part.input.token +
                                   own * part.input.head, unit);
        load_unit<T, NT>(g[k], part.output_gradient.data + b * part.output_gradient.batch +
                                   t * part.output_gradient.token +
                                   own * part.output_gradient.head, unit);
      }
    }
    unit_turn(turn, unit, b, t, c, s);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t head = group + k * groups;
      if (head >= heads) break;
      const bool other = head >= parts.heads[0];
      const NormGradientPart<T>& part = parts.part[other ? 1 : 0];
      const uint32_t own = other ? head - parts.heads[0] : head;
      const T over =
          T(1) / part.denominator[(b * parts.heads[other ? 1 : 0] + own) * rows.tokens + t];
      turn_unit<T, HALF>(g[k], unit, c, s);
      T w[8];
      load_unit<T, false>(w, part.weight, unit);
      T dot = T(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[k][i] *= over;
        const T gx = g[k][i] * x[k][i];
        sums[0][i] += other ? T(0) : gx;
        sums[1][i] += other ? gx : T(0);
        g[k][i] *= w[i];
        dot += g[k][i] * x[k][i];
      }
      const T mean = group_sum<T, LANES>(dot) * per_extent;
#pragma unroll
      for (int i = 0; i < 8; ++i) g[k][i] = (g[k][i] - x[k][i] * mean) * over;
      store_unit<T, NT>(part.input_gradient.data + b * part.input_gradient.batch +
                            t * part.input_gradient.token + own * part.input_gradient.head,
                        g[k], unit);
    }
    row += row_step;
    group += group_step;
    if (group >= groups) {
      group -= groups;
      ++row;
    }
  }
  // Across the wave's groups, then across its workgroup's waves.
#pragma unroll
  for (int mask = kWave / 2; mask >= LANES; mask >>= 1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sums[0][i] += __shfl_xor(sums[0][i], mask, kWave);
      sums[1][i] += __shfl_xor(sums[1][i], mask, kWave);
    }
  }
  constexpr int kWaves = kThreads / kWave;
  __shared__ T shared[kWaves][2][LANES][9];
  const int wave = threadIdx.x / kWave;
  if (threadIdx.x % kWave < LANES) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      shared[wave][0][u][i] = sums[0][i];
      shared[wave][1][u][i] = sums[1][i];
    }
  }
  __syncthreads();
  if (wave < 2 && threadIdx.x % kWave < LANES && holds) {
    T total[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      total[i] = shared[0][wave][u][i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) total[i] += shared[w][wave][u][i];
    }
    store_unit<T, false>(
        partials + (static_cast<uint64_t>(blockIdx.x) * 2 + wave) * turn.extent, total, unit);
  }
}

// Columns of the partial rows added up in their order: 16 columns per workgroup,
// 64 lanes to a column, each a run of rows, then the runs in a tree.
template <typename T>
__global__ __launch_bounds__(1024) void norm_weight_kernel(T* first, T* second, const T* partials,
                                                           uint32_t rows, uint32_t extent) {
  __shared__ T shared[64][17];
  const uint32_t lane = threadIdx.x % 16, run = threadIdx.x / 16;
  const uint32_t column = blockIdx.x * 16 + lane;
  const uint32_t per = (rows + 63) / 64;
  T sum = T(0);
  if (column < 2 * extent) {
    const uint32_t begin = run * per, end = begin + per < rows ? begin + per : rows;
#pragma unroll 4
    for (uint32_t r = begin; r < end; ++r) {
      sum += partials[static_cast<uint64_t>(r) * 2 * extent + column];
    }
  }
  shared[run][lane] = sum;
  for (uint32_t half = 32; half > 0; half >>= 1) {
    __syncthreads();
    if (run < half) shared[run][lane] += shared[run + half][lane];
  }
  if (run == 0 && column < 2 * extent) {
    T* target = column < extent ? first : second;
    if (target != nullptr) target[column < extent ? column : column - extent] = shared[0][lane];
  }
}

// ---------------------------------------------------------------- launchers

// Heads a lane turns with one cos and sin: as many as leave the chip full.
constexpr uint64_t kFullLanes = 256 * 2048;

bool valid_rotary(const SparHipRotary* rotary, uint64_t extent) {
  return rotary != nullptr && rotary->rotary_extent % 2 == 0 && rotary->rotary_extent <= extent &&
         std::isfinite(rotary->magnitude) &&
         (rotary->layout == SPAR_HIP_ROTARY_HALF ||
          rotary->layout == SPAR_HIP_ROTARY_INTERLEAVED) &&
         (rotary->position_dtype == SPAR_HIP_INT32 || rotary->position_dtype == SPAR_HIP_INT64);
}

bool complete_rotary(const SparHipRotary* rotary) {
  return rotary->rotary_extent == 0 ||
         (rotary->positions != nullptr && rotary->frequencies != nullptr);
}

Turn turn_of(const SparHipRotary& rotary, uint64_t extent, bool inverse) {
  return {rotary.positions, rotary.position_stride, rotary.frequencies, rotary.magnitude,
          static_cast<uint32_t>(rotary.rotary_extent / 2), static_cast<uint32_t>(extent),
          rotary.position_dtype == SPAR_HIP_INT64, inverse};
}

bool overflows(uint64_t a, uint64_t b) { return b != 0 && a > UINT64_MAX / b; }

// The largest of a call's extents, far beyond memory, so that products of two
// fit 64 bits and a head's element index 32.
bool sane(uint64_t batch, uint64_t heads, uint64_t tokens, uint64_t extent) {
  return heads < (uint64_t{1} << 24) && extent < (uint64_t{1} << 24) &&
         tokens < (uint64_t{1} << 40) && !overflows(batch, tokens) &&
         batch * tokens < (uint64_t{1} << 56);
}

Rows rows_at(uint64_t first, uint64_t batch, uint64_t tokens) {
  Rows rows{};
  rows.first = first;
  rows.tokens = tokens;
  rows.narrow = batch * tokens <= kIndex32Limit;
  if (rows.narrow) rows.by_tokens.init(static_cast<uint32_t>(tokens));
  return rows;
}

template <typename T, bool HALF, bool NT, int K>
void launch_rotary(const SparHipHeads& output, const SparHipHeads& input, uint64_t batch,
                   uint32_t heads, uint64_t tokens, const Turn& turn, hipStream_t stream) {
  const uint32_t units = units_of(turn.half, turn.extent);
  const uint32_t groups = (heads + K - 1) / K;
  FastDiv by_units, by_groups;
  by_units.init(units);
  by_groups.init(groups);
  const uint64_t per_row = static_cast<uint64_t>(units) * groups;
  const uint64_t most = kIndex32Limit / per_row;  // rows of one launch
  for (uint64_t first = 0, all = batch * tokens; first < all; first += most) {
    const uint64_t count = all - first < most ? all - first : most;
    const uint32_t items = static_cast<uint32_t>(count * per_row);
    rotary_kernel<T, HALF, NT, K><<<ceil_div_u32(items, kThreads), kThreads, 0, stream>>>(
        heads_of<T>(output), heads_of<const T>(input), turn, rows_at(first, batch, tokens), items,
        by_units, by_groups, heads);
  }
}

template <typename T>
void start_rotary(const SparHipHeads& output, const SparHipHeads& input, uint64_t batch,
                  uint32_t heads, uint64_t tokens, const Turn& turn, int layout,
                  hipStream_t stream) {
  const uint64_t lanes = batch * tokens * units_of(turn.half, turn.extent) * heads;
  const bool stream_out =
      stream_output(batch * tokens * heads * static_cast<uint64_t>(turn.extent) * sizeof(T));
  constexpr int kMany = 16 / sizeof(T);
  with_policy(layout == SPAR_HIP_ROTARY_HALF, [&](auto half) {
    with_policy(stream_out, [&](auto nt) {
      if (lanes >= kMany * kFullLanes) {
        launch_rotary<T, decltype(half)::value, decltype(nt)::value, kMany>(
            output, input, batch, heads, tokens, turn, stream);
      } else {
        launch_rotary<T, decltype(half)::value, decltype(nt)::value, 1>(output, input, batch,
                                                                        heads, tokens, turn, stream);
      }
    });
  });
}

// Lanes to a head: the power of two that holds its units.
template <typename Body>
void with_lanes(uint32_t units, Body&& body) {
  if (units <= 8) {
    body(std::integral_constant<int, 8>{});
  } else if (units <= 16) {
    body(std::integral_constant<int, 16>{});
  } else if (units <= 32) {
    body(std::integral_constant<int, 32>{});
  } else {
    body(std::integral_constant<int, 64>{});
  }
}
static_assert((SPAR_HIP_HEAD_NORM_MAX_EXTENT + 7) / 8 + 1 <= kWave);

template <typename T, bool HALF, bool NT, int LANES, int K>
void launch_norm_forward(const NormParts<T>& parts, uint64_t batch, uint64_t tokens,
                         const Turn& turn, double epsilon, hipStream_t stream) {
  const uint32_t heads = parts.heads[0] + parts.heads[1];
  const uint32_t groups = (heads + K - 1) / K;
  FastDiv by_groups;
  by_groups.init(groups);
  const uint64_t most = (kIndex32Limit / LANES - kThreads) / groups;
  for (uint64_t first = 0, all = batch * tokens; first < all; first += most) {
    const uint64_t count = all - first < most ? all - first : most;
    const uint32_t items = static_cast<uint32_t>(count * groups);
    norm_forward_kernel<T, HALF, NT, LANES, K>
        <<<ceil_div_u32(static_cast<uint64_t>(items) * LANES, kThreads), kThreads, 0, stream>>>(
            parts, turn, rows_at(first, batch, tokens), items,
            units_of(turn.half, turn.extent), by_groups, static_cast<T>(epsilon));
  }
}

template <typename T>
void start_norm_forward(const SparHipHeadNorm* parts, int part_count, uint64_t batch,
                        uint64_t tokens, const Turn& turn, int layout, double epsilon,
                        hipStream_t stream) {
  NormParts<T> all{};
  for (int p = 0; p < part_count; ++p) {
    all.part[p] = {heads_of<T>(parts[p].output), static_cast<T*>(parts[p].denominator),
                   heads_of<const T>(parts[p].input), static_cast<const T*>(parts[p].weight)};
    all.heads[p] = static_cast<uint32_t>(parts[p].heads);
  }
  const uint64_t heads = static_cast<uint64_t>(all.heads[0]) + all.heads[1];
  const bool stream_out = stream_output(batch * tokens * heads * turn.extent * sizeof(T));
  with_policy(layout == SPAR_HIP_ROTARY_HALF, [&](auto half) {
    with_policy(stream_out, [&](auto nt) {
      with_lanes(units_of(turn.half, turn.extent), [&](auto lanes) {
        constexpr int kLanes = decltype(lanes)::value;
        constexpr int kMany = 16 / sizeof(T);
        if (batch * tokens * heads * kLanes >= kMany * kFullLanes) {
          launch_norm_forward<T, decltype(half)::value, decltype(nt)::value, kLanes, kMany>(
              all, batch, tokens, turn, epsilon, stream);
        } else {
          launch_norm_forward<T, decltype(half)::value, decltype(nt)::value, kLanes, 1>(
              all, batch, tokens, turn, epsilon, stream);
        }
      });
    });
  });
}

// Workgroups of the backward, one row of partial weight gradients each: as many
// as the heads fill, at most four per CU.
constexpr uint64_t kMostPartials = 1024;

uint32_t partial_rows(uint64_t batch, uint64_t tokens, uint64_t heads) {
  const uint64_t wanted = (batch * tokens * heads + 7) / 8;
  return static_cast<uint32_t>(wanted < kMostPartials ? wanted : kMostPartials);
}

template <typename T>
void start_norm_backward(const SparHipHeadNormGradient* parts, int part_count, uint64_t batch,
                         uint64_t tokens, const Turn& turn, int layout, void* workspace,
                         hipStream_t stream) {
  NormGradientParts<T> all{};
  for (int p = 0; p < part_count; ++p) {
    all.part[p] = {heads_of<T>(parts[p].input_gradient),
                   heads_of<const T>(parts[p].output_gradient), heads_of<const T>(parts[p].input),
                   static_cast<const T*>(parts[p].weight),
                   static_cast<const T*>(parts[p].denominator)};
    all.heads[p] = static_cast<uint32_t>(parts[p].heads);
  }
  const uint32_t heads = all.heads[0] + all.heads[1];
  const uint32_t partials = partial_rows(batch, tokens, heads);
  const uint32_t units = units_of(turn.half, turn.extent);
  const bool stream_out =
      stream_output(batch * tokens * heads * static_cast<uint64_t>(turn.extent) * sizeof(T));
  if (partials > 0) {
    with_policy(layout == SPAR_HIP_ROTARY_HALF, [&](auto half) {
      with_policy(stream_out, [&](auto nt) {
        with_lanes(units, [&](auto lanes) {
          constexpr int kLanes = decltype(lanes)::value;
          constexpr int kMany = 8 / sizeof(T);
          const auto launch = [&](auto many) {
            constexpr int K = decltype(many)::value;
            const uint32_t groups = (heads + K - 1) / K;
            norm_backward_kernel<T, decltype(half)::value, decltype(nt)::value, kLanes, K>
                <<<partials, kThreads, 0, stream>>>(all, turn, rows_at(0, batch, tokens),
                                                    batch * tokens * groups, units, groups,
                                                    static_cast<T*>(workspace));
          };
          if (batch * tokens * heads * kLanes >= kMany * kMostPartials * kThreads) {
            launch(std::integral_constant<int, kMany>{});
          } else {
            launch(std::integral_constant<int, 1>{});
          }
        });
      });
    });
  }
  norm_weight_kernel<T><<<ceil_div_u32(2 * turn.extent, 16), 1024, 0, stream>>>(
      static_cast<T*>(parts[0].weight_gradient),
      part_count > 1 ? static_cast<T*>(parts[1].weight_gradient) : nullptr,
      static_cast<const T*>(workspace), partials, turn.extent);
}

bool valid_head_norm(int part_count, uint64_t extent, const SparHipRotary* rotary, int dtype) {
  return part_count >= 1 && part_count <= 2 && extent >= 1 &&
         extent <= SPAR_HIP_HEAD_NORM_MAX_EXTENT && valid_rotary(rotary, extent) &&
         valid_float_dtype(dtype);
}

}  // namespace
}  // namespace spar_hip

using namespace spar_hip;

extern "C" SparHipStatus spar_hip_launch_rotary(const SparHipHeads* output,
                                                const SparHipHeads* input, uint64_t batch,
                                                uint64_t heads, uint64_t tokens, uint64_t extent,
                                                const SparHipRotary* rotary, int inverse,
                                                int dtype, int device) {
  if (!valid_float_dtype(dtype) || !valid_rotary(rotary, extent) || inverse < 0 || inverse > 1 ||
      !sane(batch, heads, tokens, extent)) {
    return invalid();
  }
  if (batch == 0 || heads == 0 || tokens == 0 || extent == 0) return ok();
  if (output == nullptr || input == nullptr || output->data == nullptr ||
      input->data == nullptr || !complete_rotary(rotary)) {
    return invalid();
  }
  const Turn turn = turn_of(*rotary, extent, inverse != 0);
  if (overflows(units_of(turn.half, turn.extent), heads) ||
      units_of(turn.half, turn.extent) * heads > kIndex32Limit / 2) {
    return invalid();
  }
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  if (dtype == SPAR_HIP_FLOAT32) {
    start_rotary<float>(*output, *input, batch, static_cast<uint32_t>(heads), tokens, turn,
                        rotary->layout, guard.stream);
  } else {
    start_rotary<double>(*output, *input, batch, static_cast<uint32_t>(heads), tokens, turn,
                         rotary->layout, guard.stream);
  }
  return finish(guard);
}

extern "C" SparHipStatus spar_hip_launch_head_norm_rotary_forward(
    const SparHipHeadNorm* parts, int part_count, uint64_t batch, uint64_t tokens, uint64_t extent,
    const SparHipRotary* rotary, double epsilon, int dtype, int device) {
  if (!valid_head_norm(part_count, extent, rotary, dtype) || parts == nullptr ||
      !std::isfinite(epsilon) || epsilon <= 0.0) {
    return invalid();
  }
  uint64_t heads = 0;
  for (int p = 0; p < part_count; ++p) {
    if (!sane(batch, parts[p].heads, tokens, extent)) return invalid();
    heads += parts[p].heads;
  }
  if (batch == 0 || tokens == 0 || heads == 0) return ok();
  if (!complete_rotary(rotary)) return invalid();
  for (int p = 0; p < part_count; ++p) {
    if (parts[p].heads != 0 && (parts[p].output.data == nullptr ||
                                parts[p].input.data == nullptr || parts[p].weight == nullptr)) {
      return invalid();
    }
  }
  const Turn turn = turn_of(*rotary, extent, false);
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  if (dtype == SPAR_HIP_FLOAT32) {
    start_norm_forward<float>(parts, part_count, batch, tokens, turn, rotary->layout, epsilon,
                              guard.stream);
  } else {
    start_norm_forward<double>(parts, part_count, batch, tokens, turn, rotary->layout, epsilon,
                               guard.stream);
  }
  return finish(guard);
}

extern "C" SparHipStatus spar_hip_head_norm_rotary_workspace(uint64_t* bytes, uint64_t batch,
                                                             uint64_t tokens, uint64_t heads,
                                                             uint64_t extent, int dtype) {
  if (bytes == nullptr || !valid_float_dtype(dtype) || extent < 1 ||
      extent > SPAR_HIP_HEAD_NORM_MAX_EXTENT || !sane(batch, heads, tokens, extent)) {
    return invalid();
  }
  *bytes = static_cast<uint64_t>(partial_rows(batch, tokens, heads)) * 2 * extent *
           (dtype == SPAR_HIP_FLOAT32 ? sizeof(float) : sizeof(double));
  return ok();
}

extern "C" SparHipStatus spar_hip_launch_head_norm_rotary_backward(
    const SparHipHeadNormGradient* parts, int part_count, uint64_t batch, uint64_t tokens,
    uint64_t extent, const SparHipRotary* rotary, void* workspace, uint64_t workspace_bytes,
    int dtype, int device) {
  if (!valid_head_norm(part_count, extent, rotary, dtype) || parts == nullptr) return invalid();
  uint64_t heads = 0;
  for (int p = 0; p < part_count; ++p) {
    if (!sane(batch, parts[p].heads, tokens, extent) || parts[p].weight_gradient == nullptr) {
      return invalid();
    }
    heads += parts[p].heads;
  }
  const bool empty = batch == 0 || tokens == 0 || heads == 0;
  if (!empty) {
    uint64_t need = 0;
    const SparHipStatus status =
        spar_hip_head_norm_rotary_workspace(&need, batch, tokens, heads, extent, dtype);
    if (status.code != 0) return status;
    if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace) ||
        !complete_rotary(rotary)) {
      return invalid();
    }
    for (int p = 0; p < part_count; ++p) {
      if (parts[p].heads != 0 &&
          (parts[p].input_gradient.data == nullptr || parts[p].output_gradient.data == nullptr ||
           parts[p].input.data == nullptr || parts[p].weight == nullptr ||
           parts[p].denominator == nullptr)) {
        return invalid();
      }
    }
  }
  const Turn turn = turn_of(*rotary, extent, true);
  DeviceGuard guard;
  if (enter(device, guard) != hipSuccess) return runtime(guard.error);
  if (dtype == SPAR_HIP_FLOAT32) {
    start_norm_backward<float>(parts, part_count, batch, tokens, turn, rotary->layout, workspace,
                               guard.stream);
  } else {
    start_norm_backward<double>(parts, part_count, batch, tokens, turn, rotary->layout, workspace,
                                guard.stream);
  }
  return finish(guard);
}

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
// next to each other read neighbouring heads): cos and sin once for the K.  Bound by
// memory: [16, 1024, 16, 64] float32 in 26 us, 5.2 TB/s of the heads read and written
// (workgroups of 64 or 128 lanes and two heads a lane take the same, stores that stay
// in the caches 31 us); [3, 2047, 12, 80] turning 32 in pairs of neighbours in 13 us,
// 3.7 TB/s, when a launch's start and end weigh as much as its bytes.
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

// The sum over LANES neighbouring lanes, in each of them, without LDS: lanes of a quad
// change places, then quads of a half row and half rows mirror (their lanes hold equal
// sums by then), then rows and halves of the wave swap.
template <int CONTROL>
__device__ __forceinline__ float moved(float x) {
  return __uint_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_uint(x), CONTROL, 0xf, 0xf, true));
}
template <int CONTROL>
__device__ __forceinline__ double moved(double x) {
  return __hiloint2double(
      __builtin_amdgcn_update_dpp(0, __double2hiint(x), CONTROL, 0xf, 0xf, true),
      __builtin_amdgcn_update_dpp(0, __double2loint(x), CONTROL, 0xf, 0xf, true));
}

template <typename T, int LANES>
__device__ __forceinline__ T group_sum(T x) {
  static_assert(LANES >= 8 && LANES <= kWave);
  x += moved<0xb1>(x);   // quad_perm 1 0 3 2
  x += moved<0x4e>(x);   // quad_perm 2 3 0 1
  x += moved<0x141>(x);  // row_half_mirror
  if constexpr (LANES >= 16) x += moved<0x140>(x);  // row_mirror
  if constexpr (LANES >= 32) x += __shfl_xor(x, 16, kWave);
  if constexpr (LANES >= 64) x += __shfl_xor(x, 32, kWave);
  return x;
}

template <typename T>
__device__ __forceinline__ T square_sum(const T (&x)[8]) {
  return ((x[0] * x[0] + x[1] * x[1]) + (x[2] * x[2] + x[3] * x[3])) +
         ((x[4] * x[4] + x[5] * x[5]) + (x[6] * x[6] + x[7] * x[7]));
}

// LANES lanes per head, a unit each (none where a head has fewer), for K heads of one
// token of one part: cos, sin and the weight once for the K.  Groups of lanes count
// through the first part's head groups and then the second's, so that a token's
// queries and keys share the launch.  Bound by memory: 32 + 8 heads of 128 float32 for
// 4 x 4096 tokens in 124 us, 5.4 TB/s of the heads read and written; a single token of
// 16 sequences takes 5 us, the launch.  15 float64 heads of 64 for 2 x 1023 tokens 13.5 us
// (31 MB), of which cos and sin are 0.7: two workgroups a CU, each one chain of loads, sums
// and stores.  A head's elements are multiplied by 1 / d, one division a head; that rounds
// once more than dividing each of them (0.5 units in the last place).
template <typename T, bool HALF, bool NT, int LANES, int K>
__global__ __launch_bounds__(kThreads) void norm_forward_kernel(NormParts<T> parts, Turn turn,
                                                                Rows rows, uint32_t items,
                                                                uint32_t units, FastDiv by_groups,
                                                                uint32_t first_groups, T epsilon) {
  const uint32_t item = (blockIdx.x * kThreads + threadIdx.x) / LANES;
  const uint32_t u = threadIdx.x % LANES;
  if (item >= items) return;
  const uint32_t row = by_groups.div(item);
  uint32_t group = item - row * by_groups.divisor;
  uint64_t b, t;
  rows.split(row, b, t);
  Unit unit{0, 0, 0, 0, kPassed};
  if (u < units) unit = unit_at<HALF>(u, turn.half, turn.extent);
  const bool other = group >= first_groups;
  const NormPart<T>& part = parts.part[other ? 1 : 0];
  const uint32_t heads = other ? parts.heads[1] : parts.heads[0];
  const uint32_t groups = other ? by_groups.divisor - first_groups : first_groups;
  if (other) group -= first_groups;
  const T* source = part.input.data + b * part.input.batch + t * part.input.token;
  T* target = part.output.data + b * part.output.batch + t * part.output.token;
  T x[K][8], w[8];
  // In the place of a head behind the last the first of these is read, and not written:
  // any other may be written meanwhile, where the output is the input itself.
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t head = group + k * groups;
    load_unit<T, NT>(x[k], source + (head < heads ? head : group) * part.input.head, unit);
  }
  load_unit<T, false>(w, part.weight, unit);
  T c[4], s[4];
  unit_turn(turn, unit, b, t, c, s);
  T d[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    d[k] = sqrt(group_sum<T, LANES>(square_sum(x[k])) / static_cast<T>(turn.extent) + epsilon);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const T over = T(1) / d[k];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[k][i] = (x[k][i] * over) * w[i];
    turn_unit<T, HALF>(x[k], unit, c, s);
    const uint32_t head = group + k * groups;
    if (head >= heads) continue;
    if (u == 0 && part.denominator != nullptr) {
      part.denominator[(b * heads + head) * rows.tokens + t] = d[k];
    }
    store_unit<T, NT>(target + head * part.output.head, x[k], unit);
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

// Workgroups of the first part, then of the second; their groups of lanes walk the
// part's rows and head groups in a grid-stride.  Each lane keeps the weight gradient
// of its unit, which the workgroup adds up at the end into its row of `partials`: no
// atomics, and an order that only the grid decides.  Bound by memory: the tokens above in
// 188 us, 5.4 TB/s of inputs and output gradients read and gradients written; the float64
// heads above 18.4 us (47 MB), of which cos and sin are 2.3.
template <typename T, bool HALF, bool NT, int LANES, int K>
__global__ __launch_bounds__(kThreads, 3) void norm_backward_kernel(NormGradientParts<T> parts,
                                                                    Turn turn, Rows rows,
                                                                    uint64_t all_rows,
                                                                    uint32_t units,
                                                                    uint32_t first_blocks,
                                                                    T* partials) {
  constexpr uint32_t kGroups = kThreads / LANES;
  const bool other = blockIdx.x >= first_blocks;
  const NormGradientPart<T>& part = parts.part[other ? 1 : 0];
  const uint32_t heads = parts.heads[other ? 1 : 0];
  const uint32_t groups = (heads + K - 1) / K;
  const uint32_t block = other ? blockIdx.x - first_blocks : blockIdx.x;
  const uint32_t blocks = other ? gridDim.x - first_blocks : first_blocks;
  const uint32_t u = threadIdx.x % LANES;
  const bool holds = u < units;
  Unit unit{0, 0, 0, 0, kPassed};
  if (holds) unit = unit_at<HALF>(u, turn.half, turn.extent);
  const T per_extent = T(1) / static_cast<T>(turn.extent);
  T sums[8] = {}, w[8];
  load_unit<T, false>(w, part.weight, unit);
  // Items of a group lie a stride apart: its row and head group advance by the
  // stride's quotient and remainder, with no division in the loop.
  const uint64_t items = all_rows * groups;
  const uint64_t stride = static_cast<uint64_t>(blocks) * kGroups;
  uint64_t item = static_cast<uint64_t>(block) * kGroups + threadIdx.x / LANES;
  uint64_t row = item / groups;
  uint32_t group = static_cast<uint32_t>(item - row * groups);
  const uint64_t row_step = stride / groups;
  const uint32_t group_step = static_cast<uint32_t>(stride - row_step * groups);
  for (; item < items; item += stride) {
    uint64_t b, t;
    rows.split(row, b, t);
    const T* source = part.input.data + b * part.input.batch + t * part.input.token;
    const T* gradient = part.output_gradient.data + b * part.output_gradient.batch +
                        t * part.output_gradient.token;
    T x[K][8], g[K][8], over[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      // As in the forward: a head behind the last is the first of these.
      const uint32_t head = group + k * groups < heads ? group + k * groups : group;
      load_unit<T, NT>(x[k], source + head * part.input.head, unit);
      load_unit<T, NT>(g[k], gradient + head * part.output_gradient.head, unit);
      over[k] = part.denominator[(b * heads + head) * rows.tokens + t];
    }
    T c[4], s[4];
    unit_turn(turn, unit, b, t, c, s);
    T mean[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      // A head behind the last adds nothing.
      const bool counts = group + k * groups < heads;
      over[k] = T(1) / over[k];
      turn_unit<T, HALF>(g[k], unit, c, s);
      T dot = T(0);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[k][i] *= over[k];
        const T gx = g[k][i] * x[k][i];
        sums[i] += counts ? gx : T(0);
        g[k][i] *= w[i];
        dot += gx * w[i];
      }
      mean[k] = group_sum<T, LANES>(dot) * per_extent;
    }
    T* target = part.input_gradient.data + b * part.input_gradient.batch +
                t * part.input_gradient.token;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const uint32_t head = group + k * groups;
      if (head >= heads) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) g[k][i] = (g[k][i] - x[k][i] * mean[k]) * over[k];
      store_unit<T, NT>(target + head * part.input_gradient.head, g[k], unit);
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
    for (int i = 0; i < 8; ++i) sums[i] += __shfl_xor(sums[i], mask, kWave);
  }
  constexpr int kWaves = kThreads / kWave;
  __shared__ T shared[kWaves][LANES][9];
  const int wave = threadIdx.x / kWave;
  if (threadIdx.x % kWave < LANES) {
#pragma unroll
    for (int i = 0; i < 8; ++i) shared[wave][u][i] = sums[i];
  }
  __syncthreads();
  if (threadIdx.x < LANES && holds) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sums[i] = shared[0][u][i];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sums[i] += shared[w][u][i];
    }
    store_unit<T, false>(partials + static_cast<uint64_t>(blockIdx.x) * turn.extent, sums, unit);
  }
}

// The columns of a part's partial rows added up in their order (blockIdx.y: the part):
// 16 columns per workgroup, 64 lanes to a column, each a run of rows, then the runs in
// a tree.  5 us for 768 rows: one memory latency per eight rows of a run, and the tree.
template <typename T>
__global__ __launch_bounds__(1024) void norm_weight_kernel(T* first, T* second, const T* partials,
                                                           uint32_t first_rows,
                                                           uint32_t second_rows,
                                                           uint32_t extent) {
  __shared__ T shared[64][17];
  const bool other = blockIdx.y != 0;
  const uint32_t rows = other ? second_rows : first_rows;
  const T* from = partials + (other ? static_cast<uint64_t>(first_rows) * extent : 0);
  const uint32_t lane = threadIdx.x % 16, run = threadIdx.x / 16;
  const uint32_t column = blockIdx.x * 16 + lane;
  const uint32_t per = (rows + 63) / 64;
  T sum = T(0);
  if (column < extent) {
    const uint32_t begin = run * per, end = begin + per < rows ? begin + per : rows;
#pragma unroll 4
    for (uint32_t r = begin; r < end; ++r) sum += from[static_cast<uint64_t>(r) * extent + column];
  }
  shared[run][lane] = sum;
  for (uint32_t half = 32; half > 0; half >>= 1) {
    __syncthreads();
    if (run < half) shared[run][lane] += shared[run + half][lane];
  }
  if (run == 0 && column < extent) (other ? second : first)[column] = shared[0][lane];
}

// ---------------------------------------------------------------- launchers

// Heads a lane turns with one cos and sin: as many as leave the chip full.
constexpr uint64_t kFullLanes = 1 << 16;

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
  const uint32_t first_groups = (parts.heads[0] + K - 1) / K;
  const uint32_t groups = first_groups + (parts.heads[1] + K - 1) / K;
  FastDiv by_groups;
  by_groups.init(groups);
  const uint64_t most = (kIndex32Limit / LANES - kThreads) / groups;
  for (uint64_t first = 0, all = batch * tokens; first < all; first += most) {
    const uint64_t count = all - first < most ? all - first : most;
    const uint32_t items = static_cast<uint32_t>(count * groups);
    norm_forward_kernel<T, HALF, NT, LANES, K>
        <<<ceil_div_u32(static_cast<uint64_t>(items) * LANES, kThreads), kThreads, 0, stream>>>(
            parts, turn, rows_at(first, batch, tokens), items,
            units_of(turn.half, turn.extent), by_groups, first_groups, static_cast<T>(epsilon));
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

// Workgroups of the backward, one row of partial weight gradients each: as many as the
// heads fill, at most three per CU, which is what their registers let a CU hold (with
// four, the fourth waits for the others to end).
constexpr uint64_t kMostPartials = 768;

uint32_t partial_rows(uint64_t batch, uint64_t tokens, uint64_t heads) {
  const uint64_t wanted = (batch * tokens * heads + 7) / 8;
  return static_cast<uint32_t>(wanted < kMostPartials ? wanted : kMostPartials);
}

// Of these, the first part's: by its share of the heads, at least one for a part that
// has any (`heads` is their sum).
uint32_t first_rows_of(uint32_t partials, uint64_t first, uint64_t heads) {
  const uint32_t share = static_cast<uint32_t>(partials * first / heads);
  return first != 0 && share == 0 ? 1 : share;
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
  const uint32_t first = partials == 0 ? 0 : first_rows_of(partials, all.heads[0], heads);
  const uint32_t second = all.heads[1] == 0 || partials == 0 ? 0
                          : partials > first                 ? partials - first
                                                             : 1;
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
            norm_backward_kernel<T, decltype(half)::value, decltype(nt)::value, kLanes, K>
                <<<first + second, kThreads, 0, stream>>>(all, turn, rows_at(0, batch, tokens),
                                                          batch * tokens, units, first,
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
  const dim3 grid(ceil_div_u32(turn.extent, 16), part_count);
  norm_weight_kernel<T><<<grid, 1024, 0, stream>>>(
      static_cast<T*>(parts[0].weight_gradient),
      part_count > 1 ? static_cast<T*>(parts[1].weight_gradient) : nullptr,
      static_cast<const T*>(workspace), first, second, turn.extent);
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
  if (!sane(batch, heads, tokens, extent)) return invalid();
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
  if (!sane(batch, heads, tokens, extent)) return invalid();
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

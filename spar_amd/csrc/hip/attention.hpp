// What the attention kernels share: the matrix instruction, the layout of its
// operands, the rows and keys of a call, and the staging of tiles into LDS.
//
// Rows.  The query heads that read one key head are the rows of one product:
// row r = t * group + g is query t of the group's head g, so a key or value is
// read once for the whole group, and the sums of dk and dv over the group's heads
// are sums over rows.
//
// Operands.  A 16x16x4 product takes one value per lane of each operand (lane l:
// row or column l % 16, contraction index l / 16 = the lane's quarter) and yields
// four per lane: column l % 16 and rows row_of(v, quarter).  Which four indices a
// step contracts is free as long as both operands agree, and two choices follow:
//   - contracted along a head, a lane takes neighbours d = 4 W s + W quarter + i
//     (W values in 16 bytes), so that operands load in 16-byte pieces;
//   - contracted along the rows of a product's result, step v takes the rows
//     row_of(v, quarter): exactly the values the lanes hold, which thereby pass
//     from one product into the next in registers.
// A result's rows along a head may be any permutation too: block n of a chunk of
// 16 W elements holds d = 16 W c + W m + n for row m, so that a lane's operands of
// W blocks are neighbours, and its results as well.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"

namespace spar_hip {
namespace attention {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kBlock = 16;  // rows and columns of the matrix instruction

typedef double f64x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mma;

// float32 runs at 157 TFLOP/s, twice what the vector units do without packed
// instructions; products and sums are IEEE single.
template <> struct Mma<float> {
  using Acc = f32x4;
  __device__ static __forceinline__ Acc step(float a, float b, Acc c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ int row_of(int v, int quarter) { return 4 * quarter + v; }
};

template <> struct Mma<double> {
  using Acc = f64x4;
  __device__ static __forceinline__ Acc step(double a, double b, Acc c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ int row_of(int v, int quarter) { return 4 * v + quarter; }
};

template <typename T>
struct Heads {
  T* data;
  uint64_t batch, head, token;  // strides
};

template <typename T>
Heads<T> heads_of(const SparHipHeads& heads) {
  return {static_cast<T*>(heads.data), heads.strides[0], heads.strides[1], heads.strides[2]};
}

// Keys of a sequence are fewer than this, so that tokens, keys and their
// differences are 32-bit.
constexpr uint64_t kMostKeys = uint64_t{1} << 30;
constexpr int32_t kNoWindow = 1 << 30;

// The shape of a call, as the kernels take it.
struct Call {
  const void* lengths;
  bool wide_lengths;
  FastDiv group;       // query heads per key head
  uint32_t key_heads;
  uint32_t batch_heads;  // batch * key_heads
  uint32_t queries;
  uint32_t rows;       // queries * group
  uint32_t keys;
  uint32_t extent;
  int32_t window;  // kNoWindow where there is none
  int32_t sinks;
  double scale;

  __device__ __forceinline__ int32_t length(uint32_t b) const {
    if (lengths == nullptr) return static_cast<int32_t>(keys);
    const int64_t n = wide_lengths ? static_cast<const int64_t*>(lengths)[b]
                                   : static_cast<const int32_t*>(lengths)[b];
    return static_cast<int32_t>(n < 0 ? 0 : n > keys ? keys : n);
  }
  // Token of its sequence that row r's query is, less than 0 where it sees nothing.
  __device__ __forceinline__ int32_t token(uint32_t r, int32_t first) const {
    return r < rows ? first + static_cast<int32_t>(group.div(r)) : -1;
  }
  __device__ __forceinline__ bool sees(int32_t p, int32_t key) const {
    return (key <= p) & ((p - key < window) | (key < sinks));
  }
};

// The keys a tile of rows sees, as two runs: the sinks in front of the window,
// and everything from the first row's window to the last row.
struct Keys {
  int32_t sink_end, low, high;

  __device__ __forceinline__ Keys(const Call& call, int32_t first_token, int32_t last_token) {
    high = last_token + 1;
    low = first_token - call.window + 1;
    if (low < 0) low = 0;
    sink_end = call.sinks;
    if (low <= sink_end) low = sink_end = 0;
    if (last_token < 0) low = high = sink_end = 0;
  }
  __device__ __forceinline__ uint32_t tiles(int size) const {
    return static_cast<uint32_t>((sink_end + size - 1) / size + (high - low + size - 1) / size);
  }
  // First key and end of the run of tile i.
  __device__ __forceinline__ void tile(uint32_t i, int size, int32_t& begin, int32_t& end) const {
    const uint32_t sink_tiles = static_cast<uint32_t>((sink_end + size - 1) / size);
    if (i < sink_tiles) {
      begin = static_cast<int32_t>(i) * size;
      end = sink_end;
    } else {
      begin = low + static_cast<int32_t>(i - sink_tiles) * size;
      end = high;
    }
  }
};

constexpr double kLog2E = 1.44269504088896340736;
constexpr double kLn2 = 0.69314718055994530942;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ double exp2_of(double x) { return exp2(x); }
__device__ __forceinline__ float log2_of(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ double log2_of(double x) { return log2(x); }

template <typename T>
__device__ __forceinline__ T lowest() {
  return -static_cast<T>(__builtin_huge_val());
}

// Sums and maxima over the four quarters of a wave, which hold one column's rows.
template <typename T>
__device__ __forceinline__ T quarter_sum(T x) {
  x += __shfl_xor(x, 16, kWave);
  return x + __shfl_xor(x, 32, kWave);
}
template <typename T>
__device__ __forceinline__ T quarter_max(T x) {
  const T y = __shfl_xor(x, 16, kWave);
  x = x > y ? x : y;
  const T z = __shfl_xor(x, 32, kWave);
  return x > z ? x : z;
}

// 16 bytes of a head at d, without a branch, so that a batch of them is in flight at
// once: a piece behind the extent is read from the head's start, an element of a
// piece that the extent cuts (EVEN says that it cuts none) from the head's end.
// What stands there is finite where the head is, and meets zeros of the other
// operand or is not written.
template <bool EVEN, typename T>
__device__ __forceinline__ typename Vec16<T>::type load_piece(const T* head, uint32_t d,
                                                              uint32_t extent) {
  if constexpr (EVEN) {
    return loose_load(head + (d < extent ? d : 0));
  } else {
    typename Vec16<T>::type v;
#pragma unroll
    for (int i = 0; i < Vec16<T>::width; ++i) v[i] = head[d + i < extent ? d + i : extent - 1];
    return v;
  }
}

template <typename T, int W>
__device__ __forceinline__ void store_piece(T* head, uint32_t d, uint32_t extent,
                                            const T (&x)[W]) {
  if (d + W <= extent) {
    typename Vec16<T>::type v;
    if constexpr (W == Vec16<T>::width) {
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = x[i];
      loose_store<false, T>(head + d, v);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
    if (d + i < extent) head[d + i] = x[i];
  }
}

// Heads as a product's operand contracted along the head: lane l's pieces of row
// l % 16.
template <typename T, int DP>
struct Operand {
  static constexpr int W = Vec16<T>::width;
  T value[DP / 4];

  template <bool EVEN>
  __device__ __forceinline__ void load(const T* head, uint32_t extent, int quarter) {
#pragma unroll
    for (int s = 0; s < DP / (4 * W); ++s) {
      const auto piece = load_piece<EVEN>(head, 4 * W * s + W * quarter, extent);
#pragma unroll
      for (int i = 0; i < W; ++i) value[s * W + i] = piece[i];
    }
  }
  // Zeros behind the extent, and everywhere if the row is not `held`; times factor.
  __device__ __forceinline__ void finish(bool held, uint32_t extent, int quarter, T factor) {
#pragma unroll
    for (int s = 0; s < DP / (4 * W); ++s) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const bool inside = held & (4 * W * s + W * quarter + i < extent);
        value[s * W + i] = inside ? value[s * W + i] * factor : T(0);
      }
    }
  }
};

// A tile of ROWS heads in LDS, rows 16 bytes apart from a multiple of 128: 16
// lanes that read one piece of 16 rows each, or 16 pieces of one row, fall into
// different banks.  The pieces pass through registers, so that the next tile is on
// its way while the present one is used.
template <typename T, int ROWS, int DP>
struct Tile {
  static constexpr int W = Vec16<T>::width;
  static constexpr int kPitch = DP + W;
  static constexpr int kPieces = DP / W;
  static constexpr int kShare = ROWS * kPieces / kThreads;  // pieces per thread
  static_assert(ROWS * kPieces % kThreads == 0);
  alignas(16) T value[ROWS * kPitch];

  struct Stage {
    typename Vec16<T>::type piece[kShare];

    // head_of(row): the row's head.  All threads of a workgroup.
    template <bool EVEN, typename HeadOf>
    __device__ __forceinline__ void load(uint32_t extent, HeadOf&& head_of) {
#pragma unroll
      for (int j = 0; j < kShare; ++j) {
        const uint32_t at = threadIdx.x + j * kThreads;
        piece[j] = load_piece<EVEN>(head_of(at / kPieces), at % kPieces * W, extent);
      }
    }
  };

  __device__ __forceinline__ void fill(const Stage& stage) {
#pragma unroll
    for (int j = 0; j < kShare; ++j) {
      const uint32_t at = threadIdx.x + j * kThreads;
      *reinterpret_cast<typename Vec16<T>::type*>(value + at / kPieces * kPitch +
                                                  at % kPieces * W) = stage.piece[j];
    }
  }

  // The piece of row `row` that step group s contracts along the head.
  __device__ __forceinline__ typename Vec16<T>::type along(int row, int s, int quarter) const {
    return *reinterpret_cast<const typename Vec16<T>::type*>(value + row * kPitch + 4 * W * s +
                                                             W * quarter);
  }
};

// Results along a head, blocks of 16 elements by 16 columns: chunks of W blocks,
// and where DP is half a chunk more (float32), one of two.
template <typename T, int DP>
struct Along {
  static constexpr int W = Vec16<T>::width;
  static constexpr int kChunks = DP / (16 * W);
  static constexpr int kRest = DP % (16 * W) / 16;  // 0 or 2 blocks
  static_assert(kRest == 0 || kRest == 2);
  using Acc = typename Mma<T>::Acc;
  Acc block[DP / 16];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) block[n] = Acc{0, 0, 0, 0};
  }
  __device__ __forceinline__ void scale(T factor) {
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
#pragma unroll
      for (int v = 0; v < 4; ++v) block[n][v] *= factor;
    }
  }
  // += head^T weight for one head row (held in LDS, `row`) per quarter.
  __device__ __forceinline__ void add(const T* row, int m, T weight) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const auto piece =
          *reinterpret_cast<const typename Vec16<T>::type*>(row + 16 * W * c + W * m);
#pragma unroll
      for (int n = 0; n < W; ++n) {
        block[c * W + n] = Mma<T>::step(piece[n], weight, block[c * W + n]);
      }
    }
    if constexpr (kRest != 0) {
      const T* rest = row + 16 * W * kChunks + 2 * m;
      const T first = rest[0], second = rest[1];
      block[kChunks * W] = Mma<T>::step(first, weight, block[kChunks * W]);
      block[kChunks * W + 1] = Mma<T>::step(second, weight, block[kChunks * W + 1]);
    }
  }
  // Calls body(d, values) for the runs of neighbours d a lane holds: of W values,
  // of 2 in the rest.
  template <typename Body>
  __device__ __forceinline__ void visit(int quarter, Body&& body) const {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        T run[W];
#pragma unroll
        for (int n = 0; n < W; ++n) run[n] = block[c * W + n][v];
        body(16 * W * c + W * Mma<T>::row_of(v, quarter), run);
      }
    }
    if constexpr (kRest != 0) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        T run[2] = {block[kChunks * W][v], block[kChunks * W + 1][v]};
        body(16 * W * kChunks + 2 * Mma<T>::row_of(v, quarter), run);
      }
    }
  }
};

// Waves per SIMD that a kernel's registers leave room for: one computes while the
// other waits for its tile or takes exponentials.
template <typename T, int DP>
constexpr int tile_waves() {
  return DP * sizeof(T) <= 512 ? 2 : 1;
}

template <typename Body>
void with_padded_width(uint64_t extent, Body&& body) {
  if (extent <= 32) {
    body(std::integral_constant<int, 32>{});
  } else if (extent <= 64) {
    body(std::integral_constant<int, 64>{});
  } else if (extent <= 96) {
    body(std::integral_constant<int, 96>{});
  } else if (extent <= 128) {
    body(std::integral_constant<int, 128>{});
  } else if (extent <= 192) {
    body(std::integral_constant<int, 192>{});
  } else {
    body(std::integral_constant<int, SPAR_HIP_ATTENTION_MAX_EXTENT>{});
  }
}

// Calls body(integral_constant<DP>, Policy<EVEN>) with the smallest padded
// width, EVEN if 16-byte pieces divide the extent.
template <typename T, typename Body>
void with_width(uint64_t extent, Body&& body) {
  with_policy(extent % Vec16<T>::width == 0, [&](auto even) {
    with_padded_width(extent, [&](auto width) { body(width, even); });
  });
}

inline bool valid(const SparHipAttention* a) {
  constexpr uint64_t kMost = kIndex32Limit;
  if (a == nullptr || !valid_float_dtype(a->dtype) || a->key_heads == 0 || a->query_heads == 0 ||
      a->extent == 0 ||
      a->extent > SPAR_HIP_ATTENTION_MAX_EXTENT || a->query_heads % a->key_heads != 0 ||
      !__builtin_isfinite(a->scale) || a->batch > kMost || a->query_heads > kMost ||
      a->queries > kMost || a->keys >= kMostKeys ||
      a->batch * a->key_heads > kMost || a->queries * a->query_heads >= kMostKeys) {
    return false;
  }
  return a->lengths == nullptr || a->length_dtype == SPAR_HIP_INT32 ||
         a->length_dtype == SPAR_HIP_INT64;
}

inline Call call_of(const SparHipAttention& a) {
  Call call{};
  const uint64_t group = a.query_heads / a.key_heads;
  call.lengths = a.lengths;
  call.wide_lengths = a.length_dtype == SPAR_HIP_INT64;
  call.group.init(static_cast<uint32_t>(group == 0 ? 1 : group));
  call.key_heads = static_cast<uint32_t>(a.key_heads);
  call.batch_heads = static_cast<uint32_t>(a.batch * a.key_heads);
  call.queries = static_cast<uint32_t>(a.queries);
  call.rows = static_cast<uint32_t>(a.queries * group);
  call.keys = static_cast<uint32_t>(a.keys);
  call.extent = static_cast<uint32_t>(a.extent);
  call.window = a.window == 0 || a.window > kMostKeys ? kNoWindow : static_cast<int32_t>(a.window);
  call.sinks = a.window == 0 ? 0 : static_cast<int32_t>(a.sinks < a.keys ? a.sinks : a.keys);
  call.scale = a.scale;
  return call;
}

// Keys that one sequence's newest query sees at most.
inline uint64_t most_seen(const SparHipAttention& a) {
  if (a.window == 0 || a.window >= a.keys || a.sinks >= a.keys - a.window) return a.keys;
  return a.window + a.sinks;
}

}  // namespace attention
}  // namespace spar_hip

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

#include <initializer_list>
#include <type_traits>

#include "common.hpp"

namespace spar_hip {
namespace attention {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kBlock = 16;  // rows and columns of the matrix instruction

typedef double f64x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Mma;

// float32 reaches 154 TFLOP/s, twice what the vector units do without packed
// instructions; products and sums are IEEE single.  Vector instructions of any wave
// take their time, 4 cycles each, from the same pipeline (one per matrix instruction
// leaves 138 TFLOP/s, two 124), so the kernels count them: masks are formed for
// tiles at an edge alone, and addresses move in scalar registers.
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

// Workgroups of a launch: its work-items are counted in 32 bits, and those behind are
// dropped without an error.
constexpr uint64_t kMostGroups = (uint64_t{1} << 32) / kThreads - 1;

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
  // Queries of all heads and sequences.
  __host__ __device__ __forceinline__ uint64_t all_rows() const {
    return static_cast<uint64_t>(batch_heads) * rows;
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

template <typename T>
__device__ __forceinline__ T lowest_finite() {
  return sizeof(T) == 4 ? static_cast<T>(-__FLT_MAX__) : static_cast<T>(-__DBL_MAX__);
}

// Sums and maxima over the four quarters of a wave, which hold one column's rows: the
// halves and then the quarters of a half change places in registers, each lane
// combining both.  A maximum passes over NaN.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }

template <typename Combine>
__device__ __forceinline__ float over_quarters(float x, Combine&& combine) {
  const uint32_t a = __float_as_uint(x);
  const auto halves = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t h = __float_as_uint(combine(__uint_as_float(halves[0]),
                                             __uint_as_float(halves[1])));
  const auto quarters = __builtin_amdgcn_permlane16_swap(h, h, false, false);
  return combine(__uint_as_float(quarters[0]), __uint_as_float(quarters[1]));
}
template <typename Combine>
__device__ __forceinline__ double over_quarters(double x, Combine&& combine) {
  x = combine(x, __shfl_xor(x, 32, kWave));
  return combine(x, __shfl_xor(x, 16, kWave));
}
template <typename T>
__device__ __forceinline__ T quarter_sum(T x) {
  return over_quarters(x, [](T a, T b) { return a + b; });
}
template <typename T>
__device__ __forceinline__ T quarter_max(T x) {
  return over_quarters(x, [](T a, T b) { return larger(a, b); });
}

// How a call's heads can be read in 16-byte pieces.
enum class Reads {
  Single,   // pieces do not divide the extent: element by element
  Pieces,   // they do, at any address of an element
  Aligned,  // and every head starts at a multiple of 16 bytes
};

// 16 bytes of a head at d, without a branch, so that a batch of them is in flight at
// once: a piece behind the extent is read from the head's start, an element of a
// piece that the extent cuts from the head's end.  What stands there is finite
// where the head is, and meets zeros of the other operand or is not written.
template <Reads READS, typename T>
__device__ __forceinline__ typename Vec16<T>::type load_piece(const T* head, uint32_t d,
                                                              uint32_t extent) {
  if constexpr (READS != Reads::Single) {
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

  template <Reads READS>
  __device__ __forceinline__ void load(const T* head, uint32_t extent, int quarter) {
#pragma unroll
    for (int s = 0; s < DP / (4 * W); ++s) {
      const auto piece = load_piece<READS>(head, 4 * W * s + W * quarter, extent);
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

// What a piece's place in its row is mixed with.
template <int PIECES>
constexpr int kMix = PIECES % 16 == 0 ? 16 : 8;

// Tiles of ROWS heads in LDS, two or more of them: one is used while the next arrive.
// Piece p of row r lies at piece p ^ (r % 16) of the row (r % 8 where 16 pieces do not
// divide a row), so that 16 lanes that read one piece of 16 rows each, and 16 lanes
// that read 16 pieces of one row, both spread over the 64 banks without padding (with
// r % 8 every such read takes half as long again): so aligned heads go from memory
// to LDS directly, 64 neighbouring pieces of LDS per instruction, each lane asking
// for the piece that belongs there.  Others pass through registers.
template <typename T, int ROWS, int DP, Reads READS, int BUFFERS = 2>
struct Tile {
  static constexpr int W = Vec16<T>::width;
  static constexpr int kPieces = DP / W;
  static constexpr int kAll = ROWS * kPieces;
  static constexpr int kShare = (kAll + kThreads - 1) / kThreads;  // pieces per thread
  static constexpr bool kDirect = READS == Reads::Aligned;
  static_assert(kAll % kWave == 0 && kPieces % 8 == 0);
  alignas(16) T value[BUFFERS][ROWS * DP];

  struct Stage {
    typename Vec16<T>::type piece[kDirect ? 1 : kShare];
    uint32_t offset[kDirect ? kShare : 1];  // bytes, of a tile of ROWS rows
  };

  // offset_of(row): elements from a tile's base to the head of its row.  The offsets
  // of the rows in whole tiles, which most are, are computed once.
  template <typename OffsetOf>
  __device__ __forceinline__ void prepare(Stage& stage, uint32_t extent, OffsetOf&& offset_of) {
    if constexpr (kDirect) {
#pragma unroll
      for (int j = 0; j < kShare; ++j) stage.offset[j] = bytes_at(j, extent, offset_of);
    }
  }
  // Whether share j of this wave lies in the tile (the last may not).
  __device__ __forceinline__ static bool holds(int j, uint32_t wave) {
    return (j + 1) * kThreads <= kAll || j * kThreads + wave * kWave < kAll;
  }
  template <typename OffsetOf>
  __device__ __forceinline__ static uint32_t bytes_at(int j, uint32_t extent,
                                                      OffsetOf&& offset_of) {
    const uint32_t at = threadIdx.x + j * kThreads;
    const uint32_t row = at / kPieces, d = (at % kPieces ^ row % kMix<kPieces>) * W;
    return static_cast<uint32_t>(offset_of(row) + (d < extent ? d : 0)) * sizeof(T);
  }

  // Starts the way of the tile at `base` into buffer `to`; offset_of is asked where
  // the tile is not `whole`.  All threads of the workgroup.  The tile has arrived
  // after finish() and a barrier.
  template <typename OffsetOf>
  __device__ __forceinline__ void start(Stage& stage, int to, const T* base, bool whole,
                                        uint32_t extent, OffsetOf&& offset_of) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if constexpr (kDirect) {
      const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
                               (__attribute__((address_space(3))) T*)(value[to]))) +
                           wave * kWave * 16;
      const auto load = [&](int j, uint32_t offset) {
// m0 is named, although the compiler does not give it out and warns of it: it
// writes it for instructions of its own.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(lds + j * kThreads * 16), "v"(offset), "s"(base)
                     : "memory", "m0");
#pragma clang diagnostic pop
      };
      if (whole) {
#pragma unroll
        for (int j = 0; j < kShare; ++j) {
          if (holds(j, wave)) load(j, stage.offset[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kShare; ++j) {
          if (holds(j, wave)) load(j, bytes_at(j, extent, offset_of));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kShare; ++j) {
        const uint32_t at = threadIdx.x + j * kThreads;
        const uint32_t row = at / kPieces, piece = at % kPieces ^ row % kMix<kPieces>;
        if (holds(j, wave)) {
          stage.piece[j] = load_piece<READS>(base + offset_of(row), piece * W, extent);
        }
      }
    }
  }
  // The same for rows that lie anywhere: head_of(row) is the row's head.
  template <typename HeadOf>
  __device__ __forceinline__ void start_rows(Stage& stage, int to, uint32_t extent,
                                             HeadOf&& head_of) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
                             (__attribute__((address_space(3))) T*)(value[to]))) +
                         wave * kWave * 16;
#pragma unroll
    for (int j = 0; j < kShare; ++j) {
      if (!holds(j, wave)) continue;
      const uint32_t at = threadIdx.x + j * kThreads;
      const uint32_t row = at / kPieces, d = (at % kPieces ^ row % kMix<kPieces>) * W;
      const T* head = head_of(j, row);
      if constexpr (kDirect) {
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                     :
                     : "s"(lds + j * kThreads * 16), "v"(head + (d < extent ? d : 0))
                     : "memory", "m0");
#pragma clang diagnostic pop
      } else {
        stage.piece[j] = load_piece<READS>(head, d, extent);
      }
    }
  }
  __device__ __forceinline__ void finish(const Stage& stage, int to) {
    if constexpr (kDirect) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
#pragma unroll
      for (int j = 0; j < kShare; ++j) {
        if (holds(j, __builtin_amdgcn_readfirstlane(threadIdx.x / kWave))) {
          *reinterpret_cast<typename Vec16<T>::type*>(
              value[to] + (threadIdx.x + j * kThreads) * W) = stage.piece[j];
        }
      }
    }
  }
};

// Where a lane finds its pieces of a block of 16 rows of a tile.
template <typename T, int DP>
struct Lane {
  static constexpr int W = Vec16<T>::width;
  static constexpr int kChunks = DP / (16 * W);
  static constexpr int kRest = DP % (16 * W) / 16;  // 0 or 2 blocks of 16
  static_assert(kRest == 0 || kRest == 2);
  using Piece = typename Vec16<T>::type;
  int quarter, column;
  static constexpr int kMixed = kMix<DP / W>;
  int along_[kMixed / 4], across_[4], rest_[4];

  __device__ __forceinline__ explicit Lane(int lane)
      : quarter(lane / kBlock), column(lane % kBlock) {
#pragma unroll
    for (int s = 0; s < kMixed / 4; ++s) {
      along_[s] = column * DP + ((4 * s + quarter) ^ (column % kMixed)) * W;
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int row = Mma<T>::row_of(v, quarter);
      across_[v] = row * DP + (column ^ (row % kMixed)) * W;
      const int piece = 16 * kChunks + column * 2 / W;
      rest_[v] = row * DP + (piece ^ (row % kMixed)) * W + column * 2 % W;
    }
  }
  // Of row `column`, for group `step` of the contraction along the head.
  __device__ __forceinline__ Piece along(const T* block, int step) const {
    return *reinterpret_cast<const Piece*>(block + along_[step % (kMixed / 4)] +
                                           step / (kMixed / 4) * kMixed * W);
  }
  // Of row row_of(v, quarter), elements 16 W c + W column and on.
  __device__ __forceinline__ Piece across(const T* block, int v, int c) const {
    return *reinterpret_cast<const Piece*>(block + across_[v] + c * 16 * W);
  }
  __device__ __forceinline__ const T* rest(const T* block, int v) const {
    return block + rest_[v];
  }
};

// Results along a head, blocks of 16 elements by 16 columns: chunks of W blocks,
// and where DP is half a chunk more (float32), one of two.
template <typename T, int DP>
struct Along {
  static constexpr int W = Vec16<T>::width;
  static constexpr int kChunks = Lane<T, DP>::kChunks;
  static constexpr int kRest = Lane<T, DP>::kRest;
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

// 2^(base - next), of a row's old and new base.  A base is the score it was taken from
// in float32, and that rounded up to a whole number in float64, where the power is then
// an exponent: a second exponential in double would take 20 registers.
__device__ __forceinline__ float base_of(float score) { return score; }
__device__ __forceinline__ double base_of(double score) { return __builtin_ceil(score); }
__device__ __forceinline__ float shrink_of(float base, float next) { return exp2_of(base - next); }
__device__ __forceinline__ double shrink_of(double base, double next) {
  return __builtin_ldexp(1.0, static_cast<int>(larger(base - next, -2000.0)));
}

// A row's running softmax, and its sum of weights times what the keys bring: weights are
// 2^(score - base), `total` each lane's own part of their sum.  The base follows the
// row's maximum only when that has grown by 2^kSlack, so that the sum is rarely
// rescaled; sums of weights up to 2^kSlack lose nothing in floating point.  It is taken
// off finished scores: equal scores have equal weights however large they are (products
// that start from -base round every key's score differently, by steps of the base; they
// save four instructions a block, 161 us against 163 at heads of 64 and nothing at 128).
template <typename T, int DP>
struct Row {
  static constexpr int kSlack = 8;
  T base = lowest_finite<T>();  // the same in the row's four lanes; this before a score is seen
  T total = T(0);
  Along<T, DP> out;

  // Turns the scores of a block of keys into weights.
  __device__ __forceinline__ void take(T (&score)[4]) {
    T high = larger(larger(score[0], score[1]), larger(score[2], score[3]));
    if (__any(high > base + T(kSlack))) {
      high = quarter_max(high);
      const T next = high > base + T(kSlack) ? base_of(high) : base;
      const T shrink = shrink_of(base, next);
      total *= shrink;
      out.scale(shrink);
      base = next;
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      score[v] = exp2_of(score[v] - base);
      total += score[v];
    }
  }
};

// Blocks of 16 rows in a tile of keys or queries.
template <typename T, int DP>
constexpr int tile_blocks() {
  return DP * sizeof(T) <= 256 ? 2 : 1;
}

// Waves per SIMD that a kernel's registers are to leave room for.
template <typename T, int DP>
constexpr int tile_waves() {
  const int row = DP * sizeof(T);
  return (row <= 256 ? 4 : row <= 512 ? 3 : row <= 768 ? 2 : 1) - (sizeof(T) == 8 && row <= 512);
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

// The pieces along the heads of the four rows row_of(v, quarter) of a block of 16, read
// from memory in the order in which results lie along a head: what a product that
// contracts those rows takes from the lane.  head_of(row) is the row's head.
template <typename T, int DP>
struct AcrossOperand {
  using L = Lane<T, DP>;
  static constexpr int W = L::W;
  T value[4][DP / 16];

  template <Reads READS, typename HeadOf>
  __device__ __forceinline__ void load(uint32_t extent, int quarter, int column,
                                       HeadOf&& head_of) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const T* head = head_of(Mma<T>::row_of(v, quarter));
#pragma unroll
      for (int c = 0; c < L::kChunks; ++c) {
        const auto piece = load_piece<READS>(head, 16 * W * c + W * column, extent);
#pragma unroll
        for (int j = 0; j < W; ++j) value[v][c * W + j] = piece[j];
      }
      if constexpr (L::kRest != 0) {
        const uint32_t d = 16 * W * L::kChunks + 2 * column;
        value[v][L::kChunks * W] = head[d < extent ? d : 0];
        value[v][L::kChunks * W + 1] = head[d + 1 < extent ? d + 1 : 0];
      }
    }
  }
  __device__ __forceinline__ void add_to(Along<T, DP>& out, const T (&weight)[4]) const {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) {
        out.block[j] = Mma<T>::step(value[v][j], weight[v], out.block[j]);
      }
    }
  }
};

// Whether tiles of 64 rows leave so much of the chip idle that workgroups of 16 rows,
// whose waves share the keys, are faster, although every wave reads its keys itself:
// the forward of 8 heads of 128 with 256 tokens 26 us in 32 tiles and 12 us in 128,
// of 16 heads of 64 with 512 tokens and a window of 128 15 us in 128 tiles and 11 us in
// 512, of 2 heads with 634 queries of 3057 keys 23 us in 220 tiles and 24 us in 960.
inline bool spreads(uint64_t tiles) { return tiles < 192; }

// COUNT pieces read from LDS AHEAD uses before their own: the reads' latency (about
// 128 cycles) passes under the matrix instructions of the pieces before.  Left to
// itself the compiler reads a piece right before its use, into registers that the
// instructions before still occupy.  `queue` holds the first AHEAD on entry.
template <int AHEAD, typename Piece>
struct Queue {
  static constexpr int kAhead = AHEAD;
  Piece piece[AHEAD + 1];
};

__device__ __forceinline__ void keep_order() { __builtin_amdgcn_sched_barrier(0); }

template <int AHEAD, typename Piece, typename Read>
__device__ __forceinline__ void fill_queue(Queue<AHEAD, Piece>& queue, Read&& read) {
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) queue.piece[i] = read(i);
}

template <int COUNT, int AHEAD, typename Piece, typename Read, typename Use>
__device__ __forceinline__ void run_queue(Queue<AHEAD, Piece>& queue, Read&& read, Use&& use) {
  keep_order();
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    if (i + AHEAD < COUNT) queue.piece[(i + AHEAD) % (AHEAD + 1)] = read(i + AHEAD);
    keep_order();
    use(i, queue.piece[i % (AHEAD + 1)]);
    keep_order();
  }
}

// out += block^T weights of a block of 16 rows of a tile, of which the lane has the
// weights of row_of(v, quarter), v < 4.
template <typename T, int DP>
struct Across {
  using L = Lane<T, DP>;
  static constexpr int W = L::W;
  static constexpr int kPerRow = L::kChunks + (L::kRest != 0);
  static constexpr int kCount = 4 * kPerRow;
  static constexpr int kAhead = kCount < 2 ? kCount : 2;
  const L& lane;
  const T* rows;
  Queue<kAhead, typename L::Piece> queue;

  // Reads the first pieces.
  __device__ __forceinline__ Across(const L& lane_, const T* rows_) : lane(lane_), rows(rows_) {
    fill_queue(queue, [&](int i) { return read(i); });
  }
  __device__ __forceinline__ typename L::Piece read(int i) const {
    const int v = i / kPerRow, c = i % kPerRow;
    if (L::kRest != 0 && c == L::kChunks) {
      const T* rest = lane.rest(rows, v);
      typename L::Piece piece{};
      piece[0] = rest[0];
      piece[1] = rest[1];
      return piece;
    }
    return lane.across(rows, v, c);
  }
  __device__ __forceinline__ void run(Along<T, DP>& out, const T (&weight)[4]) {
    run_queue<kCount>(
        queue, [&](int i) { return read(i); },
        [&](int at, const typename L::Piece& piece) {
          const int v = at / kPerRow, c = at % kPerRow;
          const int pieces = L::kRest != 0 && c == L::kChunks ? 2 : W;
#pragma unroll
          for (int n = 0; n < W; ++n) {
            if (n >= pieces) continue;
            out.block[c * W + n] = Mma<T>::step(piece[n], weight[v], out.block[c * W + n]);
          }
        });
  }
};

// Whether heads go to LDS directly: pieces at multiples of 16 bytes, and the rows of
// a tile (of up to 32 tokens and all heads of a group) within 2^32 bytes.
template <typename T>
bool reads_aligned(const SparHipHeads& heads, uint64_t group) {
  constexpr uint64_t W = Vec16<T>::width;
  constexpr uint64_t kMost = uint64_t{1} << 24;
  return aligned16(heads.data) && heads.strides[0] % W == 0 && heads.strides[1] % W == 0 &&
         heads.strides[2] % W == 0 && heads.strides[2] <= kMost &&
         (group <= 1 || heads.strides[1] <= kMost * 8 / (group - 1));
}

// Calls body(integral_constant<DP>, integral_constant<READS>) with the smallest
// padded width and the widest reads that all of `heads` allow.
template <typename T, typename Body>
void with_width(const SparHipAttention& a, std::initializer_list<const SparHipHeads*> heads,
                Body&& body) {
  Reads reads = a.extent % Vec16<T>::width == 0 ? Reads::Aligned : Reads::Single;
  for (const SparHipHeads* h : heads) {
    if (reads == Reads::Aligned && !reads_aligned<T>(*h, a.query_heads / a.key_heads)) {
      reads = Reads::Pieces;
    }
  }
  with_padded_width(a.extent, [&](auto width) {
    if (reads == Reads::Aligned) {
      body(width, std::integral_constant<Reads, Reads::Aligned>{});
    } else if (reads == Reads::Pieces) {
      body(width, std::integral_constant<Reads, Reads::Pieces>{});
    } else {
      body(width, std::integral_constant<Reads, Reads::Single>{});
    }
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

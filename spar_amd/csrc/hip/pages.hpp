// Caches of keys and values in pages, as kernels take them.
#pragma once

#include <hip/hip_runtime.h>

#include "common.hpp"

namespace spar_hip {

// A row of a cache has room for fewer tokens than this, so that tokens are 32-bit.
constexpr uint64_t kMostRoom = uint64_t{1} << 30;

template <typename T>
struct PageHeads {
  T* data;
  uint64_t page, head, token;  // strides
};

template <typename T>
struct Pages {
  PageHeads<T> key, value;
  const int32_t* table;
  uint64_t table_stride;
  uint32_t pages;
  uint32_t room;  // tokens of a row
  FastDiv page_tokens;

  // The number that entry `entry` of row b names; held() says whether there is such a page.
  // A load's value is not looked at before that, so that it may be on its way meanwhile.
  __device__ __forceinline__ int32_t page_at(uint32_t b, uint32_t entry) const {
    return table == nullptr ? static_cast<int32_t>(b) : table[b * table_stride + entry];
  }
  __device__ __forceinline__ bool held(int32_t page) const {
    return static_cast<uint32_t>(page) < pages;
  }
};

template <typename T>
Pages<T> pages_of(const SparHipPages& cache) {
  constexpr uint64_t kMost = kIndex32Limit;
  Pages<T> made{};
  const auto heads = [](const SparHipHeads& h) {
    return PageHeads<T>{static_cast<T*>(h.data), h.strides[0], h.strides[1], h.strides[2]};
  };
  made.key = heads(cache.key);
  made.value = heads(cache.value);
  made.table = cache.table;
  made.table_stride = cache.table_stride;
  made.pages = static_cast<uint32_t>(cache.pages < kMost ? cache.pages : kMost);
  made.room = static_cast<uint32_t>(cache.table_pages * cache.page_tokens);
  made.page_tokens.init(static_cast<uint32_t>(cache.page_tokens));
  return made;
}

inline bool valid_pages(const SparHipPages* cache) {
  return cache != nullptr && cache->page_tokens != 0 && cache->page_tokens < kMostRoom &&
         cache->table_pages < kMostRoom && cache->table_pages * cache->page_tokens < kMostRoom &&
         (cache->table != nullptr || cache->table_pages <= 1);
}

// Whether the cache can hold a token at all.
inline bool has_room(const SparHipPages& cache) {
  return cache.pages != 0 && cache.table_pages != 0;
}

}  // namespace spar_hip

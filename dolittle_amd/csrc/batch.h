// Checks shared by the batch operators over caches that grow and shrink by
// sequence (batch_attention.hip, batch_cache.hip).
#pragma once

#include <cstdint>
#include <initializer_list>

#include "dl_internal.h"

namespace dl::batch {

// Most keys of a prefix or cache, and most elements of one key row over all KV
// heads: up to 64 rows (the last one's offset at most 63 * 2^26 + 2^10 bytes)
// are addressed with 32-bit offsets from a 64-bit base.
constexpr uint64_t kMostKeys = 1u << 30;
constexpr uint64_t kMostRow = 1u << 24;

inline void check_shape(const dl_batch_shape* shape) {
  require(shape != nullptr, "null shape");
  require(shape->batch && shape->rows && shape->query_heads && shape->kv_heads && shape->width && shape->capacity,
          "empty batch shape");
  require(shape->query_heads % shape->kv_heads == 0, "query heads must be a multiple of KV heads");
  require(shape->batch <= (1u << 20) && shape->rows <= (1u << 24) && shape->query_heads <= (1u << 16),
          "batch shape too large", DL_LENGTH_ERROR);
  require(shape->capacity <= kMostKeys, "capacity too large", DL_LENGTH_ERROR);
  require(shape->width <= kMostRow / shape->kv_heads, "key rows too wide", DL_LENGTH_ERROR);
}

// Whether head rows of `width` elements from these bases are whole 16-byte pieces.
inline bool whole_pieces(const dl_batch_shape* shape, uint64_t size, std::initializer_list<const void*> bases) {
  uintptr_t low = shape->width * size;
  for (const void* p : bases) low |= reinterpret_cast<uintptr_t>(p);
  return low % 16 == 0;
}

}  // namespace dl::batch

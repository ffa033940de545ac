// Shared by the kernels of the quantised key/value cache: its layout and the
// host-side checks of an mb_kv_cache.
#pragma once

#include "mb_codes.cuh"

namespace mb {

constexpr int kGroup4 = 32;  // channels that share a 4-bit scale and minimum

// A cache's layout, by value to the kernels.  Row (page, head, place) =
// (page * heads + head) * page_size + place.
struct CacheView {
  uint8_t* codes[2];  // keys, values
  uint8_t* scales[2];
  int64_t pages;
  uint32_t page_size, heads, dim;
};

__host__ __device__ inline int64_t cache_slots(const CacheView& c) {
  return c.pages * c.page_size;
}

// Row of a slot's head.  A slot fits 32 bits (checked on the host).
__device__ __forceinline__ int64_t cache_row(const CacheView& c, uint32_t slot, uint32_t head) {
  const uint32_t page = slot / c.page_size, place = slot - page * c.page_size;
  return ((int64_t)page * c.heads + head) * c.page_size + place;
}

inline CacheView cache_view(const mb_kv_cache* c) {
  return CacheView{{static_cast<uint8_t*>(c->k_codes), static_cast<uint8_t*>(c->v_codes)},
                   {static_cast<uint8_t*>(c->k_scales), static_cast<uint8_t*>(c->v_scales)},
                   c->pages,
                   (uint32_t)c->page_size,
                   (uint32_t)c->kv_heads,
                   (uint32_t)c->head_dim};
}

inline mb_status check_cache(const mb_kv_cache* c) {
  MB_REQUIRE(c != nullptr, "null cache");
  MB_REQUIRE(c->k_codes && c->v_codes && c->k_scales && c->v_scales,
             "cache pointers must not be null");
  MB_REQUIRE(aligned(c->k_codes, 16) && aligned(c->v_codes, 16) && aligned(c->k_scales, 16) &&
                 aligned(c->v_scales, 16),
             "cache pointers must be 16-byte aligned");
  MB_REQUIRE(c->bits == 8 || c->bits == 4, "bits must be 8 or 4");
  MB_REQUIRE(c->pages > 0 && c->kv_heads > 0, "pages and kv_heads must be positive");
  MB_REQUIRE(c->page_size > 0 && c->page_size % 16 == 0, "page_size must be a multiple of 16");
  MB_REQUIRE(c->head_dim > 0 && c->head_dim <= 256 &&
                 c->head_dim % (c->bits == 8 ? 16 : kGroup4) == 0,
             c->bits == 8 ? "head_dim must be a multiple of 16 up to 256"
                          : "head_dim must be a multiple of 32 up to 256");
  MB_REQUIRE(c->kv_heads <= 4096, "too many kv_heads");
  MB_REQUIRE(c->pages <= (int64_t(1) << 31) - 1 &&
                 c->pages * c->page_size <= (int64_t(1) << 32) - 2,
             "too many slots");
  return MB_OK;
}

}  // namespace mb

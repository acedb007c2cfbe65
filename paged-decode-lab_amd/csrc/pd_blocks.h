// What the cache operators share: the cache types and the block of a cache page.
#pragma once

#include <cstdint>
#include <type_traits>

#include "paged_decode.h"

namespace pd {

constexpr int kBlock = PD_BLOCK;  // slots per block, four blocks a page

inline bool valid_cache(int32_t type) { return type == PD_CACHE_BF16 || type == PD_CACHE_E4M3; }

// go(integral constant D, bool constant: e4m3) for a valid head_dim and cache type.
template <typename Go>
inline void for_cache(int head_dim, int32_t cache_type, Go go) {
  const auto with = [&](auto dim) {
    if (cache_type == PD_CACHE_E4M3)
      go(dim, std::true_type{});
    else
      go(dim, std::false_type{});
  };
  if (head_dim == 64)
    with(std::integral_constant<int, 64>{});
  else if (head_dim == 128)
    with(std::integral_constant<int, 128>{});
  else
    with(std::integral_constant<int, 256>{});
}

}  // namespace pd

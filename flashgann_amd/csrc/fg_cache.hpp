// fg_cache.hpp -- a paged key/value cache as the kernels see it.
#ifndef FG_CACHE_HPP
#define FG_CACHE_HPP

#include <cstdint>

#include "fg_host.hpp"

namespace fgk {

// n / d for 0 <= n < 2^31 without a division: d <= 2^shift, mul = ceil(2^32 *
// (2^shift / d - 1)), so (n * mul / 2^32 + n) / 2^shift is exact there and the
// sum stays below 2^32.
struct FastDiv {
    uint32_t mul, shift, d;
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

inline FastDiv fast_div(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {static_cast<uint32_t>(((1ull << 32) * ((1ull << s) - d)) / d + 1), s, d};
}

struct CacheView {
    const char *k, *v;
    int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
    uint32_t pages;
    FastDiv page_size;
};

// Checks a cache's sizes and type, its pointers and strides aside; FG_OK or a reported failure.
int check_cache_shape(const fg_kv_cache *c);

// Checks the cache and fills its view; FG_OK or a reported failure.  Without `values`, for a
// call that reads keys alone, v may be NULL.
int check_cache(const fg_kv_cache *c, CacheView *view, bool values = true);

}  // namespace fgk

#endif

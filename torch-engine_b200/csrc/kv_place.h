// Where a position of a sequence lives in a paged cache: shared by the kernels that write, read and attend to it, and
// plain C++ on the host, so that the arithmetic is checked without a GPU.
#pragma once
#include <stdint.h>

#if defined(__CUDACC__)
#define TE_HD __host__ __device__ __forceinline__
#else
#define TE_HD inline
#endif

namespace te {

// Exact division of n < 2^31 by a divisor in [1, 2^31) with one multiplication: L = ceil(log2 divisor),
// m = ceil(2^(31 + L) / divisor) < 2^32, quotient = (n * m) >> (31 + L).  m * divisor exceeds 2^(31 + L) by less than
// divisor <= 2^L, and n times that stays below 2^(31 + L): too little to carry the quotient over the next whole number.
struct FastDivisor {
    uint32_t divisor, factor;
    int32_t shift;
};
inline FastDivisor make_fast_divisor(uint32_t d) {
    int l = 0;
    while ((uint64_t(1) << l) < d) ++l;
    const uint64_t m = ((uint64_t(1) << (31 + l)) + d - 1) / d;
    return FastDivisor{d, (uint32_t)m, 31 + l};
}
TE_HD uint32_t fast_quotient(uint32_t n, const FastDivisor& f) { return (uint32_t)(((uint64_t)n * f.factor) >> f.shift); }

// The row of a page table as the descriptors give it.
struct PageRow {
    const int64_t* entries;
    int64_t max_pages;     // entries of the row
    int64_t pages;         // pages of the cache
};

// Page and slot of `position` >= 0.  False when it lies beyond the table or the table names no page of the cache.
TE_HD bool kv_place(const PageRow& row, const FastDivisor& page_size, int64_t position, int64_t& page, uint32_t& slot) {
    if (position < 0 || position >= row.max_pages * (int64_t)page_size.divisor) return false;   // the product is below 2^31 (checked by the host)
    const uint32_t i = fast_quotient((uint32_t)position, page_size);
    slot = (uint32_t)position - i * page_size.divisor;
    page = row.entries[i];
    return page >= 0 && page < row.pages;
}

}  // namespace te

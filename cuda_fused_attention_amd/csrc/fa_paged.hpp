// Host-side checks shared by the entry points that take a paged cache.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/fa_mi355x.h"

namespace fa {

inline bool misaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

inline bool bad_block_size(int b) { return b < 16 || b > (1 << 20) || (b & (b - 1)) != 0; }

// Layout of a cache: pages of a power of two of tokens (16 rows of a page are
// copied as one piece), rows of contiguous elements on 16-byte boundaries, rows of
// a page in rising order within 2^30 elements, pages at most 2^34 apart.
inline int check_paged_cache(const fa_paged_cache& c)
{
    if (c.dtype != FA_DTYPE_BF16 && c.dtype != FA_DTYPE_FP16) return hipErrorInvalidValue;
    if (c.num_blocks < 0 || c.heads_kv < 0 || c.head_dim < 1 || c.head_dim % 8 != 0) return hipErrorInvalidValue;
    if (bad_block_size(c.block_size)) return hipErrorInvalidValue;
    if (c.block_stride < 0 || c.head_stride < 0 || ((c.block_stride | c.head_stride | c.token_stride) & 7) != 0)
        return hipErrorInvalidValue;
    if (c.token_stride < c.head_dim || c.token_stride >= (1LL << 26)) return hipErrorInvalidValue;
    if (c.token_stride * c.block_size > (1LL << 30) || c.block_stride > (1LL << 34)) return hipErrorInvalidValue;
    if (c.num_blocks > 0 && c.heads_kv > 0 && (!c.k || !c.v || misaligned16(c.k) || misaligned16(c.v)))
        return hipErrorInvalidValue;
    return hipSuccess;
}

}  // namespace fa

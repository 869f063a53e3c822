// Division of cache positions by the block size as a multiply-high. Plain C++, so that the host can test it.
#pragma once

#include <stdint.h>

namespace xlite {

// m with position / block_size == mulhi(position, m) for every position below `positions`, or 0: divide. m = floor(2^32 /
// block_size) + 1 is too large by at most 1, so the product is too large by less than position * block_size / 2^32 of one
// quotient: exact while positions * block_size < 2^32. A block size of 1 has no such m (2^32 + 1 needs 33 bits).
inline uint32_t block_magic(uint32_t block_size, uint64_t positions)
{
    return block_size > 1 && positions * block_size < (1ull << 32) ? static_cast<uint32_t>((1ull << 32) / block_size) + 1 : 0u;
}

}  // namespace xlite

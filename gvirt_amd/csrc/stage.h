// Copies from global memory straight into LDS, and the layout of the tiles they fill: shared by the kernels that stage rows
// of 16-bit elements for 32x32x16 matrix products.
#pragma once

#include "common.h"

namespace xlite {
namespace stage {

// One wave-wide copy of 1 KiB into LDS at `lds_addr` + 16 * lane, from base + voff (a lane's own). The compiler sees neither
// the LDS write nor the memory counter: completion is awaited with wait<N> (at most N later copies outstanding). A register that
// a lane read wrote (the base itself, or a spilled half of it) needs five wait states before a memory instruction reads it, which
// the compiler does not insert in front of what it does not see: the copy brings them.
__device__ __forceinline__ void copy_1k(uint32_t lds_addr, uint32_t voff, const void *base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2\n\t"
                 :: "s"(lds_addr), "v"(voff), "s"(base) : "memory", "m0");
}
// the same for bytes that nobody reads again: they displace nothing on their way through the caches
__device__ __forceinline__ void copy_1k_once(uint32_t lds_addr, uint32_t voff, const void *base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2 nt\n\t"
                 :: "s"(lds_addr), "v"(voff), "s"(base) : "memory", "m0");
}
// the same from an address per lane, 16 or 4 bytes each
__device__ __forceinline__ void copy_lanes_16(uint32_t lds_addr, const void *src)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\t" :: "s"(lds_addr), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void copy_lanes_16_once(uint32_t lds_addr, const void *src)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt\n\t" :: "s"(lds_addr), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void copy_lanes_4(uint32_t lds_addr, const void *src)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\t" :: "s"(lds_addr), "v"(src) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait()
{
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(N) : "memory");
}

// address of dynamic LDS, as a scalar
__device__ __forceinline__ uint32_t lds_address(const void *p)
{
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(
        static_cast<uint32_t>((size_t)((__attribute__((address_space(3))) const unsigned char *)p)))));
}

// Tiles of rows of D 16-bit elements (64, 128 or 256), 16-byte chunks XOR-swizzled by the row so that 32 rows of one chunk (the
// operand of a product) are read without bank conflicts. A 256-byte bank window holds two rows of 64 elements, one of 128 or
// half a row of 256 (whose halves have the row's pattern).
template <int D>
__device__ __forceinline__ uint32_t pattern(uint32_t window)
{
    static_assert(D == 256 || D == 128 || D == 64, "tiles exist for rows of 64, 128 and 256 elements");
    return D >= 128 ? (((window & 3) << 2) | ((window >> 2) & 3)) : (((window & 1) << 2) | ((window >> 1) & 3));
}
// byte offset of chunk 2 ks + half of row `row`: row_offset + chunk_offset(ks)
template <int D>
__device__ __forceinline__ uint32_t row_offset(uint32_t row)
{
    return D == 64 ? (row >> 1) * 256 : row * (D * 2);
}
template <int D>
__device__ __forceinline__ uint32_t row_swizzle(uint32_t row, uint32_t half)
{
    return D == 64 ? ((((row & 1) << 3) | half) ^ pattern<D>(row >> 1)) << 4 : (half ^ pattern<D>(row)) << 4;
}
__device__ __forceinline__ uint32_t chunk_offset(uint32_t ks, uint32_t swizzle)
{
    return (((2 * (ks & 7u)) << 4) ^ swizzle) + (ks >> 3) * 256;
}
// what lane `lane` of the copy that fills rows first .. first + 1024 / (2 D) - 1 has to fetch: its row of them and chunk
template <int D>
__device__ __forceinline__ void copy_source(uint32_t lane, uint32_t first, uint32_t *row, uint32_t *chunk)
{
    if constexpr (D == 256) {
        *row = lane >> 5;
        *chunk = ((lane & 15u) ^ pattern<D>(first + (lane >> 5))) | ((lane >> 4) & 1u) << 4;
    } else if constexpr (D == 128) {
        *row = lane >> 4;
        *chunk = (lane & 15u) ^ pattern<D>(first + (lane >> 4));
    } else {
        const uint32_t c = (lane & 15u) ^ pattern<D>((first >> 1) + (lane >> 4));
        *row = 2 * (lane >> 4) + (c >> 3);
        *chunk = c & 7u;
    }
}

}  // namespace stage
}  // namespace xlite

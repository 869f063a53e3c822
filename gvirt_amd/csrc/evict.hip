// A cache that is kept to a budget: which positions stay (select_kept) and their rows moved to the front
// (compact_kv_cache, also used for the accepted path of a drafted tree).
#include <algorithm>

#include "attention_common.h"

namespace xlite {

namespace {

// ---- select_kept ------------------------------------------------------------------------------------------------------
// Per (sequence, kv head): the first `sink` and the last `recent` positions, and of the positions between them the n =
// budget - sink - recent with the largest weights; equal weights go to the lower position. A radix selection: the n-th
// largest key is found 8 bits at a time with a histogram in LDS, then one pass in position order writes the positions
// whose key is larger, and the first ones that equal it. Counts only, so the result does not depend on any order.
constexpr int kSelThreads = 1024;

// weights in the order of a descending sort: NaN first, -0 and +0 alike
__device__ __forceinline__ uint32_t weight_key(float w)
{
    w += 0.0f;
    if (w != w) {
        return 0xffffffffu;
    }
    const uint32_t b = __builtin_bit_cast(uint32_t, w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct SelectParams {
    const float *weights;
    int32_t *kept;
    int32_t *kept_lens;
    const int32_t *context_lens;
    const int32_t *block_tables;
    uint32_t n_kv_heads, block_size, max_num_block, budget, recent, sink;
};

__global__ void __launch_bounds__(kSelThreads)
select_kept_kernel(const SelectParams p)
{
    constexpr int WAVES = kSelThreads / 64;
    __shared__ uint32_t hist[256];
    __shared__ uint32_t found[2];            // the digit, and how many keys of the bins above it were taken
    __shared__ uint2 wave_count[WAVES];
    const uint32_t seq = blockIdx.x / p.n_kv_heads, kvh = blockIdx.x % p.n_kv_heads;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t length = min(static_cast<uint32_t>(max(p.context_lens[seq], 0)), p.max_num_block * p.block_size);
    int32_t *out = p.kept + static_cast<uint64_t>(blockIdx.x) * p.budget;
    const uint32_t count = min(length, p.budget);
    if (kvh == 0 && threadIdx.x == 0) {
        p.kept_lens[seq] = static_cast<int32_t>(count);
    }
    for (uint32_t i = count + threadIdx.x; i < p.budget; i += kSelThreads) {
        out[i] = -1;
    }
    if (length <= p.budget) {
        for (uint32_t i = threadIdx.x; i < length; i += kSelThreads) {
            out[i] = static_cast<int32_t>(i);
        }
        return;
    }
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    auto key_at = [&](uint32_t pos) {
        const uint32_t b = pos / p.block_size;
        const uint64_t slot = static_cast<uint64_t>(static_cast<uint32_t>(table[b])) * p.block_size + (pos - b * p.block_size);
        return weight_key(p.weights[slot * p.n_kv_heads + kvh]);
    };
    const uint32_t lo = p.sink, hi = length - p.recent;   // the judged positions
    const uint32_t n = p.budget - p.sink - p.recent;      // fewer than hi - lo: length > budget
    // ---- the n-th largest key, and how many of the keys equal to it are taken
    uint32_t threshold = 0, equal = 0;
    if (n > 0) {
        uint32_t left = n, prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (threadIdx.x < 256) {
                hist[threadIdx.x] = 0;
            }
            __syncthreads();
            for (uint32_t i = lo + threadIdx.x; i < hi; i += kSelThreads) {
                const uint32_t k = key_at(i);
                if (shift == 24 || (k >> (shift + 8)) == prefix) {
                    atomicAdd(&hist[(k >> shift) & 255u], 1u);
                }
            }
            __syncthreads();
            if (wave == 0) {
                // lane l: bins 255 - 4 l .. 252 - 4 l, in descending order
                uint32_t c[4], sum = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    c[e] = hist[255 - 4 * lane - e];
                    sum += c[e];
                }
                uint32_t incl = sum;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const uint32_t up = __shfl_up(incl, d);
                    incl += lane >= static_cast<uint32_t>(d) ? up : 0u;
                }
                uint32_t above = incl - sum;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (above < left && left <= above + c[e]) {   // exactly one bin of one lane
                        found[0] = 255 - 4 * lane - e;
                        found[1] = above;
                    }
                    above += c[e];
                }
            }
            __syncthreads();
            prefix = prefix << 8 | found[0];
            left -= found[1];
        }
        threshold = prefix;
        equal = left;
    }
    // ---- the kept positions in order
    for (uint32_t i = threadIdx.x; i < p.sink; i += kSelThreads) {
        out[i] = static_cast<int32_t>(i);
    }
    for (uint32_t i = threadIdx.x; i < p.recent; i += kSelThreads) {
        out[p.sink + n + i] = static_cast<int32_t>(hi + i);
    }
    if (n == 0) {
        return;
    }
    uint32_t above_before = 0, equal_before = 0;
    for (uint32_t i0 = lo; i0 < hi; i0 += kSelThreads) {
        const uint32_t i = i0 + threadIdx.x;
        const uint32_t k = key_at(min(i, hi - 1));
        const bool is_above = i < hi && k > threshold, is_equal = i < hi && k == threshold;
        const uint64_t above_mask = __ballot(is_above), equal_mask = __ballot(is_equal);
        __syncthreads();
        if (lane == 0) {
            wave_count[wave] = make_uint2(__builtin_popcountll(above_mask), __builtin_popcountll(equal_mask));
        }
        __syncthreads();
        uint32_t a = above_before, e = equal_before;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) {
            const uint2 c = wave_count[w];
            a += w < wave ? c.x : 0u;
            e += w < wave ? c.y : 0u;
            above_before += c.x;
            equal_before += c.y;
        }
        const uint64_t below = (1ull << lane) - 1;
        a += __builtin_popcountll(above_mask & below);
        e += __builtin_popcountll(equal_mask & below);
        if (is_above || (is_equal && e < equal)) {
            out[p.sink + a + min(e, equal)] = static_cast<int32_t>(i);
        }
    }
}

// ---- compact_kv_cache ---------------------------------------------------------------------------------------------------
// Position start + i of a sequence receives the row of position start + kept[i], kept[i] >= i, in place. The columns of a
// row are independent, so a workgroup owns a slice of the rows' bytes (or one fp32 per row: scales, weights) and walks the
// list in order, kBatch entries at a time: all of a batch is read before any of it is written, and what later batches read
// lies above everything written so far (kept[i] >= i), so one barrier per batch is all the order there is. Bound by
// memory: every moved row is read and written once.
constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;

struct CompactParams {
    unsigned char *k_cache, *v_cache;
    float *scalars[3];                  // per (slot, kv head): K scales, V scales, weights
    const int32_t *kept;
    const int32_t *kept_lens;
    const int32_t *starts;              // nullptr: 0
    const int32_t *block_tables;
    uint32_t n_kv_heads, block_size, max_num_block, max_kept;
    uint32_t per_head;                  // 1: a list per kv head, 0: one for all of them
    uint32_t row_bytes;                 // of a cache row that moves as one: a kv head's, or a position's
    uint32_t slices;                    // of a cache row
    uint32_t slice_bytes;
    uint32_t n_scalars;                 // columns of fp32: arrays x (1 | n_kv_heads)
};

// the walk: `lanes` threads per row, each with its own V at `column`
template <typename V>
__device__ __forceinline__ void move_rows(const CompactParams &p, V *data, uint64_t pitch, uint64_t column, uint32_t lanes,
                                          const int32_t *list, uint32_t count, uint32_t start, const int32_t *table)
{
    const uint32_t rows = kMoveThreads / lanes;          // rows of one instruction
    const uint32_t mine = threadIdx.x / lanes;
    const uint32_t capacity = p.max_num_block * p.block_size;
    const uint64_t at = column + threadIdx.x % lanes;
    auto row_of = [&](uint32_t pos) {
        const uint32_t b = pos / p.block_size;
        return static_cast<uint64_t>(static_cast<uint32_t>(table[b])) * p.block_size + (pos - b * p.block_size);
    };
    for (uint32_t i0 = 0; i0 < count; i0 += rows * kMoveUnroll) {
        uint32_t src[kMoveUnroll];
        bool ok[kMoveUnroll];
        V x[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; u++) {
            const uint32_t i = i0 + u * rows + mine;
            src[u] = static_cast<uint32_t>(list[min(i, count - 1)]);
            // (a row that stays where it is, and entries that break the rules: nothing is read or written)
            ok[u] = i < count && src[u] > i && src[u] < capacity - start;
        }
#pragma unroll
        for (int u = 0; u < kMoveUnroll; u++) {
            if (ok[u]) {
                x[u] = data[row_of(start + src[u]) * pitch + at];
            }
        }
        __builtin_amdgcn_s_waitcnt(0);   // the values are here, not only asked for, before anyone writes
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveUnroll; u++) {
            if (ok[u]) {
                data[row_of(start + i0 + u * rows + mine) * pitch + at] = x[u];
            }
        }
    }
}

__global__ void __launch_bounds__(kMoveThreads)
compact_kernel(const CompactParams p)
{
    const uint32_t lists = p.per_head ? p.n_kv_heads : 1u;
    const uint32_t seq = blockIdx.y / lists, head = blockIdx.y % lists;
    const uint32_t count = min(static_cast<uint32_t>(max(p.kept_lens[seq], 0)), p.max_kept);
    const uint32_t start = p.starts != nullptr ? static_cast<uint32_t>(max(p.starts[seq], 0)) : 0u;
    if (count == 0 || start >= p.max_num_block * p.block_size) {
        return;
    }
    const int32_t *list = p.kept + static_cast<uint64_t>(blockIdx.y) * p.max_kept;
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    const uint32_t part = blockIdx.x;
    if (part < 2 * p.slices) {
        unsigned char *cache = part < p.slices ? p.k_cache : p.v_cache;
        const uint64_t pitch = static_cast<uint64_t>(p.row_bytes) * (p.per_head ? p.n_kv_heads : 1u) / 16;
        const uint64_t column = (static_cast<uint64_t>(head) * p.row_bytes + (part % p.slices) * p.slice_bytes) / 16;
        move_rows<uint4>(p, reinterpret_cast<uint4 *>(cache), pitch, column, p.slice_bytes / 16, list, count, start, table);
    } else {
        const uint32_t c = part - 2 * p.slices;
        const uint32_t per_array = p.per_head ? 1u : p.n_kv_heads;
        move_rows<float>(p, p.scalars[c / per_array], p.n_kv_heads, p.per_head ? head : c % per_array, 1, list, count, start, table);
    }
}

}  // namespace

}  // namespace xlite

using namespace xlite;

extern "C" int xlite_hip_select_kept(void *stream, const float *weights, int32_t *kept, int32_t *kept_lens,
                                     const int32_t *context_lens, const int32_t *block_tables, uint32_t n_kv_heads,
                                     uint32_t block_size, uint32_t batch, uint32_t max_num_block, uint32_t budget,
                                     uint32_t recent, uint32_t sink)
{
    if (batch == 0) {
        return XLITE_HIP_OK;
    }
    XL_REQUIRE(weights && kept && kept_lens && context_lens && block_tables, "null tensor");
    XL_REQUIRE(n_kv_heads > 0 && block_size > 0 && max_num_block > 0, "zero head count or block geometry");
    XL_REQUIRE(static_cast<uint64_t>(max_num_block) * block_size < (1ull << 31), "block tables reach beyond 2^31 positions");
    XL_REQUIRE(budget > 0 && budget < (1u << 31), "budget must be positive");
    XL_REQUIRE(static_cast<uint64_t>(recent) + sink <= budget, "recent + sink must not exceed budget");
    XL_REQUIRE(static_cast<uint64_t>(batch) * n_kv_heads < (1ull << 31), "more lists than one launch takes");
    SelectParams p{weights, kept, kept_lens, context_lens, block_tables, n_kv_heads, block_size, max_num_block, budget, recent, sink};
    select_kept_kernel<<<batch * n_kv_heads, kSelThreads, 0, as_stream(stream)>>>(p);
    XL_LAUNCH_CHECK();
    return XLITE_HIP_OK;
}

extern "C" int xlite_hip_compact_kv_cache(void *stream, void *k_cache, void *v_cache, float *k_scale, float *v_scale,
                                          float *weights, const int32_t *kept, const int32_t *kept_lens, const int32_t *starts,
                                          const int32_t *block_tables, uint32_t n_kv_heads, uint32_t head_dim,
                                          uint32_t block_size, uint32_t batch, uint32_t max_num_block, uint32_t max_kept,
                                          int per_head, int kv_dtype)
{
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || kv_dtype == XLITE_HIP_KV_INT8 || kv_dtype == XLITE_HIP_KV_FP8,
               "kv cache dtype unsupported!");
    if (batch == 0 || max_kept == 0) {
        return XLITE_HIP_OK;
    }
    XL_REQUIRE(k_cache && v_cache && kept && kept_lens && block_tables, "null tensor");
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || (k_scale && v_scale), "a quantised KV cache needs k_scale and v_scale");
    XL_REQUIRE(n_kv_heads > 0 && head_dim > 0 && block_size > 0 && max_num_block > 0, "zero head count or block geometry");
    XL_REQUIRE(static_cast<uint64_t>(max_num_block) * block_size < (1ull << 31), "block tables reach beyond 2^31 positions");
    const uint64_t head_bytes = static_cast<uint64_t>(head_dim) * (kv_dtype == XLITE_HIP_KV_SAME ? 2 : 1);
    XL_REQUIRE(head_bytes % 16 == 0, "a kv head's row must be a multiple of 16 bytes");
    XL_REQUIRE((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) % 16 == 0,
               "caches must be aligned to 16 bytes");
    CompactParams p{};
    p.k_cache = static_cast<unsigned char *>(k_cache);
    p.v_cache = static_cast<unsigned char *>(v_cache);
    p.kept = kept;
    p.kept_lens = kept_lens;
    p.starts = starts;
    p.block_tables = block_tables;
    p.n_kv_heads = n_kv_heads;
    p.block_size = block_size;
    p.max_num_block = max_num_block;
    p.max_kept = max_kept;
    p.per_head = per_head ? 1u : 0u;
    const uint64_t row = head_bytes * (per_head ? 1u : n_kv_heads);
    XL_REQUIRE(row < (1ull << 31), "a position's row is too long");
    p.row_bytes = static_cast<uint32_t>(row);
    // slices of 128 bytes (a cache line), or less where the row is no multiple of it
    p.slice_bytes = row % 128 == 0 ? 128u : row % 64 == 0 ? 64u : row % 32 == 0 ? 32u : 16u;
    p.slices = p.row_bytes / p.slice_bytes;
    uint32_t arrays = 0;
    for (float *x : {kv_dtype == XLITE_HIP_KV_SAME ? nullptr : k_scale, kv_dtype == XLITE_HIP_KV_SAME ? nullptr : v_scale, weights}) {
        if (x != nullptr) {
            p.scalars[arrays++] = x;
        }
    }
    p.n_scalars = arrays * (per_head ? 1u : n_kv_heads);
    const uint64_t lists = static_cast<uint64_t>(batch) * (per_head ? n_kv_heads : 1u);
    XL_REQUIRE(lists <= 65535, "more lists than one launch takes");
    compact_kernel<<<dim3(2 * p.slices + p.n_scalars, static_cast<uint32_t>(lists)), kMoveThreads, 0, as_stream(stream)>>>(p);
    XL_LAUNCH_CHECK();
    return XLITE_HIP_OK;
}

// A cache that is kept to a budget: which positions stay (select_kept) and their rows moved to the front
// (compact_kv_cache, also used for the accepted path of a drafted tree).
#include <algorithm>

#include "attention_common.h"
#include "block_magic.h"

namespace xlite {

namespace {

// ---- select_kept ------------------------------------------------------------------------------------------------------
// Per (sequence, kv head): the first `sink` and the last `recent` positions, and of the positions between them the n =
// budget - sink - recent with the largest weights; equal weights go to the lower position. A radix selection: the n-th
// largest key is found digit by digit with histograms in LDS, then the
// positions whose key is larger, and the first ones that equal it, are written in position order. Counts only, so the result
// does not depend on any order. One workgroup per (sequence, kv head); the keys are read once, into registers.
// A weight's neighbours in memory belong to the other kv heads: the heads of a sequence run on one XCD, at the same time, so
// that its lines come from memory once and from that XCD's L2 for the other heads.
// Measured, 64 sequences x 8 heads, an eighth kept: 16 us over 4000 positions, 32 over 16000, 58 over 32000, 114 over 64000;
// one sequence of 32000 34 us. The weights of 64 x 32768 positions are 67 MB, 13 us at the rate of a copy. What bounds it: the loads,
// 27 us of the 58. A quarter's keys are converted in the loop that loads them, and the compiler has 16 loads under way only in the first
// two quarters of 64 keys: in the others every load is awaited before the next, 32 trips to memory in a row (48 with 1024 threads). It
// is not the bytes out of L2, eight times the list's because a wave's keys lie 32 bytes apart: two heads a workgroup in neighbouring
// lanes fetch half the lines and took 57 us (and 47 instead of 34 for one sequence). The histograms take 11, the ballots 3, the output 5.
constexpr uint32_t kXcds = 8;
constexpr uint32_t kSelTable = 4096;   // block-table entries in LDS
constexpr int kAhead = 16;   // loads a thread has under way

// weights in the order of a descending sort: NaN first, -0 and +0 alike; never 0, which stands for "no weight"
__device__ __forceinline__ uint32_t weight_key(float w)
{
    w += 0.0f;
    const uint32_t b = __builtin_bit_cast(uint32_t, w);
    const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return w != w ? 0xffffffffu : k;
}

struct SelectParams {
    const float *weights;
    int32_t *kept;
    int32_t *kept_lens;
    const int32_t *context_lens;
    const int32_t *block_tables;
    uint32_t n_kv_heads, block_size, max_num_block, budget, recent, sink, batch;
    uint32_t block_magic;   // see block_magic()
};

// The n-th largest of the keys (n > 0, at least n of them) and how many of those equal to it are among the n largest.
// each(f) calls f for every key of the thread (0: none). Digits of 11, 11 and 10 bits: the first one holds the sign, the
// exponent and two bits of the mantissa, so that few lanes of a wave meet in one bin (with 8 bits a dozen did, and the
// first pass took longer than the rest of the kernel together).
constexpr int kHistCopies = 4;
template <int T>
struct SelectScratch {
    uint32_t hist[kHistCopies][2048];
    uint32_t wave_sum[T / 64];
    uint32_t found[2];   // the digit, and how many keys lie in the bins above it
};
template <int T, typename EACH>
__device__ __forceinline__ void nth_largest(EACH &&each, uint32_t n, SelectScratch<T> &s, uint32_t *threshold, uint32_t *equal)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t *mine = s.hist[wave % kHistCopies];
    uint32_t left = n, prefix = 0;
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t bits = pass == 2 ? 10u : 11u;
#pragma unroll
        for (int i = 0; i < kHistCopies * 2048 / T; i++) {
            (&s.hist[0][0])[threadIdx.x + i * T] = 0;
        }
        __syncthreads();
        each([&](uint32_t k) {
            if (pass == 0 ? k != 0 : (k >> (shift + bits)) == prefix) {
                atomicAdd(&mine[(k >> shift) & ((1u << bits) - 1)], 1u);
            }
        });
        __syncthreads();
        // thread t: bins 2047 - P t, 2046 - P t, ..., in descending order
        constexpr int P = 2048 / T;
        uint32_t c[P] = {}, sum = 0;
#pragma unroll
        for (int h = 0; h < kHistCopies; h++) {
#pragma unroll
            for (int e = 0; e < P; e++) {
                c[e] += s.hist[h][2047 - P * threadIdx.x - e];
            }
        }
#pragma unroll
        for (int e = 0; e < P; e++) {
            sum += c[e];
        }
        uint32_t incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t up = __shfl_up(incl, d);
            incl += lane >= static_cast<uint32_t>(d) ? up : 0u;
        }
        if (lane == 63) {
            s.wave_sum[wave] = incl;
        }
        __syncthreads();
        uint32_t above = incl - sum;
#pragma unroll
        for (uint32_t w = 0; w < (T / 64); w++) {
            above += w < wave ? s.wave_sum[w] : 0u;
        }
#pragma unroll
        for (int e = 0; e < P; e++) {
            if (above < left && left <= above + c[e]) {   // exactly one bin of one thread
                s.found[0] = 2047 - P * threadIdx.x - e;
                s.found[1] = above;
            }
            above += c[e];
        }
        __syncthreads();
        prefix = prefix << bits | s.found[0];
        left -= s.found[1];
    }
    *threshold = prefix;
    *equal = left;
}

// T threads. KPT: keys a thread holds in registers (the judged positions fit KPT * T, the block table kSelTable; block_magic
// is there); 0: any length, the keys are read again in every pass
template <int KPT, int T>
__global__ void __launch_bounds__(T, KPT == 64 ? 4 : 1)
select_kept_kernel(const SelectParams p)
{
    __shared__ SelectScratch<T> scratch;
    __shared__ uint32_t table_lds[KPT > 0 ? kSelTable : 1];
    __shared__ uint2 counts[(KPT > 0 ? KPT : kAhead) * (T / 64)];   // (above, equal) of a wave's 64 positions, then the sums before them
    const uint32_t xcd = blockIdx.x % kXcds, place = blockIdx.x / kXcds;
    const uint32_t seq = place / p.n_kv_heads * kXcds + xcd, kvh = place % p.n_kv_heads;
    if (seq >= p.batch) {
        return;
    }
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t length = min(static_cast<uint32_t>(max(p.context_lens[seq], 0)), p.max_num_block * p.block_size);
    int32_t *out = p.kept + (static_cast<uint64_t>(seq) * p.n_kv_heads + kvh) * p.budget;
    const uint32_t count = min(length, p.budget);
    if (kvh == 0 && threadIdx.x == 0) {
        p.kept_lens[seq] = static_cast<int32_t>(count);
    }
    for (uint32_t i = count + threadIdx.x; i < p.budget; i += T) {
        out[i] = -1;
    }
    if (length <= p.budget) {
        for (uint32_t i = threadIdx.x; i < length; i += T) {
            out[i] = static_cast<int32_t>(i);
        }
        return;
    }
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    if constexpr (KPT > 0) {
        for (uint32_t i = threadIdx.x; i < ceil_div(length, p.block_size); i += T) {
            table_lds[i] = static_cast<uint32_t>(table[i]);
        }
        __syncthreads();
    }
    auto key_at = [&](uint32_t pos) {
        const uint32_t b = KPT > 0 || p.block_magic != 0 ? __umulhi(pos, p.block_magic) : pos / p.block_size;
        const uint32_t entry = KPT > 0 ? table_lds[b] : static_cast<uint32_t>(table[b]);
        const uint64_t slot = static_cast<uint64_t>(entry) * p.block_size + (pos - b * p.block_size);
        return weight_key(p.weights[slot * p.n_kv_heads + kvh]);
    };
    const uint32_t lo = p.sink, hi = length - p.recent;   // the judged positions
    const uint32_t n = p.budget - p.sink - p.recent;      // fewer than hi - lo: length > budget
    for (uint32_t i = threadIdx.x; i < p.sink; i += T) {
        out[i] = static_cast<int32_t>(i);
    }
    for (uint32_t i = threadIdx.x; i < p.recent; i += T) {
        out[p.sink + n + i] = static_cast<int32_t>(hi + i);
    }
    if (n == 0) {
        return;
    }
    const uint64_t below = (1ull << lane) - 1;
    uint32_t threshold, equal;
    if constexpr (KPT > 0) {
        // A quarter of the keys at a time, as far as the list reaches: f(j) for the keys of the quarters it has, rest(j) for the others.
        constexpr int QUARTER = KPT / 4;
        auto quarters = [&](auto &&f, auto &&rest) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < 4; g++) {
                if (lo + g * QUARTER * T < hi) {
#pragma unroll
                    for (int j = g * QUARTER; j < (g + 1) * QUARTER; j++) {
                        f(j);
                    }
                } else {
#pragma unroll
                    for (int j = g * QUARTER; j < (g + 1) * QUARTER; j++) {
                        rest(j);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);   // (all of a thread's loads under way: their addresses would take the keys' registers)
            }
        };
        auto nothing = [](int) {};
        uint32_t key[KPT];
        quarters([&](int j) {
            const uint32_t i = lo + j * T + threadIdx.x;
            const uint32_t k = key_at(min(i, hi - 1));
            key[j] = i < hi ? k : 0u;
        }, [&](int j) { key[j] = 0; });
        nth_largest<T>([&](auto &&f) {
            quarters([&](int j) { f(key[j]); }, nothing);
        }, n, scratch, &threshold, &equal);
        quarters([&](int j) {
            const uint64_t a = __ballot(key[j] > threshold), e = __ballot(key[j] == threshold);
            if (lane == 0) {
                counts[j * (T / 64) + wave] = make_uint2(__builtin_popcountll(a), __builtin_popcountll(e));
            }
        }, [&](int j) {
            if (lane == 0) {
                counts[j * (T / 64) + wave] = make_uint2(0, 0);
            }
        });
        __syncthreads();
        if (wave == 0) {   // exclusive sums in position order: lane l owns KPT / 4 consecutive entries
            constexpr int PER = (KPT * (T / 64) + 63) / 64;
            uint2 sum = make_uint2(0, 0);
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const uint2 c = counts[lane * PER + i];
                sum.x += c.x;
                sum.y += c.y;
            }
            uint2 incl = sum;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t ux = __shfl_up(incl.x, d), uy = __shfl_up(incl.y, d);
                incl.x += lane >= static_cast<uint32_t>(d) ? ux : 0u;
                incl.y += lane >= static_cast<uint32_t>(d) ? uy : 0u;
            }
            uint2 before = make_uint2(incl.x - sum.x, incl.y - sum.y);
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const uint2 c = counts[lane * PER + i];
                counts[lane * PER + i] = before;
                before.x += c.x;
                before.y += c.y;
            }
        }
        __syncthreads();
        // compared and counted anew below: kept over the barrier the ballots and positions take more registers than the keys
        uint32_t first = lo + threadIdx.x;
        asm volatile("" : "+v"(threshold), "+v"(first));
        quarters([&](int j) {
            const bool is_above = key[j] > threshold, is_equal = key[j] == threshold;
            const uint64_t am = __ballot(is_above), em = __ballot(is_equal);
            const uint2 before = counts[j * (T / 64) + wave];
            const uint32_t a = before.x + __builtin_popcountll(am & below), e = before.y + __builtin_popcountll(em & below);
            if (is_above || (is_equal && e < equal)) {
                out[p.sink + a + min(e, equal)] = static_cast<int32_t>(first + j * T);
            }
        }, nothing);
    } else {
        nth_largest<T>([&](auto &&f) {
            for (uint32_t i0 = lo + threadIdx.x; i0 < hi; i0 += kAhead * T) {
                uint32_t key[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; j++) {
                    key[j] = key_at(min(i0 + j * T, hi - 1));
                }
#pragma unroll
                for (int j = 0; j < kAhead; j++) {
                    if (i0 + j * T < hi) {
                        f(key[j]);
                    }
                }
            }
        }, n, scratch, &threshold, &equal);
        uint32_t above_before = 0, equal_before = 0;
        for (uint32_t i0 = lo; i0 < hi; i0 += kAhead * T) {
            uint32_t key[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const uint32_t i = i0 + j * T + threadIdx.x;
                key[j] = key_at(min(i, hi - 1));
                key[j] = i < hi ? key[j] : 0u;
            }
            __syncthreads();   // the counts of the round before have been read
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const uint64_t above_mask = __ballot(key[j] > threshold), equal_mask = __ballot(key[j] == threshold);
                if (lane == 0) {
                    counts[j * (T / 64) + wave] = make_uint2(__builtin_popcountll(above_mask), __builtin_popcountll(equal_mask));
                }
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kAhead; j++) {
                const bool is_above = key[j] > threshold, is_equal = key[j] == threshold;
                uint32_t a = above_before + __builtin_popcountll(__ballot(is_above) & below);
                uint32_t e = equal_before + __builtin_popcountll(__ballot(is_equal) & below);
#pragma unroll
                for (uint32_t w = 0; w < T / 64; w++) {
                    const uint2 c = counts[j * (T / 64) + w];
                    a += w < wave ? c.x : 0u;
                    e += w < wave ? c.y : 0u;
                    above_before += c.x;
                    equal_before += c.y;
                }
                if (is_above || (is_equal && e < equal)) {
                    out[p.sink + a + min(e, equal)] = static_cast<int32_t>(i0 + j * T + threadIdx.x);
                }
            }
        }
    }
}

// ---- compact_kv_cache ---------------------------------------------------------------------------------------------------
// Position start + i of a sequence receives the row of position start + kept[i], kept[i] >= i, in place. The columns of a
// row are independent, so a workgroup owns a slice of the rows' bytes (or one fp32 per row: scales, weights) and walks the
// list in order, a batch of entries at a time: all of a batch is read before any of it is written (a barrier), and what later
// batches read lies above everything written so far (kept[i] >= i), so the next batch may be read ahead of that barrier. Measured: 16
// sequences of 8192 positions cut to 2048 per head of 8 (128 elements of 16 bits, and the weights), 135 MB moved: 60 us, 4.5 TB/s
// read and written (a plain copy of as many bytes takes 52); 64 paths of 6 rows 5.5 us. What bounds it beside the bytes: the table entry
// comes from LDS or from memory by a choice of addresses, a load that the compiler awaits together with everything else, so that
// the rows of a batch are fetched one after the other; a path's few rows pay for whole batches of them.
constexpr int kMoveUnroll = 4;
constexpr uint32_t kMoveTable = 4096;   // block-table entries kept in LDS (longer tables are read from memory)

struct CompactParams {
    unsigned char *k_cache, *v_cache;
    float *scalars[3];                  // per (slot, kv head): K scales, V scales, weights
    const int32_t *kept;
    const int32_t *kept_lens;
    const int32_t *starts;              // nullptr: 0
    const int32_t *block_tables;
    uint32_t n_kv_heads, block_size, max_num_block, max_kept;
    uint32_t block_magic;               // as in SelectParams
    uint32_t per_head;                  // 1: a list per kv head, 0: one for all of them
    uint32_t row_bytes;                 // of a cache row that moves as one: a kv head's, or a position's
    uint32_t slices;                    // of a cache row
    uint32_t slice_bytes;
    uint32_t n_scalars;                 // columns of fp32: arrays x (1 | n_kv_heads)
};

// the walk: `lanes` threads per row, each with its own V at `column`
template <typename V, typename ROW>
__device__ __forceinline__ void move_rows(V *data, uint64_t pitch, uint64_t column, uint32_t lanes, const int32_t *list, uint32_t count,
                                          uint32_t start, uint32_t capacity, ROW &&row_of)
{
    constexpr int U = kMoveUnroll;
    const uint32_t rows = blockDim.x / lanes;          // rows of one instruction
    const uint32_t mine = threadIdx.x / lanes;
    V *base = data + column + threadIdx.x % lanes;
    const uint32_t batch = rows * U;
    uint32_t src[U];
    V x[U], y[U];
    bool ok[U], ok_next[U];
    auto read_list = [&](uint32_t i0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            src[u] = static_cast<uint32_t>(list[min(i0 + u * rows + mine, count - 1)]);
        }
    };
    // (a row that stays where it is, and entries that break the rules: nothing is written, and the load is one of the row
    // that stands there, whatever it holds)
    auto read_rows = [&](uint32_t i0, V (&v)[U], bool (&good)[U]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = i0 + u * rows + mine;
            good[u] = i < count && src[u] > i && src[u] < capacity - start;
            v[u] = base[row_of(start + (good[u] ? src[u] : 0u)) * pitch];
        }
    };
    read_list(0);
    read_rows(0, x, ok);
    read_list(min(batch, count - 1));
    for (uint32_t i0 = 0; i0 < count; i0 += batch) {
        read_rows(i0 + batch, y, ok_next);
        read_list(min(i0 + 2 * batch, count - 1));
        // this batch's values are here, not only asked for, before anyone writes
#pragma unroll
        for (int u = 0; u < U; u++) {
            if constexpr (sizeof(V) == 16) {
                asm volatile("" : "+v"(x[u].x), "+v"(x[u].y), "+v"(x[u].z), "+v"(x[u].w));
            } else {
                asm volatile("" : "+v"(x[u]));
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = i0 + u * rows + mine;
            if (ok[u] && start + i < capacity) {
                base[row_of(start + i) * pitch] = x[u];
            }
            x[u] = y[u];
            ok[u] = ok_next[u];
        }
    }
}

__global__ void __launch_bounds__(1024)
compact_kernel(const CompactParams p)
{
    __shared__ uint32_t table_lds[kMoveTable];
    const uint32_t lists = p.per_head ? p.n_kv_heads : 1u;
    const uint32_t seq = blockIdx.y / lists, head = blockIdx.y % lists;
    const uint32_t count = min(static_cast<uint32_t>(max(p.kept_lens[seq], 0)), p.max_kept);
    const uint32_t start = p.starts != nullptr ? static_cast<uint32_t>(max(p.starts[seq], 0)) : 0u;
    const uint32_t capacity = p.max_num_block * p.block_size;
    if (count == 0 || start >= capacity) {
        return;
    }
    const int32_t *list = p.kept + static_cast<uint64_t>(blockIdx.y) * p.max_kept;
    const int32_t *table = p.block_tables + static_cast<uint64_t>(seq) * p.max_num_block;
    const uint32_t part = blockIdx.x;
    const uint32_t first = start / p.block_size;
    for (uint32_t i = threadIdx.x; i < min(p.max_num_block - first, kMoveTable); i += blockDim.x) {
        table_lds[i] = static_cast<uint32_t>(table[first + i]);
    }
    __syncthreads();
    auto row_of = [&](uint32_t pos) {
        const uint32_t b = p.block_magic != 0 ? __umulhi(pos, p.block_magic) : pos / p.block_size;
        const uint32_t entry = b - first < kMoveTable ? table_lds[b - first] : static_cast<uint32_t>(table[b]);
        return static_cast<uint64_t>(entry) * p.block_size + (pos - b * p.block_size);
    };
    if (part < 2 * p.slices) {
        unsigned char *cache = part < p.slices ? p.k_cache : p.v_cache;
        const uint64_t pitch = static_cast<uint64_t>(p.row_bytes) * (p.per_head ? p.n_kv_heads : 1u) / 16;
        const uint64_t column = (static_cast<uint64_t>(head) * p.row_bytes + (part % p.slices) * p.slice_bytes) / 16;
        move_rows<uint4>(reinterpret_cast<uint4 *>(cache), pitch, column, p.slice_bytes / 16, list, count, start, capacity, row_of);
    } else {
        const uint32_t c = part - 2 * p.slices;
        const uint32_t per_array = p.per_head ? 1u : p.n_kv_heads;
        move_rows<float>(p.scalars[c / per_array], p.n_kv_heads, p.per_head ? head : c % per_array, 1, list, count, start, capacity, row_of);
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
    XL_REQUIRE((static_cast<uint64_t>(batch) + kXcds) * n_kv_heads < (1ull << 31), "more lists than one launch takes");
    // (the list of one head is written while the others still read the lengths)
    XL_REQUIRE(kept_lens != context_lens, "kept_lens must not be context_lens");
    SelectParams p{weights, kept, kept_lens, context_lens, block_tables, n_kv_heads, block_size, max_num_block,
                   budget, recent, sink, batch, block_magic(block_size, static_cast<uint64_t>(max_num_block) * block_size)};
    const uint64_t grid = (static_cast<uint64_t>(batch) + kXcds - 1) / kXcds * kXcds * n_kv_heads;
    const uint32_t judged = max_num_block * block_size - std::min(max_num_block * block_size, sink + recent);   // at most
    hipStream_t s = as_stream(stream);
    const dim3 g(static_cast<uint32_t>(grid));
    // The fewest keys a thread that hold the longest list: keys beyond a list's end cost their step all the same. 512 threads
    // up to 32768, where two workgroups share a compute unit (64 x 8 lists of 32000: 58 us; 1024 threads with 40 keys
    // and one workgroup 70); 1024 beyond (64000: 114 us). Reading the keys again in every pass costs 413 there with a load at a
    // time; it remains for what no workgroup can hold (100000: 490 with 16 under way) and for tables that do not fit LDS.
    const bool registers = max_num_block <= kSelTable && p.block_magic != 0;
    if (!registers) {
        select_kept_kernel<0, 1024><<<g, 1024, 0, s>>>(p);
    } else if (judged <= 4 * 1024) {
        select_kept_kernel<4, 1024><<<g, 1024, 0, s>>>(p);
    } else if (judged <= 16 * 1024) {
        select_kept_kernel<16, 1024><<<g, 1024, 0, s>>>(p);
    } else if (judged <= 64 * 512) {
        select_kept_kernel<64, 512><<<g, 512, 0, s>>>(p);
    } else if (judged <= 64 * 1024) {
        select_kept_kernel<64, 1024><<<g, 1024, 0, s>>>(p);
    } else {
        select_kept_kernel<0, 1024><<<g, 1024, 0, s>>>(p);
    }
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
    XL_REQUIRE(aligned16(k_cache) && aligned16(v_cache), "caches must be aligned to 16 bytes");
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
    p.block_magic = block_magic(block_size, static_cast<uint64_t>(max_num_block) * block_size);
    // slices of 256 bytes, or the largest power of two below that divides the row
    p.slice_bytes = std::min(256u, p.row_bytes & (~p.row_bytes + 1u));
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
    // long lists: 16 waves keep a compute unit's share of the memory busy; a path's few rows fit 4
    const uint32_t threads = max_kept > 64 ? 1024u : 256u;
    compact_kernel<<<dim3(2 * p.slices + p.n_scalars, static_cast<uint32_t>(lists)), threads, 0, as_stream(stream)>>>(p);
    XL_LAUNCH_CHECK();
    return XLITE_HIP_OK;
}

// Which path of a drafted tree the model itself takes (greedy): from node 0 on, the token of the largest logit of the node's
// row; if a child carries that token the path goes on there, otherwise the token is the sequence's next one.
// The path is not known before its logits are read, one row after the other. A few rows are all read at once by as many
// workgroups as there is room for and the walk only compares what they found (a tree of 8 over 32000 logits: 3.3 us and 3.2 us
// of walking, launch-bound); many rows would be mostly rows off the path, so that a workgroup per sequence reads those of
// its path (64 trees of up to 32 over 131072 16-bit logits, paths of up to 4, 64 MB: 23 us, 2.8 TB/s; 64 of the 256 compute units
// are at work, each in dependent trips to memory; reading all 1047 rows, 274 MB, would take 43).
#include <algorithm>

#include "attention_common.h"

namespace xlite {

namespace {

// ---- the largest logit of a row -------------------------------------------------------------------------------------------
// Values are compared, not mapped to ordered keys: a chunk of 16 bytes costs its maximum (v_maximum3: NaN wins, which is the
// order wanted) and one comparison with the thread's best; where in the chunk it lies is looked up once, at the end. With a
// 64-bit key per logit the vector instructions took longer than the memory: 10 us for a row of 131072 in one workgroup.
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

struct F32 {
    typedef float stored;
    static constexpr uint32_t kPer = 4;   // logits of 16 bytes
    static __device__ __forceinline__ float value(float x) { return x; }
    static __device__ __forceinline__ float most(const uint4 &w)
    {
        const f32x4v x = __builtin_bit_cast(f32x4v, w);
        return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[0], x[1]), __builtin_elementwise_maximum(x[2], x[3]));
    }
};
struct F16 {
    typedef uint16_t stored;
    static constexpr uint32_t kPer = 8;
    static __device__ __forceinline__ float value(uint16_t x) { return FP16::to_f32(x); }
    static __device__ __forceinline__ float most(const uint4 &w)
    {
        const f16x2v a = __builtin_elementwise_maximum(__builtin_bit_cast(f16x2v, w.x), __builtin_bit_cast(f16x2v, w.y));
        const f16x2v b = __builtin_elementwise_maximum(__builtin_bit_cast(f16x2v, w.z), __builtin_bit_cast(f16x2v, w.w));
        const f16x2v c = __builtin_elementwise_maximum(a, b);
        return static_cast<float>(__builtin_elementwise_maximum(c[0], c[1]));
    }
};
struct B16 {
    typedef uint16_t stored;
    static constexpr uint32_t kPer = 8;
    static __device__ __forceinline__ float value(uint16_t x) { return BF16::to_f32(x); }
    static __device__ __forceinline__ float most(const uint4 &w)
    {
        auto two = [](uint32_t x) { return __builtin_elementwise_maximum(BF16::lo(x), BF16::hi(x)); };
        return __builtin_elementwise_maximum(__builtin_elementwise_maximum(two(w.x), two(w.y)), __builtin_elementwise_maximum(two(w.z), two(w.w)));
    }
};

// the best of a thread, a wave, a workgroup: a value and the chunk that it was first seen in
struct Best {
    float v;
    uint32_t at;
};
// whether value a goes before value b whatever their places (NaN before everything)
__device__ __forceinline__ bool ahead(float a, float b) { return (a > b) | ((a != a) & (b == b)); }
__device__ __forceinline__ Best better(Best a, Best b)
{
    const float av = a.v, bv = b.v;   // (chosen between as values: as fields the choice becomes one of addresses, in memory)
    const uint32_t ai = a.at, bi = b.at;
    const bool take_b = ahead(bv, av) | (!ahead(av, bv) & (bi < ai));
    return Best{take_b ? bv : av, take_b ? bi : ai};
}

// A part of a row: first the logits up to the first 16-byte boundary and those behind the last one, in chunk numbers that
// keep the order (head 0, body 1 + i, tail last), then the body's chunks.
template <typename L>
struct Row {
    const typename L::stored *row;
    uint32_t vocab, head, body;   // logits ahead of the first boundary, whole chunks
    __device__ __attribute__((always_inline)) Row(const void *logits, uint64_t index, uint32_t vocab_)
    {
        const typename L::stored *r = static_cast<const typename L::stored *>(logits) + index * vocab_;
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(r) & 15u);
        const uint32_t to_boundary = ((16u - off) & 15u) / static_cast<uint32_t>(sizeof(typename L::stored));
        const uint32_t h = vocab_ < to_boundary ? vocab_ : to_boundary;
        row = r;
        vocab = vocab_;
        head = h;
        body = (vocab_ - h) / L::kPer;
    }
    __device__ __forceinline__ uint32_t first_of(uint32_t chunk) const { return chunk == 0 ? 0u : head + (chunk - 1) * L::kPer; }
    __device__ __forceinline__ uint32_t size_of(uint32_t chunk) const
    {
        const uint32_t h = head, tail = vocab - h - body * L::kPer;
        const uint32_t n = chunk > body ? tail : static_cast<uint32_t>(L::kPer);
        return chunk == 0 ? h : n;
    }
    // chunks first, first + step, ... < end of the body, and the two ragged ones (by the first 16 threads) if `ends`
    template <int U>
    __device__ __attribute__((always_inline)) Best scan(uint32_t first, uint32_t step, uint32_t end, bool ends) const
    {
        Best best{-INFINITY, 0xffffffffu};
        const uint4 *chunks = reinterpret_cast<const uint4 *>(row + head);
        for (uint32_t i0 = first; i0 < end; i0 += step * U) {
            uint4 w[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                w[u] = chunks[min(i0 + u * step, end - 1)];   // (past the end: the last one again, which changes nothing)
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float m = L::most(w[u]);
                const uint32_t at = 1 + min(i0 + u * step, end - 1);
                const bool take = ahead(m, best.v) || best.at == 0xffffffffu;
                best.v = take ? m : best.v;
                best.at = take ? at : best.at;
            }
        }
        if (ends && threadIdx.x < 16) {   // one logit per thread
            const uint32_t c = threadIdx.x < 8 ? 0u : body + 1, i = threadIdx.x & 7u;
            if (i < size_of(c)) {
                best = better(best, Best{L::value(row[first_of(c) + i]), c});
            }
        }
        return best;
    }
    // the first logit of the chunk with that value, for a whole wave (16 bytes hold at most eight)
    __device__ __forceinline__ uint32_t place(Best b, uint32_t lane) const
    {
        const uint32_t first = first_of(b.at), n = size_of(b.at);
        const float x = L::value(row[first + min(lane, n - 1)]);
        const uint64_t hits = __ballot(lane < n && (x == b.v || (x != x && b.v != b.v)));
        return first + __builtin_ctzll(hits | 1ull << 63);   // (there is one: the value came from this chunk)
    }
};

__device__ __forceinline__ Best best_of_wave(Best b)
{
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        b = better(b, Best{__shfl_xor(b.v, d), static_cast<uint32_t>(__shfl_xor(static_cast<int>(b.at), d))});
    }
    return b;
}

// the first child of `node` that carries `token`, or -1, for a whole wave (children stand behind their parent: a path grows
// with every step)
__device__ __forceinline__ int32_t child_of(const int32_t *tokens, const int32_t *parents, int32_t node, int32_t nodes, int32_t token, uint32_t lane)
{
    for (int32_t c0 = node + 1; c0 < nodes; c0 += 64) {
        const int32_t c = c0 + static_cast<int32_t>(lane);
        const int32_t at = min(c, nodes - 1);
        const int32_t parent = parents[at], carried = tokens[at];   // (one trip to memory for the two)
        const uint64_t hits = __ballot(c < nodes && parent == node && carried == token);
        if (hits != 0) {
            return c0 + __builtin_ctzll(hits);
        }
    }
    return -1;
}

struct VerifyParams {
    const void *logits;
    const int32_t *tokens, *parents, *query_start_loc, *lens;
    int32_t *accepted, *n_accepted, *next_token;
    Best *parts;              // [row][chunks]
    uint32_t vocab, max_path, parts_per_row;
};

constexpr int kPartThreads = 256;
constexpr int kWalkThreads = 1024;

// ---- few rows: every row's best, a row by several workgroups, then the walk over them ------------------------------------
template <typename L>
__global__ void __launch_bounds__(kPartThreads)
row_parts_kernel(const VerifyParams p)
{
    __shared__ Best wave_best[kPartThreads / 64];
    const Row<L> row(p.logits, blockIdx.y, p.vocab);
    const uint32_t per = ceil_div(row.body, p.parts_per_row);
    const uint32_t first = blockIdx.x * per, end = min(row.body, first + per);
    const Best b = best_of_wave(row.template scan<4>(first + threadIdx.x, kPartThreads, end, blockIdx.x == 0));
    if ((threadIdx.x & 63) == 0) {
        wave_best[threadIdx.x >> 6] = b;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        Best all = wave_best[0];
#pragma unroll
        for (int w = 1; w < kPartThreads / 64; w++) {
            all = better(all, wave_best[w]);
        }
        p.parts[static_cast<uint64_t>(blockIdx.y) * p.parts_per_row + blockIdx.x] = all;
    }
}

// one wave per sequence
template <typename L>
__global__ void __launch_bounds__(64)
walk_kernel(const VerifyParams p)
{
    const uint32_t seq = blockIdx.x, lane = threadIdx.x;
    const int32_t nodes = p.lens[seq];
    const uint64_t start = static_cast<uint32_t>(p.query_start_loc[seq]);
    int32_t *path = p.accepted + static_cast<uint64_t>(seq) * p.max_path;
    int32_t node = 0, next = -1;
    uint32_t n = 0;
    while (nodes > 0 && n < p.max_path) {
        if (lane == 0) {
            path[n] = node;
        }
        n++;
        const Best *parts = p.parts + (start + node) * p.parts_per_row;
        Best b = parts[min(lane, p.parts_per_row - 1)];
        b = best_of_wave(b);
        next = static_cast<int32_t>(Row<L>(p.logits, start + node, p.vocab).place(b, lane));
        const int32_t child = child_of(p.tokens + start, p.parents + start, node, nodes, next, lane);
        if (child < 0) {
            break;
        }
        node = child;
    }
    for (uint32_t i = n + lane; i < p.max_path; i += 64) {
        path[i] = -1;
    }
    if (lane == 0) {
        p.n_accepted[seq] = static_cast<int32_t>(n);
        p.next_token[seq] = next;
    }
}

// ---- many rows: one workgroup per sequence reads the rows of its path only ------------------------------------------------
template <typename L>
__global__ void __launch_bounds__(kWalkThreads)
walk_rows_kernel(const VerifyParams p)
{
    __shared__ Best wave_best[kWalkThreads / 64];
    const uint32_t seq = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int32_t nodes = p.lens[seq];
    const uint64_t start = static_cast<uint32_t>(p.query_start_loc[seq]);
    int32_t *path = p.accepted + static_cast<uint64_t>(seq) * p.max_path;
    int32_t node = 0, next = -1;
    uint32_t n = 0;
    while (nodes > 0 && n < p.max_path) {
        if (threadIdx.x == 0) {
            path[n] = node;
        }
        n++;
        const Row<L> row(p.logits, start + node, p.vocab);
        Best b = best_of_wave(row.template scan<8>(threadIdx.x, kWalkThreads, row.body, true));
        __syncthreads();   // (the last round's values have been read)
        if (lane == 0) {
            wave_best[wave] = b;
        }
        __syncthreads();
        b = best_of_wave(wave_best[lane % (kWalkThreads / 64)]);
        next = static_cast<int32_t>(row.place(b, lane));
        const int32_t child = child_of(p.tokens + start, p.parents + start, node, nodes, next, lane);   // the same in every wave
        if (child < 0) {
            break;
        }
        node = child;
    }
    for (uint32_t i = n + threadIdx.x; i < p.max_path; i += kWalkThreads) {
        path[i] = -1;
    }
    if (threadIdx.x == 0) {
        p.n_accepted[seq] = static_cast<int32_t>(n);
        p.next_token[seq] = next;
    }
}

// Up to so many rows all of them are read, by as many workgroups as there is room for; beyond, each sequence's workgroup
// reads the rows of its path one after the other (131072 fp32 logits, trees of 32, paths of up to 8: 12 trees all read 40 us, 13
// walked 55).
constexpr uint32_t kAllRows = 384;
uint32_t parts_per_row(uint32_t rows)
{
    return rows == 0 || rows > kAllRows ? 0u : std::max(1u, std::min(64u, 1024u / rows));
}

}  // namespace

}  // namespace xlite

using namespace xlite;

extern "C" size_t xlite_hip_verify_tree_workspace_bytes(uint32_t total_tokens)
{
    return static_cast<size_t>(total_tokens) * parts_per_row(total_tokens) * sizeof(Best);
}

extern "C" int xlite_hip_verify_tree(void *stream, const void *logits, const int32_t *tokens, const int32_t *parents,
                                     int32_t *accepted, int32_t *n_accepted, int32_t *next_token,
                                     const int32_t *query_start_loc, const int32_t *lens, uint32_t total_tokens, uint32_t vocab,
                                     uint32_t batch, uint32_t max_path, int dtype, void *workspace, size_t workspace_bytes)
{
    XL_REQUIRE(dtype == XLITE_HIP_FP16 || dtype == XLITE_HIP_BF16 || dtype == XLITE_HIP_FP32, "logits dtype unsupported!");
    if (batch == 0) {
        return XLITE_HIP_OK;
    }
    XL_REQUIRE(accepted && n_accepted && next_token && query_start_loc && lens, "null tensor");
    XL_REQUIRE(total_tokens == 0 || (logits && tokens && parents), "null tensor");
    XL_REQUIRE(max_path > 0, "accepted must hold at least one node");
    XL_REQUIRE(total_tokens == 0 || (vocab > 0 && vocab < (1u << 31)), "the vocabulary must not be empty");
    XL_REQUIRE(total_tokens < (1u << 31) && batch < (1u << 31), "more rows than one launch takes");
    XL_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == XLITE_HIP_FP32 ? 4 : 2) == 0, "logits must be aligned to their type");
    const size_t need = xlite_hip_verify_tree_workspace_bytes(total_tokens);
    if (need != 0 && (workspace == nullptr || workspace_bytes < need)) {
        return fail(XLITE_HIP_ENOSPC, __func__, "workspace too small: need " + std::to_string(need) + " bytes, have " +
                                                    std::to_string(workspace == nullptr ? 0 : workspace_bytes));
    }
    hipStream_t s = as_stream(stream);
    VerifyParams p{logits, tokens, parents, query_start_loc, lens, accepted, n_accepted, next_token, static_cast<Best *>(workspace),
                   vocab, max_path, parts_per_row(total_tokens)};
    auto launch = [&](auto type) -> int {
        using L = decltype(type);
        if (p.parts_per_row == 0) {
            walk_rows_kernel<L><<<batch, kWalkThreads, 0, s>>>(p);
        } else {
            row_parts_kernel<L><<<dim3(p.parts_per_row, total_tokens), kPartThreads, 0, s>>>(p);
            XL_LAUNCH_CHECK();
            walk_kernel<L><<<batch, 64, 0, s>>>(p);
        }
        XL_LAUNCH_CHECK();
        return XLITE_HIP_OK;
    };
    return dtype == XLITE_HIP_FP32 ? launch(F32{}) : dtype == XLITE_HIP_BF16 ? launch(B16{}) : launch(F16{});
}

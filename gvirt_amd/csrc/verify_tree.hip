// Which path of a drafted tree the model itself takes (greedy): from node 0 on, the token of the largest logit of the node's
// row; if a child carries that token the path goes on there, otherwise the token is the sequence's next one.
#include "attention_common.h"

namespace xlite {

namespace {

// logits in the order of their values, NaN above everything, -0 and +0 alike; with the index in the low half so that the
// largest of several equal ones is the one at the lowest index
__device__ __forceinline__ uint64_t ranked(float x, uint32_t i)
{
    x += 0.0f;
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const uint32_t key = x != x ? 0xffffffffu : (b & 0x80000000u ? ~b : b | 0x80000000u);
    return static_cast<uint64_t>(key) << 32 | ~i;
}

struct F32 {
    typedef float stored;
    static __device__ __forceinline__ float value(float x) { return x; }
};
struct F16 {
    typedef uint16_t stored;
    static __device__ __forceinline__ float value(uint16_t x) { return FP16::to_f32(x); }
};
struct B16 {
    typedef uint16_t stored;
    static __device__ __forceinline__ float value(uint16_t x) { return BF16::to_f32(x); }
};

constexpr int kThreads = 256;

// one workgroup per row
template <typename L>
__global__ void __launch_bounds__(kThreads)
row_choice_kernel(const typename L::stored *__restrict__ logits, int32_t *__restrict__ choice, uint32_t vocab)
{
    __shared__ uint64_t wave_best[kThreads / 64];
    const typename L::stored *row = logits + static_cast<uint64_t>(blockIdx.x) * vocab;
    uint64_t best = 0;
    for (uint32_t i = threadIdx.x; i < vocab; i += kThreads) {
        const uint64_t x = ranked(L::value(row[i]), i);
        best = x > best ? x : best;
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const uint64_t x = __shfl_xor(best, d);
        best = x > best ? x : best;
    }
    if ((threadIdx.x & 63) == 0) {
        wave_best[threadIdx.x >> 6] = best;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 64; w++) {
            best = wave_best[w] > best ? wave_best[w] : best;
        }
        choice[blockIdx.x] = static_cast<int32_t>(~static_cast<uint32_t>(best));
    }
}

// one wave per sequence
__global__ void __launch_bounds__(64)
walk_kernel(const int32_t *__restrict__ choice, const int32_t *__restrict__ tokens, const int32_t *__restrict__ parents,
            int32_t *__restrict__ accepted, int32_t *__restrict__ n_accepted, int32_t *__restrict__ next_token,
            const int32_t *__restrict__ query_start_loc, const int32_t *__restrict__ lens, uint32_t max_path)
{
    const uint32_t seq = blockIdx.x, lane = threadIdx.x;
    const int32_t nodes = lens[seq];
    const uint64_t start = static_cast<uint32_t>(query_start_loc[seq]);
    int32_t *path = accepted + static_cast<uint64_t>(seq) * max_path;
    int32_t node = 0, next = -1;
    uint32_t n = 0;
    while (nodes > 0 && n < max_path) {
        if (lane == 0) {
            path[n] = node;
        }
        n++;
        next = choice[start + node];
        // the first child with that token (children stand behind their parent: the path grows with every turn)
        int32_t child = -1;
        for (int32_t c0 = node + 1; c0 < nodes && child < 0; c0 += 64) {
            const int32_t c = c0 + static_cast<int32_t>(lane);
            const bool hit = c < nodes && parents[start + c] == node && tokens[start + c] == next;
            const uint64_t hits = __ballot(hit);
            child = hits != 0 ? c0 + __builtin_ctzll(hits) : -1;
        }
        if (child < 0) {
            break;
        }
        node = child;
    }
    for (uint32_t i = n + lane; i < max_path; i += 64) {
        path[i] = -1;
    }
    if (lane == 0) {
        n_accepted[seq] = static_cast<int32_t>(n);
        next_token[seq] = next;
    }
}

}  // namespace

}  // namespace xlite

using namespace xlite;

extern "C" size_t xlite_hip_verify_tree_workspace_bytes(uint32_t total_tokens)
{
    return static_cast<size_t>(total_tokens) * sizeof(int32_t);
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
    const size_t need = xlite_hip_verify_tree_workspace_bytes(total_tokens);
    if (need != 0 && (workspace == nullptr || workspace_bytes < need)) {
        return fail(XLITE_HIP_ENOSPC, __func__, "workspace too small: need " + std::to_string(need) + " bytes, have " +
                                                    std::to_string(workspace == nullptr ? 0 : workspace_bytes));
    }
    hipStream_t s = as_stream(stream);
    int32_t *choice = static_cast<int32_t *>(workspace);
    if (total_tokens != 0) {
        switch (dtype) {
        case XLITE_HIP_FP32:
            row_choice_kernel<F32><<<total_tokens, kThreads, 0, s>>>(static_cast<const float *>(logits), choice, vocab);
            break;
        case XLITE_HIP_BF16:
            row_choice_kernel<B16><<<total_tokens, kThreads, 0, s>>>(static_cast<const uint16_t *>(logits), choice, vocab);
            break;
        default:
            row_choice_kernel<F16><<<total_tokens, kThreads, 0, s>>>(static_cast<const uint16_t *>(logits), choice, vocab);
        }
        XL_LAUNCH_CHECK();
    }
    walk_kernel<<<batch, 64, 0, s>>>(choice, tokens, parents, accepted, n_accepted, next_token, query_start_loc, lens, max_path);
    XL_LAUNCH_CHECK();
    return XLITE_HIP_OK;
}

// C entry point of the attention over drafted trees: argument checks and kernel selection. The rows of a step are the
// nodes of one drafted tree per sequence, already written to the cache behind the cached positions; a row sees every
// cached position and those nodes whose bit its mask has:
//     out_r = sum_j [seen(r, j)] exp(q_r . k_j) v_j / sum_j [seen(r, j)] exp(q_r . k_j),   0 where nothing is seen.
// A kernel of its own streams the cache past all rows of a tree (tree_stream.hip).
// Other shapes: the walk is that of a prefill chunk with another mask, and only tiles that reach into the tree look at it, so
// the prefill kernels serve them with a mask of their own (prefill_mfma.hip, mfma_attention.hip: TREE).
#include <algorithm>

#include "attention_common.h"

using namespace xlite;

namespace {

// scratch of the 16-bit kernels, whichever serves the shape
size_t tree_bytes_16(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t batch,
                     uint32_t max_ctx)
{
    const uint32_t splits = mfma_pick_splits(total_tokens, n_heads / n_kv_heads, batch, n_kv_heads, max_ctx, 64);
    return std::max(mfma_workspace_bytes(total_tokens, n_heads, head_dim, splits + 1),
                    prefill_mfma_workspace_bytes(total_tokens, n_heads, n_kv_heads, head_dim, batch, max_ctx));
}

int run_16(hipStream_t s, const AttentionArgs &a)
{
    return prefill_mfma_supported(a) ? launch_prefill_mfma(s, a) : launch_mfma_gqa(s, a);
}

}  // namespace

extern "C" size_t xlite_hip_tree_attention_workspace_bytes(uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads,
                                                           uint32_t head_dim, uint32_t block_size, uint32_t batch,
                                                           uint32_t max_num_block, int kv_dtype)
{
    if (total_tokens == 0 || batch == 0 || n_kv_heads == 0 || n_heads % n_kv_heads != 0 || head_dim < 8 || block_size == 0) {
        return 0;
    }
    // the kernel that serves the shape, and nothing for those that would with less
    if (tree_stream_supported(n_heads, n_kv_heads, head_dim, block_size, batch, max_num_block, kv_dtype)) {
        return tree_stream_workspace_bytes(total_tokens, n_heads, n_kv_heads, head_dim, batch, block_size, max_num_block);
    }
    size_t need = tree_bytes_16(total_tokens, n_heads, n_kv_heads, head_dim, batch, max_num_block * block_size);
    AttentionArgs shape{};
    const float scale = 1.f;
    shape.n_heads = n_heads;
    shape.n_kv_heads = n_kv_heads;
    shape.head_dim = head_dim;
    shape.block_size = block_size;
    shape.max_num_block = max_num_block;
    shape.kv_dtype = kv_dtype;
    shape.k_scale = shape.v_scale = &scale;
    if (kv_dtype != XLITE_HIP_KV_SAME && !prefill_kv8_supported(shape)) {
        need += kv_dequant_bytes(n_kv_heads, head_dim, block_size, batch, max_num_block);
        need += kv_dequant_f16_io_bytes(total_tokens, n_heads, n_kv_heads, head_dim);   // bf16 models (the size does not know)
    }
    return need;
}

extern "C" int xlite_hip_tree_attention(void *stream, const void *qkv, const void *k_cache, const void *v_cache, void *output,
                                        const int32_t *tree_mask, uint32_t mask_words, const int32_t *query_start_loc,
                                        const int32_t *lens, const int32_t *cached_lens, const int32_t *block_tables,
                                        uint32_t total_tokens, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                                        uint32_t block_size, uint32_t batch, uint32_t max_num_block, int dtype, int kv_dtype,
                                        const float *k_scale, const float *v_scale, void *workspace, size_t workspace_bytes)
{
    XL_REQUIRE(dtype == XLITE_HIP_FP16 || dtype == XLITE_HIP_BF16, "qkv/kCache/vCache/output dtype unsupported!");
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || kv_dtype == XLITE_HIP_KV_INT8 || kv_dtype == XLITE_HIP_KV_FP8,
               "kv cache dtype unsupported!");
    if (batch == 0 || total_tokens == 0) {
        return XLITE_HIP_OK;
    }
    XL_REQUIRE(qkv && k_cache && v_cache && output && tree_mask && query_start_loc && lens && cached_lens && block_tables,
               "null tensor");
    XL_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0,
               "n_heads must be a positive multiple of n_kv_heads");
    XL_REQUIRE(block_size > 0 && max_num_block > 0, "block_size and max_num_block must be positive");
    XL_REQUIRE(static_cast<uint64_t>(max_num_block) * block_size < (1ull << 31), "block tables reach beyond 2^31 positions");
    XL_REQUIRE(mask_words > 0 && mask_words <= (1u << 22), "mask_words must be positive, at most 2^22");
    XL_REQUIRE(mfma_gqa_supported(head_dim), "head_dim must be 64, 128 or 256");
    XL_REQUIRE(static_cast<uint64_t>(total_tokens) * n_heads < (1ull << 31) &&
                   ceil_div(total_tokens * (n_heads / n_kv_heads), 128u) + batch <= 65535 && n_kv_heads <= 65535,
               "more rows than one launch takes");
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || (k_scale && v_scale), "a quantised KV cache needs k_scale and v_scale");
    XL_REQUIRE(kv_dtype == XLITE_HIP_KV_SAME || head_dim != 256, "quantised KV caches: head_dim must be 64 or 128");
    XL_REQUIRE(aligned16(qkv) && aligned16(k_cache) && aligned16(v_cache) && aligned16(output) && aligned16(workspace),
               "qkv, caches, output and workspace must be aligned to 16 bytes");
    AttentionArgs a{qkv, k_cache, v_cache, output, query_start_loc, lens, cached_lens, block_tables,
                    total_tokens, n_heads, n_kv_heads, head_dim, block_size, batch, max_num_block,
                    dtype, kv_dtype, k_scale, v_scale, workspace, workspace_bytes};
    a.tree_mask = reinterpret_cast<const uint32_t *>(tree_mask);
    a.mask_words = mask_words;
    hipStream_t s = as_stream(stream);
    if (tree_stream_supported(n_heads, n_kv_heads, head_dim, block_size, batch, max_num_block, kv_dtype) && workspace != nullptr &&
        workspace_bytes >= tree_stream_workspace_bytes(total_tokens, n_heads, n_kv_heads, head_dim, batch, block_size, max_num_block)) {
        return launch_tree_stream(s, a);
    }
    if (kv_dtype == XLITE_HIP_KV_SAME) {
        return run_16(s, a);
    }
    // a cache of bytes: read by the prefill kernel itself (head_dim 128; a tree is a short chunk), otherwise through an
    // fp16 copy of the blocks the batch sees
    if (prefill_kv8_supported(a)) {
        return launch_prefill_mfma(s, a);
    }
    if (const int rc = launch_kv_dequant(s, &a)) {
        return rc;
    }
    if (dtype == XLITE_HIP_FP16) {
        return run_16(s, a);
    }
    AttentionArgs f = a;
    f.dtype = XLITE_HIP_FP16;
    if (prefill_mfma_supported(f)) {
        f.io_bf16 = true;
        return launch_prefill_mfma(s, f);
    }
    void *real_out = nullptr;
    if (const int rc = launch_kv_dequant_f16_begin(s, &a, &real_out)) {
        return rc;
    }
    if (const int rc = run_16(s, a)) {
        return rc;
    }
    return launch_kv_dequant_f16_finish(s, a, real_out);
}

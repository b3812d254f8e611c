// Attention of drafted tokens over a paged cache: the entry points, and the kernels over fp16 pools (mathematics and choices in
// paged_attn_tree.hpp).  The kernels take minutes to compile, so the three kinds of pool and rows have a source file each.
#include "paged_attn_tree.hpp"

namespace lg {

hipError_t tree_launch_fp16(const TreeParams& p, int d, hipStream_t stream) {
    return tree_by_width<PackedF16, false>(p, d, stream);
}

static logismos_status_t tree_attention(bool e4m3, bool bf16, const TreeParams& p, int hq, int d, float scale,
                                        logismos_stream_t stream) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (logismos_check_paged_attn_tree_shape(p.num_seqs, p.total, p.max_q, hq, p.hkv, d, p.block_size, p.max_blocks,
                                             p.num_blocks, p.words / 2, (int)p.q_stride, (int)p.out_stride, nullptr,
                                             0) != 0)
        return bad;
    if (!p.q || !p.k_pool || !p.v_pool || !p.tables || !p.cu || !p.ctx || !p.mask || !p.out || !p.ws) return bad;
    if (e4m3 && (!p.k_exp || !p.v_exp)) return bad;
    if ((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k_pool) |
         reinterpret_cast<uintptr_t>(p.v_pool) | reinterpret_cast<uintptr_t>(p.k_exp) |
         reinterpret_cast<uintptr_t>(p.v_exp) | reinterpret_cast<uintptr_t>(p.out) |
         reinterpret_cast<uintptr_t>(p.ws)) % 16 != 0 ||
        (reinterpret_cast<uintptr_t>(p.tables) | reinterpret_cast<uintptr_t>(p.cu) |
         reinterpret_cast<uintptr_t>(p.ctx)) % 4 != 0 ||
        reinterpret_cast<uintptr_t>(p.mask) % 8 != 0)
        return bad;
    TreeParams q = p;
    q.g = hq / p.hkv;
    q.scale_log2e = scale * 1.4426950408889634f;
    if (!(scale > 0.0f) || !isfinite(q.scale_log2e)) return bad;
    hipStream_t st = static_cast<hipStream_t>(stream);
    return static_cast<logismos_status_t>(!e4m3 ? tree_launch_fp16(q, d, st)
                                          : bf16 ? tree_launch_e4m3_bf16(q, d, st)
                                                 : tree_launch_e4m3_fp16(q, d, st));
}

}  // namespace lg

extern "C" {

logismos_status_t logismos_check_paged_attn_tree_shape(int num_seqs, int total_tokens, int max_seqlen_q,
                                                       int num_q_heads, int num_kv_heads, int head_dim,
                                                       int block_size, int max_blocks_per_seq, int num_blocks,
                                                       int mask_words, int q_stride, int out_stride, char* msg,
                                                       size_t cap) {
    using lg::reject;
    if (num_seqs <= 0 || total_tokens <= 0 || max_seqlen_q <= 0)
        return reject(msg, cap, "num_seqs, total_tokens and max_seqlen_q must be positive (%d, %d, %d)", num_seqs,
                      total_tokens, max_seqlen_q);
    if (num_seqs > 65535 || total_tokens > 65535)
        return reject(msg, cap, "num_seqs and total_tokens must be <= 65535 (%d, %d)", num_seqs, total_tokens);
    if (max_seqlen_q > total_tokens)
        return reject(msg, cap, "max_seqlen_q %d exceeds total_tokens %d", max_seqlen_q, total_tokens);
    if (num_q_heads <= 0 || num_kv_heads <= 0)
        return reject(msg, cap, "num_q_heads and num_kv_heads must be positive (%d, %d)", num_q_heads, num_kv_heads);
    if (num_q_heads % num_kv_heads != 0)
        return reject(msg, cap, "num_q_heads %d is not a multiple of num_kv_heads %d", num_q_heads, num_kv_heads);
    if (head_dim <= 0 || head_dim % 32 != 0 || head_dim > 256)
        return reject(msg, cap, "head_dim must be a multiple of 32 up to 256 (%d)", head_dim);
    if (block_size <= 0 || block_size % 16 != 0)
        return reject(msg, cap, "block_size must be a positive multiple of 16 (%d)", block_size);
    if (max_blocks_per_seq <= 0 || num_blocks <= 0)
        return reject(msg, cap, "max_blocks_per_seq and num_blocks must be positive (%d, %d)", max_blocks_per_seq,
                      num_blocks);
    if ((int64_t)block_size * max_blocks_per_seq > INT32_MAX - 64 || (int64_t)block_size * num_blocks > INT32_MAX)
        return reject(msg, cap, "block_size * max_blocks_per_seq or block_size * num_blocks exceeds i32::MAX");
    if (mask_words <= 0 || mask_words > lg::kTreeMaskWords || max_seqlen_q > 64 * mask_words)
        return reject(msg, cap, "mask_words must be between 1 and %d, with a bit for each of max_seqlen_q tokens (%d, %d)",
                      lg::kTreeMaskWords, mask_words, max_seqlen_q);
    const int64_t width = (int64_t)num_q_heads * head_dim;
    if (width > (1 << 20)) return reject(msg, cap, "num_q_heads * head_dim exceeds %d", 1 << 20);
    if (q_stride < width || out_stride < width)
        return reject(msg, cap, "a stride is smaller than its row (%d and %d of %lld)", q_stride, out_stride,
                      (long long)width);
    if ((q_stride | out_stride) % 8 != 0)
        return reject(msg, cap, "strides must be multiples of 8 (%d, %d)", q_stride, out_stride);
    if (out_stride > (1 << 22)) return reject(msg, cap, "out_stride must be at most %d (%d)", 1 << 22, out_stride);
    // tiles of all units, and workgroups of the second launch
    const int64_t units = lg::packed_tiles(total_tokens, num_seqs, num_q_heads / num_kv_heads, 128) * num_kv_heads;
    const int64_t tiles = ((int64_t)block_size * max_blocks_per_seq + 31) / 32;
    if (units > (1 << 22) || tiles > INT32_MAX / units)
        return reject(msg, cap, "too many key tiles: %lld units of columns with up to %lld each", (long long)units,
                      (long long)tiles);
    return 0;
}

size_t logismos_paged_attn_tree_workspace_bytes(int total_tokens, int max_seqlen_q, int num_q_heads, int num_kv_heads,
                                                int head_dim) {
    if (total_tokens <= 0 || max_seqlen_q <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0) return 0;
    if (max_seqlen_q > total_tokens || num_q_heads % num_kv_heads != 0 || head_dim > 256) return 0;
    const int g = num_q_heads / num_kv_heads;
    const int waves = lg::tree_slot_waves(max_seqlen_q, g, 4);  // (eight: half as many workgroups)
    return (size_t)2 * lg::kTreeWorkers * (size_t)waves * (size_t)lg::tree_wave_floats(head_dim) * sizeof(float);
}

#define LOGISMOS_TREE_PARAMS                                                                                           \
    lg::TreeParams p = {};                                                                                             \
    p.q = static_cast<const unsigned short*>(q);                                                                       \
    p.k_pool = static_cast<const uint8_t*>(k_pool);                                                                    \
    p.v_pool = static_cast<const uint8_t*>(v_pool);                                                                    \
    p.tables = block_tables;                                                                                           \
    p.cu = cu_seqlens_q;                                                                                               \
    p.ctx = context_lens;                                                                                              \
    p.mask = reinterpret_cast<const uint32_t*>(tree_mask);                                                             \
    p.out = static_cast<unsigned short*>(out);                                                                         \
    p.ws = static_cast<float*>(workspace);                                                                             \
    p.num_seqs = num_seqs;                                                                                             \
    p.total = total_tokens;                                                                                            \
    p.max_q = max_seqlen_q;                                                                                            \
    p.hkv = num_kv_heads;                                                                                              \
    p.block_size = block_size;                                                                                         \
    p.max_blocks = max_blocks_per_seq;                                                                                 \
    p.num_blocks = num_blocks;                                                                                         \
    p.words = mask_words > 0 && mask_words <= lg::kTreeMaskWords ? 2 * mask_words : 0;                                 \
    p.q_stride = q_stride;                                                                                             \
    p.out_stride = out_stride;

logismos_status_t logismos_launch_paged_attn_tree_fp16(
    const void* q, const void* k_pool, const void* v_pool, const int32_t* block_tables, const int32_t* cu_seqlens_q,
    const int32_t* context_lens, const uint64_t* tree_mask, void* out, void* workspace, int num_seqs, int total_tokens,
    int max_seqlen_q, int num_q_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks_per_seq,
    int num_blocks, int mask_words, int q_stride, int out_stride, float scale, logismos_stream_t stream) {
    LOGISMOS_TREE_PARAMS
    return lg::tree_attention(false, false, p, num_q_heads, head_dim, scale, stream);
}

#define LOGISMOS_PAGED_ATTN_TREE_E4M3(name, bf16)                                                                      \
    logismos_status_t logismos_launch_paged_attn_tree_e4m3_##name(                                                     \
        const void* q, const void* k_pool, const void* k_exp, const void* v_pool, const void* v_exp,                   \
        const int32_t* block_tables, const int32_t* cu_seqlens_q, const int32_t* context_lens,                         \
        const uint64_t* tree_mask, void* out, void* workspace, int num_seqs, int total_tokens, int max_seqlen_q,       \
        int num_q_heads, int num_kv_heads, int head_dim, int block_size, int max_blocks_per_seq, int num_blocks,       \
        int mask_words, int q_stride, int out_stride, float scale, logismos_stream_t stream) {                         \
        LOGISMOS_TREE_PARAMS                                                                                           \
        p.k_exp = static_cast<const uint8_t*>(k_exp);                                                                  \
        p.v_exp = static_cast<const uint8_t*>(v_exp);                                                                  \
        return lg::tree_attention(true, bf16, p, num_q_heads, head_dim, scale, stream);                                \
    }
LOGISMOS_PAGED_ATTN_TREE_E4M3(fp16, false)
LOGISMOS_PAGED_ATTN_TREE_E4M3(bf16, true)
#undef LOGISMOS_PAGED_ATTN_TREE_E4M3
#undef LOGISMOS_TREE_PARAMS

logismos_status_t logismos_tree_mask(const int32_t* parents, int tokens, int mask_words, uint64_t* mask) {
    const logismos_status_t bad = static_cast<logismos_status_t>(hipErrorInvalidValue);
    if (tokens == 0 && mask_words > 0 && mask_words <= lg::kTreeMaskWords) return 0;
    if (!parents || !mask || tokens <= 0 || mask_words <= 0 || mask_words > lg::kTreeMaskWords ||
        tokens > 64 * mask_words)
        return bad;
    for (int i = 0; i < tokens; ++i)
        if (parents[i] < -1 || parents[i] >= i) return bad;
    for (int i = 0; i < tokens; ++i)
        for (int w = 0; w < mask_words; ++w) {
            const uint64_t above = parents[i] >= 0 ? mask[(size_t)parents[i] * mask_words + w] : 0;
            mask[(size_t)i * mask_words + w] = above | (i / 64 == w ? 1ull << (i % 64) : 0);
        }
    return 0;
}

}  // extern "C"

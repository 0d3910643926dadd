// Attention calls that see the cache through a view - 8-bit codes with page scales, a sliding window, or both: their
// argument checks (none of which needs a device) and the choice between the tuned and the plain kernel.
#include <cmath>

#include "compute_internal.h"
#include "q8.cuh"

namespace gb200 {

namespace {

constexpr uint64_t kIntLimit = (1ull << 31) - 65536;  // positions and rows, with room for a tile more in int arithmetic

bool unaligned16(const void* a, const void* b) { return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) != 0; }

int check_heads(uint32_t num_heads, uint32_t num_kv_heads, uint32_t head_dim, const std::string& what) {
    if (num_heads == 0 || num_kv_heads == 0 || num_heads % num_kv_heads != 0 || num_heads > 65535)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": num_heads must be a multiple of num_kv_heads, at most 65535");
    if (head_dim == 0 || head_dim % 8 != 0 || head_dim > 256)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": head_dim must be a multiple of 8, at most 256");
    return GRANITE_CUDA_SUCCESS;
}

// (a masked score is -infinity and has to stay that when it is scaled)
int check_scale(float scale, const std::string& what) {
    if (!(scale > 0.f) || !std::isfinite(scale)) return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": scale must be positive and finite");
    return GRANITE_CUDA_SUCCESS;
}

int check_pool(uint32_t block_size, uint32_t num_blocks, uint32_t max_blocks, const std::string& what) {
    if (block_size == 0 || num_blocks == 0 || max_blocks == 0) return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": empty pool or table");
    if ((uint64_t)block_size * max_blocks >= kIntLimit || (uint64_t)block_size * num_blocks >= kIntLimit)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": the pool or a block table spans about 2^31 tokens or more");
    return GRANITE_CUDA_SUCCESS;
}

}  // namespace

int check_decode_view(const GraniteCudaPagedDecodeArgs& a, bool contiguous, uint32_t max_seq) {
    const std::string what = contiguous ? "decode window" : "paged decode";
    if (!a.q || !a.k_cache || !a.v_cache || !a.output || (!contiguous && !a.block_tables))
        return fail(GRANITE_CUDA_NULL_POINTER, what + ": null buffer");
    if (a.batch_size == 0) return GRANITE_CUDA_SUCCESS;
    if (int rc = check_heads(a.num_heads, a.num_kv_heads, a.head_dim, what)) return rc;
    if (int rc = check_scale(a.scale, what)) return rc;
    if (a.batch_size > 65535) return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": at most 65535 sequences per call");
    if (unaligned16(a.q, a.output) || unaligned16(a.k_cache, a.v_cache))
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": Q, the caches and the output must be 16-byte aligned");
    if (contiguous) {
        if (max_seq == 0 || max_seq >= kIntLimit) return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": max_seq must be positive and below 2^31");
        return GRANITE_CUDA_SUCCESS;
    }
    return check_pool(a.block_size, a.num_blocks, a.max_blocks_per_seq, what);
}

int check_prefill_view(const GraniteCudaAttentionArgs& a) {
    const std::string what = "prefill window";
    if (!a.q || !a.k || !a.v || !a.output) return fail(GRANITE_CUDA_NULL_POINTER, what + ": null buffer");
    if (int rc = check_heads(a.num_heads, a.num_kv_heads, a.head_dim, what)) return rc;
    if (int rc = check_scale(a.scale, what)) return rc;
    if (a.q_dtype > 1 || a.out_dtype > 1) return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": dtype must be 0 (fp32) or 1 (fp16)");
    if (unaligned16(a.q, a.output) || unaligned16(a.k, a.v))
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": Q, K, V and the output must be 16-byte aligned");
    const uint32_t max_seq = a.max_seq ? a.max_seq : a.seq_kv;
    if (a.seq_kv == 0 || a.seq_kv > max_seq) return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": seq_kv must be in [1, max_seq]");
    const uint64_t batch = a.batch_size ? a.batch_size : 1;
    if ((uint64_t)a.start_pos + a.seq_q >= kIntLimit || batch * a.seq_q >= kIntLimit || batch * a.num_kv_heads * max_seq >= kIntLimit)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": positions or batch * rows reach 2^31");
    return GRANITE_CUDA_SUCCESS;
}

int check_paged_prefill_view(const GraniteCudaPagedPrefillArgs& a) {
    const std::string what = "paged prefill";
    if (!a.q || !a.k_cache || !a.v_cache || !a.block_table || !a.output) return fail(GRANITE_CUDA_NULL_POINTER, what + ": null buffer");
    if (int rc = check_heads(a.num_heads, a.num_kv_heads, a.head_dim, what)) return rc;
    if (int rc = check_scale(a.scale, what)) return rc;
    if (a.q_dtype > 1 || a.out_dtype > 1) return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": dtype must be 0 (fp32) or 1 (fp16)");
    if (unaligned16(a.q, a.output) || unaligned16(a.k_cache, a.v_cache))
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": Q, the pools and the output must be 16-byte aligned");
    if (int rc = check_pool(a.block_size, a.num_blocks, a.max_blocks_per_seq, what)) return rc;
    if ((uint64_t)a.start_pos + a.seq_q > (uint64_t)a.max_blocks_per_seq * a.block_size)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, what + ": the chunk ends beyond the block table");
    return GRANITE_CUDA_SUCCESS;
}

int launch_decode_view(granite_cuda_compute* c, const GraniteCudaPagedDecodeArgs& a, bool contiguous, uint32_t max_seq, const CacheView& view) {
    if (a.batch_size == 0) return GRANITE_CUDA_SUCCESS;
    if (view.elem == kElemInt8) return launch_paged_decode_int8(c, a, view);
    if (view.elem == kElemE4M3) return launch_paged_decode_e4m3(c, a, view);
    return launch_paged_decode_window(c, a, contiguous, max_seq, view);
}

int launch_prefill_view(granite_cuda_compute* c, const GraniteCudaAttentionArgs& a, const CacheView& view) {
    if (a.seq_q == 0) return GRANITE_CUDA_SUCCESS;
    return launch_prefill(c, a, view);
}

int launch_paged_prefill_view(granite_cuda_compute* c, const GraniteCudaPagedPrefillArgs& a, const CacheView& view) {
    if (a.seq_q == 0) return GRANITE_CUDA_SUCCESS;
    return view.elem != kElemF16 ? launch_paged_prefill_q8(c, a, view) : launch_paged_prefill(c, a, view);
}

}  // namespace gb200

// RoPE fused with the write into the 8-bit paged cache.
//
// For a page that the call touches, for one KV head and for K (rotated) or V, with x the call's rows in the page:
//     need = max |x| / qmax        scale' = max(need, scale of the page's older rows; 0 when row 0 is new)
//     new rows: round(x / scale')  older rows: round(code * (scale / scale')), only when the scale grew
// The rotation and its roundings are those of the fp16 append (rope_append.cu): adjacent pairs, tables from the
// host, both products rounded separately.  Quotients are correctly rounded: a code then depends on nothing but the
// formula above, so the same inputs give the same bytes whatever the batch around them.
//
// One block of four warps per (sequence, touched page, KV head, K or V): the scale needs the whole page before the first
// code can be written, and four float4 per thread hold a page of one head (16 rows x 128) - every input is read once, a
// row is one 512-byte load and one 128-byte store.  (One warp per page, sixteen float4 per lane: 109 us for a 4 x 2043
// token chunk - the registers leave too few warps to cover the loads.)  The older rows are only touched when the scale grows.
// Query heads are rotated by further blocks of the same launch, four 16-byte pieces per thread.  Bound by HBM for chunks (Q is
// read and written in 32 bits: three quarters of the bytes), by the chain position -> table entry -> scale -> older
// rows for a decode step.
#include "compute_internal.h"
#include "ptx.cuh"
#include "q8.cuh"

namespace gb200 {

namespace {

constexpr int kAppendThreads = 128;
constexpr int kQueryPieces = 4;  // 16-byte pieces of Q per thread
constexpr int kQueryBlock = kAppendThreads * kQueryPieces;

struct Q8AppendParams {
    float* q;
    const float* k;
    const float* v;
    const float* cos_t;
    const float* sin_t;
    uint8_t* k_pool;
    uint8_t* v_pool;
    float* k_scales;
    float* v_scales;
    const int* tables;
    const int* positions;
    int batch, new_len, hq, hkv, head_dim, block_size, max_blocks, num_blocks, table_len, start_pos;
    int pages_per_seq;      // touched pages of a sequence at most
    long long page_blocks;  // blocks that write pages; the blocks behind them rotate Q
    int tokens_per_block, blocks_per_token;  // of the Q rotation; one of the two is 1
    int* status;
};

__device__ __forceinline__ float4 rotate_quad(float4 x, float2 c, float2 s) {
    float4 r;
    r.x = __fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(x.y, s.x));
    r.y = __fadd_rn(__fmul_rn(x.x, s.x), __fmul_rn(x.y, c.x));
    r.z = __fsub_rn(__fmul_rn(x.z, c.y), __fmul_rn(x.w, s.y));
    r.w = __fadd_rn(__fmul_rn(x.z, s.y), __fmul_rn(x.w, c.y));
    return r;
}
__device__ __forceinline__ float max_abs(float4 x) { return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))); }
// 0 while every value so far is finite, NaN from then on
__device__ __forceinline__ float poison(float z, float4 x) { return fmaf(x.w, 0.f, fmaf(x.z, 0.f, fmaf(x.y, 0.f, fmaf(x.x, 0.f, z)))); }
__device__ __forceinline__ float4 finite_part(float4 x) {
    auto one = [](float v) { return fabsf(v) < INFINITY ? v : 0.f; };
    return make_float4(one(x.x), one(x.y), one(x.z), one(x.w));
}
// x / scale, correctly rounded, from the correctly rounded reciprocal: the quotient estimate and one correction by its exact
// remainder (Markstein, IBM Journal of Research and Development 34, 1990).  A division per element was two thirds of
// the kernel's instructions.  The remainder is exact while its last bit is a number: that of q times that of scale, 2^-56 scale for the
// smallest q that rounds to a code (2^-10).  Below kTinyScale both are multiplied by a power of two first, which changes nothing else.
constexpr float kTinyScale = 0x1p-90f, kTinyFactor = 0x1p64f;
__device__ __forceinline__ float over(float x, float scale, float inv) {
    const float q = __fmul_rn(x, inv);
    return fmaf(fmaf(-q, scale, x), inv, q);
}
__device__ __forceinline__ float4 times(float4 x, float f) { return make_float4(x.x * f, x.y * f, x.z * f, x.w * f); }
__device__ __forceinline__ float4 over(float4 x, float scale, float inv) {
    return make_float4(over(x.x, scale, inv), over(x.y, scale, inv), over(x.z, scale, inv), over(x.w, scale, inv));
}

// kQuads: float4 pieces of a head row for head_dim 128 (32) and 64 (16) with 16-token pages, the rows then stay in
// registers; 0: any other shape, whose rows are read twice (the second time from the caches).
template <int kElem, int kQuads>
__global__ void __launch_bounds__(kAppendThreads) q8_append_kernel(const __grid_constant__ Q8AppendParams p) {
    const int tid = threadIdx.x;
    const int quads = kQuads ? kQuads : p.head_dim / 4;
    if (blockIdx.x >= p.page_blocks) {
        // ---- rotate Q in place
        const long long blk = blockIdx.x - p.page_blocks;
        const int n = p.hq * quads;  // pieces per token
        const long long token0 = p.tokens_per_block > 1 ? blk * p.tokens_per_block : blk / p.blocks_per_token;
        const long long tokens = (long long)p.batch * p.new_len;
        const int first = (p.tokens_per_block > 1 ? 0 : (int)(blk - token0 * p.blocks_per_token) * kQueryBlock) + threadIdx.x;
        const int end = p.tokens_per_block > 1 ? (int)min((long long)p.tokens_per_block, tokens - token0) * n : n;
        float4* row = reinterpret_cast<float4*>(p.q) + token0 * n;
        float4 x[kQueryPieces];
#pragma unroll
        for (int j = 0; j < kQueryPieces; j++)
            if (first + j * kAppendThreads < end) x[j] = row[first + j * kAppendThreads];
#pragma unroll
        for (int j = 0; j < kQueryPieces; j++) {
            const int i = first + j * kAppendThreads;
            if (i >= end) break;
            const long long token = token0 + (p.tokens_per_block > 1 ? i / n : 0);
            const int b = (int)(token / p.new_len), s = (int)(token - (long long)b * p.new_len);
            const long long pos = (long long)(p.positions ? p.positions[b] : p.start_pos) + s;
            if (pos < 0 || pos >= p.table_len) continue;  // reported by the page blocks
            const size_t trig = (size_t)pos * (p.head_dim / 2) + 2 * (i % quads);
            row[i] = rotate_quad(x[j], *reinterpret_cast<const float2*>(p.cos_t + trig), *reinterpret_cast<const float2*>(p.sin_t + trig));
        }
        return;
    }

    // ---- one page of one head: task = ((sequence, page), head, K or V)
    long long task = blockIdx.x;
    const bool is_v = task & 1;
    task >>= 1;
    const int h = (int)(task % p.hkv);
    task /= p.hkv;
    const int pi = (int)(task % p.pages_per_seq);
    const long long b = task / p.pages_per_seq;
    const int start = p.positions ? p.positions[b] : p.start_pos;
    const long long room = min((long long)p.table_len, (long long)p.max_blocks * p.block_size);
    if (pi == 0 && h == 0 && !is_v && tid == 0 && (start < 0 || (long long)start + p.new_len > room))
        atomicOr(p.status, kStatusBadSeqLen);
    const AppendRows rows = append_rows(start, p.new_len, room, p.block_size, pi);
    const int r0 = rows.r0, r1 = rows.r1;
    if (r0 >= r1) return;
    const long long page0 = rows.page * p.block_size;  // position of the page's row 0
    const int phys = p.tables[(size_t)b * p.max_blocks + rows.page];
    if (phys < 0 || phys >= p.num_blocks) {
        if (tid == 0) atomicOr(p.status, kStatusBadTable);
        return;
    }
    const float4* src = reinterpret_cast<const float4*>(is_v ? p.v : p.k);
    uint32_t* pool = reinterpret_cast<uint32_t*>(is_v ? p.v_pool : p.k_pool);
    float* scales = (is_v ? p.v_scales : p.k_scales) + (size_t)phys * p.hkv + h;
    const float before = r0 > 0 ? *scales : 0.f;

    float z = 0.f;
    bool dropped = false;  // a value is not finite: all are looked at one by one then
    auto fetch = [&](int i) {  // piece i of the page: row i / quads
        const int row = i / quads, u = i - row * quads;
        const long long s = page0 + row - start;  // which of the call's tokens
        float4 x = src[(((size_t)b * p.new_len + s) * p.hkv + h) * quads + u];
        if (!is_v) {
            const size_t trig = (size_t)(page0 + row) * (p.head_dim / 2) + 2 * u;
            x = rotate_quad(x, *reinterpret_cast<const float2*>(p.cos_t + trig), *reinterpret_cast<const float2*>(p.sin_t + trig));
        }
        z = poison(z, x);
        return dropped ? finite_part(x) : x;
    };
    auto word = [&](int i) {  // where the codes of piece i live
        const int row = i / quads, u = i - row * quads;
        return pool + (((size_t)phys * p.block_size + row) * p.hkv + h) * quads + u;
    };
    const int i0 = r0 * quads, i1 = r1 * quads;
    float amax = 0.f;
    constexpr int kIts = kQuads ? 16 * kQuads / kAppendThreads : 1;
    float4 held[kIts];
    if constexpr (kQuads > 0) {
        // the loads first, none behind a branch, so that they are in flight together
        const float4* row0 = src + (((size_t)b * p.new_len + (page0 - start)) * p.hkv + h) * quads;  // (not read where it is not the call's)
        float2 cs[kIts], sn[kIts];
#pragma unroll
        for (int it = 0; it < kIts; it++) {
            const int i = it * kAppendThreads + tid, row = i / quads, u = i - row * quads;
            held[it] = make_float4(0.f, 0.f, 0.f, 0.f);
            cs[it] = sn[it] = make_float2(0.f, 0.f);
            if (i >= i0 && i < i1) {
                held[it] = row0[(size_t)row * p.hkv * quads + u];
                if (!is_v) {
                    const size_t trig = (size_t)(page0 + row) * (p.head_dim / 2) + 2 * u;
                    cs[it] = *reinterpret_cast<const float2*>(p.cos_t + trig);
                    sn[it] = *reinterpret_cast<const float2*>(p.sin_t + trig);
                }
            }
        }
#pragma unroll
        for (int it = 0; it < kIts; it++) {
            if (!is_v) held[it] = rotate_quad(held[it], cs[it], sn[it]);
            z = poison(z, held[it]);
            amax = fmaxf(amax, max_abs(held[it]));
        }
    } else {
        for (int i = i0 + tid; i < i1; i += kAppendThreads) amax = fmaxf(amax, max_abs(fetch(i)));
    }
    dropped = __syncthreads_or(z != z);
    if (dropped) {
        if (tid == 0) atomicOr(p.status, kStatusNonFinite);
        amax = 0.f;
        if (kQuads) {
#pragma unroll
            for (int it = 0; it < kIts; it++) {
                held[it] = finite_part(held[it]);
                amax = fmaxf(amax, max_abs(held[it]));
            }
        } else {
            for (int i = i0 + tid; i < i1; i += kAppendThreads) amax = fmaxf(amax, max_abs(fetch(i)));
        }
    }
#pragma unroll
    for (int sh = 16; sh > 0; sh >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, sh));
    __shared__ float s_max[kAppendThreads / 32];
    if ((tid & 31) == 0) s_max[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; w++) amax = fmaxf(amax, s_max[w]);
    float need = __fdiv_rn(amax, q8_max<kElem>());
    if (need < 1.17549435e-38f) need = 0.f;  // below the normal range: stored as zeros
    const float scale = fmaxf(before, need);
    const float up = scale < kTinyScale ? kTinyFactor : 1.f, by = scale * up;
    const float inv = scale > 0.f ? __frcp_rn(by) : 0.f;  // (scale 0: every row is zero)

    if (scale > before && r0 > 0) {
        const float ratio = __fdiv_rn(before, scale);
        for (int i = tid; i < i0; i += kAppendThreads) {
            const float4 x = q8_decode4<kElem>(*word(i));
            *word(i) = q8_encode4<kElem>(make_float4(__fmul_rn(x.x, ratio), __fmul_rn(x.y, ratio), __fmul_rn(x.z, ratio), __fmul_rn(x.w, ratio)));
        }
    }
    if (kQuads) {
        if (up != 1.f) {
#pragma unroll
            for (int it = 0; it < kIts; it++) held[it] = times(held[it], up);
        }
#pragma unroll
        for (int it = 0; it < kIts; it++) {
            const int i = it * kAppendThreads + tid;
            if (i >= i0 && i < i1) *word(i) = scale > 0.f ? q8_encode4<kElem>(over(held[it], by, inv)) : 0u;
        }
    } else {
        for (int i = i0 + tid; i < i1; i += kAppendThreads) *word(i) = scale > 0.f ? q8_encode4<kElem>(over(times(fetch(i), up), by, inv)) : 0u;
    }
    if (tid == 0) *scales = scale;
}

}  // namespace

int check_q8_append(const GraniteCudaRopeAppendArgs& a, const GraniteCudaQ8Cache& x) {
    if (!a.k || !a.v || !a.cos_table || !a.sin_table || !a.k_cache || !a.v_cache || !a.block_tables || !x.k_scales || !x.v_scales)
        return fail(GRANITE_CUDA_NULL_POINTER, "rope_paged_kv_cache_append_q8: null buffer");
    if (x.cache_dtype > 1) return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: cache_dtype must be 0 (int8) or 1 (e4m3)");
    if (a.batch_size == 0 || a.new_len == 0) return GRANITE_CUDA_SUCCESS;
    if (a.head_dim == 0 || a.head_dim % 8 != 0 || a.head_dim > 256)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: head_dim must be a multiple of 8, at most 256");
    if (a.num_kv_heads == 0 || a.block_size == 0 || a.num_blocks == 0 || a.max_blocks_per_seq == 0 || (a.q && a.num_heads == 0))
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: empty shape");
    const uintptr_t align16 = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                              reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache);
    if (align16 & 15) return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: Q, K, V and the pools must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(a.cos_table) | reinterpret_cast<uintptr_t>(a.sin_table)) & 7)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: the RoPE tables must be 8-byte aligned");
    const uint64_t limit = 1ull << 31;
    if (a.batch_size >= limit || a.new_len >= limit || a.num_heads > 65535 || a.num_kv_heads > 65535 || a.block_size >= limit ||
        a.max_blocks_per_seq >= limit || a.num_blocks >= limit || a.table_len >= limit || a.start_pos >= limit)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: a size is out of range (65535 heads, 2^31 - 1 otherwise)");
    // the kernel counts the four-element pieces of a page's head in 32 bits, a block's stride beyond the last
    if ((uint64_t)a.block_size * (a.head_dim / 4) >= limit - 65536)
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: block_size * head_dim is out of range (below about 2^33)");
    return GRANITE_CUDA_SUCCESS;
}

int launch_q8_append(granite_cuda_compute* c, const GraniteCudaRopeAppendArgs& a, const GraniteCudaQ8Cache& x) {
    if (a.batch_size == 0 || a.new_len == 0) return GRANITE_CUDA_SUCCESS;
    Q8AppendParams p{};
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.cos_t = a.cos_table;
    p.sin_t = a.sin_table;
    p.k_pool = static_cast<uint8_t*>(a.k_cache);
    p.v_pool = static_cast<uint8_t*>(a.v_cache);
    p.k_scales = x.k_scales;
    p.v_scales = x.v_scales;
    p.tables = a.block_tables;
    p.positions = a.positions;
    p.batch = (int)a.batch_size;
    p.new_len = (int)a.new_len;
    p.hq = a.q ? (int)a.num_heads : 0;
    p.hkv = (int)a.num_kv_heads;
    p.head_dim = (int)a.head_dim;
    p.block_size = (int)a.block_size;
    p.max_blocks = (int)a.max_blocks_per_seq;
    p.num_blocks = (int)a.num_blocks;
    p.table_len = (int)a.table_len;
    p.start_pos = (int)a.start_pos;
    p.status = c->d_status;
    p.pages_per_seq = (int)(((uint64_t)a.new_len + a.block_size - 2) / a.block_size) + 1;
    if ((uint64_t)a.batch_size * p.pages_per_seq >= (1ull << 31))
        return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: too many tokens for one call");
    p.page_blocks = (long long)a.batch_size * p.pages_per_seq * a.num_kv_heads * 2;
    const uint64_t pieces = (uint64_t)p.hq * (a.head_dim / 4), tokens = (uint64_t)a.batch_size * a.new_len;
    p.tokens_per_block = pieces > 0 && pieces < kQueryBlock ? (int)(kQueryBlock / pieces) : 1;
    p.blocks_per_token = (int)((pieces + kQueryBlock - 1) / kQueryBlock);
    const uint64_t q_blocks = pieces == 0 ? 0 : p.tokens_per_block > 1 ? (tokens + p.tokens_per_block - 1) / p.tokens_per_block : tokens * p.blocks_per_token;
    const uint64_t grid = (uint64_t)p.page_blocks + q_blocks;
    if (grid >= (1ull << 31)) return fail(GRANITE_CUDA_INVALID_ARGUMENT, "rope_paged_kv_cache_append_q8: too many tokens for one call");
    const int quads = a.block_size == 16 ? (a.head_dim == 128 ? 32 : a.head_dim == 64 ? 16 : 0) : 0;
    const bool e4m3 = x.cache_dtype == GRANITE_CUDA_CACHE_E4M3;
    auto kern = quads == 32   ? (e4m3 ? q8_append_kernel<kElemE4M3, 32> : q8_append_kernel<kElemInt8, 32>)
                : quads == 16 ? (e4m3 ? q8_append_kernel<kElemE4M3, 16> : q8_append_kernel<kElemInt8, 16>)
                              : (e4m3 ? q8_append_kernel<kElemE4M3, 0> : q8_append_kernel<kElemInt8, 0>);
    LaunchScope t(c, "rope_paged_kv_append_q8");
    kern<<<(unsigned)grid, kAppendThreads, 0, c->stream>>>(p);
    GB_CUDA_TRY(cudaGetLastError());
    return GRANITE_CUDA_SUCCESS;
}

}  // namespace gb200

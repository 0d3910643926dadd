// Index arithmetic of the calls that see the cache through a view, for host and device alike and without CUDA types: which keys a
// window leaves, and which key tiles a query block walks.
#pragma once
#include <stddef.h>

#ifdef __CUDACC__
#define GB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define GB_HOST_DEVICE inline
#endif

namespace gb200 {

// What a sliding window leaves of a sequence whose query sits at position `pos`: keys [0, sinks_end) and
// [lo, pos], sinks_end <= lo.  window 0: no window (sinks_end = lo = 0).
struct WindowSpan {
    int sinks_end, lo;
};
GB_HOST_DEVICE WindowSpan window_span(int pos, int window, int sinks) {
    WindowSpan s;
    s.lo = window > 0 && pos >= window ? pos - window + 1 : 0;
    s.sinks_end = sinks < s.lo ? sinks : s.lo;
    return s;
}

constexpr int kTileRows = 128;  // query rows of a block, keys of a tile

// The queries of a prefill call and what they may see: row i sits at position start_pos + i, keys are [0, seq_kv).
struct PrefillSpan {
    int seq_q, seq_kv, start_pos;
    int window, sinks;  // window 0: none
};
// The steps of the query block that starts at row q0: tiles [0, n_sink) of the sinks, then from w0, the window of its first row, to its
// diagonal.
struct WindowSteps {
    int n, n_sink, w0, lo;
};
GB_HOST_DEVICE WindowSteps window_steps(const PrefillSpan& p, int q0) {
    WindowSteps w;
    const int rows = p.seq_q - q0 < kTileRows ? p.seq_q - q0 : kTileRows, last = p.start_pos + q0 + rows;
    const int tiles = ((p.seq_kv < last ? p.seq_kv : last) + kTileRows - 1) / kTileRows;  // up to the last visible key
    w.lo = window_span(p.start_pos + q0, p.window, p.sinks).lo;
    w.w0 = w.lo / kTileRows < tiles ? w.lo / kTileRows : tiles;
    const int sink_tiles = ((p.sinks < w.lo ? p.sinks : w.lo) + kTileRows - 1) / kTileRows;
    w.n_sink = sink_tiles < w.w0 ? sink_tiles : w.w0;
    w.n = w.n_sink + tiles - w.w0;
    if (w.n < 1) {  // a block that sees nothing still runs one, masked, step
        w.n = 1;
        w.w0 = 0;
    }
    return w;
}
// Steps [chunk_begin(n, c), chunk_begin(n, c + 1)) of n are chunk c's; there are more chunks than steps in short blocks.
GB_HOST_DEVICE int chunk_begin(int n, int n_chunks, int c) { return n * c / n_chunks; }

// ---- how a prefill's key tiles are cut into chunks (host)
// A chunk's tiles run through one truncating tensor-core accumulator, 1.3e-9 of the result per key.  An fp32 output wants no more than
// 22 of them (3.6e-6): with 8, 4001 rows at 4099 under a window of 2047 are 1.4e-6 off instead of 2.9e-6 and take 369 us instead of
// 275, with 4 1.0e-6 and 462 us.  An fp16 output wants no more than 128, a twentieth of its own half step.
constexpr int kMaxChunks = 32;                       // the merge has one lane per chunk
constexpr int kMaxTilesF32 = 22, kMaxTilesF16 = 128;
constexpr size_t kMaxPartialBytes = (size_t)1 << 30;  // of a launch's partials: scratch that the object keeps
constexpr int kChunkChoices[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, kMaxChunks};

struct ChunkProblem {
    PrefillSpan span;
    int batch, num_heads, head_dim, sm_count;
    bool out_fp16;
};
inline int max_tiles(const ChunkProblem& c) { return c.out_fp16 ? kMaxTilesF16 : kMaxTilesF32; }
inline int longest_steps(const PrefillSpan& s) {
    const int blocks = (s.seq_q + kTileRows - 1) / kTileRows;
    int longest = 1;
    auto look = [&](int b) {
        const int n = window_steps(s, b * kTileRows).n;
        if (n > longest) longest = n;
    };
    for (int b = 0; b < blocks; b += 1 + blocks / 64) look(b);
    look(blocks - 1);
    return longest;
}
// Bytes of partials per chunk for one query row of every head: fp32 outputs, maximum and sum.
inline size_t row_partial_bytes(const ChunkProblem& c) { return (size_t)c.batch * c.num_heads * (c.head_dim * 4 + 8); }
// The fewest chunks whose tiles an accumulator takes; kMaxChunks where none do (an fp32 output over more than 90112 keys).
inline int wanted_chunks(const ChunkProblem& c) {
    const int longest = longest_steps(c.span);
    for (int n : kChunkChoices)
        if ((longest + n - 1) / n <= max_tiles(c)) return n;
    return kMaxChunks;
}
// Query rows that one launch takes so that the chunks it wants fit the limit on partials: all, or a multiple of a block's.
inline int rows_per_launch(const ChunkProblem& c) {
    const int n = wanted_chunks(c);
    if (n == 1 || row_partial_bytes(c) * c.span.seq_q * n <= kMaxPartialBytes) return c.span.seq_q;
    const size_t blocks = kMaxPartialBytes / (row_partial_bytes(c) * n * kTileRows);
    return blocks < 1 ? kTileRows : (int)(blocks * kTileRows) < c.span.seq_q ? (int)(blocks * kTileRows) : c.span.seq_q;
}
// How many chunks a launch's tiles are cut into: of the counts that an accumulator takes and that fit the limit, the one with the
// shortest estimate - the longest queue of any SM (items come in rounds of one per SM, a chunk costs its steps and about one and a
// half more to start and drain, 1.35 us a step) plus the merge's launch and traffic; if none is taken, the most that fit.
inline int plan_chunks(const ChunkProblem& c) {
    const long long blocks = (c.span.seq_q + kTileRows - 1) / kTileRows, items = blocks * c.batch * c.num_heads;
    const int longest = longest_steps(c.span), wanted = wanted_chunks(c);
    double best = 0;
    int chosen = 1;
    bool taken = false;
    for (int n : kChunkChoices) {
        if (n > longest || items * n >= (1ll << 31)) break;
        if (n > 1 && row_partial_bytes(c) * c.span.seq_q * n > kMaxPartialBytes) break;
        if (n < wanted && n < longest) {
            chosen = n;  // for the accumulator's sake the most so far
            continue;
        }
        const int steps = (longest + n - 1) / n;
        const double rounds = (double)((items * n + c.sm_count - 1) / c.sm_count);
        const double us = rounds * (steps + 1.5) * 1.35 + (n > 1 ? 3.0 + (double)c.batch * c.num_heads * c.span.seq_q * n * c.head_dim * 8 / 5e6 : 0.0);
        if (!taken || us < best) {
            best = us;
            chosen = n;
            taken = true;
        }
    }
    return chosen;
}

// The rows [r0, r1) of logical page `page` that an append of new_len tokens from position `start` writes, page the touched-th from the first
// page with a place for one of them: none (r0 >= r1) where `start` leaves no token in [0, room).  Any start may come, so everything is in
// 64 bits and brought into the page before it is narrowed.
struct AppendRows {
    long long page;
    int r0, r1;
};
GB_HOST_DEVICE AppendRows append_rows(long long start, long long new_len, long long room, int block_size, int touched) {
    const long long lo = start > 0 ? start : 0, hi = start + new_len < room ? start + new_len : room;
    AppendRows a;
    a.page = lo / block_size + touched;
    const long long page0 = a.page * block_size;
    const long long r0 = lo - page0, r1 = hi - page0;
    a.r0 = (int)(r0 < 0 ? 0 : r0 < block_size ? r0 : block_size);
    a.r1 = (int)(r1 < 0 ? 0 : r1 < block_size ? r1 : block_size);
    return a;
}

}  // namespace gb200

// Index arithmetic of the calls that see the cache through a view, for host and device alike and without CUDA types: which keys a
// window leaves, and which key tiles a query block walks.
#pragma once

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

// Test drivers of csrc/view_plan.h, which the kernels and their launchers share; built with the host compiler alone.
#include "../../granite_b200/csrc/view_plan.h"

using namespace gb200;

extern "C" {

void view_window_span(int pos, int window, int sinks, int* out) {
    const WindowSpan s = window_span(pos, window, sinks);
    out[0] = s.sinks_end;
    out[1] = s.lo;
}

void view_window_steps(int seq_q, int seq_kv, int start_pos, int window, int sinks, int q0, int* out) {
    const WindowSteps w = window_steps(PrefillSpan{seq_q, seq_kv, start_pos, window, sinks}, q0);
    out[0] = w.n;
    out[1] = w.n_sink;
    out[2] = w.w0;
    out[3] = w.lo;
}

void view_append_rows(long long start, long long new_len, long long room, int block_size, int touched, long long* out) {
    const AppendRows a = append_rows(start, new_len, room, block_size, touched);
    out[0] = a.page;
    out[1] = a.r0;
    out[2] = a.r1;
}

// shape: seq_q, seq_kv, start_pos, window, sinks, batch, num_heads, head_dim, sm_count, out_fp16
// out: wanted chunks and rows per launch of the call; for its last launch of that many rows: longest item, chunks, bytes of partials
void view_chunk_plan(const int* s, long long* out) {
    ChunkProblem c{{s[0], s[1], s[2], s[3], s[4]}, s[5], s[6], s[7], s[8], s[9] != 0};
    out[0] = wanted_chunks(c);
    out[1] = rows_per_launch(c);
    c.span.start_pos += c.span.seq_q - (int)out[1];
    c.span.seq_q = (int)out[1];
    out[2] = longest_steps(c.span);
    out[3] = plan_chunks(c);
    out[4] = out[3] == 1 ? 0 : (long long)(row_partial_bytes(c) * c.span.seq_q * out[3]);
}

int view_chunk_begin(int n, int n_chunks, int c) { return chunk_begin(n, n_chunks, c); }
}

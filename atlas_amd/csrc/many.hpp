// many.hpp -- launch interfaces of the operators for many continuations decoded
// together (internal): attention over shared prefixes (prefix.hip), beam search's
// selection and reordering (beam.hip), low-rank adapters (lora.hip).
#pragma once
#include <algorithm>

#include "common.hpp"

namespace atlas {

// Rows in memory: n of w bytes each, ld bytes apart (ld >= w where there are several).
struct ByteRows {
    uintptr_t p;
    long n, w, ld;
    ByteRows(const void* at, long n_, long w_, long ld_) : p((uintptr_t)at), n(n_), w(w_), ld(ld_) {}
    ByteRows(const void* at, long bytes) : ByteRows(at, 1, bytes, bytes) {}
    uintptr_t end() const { return p + (uintptr_t)(n - 1) * ld + w; }
};

// No byte of a's rows is one of b's.  (Rows of one may lie between the other's.)
inline bool rows_apart(const ByteRows& a, const ByteRows& b) {
    if (a.n <= 0 || a.w <= 0 || b.n <= 0 || b.w <= 0 || a.end() <= b.p || b.end() <= a.p) return true;
    for (long i = 0; i < a.n; ++i) {
        const uintptr_t at = a.p + (uintptr_t)i * a.ld, end = at + a.w;
        if (end <= b.p) continue;
        // of b's rows that begin before this one ends, the last ends last
        const long j = std::min((long)((end - 1 - b.p) / b.ld), b.n - 1);
        if (b.p + (uintptr_t)j * b.ld + b.w > at) return false;
    }
    return true;
}

// Scratch of a launch: the caller's, or (p null) the calling thread's.
struct Workspace {
    void* p = nullptr;
    size_t bytes = 0;
};

int prefix_attention_launch(const atlas_slot_cache& c, const atlas_prefix_batch& b, const float* q, long ld_q, int n_heads,
                            float scale, int window, float* out, long ld_out, const Workspace& ws, hipStream_t st);
// what a launch of this shape takes at most
size_t prefix_attention_workspace(const atlas_slot_cache& c, const atlas_prefix_batch& b, int n_heads, int window);

int beam_select_launch(const float* logits, long ld, int vocab, const double* scores, int n_groups, int width, int n_out,
                       uint32_t* tokens, int* parents, double* out_scores, const Workspace& ws, hipStream_t st);
size_t beam_select_workspace(int vocab, int n_groups, int width, int n_out);
int beam_reorder_launch(void* const* dst, const void* const* src, int n_states, long row_bytes, long row_stride,
                        const int* parents, int n_groups, int width, hipStream_t st);

int lora_add_launch(const atlas_lora& l, const int* adapters, const float* x, long ld_x, const float* base, long ld_base,
                    float* y, long ld_y, int n, hipStream_t st);

}  // namespace atlas

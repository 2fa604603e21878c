// many.hpp -- launch interfaces of the operators for many continuations decoded
// together (internal): attention over shared prefixes (prefix.hip), beam search's
// selection and reordering (beam.hip), low-rank adapters (lora.hip).
#pragma once
#include "common.hpp"

namespace atlas {

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

// batch_kernels.h -- the batch's kernel interface (internal).
#pragma once

#include <hip/hip_runtime.h>

#include "batch_plan.h"

namespace wick {

struct BatchArgs {
    const float *q;  // [total][heads * D] packed (may be att)
    float *att;
    // [kv_heads][prefix_capacity][D] and [sequences][kv_heads][capacity][D] of the layer,
    // f32 or bf16
    const void *pk, *pv, *k, *v;
    const BatchHeader *head;  // followed by tokens[max_tokens], then items
    const BatchToken *tokens;
    const BatchItem *items;
    float *po, *pm, *pl;  // states: [kv_heads][state_rows] x D, 1, 1
    long long state_rows;
    int prefix_capacity, capacity, group, kv_heads;
    unsigned inv_group, inv_kv_heads, inv_heads;  // batch_inverse of group, kv_heads and their product
    int shape, total;  // of the plan at the call
    int launched;      // items that the call has workgroups for
    int max_states;    // most states of a row in it
    float scale;       // log2(e) / sqrt(D)
};

// For the kernels' divisions by d >= 1.
inline unsigned batch_inverse(int d) {
    return d == 1 ? 0xffffffffu : (unsigned)(((1ull << 32) + d - 1) / d);
}

// The planned tokens' attention: `grid` workgroups over the items of every kv head.
hipError_t launch_batch_attend(int head_dim, int bf16, const BatchArgs &a, int grid, hipStream_t s);
// The split rows' states joined into att: `merges` joined tokens at the call.
hipError_t launch_batch_merge(int head_dim, const BatchArgs &a, int merges, hipStream_t s);

struct BatchAppendArgs {
    const float *ksrc, *vsrc;  // [total][kv_heads * D]
    void *k, *v;               // [sequences][kv_heads][capacity][D] of the layer
    const BatchHeader *head;   // null: rows go to positions start.. of sequence 0
    const BatchToken *tokens;
    int capacity, kv_heads, total, shape, start;
};
hipError_t launch_batch_append(int head_dim, int bf16, const BatchAppendArgs &a, hipStream_t s);

// src [kv_heads][src_capacity][D] f32, positions 0..len, to dst [kv_heads][dst_capacity][D].
hipError_t launch_batch_load(int head_dim, int bf16, const float *src, int src_capacity, void *dst, int dst_capacity,
                             int kv_heads, int len, hipStream_t s);

// dst [n][kv_heads * D] f32 from positions pos0.. of src [kv_heads][capacity][D].
hipError_t launch_batch_read(int head_dim, int bf16, const void *src, int capacity, int kv_heads, int pos0, int n,
                             float *dst, hipStream_t s);

}  // namespace wick

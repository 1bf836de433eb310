/*
 * wick_hip_batch.h -- several sequences at once over one shared prefix, on the GPU.
 *
 * wick serves one sequence per Session (src/engine.rs:101-139) and
 * keeps a prompt's positions when the next prompt begins with them (:127-132).  A
 * batch is that idea for many sequences at a time: one prefix (a system prompt, a
 * document) that all of them continue, its keys and values held and read once for
 * all, and behind it every sequence's own positions.  Without a prefix
 * (prefix 0) it is a batch of unrelated sequences.
 *
 * A step goes: wick_hip_batch_plan says which positions every sequence brings (whole
 * prompts of different lengths, single tokens, or any mix); then, per layer,
 * wick_hip_batch_append_device writes the new keys and values into the caches and
 * wick_hip_batch_attention_device attends.  The tokens of a step are packed: the rows of
 * sequence 0's tokens, then those of sequence 1, with no gaps.
 *
 * Token i of sequence s, at its position start[s] + i behind the prefix, attends as
 * Model::attention (src/model.rs:518-553) does to a context of the
 * prefix followed by the sequence's positions 0..=start[s]+i:
 *   att = softmax(q . k / sqrt(head_dim)) v.
 * q and att are f32.  The caches hold f32 (WICK_HIP_BATCH_F32) or bfloat16
 * (WICK_HIP_BATCH_BF16: keys and values are rounded to nearest when they are written,
 * half the memory and half the bytes of a step); products of either are exact to f32
 * rounding (of values of 2^-108 and above), and every sum is f32.  Scores times log2(e) that
 * leave f32's range count as infinities.  Positions that a token does not see never reach
 * its result, whatever they hold (infinities and NaN included).
 *
 * Return codes, wick_hip_last_error() and the rules on handles as in wick_hip.h: calls on
 * one handle are serialised by the caller, and work queued for one handle on several
 * streams must not overlap (its plan and its partial results are one each).
 */
#ifndef WICK_HIP_BATCH_H
#define WICK_HIP_BATCH_H

#include "wick_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define WICK_HIP_BATCH_F32 0
#define WICK_HIP_BATCH_BF16 1

typedef struct wick_hip_batch wick_hip_batch;

typedef struct wick_hip_batch_config {
    int layers;
    int heads;           /* query heads, a multiple of kv_heads */
    int kv_heads;
    int head_dim;        /* 16, 32, 64 or 128 */
    int sequences;       /* sequences of the batch */
    int capacity;        /* own positions of each sequence */
    int prefix_capacity; /* positions of the shared prefix (0: none) */
    int max_tokens;      /* most tokens of one plan, all sequences together */
    int type;            /* WICK_HIP_BATCH_F32 or WICK_HIP_BATCH_BF16 */
} wick_hip_batch_config;

/* The caches (zero-filled) and everything that later calls need, on the current HIP
 * device: no later call but the host-array ones allocates. */
int wick_hip_batch_create(const wick_hip_batch_config *cfg, wick_hip_batch **out);
void wick_hip_batch_destroy(wick_hip_batch *b);

/* Positions 0..len of every layer of `kv` (a prompt computed once, through the model
 * or by hand) become the prefix's positions 0..len.  kv has the batch's layers, kv_heads
 * and head_dim and was made on the same device.  Waits for the work queued on kv's
 * stream.  Synchronous. */
int wick_hip_batch_load_prefix(wick_hip_batch *b, const wick_hip_kv *kv, int len);

/* The prefix's positions start..start+t of `layer` from device arrays
 * [t][kv_heads*head_dim], 16-byte aligned.  Asynchronous on the handle's stream. */
int wick_hip_batch_write_prefix_device(wick_hip_batch *b, int layer, int start, int t, const float *k_dev,
                                       const float *v_dev);

/* The step that the following append and attention calls, of any layer, belong to:
 * sequence s brings t[s] tokens (0: none) at its own positions start[s]..., behind the
 * first `prefix` positions of the prefix.  start and t are host arrays [sequences],
 * read before the call returns.  Refused while the handle's stream is captured. */
int wick_hip_batch_plan(wick_hip_batch *b, const int *start, const int *t, int prefix);

/* For callers that capture append and attention calls into a graph: the number of the
 * plan's launch shape.  Graphs captured under a plan replay under any later plan of the
 * same number (single tokens whose positions move on, for example), with that plan's
 * positions, and within rounding of direct calls' results; the caller orders a replay on
 * another stream with the handle's.  Plans with the same t have the same number while it is
 * among the last 32 that were planned.  Replayed under a plan of another number graphs write
 * NaN to every captured row of att, and append nothing. */
int wick_hip_batch_shape(const wick_hip_batch *b);

/* k and v of the planned tokens, device arrays [tokens][kv_heads*head_dim], 16-byte
 * aligned, into the sequences' caches.  Asynchronous on the handle's stream. */
int wick_hip_batch_append_device(wick_hip_batch *b, int layer, const float *k_dev, const float *v_dev);

/* Attention of the planned tokens: q and att are device arrays [tokens][heads*head_dim],
 * 16-byte aligned; att may be q.  The planned positions must be in the caches.
 * Asynchronous on the handle's stream. */
int wick_hip_batch_attention_device(wick_hip_batch *b, int layer, const float *q_dev, float *att_dev);

/* The same two on host arrays.  Synchronous; they keep staging memory. */
int wick_hip_batch_append(wick_hip_batch *b, int layer, const float *k, const float *v);
int wick_hip_batch_attention(wick_hip_batch *b, int layer, const float *q, float *att);

/* Positions pos0..pos0+n of `layer` of sequence `seq` (-1: the prefix) as host arrays
 * [n][kv_heads*head_dim] (either may be NULL).  Synchronous. */
int wick_hip_batch_read(wick_hip_batch *b, int layer, int seq, int pos0, int n, float *k, float *v);

/* Launch on `stream` (a hipStream_t; NULL: the handle's own stream).  Work already
 * queued by the handle comes before what follows on the new stream, unless one of the
 * two is being captured: then the caller orders them. */
int wick_hip_batch_set_stream(wick_hip_batch *b, void *stream);

/* Wait for all work queued on the handle's stream. */
int wick_hip_batch_synchronize(wick_hip_batch *b);

/* Bytes of device and pinned host memory the handle holds beyond its caches. */
long long wick_hip_batch_scratch_bytes(const wick_hip_batch *b);

#ifdef __cplusplus
}
#endif

#endif /* WICK_HIP_BATCH_H */

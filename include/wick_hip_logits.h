/*
 * wick_hip_logits.h -- penalties, biases and grammar masks on a batch's logits, on the GPU.
 *
 * wick's sampler has a repetition penalty for one sequence
 * (src/sampler.rs:75-83).  This is that step for a batch, each row with
 * its own settings, and what serving programs put next to it: presence and frequency
 * penalties, biases on single ids, and grammars that allow a part of the vocabulary.  The
 * rows that come out go to wick_hip_sampler_sample_device or any other draw.
 *
 * Row r's logit x of id i becomes, in f32 and in this order:
 *   1. repetition, if i is among the row's tokens:  x > 0 ? x / p : x * p
 *      (the sampler's arithmetic; a p of 1 leaves x as it is)
 *   2. with c the times i is among the tokens behind the row's prompt, if c > 0:
 *      x - (frequency * c + presence)
 *   3. x + bias, if the row has a bias for i (an id given twice: the later one holds)
 *   4. minus infinity, if the row's grammar does not allow i
 * A row whose grammar allows nothing is all minus infinity.  Ids of vocab and above, among tokens
 * or biases, are passed over, as the sampler does.
 *
 * Return codes and wick_hip_last_error() as in wick_hip.h.
 */
#ifndef WICK_HIP_LOGITS_H
#define WICK_HIP_LOGITS_H

#include <stdint.h>

#include "wick_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Device arrays; a NULL array leaves its rule out. */
typedef struct wick_hip_logit_rules {
    const float *repetition;  /* [rows] */
    const float *presence;    /* [rows] */
    const float *frequency;   /* [rows] */
    const uint32_t *tokens;   /* [rows][tokens_stride]: prompt and generated ids, in order */
    const int *n_tokens;      /* [rows]: how many of them there are (with tokens: not NULL) */
    const int *n_prompt;      /* [rows]: the first n_prompt are the prompt's (NULL: none are) */
    int tokens_stride;        /* n_tokens past it counts as tokens_stride, below 0 as 0 */
    const int *bias_start;    /* [rows + 1]: row r has the entries bias_start[r]..bias_start[r+1] */
    const uint32_t *bias_ids; /* [n_bias] */
    const float *bias;        /* [n_bias] */
    int n_bias;               /* bias_start past it counts as n_bias, below 0 as 0 */
    const uint32_t *mask;     /* [masks][(vocab + 31) / 32]: bit i % 32 of word i / 32 allows id i */
    const int *mask_row;      /* [rows]: the row's mask, -1 (or any not in 0..masks) for none; NULL: mask r */
    int masks;
} wick_hip_logit_rules;

/* logits [rows][stride] to out [rows][out_stride], f32, the first vocab of each row (what is
 * behind them is neither read nor written); out may be logits (then with its stride), and may
 * not overlap it otherwise.  Asynchronous on `stream` (a hipStream_t; NULL: the default stream)
 * of the current device; allocates nothing. */
int wick_hip_logits_adjust_device(const wick_hip_logit_rules *rules, const float *logits, int rows, int vocab,
                                  int stride, float *out, int out_stride, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* WICK_HIP_LOGITS_H */

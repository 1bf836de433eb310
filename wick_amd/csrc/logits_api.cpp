// logits_api.cpp -- the C ABI of include/wick_hip_logits.h.
#include "wick_hip_logits.h"

#include <hip/hip_runtime.h>

#include <climits>

#include "attn_kernels.h"
#include "logits_kernels.h"

extern "C" int wick_hip_logits_adjust_device(const wick_hip_logit_rules *rules, const float *logits, int rows, int vocab,
                                             int stride, float *out, int out_stride, void *stream) {
    using wick::set_error;
    if (!rules || !logits || !out) return set_error(WICK_HIP_EINVAL, "null argument");
    const wick_hip_logit_rules &r = *rules;
    if (rows < 0 || vocab < 1) return set_error(WICK_HIP_EINVAL, "rows must be >= 0 and vocab >= 1 (got %d, %d)", rows, vocab);
    if (vocab > (1 << 30)) return set_error(WICK_HIP_EINVAL, "vocab must be at most 2^30 (got %d)", vocab);
    if (stride < vocab || out_stride < vocab)
        return set_error(WICK_HIP_EINVAL, "strides %d and %d must be at least vocab %d", stride, out_stride, vocab);
    if (r.tokens && !r.n_tokens) return set_error(WICK_HIP_EINVAL, "tokens without n_tokens");
    if (r.tokens_stride < 0) return set_error(WICK_HIP_EINVAL, "tokens_stride must be >= 0 (got %d)", r.tokens_stride);
    if (r.n_bias < 0) return set_error(WICK_HIP_EINVAL, "n_bias must be >= 0 (got %d)", r.n_bias);
    if (r.bias && (!r.bias_start || !r.bias_ids))
        return set_error(WICK_HIP_EINVAL, "bias without bias_start or bias_ids");
    if (r.mask && (r.masks < 1 || (!r.mask_row && r.masks < rows)))
        return set_error(WICK_HIP_EINVAL, "%d masks for %d rows", r.masks, rows);
    for (const void *p : {(const void *)logits, (const void *)out, (const void *)r.repetition, (const void *)r.presence,
                          (const void *)r.frequency, (const void *)r.tokens, (const void *)r.n_tokens,
                          (const void *)r.n_prompt, (const void *)r.bias_start, (const void *)r.bias_ids,
                          (const void *)r.bias, (const void *)r.mask, (const void *)r.mask_row})
        if (reinterpret_cast<uintptr_t>(p) & 3u) return set_error(WICK_HIP_EINVAL, "an array is not 4-byte aligned");
    if (rows == 0) return WICK_HIP_OK;
    // in place, or apart (in memory, or with every row of one between two of the other): a workgroup reads its
    // own ids only
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(logits), y0 = reinterpret_cast<uintptr_t>(out);
    const uintptr_t x1 = x0 + ((size_t)(rows - 1) * stride + vocab) * 4, y1 = y0 + ((size_t)(rows - 1) * out_stride + vocab) * 4;
    const size_t at = (y0 > x0 ? y0 - x0 : x0 - y0) / 4 % stride;  // of a row behind the other's before it
    const bool between = stride == out_stride && at >= (size_t)vocab && at <= (size_t)(stride - vocab);
    if (x0 < y1 && y0 < x1 && !between && !(x0 == y0 && (stride == out_stride || rows == 1)))
        return set_error(WICK_HIP_EINVAL, "out overlaps logits");
    wick::LogitArgs a{};
    a.r = r;
    a.x = logits;
    a.out = out;
    a.rows = rows;
    a.vocab = vocab;
    a.stride = stride;
    a.out_stride = out_stride;
    const int slab = wick::logit_slab(rows, vocab);
    a.slabs = (int)(((long long)vocab + slab - 1) / slab);
    if ((long long)rows * a.slabs > INT_MAX / 256)
        return set_error(WICK_HIP_EINVAL, "%d rows of %d logits are too many for one call", rows, vocab);
    int device;
    if (hipGetDevice(&device) != hipSuccess) return set_error(WICK_HIP_EDEVICE, "no HIP device");
    const hipError_t e = wick::launch_logits(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return set_error(WICK_HIP_EHIP, "logits kernel launch: %s", hipGetErrorString(e));
    return WICK_HIP_OK;
}

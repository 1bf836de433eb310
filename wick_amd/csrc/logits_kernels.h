// logits_kernels.h -- the logit rules' kernel interface (internal).
#pragma once

#include <hip/hip_runtime.h>

#include "wick_hip_logits.h"

namespace wick {

struct LogitArgs {
    wick_hip_logit_rules r;
    const float *x;
    float *out;  // may be x
    int rows, vocab, stride, out_stride;
    int slabs;  // workgroups of a row
};

// Ids of a workgroup for this many rows and ids (a multiple of 32).
int logit_slab(int rows, int vocab);
hipError_t launch_logits(const LogitArgs &a, hipStream_t s);

}  // namespace wick

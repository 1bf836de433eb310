// logits.hip -- the rules of include/wick_hip_logits.h in one pass over the logits.
//
// A workgroup has one row's ids [s0, s0 + SLAB).  It requests its logits and mask words,
// counts the row's tokens that fall into its slab in LDS (integer adds: any order gives
// the same counts) and applies the penalties, notes each id's last bias there and adds
// them, then writes its part of the row.  A row's tokens are read once per slab, from the L2.
//
// Bound: 8 bytes a logit and a mask bit, and the dependent reads and barriers of a workgroup (n_tokens, tokens,
// the row's settings, biases): 64 rows of 128256 with 1500 tokens each 14.2 us, where a copy of as many
// bytes, which the last-level cache holds like these, takes 10.1; one row of 49152 is the launch (3 us on the GPU).
// One LDS word an id, used for the counts and then for the biases: with a word for each the 64 rows took 18.1.
#include <hip/hip_runtime.h>

#include "logits_kernels.h"

namespace wick {
namespace {

constexpr int kT = 256;
constexpr uint32_t kSeen = 0x80000000u;

// rows of any alignment: 4 values, aligned as one
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(4)));

template <int SLAB>
__global__ __launch_bounds__(kT) void logits_kernel(LogitArgs a) {
#pragma clang fp contract(off)
    constexpr int U = SLAB / (4 * kT);  // passes of 4 ids a thread
    // first times among the generated tokens, and kSeen; then 1 + the number of the last bias
    __shared__ uint32_t note[SLAB];
    const int tid = threadIdx.x, row = blockIdx.x / a.slabs, s0 = (blockIdx.x - row * a.slabs) * SLAB;
    const wick_hip_logit_rules &r = a.r;
    const float *x = a.x + (size_t)row * a.stride;
    float *out = a.out + (size_t)row * a.out_stride;

    const int words = (a.vocab + 31) / 32;
    const uint32_t *mask = nullptr;
    if (r.mask) {
        const int m = r.mask_row ? r.mask_row[row] : row;
        if (m >= 0 && m < r.masks) mask = r.mask + (size_t)m * words;
    }
    float v[U][4];
    uint32_t allowed[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = s0 + 4 * (tid + u * kT);
        if (i + 4 <= a.vocab) {
            const f4u y = *reinterpret_cast<const f4u *>(x + i);
#pragma unroll
            for (int j = 0; j < 4; j++) v[u][j] = y[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[u][j] = i + j < a.vocab ? x[i + j] : 0.0f;
        }
        allowed[u] = ~0u;
        if (mask && i < a.vocab) allowed[u] = mask[i >> 5] >> (i & 31);
    }

    const uint32_t n = r.tokens ? min(max(r.n_tokens[row], 0), r.tokens_stride) : 0;
    const uint32_t prompt = n && r.n_prompt ? max(r.n_prompt[row], 0) : 0;
    int b0 = 0, b1 = 0;
    if (r.bias) {
        b0 = min(max(r.bias_start[row], 0), r.n_bias);
        b1 = min(max(r.bias_start[row + 1], 0), r.n_bias);
    }
    u4 *const mine = reinterpret_cast<u4 *>(note) + tid;  // mine[u * kT]: this thread's ids of pass u
    if (n > 0) {
#pragma unroll
        for (int u = 0; u < U; u++) mine[u * kT] = u4{0, 0, 0, 0};
        __syncthreads();
        const uint32_t *tokens = r.tokens + (size_t)row * r.tokens_stride;
        auto seen = [&](uint32_t i, uint32_t id) {
            const uint32_t at = id - (uint32_t)s0;
            if (at < (uint32_t)SLAB) {
                atomicOr(&note[at], kSeen);
                if (i >= prompt) atomicAdd(&note[at], 1u);
            }
        };
        const uint32_t n4 = n & ~3u;  // unsigned: a step past 2^31 tokens does not overflow
        for (uint32_t i = 4 * tid; i < n4; i += 4 * kT) {
            const u4u id = *reinterpret_cast<const u4u *>(tokens + i);
#pragma unroll
            for (int j = 0; j < 4; j++) seen(i + j, id[j]);
        }
        if (n4 + tid < n) seen(n4 + tid, tokens[n4 + tid]);
        __syncthreads();
        const float rep = r.repetition ? r.repetition[row] : 1.0f, pres = r.presence ? r.presence[row] : 0.0f,
                    freq = r.frequency ? r.frequency[row] : 0.0f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const u4 c = mine[u * kT];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float y = v[u][j];
                if (c[j]) y = y > 0.0f ? y / rep : y * rep;
                const uint32_t times = c[j] & ~kSeen;
                if (times) y -= freq * (float)times + pres;
                v[u][j] = y;
            }
        }
    }
    if (b1 > b0) {  // a thread clears its own ids, which only it has read
#pragma unroll
        for (int u = 0; u < U; u++) mine[u * kT] = u4{0, 0, 0, 0};
        __syncthreads();
        for (uint32_t i = b0 + tid; i < (uint32_t)b1; i += kT) {
            const uint32_t at = r.bias_ids[i] - (uint32_t)s0;
            if (at < (uint32_t)SLAB) atomicMax(&note[at], i - b0 + 1);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++) {
            const u4 c = mine[u * kT];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (c[j]) v[u][j] += r.bias[b0 + c[j] - 1];
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i = s0 + 4 * (tid + u * kT);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (!(allowed[u] >> j & 1)) v[u][j] = -INFINITY;
        if (i + 4 <= a.vocab) {
            *reinterpret_cast<f4u *>(out + i) = f4u{v[u][0], v[u][1], v[u][2], v[u][3]};
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < a.vocab) out[i + j] = v[u][j];
        }
    }
}

}  // namespace

// 4096 ids a workgroup read a row's tokens four times less often than 1024 do, from where
// that leaves every compute unit two workgroups (64 rows of 128256: 14.2 us with 4096, 15.5 with
// 2048, 16.0 with 8192; 8 rows of 151936, 304 workgroups of 4096: 7.6 us, with 1024 5.8).
int logit_slab(int rows, int vocab) { return (long long)rows * ((vocab + 4095) / 4096) >= 512 ? 4096 : 1024; }

hipError_t launch_logits(const LogitArgs &a, hipStream_t s) {
    const int grid = a.rows * a.slabs;
    if (logit_slab(a.rows, a.vocab) == 4096)
        logits_kernel<4096><<<grid, kT, 0, s>>>(a);
    else
        logits_kernel<1024><<<grid, kT, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace wick

// batch.hip -- attention of a batch's packed tokens over a shared prefix and the
// sequences' own positions, and the cache writes that go with it.
//
// A workgroup (BatchItem) has 32 rows of one kv head -- a row is one (token, query head)
// pair -- and walks its keys in steps of 128, each of its 4 waves 32 keys of a step.  Per
// 32 keys a wave computes
//   S^T [32 keys x 32 rows] = K Q^T,   P^T = exp2(S^T - m),   O^T [D x 32 rows] += V^T P^T
// with v_mfma_f32_32x32x16_bf16.  Its four waves' states (m, l, O) are joined through LDS.
//
// f32 products on the bf16 matrix cores.  x = x1 + x2 + x3, each part the bf16 nearest to
// what the ones before it leave (8 + 8 + 8 significant bits: exact but for the last part's
// rounding, 2^-27 of x), and x y = sum of x_i y_j.  A part of index i is at most 2^-9(i-1)
// of x, so the six products with i + j <= 4 leave out less than 2^-26 of |x y| -- under
// half the rounding of an f32 product -- and the sums are the matrix cores' f32 ones.  Six bf16
// products cost 6/16 of the f32 matrix instructions'.  A bf16 cache is its own first part:
// three products.  Infinities and values next to f32's largest have no such parts (inf - inf),
// nor may a hidden key's NaN times a weight of 0 count: either leaves a NaN or an infinity in
// its row's state, and a row with one is computed again, key by key in f32 (redo_row).
//
// Layouts.  The 32x32x16 instruction gives lane l of a wave row (or column) l % 32 and, of the
// 16 contracted indices, the 8 numbered 8 (l / 32)...  S^T leaves in lane l, for row l % 32, the keys
//   4 (l / 32) + i % 4 + 8 (i / 4),  i < 16,
// and 8 of them at a time are taken as one PV operand: the contracted index is a key either
// way, so V's operand takes the same keys in the same places and P never leaves its lane.  V's
// rows of the instruction are the dimensions d = (D / 32) (l % 32) + b, b = 0.. for the
// D / 32 instructions, so that a lane reads D / 32 adjacent values of a key, and a half
// wave a whole key.
#include <hip/hip_runtime.h>

#include "batch_kernels.h"
#include "wave_ops.h"

namespace wick {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

// A state without keys: finite, so that exp2(m - m) of two such is 1 and not NaN.
constexpr float kNoMax = -3.0e38f;
// The reference maximum is raised only when a score passes it by this (in log2 units):
// weights then stay below 2^8, and the rescaling of O is rare.
constexpr float kSlack = 8.0f;

// The parts of 8 values: part[0] + part[1] + part[2] = x (see above).
template <int PARTS>
struct Parts {
    b16x8 part[PARTS];
};

__device__ __forceinline__ Parts<3> split8(const float *x) {
    Parts<3> r;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        f32x2 v = {x[i], x[i + 1]};
#pragma unroll
        for (int p = 0; p < 3; p++) {
            const b16x2 h = __builtin_convertvector(v, b16x2);
            r.part[p][i] = h[0];
            r.part[p][i + 1] = h[1];
            v -= __builtin_convertvector(h, f32x2);
        }
    }
    return r;
}

__device__ __forceinline__ f32x16 mfma(b16x8 a, b16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// c += a b over the parts, the smallest products first.
__device__ __forceinline__ f32x16 product(const Parts<3> &a, const Parts<3> &b, f32x16 c) {
    c = mfma(a.part[2], b.part[0], c);
    c = mfma(a.part[0], b.part[2], c);
    c = mfma(a.part[1], b.part[1], c);
    c = mfma(a.part[1], b.part[0], c);
    c = mfma(a.part[0], b.part[1], c);
    return mfma(a.part[0], b.part[0], c);
}
__device__ __forceinline__ f32x16 product(const Parts<1> &a, const Parts<3> &b, f32x16 c) {
    c = mfma(a.part[0], b.part[2], c);
    c = mfma(a.part[0], b.part[1], c);
    return mfma(a.part[0], b.part[0], c);
}

// N adjacent values.
template <int N>
__device__ __forceinline__ void load_n(const float *p, float *x) {
    if constexpr (N == 1) {
        x[0] = *p;
    } else if constexpr (N == 2) {
        const f32x2 v = *reinterpret_cast<const f32x2 *>(p);
        x[0] = v[0];
        x[1] = v[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(p + i);
#pragma unroll
            for (int j = 0; j < 4; j++) x[i + j] = v[j];
        }
    }
}
template <int N>
__device__ __forceinline__ void load_n(const __bf16 *p, __bf16 *x) {
    if constexpr (N == 1) {
        x[0] = *p;
    } else if constexpr (N == 2) {
        const b16x2 v = *reinterpret_cast<const b16x2 *>(p);
        x[0] = v[0];
        x[1] = v[1];
    } else if constexpr (N == 4) {
        const b16x4 v = *reinterpret_cast<const b16x4 *>(p);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = v[j];
    } else {
        const b16x8 v = *reinterpret_cast<const b16x8 *>(p);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = v[j];
    }
}

__device__ __forceinline__ Parts<3> parts8(const float *x) { return split8(x); }
__device__ __forceinline__ Parts<1> parts8(const __bf16 *x) {
    Parts<1> r;
#pragma unroll
    for (int i = 0; i < 8; i++) r.part[0][i] = x[i];
    return r;
}

__device__ __forceinline__ float other_half(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? p[0] : p[1]);
}

template <int D>
struct Lds {
    float o[4][32][D + 4];  // the waves' O, by row
    float m[4][32], l[4][32];
    int redo[32];
};

// One row again in f32, key by key by one wave, over the item's keys that it sees: the
// definition itself, for rows with a value that the parts have no room for.  Lane d has
// the dimensions d, d + 64; o gets them unscaled.
template <int D, class T>
__device__ void redo_row(const BatchArgs &a, const BatchItem &it, const float *q, const T *pk, const T *pv, const T *k,
                         const T *v, int own_end, float *m_out, float *l_out, float *o_out) {
    const int lane = threadIdx.x & 63;
    constexpr int N = (D + 63) / 64;
    float x[N], acc[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = lane + 64 * i < D ? q[lane + 64 * i] * a.scale : 0.0f;
        acc[i] = 0.0f;
    }
    float m = kNoMax, l = 0.0f;
    for (int part = 0; part < 2; part++) {
        const T *kk = part ? k : pk, *vv = part ? v : pv;
        const int end = part ? own_end : it.p1;
        for (int key = part ? it.o0 : it.p0; key < end; key++) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (lane + 64 * i < D) s += x[i] * (float)kk[(size_t)key * D + lane + 64 * i];
            s = wave_sum(s);
            if (!(s <= m)) {  // a NaN too: it is the row's result from here on
                const float f = exp2f(m - s);
                l *= f;
#pragma unroll
                for (int i = 0; i < N; i++) acc[i] *= f;
                m = s;
            }
            const float p = exp2f(s - m);
            l += p;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (lane + 64 * i < D) acc[i] += p * (float)vv[(size_t)key * D + lane + 64 * i];
        }
    }
    *m_out = m;
    *l_out = l;
#pragma unroll
    for (int i = 0; i < N; i++)
        if (lane + 64 * i < D) o_out[lane + 64 * i] = acc[i];
}

template <int D, class T>
__global__ __launch_bounds__(256) void batch_attend_kernel(BatchArgs a) {
    constexpr int KS = D / 16;               // QK instructions per part product
    constexpr int NB = D >= 32 ? D / 32 : 1;  // 32-dimension blocks of O
    constexpr int KP = sizeof(T) == 4 ? 3 : 1;
    __shared__ Lds<D> lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const int heads = a.group * a.kv_heads;

    // the plan in memory is another one than at the call (a replayed graph)
    if (a.head->shape != a.shape) {
        const size_t n = (size_t)a.total * heads * D;
        for (size_t i = (size_t)blockIdx.x * 256 + tid; i < n; i += (size_t)gridDim.x * 256)
            a.att[i] = __builtin_nanf("");
        return;
    }
    const int work = a.head->items * a.kv_heads;
    for (int w = blockIdx.x; w < work; w += gridDim.x) {
        const BatchItem it = a.items[w / a.kv_heads];
        const int kh = w % a.kv_heads;
        const T *pk = static_cast<const T *>(a.pk) + (size_t)kh * a.prefix_capacity * D;
        const T *pv = static_cast<const T *>(a.pv) + (size_t)kh * a.prefix_capacity * D;
        const size_t own = it.seq < 0 ? 0 : ((size_t)it.seq * a.kv_heads + kh) * a.capacity * D;
        const T *ok = static_cast<const T *>(a.k) + own, *ov = static_cast<const T *>(a.v) + own;

        // a row's token and place in q and att
        auto row_at = [&](int r) {
            const int row = it.row0 + r, t = row / a.group, h = row - t * a.group;
            const int token = it.seq < 0 ? a.tokens[t].split : t;
            return ((size_t)token * heads + kh * a.group + h) * D;
        };
        const int r = min(col, it.nrows - 1);
        const int last = it.seq < 0 ? -1 : (it.row0 + r) / a.group + it.shift;  // the row's last own key
        const int first_last = it.seq < 0 ? -1 : it.row0 / a.group + it.shift;  // the first row's

        Parts<3> q[KS];
        {
            const float *src = a.q + row_at(r);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                float x[8];
                load_n<8>(src + 16 * ks + 8 * half, x);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] *= a.scale;
                q[ks] = split8(x);
            }
        }
        f32x16 o[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) o[b] = f32x16{};
        float m = kNoMax, l = 0.0f;

        for (int part = 0; part < 2; part++) {
            const T *kk = part ? ok : pk, *vv = part ? ov : pv;
            const int begin = part ? it.o0 : it.p0, end = part ? it.o1 : it.p1;
            for (int key0 = begin + 32 * wave; key0 < end; key0 += kBatchStep) {
                f32x16 s{};
                const T *krow = kk + (size_t)min(key0 + col, end - 1) * D + 8 * half;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    T x[8];
                    load_n<8>(krow + 16 * ks, x);
                    s = product(parts8(x), q[ks], s);
                }
                if (key0 + 32 > end || (part && key0 + 31 > first_last)) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int key = key0 + 4 * half + i % 4 + 8 * (i / 4);
                        if (key >= end || (part && key > last)) s[i] = -INFINITY;
                    }
                }
                float top = s[0];
#pragma unroll
                for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
                top = fmaxf(top, other_half(top));
                if (__any(top > m + kSlack)) {
                    const float to = fmaxf(m, top), f = exp2f(m - to);
                    l *= f;
#pragma unroll
                    for (int b = 0; b < NB; b++)
#pragma unroll
                        for (int i = 0; i < 16; i++) o[b][i] *= f;
                    m = to;
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    s[i] = __builtin_amdgcn_exp2f(s[i] - m);
                    l += s[i];
                }
#pragma unroll
                for (int kk2 = 0; kk2 < 2; kk2++) {
                    float p[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) p[j] = s[8 * kk2 + j];
                    const Parts<3> pp = split8(p);
                    T x[8][NB];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int key = min(key0 + 16 * kk2 + (j / 4) * 8 + 4 * half + j % 4, end - 1);
                        load_n<NB>(vv + (size_t)key * D + (D < 32 ? col % D : NB * col), x[j]);
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        T y[8];
#pragma unroll
                        for (int j = 0; j < 8; j++) y[j] = x[j][b];
                        o[b] = product(parts8(y), pp, o[b]);
                    }
                }
            }
        }
        l += other_half(l);

        // join the waves' states: O by row through LDS
        if (half == 0) {
            lds.m[wave][col] = m;
            lds.l[wave][col] = l;
        }
        if (tid < 32) lds.redo[tid] = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int d = 4 * half + i % 4 + 8 * (i / 4);
#pragma unroll
            for (int b = 0; b < NB; b++)
                if (NB * d + b < D) lds.o[wave][col][NB * d + b] = o[b][i];
        }
        __syncthreads();
        {
            // 8 threads a row, D / 8 dimensions each
            constexpr int E = D / 8;
            const int row = tid >> 3, d0 = (tid & 7) * E;
            float to = lds.m[0][row];
#pragma unroll
            for (int i = 1; i < 4; i++) to = fmaxf(to, lds.m[i][row]);
            float sum = 0.0f, acc[E];
#pragma unroll
            for (int e = 0; e < E; e++) acc[e] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float f = exp2f(lds.m[i][row] - to);
                sum += f * lds.l[i][row];
#pragma unroll
                for (int e = 0; e < E; e++) acc[e] += f * lds.o[i][row][d0 + e];
            }
            bool odd = !(fabsf(sum) < INFINITY);
#pragma unroll
            for (int e = 0; e < E; e++) odd |= !(fabsf(acc[e]) < INFINITY);
            if (odd && row < it.nrows) lds.redo[row] = 1;
            __syncthreads();
            // each thread has read its own values of all waves and nobody else's
#pragma unroll
            for (int e = 0; e < E; e++) lds.o[0][row][d0 + e] = acc[e];
            if ((tid & 7) == 0) {
                lds.m[0][row] = to;
                lds.l[0][row] = sum;
            }
        }
        __syncthreads();
        for (int rr = wave; rr < it.nrows; rr += 4)
            if (lds.redo[rr]) {
                float rm, rl;
                const int seen = it.seq < 0 ? 0 : min(it.o1, (it.row0 + rr) / a.group + it.shift + 1);
                redo_row<D, T>(a, it, a.q + row_at(rr), pk, pv, ok, ov, seen, &rm, &rl, lds.o[0][rr]);
                lds.m[0][rr] = rm;
                lds.l[0][rr] = rl;
            }
        __syncthreads();
        {
            constexpr int E = D / 8;
            const int row = tid >> 3, d0 = (tid & 7) * E;
            if (row < it.nrows) {
                const float sum = lds.l[0][row], f = it.state0 < 0 ? 1.0f / sum : 1.0f;
                float *dst;
                if (it.state0 < 0) {
                    dst = a.att + row_at(row) + d0;
                } else {
                    const size_t at = (size_t)kh * a.state_rows + it.state0 + row;
                    dst = a.po + at * D + d0;
                    if (d0 == 0) {
                        a.pm[at] = lds.m[0][row];
                        a.pl[at] = sum;
                    }
                }
#pragma unroll
                for (int e = 0; e < E; e++) dst[e] = lds.o[0][row][d0 + e] * f;
            }
        }
        __syncthreads();
    }
}

// A wave joins one row's states: weights 2^(m_i - max), att = sum w O / sum w l.  Up to 64
// states at a time have a lane each; for the sum of O, D / 4 lanes read one state.
template <int D>
__global__ __launch_bounds__(256) void batch_merge_kernel(BatchArgs a) {
    constexpr int L = D / 4, G = 64 / L;  // lanes of a state, states at once
    const int lane = threadIdx.x & 63, g = lane / L, d = 4 * (lane % L);
    const int heads = a.group * a.kv_heads;
    if (a.head->shape != a.shape) return;
    const int work = a.head->merges * heads, prefix_chunks = a.head->prefix_chunks;
    for (int w = blockIdx.x * 4 + (threadIdx.x >> 6); w < work; w += gridDim.x * 4) {
        const int i = w / heads, head = w - i * heads, kh = head / a.group, h = head - kh * a.group;
        const BatchToken t = a.tokens[i];
        const size_t base = (size_t)kh * a.state_rows;
        const int n = prefix_chunks + t.own_chunks;
        auto state = [&](int c) {
            const int row = c < prefix_chunks ? t.prefix_state + c * a.head->prefix_stride
                                              : t.own_state + (c - prefix_chunks) * t.own_stride;
            return base + row + h;
        };
        float top = kNoMax;
        for (int c = lane; c < n; c += 64) top = fmaxf(top, a.pm[state(c)]);
        top = wave_max(top);
        float sum = 0.0f;
        f32x4 acc{};
        for (int c0 = 0; c0 < n; c0 += 64) {
            float f = 0.0f;
            if (c0 + lane < n) {
                const size_t at = state(c0 + lane);
                f = exp2f(a.pm[at] - top);
                sum += f * a.pl[at];
            }
            const int m = min(64, n - c0);
            for (int c = 0; c < m; c += G) {
                const float fc = __shfl(f, min(c + g, 63), 64);
                if (c + g < m) acc += fc * *reinterpret_cast<const f32x4 *>(a.po + state(c0 + c + g) * D + d);
            }
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int x = L; x < 64; x <<= 1)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], x, 64);
        const float f = 1.0f / sum;
        if (g == 0) *reinterpret_cast<f32x4 *>(a.att + ((size_t)t.merge * heads + head) * D + d) = acc * f;
    }
}

// 4 values a thread.
__device__ __forceinline__ void store4(float *p, f32x4 v) { *reinterpret_cast<f32x4 *>(p) = v; }
__device__ __forceinline__ void store4(__bf16 *p, f32x4 v) {
    *reinterpret_cast<b16x4 *>(p) = __builtin_convertvector(v, b16x4);
}
__device__ __forceinline__ f32x4 load4(const float *p) { return *reinterpret_cast<const f32x4 *>(p); }
__device__ __forceinline__ f32x4 load4(const __bf16 *p) {
    return __builtin_convertvector(*reinterpret_cast<const b16x4 *>(p), f32x4);
}

template <int D, class T>
__global__ __launch_bounds__(256) void batch_append_kernel(BatchAppendArgs a) {
    if (a.head && a.head->shape != a.shape) return;
    const int per = a.kv_heads * D / 4;
    const long long n = (long long)a.total * per;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const int tok = (int)(i / per), e = (int)(i - (long long)tok * per), kh = e / (D / 4), d = 4 * (e % (D / 4));
        int seq = 0, pos = a.start + tok;
        if (a.head) {
            seq = a.tokens[tok].seq;
            pos = a.tokens[tok].pos;
        }
        const size_t at = (((size_t)seq * a.kv_heads + kh) * a.capacity + pos) * D + d;
        store4(static_cast<T *>(a.k) + at, load4(a.ksrc + 4 * i));
        store4(static_cast<T *>(a.v) + at, load4(a.vsrc + 4 * i));
    }
}

template <int D, class T>
__global__ __launch_bounds__(256) void batch_load_kernel(const float *src, int src_capacity, T *dst, int dst_capacity,
                                                         int len) {
    const long long n = (long long)len * D / 4;
    src += (size_t)blockIdx.y * src_capacity * D;
    dst += (size_t)blockIdx.y * dst_capacity * D;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256)
        store4(dst + 4 * i, load4(src + 4 * i));
}

template <int D, class T>
__global__ __launch_bounds__(256) void batch_read_kernel(const T *src, int capacity, int kv_heads, int pos0, int n,
                                                         float *dst) {
    const int per = kv_heads * D / 4;
    const long long all = (long long)n * per;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const int tok = (int)(i / per), e = (int)(i - (long long)tok * per), kh = e / (D / 4), d = 4 * (e % (D / 4));
        store4(dst + 4 * i, load4(src + ((size_t)kh * capacity + pos0 + tok) * D + d));
    }
}

int grid_of(long long threads) { return (int)std::min<long long>(4096, std::max<long long>(1, (threads + 255) / 256)); }

// f(D, T) for the handle's head_dim and type.
template <class F>
hipError_t dispatch(int head_dim, int bf16, F &&f) {
    switch (head_dim) {
    case 16: return bf16 ? f.template operator()<16, __bf16>() : f.template operator()<16, float>();
    case 32: return bf16 ? f.template operator()<32, __bf16>() : f.template operator()<32, float>();
    case 64: return bf16 ? f.template operator()<64, __bf16>() : f.template operator()<64, float>();
    case 128: return bf16 ? f.template operator()<128, __bf16>() : f.template operator()<128, float>();
    default: return hipErrorInvalidValue;
    }
}

struct AttendLaunch {
    const BatchArgs &a;
    int grid;
    hipStream_t s;
    template <int D, class T>
    hipError_t operator()() {
        batch_attend_kernel<D, T><<<grid, 256, 0, s>>>(a);
        return hipGetLastError();
    }
};
struct MergeLaunch {
    const BatchArgs &a;
    int grid;
    hipStream_t s;
    template <int D, class T>
    hipError_t operator()() {
        batch_merge_kernel<D><<<grid, 256, 0, s>>>(a);
        return hipGetLastError();
    }
};
struct AppendLaunch {
    const BatchAppendArgs &a;
    hipStream_t s;
    template <int D, class T>
    hipError_t operator()() {
        batch_append_kernel<D, T><<<grid_of((long long)a.total * a.kv_heads * D / 4), 256, 0, s>>>(a);
        return hipGetLastError();
    }
};
struct LoadLaunch {
    const float *src;
    int src_capacity;
    void *dst;
    int dst_capacity, kv_heads, len;
    hipStream_t s;
    template <int D, class T>
    hipError_t operator()() {
        batch_load_kernel<D, T><<<dim3(grid_of((long long)len * D / 4), kv_heads), 256, 0, s>>>(
            src, src_capacity, static_cast<T *>(dst), dst_capacity, len);
        return hipGetLastError();
    }
};
struct ReadLaunch {
    const void *src;
    int capacity, kv_heads, pos0, n;
    float *dst;
    hipStream_t s;
    template <int D, class T>
    hipError_t operator()() {
        batch_read_kernel<D, T><<<grid_of((long long)n * kv_heads * D / 4), 256, 0, s>>>(
            static_cast<const T *>(src), capacity, kv_heads, pos0, n, dst);
        return hipGetLastError();
    }
};
struct Occupancy {
    int blocks = 1;
    template <int D, class T>
    hipError_t operator()() {
        return hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, batch_attend_kernel<D, T>, 256, 0);
    }
};

}  // namespace

hipError_t launch_batch_attend(int head_dim, int bf16, const BatchArgs &a, int grid, hipStream_t s) {
    return dispatch(head_dim, bf16, AttendLaunch{a, grid, s});
}
hipError_t launch_batch_merge(int head_dim, const BatchArgs &a, int merges, hipStream_t s) {
    const long long waves = (long long)merges * a.group * a.kv_heads;
    return dispatch(head_dim, 0, MergeLaunch{a, (int)std::min<long long>(1 << 20, (waves + 3) / 4), s});
}
hipError_t launch_batch_append(int head_dim, int bf16, const BatchAppendArgs &a, hipStream_t s) {
    return dispatch(head_dim, bf16, AppendLaunch{a, s});
}
hipError_t launch_batch_load(int head_dim, int bf16, const float *src, int src_capacity, void *dst, int dst_capacity,
                             int kv_heads, int len, hipStream_t s) {
    return dispatch(head_dim, bf16, LoadLaunch{src, src_capacity, dst, dst_capacity, kv_heads, len, s});
}
hipError_t launch_batch_read(int head_dim, int bf16, const void *src, int capacity, int kv_heads, int pos0, int n,
                             float *dst, hipStream_t s) {
    return dispatch(head_dim, bf16, ReadLaunch{src, capacity, kv_heads, pos0, n, dst, s});
}
int batch_blocks_per_cu(int head_dim, int bf16) {
    Occupancy o;
    return dispatch(head_dim, bf16, o) == hipSuccess && o.blocks > 0 ? o.blocks : 1;
}

}  // namespace wick

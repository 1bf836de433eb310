// batch.hip -- attention of a batch's packed tokens over a shared prefix and the
// sequences' own positions, and the cache writes that go with it.
//
// A workgroup (BatchItem) has some rows of one kv head -- a row is one (token, query head)
// pair -- and walks its keys.  Per 32 keys a wave computes
//   S^T [keys x rows] = K Q^T,   P^T = exp2(S^T - m),   O^T [D x rows] += V^T P^T
// with the running maximum m and sum l of each row.  Items of up to 128 rows are wide: each of
// the 4 waves has 32 rows, all of them the same keys, whose operands they prepare together in
// LDS (v_mfma_f32_32x32x16_bf16).  Items of up to 16 rows are narrow: the waves have the same rows
// and every fourth 32 keys each, and join their states through LDS at the end
// (v_mfma_f32_16x16x32_bf16).
//
// f32 products on the bf16 matrix cores.  x = x1 + x2 + x3, each part the bf16 nearest to
// what the ones before it leave (8 + 8 + 8 significant bits: exact but for the last part's
// rounding, 2^-27 of x), and x y = sum of x_i y_j.  A part of index i is at most 2^-9(i-1)
// of x, so the six products with i + j <= 4 leave out about 2^-26 of |x y| -- half the
// rounding of an f32 product -- and the sums are the matrix cores' f32 ones.  Six bf16
// products cost 6/16 of the f32 matrix instructions'.  A bf16 cache is its own first part:
// three products.  (Values under 2^-108 lose low parts to underflow.)  Infinities and values
// next to f32's largest have no such parts (inf - inf), large values' sums may overflow where
// their mean does not, nor may a hidden key's NaN times a weight of 0 count: each leaves a NaN or
// an infinity in its row's state, and a row with one is computed again, key by key in f32 (redo_row).
//
// Layouts.  The 32x32x16 instruction gives lane l of a wave row (or column) l % 32 and, of the
// 16 contracted indices, the 8 numbered 8 (l / 32)...  S^T leaves in lane l, for row l % 32, the keys
//   4 (l / 32) + i % 4 + 8 (i / 4),  i < 16,
// and 8 of them at a time are taken as one PV operand: the contracted index is a key either
// way, so V's operand takes the same keys in the same places and P never leaves its lane.  V's
// rows of the instruction are the dimensions d = (D / 32) (l % 32) + b, b = 0.. for the
// D / 32 instructions, so that a lane reads D / 32 adjacent values of a key, and a half
// wave a whole key.
//
// Bound.  Wide items: the matrix cores, at the rate that the card's power leaves them (a large
// bf16 product reaches 1.16 PFLOP/s here, this instruction alone with random operands
// 1.75).  Six prompts of 697..2047 tokens (32/8 heads of 128) take 0.39 to 0.41 ms: 76.9 GFLOP, six
// times that in parts, 1.2 PFLOP/s; on a bf16 cache 53 GFLOP, three times, 0.16 ms, 1.0 PFLOP/s, where
// the weights' vector instructions are the next limit.  A tile of 32 keys (head_dim 128, f32) takes
// 4.06 us where a unit has two wide items and 2.7 where it has one, against 1.7 of products.  Narrow items:
// the latency of a step's loads, then the split of its values; HBM where there are many.
#include <hip/hip_runtime.h>

#include <type_traits>

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

// The maximum of a state without keys: f32's lowest value, so that no finite score is below it, and
// exp2(m - m) of two such is 1 and not NaN.
constexpr float kNoMax = -3.40282347e38f;
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

// The parts of 2 values, to places j and j + 1.
__device__ __forceinline__ void split2(const float *x, Parts<3> &r, int j) {
    f32x2 v = {x[0], x[1]};
#pragma unroll
    for (int p = 0; p < 3; p++) {
        const b16x2 h = __builtin_convertvector(v, b16x2);
        r.part[p][j] = h[0];
        r.part[p][j + 1] = h[1];
        v -= __builtin_convertvector(h, f32x2);
    }
}
__device__ __forceinline__ void split2(const __bf16 *x, Parts<1> &r, int j) {
    r.part[0][j] = x[0];
    r.part[0][j + 1] = x[1];
}

// The parts of 4 values.
__device__ __forceinline__ void parts4(const float *x, b16x4 (&part)[3]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        f32x2 v = {x[i], x[i + 1]};
#pragma unroll
        for (int p = 0; p < 3; p++) {
            const b16x2 h = __builtin_convertvector(v, b16x2);
            part[p][i] = h[0];
            part[p][i + 1] = h[1];
            v -= __builtin_convertvector(h, f32x2);
        }
    }
}
__device__ __forceinline__ void parts4(const __bf16 *x, b16x4 (&part)[1]) {
#pragma unroll
    for (int i = 0; i < 4; i++) part[0][i] = x[i];
}

// x / d for 0 <= x < 2^31, inv = min(2^32 / d rounded up, 2^32 - 1): off by one at most before the correction.
__device__ __forceinline__ int divide(int x, int d, unsigned inv) {
    int q = (int)__umulhi((unsigned)x, inv);
    const int r = x - q * d;
    return r < 0 ? q - 1 : r >= d ? q + 1 : q;
}

__device__ __forceinline__ float other_half(float v) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? p[0] : p[1]);
}

// Whether the plan in memory is one that the call was made for (a replayed graph's may not be).
__device__ __forceinline__ bool fits(const BatchArgs &a) { return a.head->shape == a.shape && a.head->items <= a.launched; }

// What the kernel's shape fixes.
template <int D, class T>
struct Shape {
    static constexpr int KS = D / 16;                // QK instructions per product of parts and 32 keys
    static constexpr int NB = D >= 32 ? D / 32 : 1;  // 32-dimension blocks of O
    static constexpr int KP = sizeof(T) == 4 ? 3 : 1;
    // a wide item's tile: 64 keys, or 32 where the parts of 64 would not leave room for two
    // workgroups on a CU (one of them 437 us for the six prompts, two 403; tiles of 32 keys in
    // all cases, a tile's values weighted next to the next tile's weights: eight prompts of 39..701
    // (14/2 heads of 64) 39.1 us, as it is 36.0)
    static constexpr int KT = D == 128 && KP == 3 ? 32 : 64;
    // q's third parts lie in LDS where all of them would not leave the registers for two (spilled,
    // the six prompts took 614 us)
    static constexpr int QP = D == 128 ? 2 : 3;
    static constexpr int KF = KT / 32 * KS, VF = KT / 16 * NB;  // operands of a tile: K's, V's
    // a narrow item's, with 16x16x32 instructions
    static constexpr int KS16 = D >= 32 ? D / 32 : 1, NB16 = D / 16;
};

// Operands lie as the instruction takes them: a wave reads one with its lanes side by side.
template <int D, class T>
struct Tile {
    using S = Shape<D, T>;
    b16x8 k[S::KP][S::KF][64], v[S::KP][S::VF][64];
};
template <int KP, int N>
__device__ __forceinline__ Parts<KP> read(const b16x8 (&x)[KP][N][64], int i, int lane) {
    Parts<KP> r;
#pragma unroll
    for (int p = 0; p < KP; p++) r.part[p] = x[p][i][lane];
    return r;
}

// The four waves' states of a narrow item, by row.
template <int D>
struct Join {
    float o[4][kBatchRows][D + 4];
    float m[4][kBatchRows], l[4][kBatchRows];
    int redo[kBatchRows];
};

// A tile's keys or values on their way to LDS: each wave has every fourth K operand, and
// of V's 16-key groups every fourth half.  Keys past `end` are the last one again.
template <int D, class T>
struct StageK {
    using S = Shape<D, T>;
    static constexpr int N = (S::KF + 3) / 4;
    T x[N][8];

    // k: the tile's first key, of n left
    __device__ __forceinline__ void load(const T *k, int n, int wave, int col, int half) {
        if (S::KF < 4 && wave >= S::KF) return;
        // operand wave + 4 u: 32 keys, 16 dimensions
        const int sub = S::KS >= 4 ? 0 : wave / S::KS, ks = S::KS >= 4 ? wave : wave % S::KS;
#pragma unroll
        for (int u = 0; u < N; u++)
            load_n<8>(k + 16 * (ks + 4 * u % S::KS) + (unsigned)(min(32 * (sub + 4 * u / S::KS) + col, n - 1) * D + 8 * half),
                      x[u]);
    }
    // The split into parts and the write in UNITS steps, each two values of a lane's 8.
    static constexpr int UNITS = 4 * N;
    Parts<S::KP> y;
    __device__ __forceinline__ static b16x8 *place(Tile<D, T> &t, int wave, int lane) { return &t.k[0][wave][lane]; }
    __device__ __forceinline__ void store(int i, b16x8 *at, int wave) {
        const int u = i / 4, j = 2 * (i % 4);
        if (S::KF < 4 && wave >= S::KF) return;
        split2(x[u] + j, y, j);
        if (j == 6)
#pragma unroll
            for (int p = 0; p < S::KP; p++) at[(p * S::KF + 4 * u) * 64] = y.part[p];
    }
};
template <int D, class T>
struct StageV {
    using S = Shape<D, T>;
    static constexpr int N = S::KT / 32;
    T x[N][4][S::NB];

    __device__ __forceinline__ void load(const T *v, int n, int wave, int col, int half) {
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int h = wave + 4 * u;
#pragma unroll
            for (int j = 0; j < 4; j++)
                load_n<S::NB>(v + (unsigned)(min(8 * h + 4 * half + j, n - 1) * D + (D < 32 ? col % D : S::NB * col)), x[u][j]);
        }
    }
    // The same in UNITS steps of a dimension.
    static constexpr int UNITS = N * S::NB;
    __device__ __forceinline__ static b16x4 *place(Tile<D, T> &t, int wave, int lane) {
        return reinterpret_cast<b16x4 *>(&t.v[0][wave / 2 * S::NB][lane]) + wave % 2;
    }
    __device__ __forceinline__ void store(int i, b16x4 *at) const {
        const int u = i / S::NB, b = i % S::NB;
        T y[4];
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = x[u][j][b];
        b16x4 part[S::KP];
        parts4(y, part);
#pragma unroll
        for (int p = 0; p < S::KP; p++) at[(p * S::VF + 2 * u * S::NB + b) * 128] = part[p];
    }
};

// Sums of weights times values may pass f32's range where their mean does not.  2^-32 of them never
// do: a row has less than 2^31 keys.  A row that needs it has its sums a second time at 2^-32,
// which take the place of those that overflowed; a state with any such sum has all of them
// at 2^-32 and says so by -l.
constexpr float kLow = 0x1p-32f, kLargest = 3.40282347e38f;

// low / l where sum overflowed and low did not: there the mean of finite values, which rounding may
// bring past the largest.  All others are `mean`.
__device__ __forceinline__ float mean_of(float sum, float mean, float low, float l) {
    if (fabsf(sum) < INFINITY || !(fabsf(low) < INFINITY)) return mean;
    return fminf(fmaxf(low / l, -kLargest), kLargest);
}

// One row again in f32, key by key by one wave, over the item's keys that it sees, for rows with a
// value that the parts, or the sums, have no room for.  Lane d has the dimensions d, d + 64.
template <int D, class T>
__device__ __noinline__ void redo_row(const float *q, float scale, const T *pk, const T *pv, int p0, int p1, const T *k,
                                      const T *v, int o0, int o1, bool direct, float *dst, float *m_out, float *l_out) {
    const int lane = threadIdx.x & 63;
    constexpr int N = (D + 63) / 64;
    float x[N], acc[N], low[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = lane + 64 * i < D ? q[lane + 64 * i] * scale : 0.0f;
        acc[i] = low[i] = 0.0f;
    }
    float m = kNoMax, l = 0.0f;
    for (int part = 0; part < 2; part++) {
        const T *kk = part ? k : pk, *vv = part ? v : pv;
        const int end = part ? o1 : p1;
        for (int key = part ? o0 : p0; key < end; key++) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (lane + 64 * i < D) s += x[i] * (float)kk[(size_t)key * D + lane + 64 * i];
            s = wave_sum(s);
            if (!(s <= m)) {  // a NaN too: it is the row's result from here on
                const float f = exp2f(m - s);
                l *= f;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    acc[i] *= f;
                    low[i] *= f;
                }
                m = s;
            }
            const float p = exp2f(s - m);
            l += p;
#pragma unroll
            for (int i = 0; i < N; i++)
                if (lane + 64 * i < D) {
                    const float y = (float)vv[(size_t)key * D + lane + 64 * i];
                    acc[i] += p * y;
                    low[i] += p * kLow * y;
                }
        }
    }
    bool over = false;
#pragma unroll
    for (int i = 0; i < N; i++) over |= !(fabsf(acc[i]) < INFINITY) && fabsf(low[i]) < INFINITY;
    const bool scaled = !direct && __any(over);
#pragma unroll
    for (int i = 0; i < N; i++)
        if (lane + 64 * i < D)
            dst[lane + 64 * i] = direct    ? mean_of(acc[i], acc[i] / l, low[i], l * kLow)
                                 : !scaled ? acc[i]
                                           : fabsf(acc[i]) < INFINITY ? acc[i] * kLow : low[i];
    if (!direct && lane == 0) {
        *m_out = m;
        *l_out = scaled ? -l : l;
    }
}

// The softmax state of a wave's 32 rows (row lane % 32), and what a tile of 32 keys does to it.
template <int D, class T>
struct Rows {
    using S = Shape<D, T>;
    Parts<S::QP> q[S::KS];
    b16x8 *rest;  // q's third parts where they are not in registers
    f32x16 o[S::NB];
    float m, l;  // l: of the keys in this lane

    __device__ __forceinline__ void begin(const float *src, float scale, int half, b16x8 *third) {
        rest = third;
#pragma unroll
        for (int ks = 0; ks < S::KS; ks++) {
            float x[8];
            load_n<8>(src + 16 * ks + 8 * half, x);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= scale;
            const Parts<3> y = split8(x);
#pragma unroll
            for (int p = 0; p < S::QP; p++) q[ks].part[p] = y.part[p];
            if constexpr (S::QP < 3) rest[64 * ks] = y.part[2];
        }
#pragma unroll
        for (int b = 0; b < S::NB; b++) o[b] = f32x16{};
        m = kNoMax;
        l = 0.0f;
    }

    __device__ __forceinline__ Parts<3> query(int ks) const {
        Parts<3> r;
#pragma unroll
        for (int p = 0; p < S::QP; p++) r.part[p] = q[ks].part[p];
        if constexpr (S::QP < 3) r.part[2] = rest[64 * ks];
        return r;
    }

    // scores s of the keys key0..: keys past `last` are hidden, the reference maximum follows
    template <bool MASK>
    __device__ __forceinline__ void scores(f32x16 &s, int key0, int half, int last) {
        if constexpr (MASK) {
            const int left = last - key0 - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = i % 4 + 8 * (i / 4) > left ? -INFINITY : s[i];
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
        top = fmaxf(top, other_half(top));
        if (__any(top > m + kSlack)) {
            const float to = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - to);
            l *= f;
#pragma unroll
            for (int b = 0; b < S::NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] *= f;
            m = to;
        }
    }

    // the weights of scores s[8 kk + j], s[8 kk + j + 1] and their parts
    __device__ __forceinline__ void weight2(f32x16 &s, Parts<3> &w, int kk, int j) {
        float p[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            p[i] = __builtin_amdgcn_exp2f(s[8 * kk + j + i] - m);
            l += p[i];
        }
        split2(p, w, j);
    }
};

__device__ __forceinline__ f32x4 mfma16(b16x8 a, b16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 product(const Parts<3> &a, const Parts<3> &b, f32x4 c) {
    c = mfma16(a.part[2], b.part[0], c);
    c = mfma16(a.part[0], b.part[2], c);
    c = mfma16(a.part[1], b.part[1], c);
    c = mfma16(a.part[1], b.part[0], c);
    c = mfma16(a.part[0], b.part[1], c);
    return mfma16(a.part[0], b.part[0], c);
}
__device__ __forceinline__ f32x4 product(const Parts<1> &a, const Parts<3> &b, f32x4 c) {
    c = mfma16(a.part[0], b.part[2], c);
    c = mfma16(a.part[0], b.part[1], c);
    return mfma16(a.part[0], b.part[0], c);
}

// Up to 16 rows (row lane % 16) against 32 keys at a time, the operands straight from
// memory.  The 16x16x32 instruction gives lane l row or column l % 16 and the contracted indices
// 8 (l / 16)..; scores leave it with keys 4 (l / 16) + i of each 16, so V's operand takes
// keys 4 (l / 16) + j and, for j >= 4, 16 + 4 (l / 16) + j - 4.
template <int D, class T>
struct Few {
    using S = Shape<D, T>;
    static constexpr int KS = S::KS16, NB = S::NB16;
    Parts<3> q[KS];
    f32x4 o[NB];
    float m, l;
    T k[2][KS][8], v[8][NB];

    __device__ __forceinline__ void begin(const float *src, float scale, int quad) {
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            float x[8] = {};
            if (D >= 32 || quad < 2) load_n<8>(src + 32 * ks + 8 * quad, x);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= scale;
            q[ks] = split8(x);
        }
#pragma unroll
        for (int b = 0; b < NB; b++) o[b] = f32x4{};
        m = kNoMax;
        l = 0.0f;
    }

    // of n keys left at p
    __device__ __forceinline__ void load_k(const T *p, int n, int col, int quad) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const unsigned at = min(16 * u + col, n - 1) * D + 8 * (D >= 32 ? quad : quad & 1);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) load_n<8>(p + 32 * ks + at, k[u][ks]);
        }
    }
    __device__ __forceinline__ void load_v(const T *p, int n, int col, int quad) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            load_n<NB>(p + (unsigned)(min(16 * (j / 4) + 4 * quad + j % 4, n - 1) * D + NB * col), v[j]);
    }

    __device__ __forceinline__ void scores(f32x4 (&s)[2]) const {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            s[u] = f32x4{};
#pragma unroll
            for (int ks = 0; ks < KS; ks++) s[u] = product(parts8(k[u][ks]), q[ks], s[u]);  // 16 dimensions: q's rest is 0
        }
    }

    // keys past `left` of the 32 are hidden
    __device__ __forceinline__ void values(f32x4 (&s)[2], bool mask, int left) {
        if (mask) {
#pragma unroll
            for (int i = 0; i < 8; i++) s[i / 4][i % 4] = 16 * (i / 4) + i % 4 > left ? -INFINITY : s[i / 4][i % 4];
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; i++) top = fmaxf(top, s[i / 4][i % 4]);
        top = rows_max(top);
        if (__any(top > m + kSlack)) {
            const float to = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - to);
            l *= f;
#pragma unroll
            for (int b = 0; b < NB; b++) o[b] *= f;
            m = to;
        }
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[i] = __builtin_amdgcn_exp2f(s[i / 4][i % 4] - m);
            l += p[i];
        }
        const Parts<3> w = split8(p);
#pragma unroll
        for (int b = 0; b < NB; b++) {
            T y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = v[j][b];
            o[b] = product(parts8(y), w, o[b]);
        }
    }
};

template <int D, class T>
__global__ __launch_bounds__(256, 2) void batch_attend_kernel(BatchArgs a) {
    using S = Shape<D, T>;
    constexpr int KS = S::KS, NB = S::NB, KT = S::KT;
    __shared__ union {
        Join<D> join;
        struct {
            Tile<D, T> tile;
            b16x8 third[S::QP < 3 ? 4 : 1][S::QP < 3 ? KS : 1][64];
        };
    } lds;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // the same in all lanes
    const int heads = a.group * a.kv_heads;

    if (!fits(a)) {
        const size_t n = (size_t)a.total * heads * D;
        for (size_t i = (size_t)blockIdx.x * 256 + tid; i < n; i += (size_t)gridDim.x * 256)
            a.att[i] = __builtin_nanf("");
        return;
    }
    if ((int)blockIdx.x >= a.head->items * a.kv_heads) return;
    {
        const int item = divide(blockIdx.x, a.kv_heads, a.inv_kv_heads), kh = blockIdx.x - item * a.kv_heads;
        const BatchItem it = a.items[item];
        const T *pk = static_cast<const T *>(a.pk) + (size_t)kh * a.prefix_capacity * D;
        const T *pv = static_cast<const T *>(a.pv) + (size_t)kh * a.prefix_capacity * D;
        const size_t own = it.seq < 0 ? 0 : ((size_t)it.seq * a.kv_heads + kh) * a.capacity * D;
        const T *ok = static_cast<const T *>(a.k) + own, *ov = static_cast<const T *>(a.v) + own;
        const bool direct = it.state0 < 0;

        // row r of the item: its place in q and att, its last own key, its states
        auto row_at = [&](int r) {
            const int row = it.row0 + r, t = divide(row, a.group, a.inv_group), h = row - t * a.group;
            const int token = it.seq >= 0 ? t : it.seq == -1 ? t + it.shift : a.tokens[t].split;
            return ((size_t)token * heads + kh * a.group + h) * D;
        };
        auto last_of = [&](int r) { return it.seq < 0 ? -1 : divide(it.row0 + r, a.group, a.inv_group) + it.shift; };
        auto state_at = [&](int r) { return (size_t)kh * a.state_rows + it.state0 + r; };
        auto redo = [&](int r) {
            const size_t at = direct ? 0 : state_at(r);
            redo_row<D, T>(a.q + row_at(r), a.scale, pk, pv, it.p0, it.p1, ok, ov, it.o0, min(it.o1, last_of(r) + 1), direct,
                           direct ? a.att + row_at(r) : a.po + at * D, a.pm + at, a.pl + at);
        };

        if (it.nrows > kBatchRows) {
            // this wave's rows
            const int r0 = 32 * wave, nr = min(32, it.nrows - r0);
            const int r = max(0, min(r0 + col, it.nrows - 1));
            const int last = last_of(r), first_last = last_of(min(r0, it.nrows - 1)),
                      end_last = last_of(min(r0 + 32, it.nrows) - 1);
            Rows<D, T> st;

            // The tiles of the prefix, then those of the own keys.  While the scores of a tile
            // are summed, its values are split into parts and written to LDS; while its values
            // are, the next tile's keys.
            StageK<D, T> sk;
            StageV<D, T> sv;
            const int tp = (it.p1 - it.p0 + KT - 1) / KT, tiles = tp + (it.o1 - it.o0 + KT - 1) / KT;
            auto first_key = [&](int t) { return t >= tp ? it.o0 + (t - tp) * KT : it.p0 + t * KT; };
            auto load_k = [&](int t) {
                const bool o = t >= tp;
                const int key = first_key(t);
                sk.load((o ? ok : pk) + (size_t)key * D, (o ? it.o1 : it.p1) - key, wave, col, half);
            };
            auto load_v = [&](int t) {
                const bool o = t >= tp;
                const int key = first_key(t);
                sv.load((o ? ov : pv) + (size_t)key * D, (o ? it.o1 : it.p1) - key, wave, col, half);
            };
            b16x8 *const kat = sk.place(lds.tile, wave, lane);
            b16x4 *const vat = sv.place(lds.tile, wave, lane);
            load_k(0);
            load_v(0);
            st.begin(a.q + row_at(r), a.scale, half, &lds.third[S::QP < 3 ? wave : 0][0][lane]);
#pragma unroll
            for (int i = 0; i < sk.UNITS; i++) sk.store(i, kat, wave);
            load_k(min(1, tiles - 1));  // past the last tile the last one again: no one reads it
            __syncthreads();
            // a tile for this wave; MASK: some of its keys are past the end or hidden from some rows
            auto tile = [&](auto mask, int t, int tile0, int seen, bool second) {
                constexpr bool MASK = decltype(mask)::value;
                f32x16 s[KT / 32];
                {
                    // one group: an operand's products, the next operand's read, a share of the split
                    constexpr int G = S::KF;
                    Parts<S::KP> x = read(lds.tile.k, 0, lane), y;
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        if (g + 1 < G) y = read(lds.tile.k, g + 1, lane);
                        if (g % KS == 0) s[g / KS] = f32x16{};
                        s[g / KS] = product(x, st.query(g % KS), s[g / KS]);
#pragma unroll
                        for (int i = g * sv.UNITS / G; i < (g + 1) * sv.UNITS / G; i++) sv.store(i, vat);
                        x = y;
                    }
                }
                load_v(min(t + 1, tiles - 1));
                __syncthreads();
                constexpr int G = 2 * NB, UNITS = sk.UNITS * 32 / KT;  // of a 32-key part
#pragma unroll
                for (int sub = 0; sub < KT / 32; sub++) {
                    if (MASK && sub > 0 && !second) {  // no key of it is seen
#pragma unroll
                        for (int i = 0; i < UNITS; i++) sk.store(sub * UNITS + i, kat, wave);
                        break;
                    }
                    Parts<S::KP> x = read(lds.tile.v, sub * G, lane), y;
                    st.template scores<MASK>(s[sub], tile0 + 32 * sub, half, seen);
                    Parts<3> w8[2];
#pragma unroll
                    for (int j = 0; j < 8; j += 2) st.weight2(s[sub], w8[0], 0, j);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        if (g + 1 < G) y = read(lds.tile.v, sub * G + g + 1, lane);
                        st.o[g % NB] = product(x, w8[g / NB], st.o[g % NB]);
                        if (g < NB)
#pragma unroll
                            for (int j = g * 4 / NB; j < (g + 1) * 4 / NB; j++) st.weight2(s[sub], w8[1], 1, 2 * j);
#pragma unroll
                        for (int i = g * UNITS / G; i < (g + 1) * UNITS / G; i++) sk.store(sub * UNITS + i, kat, wave);
                        x = y;
                    }
                }
                load_k(min(t + 2, tiles - 1));
                __syncthreads();
            };
            // One loop after the other, so that O stays where it is: of the prefix and then of the
            // own keys the tiles that all rows of the wave see whole, those that they see in
            // part, and last the tiles that the other waves still need.
            int t = 0;
            for (int part = 0; part < 2; part++) {
                const int begin = part ? it.o0 : it.p0, end = part ? it.o1 : it.p1;
                // keys that every row sees, and that any row does
                const int all = max(0, (part ? min(end, first_last + 1) : end) - begin);
                const int any = max(0, (part ? min(end, end_last + 1) : end) - begin);
                if (nr <= 0) break;
                const int t0 = t;
                for (const int stop = t0 + all / KT; t < stop; t++) tile(std::false_type{}, t, 0, 0, true);
                for (const int stop = t0 + (any + KT - 1) / KT; t < stop; t++)
                    tile(std::true_type{}, t, begin + (t - t0) * KT, part ? min(last, end - 1) : end - 1,
                         any - (t - t0) * KT > 32);
            }
            for (; t < tiles; t++) {
#pragma unroll
                for (int i = 0; i < sv.UNITS; i++) sv.store(i, vat);
                load_v(min(t + 1, tiles - 1));
                __syncthreads();
#pragma unroll
                for (int i = 0; i < sk.UNITS; i++) sk.store(i, kat, wave);
                load_k(min(t + 2, tiles - 1));
                __syncthreads();
            }
            const float sum = st.l + other_half(st.l);
            // 0 though there are keys: their scores left f32 as sums of parts (or are -infinity)
            bool odd = !(fabsf(sum) < INFINITY) || (sum == 0.0f && (it.p1 > it.p0 || last >= it.o0));
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) odd |= !(fabsf(st.o[b][i]) < INFINITY);
            const unsigned long long odds = __ballot(odd && col < nr);
            const unsigned again = (unsigned)odds | (unsigned)(odds >> 32);
            if (col < nr && !(again >> col & 1)) {
                const float f = direct ? 1.0f / sum : 1.0f;
                float *dst = direct ? a.att + row_at(r) : a.po + state_at(r) * D;
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    float x[4 * NB];  // dimensions NB (4 half + 8 g)...
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int b = 0; b < NB; b++) x[NB * i + b] = st.o[b][4 * g + i] * f;
                    if (NB * (4 * half + 8 * g) < D) {
#pragma unroll
                        for (int i = 0; i < 4 * NB; i += 4)
                            *reinterpret_cast<f32x4 *>(dst + NB * (4 * half + 8 * g) + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
                    }
                }
                if (!direct && half == 0) {
                    a.pm[state_at(r)] = st.m;
                    a.pl[state_at(r)] = sum;
                }
            }
            for (int i = 0; i < 32; i++)
                if (again >> i & 1) redo(r0 + i);
            return;
        }

        {
            const int c = lane & 15, quad = lane >> 4, r = min(c, it.nrows - 1);
            const int last = last_of(r), first_last = last_of(0);
            // this wave's tiles: every fourth 32 keys of the prefix, then of the own keys
            const int np = max(0, (it.p1 - it.p0 - 32 * wave + 127) / 128);
            const int tiles = np + max(0, (it.o1 - it.o0 - 32 * wave + 127) / 128);
            auto first_key = [&](int t) { return 32 * wave + (t < np ? it.p0 + 128 * t : it.o0 + 128 * (t - np)); };
            Few<D, T> st;
            // a step's values are requested before its scores are summed, the next step's keys before
            // its weights are taken.  Both a whole step ahead, where there are registers for it, took
            // 12.9 us against 13.4 for 16 tokens over a prefix of 4001, but 9.05 against 8.6 for 4
            // over 1025 and 4.95 against 4.7 for three short prompts.
            auto load_k = [&](int t) {
                const int key = first_key(t);
                st.load_k((t < np ? pk : ok) + (size_t)key * D, (t < np ? it.p1 : it.o1) - key, c, quad);
            };
            if (tiles > 0) load_k(0);
            st.begin(a.q + row_at(r), a.scale, quad);
            for (int t = 0; t < tiles; t++) {
                const bool o = t >= np;
                const int key0 = first_key(t), end = o ? it.o1 : it.p1;
                st.load_v((o ? ov : pv) + (size_t)key0 * D, end - key0, c, quad);
                f32x4 s[2];
                st.scores(s);
                if (t + 1 < tiles) load_k(t + 1);
                st.values(s, key0 + 32 > end || (o && key0 + 31 > first_last),
                          (o ? min(last, end - 1) : end - 1) - key0 - 4 * quad);
            }
            const float l = rows_sum(st.l);
            // join the waves' states: O by row through LDS
            Join<D> &j = lds.join;
            if (quad == 0) {
                j.m[wave][c] = st.m;
                j.l[wave][c] = l;
            }
            if (tid < kBatchRows) j.redo[tid] = 0;
            constexpr int NB16 = S::NB16;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int b = 0; b < NB16; b++) j.o[wave][c][NB16 * (4 * quad + i) + b] = st.o[b][i];
        }
        Join<D> &j = lds.join;
        __syncthreads();
        // 16 threads a row, D / 16 dimensions each
        constexpr int E = D / 16;
        const int row = tid >> 4, d0 = (tid & 15) * E;
        float to = j.m[0][row];
#pragma unroll
        for (int i = 1; i < 4; i++) to = fmaxf(to, j.m[i][row]);
        float sum = 0.0f, acc[E];
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float f = __builtin_amdgcn_exp2f(j.m[i][row] - to);
            sum += f * j.l[i][row];
#pragma unroll
            for (int e = 0; e < E; e++) acc[e] += f * j.o[i][row][d0 + e];
        }
        bool odd = !(fabsf(sum) < INFINITY);
        if (__any(sum == 0.0f)) odd |= sum == 0.0f && (it.p1 > it.p0 || last_of(row) >= it.o0);
#pragma unroll
        for (int e = 0; e < E; e++) odd |= !(fabsf(acc[e]) < INFINITY);
        if (odd && row < it.nrows) j.redo[row] = 1;
        __syncthreads();
        if (row < it.nrows && !j.redo[row]) {
            const float f = direct ? 1.0f / sum : 1.0f;
            float *dst = direct ? a.att + row_at(row) + d0 : a.po + state_at(row) * D + d0;
            if (!direct && d0 == 0) {
                a.pm[state_at(row)] = to;
                a.pl[state_at(row)] = sum;
            }
#pragma unroll
            for (int e = 0; e < E; e++) dst[e] = acc[e] * f;
        }
        for (int i = wave; i < it.nrows; i += 4)
            if (j.redo[i]) redo(i);
    }
}

// State c of a row.  base: state row 0 of the row's kv head, and the head in the group.
__device__ __forceinline__ size_t state_of(const BatchToken &t, size_t base, int prefix_chunks, int stride, int c) {
    return base + (c < prefix_chunks ? t.prefix_state + (size_t)c * stride
                                     : t.own_state + (size_t)(c - prefix_chunks) * t.own_stride);
}

// The running sums of a row's states c = first, first + G, ...: `B` of them on their way at a time.
template <int D, int G, int B>
__device__ __forceinline__ void join_states(const BatchArgs &a, const BatchToken &t, size_t base, int prefix_chunks,
                                            int stride, int first, int n, int d, float &m, float &l, f32x4 &acc) {
    for (int c0 = first; c0 < n; c0 += B * G) {
        f32x4 o[B];
        float mm[B], ll[B], top = m;
#pragma unroll
        for (int b = 0; b < B; b++) {
            const size_t at = state_of(t, base, prefix_chunks, stride, min(c0 + b * G, n - 1));
            o[b] = *reinterpret_cast<const f32x4 *>(a.po + at * D + d);
            mm[b] = a.pm[at];
            ll[b] = a.pl[at];
        }
#pragma unroll
        for (int b = 0; b < B; b++) top = fmaxf(top, mm[b]);
        const float old = exp2f(m - top);
        l *= old;
        acc *= old;
        m = top;
#pragma unroll
        for (int b = 0; b < B; b++)
            if (c0 + b * G < n) {
                const float f = exp2f(mm[b] - top);
                l += f * fabsf(ll[b]);
                acc += (ll[b] < 0.0f ? f / kLow : f) * o[b];
            }
    }
}

// The values of a row's `mean` again whose sum overflowed, from sums at 2^-32, state after state.
__device__ __forceinline__ f32x4 join_low(const BatchArgs &a, const BatchToken &t, size_t base, int prefix_chunks,
                                          int stride, int n, int D, int d, f32x4 sum, f32x4 mean) {
    float top = kNoMax, l = 0.0f;
    f32x4 low{};
    for (int c = 0; c < n; c++) top = fmaxf(top, a.pm[state_of(t, base, prefix_chunks, stride, c)]);
    for (int c = 0; c < n; c++) {
        const size_t at = state_of(t, base, prefix_chunks, stride, c);
        const float f = exp2f(a.pm[at] - top), ll = a.pl[at];
        l += f * kLow * fabsf(ll);
        low += (ll < 0.0f ? f : f * kLow) * *reinterpret_cast<const f32x4 *>(a.po + at * D + d);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) mean[e] = mean_of(sum[e], mean[e], low[e], l);
    return mean;
}
__device__ __forceinline__ bool finite(f32x4 x) {
    return fabsf(x[0]) < INFINITY && fabsf(x[1]) < INFINITY && fabsf(x[2]) < INFINITY && fabsf(x[3]) < INFINITY;
}

// W waves join one row's states: with the largest m, weights 2^(m_i - m), att = sum w O /
// sum w l.  D / 4 lanes read a state, 8 states in flight each; their running sums are
// joined last, always in the same order.  Bound by the states' reads and its own launch: 1024 rows of
// 28 states of 128 dimensions 7.6 us (one state after the other, as the first version read them, 19).
// Four waves where one would need several rounds of its 8: there 72.5 us a step against 74.4 with one.
template <int D, int W>
__global__ __launch_bounds__(256) void batch_merge_kernel(BatchArgs a) {
    constexpr int L = D / 4, G = 64 * W / L, B = 8;  // lanes of a state, states at once, and on their way
    __shared__ float part[W > 1 ? W : 1][D + 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = 4 * (lane % L);
    const int g = (W > 1 ? wave * (64 / L) : 0) + lane / L;
    const int heads = a.group * a.kv_heads;
    if (!fits(a)) return;
    const int work = a.head->merges * heads, prefix_chunks = a.head->prefix_chunks, stride = a.head->prefix_stride;
    constexpr int R = 4 / W;  // rows of a workgroup
    for (int w = blockIdx.x * R + (W > 1 ? 0 : wave); w < work; w += gridDim.x * R) {
        const int i = divide(w, heads, a.inv_heads), head = w - i * heads, kh = divide(head, a.group, a.inv_group),
                  h = head - kh * a.group;
        const BatchToken t = a.tokens[i];
        const size_t base = (size_t)kh * a.state_rows + h;
        const int n = prefix_chunks + t.own_chunks;
        float m = kNoMax, l = 0.0f;
        f32x4 acc{};
        join_states<D, G, B>(a, t, base, prefix_chunks, stride, g, n, d, m, l, acc);
        float top = m;
#pragma unroll
        for (int x = L; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        float f = exp2f(m - top);
        l *= f;
        acc *= f;
#pragma unroll
        for (int x = L; x < 64; x <<= 1) {
            l += __shfl_xor(l, x, 64);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], x, 64);
        }
        if constexpr (W > 1) {
            if (lane < L) {
#pragma unroll
                for (int e = 0; e < 4; e++) part[wave][d + e] = acc[e];
                if (lane == 0) {
                    part[wave][D] = top;
                    part[wave][D + 1] = l;
                }
            }
            __syncthreads();
            float all = part[0][D];
#pragma unroll
            for (int x = 1; x < W; x++) all = fmaxf(all, part[x][D]);
            l = 0.0f;
            acc = f32x4{};
#pragma unroll
            for (int x = 0; x < W; x++) {
                f = exp2f(part[x][D] - all);
                l += f * part[x][D + 1];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[e] += f * part[x][d + e];
            }
            __syncthreads();
        }
        if (lane < L && (W == 1 || wave == 0)) {
            f32x4 y = acc * (1.0f / l);
            if (!finite(acc)) y = join_low(a, t, base, prefix_chunks, stride, n, D, d, acc, y);
            *reinterpret_cast<f32x4 *>(a.att + ((size_t)t.merge * heads + head) * D + d) = y;
        }
    }
}

// The same for few states: D / 4 lanes have a row, 4 states in flight, nothing to join across lanes.
// 16 prompts of 12..161 tokens behind a prefix of 1500 (20 thousand rows) 102.4 us a step, 106.8
// with a wave a row; 4 tokens over 300 (36 rows) 8.1 and 8.6; but 16 tokens of 14 states 14.5 and 13.4.
template <int D>
__global__ __launch_bounds__(256) void batch_merge_rows_kernel(BatchArgs a) {
    constexpr int L = D / 4, R = 256 / L;  // lanes of a row, rows of a workgroup
    const int d = 4 * (threadIdx.x % L), heads = a.group * a.kv_heads;
    if (!fits(a)) return;
    const int work = a.head->merges * heads, prefix_chunks = a.head->prefix_chunks, stride = a.head->prefix_stride;
    for (int w = blockIdx.x * R + threadIdx.x / L; w < work; w += gridDim.x * R) {
        const int i = divide(w, heads, a.inv_heads), head = w - i * heads, kh = divide(head, a.group, a.inv_group);
        const BatchToken t = a.tokens[i];
        const size_t base = (size_t)kh * a.state_rows + (head - kh * a.group);
        const int n = prefix_chunks + t.own_chunks;
        float m = kNoMax, l = 0.0f;
        f32x4 acc{};
        join_states<D, 1, 4>(a, t, base, prefix_chunks, stride, 0, n, d, m, l, acc);
        f32x4 y = acc * (1.0f / l);
        if (!finite(acc)) y = join_low(a, t, base, prefix_chunks, stride, n, D, d, acc, y);
        *reinterpret_cast<f32x4 *>(a.att + ((size_t)t.merge * heads + head) * D + d) = y;
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
    long long rows;
    hipStream_t s;
    template <int D, class T>
    hipError_t operator()() {
        if (a.max_states <= 8)
            batch_merge_rows_kernel<D><<<(int)std::min<long long>(1 << 20, (rows + 1024 / D - 1) / (1024 / D)), 256, 0, s>>>(a);
        else if (a.max_states > 256 / D * 8)  // one wave's round
            batch_merge_kernel<D, 4><<<(int)std::min<long long>(1 << 20, rows), 256, 0, s>>>(a);
        else
            batch_merge_kernel<D, 1><<<(int)std::min<long long>(1 << 20, (rows + 3) / 4), 256, 0, s>>>(a);
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

}  // namespace

hipError_t launch_batch_attend(int head_dim, int bf16, const BatchArgs &a, int grid, hipStream_t s) {
    return dispatch(head_dim, bf16, AttendLaunch{a, grid, s});
}
hipError_t launch_batch_merge(int head_dim, const BatchArgs &a, int merges, hipStream_t s) {
    return dispatch(head_dim, 0, MergeLaunch{a, (long long)merges * a.group * a.kv_heads, s});
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

}  // namespace wick

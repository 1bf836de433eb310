// batch_plan.h -- how a batch's step is cut into workgroups (host code, no HIP).
//
// A row is one (token, query head of a kv head's group) pair, numbered token * group +
// head over the packed tokens; every kv head has the same rows and the same cut.  An
// item is one workgroup's work for each kv head: a block of rows against a range of the
// prefix's keys and a range of its sequence's own keys.
//   whole items   rows of one sequence against all the keys that they see; att is
//                 written directly.  For sequences with many rows, where such items
//                 alone fill the GPU.
//   split items   the keys dealt to several items, each leaving partial states
//                 (m, l, O) that a second launch joins.  The rows of all split
//                 sequences together go against the prefix (a block's rows read a
//                 prefix key once for all of its sequences), each sequence's rows
//                 against its own keys.
#pragma once

#include <algorithm>
#include <climits>
#include <cstdint>
#include <vector>

namespace wick {

constexpr int kBatchRows = 32;   // rows of an item
constexpr int kBatchStep = 128;  // keys a workgroup takes at a time: 4 waves x 32

// One workgroup's work (device layout).
struct BatchItem {
    int row0, nrows;   // rows [row0, row0 + nrows): of the packed tokens (seq >= 0) or of
                       // the split tokens (seq < 0, found through BatchToken::split)
    int seq;           // sequence of the own keys; -1: prefix keys only
    int p0, p1;        // prefix keys
    int o0, o1;        // own keys; row r sees those up to r / group + shift
    int shift;
    int state0;        // first state row; -1: the rows' att is written
    int pad[7];
};
static_assert(sizeof(BatchItem) == 64, "one cache line each");

// Device layout: entry i < total says where packed token i goes; entry i < splits
// describes split token i; entry i < merges describes joined token i.
struct BatchToken {
    int seq, pos;       // the token's place in the caches
    int split;          // the packed token of split token i
    int merge;          // the packed token of joined token i
    int prefix_state;   // its rows' first state row against the prefix, chunk 0
    int own_state;      // its rows' first state row against its own keys, chunk 0
    int own_stride;     // state rows from one own chunk to the next
    int own_chunks;
};
static_assert(sizeof(BatchToken) == 32, "");

struct BatchHeader {
    int shape;           // wick_hip_batch_shape()
    int items, total, merges;
    int prefix_chunks, prefix_stride;  // state rows from one prefix chunk to the next
    int pad[10];
};
static_assert(sizeof(BatchHeader) == 64, "");

// What a handle was made for.
struct BatchLimits {
    int group, kv_heads, sequences, capacity, prefix_capacity, max_tokens;
    int workgroups;  // resident at once
};

// Most items and state rows (per kv head) of any plan.  Split sequences have together at
// most `workgroups` blocks of whole rows over all kv heads (with more they are whole) and one
// ragged block each; their items are at most `workgroups` over all kv heads, or a block against
// the prefix and one against its own keys where that is more.
inline int64_t batch_max_items(const BatchLimits &c) {
    const int64_t rows = (int64_t)c.max_tokens * c.group;
    return 2 * (rows / kBatchRows + std::min(c.sequences, c.max_tokens) + 1) + c.workgroups / c.kv_heads + 1;
}
inline int64_t batch_max_state_rows(const BatchLimits &c) {
    const int64_t rows = (int64_t)c.max_tokens * c.group, few = std::min(c.sequences, c.max_tokens);
    const int64_t blocks = std::min(rows / kBatchRows, (int64_t)c.workgroups / c.kv_heads + few) + few + 1;
    return (2 * blocks + c.workgroups / c.kv_heads + 1) * kBatchRows;
}

struct BatchPlan {
    BatchHeader head{};
    std::vector<BatchItem> items;
    std::vector<BatchToken> tokens;  // [total]
    int64_t state_rows = 0;
};

inline int batch_blocks(int64_t rows) { return (int)((rows + kBatchRows - 1) / kBatchRows); }

// The plan of a step; start and t as wick_hip_batch_plan has them, already checked.
inline BatchPlan batch_plan(const BatchLimits &c, const int *start, const int *t, int prefix) {
    BatchPlan p;
    int total = 0;
    for (int s = 0; s < c.sequences; s++) total += t[s];
    p.head.total = total;
    p.tokens.assign(total, BatchToken{});
    int64_t whole_blocks = 0;
    for (int s = 0; s < c.sequences; s++) {
        const int64_t rows = (int64_t)t[s] * c.group;
        if (rows >= kBatchRows) whole_blocks += batch_blocks(rows);
    }
    const bool wholes = whole_blocks * c.kv_heads >= c.workgroups;
    auto whole = [&](int s) { return wholes && (int64_t)t[s] * c.group >= kBatchRows; };

    // the split rows, and the shortest key range per item that keeps them within the
    // resident workgroups
    int splits = 0, longest = prefix;
    for (int s = 0; s < c.sequences; s++)
        if (!whole(s) && t[s] > 0) {
            splits += t[s];
            longest = std::max(longest, start[s] + t[s]);
        }
    const int64_t split_rows = (int64_t)splits * c.group;
    auto chunks = [](int keys, int len) { return (keys + len - 1) / len; };
    auto count = [&](int len) {
        int64_t n = prefix ? (int64_t)batch_blocks(split_rows) * chunks(prefix, len) : 0;
        for (int s = 0; s < c.sequences; s++)
            if (!whole(s) && t[s] > 0)
                n += (int64_t)batch_blocks((int64_t)t[s] * c.group) * chunks(start[s] + t[s], len);
        return n;
    };
    const int64_t most = std::max(1, c.workgroups / c.kv_heads);
    int lo = 1, hi = std::max(1, chunks(longest, kBatchStep));  // in steps
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (count(mid * kBatchStep) <= most)
            hi = mid;
        else
            lo = mid + 1;
    }
    const int len = lo * kBatchStep;

    auto even = [&](int keys, int n) {  // n ranges over keys, in steps
        return chunks(chunks(keys, n), kBatchStep) * kBatchStep;
    };
    if (prefix && splits) {
        const int part = even(prefix, chunks(prefix, len)), n = chunks(prefix, part);
        p.head.prefix_chunks = n;
        p.head.prefix_stride = (int)split_rows;
        for (int k = 0; k < n; k++)
            for (int64_t r = 0; r < split_rows; r += kBatchRows) {
                BatchItem it{};
                it.row0 = (int)r;
                it.nrows = (int)std::min<int64_t>(kBatchRows, split_rows - r);
                it.seq = -1;
                it.p0 = k * part;
                it.p1 = std::min(prefix, it.p0 + part);
                it.state0 = (int)(p.state_rows + r);
                p.items.push_back(it);
                if (r + kBatchRows >= split_rows) p.state_rows += split_rows;
            }
    }
    int token = 0, split = 0;
    for (int s = 0; s < c.sequences; s++) {
        for (int i = 0; i < t[s]; i++) {
            p.tokens[token + i].seq = s;
            p.tokens[token + i].pos = start[s] + i;
        }
        const int keys = start[s] + t[s], rows = t[s] * c.group, shift = start[s] - token;
        const int64_t row0 = (int64_t)token * c.group;
        auto block = [&](int r, int o0, int o1, int64_t state0, int p1) {
            BatchItem it{};
            it.row0 = (int)(row0 + r);
            it.nrows = std::min(kBatchRows, rows - r);
            it.seq = s;
            it.p1 = p1;
            it.o0 = o0;
            // no key past the last one that the block's last row sees
            it.o1 = std::min(o1, (int)((row0 + r + it.nrows - 1) / c.group) + shift + 1);
            it.o1 = std::max(it.o0, it.o1);
            it.shift = shift;
            it.state0 = (int)state0;
            p.items.push_back(it);
        };
        if (t[s] > 0 && whole(s)) {
            for (int r = 0; r < rows; r += kBatchRows) block(r, 0, keys, -1, prefix);
        } else if (t[s] > 0) {
            const int part = even(keys, chunks(keys, len)), n = chunks(keys, part);
            const bool direct = n == 1 && !prefix;
            for (int i = 0; i < t[s] && !direct; i++) {
                BatchToken &m = p.tokens[split];
                m.split = m.merge = token + i;
                m.prefix_state = split * c.group;
                m.own_state = (int)(p.state_rows + (int64_t)i * c.group);
                m.own_stride = rows;
                m.own_chunks = n;
                split++;
            }
            for (int k = 0; k < n; k++) {
                for (int r = 0; r < rows; r += kBatchRows)
                    block(r, k * part, std::min(keys, (k + 1) * part), direct ? -1 : p.state_rows + r, 0);
                if (!direct) p.state_rows += rows;
            }
        }
        token += t[s];
    }
    p.head.merges = split;
    // the longest items first
    std::stable_sort(p.items.begin(), p.items.end(), [](const BatchItem &a, const BatchItem &b) {
        const int x = a.p1 - a.p0 + a.o1 - a.o0, y = b.p1 - b.p0 + b.o1 - b.o0;
        return x / kBatchStep > y / kBatchStep;
    });
    p.head.items = (int)p.items.size();
    return p;
}

}  // namespace wick

// batch_plan.h -- how a batch's step is cut into workgroups (host code, no HIP).
//
// A row is one (token, query head of a kv head's group) pair, numbered token * group +
// head over the packed tokens; every kv head has the same rows and the same cut.  An
// item is one workgroup's work for each kv head: a block of rows against a range of the
// prefix's keys and a range of its sequence's own keys.  A block of up to 16 rows is
// narrow (the four waves share the keys), one of up to 128 wide (the waves share the rows).
//   whole items   rows of one sequence against all the keys that they see; att is
//                 written directly.
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

constexpr int kBatchRows = 16;   // rows of a narrow item
constexpr int kBatchWide = 128;  // rows of a wide item: 4 waves x 32
constexpr int kBatchStep = 128;  // keys a narrow item takes at a time: 4 waves x 32
constexpr int kBatchFew = 48;    // rows up to which narrow items share them
constexpr int kBatchBig = 64;    // rows from which a sequence is a candidate for whole items

// One workgroup's work (device layout).
struct BatchItem {
    int row0, nrows;   // rows [row0, row0 + nrows): of the packed tokens (seq >= 0) or of
                       // the split tokens (seq < 0, found through BatchToken::split)
    int seq;           // sequence of the own keys; -1: prefix keys only, split token i is packed
                       // token i + shift; -2: prefix keys only, it is BatchToken::split of i
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
    int max_states;                    // most states of a row
    int most_items;                    // of any plan for the same t
    int pad[8];
};
static_assert(sizeof(BatchHeader) == 64, "");

// What a handle was made for.
struct BatchLimits {
    int group, kv_heads, sequences, capacity, prefix_capacity, max_tokens;
    int cus;  // the GPU's compute units
};

// Most items and state rows (per kv head) of any plan.  A sequence of kBatchBig rows or more
// is split only where its longest item would cost twice the target, which the sum of its
// items' costs (half the longest each, or more) allows for cus / kv_heads blocks
// together; the others have less than kBatchBig rows each.
inline int64_t batch_max_items(const BatchLimits &c) {
    const int64_t rows = (int64_t)c.max_tokens * c.group;
    return 2 * (rows / kBatchRows + std::min(c.sequences, c.max_tokens) + 1) + c.cus / c.kv_heads + 1;
}
inline int64_t batch_max_state_rows(const BatchLimits &c) {
    const int64_t rows = (int64_t)c.max_tokens * c.group, few = std::min(c.sequences, c.max_tokens);
    const int64_t slots = c.cus / c.kv_heads + 1;
    const int64_t split = std::min(rows, kBatchWide * slots + (kBatchBig + kBatchWide) * few);
    return 2 * kBatchWide * slots + 2 * split + 2 * kBatchWide;
}

struct BatchPlan {
    BatchHeader head{};
    std::vector<BatchItem> items;
    std::vector<BatchToken> tokens;  // [total]
    int64_t state_rows = 0;
};

constexpr double kPlanItem = 2.0;       // an item's cost besides its keys'
constexpr double kPlanWhole = 2.0;      // targets that a whole item may cost
constexpr double kPlanLeastWide = 4.0;  // least cost of a range of keys
constexpr double kPlanLeastNarrow = 1.0;
constexpr double kPlanShare = 1.0;      // compute units' shares of the sum that the target is one of

// Cost of a block of `rows` rows against `keys` keys, in tiles of a wave: a wide item's waves
// all take every 32 keys, a narrow one's every fourth; and what an item costs besides.
inline double batch_cost(int64_t rows, int64_t keys) {
    return keys / (rows > kBatchRows ? 32.0 : 128.0);
}
// Rows of a block where `rows` are cut into blocks.
inline int batch_block(int64_t rows) { return rows <= kBatchFew ? kBatchRows : kBatchWide; }

// The plan of a step; start and t as wick_hip_batch_plan has them, already checked.
inline BatchPlan batch_plan(const BatchLimits &c, const int *start, const int *t, int prefix) {
    BatchPlan p;
    int total = 0;
    for (int s = 0; s < c.sequences; s++) total += t[s];
    p.head.total = total;
    p.tokens.assign(total, BatchToken{});
    auto rows_of = [&](int s) { return (int64_t)t[s] * c.group; };
    auto blocks = [](int64_t rows) { return (rows + batch_block(rows) - 1) / batch_block(rows); };
    auto big = [&](int s) { return rows_of(s) >= kBatchBig; };

    // what all items cost together, the big sequences in whole ones; the target is a
    // compute unit's share
    double sum = 0.0;
    int64_t small_rows = 0;
    for (int s = 0; s < c.sequences; s++) {
        const int64_t rows = rows_of(s);
        if (big(s)) {
            const double keys = (double)prefix + start[s] + 0.5 * t[s];
            sum += blocks(rows) * (keys / 32.0 + kPlanItem);
        } else if (rows) {
            sum += blocks(rows) * (batch_cost(batch_block(rows), start[s] + t[s]) + kPlanItem);
            small_rows += rows;
        }
    }
    if (prefix && small_rows) sum += blocks(small_rows) * (batch_cost(batch_block(small_rows), prefix) + kPlanItem);
    // no plan of the same t has more items: a block's ranges are at most its cost over the
    // target and one more, the last rows' excess over the average another one
    int64_t base = 0;
    for (int s = 0; s < c.sequences; s++) base += 2 * blocks(rows_of(s)) + 1;
    p.head.most_items = (int)std::min<int64_t>(batch_max_items(c), c.cus / c.kv_heads + 1 + 2 * base);
    const double target = sum * c.kv_heads / (c.cus * kPlanShare);
    auto whole = [&](int s) { return big(s) && batch_cost(kBatchWide, (int64_t)prefix + start[s] + t[s]) <= kPlanWhole * target; };

    // n even ranges over the keys of a block of `rows` rows, each near the target, in steps
    auto range = [&](int64_t rows, int keys) {
        const bool wide = batch_block(rows) == kBatchWide;
        const double least = wide ? kPlanLeastWide : kPlanLeastNarrow;
        const int n = std::max(1, (int)(batch_cost(batch_block(rows), keys) / std::max(target, least) + 0.999));
        const int part = (keys + n - 1) / n;
        const int step = wide ? 32 : kBatchStep;
        return (part + step - 1) / step * step;
    };
    auto chunks = [](int keys, int len) { return (keys + len - 1) / len; };

    int64_t split_rows = 0;
    std::vector<int> split_token;
    for (int s = 0, token = 0; s < c.sequences; token += t[s++])
        if (!whole(s)) {
            split_rows += rows_of(s);
            for (int i = 0; i < t[s]; i++) split_token.push_back(token + i);
        }
    if (prefix && split_rows) {
        const int part = range(split_rows, prefix), n = chunks(prefix, part), step = batch_block(split_rows);
        p.head.prefix_chunks = n;
        p.head.prefix_stride = (int)split_rows;
        for (int k = 0; k < n; k++) {
            for (int64_t r = 0; r < split_rows; r += step) {
                BatchItem it{};
                it.row0 = (int)r;
                it.nrows = (int)std::min<int64_t>(step, split_rows - r);
                const int first = (int)(r / c.group), end = (int)((r + it.nrows - 1) / c.group);
                it.shift = split_token[first] - first;
                it.seq = split_token[end] - end == it.shift ? -1 : -2;  // they ascend
                it.p0 = k * part;
                it.p1 = std::min(prefix, it.p0 + part);
                it.state0 = (int)(p.state_rows + r);
                p.items.push_back(it);
            }
            p.state_rows += split_rows;
        }
    }
    int token = 0, split = 0;
    for (int s = 0; s < c.sequences; s++) {
        for (int i = 0; i < t[s]; i++) {
            p.tokens[token + i].seq = s;
            p.tokens[token + i].pos = start[s] + i;
        }
        const int keys = start[s] + t[s], rows = (int)rows_of(s), shift = start[s] - token;
        const int64_t row0 = (int64_t)token * c.group;
        const int step = batch_block(rows);
        // rows [r, r + step) against own keys [o0, o1), as far as the last row sees them
        auto block = [&](int r, int o0, int o1, int64_t state0, int p1) {
            BatchItem it{};
            it.row0 = (int)(row0 + r);
            it.nrows = std::min(step, rows - r);
            it.seq = s;
            it.p1 = p1;
            it.o0 = o0;
            it.o1 = std::min(o1, (int)((row0 + r + it.nrows - 1) / c.group) + shift + 1);
            it.shift = shift;
            it.state0 = (int)state0;
            if (it.o1 > it.o0) p.items.push_back(it);
        };
        if (rows && whole(s)) {
            for (int r = 0; r < rows; r += step) block(r, 0, keys, -1, prefix);
        } else if (rows) {
            const int part = range(rows, keys), n = chunks(keys, part);
            const bool direct = n == 1 && !prefix;
            for (int i = 0; i < t[s] && !direct; i++) {
                BatchToken &m = p.tokens[split];
                m.split = m.merge = token + i;
                m.prefix_state = split * c.group;
                m.own_state = (int)(p.state_rows + (int64_t)i * c.group);
                m.own_stride = rows;
                m.own_chunks = (start[s] + i) / part + 1;  // those in which it sees a key
                p.head.max_states = std::max(p.head.max_states, p.head.prefix_chunks + m.own_chunks);
                split++;
            }
            for (int k = 0; k < n; k++) {
                for (int r = 0; r < rows; r += step)
                    block(r, k * part, std::min(keys, (k + 1) * part), direct ? -1 : p.state_rows + r, 0);
                if (!direct) p.state_rows += rows;
            }
        }
        token += t[s];
    }
    p.head.merges = split;
    // the costliest items first
    std::stable_sort(p.items.begin(), p.items.end(), [](const BatchItem &a, const BatchItem &b) {
        const auto cost = [](const BatchItem &x) {
            return (int)batch_cost(x.nrows, (int64_t)x.p1 - x.p0 + x.o1 - x.o0);
        };
        return cost(a) > cost(b);
    });
    p.head.items = (int)p.items.size();
    return p;
}

}  // namespace wick

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
// Rows up to which narrow items share them.  Of a sequence: 64 rows (32/4 heads of 64) over 16000
// keys 20.8 us, as one wide item 24.1; 96 rows 30.3, as a wide one 26.9.
constexpr int kBatchFew = 64;
// Of several sequences against the prefix: narrow items each split f32 keys into parts again.  48 rows
// (32/8 heads of 128) over a prefix of 32768 103 us, as a wide item 81; 33 to 64 rows over 8000 to
// 24000 take from 3% less to 17% more as narrow ones.  A bf16 cache's keys need no split: 64 rows over
// 16000 30.4 us, as a wide item 35.5.
inline int batch_few(bool bf16) { return bf16 ? 64 : 32; }

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
    int few;  // batch_few() of the cache's type
};

// Most items and state rows (per kv head) of any plan.  The cut prices every block in the shape it
// is cut in, and a range costs the target or more, so the ranges of all blocks are at most their
// costs over the target -- 2 cus / kv_heads together, or half of that without wide blocks -- and one
// more a block.  Two more where a wide block's own keys end inside a range, which the average of
// its rows' keys also prices half a range too low.  Blocks: a sequence of r rows has up to r / 16 + 1
// of its own (wide ones an eighth of that), all split rows together up to r / 16 + 1 against the prefix.
// A big sequence is split only where its longest item costs more than 1 / kPlanLone
// of a unit's share, and its items cost half the longest each or more, so that the split
// ones have at most 2.6 cus / kv_heads blocks together; steps without wide blocks have fewer
// than 2 cus / kv_heads of them; other sequences have up to kBatchFew rows.
inline int64_t batch_max_items(const BatchLimits &c) {
    const int64_t rows = (int64_t)c.max_tokens * c.group;
    return 2 * (rows / kBatchRows + std::min(c.sequences, c.max_tokens) + 1) + 2 * c.cus / c.kv_heads + 1;
}
inline int64_t batch_max_state_rows(const BatchLimits &c) {
    const int64_t rows = (int64_t)c.max_tokens * c.group, few = std::min(c.sequences, c.max_tokens);
    const int64_t slots = c.cus / c.kv_heads + 1;
    const int64_t split = std::min(rows, 3 * kBatchWide * slots + (kBatchFew + kBatchWide) * few);
    // the least range is kBatchStep keys for either kind of block (kPlanLeastWide, kPlanLeastNarrow)
    auto ranges_of = [](int64_t keys) { return (keys + kBatchStep - 1) / kBatchStep; };
    const int64_t ranges = ranges_of(c.prefix_capacity) + ranges_of(c.capacity);
    return std::min(6 * kBatchWide * slots + 2 * split + 2 * kBatchWide, rows * ranges);
}

struct BatchPlan {
    BatchHeader head{};
    std::vector<BatchItem> items;
    std::vector<BatchToken> tokens;  // [total]
    int64_t state_rows = 0;
};

// The constants of the plan, in tiles of 32 keys by a wide item (about 2 us at head_dim 128).
constexpr double kPlanItem = 2.0;  // an item's cost besides its keys'
// What leaving states and joining them costs a step, and what a tile of a lone wide item on a
// unit takes against one of two.  16 prompts of 12..161 tokens behind a prefix of 1500 (16/8 heads
// of 128): split 105 us, whole 128; one prompt of 512: 28.3 and 43.7; of 1000 (32/8 of 128) 74 and 79, but
// 56 and 47 on a bf16 cache; of 2000 (14/2 of 64) 62 and 78.  Eight prompts of 33..701 (14/2 of 64) with a
// price of 0, 6, 12 and 18: 38.3, 37.4, 39.9 and 37.1.
constexpr double kPlanJoin = 18.0, kPlanLone = 1.3;
constexpr double kPlanLeastWide = 4.0, kPlanLeastNarrow = 1.0;  // least cost of a range of keys
static_assert(32 * kPlanLeastWide == kBatchStep && 128 * kPlanLeastNarrow == kBatchStep, "batch_max_state_rows counts on it");
// Ranges up to which small sequences are not cut, to save the second launch: four tokens behind a
// prefix of 100 (9/3 heads of 64) 6.8 us, cut 9.0; of 200 8.2 and 9.2; of 300 9.5 and 9.3.
constexpr double kPlanAlone = 1.6;
// Wide items to cut for each compute unit (narrow ones: one): 64 tokens over a prefix of 32768
// (32/8 heads of 128, bf16) 126 us with two, 136 with 1.5, 142 with 2.5.
constexpr double kPlanWideItems = 2.0;

// Cost of a block of `rows` rows against `keys` keys, in tiles of a wave: a wide item's waves
// all take every 32 keys, a narrow one's every fourth; and what an item costs besides.
inline double batch_cost(int64_t rows, int64_t keys) {
    return keys / (rows > kBatchRows ? 32.0 : 128.0);
}

// The plan of a step; start and t as wick_hip_batch_plan has them, already checked.
inline BatchPlan batch_plan(const BatchLimits &c, const int *start, const int *t, int prefix) {
    BatchPlan p;
    int total = 0;
    for (int s = 0; s < c.sequences; s++) total += t[s];
    p.head.total = total;
    p.tokens.assign(total, BatchToken{});
    auto rows_of = [&](int s) { return (int64_t)t[s] * c.group; };
    auto chunks = [](int64_t keys, int64_t len) { return (keys + len - 1) / len; };

    // Narrow blocks for a step that would leave units idle with wide ones, cut as finely as
    // they may be, if one round of narrow ones holds it: 16 tokens over a prefix of 4001 (14/2
    // heads of 64) 12.6 us, 15.2 with wide blocks; one prompt of 512 (16/8 of 128) 25.1 and 29.5; of
    // 1000 (32/8 of 128) 98.7 and 80.8; eight of 50..100 (32/4 of 64) 14.2 and 10.9.
    int64_t most_wide = 0, least_narrow = 0, small_rows = 0;
    for (int s = 0; s < c.sequences; s++) {
        const int64_t rows = rows_of(s), keys = (int64_t)start[s] + t[s];
        least_narrow += chunks(rows, kBatchRows);
        if (rows > kBatchFew)
            most_wide += chunks(rows, kBatchWide) * chunks(prefix + keys, (int64_t)(32 * kPlanLeastWide));
        else
            small_rows += rows;
    }
    if (small_rows > c.few)
        most_wide += chunks(small_rows, kBatchWide) * chunks(prefix, (int64_t)(32 * kPlanLeastWide));
    const bool wides = std::max(most_wide, least_narrow) * c.kv_heads >= 2 * c.cus;
    auto block_of = [&](int64_t rows) { return wides && rows > kBatchFew ? kBatchWide : kBatchRows; };
    auto shared_of = [&](int64_t rows) { return wides && rows > c.few ? kBatchWide : kBatchRows; };  // against the prefix
    auto blocks = [&](int64_t rows) { return chunks(rows, block_of(rows)); };
    auto big = [&](int s) { return block_of(rows_of(s)) == kBatchWide; };

    // what all items cost together, the big sequences in whole ones; a compute unit's share
    // of it is what the step takes at best
    double sum = 0.0;
    // Few keys for every sequence that is not big: each takes all of its own, the prefix
    // again and again, which costs less than the second launch
    double alone_most = 0.0, alone_sum = 0.0;
    // no plan of the same t has more items: a block's ranges are at most its cost over the
    // target and one more, the last rows' excess over the average another one
    int64_t base = 0;
    small_rows = 0;
    for (int s = 0; s < c.sequences; s++) {
        const int64_t rows = rows_of(s);
        if (big(s)) {
            const double keys = (double)prefix + start[s] + 0.5 * t[s];
            sum += blocks(rows) * (keys / 32.0 + kPlanItem);
        } else if (rows) {
            sum += blocks(rows) * (batch_cost(kBatchRows, start[s] + t[s]) + kPlanItem);
            small_rows += rows;
            const double cost = batch_cost(kBatchRows, (int64_t)prefix + start[s] + t[s]);
            alone_most = std::max(alone_most, cost);
            alone_sum += blocks(rows) * (cost + kPlanItem);
        }
        base += 2 * chunks(rows, kBatchRows) + 1;
    }
    // the rows of the sequences that are not big, against the prefix in blocks of this shape
    auto with_shared = [&](int block) {
        return prefix && small_rows ? sum + chunks(small_rows, block) * (batch_cost(block, prefix) + kPlanItem) : sum;
    };
    const double share = with_shared(shared_of(small_rows)) * c.kv_heads / c.cus;
    p.head.most_items = (int)std::min<int64_t>(batch_max_items(c), 2 * c.cus / c.kv_heads + 1 + 2 * base);
    const bool alone = alone_most <= kPlanAlone && alone_sum * c.kv_heads <= kPlanAlone * c.cus;
    auto whole = [&](int s) {
        return big(s) ? kPlanLone * batch_cost(kBatchWide, (int64_t)prefix + start[s] + t[s]) <= share + kPlanJoin : alone;
    };

    int64_t split_rows = 0;
    std::vector<int> split_token;
    for (int s = 0, token = 0; s < c.sequences; token += t[s++])
        if (!whole(s)) {
            split_rows += rows_of(s);
            for (int i = 0; i < t[s]; i++) split_token.push_back(token + i);
        }
    // What a range should cost.  Split big sequences make the blocks of all split rows wide: there the
    // other sequences' few rows add up to a wide block, not the narrow ones of a step of their own.
    const double cut = with_shared(shared_of(alone ? small_rows : split_rows)) * c.kv_heads / c.cus;
    const double target = wides ? cut / kPlanWideItems : cut;

    // n even ranges over the keys of a block, each near the target, in steps
    auto range = [&](int block, int keys) {
        const bool wide = block == kBatchWide;
        const double least = wide ? kPlanLeastWide : kPlanLeastNarrow;
        const int n = std::max(1, (int)(batch_cost(block, keys) / std::max(target, least) + 0.999));
        const int part = (keys + n - 1) / n;
        const int step = wide ? 32 : kBatchStep;
        return (part + step - 1) / step * step;
    };
    if (prefix && split_rows) {
        const int step = shared_of(split_rows), part = range(step, prefix), n = (int)chunks(prefix, part);
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
        const int step = block_of(rows);
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
            const int part = range(step, keys), n = (int)chunks(keys, part);
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

// Checks batch_plan(): every (row, key) pair that a token sees lies in exactly one item, in
// bounds; states of different items do not meet; every joined row's states are those that
// its items write; the plan stays within what a handle allocates.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>

#include "batch_plan.h"

using namespace wick;

static int bad(const char *what, int k) {
    std::printf("case %d: %s\n", k, what);
    return 1;
}

static int check(const BatchLimits &c, const std::vector<int> &start, const std::vector<int> &t, int prefix, int k) {
    const BatchPlan p = batch_plan(c, start.data(), t.data(), prefix);
    int total = 0;
    for (int x : t) total += x;
    if (p.head.total != total || (int)p.tokens.size() != total) return bad("token count", k);
    if (p.head.items != (int)p.items.size() || p.head.items > batch_max_items(c)) return bad("item count", k);
    if (p.state_rows > batch_max_state_rows(c)) return bad("state rows", k);
    std::vector<int> seq(total), pos(total);
    for (int s = 0, i = 0; s < c.sequences; s++)
        for (int j = 0; j < t[s]; j++, i++) {
            seq[i] = s;
            pos[i] = start[s] + j;
            if (p.tokens[i].seq != s || p.tokens[i].pos != pos[i]) return bad("token place", k);
        }
    // per packed row: times each prefix key and each own key is in an item
    const int rows = total * c.group;
    std::vector<std::vector<int>> pre(rows, std::vector<int>(prefix, 0)), own(rows);
    for (int r = 0; r < rows; r++) own[r].assign(pos[r / c.group] + 1, 0);
    std::map<int, int> state;  // state row -> packed row
    std::vector<int> direct(rows, 0);
    std::map<int, std::vector<int>> of_row;
    for (const BatchItem &it : p.items) {
        if (it.nrows < 1 || it.nrows > kBatchWide || it.row0 < 0) return bad("item rows", k);
        if (it.p0 < 0 || it.p1 > prefix || it.p0 > it.p1 || it.o0 < 0 || it.o0 > it.o1) return bad("item keys", k);
        if (it.seq < 0 && it.o0 != it.o1) return bad("own keys without a sequence", k);
        if (it.seq >= 0 && it.o1 > start[it.seq] + t[it.seq]) return bad("own keys past the end", k);
        for (int r = 0; r < it.nrows; r++) {
            const int row = it.row0 + r, tok = it.seq == -2   ? p.tokens[row / c.group].split
                                       : it.seq < 0 ? row / c.group + it.shift
                                                    : row / c.group;
            if (tok < 0 || tok >= total) return bad("item token", k);
            const int packed = tok * c.group + row % c.group;
            if (it.seq >= 0 && seq[tok] != it.seq) return bad("item sequence", k);
            for (int j = it.p0; j < it.p1; j++) pre[packed][j]++;
            const int last = row / c.group + it.shift;
            if (it.seq >= 0 && last != pos[tok]) return bad("last key", k);
            for (int j = it.o0; j < it.o1 && j <= last; j++) own[packed][j]++;
            if (it.state0 < 0) {
                direct[packed]++;
            } else {
                const int at = it.state0 + r;
                if (at >= p.state_rows || state.count(at)) return bad("state rows meet", k);
                state[at] = packed;
                if (it.seq < 0 || last >= it.o0) of_row[packed].push_back(at);
            }
        }
    }
    for (int r = 0; r < rows; r++) {
        for (int n : pre[r])
            if (n != 1) return bad("prefix key", k);
        for (int n : own[r])
            if (n != 1) return bad("own key", k);
        if (direct[r] > 1 || (direct[r] == 1) != (of_row.count(r) == 0)) return bad("att written once", k);
    }
    size_t joined = 0;
    for (int i = 0; i < p.head.merges; i++) {
        const BatchToken &m = p.tokens[i];
        for (int h = 0; h < c.group; h++) {
            std::vector<int> want;
            for (int n = 0; n < p.head.prefix_chunks; n++) want.push_back(m.prefix_state + n * p.head.prefix_stride + h);
            for (int n = 0; n < m.own_chunks; n++) want.push_back(m.own_state + n * m.own_stride + h);
            // a block's later rows may see a range of keys that this one does not: such a
            // state holds no keys and is left out
            std::vector<int> &have = of_row[m.merge * c.group + h];
            std::sort(want.begin(), want.end());
            std::sort(have.begin(), have.end());
            if (want != have) return bad("joined states", k);
            joined += have.size();
        }
    }
    size_t rows_joined = 0;
    for (const auto &x : of_row) rows_joined += x.second.size();
    if (joined != rows_joined) return bad("states that nothing joins", k);
    return 0;
}

int main() {
    std::mt19937 g(7);
    auto pick = [&](int lo, int hi) { return (int)(lo + g() % (unsigned)(hi - lo + 1)); };
    int wholes = 0, splits = 0;
    for (int k = 0; k < 400; k++) {
        BatchLimits c{};
        c.group = pick(1, 9);
        c.kv_heads = pick(1, 8);
        c.sequences = pick(1, 12);
        c.capacity = pick(1, 300);
        c.prefix_capacity = k % 3 ? pick(0, 900) : 0;
        c.cus = k % 4 == 0 ? 16 : k % 4 == 1 ? 256 : k % 4 == 2 ? 1 : 64;
        c.few = batch_few(k / 4 % 2);
        const bool single = k % 5 == 0;
        std::vector<int> start(c.sequences), t(c.sequences);
        int total = 0;
        for (int s = 0; s < c.sequences; s++) {
            start[s] = pick(0, c.capacity - 1);
            t[s] = single ? 1 : pick(0, 3) == 0 ? 0 : pick(0, c.capacity - start[s]);
            total += t[s];
        }
        c.max_tokens = std::max(1, total);
        const int prefix = c.prefix_capacity ? pick(0, c.prefix_capacity) : 0;
        if (check(c, start, t, prefix, k)) return 1;
        const BatchPlan p = batch_plan(c, start.data(), t.data(), prefix);
        // graphs of this plan's t replay under plans for other positions
        for (int j = 0; j < 4; j++) {
            std::vector<int> other(c.sequences);
            for (int s = 0; s < c.sequences; s++) other[s] = j == 0 ? c.capacity - t[s] : pick(0, c.capacity - t[s]);
            const BatchPlan q = batch_plan(c, other.data(), t.data(), j == 1 ? 0 : c.prefix_capacity);
            if (q.head.items > p.head.most_items) return bad("more items than a captured call launches", k);
        }
        for (const BatchItem &it : p.items) (it.state0 < 0 ? wholes : splits)++;
    }
    if (!wholes || !splits) return bad("both kinds of items", -1);
    std::printf("ok\n");
    return 0;
}

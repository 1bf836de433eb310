// Checks that the plans of batch_plan() stay within what a handle allocates and what a captured
// call launches, over steps of every kind: only sizes are looked at, so prefixes are as long as
// in use.  argv[1]: steps to draw, argv[2]: the seed.
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <string>

#include "batch_plan.h"

using namespace wick;

static std::string text(const std::vector<int> &x) {
    std::string s;
    for (int v : x) s += (s.empty() ? "" : ",") + std::to_string(v);
    return s;
}

// Sizes of one step against the bounds of its handle; the items a captured call launches must do for
// the same tokens at any place.
static int check(BatchLimits c, const std::vector<int> &start, const std::vector<int> &t, int prefix, int spare) {
    int total = 0;
    for (int x : t) total += x;
    c.sequences = (int)t.size();
    c.max_tokens = std::max(1, total) + spare;
    const BatchPlan p = batch_plan(c, start.data(), t.data(), prefix);
    const char *what = nullptr;
    // the smallest handle that takes the step
    BatchLimits tight = c;
    tight.prefix_capacity = prefix;
    tight.capacity = 1;
    for (size_t i = 0; i < t.size(); i++) tight.capacity = std::max(tight.capacity, start[i] + t[i]);
    if (p.state_rows > batch_max_state_rows(tight)) what = "more state rows than the smallest handle holds";
    if (p.head.items != (int)p.items.size()) what = "item count";
    if (p.head.items > batch_max_items(c)) what = "more items than a handle holds";
    if (p.head.items > p.head.most_items) what = "more items than a captured call launches";
    if (p.head.most_items > batch_max_items(c)) what = "a captured call of more items than a handle holds";
    if (p.state_rows > batch_max_state_rows(c)) what = "more state rows than a handle holds";
    const std::vector<int> none(t.size(), 0);
    if (batch_plan(c, none.data(), t.data(), 0).head.most_items != p.head.most_items) what = "a captured call depends on the place";
    if (!what) return 0;
    std::printf("%s: group %d kv_heads %d few %d cus %d start %s t %s prefix %d max_tokens %d: items %d, handle %lld, captured %d; "
                "state rows %lld of %lld\n",
                what, c.group, c.kv_heads, c.few, c.cus, text(start).c_str(), text(t).c_str(), prefix, c.max_tokens, p.head.items,
                (long long)batch_max_items(c), p.head.most_items, (long long)p.state_rows, (long long)batch_max_state_rows(c));
    return 1;
}

int main(int argc, char **argv) {
    const int steps = argc > 1 ? std::atoi(argv[1]) : 20000;
    std::mt19937 g(argc > 2 ? std::atoi(argv[2]) : 1);
    const int shapes[][2] = {{3, 3}, {7, 2}, {2, 8}, {8, 4}, {4, 8}};  // group, kv_heads
    auto limits = [](int group, int kv_heads, bool bf16) {
        BatchLimits c{};
        c.group = group;
        c.kv_heads = kv_heads;
        c.capacity = 4000;
        c.prefix_capacity = 200000;
        c.cus = 256;
        c.few = batch_few(bf16);
        return c;
    };
    int bad = 0;
    // a prompt beside a few single tokens, behind a long prefix
    for (bool bf16 : {false, true}) {
        bad += check(limits(4, 8, bf16), {142, 52, 0}, {1, 1, 32}, 8764, 0);
        bad += check(limits(7, 2, bf16), {9, 0}, {18, 1}, 35263, 0);
        bad += check(limits(8, 4, bf16), {0, 100, 100}, {15, 1, 1}, 24000, 0);
        bad += check(limits(3, 3, bf16), {0, 100, 100, 100, 100, 100}, {38, 1, 1, 1, 1, 1}, 24000, 0);
        bad += check(limits(4, 8, bf16), {0, 100, 100, 100}, {30, 1, 1, 1}, 16384, 0);
        bad += check(limits(2, 8, bf16), {0, 100, 100, 100}, {62, 1, 1, 1}, 16384, 0);
        bad += check(limits(7, 2, bf16), {0, 100, 100, 100}, {16, 1, 1, 1}, 32768, 0);
        bad += check(limits(3, 3, bf16), {0, 100, 100, 100}, {40, 1, 1, 1}, 32768, 0);
        bad += check(limits(8, 4, bf16), {0, 100, 100}, {15, 1, 1}, 32768, 5000);
        bad += check(limits(7, 2, bf16), {0, 100, 100, 100}, {16, 1, 1, 1}, 60000, 5000);
    }
    // a handle holds states for its own rows and positions: four tokens of three rows against up to three
    // ranges of 300 prefix positions and one of 61
    BatchLimits four = limits(3, 3, false);
    four.sequences = four.max_tokens = 4;
    four.capacity = 61;
    four.prefix_capacity = 300;
    if (batch_max_state_rows(four) > 4 * 3 * (3 + 1)) {
        std::printf("%lld state rows for four tokens\n", (long long)batch_max_state_rows(four));
        bad++;
    }
    auto pick = [&](int lo, int hi) { return (int)(lo + g() % (unsigned)(hi - lo + 1)); };
    auto spread = [&](int lo, int hi) {  // over the logarithm, lo >= 1
        return std::min(hi, (int)std::exp(std::log((double)lo) + (g() / 4294967296.0) * std::log((hi + 1.0) / lo)));
    };
    for (int k = 0; k < steps && bad < 20; k++) {
        const int *s = shapes[pick(0, 4)];
        BatchLimits c = limits(s[0], s[1], pick(0, 1));
        if (pick(0, 2) == 0) {
            c.group = spread(1, 128);
            c.kv_heads = spread(1, 16);
        }
        if (pick(0, 7) == 0) c.cus = spread(1, 304);
        // prompts, prompts that go on and single tokens, in any order; some sequences bring nothing
        const int prompts = pick(0, 2) == 0 ? spread(1, 20) : pick(0, 2), singles = pick(0, 3) == 0 ? spread(1, 64) : pick(0, 5);
        const int longest = spread(1, prompts > 2 ? 700 : 2000);
        std::vector<int> t, start;
        for (int i = 0; i < prompts; i++) t.push_back(spread(1, longest));
        for (int i = 0; i < singles; i++) t.push_back(1);
        if (t.empty() || pick(0, 3) == 0) t.push_back(0);
        for (size_t i = t.size(); i > 1; i--) std::swap(t[i - 1], t[pick(0, (int)i - 1)]);
        const bool fresh = pick(0, 1);
        for (int x : t) start.push_back(x > 1 && fresh ? 0 : pick(0, 1) ? spread(1, c.capacity - x + 1) - 1 : pick(0, c.capacity - x));
        const int prefix = pick(0, 5) == 0 ? 0 : spread(1, 200000);
        bad += check(c, start, t, prefix, pick(0, 1) ? 0 : spread(1, 100000));
    }
    if (bad) return 1;
    std::printf("ok\n");
    return 0;
}

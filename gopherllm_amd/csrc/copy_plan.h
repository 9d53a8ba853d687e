// copy_plan.h -- the order in which ranges of rows are copied within a cache so
// that every row is read before it is written.  Host arithmetic only, so it is
// tested without a device.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

namespace gllm {

constexpr int kCopyMost = 4096;  // moves of a call

struct RowMove {
    int src, dst, rows;
};

// First `staged` is read into a workspace, then `moves` are made, then `staged` is
// written from there.
struct CopyPlan {
    bool ok;      // false: two destinations share a row
    bool apart;   // no move writes what any reads: `moves` in any order, otherwise one after another
    std::vector<RowMove> moves, staged;  // without those that do nothing
};

// same: source and destination are one cache.
inline CopyPlan copy_plan(const int32_t* m, int n, bool same) {
    CopyPlan p{true, true, {}, {}};
    std::vector<RowMove> to;
    for (int i = 0; i < n; i++)
        if (m[3 * i + 2] > 0) to.push_back({m[3 * i], m[3 * i + 1], m[3 * i + 2]});
    std::sort(to.begin(), to.end(), [](const RowMove& a, const RowMove& b) { return a.dst < b.dst; });
    for (size_t i = 1; i < to.size(); i++)
        if (to[i].dst < to[i - 1].dst + to[i - 1].rows) {
            p.ok = false;
            return p;
        }
    for (const RowMove& x : to)
        if (!same || x.src != x.dst) p.moves.push_back(x);
    if (!same) return p;
    // move i reads rows that move j writes: i goes before j.  The destinations are
    // sorted and apart, so those that a source meets lie together.
    const int k = (int)p.moves.size();
    std::vector<std::vector<int>> after(k), before(k);
    std::vector<int> waits(k, 0);
    bool any = false;
    for (int i = 0; i < k; i++) {
        const RowMove& x = p.moves[i];
        int lo = 0, hi = k;  // the first destination that ends past the source's first row
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (p.moves[mid].dst + p.moves[mid].rows <= x.src) lo = mid + 1;
            else hi = mid;
        }
        for (int j = lo; j < k && p.moves[j].dst < x.src + x.rows; j++) {
            any = true;
            if (j == i) continue;  // over its own rows: copied from the right end
            after[i].push_back(j);
            before[j].push_back(i);
            waits[j]++;
        }
    }
    if (!any) return p;
    p.apart = false;
    std::vector<RowMove> order;
    std::vector<int> ready, seen(k, -1);
    std::vector<bool> done(k, false);
    for (int i = 0; i < k; i++)
        if (!waits[i]) ready.push_back(i);
    int first = 0;  // all before it are done
    for (size_t at = 0, left = k; left; left--) {
        int i;
        if (at < ready.size()) {
            i = ready[at++];
            order.push_back(p.moves[i]);
        } else {
            // The rest wait for circles or are in one.  Up from one of them to what it waits
            // for, until a move comes again: its circle's shortest is set aside, so its rows are free.
            while (done[first]) first++;
            const auto up = [&](int j) {
                while (done[before[j].back()]) before[j].pop_back();
                return before[j].back();
            };
            int j = first;
            for (; seen[j] != (int)left; j = up(j)) seen[j] = (int)left;
            i = j;
            for (int c = up(j); c != j; c = up(c))
                if (p.moves[c].rows < p.moves[i].rows) i = c;
            p.staged.push_back(p.moves[i]);
        }
        done[i] = true;
        for (int j : after[i])
            if (--waits[j] == 0 && !done[j]) ready.push_back(j);
    }
    p.moves = order;
    return p;
}

}  // namespace gllm

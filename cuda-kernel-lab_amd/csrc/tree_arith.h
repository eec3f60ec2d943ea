// tree_arith.h -- how the attention of drafted tokens is cut over the workgroups: arithmetic alone, for the
// kernels and (compiled by the host compiler) for tests.
//
// The rows of a sequence for one kv head (its n tokens times the G query heads of the head, a token's heads
// together) are cut into groups of as many tokens as fill a workgroup's rows. Each (sequence, group) is an item; its
// units are `extra` for its start and `weight` for each page that its tokens may see. The units of all items, in the order of
// sequences, groups and pages, are cut into ranges, and workgroup (g, kv head) takes range g: pieces of items, one after
// the other; a page belongs to the range that holds its first unit. An item inside one range is written by its
// workgroup. Of an item cut by range boundaries, the piece that starts it goes to partial slot 2 w + 1 of its
// workgroup w = g Hkv + kv head, every later piece to slot 2 w of its.
#pragma once

#include <cstdint>

#include "range_arith.h"

namespace pdattn {

// x / d for x >= 0, 0 < d < 2^16, in 32 bits (a 64-bit division is some hundred instructions).
PD_RANGE_FN int64_t tree_div(int64_t x, uint32_t d) {
    const uint64_t u = (uint64_t)x;
    if (u >> 32 == 0) return (int64_t)((uint32_t)u / d);
    uint64_t q = 0;
    uint32_t rest = 0;
    for (int i = 48; i >= 0; i -= 16) {
        rest = rest << 16 | (uint32_t)(u >> i & 0xFFFF);
        q = q << 16 | rest / d;
        rest %= d;
    }
    return (int64_t)q;
}

// One sequence of the batch as the kernels see it. Positions count from the sequence's first cached token.
struct TreeSeq {
    int len, n, ctx;     // cached tokens, new ones among them, those before them (below 0: n > len)
    int np;              // pages
    int s, w0;           // attended pages: [0, s) and [w0, np)
    int groups;
    // pages of group j: u0 + st (j >> cl). Chains: later tokens see more pages, a page more every 16 tokens.
    int u0, st, cl;
    int wt, wl;          // units of a page of a group, and of the last group
    int extra;           // units of a group's start
    PD_RANGE_FN int attended() const { return s + np - w0; }
    // the page at place i of the attended ones
    PD_RANGE_FN int page(int i) const { return i < s ? i : i - s + w0; }
    // the places of pages below page p (those before it in the order of places)
    PD_RANGE_FN int below(int p) const { return p <= s ? p : p <= w0 ? s : s + p - w0; }
    PD_RANGE_FN int weight(int j) const { return j == groups - 1 ? wl : wt; }
    PD_RANGE_FN int pages(int j) const { return u0 + st * (j >> cl); }
    PD_RANGE_FN int units(int j) const { return pages(j) * weight(j) + extra; }
    // the first page of group j whose first unit is x or later
    PD_RANGE_FN int first_page(int j, int x) const {
        const int k = weight(j), y = x - extra;
        return y <= 0 ? 0 : k == 1 ? y : (int)(((uint32_t)y + (uint32_t)k - 1u) / (uint32_t)k);
    }
    // the first unit of the last page of group j
    PD_RANGE_FN int last_unit(int j) const { return extra + (pages(j) - 1) * weight(j); }
    // units of the groups before j
    PD_RANGE_FN int64_t before(int j) const {
        const int64_t m = j >> cl;
        int64_t sum = (int64_t)u0 * j;
        if (st) sum += st * ((m * (m - 1) / 2 << cl) + (j - (m << cl)) * m);
        sum = sum * wt + (int64_t)extra * j;
        return j == groups && j > 0 ? sum - (int64_t)pages(j - 1) * (wt - wl) : sum;
    }
    PD_RANGE_FN int64_t total() const { return before(groups); }
    // the group that holds the sequence's unit x
    PD_RANGE_FN int group_of(int64_t x) const {
        if (groups <= 1) return 0;
        int lo = 0, hi = groups - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (before(mid) <= x) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    }
};

// From the device's tables as they are (no trust in them: never a negative count). 2^tl tokens per group; causal: no
// token sees drafted keys after its own. weight: units of a page; of a group that fills at most half of its rows three
// quarters of that (rounded up). extra: units of a group's start.
PD_RANGE_FN TreeSeq tree_seq(int ip0, int ip1, int last, int q0, int q1, int n_tokens, int tl, int window, int sink, bool causal,
                             int weight = 1, int extra = 0) {
    TreeSeq t;
    t.np = ip1 > ip0 ? ip1 - ip0 : 0;
    t.len = t.np > 0 ? (t.np - 1) * 16 + (last < 1 ? 1 : last > 16 ? 16 : last) : 0;
    const int a = q0 < 0 ? 0 : q0 > n_tokens ? n_tokens : q0, b = q1 < 0 ? 0 : q1 > n_tokens ? n_tokens : q1;
    t.n = b > a ? b - a : 0;
    t.ctx = t.len - t.n;
    t.groups = (int)(((int64_t)t.n + (1 << tl) - 1) >> tl);
    t.wt = weight;
    t.wl = t.n - ((int64_t)(t.groups - 1) << tl) <= (1 << tl) / 2 ? weight - weight / 4 : weight;
    t.extra = extra;
    t.s = t.w0 = 0;
    if (window > 0) {
        // a token at position ctx or later sees, below the context, only keys from ctx - window + 1 on
        const int first = t.ctx - window + 1;
        const int w0 = first > 0 ? first / 16 : 0;
        const int s = sink > 0 ? (int)(((int64_t)sink + 15) / 16) : 0;
        if (w0 > s) {
            t.s = s;
            t.w0 = w0;
        }
    }
    // A sequence without pages still has its rows to write: one page an item at least.
    t.u0 = t.attended() > 0 ? t.attended() : 1;
    t.st = 0;
    t.cl = 0;
    if (causal && t.groups > 1 && t.ctx >= 0 && (int64_t)2 * t.n > t.ctx) {
        // Tokens of group j see the keys below ctx + (j + 1) 2^tl. (Where the context is most of them, equal units are
        // better: the groups' cuts then fall on the same keys, which their workgroups read together, through one L2. A
        // chain of 512 on 2 x 8192 tokens: 164 us, with their own units 191.)
        const int sl = tl > 4 ? tl : 4;   // a step is 16 tokens or a group
        t.u0 = t.below((t.ctx + (1 << sl) + 15) >> 4);
        t.st = 1 << (sl - 4);
        t.cl = sl - tl;
    }
    return t;
}

// The blocks of a wave: block i starts at place first + step i and has `width` places, those below p1. Places [a0, a1) hold
// pages whose every key is seen by every row: the blocks inside them are `plain`, and come first; then those behind
// them, then those before (the order of blocks does not matter to a softmax, and two loops without a branch inside do).
struct TreeOrder {
    int n, b0, plain;
    PD_RANGE_FN int block(int i) const { return i + b0 < n ? i + b0 : i + b0 - n; }
};
PD_RANGE_FN TreeOrder tree_order(int first, int step, int width, int p1, int a0, int a1) {
    TreeOrder o;
    o.n = first < p1 ? (p1 - first + step - 1) / step : 0;
    if (a1 > p1) a1 = p1;
    o.b0 = a0 > first ? (a0 - first + step - 1) / step : 0;
    const int b1 = a1 >= first + width ? (a1 - first - width) / step + 1 : 0;
    o.plain = b1 > o.b0 ? b1 - o.b0 : 0;
    if (o.plain == 0) o.b0 = 0;
    return o;
}

// The cut of `units` into ranges: at most `most`, of at least `least` units on average. With two workgroups on a CU the
// one that came first issues first: where all `most` ranges are used, the first half of them is longer, `early` to
// `late`.
struct TreeCuts {
    int64_t step;                           // units = step total + rest
    int rest;
    int ranges, early, late, half, total;   // half: ranges of the first kind; total: the sum of their weights, below 2^15
    PD_RANGE_FN int64_t start(int g) const {   // units w / total
        const int w = g <= half ? early * g : early * half + late * (g - half);
        return step * w + (uint32_t)rest * (uint32_t)w / (uint32_t)total;
    }
    // the range that holds unit x: a guess in 32-bit floats, put right
    PD_RANGE_FN int of(int64_t x) const {
        const float y = (float)x / ((float)step + (float)rest / (float)total), e = (float)(early * half);
        int g = (int)(y < e ? y / (float)early : (float)half + (y - e) / (float)late);
        g = g < 0 ? 0 : g >= ranges ? ranges - 1 : g;
        while (g > 0 && start(g) > x) --g;
        while (g + 1 < ranges && start(g + 1) <= x) ++g;
        return g;
    }
};
PD_RANGE_FN TreeCuts tree_cuts(int64_t units, int most, int least, int early, int late) {
    TreeCuts c;
    const int64_t r = tree_div(units, (uint32_t)least);
    c.ranges = units <= 0 ? 0 : r < 1 ? 1 : r > most ? most : (int)r;
    c.half = c.ranges == most ? most / 2 : 0;
    c.early = early;
    c.late = c.half > 0 ? late : 1;
    c.total = c.half > 0 ? early * c.half + late * (c.ranges - c.half) : c.ranges;
    c.step = c.total > 0 ? tree_div(units, (uint32_t)c.total) : 0;
    c.rest = (int)(units - c.step * c.total);
    return c;
}

// The partial slot (0 or 1) of a piece that holds pages [p0, p1) of its item's `pages`, or -1: the whole item.
PD_RANGE_FN int tree_slot(int p0, int p1, int pages) { return p0 > 0 ? 0 : p1 < pages ? 1 : -1; }

}  // namespace pdattn

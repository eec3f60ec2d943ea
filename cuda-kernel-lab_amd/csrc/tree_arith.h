// tree_arith.h -- how the attention of drafted tokens is cut over the workgroups: arithmetic alone, for the
// kernels and (compiled by the host compiler) for tests.
//
// The rows of a sequence for one kv head (its n tokens times the G query heads of the head, a token's heads
// together) are cut into groups of as many tokens as fill a workgroup's rows. Each (sequence, group) is an item; its
// units are the pages that the sequence attends. The units of all items, in the order of sequences, groups and
// pages, are cut into equal ranges, and workgroup (g, kv head) takes range g: pieces of items, one after the
// other. An item inside one range is written by its workgroup. Of an item cut by range boundaries, the piece that
// starts it goes to partial slot 2 w + 1 of its workgroup w = g Hkv + kv head, every later piece to slot 2 w of its.
#pragma once

#include <cstdint>

#include "range_arith.h"

namespace pdattn {

// One sequence of the batch as the kernels see it. Positions count from the sequence's first cached token.
struct TreeSeq {
    int len, n, ctx;     // cached tokens, new ones among them, those before them (below 0: n > len)
    int np;              // pages
    int s, w0;           // attended pages: [0, s) and [w0, np)
    int groups;
    // attended pages, and the units of one of its items: a sequence without pages still has its rows to write
    PD_RANGE_FN int attended() const { return s + np - w0; }
    PD_RANGE_FN int units() const { return attended() > 0 ? attended() : 1; }
    PD_RANGE_FN int64_t total() const { return (int64_t)groups * units(); }
    // the page at place i of the attended ones
    PD_RANGE_FN int page(int i) const { return i < s ? i : i - s + w0; }
};

// From the device's tables as they are (no trust in them: never a negative count). page_tokens = 16; tpg: tokens
// per group.
PD_RANGE_FN TreeSeq tree_seq(int ip0, int ip1, int last, int q0, int q1, int n_tokens, int tpg, int window, int sink) {
    TreeSeq t;
    t.np = ip1 > ip0 ? ip1 - ip0 : 0;
    t.len = t.np > 0 ? (t.np - 1) * 16 + (last < 1 ? 1 : last > 16 ? 16 : last) : 0;
    const int a = q0 < 0 ? 0 : q0 > n_tokens ? n_tokens : q0, b = q1 < 0 ? 0 : q1 > n_tokens ? n_tokens : q1;
    t.n = b > a ? b - a : 0;
    t.ctx = t.len - t.n;
    t.groups = (t.n + tpg - 1) / tpg;
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
    return t;
}

// The attended pages of a sequence below page `p` (those before it in the order of places).
PD_RANGE_FN int tree_places_below(const TreeSeq& t, int p) { return p <= t.s ? p : p <= t.w0 ? t.s : t.s + p - t.w0; }

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

// Ranges that `units` are cut into: at most `most`, of at least `least` units each.
PD_RANGE_FN int tree_ranges(int64_t units, int most, int least) {
    const int64_t r = units / least;
    return r < 1 ? 1 : r > most ? most : (int)r;
}
PD_RANGE_FN int64_t tree_range_start(int64_t units, int ranges, int g) { return units * g / ranges; }
// The range that holds unit x.
PD_RANGE_FN int tree_range_of(int64_t units, int ranges, int64_t x) { return (int)(((x + 1) * ranges - 1) / units); }

// The partial slot of a piece that starts `skip` units into its item and takes `take` of its `units`, or -1: the
// whole item.
PD_RANGE_FN int tree_slot(int skip, int take, int units) { return skip > 0 ? 0 : take < units ? 1 : -1; }

}  // namespace pdattn

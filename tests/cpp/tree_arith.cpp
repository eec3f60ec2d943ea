// The cut of the attention of drafted tokens over workgroups (csrc/tree_arith.h), for tests/test_tree_arithmetic.py.
#include "../../cuda-kernel-lab_amd/csrc/tree_arith.h"

using namespace pdattn;

namespace {
TreeSeq seq(const int* a) { return tree_seq(a[0], a[1], a[2], a[3], a[4], a[5], __builtin_ctz(a[6]), a[7], a[8], a[9] != 0); }
}  // namespace

// a: ip0, ip1, last, q0, q1, n_tokens, tokens per group (a power of two), window, sink, causal; out: len, n, ctx, np, s, w0, groups, attended
extern "C" void t_seq(const int* a, int* out) {
    const TreeSeq t = seq(a);
    const int v[] = {t.len, t.n, t.ctx, t.np, t.s, t.w0, t.groups, t.attended()};
    for (int i = 0; i < 8; ++i) out[i] = v[i];
}
extern "C" int t_page(const int* a, int i) { return seq(a).page(i); }
extern "C" int t_below(const int* a, int page) { return seq(a).below(page); }
extern "C" int t_units(const int* a, int j) { return seq(a).units(j); }
extern "C" long long t_before(const int* a, int j) { return seq(a).before(j); }
extern "C" int t_group(const int* a, long long x) { return seq(a).group_of(x); }
extern "C" int t_ranges(long long units, int most, int least, int early, int late) {
    return tree_cuts(units, most, least, early, late).ranges;
}
extern "C" long long t_start(long long units, int most, int least, int early, int late, int g) {
    return tree_cuts(units, most, least, early, late).start(g);
}
extern "C" int t_of(long long units, int most, int least, int early, int late, long long x) {
    return tree_cuts(units, most, least, early, late).of(x);
}
// the same with `weight` units a page and `extra` an item; a as above
extern "C" void t_weighted(const int* a, int weight, int extra, int j, int x, int* out) {
    const TreeSeq t = tree_seq(a[0], a[1], a[2], a[3], a[4], a[5], __builtin_ctz(a[6]), a[7], a[8], a[9] != 0, weight, extra);
    const long long v[] = {t.units(j), t.before(j), t.total(), t.group_of(t.before(j) + x), t.first_page(j, x), t.groups, t.last_unit(j)};
    for (int i = 0; i < 7; ++i) out[i] = (int)v[i];
}
extern "C" int t_slot(int skip, int take, int units) { return tree_slot(skip, take, units); }
// out: blocks, the plain ones among them; order[i]: the i-th block
extern "C" void t_order(int first, int step, int width, int p1, int a0, int a1, int* out, int* order) {
    const TreeOrder o = tree_order(first, step, width, p1, a0, a1);
    out[0] = o.n;
    out[1] = o.plain;
    for (int i = 0; i < o.n; ++i) order[i] = o.block(i);
}

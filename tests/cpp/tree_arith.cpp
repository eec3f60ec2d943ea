// The cut of the attention of drafted tokens over workgroups (csrc/tree_arith.h), for tests/test_tree_arithmetic.py.
#include "../../cuda-kernel-lab_amd/csrc/tree_arith.h"

using namespace pdattn;

// out: len, n, ctx, np, s, w0, groups, attended, units
extern "C" void t_seq(int ip0, int ip1, int last, int q0, int q1, int n_tokens, int tpg, int window, int sink, int* out) {
    const TreeSeq t = tree_seq(ip0, ip1, last, q0, q1, n_tokens, tpg, window, sink);
    const int v[] = {t.len, t.n, t.ctx, t.np, t.s, t.w0, t.groups, t.attended(), t.units()};
    for (int i = 0; i < 9; ++i) out[i] = v[i];
}
extern "C" int t_page(int ip0, int ip1, int last, int q0, int q1, int n_tokens, int tpg, int window, int sink, int i) {
    return tree_seq(ip0, ip1, last, q0, q1, n_tokens, tpg, window, sink).page(i);
}
extern "C" int t_ranges(long long units, int most, int least) { return tree_ranges(units, most, least); }
extern "C" long long t_start(long long units, int ranges, int g) { return tree_range_start(units, ranges, g); }
extern "C" int t_of(long long units, int ranges, long long x) { return tree_range_of(units, ranges, x); }
extern "C" int t_slot(int skip, int take, int units) { return tree_slot(skip, take, units); }
// out: blocks, the plain ones among them; order[i]: the i-th block
extern "C" void t_order(int first, int step, int width, int p1, int a0, int a1, int* out, int* order) {
    const TreeOrder o = tree_order(first, step, width, p1, a0, a1);
    out[0] = o.n;
    out[1] = o.plain;
    for (int i = 0; i < o.n; ++i) order[i] = o.block(i);
}
extern "C" int t_below(int ip0, int ip1, int last, int q0, int q1, int n_tokens, int tpg, int window, int sink, int page) {
    return tree_places_below(tree_seq(ip0, ip1, last, q0, q1, n_tokens, tpg, window, sink), page);
}

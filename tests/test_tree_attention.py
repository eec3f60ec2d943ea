"""Attention of drafted tokens (pdattn_tree_attention).

CPU: the 64-bit restatement (oracle.tree_attention) against dense softmaxes of its own over explicit boolean masks,
with planted mistakes; the refusals. GPU: the library against the restatement: trees, chains and single tokens,
every group size, lengths from 1 on, scores capped, biased and windowed, rows that see nothing, bits of NaN and
infinity where a token does not look, and what the documentation allows beyond that.
"""
import numpy as np
import pytest
from scipy.special import logsumexp, softmax

import oracle
import pdattn
from _draft import DeviceDraft, check_attention, make_draft, oracle_attention, pack

SLOPES = lambda Hq: [2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)]  # noqa: E731


# ---- CPU: the restatement --------------------------------------------------------------------------

def _dense(dr, soft_cap=0.0, slopes=None, window=0, sink=0):
    """The same attention by another road: ancestors found by walking the parents, one [tokens, keys] matrix."""
    bt = dr.bt
    out, lse = np.zeros((dr.n_tokens, bt.Hq, 128)), np.zeros((dr.n_tokens, bt.Hq))
    for b in range(bt.B):
        q0, n, L = int(dr.q_indptr[b]), len(dr.parent[b]), bt.lens[b]
        ctx = L - n
        see, pos = np.zeros((n, L), bool), np.arange(L, dtype=np.int64)
        see[:, :ctx] = True
        for i in range(n):
            line = list(range(i + 1))
            if dr.mask is not None:
                line, p = [], i
                while p >= 0:
                    line.append(p)
                    p = dr.parent[b][p]
                pos[ctx + i] = ctx + len(line) - 1
            see[i, [ctx + p for p in line]] = True
        pages = bt.indices[bt.indptr[b]:bt.indptr[b + 1]]
        for h in range(bt.Hq):
            K = bt.k[pages, :, h // bt.G].reshape(-1, 128)[:L].astype(np.float64)
            V = bt.v[pages, :, h // bt.G].reshape(-1, 128)[:L].astype(np.float64)
            x = dr.q[q0:q0 + n, h].astype(np.float64) @ K.T / np.sqrt(128)
            if soft_cap:
                x = soft_cap * np.tanh(x / soft_cap)
            far = pos[ctx:, None] - pos[None]
            if slopes is not None:
                x = x - slopes[h] * far
            ok = see & ((far < window) | (np.arange(L) < sink)) if window else see
            x = np.where(ok, x, -np.inf)
            lse[q0:q0 + n, h], out[q0:q0 + n, h] = logsumexp(x, 1), softmax(x, 1) @ V
    return out, lse


CPU_CASES = [dict(ctx=[37, 16, 1], new=[9, 1, 5], Hq=8, Hkv=2), dict(ctx=[40], new=[33], Hq=4, Hkv=4),
             dict(ctx=[21, 30], new=[6, 12], Hq=4, Hkv=2, tree=False)]
CPU_SCORES = [dict(), dict(soft_cap=2.0), dict(slopes=True), dict(window=7, sink=3), dict(soft_cap=1.5, slopes=True, window=12)]


def _agrees(case, score, fault="none"):
    dr = make_draft(seed=3, **case)
    score = dict(score, slopes=SLOPES(case["Hq"])) if score.get("slopes") else score
    out, lse, _ = oracle_attention(dr, fault=fault, **score)
    ro, rl = _dense(dr, **score)
    return np.allclose(out, ro, atol=1e-9) and np.allclose(lse, rl, atol=1e-9)


@pytest.mark.parametrize("case", CPU_CASES)
@pytest.mark.parametrize("score", CPU_SCORES)
def test_restatement_matches_dense(case, score):
    assert _agrees(case, score)


@pytest.mark.parametrize("fault", [f for f in oracle.TREE_FAULTS if f != "none"])
def test_planted_fault_is_caught(fault):
    assert not all(_agrees(case, score, fault) for case in CPU_CASES for score in CPU_SCORES)


def test_restatement_without_drafts_is_the_decode_oracle(oracle_lib):
    dr = make_draft([36, 16, 299], [1, 1, 1], 8, 2, seed=5, tree=False)
    bt = dr.bt
    out, lse, _ = oracle_attention(dr)
    ro, rl = oracle.decode(dr.q, bt.k, bt.v, bt.indptr, bt.indices, bt.last, 8, 2)
    assert np.allclose(out, ro, atol=1e-9) and np.allclose(lse, rl, atol=1e-9)


# ---- CPU: refusals -----------------------------------------------------------------------------------

def _fake(**kw):
    a = 1 << 20   # an aligned stand-in: a refused call touches no device memory
    base = dict(B=2, Hq=8, Hkv=2, n_tokens=4, q_indptr=a, max_tokens=3)
    base.update(kw)
    ptrs = [base.pop(k, a) for k in ("q", "k", "v", "indptr", "indices", "last")]
    return pdattn.make_tree_params(*ptrs, **base)


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), 1), (dict(n_tokens=-1), 1), (dict(Hq=6, Hkv=2), 2), (dict(Hq=9, Hkv=2), 2), (dict(Hq=0), 1),
    (dict(q_indptr=None), 1),                                       # four tokens of two sequences
    (dict(max_tokens=0), 1), (dict(mask=1 << 20, mask_words=0), 1),
    (dict(mask=1 << 20, mask_words=16, max_tokens=513), 2), (dict(depth=1 << 20, max_tokens=513), 2),
    (dict(sm_scale=float("nan")), 1), (dict(sm_scale=float("inf")), 1), (dict(soft_cap=-1.0), 1),
    (dict(soft_cap=float("inf")), 1), (dict(soft_cap=float("nan")), 1), (dict(window=-1), 1), (dict(sink=-1), 1),
    (dict(q=None), 1), (dict(k=None), 1), (dict(indptr=None), 1), (dict(indices=None), 1), (dict(last=None), 1),
    (dict(q=(1 << 20) + 8), 1), (dict(v=(1 << 20) + 2), 1), (dict(n_tokens=1 << 28, Hq=64, Hkv=8), 1),
])
def test_refusals(kw, status):
    p = _fake(**kw)
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.tree_attention(p, 1 << 20, 1 << 20, pdattn.Workspace(1 << 20, 1 << 40, 0))
    assert e.value.status == status
    assert pdattn.tree_workspace_size(p) == 0


@pytest.mark.parametrize("out,lse", [(None, 1 << 20), (1 << 20, None), ((1 << 20) + 4, 1 << 20)])
def test_refused_outputs(out, lse):
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.tree_attention(_fake(), out, lse, pdattn.Workspace(1 << 20, 1 << 40, 0))
    assert e.value.status == 1


@pytest.mark.parametrize("off", [0, 4 * 8 * 256 - 16, 16 - 4 * 8 * 256])
def test_an_output_over_the_queries_is_refused(off):
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.tree_attention(_fake(q=1 << 24), (1 << 24) + off, 1 << 20, pdattn.Workspace(1 << 20, 1 << 40, 0))
    assert e.value.status == 1 and "overlaps" in str(e.value)


def test_nothing_to_do():
    ws = pdattn.Workspace()
    pdattn.tree_attention(_fake(B=0, n_tokens=0), 1 << 20, 1 << 20, ws)
    pdattn.tree_attention(_fake(n_tokens=0), 1 << 20, 1 << 20, ws)
    assert not ws.base and pdattn.tree_workspace_size(_fake(n_tokens=0)) == 0


# ---- GPU: the library against the restatement ----------------------------------------------------------

def _run(dr, tag, single=False, max_tokens=None, **score):
    print(f"tree {tag}", flush=True)
    dd = DeviceDraft(dr)
    out, lse = dd.run(single=single, max_tokens=max_tokens, **score)
    off = check_attention(out, lse, oracle_attention(dr, **score), tag)
    print(f"tree {tag}: {off[0]:.3f} / {off[1]:.3f} of the tolerances", flush=True)
    return dd


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(8, 8), (8, 4), (16, 4), (16, 2), (32, 32), (2, 1), (3, 3)])
@pytest.mark.parametrize("tree", [True, False])
def test_heads(Hq, Hkv, tree):
    dr = make_draft([300, 17, 64, 5], [7, 16, 1, 33], Hq, Hkv, seed=Hq + Hkv, tree=tree)
    _run(dr, f"heads {Hq}/{Hkv} tree={tree}")


# contexts at the edges of pages and of 32-key blocks, drafts that start and end in the middle of both
@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new", [([0, 0, 0], [1, 16, 40]), ([1, 15, 16, 17], [1, 1, 2, 31]),
                                     ([31, 32, 33, 47], [33, 32, 17, 1]), ([127, 128, 129], [64, 65, 63]),
                                     ([1000, 2, 515, 0], [3, 100, 1, 5]), ([2047], [129])])
@pytest.mark.parametrize("tree", [True, False])
def test_lengths(ctx, new, tree):
    dr = make_draft(ctx, new, 8, 2, seed=sum(ctx) + 7, tree=tree)
    _run(dr, f"lengths {ctx} + {new} tree={tree}")


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (16, 2)])
@pytest.mark.parametrize("score", [dict(soft_cap=5.0), dict(slopes=True), dict(window=100, sink=3), dict(window=16),
                                   dict(window=1), dict(window=70, sink=50), dict(soft_cap=3.0, slopes=True, window=333, sink=20)])
@pytest.mark.parametrize("tree", [True, False])
def test_scores(Hq, Hkv, score, tree):
    score = dict(score, slopes=SLOPES(Hq)) if score.get("slopes") else score
    dr = make_draft([400, 60, 3, 1100], [13, 40, 5, 1], Hq, Hkv, seed=11, tree=tree)
    _run(dr, f"scores {Hq}/{Hkv} {sorted(score)} tree={tree}", **score)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 4), (8, 2), (16, 2)])
@pytest.mark.parametrize("score", [dict(), dict(soft_cap=5.0), dict(slopes=True), dict(window=100, sink=3)])
def test_one_token_per_sequence(Hq, Hkv, score):
    """The decode form: no q_indptr, no mask."""
    score = dict(score, slopes=SLOPES(Hq)) if score.get("slopes") else score
    dr = make_draft([0, 15, 300, 1500, 33], [1] * 5, Hq, Hkv, seed=13, tree=False)
    _run(dr, f"decode {Hq}/{Hkv} {sorted(score)}", single=True, **score)


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [True, False])
def test_sequences_without_tokens_and_without_pages(tree):
    """A sequence with no new token, one with nothing cached but them, one with no page at all though it has tokens."""
    dr = make_draft([50, 20, 0, 70], [3, 0, 6, 2], 8, 2, seed=17, tree=tree)
    _run(dr, f"no tokens tree={tree}")
    bt = dr.bt   # sequence 2's tokens lose their pages
    cut = int(bt.indptr[3] - bt.indptr[2])
    bt.indices = np.delete(bt.indices, np.arange(int(bt.indptr[2]), int(bt.indptr[3])))
    bt.indptr = bt.indptr.copy()
    bt.indptr[3:] -= cut
    bt.last = bt.last.copy()
    bt.last[2] = 0
    dd = _run(dr, f"no pages tree={tree}")
    assert np.isneginf(dd.lse.cpu().numpy()[3:9]).all()


@pytest.mark.gpu
def test_rows_that_see_nothing():
    """Mask rows of zeros: with an empty context the row sees no key; with one it sees the context alone."""
    dr = make_draft([0, 40], [20, 20], 8, 2, seed=19)
    dr.mask[3], dr.mask[7], dr.mask[25] = 0, 0, 0
    dd = _run(dr, "nothing seen")
    assert np.isneginf(dd.lse.cpu().numpy()[3]).all() and np.isfinite(dd.lse.cpu().numpy()[25]).all()


@pytest.mark.gpu
def test_a_window_that_leaves_nothing():
    """Depths that put a token far behind the context, whose window then holds only keys it does not see."""
    dr = make_draft([10, 100], [5, 5], 4, 2, seed=23)
    dr.depth[:] = 400
    dr.mask[:] = 0
    _run(dr, "empty window", window=8)


@pytest.mark.gpu
def test_arbitrary_masks_and_depths():
    """Bits that are no tree (later tokens, not the token itself), depths out of order and below 0."""
    dr = make_draft([35, 3, 90], [40, 64, 7], 8, 2, seed=29)
    rng = np.random.default_rng(1)
    dr.mask = pack(rng.random((dr.n_tokens, 64)) < 0.4)
    dr.depth = rng.integers(-3, 50, dr.n_tokens).astype(np.int32)
    _run(dr, "arbitrary", window=30, sink=2, slopes=SLOPES(8))


@pytest.mark.gpu
@pytest.mark.parametrize("words,new", [(1, [40, 12]), (2, [40, 12]), (5, [40, 12]), (16, [512, 31])])
def test_mask_words(words, new):
    """Fewer words than the tokens (their bits count as 0), more than needed, and the most tokens."""
    rng = np.random.default_rng(words)
    dr = make_draft([33, 50], new, 4, 2, seed=31, tree=False)
    dr.mask = pack(rng.random((dr.n_tokens, 32 * words)) < 0.5)
    _run(dr, f"words {words}")


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new", [([600, 0], [700, 513]), ([5], [1300])])
def test_long_chains(ctx, new):
    """More tokens of a sequence than a mask may have: a chunk of a prefill."""
    dr = make_draft(ctx, new, 4, 2, seed=37, tree=False)
    _run(dr, f"chain {ctx} + {new}")


@pytest.mark.gpu
def test_depths_without_a_mask():
    dr = make_draft([70, 9], [20, 33], 8, 2, seed=41)
    dr.mask = None
    _run(dr, "depths alone", window=25, slopes=SLOPES(8))


@pytest.mark.gpu
def test_tokens_past_the_masks_limit_are_not_seen():
    """max_tokens says 512, a sequence has 530: keys past the limit are not seen, and nothing else changes."""
    dr = make_draft([20], [530], 2, 2, seed=43, words=16)
    dr.mask = pack(np.random.default_rng(3).random((530, 512)) < 0.5)
    _run(dr, "past the limit", max_tokens=512)


@pytest.mark.gpu
@pytest.mark.parametrize("sm_scale", [0.0, -0.3, 1.0, 8.0])
@pytest.mark.parametrize("soft_cap", [0.0, 4.0])
def test_scales(sm_scale, soft_cap):
    """Scores in the hundreds (a softmax close to an argmax), all alike, and of the other sign."""
    dr = make_draft([200, 30], [9, 20], 8, 2, seed=47)
    _run(dr, f"scale {sm_scale} cap {soft_cap}", sm_scale=sm_scale, soft_cap=soft_cap)


def _poison(dr, rng):
    """NaN and infinities in every cache slot past the sequences' ends."""
    bt = dr.bt
    bad = np.array([np.nan, np.inf, -np.inf], np.float16)
    for b in range(bt.B):
        if bt.indptr[b + 1] > bt.indptr[b] and bt.last[b] < 16:
            page = bt.indices[bt.indptr[b + 1] - 1]
            for c in (bt.k, bt.v):
                c[page, bt.last[b]:] = rng.choice(bad, c[page, bt.last[b]:].shape)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [dict(), dict(soft_cap=5.0, slopes=True), dict(window=40, sink=5)])
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (16, 2)])
def test_bits_past_the_end(score, Hq, Hkv):
    score = dict(score, slopes=SLOPES(Hq)) if score.get("slopes") else score
    dr = make_draft([37, 101, 0, 250], [5, 30, 3, 17], Hq, Hkv, seed=53)
    _poison(dr, np.random.default_rng(2))
    _run(dr, f"poisoned ends {sorted(score)}", **score)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["nan", "inf"])
@pytest.mark.parametrize("Hq,Hkv,new", [(4, 4, 12), (16, 2, 40), (16, 2, 3), (8, 2, 64)])
def test_a_drafted_token_of_nan_reaches_only_those_who_see_it(kind, Hq, Hkv, new):
    """K and V of some drafted tokens hold NaN (infinity): a row that does not see them is as without them."""
    dr = make_draft([50, 20], [new, new], Hq, Hkv, seed=59)
    bt, bad = dr.bt, (np.nan if kind == "nan" else np.inf)
    rng = np.random.default_rng(4)
    struck = np.zeros(dr.n_tokens, bool)
    for b in range(bt.B):
        q0, n = int(dr.q_indptr[b]), len(dr.parent[b])
        ctx = bt.lens[b] - n
        for j in rng.choice(np.arange(1, n), 2, replace=False):
            pos = ctx + j
            page = bt.indices[bt.indptr[b] + pos // 16]
            bt.v[page, pos % 16, :, ::3] = bad
            if kind == "nan":
                bt.k[page, pos % 16] = bad
            seen = dr.mask.view(np.uint32)[q0:q0 + n, j // 32] >> np.uint32(j % 32) & 1
            struck[q0:q0 + n] |= seen != 0
    print(f"tree {kind} in drafts", flush=True)
    out, lse = DeviceDraft(dr).run()
    assert struck.any() and not struck.all()
    with np.errstate(invalid="ignore"):
        ref = oracle_attention(dr)
    check_attention(out, lse, ref, f"{kind} unseen", rows=~struck)
    if kind == "nan":
        assert np.isnan(out[struck]).all() and np.isnan(lse[struck]).all()
    else:   # (V alone: lse is untouched, the struck dims are infinite, the others not)
        assert np.isfinite(lse).all() and np.isfinite(out[struck][..., 1::3]).all()
        assert not np.isfinite(out[struck][..., ::3]).any()


@pytest.mark.gpu
def test_nan_outside_the_window():
    """Keys of NaN before the window and past the kept first keys, in the window of some rows and not of others."""
    dr = make_draft([200], [24], 8, 2, seed=61, tree=False)
    bt = dr.bt
    pages = bt.indices[bt.indptr[0]:bt.indptr[1]]
    for pos in range(5, 157):   # the first row's window of 50 starts at 151, the seventh's at 157
        bt.k[pages[pos // 16], pos % 16], bt.v[pages[pos // 16], pos % 16] = np.nan, np.nan
    print("tree nan outside the window", flush=True)
    out, lse = DeviceDraft(dr).run(window=50, sink=5)
    rows = np.arange(24) >= 6
    with np.errstate(invalid="ignore"):
        check_attention(out, lse, oracle_attention(dr, window=50, sink=5), "nan outside", rows=rows)
    assert np.isnan(lse[~rows]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tree", [True, False])
def test_rows_behind_the_last_sequence_stay(tree):
    import torch
    dr = make_draft([30, 80], [4, 9], 8, 2, seed=67, tree=tree, extra_rows=6)
    dr.q[13:] = np.nan
    dd = DeviceDraft(dr)
    dd.out.fill_(7.0)
    dd.lse.fill_(-3.0)
    out, lse = dd.run()
    assert np.all(out[13:] == 7.0) and np.all(lse[13:] == -3.0)
    check_attention(out, lse, oracle_attention(dr), "behind", rows=slice(0, 13))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_many_sequences():
    """More sequences than one pass of a workgroup's scan holds, most of them tiny."""
    rng = np.random.default_rng(5)
    ctx, new = rng.integers(0, 40, 1500), rng.integers(0, 4, 1500)
    ctx[700], new[700] = 900, 60
    dr = make_draft(ctx.tolist(), new.tolist(), 4, 2, seed=71)
    _run(dr, "1500 sequences")


@pytest.mark.gpu
@pytest.mark.parametrize("score", [dict(), dict(soft_cap=20.0, slopes=True), dict(window=900, sink=4)])
def test_long_context(score):
    """Contexts cut over many workgroups, beside short ones."""
    score = dict(score, slopes=SLOPES(8)) if score.get("slopes") else score
    dr = make_draft([9000, 60, 3500], [10, 21, 2], 8, 2, seed=73)
    _run(dr, f"long {sorted(score)}", **score)


@pytest.mark.gpu
def test_same_bits_every_time():
    import torch
    dr = make_draft([2500, 60, 900], [24, 5, 40], 16, 4, seed=79)
    dd = DeviceDraft(dr)
    first = [x.copy() for x in dd.run(soft_cap=30.0)]
    for _ in range(5):
        again = dd.run(soft_cap=30.0)
        assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(first, again))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_max_tokens_is_a_hint():
    """Another max_tokens than the batch's may choose another kernel, not another result."""
    dr = make_draft([300, 20, 77], [5, 30, 1], 8, 2, seed=83)
    ref = oracle_attention(dr)
    for most in (1, 2, 5, 30, 200, 512):
        print(f"tree max_tokens {most}", flush=True)
        out, lse = DeviceDraft(dr).run(max_tokens=most)
        check_attention(out, lse, ref, f"max_tokens {most}")


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1, 2 ** 28, 2 ** 29 + 1, 2 ** 31 - 1])
def test_any_max_tokens_of_a_chain(most):
    _run(make_draft([300, 20, 77], [5, 30, 1], 8, 2, seed=85, tree=False), f"max_tokens {most}", max_tokens=most)


@pytest.mark.gpu
def test_on_another_stream_and_in_a_graph():
    """A captured call replayed with other lengths, trees and pages in the same buffers, eager calls between."""
    import torch
    from _gpu import device
    shapes = [([300, 40], [8, 20]), ([120, 7], [16, 12]), ([33, 250], [20, 8])]
    drafts = [make_draft(c, n, 8, 2, seed=89 + i) for i, (c, n) in enumerate(shapes)]
    refs = [oracle_attention(d) for d in drafts]
    pages = max(d.bt.num_pages for d in drafts)
    dev = device()
    k = torch.zeros(pages, 16, 2, 128, dtype=torch.float16, device=dev)
    v, q = torch.zeros_like(k), torch.zeros(28, 8, 128, dtype=torch.float16, device=dev)
    indptr, q_indptr = (torch.zeros(3, dtype=torch.int32, device=dev) for _ in range(2))
    last, indices = torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros(pages, dtype=torch.int32, device=dev)
    mask, depth = torch.zeros(28, 1, dtype=torch.int32, device=dev), torch.zeros(28, dtype=torch.int32, device=dev)
    out, lse = torch.zeros(28, 8, 128, dtype=torch.float16, device=dev), torch.zeros(28, 8, device=dev)
    p = pdattn.make_tree_params(q, k, v, indptr, indices, last, 2, 8, 2, q_indptr=q_indptr, max_tokens=20, mask=mask, depth=depth)
    ws_mem = torch.empty(pdattn.tree_workspace_size(p), dtype=torch.uint8, device=dev)
    ws = pdattn.Workspace(ws_mem.data_ptr(), ws_mem.numel(), 0)

    def put(d):
        for buf, x in ((k, d.bt.k), (v, d.bt.v), (q, d.q), (indptr, d.bt.indptr), (q_indptr, d.q_indptr), (last, d.bt.last),
                       (indices, d.bt.indices), (mask, d.mask), (depth, d.depth)):
            x = torch.from_numpy(np.ascontiguousarray(x)).to(dev).to(buf.dtype)
            buf[:x.shape[0]].copy_(x)

    put(drafts[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pdattn.tree_attention(p, out, lse, ws, side)
    side.synchronize()
    check_attention(out.float().cpu(), lse.cpu(), refs[0], "side stream")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pdattn.tree_attention(p, out, lse, ws, side)
    for turn in range(6):
        i = turn % 3
        put(drafts[i])
        out.fill_(float("nan"))
        lse.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.float().cpu().numpy(), lse.cpu().numpy()
        check_attention(*got, refs[i], f"replay {turn}")
        pdattn.tree_attention(p, out, lse, ws, torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert np.array_equal(got[0], out.float().cpu().numpy()) and np.array_equal(got[1], lse.cpu().numpy())


@pytest.mark.gpu
def test_workspace_of_the_caller():
    """One byte too few is refused before anything runs; the size asked for is enough, filled with anything."""
    import torch
    dr = make_draft([700, 50], [6, 30], 8, 2, seed=97)
    dd = DeviceDraft(dr)
    p = dd.params()
    need = pdattn.tree_workspace_size(p)
    mem = torch.full((need + 4096,), 0xFF, dtype=torch.uint8, device=dd.q.device)
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.tree_attention(p, dd.out, dd.lse, pdattn.Workspace(mem.data_ptr(), need - 1, 0))
    assert e.value.status == 4
    pdattn.tree_attention(p, dd.out, dd.lse, pdattn.Workspace(mem.data_ptr(), need, 0))
    torch.cuda.synchronize()
    assert bool((mem[need:] == 0xFF).all())
    check_attention(dd.out.float().cpu(), dd.lse.cpu(), oracle_attention(dr), "caller's workspace")


@pytest.mark.gpu
def test_a_plan_in_the_same_workspace_is_refused_afterwards():
    """The partial states are written where the plan's schedule lay: the library knows."""
    import torch
    from _gpu import DeviceBatch
    from pdattn import inputs
    dr = make_draft([700, 50], [6, 30], 8, 2, seed=101)
    dd = DeviceDraft(dr)
    p = dd.params()
    bt = inputs.make_batch([1000, 64], 8, 2, seed=3)
    db, plan = DeviceBatch(bt), pdattn.Plan(bt.indptr, bt.last, 2, 8, 2)
    mem = torch.empty(max(plan.workspace_bytes, pdattn.tree_workspace_size(p)), dtype=torch.uint8, device=dd.q.device)
    plan.upload(mem, mem.numel())
    pdattn.tree_attention(p, dd.out, dd.lse, pdattn.Workspace(mem.data_ptr(), mem.numel(), 0))
    with pytest.raises(pdattn.PdattnError) as e:
        plan.run(db.q, db.k, db.v, db.indptr, db.indices, db.last, db.out, db.lse, mem, mem.numel())
    assert e.value.status == 6
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_far_pages():
    """Page ids past 32 bits of cache bytes."""
    import torch
    dr = make_draft([260, 33], [20, 7], 8, 2, seed=103)
    dd = DeviceDraft(dr)
    far = torch.zeros(600_000, 16, 2, 128, dtype=torch.float16, device=dd.q.device)   # 4.9 GB
    farv = torch.zeros_like(far)
    ids = torch.randperm(dr.bt.num_pages, device=dd.q.device) + 599_000
    ids[0] = 599_999
    order = torch.from_numpy(dr.bt.indices.astype(np.int64)).to(dd.q.device)
    far[ids], farv[ids] = dd.db.k[order], dd.db.v[order]
    dd.db.k, dd.db.v, dd.db.indices = far, farv, ids.int()
    print("tree far pages", flush=True)
    out, lse = dd.run()
    check_attention(out, lse, oracle_attention(dr), "far pages")

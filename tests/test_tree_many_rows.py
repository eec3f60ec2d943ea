"""Attention of drafted tokens: batches of many rows per sequence, many sequences, long pieces, and calls side by side."""
import numpy as np
import pdattn
import pytest
import torch
from _draft import DeviceDraft, check_attention, make_draft, oracle_attention


def _check(dr, tag, **kw):
    print(f"tree {tag}", flush=True)
    dd = DeviceDraft(dr)
    out, lse = dd.run(**kw)
    check_attention(out, lse, oracle_attention(dr), tag)
    return dd


# more than 128 rows of a kv head on average; contexts that end at, before and behind pages and 64-key blocks
@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new", [([0], [40]), ([0, 1], [64, 60]), ([63, 64, 65], [64, 63, 65]), ([15, 16, 17], [100, 33, 34]),
                                     ([500, 3], [90, 1]), ([1000], [257]), ([2049, 130], [65, 128]), ([127, 70], [128, 129])])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (16, 2), (2, 2)])
@pytest.mark.parametrize("tree", [True, False])
def test_many_rows(ctx, new, Hq, Hkv, tree):
    if Hq == Hkv:
        new = [3 * n for n in new]
        if tree and max(new) > 512:
            new = [min(n, 512) for n in new]
    _check(make_draft(ctx, new, Hq, Hkv, seed=sum(ctx) + sum(new), tree=tree), f"many rows {ctx} + {new} {Hq}/{Hkv} tree={tree}")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["nan", "inf"])
@pytest.mark.parametrize("where", ["k", "v"])
def test_many_rows_with_a_drafted_token_of_nan(kind, where):
    """A drafted key or value that is not finite reaches the rows whose mask has it, and no other."""
    dr = make_draft([200, 33], [70, 64], 8, 2, seed=29)
    bt = dr.bt
    for b, j in ((0, 41), (1, 5)):
        at = bt.lens[b] - int(dr.q_indptr[b + 1] - dr.q_indptr[b]) + j
        page = bt.indices[bt.indptr[b] + at // 16]
        x = bt.k if where == "k" else bt.v
        x[page, at % 16] = np.nan if kind == "nan" else np.inf
    out, lse = DeviceDraft(dr).run()
    ref = oracle_attention(dr)
    words = dr.mask.view(np.uint32)
    hit = np.zeros(dr.n_tokens, bool)
    for b, j in ((0, 41), (1, 5)):
        rows = slice(int(dr.q_indptr[b]), int(dr.q_indptr[b + 1]))
        hit[rows] = words[rows, j // 32] >> (j % 32) & 1
    assert 0 < hit.sum() < dr.n_tokens / 2
    check_attention(out, lse, ref, f"{kind} in {where}", rows=~hit)
    assert not np.isfinite(out[hit]).all(axis=(1, 2)).any()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [64, 70])
def test_values_behind_the_last_key_may_be_anything(new):
    """Elements of the last page behind the sequence's end are not read into any result."""
    dr = make_draft([101, 55], [new, new + 1], 8, 2, seed=31)
    bt = dr.bt
    ref = oracle_attention(dr)
    for b in range(2):
        page = bt.indices[bt.indptr[b + 1] - 1]
        assert bt.last[b] < 16
        bt.k[page, bt.last[b]:] = np.nan
        bt.v[page, bt.last[b]:] = np.inf
    out, lse = DeviceDraft(dr).run()
    check_attention(out, lse, ref, "behind the end")


@pytest.mark.gpu
@pytest.mark.parametrize("B", [63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("new,Hq", [(1, 2), (2, 8), (9, 16), (20, 16)])
def test_sequence_counts(B, new, Hq):
    """The search of a range's first sequence, at the edges of what a wave or a workgroup looks at in one go."""
    rng = np.random.default_rng(B + new)
    ctx = rng.integers(0, 60, B).tolist()
    n = rng.integers(0, 2 * new, B)
    n[-1] = new
    _check(make_draft(ctx, n.tolist(), Hq, 2, seed=B, tree=bool(B & 1)), f"{B} sequences of {new}, {Hq} heads")


@pytest.mark.gpu
def test_long_pieces():
    """Enough heads that one workgroup has more than 64 blocks of a sequence (three heads are checked)."""
    from _gpu import device
    dev = device()
    ctx, n, H = 17500, 130, 64
    pages = (ctx + n + 15) // 16
    g = torch.Generator(device=dev).manual_seed(37)
    k = torch.randn(pages, 16, H, 128, generator=g, device=dev, dtype=torch.float16)
    v = torch.randn(pages, 16, H, 128, generator=g, device=dev, dtype=torch.float16)
    q = torch.randn(n, H, 128, generator=g, device=dev, dtype=torch.float16)
    order = torch.randperm(pages, generator=g, device=dev).int()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    p = pdattn.make_tree_params(q, k, v, i32(0, pages), order, i32((ctx + n - 1) % 16 + 1), 1, H, H, q_indptr=i32(0, n), max_tokens=n)
    out = torch.full((n, H, 128), float("nan"), dtype=torch.float16, device=dev)
    lse = torch.full((n, H), float("nan"), device=dev)
    ws = pdattn.Workspace()
    pdattn.tree_attention(p, out, lse, ws)
    torch.cuda.synchronize()
    pdattn.workspace_release(ws)
    heads = [0, 37, 63]
    import oracle
    ref = oracle.tree_attention(q[:, heads].cpu().numpy(), k[:, :, heads].cpu().numpy(), v[:, :, heads].cpu().numpy(),
                                np.array([0, pages], np.int32), order.cpu().numpy(), np.array([(ctx + n - 1) % 16 + 1], np.int32),
                                3, 3, np.array([0, n], np.int32), None, None)
    check_attention(out[:, heads].float().cpu().numpy(), lse[:, heads].cpu().numpy(), ref, "long pieces")


@pytest.mark.gpu
def test_two_graphs_share_a_workspace():
    """Captured one after the other into the same workspace and replayed in turns, with eager calls between."""
    drafts = [make_draft([300, 20], [70, 60], 8, 2, seed=41), make_draft([64, 700, 3], [5, 9, 2], 8, 2, seed=43)]
    refs = [oracle_attention(d) for d in drafts]
    dds = [DeviceDraft(d) for d in drafts]
    ps = [dd.params() for dd in dds]
    ws = pdattn.Workspace()
    pdattn.workspace_reserve(ws, max(pdattn.tree_workspace_size(p) for p in ps))
    side, graphs = torch.cuda.Stream(), []
    side.wait_stream(torch.cuda.current_stream())
    for p, dd in zip(ps, dds):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pdattn.tree_attention(p, dd.out, dd.lse, ws, side)
        graphs.append(graph)
    for turn in (0, 1, 1, 0, 1, 0):
        dd = dds[turn]
        dd.out.fill_(float("nan"))
        dd.lse.fill_(float("nan"))
        torch.cuda.synchronize()
        graphs[turn].replay()
        torch.cuda.synchronize()
        check_attention(dd.out.float().cpu().numpy(), dd.lse.cpu().numpy(), refs[turn], f"graph {turn}")
        other = dds[1 - turn]
        pdattn.tree_attention(ps[1 - turn], other.out, other.lse, ws)
        torch.cuda.synchronize()
        check_attention(other.out.float().cpu().numpy(), other.lse.cpu().numpy(), refs[1 - turn], "eager")
    del graphs
    pdattn.workspace_release(ws)


@pytest.mark.gpu
def test_two_streams_with_their_own_workspaces():
    drafts = [make_draft([900, 20], [40, 60], 8, 2, seed=47), make_draft([64, 1500], [5, 9], 8, 2, seed=53)]
    refs = [oracle_attention(d) for d in drafts]
    dds = [DeviceDraft(d) for d in drafts]
    ps = [dd.params() for dd in dds]
    wss = [pdattn.Workspace() for _ in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(8):
        for p, dd, ws, s in zip(ps, dds, wss, streams):
            pdattn.tree_attention(p, dd.out, dd.lse, ws, s)
    torch.cuda.synchronize()
    for dd, ref, ws in zip(dds, refs, wss):
        check_attention(dd.out.float().cpu().numpy(), dd.lse.cpu().numpy(), ref, "two streams")
        pdattn.workspace_release(ws)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,new", [(8, 2, 64), (8, 2, 20), (16, 2, 33), (4, 4, 5), (1200, 300, 50)])
def test_the_scores_do_not_change_the_workspace(Hq, Hkv, new):
    """A workspace sized for plain scores serves changed ones, masks and chains, and a graph of either."""
    base = dict(B=2, Hq=Hq, Hkv=Hkv, n_tokens=2 * new, q_indptr=1 << 20, max_tokens=new)
    ptrs = [1 << 20] * 6
    sizes = {pdattn.tree_workspace_size(pdattn.make_tree_params(*ptrs, **base, **kw))
             for kw in (dict(), dict(soft_cap=5.0), dict(window=50), dict(slopes=1 << 20), dict(mask=1 << 20, mask_words=2))}
    assert len(sizes) == 1 and min(sizes) > 0
    if Hkv > 4:
        return
    dr = make_draft([100, 400], [new, new], Hq, Hkv, seed=61)
    mem = torch.empty(min(sizes), dtype=torch.uint8, device="cuda")
    ws, dd = pdattn.Workspace(mem.data_ptr(), mem.numel(), 0), DeviceDraft(dr)
    for kw in (dict(), dict(soft_cap=5.0, window=70)):
        pdattn.tree_attention(dd.params(**kw), dd.out, dd.lse, ws)
        torch.cuda.synchronize()
        check_attention(dd.out.float().cpu().numpy(), dd.lse.cpu().numpy(), oracle_attention(dr, **kw), f"scores {kw}")

"""The operators of a speculative decoding step in a run, as a serving loop uses them: the drafted tokens' rotary
positions and append, their attention, the accepted path's rows to the front, and the next step on the shortened
sequences -- against the restatements in 64 bits on host copies of the same caches."""
import numpy as np
import pytest

import oracle
import pdattn
from _draft import check_attention, random_tree, tree_rows
from pdattn import inputs

pytestmark = pytest.mark.gpu


def _table(lens, spare, rng):
    """A page table for sequences that will grow to lens + spare tokens: pages are given out once."""
    pages = [-(-(n + spare) // 16) for n in lens]
    ids = rng.permutation(sum(pages)).astype(np.int32)
    return np.split(ids, np.cumsum(pages)[:-1])


def _csr(own, lens):
    need = [-(-n // 16) for n in lens]
    indptr = np.concatenate([[0], np.cumsum(need)]).astype(np.int32)
    indices = np.concatenate([p[:n] for p, n in zip(own, need)]).astype(np.int32)
    last = np.array([n - (p - 1) * 16 if p else 0 for n, p in zip(lens, need)], np.int32)
    return indptr, indices, last


@pytest.mark.parametrize("Hq,Hkv,score,rotary", [(8, 2, dict(), 128), (16, 2, dict(soft_cap=20.0, window=120, sink=4), 64),
                                                 (4, 4, dict(slopes=True), 32)])
def test_three_steps(Hq, Hkv, score, rotary):
    import torch
    from _gpu import device
    dev, rng = device(), np.random.default_rng(Hq)
    lens, n_draft = [150, 33, 1, 400], [12, 5, 20, 1]
    own = _table(lens, 100, rng)
    pages = sum(len(p) for p in own)
    kc, vc = (rng.standard_normal((pages, 16, Hkv, 128)).astype(np.float16) for _ in range(2))
    k, v = torch.from_numpy(kc.copy()).to(dev), torch.from_numpy(vc.copy()).to(dev)
    put = lambda x, t=np.int32: torch.from_numpy(np.ascontiguousarray(x, dtype=t)).to(dev)  # noqa: E731
    freq, scale = pdattn.rope_frequencies(rotary, 10000.0, pdattn.ROPE_LINEAR, 2.0)
    f, ws = put(freq, np.float64), pdattn.Workspace()
    if score.get("slopes"):
        score = dict(score, slopes=[2.0 ** (-2 * (h + 1)) for h in range(Hq)])
    on_gpu = dict(score, slopes=put(score["slopes"], np.float32)) if "slopes" in score else score
    for step in range(3):
        # draft: a tree per sequence, appended behind the cached tokens
        parent = [random_tree(n, rng) for n in n_draft]
        rows = [tree_rows(p, 1) for p in parent]
        mask, depth = (np.concatenate([r[i] for r in rows]).astype(np.int32) for i in (0, 1))
        q_indptr = np.concatenate([[0], np.cumsum(n_draft)]).astype(np.int32)
        seqs = np.repeat(np.arange(4), n_draft)
        index = np.arange(len(seqs)) - q_indptr[seqs]
        ctx = np.array(lens)[seqs]
        full = [a + n for a, n in zip(lens, n_draft)]
        indptr, indices, last = _csr(own, full)
        qkv = rng.standard_normal((len(seqs), Hq + 2 * Hkv, 128)).astype(np.float16)
        d_qkv = torch.from_numpy(qkv).to(dev)
        q = torch.empty(len(seqs), Hq, 128, dtype=torch.float16, device=dev)
        d = [put(x) for x in (indptr, indices, last, q_indptr, seqs, ctx + index, ctx + depth)]
        p = pdattn.make_rope_append_params(d_qkv[:, :Hq], d_qkv[:, Hq:Hq + Hkv], d_qkv[:, Hq + Hkv:], q, k, v, d[0], d[1], d[4],
                                           d[5], f, 4, rotary_dim=rotary, scale=scale, rope_positions=d[6])
        # attention of the drafted tokens
        out = torch.empty_like(q)
        lse = torch.empty(len(seqs), Hq, device=dev)
        tp = pdattn.make_tree_params(q, k, v, d[0], d[1], d[2], 4, Hq, Hkv, q_indptr=d[3], max_tokens=max(n_draft),
                                     mask=put(mask.reshape(-1, 1)), depth=put(depth), **on_gpu)
        # the accepted path: from a node to its root
        paths = []
        for n, par in zip(n_draft, parent):
            line, i = [], int(rng.integers(0, n))
            while i >= 0:
                line.append(i)
                i = par[i]
            paths.append(line[::-1])
        aip = np.concatenate([[0], np.cumsum([len(x) for x in paths])]).astype(np.int32)
        d_aip, d_acc = put(aip), put(np.concatenate(paths))
        print(f"step {step}", flush=True)
        pdattn.rope_append_kv(p)
        pdattn.tree_attention(tp, out, lse, ws)
        pdattn.accept_kv(k, v, d[0], d[1], d[2], d[3], d_aip, d_acc, 4, Hkv)
        torch.cuda.synchronize()
        # the host's copies: q and the new k as the library rounded them (their own tests hold the rotation)
        exact = oracle.rope(qkv[:, :Hq + Hkv], ctx + depth, freq, rotary, False, scale)
        qh = q.cpu().numpy()
        assert np.abs(qh - exact[:, :Hq]).max() < 2 ** -8
        kn = exact[:, Hq:].astype(np.float16)
        kc, vc, bad = oracle.append_kv(kc, vc, kn, qkv[:, Hq + Hkv:], seqs, ctx + index, indptr, indices)
        assert bad == 0
        ref = oracle.tree_attention(qh, kc, vc, indptr, indices, last, Hq, Hkv, q_indptr, mask.reshape(-1, 1), depth, **score)
        kc, vc, bad = oracle.accept_kv(kc, vc, indptr, indices, last, q_indptr, aip, np.concatenate(paths))
        got = k.cpu().numpy()
        # (a rotated key may round the other way once in a while: half a step of fp16 and a little)
        assert bad == 0 and np.array_equal(v.cpu().numpy().view(np.uint16), vc.view(np.uint16))
        assert np.mean(got != kc) < 1e-3 and np.abs(got.astype(np.float64) - kc).max() < 2 ** -8
        check_attention(out.float().cpu(), lse.cpu(), ref, f"step {step}")
        kc = got.copy()   # go on from the same keys
        lens = [a + len(x) for a, x in zip(lens, paths)]
    pdattn.workspace_release(ws)
    # an ordinary decode over what the steps left
    bt = inputs.Batch(lens, Hq, Hkv, *_csr(own, lens), pages, 0)
    q1 = rng.standard_normal((4, Hq, 128)).astype(np.float16)
    tables = [put(x) for x in (bt.indptr, bt.indices, bt.last)]
    dq, out, lse = torch.from_numpy(q1).to(dev), torch.empty(4, Hq, 128, dtype=torch.float16, device=dev), torch.empty(4, Hq, device=dev)
    nc, ct = pdattn.plan_chunks(Hq // Hkv, 4, Hkv, max(lens))
    ws = pdattn.Workspace()
    pdattn.decode_attention_balanced(pdattn.make_params(dq, k, v, *tables, 4, Hq, Hkv, nc, ct), Hq // Hkv, out, lse, ws)
    torch.cuda.synchronize()
    pdattn.workspace_release(ws)
    ref = oracle.tree_attention(q1, kc, vc, bt.indptr, bt.indices, bt.last, Hq, Hkv)
    check_attention(out.float().cpu(), lse.cpu(), ref, "decode after the steps")
